// Attention of a few rows per sequence over a paged bf16 cache (head size 64 or 128): the step of one new
// token, and drafts to verify, up to 64 (row, query head) pairs per key head.
//
//   out = sum_j softmax_j(scale * q . k[j]) v[j] over the positions j that the row sees
//
// Every key and value is read once from HBM and used for all pairs of its head: 2 to 64 multiply-adds per
// element, so the bound is HBM and the tensor work only has to keep up with it. The pairs are far fewer than the
// 128 rows of a tcgen05 tile, so the products are warp-level mma.m16n8k16 with the pairs as the 16 rows and the
// accumulators in registers.
//
// The work is one list: the 64-position tiles of (sequence 0, key head 0), then those of head 1, and so on. Every
// CTA takes an equal, consecutive share of it, as many CTAs as the SMs hold at once, whatever the lengths are:
// no SM waits for a long sequence, and a CTA's ring of TMA copies (out of the pages, 128-byte swizzle, no
// multicast) runs on from one (sequence, head) to the next. Four warps per 16 pairs take 16 positions of a
// tile each, with a running maximum and sum of their own, and are joined through shared memory. A (sequence,
// head) that shares end in is left as partials in the workspace, one per share, and join_kernel joins
// them in order: equal calls give equal bits, and no atomics or waits between CTAs are needed.
// Every mbarrier wait is bounded: one that gives up ends its sequences with SSB_ROW_DEVICE_TIMEOUT.
#include <algorithm>

#include "ssb_decoder.cuh"
#include "ssb_tma.cuh"
#include "ssb_tma_map.cuh"

namespace ssb {

namespace {

constexpr int kGroups = 4;  // warps that share a tile, 16 positions each
constexpr int kMaxStages = 8;
// A CTA's share is at least this many tiles: below it the join costs more than the tiles' latency.
constexpr int kMinTiles = 2;

template <int D> constexpr int stage_bytes() { return 2 * kTile * D * 2; }
template <int MT> constexpr int step_threads() { return (kGroups * MT + 1) * 32; }

__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 2^x with a relative error of 2^-22; -inf gives 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool bf16_pair_not_finite(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// What the shares of a call are: `total` tiles in `shares` equal parts.
struct Plan {
    int64_t total;
    int shares;
    __device__ __forceinline__ int64_t begin(int i) const { return i < shares ? total * i / shares : total; }
};

__device__ __forceinline__ Span span_of(const AttendArgs & g, const Sequence & q) {
    return span_of(q.length - q.n, q.length - 1, g.window, g.sinks);
}
__device__ __forceinline__ int tiles_of(const AttendArgs & g, const Sequence & q) {
    return q.ok && q.n > 0 ? span_of(g, q).tiles : 0;
}

// The place in the list where a share begins, and the walk over it, unit by unit ((sequence, key head) pairs).
struct Walk {
    int seq, head, tiles;  // the unit, and its tiles
    int64_t unit_at;       // its first tile's place in the list
    Sequence q;
    __device__ __forceinline__ void next(const AttendArgs & g) {
        unit_at += tiles;
        if (++head < g.kv.kv_heads) return;
        head = 0;
        do {
            q = sequence(g.kv, ++seq);
            tiles = tiles_of(g, q);
        } while (tiles == 0 && seq + 1 < g.kv.seqs);
    }
};

// The partials of a share in the workspace: slot 0 of a unit that began in an earlier share, slot 1 of one
// that begins in this share and ends in a later one.
struct PartHead {
    int unit;  // or -1
    int ends;  // the unit ends in this share
    int bad;   // bits that refuse the sequence
    int unused;
};
__device__ __forceinline__ PartHead * part_head(const AttendArgs & g, int share, int slot) {
    return static_cast<PartHead *>(g.workspace) + share * 2 + slot;
}
// After the heads of all shares: per slot, (maximum, sum) of each pair and then their outputs.
__device__ __forceinline__ float * part_data(const AttendArgs & g, int share, int slot, int pairs) {
    return reinterpret_cast<float *>(static_cast<PartHead *>(g.workspace) + (size_t) g.max_shares * 2) +
           (size_t) (share * 2 + slot) * pairs * (g.kv.head_dim + 2);
}

__device__ __forceinline__ void store_pair(const AttendArgs & g, int64_t row, int head, int at, float x, float y) {
    __nv_bfloat16 * dst = static_cast<__nv_bfloat16 *>(g.out) + row * g.out_ld + (int64_t) head * g.kv.head_dim + at;
    if (g.vec_out) *reinterpret_cast<uint32_t *>(dst) = pack_bf16(x, y);
    else dst[0] = narrow<__nv_bfloat16>(x), dst[1] = narrow<__nv_bfloat16>(y);
}

// What a refused sequence's rows hold: 0, or NaN where the device did not answer.
__device__ __forceinline__ float refused_value(int bad) { return bad & 2 ? __int_as_float(0x7fc00000) : 0.0f; }

__device__ __forceinline__ void report(const AttendArgs & g, int seq, int head, int bad) {
    if (!g.kv.status) return;
    if (bad & 2) g.kv.status[seq] = SSB_ROW_DEVICE_TIMEOUT;
    else if (head == 0) g.kv.status[seq] = bad ? SSB_ROW_INVALID_ROW : SSB_ROW_OK;
}

template <int D, int MT>
__global__ void __launch_bounds__(step_threads<MT>(), MT == 1 ? 2 : 1)
    step_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ AttendArgs g, int stages, int pairs) {
    constexpr int kPitch = D + 8, kThreads = step_threads<MT>(), kConsumers = kThreads - 32;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char * smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    float * room = reinterpret_cast<float *>(smem + (size_t) stages * stage_bytes<D>());  // [pairs][kPitch]
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
    __shared__ float2 stat[16 * MT];
    __shared__ int64_t s_scan[kThreads / 32];
    __shared__ int64_t s_at;
    __shared__ int s_seq, s_idle, s_dead;
    __shared__ int s_refused[kMaxStages];  // per tile: its unit has a page outside the pool
    const KvArgs & kv = g.kv;
    const int tid = (int) threadIdx.x, warp = warp_id(), lane = lane_id(), me = (int) blockIdx.x;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // join_kernel may be set up meanwhile
    // ---- every CTA adds up the tiles of all sequences and finds where its share begins
    const int chunk = (kv.seqs + kThreads - 1) / kThreads;
    const int c0 = min(tid * chunk, kv.seqs), c1 = min(c0 + chunk, kv.seqs);
    int64_t mine = 0;
    bool idle = false;
    if (tid == 0) {
        for (int s = 0; s < stages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], kGroups * MT);
        s_idle = s_dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    for (int s = c0; s < c1; s++) {
        const int n = tiles_of(g, sequence(kv, s));
        mine += n;
        idle |= n == 0 && s % (int) gridDim.x == me;
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) s_scan[warp] = upto;
    __syncthreads();
    if (idle) s_idle = 1;
    Plan plan;
    plan.total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; w++) {
        if (w < warp) upto += s_scan[w];
        plan.total += s_scan[w];
    }
    plan.total *= kv.kv_heads;
    plan.shares = (int) min((int64_t) gridDim.x, (plan.total + kMinTiles - 1) / kMinTiles);
    const int64_t begin = plan.begin(me), end = plan.begin(me + 1);
    int64_t at = (upto - mine) * kv.kv_heads;
    if (begin < end && at <= begin && begin < upto * kv.kv_heads) {
        for (int s = c0; s < c1; s++) {
            const int64_t past = at + (int64_t) tiles_of(g, sequence(kv, s)) * kv.kv_heads;
            if (begin < past) {
                s_seq = s;
                s_at = at;
                break;
            }
            at = past;
        }
    }
    __syncthreads();
    Walk walk{};
    if (begin < end) {
        walk.seq = s_seq;
        walk.q = sequence(kv, walk.seq);
        walk.tiles = tiles_of(g, walk.q);
        walk.head = (int) ((begin - s_at) / walk.tiles);
        walk.unit_at = s_at + (int64_t) walk.head * walk.tiles;
    }
    auto dead = [&]() { return *reinterpret_cast<volatile int *>(&s_dead) != 0; };
    const int box = kv.page_size < kTile ? kv.page_size : kTile;  // positions of one TMA copy: a piece of a tile
    if (warp == kGroups * MT) {
        // ---- producer: lane l looks up and copies piece l of every 32
        const int per_tile = kTile / box, batch = 32 / per_tile;
        int last_use[kMaxStages];
#pragma unroll
        for (int s = 0; s < kMaxStages; s++) last_use[s] = -1;
        int it = 0;
        for (int64_t now = begin; now < end && !__any_sync(0xffffffffu, dead()); walk.next(g)) {
            const Span span = span_of(g, walk.q);
            const int32_t * table = kv.table + (int64_t) walk.seq * kv.table_ld;
            const int t0 = (int) (now - walk.unit_at), t1 = (int) min((int64_t) walk.tiles, end - walk.unit_at);
            bool ok = true;
            for (int t = t0; t < t1 && ok; t += batch) {
                const int my_tile = t + lane / per_tile;
                const int from = span.base(my_tile) + lane % per_tile * box;
                // only pieces that hold a seen position: the table's other entries may be anything
                const bool wanted = my_tile < t1 && from < span.hi && (from + box > span.first || from < span.sinks);
                const int page = wanted ? table[from >> kv.page_shift] : 0;
                const bool valid = wanted && (unsigned) page < (unsigned) kv.pages;
                const bool refuse = __any_sync(0xffffffffu, wanted && !valid);
                const uint32_t votes = __ballot_sync(0xffffffffu, valid);
                const int stop = min(t1, t + batch);
                for (int u = t; u < stop; u++, it++) {
                    const int s = it % stages;
                    const bool ready = it < stages || mbar_wait(&empty[s], (uint32_t) (it / stages - 1) & 1u);
                    if (!__all_sync(0xffffffffu, ready)) {
                        ok = false;
                        break;
                    }
                    const uint32_t of_tile = (per_tile == 1 ? 1u : (1u << per_tile) - 1u) << ((u - t) * per_tile);
                    if (lane == 0) {
                        s_refused[s] = refuse;  // read by the consumers once the barrier's phase has ended
                        mbar_expect(&full[s], (uint32_t) (__popc(votes & of_tile) * 2 * box * D * 2));
                    }
                    __syncwarp();
                    if (valid && my_tile == u) {
                        unsigned char * dst = smem + (size_t) s * stage_bytes<D>() + lane % per_tile * box * D * 2;
                        const int slot = from & (kv.page_size - 1);
                        tma_load_5d(dst, &map_k, 0, slot, 0, walk.head, page, &full[s]);
                        tma_load_5d(dst + kTile * D * 2, &map_v, 0, slot, 0, walk.head, page, &full[s]);
                    }
#pragma unroll
                    for (int i = 0; i < kMaxStages; i++)
                        if (i == s) last_use[i] = it / stages;
                }
            }
            if (!ok) {
                if (lane == 0) atomicOr(&s_dead, 1);
                break;
            }
            now = walk.unit_at + t1;
            if (now >= end) break;
        }
        __syncwarp();
        if (dead()) {  // let the copies in flight land before the shared memory is given up
#pragma unroll
            for (int s = 0; s < kMaxStages; s++)
                if (last_use[s] >= 0) mbar_wait(&full[s], (uint32_t) last_use[s] & 1u);
        }
    } else {
        // ---- consumers
        const int mt = warp % MT, kg = warp / MT;
        const int r0 = mt * 16 + lane / 4;  // this thread's pairs: r0 and r0 + 8
        // this warp's 16 positions within a tile: their rows in the tile's [piece][half][position] layout
        const int row = kg * 16;
        const uint32_t row_at = (uint32_t) (row / box * (box * D * 2) + row % box * 128);
        const uint32_t half_at = (uint32_t) box * 128;
        const int k_row = (lane & 7) + (lane >> 4) * 8, k_chunk = lane >> 3 & 1;
        const int v_row = (lane & 7) + (lane >> 3 & 1) * 8, v_chunk = lane >> 4;
        PartHead part[2] = {{-1, 0, 0, 0}, {-1, 0, 0, 0}};
        int it = 0;
        for (int64_t now = begin; now < end; walk.next(g)) {
            const Span span = span_of(g, walk.q);
            const int t0 = (int) (now - walk.unit_at), t1 = (int) min((int64_t) walk.tiles, end - walk.unit_at);
            const int rows = walk.q.n * g.group;  // (row, query head) pairs of this unit
            const int p_first = walk.q.length - walk.q.n, p_last = walk.q.length - 1;
            // the pairs of this warp's 16 rows as the A operand, for all of the head
            uint32_t qa[D / 16][4];
            int position[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int m = r0 + 8 * i;
                position[i] = p_first + (m < rows ? m : rows - 1) / g.group;
                const __nv_bfloat16 * src = static_cast<const __nv_bfloat16 *>(g.q) +
                                            (int64_t) (walk.q.start + m / g.group) * g.q_ld +
                                            (int64_t) (walk.head * g.group + m % g.group) * D + lane % 4 * 2;
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++) {
                    qa[ks][i] = m < rows ? *reinterpret_cast<const uint32_t *>(src + ks * 16) : 0u;
                    qa[ks][2 + i] = m < rows ? *reinterpret_cast<const uint32_t *>(src + ks * 16 + 8) : 0u;
                }
            }
            float o[D / 8][4];
            float top[2] = {-kInf, -kInf}, sum[2] = {0.0f, 0.0f};
            int bad = 0;
#pragma unroll
            for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            for (int t = t0; t < t1; t++, it++) {
                const int s = it % stages;
                const bool ok = !dead() && mbar_wait(&full[s], (uint32_t) (it / stages) & 1u);
                if (!__all_sync(0xffffffffu, ok)) {  // the rest of the share is refused, unit by unit
                    if (lane == 0) atomicOr(&s_dead, 1);
                    bad |= 2;
                    break;
                }
                bad |= *reinterpret_cast<volatile int *>(&s_refused[s]);
                const uint32_t keys = smem_addr(smem) + (uint32_t) s * stage_bytes<D>() + row_at, values = keys + kTile * D * 2;
                float c[2][4] = {};
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++) {
                    const int chunk = ks * 2 + k_chunk;
                    uint32_t b[4];
                    ldmatrix(b, keys + (uint32_t) (chunk / 8) * half_at + (uint32_t) (k_row * 128 + ((chunk % 8) ^ (k_row & 7)) * 16));
                    mma(c[0], qa[ks], b[0], b[1]);
                    mma(c[1], qa[ks], b[2], b[3]);
                }
                const int base = span.base(t) + row;  // the warp's first position
                const bool whole = base + 15 <= p_first && (g.window == 0 || base > p_last - g.window || base + 15 < g.sinks);
                float new_top[2] = {top[0], top[1]};
#pragma unroll
                for (int nt = 0; nt < 2; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = c[nt][e] * g.scale_log2;
                        if (!whole && !sees(position[e / 2], base + nt * 8 + lane % 4 * 2 + e % 2, g.window, g.sinks)) x = -kInf;
                        c[nt][e] = x;
                        new_top[e / 2] = fmaxf(new_top[e / 2], x);
                    }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    new_top[i] = fmaxf(new_top[i], shfl_xor(new_top[i], 1));
                    new_top[i] = fmaxf(new_top[i], shfl_xor(new_top[i], 2));
                }
                if (__any_sync(0xffffffffu, new_top[0] != top[0] || new_top[1] != top[1])) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float a = new_top[i] == top[i] ? 1.0f : ex2(top[i] - new_top[i]);
                        top[i] = new_top[i];
                        sum[i] *= a;
#pragma unroll
                        for (int j = 0; j < D / 8; j++) o[j][2 * i] *= a, o[j][2 * i + 1] *= a;
                    }
                }
                const float ref[2] = {top[0] == -kInf ? 0.0f : top[0], top[1] == -kInf ? 0.0f : top[1]};
#pragma unroll
                for (int nt = 0; nt < 2; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        c[nt][e] = ex2(c[nt][e] - ref[e / 2]);
                        sum[e / 2] += c[nt][e];
                    }
                // the weights rounded to bf16 for the product: half a step of the output's own type
                const uint32_t pa[4] = {pack_bf16(c[0][0], c[0][1]), pack_bf16(c[0][2], c[0][3]), pack_bf16(c[1][0], c[1][1]),
                                        pack_bf16(c[1][2], c[1][3])};
                bool apart = false;  // a value that some row must not see is not finite: 0 times it would reach the row
                if (!whole) {
                    bool found = false;
#pragma unroll
                    for (int i = 0; i < 16 * D / 8 / 32; i++) {
                        const int e = lane + 32 * i, r = e / (D / 8), chunk = e % (D / 8);
                        uint4 x;
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                                     : "r"(values + (uint32_t) (chunk / 8) * half_at + (uint32_t) (r * 128 + chunk % 8 * 16)));
                        found |= bf16_pair_not_finite(x.x) | bf16_pair_not_finite(x.y) | bf16_pair_not_finite(x.z) | bf16_pair_not_finite(x.w);
                    }
                    apart = __any_sync(0xffffffffu, found);
                }
                if (!apart) {
#pragma unroll
                    for (int n2 = 0; n2 < D / 16; n2++) {
                        const int chunk = n2 * 2 + v_chunk;
                        uint32_t b[4];
                        ldmatrix_trans(b, values + (uint32_t) (chunk / 8) * half_at + (uint32_t) (v_row * 128 + ((chunk % 8) ^ (v_row & 7)) * 16));
                        mma(o[2 * n2], pa, b[0], b[1]);
                        mma(o[2 * n2 + 1], pa, b[2], b[3]);
                    }
                } else {
                    for (int j = 0; j < 16; j++) {  // one position at a time, for the rows that see it
                        const int from = (lane & ~3) | (j % 8 / 2);
                        float w[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const uint32_t pair = __shfl_sync(0xffffffffu, j < 8 ? pa[i] : pa[2 + i], from);
                            w[i] = j % 2 ? bf16_hi(pair) : bf16_lo(pair);
                        }
                        const bool see0 = sees(position[0], base + j, g.window, g.sinks), see1 = sees(position[1], base + j, g.window, g.sinks);
#pragma unroll
                        for (int n = 0; n < D / 8; n++) {
                            uint32_t pair;
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pair)
                                         : "r"(values + (uint32_t) (n / 8) * half_at + (uint32_t) (j * 128 + ((n % 8) ^ (j & 7)) * 16 + lane % 4 * 4)));
                            if (see0) o[n][0] += w[0] * bf16_lo(pair), o[n][1] += w[0] * bf16_hi(pair);
                            if (see1) o[n][2] += w[1] * bf16_lo(pair), o[n][3] += w[1] * bf16_hi(pair);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                sum[i] += shfl_xor(sum[i], 1);
                sum[i] += shfl_xor(sum[i], 2);
            }
            // the four warps of 16 pairs joined into the first, one after the other
            for (int from = 1; from < kGroups; from++) {
                if (kg == from) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int m = r0 + 8 * i;
                        if (m >= rows) continue;
                        if (lane % 4 == 0) stat[m] = make_float2(top[i], sum[i]);
#pragma unroll
                        for (int n = 0; n < D / 8; n++)
                            *reinterpret_cast<float2 *>(room + m * kPitch + n * 8 + lane % 4 * 2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
                    }
                }
                bar_sync(1, kConsumers);
                if (kg == 0) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int m = r0 + 8 * i;
                        if (m >= rows) continue;
                        const float2 other = stat[m];
                        const float t = fmaxf(top[i], other.x), ref = t == -kInf ? 0.0f : t;
                        const float a = ex2(top[i] - ref), b = ex2(other.x - ref);
                        top[i] = t;
                        sum[i] = sum[i] * a + other.y * b;
#pragma unroll
                        for (int n = 0; n < D / 8; n++) {
                            const float2 x = *reinterpret_cast<const float2 *>(room + m * kPitch + n * 8 + lane % 4 * 2);
                            o[n][2 * i] = o[n][2 * i] * a + x.x * b, o[n][2 * i + 1] = o[n][2 * i + 1] * a + x.y * b;
                        }
                    }
                }
                bar_sync(1, kConsumers);
            }
            if (dead()) bad |= 2;
            if (kg == 0) {
                const bool begins = t0 == 0, ends = t1 == walk.tiles;
                if (begins && ends) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int m = r0 + 8 * i;
                        if (m >= rows) continue;
                        const int64_t out_row = walk.q.start + m / g.group;
                        const int h = walk.head * g.group + m % g.group;
                        const bool blank = bad || position[i] < 0;
                        const float inv = 1.0f / sum[i], fill = refused_value(bad);
#pragma unroll
                        for (int n = 0; n < D / 8; n++)
                            store_pair(g, out_row, h, n * 8 + lane % 4 * 2, blank ? fill : o[n][2 * i] * inv, blank ? fill : o[n][2 * i + 1] * inv);
                        if (g.lse && lane % 4 == 0)
                            g.lse[out_row * g.q_heads + h] = blank ? -kInf : (top[i] == -kInf ? 0.0f : top[i]) * kLn2 + logf(sum[i]);
                    }
                    if (tid == 0) report(g, walk.seq, walk.head, bad);
                } else {
                    const int slot = begins ? 1 : 0;
                    part[slot] = {walk.seq * kv.kv_heads + walk.head, ends, bad, 0};
                    float * data = part_data(g, me, slot, pairs);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int m = r0 + 8 * i;
                        if (m >= rows) continue;
                        if (lane % 4 == 0) *reinterpret_cast<float2 *>(data + 2 * m) = make_float2(top[i], sum[i]);
#pragma unroll
                        for (int n = 0; n < D / 8; n++)
                            *reinterpret_cast<float2 *>(data + 2 * pairs + m * D + n * 8 + lane % 4 * 2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
                    }
                }
            }
            now = walk.unit_at + t1;
            if (now >= end) break;
        }
        if (tid == 0) {
            *part_head(g, me, 0) = part[0];
            *part_head(g, me, 1) = part[1];
        }
    }
    __syncthreads();
    if (s_idle) {  // sequences with nothing to read: idle or refused rows, or none
        for (int s = me; s < kv.seqs; s += (int) gridDim.x) {
            const Sequence q = sequence(kv, s);
            if (tiles_of(g, q) > 0) continue;
            for (int64_t e = tid; e < (int64_t) q.n * g.q_heads * (D / 2); e += kThreads) {
                const int64_t pair = e / (D / 2);
                store_pair(g, q.start + pair / g.q_heads, (int) (pair % g.q_heads), (int) (e % (D / 2)) * 2, 0.0f, 0.0f);
            }
            if (g.lse)
                for (int64_t e = tid; e < (int64_t) q.n * g.q_heads; e += kThreads) g.lse[q.start * (int64_t) g.q_heads + e] = -kInf;
            if (tid == 0 && kv.status) kv.status[s] = q.ok ? SSB_ROW_OK : SSB_ROW_INVALID_ROW;
        }
    }
}

// Joins the partials of the unit that begins in share `blockIdx.x` and ends in a later one: those of the
// following shares' slot 0, up to the one that says it ends.
constexpr int kJoinThreads = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttendArgs g, int pairs) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the shares are written
    const int share = (int) blockIdx.x, tid = (int) threadIdx.x;
    const PartHead head = *part_head(g, share, 1);
    if (head.unit < 0) return;
    const KvArgs & kv = g.kv;
    int bad = head.bad, last = share;
    for (bool ends = false; !ends && last + 1 < g.max_shares;) {
        const PartHead next = *part_head(g, ++last, 0);
        bad |= next.bad;
        ends = next.ends;
    }
    const int seq = head.unit / kv.kv_heads, kv_head = head.unit % kv.kv_heads;
    const Sequence q = sequence(kv, seq);
    const int rows = q.n * g.group;
    for (int e = tid; e < rows * (D / 4); e += kJoinThreads) {
        const int m = e / (D / 4), c = e % (D / 4) * 4;
        float top = -kInf, sum = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int i = share; i <= last; i++) {
            const float * data = part_data(g, i, i == share, pairs);
            const float2 s = *reinterpret_cast<const float2 *>(data + 2 * m);
            const float4 x = *reinterpret_cast<const float4 *>(data + 2 * pairs + m * D + c);
            const float t = fmaxf(top, s.x), ref = t == -kInf ? 0.0f : t;
            const float a = ex2(top - ref), b = ex2(s.x - ref);
            top = t;
            sum = sum * a + s.y * b;
            o.x = o.x * a + x.x * b, o.y = o.y * a + x.y * b, o.z = o.z * a + x.z * b, o.w = o.w * a + x.w * b;
        }
        const bool blank = bad || q.length - q.n + m / g.group < 0;
        const float inv = 1.0f / sum, fill = refused_value(bad);
        const int64_t out_row = q.start + m / g.group;
        const int h = kv_head * g.group + m % g.group;
        store_pair(g, out_row, h, c, blank ? fill : o.x * inv, blank ? fill : o.y * inv);
        store_pair(g, out_row, h, c + 2, blank ? fill : o.z * inv, blank ? fill : o.w * inv);
        if (g.lse && c == 0) g.lse[out_row * g.q_heads + h] = blank ? -kInf : (top == -kInf ? 0.0f : top) * kLn2 + logf(sum);
    }
    if (tid == 0) report(g, seq, kv_head, bad);
}

constexpr int kMaxPairs = 64;  // (row, query head) pairs of one key head

template <int D, int MT>
cudaError_t launch(AttendArgs a, int sm_count, cudaStream_t stream) {
    CUtensorMap maps[2];
    const int box = a.kv.page_size < kTile ? a.kv.page_size : kTile;
    if (!page_map(&maps[0], a.kv.k, a.kv, D, box) || !page_map(&maps[1], a.kv.v, a.kv, D, box)) return cudaErrorInvalidValue;
    // as many CTAs as the SMs hold at once: two where 16 pairs leave room for two rings of three tiles
    constexpr int kPerSm = MT == 1 ? 2 : 1;
    constexpr size_t kBudget = (kPerSm == 2 ? 113 : 226) * 1024 - 2048;  // less the static shared memory
    int pairs = (a.kv.max_rows * a.group + 1) / 2 * 2;  // even: the partials' vectors stay aligned
    const size_t room = (size_t) pairs * (D + 8) * sizeof(float) + 1024;
    int stages = (int) ((kBudget - room) / stage_bytes<D>());
    stages = stages < kMaxStages ? stages : kMaxStages;
    const size_t smem = (size_t) stages * stage_bytes<D>() + room;
    // no more shares than the longest sequences could fill
    const int64_t reach = a.window > 0 ? std::min<int64_t>(a.kv.max_length, (int64_t) a.window + a.sinks + a.kv.max_rows + 2 * kTile) : a.kv.max_length;
    const int64_t tiles = (reach + kTile - 1) / kTile * a.kv.kv_heads * a.kv.seqs;
    const int64_t most = std::max<int64_t>(1, (tiles + kMinTiles - 1) / kMinTiles);
    const int shares = (int) std::min<int64_t>(kPerSm * sm_count, most);
    a.max_shares = shares;
    const void * kernel = (const void *) step_kernel<D, MT>;
    cudaError_t e = set_max_dynamic_smem(kernel, smem);
    if (e != cudaSuccess) return e;
    step_kernel<D, MT><<<shares, step_threads<MT>(), smem, stream>>>(maps[0], maps[1], a, stages, pairs);
    e = cudaGetLastError();
    if (e != cudaSuccess || shares == 1) return e;
    // launched while the shares still run, and waiting for them on the device
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned) shares);
    config.blockDim = dim3(kJoinThreads);
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, join_kernel<D>, a, pairs);
}

template <int D> cudaError_t launch(const AttendArgs & a, int sm_count, cudaStream_t stream) {
    const int64_t pairs = (int64_t) a.kv.max_rows * a.group;
    return pairs <= 16 ? launch<D, 1>(a, sm_count, stream) : pairs <= 32 ? launch<D, 2>(a, sm_count, stream) : launch<D, 4>(a, sm_count, stream);
}

}  // namespace

bool attend_step_takes(const AttendArgs & a) {
    return (int64_t) a.kv.max_rows * a.group <= kMaxPairs && tensor_core_takes(a);
}

// Two slots of every share: at most 2 CTAs per SM of 16 pairs, or 1 of 64.
int64_t attend_workspace_bytes(int sm_count) {
    return (int64_t) sm_count * (2 * 2 * sizeof(PartHead) + 2 * kMaxPairs * (128 + 2) * sizeof(float));
}

cudaError_t launch_attend_step(const AttendArgs & a, int sm_count, cudaStream_t stream) {
    return a.kv.head_dim == 64 ? launch<64>(a, sm_count, stream) : launch<128>(a, sm_count, stream);
}

}  // namespace ssb

// Attention of a few rows per sequence over a paged cache (head size 64 or 128): the step of one new token, and
// drafts to verify, up to 64 (row, query head) pairs per key head.
//
//   out = sum_j softmax_j(scale * q . k[j]) v[j] over the positions j that the row sees
//
// Every key and value is read once from HBM and used for all pairs of its head: 2 to 64 multiply-adds per
// element, so the bound is HBM and the arithmetic only has to keep up with it. The pairs are far fewer than the
// 128 rows of a tcgen05 tile, so bf16 products are warp-level mma.m16n8k16 with the pairs as the 16 rows and the
// accumulators in registers. fp32 products of up to 4 pairs are the FMA pipes', a lane per position for the scores and a
// lane per elements of the head for the output; of more pairs they are mma.m16n8k8 of tf32, three for each: a value is the sum
// of its 11 leading bits and the rest, and the product of two rests, 2^-22 of the product at most, is left out.
//
// The work is one list: the tiles of (sequence 0, key head 0), 64 positions of bf16 or 32 of fp32 each, then those of
// head 1, and so on. Every CTA takes an equal, consecutive share of it, as many CTAs as the SMs hold at once,
// whatever the lengths are: no SM waits for a long sequence, and a CTA's ring of TMA copies (out of the pages,
// 128-byte swizzle, no multicast) runs on from one (sequence, head) to the next. (Shares within a cluster per
// sequence and head, joined through distributed shared memory, took 1.5 times as long on 64 ragged streams: CTAs
// of short sequences left and started too often, and of clusters of 16 the GPU held 7 at once.) Two or three
// warps per 16 pairs take the tiles in turn, with a running maximum and sum of their own, and are joined
// through shared memory. A (sequence, head) that shares end in is left as partials in the workspace, one per
// share, and join_kernel joins them in order: equal calls give equal bits, and no atomics or waits between CTAs
// are needed. Every mbarrier wait is bounded: one that gives up ends its share, whose sequences become SSB_ROW_DEVICE_TIMEOUT.
//
// Measured, 8 key heads of 128 elements: one stream at 120001 positions 86 us (5.7 TB/s, launch and join included),
// 64 streams of up to 8000 positions 162 us (6.4 TB/s, 98% of a copy's rate), 128 dialogues under a window of 2000
// 160 us (6.3 TB/s), 24 streams with up to 5 drafts on 4 query heads per key head 57 us (4.0 TB/s: two CTAs of two tiles
// each per SM; their start and last units are 20 us of it; three tiles in one CTA took 61), one stream at 37 positions 7.6 us (latency: length,
// page, tile, one after the other), 16 streams of fp32 43 us (4.7 TB/s); the 24 streams with drafts in fp32 308 us
// (1.4 TB/s: the tf32 products and what splits and adds up their numbers; on the FMA pipes 736).
#include <algorithm>

#include "ssb_decoder.cuh"
#include "ssb_tma.cuh"
#include "ssb_tma_map.cuh"

namespace ssb {

namespace {

// Warps per 16 pairs. Each takes a tile of its own, every kGroups-th: with 16 positions of the same tile each, a
// warp's chain of product, maximum, weights and product took 2200 clocks per tile of 32 KB, that HBM brings an SM
// in 1400; a warp takes 2100 for a tile of its own, and six of an SM are at one each. Two groups fit an SM twice up to 32 pairs
// (head size 128: 28 of bf16, 20 of fp32); three groups of up to 16 pairs do at head size 64, and at 128 up to 6 of bf16, which
// one CTA of three still beats up to 10 pairs (24 streams of 300 to 4001 positions: 10 pairs 47 us, 50 with two groups twice;
// 16 pairs 54 and 51). The ring's stages are a multiple
// of the groups, so that a stage is always the same group's: a barrier's parity tells a phase only to who has seen
// the one before.
template <typename T, int D, int MT, int MP> constexpr int groups() { return MT == 1 && (D == 64 || MP < 16) ? 3 : 2; }
constexpr int kMaxStages = 8;
// A CTA's share is at least this many tiles: a tile per group, since more shares would bring more partials to join and
// no earlier end. Where no unit can have more than two tiles per group, shares are of whole units and nothing is left
// to join: drafts of 12 streams at up to 163 positions take 9.6 us, and took 14.1 with parts and their join.
constexpr int kMinTiles = 3, kWholeTiles = 6;
// What a unit costs besides its tiles, in tiles: shares of many short units would end last otherwise.
constexpr int kUnitCost = 2;

// Positions of a tile: 64 of bf16, 32 of fp32, keys and values 256 D bytes either way.
template <typename T> constexpr int tile_of() { return sizeof(T) == 2 ? 64 : 32; }
template <int D> constexpr int stage_bytes() { return 256 * D; }
template <typename T, int D, int MT, int MP> constexpr int step_threads() { return (groups<T, D, MT, MP>() * MT + 1) * 32; }
// bf16, and more than 4 pairs of fp32: at 24 streams of 300 to 4001 positions 6 pairs take 205 us so (head size 128; 97 at 64),
// 302 (115) on the FMA pipes; 4 pairs take 129 (81) there
template <typename T, int MP> constexpr bool by_tensor_cores() { return sizeof(T) == 2 || MP == 16; }

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
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An fp32 value as the sum of two of 11 bits and more: `high` is it rounded to tf32, `low` the exact rest, of which the
// product takes the first 11 bits, all but one. Not finite: `low` is NaN. From kSplitLimit on, where rounding leaves the range,
// `high` is infinite and `low` minus that.
constexpr float kSplitLimit = 0x1.ffep127f;
__device__ __forceinline__ void split(uint32_t x, uint32_t & high, uint32_t & low) {
    high = (x + 0x1000u) & 0xffffe000u;
    low = __float_as_uint(__uint_as_float(x) - __uint_as_float(high));
}
template <int N> __device__ __forceinline__ void split(const uint32_t (&x)[N], uint32_t (&high)[N], uint32_t (&low)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) split(x[i], high[i], low[i]);
}
// The larger size, or NaN where either is.
__device__ __forceinline__ float max_size(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(fabsf(b)));
    return y;
}
__device__ __forceinline__ float load_shared(uint32_t at) {
    float x;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at));
    return x;
}
__device__ __forceinline__ float2 load_shared2(uint32_t at) {
    float2 x;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at));
    return x;
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// The n lowest bits of 64, for any n.
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }
__device__ __forceinline__ bool bf16_pair_not_finite(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// Named barriers of a hand-over from one group's slot to the group that joins.
__device__ __forceinline__ int slot_full(int from, int joiner) { return 1 + from * 2 + (joiner > from ? joiner - 1 : joiner); }
__device__ __forceinline__ int slot_free(int from, int joiner) { return 6 + slot_full(from, joiner); }

// What the shares of a call are: `total` tiles, kUnitCost more for every unit (or as many as there are units, where they
// stay whole), in `shares` equal parts.
struct Plan {
    int64_t total;
    int shares;
    int64_t each;  // of a share; the first `more` have one more
    int more;
    __device__ __forceinline__ int64_t begin(int i) const { return i < shares ? i * each + min(i, more) : total; }
};

template <int kTile> __device__ __forceinline__ SpanOf<kTile> span_of(const AttendArgs & g, const Sequence & q) {
    return span_of<kTile>(q.length - q.n, q.length - 1, g.window, g.sinks);
}
template <int kTile> __device__ __forceinline__ int tiles_of(const AttendArgs & g, const Sequence & q) {
    return q.ok && q.n > 0 ? span_of<kTile>(g, q).tiles : 0;
}
// A unit's length in the list, of which the first cost_before() places are no tiles.
__device__ __forceinline__ int cost_before(const AttendArgs & g) { return g.whole_units ? 0 : kUnitCost; }
__device__ __forceinline__ int unit_cost(const AttendArgs & g, int tiles) { return g.whole_units ? 1 : tiles + kUnitCost; }
template <int kTile> __device__ __forceinline__ int64_t cost_of(const AttendArgs & g, const Sequence & q) {
    const int tiles = tiles_of<kTile>(g, q);
    return tiles > 0 ? (int64_t) unit_cost(g, tiles) * g.kv.kv_heads : 0;
}

// The walk over a share, unit by unit ((sequence, key head) pairs), the next sequence's numbers on their way.
template <int kTile> struct Walk {
    int seq, head, tiles;  // the unit, and its tiles
    int64_t at, end;       // the unit's place in the list, and the share's end
    Sequence q;
    SequenceNumbers ahead;
    __device__ __forceinline__ void start(const AttendArgs & g, int s, const SequenceNumbers & numbers, int64_t seq_at, int64_t begin, int64_t stop) {
        seq = s;
        q = sequence(g.kv, numbers);
        ahead = sequence_numbers(g.kv, min(s + 1, g.kv.seqs - 1));
        tiles = tiles_of<kTile>(g, q);
        const int64_t into = begin - seq_at;  // below 2^25 tiles times 2^10 heads
        const int each = unit_cost(g, tiles);
        head = into <= INT32_MAX ? (int) ((uint32_t) into / (uint32_t) each) : (int) (into / each);
        at = seq_at + (int64_t) head * each;
        end = stop;
    }
    // the unit's tiles that are this share's: from `now` (the share's begin, or a unit's) on
    __device__ __forceinline__ int first_tile(const AttendArgs & g, int64_t now) const {
        return g.whole_units ? 0 : (int) max(now - at - kUnitCost, (int64_t) 0);
    }
    __device__ __forceinline__ int last_tile(const AttendArgs & g) const {
        return g.whole_units ? tiles : (int) min((int64_t) tiles, max(end - at - kUnitCost, (int64_t) 0));
    }
    // whether the share has tiles of a later unit
    __device__ __forceinline__ bool more(const AttendArgs & g) const { return end - (at + unit_cost(g, tiles)) > cost_before(g); }
    __device__ __forceinline__ void next(const AttendArgs & g) {
        at += unit_cost(g, tiles);
        if (++head < g.kv.kv_heads) return;
        head = 0;
        do {
            q = sequence(g.kv, ahead);
            ahead = sequence_numbers(g.kv, min(++seq + 1, g.kv.seqs - 1));
            tiles = tiles_of<kTile>(g, q);
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

template <typename T> __device__ __forceinline__ void store_two(const AttendArgs & g, T * dst, float x, float y);
template <> __device__ __forceinline__ void store_two<__nv_bfloat16>(const AttendArgs & g, __nv_bfloat16 * dst, float x, float y) {
    if (g.vec_out) *reinterpret_cast<uint32_t *>(dst) = pack_bf16(x, y);
    else dst[0] = narrow<__nv_bfloat16>(x), dst[1] = narrow<__nv_bfloat16>(y);
}
template <> __device__ __forceinline__ void store_two<float>(const AttendArgs & g, float * dst, float x, float y) {
    if (g.vec_out) *reinterpret_cast<float2 *>(dst) = make_float2(x, y);
    else dst[0] = x, dst[1] = y;
}
template <typename T> __device__ __forceinline__ void store_pair(const AttendArgs & g, int64_t row, int head, int at, float x, float y) {
    store_two(g, static_cast<T *>(g.out) + row * g.out_ld + (int64_t) head * g.kv.head_dim + at, x, y);
}

// A wait that the wait-limit test build (SSB_WAIT_TEST) lets run out for one warp of a group alone: for the fifth tile of sequence
// 2's second key head.
__device__ __forceinline__ bool late(int seq, int head, int tile, bool one) {
#ifdef SSB_WAIT_TEST
    if (one && seq == 2 && head == 1 && tile == 4) {
        for (const long long t0 = clock64(); clock64() - t0 <= kWaitCycles;) {}
        return true;
    }
#endif
    return false;
}

// MP: the most pairs of a warp.
template <typename T, int D, int MT, int MP>
__global__ void __launch_bounds__(step_threads<T, D, MT, MP>(), MT <= 2 ? 2 : 1)
    step_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ AttendArgs g, int stages, int pairs) {
    constexpr int kTile = tile_of<T>(), kBytes = sizeof(T);
    constexpr int kPitch = D + 8, kQueryPitch = D * kBytes + 16, kGroups = groups<T, D, MT, MP>(), kThreads = step_threads<T, D, MT, MP>();
    constexpr int kHandOver = 2 * MT * 32;  // threads of the two sides of a hand-over between a unit's warps
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char * smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    // [2][pairs][kQueryPitch]; a product reads 16 rows for every 16 pairs, those past the last for nobody
    unsigned char * query = smem + (size_t) stages * stage_bytes<D>();
    float * room = reinterpret_cast<float *>(query + (size_t) 2 * pairs * kQueryPitch);  // [kGroups][pairs][kPitch]
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
    __shared__ float2 stat[kGroups][16 * MT];
    __shared__ int64_t s_scan[kThreads / 32];
    __shared__ int64_t s_at, s_begin, s_end;
    __shared__ SequenceNumbers s_numbers;
    __shared__ int s_seq, s_idle, s_dead;
    __shared__ __align__(8) uint64_t query_full[2], query_empty[2];
    __shared__ PartHead s_part[2];
    __shared__ int s_bad[kGroups];  // what refuses the unit, from the warps that hand over their part of it
    constexpr bool kFma = !by_tensor_cores<T, MP>();
    __shared__ __align__(16) float s_weight[kFma ? kGroups * MT : 1][kFma ? MP : 1][kFma ? kTile : 4];  // a warp's weights
    __shared__ int s_refused[kMaxStages];  // per tile: its unit has a page outside the pool
    const KvArgs & kv = g.kv;
    const int tid = (int) threadIdx.x, warp = warp_id(), lane = lane_id(), me = (int) blockIdx.x;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // join_kernel may be set up meanwhile
    if (tid == kThreads - 1) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
    // ---- every CTA adds up the tiles of all sequences and finds where its share begins
    const int chunk = (kv.seqs + kThreads - 1) / kThreads;
    const int c0 = min(tid * chunk, kv.seqs), c1 = min(c0 + chunk, kv.seqs);
    SequenceNumbers numbers = sequence_numbers(kv, min(c0, kv.seqs - 1));  // on their way during the set-up
    int64_t mine = 0;
    bool idle = false;
    if (tid == 0) {
        for (int s = 0; s < stages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], MT);
        for (int s = 0; s < 2; s++) mbar_init(&query_full[s], 32), mbar_init(&query_empty[s], kGroups * MT);
        s_idle = s_dead = 0;
        s_part[0] = s_part[1] = {-1, 0, 0, 0};
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    for (int s = c0; s < c1; s++) {
        if (s > c0) numbers = sequence_numbers(kv, s);
        const int64_t n = cost_of<kTile>(g, sequence(kv, numbers));
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
    const int least = g.whole_units ? 1 : kMinTiles + kUnitCost;  // of a share
    plan.shares = (int) min((int64_t) gridDim.x, (plan.total + least - 1) / least);
    if (plan.shares == 0) {
        plan.each = plan.more = 0;
    } else if (plan.total <= INT32_MAX) {
        plan.each = (uint32_t) plan.total / (uint32_t) plan.shares;
        plan.more = (int) ((uint32_t) plan.total - (uint32_t) plan.each * (uint32_t) plan.shares);
    } else {
        plan.each = plan.total / plan.shares;
        plan.more = (int) (plan.total - plan.each * plan.shares);
    }
    const int64_t begin = plan.begin(me), end = plan.begin(me + 1);
    int64_t at = upto - mine;
    if (begin < end && at <= begin && begin < upto) {
        for (int s = c0; s < c1; s++) {
            if (chunk > 1) numbers = sequence_numbers(kv, s);
            const int64_t past = at + cost_of<kTile>(g, sequence(kv, numbers));
            if (begin < past) {
                s_seq = s;
                s_at = at, s_begin = begin, s_end = end;
                s_numbers = numbers;
                break;
            }
            at = past;
        }
    }
    __syncthreads();
    Walk<kTile> walk{};
    if (begin < end) walk.start(g, s_seq, s_numbers, s_at, begin, end);
    auto dead = [&]() { return *reinterpret_cast<volatile int *>(&s_dead) != 0; };
    const int box = kv.page_size < kTile ? kv.page_size : kTile;  // positions of one TMA copy: a piece of a tile
    if (warp == kGroups * MT) {
        // ---- producer: lane l looks up and copies piece l of every 32
        const int per_tile = kTile / box, batch = 32 / per_tile;
        int it = 0, unit = 0, issued = 0;
        int64_t now = begin;
        for (bool more = begin < end; more && !__any_sync(0xffffffffu, dead()); unit++) {
            const int t0 = walk.first_tile(g, now), t1 = walk.last_tile(g);
            const auto span = span_of<kTile>(g, walk.q);
            const int32_t * table = kv.table + (int64_t) walk.seq * kv.table_ld;
            bool ok = true, queries = false;
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
                    const bool issue = !left_out(walk.seq, walk.head, u);
                    if (lane == 0 && issue) {
                        s_refused[s] = refuse;  // read by the consumers once the barrier's phase has ended
                        mbar_expect(&full[s], (uint32_t) (__popc(votes & of_tile) * 2 * box * D * kBytes));
                    }
                    __syncwarp();
                    if (valid && issue && my_tile == u) {
                        unsigned char * dst = smem + (size_t) s * stage_bytes<D>() + lane % per_tile * box * D * kBytes;
                        const int slot = from & (kv.page_size - 1);
                        tma_load_5d(dst, &map_k, 0, slot, 0, walk.head, page, &full[s]);
                        tma_load_5d(dst + kTile * D * kBytes, &map_v, 0, slot, 0, walk.head, page, &full[s]);
                    }
                    issued = it + 1;
                    if (queries) continue;
                    // behind the unit's first tile, its pairs
                    queries = true;
                    const bool free = unit < 2 || mbar_wait(&query_empty[unit & 1], (uint32_t) (unit / 2 - 1) & 1u);
                    if (!__all_sync(0xffffffffu, free)) {
                        ok = false;
                        break;
                    }
                    const int rows = walk.q.n * g.group;
                    unsigned char * dst = query + (unit & 1) * pairs * kQueryPitch;
                    for (int e = lane; e < rows * (D / 4); e += 32) {  // rows past them hold anything, for nobody
                        const int m = e / (D / 4), c = e % (D / 4) * 4;
                        const T * src = static_cast<const T *>(g.q) + (int64_t) (walk.q.start + m / g.group) * g.q_ld +
                                        (int64_t) (walk.head * g.group + m % g.group) * D + c;
                        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(dst + m * kQueryPitch + c * kBytes)), "l"(src), "n"(4 * kBytes) : "memory");
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(&query_full[unit & 1])) : "memory");
                }
            }
            if (!ok) {
                if (lane == 0) atomicOr(&s_dead, 1);
                break;
            }
            more = walk.more(g);
            if (more) {
                walk.next(g);
                now = walk.at;
            }
        }
        __syncwarp();
        asm volatile("cp.async.wait_all;" ::: "memory");
        // The copies in flight land before the shared memory is given up, whichever warp's wait ran out and however late:
        // a consumer may give up when this warp has issued its last copy. (Else this warp has nothing else to do.)
        for (int i = max(0, issued - stages); i < issued; i++) mbar_wait(&full[i % stages], (uint32_t) (i / stages) & 1u);
    } else if constexpr (!kFma) {
        // ---- consumers whose products are the tensor cores'
        const int mt = warp % MT, kg = warp / MT;
        const int r0 = mt * 16 + lane / 4;  // this thread's pairs: r0 and r0 + 8
        const int pair_row[2] = {r0 / g.group, (r0 + 8) / g.group};  // their rows in the sequence, and query heads
        const int pair_head[2] = {r0 % g.group, (r0 + 8) % g.group};
        // a tile is [piece][column block of 128 bytes][position]: where its groups of 16 positions start
        const int box_shift = __ffs(box) - 1;
        const uint32_t half_at = (uint32_t) box * 128;
        auto rows_at = [&](int r) { return (uint32_t) ((r >> box_shift) * (box * D * kBytes) + (r & (box - 1)) * 128); };
        uint32_t group_at[kTile / 16];
#pragma unroll
        for (int kk = 0; kk < kTile / 16; kk++) group_at[kk] = rows_at(kk * 16);
        const int k_row = (lane & 7) + (lane >> 4) * 8, k_chunk = lane >> 3 & 1;
        const int v_row = (lane & 7) + (lane >> 3 & 1) * 8, v_chunk = lane >> 4;
        const uint32_t query_at = smem_addr(query) + (uint32_t) ((mt * 16 + (lane & 15)) * kQueryPitch + (lane >> 4) * 16);
        // scores in units of the base 2 logarithm; not 0 (tma_takes), so that 2^(-inf * scale) stays 0
        const float scale = fabsf(g.scale_log2);
        const uint32_t sign = g.scale_log2 < 0.0f ? (kBytes == 2 ? 0x80008000u : 0x80000000u) : 0u;
        int it = 0, unit = 0, owed = 0;  // owed: the group that has this one's slot of `room`, 0 for none
        int64_t now = begin;
        bool more = begin < end, entered = false;
        while (more) {
            if (entered) {
                walk.next(g);
                now = walk.at;
                unit++;
            }
            entered = true;
            more = walk.more(g);
            const auto span = span_of<kTile>(g, walk.q);
            const int t0 = walk.first_tile(g, now), t1 = walk.last_tile(g);
            const int rows = walk.q.n * g.group;  // (row, query head) pairs of this unit
            const int p_first = walk.q.length - walk.q.n, p_last = walk.q.length - 1;
            // what this thread's rows see: seen_n positions from seen_from, and the sinks
            int position[2], seen_from[2], seen_n[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                position[i] = p_first + min(pair_row[i], walk.q.n - 1);
                seen_from[i] = g.window > 0 ? max(position[i] - g.window + 1, 0) : 0;
                seen_n[i] = max(position[i] + 1 - seen_from[i], 0);
            }
            auto visible = [&](int i, int j) { return (unsigned) (j - seen_from[i]) < (unsigned) seen_n[i] || (j < g.sinks && j <= position[i]); };
            const bool fed = __all_sync(0xffffffffu, !dead() && mbar_wait(&query_full[unit & 1], (uint32_t) (unit / 2) & 1u));
            if (!fed && lane == 0) atomicOr(&s_dead, 1);
            const uint32_t queries = query_at + (uint32_t) ((unit & 1) * pairs * kQueryPitch);
            float o[D / 8][4];
            float top[2] = {-kInf, -kInf}, sum[2] = {0.0f, 0.0f};
            int bad = 0;
#pragma unroll
            for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            const int it_after = it + t1 - t0;  // wherever the loop ends
            for (int t = t0; t < t1; t++, it++) {
                if (it % kGroups != kg) continue;
                const int s = it % stages;
                const bool ok = !dead() && !late(walk.seq, walk.head, t, MT > 1 && mt == (rows - 1) / 16) && mbar_wait(&full[s], (uint32_t) (it / stages) & 1u);
                if (!__all_sync(0xffffffffu, ok)) {
                    if (lane == 0) atomicOr(&s_dead, 1);
                    break;
                }
                bad |= *reinterpret_cast<volatile int *>(&s_refused[s]);
                const uint32_t keys = smem_addr(smem) + (uint32_t) s * stage_bytes<D>(), values = keys + kTile * D * kBytes;
                float c[kTile / 8][4] = {};
                // fp32: a tensor core cuts its sums off where an addition rounds, so that a sum of many is off in one direction
                // (an output of 4000 positions by 4e-6, ten times what fp32 additions make it); four products at a time, and
                // the small ones apart, are added up here, and an output's eight positions below (2.3e-7)
                constexpr int kSmall = kBytes == 4 ? kTile / 8 : 1;
                float small[kSmall][4] = {}, four[kSmall][4] = {};
#pragma unroll
                for (int ks = 0; ks < D * kBytes / 32; ks++) {  // 32 bytes of the head: 16 elements of bf16, 8 of fp32
                    uint32_t qa[4];
                    ldmatrix(qa, queries + ks * 32);
                    if (sign != 0) qa[0] ^= sign, qa[1] ^= sign, qa[2] ^= sign, qa[3] ^= sign;
                    const int chunk = ks * 2 + k_chunk;
                    const uint32_t at = keys + (uint32_t) (chunk / 8) * half_at + (uint32_t) (k_row * 128 + ((chunk % 8) ^ (k_row & 7)) * 16);
                    if constexpr (kBytes == 2) {
#pragma unroll
                        for (int kk = 0; kk < kTile / 16; kk++) {
                            uint32_t b[4];
                            ldmatrix(b, at + group_at[kk]);
                            mma(c[2 * kk], qa, b[0], b[1]);
                            mma(c[2 * kk + 1], qa, b[2], b[3]);
                        }
                    } else {
                        uint32_t qh[4], ql[4], kh[kTile / 16][4], kl[kTile / 16][4];
                        split(qa, qh, ql);
#pragma unroll
                        for (int kk = 0; kk < kTile / 16; kk++) {
                            uint32_t b[4];
                            ldmatrix(b, at + group_at[kk]);
                            split(b, kh[kk], kl[kk]);
                        }
#pragma unroll
                        for (int nt = 0; nt < kTile / 8; nt++) mma_tf32(small[nt], qh, kl[nt / 2][nt % 2 * 2], kl[nt / 2][nt % 2 * 2 + 1]);
#pragma unroll
                        for (int nt = 0; nt < kTile / 8; nt++) mma_tf32(four[nt], qh, kh[nt / 2][nt % 2 * 2], kh[nt / 2][nt % 2 * 2 + 1]);
#pragma unroll
                        for (int nt = 0; nt < kTile / 8; nt++) mma_tf32(small[nt], ql, kh[nt / 2][nt % 2 * 2], kh[nt / 2][nt % 2 * 2 + 1]);
                        if (ks % 4 != 3) continue;
#pragma unroll
                        for (int nt = 0; nt < kTile / 8; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                c[nt][e] += ks == D / 8 - 1 ? four[nt][e] + small[nt][e] : four[nt][e];
                                four[nt][e] = 0.0f;
                            }
                    }
                }
                const int base = span.base(t);
                const bool whole = base + kTile - 1 <= p_first && (g.window == 0 || base > p_last - g.window || base + kTile - 1 < g.sinks);
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        // the tile's positions that row i sees, a bit each, this thread's at the bits 8 nt and 8 nt + 1
                        const uint64_t bits = ((bits_below(seen_from[i] + seen_n[i] - base) & ~bits_below(seen_from[i] - base)) |
                                               bits_below(min(g.sinks, position[i] + 1) - base)) >> (lane % 4 * 2);
                        const uint32_t low = (uint32_t) bits, high = (uint32_t) (bits >> 32);
#pragma unroll
                        for (int nt = 0; nt < kTile / 8; nt++)
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                if (!((nt < 4 ? low : high) >> (nt % 4 * 8 + e) & 1u)) c[nt][2 * i + e] = -kInf;
                    }
                }
                if constexpr (kBytes == 4) {  // a value that is not finite makes its parts' product NaN: those one by one
#pragma unroll
                    for (int nt = 0; nt < kTile / 8; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (c[nt][e] == c[nt][e]) continue;
                            const int m = r0 + e / 2 * 8, j = nt * 8 + lane % 4 * 2 + e % 2;
                            if (m >= rows) continue;
                            const float * q_row = reinterpret_cast<const float *>(query + (size_t) ((unit & 1) * pairs + m) * kQueryPitch);
                            float s = 0.0f;
                            for (int d = 0; d < D; d++)
                                s += q_row[d] * load_shared(keys + rows_at(j) + (uint32_t) (d / 32) * half_at + (uint32_t) (((d / 4 % 8) ^ (j & 7)) * 16 + d % 4 * 4));
                            c[nt][e] = sign ? -s : s;
                        }
                }
                float new_top[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    new_top[i] = fmaxf(c[0][2 * i], c[0][2 * i + 1]);
#pragma unroll
                    for (int nt = 1; nt < kTile / 8; nt++) new_top[i] = fmaxf(new_top[i], fmaxf(c[nt][2 * i], c[nt][2 * i + 1]));
                    new_top[i] = fmaxf(new_top[i], shfl_xor(new_top[i], 1));
                    new_top[i] = fmaxf(top[i], fmaxf(new_top[i], shfl_xor(new_top[i], 2)) * scale);
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
                // the weights rounded to bf16 for the product: half a step of the output's own type
                uint32_t pa[kTile / 16][4];  // (bf16)
#pragma unroll
                for (int nt = 0; nt < kTile / 8; nt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) c[nt][e] = ex2(fmaf(c[nt][e], scale, -ref[e / 2]));
                    sum[0] += c[nt][0] + c[nt][1];
                    sum[1] += c[nt][2] + c[nt][3];
                    if constexpr (kBytes == 2) {
                        pa[nt / 2][nt % 2 * 2] = pack_bf16(c[nt][0], c[nt][1]);
                        pa[nt / 2][nt % 2 * 2 + 1] = pack_bf16(c[nt][2], c[nt][3]);
                    }
                }
                if constexpr (kBytes == 4) {
                    // Eight positions at a time, the first of each two as the product's columns 0 to 3 and the second as
                    // 4 to 7: the scores are then where the product takes its weights. Values that no row sees are cleared;
                    // where one of the others is not finite, or its split is not, the eight are taken one at a time,
                    // for the rows that see them.
#pragma unroll
                    for (int nt = 0; nt < kTile / 8; nt++) {
                        const int p = base + nt * 8 + lane % 4 * 2, r = lane % 4 * 2;
                        const bool keep[2] = {whole || span.seen(p), whole || span.seen(p + 1)};
                        if (!whole && !__any_sync(0xffffffffu, keep[0] || keep[1])) continue;
                        const uint32_t at = values + rows_at(nt * 8);
                        uint32_t v[D / 8][2];
                        float most = 0.0f;
#pragma unroll
                        for (int n = 0; n < D / 8; n++)
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const int chunk = n * 2 + lane / 16;
                                const float x = load_shared(at + (uint32_t) (chunk / 8) * half_at + (uint32_t) ((r + i) * 128 + ((chunk % 8) ^ (r + i)) * 16 + lane / 4 % 4 * 4));
                                v[n][i] = keep[i] ? __float_as_uint(x) : 0u;
                            }
                        const uint32_t w[4] = {__float_as_uint(c[nt][0]), __float_as_uint(c[nt][2]), __float_as_uint(c[nt][1]), __float_as_uint(c[nt][3])};
                        uint32_t wh[4], wl[4];
                        split(w, wh, wl);
#pragma unroll
                        for (int n = 0; n < D / 8; n++)
#pragma unroll
                            for (int i = 0; i < 2; i++) most = max_size(most, __uint_as_float(v[n][i]));
                        if (__any_sync(0xffffffffu, !(most < kSplitLimit))) {
                            for (int j = 0; j < 8; j++) {
                                const int from = (lane & ~3) | (j / 2);
                                const float w0 = __shfl_sync(0xffffffffu, j % 2 ? c[nt][1] : c[nt][0], from);
                                const float w1 = __shfl_sync(0xffffffffu, j % 2 ? c[nt][3] : c[nt][2], from);
                                const bool see0 = visible(0, base + nt * 8 + j), see1 = visible(1, base + nt * 8 + j);
#pragma unroll
                                for (int n = 0; n < D / 8; n++) {
                                    const int chunk = n * 2 + lane % 4 / 2;
                                    const float2 x = load_shared2(at + (uint32_t) (chunk / 8) * half_at + (uint32_t) (j * 128 + ((chunk % 8) ^ j) * 16 + lane % 2 * 8));
                                    if (see0) o[n][0] += w0 * x.x, o[n][1] += w0 * x.y;
                                    if (see1) o[n][2] += w1 * x.x, o[n][3] += w1 * x.y;
                                }
                            }
                            continue;
                        }
#pragma unroll
                        for (int n0 = 0; n0 < D / 8; n0 += 4) {
                            uint32_t vh[4][2], vl[4][2];
                            float eight[4][4] = {};
#pragma unroll
                            for (int n = 0; n < 4; n++) split(v[n0 + n], vh[n], vl[n]);
#pragma unroll
                            for (int n = 0; n < 4; n++) mma_tf32(eight[n], wh, vl[n][0], vl[n][1]);
#pragma unroll
                            for (int n = 0; n < 4; n++) mma_tf32(eight[n], wl, vh[n][0], vh[n][1]);
#pragma unroll
                            for (int n = 0; n < 4; n++) mma_tf32(eight[n], wh, vh[n][0], vh[n][1]);
#pragma unroll
                            for (int n = 0; n < 4; n++)
#pragma unroll
                                for (int e = 0; e < 4; e++) o[n0 + n][e] += eight[n][e];
                        }
                    }
                } else {
                // A value that its weight of 0 must keep out has to be finite. Positions that no row sees are
                // cleared as they are loaded; those that some rows see and others do not are looked through, and
                // taken one at a time, for the rows that see them, where they are not finite.
                bool apart = false;
                if (!whole && walk.q.n > 1) {
                    bool found = false;
#pragma unroll
                    for (int side = 0; side < 2; side++) {  // seen by the later rows only, and by the earlier ones only
                        const int j0 = max(side == 0 ? p_first + 1 : span.first, base);
                        const int j1 = min(side == 0 ? span.hi : (g.window > 0 ? p_last - g.window + 1 : 0), base + kTile);
                        for (int e = lane; e < (j1 - j0) * (D / 8); e += 32) {
                            const int r = j0 - base + e / (D / 8), chunk = e % (D / 8);
                            uint4 x;
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                                         : "r"(values + rows_at(r) + (uint32_t) (chunk / 8) * half_at + (uint32_t) (chunk % 8 * 16)));
                            found |= bf16_pair_not_finite(x.x) | bf16_pair_not_finite(x.y) | bf16_pair_not_finite(x.z) | bf16_pair_not_finite(x.w);
                        }
                    }
                    apart = __any_sync(0xffffffffu, found);
                }
                if (whole) {
#pragma unroll
                    for (int kk = 0; kk < kTile / 16; kk++)
#pragma unroll
                        for (int n2 = 0; n2 < D / 16; n2++) {
                            const int chunk = n2 * 2 + v_chunk;
                            uint32_t b[4];
                            ldmatrix_trans(b, values + group_at[kk] + (uint32_t) (chunk / 8) * half_at + (uint32_t) (v_row * 128 + ((chunk % 8) ^ (v_row & 7)) * 16));
                            mma(o[2 * n2], pa[kk], b[0], b[1]);
                            mma(o[2 * n2 + 1], pa[kk], b[2], b[3]);
                        }
                } else if (!apart) {
#pragma unroll
                    for (int kk = 0; kk < kTile / 16; kk++) {
                        uint32_t keep[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int j = base + kk * 16 + i * 8 + lane % 4 * 2;
                            keep[i] = (span.seen(j) ? 0xffffu : 0u) | (span.seen(j + 1) ? 0xffff0000u : 0u);
                        }
                        if (!__any_sync(0xffffffffu, (keep[0] | keep[1]) != 0)) continue;
#pragma unroll
                        for (int n2 = 0; n2 < D / 16; n2++) {
                            const int chunk = n2 * 2 + v_chunk;
                            uint32_t b[4];
                            ldmatrix_trans(b, values + group_at[kk] + (uint32_t) (chunk / 8) * half_at + (uint32_t) (v_row * 128 + ((chunk % 8) ^ (v_row & 7)) * 16));
                            mma(o[2 * n2], pa[kk], b[0] & keep[0], b[1] & keep[1]);
                            mma(o[2 * n2 + 1], pa[kk], b[2] & keep[0], b[3] & keep[1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int kk = 0; kk < kTile / 16; kk++)
                        for (int j = 0; j < 16; j++) {
                            const int from = (lane & ~3) | (j % 8 / 2), p = base + kk * 16 + j;
                            float w[2];
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const uint32_t pair = __shfl_sync(0xffffffffu, j < 8 ? pa[kk][i] : pa[kk][2 + i], from);
                                w[i] = j % 2 ? bf16_hi(pair) : bf16_lo(pair);
                            }
                            const bool see0 = visible(0, p), see1 = visible(1, p);
#pragma unroll
                            for (int n = 0; n < D / 8; n++) {
                                uint32_t pair;
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pair)
                                             : "r"(values + group_at[kk] + (uint32_t) (n / 8) * half_at + (uint32_t) (j * 128 + ((n % 8) ^ (j & 7)) * 16 + lane % 4 * 4)));
                                if (see0) o[n][0] += w[0] * bf16_lo(pair), o[n][1] += w[0] * bf16_hi(pair);
                                if (see1) o[n][2] += w[1] * bf16_lo(pair), o[n][3] += w[1] * bf16_hi(pair);
                            }
                        }
                }
                }  // (bf16)
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
            it = it_after;
            if (lane == 0) mbar_arrive(&query_empty[unit & 1]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                sum[i] += shfl_xor(sum[i], 1);
                sum[i] += shfl_xor(sum[i], 2);
            }
            // The groups that had tiles of this unit hand over to the one that had the last (`it` is past it), each in a
            // slot of its own, and go on with the next unit; so the joins go round the groups.
            const int joiner = (it - 1) % kGroups, others = min(t1 - t0, kGroups) - 1;
            const int behind = (joiner - kg + kGroups) % kGroups;  // how many tiles before the joiner's last this one's was
            if (behind > others) continue;
            if (behind > 0) {
                if (owed) bar_sync(slot_free(kg, owed - 1), kHandOver);
                owed = joiner + 1;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int m = r0 + 8 * i;
                    if (m >= rows) continue;
                    if (lane % 4 == 0) stat[kg][m] = make_float2(top[i], sum[i]);
                    float * slot = room + (size_t) (kg * pairs + m) * kPitch + lane % 4 * 2;
#pragma unroll
                    for (int n = 0; n < D / 8; n++) *reinterpret_cast<float2 *>(slot + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
                }
                if (mt == 0 && lane == 0) s_bad[kg] = bad;
                bar_arrive(slot_full(kg, joiner), kHandOver);
                continue;
            }
            for (int i = 1; i <= others; i++) {
                const int from = (joiner - i + kGroups) % kGroups;
                bar_sync(slot_full(from, joiner), kHandOver);
                bad |= *reinterpret_cast<volatile int *>(&s_bad[from]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int m = r0 + 8 * i;
                    if (m >= rows) continue;
                    const float2 other = stat[from][m];
                    const float t = fmaxf(top[i], other.x), ref = t == -kInf ? 0.0f : t;
                    const float a = ex2(top[i] - ref), b = ex2(other.x - ref);
                    top[i] = t;
                    sum[i] = sum[i] * a + other.y * b;
                    const float * slot = room + (size_t) (from * pairs + m) * kPitch + lane % 4 * 2;
#pragma unroll
                    for (int n = 0; n < D / 8; n++) {
                        const float2 x = *reinterpret_cast<const float2 *>(slot + n * 8);
                        o[n][2 * i] = o[n][2 * i] * a + x.x * b, o[n][2 * i + 1] = o[n][2 * i + 1] * a + x.y * b;
                    }
                }
                bar_arrive(slot_free(from, joiner), kHandOver);
            }
            const bool begins = t0 == 0, ends = t1 == walk.tiles;
            if (begins && ends) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int m = r0 + 8 * i;
                    if (m >= rows) continue;
                    const int64_t out_row = walk.q.start + pair_row[i];
                    const int h = walk.head * g.group + pair_head[i];
                    const bool blank = bad || position[i] < 0;
                    const float inv = 1.0f / sum[i];
                    T * dst = static_cast<T *>(g.out) + out_row * g.out_ld + (int64_t) h * D + lane % 4 * 2;
#pragma unroll
                    for (int n = 0; n < D / 8; n++) {
                        const float x = blank ? 0.0f : o[n][2 * i] * inv, y = blank ? 0.0f : o[n][2 * i + 1] * inv;
                        store_two(g, dst + n * 8, x, y);
                    }
                    if (g.lse && lane % 4 == 0)
                        g.lse[out_row * g.q_heads + h] = blank ? -kInf : (top[i] == -kInf ? 0.0f : top[i]) * kLn2 + logf(sum[i]);
                }
                if (mt == 0 && lane == 0) raise_status(kv, walk.seq, bad);
            } else {
                const int slot = begins ? 1 : 0;
                if (mt == 0 && lane == 0) s_part[slot] = {walk.seq * kv.kv_heads + walk.head, ends, bad, 0};
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
        if (owed) bar_sync(slot_free(kg, owed - 1), kHandOver);  // every arrival has its wait
    } else {
        // ---- consumers of few pairs of fp32: products by the FMA pipes, 2 MP of them for every element that HBM brings
        const int mt = warp % MT, kg = warp / MT, m0 = mt * MP;
        const int box_shift = __ffs(box) - 1;
        auto row_at = [&](int r) { return (uint32_t) ((r >> box_shift) * (box * D * 4) + (r & (box - 1)) * 128); };
        const uint32_t block_at = (uint32_t) box * 128;  // a tile is [piece][column block][position]
        constexpr int kPer = D / 32;  // elements of the output of a lane, for each pair
        const uint32_t column = (uint32_t) (lane * kPer / 32) * block_at, in_block = (uint32_t) (lane * kPer % 32 * 4);
        float (*weights)[kTile] = s_weight[warp];
        int it = 0, unit = 0, owed = 0;
        int64_t now = begin;
        bool more = begin < end, entered = false;
        while (more) {
            if (entered) {
                walk.next(g);
                now = walk.at;
                unit++;
            }
            entered = true;
            more = walk.more(g);
            const auto span = span_of<kTile>(g, walk.q);
            const int t0 = walk.first_tile(g, now), t1 = walk.last_tile(g);
            const int mine = min(walk.q.n * g.group - m0, MP);  // pairs of this warp
            const int p_first = walk.q.length - walk.q.n, p_last = walk.q.length - 1;
            auto position = [&](int m) { return p_first + (m0 + m) / g.group; };
            const bool fed = __all_sync(0xffffffffu, !dead() && mbar_wait(&query_full[unit & 1], (uint32_t) (unit / 2) & 1u));
            if (!fed && lane == 0) atomicOr(&s_dead, 1);
            const unsigned char * queries = query + (size_t) ((unit & 1) * pairs + m0) * kQueryPitch;
            float o[MP][kPer], top[MP], sum[MP];
            int bad = 0;
#pragma unroll
            for (int m = 0; m < MP; m++) {
                top[m] = -kInf, sum[m] = 0.0f;
#pragma unroll
                for (int d = 0; d < kPer; d++) o[m][d] = 0.0f;
            }
            const int it_after = it + t1 - t0;
            for (int t = t0; t < t1; t++, it++) {
                if (it % kGroups != kg) continue;
                const int s = it % stages;
                const bool ok = !dead() && mbar_wait(&full[s], (uint32_t) (it / stages) & 1u);
                if (!__all_sync(0xffffffffu, ok)) {
                    if (lane == 0) atomicOr(&s_dead, 1);
                    break;
                }
                bad |= *reinterpret_cast<volatile int *>(&s_refused[s]);
                const unsigned char * keys = smem + (size_t) s * stage_bytes<D>(), * values = keys + kTile * D * 4;
                // scores: a lane per position
                float x[MP];
#pragma unroll
                for (int m = 0; m < MP; m++) x[m] = 0.0f;
                const unsigned char * key = keys + row_at(lane);
#pragma unroll 1
                for (int block = 0; block < D / 32; block++) {
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        const float4 k = *reinterpret_cast<const float4 *>(key + block * block_at + ((c ^ (lane & 7)) * 16));
#pragma unroll
                        for (int m = 0; m < MP; m++) {
                            if (MP > 2 && m >= mine) break;
                            const float4 y = *reinterpret_cast<const float4 *>(queries + m * kQueryPitch + block * 128 + c * 16);
                            x[m] += k.x * y.x + k.y * y.y + k.z * y.z + k.w * y.w;
                        }
                    }
                }
                const int base = span.base(t), p = base + lane;
                const bool whole = base + kTile - 1 <= p_first && (g.window == 0 || base > p_last - g.window || base + kTile - 1 < g.sinks);
#pragma unroll
                for (int m = 0; m < MP; m++) {
                    if (m >= mine) break;
                    const bool hidden = !whole && !(span.seen(p) && sees(position(m), p, g.window, g.sinks));
                    x[m] = hidden ? -kInf : x[m] * g.scale_log2;
                    float most = x[m];
#pragma unroll
                    for (int i = 16; i > 0; i /= 2) most = fmaxf(most, shfl_xor(most, i));
                    most = fmaxf(top[m], most);
                    const float ref = most == -kInf ? 0.0f : most;
                    if (most != top[m]) {
                        const float a = ex2(top[m] - ref);
                        top[m] = most;
                        sum[m] *= a;
#pragma unroll
                        for (int d = 0; d < kPer; d++) o[m][d] *= a;
                    }
                    const float w = hidden ? 0.0f : ex2(x[m] - ref);
                    sum[m] += w;  // this lane's positions
                    weights[m][lane] = hidden ? -1.0f : w;
                }
                __syncwarp();
                // values: a lane per kPer elements. A weight below 0 is a position that the row does not see: whatever
                // lies there, NaN included, stays out.
                for (int j = 0; j < kTile; j += 4) {
                    float v[4][kPer];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const unsigned char * at = values + row_at(j + i) + column + (((in_block / 16) ^ ((j + i) & 7)) * 16 + in_block % 16);
                        if (kPer == 4) *reinterpret_cast<float4 *>(v[i]) = *reinterpret_cast<const float4 *>(at);
                        else *reinterpret_cast<float2 *>(v[i]) = *reinterpret_cast<const float2 *>(at);
                    }
#pragma unroll
                    for (int m = 0; m < MP; m++) {
                        if (m >= mine) break;
                        const float4 w = *reinterpret_cast<const float4 *>(&weights[m][j]);
                        const float ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (whole || ws[i] >= 0.0f) {
#pragma unroll
                                for (int d = 0; d < kPer; d++) o[m][d] += ws[i] * v[i][d];
                            }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
            it = it_after;
            if (lane == 0) mbar_arrive(&query_empty[unit & 1]);
#pragma unroll
            for (int m = 0; m < MP; m++) {
                if (m >= mine) break;
#pragma unroll
                for (int i = 16; i > 0; i /= 2) sum[m] += shfl_xor(sum[m], i);
            }
            const int joiner = (it - 1) % kGroups, others = min(t1 - t0, kGroups) - 1;
            const int behind = (joiner - kg + kGroups) % kGroups;
            if (behind > others) continue;
            if (behind > 0) {  // hands over, as above
                if (owed) bar_sync(slot_free(kg, owed - 1), kHandOver);
                owed = joiner + 1;
#pragma unroll
                for (int m = 0; m < MP; m++) {
                    if (m >= mine) break;
                    if (lane == 0) stat[kg][m0 + m] = make_float2(top[m], sum[m]);
                    float * slot = room + (size_t) (kg * pairs + m0 + m) * kPitch + lane * kPer;
#pragma unroll
                    for (int d = 0; d < kPer; d++) slot[d] = o[m][d];
                }
                if (mt == 0 && lane == 0) s_bad[kg] = bad;
                bar_arrive(slot_full(kg, joiner), kHandOver);
                continue;
            }
            for (int i = 1; i <= others; i++) {
                const int from = (joiner - i + kGroups) % kGroups;
                bar_sync(slot_full(from, joiner), kHandOver);
                bad |= *reinterpret_cast<volatile int *>(&s_bad[from]);
#pragma unroll
                for (int m = 0; m < MP; m++) {
                    if (m >= mine) break;
                    const float2 other = stat[from][m0 + m];
                    const float most = fmaxf(top[m], other.x), ref = most == -kInf ? 0.0f : most;
                    const float a = ex2(top[m] - ref), b = ex2(other.x - ref);
                    top[m] = most;
                    sum[m] = sum[m] * a + other.y * b;
                    const float * slot = room + (size_t) (from * pairs + m0 + m) * kPitch + lane * kPer;
#pragma unroll
                    for (int d = 0; d < kPer; d++) o[m][d] = o[m][d] * a + slot[d] * b;
                }
                bar_arrive(slot_free(from, joiner), kHandOver);
            }
            const bool begins = t0 == 0, ends = t1 == walk.tiles, entire = begins && ends;
            const int slot = begins ? 1 : 0;
            float * data = part_data(g, me, slot, pairs);
#pragma unroll
            for (int m = 0; m < MP; m++) {
                if (m >= mine) break;
                if (entire) {
                    const int64_t out_row = walk.q.start + (m0 + m) / g.group;
                    const int h = walk.head * g.group + (m0 + m) % g.group;
                    const bool blank = bad || position(m) < 0;
                    const float inv = 1.0f / sum[m];
#pragma unroll
                    for (int d = 0; d < kPer; d += 2)
                        store_pair<T>(g, out_row, h, lane * kPer + d, blank ? 0.0f : o[m][d] * inv, blank ? 0.0f : o[m][d + 1] * inv);
                    if (g.lse && lane == 0)
                        g.lse[out_row * g.q_heads + h] = blank ? -kInf : (top[m] == -kInf ? 0.0f : top[m]) * kLn2 + logf(sum[m]);
                } else {
                    if (lane == 0) *reinterpret_cast<float2 *>(data + 2 * (m0 + m)) = make_float2(top[m], sum[m]);
#pragma unroll
                    for (int d = 0; d < kPer; d++) data[2 * pairs + (m0 + m) * D + lane * kPer + d] = o[m][d];
                }
            }
            if (mt == 0 && lane == 0) {
                if (entire) raise_status(kv, walk.seq, bad);
                else s_part[slot] = {walk.seq * kv.kv_heads + walk.head, ends, bad, 0};
            }
        }
        if (owed) bar_sync(slot_free(kg, owed - 1), kHandOver);  // every arrival has its wait
    }
    __syncthreads();
    if (s_dead) {
        // A wait gave up, here or there, for one warp of a unit or for all: the share is lost as a whole. What ended in it is NaN,
        // what it was a part of is for the join. (To carry this along with the units, warp by warp, cost 20 pairs of bf16 2 us of 57.)
        if (tid < 2 && s_part[tid].unit >= 0) s_part[tid].bad |= 2;
        walk.start(g, s_seq, s_numbers, s_at, s_begin, s_end);
        for (int64_t now = s_begin;; now = walk.at) {
            if (walk.first_tile(g, now) == 0 && walk.last_tile(g) == walk.tiles) {
                const int rows = walk.q.n * g.group;
                for (int e = tid; e < rows * (D / 2); e += kThreads) {
                    const int m = e / (D / 2);
                    store_pair<T>(g, walk.q.start + m / g.group, walk.head * g.group + m % g.group, e % (D / 2) * 2, refused_value(2), refused_value(2));
                }
                if (g.lse)
                    for (int m = tid; m < rows; m += kThreads) g.lse[(int64_t) (walk.q.start + m / g.group) * g.q_heads + walk.head * g.group + m % g.group] = -kInf;
                if (tid == 0) raise_status(kv, walk.seq, 2);
            }
            if (!walk.more(g)) break;
            walk.next(g);
        }
    }
    if (tid < 2) *part_head(g, me, tid) = s_part[tid];
    if (s_idle) {  // sequences with nothing to read: idle or refused rows, or none
        for (int s = me; s < kv.seqs; s += (int) gridDim.x) {
            const Sequence q = sequence(kv, s);
            if (tiles_of<kTile>(g, q) > 0) continue;
            for (int64_t e = tid; e < (int64_t) q.n * g.q_heads * (D / 2); e += kThreads) {
                const int64_t pair = e / (D / 2);
                store_pair<T>(g, q.start + pair / g.q_heads, (int) (pair % g.q_heads), (int) (e % (D / 2)) * 2, 0.0f, 0.0f);
            }
            if (g.lse)
                for (int64_t e = tid; e < (int64_t) q.n * g.q_heads; e += kThreads) g.lse[q.start * (int64_t) g.q_heads + e] = -kInf;
            if (tid == 0) raise_status(kv, s, q.ok ? 0 : 1);
        }
    }
    statuses_cleared();
}

// Joins the partials of the unit that begins in share `blockIdx.x` and ends in a later one: those of the
// following shares' slot 0, up to the one that says it ends. A block takes 8 pairs, a warp one of them, or several
// warps where there are fewer (a block of 256 threads for pair after pair took 27 us longer for 20 pairs).
constexpr int kJoinWarps = 8;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ AttendArgs g, int pairs) {
    constexpr int kPer = D / 32;  // elements of a lane
    __shared__ float s_out[kJoinWarps][D];
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the shares are written
    const int share = (int) blockIdx.x, warp = warp_id(), lane = lane_id();
    const PartHead head = *part_head(g, share, 1);
    if (head.unit < 0) return;
    const KvArgs & kv = g.kv;
    const int seq = head.unit / kv.kv_heads, kv_head = head.unit % kv.kv_heads;
    const Sequence q = sequence(kv, seq);
    int bad = head.bad, last = g.max_shares - 1;  // the share the unit ends in: the first of the following that says so
    for (int i = share + 1; i < g.max_shares; i += 32) {
        PartHead next{-1, 0, 0, 0};
        if (i + lane < g.max_shares) next = *part_head(g, i + lane, 0);
        const uint32_t ends = __ballot_sync(0xffffffffu, next.unit == head.unit && next.ends);
        const int stop = ends ? __ffs(ends) - 1 : 31;
        if (lane <= stop && next.unit == head.unit) bad |= next.bad;
        if (ends) {
            last = i + stop;
            break;
        }
    }
    bad = __reduce_or_sync(0xffffffffu, bad);
    const int parts = last - share + 1, rows = q.n * g.group;
    const int m0 = (int) blockIdx.y * kJoinWarps, here = min(rows - m0, kJoinWarps);
    const int sharing = here <= 1 ? 8 : here <= 2 ? 4 : here <= 4 ? 2 : 1;  // warps of a pair
    const int m = m0 + warp / sharing, mine = warp % sharing;
    const bool on = m < rows;
    auto data = [&](int i) { return part_data(g, share + i, i == 0, pairs); };
    float top = -kInf, sum = 0.0f, o[kPer] = {};
    if (on) {
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, data(i)[2 * m]);
#pragma unroll
        for (int x = 16; x > 0; x /= 2) top = fmaxf(top, shfl_xor(top, x));
        const float ref = top == -kInf ? 0.0f : top;
        for (int i = lane; i < parts; i += 32) {
            const float2 s = *reinterpret_cast<const float2 *>(data(i) + 2 * m);
            sum += s.y * ex2(s.x - ref);
        }
#pragma unroll
        for (int x = 16; x > 0; x /= 2) sum += shfl_xor(sum, x);
#pragma unroll 8
        for (int i = mine; i < parts; i += sharing) {
            const float * from = data(i);
            const float w = ex2(from[2 * m] - ref);
            float x[kPer];
            if (kPer == 4) *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(from + 2 * pairs + m * D + lane * kPer);
            else *reinterpret_cast<float2 *>(x) = *reinterpret_cast<const float2 *>(from + 2 * pairs + m * D + lane * kPer);
#pragma unroll
            for (int e = 0; e < kPer; e++) o[e] += x[e] * w;
        }
        if (mine > 0) {
#pragma unroll
            for (int e = 0; e < kPer; e++) s_out[warp][lane * kPer + e] = o[e];
        }
    }
    __syncthreads();
    if (on && mine == 0) {
        for (int w = 1; w < sharing; w++) {
#pragma unroll
            for (int e = 0; e < kPer; e++) o[e] += s_out[warp + w][lane * kPer + e];
        }
        const bool blank = bad || q.length - q.n + m / g.group < 0;
        const float inv = 1.0f / sum, fill = refused_value(bad);
        const int64_t out_row = q.start + m / g.group;
        const int h = kv_head * g.group + m % g.group;
#pragma unroll
        for (int e = 0; e < kPer; e += 2)
            store_pair<T>(g, out_row, h, lane * kPer + e, blank ? fill : o[e] * inv, blank ? fill : o[e + 1] * inv);
        if (g.lse && lane == 0) g.lse[out_row * g.q_heads + h] = blank ? -kInf : (top == -kInf ? 0.0f : top) * kLn2 + logf(sum);
    }
    if (threadIdx.x == 0 && blockIdx.y == 0) raise_status(kv, seq, bad);
}

// (row, query head) pairs of one key head. More take the prompt kernel: with eight blocks of 16 pairs on a tile, 64 rows of
// 2 query heads per key head took 48 us on 8 streams of up to 2000 positions, where the prompt kernel takes 27.
constexpr int kMaxPairs = 64;

template <typename T, int D, int MT, int MP>
cudaError_t launch(AttendArgs a, int sm_count, cudaStream_t stream) {
    constexpr int kTile = tile_of<T>();
    CUtensorMap maps[2];
    const int box = a.kv.page_size < kTile ? a.kv.page_size : kTile;
    if (!page_maps(maps, a.kv, D, box, D * (int) sizeof(T) / 128, sizeof(T))) return cudaErrorInvalidValue;
    // as many CTAs as the SMs hold at once: two where a ring of a tile per group fits twice, else one with a
    // ring as long as fits
    int pairs = (a.kv.max_rows * a.group + 1) / 2 * 2;  // even: the partials' vectors stay aligned
    constexpr int G = groups<T, D, MT, MP>();
    const size_t query = (size_t) 2 * pairs * (D * sizeof(T) + 16), slots = (size_t) G * pairs * (D + 8) * sizeof(float);
    // a product that reads 16 rows from the last query's must end within the shared memory
    const size_t room = std::max(query + slots, (size_t) (pairs + 16 * MT) * (D * sizeof(T) + 16)) + 1024;
    constexpr size_t weights = by_tensor_cores<T, MP>() ? 0 : (size_t) G * MT * MP * kTile * 4;
    auto ring = [&](size_t budget) {
        const int n = (int) ((budget * 1024 - 2048 - weights - room) / stage_bytes<D>());  // less the static shared memory
        return (n < kMaxStages ? n : kMaxStages) / G * G;
    };
    const int per_sm = MT <= 2 && ring(113) >= G ? 2 : 1;
    int stages = ring(per_sm == 2 ? 113 : 226);
    const size_t smem = (size_t) stages * stage_bytes<D>() + room;
    // no more shares than the longest sequences could fill
    const int64_t reach = a.window > 0 ? std::min<int64_t>(a.kv.max_length, (int64_t) a.window + a.sinks + a.kv.max_rows + 2 * kTile) : a.kv.max_length;
    const int64_t longest = (reach + kTile - 1) / kTile, units = (int64_t) a.kv.kv_heads * a.kv.seqs;
    a.whole_units = longest <= kWholeTiles;
    const int64_t most = a.whole_units ? units : units * ((longest + kMinTiles - 1) / kMinTiles);
    const int shares = (int) std::min<int64_t>(per_sm * sm_count, most);
    a.max_shares = shares;
    const void * kernel = (const void *) step_kernel<T, D, MT, MP>;
    cudaError_t e = set_max_dynamic_smem(kernel, smem);
    if (e != cudaSuccess) return e;
    void * params[] = {&maps[0], &maps[1], &a, &stages, &pairs};
    e = launch_cluster(kernel, (unsigned) shares, 1, step_threads<T, D, MT, MP>(), smem, stream, params, &a.kv);
    if (e != cudaSuccess || shares == 1 || a.whole_units) return e;  // nothing is split
    // launched while the shares still run, and waiting for them on the device
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned) shares, (unsigned) (pairs + kJoinWarps - 1) / kJoinWarps);
    config.blockDim = dim3(kJoinWarps * 32);
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, join_kernel<T, D>, a, pairs);
}

template <int D> cudaError_t launch(const AttendArgs & a, bool bf16, int sm_count, cudaStream_t stream) {
    using B = __nv_bfloat16;
    const int64_t pairs = (int64_t) a.kv.max_rows * a.group;
    if (bf16 && pairs <= 10) return launch<B, D, 1, 10>(a, sm_count, stream);
    if (bf16) return pairs <= 16 ? launch<B, D, 1, 16>(a, sm_count, stream) : pairs <= 32 ? launch<B, D, 2, 16>(a, sm_count, stream) : launch<B, D, 4, 16>(a, sm_count, stream);
    if (pairs <= 4) return pairs <= 2 ? launch<float, D, 1, 2>(a, sm_count, stream) : launch<float, D, 1, 4>(a, sm_count, stream);
    return pairs <= 16 ? launch<float, D, 1, 16>(a, sm_count, stream) : pairs <= 32 ? launch<float, D, 2, 16>(a, sm_count, stream) : launch<float, D, 4, 16>(a, sm_count, stream);
}

}  // namespace

bool attend_step_takes(const AttendArgs & a, bool bf16) {
    return (int64_t) a.kv.max_rows * a.group <= kMaxPairs && tma_takes(a, bf16 ? 2 : 4);
}

// Two slots of every share: at most 2 CTAs per SM of 32 pairs, or 1 of 64.
int64_t attend_workspace_bytes(int sm_count) {
    return (int64_t) sm_count * (2 * 2 * sizeof(PartHead) + 2 * kMaxPairs * (128 + 2) * sizeof(float));
}

cudaError_t launch_attend_step(const AttendArgs & a, bool bf16, int sm_count, cudaStream_t stream) {
    return a.kv.head_dim == 64 ? launch<64>(a, bf16, sm_count, stream) : launch<128>(a, bf16, sm_count, stream);
}

}  // namespace ssb

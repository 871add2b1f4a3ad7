// Attention of a few rows per sequence over a paged bf16 cache (head size 64 or 128): the step of one new
// token, and drafts to verify, up to 64 (row, query head) pairs per key head.
//
//   out = sum_j softmax_j(scale * q . k[j]) v[j] over the positions j that the row sees
//
// Every key and value is read once from HBM and used for all pairs of its head: 2 to 64 multiply-adds per
// element, so the bound is HBM and the tensor work only has to keep up with it. The pairs are far fewer than the
// 128 rows of a tcgen05 tile, so the products are warp-level mma.m16n8k16 with the pairs as the 16 rows and the
// accumulators in registers. A producer warp keeps a ring of 64-position tiles in flight with TMA copies out
// of the pages (128-byte swizzle, no multicast); four warps per 16 pairs take 16 positions of a tile each,
// with a running maximum and sum of their own. At the end the four are joined through shared memory, and
// the CTAs of a cluster, which share the tiles of one (sequence, key head), through distributed shared memory.
// Every mbarrier wait is bounded: one that gives up ends the kernel with SSB_ROW_DEVICE_TIMEOUT.
#include "ssb_decoder.cuh"
#include "ssb_tma.cuh"
#include "ssb_tma_map.cuh"

namespace ssb {

namespace {

namespace cg = cooperative_groups;

constexpr int kGroups = 4;       // warps that share a tile, 16 positions each
constexpr int kMaxStages = 8;
constexpr int kMaxRanks = 16;

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

template <int D, int MT>
__global__ void __launch_bounds__(step_threads<MT>(), MT == 1 ? 2 : 1)
    step_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ AttendArgs g, int stages) {
    constexpr int kHalves = D / 64, kPairs = 16 * MT, kPitch = D + 8;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char * smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
    __shared__ float2 stat[2][kPairs];
    __shared__ float share[kMaxRanks * kPairs];
    __shared__ int s_bad;  // 1: a page outside the pool, 2: a wait gave up
    const KvArgs & kv = g.kv;
    auto cluster = cg::this_cluster();
    const int ranks = (int) cluster.num_blocks(), rank = (int) cluster.block_rank();
    const int unit = (int) (blockIdx.x / (unsigned) ranks);
    const int head = unit % kv.kv_heads, seq = unit / kv.kv_heads;
    const int tid = (int) threadIdx.x, warp = warp_id(), lane = lane_id();
    const Sequence q = sequence(kv, seq);
    const bool reports = kv.status && head == 0 && rank == 0 && tid == 0;
    const int rows = q.n * g.group;
    if (rows == 0) {
        if (reports) kv.status[seq] = q.ok ? SSB_ROW_OK : SSB_ROW_INVALID_ROW;
        return;
    }
    const int first = q.length - q.n;
    const Span span = span_of(first, q.length - 1, g.window, g.sinks);
    const int tiles = q.ok ? span.tiles : 0;
    const int t0 = (int) ((int64_t) tiles * rank / ranks), t1 = (int) ((int64_t) tiles * (rank + 1) / ranks);
    if (tid == 0) {
        for (int s = 0; s < stages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], kGroups * MT);
        s_bad = q.ok ? 0 : 1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    auto gave_up = [&]() { return (*reinterpret_cast<volatile int *>(&s_bad) & 2) != 0; };
    const int box = kv.page_size < kTile ? kv.page_size : kTile;  // positions of one TMA copy: a piece of a tile

    float o[D / 8][4];
    float top[2] = {-kInf, -kInf}, sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    const int mt = warp % MT, kg = warp / MT;
    const int r0 = mt * 16 + lane / 4;  // this thread's pairs: r0 and r0 + 8

    if (warp == kGroups * MT) {
        // ---- producer: lane l looks up and copies piece l of every 32
        const int per_tile = kTile / box;
        const int32_t * table = kv.table + (int64_t) seq * kv.table_ld;
        int last_use[kMaxStages];
#pragma unroll
        for (int s = 0; s < kMaxStages; s++) last_use[s] = -1;
        for (int t = t0; t < t1 && !gave_up(); t += 32 / per_tile) {
            const int mine = t + lane / per_tile;
            const int at = span.base(mine) + lane % per_tile * box;
            // only pieces that hold a seen position: the table's other entries may be anything
            const bool wanted = mine < t1 && at < span.hi && (at + box > span.first || at < span.sinks);
            const int page = wanted ? table[at >> kv.page_shift] : 0;
            const bool valid = wanted && (unsigned) page < (unsigned) kv.pages;
            if (wanted && !valid) atomicOr(&s_bad, 1);
            const uint32_t votes = __ballot_sync(0xffffffffu, valid);
            const int end = min(t1, t + 32 / per_tile);
            for (int u = t; u < end; u++) {
                const int it = u - t0, s = it % stages;
                const bool ready = it < stages || mbar_wait(&empty[s], (uint32_t) (it / stages - 1) & 1u);
                if (!__all_sync(0xffffffffu, ready)) {
                    if (lane == 0) atomicOr(&s_bad, 2);
                    break;
                }
                const uint32_t of_tile = (per_tile == 1 ? 1u : (1u << per_tile) - 1u) << ((u - t) * per_tile);
                if (lane == 0) mbar_expect(&full[s], (uint32_t) (__popc(votes & of_tile) * 2 * box * D * 2));
                __syncwarp();
                if (valid && mine == u) {
                    unsigned char * dst = smem + (size_t) s * stage_bytes<D>() + lane % per_tile * box * D * 2;
                    const int slot = at & (kv.page_size - 1);
                    tma_load_5d(dst, &map_k, 0, slot, 0, head, page, &full[s]);
                    tma_load_5d(dst + kTile * D * 2, &map_v, 0, slot, 0, head, page, &full[s]);
                }
#pragma unroll
                for (int i = 0; i < kMaxStages; i++)
                    if (i == s) last_use[i] = it / stages;
            }
        }
        __syncwarp();
        if (gave_up()) {  // let the copies in flight land before the shared memory is given up
#pragma unroll
            for (int s = 0; s < kMaxStages; s++)
                if (last_use[s] >= 0) mbar_wait(&full[s], (uint32_t) last_use[s] & 1u);
        }
    } else {
        // ---- consumers. The pairs of this warp's 16 rows as the A operand, for all of the head.
        uint32_t qa[D / 16][4];
        int position[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int m = r0 + 8 * i;
            position[i] = first + (m < rows ? m : rows - 1) / g.group;
            const __nv_bfloat16 * src = static_cast<const __nv_bfloat16 *>(g.q) + (int64_t) (q.start + m / g.group) * g.q_ld +
                                        (int64_t) (head * g.group + m % g.group) * D + lane % 4 * 2;
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++) {
                qa[ks][i] = m < rows ? *reinterpret_cast<const uint32_t *>(src + ks * 16) : 0u;
                qa[ks][2 + i] = m < rows ? *reinterpret_cast<const uint32_t *>(src + ks * 16 + 8) : 0u;
            }
        }
        const int p_first = first, p_last = q.length - 1;
        // this warp's 16 positions within a tile: their rows in the tile's [piece][half][position] layout
        const int row = kg * 16;
        const uint32_t row_at = (uint32_t) (row / box * (box * D * 2) + row % box * 128);
        const uint32_t half_at = (uint32_t) box * 128;
        const int k_row = (lane & 7) + (lane >> 4) * 8, k_chunk = lane >> 3 & 1;
        const int v_row = (lane & 7) + (lane >> 3 & 1) * 8, v_chunk = lane >> 4;
        for (int t = t0; t < t1; t++) {
            const int it = t - t0, s = it % stages;
            bool ok = mbar_wait(&full[s], (uint32_t) (it / stages) & 1u);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok || gave_up()) {
                if (lane == 0) atomicOr(&s_bad, 2);
                break;
            }
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
    }
    __syncthreads();
    // the four warps of a row block joined: 2 and 3 into 0 and 1, then 1 into 0
    float * room = reinterpret_cast<float *>(smem);  // two slots of [kPairs][kPitch], over the ring
#pragma unroll
    for (int half = kGroups / 2; half >= 1; half /= 2) {
        if (kg >= half && kg < 2 * half && warp < kGroups * MT) {
            float * slot = room + (size_t) (kg - half) * kPairs * kPitch;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int m = r0 + 8 * i;
                if (m >= rows) continue;
                if (lane % 4 == 0) stat[kg - half][m] = make_float2(top[i], sum[i]);
#pragma unroll
                for (int n = 0; n < D / 8; n++)
                    *reinterpret_cast<float2 *>(slot + m * kPitch + n * 8 + lane % 4 * 2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            }
        }
        __syncthreads();
        if (kg < half) {
            const float * slot = room + (size_t) kg * kPairs * kPitch;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int m = r0 + 8 * i;
                if (m >= rows) continue;
                const float2 other = stat[kg][m];
                const float t = fmaxf(top[i], other.x), ref = t == -kInf ? 0.0f : t;
                const float a = ex2(top[i] - ref), b = ex2(other.x - ref);
                top[i] = t;
                sum[i] = sum[i] * a + other.y * b;
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    const float2 x = *reinterpret_cast<const float2 *>(slot + m * kPitch + n * 8 + lane % 4 * 2);
                    o[n][2 * i] = o[n][2 * i] * a + x.x * b, o[n][2 * i + 1] = o[n][2 * i + 1] * a + x.y * b;
                }
            }
        }
        __syncthreads();
    }
    if (kg == 0) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int m = r0 + 8 * i;
            if (m >= rows) continue;
            if (lane % 4 == 0) stat[0][m] = make_float2(top[i], sum[i]);
#pragma unroll
            for (int n = 0; n < D / 8; n++)
                *reinterpret_cast<float2 *>(room + m * kPitch + n * 8 + lane % 4 * 2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
    }
    const Partial partial{room, kPitch, stat[0], share, &s_bad};
    const int refused = join_cluster(
        partial, rows, D,
        [&](int m, int c, float4 x) {
            if (first + m / g.group < 0) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            store4(static_cast<__nv_bfloat16 *>(g.out) + (int64_t) (q.start + m / g.group) * g.out_ld +
                       (int64_t) (head * g.group + m % g.group) * D + c, x, g.vec_out);
        },
        [&](int m, float lse) {
            if (g.lse) g.lse[(int64_t) (q.start + m / g.group) * g.q_heads + head * g.group + m % g.group] = first + m / g.group < 0 ? -kInf : lse;
        });
    if (reports) kv.status[seq] = refused == 0 ? SSB_ROW_OK : (refused & 2 ? SSB_ROW_DEVICE_TIMEOUT : SSB_ROW_INVALID_ROW);
}

template <int D, int MT>
cudaError_t launch(const AttendArgs & a, int sm_count, cudaStream_t stream) {
    CUtensorMap maps[2];
    if (!page_map(&maps[0], a.kv.k, a.kv, D, min(a.kv.page_size, kTile)) || !page_map(&maps[1], a.kv.v, a.kv, D, min(a.kv.page_size, kTile)))
        return cudaErrorInvalidValue;
    const void * kernel = (const void *) step_kernel<D, MT>;
    // tiles of the longest sequence, and how many CTAs share them: enough to cover the SMs twice where there
    // are tiles for it, and no CTA with more than 16 tiles while others would be done (lengths are ragged)
    const int tiles = (int) (((int64_t) (a.window > 0 ? min(a.kv.max_length, a.window + a.sinks + a.kv.max_rows + kTile) : a.kv.max_length) + kTile - 1) / kTile);
    const int64_t units = (int64_t) a.kv.kv_heads * a.kv.seqs;
    int split = 1;
    while (split < kMaxRanks && ((units * split < sm_count && split * 2 <= tiles) || tiles > 16 * split)) split *= 2;
    const int stages = units * split <= sm_count ? 6 : 3;
    const size_t smem = (size_t) stages * stage_bytes<D>() + 1024;
    cudaError_t e = set_max_dynamic_smem(kernel, smem);
    if (e == cudaSuccess && split > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    if (units * split > INT32_MAX) return cudaErrorInvalidValue;
    AttendArgs args = a;
    int st = stages;
    void * params[] = {&maps[0], &maps[1], &args, &st};
    return launch_cluster(kernel, (unsigned) (units * split), split, step_threads<MT>(), smem, stream, params);
}

template <int D> cudaError_t launch(const AttendArgs & a, int sm_count, cudaStream_t stream) {
    const int64_t pairs = (int64_t) a.kv.max_rows * a.group;
    return pairs <= 16 ? launch<D, 1>(a, sm_count, stream) : pairs <= 32 ? launch<D, 2>(a, sm_count, stream) : launch<D, 4>(a, sm_count, stream);
}

}  // namespace

bool attend_step_takes(const AttendArgs & a) {
    return (int64_t) a.kv.max_rows * a.group <= 64 && tensor_core_takes(a);
}

cudaError_t launch_attend_step(const AttendArgs & a, int sm_count, cudaStream_t stream) {
    return a.kv.head_dim == 64 ? launch<64>(a, sm_count, stream) : launch<128>(a, sm_count, stream);
}

}  // namespace ssb

// Attention over the paged cache for any type, head size (to 256) and alignment: the kernel of fp32 prompts and of the
// head sizes and alignments that the step and prompt kernels do not take.
//
//   out = sum_j softmax_j(scale * q . k[j]) v[j] over the positions j that the row sees
//
// A row block is up to kRows (row, query head) pairs that read one key head, so each key and value is loaded
// once for all of them. A CTA walks tiles of 64 positions with a running maximum and sum per row; the CTAs of
// a cluster take consecutive shares of the tiles and join their partials through distributed shared memory,
// in rank order (no scratch, no atomics: equal calls give equal bits). Scores: four threads per position, a
// quarter of the head each. Values: one thread per element of the head, for all rows. The loads are not ahead of
// the arithmetic, whose shared-memory reads bound it: 8 ragged prompts of up to 6000 bf16 rows take it 114 ms
// (9 TFLOP/s), one stream at 120001 bf16 positions 1.9 ms.
#include "ssb_decoder.cuh"

namespace ssb {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kRows = 16;

// Shared memory, in floats: the key tile's rows are padded to D + 16 so that the quarters which eight threads
// read at once fall into different banks.
template <int D> struct Layout {
    static constexpr int kPitch = D + 16;
    static constexpr int kKey = 0;
    static constexpr int kValue = kKey + kTile * kPitch;
    static constexpr int kQuery = kValue + kTile * D;
    static constexpr int kWeight = kQuery + kRows * kPitch;
    static constexpr int kStat = kWeight + kRows * kTile;  // float2 per row
    static constexpr int kAlpha = kStat + 2 * kRows;
    static constexpr int kShare = kAlpha + kRows;          // [16 ranks][kRows]
    static constexpr int kFloats = kShare + 16 * kRows;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attend_kernel(const __grid_constant__ AttendArgs g, int row_blocks) {
    using L = Layout<D>;
    extern __shared__ __align__(16) float smem[];
    __shared__ int s_bad;
    const KvArgs & kv = g.kv;
    auto cluster = cg::this_cluster();
    const int ranks = (int) cluster.num_blocks(), rank = (int) cluster.block_rank();
    const int unit = (int) (blockIdx.x / (unsigned) ranks);
    const int block = unit % row_blocks, head = unit / row_blocks % kv.kv_heads, seq = unit / row_blocks / kv.kv_heads;
    const int tid = (int) threadIdx.x, warp = warp_id(), lane = lane_id();
    const bool reports = kv.status && block == 0 && head == 0 && rank == 0 && tid == 0;
    const Sequence q = sequence(kv, seq);
    const int pairs = q.n * g.group;  // (row, query head) pairs of this key head
    const int m0 = block * kRows;
    // the whole sequence is refused for a bad page that any of its rows sees, whichever block meets it
    bool ok = q.ok;
    if (ok && q.n > 0) ok = pages_ok(kv, seq, span_of(q.length - q.n, q.length - 1, g.window, g.sinks));
    if (reports) kv.status[seq] = ok ? SSB_ROW_OK : SSB_ROW_INVALID_ROW;
    if (m0 >= pairs) return;
    const int rows = min(kRows, pairs - m0), dim = kv.head_dim;
    const int first = q.length - q.n;  // the position of the sequence's first row
    const Span span = span_of(first + m0 / g.group, first + (m0 + rows - 1) / g.group, g.window, g.sinks);
    const int tiles = ok ? span.tiles : 0;

    float * keys = smem + L::kKey, * values = smem + L::kValue, * query = smem + L::kQuery, * weight = smem + L::kWeight;
    float2 * stat = reinterpret_cast<float2 *>(smem + L::kStat);
    float * alpha = smem + L::kAlpha;
    auto row_of = [&](int m) { return q.start + (m0 + m) / g.group; };
    auto head_of = [&](int m) { return head * g.group + (m0 + m) % g.group; };
    auto position_of = [&](int m) { return first + (m0 + m) / g.group; };

    for (int e = tid; e < kRows * (D / 4); e += kThreads) {
        const int m = e / (D / 4), c = e % (D / 4) * 4;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (m < rows && c < dim) {
            x = load4(static_cast<const T *>(g.q) + (int64_t) row_of(m) * g.q_ld + (int64_t) head_of(m) * dim + c, g.vec_q);
            x.x *= g.scale_log2, x.y *= g.scale_log2, x.z *= g.scale_log2, x.w *= g.scale_log2;
        }
        *reinterpret_cast<float4 *>(query + m * L::kPitch + c) = x;
    }
    if (tid < kRows) stat[tid] = make_float2(-kInf, 0.0f);
    if (tid == 0) s_bad = ok ? 0 : 1;

    constexpr int kParts = kThreads / D;  // parts of a tile's positions in the value product
    constexpr int kPart = kTile / kParts;
    const int vc = tid % D, vp = tid / D;
    float acc[kRows];
#pragma unroll
    for (int m = 0; m < kRows; m++) acc[m] = 0.0f;

    const int t0 = (int) ((int64_t) tiles * rank / ranks), t1 = (int) ((int64_t) tiles * (rank + 1) / ranks);
    for (int t = t0; t < t1; t++) {
        const int base = span.base(t);
        __syncthreads();
        for (int e = tid; e < kTile * (D / 4); e += kThreads) {
            const int j = e / (D / 4), c = e % (D / 4) * 4, p = base + j;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
            if (c < dim && span.seen(p)) {
                const int page = kv.table[(int64_t) seq * kv.table_ld + (p >> kv.page_shift)];
                const int64_t at = pool_offset(kv, page, p & (kv.page_size - 1), head) + c;
                x = load4(static_cast<const T *>(kv.k) + at, g.vec_cache);
                y = load4(static_cast<const T *>(kv.v) + at, g.vec_cache);
            }
            *reinterpret_cast<float4 *>(keys + j * L::kPitch + c) = x;
            *reinterpret_cast<float4 *>(values + j * D + c) = y;
        }
        __syncthreads();
        {  // scores: thread (position, quarter); a quarter is every fourth group of four elements
            const int j = tid / 4, part = tid % 4, p = base + j;
            float s[kRows];
#pragma unroll
            for (int m = 0; m < kRows; m++) s[m] = 0.0f;
            for (int c = part * 4; c < D; c += 16) {
                const float4 x = *reinterpret_cast<const float4 *>(keys + j * L::kPitch + c);
#pragma unroll
                for (int m = 0; m < kRows; m++) {
                    if (m >= rows) break;
                    const float4 y = *reinterpret_cast<const float4 *>(query + m * L::kPitch + c);
                    s[m] += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
                }
            }
#pragma unroll
            for (int m = 0; m < kRows; m++) {
                if (m >= rows) break;
                s[m] += shfl_xor(s[m], 1);
                s[m] += shfl_xor(s[m], 2);
                // a hidden position is told from one whose score is -inf by a weight below 0
                if (part == 0) weight[m * kTile + j] = span.seen(p) && sees(position_of(m), p, g.window, g.sinks) ? s[m] : -kInf;
            }
        }
        __syncthreads();
        for (int m = warp; m < rows; m += kThreads / 32) {
            const float2 old = stat[m];
            float x[2];
            bool hidden[2];
            float top = old.x;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int p = base + lane + 32 * i;
                x[i] = weight[m * kTile + lane + 32 * i];
                hidden[i] = !(span.seen(p) && sees(position_of(m), p, g.window, g.sinks));
                top = fmaxf(top, x[i]);
            }
#pragma unroll
            for (int o = 16; o > 0; o /= 2) top = fmaxf(top, shfl_xor(top, o));
            const float ref = top == -kInf ? 0.0f : top;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float w = hidden[i] ? 0.0f : exp2f(x[i] - ref);
                sum += w;
                weight[m * kTile + lane + 32 * i] = hidden[i] ? -1.0f : w;
            }
#pragma unroll
            for (int o = 16; o > 0; o /= 2) sum += shfl_xor(sum, o);
            if (lane == 0) {
                const float a = exp2f(old.x - ref);
                alpha[m] = a;
                stat[m] = make_float2(top, old.y * a + sum);
            }
        }
        __syncthreads();
        // values: thread (element, part of the positions). A weight below 0 is a position that the row does
        // not see: whatever lies there, NaN included, stays out.
#pragma unroll
        for (int m = 0; m < kRows; m++) {
            if (m >= rows) break;
            acc[m] *= alpha[m];
        }
        for (int j = vp * kPart; j < (vp + 1) * kPart; j += 4) {
            const float y0 = values[j * D + vc], y1 = values[(j + 1) * D + vc], y2 = values[(j + 2) * D + vc], y3 = values[(j + 3) * D + vc];
#pragma unroll
            for (int m = 0; m < kRows; m++) {
                if (m >= rows) break;
                const float4 w = *reinterpret_cast<const float4 *>(weight + m * kTile + j);
                if (w.x >= 0.0f) acc[m] += w.x * y0;
                if (w.y >= 0.0f) acc[m] += w.y * y1;
                if (w.z >= 0.0f) acc[m] += w.z * y2;
                if (w.w >= 0.0f) acc[m] += w.w * y3;
            }
        }
    }
    // the parts of each element added up in shared memory (over the key tile), then the cluster's join
    __syncthreads();
    float * out = keys;
#pragma unroll
    for (int part = 0; part < kParts; part++) {
        if (vp == part) {
#pragma unroll
            for (int m = 0; m < kRows; m++) {
                if (m >= rows) break;
                out[m * D + vc] = part == 0 ? acc[m] : out[m * D + vc] + acc[m];
            }
        }
        __syncthreads();
    }
    const Partial partial{out, D, stat, smem + L::kShare, &s_bad};
    join_cluster(
        partial, rows, dim,
        [&](int m, int c, float4 o) {
            if (position_of(m) < 0) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            store4(static_cast<T *>(g.out) + (int64_t) row_of(m) * g.out_ld + (int64_t) head_of(m) * dim + c, o, g.vec_out);
        },
        [&](int m, float lse) {
            if (g.lse) g.lse[(int64_t) row_of(m) * g.q_heads + head_of(m)] = position_of(m) < 0 ? -kInf : lse;
        });
}

template <typename T, int D>
cudaError_t launch(const AttendArgs & a, int sm_count, cudaStream_t stream) {
    const void * kernel = (const void *) attend_kernel<T, D>;
    const size_t smem = Layout<D>::kFloats * sizeof(float);
    cudaError_t e = set_max_dynamic_smem(kernel, smem);
    if (e != cudaSuccess) return e;
    const int row_blocks = (int) (((int64_t) a.kv.max_rows * a.group + kRows - 1) / kRows);
    const int64_t units = (int64_t) row_blocks * a.kv.kv_heads * a.kv.seqs;
    int split = 1;
    while (split < 8 && split * 4 * kTile < a.kv.max_length && units * split < 4 * sm_count) split *= 2;
    if (units * split > INT32_MAX) return cudaErrorInvalidValue;
    AttendArgs args = a;
    int blocks = row_blocks;
    void * params[] = {&args, &blocks};
    return launch_cluster(kernel, (unsigned) (units * split), split, kThreads, smem, stream, params);
}

}  // namespace

cudaError_t launch_attend(const AttendArgs & a, bool bf16, int sm_count, cudaStream_t stream) {
    using B = __nv_bfloat16;
    const int d = a.kv.head_dim;
    if (attend_step_takes(a, bf16)) return launch_attend_step(a, bf16, sm_count, stream);
    if (bf16 && attend_prompt_takes(a)) return launch_attend_prompt(a, sm_count, stream);
    if (bf16) return d <= 64 ? launch<B, 64>(a, sm_count, stream) : d <= 128 ? launch<B, 128>(a, sm_count, stream) : launch<B, 256>(a, sm_count, stream);
    return d <= 64 ? launch<float, 64>(a, sm_count, stream) : d <= 128 ? launch<float, 128>(a, sm_count, stream) : launch<float, 256>(a, sm_count, stream);
}

}  // namespace ssb

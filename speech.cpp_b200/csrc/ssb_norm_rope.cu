// Query and key heads normed and rotated, keys and values appended to the paged cache, in one pass.
//
//   x' = x / sqrt(mean(x^2) + eps) * weight;   (a, b) -> (a cos t - b sin t, b cos t + a sin t)
//
// One CTA per row (and, for few rows, per part of its heads): the row's angles t = position * inv_freq[i] are
// reduced to [-pi, pi] in 64 bits, since at position 10^6 a product in 32 bits is off by up to 0.03, and
// their cosines and sines are left in shared memory for all heads. A head is held by `lanes` threads, each with
// four adjacent elements a and the four elements b they pair with, so the norm is one shuffle reduction and
// the rotation needs no exchange. Every element is read once and written once: the bound is HBM, and for a
// row or two the latency of row_start -> length -> table -> store. The row's first elements are loaded before those
// are looked up. Head sizes of 64 and 128 have kernels of their own, since the general one was bound by its
// instructions (84% of the issue slots). Measured, 16 query and 8 key heads of 128, replays of a graph: 13500 fp32 rows
// 72.6 us (6.1 TB/s, 93% of a copy's rate; 80.6 before; between calls on other operands 79.4 us, 5.6 TB/s, 85%), as many bf16 rows
// 68 us, 256 bf16 rows 3.7 us, one row 2.8 us.
#include "ssb_decoder.cuh"

namespace ssb {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxHalf = 128;  // pairs of a head of 256 elements

// The sequence that row r belongs to, or s = -1. Where the starts rise it is the last one that starts at r or before, found 32 ways at
// a time by the warp. One that this finds but that may not have the row (it has too many rows, or less than none) is refused for its
// own rows only: the row may be another's, so the CTA looks through all of them then. (So it does for rows behind the last sequence:
// 256 rows and as many behind them take 4.8 us, 3.8 without those.)
struct RowOf {
    int s;
    Sequence q;
};
__device__ __forceinline__ RowOf sequence_of(const KvArgs & a, int r) {
    RowOf x;
    auto take = [&](int s) {
        x.s = s;
        x.q = sequence(a, s);
        return x.q.rows_ok && r >= x.q.start && r < x.q.start + x.q.n;
    };
    if (!a.row_start) {
        const int s = r / a.max_rows;
        if (s >= a.seqs || !take(s)) x.s = -1;
        return x;
    }
    int lo = 0, n = a.seqs;  // the answer lies in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int at = lo + (int) lane_id() * step;
        const bool below = (int) lane_id() * step < n && a.row_start[at] <= r;
        const uint32_t votes = __ballot_sync(0xffffffffu, below);
        const int last = votes ? 31 - __clz(votes) : 0;
        lo += last * step;
        n = min(step, n - last * step);
    }
    if (take(lo)) return x;
    __shared__ int s_owner[kRopeThreads / 32];
    int owner = -1;
#pragma unroll 4
    for (int s = (int) threadIdx.x; s < a.seqs; s += kRopeThreads) {  // (loads that wait for no other)
        const int start = a.row_start[s], end = a.row_start[s + 1];
        if (start >= 0 && start <= r && r < end && end <= a.rows && end - start <= a.max_rows) owner = max(owner, s);
    }
    owner = __reduce_max_sync(0xffffffffu, owner);
    if (lane_id() == 0) s_owner[warp_id()] = owner;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRopeThreads / 32; w++) owner = max(owner, s_owner[w]);
    if (owner >= 0 && take(owner)) return x;
    x.s = -1;
    return x;
}

// Element offsets of chunk c (of head_dim / 8) of a head: the four elements at `a` and the four at `b`, which
// in the rotated part are the pairs' halves.
__device__ __forceinline__ void chunk_at(int c, int dim, int rope, int & a, int & b) {
    if (c < rope / 8) {
        a = 4 * c, b = rope / 2 + 4 * c;
    } else {
        a = rope + 4 * (c - rope / 8), b = a + (dim - rope) / 2;
    }
}

// kLanes: threads of a head, for heads of 8 kLanes elements where all of them load and store four at a time; 0: `lanes_any`
// threads, any size and alignment.
template <typename T, typename TC, int kLanes>
__global__ void __launch_bounds__(kRopeThreads) norm_rope_kernel(const __grid_constant__ NormRopeArgs g, int lanes_any, int parts) {
    const int lanes = kLanes ? kLanes : lanes_any;
    const KvArgs & kv = g.kv;
    const int tid = (int) threadIdx.x;
    const int row_ctas = kv.rows * parts;
    if ((int) blockIdx.x >= row_ctas) {
        // the sequences' statuses, one warp each
        const int s = ((int) blockIdx.x - row_ctas) * (kRopeThreads / 32) + tid / 32;
        if (s >= kv.seqs) return;
        const Sequence q = sequence(kv, s);
        bool ok = q.ok;
        if (q.ok && q.n > 0 && q.length > 0) {
            const int first = max(q.length - q.n, 0) >> kv.page_shift, last = (q.length - 1) >> kv.page_shift;
            for (int i = first + (int) lane_id(); i <= last; i += 32)
                ok &= (unsigned) kv.table[(int64_t) s * kv.table_ld + i] < (unsigned) kv.pages;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (lane_id() == 0) kv.status[s] = ok ? SSB_ROW_OK : SSB_ROW_INVALID_ROW;
        return;
    }
    const int r = (int) blockIdx.x / parts, part = (int) blockIdx.x - r * parts;
    __shared__ __align__(16) float2 turn[kRopeMaxHalf];  // cosine and sine of each pair's angle
    const int dim = kLanes ? 8 * kLanes : kv.head_dim, chunks = dim / 8;
    const bool vec_in = kLanes || g.vec_in, vec_out = kLanes || g.vec_out, vec_cache = kLanes || g.vec_cache, vec_weight = kLanes || g.vec_weight;
    const int slots = kRopeThreads / lanes;  // heads of one pass
    const int c = tid % lanes;
    const bool held = kLanes || c < chunks;
    int ia, ib;
    chunk_at(held ? c : 0, dim, g.rope_dim, ia, ib);
    const bool rotated = ia < g.rope_dim;
    const int heads = g.q_heads + 2 * kv.kv_heads;
    // head h of the row: a query, key or value head (0, 1, 2), and its number there
    auto kind_of = [&](int h) { return h < g.q_heads ? 0 : (h < g.q_heads + kv.kv_heads ? 1 : 2); };
    auto number_of = [&](int h, int kind) { return kind == 0 ? h : h - g.q_heads - (kind == 2 ? kv.kv_heads : 0); };
    const T * q_row = static_cast<const T *>(g.q) + (int64_t) r * g.q_ld, * k_row = static_cast<const T *>(g.k) + (int64_t) r * g.k_ld;
    const T * v_row = static_cast<const T *>(g.v) + (int64_t) r * g.v_ld;
    auto load = [&](int h, float4 & x, float4 & y) {
        if (!held || h >= heads) return;
        const int kind = kind_of(h);
        const T * src = (kind == 0 ? q_row : kind == 1 ? k_row : v_row) + number_of(h, kind) * dim;
        x = load4(src + ia, vec_in), y = load4(src + ib, vec_in);
    };
    // the first heads' elements, on their way while the row's sequence, page and angles are looked up
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
    load(part * slots + tid / lanes, x, y);
    const RowOf found = sequence_of(kv, r);
    if (found.s < 0) return;
    const int s = found.s;
    const Sequence q = found.q;
    const int p = q.length - q.n + (r - q.start);
    int page = -1;
    if (q.ok && p >= 0) page = kv.table[(int64_t) s * kv.table_ld + (p >> kv.page_shift)];
    const bool live = (unsigned) page < (unsigned) kv.pages;  // else idle, or refused

    const double at = (double) (g.positions ? g.positions[r] : p);
    for (int i = tid; i < g.rope_dim / 2; i += kRopeThreads) {
        const double t = at * g.inv_freq[i];
        const double turns = rint(t * 0.15915494309189535);  // 1 / (2 pi)
        const float x = (float) fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, t));
        float sn, cs;
        sincosf(x, &sn, &cs);
        turn[i] = make_float2(cs, sn);
    }
    __syncthreads();

    T * out_row = static_cast<T *>(g.q_out) + (int64_t) r * g.q_out_ld;
    if (!live) {  // idle or refused: its queries are 0 and the cache is left alone
        const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int h = part * slots + tid / lanes; held && h < g.q_heads; h += parts * slots)
            store4(out_row + h * dim + ia, none, vec_out), store4(out_row + h * dim + ib, none, vec_out);
        return;
    }
    const int64_t slot_at = (int64_t) page * kv.page_stride + (int64_t) (p & (kv.page_size - 1)) * kv.position_stride;
    const float per_element = 1.0f / (float) dim;
    for (int h0 = part * slots; h0 < heads; h0 += parts * slots) {
        const int h = h0 + tid / lanes;
        const int kind = kind_of(h), hk = number_of(h, kind);
        if (h0 != part * slots) load(h, x, y);
        const float * weight = kind == 0 ? g.q_weight : kind == 1 ? g.k_weight : nullptr;
        if (h0 < g.q_heads + kv.kv_heads) {  // some head of this pass is normed and rotated
            float sum = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
#pragma unroll
            for (int o = kLanes ? kLanes / 2 : 16; o > 0; o /= 2)
                if (kLanes || o < lanes) sum += shfl_xor(sum, o);
            if (weight && held) {
                const float inv = rsqrtf(fmaf(sum, per_element, g.eps));
                const float4 wx = load4(weight + ia, vec_weight), wy = load4(weight + ib, vec_weight);
                x.x *= inv * wx.x, x.y *= inv * wx.y, x.z *= inv * wx.z, x.w *= inv * wx.w;
                y.x *= inv * wy.x, y.y *= inv * wy.y, y.z *= inv * wy.z, y.w *= inv * wy.w;
            }
            if (kind < 2 && rotated && held) {
                const float4 * at = reinterpret_cast<const float4 *>(turn + (g.interleaved ? ia / 2 : ia));
                if (g.interleaved) {
                    const float4 a = at[0], b = *reinterpret_cast<const float4 *>(turn + ib / 2);
                    x = make_float4(x.x * a.x - x.y * a.y, x.y * a.x + x.x * a.y, x.z * a.z - x.w * a.w, x.w * a.z + x.z * a.w);
                    y = make_float4(y.x * b.x - y.y * b.y, y.y * b.x + y.x * b.y, y.z * b.z - y.w * b.w, y.w * b.z + y.z * b.w);
                } else {
                    const float4 a = at[0], b = at[1], u = x;
                    x = make_float4(u.x * a.x - y.x * a.y, u.y * a.z - y.y * a.w, u.z * b.x - y.z * b.y, u.w * b.z - y.w * b.w);
                    y = make_float4(y.x * a.x + u.x * a.y, y.y * a.z + u.y * a.w, y.z * b.x + u.z * b.y, y.w * b.z + u.w * b.w);
                }
            }
        }
        if (!held || h >= heads) continue;
        if (kind == 0) {
            T * dst = out_row + h * dim;
            store4(dst + ia, x, vec_out), store4(dst + ib, y, vec_out);
        } else {
            TC * dst = static_cast<TC *>(kind == 1 ? kv.k : kv.v) + slot_at + (int64_t) hk * kv.head_stride;
            store4(dst + ia, x, vec_cache), store4(dst + ib, y, vec_cache);
        }
    }
}

template <typename T, typename TC>
cudaError_t launch(const NormRopeArgs & a, int sm_count, cudaStream_t stream) {
    int lanes = 2;
    while (lanes * 8 < a.kv.head_dim) lanes *= 2;
    const int slots = kRopeThreads / lanes, heads = a.q_heads + 2 * a.kv.kv_heads;
    // few rows: a CTA per pass over the heads, so that their loads go out together; many: a row's angles are
    // worked out once
    const int parts = a.kv.rows < 4 * sm_count ? (heads + slots - 1) / slots : 1;
    const int64_t status_ctas = a.kv.status ? (a.kv.seqs + kRopeThreads / 32 - 1) / (kRopeThreads / 32) : 0;
    const int64_t grid = (int64_t) a.kv.rows * parts + status_ctas;
    if (grid == 0) return cudaSuccess;
    const bool vec = a.vec_in && a.vec_out && a.vec_cache && a.vec_weight;
    if (vec && a.kv.head_dim == 128) norm_rope_kernel<T, TC, 16><<<(unsigned) grid, kRopeThreads, 0, stream>>>(a, lanes, parts);
    else if (vec && a.kv.head_dim == 64) norm_rope_kernel<T, TC, 8><<<(unsigned) grid, kRopeThreads, 0, stream>>>(a, lanes, parts);
    else norm_rope_kernel<T, TC, 0><<<(unsigned) grid, kRopeThreads, 0, stream>>>(a, lanes, parts);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeArgs & a, bool bf16, bool cache_bf16, int sm_count, cudaStream_t stream) {
    using B = __nv_bfloat16;
    if (bf16) return cache_bf16 ? launch<B, B>(a, sm_count, stream) : launch<B, float>(a, sm_count, stream);
    return cache_bf16 ? launch<float, B>(a, sm_count, stream) : launch<float, float>(a, sm_count, stream);
}

}  // namespace ssb

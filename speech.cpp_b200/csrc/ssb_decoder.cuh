// Device pieces shared by the decoder-step kernels: where a sequence's rows and pages are, which
// positions a block of rows sees, and the join of partial attentions across a thread-block cluster.
#pragma once

#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_bf16.h>

#include "ssb_device.cuh"
#include "ssb_kernels.h"

namespace ssb {
namespace {

constexpr float kLn2 = 0.6931471805599453f;

struct Sequence {
    int start;   // first row
    int n;       // rows
    int length;  // cached positions, the new rows included
    bool rows_ok;  // the rows exist and are as many as the launch covers
    bool ok;       // and the length is within the bound
};

struct SequenceNumbers {
    int start, end, length;
};
__device__ __forceinline__ SequenceNumbers sequence_numbers(const KvArgs & a, int s) {
    const int start = a.row_start ? a.row_start[s] : s * a.max_rows;
    return {start, a.row_start ? a.row_start[s + 1] : start + a.max_rows, a.length[s]};
}
__device__ __forceinline__ Sequence sequence(const KvArgs & a, const SequenceNumbers & x) {
    Sequence q;
    q.start = x.start;
    q.length = x.length;
    q.rows_ok = x.start >= 0 && x.end >= x.start && x.end <= a.rows && x.end - x.start <= a.max_rows;
    q.n = q.rows_ok ? x.end - x.start : 0;
    q.ok = q.rows_ok && q.length >= 0 && q.length <= a.max_length;
    return q;
}
__device__ __forceinline__ Sequence sequence(const KvArgs & a, int s) { return sequence(a, sequence_numbers(a, s)); }

// A call's statuses are cleared in stream order before the kernel whose CTAs share a sequence, and those only raise
// them: what one CTA refuses, another that knows nothing of it cannot report as good. `bad`: 1 refused, 2 a wait gave up.
// The kernel starts while they are cleared (a programmatic dependency) and waits for that here, and before it ends: a step that
// asks for statuses takes 8.3 us instead of 7.6 (one stream at 37 positions), and 10.3 behind a memset.
static_assert(SSB_ROW_OK == 0 && SSB_ROW_INVALID_ROW < SSB_ROW_DEVICE_TIMEOUT, "statuses are cleared to 0 and get larger as they get worse");
__device__ __forceinline__ void statuses_cleared() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void raise_status(const KvArgs & a, int seq, int bad) {
    if (!bad || !a.status) return;
    statuses_cleared();
    atomicMax(a.status + seq, bad & 2 ? (int) SSB_ROW_DEVICE_TIMEOUT : (int) SSB_ROW_INVALID_ROW);
}
__global__ void clear_kernel(int32_t * status, int n) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int i = (int) (blockIdx.x * blockDim.x + threadIdx.x);
    if (i < n) status[i] = SSB_ROW_OK;
}

// Element offset of (page, slot, head) in the pool: 64-bit, a long cache passes 2^31 elements.
__device__ __forceinline__ int64_t pool_offset(const KvArgs & a, int page, int slot, int head) {
    return (int64_t) page * a.page_stride + (int64_t) slot * a.position_stride + (int64_t) head * a.head_stride;
}

// The positions that rows at positions p_first..p_last see between them, [0, sinks) and [first, hi), as tiles
// of kTile positions (64 but for fp32 steps) that start at multiples of kTile: first the sinks' (none where they
// run into the rest), then the rest's from lo on. A tile may hold positions that nobody sees; those are not to be
// read.
constexpr int kTile = 64;
template <int kTile> struct SpanOf {
    int sinks, first, lo, hi, sink_tiles, tiles;
    __device__ __forceinline__ int base(int t) const { return t < sink_tiles ? t * kTile : lo + (t - sink_tiles) * kTile; }
    __device__ __forceinline__ bool seen(int j) const { return j < hi && (j >= first || j < sinks); }
};

using Span = SpanOf<kTile>;

template <int kTile = ::ssb::kTile> __device__ __forceinline__ SpanOf<kTile> span_of(int p_first, int p_last, int window, int sinks) {
    SpanOf<kTile> s;
    s.hi = p_last + 1 > 0 ? p_last + 1 : 0;
    s.first = window > 0 && p_first - window + 1 > 0 ? p_first - window + 1 : 0;
    s.lo = s.first / kTile * kTile;
    s.sinks = sinks < s.hi ? sinks : s.hi;
    if (s.lo <= s.sinks) s.lo = 0;
    s.sink_tiles = s.lo == 0 ? 0 : (s.sinks + kTile - 1) / kTile;
    s.tiles = s.sink_tiles + (s.hi - s.lo + kTile - 1) / kTile;
    return s;
}

__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
    return j <= p && (window == 0 || j > p - window || j < sinks);
}

// Whether every table entry of the pages that hold some position of `s` names a page of the pool. All
// threads of the CTA take part and get the answer.
__device__ __forceinline__ bool pages_ok(const KvArgs & a, int seq, const Span & s) {
    const int32_t * table = a.table + (int64_t) seq * a.table_ld;
    bool ok = true;
    const int sink_pages = (s.sinks + a.page_size - 1) >> a.page_shift;
    const int first = s.first >> a.page_shift, last = (s.hi + a.page_size - 1) >> a.page_shift;
    for (int i = (int) threadIdx.x; i < sink_pages; i += (int) blockDim.x) ok &= (unsigned) table[i] < (unsigned) a.pages;
    for (int i = first + (int) threadIdx.x; i < last; i += (int) blockDim.x)
        ok &= (unsigned) table[i] < (unsigned) a.pages;
    return __syncthreads_and(ok) != 0;
}

// A tile or step whose copies the wait-limit test build (SSB_WAIT_TEST) never issues, so that the bounded waits for them run out.
__device__ __forceinline__ bool left_out(int seq, int head, int tile) {
#ifdef SSB_WAIT_TEST
    return seq == 1 && head == 1 && tile == 2;
#else
    return false;
#endif
}

// What a refused sequence's rows hold: 0, or NaN where the device did not answer.
__device__ __forceinline__ float refused_value(int bad) { return bad & 2 ? __int_as_float(0x7fc00000) : 0.0f; }

constexpr int kMaxRanks = 8;  // of a cluster: the portable size

// What a CTA leaves for the join of its cluster: `rows` rows of unnormalized output (row m at out + m * ld),
// each row's maximum score (base 2 logarithm units) and sum of weights, and bits that refuse the sequence.
struct Partial {
    float * out;
    int ld;
    float2 * stat;  // [rows] (maximum, sum)
    float * share;  // [cluster size * rows] scratch
    int * bad;
};

// Joins the partials of the cluster's CTAs, in rank order whatever their timing, and hands element
// groups of four to `store(m, c, float4)` and the log-sum-exps to `store_lse(m, lse)`, spread over the
// ranks. Returns every rank's refusing bits, the same to all. A row with no visible position is the caller's.
template <typename Store, typename StoreLse>
__device__ __forceinline__ int join_cluster(const Partial & p, int rows, int dim, Store store, StoreLse store_lse) {
    namespace cg = cooperative_groups;
    auto cluster = cg::this_cluster();
    const int ranks = (int) cluster.num_blocks(), rank = (int) cluster.block_rank();
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    int refused = 0;
#pragma unroll
    for (int r = 0; r < kMaxRanks; r++)
        if (r < ranks) refused |= *cluster.map_shared_rank(p.bad, r);
    for (int m = (int) threadIdx.x; m < rows; m += (int) blockDim.x) {
        float2 stat[kMaxRanks];  // all on their way at once, as below
#pragma unroll
        for (int r = 0; r < kMaxRanks; r++) stat[r] = r < ranks ? cluster.map_shared_rank(p.stat, r)[m] : make_float2(-kInf, 0.0f);
        float top = -kInf;
#pragma unroll
        for (int r = 0; r < kMaxRanks; r++) top = fmaxf(top, stat[r].x);
        const float ref = top == -kInf ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < kMaxRanks; r++) {
            stat[r].x = exp2f(stat[r].x - ref);
            sum += stat[r].y * stat[r].x;
        }
        const float inv = 1.0f / sum;
#pragma unroll
        for (int r = 0; r < kMaxRanks; r++)
            if (r < ranks) p.share[r * rows + m] = stat[r].x * inv;
        if (rank == 0) store_lse(m, refused ? -kInf : ref * kLn2 + logf(sum));
    }
    __syncthreads();
    const int groups = dim / 4;
    const float fill = refused_value(refused);
#pragma unroll 2
    for (int e = rank * (int) blockDim.x + (int) threadIdx.x; e < rows * groups; e += ranks * (int) blockDim.x) {
        const int m = e / groups, c = (e - m * groups) * 4;
        float4 x[kMaxRanks];
#pragma unroll
        for (int r = 0; r < kMaxRanks; r++)
            x[r] = r < ranks ? *reinterpret_cast<const float4 *>(cluster.map_shared_rank(p.out, r) + m * p.ld + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < kMaxRanks; r++) {
            if (r >= ranks) break;
            const float w = p.share[r * rows + m];
            o.x += x[r].x * w, o.y += x[r].y * w, o.z += x[r].z * w, o.w += x[r].w * w;
        }
        store(m, c, refused ? make_float4(fill, fill, fill, fill) : o);
    }
    if (ranks > 1) cluster.sync();  // no rank leaves while another reads its shared memory
    return refused;
}

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four adjacent elements, widened; `vec` where the address is a multiple of their size.
__device__ __forceinline__ float4 load4(const float * p, bool vec) {
    return vec ? *reinterpret_cast<const float4 *>(p) : make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16 * p, bool vec) {
    if (!vec) return make_float4(widen(p[0]), widen(p[1]), widen(p[2]), widen(p[3]));
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    return make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
}
__device__ __forceinline__ void store4(float * p, const float4 & x, bool vec) {
    if (vec) *reinterpret_cast<float4 *>(p) = x;
    else p[0] = x.x, p[1] = x.y, p[2] = x.z, p[3] = x.w;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void store4(__nv_bfloat16 * p, const float4 & x, bool vec) {
    if (vec) *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
    else p[0] = narrow<__nv_bfloat16>(x.x), p[1] = narrow<__nv_bfloat16>(x.y), p[2] = narrow<__nv_bfloat16>(x.z), p[3] = narrow<__nv_bfloat16>(x.w);
}

// Launches `kernel` with `blocks` CTAs in clusters of `size`. One that raises statuses (see raise_status) has them cleared first.
inline cudaError_t launch_cluster(const void * kernel, unsigned blocks, int size, int threads, size_t smem, cudaStream_t stream,
                                  void ** params, const KvArgs * raises = nullptr) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3((unsigned) threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    config.attrs = attributes;
    if (size > 1) {
        cudaLaunchAttribute & cluster = attributes[config.numAttrs++];
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = (unsigned) size;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    }
    if (raises && raises->status) {
        clear_kernel<<<(raises->seqs + 255) / 256, 256, 0, stream>>>(raises->status, raises->seqs);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        cudaLaunchAttribute & early = attributes[config.numAttrs++];
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
    }
    return cudaLaunchKernelExC(&config, kernel, params);
}

}  // namespace
}  // namespace ssb

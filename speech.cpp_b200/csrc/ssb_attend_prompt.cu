// Attention of many rows per sequence over a paged bf16 cache (head size 64 or 128): prompts, and blocks of them.
//
//   out = sum_j softmax_j(scale * q . k[j]) v[j] over the positions j that the row sees
//
// 4 D multiply-adds per (row, position) pair of a query head, so the bound is the tensor cores, and next to them the
// 16 exponentials per clock of an SM: both take about 1000 clocks for 128 x 128 scores at D = 128. The (row, query
// head) pairs that read one key head are one list, cut into tiles of 128 rows of a tcgen05 product; a CTA holds
// two of them and walks the tiles of 128 positions that they see:
//   warps 0-3, 4-7  one tile each, a thread per pair: the scores from tensor memory, the mask where the tile needs
//                   one, the running maximum, the weights in bf16 back over the scores, and their fp32 sum. The
//                   output in tensor memory is rescaled only when the maximum has grown by a factor of 256 since
//                   the last time; until then the weights are relative to the older maximum. They are taken 256 times
//                   smaller, so that none is above 1: a finite value times its weight stays finite.
//   warp 8          TMA copies of keys and values out of the pages into a ring (128-byte swizzle, no multicast)
//   warp 9          one thread issues the products: scores = Q K^T with both operands in shared memory, output +=
//                   P V with P in tensor memory and V taken as it lies (its rows are the inner dimension). While one
//                   tile's weights are worked out, the other's products run.
// Where there are fewer CTAs than SMs, the CTAs of a cluster share the positions and join their partials through
// distributed shared memory, in rank order.
//
// Measured (D = 128, replays of a graph): 8 prompts of 1000 to 6001 rows, 32 query and 8 key heads, 1025 us, 986 TFLOP/s of the
// products that the masks leave (1181 us and 856 TFLOP/s between calls on other operands); a step is bound by its chain (scores, maximum, exponentials, product, next scores:
// 1900 clocks of softmax and 1300 of products and waits) with the other tile's chain beside it, and about 10000
// clocks a CTA (1 in 7) go before and after the steps. 512 rows behind 4000 positions: 35 us on 128 CTAs, a
// third of it the join. 16001 rows under a window of 1024 and 4 sinks: 239 us, 3 of a CTA's 10 steps at an edge.
// One value that is not finite and that only some of a CTA's rows see costs much: those 256 pairs go over their positions
// one by one, the 512 rows 29 ms and 8 prompts of 2000 rows 39 ms with one such value.
// Every mbarrier wait is bounded; one that gives up ends the rows of its CTA, and of the cluster that shares them, as NaN with
// SSB_ROW_DEVICE_TIMEOUT.
#include <algorithm>

#include "ssb_decoder.cuh"
#include "ssb_tma.cuh"
#include "ssb_tma_map.cuh"

namespace ssb {

namespace {

namespace cg = cooperative_groups;

constexpr int kRows = 128;            // pairs of a tile: lanes of tensor memory
constexpr int kKeys = 128;            // positions of a step
constexpr int kThreads = 384;         // three warpgroups: two of softmax, one of the producer and the product warp
// Registers of a thread while the loop runs: the launch's 168 are split anew (2 x 224 + 56 = 3 x 168), since a
// softmax thread holds a row of 128 scores.
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56, kLaunchRegs = 168;
static_assert(2 * kSoftmaxRegs + kOtherRegs == 3 * kLaunchRegs, "no more than the launch has");
constexpr int kCtaRows = 2 * kRows;
constexpr float kRescale = 8.0f;      // log2 of the growth that rescales the output (256 below)
constexpr int kTmemColumns = 512;     // two tiles' scores (128 each, the weights over them) and outputs (D each)

template <int D> constexpr int slot_bytes() { return kKeys * D * 2; }
template <int D> constexpr int slots() { return D == 128 ? 4 : 8; }

// Shared-memory matrix descriptors of bf16 tiles with 128-byte swizzle, in two words: the address and the leading
// offset in units of 16 bytes below, the stride offset, the version (1) and the layout (2) above. Rows are 128
// bytes, 8 of them a block of 1024 bytes, the stride. A step along a tile adds its offset / 16 to the lower word,
// which is all that is left to do between two products: with whole descriptors built for each, the one thread
// took 110 clocks a product, that takes the tensor cores 64.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// Inner dimension along the rows' 128 bytes (the leading offset is not used), or across the rows, where the outer
// dimension's next 64 elements lie `next` bytes on. (In a cluster an address has its CTA's rank above its 18 bits.)
__device__ __forceinline__ uint32_t k_major(uint32_t addr) { return ((addr >> 4) & 0x3fffu) | (1u << 16); }
__device__ __forceinline__ uint32_t mn_major(uint32_t addr, uint32_t next) { return ((addr >> 4) & 0x3fffu) | ((next >> 4) << 16); }

// Instruction descriptor of kind::f16: D f32, A and B bf16, B's inner dimension across its rows where `b_mn`.
__host__ __device__ constexpr uint32_t instruction(int m, int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t) b_mn << 16) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (m >> 4) << 24);
}

template <bool kAdd> __device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "n"(kDescHigh), "r"(idesc), "n"((int) kAdd)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "n"(kDescHigh), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t * bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// One lane of the warp, the same each time.
__device__ __forceinline__ bool elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 32 columns of the warp's 32 lanes of tensor memory (thread t: lane base + t); wait_ld() before they are used.
__device__ __forceinline__ void tmem_load(uint32_t (&r)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// Ties the registers to a point after the wait: nothing may use them before it.
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.wait::ld.sync.aligned;"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
          "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
          "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
          "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
            addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// The same for registers of loads that one wait has covered.
__device__ __forceinline__ void after_wait(uint32_t (&r)[32]) {
    asm volatile(
        ""
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
          "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
          "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
          "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 2^x with a relative error of 2^-22; -inf gives 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 values in one register pair, for the instructions that work on both at once.
__device__ __forceinline__ uint64_t two(uint32_t a, uint32_t b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint64_t two(float a, float b) { return two(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ float2 apart_of(uint64_t d) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(d));
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// The n lowest bits, for any n.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
// Adds 0 times each of eight bf16 values: NaN where one is not finite.
__device__ __forceinline__ void add_nothing(__nv_bfloat162 & sum, const uint4 & v) {
    const __nv_bfloat162 zero = __floats2bfloat162_rn(0.0f, 0.0f);
    sum = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&v.x), zero, sum);
    sum = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&v.y), zero, sum);
    sum = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&v.z), zero, sum);
    sum = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&v.w), zero, sum);
}

// The positions that a block of rows sees, in steps of kKeys (see Span, whose tiles are of kTile).
struct Steps {
    int sinks, first, lo, hi, sink_steps, steps;
    __device__ __forceinline__ int base(int t) const { return t < sink_steps ? t * kKeys : lo + (t - sink_steps) * kKeys; }
    __device__ __forceinline__ bool seen(int j) const { return j < hi && (j >= first || j < sinks); }
};
__device__ __forceinline__ Steps steps_of(const Span & span) {
    Steps s;
    s.hi = span.hi, s.first = span.first, s.sinks = span.sinks;
    s.lo = s.first / kKeys * kKeys;
    if (s.lo <= s.sinks) s.lo = 0;
    s.sink_steps = s.lo == 0 ? 0 : (s.sinks + kKeys - 1) / kKeys;
    s.steps = s.sink_steps + (s.hi - s.lo + kKeys - 1) / kKeys;
    return s;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ AttendArgs g, int row_blocks) {
    constexpr int kHalves = D / 64, kSlots = slots<D>();
    constexpr uint32_t kHalfBytes = kKeys * 128;  // 64 elements of every position
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char * smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    unsigned char * query = smem;                                            // [2 tiles][half][128 rows][128 bytes]
    unsigned char * ring = smem + (size_t) 2 * kRows * D * 2;                // [kSlots][half][128 positions][128 bytes]
    __shared__ __align__(8) uint64_t full[kSlots], empty[kSlots], scores_full[2], weights_full[2][2], out_full;
    __shared__ float2 stat[kCtaRows];
    __shared__ float share[8 * kCtaRows];
    __shared__ uint32_t s_tmem;
    __shared__ int s_bad;    // bits that refuse the rows: 1 a page outside the pool or a bad length, 2 a wait gave up
    __shared__ int s_apart;  // a value that only some rows see is not finite
    const KvArgs & kv = g.kv;
    auto cluster = cg::this_cluster();
    const int ranks = (int) cluster.num_blocks(), rank = (int) cluster.block_rank();
    const int unit = (int) (blockIdx.x / (unsigned) ranks);
    // the last rows of a sequence see the most: they start first
    const int block = row_blocks - 1 - unit / (kv.kv_heads * kv.seqs);
    const int head = unit % kv.kv_heads, seq = unit / kv.kv_heads % kv.seqs;
    const int tid = (int) threadIdx.x, warp = warp_id(), lane = lane_id();
    const Sequence q = sequence(kv, seq);
    const int pairs = q.n * g.group, m0 = block * kCtaRows;
    if (m0 >= pairs) {
        if (block == 0 && head == 0 && rank == 0 && tid == 0) raise_status(kv, seq, q.ok ? 0 : 1);  // no rows at all
        statuses_cleared();
        return;
    }
    const int first = q.length - q.n;  // the position of the sequence's first row
    const int rows = min(kCtaRows, pairs - m0);
    const Steps span = steps_of(span_of(first + m0 / g.group, first + (m0 + rows - 1) / g.group, g.window, g.sinks));
    // the queries into their swizzled places, a row past the last as zeros; the scale's sign folded in
    const uint32_t sign = g.scale_log2 < 0.0f ? 0x80008000u : 0u;
    constexpr int kChunks = D / 8, kPass = kThreads / kChunks, kPasses = (kCtaRows + kPass - 1) / kPass;
    const int chunk = tid % kChunks;
    uint4 queries[kPasses];  // on their way while the pages are looked through
    {
        const bool wide = (reinterpret_cast<uintptr_t>(g.q) | (uintptr_t) (g.q_ld * 2)) % 16 == 0;
#pragma unroll
        for (int i = 0; i < kPasses; i++) {
            const int m = i * kPass + tid / kChunks;
            queries[i] = make_uint4(0u, 0u, 0u, 0u);
            if (m >= rows) continue;
            const __nv_bfloat16 * src = static_cast<const __nv_bfloat16 *>(g.q) + (int64_t) (q.start + (m0 + m) / g.group) * g.q_ld +
                                        (int64_t) (head * g.group + (m0 + m) % g.group) * D + chunk * 8;
            if (wide) {
                queries[i] = *reinterpret_cast<const uint4 *>(src);
            } else {
                const uint2 a = reinterpret_cast<const uint2 *>(src)[0], b = reinterpret_cast<const uint2 *>(src)[1];
                queries[i] = make_uint4(a.x, a.y, b.x, b.y);
            }
        }
    }
    int t0 = (int) ((int64_t) span.steps * rank / ranks), t1 = (int) ((int64_t) span.steps * (rank + 1) / ranks);
    // slot and phase of the keys (index 2 (t - t0)) and the values (one more) of step t
    auto slot_of = [&](int index) { return index % kSlots; };
    auto phase_of = [&](int index) { return (uint32_t) (index / kSlots) & 1u; };

    // The producer's: lane l copies piece l of a step's keys or values.
    const int box = min(kv.page_size, kKeys), per_step = kKeys / box;
    const int32_t * table = kv.table + (int64_t) seq * kv.table_ld;
    auto place = [&](int t) { return span.base(t) + lane * box; };
    auto page_of = [&](int t) {  // only of pieces that hold a seen position, the table's other entries may be anything; else -1
        const int from = place(t);
        const bool wanted = t < t1 && lane < per_step && from < span.hi && (from + box > span.first || from < span.sinks);
        return wanted ? table[from >> kv.page_shift] : -1;
    };
    auto copy = [&](int index, int t, int page) {
        const int s = slot_of(index);
        if (left_out(seq, head, t) && block > 0 && block == row_blocks - 1) return;
        const bool wanted = (unsigned) page < (unsigned) kv.pages;
        const int copies = __popc(__ballot_sync(0xffffffffu, wanted));
        if (lane == 0) mbar_expect(&full[s], (uint32_t) (copies * box * D * 2));
        __syncwarp();
        if (!wanted) return;
        unsigned char * dst = ring + (size_t) s * slot_bytes<D>() + lane * box * 128;
        for (int half = 0; half < kHalves; half++)
            tma_load_5d(dst + half * kHalfBytes, index & 1 ? &map_v : &map_k, 0, place(t) & (kv.page_size - 1), half, head, page, &full[s]);
    };
    int issued = 0, next = -1;  // copies, and the page of the next step's piece
    if (warp == 8) {
        // the first copies wait for nothing but these: they run while the queries load and the pages are looked through
        if (lane == 0) {
            for (int s = 0; s < kSlots; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], 2);
            for (int i = 0; i < 2; i++) mbar_init(&scores_full[i], 1), mbar_init(&weights_full[i][0], 4), mbar_init(&weights_full[i][1], 4);
            mbar_init(&out_full, 1);
            s_bad = 0;
            s_apart = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (q.ok) {
            next = page_of(t0);
            for (int t = t0; t < t1 && issued < kSlots; t++) {
                const int page = next;
                next = page_of(t + 1);
                for (int which = 0; which < 2; which++) copy(issued++, t, page);
            }
        }
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "n"(kTmemColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    bool ok = q.ok;
    if (ok) ok = pages_ok(kv, seq, span_of(first, q.length - 1, g.window, g.sinks));
    if (!ok) t1 = t0;
    if (tid == 8 * 32 && !ok) s_bad = 1;
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
        const int m = i * kPass + tid / kChunks, r = m % kRows;
        if (m >= kCtaRows) continue;
        *reinterpret_cast<uint4 *>(query + m / kRows * (kRows * D * 2) + chunk / 8 * (kRows * 128) + r * 128 + ((chunk % 8) ^ (r & 7)) * 16) =
            make_uint4(queries[i].x ^ sign, queries[i].y ^ sign, queries[i].z ^ sign, queries[i].w ^ sign);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;
    auto dead = [&]() { return (*reinterpret_cast<volatile int *>(&s_bad) & 2) != 0; };
    auto give_up = [&]() { atomicOr(&s_bad, 2); };
    // what the epilogue takes its rows from; the softmax warps' row
    const int tile = warp / 4, m = tid;  // (warps 0-7)
    float top = -kInf, sum = 0.0f;
    int position = 0, seen_from = 0;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 8) {
            // ---- producer, from where its first copies ended
            bool alive = ok;
            for (int t = t0 + issued / 2; t < t1 && alive; t++) {
                const int page = next;
                next = page_of(t + 1);
                for (int which = 0; which < 2; which++) {
                    const bool ready = mbar_wait(&empty[slot_of(issued)], phase_of(issued - kSlots));
                    if (!__all_sync(0xffffffffu, ready && !dead())) {
                        alive = false;
                        break;
                    }
                    copy(issued++, t, page);
                }
            }
            if (ok && !alive && lane == 0) give_up();
            // The copies in flight land before the shared memory is given up, whichever warp's wait ran out and however late:
            // the last steps' copies may all be issued when the products give up on one of them. (Else they are there already,
            // or this warp has nothing else to do.)
            for (int i = max(0, issued - kSlots); i < issued; i++) mbar_wait(&full[slot_of(i)], phase_of(i));
        } else if (warp == 9) {
            // ---- products, all in one thread's order, so that a tile's next scores come after the product that reads the
            // weights which they overwrite. The tiles take turns: one's products run while the other's weights are worked
            // out, and little but the wait for them stands between two turns: a step of both tiles takes 3240 clocks at
            // D = 128 (2 x 1024 of products), where a loop that looked for what had become possible took 5500.
            if (t1 > t0) {
                const bool leader = elect();  // all lanes walk the loop, which keeps its numbers in uniform registers
                const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
                constexpr uint32_t kScores = instruction(kRows, kKeys, false), kOutput = instruction(kRows, D, true);
                const uint32_t query_desc = k_major(smem_addr(query)), ring_desc = k_major(smem_addr(ring));
                const uint32_t value_desc = mn_major(smem_addr(ring), kHalfBytes);
                auto scores = [&](int tile, int index) {  // with the keys at `index` of the ring
                    const uint32_t a = query_desc + (uint32_t) (tile * (kRows * D * 2 / 16));
                    const uint32_t b = ring_desc + (uint32_t) (slot_of(index) * (slot_bytes<D>() / 16));
                    const uint32_t d = tmem + (uint32_t) (tile * kKeys);
                    if (!leader) return;
                    mma_ss<false>(d, a, b, kScores);
    #pragma unroll
                    for (int k = 1; k < D / 16; k++)
                        mma_ss<true>(d, a + (uint32_t) ((k / 4 * kRows * 128 + k % 4 * 32) / 16), b + (uint32_t) ((k / 4 * kHalfBytes + k % 4 * 32) / 16), kScores);
                    commit(&scores_full[tile]);
                    commit(&empty[slot_of(index)]);
                };
                auto output = [&](int tile, int index, int half, uint32_t add) {  // with half of the values at `index`
                    const uint32_t b = value_desc + (uint32_t) (slot_of(index) * (slot_bytes<D>() / 16) + half * (kKeys * 64 / 16));
                    const uint32_t d = tmem + (uint32_t) (2 * kKeys + tile * D), a = tmem + (uint32_t) (tile * kKeys + half * (kKeys / 4));
                    if (!leader) return;
                    mma_ts(d, a, b, kOutput, add);
    #pragma unroll
                    for (int k = 1; k < kKeys / 32; k++) mma_ts(d, a + (uint32_t) (k * 8), b + (uint32_t) (k * 2048 / 16), kOutput, 1u);
                };
                const int all = t1 - t0;
                bool alive = __all_sync(0xffffffffu, mbar_wait(&full[0], 0u));
                fence_after();
                if (alive) scores(0, 0), scores(1, 0);
                alive = __all_sync(0xffffffffu, alive && mbar_wait(&full[slot_of(1)], 0u));
                for (int t = 0; t < all && alive; t++) {
                    const int index = 2 * t;
                    const bool more = t + 1 < all;
    #pragma unroll
                    for (int tile = 0; tile < 2; tile++) {
    #pragma unroll
                        for (int half = 0; half < 2 && alive; half++) {
                            alive = __all_sync(0xffffffffu, mbar_wait(&weights_full[tile][half], (uint32_t) t & 1u));
                            if (!alive) break;
                            fence_after();
                            output(tile, index + 1, half, half == 0 ? (uint32_t) t : 1u);
                            // the next step's keys and then its values, where this warp waits for weights anyway
                            if (half == 0 && more) alive = __all_sync(0xffffffffu, mbar_wait(&full[slot_of(index + 2 + tile)], phase_of(index + 2 + tile)));
                        }
                        if (!alive) break;
                        if (more) scores(tile, index + 2);
                        if (leader) commit(&empty[slot_of(index + 1)]);
                    }
                }
                if (!alive && leader) give_up();
                if (leader) commit(&out_full);  // after every product issued
                mbar_wait(&out_full, 0u);
            }
            __syncwarp();
        }
        fence_before();
        __syncthreads();
        // only now: a warp that took its registers back earlier could take those that a softmax warp still waits for
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLaunchRegs));
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ---- softmax of a tile, a thread per pair
        const int p_low = first + (m0 + tile * kRows) / g.group, p_high = first + (m0 + min(rows, (tile + 1) * kRows) - 1) / g.group;
        const int p_first = first + m0 / g.group, p_last = first + (m0 + rows - 1) / g.group;  // of the CTA
        position = first + (m0 + min(m, rows - 1)) / g.group;
        seen_from = g.window > 0 ? max(position - g.window + 1, 0) : 0;
        const float scale = fabsf(g.scale_log2);  // not 0 (tma_takes): a hidden score of -inf stays -inf
        const uint32_t lanes = tmem + ((uint32_t) (warp % 4 * 32) << 16);
        const uint32_t mine = lanes + (uint32_t) (tile * kKeys), out = lanes + (uint32_t) (2 * kKeys + tile * D);
        for (int t = t0; t < t1; t++) {
            const int base = span.base(t);
            const bool whole = base + kKeys - 1 <= p_low && (g.window == 0 || base > p_high - g.window || base + kKeys - 1 < g.sinks);
            uint32_t visible[4];  // the columns of this step that the row sees, a bit each
            if (!whole) {
                const int from = seen_from - base, count = max(position + 1 - seen_from, 0), sinks = min(g.sinks, position + 1) - base;
#pragma unroll
                for (int c = 0; c < 4; c++) visible[c] = bits_below(from + count - c * 32) & ~bits_below(from - c * 32) | bits_below(sinks - c * 32);
            }
            // whether some position of the step is seen by none or only some of the CTA's rows
            const bool edge = base + kKeys - 1 > p_first || (g.window > 0 && base <= p_last - g.window && base + kKeys - 1 >= g.sinks);
            if (edge) {
                // Values that a weight of 0 must keep out have to be finite: those of positions that no row of the
                // CTA sees are cleared, those that only some rows see are looked through. A thread per position;
                // both tiles do the same, while the scores are worked out. (The slot's phase before is over: its product came
                // before the last step's scores.)
                const int index = 2 * (t - t0) + 1, p = base + tid % kKeys;
                const bool there = !dead() && mbar_wait(&full[slot_of(index)], phase_of(index));
                unsigned char * value = ring + (size_t) slot_of(index) * slot_bytes<D>() + tid % kKeys * 128;
                if (there && !span.seen(p)) {
#pragma unroll
                    for (int c = 0; c < D / 8; c++) *reinterpret_cast<uint4 *>(value + c / 8 * kHalfBytes + c % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
                } else if (there && !(p <= p_first && (g.window == 0 || p > p_last - g.window || p < g.sinks))) {
                    __nv_bfloat162 sum = __floats2bfloat162_rn(0.0f, 0.0f);
#pragma unroll
                    for (int c = 0; c < D / 8; c++) add_nothing(sum, *reinterpret_cast<const uint4 *>(value + c / 8 * kHalfBytes + c % 8 * 16));
                    if (__low2float(sum) != 0.0f || __high2float(sum) != 0.0f) s_apart = 1;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            const bool got = !dead() && mbar_wait(&scores_full[tile], (uint32_t) (t - t0) & 1u);
            if (!__all_sync(0xffffffffu, got)) {
                if (lane == 0) give_up();
                break;
            }
            fence_after();
            uint32_t x[4][32];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_load(x[c], mine + (uint32_t) (c * 32));
            tmem_wait_load(x[0]);
#pragma unroll
            for (int c = 1; c < 4; c++) after_wait(x[c]);
            if (!whole) {
#pragma unroll
                for (int c = 0; c < kKeys; c++)
                    if (!(visible[c / 32] >> (c % 32) & 1u)) x[c / 32][c % 32] = 0xff800000u;
            }
            float most[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
            for (int c = 0; c < kKeys; c += 2)
                most[c / 2 % 4] = fmaxf(most[c / 2 % 4], fmaxf(__uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1])));
            const float new_top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * scale;
            const bool grown = new_top > top + kRescale || (top == -kInf && new_top > -kInf);
            if (__any_sync(0xffffffffu, grown)) {
                const float a = grown ? ex2(top - new_top) : 1.0f;
                if (grown) top = new_top;
                sum *= a;
                if (t > t0) {  // the output through the step before is complete: its product came before these scores'
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t o[32];
                        tmem_load(o, out + (uint32_t) (c * 32));
                        tmem_wait_load(o);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
                        tmem_store32(out + (uint32_t) (c * 32), o);
                    }
                    tmem_wait_store();
                }
            }
            const float ref = top == -kInf ? 0.0f : top + kRescale;
            // the weights, rounded to bf16 for the product (half a step of the output's own type), over the scores; the
            // product starts with the first half of them
            const uint64_t scales = two(scale, scale), refs = two(-ref, -ref);
            uint64_t part[2] = {0, 0};  // sums of the even and the odd columns
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float2 s = apart_of(fma2(two(x[c][2 * i], x[c][2 * i + 1]), scales, refs));
                    const float a = ex2(s.x), b = ex2(s.y);
                    part[i % 2] = add2(part[i % 2], two(a, b));
                    w[i] = pack_bf16(a, b);
                }
                tmem_store16(mine + (uint32_t) (c * 16), w);
                if (c % 2 == 0) continue;
                tmem_wait_store();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&weights_full[tile][c / 2]);
            }
            const float2 total = apart_of(add2(part[0], part[1]));
            sum += total.x + total.y;
        }
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLaunchRegs));
        fence_before();
        __syncthreads();
    }
    fence_after();

    // ---- epilogue: warps 0-7, a thread per pair, 32 elements at a time
    const int bad = s_bad;
    const bool live = warp < 8 && m < rows;
    const int64_t out_row = q.start + (m0 + m) / g.group;
    const int out_head = head * g.group + (m0 + m) % g.group;
    const bool apart = s_apart != 0;
    const float scale = g.scale_log2;
    const __nv_bfloat16 * q_row = static_cast<const __nv_bfloat16 *>(g.q) + out_row * g.q_ld + (int64_t) out_head * D;
    auto each_seen = [&](auto && visit) {  // the positions of this CTA's steps that the pair sees, one after the other
        for (int t = t0; t < t1; t++)
            for (int p = span.base(t); p < span.base(t) + kKeys; p++) {
                if (!span.seen(p) || !sees(position, p, g.window, g.sinks)) continue;
                const int page = kv.table[(int64_t) seq * kv.table_ld + (p >> kv.page_shift)];
                const int64_t at = pool_offset(kv, page, p & (kv.page_size - 1), head);
                float s = 0.0f;
                for (int c = 0; c < D; c += 4) {
                    const float4 a = load4(q_row + c, true), b = load4(static_cast<const __nv_bfloat16 *>(kv.k) + at + c, true);
                    s += a.x * b.x + a.y * b.y + a.z * b.z + a.w * b.w;
                }
                visit(s * scale, at);
            }
    };
    float shift = kRescale;  // what the weights are relative to is the maximum and this
    if (live && apart && !bad) {  // pair by pair, without the positions that it does not see
        top = -kInf, shift = 0.0f;
        each_seen([&](float s, int64_t) { top = fmaxf(top, s); });
        const float ref = top == -kInf ? 0.0f : top;
        sum = 0.0f;
        each_seen([&](float s, int64_t) { sum += ex2(s - ref); });
    }
    if (ranks > 1 && live) stat[m] = make_float2(top + shift, sum);
    const bool blank = bad || position < 0;
    const float ref = top == -kInf ? 0.0f : top + shift, inv = 1.0f / sum;
    const float fill = refused_value(bad);
    constexpr int kPitch = D + 4;
    float * partial = reinterpret_cast<float *>(smem);  // [kCtaRows][kPitch], over the queries and the ring
    if (warp < 8) {
        const uint32_t out = tmem + ((uint32_t) (warp % 4 * 32) << 16) + (uint32_t) (2 * kKeys + tile * D);
        unsigned char * rows_at = query + (size_t) warp * 32 * D * 2;  // this warp's rows, over the queries
#pragma unroll 1
        for (int c = 0; c < D / 32; c++) {
            __syncwarp();
            uint32_t x[32];
            tmem_load(x, out + (uint32_t) (c * 32));
            tmem_wait_load(x);
            if (t1 == t0) {  // no step: nothing was written there
#pragma unroll
                for (int i = 0; i < 32; i++) x[i] = 0u;
            }
            if (live && apart && !bad) {
                float o[32];
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] = 0.0f;
                each_seen([&](float s, int64_t at) {
                    const float w = ex2(s - ref);
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] += w * widen(static_cast<const __nv_bfloat16 *>(kv.v)[at + c * 32 + i]);
                });
#pragma unroll
                for (int i = 0; i < 32; i++) x[i] = __float_as_uint(o[i]);
            }
            if (ranks > 1) {
                if (!live) continue;
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    *reinterpret_cast<uint4 *>(partial + m * kPitch + c * 32 + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {  // 16 bytes each, swizzled by the row: neighbours fall into different banks
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    y[e] = blank ? pack_bf16(fill, fill)
                                 : pack_bf16(__uint_as_float(x[i * 8 + e * 2]) * inv, __uint_as_float(x[i * 8 + e * 2 + 1]) * inv);
                *reinterpret_cast<uint4 *>(rows_at + lane * D * 2 + (((c * 4 + i) ^ (lane & 7)) * 16)) = make_uint4(y[0], y[1], y[2], y[3]);
            }
        }
        if (ranks == 1) {  // out by whole rows, D / 8 threads each
            __syncwarp();
            const int64_t row_offset = out_row * g.out_ld + (int64_t) out_head * D;
            const bool wide = (reinterpret_cast<uintptr_t>(g.out) | (uintptr_t) (g.out_ld * 2)) % 16 == 0;
            constexpr int kChunks = D / 8;
#pragma unroll 4
            for (int i = 0; i < kChunks; i++) {
                const int r = i * (32 / kChunks) + lane / kChunks, c = lane % kChunks;
                const int64_t at = __shfl_sync(0xffffffffu, row_offset, r);
                if (tile * kRows + warp % 4 * 32 + r >= rows) continue;
                const uint4 y = *reinterpret_cast<const uint4 *>(rows_at + r * D * 2 + ((c ^ (r & 7)) * 16));
                __nv_bfloat16 * dst = static_cast<__nv_bfloat16 *>(g.out) + at + c * 8;
                if (wide) {
                    *reinterpret_cast<uint4 *>(dst) = y;
                } else {
                    store4(dst, make_float4(bf16_lo(y.x), bf16_hi(y.x), bf16_lo(y.y), bf16_hi(y.y)), g.vec_out);
                    store4(dst + 4, make_float4(bf16_lo(y.z), bf16_hi(y.z), bf16_lo(y.w), bf16_hi(y.w)), g.vec_out);
                }
            }
        }
        if (live && ranks == 1 && g.lse)
            g.lse[out_row * g.q_heads + out_head] = blank ? -kInf : (top == -kInf ? 0.0f : top) * kLn2 + logf(shift > 0.0f ? sum * 256.0f : sum);
        fence_before();
    }
    int refused = bad;
    if (ranks > 1) {
        const Partial mine{partial, kPitch, stat, share, &s_bad};
        refused = join_cluster(
            mine, rows, D,
            [&](int r, int c, float4 o) {
                if (first + (m0 + r) / g.group < 0) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                store4(static_cast<__nv_bfloat16 *>(g.out) + (int64_t) (q.start + (m0 + r) / g.group) * g.out_ld +
                           (int64_t) (head * g.group + (m0 + r) % g.group) * D + c, o, g.vec_out);
            },
            [&](int r, float lse) {
                if (g.lse)
                    g.lse[(int64_t) (q.start + (m0 + r) / g.group) * g.q_heads + head * g.group + (m0 + r) % g.group] =
                        first + (m0 + r) / g.group < 0 ? -kInf : lse;
            });
    } else {
        __syncthreads();
    }
    if (rank == 0 && tid == 0) raise_status(kv, seq, refused);
    statuses_cleared();
    if (warp == 9) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemColumns) : "memory");
    }
}

template <int D>
cudaError_t launch(const AttendArgs & a, int sm_count, cudaStream_t stream) {
    CUtensorMap maps[2];
    const int box = std::min(a.kv.page_size, kKeys);
    if (!page_maps(maps, a.kv, D, box, 1, 2)) return cudaErrorInvalidValue;
    const void * kernel = (const void *) prompt_kernel<D>;
    const size_t smem = (size_t) 2 * kRows * D * 2 + (size_t) slots<D>() * slot_bytes<D>() + 1024;
    static_assert((size_t) kCtaRows * (D + 4) * 4 <= (size_t) 2 * kRows * D * 2 + (size_t) slots<D>() * slot_bytes<D>(), "the partials fit");
    cudaError_t e = set_max_dynamic_smem(kernel, smem);
    if (e != cudaSuccess) return e;
    int row_blocks = (int) (((int64_t) a.kv.max_rows * a.group + kCtaRows - 1) / kCtaRows);
    const int64_t units = (int64_t) row_blocks * a.kv.kv_heads * a.kv.seqs;
    const int64_t reach = a.window > 0 ? std::min<int64_t>(a.kv.max_length, (int64_t) a.window + a.sinks + kCtaRows) : a.kv.max_length;
    int split = 1;
    while (split < 8 && units * split * 2 <= sm_count && (int64_t) split * 2 * kKeys <= reach) split *= 2;
    if (units * split > INT32_MAX) return cudaErrorInvalidValue;
    AttendArgs args = a;
    void * params[] = {&maps[0], &maps[1], &args, &row_blocks};
    return launch_cluster(kernel, (unsigned) (units * split), split, kThreads, smem, stream, params, &a.kv);
}

}  // namespace

bool attend_prompt_takes(const AttendArgs & a) { return tma_takes(a, 2); }

cudaError_t launch_attend_prompt(const AttendArgs & a, int sm_count, cudaStream_t stream) {
    return a.kv.head_dim == 64 ? launch<64>(a, sm_count, stream) : launch<128>(a, sm_count, stream);
}

}  // namespace ssb

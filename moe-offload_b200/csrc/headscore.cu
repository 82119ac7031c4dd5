// Log-probabilities of given tokens, entropy and alternatives straight from hidden rows [T, H] and
// the LM head [V, H] (prompt scoring), without [T, V] logits in memory.
//
//   score_kernel   the product X . W^T on the tensor cores: a pair of CTAs (tcgen05 cta_group::2) makes
//                  a tile of 256 rows x up to 256 vocabulary entries, fp32 accumulators in TMEM, and
//                  consumes it where it lies: every row keeps its running softmax statistics
//                  and a list of its largest logits. A pair stays with one block of 256 rows and walks
//                  every P-th vocabulary tile; pairs of different row blocks walk the same tiles side
//                  by side, so the head is read from HBM once and from L2 after that. Up to 128 rows,
//                  where the head's bytes are the bound, every CTA works alone on tiles of 128 rows: a
//                  pair would take twice as long for the same bytes.
//                  The parts share a bound on candidates through kBins maxima a row (clear_kernel).
//   finish_kernel  one CTA per row: joins the parts, sums the leading candidates' and the target's
//                  logits again in 64 bits, exactly as the LM head does, corrects the statistics by
//                  them and orders the alternatives.
//   exact_kernel   rows whose order the candidates do not settle (near-equal logits, values that are not
//                  finite): all V logits in 64 bits. It reads the rows' number and ends when there are none.
//
// B200, head 248,320 x 3,072, as graphs: one row 242 to 250 us by the box (0.95 to 0.98 of the copy rate), 256 rows
// 337 to 360 us, 2,048 rows 2.25 to 2.7 ms by the power limit (2.20 ms at the sustained rate of the tensor cores).
// With the upper 40 % of the ids 3.3 higher 264 us, 471 us and 2.6 ms; rising by 40 from the first id to the last,
// where every tile fills the lists, 279 us, 1.56 ms and 5.2 ms.
//
// A tensor-core logit carries the rounding of H / 16 fp32 accumulations. That moves the log of the sum
// of e^logit by the probability-weighted mean of those errors, a few 1e-7; it must not move an id or a
// logit that is returned, hence the second sum. The errors go by the sums of magnitudes sum_h |x_h w_vh|,
// not by the logits: a candidate list is enough when the n-th exact logit lies above the best logit outside
// by what the accumulations may lose of kSpread times the largest such sum among the row's candidates, and by kMargin
// times the largest error seen among them. For N(0, 1) rows on a head of 248,320 x 3,072 that is 0.004 beside the
// 0.05 to 0.07 that lie between the n-th and the (n + 8)-th logit (n = 32, 20), so that hardly a row
// is left to exact_kernel. An entry outside whose magnitudes exceed those of all candidates by more than kSpread may
// be missed: nothing here has seen it.
#include <cooperative_groups.h>

#include "common.cuh"
#include "internal.h"
#include "tcgen05.cuh"
#include "toplist.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kM = 128;                // rows of X per CTA (TMEM lanes); a pair's MMA has M = 256
constexpr int kN = 256;                // vocabulary entries per tile, at most (MMA N)
constexpr int kK = 64;                 // K per stage: 128 bytes, the swizzle's width
constexpr int kThreads = 320;          // TMA warp, MMA warp, 8 epilogue warps
constexpr int kEpiWarps = 8;           // each 32 rows (its TMEM lanes) x half of the columns
constexpr int kHalves = 2;
constexpr uint32_t kABytes = kM * 128;
constexpr uint32_t kTmemCols = 512;    // two accumulators of kN columns: one fills while one is read

constexpr int kSlots = 160;            // a row's list in one part: a first tile whole (128), and 32 more
constexpr int kPad = 8;                // kept beyond n, to tell whether the order of the n is settled
constexpr int kKeep = kTopMax + kPad;  // at most
constexpr int kBins = 64;              // disjoint maxima of a row, for a bound on its keep-th largest logit
constexpr int kMaxGroup = 8;           // 256-row blocks per launch: 74 / 8 = 9 parts, 144 of 148 CTAs busy
constexpr float kMargin = 16.f, kSpread = 4.f;         // see above
constexpr int kExCluster = 8, kMaxClusters = 32;       // exact_kernel: CTAs per cluster, clusters at most

struct ScoreArgs {
    int T, V, H;                       // rows of this launch
    int blocks, parts;                 // row blocks (256 or 128 rows), vocabulary parts
    int width, xbox;                   // vocabulary entries per tile, rows of X per load
    int keep;                          // entries a list has to keep
    uint2 *lists;                      // [128-row blocks][parts][kHalves][kSlots][kM] (value, index)
    float4 *stats;                     // [128-row blocks][parts][kHalves][kM] m, s, w, entries (as int bits)
    unsigned *bins;                    // [128-row blocks][kBins][kM] order images of maxima, 0 before the launch
    int *redo;                         // [0]: rows for exact_kernel, then its counters
};

template <bool kPair>
struct ScoreSmem {
    static constexpr int kStages = kPair ? 6 : 4;
    static constexpr uint32_t kStageBytes = kABytes + (kPair ? kN / 2 : kN) * 128; // (a pair's CTAs hold half of W each)
    static constexpr size_t bars = (size_t)kStages * kStageBytes;
    // full, empty [kStages]; acc_full, acc_empty [2]; drain; TMEM slot, abort flag
    static constexpr size_t alloc = bars + (2 * kStages + 5) * 8 + 16 + 1024;
};

MOE_D void mma_bf16_ss(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

// ---- pair forms (cta_group::2): the CTA of rank 0 issues for both, its barriers collect both CTAs'
// loads and both CTAs' epilogues

// D (both CTAs' TMEM, 128 rows each) += A (128 rows in each CTA's shared memory) . B (half of the rows in
// each); the descriptors hold the offsets in either CTA
MOE_D void mma_bf16_pair(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

// arrives at the same barrier of both CTAs once the MMAs issued so far are done
MOE_D void mma_commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// at this CTA's alone
MOE_D void mma_commit_pair_local(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

// shared::cluster address of a variable of the pair's first CTA
MOE_D uint32_t first_cta_addr(const void *p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_addr(p)));
    return r;
}

// 2-D tiled load into this CTA, completing on a barrier of the pair's first CTA
MOE_D void tma_load_2d_pair(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

MOE_D void arrive_first_cta(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// 32 columns of this warp's 32 TMEM lanes; r holds them after tmem_wait (nothing may touch it before)
MOE_D void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
MOE_D void tmem_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// order-preserving image of a float that is no NaN (-0 below +0: both forms of a zero logit are
// brought to +0 before); 0 is below all
MOE_D uint32_t order_of(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

MOE_D float value_of(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }

// the largest float below an image's (the image between those of -1e-45 and +0 is that of -0, equal to
// +0); -inf for none
MOE_D float value_below(uint32_t o) { return o > 0x00800000u ? value_of(o - (o == 0x80000000u ? 2u : 1u)) : -INFINITY; }

// A row's statistics while its tiles go by, in steps of 2: sums over 2^(x log2(e) - r) with r a whole
// number near log2(e) times the largest value m, which the sums leave out (as SoftRun does). r is exact,
// rescaling by it too, and one FMA makes an exponent. The fp32 constant is 1.3e-8 off: run2_end takes m by the
// same constant, so that only the differences from m see it. (2^t overflows where the FMA and r may lie 128
// apart: logits from 2^30 on.)
struct Run2 {
    float m, r, s, w;                  // w: sum of t 2^t, t the exponents
};
// 32 values, top their largest (NaN left out). Columns that are not there hold kAbsent, not -inf: 0 x inf
// would be NaN (and is, for a logit that is -inf). Where the largest value changes, the old one takes the
// place of the new one among the values.
constexpr float kAbsent = -1e30f;
MOE_D void run2_add(Run2 &a, uint32_t (&x)[32], float top) {
    float s[4] = {a.s, 0.f, 0.f, 0.f}, w[4] = {a.w, 0.f, 0.f, 0.f};
    if (__any_sync(0xffffffffu, top > a.m)) {
        bool more = top > a.m;
        const float old = fmaxf(a.m, kAbsent), want = floorf(top * kLog2e);
        if (more && !(want <= a.r + 40.f && a.m > -INFINITY)) {
            const float d = a.m > -INFINITY ? fmaxf(a.r - want, kSoftFar) : 0.f, f = fast_pow2(d);
            w[0] = f * (w[0] + d * s[0]);
            s[0] *= f;                            // (nothing in the sums yet: 0, or NaN)
            a.r = want;
        }
        if (more) a.m = top;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const bool here = more && __uint_as_float(x[i]) == top;
            x[i] = here ? __float_as_uint(old) : x[i];
            more = more && !here;
        }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const float t = fmaf(__uint_as_float(x[i]), kLog2e, -a.r), e = fast_pow2(t);
        s[i & 3] += e;
        w[i & 3] = fmaf(t, e, w[i & 3]);
    }
    a.s = (s[0] + s[1]) + (s[2] + s[3]);
    a.w = (w[0] + w[1]) + (w[2] + w[3]);
}

MOE_D Soft run2_end(const Run2 &a) {
    if (a.m == -INFINITY) return Soft{a.m, a.s, 0.f};
    const float ln2 = 0.6931471805599453f;
    // r and m on the same scale, that of the rounded log2(e)
    const float d = (float)(((double)a.r - (double)a.m * (double)kLog2e) * 0.6931471805599453), f = expf(d);
    return Soft{a.m, f * a.s, f * fmaf(ln2, a.w, d * a.s)};
}

// A bound that at least keep of the row's logits reach, from its maxima so far in kBins disjoint sets
// of vocabulary entries (kM apart): their keep-th largest, or a little less. 0: fewer maxima than that.
MOE_D uint32_t bins_bound(const uint32_t (&o)[kBins], int keep) {
    uint32_t lo = 0xffffffffu, hi = 0u;
    int reach = 0;
#pragma unroll
    for (int i = 0; i < kBins; ++i) {
        hi = max(hi, o[i]);
        lo = min(lo, o[i] - 1u);                  // (0 - 1: the largest)
        reach += o[i] ? 1 : 0;
    }
    if (reach < keep) return 0u;
    // reach >= keep bins reach lo, fewer reach hi
    lo += 1u;
    hi += 1u;
#pragma unroll 1
    while (reach > keep + 4 && hi - lo > 1u) {
        const uint32_t mid = lo + (hi - lo) / 2u;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kBins; ++i) n += o[i] >= mid ? 1 : 0;
        if (n >= keep) {
            lo = mid;
            reach = n;
        } else {
            hi = mid;
        }
    }
    return lo;
}

// A row's list cut to its keep largest entries (equal ones: the lower index), in their order, by the whole
// warp: list is the row's own, of n >= keep entries. Returns the smallest value kept. What is dropped, and what
// comes later and does not exceed that value, has keep entries of this list before it, so it is none of the
// row's keep largest. Out of line: few rows need it (a part's entries above the bound outnumber its list: a
// vocabulary in blocks or in order, or a first tile before the other parts have told their maxima).
__device__ __noinline__ float cut_list(uint2 *list, int n, int keep) {
    constexpr int kPer = kSlots / 32;
    const int lane = threadIdx.x & 31;
    uint2 e[kPer];
    uint32_t o[kPer];
    __syncwarp();                                 // the row's lane has written its entries
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = lane + 32 * i;
        e[i] = at < n ? list[at * kM] : make_uint2(0u, 0u);
        o[i] = at < n ? order_of(__uint_as_float(e[i].x)) : 0u;
    }
    uint32_t t = 0u;                              // the largest image that keep entries reach
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t u = t | (1u << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) c += o[i] >= u ? 1 : 0;
        if (__reduce_add_sync(0xffffffffu, c) >= keep) t = u;
    }
    int over = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) over += o[i] > t ? 1 : 0;
    int ties = keep - __reduce_add_sync(0xffffffffu, over), to = 0;
    const unsigned before = (1u << lane) - 1u;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {              // (all entries are in registers: they may move up in place)
        const unsigned equal = __ballot_sync(0xffffffffu, o[i] == t);
        const bool in = o[i] > t || (o[i] == t && __popc(equal & before) < ties);
        ties -= min(ties, __popc(equal));
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (in) list[(to + __popc(who & before)) * kM] = e[i];
        to += __popc(who);
    }
    __syncwarp();
    return value_of(t);
}

// Clears the bins and lets score_kernel start meanwhile: only its epilogue needs them.
__global__ void clear_kernel(uint4 *bins) {
    pdl_launch_dependents();
    bins[blockIdx.x * blockDim.x + threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
}

template <bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    score_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, ScoreArgs a) {
    using SL = ScoreSmem<kPair>;
    constexpr int kStages = SL::kStages, kCtas = kPair ? 2 : 1;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + SL::bars);
    uint64_t *empty = full + kStages;
    uint64_t *acc_full = empty + kStages;
    uint64_t *acc_empty = acc_full + 2;
    uint64_t *drain = acc_empty + 2;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(drain + 1);
    // set by the first failed wait of any role of the CTA: the others stop, and what was issued is drained
    volatile int *abort = reinterpret_cast<volatile int *>(tslot + 1);
    cg::cluster_group pair = cg::this_cluster();
    const int rank = kPair ? (int)pair.block_rank() : 0;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);          // (known to be uniform)
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 1);              // (used in a pair's first CTA)
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], kCtas * kEpiWarps);         // (in the first CTA, by both)
        }
        mbar_init(drain, 1);
        *abort = 0;
        fence_barrier_init();
        if (kPair) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (blockIdx.x == 0)
            for (int i = 0; i <= kMaxClusters; ++i) a.redo[i] = 0;
    }
    if (warp == 1) {
        if (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tslot)),
                         "r"(kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tslot)),
                         "r"(kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        }
    }
    {
        // rows of X that no load will fill: zeros (their results are not read, but the tensor cores spend power
        // on what is there)
        const int row0 = (blockIdx.x / kCtas % a.blocks * kCtas + rank) * kM;
        const int from = min(max((a.T - row0 + a.xbox - 1) / a.xbox, 0) * a.xbox, kM) * 128;
        for (int s = 0; s < kStages; ++s)
            for (int i = from + 16 * tid; i < (int)kABytes; i += 16 * kThreads)
                *reinterpret_cast<uint4 *>(smem + (size_t)s * SL::kStageBytes + i) = make_uint4(0u, 0u, 0u, 0u);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    if (kPair) pair.sync();                      // both CTAs' barriers are there
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    const int unit = blockIdx.x / kCtas, block = unit % a.blocks, part = unit / a.blocks;
    const int tiles = (a.V + a.width - 1) / a.width, nkb = (a.H + kK - 1) / kK;

    // The two control warps run in step with one lane elected to issue, and with the stages unrolled: beside
    // eight busy epilogue warps their own instructions are what limits them (512 cycles a K block)
    if (warp == 0) {
        // ---- TMA, in each CTA for its own shared memory: 128 rows of X and the tile's rows of W (a pair: half of
        // them). Rows and columns of a box outside the arrays arrive as zeros, which costs
        // the TMA unit as much as data (one row in a box of 128 made the one-row case 1.4 times slower):
        // a few rows come in boxes of 32, and boxes of X wholly outside are left as they are
        const int row0 = (block * kCtas + rank) * kM;
        auto boxes = [&](int r0) { return min(max((a.T - r0 + a.xbox - 1) / a.xbox, 0), kM / a.xbox); };
        const int nx = boxes(row0), wrows = a.width / kCtas;
        uint32_t bytes = (uint32_t)nx * a.xbox * 128u + (uint32_t)wrows * 128u;
        if (kPair)                               // the first CTA's barrier counts both CTAs' bytes
            bytes = (uint32_t)(boxes(block * 2 * kM) + boxes(block * 2 * kM + kM)) * a.xbox * 128u + (uint32_t)a.width * 128u;
        const uint32_t full0 = kPair ? first_cta_addr(full) : smem_addr(full);
        const int kend = nkb * kK;
        uint32_t phase = 1, g = 0;
        int v = part, x = 0;
        bool stop = v >= tiles;
        while (!stop) {
#pragma unroll
            for (int s = 0; s < kStages; ++s) {
                if (stop) continue;
                if (!wait_or_abort_step(&empty[s], phase, abort)) {
                    stop = true;
                    continue;
                }
                if (elect_lane()) {
                    unsigned char *st = smem + (size_t)s * SL::kStageBytes;
                    const int w0 = v * a.width + rank * wrows;
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
                    if (kPair) {
                        tma_load_2d_pair(st + kABytes, &map_w, x, w0, full0 + 8u * s);
                        for (int i = 0; i < nx; ++i)
                            tma_load_2d_pair(st + (size_t)i * a.xbox * 128, &map_x, x, row0 + i * a.xbox, full0 + 8u * s);
                    } else {
                        tma_load_2d(st + kABytes, &map_w, x, w0, &full[s]);
                        for (int i = 0; i < nx; ++i)
                            tma_load_2d(st + (size_t)i * a.xbox * 128, &map_x, x, row0 + i * a.xbox, &full[s]);
                    }
                }
                __syncwarp();
                ++g;
                x += kK;
                if (x >= kend) {
                    x = 0;
                    v += a.parts;
                    stop = v >= tiles;
                }
            }
            phase ^= 1u;
        }
        // nothing may still arrive here when the CTA ends: the last round's releases (each follows the
        // loads and MMAs of its stage), or after an abort the loads themselves
        if (!aborted(abort)) {
            for (uint32_t i = g > (uint32_t)kStages ? g - kStages : 0u; i < g; ++i)
                if (!wait_or_abort_step(&empty[i % kStages], (i / kStages) & 1u, abort)) break;
        } else if (rank == 0) {
            for (uint32_t i = g > (uint32_t)kStages ? g - kStages : 0u; i < g; ++i)
                mbar_wait(&full[i % kStages], (i / kStages) & 1u);
        }
    } else if (warp == 1 && rank == 0) {
        // ---- MMA (a pair's first CTA issues for both)
        const uint32_t idesc = instr_desc_bf16(kCtas * kM, a.width);
        const uint64_t desc0 = desc_sw128(smem_addr(smem));         // (16-byte units in the low bits)
        uint32_t phase = 0, it = 0;
        int v = part, kb = 0;
        bool stop = v >= tiles, issued = false;
        while (!stop) {
#pragma unroll
            for (int s = 0; s < kStages; ++s) {
                if (stop) continue;
                const uint32_t b = it & 1u;
                if (kb == 0 && !wait_or_abort_step(&acc_empty[b], ((it >> 1) & 1u) ^ 1u, abort)) {
                    stop = true;
                    continue;
                }
                if (!wait_or_abort_step(&full[s], phase, abort)) {
                    stop = true;
                    continue;
                }
                tc_fence_after();
                const bool last = kb + 1 == nkb;
                if (elect_lane()) {
                    const uint64_t da = desc0 + (s * SL::kStageBytes) / 16u, db = da + kABytes / 16u;
                    const uint32_t d = tmem + b * kN;
#pragma unroll
                    for (int j = 0; j < kK / 16; ++j) {
                        if (kPair) mma_bf16_pair(d, da + 2u * j, db + 2u * j, idesc, j > 0 ? 1u : (uint32_t)kb);
                        else mma_bf16_ss(d, da + 2u * j, db + 2u * j, idesc, j > 0 ? 1u : (uint32_t)kb);
                    }
                    if (kPair) mma_commit_pair(&empty[s]);
                    else mma_commit(&empty[s]);
                    if (last) {
                        if (kPair) mma_commit_pair(&acc_full[b]);
                        else mma_commit(&acc_full[b]);
                    }
                }
                __syncwarp();
                issued = true;
                ++kb;
                if (last) {
                    kb = 0;
                    ++it;
                    v += a.parts;
                    stop = v >= tiles;
                }
            }
            phase ^= 1u;
        }
        if (aborted(abort) && issued) {
            if (elect_lane()) {
                if (kPair) mma_commit_pair_local(drain);
                else mma_commit(drain);
            }
            __syncwarp();
            mbar_wait(drain, 0);
        }
    } else if (warp >= 2) {
        // ---- epilogue: thread = row, the tile's columns 0 .. 127 or the rest
        pdl_wait();                              // the bins are clear
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int cols = half ? a.width - kN / 2 : min(a.width, kN / 2);
        const int mblock = block * kCtas + rank, lrow = quarter * 32 + lane, row = mblock * kM + lrow;
        const int slice = (mblock * a.parts + part) * kHalves + half;
        uint2 *list = a.lists + (size_t)slice * kSlots * kM + lrow;
        unsigned *bins = a.bins + (size_t)mblock * kBins * kM + lrow;
        const bool any = mblock * kM + quarter * 32 < a.T;          // a row of this warp is there
        constexpr int kSets = kN / 2 / 32;
        Run2 run{-INFINITY, 0.f, 0.f, 0.f};
        float least = row < a.T ? kAbsent : INFINITY;                // appended: what is above it
        float reach = INFINITY;                  // the bound that the entries from base on all reach
        int count = 0, base = 0;
        float tops[kSets], told[kSets];          // largest values of the four sets of 32 columns; last told
#pragma unroll
        for (int j = 0; j < kSets; ++j) tops[j] = told[j] = -INFINITY;
        uint32_t it = 0;
        for (int v = part; v < tiles; v += a.parts, ++it) {
            const uint32_t b = it & 1u;
            if (aborted(abort) || !wait_or_abort(&acc_full[b], (it >> 1) & 1u, abort)) break;
            tc_fence_after();
            const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + b * kN + half * (kN / 2);
            const int col0 = v * a.width + half * (kN / 2);
            const int inside = min(cols, a.V - col0);               // columns that are there
            auto mask = [&](int j, uint32_t (&x)[32]) {
                if (32 * j + 32 > inside) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (32 * j + i >= inside) x[i] = __float_as_uint(kAbsent);
                }
            };
            auto tell = [&]() {
                if (row >= a.T) return;
#pragma unroll
                for (int j = 0; j < kSets; ++j) {
                    if (tops[j] > told[j])
                        atomicMax(&bins[(((part * kHalves + half) * kSets + j) % kBins) * kM], order_of(tops[j] + 0.f));
                    told[j] = tops[j];
                }
            };
            // Before the tiles 0, 1, 4, 16, .. each part takes a bound on what is worth a place in its list from
            // the row's maxima that the parts have told each other. It may miss what others have just
            // told: any such bound is a valid one, and the entries above the last are there in any case.
            auto look = [&]() {
                uint32_t o[kBins];
#pragma unroll
                for (int i = 0; i < kBins; ++i) o[i] = __ldcg(&bins[i * kM]);
                const uint32_t bound = bins_bound(o, a.keep);
                const float below = value_below(bound);
                if (below > least) {
                    least = below;                                   // (those equal to the bound: by index)
                    reach = value_of(bound);
                    base = count;
                }
            };
            // a set of columns: statistics (pass 0, 2), candidates (pass 1, 2)
            auto take = [&](int j, uint32_t (&x)[32], int pass) {
                mask(j, x);
                float top[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = __uint_as_float(x[16 * h]);
#pragma unroll
                    for (int i = 1; i < 16; ++i) top[h] = fmaxf(top[h], __uint_as_float(x[16 * h + i]));
                    if (pass != 0 && __any_sync(0xffffffffu, top[h] > least)) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float value = __uint_as_float(x[16 * h + i]);
                            if (value > least) {                    // (+ 0: no -0 in a list)
                                list[count * kM] = make_uint2(__float_as_uint(value + 0.f),
                                                              (uint32_t)(col0 + 32 * j + 16 * h + i));
                                ++count;
                            }
                        }
                        // keep entries that reach the bound: more that only equal it come behind them by index
                        if (count - base >= a.keep) least = fmaxf(least, reach < INFINITY ? reach : kAbsent);
                    }
                }
                // 32 more have to fit
                for (unsigned full = __ballot_sync(0xffffffffu, count > kSlots - 32); full;
                     full &= full - 1) {
                    const int of = __ffs(full) - 1;
                    const float bound = cut_list(list + (of - lane), __shfl_sync(0xffffffffu, count, of), a.keep);
                    if (lane == of) {
                        count = base = a.keep;
                        least = fmaxf(least, bound);
                    }
                }
                if (pass != 1) run2_add(run, x, fmaxf(top[0], top[1]));
                return fmaxf(top[0], top[1]);
            };
            if (any && inside > 0) {
                uint32_t xa[32], xb[32];
                // the first tile: its maxima are told, its statistics taken while the others tell theirs, and
                // its candidates only then
                int pass = 2;
                if (it == 0) {
#pragma unroll
                    for (int j = 0; j < kSets; ++j) {
                        tmem_ld32(taddr + 32 * j, xa);
                        tmem_wait(xa);
                        mask(j, xa);
#pragma unroll
                        for (int i = 0; i < 32; ++i) tops[j] = fmaxf(tops[j], __uint_as_float(xa[i]));
                        if (32 * j >= inside) tops[j] = -INFINITY;
                    }
                    tell();
                    pass = 0;
                } else if ((it & (it - 1u)) == 0u && (it & 0x55555555u)) {
                    look();
                }
#pragma unroll 1
                for (;; pass = 1) {
                    if (pass == 1) look();
                    // the next set is on its way while one is taken
                    tmem_ld32(taddr, xa);
#pragma unroll 1
                    for (int j = 0; 32 * j < inside; j += 2) {
                        tmem_wait(xa);
                        tmem_ld32(taddr + 32 * (j + 1), xb);
                        const float ta = take(j, xa, pass);
                        tmem_wait(xb);
                        if (j + 2 < kSets) tmem_ld32(taddr + 32 * (j + 2), xa);
                        const float tb = 32 * (j + 1) < inside ? take(j + 1, xb, pass) : -INFINITY;
#pragma unroll
                        for (int k = 0; k < kSets; ++k)
                            tops[k] = fmaxf(tops[k], k == j ? ta : k == j + 1 ? tb : -INFINITY);
                    }
                    tmem_wait(xa);
                    if (pass != 0) break;
                }
                if ((it & (it + 1u)) == 0u && ((it + 1u) & 0x55555555u)) tell();     // the next tile looks
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (kPair) arrive_first_cta(first_cta_addr(&acc_empty[b]));
                else mbar_arrive(&acc_empty[b]);
            }
        }
        if (row < a.T) {
            const Soft s = run2_end(run);
            a.stats[(size_t)slice * kM + lrow] = make_float4(s.m, s.s, s.w, __int_as_float(count));
        }
    }
    __syncwarp();
    tc_fence_before();
    if (kPair) pair.sync();                      // neither CTA's memory goes while the other may reach it
    else __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        if (kPair)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

// ------------------------------------------------------------------ exact logits

// x as floats: the elements 8 c .. 8 c + 3 of every chunk c of 8, then the elements 8 c + 4 .. 8 c + 7, so
// that a warp's 16-byte reads of consecutive chunks do not meet in a bank
MOE_D void stage_row(const uint16_t *x, int H, float4 *xs) {
    const int nch = H / 8;
    for (int c = threadIdx.x; c < nch; c += blockDim.x) {
        const uint4 q = __ldg(reinterpret_cast<const uint4 *>(x) + c);
        xs[c] = make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16),
                            __uint_as_float(q.y & 0xffff0000u));
        xs[nch + c] = make_float4(__uint_as_float(q.z << 16), __uint_as_float(q.z & 0xffff0000u),
                                  __uint_as_float(q.w << 16), __uint_as_float(q.w & 0xffff0000u));
    }
}

// A warp's dot product of a head row with the staged row: the products (exact in fp32) summed in
// 64 bits in the LM head's order, rounded once. size: the sum of their magnitudes.
template <bool kSize>
MOE_D float exact_logit(const uint16_t *w, const float4 *xs, int H, float &size) {
    const int lane = threadIdx.x & 31, nch = H / 8;
    const uint4 *wr = reinterpret_cast<const uint4 *>(w);
    double acc = 0.0;
    float mag = 0.f;
    auto add = [&](float p) {
        acc += (double)p;
        if (kSize) mag += fabsf(p);
    };
#pragma unroll 4
    for (int c = lane; c < nch; c += 32) {
        const uint4 q = __ldg(wr + c);
        const float4 a = xs[c], b = xs[nch + c];
        add(__uint_as_float(q.x << 16) * a.x);
        add(__uint_as_float(q.x & 0xffff0000u) * a.y);
        add(__uint_as_float(q.y << 16) * a.z);
        add(__uint_as_float(q.y & 0xffff0000u) * a.w);
        add(__uint_as_float(q.z << 16) * b.x);
        add(__uint_as_float(q.z & 0xffff0000u) * b.y);
        add(__uint_as_float(q.w << 16) * b.z);
        add(__uint_as_float(q.w & 0xffff0000u) * b.w);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        acc += __shfl_xor_sync(0xffffffffu, acc, off);
        if (kSize) mag += __shfl_xor_sync(0xffffffffu, mag, off);
    }
    if (kSize) size = mag;
    return (float)acc;
}
MOE_D float exact_logit(const uint16_t *w, const float4 *xs, int H) {
    float none;
    return exact_logit<false>(w, xs, H, none);
}

// ------------------------------------------------------------------ one row's parts joined

constexpr int kCand = 1024;            // candidates that are ranked at once
constexpr int kMaxLists = 512;         // lists of a row, at most
constexpr int kGroups = 64;            // disjoint sets of entries whose maxima bound the candidates

struct FinishArgs {
    const uint16_t *head, *x;          // x: this launch's first row
    int V, H, n;
    int parts, keep;
    const uint2 *lists;
    const float4 *stats;
    const int32_t *targets;
    float *logprob, *entropy;
    int32_t *top_ids;
    float *top_logprobs;
    int *redo;                         // [0] count, counters of exact_kernel, (row, bits of m, bits of lse - m) ..
};

// Candidates where more than kCand entries reach tau: those above a bound on (value, index). Out of line: rows of
// ties (a padded batch) and lists whose large entries lie in few places need it.
template <int kT>
__device__ __noinline__ void recollect(const uint2 *lists, const int *counts, int nlists, float tau, int keep,
                                       unsigned long long *cand, int *ncand, unsigned long long *shared_bound) {
    constexpr int kW = kT / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto entries = [&](auto &&f) {
        for (int l = warp; l < nlists; l += kW)
#pragma unroll
            for (int i = 0; i < kSlots / 32; ++i) {
                const uint2 e = lane + 32 * i < counts[l] ? lists[((size_t)l * kSlots + lane + 32 * i) * kM]
                                                          : make_uint2(0xff800000u, 0u);           // -inf
                const float value = __uint_as_float(e.x);
                if (value >= tau && value > -INFINITY) f(top_key(value, (int)e.y));
            }
    };
    auto collect = [&](unsigned long long bound) {
        __syncthreads();                         // (ncand has been read)
        if (tid == 0) *ncand = 0;
        __syncthreads();
        entries([&](unsigned long long k) {
            if (k < bound) return;
            const int at = atomicAdd(ncand, 1);
            if (at < kCand) cand[at] = k;
        });
        __syncthreads();
    };
    // the keep-th largest of the threads' best entries
    unsigned long long best = 0ull;
    entries([&](unsigned long long k) { best = k > best ? k : best; });
    __syncthreads();
    cand[tid] = best;
    __syncthreads();
    int r = 0;
    for (int j = 0; j < kT; ++j) r += (cand[j] > best || (cand[j] == best && j < tid)) ? 1 : 0;
    if (r == keep - 1) *shared_bound = best;
    __syncthreads();
    collect(*shared_bound);
    if (*ncand <= kCand) return;
    // crowded in a few threads: a bound bit by bit, which keep to kCand keys reach (they differ)
    unsigned long long bound = 0ull;
    int reach = 0;
    for (int bit = 63; bit >= 0 && !(reach >= keep && reach <= kCand); --bit) {
        const unsigned long long u = bound | (1ull << bit);
        int c = 0;
        entries([&](unsigned long long k) { c += k >= u ? 1 : 0; });
        c = __reduce_add_sync(0xffffffffu, c);
        __syncthreads();
        if (tid == 0) *ncand = 0;
        __syncthreads();
        if (lane == 0) atomicAdd(ncand, c);
        __syncthreads();
        if (*ncand >= keep) {
            bound = u;
            reach = *ncand;
        }
    }
    collect(bound);
}

// kT: 512 threads for few rows (latency), 128 for many (the rows' own instructions are the bound then:
// 98 us for 2,048 rows, 116 with 512)
template <int kT>
__global__ void __launch_bounds__(kT) finish_kernel(FinishArgs p) {
    constexpr int kW = kT / 32;
    extern __shared__ float4 xs[];                                  // the row (stage_row)
    __shared__ unsigned long long cand[kCand], lead[kKeep];
    __shared__ float peaks[kMaxLists], groups[kGroups], exact[kKeep + 1], sizes[kW];
    __shared__ unsigned long long bound_s;
    __shared__ int counts[kMaxLists];
    __shared__ Soft softs[kW];
    __shared__ float tau_s;
    __shared__ int ncand;
    const int row = blockIdx.x, block = row / kM, lrow = row % kM;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nlists = p.parts * kHalves;
    const float4 *stats = p.stats + (size_t)block * nlists * kM + lrow;
    const uint2 *lists = p.lists + (size_t)block * nlists * kSlots * kM + lrow;
    stage_row(p.x + (size_t)row * p.H, p.H, xs);
    pdl_launch_dependents();
    pdl_wait();                                                     // score_kernel's lists and statistics
    if (tid == 0) {
        ncand = 0;
        tau_s = -INFINITY;
    }
    __syncthreads();

    // statistics, in a fixed order
    Soft st = soft_none();
    for (int l = tid; l < nlists; l += kT) {
        const float4 f = stats[(size_t)l * kM];
        st = soft_merge(st, Soft{f.x, f.y, f.z});
        peaks[l] = f.x;
        counts[l] = min(__float_as_int(f.w), kSlots);
    }
    st = soft_warp(st);
    if (lane == 0) softs[warp] = st;
    __syncthreads();

    // the leading candidates: the keep-th largest of kGroups disjoint maxima is a bound that keep entries
    // reach. With enough lists their own maxima do, and only the lists that reach the bound are read;
    // else those of the threads, which hold the entries of 2 lists a warp
    constexpr int kPer = kSlots / 32;
    const bool by_list = nlists >= 2 * p.keep;
    uint2 held[2][kPer];
    auto load_list = [&](int l, uint2 (&e)[kPer]) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            e[i] = l < nlists && lane + 32 * i < counts[l] ? lists[((size_t)l * kSlots + lane + 32 * i) * kM]
                                                           : make_uint2(0xff800000u, 0u);          // -inf
    };
    if (by_list) {
        if (tid < kGroups) {
            float top = tid < nlists ? peaks[tid] : -INFINITY;
            for (int l = tid + kGroups; l < nlists; l += kGroups) top = fmaxf(top, peaks[l]);
            groups[tid] = top;
        }
    } else {
        float top = -INFINITY;
        for (int l = warp; l < nlists; l += 2 * kW) {
            load_list(l, held[0]);
            load_list(l + kW, held[1]);
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                top = fmaxf(top, fmaxf(__uint_as_float(held[0][i].x), __uint_as_float(held[1][i].x)));
        }
#pragma unroll
        for (int off = kT / kGroups / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (tid % (kT / kGroups) == 0) groups[tid / (kT / kGroups)] = top;
    }
    __syncthreads();
    if (tid < kGroups) {
        const float mine = groups[tid];
        int r = 0;
#pragma unroll 16
        for (int j = 0; j < kGroups; ++j) r += (groups[j] > mine || (groups[j] == mine && j < tid)) ? 1 : 0;
        if (r == p.keep - 1) tau_s = mine;
    }
    st = soft_warp(lane < kW ? softs[lane] : soft_none());
    __syncthreads();
    const float tau = tau_s;
    const bool one_round = nlists <= 2 * kW;                         // held still has all entries
    // every entry that may reach tau
    for (int l = warp; l < nlists; l += 2 * kW) {
        if (by_list || !one_round) {
            const bool a = !by_list || peaks[l] >= tau;
            const bool b = l + kW < nlists && (!by_list || peaks[l + kW] >= tau);
            if (!a && !b) continue;
            load_list(a ? l : nlists, held[0]);
            load_list(b ? l + kW : nlists, held[1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const float value = __uint_as_float(held[h][i].x);
                if (value >= tau && value > -INFINITY) {
                    const int at = atomicAdd(&ncand, 1);
                    if (at < kCand) cand[at] = top_key(value, (int)held[h][i].y);
                }
            }
    }
    __syncthreads();
    if (ncand > kCand) recollect<kT>(lists, counts, nlists, tau, p.keep, cand, &ncand, &bound_s);
    const int have = ncand;
    for (int i = tid; i < have; i += kT) {
        const unsigned long long k = cand[i];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < have; ++j) r += cand[j] > k ? 1 : 0;
        if (r < p.keep) lead[r] = k;
    }
    __syncthreads();

    // the leading ones' and the target's logits again, in 64 bits
    const int lead_n = min(have, p.keep);
    const int target = p.targets ? p.targets[row] : -1;
    const bool has_target = target >= 0 && target < p.V;
    float widest = 0.f;                          // the largest sum of magnitudes behind a leading one
    for (int i = warp; i <= lead_n; i += kW) {
        const int id = i < lead_n ? top_index(lead[i]) : target;
        const bool in = id >= 0 && id < p.V;
        float mine = 0.f;
        const float l = in ? exact_logit<true>(p.head + (size_t)id * p.H, xs, p.H, mine) : 0.f;
        if (lane == 0) exact[i] = l;
        if (i < lead_n) widest = fmaxf(widest, mine);
    }
    if (lane == 0) sizes[warp] = widest;
    __syncthreads();
    if (warp != 0) return;
    widest = lane < kW ? sizes[lane] : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) widest = fmaxf(widest, __shfl_xor_sync(0xffffffffu, widest, off));
    // Each of the tensor cores' H / 16 steps loses at most 2^-23 of what it holds
    const float loss = (float)((p.H + 15) / 16) * 1.1920929e-7f;

    // Statistics relative to the exact logit of the leading candidate, which they leave out, with the
    // others' exact logits in place of the tensor cores'. The tensor cores' accumulation rounds towards zero:
    // logits come out smaller by a share that the candidates show (rho, some 1e-6), and the sums over
    // the rest are moved by it to first order: sum a e^(a - m) is known, and the entropy's sum takes the
    // rest's mean for its values.
    float err = 0.f, gain = 0.f, size = 0.f;
    Soft sum{0.f, 0.f, 0.f}, near_sum{0.f, 0.f, 0.f};
    const bool fine = st.m < INFINITY && st.m > -INFINITY && st.s < INFINITY && st.w > -INFINITY && lead_n > 0;
    if (fine) {
        sum.m = exact[0];
        for (int i = lane; i < lead_n; i += 32) {
            const float near = top_value(lead[i]), x = exact[i];
            err = fmaxf(err, fabsf(x - near));
            if (i > 0) {
                gain += near < 0.f ? near - x : x - near;
                size += fabsf(near);
                const float dx = fmaxf(x - sum.m, kSoftFar), dn = fmaxf(near - sum.m, kSoftFar);
                const float ex = expf(dx), en = expf(dn);
                sum.s += ex;
                sum.w += dx * ex;
                near_sum.s += en;
                near_sum.w += dn * en;
            }
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            sum.s += __shfl_xor_sync(0xffffffffu, sum.s, off);
            sum.w += __shfl_xor_sync(0xffffffffu, sum.w, off);
            near_sum.s += __shfl_xor_sync(0xffffffffu, near_sum.s, off);
            near_sum.w += __shfl_xor_sync(0xffffffffu, near_sum.w, off);
            gain += __shfl_xor_sync(0xffffffffu, gain, off);
            size += __shfl_xor_sync(0xffffffffu, size, off);
            err = fmaxf(err, __shfl_xor_sync(0xffffffffu, err, off));
        }
        const float d = st.m - sum.m, f = expf(d);
        const float rs = fmaf(f, st.s, -near_sum.s), rw = f * (st.w + d * st.s) - near_sum.w;     // the rest
        if (rs > 0.f) {
            // A share larger than the loss is no share: the candidates' sums cancel, their errors have nothing to
            // do with their size, and the rest stays.
            const float rho = fabsf(gain) <= loss * size && size > 0.f ? gain / size : 0.f;
            const float moved = rho * fmaf(sum.m, rs, rw);
            sum.s += rs + moved;
            sum.w += rw + moved * (1.f + rw / rs);
        }
    } else {
        sum.m = __int_as_float(0x7fffffff);
    }
    const float rest = soft_log_rest(sum);
    if (lane == 0) {
        p.entropy[row] = soft_entropy(sum);
        if (p.targets) {
            if (!has_target && target != -1) atomicOr(&g_moe_device_error, MOE_DEVERR_BAD_INPUT);
            p.logprob[row] = has_target ? (exact[lead_n] - sum.m) - rest : __int_as_float(0x7fffffff);
        }
    }
    if (p.n == 0) return;
    // order by the exact logits (lead_n <= 64 entries: two a lane)
    unsigned long long key[2], nth = 0ull;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = lane + 32 * h;
        key[h] = i < lead_n ? top_key(exact[i], top_index(lead[i])) : 0ull;
    }
    int rank[2] = {0, 0};
    for (int j = 0; j < lead_n; ++j) {
        const unsigned long long o = __shfl_sync(0xffffffffu, key[j >> 5], j & 31);
        rank[0] += o > key[0] ? 1 : 0;
        rank[1] += o > key[1] ? 1 : 0;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned who = __ballot_sync(0xffffffffu, key[h] != 0ull && rank[h] == p.n - 1);
        if (who) nth = __shfl_sync(0xffffffffu, key[h], __ffs(who) - 1);
    }
    // settled: there is nothing outside the candidates, or it cannot reach the n-th (a row of zeros: no error)
    const float outside = lead_n > 0 ? top_value(lead[lead_n - 1]) : INFINITY;
    const float margin = fmaxf(kMargin * err, kSpread * loss * widest);
    const bool settled = fine && lead_n >= p.n &&
                         (lead_n == p.V || (margin == 0.f ? top_value(nth) >= outside : top_value(nth) > outside + margin));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (key[h] != 0ull && rank[h] < p.n) {
            p.top_ids[(size_t)row * p.n + rank[h]] = top_index(key[h]);
            p.top_logprobs[(size_t)row * p.n + rank[h]] = (top_value(key[h]) - sum.m) - rest;
        }
    }
    if (!settled && lane == 0) {
        const int at = atomicAdd(p.redo, 1);
        int *r = p.redo + 1 + kMaxClusters + 3 * at;
        r[0] = row;
        r[1] = __float_as_int(sum.m);
        r[2] = __float_as_int(rest);
    }
}

// ------------------------------------------------------------------ rows the candidates do not settle

constexpr int kExThreads = 512, kExWarps = kExThreads / 32;

struct ExactArgs {
    const uint16_t *head, *x;
    int V, H, n;
    int *redo;
    unsigned long long *lists;         // [clusters][32]
    int32_t *top_ids;
    float *top_logprobs;
};

// Clusters of kExCluster CTAs take the rows in turn; fewer rows than clusters are split, each cluster
// taking a share of the vocabulary, and the one that ends last joins the shares' lists.
__global__ void __cluster_dims__(kExCluster, 1, 1) __launch_bounds__(kExThreads) exact_kernel(ExactArgs p) {
    extern __shared__ float4 xs[];
    __shared__ unsigned long long lists[kExWarps][32], gathered[kExCluster][32];
    pdl_wait();
    const int rows = *p.redo;
    if (rows == 0) return;                                          // the same for every CTA
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int clusters = gridDim.x / kExCluster, me = blockIdx.x / kExCluster;
    const int shares = rows < clusters ? clusters / rows : 1;
    for (int unit = me; unit < rows * shares; unit += clusters) {
        const int i = unit / shares, share = unit % shares;
        const int *r = p.redo + 1 + kMaxClusters + 3 * i;
        const int row = r[0];
        stage_row(p.x + (size_t)row * p.H, p.H, xs);
        __syncthreads();
        unsigned long long list = 0ull;
        const int step = shares * kExCluster * kExWarps;
        for (int v = (share * kExCluster + rank) * kExWarps + warp; v < p.V; v += step) {
            const unsigned long long k = top_key(exact_logit(p.head + (size_t)v * p.H, xs, p.H), v);
            list = top_insert(list, k);
        }
        lists[warp][lane] = list;
        __syncthreads();
        for (int h = kExWarps / 2; h > 0; h >>= 1) {
            if (warp < h) {
                list = top_merge(list, lists[warp + h][lane]);
                lists[warp][lane] = list;
            }
            __syncthreads();
        }
        cluster.sync();                                             // the first CTA has begun, and read the last row's
        if (warp == 0) cluster.map_shared_rank(&gathered[0][0], 0)[rank * 32 + lane] = list;
        cluster.sync();
        if (rank == 0 && warp == 0) {
            for (int q = 1; q < kExCluster; ++q) list = top_merge(list, gathered[q][lane]);
            bool mine = true;
            if (shares > 1) {
                p.lists[me * 32 + lane] = list;
                __threadfence();
                __syncwarp();
                int before = 0;
                if (lane == 0) before = atomicAdd(p.redo + 1 + i, 1);
                before = __shfl_sync(0xffffffffu, before, 0);
                __threadfence();
                mine = before == shares - 1;
                if (mine)
                    for (int q = 0; q < shares; ++q)
                        if (q != share) list = top_merge(list, __ldcg(p.lists + (i * shares + q) * 32 + lane));
            }
            if (mine && lane < p.n) {
                const float m = __int_as_float(r[1]), rest = __int_as_float(r[2]);
                p.top_ids[(size_t)row * p.n + lane] = top_index(list);
                p.top_logprobs[(size_t)row * p.n + lane] = (top_value(list) - m) - rest;
            }
        }
        __syncthreads();
    }
}

struct Plan {
    int sms;
    bool paired;                       // 256-row blocks by CTA pairs, or one of 128 rows
    size_t lists, stats, bins, exact, redo, bytes;     // offsets
};

int make_plan(int T, Plan &pl) {
    int dev = 0;
    MOE_CUDA_TRY(cudaGetDevice(&dev));
    MOE_CUDA_TRY(cudaDeviceGetAttribute(&pl.sms, cudaDevAttrMultiProcessorCount, dev));
    if (pl.sms < 2 * kMaxGroup || pl.sms * kHalves > kMaxLists)
        return moe_set_error(MOE_ENODEV, "head logprobs: a device of %d SMs (%d to %d)", pl.sms, 2 * kMaxGroup,
                             kMaxLists / kHalves);
    pl.paired = T > kM;
    // 128-row blocks x parts is at most the number of SMs in every launch
    const size_t slices = (size_t)pl.sms * kHalves;
    const int rows = T < kMaxGroup * 2 * kM ? T : kMaxGroup * 2 * kM;
    const size_t mblocks = pl.paired ? 2 * (((size_t)rows + 2 * kM - 1) / (2 * kM)) : 1;
    pl.lists = 0;
    pl.stats = al256(slices * kSlots * kM * sizeof(uint2));
    pl.bins = pl.stats + al256(slices * kM * sizeof(float4));
    pl.exact = pl.bins + al256(mblocks * kBins * kM * sizeof(unsigned));
    pl.redo = pl.exact + al256((size_t)kMaxClusters * 32 * sizeof(unsigned long long));
    pl.bytes = pl.redo + al256((1 + kMaxClusters + 3 * (size_t)rows) * sizeof(int));
    return MOE_OK;
}

template <bool kPair>
int launch_score(const CUtensorMap &mx, const CUtensorMap &mw, const ScoreArgs &a, cudaStream_t st) {
    auto kern = score_kernel<kPair>;
    const size_t smem = ScoreSmem<kPair>::alloc;
    MOE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.blocks * a.parts * (kPair ? 2 : 1)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kPair ? 2 : 1;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    MOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, mx, mw, a));
    return MOE_OK;
}

}  // namespace

extern "C" size_t moe_head_logprobs_workspace_bytes(int T, int V, int n) {
    Plan pl;
    if (T <= 0 || V <= 0 || n < 0 || make_plan(T, pl) != MOE_OK) return 0;
    return pl.bytes;
}

extern "C" int moe_head_logprobs(const void *head, int V, int H, const void *x, int T, const int32_t *targets, int n,
                                 float *logprob, float *entropy, int32_t *top_ids, float *top_logprobs,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = moe_logprobs_check("head logprobs", T, V, targets, n, logprob, entropy, top_ids, top_logprobs))
        return rc;
    if (!head || !x || H <= 0 || H % 8 || H > 8192)
        return moe_set_error(MOE_EINVAL, "head logprobs: head and x must be set, H=%d a multiple of 8 up to 8192", H);
    if ((reinterpret_cast<uintptr_t>(head) | reinterpret_cast<uintptr_t>(x)) & 15)
        return moe_set_error(MOE_EINVAL, "head logprobs: head and x must be 16-byte aligned");
    Plan pl;
    if (int rc = make_plan(T, pl)) return rc;
    if (!workspace || workspace_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return moe_set_error(MOE_EINVAL, "head logprobs: a 16-byte aligned workspace of %zu bytes is needed", pl.bytes);
    char *ws = static_cast<char *>(workspace);
    uint2 *lists = reinterpret_cast<uint2 *>(ws + pl.lists);
    float4 *stats = reinterpret_cast<float4 *>(ws + pl.stats);
    int *redo = reinterpret_cast<int *>(ws + pl.redo);
    cudaStream_t st = as_stream(stream);
    unsigned *bins = reinterpret_cast<unsigned *>(ws + pl.bins);
    CUtensorMap mw, mx;
    int rc;
    for (int t0 = 0; t0 < T; t0 += kMaxGroup * 2 * kM) {
        const int rows = T - t0 < kMaxGroup * 2 * kM ? T - t0 : kMaxGroup * 2 * kM;
        const int ctas = pl.paired ? 2 : 1, blocks = (rows + ctas * kM - 1) / (ctas * kM);
        int parts = pl.sms / ctas / blocks;
        // the tile width that leaves the busiest part the fewest entries (V = 248,320 over 148 parts: 7 tiles of
        // 256, or 7 of 240, 6 % less)
        int width = kN;
        long long most = -1;
        for (int w = kN; w >= 192; w -= 16 * ctas) {
            const int tiles = (V + w - 1) / w;
            const long long m = (long long)((tiles + parts - 1) / parts) * w;
            if (most < 0 || m < most) {
                most = m;
                width = w;
            }
        }
        if (parts > (V + width - 1) / width) parts = (V + width - 1) / width;
        const int xbox = rows >= kM ? kM : 32;
        const uint16_t *xr = static_cast<const uint16_t *>(x) + (size_t)t0 * H;
        rc = make_map("head logprobs", &mw, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, head, (uint64_t)H, (uint64_t)V, kK,
                      (uint32_t)(width / ctas));
        if (!rc)
            rc = make_map("head logprobs", &mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, xr, (uint64_t)H, (uint64_t)rows, kK,
                          (uint32_t)xbox);
        if (rc) return rc;
        const ScoreArgs sa{rows, V, H, blocks, parts, width, xbox, n + kPad, lists, stats, bins, redo};
        constexpr int kClear = 256;                                  // 16 bytes a thread
        clear_kernel<<<blocks * ctas * (kBins * kM / 4 / kClear), kClear, 0, st>>>(reinterpret_cast<uint4 *>(bins));
        MOE_CUDA_TRY(cudaGetLastError());
        if ((rc = pl.paired ? launch_score<true>(mx, mw, sa, st) : launch_score<false>(mx, mw, sa, st))) return rc;
        int32_t *ids = n ? top_ids + (size_t)t0 * n : nullptr;
        float *tl = n ? top_logprobs + (size_t)t0 * n : nullptr;
        const FinishArgs fa{static_cast<const uint16_t *>(head), xr, V, H, n, parts, n + kPad, lists, stats,
                            targets ? targets + t0 : nullptr, logprob ? logprob + t0 : nullptr, entropy + t0, ids, tl,
                            redo};
        // both launched ahead of their predecessor's end (what they read of it they wait for)
        const size_t xbytes = (size_t)H * sizeof(float);
        if (rows > 4 * pl.sms)
            MOE_CUDA_TRY(launch_pdl(finish_kernel<128>, dim3((unsigned)rows), dim3(128), xbytes, st, fa));
        else if (rows > pl.sms)
            MOE_CUDA_TRY(launch_pdl(finish_kernel<256>, dim3((unsigned)rows), dim3(256), xbytes, st, fa));
        else
            MOE_CUDA_TRY(launch_pdl(finish_kernel<512>, dim3((unsigned)rows), dim3(512), xbytes, st, fa));
        if (n > 0) {
            const int clusters = pl.sms / kExCluster < kMaxClusters ? pl.sms / kExCluster : kMaxClusters;
            const ExactArgs ea{static_cast<const uint16_t *>(head), xr, V, H, n, redo,
                               reinterpret_cast<unsigned long long *>(ws + pl.exact), ids, tl};
            MOE_CUDA_TRY(launch_pdl(exact_kernel, dim3((unsigned)(clusters * kExCluster)), dim3(kExThreads),
                                    xbytes, st, ea));
        }
    }
    return MOE_OK;
}

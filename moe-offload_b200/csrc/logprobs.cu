// Log-probabilities of given tokens, entropy and the n most likely alternatives of rows of
// logits [T, V] fp32 that are in memory (a decode step's answer to a request's `logprobs`).
//
//   lse = log sum_v e^l_v      logprob = l_target - lse      entropy = lse - sum_v p_v l_v
//
// One pass over the row (4 V bytes: HBM, or L2 right after the LM head) by a cluster of up to 8
// CTAs, one launch, no workspace. Every thread keeps the softmax statistics of its elements
// (toplist.cuh) and, for the alternatives, the largest element of each of the 32 residues of the
// index mod 32. The n-th largest of the row's 32 residue maxima is a bound tau that at least n
// elements reach, and hardly more do (31 expected for n = 20 of independent logits), so only the
// threads whose own maximum reaches tau look at their elements again (at one batch of 16, unless
// another batch of theirs reaches tau too); the few that reach it are ranked by counting. No
// running list, no sort.
// B200, n = 20: 512 rows of 248,320 100 us (0.78 of the copy rate), one row 9.9 us, which is latency.
// Ties at tau (a mask that leaves fewer than n tokens, a row of equal logits) are taken in index
// order from the start of the row; a row whose large elements crowd into fewer than n residues
// takes n passes.
#include <cooperative_groups.h>

#include "common.cuh"
#include "internal.h"
#include "toplist.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kMaxCluster = 8;
constexpr int kBatch = 4;              // chunks of 4 elements a thread has in flight
constexpr int kCand = 256;             // elements above (or equal to) tau that are ranked at once

struct LogprobArgs {
    const float *logits;
    int T, V, n;
    const int32_t *targets;
    float *logprob, *entropy;
    int32_t *top_ids;
    float *top_logprobs;
};

// The row as chunks of 4 elements at 16-byte boundaries: chunk c holds the elements 4 c - a ..
// 4 c - a + 3 (a: elements between the boundary below the row and the row), -inf outside the row.
struct Row {
    const float *p;
    int a, V;
    MOE_D float at(int i) const { return (i >= 0 && i < V) ? __ldg(p + i) : -INFINITY; }
};

// kBatch chunks c, c + kT, ...; lo, hi: the chunks that lie wholly inside the row and this
// CTA's part; end: the part's end
template <int kT>
MOE_D void load_batch(const Row &row, int c, int lo, int hi, int end, float (&v)[4 * kBatch]) {
    if (c >= lo && c + (kBatch - 1) * kT < hi) {
        const float4 *q = reinterpret_cast<const float4 *>(row.p - row.a) + c;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const float4 f = __ldg(q + j * kT);
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int cc = c + j * kT;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * j + i] = cc < end ? row.at(4 * cc - row.a + i) : -INFINITY;
        }
    }
}

// what a warp adds to the row's sums, relative to the row's largest value m: s, w as in Soft, and
// how many threads hold m itself
struct WarpSum {
    float s, w;
    int peaks;
};

template <int kT>
struct Shared {
    static constexpr int kWarps = kT / 32;
    float res[kWarps][32];                       // residue maxima of the warps
    float part_res[kMaxCluster][32];             // of the cluster's CTAs (written by them)
    // gathered in the cluster's first CTA: every warp's sums and the candidates of the row
    WarpSum sums[kMaxCluster * kWarps];
    unsigned long long above[kCand], equal[kCand], out[kTopMax];
    int nabove, nequal;
    int scan[kWarps];
    unsigned long long best[kWarps];
};

// appends the keys of the lanes with ok to a list of the first CTA, as far as it reaches
MOE_D void append(unsigned long long *list, int *count, bool ok, unsigned long long key) {
    const unsigned who = __ballot_sync(0xffffffffu, ok);
    if (!who) return;
    const int lane = threadIdx.x & 31;
    int base = 0;
    if (lane == __ffs(who) - 1) base = atomicAdd(count, __popc(who));
    base = __shfl_sync(0xffffffffu, base, __ffs(who) - 1);
    const int at = base + __popc(who & ((1u << lane) - 1u));
    if (ok && at < kCand) list[at] = key;
}

// scatters the m keys of a list to out by their rank (+ from) among themselves, ranks below n
template <int kT>
MOE_D void rank_out(const unsigned long long *list, int m, int from, int n, unsigned long long *out) {
    for (int i = threadIdx.x; i < m; i += kT) {
        const unsigned long long k = list[i];
        int r = from;
        for (int j = 0; j < m; ++j) r += list[j] > k;
        if (r < n) out[r] = k;
    }
}

// kT threads a CTA (a cluster of several CTAs needs a warp for each: 512)
template <int kT>
__global__ void __launch_bounds__(kT) logprobs_kernel(LogprobArgs p) {
    constexpr int kWarps = kT / 32;
    __shared__ Shared<kT> sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int t = blockIdx.x / parts;
    const float *base = p.logits + (size_t)t * p.V;
    const Row row{base, (int)((reinterpret_cast<uintptr_t>(base) >> 2) & 3), p.V};
    const int chunks = (p.V + row.a + 3) / 4;
    const int per = (chunks + parts - 1) / parts;
    const int c0 = min(part * per, chunks), c1 = min(c0 + per, chunks);
    const int lo = max(c0, row.a ? 1 : 0), hi = min(c1, (p.V + row.a) / 4);
    if (tid == 0) sh.nabove = sh.nequal = 0;
    if (parts > 1) cluster.barrier_arrive();     // waited for before the first store to another CTA

    // ---- the pass over the row. best: the batch with the thread's first largest element, peak that
    // element, next: the largest element of its other batches
    SoftRun run = run_none();
    float res[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    float next = -INFINITY;
    int best = c0 + tid;
#pragma unroll 1
    for (int c = c0 + tid; c < c1; c += kT * kBatch) {
        float v[4 * kBatch];
        load_batch<kT>(row, c, lo, hi, c1, v);
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = v[i];
#pragma unroll
            for (int j = 1; j < kBatch; ++j) q[i] = fmaxf(q[i], v[4 * j + i]);
            res[i] = fmaxf(res[i], q[i]);
        }
        const float top = fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3]));
        next = fmaxf(next, fminf(run.m, top));
        if (top > run.m) best = c;
        run_add(run, v, top);
    }
    const float peak = run.m;
    // lanes l, l + 8, l + 16, l + 24 hold the same residues 4 (l mod 8) .. + 3
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        res[i] = fmaxf(res[i], __shfl_xor_sync(0xffffffffu, res[i], 8));
        res[i] = fmaxf(res[i], __shfl_xor_sync(0xffffffffu, res[i], 16));
    }
    if (lane < 8) *reinterpret_cast<float4 *>(&sh.res[warp][4 * lane]) = make_float4(res[0], res[1], res[2], res[3]);
    __syncthreads();
    // ---- the cluster's CTAs exchange their residue maxima
    float top = sh.res[0][lane];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sh.res[w][lane]);
    if (parts > 1) {
        cluster.barrier_wait();
        if (warp < parts) cluster.map_shared_rank(&sh.part_res[0][0], warp)[part * 32 + lane] = top;
        cluster.sync();
        top = sh.part_res[0][lane];
        for (int q = 1; q < parts; ++q) top = fmaxf(top, sh.part_res[q][lane]);
    }
    float m = top;                               // the row's largest value
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));

    // ---- the sums relative to m; all its occurrences are left out and counted
    {
        // (a thread without a finite logit has no reference: nothing, or a NaN, to pass on)
        const float d = fmaxf(run.r - m, kSoftFar), f = peak > -INFINITY ? expf(d) : 0.f;
        const float e = fmaxf(peak - m, kSoftFar), g = peak == m ? 0.f : expf(e);
        WarpSum a{fmaf(f, run.s, g), fmaf(f, fmaf(d, run.s, run.w), e * g), peak == m};
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            a.s += __shfl_xor_sync(0xffffffffu, a.s, off);
            a.w += __shfl_xor_sync(0xffffffffu, a.w, off);
            a.peaks += __shfl_xor_sync(0xffffffffu, a.peaks, off);
        }
        if (lane == 0) cluster.map_shared_rank(sh.sums, 0)[part * kWarps + warp] = a;
    }
    float tau = -INFINITY;
    if (p.n > 0) {
        int r = 0;                               // rank among the 32 residues, equal ones by lane
#pragma unroll 4
        for (int j = 0; j < 32; ++j) {
            const float o = __shfl_sync(0xffffffffu, top, j);
            r += (o > top || (o == top && j < lane)) ? 1 : 0;
        }
        tau = __shfl_sync(0xffffffffu, top, __ffs(__ballot_sync(0xffffffffu, r == p.n - 1)) - 1);
        // ---- the threads whose maximum reaches tau look again
        unsigned long long *above = cluster.map_shared_rank(sh.above, 0), *equal = cluster.map_shared_rank(sh.equal, 0);
        int *nabove = cluster.map_shared_rank(&sh.nabove, 0), *nequal = cluster.map_shared_rank(&sh.nequal, 0);
        const bool mine = peak >= tau && peak > -INFINITY;
        if (__ballot_sync(0xffffffffu, mine)) {
            float v[4 * kBatch];
            if (mine) load_batch<kT>(row, best, lo, hi, c1, v);
#pragma unroll
            for (int i = 0; i < 4 * kBatch; ++i) {
                // (lanes that do not take part hold nothing: -inf is neither above tau nor equal to it)
                const float x = mine ? v[i] : -INFINITY;
                if (__ballot_sync(0xffffffffu, x >= tau && x > -INFINITY)) {
                    const unsigned long long k = top_key(x, 4 * (best + (i >> 2) * kT) - row.a + (i & 3));
                    append(above, nabove, x > tau, k);
                    append(equal, nequal, x == tau && tau > -INFINITY, k);
                }
            }
            // their other batches: the whole warp for one thread at a time, 128 elements a step
            unsigned who = __ballot_sync(0xffffffffu, mine && next >= tau && next > -INFINITY);
            while (who) {
                const int owner = __ffs(who) - 1;
                who &= who - 1;
                const int ob = __shfl_sync(0xffffffffu, best, owner);
                for (int c = c0 + 32 * warp + owner; c < c1; c += kT * 32) {
                    float x[4];
                    int at[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int cc = c + kT * (8 * j + (lane >> 2));
                        const bool done = cc >= ob && cc < ob + kT * kBatch;       // the batch from above
                        at[j] = 4 * cc - row.a + (lane & 3);
                        x[j] = cc < c1 && !done ? row.at(at[j]) : -INFINITY;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        append(above, nabove, x[j] > tau, top_key(x[j], at[j]));
                        append(equal, nequal, x[j] == tau && tau > -INFINITY, top_key(x[j], at[j]));
                    }
                }
            }
        }
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    if (part != 0) return;                       // only the first CTA's shared memory is used from here

    const int n = p.n;
    if (n > 0) {
        const int na = sh.nabove, ne = sh.nequal;
        if (na <= kCand) {
            rank_out<kT>(sh.above, na, 0, n, sh.out);
            if (tau > -INFINITY && ne <= kCand) {
                rank_out<kT>(sh.equal, ne, na, n, sh.out);
            } else {
                // the first of the elements equal to tau, in index order (NaN counts as -inf)
                const unsigned long long key0 = top_key(tau, 0) >> 32;
                for (int i0 = 0, found = na; i0 < p.V && found < n; i0 += kT) {
                    const int i = i0 + tid;
                    const unsigned long long k = i < p.V ? top_key(__ldg(base + i), i) : 0ull;
                    const bool ok = (k >> 32) == key0;
                    const unsigned who = __ballot_sync(0xffffffffu, ok);
                    if (lane == 0) sh.scan[warp] = __popc(who);
                    __syncthreads();
                    int before = found + __popc(who & ((1u << lane) - 1u));
                    for (int w = 0; w < kWarps; ++w) {
                        before += w < warp ? sh.scan[w] : 0;
                        found += sh.scan[w];
                    }
                    if (ok && before < n) sh.out[before] = k;
                    __syncthreads();
                }
            }
        } else {
            // more than kCand elements above tau: the largest below the last one, n times
            unsigned long long last = ~0ull;
            for (int r = 0; r < n; ++r) {
                unsigned long long b = 0ull;
                for (int i = tid; i < p.V; i += kT) {
                    const unsigned long long k = top_key(__ldg(base + i), i);
                    if (k < last && k > b) b = k;
                }
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) {
                    const unsigned long long o = __shfl_xor_sync(0xffffffffu, b, off);
                    b = o > b ? o : b;
                }
                if (lane == 0) sh.best[warp] = b;
                __syncthreads();
                for (int w = 0; w < kWarps; ++w) b = sh.best[w] > b ? sh.best[w] : b;
                last = b;
                if (tid == 0) sh.out[r] = b;
                __syncthreads();
            }
        }
        __syncthreads();
    }
    if (warp == 0) {
        Soft all{m, 0.f, 0.f};
        int peaks = 0;
        for (int i = lane; i < parts * kWarps; i += 32) {
            all.s += sh.sums[i].s;
            all.w += sh.sums[i].w;
            peaks += sh.sums[i].peaks;
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            all.s += __shfl_xor_sync(0xffffffffu, all.s, off);
            all.w += __shfl_xor_sync(0xffffffffu, all.w, off);
            peaks += __shfl_xor_sync(0xffffffffu, peaks, off);
        }
        all.s += (float)(peaks - 1);             // Soft leaves one occurrence of m out
        const float rest = soft_log_rest(all);
        if (lane < n) {
            const unsigned long long k = sh.out[lane];
            p.top_ids[(size_t)t * n + lane] = top_index(k);
            p.top_logprobs[(size_t)t * n + lane] = (top_value(k) - all.m) - rest;
        }
        if (lane == 0) {
            p.entropy[t] = soft_entropy(all);
            if (p.targets) {
                const int id = p.targets[t];
                const bool in = id >= 0 && id < p.V;
                if (!in && id != -1) atomicOr(&g_moe_device_error, MOE_DEVERR_BAD_INPUT);
                p.logprob[t] = in ? (__ldg(base + id) - all.m) - rest : __int_as_float(0x7fffffff);
            }
        }
    }
}

int launch_logprobs(const LogprobArgs &p, cudaStream_t stream) {
    const int T = p.T, V = p.V;
    // A CTA's work behind the pass over its elements is a chain of some 5,000 cycles, whatever it has read. So:
    // a cluster only as far as the rows leave SMs free (T = 64, V = 248,320: 21.5 us with 4 CTAs a row, 25.6
    // with 2, 29.7 with 8; T = 1: 10.2 with 8, 23.6 with 1), and fewer threads for many short rows
    // (2,048 x 1,000: 17 us with 128, 25 with 256, 42 with 512; 2,048 x 50,021: 83, 87, 100;
    // 2,048 x 248,320: 414, 357, 346).
    int parts = 1, threads = 512;
    if (V <= 16384) {
        threads = T >= 148 ? 128 : 256;
    } else if (T >= 296) {
        threads = V <= 131072 ? 256 : 512;
    } else {
        while (parts < kMaxCluster && T * parts < 148 && V / (2 * parts) >= 14336) parts *= 2;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)T * (unsigned)parts);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;            // (a CTA alone is a cluster of one)
    auto kern = threads == 512 ? logprobs_kernel<512> : threads == 256 ? logprobs_kernel<256> : logprobs_kernel<128>;
    MOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return MOE_OK;
}

}  // namespace

int moe_logprobs_check(const char *who, int T, int V, const int32_t *targets, int n, const float *logprob,
                       const float *entropy, const int32_t *top_ids, const float *top_logprobs) {
    if (T <= 0 || V <= 0 || T > (1 << 24) || V > (1 << 30))
        return moe_set_error(MOE_EINVAL, "%s: bad sizes T=%d V=%d (T <= 2^24, V <= 2^30)", who, T, V);
    if (n < 0 || n > kTopMax || n > V)
        return moe_set_error(MOE_EINVAL, "%s: n=%d alternatives (0 to min(V, %d) = %d)", who, n, kTopMax,
                             V < kTopMax ? V : kTopMax);
    if (!entropy || (targets && !logprob) || (!targets && logprob) || (n > 0 && (!top_ids || !top_logprobs)))
        return moe_set_error(MOE_EINVAL, "%s: null pointer", who);
    return MOE_OK;
}

extern "C" int moe_token_logprobs(const float *logits, int T, int V, const int32_t *targets, int n, float *logprob,
                                  float *entropy, int32_t *top_ids, float *top_logprobs, void *stream) {
    if (int rc = moe_logprobs_check("token logprobs", T, V, targets, n, logprob, entropy, top_ids, top_logprobs))
        return rc;
    if (!logits || (reinterpret_cast<uintptr_t>(logits) & 3))
        return moe_set_error(MOE_EINVAL, "token logprobs: logits must be 4-byte aligned and not null");
    return launch_logprobs(LogprobArgs{logits, T, V, n, targets, logprob, entropy, top_ids, top_logprobs},
                           as_stream(stream));
}

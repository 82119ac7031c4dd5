// Log-probabilities of given tokens, entropy and the n most likely alternatives of rows of
// logits [T, V] fp32 that are in memory (a decode step's answer to a request's `logprobs`).
//
//   lse = log sum_v e^l_v      logprob = l_target - lse      entropy = lse - sum_v p_v l_v
//
// One pass over the row (4 V bytes: HBM, or L2 right after the LM head): every thread keeps the
// softmax statistics of its elements (toplist.cuh) and its own largest element. The n largest
// elements of a CTA's part all belong to the n threads with the largest maxima, so only those
// threads' elements (V / threads each) are looked at a second time, instead of every element being
// held against a running list. A row is shared by a cluster of up to 8 CTAs when there are few
// rows; they join through distributed shared memory, so there is no workspace, no counter to
// reset and one launch.
#include <cooperative_groups.h>

#include "common.cuh"
#include "internal.h"
#include "toplist.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

struct LogprobArgs {
    const float *logits;
    int T, V, n;
    const int32_t *targets;
    float *logprob, *entropy;
    int32_t *top_ids;
    float *top_logprobs;
};

// 4 consecutive logits at virtual index 4 c - a (a: elements between the 16-byte boundary below
// the row and the row), -inf outside the row; returns the index of v[0]
MOE_D int load4(const float *row, int a, int V, int c, float (&v)[4]) {
    const int i0 = 4 * c - a;
    if (i0 >= 0 && i0 + 4 <= V) {
        const float4 q = __ldg(reinterpret_cast<const float4 *>(row + i0));
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (i0 + i >= 0 && i0 + i < V) ? __ldg(row + i0 + i) : -INFINITY;
    }
    return i0;
}

__global__ void __launch_bounds__(kThreads) logprobs_kernel(LogprobArgs p) {
    __shared__ unsigned long long lists[kWarps][32];
    __shared__ Soft softs[kWarps];
    __shared__ unsigned long long cta_list[32];
    __shared__ Soft cta_soft;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int t = blockIdx.x / parts;
    const float *row = p.logits + (size_t)t * p.V;
    const int a = (int)((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
    const int chunks = (p.V + a + 3) / 4;
    const int per = (chunks + parts - 1) / parts;
    const int c0 = min(part * per, chunks), c1 = min(c0 + per, chunks);

    Soft st = soft_none();
    // the first in-range index of the thread, for a thread whose elements are all -inf
    int at = c0 + tid < c1 ? max(4 * (c0 + tid) - a, 0) : -1;
#pragma unroll 4
    for (int c = c0 + tid; c < c1; c += kThreads) {
        float v[4];
        const int i0 = load4(row, a, p.V, c, v);
        soft_add(st, at, v, i0);
    }
    unsigned long long list = 0ull;
    if (p.n > 0) {
        // the CTA's 32 best thread maxima, sorted
        list = top_sort(at >= 0 ? top_key(st.m, at) : 0ull);
        lists[warp][lane] = list;
    }
    const Soft ws = soft_warp(st);
    if (lane == 0) softs[warp] = ws;
    __syncthreads();
    if (warp == 0) {
        const Soft b = soft_warp(lane < kWarps ? softs[lane] : soft_none());
        if (lane == 0) cta_soft = b;
    }
    if (p.n > 0) {
        for (int h = kWarps / 2; h > 0; h >>= 1) {
            if (warp < h) {
                list = top_merge(list, lists[warp + h][lane]);
                lists[warp][lane] = list;
            }
            __syncthreads();
        }
        // every element that is among the CTA's n largest belongs to one of the first n of these
        // threads and is not below the n-th of them
        const unsigned long long floor_key = lists[0][p.n - 1];
        list = 0ull;
        for (int o = warp; o < p.n; o += kWarps) {
            const unsigned long long ok = lists[0][o];
            if (!ok) break;
            const int oc = (top_index(ok) + a) >> 2;                 // a chunk of the owner
            const int first = c0 + (oc - c0) % kThreads;             // its first one
            for (int c = first; c < c1; c += kThreads * 8) {         // 8 chunks of 4 elements a pass
                const int cc = c + kThreads * (lane >> 2), i = 4 * cc - a + (lane & 3);
                unsigned long long k = 0ull;
                if (cc < c1 && i >= 0 && i < p.V) k = top_key(__ldg(row + i), i);
                list = top_insert(list, k, __ballot_sync(0xffffffffu, k >= floor_key && k != 0ull));
            }
        }
        __syncthreads();
        lists[warp][lane] = list;
        __syncthreads();
        for (int h = kWarps / 2; h > 0; h >>= 1) {
            if (warp < h) {
                list = top_merge(list, lists[warp + h][lane]);
                lists[warp][lane] = list;
            }
            __syncthreads();
        }
        if (warp == 0) cta_list[lane] = list;
    }
    if (parts > 1) cluster.sync();
    if (part == 0 && warp == 0) {
        __syncwarp();
        Soft all = lane < parts ? *cluster.map_shared_rank(&cta_soft, lane) : soft_none();
        all = soft_warp(all);
        const float rest = soft_log_rest(all);
        if (p.n > 0) {
            unsigned long long other[kMaxCluster];
#pragma unroll
            for (int r = 1; r < kMaxCluster; ++r)
                other[r] = r < parts ? cluster.map_shared_rank(cta_list, r)[lane] : 0ull;
#pragma unroll
            for (int r = 1; r < kMaxCluster; ++r)
                if (r < parts) list = top_merge(list, other[r]);
            if (lane < p.n) {
                p.top_ids[(size_t)t * p.n + lane] = top_index(list);
                p.top_logprobs[(size_t)t * p.n + lane] = (top_value(list) - all.m) - rest;
            }
        }
        if (lane == 0) {
            p.entropy[t] = soft_entropy(all);
            if (p.targets) {
                const int id = p.targets[t];
                const bool in = id >= 0 && id < p.V;
                if (!in && id != -1) atomicOr(&g_moe_device_error, MOE_DEVERR_BAD_INPUT);
                p.logprob[t] = in ? (__ldg(row + id) - all.m) - rest : __int_as_float(0x7fffffff);
            }
        }
    }
    if (parts > 1) cluster.sync();               // the others' shared memory stays until it is read
}

}  // namespace

int moe_token_logprobs_launch(const float *logits, int T, int V, const int32_t *targets, int n, float *logprob,
                              float *entropy, int32_t *top_ids, float *top_logprobs, void *stream) {
    int parts = 1;
    while (parts < kMaxCluster && (long long)T * parts < 296 && V / (2 * parts) >= 4096) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)T * (unsigned)parts);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const LogprobArgs p{logits, T, V, n, targets, logprob, entropy, top_ids, top_logprobs};
    MOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, logprobs_kernel, p));
    return MOE_OK;
}

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
    return moe_token_logprobs_launch(logits, T, V, targets, n, logprob, entropy, top_ids, top_logprobs, stream);
}

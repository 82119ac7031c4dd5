// Low-rank adapters of many requests beside a shared projection:
//
//   out[t] = y[t] + scale[a] * (x[t] . A[a]^T) . B[a]^T,   a = ids[t]   (a = -1: out[t] = y[t])
//
// with A [adapters, rank, K], B [adapters, N, rank] bf16 and y the projection's own output (bf16,
// or the LM head's fp32 logits). Both products are summed in fp32; the result is rounded once.
#include "common.cuh"

namespace {

constexpr int kThreads = 256;

struct AdapterArgs {
    const uint16_t *x;
    int T, K, N;
    const uint16_t *a, *b;
    const float *scale;
    int adapters, rank;
    const int32_t *ids;
    const void *y;
    void *out;
};

template <bool kFp32>
__global__ void __launch_bounds__(kThreads) adapter_kernel(AdapterArgs p) {
    __shared__ float u[128];
    const int t = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int id = p.ids[t];
    if (id < -1 || id >= p.adapters) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(&g_moe_device_error, MOE_DEVERR_BAD_INPUT);
        id = -1;
    }
    if (id >= 0) {
        for (int j = warp; j < p.rank; j += kThreads / 32) {
            const uint16_t *ar = p.a + ((size_t)id * p.rank + j) * p.K, *xr = p.x + (size_t)t * p.K;
            float s = 0.f;
            for (int k = lane; k < p.K; k += 32) s = fmaf(bf16_bits_to_f32(ar[k]), bf16_bits_to_f32(xr[k]), s);
            for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            if (lane == 0) u[j] = s * p.scale[id];
        }
        __syncthreads();
    }
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= p.N) return;
    const size_t at = (size_t)t * p.N + i;
    if (id < 0) {
        if (kFp32) static_cast<float *>(p.out)[at] = static_cast<const float *>(p.y)[at];
        else static_cast<uint16_t *>(p.out)[at] = static_cast<const uint16_t *>(p.y)[at];
        return;
    }
    const uint16_t *br = p.b + ((size_t)id * p.N + i) * p.rank;
    float s = 0.f;
    for (int j = 0; j < p.rank; ++j) s = fmaf(bf16_bits_to_f32(br[j]), u[j], s);
    if (kFp32) static_cast<float *>(p.out)[at] = static_cast<const float *>(p.y)[at] + s;
    else static_cast<uint16_t *>(p.out)[at] = f32_to_bf16_bits(bf16_bits_to_f32(static_cast<const uint16_t *>(p.y)[at]) + s);
}

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p < q + nb && q < p + na;
}

}  // namespace

extern "C" int moe_adapter_add(const void *x, int T, int K, int N, const void *a, const void *b, const float *scale,
                               int adapters, int rank, const int32_t *ids, const void *y, int y_fp32, void *out,
                               void *stream) {
    if (!x || !a || !b || !scale || !ids || !y || !out) return moe_set_error(MOE_EINVAL, "adapters: null pointer");
    if (T <= 0 || K <= 0 || K % 8 || N <= 0 || adapters <= 0 || rank <= 0 || rank > 128 || rank % 8)
        return moe_set_error(MOE_EINVAL,
                             "adapters: bad sizes T=%d K=%d N=%d adapters=%d rank=%d (K and rank multiples of 8, "
                             "rank up to 128)", T, K, N, adapters, rank);
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15)
        return moe_set_error(MOE_EINVAL, "adapters: x, a and b must be 16-byte aligned");
    const size_t es = y_fp32 ? 4 : 2, ny = (size_t)T * N * es;
    if ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out)) & (es - 1))
        return moe_set_error(MOE_EINVAL, "adapters: y and out must be aligned to their %zu-byte values", es);
    if ((out != y && overlap(out, ny, y, ny)) || overlap(out, ny, x, (size_t)T * K * 2) ||
        overlap(out, ny, a, (size_t)adapters * rank * K * 2) || overlap(out, ny, b, (size_t)adapters * rank * N * 2) ||
        overlap(out, ny, scale, (size_t)adapters * 4) || overlap(out, ny, ids, (size_t)T * 4))
        return moe_set_error(MOE_EINVAL, "adapters: out may be y itself, but not overlap it or another input");
    if (T > 65535) return moe_set_error(MOE_EINVAL, "adapters: T=%d rows (at most 65535)", T);
    const AdapterArgs p{static_cast<const uint16_t *>(x), T, K, N, static_cast<const uint16_t *>(a),
                        static_cast<const uint16_t *>(b), scale, adapters, rank, ids, y, out};
    const dim3 grid((unsigned)((N + kThreads - 1) / kThreads), (unsigned)T);
    if (y_fp32) adapter_kernel<true><<<grid, kThreads, 0, as_stream(stream)>>>(p);
    else adapter_kernel<false><<<grid, kThreads, 0, as_stream(stream)>>>(p);
    MOE_CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

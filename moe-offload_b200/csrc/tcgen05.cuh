// tcgen05 (5th-generation tensor core), tiled TMA and mbarrier helpers shared by the tensor-core
// kernels (prefill.cu, headscore.cu).
#pragma once

#include <cuda.h>

#include "common.cuh"

// Shared-memory matrix descriptor for a K-major operand in the 128-byte-swizzle layout: rows
// of 128 bytes (64 bf16 of K), 8-row groups 1024 bytes apart (stride byte offset), descriptor
// version 1 (bits 46-47), layout type 2 = SWIZZLE_128B (bits 61-63). The K = 16 steps inside
// a 64-wide block advance the start address by 32 bytes.
MOE_D uint64_t desc_sw128(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

// instruction descriptor, kind::f16: D f32, A and B bf16, both K-major, M x N
MOE_HD uint32_t instr_desc_bf16(int m, int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

MOE_D void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

MOE_D void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
MOE_D void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

MOE_D void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Bounded wait that also gives up once another warp of the CTA has aborted (the flag is
// polled every 1024 tries). On its own timeout it records the device error and raises the
// CTA's abort flag. Warp-uniform result: every lane of the calling warp must call it.
MOE_D bool wait_or_abort(uint64_t *bar, uint32_t parity, volatile int *abort) {
    bool ok = false, gave_up = false;
#pragma unroll 1
    for (uint32_t i = 0; i < kMbarSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) {
            ok = true;
            break;
        }
        if ((i & 1023u) == 1023u && *abort) {
            gave_up = true;
            break;
        }
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {                                             // warp-uniform branch
        const bool timed_out = !__any_sync(0xffffffffu, gave_up);
        if ((threadIdx.x & 31) == 0) {
            if (timed_out) atomicOr(&g_moe_device_error, MOE_DEVERR_MBAR_TIMEOUT);
            *abort = 1;
        }
    }
    return ok;
}

// The same without the vote, for a warp whose lanes all poll one barrier in step (the lanes see the same
// phase): a few instructions when the barrier is ready.
MOE_D bool wait_or_abort_step(uint64_t *bar, uint32_t parity, volatile int *abort) {
    if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
    for (uint32_t i = 0; i < kMbarSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && *abort) return false;
    }
    atomicOr(&g_moe_device_error, MOE_DEVERR_MBAR_TIMEOUT);
    *abort = 1;
    return false;
}

// true in one lane of the (converged) warp
MOE_D bool elect_lane() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}

MOE_D bool aborted(volatile int *abort) { return __any_sync(0xffffffffu, *abort != 0); }

// 2-D tiled TMA load (no multicast) completing on an mbarrier; x is the innermost coordinate
MOE_D void tma_load_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
            "r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}

// 2-D tensor map over a row-major [rows][cols] array with a box of box_cols x box_rows
// elements and 128-byte swizzling (box_cols * element size = 128 bytes)
static inline int make_map(const char *who, CUtensorMap *m, CUtensorMapDataType dt, size_t esize, const void *base,
                           uint64_t cols, uint64_t rows, uint32_t box_cols, uint32_t box_rows) {
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {cols * esize};
    const cuuint32_t box[2] = {box_cols, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    // the driver entry point is looked up through the runtime, so the library does not link
    // libcuda directly (it loads on hosts without a driver; calls then fail with an error)
    using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn encode = nullptr;
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        MOE_CUDA_TRY(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess || !fn)
            return moe_set_error(MOE_ECUDA, "%s: cuTensorMapEncodeTiled not available from the driver", who);
        encode = reinterpret_cast<EncodeFn>(fn);
    }
    const CUresult r = encode(m, dt, 2, const_cast<void *>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return moe_set_error(MOE_ECUDA, "%s: cuTensorMapEncodeTiled failed (%d)", who, (int)r);
    return MOE_OK;
}

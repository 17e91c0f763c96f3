/*
 * ring.cuh -- barriers, bounded waits and tensor copies of the kernels with shared-memory rings beside the attention (experts_umma.cu,
 * adapters.cu).
 *
 * Every wait is bounded: one that runs out raises the block's abort flag and leaves a code in the file's error words (hy3a_layer_sync).
 */
#ifndef HY3A_RING_CUH
#define HY3A_RING_CUH

#include <cuda.h>

#include "layer.h"

namespace hy3a_ring {

__device__ __forceinline__ unsigned smem_u32(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect_tx(unsigned bar, unsigned bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ bool mbar_try(unsigned bar, unsigned parity, unsigned hint_ns) {
    unsigned ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity), "r"(hint_ns) : "memory");
    return ok != 0;
}
/* Waits until the phase of that parity is over; false once anything in the block has given up.  A wait gives up after half a second and many polls. */
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, volatile int *abort_flag, unsigned *err, unsigned where) {
    if (mbar_try(bar, parity, 2000u)) return true;
    unsigned long long t0, t1;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    for (unsigned i = 0; i < (1u << 22); i++) {
        if (mbar_try(bar, parity, 20000u)) return true;
        if (*abort_flag) return false;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
        if (i >= (1u << 13) && t1 - t0 > 500000000ull) break;
    }
    *abort_flag = 1;
    if (atomicCAS(err, 0u, 2u) == 0u) err[1] = where;
    return false;
}
/* one wait that nothing ends (hy3a_layer_wait_out) */
__device__ __forceinline__ void wait_out(unsigned *err, unsigned where) {
    __shared__ alignas(8) unsigned long long s_bar;
    __shared__ int s_abort;
    s_abort = 0;
    mbar_init(smem_u32(&s_bar), 1);
    mbar_wait(smem_u32(&s_bar), 0u, &s_abort, err, where);
}
__device__ __forceinline__ unsigned elect_one() {
    unsigned p;
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}" : "=r"(p));
    return p;
}

/* ---- tensor maps (host) ---- */
typedef CUresult (*encode_tiled_fn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                    CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
/* the driver's encoder, NULL if it has none */
static inline encode_tiled_fn encoder() {
    static const encode_tiled_fn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return (encode_tiled_fn)p;
    }();
    return fn;
}
/* 16-bit elements, [depth][rows][inner] with dense depths (rank 3), or [rows][inner] (rank 2), rows `stride` elements apart; boxes of box_rows x
 * box_inner (128 bytes) */
static inline bool encode(CUtensorMap *m, int rank, const void *base, size_t inner, size_t rows, size_t depth, size_t stride, int box_inner, int box_rows) {
    const encode_tiled_fn enc = encoder();
    const cuuint64_t dims[3] = {inner, rows, depth}, strides[2] = {2 * stride, 2 * stride * rows};
    const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows, 1}, one[3] = {1, 1, 1};
    /* (16-bit types are moved alike) */
    return enc && enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

} /* namespace hy3a_ring */
#endif

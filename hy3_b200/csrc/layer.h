/*
 * layer.h -- what the operators beside the attention share (route.cu, experts.cu, adapters.cu, quantize4.cu, linear4.cu, logprobs.cu): the device check and
 * launch attributes on the host; 16-byte loads, conversions and the warp-level matrix product on the device.
 *
 * The warp-level product takes its fragments straight from global memory.  mma.m16n8k16 wants of lane (g = lane / 4, t = lane % 4) the
 * k's {2t, 2t+1, 2t+8, 2t+9} of rows g and g + 8 of A and of column g of B.  A sum does not mind the order of its terms, so k is
 * renamed: lane t loads k = 16t .. 16t+15 of a block of 64 as 32 bytes, four at a time of which are the steps' shares.  Both operands use the
 * same names, four lanes read a line of 128 bytes of a row, and no shared memory is touched.  (Blocks of 32 k's, 16 bytes a lane, touch
 * eight half lines an instruction: 1 row of 192 experts 57.7 us a pass instead of 55.1, adapters of 64 rows 24.9 instead of 23.4.)
 */
#ifndef HY3A_LAYER_H
#define HY3A_LAYER_H

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>

#include "ctx.h"

/* The current device's number and SM count; refuses devices that sm_100a code cannot run on. */
int hy3a_layer_device(const char *who, int *device, int *sms);

/* Whether sizes of a matrix in 4 bits are in their limits: 0 or HY3A_EINVAL. */
int hy3a_quant4_sizes(const char *who, int out_width, int width, int group);

/* Where the files' error words {code, where} of the first wait that ran out lie on the current device (hy3a_layer_sync reads and clears them) */
cudaError_t hy3a_experts_words(unsigned **words);
cudaError_t hy3a_adapters_words(unsigned **words);
cudaError_t hy3a_linear4_words(unsigned **words);
cudaError_t hy3a_linear4_many_words(unsigned **words);
/* a launch of the file's with one wait that runs out */
cudaError_t hy3a_experts_wait_out(void *stream);
cudaError_t hy3a_adapters_wait_out(void *stream);
cudaError_t hy3a_linear4_wait_out(void *stream);
cudaError_t hy3a_linear4_many_wait_out(void *stream);

/* launch configuration with programmatic stream serialisation: the kernels wait (pdl_wait) before they touch memory */
struct hy3a_launch {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    hy3a_launch(dim3 grid, dim3 block, size_t smem, void *stream) : cfg(), attr() {
        cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t)stream;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr; cfg.numAttrs = 1;
    }
    void cluster(int x, int y = 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = x; attr[1].val.clusterDim.y = y; attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
};

namespace hy3a_layer {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class T> struct type;
template <> struct type<__nv_bfloat16> {
    static constexpr int code = HY3A_BF16;
    static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ __nv_bfloat16 cut(float v) { return __float2bfloat16_rz(v); }
    static __device__ __forceinline__ __nv_bfloat16 step_down(__nv_bfloat16 v) { return __ushort_as_bfloat16(__bfloat16_as_ushort(v) - 1); }      /* next towards 0, of what is not 0 */
    static __device__ __forceinline__ __nv_bfloat16 least(float v) { return __ushort_as_bfloat16(v < 0.f ? 0x8080 : 0x0080); }                      /* smallest normal number of v's sign */
    static __device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
template <> struct type<__half> {
    static constexpr int code = HY3A_F16;
    static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ __half cut(float v) { return __float2half_rz(v); }
    static __device__ __forceinline__ __half step_down(__half v) { return __ushort_as_half(__half_as_ushort(v) - 1); }
    static __device__ __forceinline__ __half least(float v) { return __ushort_as_half(v < 0.f ? 0x8001 : 0x0001); }      /* (subnormal: the normal ones begin at 2^-14) */
    static __device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
template <> struct type<float> {
    static constexpr int code = HY3A_F32;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};

__device__ __forceinline__ uint4 load_row(const void *p) { return *reinterpret_cast<const uint4 *>(p); }
__device__ __forceinline__ uint4 zero16() { return make_uint4(0, 0, 0, 0); }

/* 16 k's of a row, of which `left` (a multiple of 8) are there, the others 0.  WIDE: rows start on 32-byte boundaries and are multiples of 16.
 * ONCE: not kept in L1 (weights). */
struct k16 { unsigned v[8]; };
template <bool WIDE, bool ONCE> __device__ __forceinline__ k16 load16(const void *p, int left) {
    k16 r;
#pragma unroll
    for (int i = 0; i < 8; i++) r.v[i] = 0u;
    if (WIDE) {
        if (left > 0) {
            if (ONCE) asm("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]), "=r"(r.v[7]) : "l"(p));
            else asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]), "=r"(r.v[7]) : "l"(p));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (left > 8 * i) {
                const char *q = reinterpret_cast<const char *>(p) + 16 * i;
                if (ONCE) asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.v[4 * i]), "=r"(r.v[4 * i + 1]), "=r"(r.v[4 * i + 2]), "=r"(r.v[4 * i + 3]) : "l"(q));
                else asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.v[4 * i]), "=r"(r.v[4 * i + 1]), "=r"(r.v[4 * i + 2]), "=r"(r.v[4 * i + 3]) : "l"(q));
            }
        }
    }
    return r;
}
/* a block of 64 k's: rows g (lo) and g + 8 (hi) of A, column g of B, 16 k's each */
template <class T> __device__ __forceinline__ void mma64(float (&d)[4], const k16 &lo, const k16 &hi, const k16 &b) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) type<T>::mma(d, lo.v[i], hi.v[i], lo.v[i + 1], hi.v[i + 1], b.v[i], b.v[i + 1]);
}
/* the same of 32 k's, 8 each (operands in shared memory) */
template <class T> __device__ __forceinline__ void mma32(float (&d)[4], const uint4 &lo, const uint4 &hi, const uint4 &b) {
    type<T>::mma(d, lo.x, hi.x, lo.y, hi.y, b.x, b.y);
    type<T>::mma(d, lo.z, hi.z, lo.w, hi.w, b.z, b.w);
}
/* whether rows of so many 16-bit elements, at these strides and addresses, can be loaded 32 bytes at a time */
static inline bool wide_rows(std::initializer_list<const void *> p, std::initializer_list<size_t> n) {
    for (const void *q : p) if ((uintptr_t)q & 31) return false;
    for (size_t k : n) if (k & 15) return false;
    return true;
}

} /* namespace hy3a_layer */
#endif

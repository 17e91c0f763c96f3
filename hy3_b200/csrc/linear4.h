/* linear4.h -- what the kernels of hy3a_linear4 share (linear4.cu: few rows; linear4_umma.cu: many). */
#ifndef HY3A_LINEAR4_H
#define HY3A_LINEAR4_H

#include "layer.h"

struct linear4_args {
    const void *x;            /* [rows][width], 16-bit type T */
    size_t x_stride;
    const uint8_t *codes;     /* [out_width][width / 2] */
    const void *scales;       /* [out_width][groups], T */
    void *out;                /* [rows][out_width], T or fp32 */
    size_t out_stride;
    int rows, width, out_width, group, groups;
    int wide;                 /* out is fp32 */
};

/* linear4_umma.cu: any number of rows; *what: why, where it is not CUDA's error */
cudaError_t hy3a_linear4_launch_many(const linear4_args &a, int dtype, int device, void *stream, const char **what);

namespace hy3a_layer {

/* Codes become numbers of the rows' type by their bits: with a code c in the lowest bits of the mantissa, 0x4300 | c is 128 + c in bf16 and 0x6400 | c is 1024 + c in
 * fp16 (with c four bits higher 1024 + 16 c), and the subtraction of 128 + 8, or 1024 + 8, is exact.  A word's codes k = 0 .. 7 come as the pairs (0, 4), (1, 5),
 * (2, 6), (3, 7). */
__device__ __forceinline__ unsigned and_or(unsigned a, unsigned mask, unsigned bits) {
    unsigned r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
}
template <class T> struct steps;
template <> struct steps<__nv_bfloat16> {
    /* the same as the pairs (0, 1), (2, 3), (4, 5), (6, 7) */
    static __device__ __forceinline__ void in_order(unsigned w, unsigned (&v)[4]) {
        const unsigned odd = w >> 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned c = and_or(__byte_perm(w, odd, 0x4400 + 0x1111 * i), 0x000f000fu, 0x43004300u);
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(v[i]) : "r"(c), "r"(0x43084308u));
        }
    }
    static __device__ __forceinline__ void of(unsigned w, unsigned (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned c = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(v[i]) : "r"(c), "r"(0x43084308u));
        }
    }
    /* the same in units of 1 / kPerStep, in 9 operations a word and not 11: a nibble in bits 0-3 or 4-7 of a 16-bit number is that many 2^-133 or 2^-129 as it stands (subnormal, or of the lowest exponent) */
    static constexpr float kPerStep = 64.f;
    static __device__ __forceinline__ void parts(unsigned w, unsigned (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const unsigned u = i ? w >> 8 : w;
            asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v[i]) : "r"(u & 0x000f000fu), "r"(0x7f007f00u) /* 2^127 */, "r"(0xbe00be00u) /* -1 / 8 */);
            asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v[i + 1]) : "r"(u & 0x00f000f0u), "r"(0x7d007d00u) /* 2^123 */, "r"(0xbe00be00u));
        }
    }
};
template <> struct steps<__half> {
    static __device__ __forceinline__ void in_order(unsigned w, unsigned (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned c = and_or(__byte_perm(w, 0, 0x1111 * i), 0x00f0000fu, 0x64006400u);       /* 1024 + c, 1024 + 16 c */
            asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v[i]) : "r"(c), "r"(0x2c003c00u) /* 1, 1 / 16 */, "r"(0xd480e408u) /* -1032, -72 */);
        }
    }
    static __device__ __forceinline__ void of(unsigned w, unsigned (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const unsigned u = i ? w >> 8 : w, lo = and_or(u, 0x000f000fu, 0x64006400u), hi = and_or(u, 0x00f000f0u, 0x64006400u);
            asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(v[i]) : "r"(lo), "r"(0x64086408u));
            asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v[i + 1]) : "r"(hi), "r"(0x2c002c00u) /* 1 / 16 */, "r"(0xd480d480u) /* -72 */);
        }
    }
    static constexpr float kPerStep = 1.f;
    static __device__ __forceinline__ void parts(unsigned w, unsigned (&v)[4]) { of(w, v); }
};

/* whether row t of x has a NaN, for a warp */
template <class T> __device__ __forceinline__ bool has_nan(const linear4_args &a, int t) {
    const uint4 *const x = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.x) + (size_t)t * a.x_stride);
    constexpr unsigned kInf = type<T>::code == HY3A_BF16 ? 0x7f80u : 0x7c00u;
    /* (rows that nobody wrote have theirs early) */
#pragma unroll 1
    for (int i0 = threadIdx.x & 31, n = a.width / 8; __any_sync(0xffffffffu, i0 < n); i0 += 128) {
        bool is = false;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (i0 + 32 * u >= n) continue;
            const uint4 v = x[i0 + 32 * u];
            const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) is |= (w[j] & 0x7fffu) > kInf || (w[j] >> 16 & 0x7fffu) > kInf;
        }
        if (__any_sync(0xffffffffu, is)) return true;
    }
    return false;
}
/* out[t][o] from the definition, by a warp; weights in eighths, which are exact: 8 steps of a scale from 2^125 on are beyond fp32 where their products with x need not be */
template <class T> __device__ __forceinline__ float plain(const linear4_args &a, int t, int o) {
    const uint4 *const x = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.x) + (size_t)t * a.x_stride), *const codes = reinterpret_cast<const uint4 *>(a.codes + (size_t)o * (a.width / 2));
    const T *const scales = reinterpret_cast<const T *>(a.scales) + (size_t)o * a.groups;
    float sum = 0.f;
#pragma unroll 1
    for (int i = threadIdx.x & 31; i < a.width / 32; i += 32) {         /* 32 k's, of one group */
        const uint4 c = codes[i];
        const unsigned w[4] = {c.x, c.y, c.z, c.w};
        const float s = 0.125f * type<T>::up(scales[i * 32 / a.group]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint4 v = x[4 * i + j];
            const unsigned pairs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const unsigned short u = (unsigned short)(k % 2 ? pairs[k / 2] >> 16 : pairs[k / 2]);
                sum = fmaf((float)((int)(w[j] >> (4 * k) & 15u) - 8) * s, type<T>::up(*reinterpret_cast<const T *>(&u)), sum);
            }
        }
    }
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    return 8.f * sum;
}
} /* namespace hy3a_layer */
#endif

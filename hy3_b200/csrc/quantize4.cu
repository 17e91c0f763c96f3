/*
 * quantize4.cu -- weights to 4 bits with a scale for each group of neighbours in a row (hy3a_quantize4).
 *
 *      ext = the group's largest value if that is larger than minus its smallest, else its smallest;   s = ext / -8, rounded to the scales' type
 *      q = min(max(rint(w / s), -8), 7) + 8
 *
 * so that the value of the largest magnitude is 8 steps from 0, on the side that has 8.  Codes are counted in steps of the rounded scale, with IEEE division.
 *
 * A lane takes 16 neighbours, two to eight lanes meet for a group.  What bounds it is memory, if the instructions stay below that.
 */
#include "layer.h"

namespace {

using namespace hy3a_layer;

constexpr int kThreads = 256;

struct quantize_args {
    const void *w;
    size_t stride;
    uint8_t *codes;
    void *scales;
    size_t out;
    int units;           /* of 16 values in a row, */
    int padded;          /* and in a row of full groups */
    int groups;
};

__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

template <class W> __device__ __forceinline__ void load_values(const W *p, float (&v)[16]) {
    constexpr int kOf = 16 / sizeof(W);        /* values in 16 bytes */
#pragma unroll
    for (int i = 0; i < 16 / kOf; i++) {
        const uint4 raw = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
        const W *const r = reinterpret_cast<const W *>(&raw);
#pragma unroll
        for (int j = 0; j < kOf; j++) v[i * kOf + j] = type<W>::up(r[j]);
    }
}

/* GROUP: values of a group */
template <class W, class S, int GROUP>
__global__ void __launch_bounds__(kThreads) hy3a_quantize4_kernel(const quantize_args a) {
    constexpr int kLanes = GROUP / 16;
    pdl_release();
    pdl_wait();
    const size_t total = a.out * a.padded, step = (size_t)gridDim.x * kThreads;
    /* (the last lanes of a warp that have nothing left still meet the others) */
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i - (threadIdx.x & 31) < total; i += step) {
        const size_t row = i / a.padded;
        const int unit = (int)(i - row * a.padded);
        const bool here = i < total && unit < a.units;
        float v[16];
        if (here) load_values(reinterpret_cast<const W *>(a.w) + row * a.stride + (size_t)unit * 16, v);
        else {
#pragma unroll
            for (int j = 0; j < 16; j++) v[j] = 0.f;
        }
        /* 0 among the values changes neither bound that counts */
        float hi = 0.f, lo = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j++) { hi = max_nan(hi, v[j]); lo = min_nan(lo, v[j]); }
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) {
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        }
        const S s = type<S>::down(__fadd_rn((hi > -lo ? hi : lo) * -0.125f, 0.f));       /* (no -0) */
        const float step_size = type<S>::up(s);
        unsigned word[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const float t = fminf(fmaxf(rintf(__fdiv_rn(v[j], step_size)), -8.f), 7.f);
            word[j / 8] |= (unsigned)((int)t + 8) << (4 * (j % 8));
        }
        /* a group whose scale is 0 or not finite has no steps */
        if (!(fabsf(step_size) > 0.f && fabsf(step_size) < INFINITY)) word[0] = word[1] = 0x88888888u;
        if (!here) continue;
        *reinterpret_cast<uint2 *>(a.codes + (row * a.units + unit) * 8) = make_uint2(word[0], word[1]);
        if (unit % kLanes == 0) reinterpret_cast<S *>(a.scales)[row * a.groups + unit / kLanes] = s;
    }
}

template <class W, class S>
cudaError_t launch(const quantize_args &a, int group, int sms, void *stream) {
    const size_t blocks = (a.out * a.padded + kThreads - 1) / kThreads, most = (size_t)sms * 8;
    hy3a_launch l(dim3((unsigned)(blocks < most ? blocks : most)), dim3(kThreads), 0, stream);
    if (group == 32) return cudaLaunchKernelEx(&l.cfg, hy3a_quantize4_kernel<W, S, 32>, a);
    if (group == 64) return cudaLaunchKernelEx(&l.cfg, hy3a_quantize4_kernel<W, S, 64>, a);
    return cudaLaunchKernelEx(&l.cfg, hy3a_quantize4_kernel<W, S, 128>, a);
}
template <class W>
cudaError_t launch_type(const quantize_args &a, int dtype, int group, int sms, void *stream) {
    return dtype == HY3A_BF16 ? launch<W, __nv_bfloat16>(a, group, sms, stream) : launch<W, __half>(a, group, sms, stream);
}

} /* namespace */

extern "C" int hy3a_quantize4(void *stream, int w_dtype, int out_width, int width, int group, const void *w, size_t w_stride, int dtype, void *codes, void *scales) {
    if (w_dtype != HY3A_F32 && w_dtype != HY3A_F16 && w_dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "quantize4: w_dtype %d not in {0,1,2}", w_dtype);
    if (dtype != HY3A_F16 && dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "quantize4: dtype %d not in {1,2}", dtype);
    int rc = hy3a_quant4_sizes("quantize4", out_width, width, group);
    if (rc) return rc;
    if (out_width == 0) return HY3A_OK;
    if (!w || !codes || !scales) return hy3a_fail(NULL, HY3A_EINVAL, "quantize4: NULL argument");
    const size_t el = w_dtype == HY3A_F32 ? 4 : 2;
    if (((uintptr_t)w | (uintptr_t)codes) & 15) return hy3a_fail(NULL, HY3A_EINVAL, "quantize4: w and codes have to be 16-byte aligned");
    if ((uintptr_t)scales & 1) return hy3a_fail(NULL, HY3A_EINVAL, "quantize4: scales are not aligned to their type");
    if (w_stride * el % 16) return hy3a_fail(NULL, HY3A_EINVAL, "quantize4: rows of w have to start on 16-byte boundaries");
    int dev, sms;
    if ((rc = hy3a_layer_device("quantize4", &dev, &sms))) return rc;
    const int groups = (width + group - 1) / group;
    const quantize_args a = {w, w_stride, (uint8_t *)codes, scales, (size_t)out_width, width / 16, groups * (group / 16), groups};
    const cudaError_t e = w_dtype == HY3A_F32 ? launch_type<float>(a, dtype, group, sms, stream)
                        : (w_dtype == HY3A_F16 ? launch_type<__half>(a, dtype, group, sms, stream) : launch_type<__nv_bfloat16>(a, dtype, group, sms, stream));
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "quantize4: %s", cudaGetErrorString(e));
    return HY3A_OK;
}

/*
 * quantize4.cu -- weights to 4 bits with a scale for each group of neighbours in a row (hy3a_quantize4).
 *
 *      ext = the group's largest value if that is larger than minus its smallest, else its smallest;   s = ext / -8, rounded to the scales' type
 *      q = min(max(rint(w / s), -8), 7) + 8
 *
 * so that the value of the largest magnitude is 8 steps from 0, on the side that has 8.  Codes are counted in steps of the rounded scale, with IEEE division.
 *
 * A lane takes 32 neighbours, one to four lanes meet for a group, and the next ones' values are on their way meanwhile.  Memory bounds it (120832 x 4096 bf16: 204 to 207 us, 6.1 TB/s; fp32, whose quotients are looked at one by one, 457 us, 4.9 TB/s), if the instructions stay
 * below that: a division and two conversions for each value keep the unit of special functions busy for three times as long (572 us), 16 values a lane are 290 us.
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
    int out;
    int units;           /* of 32 values in a row, */
    int padded;          /* and in a row of full groups */
    int groups;
    int shift;           /* 2^shift threads take a row */
};

__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

/* 32 values and the bounds of theirs (and 0, which changes neither bound that counts); those of 16 bits are compared two at a time */
template <class W> struct values;
template <> struct values<float> {
    uint4 raw[8];
    __device__ __forceinline__ void load(const void *p) {
#pragma unroll
        for (int i = 0; i < 8; i++) raw[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ float at(int j) const { const uint4 &r = raw[j / 4]; return __uint_as_float(j % 4 == 0 ? r.x : (j % 4 == 1 ? r.y : (j % 4 == 2 ? r.z : r.w))); }
    __device__ __forceinline__ void bounds(float &hi, float &lo) const {
        hi = lo = 0.f;
#pragma unroll
        for (int j = 0; j < 32; j++) { hi = max_nan(hi, at(j)); lo = min_nan(lo, at(j)); }
    }
};
template <class W> struct values16 {
    uint4 raw[4];
    __device__ __forceinline__ void load(const void *p) {
#pragma unroll
        for (int i = 0; i < 4; i++) raw[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ unsigned word(int i) const { const uint4 &r = raw[i / 4]; return i % 4 == 0 ? r.x : (i % 4 == 1 ? r.y : (i % 4 == 2 ? r.z : r.w)); }
    __device__ __forceinline__ float at(int j) const {
        const unsigned short u = (unsigned short)(j % 2 ? word(j / 2) >> 16 : word(j / 2));
        return type<W>::up(*reinterpret_cast<const W *>(&u));
    }
    template <class Max, class Min> __device__ __forceinline__ void bounds_by(float &hi, float &lo, const Max &most, const Min &least) const {
        unsigned h = 0u, l = 0u;
#pragma unroll
        for (int i = 0; i < 16; i++) { h = most(h, word(i)); l = least(l, word(i)); }
        const unsigned short a[4] = {(unsigned short)h, (unsigned short)(h >> 16), (unsigned short)l, (unsigned short)(l >> 16)};
        hi = max_nan(type<W>::up(*reinterpret_cast<const W *>(&a[0])), type<W>::up(*reinterpret_cast<const W *>(&a[1])));
        lo = min_nan(type<W>::up(*reinterpret_cast<const W *>(&a[2])), type<W>::up(*reinterpret_cast<const W *>(&a[3])));
    }
};
template <> struct values<__nv_bfloat16> : values16<__nv_bfloat16> {
    __device__ __forceinline__ void bounds(float &hi, float &lo) const {
        bounds_by(hi, lo, [](unsigned a, unsigned b) { unsigned r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; },
                  [](unsigned a, unsigned b) { unsigned r; asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; });
    }
};
template <> struct values<__half> : values16<__half> {
    __device__ __forceinline__ void bounds(float &hi, float &lo) const {
        bounds_by(hi, lo, [](unsigned a, unsigned b) { unsigned r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; },
                  [](unsigned a, unsigned b) { unsigned r; asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; });
    }
};

/* 8 + the steps of v, by the definition; a group whose scale is 0 or not finite has none */
__device__ __noinline__ unsigned code_of(float v, float s) {
    if (!(fabsf(s) > 0.f && fabsf(s) < INFINITY)) return 8u;
    return (unsigned)((int)fminf(fmaxf(rintf(__fdiv_rn(v, s)), -8.f), 7.f) + 8);
}

/* r = 3 2^22 + 8 + rint(w / s): the code in its last bits; off: how far w / s is from what it was rounded to.  Two at a time. */
constexpr float kMagic = 12582920.f;
struct f2 { float x, y; };
__device__ __forceinline__ unsigned long long bits(f2 v) { unsigned long long r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y)); return r; }
__device__ __forceinline__ f2 pair(unsigned long long v) { f2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { unsigned long long r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c))); return pair(r); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { unsigned long long r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b))); return pair(r); }
__device__ __forceinline__ void rounded(f2 w, float inverse, f2 &r, f2 &off) {
    r = fma2(w, {inverse, inverse}, {kMagic, kMagic});
    off = fma2(w, {-inverse, -inverse}, add2(r, {-kMagic, -kMagic}));
}

/* GROUP: values of a group.  A row is taken by 2^shift threads of a block. */
template <class W, class S, int GROUP>
__global__ void __launch_bounds__(kThreads) hy3a_quantize4_kernel(const quantize_args a) {
    constexpr int kLanes = GROUP / 32;
    const int first = threadIdx.x & ((1 << a.shift) - 1), step = gridDim.x << (8 - a.shift);       /* (in a row; rows) */
    int row = (blockIdx.x << (8 - a.shift)) + (threadIdx.x >> a.shift), unit = first;
    pdl_release();
    pdl_wait();
    /* the next values are on their way while these are worked on */
    values<W> next;
    const auto load = [&]() { if (row < a.out && unit < a.units) next.load(reinterpret_cast<const W *>(a.w) + (size_t)row * a.stride + (size_t)unit * 32); };
    load();
    /* (lanes meet by groups, and the threads of a row go as far as its groups: those of a warp have the same number of turns) */
    while (__any_sync(0xffffffffu, row < a.out)) {
        const values<W> v = next;
        const int row_now = row, unit_now = unit;
        const bool here = row < a.out && unit < a.units;
        unit += 1 << a.shift;
        if (unit - first >= a.padded) { unit = first; row += step; }
        load();
        float hi = 0.f, lo = 0.f;
        if (here) v.bounds(hi, lo);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) {
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        }
        if (here) {
            const float far = hi > -lo ? hi : lo;
            const S s = type<S>::down(__fadd_rn(far * -0.125f, 0.f));       /* (no -0) */
            const float step_size = type<S>::up(s), inverse = __fdividef(1.f, step_size);
            /* A product with 1 / s is off by 2^-19 at most.  Quotients of numbers of 16 bits are in the middle between two codes, or 2^-13 and more beside it, so that
             * products are as good once they are rounded to multiples of 2^-16.  Of fp32 values, whose quotients are off by 2^-21 and may be any, those within 2^-18 of the middle are divided.
             * Steps are more than 8 and a little where the scale is subnormal, and 1 / s is no use where it is 0 or not finite. */
            const bool regular = fabsf(fmaf(far, inverse, 8.f)) < 0.4f;
            constexpr float kNear = 0.5f - 0x1p-18f;
            unsigned word[4];
#pragma unroll
            for (int h = 0; h < 4; h++) {
                /* codes k and k + 4 of a word as the 16-bit halves of one number, 8 + 8 at most */
                float off = 0.f;
                word[h] = 0u;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    f2 r, e;
                    if (sizeof(W) == 2) r = add2(fma2({v.at(8 * h + k), v.at(8 * h + k + 4)}, {inverse, inverse}, {192.f, 192.f}), {kMagic - 192.f, kMagic - 192.f});      /* (192 + t: steps of 2^-16) */
                    else {
                        rounded({v.at(8 * h + k), v.at(8 * h + k + 4)}, inverse, r, e);
                        off = fmaxf(off, fmaxf(fabsf(e.x), fabsf(e.y)));
                    }
                    unsigned c = __byte_perm(__float_as_uint(r.x), __float_as_uint(r.y), 0x5410);
                    asm("min.u16x2 %0, %0, %1;" : "+r"(c) : "r"(0x000f000fu));
                    word[h] += c << (4 * k);
                }
                if (!regular || !(off < kNear)) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const f2 w = {v.at(8 * h + k), v.at(8 * h + k + 4)};
                        f2 r, e;
                        rounded(w, inverse, r, e);
                        if (!regular || !(fabsf(e.x) < kNear)) word[h] = (word[h] & ~(15u << (4 * k))) | code_of(w.x, step_size) << (4 * k);
                        if (!regular || !(fabsf(e.y) < kNear)) word[h] = (word[h] & ~(15u << (4 * k + 16))) | code_of(w.y, step_size) << (4 * k + 16);
                    }
                }
            }
            *reinterpret_cast<uint4 *>(a.codes + ((size_t)row_now * a.units + unit_now) * 16) = make_uint4(word[0], word[1], word[2], word[3]);
            if (unit_now % kLanes == 0) reinterpret_cast<S *>(a.scales)[(size_t)row_now * a.groups + unit_now / kLanes] = s;
        }
    }
}

template <class W, class S>
cudaError_t launch(const quantize_args &a, int group, int sms, void *stream) {
    const int blocks = (a.out + (kThreads >> a.shift) - 1) / (kThreads >> a.shift);
    hy3a_launch l(dim3(blocks < sms * 8 ? blocks : sms * 8), dim3(kThreads), 0, stream);
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
    quantize_args a = {w, w_stride, (uint8_t *)codes, scales, out_width, width / 32, groups * (group / 32), groups, 2};
    while (a.shift < 8 && (1 << a.shift) < a.padded) a.shift++;
    const cudaError_t e = w_dtype == HY3A_F32 ? launch_type<float>(a, dtype, group, sms, stream)
                        : (w_dtype == HY3A_F16 ? launch_type<__half>(a, dtype, group, sms, stream) : launch_type<__nv_bfloat16>(a, dtype, group, sms, stream));
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "quantize4: %s", cudaGetErrorString(e));
    return HY3A_OK;
}

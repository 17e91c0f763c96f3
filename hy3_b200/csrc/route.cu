/*
 * route.cu -- routing of rows to experts (hy3a_route), and the device check of the operators beside the attention.
 *
 * s = sigmoid(l) or softmax(l); c = s + bias picks; w = s (renormalised, scaled) weighs.  The selection is a matter of exact values: c
 * is computed with IEEE division and CUDA's expf, the softmax's denominator is summed in 64 bits and rounded once (its value then
 * does not hang on the order of the sum), and ties go to the lowest index.
 *
 * A warp takes a row, a lane every 32nd expert.  What bounds it is the number of instructions (a row of 256 logits is 512 to 1024 bytes), so the top
 * k are not looked for k times over all values: the k-th largest of the 32 lanes' maxima is no larger than the k-th largest value, and the
 * few values (10 or so of 192) that reach it are packed into a lane each and ranked.  A softmax without bias is selected by exp(l - max), and
 * only what reaches the threshold is divided: the quotients are in the same order, except that neighbours may round to one, so the threshold
 * is lowered by more than a rounding.  Rows where more than 32 values reach it (many equal ones) take k searches.
 * 16384 rows of 256 logits in 8 groups take 17.6 us a pass (8.9 MB, 1.4 us of memory); up to 2048 rows of 192 the pass is the host's call (5.4).
 */
#include <atomic>

#include "layer.h"

int hy3a_layer_device(const char *who, int *device, int *sms) {
    static std::atomic<int> known[64];      /* per device: 0 not asked yet, -1 another architecture, else its SM count */
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "%s: no CUDA device (%s): this library has no CPU path", who, cudaGetErrorString(e));
    int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        int major = 0, minor = 0;
        if ((e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev)) != cudaSuccess ||
            (e = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev)) != cudaSuccess ||
            (e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
            return hy3a_fail(NULL, HY3A_ECUDA, "%s: %s", who, cudaGetErrorString(e));
        if (major != 10 || minor != 0) n = -1;
        if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    }
    if (n < 0) return hy3a_fail(NULL, HY3A_EDEVICE, "%s: device %d is not of compute capability 10.0; the kernels are built for sm_100a only", who, dev);
    *device = dev;
    *sms = n;
    return 0;
}

namespace {

using namespace hy3a_layer;

constexpr int kWarps = 4;             /* rows per block, a warp each */
constexpr int kMaxExperts = 1024, kMaxTopK = 32, kMaxGroups = 32;

/* order of floats as unsigned numbers; no c is -0 (s >= +0, and x + -x rounds to +0) */
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned u = __float_as_uint(v);
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

struct route_args {
    const void *logits;
    size_t stride;
    const float *bias;
    int rows, experts, top_k, softmax, groups, top_groups, renormalize, group_size, group_shift /* 2^shift lanes scan a group */, group_skew;
    unsigned group_magic;            /* 2^32 / group_size, rounded up: x / group_size is the upper half of x * group_magic for x < 1024 and group_size > 1 */
    float scale;
    int *ids;
    float *weights;
};

__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

/* the two best of two pairs */
__device__ __forceinline__ void two_best(float &a, float &b, float c, float d) {
    const float lo = fminf(a, c);
    a = fmaxf(a, c);
    b = fmaxf(lo, fmaxf(b, d));
}

constexpr float kLowest = -3.402823466e38f;
/* what a pick counts for: below everything that is open, but open, if it is NaN, so that a row of NaN keeps ids in range and shows NaN weights */
__device__ __forceinline__ unsigned key_of(float c, bool open) { return !open || c == -INFINITY ? 0u : ordered(isnan(c) ? kLowest : c); }

/* One warp per row; lane i holds experts i, i + 32, ... (coalesced), VPL of them.  QUOTIENT: softmax without bias. */
template <class T, int VPL, bool GROUPED, bool QUOTIENT>
__global__ void __launch_bounds__(32 * kWarps) hy3a_route_kernel(const route_args a) {
    __shared__ float s_pick[GROUPED ? kWarps : 1][GROUPED ? 32 * VPL : 1];
    __shared__ uint4 s_few[kWarps][32];                  /* {key, score, expert} of what reaches the threshold */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * kWarps + warp;
    pdl_release();
    pdl_wait();
    if (row >= a.rows) return;
    const T *l = reinterpret_cast<const T *>(a.logits) + (size_t)row * a.stride;
    float s[VPL];                                       /* scores; QUOTIENT: numerators */
    unsigned key[VPL];                                  /* order of picks, 0: closed */
#pragma unroll
    for (int j = 0; j < VPL; j++) s[j] = lane + 32 * j < a.experts ? type<T>::up(l[lane + 32 * j]) : -INFINITY;
    unsigned open = 0;                /* bit j: not closed by a logit of -inf (and there) */
#pragma unroll
    for (int j = 0; j < VPL; j++) open |= s[j] == -INFINITY ? 0u : 1u << j;
    float d = 1.f;                    /* denominator */
    bool row_nan = false;
    if (QUOTIENT || a.softmax) {
        float m = s[0];
#pragma unroll
        for (int j = 1; j < VPL; j++) m = max_nan(m, s[j]);       /* a row with a NaN has no softmax */
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < VPL; j++) {
            s[j] = lane + 32 * j < a.experts ? expf(__fsub_rn(s[j], m)) : 0.f;
            sum += (double)s[j];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        d = (float)sum;
        row_nan = isnan(d);           /* also of a row without open experts, and of one with +inf */
        if (!QUOTIENT) {
#pragma unroll
            for (int j = 0; j < VPL; j++) s[j] = __fdiv_rn(s[j], d);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPL; j++) s[j] = __fdiv_rn(1.f, __fadd_rn(1.f, expf(-s[j])));
    }
#pragma unroll
    for (int j = 0; j < VPL; j++) {
        const int e = lane + 32 * j;
        if (QUOTIENT) {
            const float v = row_nan ? 0.f : s[j];       /* numerators of a NaN row count alike: its quotients all are NaN */
            key[j] = (open >> j) & 1 ? __float_as_uint(v) + 1u : 0u;
            if (GROUPED) s_pick[warp][e] = (open >> j) & 1 ? v : -INFINITY;
        } else {
            const float c = a.bias && e < a.experts ? __fadd_rn(s[j], a.bias[e]) : s[j];
            key[j] = key_of(c, (open >> j) & 1);
            if (GROUPED) s_pick[warp][e] = !((open >> j) & 1) ? -INFINITY : (isnan(c) ? kLowest : c);
        }
    }
    if (GROUPED) {
        /* a group stands with the sum of its two best open experts: `per` lanes scan each group, and meet */
        const int size = a.group_size, shift = a.group_shift, per = 1 << shift, grp = lane >> shift, sub = lane & (per - 1);
        float b1 = -INFINITY, b2 = -INFINITY;
        __syncwarp();
        if (grp < a.groups) {
            const float *p = s_pick[warp] + grp * size;
            int i = sub + (a.group_skew ? lane - sub : 0);       /* groups of 32 would all start in the same bank */
            for (int q = sub; q < size; q += per) {
                const float v = p[i];
                b2 = fmaxf(b2, fminf(b1, v));
                b1 = fmaxf(b1, v);
                i += per;
                if (i >= size) i -= size;
            }
        }
        for (int o = 1; o < per; o <<= 1) {
            const float c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
            two_best(b1, b2, c1, c2);
        }
        if (QUOTIENT) {
            b1 = b1 == -INFINITY ? b1 : (row_nan ? kLowest : __fdiv_rn(b1, d));
            b2 = b2 == -INFINITY ? b2 : (row_nan ? kLowest : __fdiv_rn(b2, d));
        }
        const float stands = b2 == -INFINITY ? b1 : fmaxf(__fadd_rn(b1, b2), kLowest);      /* (two NaN: still before a group without open experts) */
        /* groups that come before this one: better, or as good with a lower index (o > mine, or o >= mine: a key is at least 1) */
        const unsigned mine = ordered(stands);
        int before = 0;
        for (int g = 0; g < a.groups; g++) before += __shfl_sync(0xffffffffu, mine, g << shift) > mine - (g < grp);
        const unsigned kept = __ballot_sync(0xffffffffu, before < a.top_groups);
#pragma unroll
        for (int j = 0; j < VPL; j++) {
            const int g = size == 1 ? lane + 32 * j : (int)__umulhi((unsigned)(lane + 32 * j), a.group_magic);      /* (past the last expert: any, it is closed) */
            if (!((kept >> ((g << shift) & 31)) & 1)) key[j] = 0u;
        }
    }
    /* the k-th largest of the lanes' maxima (equal ones leave together: then of more than k) */
    unsigned m = key[0], least = 0;
#pragma unroll
    for (int j = 1; j < VPL; j++) m = max(m, key[j]);
    for (int r = 0; r < a.top_k; r++) {
        least = __reduce_max_sync(0xffffffffu, m);
        if (m == least) m = 0u;
    }
    if (QUOTIENT && least) {
        /* quotients of numerators that differ by less than 2^-22 may be equal; near the subnormal numbers by more: then everything counts */
        const float t = __uint_as_float(least - 1u);
        least = t > 1e-30f ? __float_as_uint(t * (1.f - 9.5367e-7f)) + 1u : 1u;
    }
    least = max(least, 1u);
    int n = 0;
#pragma unroll
    for (int j = 0; j < VPL; j++) {
        const bool in = key[j] >= least;
        const unsigned all = __ballot_sync(0xffffffffu, in);
        const int at = n + __popc(all & ((1u << lane) - 1u));
        if (in && at < 32) s_few[warp][at] = make_uint4(key[j], __float_as_uint(s[j]), lane + 32 * j, 0u);
        n += __popc(all);
    }
    int my_id = -1, rank = lane;                        /* the rank-th choice: expert and weight */
    float my_w = 0.f;
    if (n <= 32) {
        __syncwarp();
        const uint4 few = s_few[warp][lane];
        unsigned k = lane < n ? few.x : 0u;
        float w = __uint_as_float(few.y);
        if (QUOTIENT) {
            w = __fdiv_rn(w, d);
            if (k) k = key_of(w, true);
        }
        /* (the list is in the order of the experts) */
        rank = 0;
#pragma unroll 4
        for (int i = 0; i < n; i++) rank += __shfl_sync(0xffffffffu, k, i) > k - (k && i < lane);      /* larger, or as large and before it */
        if (lane < n) { my_id = (int)few.z; my_w = w; }
        else rank = lane;                               /* (lanes past the list: the choices that are left) */
    } else {
        if (QUOTIENT) {
#pragma unroll
            for (int j = 0; j < VPL; j++) {
                s[j] = __fdiv_rn(s[j], d);
                if (key[j]) key[j] = key_of(s[j], true);
            }
        }
        for (int r = 0; r < a.top_k; r++) {
            unsigned top = key[0];
#pragma unroll
            for (int j = 1; j < VPL; j++) top = max(top, key[j]);
            const unsigned best = __reduce_max_sync(0xffffffffu, top);
            if (best == 0u) break;                      /* only closed experts are left */
            int e = 0x7fffffff;
#pragma unroll
            for (int j = VPL - 1; j >= 0; j--) if (key[j] == best) e = lane + 32 * j;
            const int id = __reduce_min_sync(0xffffffffu, e);
            float w = 0.f;
#pragma unroll
            for (int j = 0; j < VPL; j++) if (lane + 32 * j == id) { key[j] = 0u; w = s[j]; }
            w = __shfl_sync(0xffffffffu, w, id & 31);
            if (lane == r) { my_id = id; my_w = w; }
        }
    }
    if (rank >= a.top_k) my_w = 0.f;
    if (a.renormalize) {
        float sum = my_w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        my_w = __fdiv_rn(my_w, __fadd_rn(sum, 1e-20f));
    }
    if (rank < a.top_k) {
        a.ids[(size_t)row * a.top_k + rank] = my_id;
        a.weights[(size_t)row * a.top_k + rank] = my_w * a.scale;
    }
}

template <class T, int VPL>
cudaError_t launch_vpl(const route_args &a, void *stream) {
    hy3a_launch l(dim3((a.rows + kWarps - 1) / kWarps), dim3(32 * kWarps), 0, stream);
    const bool quotient = a.softmax && !a.bias;
    if (a.groups > 1) return quotient ? cudaLaunchKernelEx(&l.cfg, hy3a_route_kernel<T, VPL, true, true>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_route_kernel<T, VPL, true, false>, a);
    return quotient ? cudaLaunchKernelEx(&l.cfg, hy3a_route_kernel<T, VPL, false, true>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_route_kernel<T, VPL, false, false>, a);
}
template <class T>
cudaError_t launch_type(const route_args &a, void *stream) {
    const int n = (a.experts + 31) / 32;
    if (n <= 1) return launch_vpl<T, 1>(a, stream);
    if (n <= 2) return launch_vpl<T, 2>(a, stream);
    if (n <= 4) return launch_vpl<T, 4>(a, stream);
    if (n <= 6) return launch_vpl<T, 6>(a, stream);
    if (n <= 8) return launch_vpl<T, 8>(a, stream);
    if (n <= 16) return launch_vpl<T, 16>(a, stream);
    return launch_vpl<T, 32>(a, stream);
}

} /* namespace */

extern "C" int hy3a_route(void *stream, int dtype, int rows, int experts, const void *logits, size_t stride, const float *bias, int top_k, int score,
                          int groups, int top_groups, int renormalize, float scale, int *ids, float *weights) {
    if (dtype != HY3A_F32 && dtype != HY3A_F16 && dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "route: dtype %d not in {0,1,2}", dtype);
    if (rows < 0) return hy3a_fail(NULL, HY3A_EINVAL, "route: rows %d < 0", rows);
    if (experts < 1 || experts > kMaxExperts) return hy3a_fail(NULL, HY3A_EINVAL, "route: experts %d not in [1,%d]", experts, kMaxExperts);
    if (top_k < 1 || top_k > kMaxTopK || top_k > experts) return hy3a_fail(NULL, HY3A_EINVAL, "route: top_k %d not in [1,%d]", top_k, experts < kMaxTopK ? experts : kMaxTopK);
    if (score != HY3A_SCORE_SIGMOID && score != HY3A_SCORE_SOFTMAX) return hy3a_fail(NULL, HY3A_EINVAL, "route: score %d not in {0,1}", score);
    if (groups < 1 || groups > kMaxGroups || experts % groups) return hy3a_fail(NULL, HY3A_EINVAL, "route: groups %d: a divisor of %d experts up to %d", groups, experts, kMaxGroups);
    if (top_groups < 1 || top_groups > groups) return hy3a_fail(NULL, HY3A_EINVAL, "route: top_groups %d not in [1,%d]", top_groups, groups);
    if (top_k > experts / groups * top_groups) return hy3a_fail(NULL, HY3A_EINVAL, "route: top_k %d, but %d groups of %d experts stay", top_k, top_groups, experts / groups);
    if (rows == 0) return HY3A_OK;
    if (!logits || !ids || !weights) return hy3a_fail(NULL, HY3A_EINVAL, "route: NULL argument");
    const size_t el = dtype == HY3A_F32 ? 4 : 2;
    if (((uintptr_t)logits & (el - 1)) || (((uintptr_t)bias | (uintptr_t)ids | (uintptr_t)weights) & 3)) return hy3a_fail(NULL, HY3A_EINVAL, "route: a pointer is not aligned to its type");
    int dev, sms, rc = hy3a_layer_device("route", &dev, &sms);
    if (rc) return rc;
    const int size = experts / groups;
    int shift = 5;
    while ((groups << shift) > 32) shift--;
    const route_args a = {logits, stride, bias, rows, experts, top_k, score == HY3A_SCORE_SOFTMAX, groups, top_groups, renormalize != 0,
                          experts / groups, shift, size >= 32 && size % (1 << shift) == 0, (unsigned)(((1ull << 32) + experts / groups - 1) / (experts / groups)), scale, ids, weights};
    const cudaError_t e = dtype == HY3A_F32 ? launch_type<float>(a, stream) : (dtype == HY3A_F16 ? launch_type<__half>(a, stream) : launch_type<__nv_bfloat16>(a, stream));
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "route: %s", cudaGetErrorString(e));
    return HY3A_OK;
}

extern "C" int hy3a_layer_sync(void *stream) {
    unsigned err[2][2] = {{0, 0}, {0, 0}};
    cudaError_t e = cudaStreamSynchronize((cudaStream_t)stream);
    if (e == cudaSuccess) e = hy3a_experts_error(err[0]);
    if (e == cudaSuccess) e = hy3a_adapters_error(err[1]);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "layer_sync: %s", cudaGetErrorString(e));
    for (int i = 0; i < 2; i++)
        if (err[i][0]) return hy3a_fail(NULL, HY3A_ETIMEOUT, "%s: a device-side bounded wait ran out (code %u, where %u): outputs since the last check are not valid", i ? "adapters" : "experts", err[i][0], err[i][1]);
    return HY3A_OK;
}

extern "C" int hy3a_layer_wait_out(void *stream, int which) {
    if (which != 0 && which != 1) return hy3a_fail(NULL, HY3A_EINVAL, "layer_wait_out: which %d not in {0,1}", which);
    int dev, sms, rc = hy3a_layer_device("layer_wait_out", &dev, &sms);
    if (rc) return rc;
    const cudaError_t e = which ? hy3a_adapters_wait_out(stream) : hy3a_experts_wait_out(stream);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "layer_wait_out: %s", cudaGetErrorString(e));
    return HY3A_OK;
}

/*
 * adapters.cu -- low-rank adapters of many requests beside a shared projection (hy3a_adapters):
 *
 *      out[t] = base[t] + scales[a] * B_a (A_a x[t]),   a = ids[t]
 *
 * Two launches:
 *   1. reduce   u[s][t] = A_a x[t] over the s-th cut of the width, fp32 (no cut is added to another here: the order of the sum is fixed);
 *   2. expand   sums the cuts, and adds B_a (scales[a] u[t]) to base.  u enters the product as two numbers of the rows' type, a rounded
 *               value and the rest, so that an fp32 result keeps about 17 (bf16) or 22 (fp16) bits of it; each row of u is brought to a
 *               largest value in [1, 2) first and back afterwards, which keeps fp16 in range.
 * Both walk tiles of rows, and for a tile the adapters that occur in it: neighbouring rows of one request cost one pass, a batch of
 * requests with an adapter each one pass per adapter, and no sorting is needed.
 */
#include <math.h>

#include <algorithm>

#include "layer.h"

namespace {

using namespace hy3a_layer;

constexpr int kMaxRank = 256;
constexpr int kReduceWarps = 4;       /* warps of a reduce block: one 16-rank block each */
constexpr int kExpandWarps = 4, kExpandCols = 64 /* columns of a warp */;

struct adapter_args {
    const void *x, *base, *a, *b;
    size_t x_stride, base_stride, out_stride;
    const int *ids;
    const float *scales;
    void *out;
    float *u;            /* [cuts][rows][rank] */
    int rows, width, out_width, adapters, rank, cuts, cut;   /* cut: k's of one, a multiple of 32 */
};

/* ---- 1. reduce: block = (8 rows, a cut, up to 4 blocks of 16 ranks) ---------------------------------------------------- */
template <class T>
__global__ void __launch_bounds__(32 * kReduceWarps) hy3a_adapters_reduce_kernel(const adapter_args a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int t0 = blockIdx.x * 8, cut = blockIdx.y, r0 = (blockIdx.z * kReduceWarps + warp) * 16;
    pdl_release();
    pdl_wait();
    if (r0 >= a.rank) return;
    const int row = t0 + g;
    int id = row < a.rows ? a.ids[row] : -1;
    if (id < 0 || id >= a.adapters) id = -1;
    const T *x = reinterpret_cast<const T *>(a.x) + (size_t)(row < a.rows ? row : 0) * a.x_stride;
    const int k_end = min(a.width, (cut + 1) * a.cut);
    float u[4] = {};                      /* of the adapter of each column's row */
    unsigned todo = __ballot_sync(0xffffffffu, id >= 0);
    while (todo) {
        const int ad = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
        const unsigned mine = __ballot_sync(0xffffffffu, id == ad);
        todo &= ~mine;
        const T *w = reinterpret_cast<const T *>(a.a) + ((size_t)ad * a.rank + r0 + g) * a.width;
        const bool has_lo = r0 + g < a.rank, has_hi = r0 + 8 + g < a.rank;
        float acc[4] = {};
        for (int kb = cut * a.cut; kb < k_end; kb += 32 * 4) {
            uint4 lo[4], hi[4], v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = kb + 32 * i + t * 8;
                lo[i] = has_lo && k < k_end ? load_row(w + k) : zero16();
                hi[i] = has_hi && k < k_end ? load_row(w + (size_t)8 * a.width + k) : zero16();
                v[i] = id == ad && k < k_end ? load_row(x + k) : zero16();
            }
#pragma unroll
            for (int i = 0; i < 4; i++) mma32<T>(acc, lo[i], hi[i], v[i]);
        }
        /* columns 2t and 2t + 1 belong to the rows of lanes 8t and 8t + 4 */
        const bool c0 = (mine >> (8 * t)) & 1, c1 = (mine >> (8 * t + 4)) & 1;
        if (c0) { u[0] = acc[0]; u[2] = acc[2]; }
        if (c1) { u[1] = acc[1]; u[3] = acc[3]; }
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int r = r0 + g + (c >> 1) * 8, tt = t0 + 2 * t + (c & 1);
        if (r < a.rank && tt < a.rows) a.u[((size_t)cut * a.rows + tt) * a.rank + r] = u[c];
    }
}

/* ---- 2. expand: block = (TOK rows, 256 columns), a warp 64 columns of them ------------------------------------------------
 * A's rows are columns of the output: row g of the j-th product is column 8g + 2j, row g + 8 the one behind it, so that a lane ends up
 * with 8 neighbouring columns of a row. */
template <class T, class O, int TOK>
__global__ void __launch_bounds__(32 * kExpandWarps) hy3a_adapters_expand_kernel(const adapter_args a) {
    extern __shared__ uint4 s_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int pitch = (a.rank + 31) / 32 * 32 + 8;               /* elements of a row of u: 16 bytes more than a multiple of 64 */
    T *s_hi = reinterpret_cast<T *>(s_raw), *s_lo = s_hi + TOK * pitch;
    __shared__ float s_back[TOK];
    __shared__ int s_id[TOK];
    const int t0 = blockIdx.x * TOK, n0 = (blockIdx.y * kExpandWarps + warp) * kExpandCols;
    pdl_release();
    pdl_wait();
    for (int i = warp; i < TOK; i += kExpandWarps) {             /* a warp per row: sums the cuts, scales, splits */
        const int row = t0 + i;
        int id = row < a.rows ? a.ids[row] : -1;
        if (id < 0 || id >= a.adapters) id = -1;
        float v[kMaxRank / 32], m = 0.f;
        const float scale = id >= 0 ? a.scales[id] : 0.f;
#pragma unroll
        for (int j = 0; j < kMaxRank / 32; j++) {
            const int r = lane + 32 * j;
            v[j] = 0.f;
            if (id >= 0 && r < a.rank) {
                for (int c = 0; c < a.cuts; c++) v[j] += a.u[((size_t)c * a.rows + row) * a.rank + r];
                v[j] *= scale;
                if (fabsf(v[j]) <= 3.402823466e38f) m = fmaxf(m, fabsf(v[j]));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        /* 2^-floor(log2 m) of the largest finite value; subnormal or no values stay as they are */
        const int ex = (int)(__float_as_uint(m) >> 23);
        const bool usual = ex > 0 && ex < 254;
        const float to = usual ? __uint_as_float((unsigned)(254 - ex) << 23) : 1.f;
        if (lane == 0) { s_id[i] = id; s_back[i] = usual ? __uint_as_float((unsigned)ex << 23) : 1.f; }
#pragma unroll
        for (int j = 0; j < kMaxRank / 32; j++) {
            const int r = lane + 32 * j;
            if (r < pitch - 8) {
                const float f = v[j] * to;
                const T hi = type<T>::down(f);
                s_hi[i * pitch + r] = hi;
                s_lo[i * pitch + r] = type<T>::down(isinf(type<T>::up(hi)) ? 0.f : f - type<T>::up(hi));
            }
        }
    }
    __syncthreads();
    if (n0 >= a.out_width) return;
    constexpr int NG = TOK / 8;
    float acc[NG][4][4] = {};
    /* lane i keeps the id of row i of the tile (TOK <= 32) */
    const int my = lane < TOK ? s_id[lane] : -1;
    const unsigned any = __ballot_sync(0xffffffffu, my >= 0);
    /* 32 ranks of an adapter's rows n0 + 8g .. n0 + 8g + 7, and 8 rows of u against them */
    auto load_b = [&](int ad, int r, uint4 (&f)[8]) {
        const T *w = reinterpret_cast<const T *>(a.b) + ((size_t)ad * a.out_width + n0 + g * 8) * a.rank + r;
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = r < a.rank && n0 + g * 8 + j < a.out_width ? load_row(w + (size_t)j * a.rank) : zero16();
    };
    auto multiply = [&](float (&d)[4][4], int i, int r, const uint4 (&f)[8]) {
        const uint4 hi = *reinterpret_cast<const uint4 *>(s_hi + (8 * i + g) * pitch + r), lo = *reinterpret_cast<const uint4 *>(s_lo + (8 * i + g) * pitch + r);
#pragma unroll
        for (int j = 0; j < 4; j++) { mma32<T>(d[j], f[2 * j], f[2 * j + 1], lo); mma32<T>(d[j], f[2 * j], f[2 * j + 1], hi); }
    };
    const int first = __shfl_sync(0xffffffffu, my, any ? __ffs(any) - 1 : 0);
    if (__ballot_sync(0xffffffffu, my == first) == any) {
        /* one adapter in the tile: its rows' u are the only ones that are not 0 */
        for (int r0 = 0; r0 < a.rank; r0 += 32) {
            uint4 f[8];
            load_b(first, r0 + t * 8, f);
#pragma unroll
            for (int i = 0; i < NG; i++) if ((any >> (8 * i)) & 0xff) multiply(acc[i], i, r0 + t * 8, f);
        }
    } else {
        /* several: each group of 8 rows takes the columns of its own (an adapter that is not finite must not reach the others' rows) */
#pragma unroll
        for (int i = 0; i < NG; i++) {
            unsigned todo = any & (0xffu << (8 * i));
            while (todo) {
                const int ad = __shfl_sync(0xffffffffu, my, __ffs(todo) - 1);
                const unsigned mine = __ballot_sync(0xffffffffu, my == ad);
                todo &= ~mine;
                float d[4][4] = {};
                for (int r0 = 0; r0 < a.rank; r0 += 32) {
                    uint4 f[8];
                    load_b(ad, r0 + t * 8, f);
                    multiply(d, i, r0 + t * 8, f);
                }
                const bool c0 = (mine >> (8 * i + 2 * t)) & 1, c1 = (mine >> (8 * i + 2 * t + 1)) & 1;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (c0) { acc[i][j][0] = d[j][0]; acc[i][j][2] = d[j][2]; }
                    if (c1) { acc[i][j][1] = d[j][1]; acc[i][j][3] = d[j][3]; }
                }
            }
        }
    }
    const int n = n0 + g * 8;
    if (n >= a.out_width) return;
#pragma unroll
    for (int i = 0; i < NG; i++) {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int tt = 8 * i + 2 * t + c, row = t0 + tt;
            if (row >= a.rows) continue;
            const O *base = reinterpret_cast<const O *>(a.base) + (size_t)row * a.base_stride + n;
            O *out = reinterpret_cast<O *>(a.out) + (size_t)row * a.out_stride + n;
            const float back = s_back[tt];
            const bool with = s_id[tt] >= 0;
            constexpr int PER = 16 / sizeof(O);
#pragma unroll
            for (int q = 0; q < 8 / PER; q++) {
                uint4 raw = *reinterpret_cast<const uint4 *>(base + q * PER);
                O *o = reinterpret_cast<O *>(&raw);
#pragma unroll
                for (int z = 0; z < PER; z++) {
                    const int col = q * PER + z;                       /* column col = row (col & 1) * 8 + g of product col >> 1 */
                    if (with) o[z] = type<O>::down(type<O>::up(o[z]) + back * acc[i][col >> 1][(col & 1) * 2 + c]);
                }
                *reinterpret_cast<uint4 *>(out + q * PER) = raw;
            }
        }
    }
}

/* Cuts of the width: enough blocks to fill the device where there are few rows, none shorter than 256. */
int cuts_of(int rows, int width, int rank, int sms) {
    const long long blocks = (long long)((rows + 7) / 8) * ((rank + 16 * kReduceWarps - 1) / (16 * kReduceWarps));
    long long c = (4ll * sms + blocks - 1) / blocks;
    c = std::min<long long>(c, (width + 255) / 256);
    return (int)std::max<long long>(1, std::min<long long>(c, 32));
}

template <class T, class O>
cudaError_t launch(const adapter_args &a, void *stream) {
    cudaError_t e;
    {   hy3a_launch l(dim3((a.rows + 7) / 8, a.cuts, (a.rank + 16 * kReduceWarps - 1) / (16 * kReduceWarps)), dim3(32 * kReduceWarps), 0, stream);
        if ((e = cudaLaunchKernelEx(&l.cfg, hy3a_adapters_reduce_kernel<T>, a)) != cudaSuccess) return e; }
    const int pitch = (a.rank + 31) / 32 * 32 + 8, cols = kExpandWarps * kExpandCols, ny = (a.out_width + cols - 1) / cols;
    if (a.rows <= 256) {
        hy3a_launch l(dim3((a.rows + 7) / 8, ny), dim3(32 * kExpandWarps), (size_t)2 * 8 * pitch * sizeof(T), stream);
        return cudaLaunchKernelEx(&l.cfg, hy3a_adapters_expand_kernel<T, O, 8>, a);
    }
    hy3a_launch l(dim3((a.rows + 31) / 32, ny), dim3(32 * kExpandWarps), (size_t)2 * 32 * pitch * sizeof(T), stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_adapters_expand_kernel<T, O, 32>, a);
}

int check_sizes(const char *who, int rows, int width, int rank) {
    if (rows < 0) return hy3a_fail(NULL, HY3A_EINVAL, "%s: rows %d < 0", who, rows);
    if (width < 8 || width % 8) return hy3a_fail(NULL, HY3A_EINVAL, "%s: width %d is no multiple of 8", who, width);
    if (rank < 8 || rank % 8 || rank > kMaxRank) return hy3a_fail(NULL, HY3A_EINVAL, "%s: rank %d is no multiple of 8 up to %d (fill smaller ones up with zeros)", who, rank, kMaxRank);
    return 0;
}
constexpr int kMostCuts = 32;

} /* namespace */

extern "C" {

size_t hy3a_adapters_workspace(int rows, int width, int rank) {
    if (check_sizes("adapters_workspace", rows, width, rank)) return 0;
    return (size_t)std::min(kMostCuts, (width + 255) / 256) * rows * rank * sizeof(float);
}

int hy3a_adapters(void *stream, int dtype, int rows, int width, int out_width, int adapters, int rank, const void *x, size_t x_stride, int base_dtype,
                  const void *base, size_t base_stride, const void *a_, const void *b_, const int *ids, const float *scales, void *out,
                  size_t out_stride, void *work, size_t work_bytes) {
    if (dtype != HY3A_F16 && dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: dtype %d not in {1,2}", dtype);
    if (base_dtype != dtype && base_dtype != HY3A_F32) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: base_dtype %d is neither the rows' (%d) nor fp32", base_dtype, dtype);
    int rc = check_sizes("adapters", rows, width, rank);
    if (rc) return rc;
    if (out_width < 8 || out_width % 8) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: out_width %d is no multiple of 8", out_width);
    if (adapters < 1) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: %d adapters", adapters);
    if (rows == 0) return HY3A_OK;
    if (!x || !base || !a_ || !b_ || !ids || !scales || !out || !work) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: NULL argument");
    if (((uintptr_t)x | (uintptr_t)base | (uintptr_t)a_ | (uintptr_t)b_ | (uintptr_t)out | (uintptr_t)work) & 15) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: pointers must be 16-byte aligned");
    if (((uintptr_t)ids | (uintptr_t)scales) & 3) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: ids and scales must be 4-byte aligned");
    if ((x_stride & 7) || ((base_stride | out_stride) & (base_dtype == HY3A_F32 ? 3 : 7))) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: rows must start on 16-byte boundaries");
    if (out_stride < (size_t)out_width && rows > 1) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: out rows of %d overlap at a stride of %zu", out_width, out_stride);
    int dev, sms;
    if ((rc = hy3a_layer_device("adapters", &dev, &sms))) return rc;
    const int cuts = cuts_of(rows, width, rank, sms);
    const size_t need = (size_t)cuts * rows * rank * sizeof(float);
    if (work_bytes < need) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: the workspace has %zu bytes, %zu are needed (hy3a_adapters_workspace)", work_bytes, need);
    const int cut = ((width + cuts - 1) / cuts + 31) / 32 * 32;
    const adapter_args a = {x, base, a_, b_, x_stride, base_stride, out_stride, ids, scales, out, (float *)work, rows, width, out_width, adapters, rank,
                            (width + cut - 1) / cut, cut};
    cudaError_t e;
    if (dtype == HY3A_F16) e = base_dtype == HY3A_F32 ? launch<__half, float>(a, stream) : launch<__half, __half>(a, stream);
    else e = base_dtype == HY3A_F32 ? launch<__nv_bfloat16, float>(a, stream) : launch<__nv_bfloat16, __nv_bfloat16>(a, stream);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "adapters: %s", cudaGetErrorString(e));
    return HY3A_OK;
}

} /* extern "C" */

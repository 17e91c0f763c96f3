/*
 * adapters.cu -- low-rank adapters of many requests beside a shared projection (hy3a_adapters):
 *
 *      out[t] = base[t] + scales[a] * B_a (A_a x[t]),   a = ids[t]
 *
 * Two launches:
 *   1. reduce   u[s][t] = A_a x[t] over the s-th 1024 of the width, fp32;
 *   2. expand   sums the cuts in their order, and adds B_a (scales[a] u[t]) to base.  u enters the product as two numbers of the rows'
 *               type, a rounded value and the rest, so that an fp32 result keeps about 17 (bf16) or 22 (fp16) bits of it; each row of u is
 *               brought to a largest value in [1, 2) first and back afterwards, which keeps fp16 in range.
 * Both walk tiles of rows and need no sorting.  Long inputs (prompts: neighbouring rows share an adapter) take tiles of 32 rows and go
 * through the adapters that occur in one; short ones (a row per request) tiles of 8, and each adapter of a tile is a block of its own, so
 * that no block waits for one adapter's weights after another's.
 */
#include <math.h>

#include <algorithm>
#include <atomic>

#include "layer.h"

namespace {

using namespace hy3a_layer;

constexpr int kMaxRank = 256;
constexpr int kCut = 1024;           /* k's of a reduce block: 128 of each of its 8 warps */
constexpr int kReduceWarps = 8, kExpandWarps = 4, kExpandCols = 64 /* columns of a warp at a time */;

struct adapter_args {
    const void *x, *base, *a, *b;
    size_t x_stride, base_stride, out_stride;
    const int *ids;
    const float *scales;
    void *out;
    float *u;            /* [cuts][rows][rank] */
    int rows, width, out_width, adapters, rank, cuts, span /* columns of an expand block */;
};

__device__ __forceinline__ int id_of(const adapter_args &a, int row) {
    const int id = row < a.rows ? a.ids[row] : -1;
    return id >= 0 && id < a.adapters ? id : -1;
}
/* the n-th adapter that occurs among the lanes' ids (uniform), -1 if there are fewer */
__device__ __forceinline__ int nth_adapter(int id, unsigned todo, int n) {
    for (;; n--) {
        if (!todo) return -1;
        const int ad = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
        if (n == 0) return ad;
        todo &= ~__ballot_sync(0xffffffffu, id == ad);
    }
}

/* ---- 1. reduce: block = (8 G rows, 16 RB ranks, a cut); SPLIT: and one of the tile's adapters -------------------------------- */
template <class T, int G, int RB, bool SPLIT>
__global__ void __launch_bounds__(32 * kReduceWarps) hy3a_adapters_reduce_kernel(const adapter_args a) {
    __shared__ float s_sum[kReduceWarps][RB][G][4][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rank_blocks = (a.rank + 16 * RB - 1) / (16 * RB), cut = blockIdx.y / rank_blocks, r0 = (blockIdx.y - cut * rank_blocks) * 16 * RB, t0 = blockIdx.x * 8 * G;
    pdl_release();
    pdl_wait();
    const int id = lane < 8 * G ? id_of(a, t0 + lane) : -1;
    unsigned todo = __ballot_sync(0xffffffffu, id >= 0);
    if (SPLIT) {
        const int ad = nth_adapter(id, todo, blockIdx.z);
        if (ad < 0) return;
        todo = __ballot_sync(0xffffffffu, id == ad);
    }
    const int k0 = cut * kCut + warp * (kCut / kReduceWarps) + t * 8;
    while (todo) {
        const int ad = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
        const unsigned mine = __ballot_sync(0xffffffffu, id == ad);
        todo &= ~mine;
        const T *w = reinterpret_cast<const T *>(a.a) + ((size_t)ad * a.rank + r0 + g) * a.width;
        float acc[RB][G][4] = {};
#pragma unroll
        for (int i = 0; i < kCut / kReduceWarps / 32; i++) {
            const int k = k0 + 32 * i;
            uint4 lo[RB], hi[RB];
#pragma unroll
            for (int b = 0; b < RB; b++) {
                lo[b] = r0 + 16 * b + g < a.rank && k < a.width ? load_row(w + (size_t)16 * b * a.width + k) : zero16();
                hi[b] = r0 + 16 * b + 8 + g < a.rank && k < a.width ? load_row(w + (size_t)(16 * b + 8) * a.width + k) : zero16();
            }
#pragma unroll
            for (int j = 0; j < G; j++) {
                const bool on = (mine >> (8 * j + g)) & 1;
                const uint4 x = on && k < a.width ? load_row(reinterpret_cast<const T *>(a.x) + (size_t)(t0 + 8 * j + g) * a.x_stride + k) : zero16();
#pragma unroll
                for (int b = 0; b < RB; b++) mma32<T>(acc[b][j], lo[b], hi[b], x);
            }
        }
#pragma unroll
        for (int b = 0; b < RB; b++)
#pragma unroll
            for (int j = 0; j < G; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) s_sum[warp][b][j][c][lane] = acc[b][j][c];
        __syncthreads();
        /* accumulator c of lane (g, t): rank g or g + 8 (c >= 2), row 2t + (c & 1) */
        for (int i = tid; i < 8 * G * 16 * RB; i += 32 * kReduceWarps) {
            const int tt = i / (16 * RB), r = i % (16 * RB);
            if (!((mine >> tt) & 1) || r0 + r >= a.rank) continue;
            const int c = ((r >> 3) & 1) * 2 + (tt & 1), from = (r & 7) * 4 + ((tt & 7) >> 1);
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < kReduceWarps; v++) sum += s_sum[v][r >> 4][tt >> 3][c][from];
            a.u[((size_t)cut * a.rows + t0 + tt) * a.rank + r0 + r] = sum;
        }
        if (!SPLIT) __syncthreads();
    }
}

/* Puts a tile's u into shared memory: the cuts' sum, the scale, the split into two numbers; neighbouring threads share a row, four ranks each
 * at a time.  `any`: the rows that have an adapter (the others get zeros). */
template <class T, int TOK, int THREADS>
__device__ __forceinline__ void put_u(const adapter_args &a, unsigned any, int t0, int pitch, T *s_hi, T *s_lo, float *s_back) {
    constexpr int PT = THREADS / TOK, NQ = kMaxRank / 4 / PT;
    const int i = threadIdx.x / PT, sub = threadIdx.x % PT;
    const bool on = (any >> i) & 1;
    const float scale = on ? a.scales[a.ids[t0 + i]] : 0.f;
    const float *u = a.u + (size_t)(t0 + i) * a.rank;
    float4 v[NQ];
    float m = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const int r = 4 * (sub + PT * q);
        v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on && r < a.rank) {
#pragma unroll 4
            for (int c = 0; c < a.cuts; c++) {
                const float4 w = *reinterpret_cast<const float4 *>(u + (size_t)c * a.rows * a.rank + r);
                v[q].x += w.x; v[q].y += w.y; v[q].z += w.z; v[q].w += w.w;
            }
            v[q].x *= scale; v[q].y *= scale; v[q].z *= scale; v[q].w *= scale;
        }
        const float big = 3.402823466e38f, x[4] = {fabsf(v[q].x), fabsf(v[q].y), fabsf(v[q].z), fabsf(v[q].w)};
#pragma unroll
        for (int z = 0; z < 4; z++) if (x[z] <= big) m = fmaxf(m, x[z]);
    }
#pragma unroll
    for (int o = 1; o < PT; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    /* 2^-floor(log2 m) of the largest finite value; subnormal or no values stay as they are */
    const int ex = (int)(__float_as_uint(m) >> 23);
    const bool usual = ex > 0 && ex < 254;
    const float to = usual ? __uint_as_float((unsigned)(254 - ex) << 23) : 1.f;
    if (sub == 0) s_back[i] = usual ? __uint_as_float((unsigned)ex << 23) : 1.f;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const int r = 4 * (sub + PT * q);
        if (r < pitch - 8) {
            const float f[4] = {v[q].x * to, v[q].y * to, v[q].z * to, v[q].w * to};
            T hi[4], lo[4];
#pragma unroll
            for (int z = 0; z < 4; z++) { hi[z] = type<T>::down(f[z]); lo[z] = type<T>::down(isinf(type<T>::up(hi[z])) ? 0.f : f[z] - type<T>::up(hi[z])); }
            *reinterpret_cast<uint2 *>(s_hi + i * pitch + r) = *reinterpret_cast<const uint2 *>(hi);
            *reinterpret_cast<uint2 *>(s_lo + i * pitch + r) = *reinterpret_cast<const uint2 *>(lo);
        }
    }
}

/* The columns of the output are the M side of the second product; which of a warp's 64 is which row of it is free, and chosen so that a
 * lane's values of an output row lie together: column `col` (0-7) of group g, which is row (col & 1) * 8 + g of product col >> 1.  An
 * instruction of the warp then moves 128 contiguous bytes of each of four rows: fp32 two runs of 4 columns a lane, 16-bit types one of 8. */
template <class O> __device__ __forceinline__ int column(int g, int col) { return sizeof(O) == 4 ? (col & 4) * 8 + g * 4 + (col & 3) : g * 8 + col; }

/* ---- 2. expand, short inputs: block = (8 rows, 256 columns, one of the tile's adapters) -----------------------------------
 * A warp's part of base is on its way before u is put together. */
template <class T, class O>
__global__ void __launch_bounds__(32 * kExpandWarps) hy3a_adapters_expand_kernel(const adapter_args a) {
    extern __shared__ uint4 s_raw[];
    constexpr int PER = 16 / sizeof(O), NB = 8 / PER;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int pitch = (a.rank + 31) / 32 * 32 + 8;               /* elements of a row of u: 16 bytes more than a multiple of 64 */
    T *s_hi = reinterpret_cast<T *>(s_raw), *s_lo = s_hi + 8 * pitch;
    __shared__ float s_back[8];
    const int t0 = blockIdx.x * 8, n0 = blockIdx.y * a.span + warp * kExpandCols, n_end = a.out_width;
    pdl_release();
    pdl_wait();
    /* lane i keeps the id of row i of the tile */
    const int my = lane < 8 ? id_of(a, t0 + lane) : -1;
    unsigned any = __ballot_sync(0xffffffffu, my >= 0);
    const unsigned none = __ballot_sync(0xffffffffu, lane < 8 && t0 + lane < a.rows && my < 0);
    const int ad = nth_adapter(my, any, blockIdx.z);
    if (ad < 0 && blockIdx.z > 0) return;
    any = __ballot_sync(0xffffffffu, my >= 0 && my == ad);
    const unsigned rows = any | (blockIdx.z == 0 ? none : 0u);       /* rows without an adapter go with the first */
    uint4 held[2][NB];
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int q = 0; q < NB; q++) {
            const int n = n0 + column<O>(g, q * PER);
            held[c][q] = ((rows >> (2 * t + c)) & 1) && n < n_end ? load_row(reinterpret_cast<const O *>(a.base) + (size_t)(t0 + 2 * t + c) * a.base_stride + n) : zero16();
        }
    put_u<T, 8, 32 * kExpandWarps>(a, any, t0, pitch, s_hi, s_lo, s_back);
    __syncthreads();
    float acc[4][4] = {};
    if (any) {
        const T *w = reinterpret_cast<const T *>(a.b) + ((size_t)ad * a.out_width + n0) * a.rank;
        for (int r = t * 8; r < (a.rank + 31) / 32 * 32; r += 32) {
            uint4 f[8];
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = r < a.rank && n0 + column<O>(g, j) < n_end ? load_row(w + (size_t)column<O>(g, j) * a.rank + r) : zero16();
            const uint4 hi = *reinterpret_cast<const uint4 *>(s_hi + g * pitch + r), lo = *reinterpret_cast<const uint4 *>(s_lo + g * pitch + r);
#pragma unroll
            for (int j = 0; j < 4; j++) { mma32<T>(acc[j], f[2 * j], f[2 * j + 1], lo); mma32<T>(acc[j], f[2 * j], f[2 * j + 1], hi); }
        }
    }
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const int tt = 2 * t + c;
        if (!((rows >> tt) & 1)) continue;
        O *out = reinterpret_cast<O *>(a.out) + (size_t)(t0 + tt) * a.out_stride;
        const float back = s_back[tt];
        const bool with = (any >> tt) & 1;
#pragma unroll
        for (int q = 0; q < NB; q++) {
            const int n = n0 + column<O>(g, q * PER);
            O *o = reinterpret_cast<O *>(&held[c][q]);
#pragma unroll
            for (int z = 0; z < PER; z++)
                if (with) o[z] = type<O>::down(type<O>::up(o[z]) + back * acc[(q * PER + z) >> 1][(z & 1) * 2 + c]);
            if (n < n_end) *reinterpret_cast<uint4 *>(out + n) = held[c][q];
        }
    }
}

/* ---- 2. expand, long inputs: block = (32 rows, `span` columns in tiles of 128) --------------------------------------------
 * Units (column tile, adapter of the row tile, 32 ranks) go through a ring of 4 stages filled by cp.async: 128 rows of B of 32 ranks, and with
 * the last unit of a column tile the tile of base.  A warp has 16 rows x 32 columns; a lane 4 neighbouring columns of each of its rows. */
constexpr int kLongRows = 32, kLongCols = 128, kLongStages = 4, kLongThreads = 256, kLongSpan = 512;
template <class O> struct long_stage {
    static constexpr int pitch = kLongCols * sizeof(O) + 16, b_bytes = kLongCols * 64, bytes = b_bytes + kLongRows * pitch;
};
__device__ __forceinline__ void copy_async(void *dst, const void *src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
/* 16-byte chunk c of row n of a stage's 32 ranks of B: pairs of rows share 128 bytes, and trade places so that rows 4 apart do not meet in a bank */
__device__ __forceinline__ int chunk_of(int n, int c) { return (n >> 1) * 128 + (((n ^ (n >> 2)) & 1) << 6) + c * 16; }
template <class T, class O>
__global__ void __launch_bounds__(kLongThreads, 2) hy3a_adapters_expand_long_kernel(const adapter_args a) {
    extern __shared__ uint4 s_raw[];
    using stage = long_stage<O>;
    uint8_t *ring = reinterpret_cast<uint8_t *>(s_raw);
    const int chunks = (a.rank + 31) >> 5, pitch = chunks * 32 + 8;      /* elements of a row of u: 16 bytes more than a multiple of 64 */
    T *s_hi = reinterpret_cast<T *>(ring + kLongStages * stage::bytes), *s_lo = s_hi + kLongRows * pitch;
    __shared__ float s_back[kLongRows];
    __shared__ int s_adapter[kLongRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int t0 = blockIdx.x * kLongRows, c_begin = blockIdx.y * a.span, c_end = min(a.out_width, c_begin + a.span);
    const int tok = (warp & 1) * 16, col = (warp >> 1) * 32;             /* the warp's part of a tile */
    pdl_release();
    pdl_wait();
    const int my = id_of(a, t0 + lane);
    const unsigned any = __ballot_sync(0xffffffffu, my >= 0);
    int n_ad = 0;                                                        /* adapters of the tile */
    for (unsigned todo = any; todo; n_ad++) {
        const int ad = __shfl_sync(0xffffffffu, my, __ffs(todo) - 1);
        todo &= ~__ballot_sync(0xffffffffu, my == ad);
        if (tid == 0) s_adapter[n_ad] = ad;
    }
    __syncthreads();
    const int tiles = (c_end - c_begin + kLongCols - 1) / kLongCols, per = max(1, n_ad * chunks);
    /* the thread's 16-byte pieces of a stage, as far as they do not depend on the unit */
    constexpr int PER = 16 / sizeof(O), QR = kLongCols / PER /* pieces of a row of base */, NBASE = kLongRows * QR / kLongThreads, STEP = kLongThreads / QR;
    const int bn = tid >> 2, br = (tid & 3) * 8, row0 = tid / QR, c_in = (tid % QR) * PER;
    const T *b_at = reinterpret_cast<const T *>(a.b) + (size_t)(c_begin + bn) * a.rank + br;
    const O *base_at = reinterpret_cast<const O *>(a.base) + (size_t)(t0 + row0) * a.base_stride + c_begin + c_in;
    const size_t ad_size = (size_t)a.out_width * a.rank;
    int f_c0 = c_begin, f_k = 0, f_r0 = 0;              /* the next unit to fetch: column, adapter of the tile, rank */
    const T *f_b = b_at + (n_ad ? s_adapter[0] : 0) * ad_size;
    auto fetch = [&](int slot) {
        uint8_t *st = ring + slot * stage::bytes;
        if (f_c0 < c_end) {
            if (n_ad) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const bool on = f_c0 + bn + 64 * i < c_end && f_r0 + br < a.rank;
                    copy_async(st + chunk_of(bn + 64 * i, tid & 3), on ? f_b + 64 * i * a.rank : reinterpret_cast<const T *>(a.b), on);
                }
                f_b += 32;
                f_r0 += 32;
            }
            if (f_r0 >= a.rank || !n_ad) {
                f_r0 = 0;
                if (++f_k >= n_ad) {
                    f_k = 0;
#pragma unroll
                    for (int i = 0; i < NBASE; i++) {
                        const bool on = t0 + row0 + STEP * i < a.rows && f_c0 + c_in < c_end;
                        copy_async(st + stage::b_bytes + (row0 + STEP * i) * stage::pitch + c_in * sizeof(O), on ? base_at + (size_t)(STEP * i) * a.base_stride : reinterpret_cast<const O *>(a.base), on);
                    }
                    f_c0 += kLongCols;
                    base_at += kLongCols;
                    b_at += (size_t)kLongCols * a.rank;
                }
                f_b = b_at + (n_ad ? s_adapter[f_k] : 0) * ad_size;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int u = 0; u < kLongStages - 1; u++) fetch(u);
    put_u<T, kLongRows, kLongThreads>(a, any, t0, pitch, s_hi, s_lo, s_back);
    const T *u_hi = s_hi + (tok + g) * pitch + t * 8, *u_lo = s_lo + (tok + g) * pitch + t * 8;
    O *out = reinterpret_cast<O *>(a.out) + (size_t)(t0 + tok + 2 * t) * a.out_stride + c_begin + col + 4 * g;
    int slot = 0;
    for (int tile = 0; tile < tiles; tile++) {
        float acc[2][2][4] = {};
        const uint8_t *st = ring;
        int k = 0, r = 0;
        for (int in = 0; in < per; in++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kLongStages - 2) : "memory");
            __syncthreads();                   /* the unit is there for all, and the one before it has been read by all */
            fetch((slot + kLongStages - 1) % kLongStages);
            st = ring + slot * stage::bytes;
            slot = (slot + 1) % kLongStages;
            if (!n_ad) break;
            const unsigned mine = n_ad == 1 ? any : __ballot_sync(0xffffffffu, my == s_adapter[k]);
            if ((mine >> tok) & 0xffff) {
                /* product m of the warp's two: its row g is column 4g + 2m, row g + 8 the one behind it */
                uint4 f[4];
#pragma unroll
                for (int j = 0; j < 4; j++) f[j] = *reinterpret_cast<const uint4 *>(st + chunk_of(col + 4 * g + j, t));
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint4 hi = *reinterpret_cast<const uint4 *>(u_hi + 8 * i * pitch + r), lo = *reinterpret_cast<const uint4 *>(u_lo + 8 * i * pitch + r);
                    if (n_ad == 1) {
#pragma unroll
                        for (int m = 0; m < 2; m++) { mma32<T>(acc[m][i], f[2 * m], f[2 * m + 1], lo); mma32<T>(acc[m][i], f[2 * m], f[2 * m + 1], hi); }
                    } else {
                        /* an adapter that is not finite must not reach the others' rows: only its own columns are taken */
                        const bool c0 = (mine >> (tok + 8 * i + 2 * t)) & 1, c1 = (mine >> (tok + 8 * i + 2 * t + 1)) & 1;
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            float d[4] = {acc[m][i][0], acc[m][i][1], acc[m][i][2], acc[m][i][3]};
                            mma32<T>(d, f[2 * m], f[2 * m + 1], lo);
                            mma32<T>(d, f[2 * m], f[2 * m + 1], hi);
                            if (c0) { acc[m][i][0] = d[0]; acc[m][i][2] = d[2]; }
                            if (c1) { acc[m][i][1] = d[1]; acc[m][i][3] = d[3]; }
                        }
                    }
                }
            }
            if ((r += 32) >= a.rank) { r = 0; k++; }
        }
        const bool in_columns = c_begin + tile * kLongCols + col + 4 * g < c_end;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int row = tok + 8 * i + 2 * t + c;
                struct alignas(4 * sizeof(O)) four { O v[4]; };
                four o = *reinterpret_cast<const four *>(st + stage::b_bytes + row * stage::pitch + (col + 4 * g) * sizeof(O));
                if ((any >> row) & 1) {
                    const float back = s_back[row];
#pragma unroll
                    for (int z = 0; z < 4; z++) o.v[z] = type<O>::down(type<O>::up(o.v[z]) + back * acc[z >> 1][i][(z & 1) * 2 + c]);
                }
                if (t0 + row < a.rows && in_columns) *reinterpret_cast<four *>(out + (size_t)(8 * i + c) * a.out_stride) = o;
            }
        out += kLongCols;
    }
}

constexpr int kShort = 256;           /* rows up to which a tile's adapters are blocks of their own */

template <class T, class O>
cudaError_t launch(adapter_args a, int device, int sms, void *stream) {
    cudaError_t e;
    const int pitch = (a.rank + 31) / 32 * 32 + 8, rank_blocks = (a.rank + 15) / 16;
    if (a.rows <= kShort) {
        const int tiles = (a.rows + 7) / 8, z = std::min({8, a.rows, a.adapters});
        {   hy3a_launch l(dim3(tiles, a.cuts * rank_blocks, z), dim3(32 * kReduceWarps), 0, stream);
            if ((e = cudaLaunchKernelEx(&l.cfg, hy3a_adapters_reduce_kernel<T, 1, 1, true>, a)) != cudaSuccess) return e; }
        a.span = kExpandWarps * kExpandCols;
        hy3a_launch l(dim3(tiles, (a.out_width + a.span - 1) / a.span, z), dim3(32 * kExpandWarps), (size_t)2 * 8 * pitch * sizeof(T), stream);
        return cudaLaunchKernelEx(&l.cfg, hy3a_adapters_expand_kernel<T, O>, a);
    }
    constexpr int kMostSmem = kLongStages * long_stage<O>::bytes + 2 * kLongRows * (kMaxRank + 8) * sizeof(T);
    static std::atomic<bool> ready[64];       /* shared memory allowed, per device */
    if (device >= 64 || !ready[device].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(hy3a_adapters_expand_long_kernel<T, O>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem)) != cudaSuccess) return e;
        if (device < 64) ready[device].store(true, std::memory_order_release);
    }
    const int tiles = (a.rows + kLongRows - 1) / kLongRows;
    {   hy3a_launch l(dim3(tiles, a.cuts * ((rank_blocks + 1) / 2)), dim3(32 * kReduceWarps), 0, stream);
        if ((e = cudaLaunchKernelEx(&l.cfg, hy3a_adapters_reduce_kernel<T, kLongRows / 8, 2, false>, a)) != cudaSuccess) return e; }
    a.span = kLongSpan;
    hy3a_launch l(dim3(tiles, (a.out_width + a.span - 1) / a.span), dim3(kLongThreads), kLongStages * long_stage<O>::bytes + (size_t)2 * kLongRows * pitch * sizeof(T), stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_adapters_expand_long_kernel<T, O>, a);
}

int check_sizes(const char *who, int rows, int width, int rank) {
    if (rows < 0) return hy3a_fail(NULL, HY3A_EINVAL, "%s: rows %d < 0", who, rows);
    if (width < 8 || width % 8) return hy3a_fail(NULL, HY3A_EINVAL, "%s: width %d is no multiple of 8", who, width);
    if (rank < 8 || rank % 8 || rank > kMaxRank) return hy3a_fail(NULL, HY3A_EINVAL, "%s: rank %d is no multiple of 8 up to %d (fill smaller ones up with zeros)", who, rank, kMaxRank);
    return 0;
}
int cuts_of(int width) { return (width + kCut - 1) / kCut; }

} /* namespace */

extern "C" {

size_t hy3a_adapters_workspace(int rows, int width, int rank) {
    if (check_sizes("adapters_workspace", rows, width, rank)) return 0;
    return (size_t)cuts_of(width) * rows * rank * sizeof(float);
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
    const size_t need = hy3a_adapters_workspace(rows, width, rank);
    if (work_bytes < need) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: the workspace has %zu bytes, %zu are needed (hy3a_adapters_workspace)", work_bytes, need);
    const adapter_args a = {x, base, a_, b_, x_stride, base_stride, out_stride, ids, scales, out, (float *)work, rows, width, out_width, adapters, rank, cuts_of(width), 0};
    cudaError_t e;
    if (dtype == HY3A_F16) e = base_dtype == HY3A_F32 ? launch<__half, float>(a, dev, sms, stream) : launch<__half, __half>(a, dev, sms, stream);
    else e = base_dtype == HY3A_F32 ? launch<__nv_bfloat16, float>(a, dev, sms, stream) : launch<__nv_bfloat16, __nv_bfloat16>(a, dev, sms, stream);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "adapters: %s", cudaGetErrorString(e));
    return HY3A_OK;
}

} /* extern "C" */

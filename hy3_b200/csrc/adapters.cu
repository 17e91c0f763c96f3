/*
 * adapters.cu -- low-rank adapters of many requests beside a shared projection (hy3a_adapters):
 *
 *      out[t] = base[t] + scales[a] * B_a (A_a x[t]),   a = ids[t]
 *
 * u = A_a x enters the second product as two numbers of the rows' type, the next smaller value and the rest, which leave 2^-16 (bf16) or 2^-22 (fp16) of a
 * row's largest; each row of u is brought to a largest value in [1, 2) first and back afterwards, which keeps fp16 in range.  bf16 rows on an fp32 base take a
 * third number (2^-24): two left an error of 1e-6 of the result.  The numbers have the sign of u, and none is 0 unless u is: an infinite weight meets each of
 * them, and gives the infinity that it gives with u (rounded to nearest they leave half as much, and NaN there).
 *
 * Rows are worked on in tiles of one adapter, so that its weights are read once for all of a tile, whatever the order of the rows:
 *   up to 8 rows        one launch: clusters of blocks for each adapter that occurs (short kernel);
 *   up to kShort rows   one launch: the rows are listed by adapter within it, in tiles of 8, and each tile is a cluster's or a few clusters';
 *   more                listed by a launch of their own (grouping.cuh) in tiles of 64; 1. reduce: u[s][t] = A_a x[t] over the s-th 2048 of the width, fp32; 2. expand.
 * Parts of u are added in their order wherever they meet.
 */
#include <math.h>

#include <algorithm>
#include <atomic>

#include "grouping.cuh"
#include "ring.cuh"

namespace {

using namespace hy3a_layer;
using namespace hy3a_ring;

constexpr int kMaxRank = 256, kMaxWidth = 1 << 20;
constexpr int kCut = 2048;           /* k's of a reduce block: 256 of each of its 8 warps (1024: 2048 rows on 8192 -> 4096 48.4 -> 55.7 us a pass, 512 of width 4096 25.0 -> 23.5) */
constexpr int kReduceWarps = 8, kExpandCols = 64 /* columns of a warp at a time */;
constexpr int kLongRows = 64, kLongCols = 128, kLongStages = 4;

/* `count` listed rows from `first` on, all of one adapter (-1: none) */
struct adapter_tile { int adapter, first, count, unused; };

struct adapter_args {
    const void *x, *base, *a, *b;
    size_t x_stride, base_stride, out_stride;
    const int *ids;
    const float *scales;
    void *out;
    float *u;            /* [cuts][rows][rank], in the order of the list */
    int *list;           /* [rows] rows, adapter by adapter (those without one behind the others) */
    adapter_tile *tiles; /* [*n_tiles] */
    int *n_tiles;
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

__device__ __forceinline__ float4 peer_value(unsigned addr, unsigned rank) {
    unsigned p;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(p) : "memory");
    return v;
}
/* the lanes (rows) of an adapter, none for -1 */
__device__ __forceinline__ unsigned rows_of(int id, int ad) { return __ballot_sync(0xffffffffu, id >= 0 && id == ad); }

/* ---- plan ---------------------------------------------------------------------------------------------------------------- */
constexpr int kPlanShared = 512;                          /* rows from which the blocks of a cluster share them: their warps take turns (2048 rows 11.5 us with one block) */
constexpr int kMaxListed = 2 * kGroupThreads - 1;       /* adapters whose rows can be listed */
template <int BLOCKS>
__global__ void __launch_bounds__(kGroupThreads) hy3a_adapters_plan_kernel(const adapter_args a) {
    pdl_release();
    const int tiles = group_items<BLOCKS, 2, true>(
        a.rows, a.adapters + 1, kLongRows, [&](int i) { const int id = a.ids[i]; return id >= 0 && id < a.adapters ? id : a.adapters; },
        [&](int ad, int p0, int n, int first, int count) { for (int j = 0; j < count; j++) a.tiles[first + j] = {ad < a.adapters ? ad : -1, p0 + j * kLongRows, min(kLongRows, n - j * kLongRows), 0}; },
        [&](int i, int p) { a.list[p] = i; });
    if (threadIdx.x == 0 && (BLOCKS == 1 || cluster_rank() == 0)) *a.n_tiles = tiles;
}

/* ---- long inputs, 1. reduce: block = (8 G rows of a tile, 16 RB ranks, a cut) ---------------------------------------------- */
template <class T, int G, int RB, bool WIDE>
__global__ void __launch_bounds__(32 * kReduceWarps, 2) hy3a_adapters_reduce_kernel(const adapter_args a) {
    __shared__ float s_sum[kReduceWarps][RB][G][4][32];
    constexpr int PARTS = kLongRows / (8 * G);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rank_blocks = (a.rank + 16 * RB - 1) / (16 * RB), cut = blockIdx.y / rank_blocks, r0 = (blockIdx.y - cut * rank_blocks) * 16 * RB, tile = blockIdx.x / PARTS;
    pdl_release();
    pdl_wait();
    const adapter_tile d = a.tiles[tile];        /* (the table has a line for each block that is launched; asked for together) */
    if (tile >= *a.n_tiles) return;
    const int p0 = d.first + ((int)blockIdx.x - tile * PARTS) * 8 * G, count = d.first + d.count - p0;
    if (d.adapter < 0 || count <= 0) return;
    const int k0 = cut * kCut + warp * (kCut / kReduceWarps) + t * 16;
    const T *w = reinterpret_cast<const T *>(a.a) + ((size_t)d.adapter * a.rank + r0 + g) * a.width, *x[G];
#pragma unroll
    for (int j = 0; j < G; j++) x[j] = reinterpret_cast<const T *>(a.x) + (size_t)a.list[p0 + min(8 * j + g, count - 1)] * a.x_stride;
    float acc[RB][G][4] = {};
#pragma unroll
    for (int i = 0; i < kCut / kReduceWarps / 64; i++) {
        const int k = k0 + 64 * i;
        k16 lo[RB], hi[RB];
#pragma unroll
        for (int b = 0; b < RB; b++) {
            lo[b] = load16<WIDE, false>(w + (size_t)16 * b * a.width + k, r0 + 16 * b + g < a.rank ? a.width - k : 0);
            hi[b] = load16<WIDE, false>(w + (size_t)(16 * b + 8) * a.width + k, r0 + 16 * b + 8 + g < a.rank ? a.width - k : 0);
        }
#pragma unroll
        for (int j = 0; j < G; j++) {
            const k16 v = load16<WIDE, false>(x[j] + k, a.width - k);
#pragma unroll
            for (int b = 0; b < RB; b++) mma64<T>(acc[b][j], lo[b], hi[b], v);
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
        if (tt >= count || r0 + r >= a.rank) continue;
        const int c = ((r >> 3) & 1) * 2 + (tt & 1), from = (r & 7) * 4 + ((tt & 7) >> 1);
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < kReduceWarps; v++) sum += s_sum[v][r >> 4][tt >> 3][c][from];
        a.u[((size_t)cut * a.rows + p0 + tt) * a.rank + r0 + r] = sum;
    }
}

/* the value of the rows' type next below |f| with f's sign, but not 0, and what it leaves of f (0, infinities and NaN: themselves; an infinity leaves 1) */
template <class T> __device__ __forceinline__ T below(float &f) {
    T t = type<T>::cut(f);
    if (type<T>::up(t) == f && f != 0.f && !isinf(f)) t = type<T>::step_down(t);
    if (type<T>::up(t) == 0.f && f != 0.f) { t = type<T>::least(f); f = 2.f * type<T>::up(t); }
    f = isinf(f) ? copysignf(1.f, f) : f - type<T>::up(t);
    return t;
}
/* the nearest one, but 0 of 0 alone */
template <class T> __device__ __forceinline__ T nearest(float f) {
    const T t = type<T>::down(f);
    return type<T>::up(t) == 0.f && f != 0.f ? type<T>::least(f) : t;
}
/* numbers of the rows' type that stand for one of u */
template <class T, class O> constexpr int kTermsOf = sizeof(O) == 4 && type<T>::code == HY3A_BF16 ? 3 : 2;

/* Puts a tile's u into shared memory: the sum of its parts (u(part, row, rank): four ranks), in their order, the scale, the split into TERMS numbers;
 * neighbouring threads share a row, four ranks each at a time.  `any`: the rows that have an adapter (the others get zeros); `ranks`: how many are
 * written, those past the last as zeros; place(term, row, rank): where four go. */
template <class T, int TOK, int THREADS, int TERMS, int NQ, class U, class P>
__device__ __forceinline__ void put_u_of(const adapter_args &a, const U &u, int parts, float scale, unsigned long long any, int ranks, const P &place, float *s_back) {
    constexpr int PT = THREADS / TOK;
    const int i = threadIdx.x / PT, sub = threadIdx.x % PT;
    const bool on = (any >> i) & 1;
    float4 v[NQ];
    float m = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; q++) v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int c = 0; c < parts; c++) {
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const int r = 4 * (sub + PT * q);
            const float4 w = on && r < a.rank ? u(c, i, r) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[q].x += w.x; v[q].y += w.y; v[q].z += w.z; v[q].w += w.w;
        }
    }
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        v[q].x *= scale; v[q].y *= scale; v[q].z *= scale; v[q].w *= scale;
        const float big = 3.402823466e38f, x[4] = {fabsf(v[q].x), fabsf(v[q].y), fabsf(v[q].z), fabsf(v[q].w)};
#pragma unroll
        for (int z = 0; z < 4; z++) if (x[z] <= big) m = fmaxf(m, x[z]);
    }
#pragma unroll
    for (int o = 1; o < PT; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    /* 2^-floor(log2 m) of the largest finite value, as far as fp32 has that and its inverse (no value: 1) */
    const unsigned ex = m > 0.f ? (unsigned)min(max((int)(254u - (__float_as_uint(m) >> 23)), 1), 253) : 127u;
    const float to = __uint_as_float(ex << 23);
    if (sub == 0) s_back[i] = __uint_as_float((254u - ex) << 23);
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const int r = 4 * (sub + PT * q);
        if (r < ranks) {
            float f[4] = {v[q].x * to, v[q].y * to, v[q].z * to, v[q].w * to};
#pragma unroll
            for (int k = 0; k < TERMS; k++) {
                T part[4];
#pragma unroll
                for (int z = 0; z < 4; z++) part[z] = k < TERMS - 1 ? below<T>(f[z]) : nearest<T>(f[z]);
                *reinterpret_cast<uint2 *>(place(k, i, r)) = *reinterpret_cast<const uint2 *>(part);
            }
        }
    }
}
template <class T, int TOK, int THREADS, int TERMS, class U, class P>
__device__ __forceinline__ void put_u(const adapter_args &a, const U &u, int parts, float scale, unsigned long long any, int ranks, const P &place, float *s_back) {
    constexpr int MOST = kMaxRank * TOK / 4 / THREADS;             /* four ranks at a time of a thread, at the largest rank */
    if (a.rank <= kMaxRank / 8) put_u_of<T, TOK, THREADS, TERMS, (MOST + 7) / 8>(a, u, parts, scale, any, ranks, place, s_back);
    else if (a.rank <= kMaxRank / 2) put_u_of<T, TOK, THREADS, TERMS, (MOST + 1) / 2>(a, u, parts, scale, any, ranks, place, s_back);
    else put_u_of<T, TOK, THREADS, TERMS, MOST>(a, u, parts, scale, any, ranks, place, s_back);
}

/* The columns of the output are the M side of the second product; which of a warp's 64 is which row of it is free, and chosen so that a
 * lane's values of an output row lie together: column `col` (0-7) of group g, which is row (col & 1) * 8 + g of product col >> 1.  An
 * instruction of the warp then moves 128 contiguous bytes of each of four rows: fp32 two runs of 4 columns a lane, 16-bit types one of 8. */
template <class O> __device__ __forceinline__ int column(int g, int col) { return sizeof(O) == 4 ? (col & 4) * 8 + g * 4 + (col & 3) : g * 8 + col; }

/* ---- short inputs: cluster of 8 blocks = (a tile of 8 rows of one adapter, 8 x `span` columns) ----------------------------------
 * LISTED: each block lists the rows by adapter itself, 256 at a time (blockIdx.x), and takes the tile of its number (a launch that lists them took
 * 5 us: 64 rows of a few prompts on 4096 -> 10240 11.9 with it, 10.4 without; 16 rows of as many requests on 8192 -> 4096 12.3, 10.3); otherwise (up to 8 rows) a
 * warp finds the adapter of its number among them.
 * Each block multiplies the rows by an eighth of A's width, the blocks meet in shared memory, and each adds its columns: one launch, u never
 * leaves the chip, and A is read once for 8 x span columns.  B is asked of L2 and base of memory before the first product begins. */
constexpr int kShortBlocks = 8, kShortWarps = 8, kShortListed = 32 * kShortWarps;
/* clusters for which a listed input's columns are divided: about as many as fit at once (two blocks an SM).  us a pass with 32 / 64 / 96: 64 rows of a few
 * prompts on 4096 -> 10240 10.4 / 14.2 / 14.1, of as many requests 12.3 / 15.1 / 20.2, on 8192 -> 4096 17.7 / 22.5 / 25.1. */
constexpr int kShortClusters = 32;
template <class T, class O, bool WIDE, bool LISTED>
__global__ void __launch_bounds__(32 * kShortWarps, 2) hy3a_adapters_short_kernel(const adapter_args a) {
    constexpr int PER = 16 / sizeof(O), NB = 8 / PER, RB = 4;            /* blocks of 16 ranks at a time */
    constexpr int TERMS = kTermsOf<T, O>;
    __shared__ float s_sum[kShortWarps][RB][4][32];
    __shared__ alignas(16) float s_part[8 * kMaxRank];                   /* [row][rank] of the block's share of the width */
    __shared__ alignas(16) uint8_t s_u_raw[TERMS * 8 * (kMaxRank + 8) * sizeof(T)];
    __shared__ float s_back[8];
    const int pitch = (a.rank + 31) / 32 * 32 + 8;                       /* elements of a row of u: 16 bytes more than a multiple of 64 */
    T *s_u = reinterpret_cast<T *>(s_u_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int share = blockIdx.y % kShortBlocks;
    pdl_release();
    pdl_wait();
    /* lane i (and i + 8, ...) keeps row i of the tile */
    int row, ad, group = blockIdx.y / kShortBlocks, span = a.span;
    unsigned rows, any;                                                  /* the block's rows, and those with an adapter */
    if (LISTED) {
        __shared__ alignas(16) int s_id[kShortListed];
        __shared__ int s_heads[kShortWarps], s_row[8], s_tile[2] /* adapter, place of its first row among the adapter's */, s_rows;
        const int first = blockIdx.x * kShortListed, my = id_of(a, first + tid), listed = min(kShortListed, a.rows - first);
        s_id[tid] = my;
        if (tid == 0) s_rows = 0;
        __syncthreads();
        /* the row's place among its adapter's; every eighth of them begins a tile, and the block takes the one of its number */
        int place = 0;
#pragma unroll 8
        for (int i = 0, n = tid < listed ? tid : 0; i < n; i += 4) {
            const int4 id = *reinterpret_cast<const int4 *>(s_id + i);
            place += (id.x == my) + (i + 1 < tid && id.y == my) + (i + 2 < tid && id.z == my) + (i + 3 < tid && id.w == my);
        }
        const bool head = tid < listed && (place & 7) == 0;
        const unsigned heads = __ballot_sync(0xffffffffu, head);
        if (lane == 0) s_heads[warp] = __popc(heads);
        __syncthreads();
        int before = 0, tiles = 0;
        for (int w = 0; w < kShortWarps; w++) { tiles += s_heads[w]; if (w < warp) before += s_heads[w]; }
        const int groups = max(1, min(kShortClusters / tiles, (a.out_width + kShortBlocks * span - 1) / (kShortBlocks * span))), tile = blockIdx.z % tiles;
        group = blockIdx.z / tiles;
        if (group >= groups) return;                                     /* (so do the cluster's others) */
        const int each = (a.out_width + kShortBlocks * groups - 1) / (kShortBlocks * groups), pass = each <= kShortWarps * kExpandCols ? kExpandCols : kShortWarps * kExpandCols;
        span = (each + pass - 1) / pass * pass;
        if (head && before + __popc(heads & ((1u << lane) - 1u)) == tile) { s_tile[0] = my; s_tile[1] = place; }
        __syncthreads();
        ad = s_tile[0];
        const int at = place - s_tile[1];
        const bool mine = tid < listed && my == ad && at >= 0 && at < 8;
        if (mine) { s_row[at] = first + tid; atomicAdd(&s_rows, 1); }
        __syncthreads();
        const int count = s_rows;
        row = s_row[min(lane & 7, count - 1)];
        rows = (1u << count) - 1u;
        any = ad < 0 ? 0u : rows;
    } else {
        row = min(lane & 7, a.rows - 1);
        const int my = lane < 8 ? id_of(a, lane) : -1;
        const unsigned with = __ballot_sync(0xffffffffu, my >= 0), none = __ballot_sync(0xffffffffu, lane < 8 && lane < a.rows && my < 0);
        ad = nth_adapter(my, with, blockIdx.z);
        if (ad < 0 && blockIdx.z > 0) return;
        any = rows_of(my, ad);
        rows = any | (blockIdx.z == 0 ? none : 0u);                      /* rows without an adapter go with the first */
    }
    const int c_begin = (group * kShortBlocks + share) * span, n_end = min(a.out_width, c_begin + span);
    const int row_g = __shfl_sync(0xffffffffu, row, g), row_t[2] = {__shfl_sync(0xffffffffu, row, 2 * t), __shfl_sync(0xffffffffu, row, 2 * t + 1)};
    const T *const b = reinterpret_cast<const T *>(a.b) + (size_t)(ad < 0 ? 0 : ad) * a.out_width * a.rank;
    if (any && c_begin < n_end)
        for (size_t i = (size_t)tid * 64, n = (size_t)(n_end - c_begin) * a.rank; i < n; i += 32 * kShortWarps * 64)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(b + (size_t)c_begin * a.rank + i));
    uint4 held[2][NB];
    auto fetch_base = [&](int n0) {
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int q = 0; q < NB; q++) {
                const int n = n0 + column<O>(g, q * PER);
                held[c][q] = ((rows >> (2 * t + c)) & 1) && n < n_end ? load_row(reinterpret_cast<const O *>(a.base) + (size_t)row_t[c] * a.base_stride + n) : zero16();
            }
    };
    int n0 = c_begin + warp * kExpandCols;
    fetch_base(n0);
    if (any) {
        const int slice = ((a.width + kShortBlocks - 1) / kShortBlocks + 63) / 64 * 64, k_begin = share * slice, k_end = min(a.width, k_begin + slice);
        const T *x = reinterpret_cast<const T *>(a.x) + (size_t)row_g * a.x_stride;
        const bool on = (any >> g) & 1;
        for (int r0 = 0; r0 < a.rank; r0 += 16 * RB) {
            const T *w = reinterpret_cast<const T *>(a.a) + ((size_t)ad * a.rank + r0 + g) * a.width;
            float acc[RB][4] = {};
            for (int kb = k_begin + warp * 64; kb < k_end; kb += 64 * kShortWarps) {
                const int k = kb + t * 16, left = k_end - k;
                k16 lo[RB], hi[RB];
#pragma unroll
                for (int i = 0; i < RB; i++) {
                    lo[i] = load16<WIDE, false>(w + (size_t)16 * i * a.width + k, r0 + 16 * i + g < a.rank ? left : 0);
                    hi[i] = load16<WIDE, false>(w + (size_t)(16 * i + 8) * a.width + k, r0 + 16 * i + 8 + g < a.rank ? left : 0);
                }
                const k16 v = load16<WIDE, false>(x + k, on ? left : 0);
#pragma unroll
                for (int i = 0; i < RB; i++) mma64<T>(acc[i], lo[i], hi[i], v);
            }
            if (r0) __syncthreads();
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) s_sum[warp][i][c][lane] = acc[i][c];
            __syncthreads();
            /* accumulator c of lane (g, t): rank g or g + 8 (c >= 2), row 2t + (c & 1) */
            for (int i = tid; i < 8 * 16 * RB; i += 32 * kShortWarps) {
                const int tt = i / (16 * RB), r = i % (16 * RB), c = ((r >> 3) & 1) * 2 + (tt & 1), from = (r & 7) * 4 + (tt >> 1);
                float sum = 0.f;
#pragma unroll
                for (int v = 0; v < kShortWarps; v++) sum += s_sum[v][r >> 4][c][from];
                if (r0 + r < a.rank) s_part[tt * a.rank + r0 + r] = sum;
            }
        }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const unsigned part = (unsigned)__cvta_generic_to_shared(s_part);
    put_u<T, 8, 32 * kShortWarps, TERMS>(a, [&](int c, int i, int r) { return peer_value(part + (unsigned)(i * a.rank + r) * 4u, (unsigned)c); }, kShortBlocks, ad < 0 ? 0.f : a.scales[ad], any, pitch - 8,
                                               [&](int k, int i, int r) { return s_u + (k * 8 + i) * pitch + r; }, s_back);
    __syncwarp();
    cluster_arrive();                        /* the others' shares have been read */
    __syncthreads();
    for (; n0 < n_end; n0 += kShortWarps * kExpandCols) {
        float acc[4][4] = {};
        if (any) {
            const T *w = b + (size_t)n0 * a.rank;
            for (int r = t * 8; r < (a.rank + 31) / 32 * 32; r += 32) {
                uint4 f[8];
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] = r < a.rank && n0 + column<O>(g, j) < n_end ? load_row(w + (size_t)column<O>(g, j) * a.rank + r) : zero16();
#pragma unroll
                for (int k = TERMS - 1; k >= 0; k--) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(s_u + (k * 8 + g) * pitch + r);
#pragma unroll
                    for (int j = 0; j < 4; j++) mma32<T>(acc[j], f[2 * j], f[2 * j + 1], v);
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int tt = 2 * t + c;
            if (!((rows >> tt) & 1)) continue;
            O *out = reinterpret_cast<O *>(a.out) + (size_t)row_t[c] * a.out_stride;
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
        if (n0 + kShortWarps * kExpandCols < n_end) fetch_base(n0 + kShortWarps * kExpandCols);
    }
    __syncwarp();
    cluster_wait();
}

/* ---- 2. expand, long inputs: block = (a tile of up to 64 rows, some tiles of 128 columns, 256 in 16-bit types), two an SM -------------------
 * Base and output are what this kernel has to move (168 MB for 2048 rows of 10240 in fp32, of 50 us a pass in all; a copy of as many bytes by rows of 128
 * in this form runs at 5.6 TB/s).  Columns are the M side of tcgen05.mma, rows the N side: an accumulator's lane is a column of the output, so that a
 * warp adds base and stores straight from tensor memory, 128 bytes of a row at a time, whatever rows the list names.  In 16-bit types a lane has
 * two neighbouring columns, one in each of two accumulators: B's columns come in by their parity.  Warps 0-7 prepare u and then move the quarter w % 4 of
 * the columns of rows 32 (w / 4) ..; warp 8 fetches B (128 columns x 64 ranks a stage, 128-byte swizzle), warp 9 multiplies, into two sets of accumulators in turn.
 * Measured beside it, 2048 rows on 4096 -> 10240 with 32 / 128 ranks: warp-level products over a ring of tensor copies 63 / 159, this 50 / 78; base and
 * output through shared memory by a bulk copy of each row, one block an SM, 67 / 92. */
constexpr int kLongWarps = 8, kLongThreads = 32 * (kLongWarps + 2), kStageBytes = kLongCols * 128;
enum { A_FULL = 0, A_EMPTY = kLongStages, A_TFULL = 2 * kLongStages, A_TEMPTY = A_TFULL + 2, A_COUNT = A_TEMPTY + 2 };
__device__ unsigned g_err[2];         /* {code, where} of the first wait that ran out, until hy3a_layer_sync reads it */

__device__ __forceinline__ void tma_load(unsigned dst, const CUtensorMap *map, unsigned bar, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
/* K-major operand, 128-byte swizzle: 8-row groups 1024 B apart, descriptor version 1, layout 2 */
__device__ __forceinline__ unsigned long long make_desc(unsigned saddr) {
    return (unsigned long long)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | ((unsigned long long)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void umma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(unsigned bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void tmem_ld8(unsigned taddr, unsigned (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
template <class T, class O>
__global__ void __launch_bounds__(kLongThreads, 2) hy3a_adapters_expand_long_kernel(const __grid_constant__ CUtensorMap tm_b, const adapter_args a, int stages, int blocks) {
    extern __shared__ uint8_t s_bytes[];
    constexpr int TERMS = kTermsOf<T, O>, PER = 4 / sizeof(O) /* columns of a lane */, COLS = kLongCols * PER, ACC = kLongRows * PER /* columns of tensor memory of a unit */;
    uint8_t *ring = s_bytes + ((1024u - (smem_u32(s_bytes) & 1023u)) & 1023u), *s_u = ring + stages * kStageBytes;      /* u: [term][64 ranks][row] */
    __shared__ float s_back[kLongRows];
    __shared__ size_t s_base[kLongRows], s_out[kLongRows];               /* where the rows begin, in words of 4 bytes */
    __shared__ alignas(8) unsigned long long s_bar[A_COUNT];
    __shared__ unsigned s_tmem;
    __shared__ int s_abort_flag;
    volatile int *s_abort = &s_abort_flag;
    const unsigned bar0 = smem_u32(s_bar);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, panels = (a.rank + 63) >> 6, across = (a.out_width + COLS - 1) / COLS;
    if (tid == 0) {
        s_abort_flag = 0;
        for (int i = 0; i < stages; i++) { mbar_init(bar0 + 8 * (A_FULL + i), 1); mbar_init(bar0 + 8 * (A_EMPTY + i), 1); }
        for (int i = 0; i < 2; i++) { mbar_init(bar0 + 8 * (A_TFULL + i), 1); mbar_init(bar0 + 8 * (A_TEMPTY + i), kLongWarps); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kLongWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(2u * ACC) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = s_tmem;
    pdl_release();                           /* not before the tensor memory is there: the next kernel could take it and wait for this one */
    pdl_wait();
    /* the column tiles of a row tile are divided among as many blocks as fit at once */
    const int tiles = *a.n_tiles, groups = max(1, min(blocks / tiles, across)), span = (across + groups - 1) / groups, c_first = ((int)blockIdx.x / tiles) * span;
    const int columns = (int)blockIdx.x / tiles < groups ? min(span, across - c_first) : 0;
    const adapter_tile d = a.tiles[(int)blockIdx.x % tiles];
    const int ad = d.adapter;
    if (tid < kLongRows) {
        const int row = a.list[d.first + min(tid, d.count - 1)];
        s_base[tid] = (size_t)row * (a.base_stride / PER);
        s_out[tid] = (size_t)row * (a.out_stride / PER);
    }
    __syncthreads();
    if (columns > 0 && (ad >= 0 || warp < kLongWarps)) {
        if (warp == kLongWarps) {
            if (lane == 0) {
                int st = 0;
                unsigned ph = 0;
                bool ok = true;
                for (int c = 0; c < columns && ok; c++)
                    for (int p = 0; p < panels * PER; p++) {
                        if (!(ok = mbar_wait(bar0 + 8 * (A_EMPTY + st), ph ^ 1u, s_abort, g_err, 30u))) break;
                        mbar_expect_tx(bar0 + 8 * (A_FULL + st), kStageBytes);
                        tma_load(smem_u32(ring) + st * kStageBytes, &tm_b, bar0 + 8 * (A_FULL + st), p / PER * 64, p % PER, (c_first + c) * kLongCols, ad);
                        if (++st == stages) { st = 0; ph ^= 1u; }
                    }
                for (int i = 0; i < stages && ok; i++) {                 /* the last commits have reached their barriers before the block ends */
                    ok = mbar_wait(bar0 + 8 * (A_EMPTY + st), ph ^ 1u, s_abort, g_err, 34u);
                    if (++st == stages) { st = 0; ph ^= 1u; }
                }
            }
        } else if (warp == kLongWarps + 1) {
            asm volatile("bar.sync 1, %0;" ::"n"(32 * (kLongWarps + 1)) : "memory");
            if (lane == 0) {
                constexpr unsigned kType = type<T>::code == HY3A_BF16 ? (1u << 7) | (1u << 10) : 0u;
                const unsigned idesc = (1u << 4) | kType | (((unsigned)(d.count + 15) >> 4) << 18) | ((kLongCols >> 4) << 24);
                int st = 0;
                unsigned ph = 0;
                bool ok = true;
                for (int c = 0; c < columns && ok; c++) {
                    const int buf = c & 1;
                    if (!(ok = mbar_wait(bar0 + 8 * (A_TEMPTY + buf), ((c >> 1) & 1) ^ 1, s_abort, g_err, 32u))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    for (int p = 0; p < panels * PER; p++) {
                        if (!(ok = mbar_wait(bar0 + 8 * (A_FULL + st), ph, s_abort, g_err, 31u))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const int panel = p / PER, steps = min(4, (a.rank - panel * 64 + 15) >> 4);
                        const unsigned long long da = make_desc(smem_u32(ring) + st * kStageBytes);
                        for (int k = TERMS - 1; k >= 0; k--) {
                            const unsigned long long db = make_desc(smem_u32(s_u) + (k * panels + panel) * kLongRows * 128);
                            for (int i = 0; i < steps; i++) umma(tmem + buf * ACC + p % PER * kLongRows, da + 2 * i, db + 2 * i, idesc, panel > 0 || k < TERMS - 1 || i > 0);
                        }
                        umma_commit(bar0 + 8 * (A_EMPTY + st));
                        if (++st == stages) { st = 0; ph ^= 1u; }
                    }
                    if (ok) umma_commit(bar0 + 8 * (A_TFULL + buf));
                }
            }
        } else {
            const int r0 = (warp >> 2) * 32, count = d.count - r0;
            if (ad >= 0) {
                put_u<T, kLongRows, 32 * kLongWarps, TERMS>(a, [&](int c, int i, int r) { return *reinterpret_cast<const float4 *>(a.u + ((size_t)c * a.rows + d.first + i) * a.rank + r); },
                                                            a.cuts, a.scales[ad], ~0ull >> (kLongRows - d.count), (a.rank + 15) & ~15,
                                                            [&](int k, int i, int r) { return s_u + (k * panels + (r >> 6)) * kLongRows * 128 + i * 128 + ((((r >> 3) & 7) ^ (i & 7)) << 4) + (r & 7) * 2; }, s_back);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("bar.sync 1, %0;" ::"n"(32 * (kLongWarps + 1)) : "memory");
            }
            for (int c = 0; c < columns; c++) {
                const int n = (c_first + c) * COLS + (warp & 3) * 32 * PER + lane * PER, buf = c & 1;
                const bool in = n < a.out_width, whole = count >= 32 && n + (32 - lane) * PER <= a.out_width;
                const unsigned *const base = reinterpret_cast<const unsigned *>(reinterpret_cast<const O *>(a.base) + n);
                unsigned *const out = reinterpret_cast<unsigned *>(reinterpret_cast<O *>(a.out) + n);
                unsigned held[32];
                if (whole) {
#pragma unroll
                    for (int j = 0; j < 32; j++) held[j] = base[s_base[r0 + j]];
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++) if (in && j < count) held[j] = base[s_base[r0 + j]];
                }
                if (ad < 0) {
#pragma unroll
                    for (int j = 0; j < 32; j++) if (in && j < count) out[s_out[r0 + j]] = held[j];
                    continue;
                }
                if (!mbar_wait(bar0 + 8 * (A_TFULL + buf), (c >> 1) & 1, s_abort, g_err, 33u)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                constexpr int STEP = 16 / PER;
#pragma unroll
                for (int h = 0; h < 32; h += STEP) {
                    if (h >= count) continue;
                    unsigned v[2][8];                /* rows and the 8 behind them, or a row's two columns */
                    const unsigned at = tmem + ((unsigned)((warp & 3) * 32) << 16) + buf * ACC + r0 + h;
                    tmem_ld8(at, v[0]);
                    tmem_ld8(at + (PER == 2 ? kLongRows : 8), v[1]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    auto sum = [&](int j) {
                        const float by = s_back[r0 + h + j];
                        unsigned o = held[h + j];
                        O *const e = reinterpret_cast<O *>(&o);
#pragma unroll
                        for (int z = 0; z < PER; z++) e[z] = type<O>::down(type<O>::up(e[z]) + by * __uint_as_float(PER == 2 ? v[z][j & 7] : v[j >> 3][j & 7]));
                        out[s_out[r0 + h + j]] = o;
                    };
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < STEP; j++) sum(j);
                    } else {
#pragma unroll
                        for (int j = 0; j < STEP; j++) if (in && h + j < count) sum(j);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar0 + 8 * (A_TEMPTY + buf));
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*s_abort) for (int i = 0; i < 10000; i++) __nanosleep(1000);      /* copies of the unit that was given up are still on their way */
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == kLongWarps + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * ACC) : "memory");
}

/* Rows up to which the short kernel is taken (us a pass, short / long): 128, 160, 200 and 256 rows of as many requests on 8192 -> 4096 27.5 / 28.4, 28.9 / 29.1,
 * 30.5 / 29.7, 32.3 / 30.5; of 7 prompts on 4096 -> 10240 14.5 / 16.0, 15.1 / 16.2, 15.6 / 16.4, 22.6 / 17.9; of 40 adapters on 600 -> 5000 11.5 / 15.4, 14.2 / 16.7,
 * 18.4 / 17.6, 22.0 / 18.5. */
constexpr int kShort = 192;

template <class T, class O, bool LISTED>
cudaError_t launch_short(adapter_args a, bool wide, void *stream) {
    a.span = LISTED ? 512 : 256;           /* at least, where the kernel chooses */
    const int groups = (a.out_width + kShortBlocks * a.span - 1) / (kShortBlocks * a.span), chunk = std::min(a.rows, kShortListed);
    hy3a_launch l(LISTED ? dim3((a.rows + kShortListed - 1) / kShortListed, kShortBlocks, std::max(kShortClusters, chunk / 8 + std::min(chunk, a.adapters + 1)))
                         : dim3(1, kShortBlocks * groups, std::min(a.rows, a.adapters)), dim3(32 * kShortWarps), 0, stream);
    l.cluster(1, kShortBlocks);
    return wide ? cudaLaunchKernelEx(&l.cfg, hy3a_adapters_short_kernel<T, O, true, LISTED>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_adapters_short_kernel<T, O, false, LISTED>, a);
}
/* B as [adapter][column / per][column % per][rank]; boxes of 128 columns that are `per` apart, of 64 ranks */
bool encode_columns(CUtensorMap *m, const adapter_args &a, int per) {
    const encode_tiled_fn enc = encoder();
    const cuuint64_t line = (cuuint64_t)a.rank * 2, dims[4] = {(cuuint64_t)a.rank, (cuuint64_t)per, (cuuint64_t)(a.out_width / per), (cuuint64_t)a.adapters}, strides[3] = {line, line * per, line * a.out_width};
    const cuuint32_t box[4] = {64, 1, kLongCols, 1}, one[4] = {1, 1, 1, 1};
    return enc && enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(a.b), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <class T, class O>
cudaError_t launch(const adapter_args &a, int device, int sms, void *stream, const char **what) {
    cudaError_t e;
    const bool wide = wide_rows({a.x, a.a}, {a.x_stride, (size_t)a.width});
    if (a.rows <= 8) return launch_short<T, O, false>(a, wide, stream);
    /* (the plan's array holds no more adapters: beyond, tiles of 8 rows read A and B for each.  us a pass with 2047 / 2048 adapters of rank 64 on 8192 -> 4096: 2048 rows
     * of 7 prompts 121 / 326, of as many requests 416 / 784, 300 rows of as many requests 93 / 121) */
    if (a.rows <= kShort || a.adapters > kMaxListed) return launch_short<T, O, true>(a, wide, stream);
    const bool shared = a.rows >= kPlanShared;
    {   hy3a_launch l(dim3(shared ? kGroupCluster : 1), dim3(kGroupThreads), 0, stream);
        if (shared) l.cluster(kGroupCluster);
        if ((e = shared ? cudaLaunchKernelEx(&l.cfg, hy3a_adapters_plan_kernel<kGroupCluster>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_adapters_plan_kernel<1>, a)) != cudaSuccess) return e; }
    constexpr int kTerms = kTermsOf<T, O>, kMostSmem = 1024 + kLongStages * kStageBytes + kTerms * (kMaxRank / 64) * kLongRows * 128, kHalf = 113000 /* of an SM, static shared memory left out */;
    static std::atomic<bool> ready[64];       /* shared memory allowed, per device */
    if (device >= 64 || !ready[device].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(hy3a_adapters_expand_long_kernel<T, O>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem)) != cudaSuccess) return e;
        if (device < 64) ready[device].store(true, std::memory_order_release);
    }
    CUtensorMap tm_b;
    if (!encode_columns(&tm_b, a, 4 / sizeof(O))) {
        *what = "no tensor map (cuTensorMapEncodeTiled)";
        return cudaErrorInvalidValue;
    }
    /* most tiles that there can be: every adapter's last one, and a tile has a row at least (the table has a line more than rows) */
    const int tiles = std::min(a.rows, a.rows / kLongRows + std::min(a.rows, a.adapters + 1)), rank_blocks = (a.rank + 31) / 32;
    {   hy3a_launch l(dim3(kLongRows / 16 * tiles, a.cuts * rank_blocks), dim3(32 * kReduceWarps), 0, stream);
        if ((e = wide ? cudaLaunchKernelEx(&l.cfg, hy3a_adapters_reduce_kernel<T, 2, 2, true>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_adapters_reduce_kernel<T, 2, 2, false>, a)) != cudaSuccess) return e; }
    /* two blocks an SM while u leaves room for two stages at least */
    const int u_bytes = kTerms * ((a.rank + 63) / 64) * kLongRows * 128, room = (kHalf - 1024 - u_bytes) / kStageBytes, stages = room < 2 ? kLongStages : std::min(kLongStages, room), blocks = (room < 2 ? 1 : 2) * sms;
    hy3a_launch l(dim3(std::max(blocks, tiles)), dim3(kLongThreads), 1024 + stages * kStageBytes + u_bytes, stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_adapters_expand_long_kernel<T, O>, tm_b, a, stages, blocks);
}

int check_sizes(const char *who, int rows, int width, int rank) {
    if (rows < 0) return hy3a_fail(NULL, HY3A_EINVAL, "%s: rows %d < 0", who, rows);
    if (width < 8 || width % 8) return hy3a_fail(NULL, HY3A_EINVAL, "%s: width %d is no multiple of 8", who, width);
    if (width > kMaxWidth) return hy3a_fail(NULL, HY3A_EINVAL, "%s: width %d is over %d", who, width, kMaxWidth);
    if (rank < 8 || rank % 8 || rank > kMaxRank) return hy3a_fail(NULL, HY3A_EINVAL, "%s: rank %d is no multiple of 8 up to %d (fill smaller ones up with zeros)", who, rank, kMaxRank);
    return 0;
}
int cuts_of(int width) { return (width + kCut - 1) / kCut; }
/* workspace: offsets of its parts, in bytes (a tile has a row at least) */
struct workspace { size_t list, tiles, u, total; };
workspace layout(int rows, int width, int rank) {
    auto up256 = [](size_t n) { return (n + 255) & ~(size_t)255; };
    workspace w;
    w.list = 256;                             /* the number of tiles lies before it */
    w.tiles = w.list + up256((size_t)rows * sizeof(int));
    w.u = w.tiles + up256((size_t)(rows + 1) * sizeof(adapter_tile));
    w.total = w.u + up256((size_t)cuts_of(width) * rows * rank * sizeof(float));
    return w;
}

} /* namespace */

static __global__ void hy3a_adapters_wait_out_kernel() { wait_out(g_err, 39u); }
cudaError_t hy3a_adapters_wait_out(void *stream) {
    hy3a_adapters_wait_out_kernel<<<1, 1, 0, (cudaStream_t)stream>>>();
    return cudaGetLastError();
}
cudaError_t hy3a_adapters_error(unsigned *err) {
    const unsigned none[2] = {0, 0};
    cudaError_t e = cudaMemcpyFromSymbol(err, g_err, sizeof(none));
    if (e == cudaSuccess && err[0]) e = cudaMemcpyToSymbol(g_err, none, sizeof(none));
    return e;
}

extern "C" {

size_t hy3a_adapters_workspace(int rows, int width, int rank) {
    if (check_sizes("adapters_workspace", rows, width, rank)) return 0;
    return layout(rows, width, rank).total;
}

int hy3a_adapters(void *stream, int dtype, int rows, int width, int out_width, int adapters, int rank, const void *x, size_t x_stride, int base_dtype,
                  const void *base, size_t base_stride, const void *a_, const void *b_, const int *ids, const float *scales, void *out,
                  size_t out_stride, void *work, size_t work_bytes) {
    if (dtype != HY3A_F16 && dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: dtype %d not in {1,2}", dtype);
    if (base_dtype != dtype && base_dtype != HY3A_F32) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: base_dtype %d is neither the rows' (%d) nor fp32", base_dtype, dtype);
    int rc = check_sizes("adapters", rows, width, rank);
    if (rc) return rc;
    if (out_width > kMaxWidth) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: out_width %d is over %d", out_width, kMaxWidth);
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
    const workspace w = layout(rows, width, rank);
    if (work_bytes < w.total) return hy3a_fail(NULL, HY3A_EINVAL, "adapters: the workspace has %zu bytes, %zu are needed (hy3a_adapters_workspace)", work_bytes, w.total);
    char *m = (char *)work;
    const adapter_args a = {x, base, a_, b_, x_stride, base_stride, out_stride, ids, scales, out, (float *)(m + w.u), (int *)(m + w.list), (adapter_tile *)(m + w.tiles), (int *)m,
                            rows, width, out_width, adapters, rank, cuts_of(width), 0};
    cudaError_t e;
    const char *what = NULL;
    if (dtype == HY3A_F16) e = base_dtype == HY3A_F32 ? launch<__half, float>(a, dev, sms, stream, &what) : launch<__half, __half>(a, dev, sms, stream, &what);
    else e = base_dtype == HY3A_F32 ? launch<__nv_bfloat16, float>(a, dev, sms, stream, &what) : launch<__nv_bfloat16, __nv_bfloat16>(a, dev, sms, stream, &what);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "adapters: %s", what ? what : cudaGetErrorString(e));
    return HY3A_OK;
}

} /* extern "C" */

/*
 * experts.cu -- gated feed-forward networks of routed experts (hy3a_experts):
 *
 *      y[t] = sum_j w[t][j] * down_e (silu(gate_e x[t]) * (up_e x[t])),   e = ids[t][j]
 *
 * A slot is a (row, choice) pair, t * top_k + j.  Four launches, all on the stream, nothing read back:
 *   1. plan      counts the slots of each held expert, lists them expert by expert, and cuts the lists into tiles;
 *   2. gate/up   h = silu(gate x) * (up x) of every listed slot, rounded once to the rows' type (it is the next product's operand; fp16 rows take a launch
 *                for that, which brings each slot's h near the top of the type's range first: products of two sums may be beyond it, and below);
 *   3. down      y of every listed slot, fp32;
 *   4. combine   sums a row's slots in the order of j, fp32, and rounds once.
 * Fewer than 32 slots take no plan: gate / up (and the range), and down with the sum.
 * Slots whose id is outside [first_expert, first_expert + held) are left out everywhere.  The place of a slot within its expert's list
 * comes from an atomic and may differ from run to run; no sum depends on it, so results do not.
 */
#include <math.h>

#include <algorithm>

#include "experts.h"
#include "grouping.cuh"

namespace {

using namespace hy3a_layer;

constexpr int kMaxHeld = kGroupThreads;
constexpr int kFewMost = 32;           /* slots of a call below which its products run here */

/* ---- workspace: offsets of its parts, in bytes ------------------------------------------------------------------------ */
struct workspace {
    size_t row, place, tiles, h, back, y, total;
};
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
workspace layout(long long slots, int hidden, int inter, int held) {
    workspace w;
    w.row = 0;
    w.place = w.row + up256((size_t)slots * 4);
    w.tiles = w.place + up256((size_t)slots * 4);
    w.h = w.tiles + 256 + up256(((size_t)slots / kTileSlots + (slots < held ? slots : held)) * sizeof(expert_tile));     /* their number, then the table */
    w.back = w.h + up256((size_t)slots * inter * (slots < kFewMost ? 4 : 2));
    w.y = w.back + up256((size_t)slots * 4);
    w.total = w.y + up256((size_t)slots * std::max(hidden, inter) * 4);        /* y, and before it h in fp32 */
    return w;
}

__device__ __forceinline__ int local_expert(const expert_args &a, int id) {
    const int e = id - a.first;
    return id >= 0 && e >= 0 && e < a.held ? e : -1;
}

/* ---- 1. plan ------------------------------------------------------------------------------------------------------------ */
template <int BLOCKS>
__global__ void __launch_bounds__(kGroupThreads) hy3a_experts_plan_kernel(const expert_args a) {
    pdl_release();
    const int tiles = group_items<BLOCKS, 1, false>(
        a.slots, a.held, kTileSlots, [&](int i) { const int e = local_expert(a, a.ids[i]); if (e < 0) a.place[i] = -1; return e; },
        [&](int e, int p0, int n, int first, int count) { for (int j = 0; j < count; j++) a.tiles[first + j] = {e, first, count, p0, n}; },
        [&](int i, int p) { a.row[p] = i / a.top_k; a.place[i] = p; });
    if (threadIdx.x == 0 && (BLOCKS == 1 || cluster_rank() == 0)) *a.n_tiles = tiles;
}

/* ---- fp16 rows, between gate / up and down: h as fp16 holds it ------------------------------------------------------------
 * The products of two sums may be beyond the type's range, or so small that it keeps few of their bits, where the result is neither.  A warp takes a slot (a
 * block, up to two slots an SM), and brings its largest value into [2^14, 2^15) on the way to fp16: 2^-38 of it is kept.  us a pass, without / with it: 1 row
 * of 192 experts 54.1 / 57.0, 8 rows 313 / 318, 2048 rows 1277 / 1344, 8192 rows on 24 held experts 377 / 413, 333 rows of 10 small ones 22.6 / 27.0.  Two blocks an SM find room beside gate / up, and
 * are there when it ends. */
/* the larger of m and |v|, if that is finite */
__device__ __forceinline__ float most_finite(float m, float v) { return fabsf(v) <= 3.402823466e38f ? fmaxf(m, fabsf(v)) : m; }
constexpr int kRangeThreads = 256, kRangeBlocks = 2 /* an SM */;
/* EACH: threads of a slot, 32 or, if there are no more slots than blocks, all of a block */
template <bool FEW, int EACH>
__global__ void __launch_bounds__(kRangeThreads) hy3a_experts_range_kernel(const expert_args a) {
    pdl_release();                          /* (gate / up let this launch begin behind its own wait: the plan is complete, here and for `down`) */
    const int sub = threadIdx.x % EACH, quads = a.inter >> 2, tiles = FEW ? 0 : *a.n_tiles;
    const int listed = FEW ? a.slots : (tiles ? a.tiles[tiles - 1].p0 + a.tiles[tiles - 1].count : 0);      /* (few: those without an expert too, nobody reads theirs) */
    pdl_wait();
    for (int p = (blockIdx.x * kRangeThreads + threadIdx.x) / EACH; p < listed; p += gridDim.x * kRangeThreads / EACH) {
        const float4 *const from = reinterpret_cast<const float4 *>(a.wide + (size_t)p * a.inter);
        float most = 0.f;
#pragma unroll 4
        for (int i = sub; i < quads; i += EACH) {
            const float4 v = from[i];
            most = most_finite(most_finite(most_finite(most_finite(most, v.x), v.y), v.z), v.w);
        }
        most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        if (EACH > 32) {
            __shared__ float s_most[kRangeThreads / 32];
            if ((sub & 31) == 0) s_most[sub >> 5] = most;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kRangeThreads / 32; w++) most = fmaxf(most, s_most[w]);
        }
        /* 2^n that does it, at most 2^100; and its inverse */
        const int n = most > 0.f ? min(141 - (int)(__float_as_uint(most) >> 23), 100) : 0;
        const float by = __uint_as_float((unsigned)(127 + n) << 23);
        if (sub == 0) a.back[p] = __uint_as_float((unsigned)(127 - n) << 23);
        __half *const h = reinterpret_cast<__half *>(a.h) + (size_t)p * a.inter;
#pragma unroll 4
        for (int i = sub; i < quads; i += EACH) {
            const float4 v = from[i];
            const float f[4] = {v.x * by, v.y * by, v.z * by, v.w * by};
            __half one[4], rest[4];
#pragma unroll
            for (int z = 0; z < 4; z++) {
                one[z] = __float2half_rn(f[z]);
                rest[z] = __float2half_rn(isinf(f[z]) ? 0.f : f[z] - __half2float(one[z]));
            }
            *reinterpret_cast<uint2 *>(h + 4 * i) = *reinterpret_cast<const uint2 *>(one);
            if (FEW) *reinterpret_cast<uint2 *>(h + (size_t)a.slots * a.inter + 4 * i) = *reinterpret_cast<const uint2 *>(rest);
        }
    }
}

/* ---- calls with few slots (at most 31; the others: experts_umma.cu) -----------------------------------------------------
 * Two launches (fp16 rows three), without a plan: every warp sees all slots.  The first slot of an expert leads, and takes the expert's other slots along, 8 at a
 * time (more than 8 read the weights again, from L2).  h enters the second product as two numbers of the rows' type, the rounded value and the
 * rest: with so few values the error that one number leaves is now and then more than half as large again as that of the result's own rounding.
 * Fragments come straight from global memory (layer.h), 8 loads of 32 bytes in flight a lane. */
constexpr int kFewWarps = 8, kFewLoads = 4 /* k blocks of 64 in flight */;
/* lane s: expert of slot s (-1: none), the slots of the same expert */
__device__ __forceinline__ int few_slots(const expert_args &a, unsigned &same) {
    const int lane = threadIdx.x & 31, e = lane < a.slots ? local_expert(a, a.ids[lane]) : -1;
    same = __match_any_sync(0xffffffffu, e);
    return e;
}
/* position of the n-th set bit, -1 if there are fewer */
__device__ __forceinline__ int nth_bit(unsigned bits, int n) {
    for (; n > 0; n--) bits &= bits - 1;
    return bits ? __ffs(bits) - 1 : -1;
}
template <class T, bool WIDE> __device__ __forceinline__ void few_load(k16 (&lo)[kFewLoads], k16 (&hi)[kFewLoads], const T *w_lo, const T *w_hi, bool has_lo, bool has_hi, int k, int step, int K) {
#pragma unroll
    for (int u = 0; u < kFewLoads; u++) {
        lo[u] = load16<WIDE, true>(w_lo + k + u * step, has_lo ? K - k - u * step : 0);
        hi[u] = load16<WIDE, true>(w_hi + k + u * step, has_hi ? K - k - u * step : 0);
    }
}
template <class T, bool WIDE> __device__ __forceinline__ void few_multiply(float (&acc)[4], const k16 (&lo)[kFewLoads], const k16 (&hi)[kFewLoads], const T *row, int k, int step, int K) {
#pragma unroll
    for (int u = 0; u < kFewLoads; u++) mma64<T>(acc, lo[u], hi[u], load16<WIDE, false>(row + k + u * step, row ? K - k - u * step : 0));
}

/* h of one expert's slots, 8 of its rows: block = (8 pairs of gate and up rows, slot that may lead); the warps share the k's, and their sums
 * meet in shared memory in a fixed order.  Rows 0-7 of A are gate rows, rows 8-15 the up rows of the same index: both halves of a pair lie in
 * one lane. */
template <class T, bool WIDE>
__global__ void __launch_bounds__(32 * kFewWarps, 3) hy3a_experts_few_up_kernel(const expert_args a) {
    __shared__ float s_sum[kFewWarps][4][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_release();                          /* behind the wait: what the next kernel reads before its own is complete */
    unsigned same;
    const int mine = few_slots(a, same), e = __shfl_sync(0xffffffffu, mine, blockIdx.y);
    const unsigned slots = __shfl_sync(0xffffffffu, same, blockIdx.y);
    if (e < 0 || (int)blockIdx.y != __ffs(slots) - 1) return;
    const int K = a.hidden, M = a.inter, m0 = blockIdx.x * 8, step = 64 * kFewWarps;
    const bool has = m0 + g < M;
    const T *gate = reinterpret_cast<const T *>(a.gate) + ((size_t)e * M + m0 + g) * K, *up = reinterpret_cast<const T *>(a.up) + ((size_t)e * M + m0 + g) * K;
    for (int base = 0; base < __popc(slots); base += 8) {
        const int s = nth_bit(slots, base + g);
        const T *x = s >= 0 ? reinterpret_cast<const T *>(a.x) + (size_t)(s / a.top_k) * a.x_stride : nullptr;
        float acc[4] = {};
        for (int kb = warp * 64; kb < K; kb += step * kFewLoads) {
            k16 lo[kFewLoads], hi[kFewLoads];
            few_load<T, WIDE>(lo, hi, gate, up, has, has, kb + t * 16, step, K);
            few_multiply<T, WIDE>(acc, lo, hi, x, kb + t * 16, step, K);
        }
        if (base) __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; c++) s_sum[warp][c][lane] = acc[c];
        __syncthreads();
        /* accumulator c of lane (g, t): row g (c < 2) or g + 8, column 2t + (c & 1) */
        if (tid < 64) {
            const int m = tid & 7, col = tid >> 3, from = m * 4 + (col >> 1), c = col & 1, to = nth_bit(slots, base + col);
            float lo = 0.f, hi = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; w++) { lo += s_sum[w][c][from]; hi += s_sum[w][2 + c][from]; }
            if (to >= 0 && m0 + m < M) {
                const float v = __fdividef(lo, 1.f + __expf(-lo)) * hi;
                const size_t at = (size_t)to * M + m0 + m;
                if (type<T>::code == HY3A_F16) a.wide[at] = v;
                else {
                    const T h = type<T>::down(v);
                    reinterpret_cast<T *>(a.h)[at] = h;
                    reinterpret_cast<T *>(a.h)[at + (size_t)a.slots * M] = type<T>::down(isinf(type<T>::up(h)) ? 0.f : v - type<T>::up(h));
                }
            }
        }
    }
}

/* out: block = 16 columns; its warps take the experts in turn, or shares of their k's where there are fewer experts than warps, and the slots'
 * sums are weighed and added up in shared memory, in the order of the choices.  The first weights are on their way before the wait for h. */
template <class T, bool WIDE>
__global__ void __launch_bounds__(32 * kFewWarps, 2) hy3a_experts_few_down_kernel(const expert_args a) {
    __shared__ float s_y[kFewWarps][kFewMost][16];                         /* [share of the k's][slot][column] */
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned same;
    const int mine = few_slots(a, same);
    const unsigned any = __ballot_sync(0xffffffffu, mine >= 0), leaders = __ballot_sync(0xffffffffu, mine >= 0 && lane == __ffs(same) - 1);
    const int n = __popc(leaders), shares = n ? max(1, kFewWarps / n) : 1;
    const int K = a.inter, M = a.hidden, m0 = blockIdx.x * 16, step = shares * 64;
    const size_t rest = (size_t)a.slots * K;
    bool waited = false;
    for (int unit = warp; unit < n * shares; unit += kFewWarps) {
        const int which = unit / shares, share = unit - which * shares, lead = nth_bit(leaders, which);
        const int e = __shfl_sync(0xffffffffu, mine, lead);
        const unsigned slots = __shfl_sync(0xffffffffu, same, lead);
        const T *w_lo = reinterpret_cast<const T *>(a.down) + ((size_t)e * M + m0 + g) * K, *w_hi = w_lo + (size_t)8 * K;
        const bool has_lo = m0 + g < M, has_hi = m0 + 8 + g < M;
        for (int base = 0; base < __popc(slots); base += 8) {
            const int s = nth_bit(slots, base + g);
            const T *h = s >= 0 ? reinterpret_cast<const T *>(a.h) + (size_t)s * K : nullptr;
            float acc[4] = {}, acc_rest[4] = {};
            for (int kb = share * 64; kb < K; kb += step * kFewLoads) {
                k16 lo[kFewLoads], hi[kFewLoads];
                few_load<T, WIDE>(lo, hi, w_lo, w_hi, has_lo, has_hi, kb + t * 16, step, K);
                if (!waited) { pdl_wait(); waited = true; }
                const int k = kb + t * 16;
#pragma unroll
                for (int u = 0; u < kFewLoads; u++) {
                    const int left = h ? K - k - u * step : 0;
                    const k16 v = load16<WIDE, false>(h + k + u * step, left), r = load16<WIDE, false>(h + rest + k + u * step, left);
                    mma64<T>(acc, lo[u], hi[u], v);
                    mma64<T>(acc_rest, lo[u], hi[u], r);
                }
            }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int to = nth_bit(slots, base + 2 * t + (c & 1));
                /* (an infinite weight meets both numbers of h, whose signs may differ: then the first has it) */
                const float y = fabsf(acc[c]) <= 3.402823466e38f ? acc[c] + acc_rest[c] : acc[c];
                if (to >= 0) s_y[share][to][g + (c >> 1) * 8] = type<T>::code == HY3A_F16 ? a.back[to] * y : y;
            }
        }
    }
    if (!waited) pdl_wait();
    pdl_release();
    __syncthreads();
    const int m = tid & 15;
    if (m0 + m >= M) return;
    for (int row = tid >> 4; row < a.rows; row += 2 * kFewWarps) {
        float sum = 0.f;
        for (int j = 0; j < a.top_k; j++) {
            const int s = row * a.top_k + j;
            if (!((any >> s) & 1)) continue;
            float y = 0.f;
            for (int i = 0; i < shares; i++) y += s_y[i][s][m];
            sum += a.weights[s] * y;
        }
        reinterpret_cast<T *>(a.out)[(size_t)row * a.out_stride + m0 + m] = type<T>::down(sum);
    }
}

/* ---- 4. combine: a thread per 8 columns of a row ------------------------------------------------------------------------
 * (The weights and places come from launches that are complete before `down` lets this one begin.)  Bound by the chain of its loads and by memory: 39 us by
 * itself for 8192 rows of 4096 with a slot each, whose 201 MB take 31. */
template <class T>
__global__ void __launch_bounds__(256) hy3a_experts_combine_kernel(const expert_args a) {
    pdl_release();
    const int row = blockIdx.x, d = (blockIdx.y * 256 + threadIdx.x) * 8, lane = threadIdx.x & 31;
    const size_t s0 = (size_t)row * a.top_k;
    const int place = lane < a.top_k ? a.place[s0 + lane] : -1;
    const float w_lane = lane < a.top_k ? a.weights[s0 + lane] : 0.f;
    unsigned todo = __ballot_sync(0xffffffffu, place >= 0);
    const bool in = d < a.hidden;
    pdl_wait();
    float sum[8] = {};
#pragma unroll 4
    while (todo) {                            /* (in the order of the choices) */
        const int j = __ffs(todo) - 1;
        todo &= todo - 1;
        const float w = __shfl_sync(0xffffffffu, w_lane, j);
        const size_t p = (size_t)__shfl_sync(0xffffffffu, place, j);
        if (!in) continue;
        const float4 *const y = reinterpret_cast<const float4 *>(a.y + p * a.hidden + d), lo = y[0], hi = y[1];
        sum[0] += w * lo.x; sum[1] += w * lo.y; sum[2] += w * lo.z; sum[3] += w * lo.w;
        sum[4] += w * hi.x; sum[5] += w * hi.y; sum[6] += w * hi.z; sum[7] += w * hi.w;
    }
    if (!in) return;
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = type<T>::down(sum[i]);
    *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + (size_t)row * a.out_stride + d) = *reinterpret_cast<const uint4 *>(o);
}

template <class T>
cudaError_t launch_few(const expert_args &a, void *stream) {
    hy3a_launch l(dim3((a.inter + 7) / 8, a.slots), dim3(32 * kFewWarps), 0, stream);
    const bool wide_up = wide_rows({a.x, a.gate, a.up}, {a.x_stride, (size_t)a.hidden}), wide_down = wide_rows({a.down}, {(size_t)a.inter});
    const cudaError_t e = wide_up ? cudaLaunchKernelEx(&l.cfg, hy3a_experts_few_up_kernel<T, true>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_experts_few_up_kernel<T, false>, a);
    if (e != cudaSuccess) return e;
    if (type<T>::code == HY3A_F16) {
        hy3a_launch r(dim3(a.slots), dim3(kRangeThreads), 0, stream);
        const cudaError_t e = cudaLaunchKernelEx(&r.cfg, hy3a_experts_range_kernel<true, kRangeThreads>, a);
        if (e != cudaSuccess) return e;
    }
    hy3a_launch d(dim3((a.hidden + 15) / 16), dim3(32 * kFewWarps), 0, stream);
    return wide_down ? cudaLaunchKernelEx(&d.cfg, hy3a_experts_few_down_kernel<T, true>, a) : cudaLaunchKernelEx(&d.cfg, hy3a_experts_few_down_kernel<T, false>, a);
}
template <class T>
cudaError_t launch(const expert_args &a, int device, int sms, void *stream, const char **what) {
    /* us a pass, few / umma: bf16, 8 of 192 experts of 4096 x 1536 for 1, 2, 3 rows 54.4 / 67.5, 94.5 / 110, 137 / 149; fp16, the same for 1, 3 rows 57.3 / 70.5,
     * 141 / 153, 3 of 10 of 1032 x 200 for 1, 10 rows 11.3 / 17.2, 12.4 / 18.1 */
    if (a.slots < kFewMost) return launch_few<T>(a, stream);
    cudaError_t e;
    const bool shared = a.slots >= kGroupShared;
    {   hy3a_launch l(dim3(shared ? kGroupCluster : 1), dim3(kGroupThreads), 0, stream);
        if (shared) l.cluster(kGroupCluster);
        if ((e = shared ? cudaLaunchKernelEx(&l.cfg, hy3a_experts_plan_kernel<kGroupCluster>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_experts_plan_kernel<1>, a)) != cudaSuccess) return e; }
    if ((e = hy3a_experts_launch_umma(a, type<T>::code, device, sms, stream, what)) != cudaSuccess) return e;
    hy3a_launch l(dim3(a.rows, (a.hidden / 8 + 255) / 256), dim3(256), 0, stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_experts_combine_kernel<T>, a);
}

/* tiles are counted in 32 bits: 2^28 slots in tiles of 256, times 2^16 weight rows in tiles of 128 (pairs) */
constexpr int kMaxWidth = 65536;
int check_sizes(const char *who, int rows, int top_k, int hidden, int inter, int held) {
    if (rows < 0) return hy3a_fail(NULL, HY3A_EINVAL, "%s: rows %d < 0", who, rows);
    if (top_k < 1 || top_k > 32) return hy3a_fail(NULL, HY3A_EINVAL, "%s: top_k %d not in [1,32]", who, top_k);
    if (hidden < 8 || hidden % 8 || inter < 8 || inter % 8) return hy3a_fail(NULL, HY3A_EINVAL, "%s: hidden %d and inter %d have to be multiples of 8", who, hidden, inter);
    if (held < 1 || held > kMaxHeld) return hy3a_fail(NULL, HY3A_EINVAL, "%s: %d experts held, not in [1,%d]", who, held, kMaxHeld);
    if (hidden > kMaxWidth || inter > kMaxWidth) return hy3a_fail(NULL, HY3A_EINVAL, "%s: hidden %d or inter %d is over %d", who, hidden, inter, kMaxWidth);
    if ((long long)rows * top_k >= 1ll << 28) return hy3a_fail(NULL, HY3A_EINVAL, "%s: %d rows of %d slots are too many", who, rows, top_k);
    return 0;
}

} /* namespace */

cudaError_t hy3a_experts_launch_range(const expert_args &a, int sms, void *stream) {
    const int most = kRangeBlocks * sms, each = kRangeThreads / 32;
    hy3a_launch l(dim3(a.slots <= most ? a.slots : std::min((a.slots + each - 1) / each, most)), dim3(kRangeThreads), 0, stream);
    return a.slots <= most ? cudaLaunchKernelEx(&l.cfg, hy3a_experts_range_kernel<false, kRangeThreads>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_experts_range_kernel<false, 32>, a);
}

extern "C" {

size_t hy3a_experts_workspace(int rows, int top_k, int hidden, int inter, int held) {
    if (check_sizes("experts_workspace", rows, top_k, hidden, inter, held)) return 0;
    return layout((long long)rows * top_k, hidden, inter, held).total;
}

int hy3a_experts(void *stream, int dtype, int rows, int top_k, int hidden, int inter, int held, int first_expert, const void *x, size_t x_stride,
                 const int *ids, const float *weights, const void *gate, const void *up, const void *down, void *out, size_t out_stride,
                 void *work, size_t work_bytes) {
    if (dtype != HY3A_F16 && dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "experts: dtype %d not in {1,2}", dtype);
    int rc = check_sizes("experts", rows, top_k, hidden, inter, held);
    if (rc) return rc;
    if (first_expert < 0 || first_expert > 0x7fffffff - held) return hy3a_fail(NULL, HY3A_EINVAL, "experts: first_expert %d", first_expert);
    if (rows == 0) return HY3A_OK;
    if (!x || !ids || !weights || !gate || !up || !down || !out || !work) return hy3a_fail(NULL, HY3A_EINVAL, "experts: NULL argument");
    if (((uintptr_t)x | (uintptr_t)gate | (uintptr_t)up | (uintptr_t)down | (uintptr_t)out) & 15) return hy3a_fail(NULL, HY3A_EINVAL, "experts: pointers must be 16-byte aligned");
    if (((uintptr_t)ids | (uintptr_t)weights) & 3) return hy3a_fail(NULL, HY3A_EINVAL, "experts: ids and weights must be 4-byte aligned");
    if ((uintptr_t)work & 255) return hy3a_fail(NULL, HY3A_EINVAL, "experts: the workspace must be 256-byte aligned");
    if ((x_stride & 7) || (out_stride & 7)) return hy3a_fail(NULL, HY3A_EINVAL, "experts: row strides must be multiples of 8");
    if (x_stride < (size_t)hidden && rows > 1) return hy3a_fail(NULL, HY3A_EINVAL, "experts: x rows of %d overlap at a stride of %zu", hidden, x_stride);
    if (out_stride < (size_t)hidden && rows > 1) return hy3a_fail(NULL, HY3A_EINVAL, "experts: out rows of %d overlap at a stride of %zu", hidden, out_stride);
    const workspace w = layout((long long)rows * top_k, hidden, inter, held);
    if (work_bytes < w.total) return hy3a_fail(NULL, HY3A_EINVAL, "experts: the workspace has %zu bytes, %zu are needed (hy3a_experts_workspace)", work_bytes, w.total);
    int dev, sms;
    if ((rc = hy3a_layer_device("experts", &dev, &sms))) return rc;
    char *b = (char *)work;
    expert_args a = {x, x_stride, ids, weights, gate, up, down, out, out_stride, rows, top_k, hidden, inter, held, first_expert, rows * top_k,
                     (int *)(b + w.row), (int *)(b + w.place), (expert_tile *)(b + w.tiles + 256), (int *)(b + w.tiles), b + w.h, (float *)(b + w.y), (float *)(b + w.back), (float *)(b + w.y)};
    const char *what = NULL;
    const cudaError_t e = dtype == HY3A_F16 ? launch<__half>(a, dev, sms, stream, &what) : launch<__nv_bfloat16>(a, dev, sms, stream, &what);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "experts: %s", what ? what : cudaGetErrorString(e));
    return HY3A_OK;
}

} /* extern "C" */

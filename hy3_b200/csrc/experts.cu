/*
 * experts.cu -- gated feed-forward networks of routed experts (hy3a_experts):
 *
 *      y[t] = sum_j w[t][j] * down_e (silu(gate_e x[t]) * (up_e x[t])),   e = ids[t][j]
 *
 * A slot is a (row, choice) pair, t * top_k + j.  Four launches, all on the stream, nothing read back:
 *   1. plan      counts the slots of each held expert, lists them expert by expert, and cuts the lists into tiles;
 *   2. gate/up   h = silu(gate x) * (up x) of every listed slot, rounded once to the rows' type (it is the next product's operand);
 *   3. down      y of every listed slot, fp32 (few slots) or in fixed point (experts.h);
 *   4. combine   sums a row's slots in the order of j, fp32, and rounds once.
 * Slots whose id is outside [first_expert, first_expert + held) are left out everywhere.  The place of a slot within its expert's list
 * comes from an atomic and may differ from run to run; no sum depends on it, so results do not.
 */
#include <math.h>

#include "experts.h"

namespace {

using namespace hy3a_layer;

constexpr int kFewMost = 32;           /* slots of a call below which its products run here */

/* ---- workspace: offsets of its parts, in bytes ------------------------------------------------------------------------ */
struct workspace {
    size_t off, active, row, place, tiles, h, y, scale, total;
};
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
workspace layout(long long slots, int hidden, int inter, int held) {
    workspace w;
    w.off = 0;
    w.active = w.off + up256(((size_t)held + 1) * 4);
    w.row = w.active + up256(((size_t)held + 1) * 4);
    w.place = w.row + up256((size_t)slots * 4);
    w.tiles = w.place + up256((size_t)slots * 4);
    w.h = w.tiles + 256 + up256(((size_t)slots / kTileSlots + (slots < held ? slots : held)) * sizeof(expert_tile));     /* their number, then the table */
    w.y = w.h + up256((size_t)slots * inter * 2);
    const bool few = slots < kFewMost;
    w.scale = w.y + up256((size_t)slots * hidden * (few ? 4 : 2));
    w.total = w.scale + (few ? 0 : up256((size_t)slots * ((hidden + 31) / 32) * 4));
    return w;
}

__device__ __forceinline__ int local_expert(const expert_args &a, int id) {
    const int e = id - a.first;
    return id >= 0 && e >= 0 && e < a.held ? e : -1;
}

/* ---- 1. plan: one block, or a cluster of 8 that share the slots ---------------------------------------------------------
 * Each block counts its part of the slots, all read all counts, and each lists its part.  65 536 slots: 37 us with one block, TWO with 8. */
constexpr int kPlanThreads = 1024, kMaxHeld = 1024, kPlanCluster = 8, kPlanShared = 4096;      /* slots from which blocks share them */
__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int peer_value(const int *p, unsigned rank) {
    unsigned a = (unsigned)__cvta_generic_to_shared(p);
    int v;
    asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(a) : "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
template <int BLOCKS>
__global__ void __launch_bounds__(kPlanThreads) hy3a_experts_plan_kernel(const expert_args a) {
    __shared__ int s_count[kMaxHeld], s_next[kMaxHeld], s_warp[3][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned me = BLOCKS > 1 ? cluster_rank() : 0;
    const int per = (a.slots + BLOCKS - 1) / BLOCKS, begin = min(a.slots, (int)me * per), end = min(a.slots, begin + per);
    pdl_release();
    for (int e = tid; e < a.held; e += kPlanThreads) s_count[e] = 0;
    __syncthreads();
    pdl_wait();
#pragma unroll 4
    for (int i = begin + tid; i < end; i += kPlanThreads) {
        const int e = local_expert(a, a.ids[i]);
        if (e >= 0) atomicAdd(&s_count[e], 1);
    }
    if (BLOCKS > 1) cluster_sync(); else __syncthreads();
    /* a thread per expert: its slots, those of the blocks before this one, its tiles; exclusive sums over the experts */
    int n = 0, earlier = 0;
    if (tid < a.held) {
        if (BLOCKS == 1) n = s_count[tid];
        else {
#pragma unroll
            for (int r = 0; r < BLOCKS; r++) {
                const int c = peer_value(&s_count[tid], r);
                n += c;
                if (r < (int)me) earlier += c;
            }
        }
    }
    const int tiles = (n + kTileSlots - 1) / kTileSlots;
    int sum[3] = {n, tiles, n > 0};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < 3; i++) {
            const int u = __shfl_up_sync(0xffffffffu, sum[i], o);
            if (lane >= o) sum[i] += u;
        }
#pragma unroll
    for (int i = 0; i < 3; i++) if (lane == 31) s_warp[i][warp] = sum[i];
    __syncthreads();
    int total[3];
#pragma unroll
    for (int i = 0; i < 3; i++) {
        int w = s_warp[i][lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        total[i] = __shfl_sync(0xffffffffu, w, 31);
        const int before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
        sum[i] += warp ? before : 0;
    }
    const int p0 = sum[0] - n, first = sum[1] - tiles, at = sum[2] - (n > 0);
    if (tid < a.held) {
        s_next[tid] = p0 + earlier;           /* where the block's next slot of the expert goes */
        if (me == 0) {
            a.off[tid] = p0;
            if (n > 0) a.active[1 + at] = tid;
            for (int j = 0; j < tiles; j++) a.tiles[first + j] = {tid, first, tiles, p0, n};
        }
    }
    if (tid == 0 && me == 0) { a.off[a.held] = total[0]; a.active[0] = total[2]; *a.n_tiles = total[1]; }
    __syncthreads();
#pragma unroll 4
    for (int i = begin + tid; i < end; i += kPlanThreads) {
        const int e = local_expert(a, a.ids[i]);
        if (e >= 0) {
            const int p = atomicAdd(&s_next[e], 1);
            a.row[p] = i / a.top_k;
            a.place[i] = p;
        }
    }
    if (BLOCKS > 1) cluster_sync();           /* nobody leaves while its counts are read */
}

/* ---- 2. and 3. of calls with few slots (the others: experts_umma.cu) ------------------------------------------------------------------------------------
 * A block takes one expert and 16 of its weight rows, 8 warps share the k's, fragments come straight from global memory (layer.h), and
 * the warps' sums meet in shared memory in a fixed order.  Up to 32 slots go through together.  Rows 0-7 of the gate / up product's A
 * are gate rows, rows 8-15 the up rows of the same index, so that both halves of a pair lie in one lane. */
constexpr int kFewWarps = 8, kFewSlots = 32, kUnroll = 4;
template <class T, bool DOWN>
__global__ void __launch_bounds__(32 * kFewWarps) hy3a_experts_few_kernel(const expert_args a) {
    __shared__ float s_sum[kFewWarps][kFewSlots / 8][4][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_release();
    pdl_wait();
    if (blockIdx.y >= a.active[0]) return;
    const int e = a.active[1 + blockIdx.y], p0 = a.off[e], count = a.off[e + 1] - p0;
    const int K = DOWN ? a.inter : a.hidden, M = DOWN ? a.hidden : a.inter;
    const int m0 = blockIdx.x * (DOWN ? 16 : 8), r_lo = m0 + g, r_hi = DOWN ? m0 + 8 + g : r_lo;
    const T *w_lo = reinterpret_cast<const T *>(DOWN ? a.down : a.gate) + ((size_t)e * M + r_lo) * K;
    const T *w_hi = reinterpret_cast<const T *>(DOWN ? a.down : a.up) + ((size_t)e * M + r_hi) * K;
    const bool has_lo = r_lo < M, has_hi = r_hi < M;
    for (int base = 0; base < count; base += kFewSlots) {
        const int groups = min(kFewSlots / 8, (count - base + 7) >> 3);
        const T *row[kFewSlots / 8];
#pragma unroll
        for (int i = 0; i < kFewSlots / 8; i++) {
            const int p = p0 + base + 8 * i + g;
            row[i] = nullptr;
            if (base + 8 * i + g < count) row[i] = DOWN ? reinterpret_cast<const T *>(a.h) + (size_t)p * a.inter : reinterpret_cast<const T *>(a.x) + (size_t)a.row[p] * a.x_stride;
        }
        float acc[kFewSlots / 8][4] = {};
        for (int kb = warp * 32; kb < K; kb += 32 * kFewWarps * kUnroll) {
            const int k0 = kb + t * 8;
            uint4 lo[kUnroll], hi[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; u++) {
                const int k = k0 + u * 32 * kFewWarps;
                lo[u] = has_lo && k < K ? load_once(w_lo + k) : zero16();
                hi[u] = has_hi && k < K ? load_once(w_hi + k) : zero16();
            }
#pragma unroll
            for (int i = 0; i < kFewSlots / 8; i++) {
                if (i < groups) {
#pragma unroll
                    for (int u = 0; u < kUnroll; u++) {
                        const int k = k0 + u * 32 * kFewWarps;
                        mma32<T>(acc[i], lo[u], hi[u], row[i] && k < K ? load_row(row[i] + k) : zero16());
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kFewSlots / 8; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) s_sum[warp][i][c][lane] = acc[i][c];
        __syncthreads();
        /* accumulator c of lane (g, t): row g (c < 2) or g + 8, column 2t + (c & 1) */
        const int m = tid & 7, col = tid >> 3, from = m * 4 + ((col & 7) >> 1), c0 = col & 1, i = col >> 3;
        if (base + col < count) {
            float lo = 0.f, hi = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; w++) { lo += s_sum[w][i][c0][from]; hi += s_sum[w][i][2 + c0][from]; }
            const int p = p0 + base + col;
            if (DOWN) {
                float *y = a.y + (size_t)p * a.hidden + m0;
                if (m0 + m < M) y[m] = lo;
                if (m0 + 8 + m < M) y[8 + m] = hi;
            } else if (m0 + m < M) {
                reinterpret_cast<T *>(a.h)[(size_t)p * a.inter + m0 + m] = type<T>::down(__fdividef(lo, 1.f + __expf(-lo)) * hi);
            }
        }
        __syncthreads();
    }
}

/* ---- 4. combine: a thread per 8 columns of a row; FIXED: y is a.q and a.q_scale (experts.h) ------------------------------ */
template <class T, bool FIXED>
__global__ void __launch_bounds__(256) hy3a_experts_combine_kernel(const expert_args a) {
    pdl_release();
    pdl_wait();
    const int row = blockIdx.x, d = (blockIdx.y * 256 + threadIdx.x) * 8, lane = threadIdx.x & 31;
    const size_t s0 = (size_t)row * a.top_k;
    const bool mine = lane < a.top_k && local_expert(a, a.ids[s0 + lane]) >= 0;
    const float w_lane = mine ? a.weights[s0 + lane] : 0.f;
    const int place = mine ? a.place[s0 + lane] : 0;
    unsigned todo = __ballot_sync(0xffffffffu, mine);
    const bool in = d < a.hidden;
    float sum[8] = {};
#pragma unroll 4
    while (todo) {                            /* (in the order of the choices) */
        const int j = __ffs(todo) - 1;
        todo &= todo - 1;
        const float w = __shfl_sync(0xffffffffu, w_lane, j);
        const size_t p = (size_t)__shfl_sync(0xffffffffu, place, j);
        if (!in) continue;
        if (FIXED) {
            const uint4 v = *reinterpret_cast<const uint4 *>(a.q + p * a.hidden + d);
            const float scale = a.q_scale[p * ((a.hidden + 31) >> 5) + (d >> 5)];
            const unsigned u[4] = {v.x, v.y, v.z, v.w};
            if (scale >= 0.f) {
                const float ws = w * scale;
#pragma unroll
                for (int i = 0; i < 4; i++) { sum[2 * i] += ws * (float)(short)(u[i] & 0xffff); sum[2 * i + 1] += ws * (float)(short)(u[i] >> 16); }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) { sum[2 * i] += w * __uint_as_float(u[i] << 16); sum[2 * i + 1] += w * __uint_as_float(u[i] & 0xffff0000u); }
            }
        } else {
            const float4 *y = reinterpret_cast<const float4 *>(a.y + p * a.hidden + d);
            const float4 v0 = y[0], v1 = y[1];
            sum[0] += w * v0.x; sum[1] += w * v0.y; sum[2] += w * v0.z; sum[3] += w * v0.w;
            sum[4] += w * v1.x; sum[5] += w * v1.y; sum[6] += w * v1.z; sum[7] += w * v1.w;
        }
    }
    if (!in) return;
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = type<T>::down(sum[i]);
    *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + (size_t)row * a.out_stride + d) = *reinterpret_cast<const uint4 *>(o);
}

template <class T>
cudaError_t launch_few(const expert_args &a, void *stream) {
    cudaError_t e;
    const int most = a.slots < a.held ? a.slots : a.held;       /* experts that can have slots */
    {   hy3a_launch l(dim3((a.inter + 7) / 8, most), dim3(32 * kFewWarps), 0, stream);
        if ((e = cudaLaunchKernelEx(&l.cfg, hy3a_experts_few_kernel<T, false>, a)) != cudaSuccess) return e; }
    hy3a_launch l(dim3((a.hidden + 15) / 16, most), dim3(32 * kFewWarps), 0, stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_experts_few_kernel<T, true>, a);
}
template <class T>
cudaError_t launch(const expert_args &a, int device, int sms, void *stream, const char **what) {
    cudaError_t e;
    const bool shared = a.slots >= kPlanShared, few = a.slots < kFewMost;
    {   hy3a_launch l(dim3(shared ? kPlanCluster : 1), dim3(kPlanThreads), 0, stream);
        if (shared) l.cluster(kPlanCluster);
        if ((e = shared ? cudaLaunchKernelEx(&l.cfg, hy3a_experts_plan_kernel<kPlanCluster>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_experts_plan_kernel<1>, a)) != cudaSuccess) return e; }
    /* a handful of slots (bf16, 192 experts of 4096 x 1536; us a pass, few / umma): 8 slots 74 / 83, 64 slots 390 / 343 */
    if (few) e = launch_few<T>(a, stream);
    else e = hy3a_experts_launch_umma(a, type<T>::code, device, sms, stream, what);
    if (e != cudaSuccess) return e;
    hy3a_launch l(dim3(a.rows, (a.hidden / 8 + 255) / 256), dim3(256), 0, stream);
    return few ? cudaLaunchKernelEx(&l.cfg, hy3a_experts_combine_kernel<T, false>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_experts_combine_kernel<T, true>, a);
}

int check_sizes(const char *who, int rows, int top_k, int hidden, int inter, int held) {
    if (rows < 0) return hy3a_fail(NULL, HY3A_EINVAL, "%s: rows %d < 0", who, rows);
    if (top_k < 1 || top_k > 32) return hy3a_fail(NULL, HY3A_EINVAL, "%s: top_k %d not in [1,32]", who, top_k);
    if (hidden < 8 || hidden % 8 || inter < 8 || inter % 8) return hy3a_fail(NULL, HY3A_EINVAL, "%s: hidden %d and inter %d have to be multiples of 8", who, hidden, inter);
    if (held < 1 || held > kMaxHeld) return hy3a_fail(NULL, HY3A_EINVAL, "%s: %d experts held, not in [1,%d]", who, held, kMaxHeld);
    if ((long long)rows * top_k > 0x7fffffffll / 2) return hy3a_fail(NULL, HY3A_EINVAL, "%s: %d rows of %d slots are too many", who, rows, top_k);
    return 0;
}

} /* namespace */

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
                     (int *)(b + w.off), (int *)(b + w.active), (int *)(b + w.row), (int *)(b + w.place), (expert_tile *)(b + w.tiles + 256), (int *)(b + w.tiles),
                     b + w.h, (float *)(b + w.y), (short *)(b + w.y), (float *)(b + w.scale)};
    const char *what = NULL;
    const cudaError_t e = dtype == HY3A_F16 ? launch<__half>(a, dev, sms, stream, &what) : launch<__nv_bfloat16>(a, dev, sms, stream, &what);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "experts: %s", what ? what : cudaGetErrorString(e));
    return HY3A_OK;
}

} /* extern "C" */

/*
 * logprobs.cu -- log probabilities of given tokens, entropy and the best alternatives of rows of logits (hy3a_logprobs).
 *
 *      log p_i = (l_i - m) - log Z,   Z = sum e^(l_i - m),   H = log Z + (sum e^(l_i - m) (m - l_i)) / Z,   m = max l
 *
 * in one pass, with running m.  The logits that equal m are counted (n) and the others' exponentials added up (S), so that log Z = log1p(S) where the largest stands
 * alone: a token that is nearly certain keeps the digits of its log probability.  The terms of H are all positive.
 *
 * A row is a block's, or the blocks' of a cluster where rows are few.  A warp shares m, so that it seldom rises: past the first vectors nearly all take the
 * branch without it.
 *
 * The top k are found without a second pass over the row: a thread keeps its largest logit and the vector of 16 bytes that had it; the k-th largest of 128
 * such keys, of four threads each, is no larger than the k-th largest logit; the few threads whose own key reaches it look through their vectors again, and the few logits
 * that reach it are ranked by (value, lowest index).  Rows with a NaN or an infinity, and rows where too many reach it, are searched k times instead.
 */
#include <math.h>

#include "layer.h"

namespace {

using namespace hy3a_layer;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxTopK = 32, kMaxVocab = 1 << 24, kMaxAsked = 1024, kMaxRows = 1 << 27, kList = 1024 /* logits that can be ranked */;
constexpr int kKeys = 128;                    /* groups of threads among whose largest logits the threshold is looked for */
constexpr float kLog2e = 1.4426950408889634f, kLowest = -3.402823466e38f;

struct logprobs_args {
    const void *logits;
    size_t stride;
    const int *tokens;
    float *asked_logp, *entropy, *top_logp;
    int *top_ids;
    int rows, vocab, asked, top_k, cluster;
};

__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void meet(int cluster) {
    if (cluster > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else __syncthreads();
}
__device__ __forceinline__ unsigned peer(const void *p, unsigned rank) {
    unsigned a = (unsigned)__cvta_generic_to_shared(p);
    asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(a) : "r"(rank));
    return a;
}
__device__ __forceinline__ float peer_float(const float *p, unsigned rank) { float v; asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer(p, rank)) : "memory"); return v; }
__device__ __forceinline__ float ex2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float warp_max(float v) { float r; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }      /* (not of NaN) */
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

/* What is kept of some logits: their maximum m, how many equal it, the sum of e^(l - m) of the others, and of e^(l - m) (m - l). */
struct part { float m, n, s, t; };
/* p seen from a maximum that is no smaller: n and s of the logits below it go to s */
__device__ __forceinline__ void raise(part &p, float m) {
    if (p.m == m) return;             /* (also: no logits on either side) */
    const float rise = fminf(m - p.m, 200.f), f = ex2(-rise * kLog2e), all = p.n + p.s;       /* (e^-200 is 0, and so is 0 times it) */
    p.t = p.m == -INFINITY ? p.t : f * fmaf(rise, all, p.t);         /* (where none was open, s and t are 0, or NaN) */
    p.s = p.m == -INFINITY ? p.s : f * all;
    p.n = 0.f;
    p.m = m;
}

/* Logits as vectors of 16 bytes, numbered from the boundary at or before the row's first: of the first and the last one only some values are the row's. */
template <class T> struct row_of {
    static constexpr int kOf = 16 / sizeof(T);
    const T *base;               /* the boundary */
    int skip, end;               /* the row's values are [skip, end) from there */
    int vectors;
    __device__ __forceinline__ row_of(const logprobs_args &a, int row) {
        const T *p = reinterpret_cast<const T *>(a.logits) + (size_t)row * a.stride;
        skip = (int)(((uintptr_t)p & 15) / sizeof(T));
        base = p - skip;
        end = skip + a.vocab;
        vectors = (end + kOf - 1) / kOf;
    }
    /* vector i, -inf in place of what is not the row's */
    __device__ __forceinline__ void load(int i, float (&v)[kOf]) const {
        if (i >= vectors || i < 0) {
#pragma unroll
            for (int j = 0; j < kOf; j++) v[j] = -INFINITY;
        } else if ((i == 0 && skip) || (i + 1) * kOf > end) {
#pragma unroll
            for (int j = 0; j < kOf; j++) v[j] = i * kOf + j >= skip && i * kOf + j < end ? type<T>::up(base[i * kOf + j]) : -INFINITY;
        } else {
            uint4 raw;
            asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w) : "l"(base + (size_t)i * kOf));
            const T *const r = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int j = 0; j < kOf; j++) v[j] = type<T>::up(r[j]);
        }
    }
};

/* order of floats as unsigned numbers, NaN below all but what is closed (0) */
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned u = __float_as_uint(isnan(v) ? kLowest : v + 0.f);       /* (-0 is 0) */
    return v == -INFINITY ? 0u : u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ unsigned long long key_of(float v, int i) { return (unsigned long long)ordered(v) << 32 | (0xffffffffu - (unsigned)i); }
__device__ __forceinline__ bool closed(unsigned long long key) { return (key >> 32) == 0; }

/* parts of two sets of logits as one's */
__device__ __forceinline__ void join(part &p, part q) {
    const float m = fmaxf(p.m, q.m);
    raise(p, m);
    raise(q, m);
    p.n += q.n; p.s += q.s; p.t += q.t;
}
__device__ __forceinline__ unsigned long long warp_max(unsigned long long key) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32) == hi ? (unsigned)key : 0u);
    return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ void order(unsigned long long &a, unsigned long long &b) { if (a < b) { const unsigned long long c = a; a = b; b = c; } }
/* the k-th largest of kKeys keys, 0 if fewer are open; one warp */
__device__ __forceinline__ unsigned long long kth_largest(const unsigned long long *keys, int k) {
    static_assert(kKeys == 128, "four keys a lane");
    const int lane = threadIdx.x & 31;
    unsigned long long q[4], most = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) q[j] = keys[lane + 32 * j];
    order(q[0], q[1]); order(q[2], q[3]); order(q[0], q[2]); order(q[1], q[3]); order(q[1], q[2]);
    for (int i = 0; i < k; i++) {
        most = warp_max(q[0]);
        if (closed(most)) return 0;
        if (q[0] == most) { q[0] = q[1]; q[1] = q[2]; q[2] = q[3]; q[3] = 0; }
    }
    return most;
}

template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads, 2) hy3a_logprobs_kernel(const logprobs_args a) {
    constexpr int kOf = row_of<T>::kOf, kAtOnce = 32 / kOf;        /* vectors of a thread that are on their way together */
    __shared__ part s_part[kWarps], s_all;
    __shared__ float s_max, s_log;
    __shared__ unsigned long long s_key[TOP ? kKeys : 1], s_threshold, s_list[TOP ? kList : 1];
    __shared__ unsigned s_listed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cluster = a.cluster, me = cluster > 1 ? (int)cluster_rank() : 0, row = blockIdx.x / cluster;
    pdl_release();
    pdl_wait();
    const row_of<T> r(a, row);
    const int per = (r.vectors + cluster - 1) / cluster, first = me * per, last = min(r.vectors, first + per);       /* the block's vectors */
    if (tid == 0) s_listed = 0;

    part p = {-INFINITY, 0.f, 0.f, 0.f};
    float best = -INFINITY;                /* the thread's largest logit, */
    int best_at = 0;                       /* and the first vector that has it */
    for (int i0 = first + warp * 32; i0 < last; i0 += kThreads * kAtOnce) {
        float v[kAtOnce][kOf];
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int i = i0 + u * kThreads + lane;
            r.load(i < last ? i : -1, v[u]);
        }
        float most = -INFINITY;
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            float vm = v[u][0];
#pragma unroll
            for (int j = 1; j < kOf; j++) vm = fmaxf(vm, v[u][j]);
            if (TOP && vm > best) { best = vm; best_at = i0 + u * kThreads + lane; }
            most = fmaxf(most, vm);
        }
        if (__any_sync(0xffffffffu, most >= p.m)) {
            const float m = warp_max(fmaxf(most, p.m));
            raise(p, m);
#pragma unroll
            for (int u = 0; u < kAtOnce; u++)
#pragma unroll
                for (int j = 0; j < kOf; j++) {
                    const float d = v[u][j] == -INFINITY ? -200.f : max_nan(v[u][j] - m, -200.f);
                    const float e = d == 0.f ? 0.f : ex2(d * kLog2e);
                    p.n += d == 0.f ? 1.f : 0.f;
                    p.s += e;
                    p.t = fmaf(e, -d, p.t);
                }
        } else {
#pragma unroll
            for (int u = 0; u < kAtOnce; u++)
#pragma unroll
                for (int j = 0; j < kOf; j++) {
                    const float d = max_nan(v[u][j] - p.m, -200.f);
                    const float e = ex2(d * kLog2e);
                    p.s += e;
                    p.t = fmaf(e, -d, p.t);
                }
        }
    }
    p.n = warp_sum(p.n); p.s = warp_sum(p.s); p.t = warp_sum(p.t);
    if (lane == 0) s_part[warp] = p;
    const unsigned long long mine = TOP ? key_of(best, best_at) : 0;        /* (here a key has the vector's number for the logit's) */
    if (TOP) {
        unsigned long long key = mine;
#pragma unroll
        for (int o = 1; o < kThreads / kKeys; o <<= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
            key = other > key ? other : key;
        }
        if (tid % (kThreads / kKeys) == 0) s_key[tid / (kThreads / kKeys)] = key;
    }
    __syncthreads();
    if (warp == 0) {
        part q = lane < kWarps ? s_part[lane] : part{-INFINITY, 0.f, 0.f, 0.f};
        raise(q, warp_max(q.m));
        q.n = warp_sum(q.n); q.s = warp_sum(q.s); q.t = warp_sum(q.t);
        if (lane == 0) s_all = q;
    } else if (TOP && warp == 1) {
        const unsigned long long key = kth_largest(s_key, a.top_k);
        if (lane == 0) s_threshold = key;
    }
    meet(cluster);
    if (TOP) {
        /* what each block is sure of, all may rely on */
        unsigned long long threshold = s_threshold;
        for (int c = 0; c < cluster; c++) {
            if (cluster == 1) break;
            unsigned long long other;
            asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(other) : "r"(peer(&s_threshold, c)) : "memory");
            threshold = other > threshold ? other : threshold;
        }
        if (!closed(mine) && mine >= threshold) {
            const unsigned count = peer(&s_listed, 0), list = peer(s_list, 0);
            for (int i0 = first + tid; i0 < last; i0 += kThreads * kAtOnce) {
                float v[kAtOnce][kOf];
#pragma unroll
                for (int u = 0; u < kAtOnce; u++) r.load(i0 + u * kThreads < last ? i0 + u * kThreads : -1, v[u]);
#pragma unroll
                for (int u = 0; u < kAtOnce; u++)
#pragma unroll
                    for (int j = 0; j < kOf; j++) {
                        const int i = i0 + u * kThreads;
                        if (v[u][j] == -INFINITY || key_of(v[u][j], i) < threshold) continue;
                        unsigned at;
                        asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(count) : "memory");
                        if (at < kList) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(list + 8 * at), "l"(key_of(v[u][j], i * kOf + j - r.skip)) : "memory");
                    }
            }
        }
    }
    if (me == 0 && tid == 0) {
        part q = s_all;
        for (int c = 1; c < cluster; c++) {
            const part o = {peer_float(&s_all.m, c), peer_float(&s_all.n, c), peer_float(&s_all.s, c), peer_float(&s_all.t, c)};
            join(q, o);
        }
        const bool none = q.m == -INFINITY && !isnan(q.s);             /* nothing is open */
        s_max = q.m;
        s_log = none ? 0.f : (q.n == 1.f ? log1pf(q.s) : logf(q.n + q.s));
        a.entropy[row] = none ? 0.f : s_log + q.t / (q.n + q.s);
    }
    meet(cluster);
    if (me != 0) return;

    const float m = s_max, log_all = s_log;
    /* (a closed logit has -inf, also where nothing is open, and NaN where the sum is one) */
    const auto logp = [&](float l) { return l == -INFINITY && !isnan(log_all) ? -INFINITY : (l - m) - log_all; };
    for (int j = tid; j < a.asked; j += kThreads) {
        const int token = a.tokens[(size_t)row * a.asked + j];
        float v = token == -1 ? 0.f : NAN;
        if (token >= 0 && token < a.vocab) v = logp(type<T>::up(reinterpret_cast<const T *>(a.logits)[(size_t)row * a.stride + token]));
        a.asked_logp[(size_t)row * a.asked + j] = v;
    }
    if (!TOP) return;
    int *const ids = a.top_ids + (size_t)row * a.top_k;
    float *const top = a.top_logp + (size_t)row * a.top_k;
    const auto put = [&](int rank, unsigned long long key) {
        const unsigned u = (unsigned)(key >> 32);
        ids[rank] = closed(key) ? -1 : (int)(0xffffffffu - (unsigned)key);
        top[rank] = closed(key) ? -INFINITY : logp(__uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u));
    };
    const unsigned n = s_listed;
    if (n <= kList && !isnan(log_all)) {
        for (unsigned i = tid; i < n; i += kThreads) {
            const unsigned long long key = s_list[i];
            int rank = 0;
            for (unsigned j = 0; j < n; j++) rank += s_list[j] > key;
            if (rank < a.top_k) put(rank, key);
        }
        for (int i = (int)n + tid; i < a.top_k; i += kThreads) put(i, 0);
        return;
    }
    unsigned long long before = ~0ull;
    for (int k = 0; k < a.top_k; k++) {
        unsigned long long most = 0;
        for (int i = tid; i < r.vectors; i += kThreads) {
            float v[kOf];
            r.load(i, v);
#pragma unroll
            for (int j = 0; j < kOf; j++) {
                const unsigned long long key = key_of(v[j], i * kOf + j - r.skip);
                if (!closed(key) && key < before && key > most) most = key;
            }
        }
        most = warp_max(most);
        __syncthreads();                     /* (the last round's have been read) */
        if (lane == 0) s_key[warp] = most;
        __syncthreads();
        before = warp_max(lane < kWarps ? s_key[lane] : 0);
        if (tid == 0) put(k, before);
        /* (once nothing is left, it stays so: no key is below 0) */
    }
}

template <class T>
cudaError_t launch(const logprobs_args &a, void *stream) {
    hy3a_launch l(dim3((unsigned)a.rows * a.cluster), dim3(kThreads), 0, stream);
    if (a.cluster > 1) l.cluster(a.cluster);
    return a.top_k ? cudaLaunchKernelEx(&l.cfg, hy3a_logprobs_kernel<T, true>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_logprobs_kernel<T, false>, a);
}

} /* namespace */

extern "C" int hy3a_logprobs(void *stream, int dtype, int rows, int vocab, const void *logits, size_t stride, const int *tokens, int asked, int top_k,
                             float *asked_logp, float *entropy, int *top_ids, float *top_logp) {
    if (dtype != HY3A_F32 && dtype != HY3A_F16 && dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "logprobs: dtype %d not in {0,1,2}", dtype);
    if (rows < 0 || rows > kMaxRows) return hy3a_fail(NULL, HY3A_EINVAL, "logprobs: rows %d not in [0,%d]", rows, kMaxRows);
    if (vocab < 1 || vocab > kMaxVocab) return hy3a_fail(NULL, HY3A_EINVAL, "logprobs: vocab %d not in [1,%d]", vocab, kMaxVocab);
    if (asked < 0 || asked > kMaxAsked) return hy3a_fail(NULL, HY3A_EINVAL, "logprobs: asked %d not in [0,%d]", asked, kMaxAsked);
    if (top_k < 0 || top_k > kMaxTopK || top_k > vocab) return hy3a_fail(NULL, HY3A_EINVAL, "logprobs: top_k %d not in [0,%d]", top_k, vocab < kMaxTopK ? vocab : kMaxTopK);
    if (rows == 0) return HY3A_OK;
    if (!logits || !entropy || (asked && (!tokens || !asked_logp)) || (top_k && (!top_ids || !top_logp))) return hy3a_fail(NULL, HY3A_EINVAL, "logprobs: NULL argument");
    const size_t el = dtype == HY3A_F32 ? 4 : 2;
    if (((uintptr_t)logits & (el - 1)) || (((uintptr_t)tokens | (uintptr_t)asked_logp | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_logp) & 3))
        return hy3a_fail(NULL, HY3A_EINVAL, "logprobs: a pointer is not aligned to its type");
    int dev, sms, rc = hy3a_layer_device("logprobs", &dev, &sms);
    if (rc) return rc;
    /* Blocks of a row: as many as fit on the device at once for all rows (two an SM), up to a portable cluster, and with a step of the loop for each at least. */
    int cluster = 8;
    while (cluster > 1 && ((long long)rows * cluster > 2 * sms || (size_t)vocab * el < (size_t)cluster * kThreads * 128)) cluster >>= 1;
    const logprobs_args a = {logits, stride, tokens, asked_logp, entropy, top_logp, top_ids, rows, vocab, asked, top_k, cluster};
    const cudaError_t e = dtype == HY3A_F32 ? launch<float>(a, stream) : (dtype == HY3A_F16 ? launch<__half>(a, stream) : launch<__nv_bfloat16>(a, stream));
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "logprobs: %s", cudaGetErrorString(e));
    return HY3A_OK;
}

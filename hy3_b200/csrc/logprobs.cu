/*
 * logprobs.cu -- log probabilities of given tokens, entropy and the best alternatives of rows of logits (hy3a_logprobs).
 *
 *      log p_i = (l_i - m) - log Z,   Z = sum e^(l_i - m),   H = log Z + (sum e^(l_i - m) (m - l_i)) / Z,   m = max l
 *
 * in one pass, with running m.  The logits that equal m are counted (n) and the others' exponentials added up (S), so that log Z = log1p(S) where the largest stands
 * alone: a token that is nearly certain keeps the digits of its log probability.  The terms of H are all positive.
 *
 * Memory bounds it where rows are many and long (2048 x 120832 fp32: 151 to 160 us, 6.2 to 6.5 TB/s; bf16 rows, 106 us, are bound by the exponentials and 10 instructions a pair of logits), the chain of loads, meetings and
 * ranking where they are few (1 x 120832, top 20: 7.3 to 7.8 us).  A row is a block's, or the blocks' of a cluster where rows are few.  A warp shares m, so that it seldom rises: past the first vectors nearly all take the
 * branch without it, and of those that raise it only the vectors that have the new m are looked at logit by logit.
 *
 * The top k are found without a second pass over the row: a thread keeps its largest logit and the vector of 16 bytes that had it; the k-th largest of 32
 * such keys, of the threads of a lane each, is no larger than the k-th largest logit; the vectors of the few threads whose own key reaches it are looked through again (the last
 * ones are still in registers), and the few logits that reach it are ranked by (value, lowest index).  Rows with a NaN or an infinity, and rows where too many reach
 * it, are searched k times instead.
 */
#include <math.h>

#include "layer.h"

namespace {

using namespace hy3a_layer;

/* Threads of a block: 64 where a row is a round or two of their loads, else four blocks an SM where there are more rows than SMs, so that one's end runs beside the others' loads; else one, and the blocks of a cluster for a row where rows
 * are fewer still: 131072 fp32 logits are one round of loads for 8 of them. */
constexpr int kSmall = 64, kAlone = 256, kShared = 512, kMaxCluster = 8;
constexpr int kMaxTopK = 32, kMaxVocab = 1 << 24, kMaxAsked = 1024, kMaxRows = 1 << 27, kList = 1024 /* logits that can be ranked */;
/* Up to this k the threshold is the k-th of the lanes' largest keys, above it of their two largest: the 32nd of 32 lets many through (4856 x 4362 fp32: 63 us with two, 78 with one; top 28 62 and 60, top 20 59 and 54) */
constexpr int kOneKey = 28;
constexpr float kLog2e = 1.4426950408889634f;

struct logprobs_args {
    const void *logits;
    size_t stride;
    const int *tokens;
    float *asked_logp, *entropy, *top_logp;
    int *top_ids;
    int rows, vocab, asked, top_k, cluster /* blocks of a row; 0: one by itself; -1: a small one */;
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
__device__ __forceinline__ float ex2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float warp_max(float v) { float r; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }      /* (not of NaN) */
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

/* What is kept of some logits: their maximum m, how many equal it, the sum of e^(l - m) of the others, and of e^(l - m) (m - l). */
struct __align__(16) part { float m, n, s, t; };
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
    __device__ __forceinline__ uint4 load(int i) const {
        constexpr unsigned kClosed = sizeof(T) == 4 ? 0xff800000u : (type<T>::code == HY3A_BF16 ? 0xff80ff80u : 0xfc00fc00u);
        uint4 raw = make_uint4(kClosed, kClosed, kClosed, kClosed);
        const int at = i * kOf;
        if (i >= 0 && at >= skip && at + kOf <= end)
            asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w) : "l"(base + at));
        else if (i >= 0 && at < end) {
            /* an edge, shifted in from above (rare: in few instructions) */
#pragma unroll 1
            for (int j = 0; j < kOf; j++) {
                unsigned v = kClosed;
                if (at + j >= skip && at + j < end) v = bits_of(base + at + j);
                const auto next = [](unsigned lo, unsigned hi) { return sizeof(T) == 4 ? hi : __funnelshift_r(lo, hi, 16); };
                raw = make_uint4(next(raw.x, raw.y), next(raw.y, raw.z), next(raw.z, raw.w), next(raw.w, v));
            }
        }
        return raw;
    }
    static __device__ __forceinline__ unsigned bits_of(const T *p) { return sizeof(T) == 4 ? *reinterpret_cast<const unsigned *>(p) : *reinterpret_cast<const unsigned short *>(p); }
};
/* the u-th of several vectors */
template <int N> __device__ __forceinline__ uint4 pick(const uint4 (&raw)[N], int u) {
    uint4 r = raw[0];
#pragma unroll
    for (int k = 1; k < N; k++) if (u == k) r = raw[k];
    return r;
}
/* a vector's logits, and the largest of them that is a number */
template <class T> __device__ __forceinline__ void logits_of(const uint4 &r, float (&v)[4]) { v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w); }
__device__ __forceinline__ float largest(const uint4 &r, float) { return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w))); }
template <class T> __device__ __forceinline__ void logits_of16(const uint4 &r, float (&v)[8]) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const unsigned short u[2] = {(unsigned short)w[i], (unsigned short)(w[i] >> 16)};
        v[2 * i] = type<T>::up(*reinterpret_cast<const T *>(&u[0]));
        v[2 * i + 1] = type<T>::up(*reinterpret_cast<const T *>(&u[1]));
    }
}
template <class T> __device__ __forceinline__ void logits_of(const uint4 &r, float (&v)[8]) { logits_of16<T>(r, v); }
__device__ __forceinline__ unsigned largest2(unsigned a, unsigned b, __nv_bfloat16) { unsigned r; asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ unsigned largest2(unsigned a, unsigned b, __half) { unsigned r; asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
template <class T> __device__ __forceinline__ float largest(const uint4 &r, T t) {
    const unsigned m = largest2(largest2(r.x, r.y, t), largest2(r.z, r.w, t), t);
    const unsigned short u[2] = {(unsigned short)m, (unsigned short)(m >> 16)};
    return fmaxf(type<T>::up(*reinterpret_cast<const T *>(&u[0])), type<T>::up(*reinterpret_cast<const T *>(&u[1])));
}

/* order of floats as unsigned numbers, NaN below all but what is closed (0) */
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned u = __float_as_uint(v + 0.f);       /* (-0 is 0) */
    return v == -INFINITY ? 0u : isnan(v) ? 1u /* a NaN seen from value_of too */ : u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ unsigned long long key_of(float v, int i) { return (unsigned long long)ordered(v) << 32 | (0xffffffffu - (unsigned)i); }
__device__ __forceinline__ float value_of(unsigned long long key) { const unsigned u = (unsigned)(key >> 32); return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
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
/* the k-th largest of the lanes' keys, 0 if fewer are open */
__device__ __forceinline__ unsigned long long kth_largest(unsigned long long key, int k) {
    int before = 0;
#pragma unroll
    for (int i = 1; i < 32; i++) before += __shfl_xor_sync(0xffffffffu, key, i) > key;
    const unsigned at = __ballot_sync(0xffffffffu, before == k - 1 && !closed(key));        /* (open keys differ) */
    return at ? __shfl_sync(0xffffffffu, key, __ffs(at) - 1) : 0;
}
/* the same of two keys a lane, `key` the larger */
__device__ __forceinline__ unsigned long long kth_largest(unsigned long long key, unsigned long long second, int k) {
    int before = 0, before2 = 1;
#pragma unroll 4
    for (int i = 1; i < 32; i++) {
        const unsigned long long a = __shfl_xor_sync(0xffffffffu, key, i), b = __shfl_xor_sync(0xffffffffu, second, i);
        before += (a > key) + (b > key);
        before2 += (a > second) + (b > second);
    }
    const unsigned at = __ballot_sync(0xffffffffu, before == k - 1 && !closed(key)), at2 = __ballot_sync(0xffffffffu, before2 == k - 1 && !closed(second));
    return at ? __shfl_sync(0xffffffffu, key, __ffs(at) - 1) : at2 ? __shfl_sync(0xffffffffu, second, __ffs(at2) - 1) : 0;
}
/* two numbers at a time */
struct f2 { float x, y; };
__device__ __forceinline__ unsigned long long bits(f2 v) { unsigned long long r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y)); return r; }
__device__ __forceinline__ f2 pair(unsigned long long v) { f2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { unsigned long long r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c))); return pair(r); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { unsigned long long r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b))); return pair(r); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { unsigned long long r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b))); return pair(r); }

/* a load that stays where it stands */
__device__ __forceinline__ float load_now(const float *p) { float v; asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p)); return v; }
template <class T> __device__ __forceinline__ T load_now(const T *p) { unsigned short v; asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p)); return *reinterpret_cast<T *>(&v); }

/* What a thread has of its logits so far; the sums in two halves. */
struct running {
    float m, n;
    f2 s, t;
    __device__ __forceinline__ part all() const { return {m, n, s.x + s.y, t.x + t.y}; }
    /* logits below m */
    template <int N> __device__ __forceinline__ void add_below(const float (&v)[N]) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            f2 d = fma2({v[j], v[j + 1]}, {-1.f, -1.f}, {m, m});
            d = {min_nan(d.x, 200.f), min_nan(d.y, 200.f)};         /* (e^-200 is 0, and so is 0 times it) */
            const f2 a = mul2(d, {-kLog2e, -kLog2e}), e = {ex2(a.x), ex2(a.y)};
            s = add2(s, e);
            t = fma2(e, d, t);
        }
    }
    /* logits up to m, -inf among them also where m is that */
    template <int N> __device__ __forceinline__ void add(const float (&v)[N]) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float d = v[j] == -INFINITY ? 200.f : min_nan(m - v[j], 200.f), e = d == 0.f ? 0.f : ex2(d * -kLog2e);
            n += d == 0.f ? 1.f : 0.f;
            s.x += e;
            t.x = fmaf(e, d, t.x);
        }
    }
};

template <class T, bool TOP, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == kShared ? 1 : 1024 / kThreads) hy3a_logprobs_kernel(const logprobs_args a) {
    constexpr int kWarps = kThreads / 32, kOf = row_of<T>::kOf, kAtOnce = 8;        /* vectors of a thread that are on their way together */
    constexpr bool kCluster = kThreads == kShared;
    __shared__ part s_part[kWarps], s_all[kMaxCluster];
    __shared__ float s_max, s_log;
    __shared__ unsigned long long s_key[TOP ? kThreads : 1], s_lanes[TOP && kCluster ? kMaxCluster : 1][32];
    __shared__ __align__(16) unsigned long long s_list[TOP ? kList : 2];
    __shared__ unsigned s_listed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cluster = kCluster ? a.cluster : 1, me = kCluster ? (int)cluster_rank() : 0, row = kCluster ? blockIdx.x / cluster : blockIdx.x;
    pdl_release();
    pdl_wait();
    const row_of<T> r(a, row);
    const int per = (r.vectors + cluster - 1) / cluster, first = me * per, last = min(r.vectors, first + per);       /* the block's vectors */
    if (tid == 0) s_listed = 0;
    if (kCluster) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

    int token = -1;           /* (loaded here, its logit behind the loop, both used at the end) */
    if (me == 0 && tid < a.asked) asm volatile("ld.global.s32 %0, [%1];" : "=r"(token) : "l"(a.tokens + (size_t)row * a.asked + tid));
    running p = {-INFINITY, 0.f, {0.f, 0.f}, {0.f, 0.f}};
    float best = -INFINITY;                /* the thread's largest logit, */
    int best_at = 0;                       /* and the first vector that has it */
    uint4 raw[kAtOnce];                    /* (the last ones stay) */
    int i0 = first + warp * 32;
    for (;; i0 += kThreads * kAtOnce) {
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int i = i0 + u * kThreads + lane;
            raw[u] = r.load(i < last ? i : -1);
        }
        /* vectors that there are, the same for a warp (small blocks alone look: rows of many vectors take 4 to 10% longer where each is asked for) */
        const int here = kThreads == kSmall ? (last - i0 + kThreads - 1) / kThreads : kAtOnce;
        float most = -INFINITY;
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            if (u >= here) break;
            const float vm = largest(raw[u], T());
            if (TOP && vm > best) { best = vm; best_at = i0 + u * kThreads + lane; }
            most = fmaxf(most, vm);
        }
        /* where m rises, the vectors that have it (or all, as long as nothing is open) are looked at logit by logit, one piece of code for all: code that is run once is fetched once */
        unsigned with_m = 0u;
        if (__any_sync(0xffffffffu, most >= p.m)) {
            part q = p.all();
            raise(q, warp_max(fmaxf(most, p.m)));
            p = {q.m, q.n, {q.s, 0.f}, {q.t, 0.f}};
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                if (u >= here) break;
                with_m |= __any_sync(0xffffffffu, largest(raw[u], T()) >= p.m || p.m == -INFINITY) ? 1u << u : 0u;
            }
            for (unsigned todo = with_m; todo; todo &= todo - 1) {
                float v[kOf];
                logits_of<T>(pick(raw, __ffs(todo) - 1), v);
                p.add(v);
            }
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            if (u >= here) break;
            if ((with_m >> u) & 1) continue;
            float v[kOf];
            logits_of<T>(raw[u], v);
            p.add_below(v);
        }
        if (i0 + kThreads * kAtOnce >= last) break;
    }
    const T *const logits = reinterpret_cast<const T *>(a.logits) + (size_t)row * a.stride;
    T token_logit = type<T>::down(0.f);
    if (me == 0 && token >= 0 && token < a.vocab) token_logit = load_now(logits + token);
    part q = p.all();
    q.n = warp_sum(q.n); q.s = warp_sum(q.s); q.t = warp_sum(q.t);
    if (lane == 0) s_part[warp] = q;
    if (TOP) s_key[tid] = key_of(best, best_at);        /* (here a key has the vector's number for the logit's) */
    __syncthreads();
    if (kCluster) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");              /* all blocks are there: they write to each other now */
    if (warp == 0) {
        q = lane < kWarps ? s_part[lane] : part{-INFINITY, 0.f, 0.f, 0.f};
        raise(q, warp_max(q.m));
        q.n = warp_sum(q.n); q.s = warp_sum(q.s); q.t = warp_sum(q.t);
        if (lane == 0) {
            if (kCluster) asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(peer(&s_all[me], 0)), "f"(q.m), "f"(q.n), "f"(q.s), "f"(q.t) : "memory");
            else s_all[0] = q;
        }
    } else if (TOP && warp == 1) {
        unsigned long long key = s_key[lane], second = 0;
#pragma unroll
        for (int w = 1; w < kWarps; w++) {
            const unsigned long long other = s_key[32 * w + lane], less = other > key ? key : other;
            if (!kCluster) second = less > second ? less : second;
            key = other > key ? other : key;
        }
        /* (the block's threshold, or what the cluster's blocks find it from each) */
        if (!kCluster) {
            key = a.top_k > kOneKey ? kth_largest(key, second, a.top_k) : kth_largest(key, a.top_k);
            if (lane == 0) s_lanes[0][0] = key;
        }
        else for (int c = 0; c < cluster; c++) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(peer(&s_lanes[me][lane], c)), "l"(key) : "memory");
    }
    meet(cluster);
    if (TOP) {
        /* the largest of each lane's threads, in all blocks; every warp finds the k-th of them (0: fewer are open) */
        unsigned long long key = s_lanes[0][kCluster ? lane : 0];
        if (kCluster) {
            for (int c = 1; c < cluster; c++) key = s_lanes[c][lane] > key ? s_lanes[c][lane] : key;
            key = kth_largest(key, a.top_k);
        }
        const float least = closed(key) ? -INFINITY : value_of(key);
        const int least_at = closed(key) ? -1 : (int)(0xffffffffu - (unsigned)key);
        const auto reaches = [&](float l, int i) { return l > least || (l == least && i <= least_at); };
        const bool mine = reaches(best, best_at);
        const unsigned who = __ballot_sync(0xffffffffu, mine), count = peer(&s_listed, 0), list = peer(s_list, 0);
        const auto take = [&](const uint4 &of, int vector) {
            float v[kOf];
            logits_of<T>(of, v);
#pragma unroll
            for (int j = 0; j < kOf; j++) {
                if (!reaches(v[j], vector)) continue;
                unsigned at;
                asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(count) : "memory");
                if (at < kList) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(list + 8 * at), "l"(key_of(v[j], vector * kOf + j - r.skip)) : "memory");
            }
        };
        /* The last round's vectors are still there; those of the rounds before are read again: by the thread, round after round, or by eight lanes for each, 64 vectors at a time, where that is fewer loads one
         * behind the other (403 rows of 115189 in fp32, top 1: 43.5 us, and 55.5 by threads alone). */
        const int from = first + warp * 32, rounds = (i0 - from) / (kThreads * kAtOnce), threads = __popc(who);
        const bool together = kThreads != kSmall && (threads + 3) / 4 * ((rounds + 7) / 8) < rounds;
        if (mine)
            for (int i = i0 + lane;;) {
                unsigned todo = 0u;
#pragma unroll
                for (int u = 0; u < kAtOnce; u++) todo |= reaches(largest(raw[u], T()), i + u * kThreads) ? 1u << u : 0u;
                for (; todo; todo &= todo - 1) take(pick(raw, __ffs(todo) - 1), i + (__ffs(todo) - 1) * kThreads);
                i -= kThreads * kAtOnce;
                if (together || i < first) break;
#pragma unroll
                for (int u = 0; u < kAtOnce; u++) raw[u] = r.load(i + u * kThreads);
            }
        if (together) {
            __syncwarp();
            if (mine) s_key[warp * 32 + __popc(who & ((1u << lane) - 1u))] = lane;
            __syncwarp();
#pragma unroll 1
            for (int c = lane >> 3; c < threads; c += 4) {
                const int at = from + (int)s_key[warp * 32 + c];
#pragma unroll 1
                for (int n = lane & 7; n < rounds * kAtOnce; n += 8 * kAtOnce) {
                    unsigned todo = 0u;
#pragma unroll
                    for (int u = 0; u < kAtOnce; u++) raw[u] = r.load(n + 8 * u < rounds * kAtOnce ? at + (n + 8 * u) * kThreads : -1);
#pragma unroll
                    for (int u = 0; u < kAtOnce; u++) todo |= reaches(largest(raw[u], T()), at + (n + 8 * u) * kThreads) ? 1u << u : 0u;
                    for (; todo; todo &= todo - 1) take(pick(raw, __ffs(todo) - 1), at + (n + 8 * (__ffs(todo) - 1)) * kThreads);
                }
            }
        }
    }
    if (me == 0 && tid == 0) {
        q = s_all[0];
        for (int c = 1; c < cluster; c++) join(q, s_all[c]);
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
        if (j != tid) {
            token = a.tokens[(size_t)row * a.asked + j];
            if (token >= 0 && token < a.vocab) token_logit = logits[token];
        }
        a.asked_logp[(size_t)row * a.asked + j] = token >= 0 && token < a.vocab ? logp(type<T>::up(token_logit)) : (token == -1 ? 0.f : NAN);
    }
    if (!TOP) return;
    int *const ids = a.top_ids + (size_t)row * a.top_k;
    float *const top = a.top_logp + (size_t)row * a.top_k;
    const auto put = [&](int at, unsigned long long key) {
        ids[at] = closed(key) ? -1 : (int)(0xffffffffu - (unsigned)key);
        top[at] = closed(key) ? -INFINITY : logp(value_of(key));
    };
    const unsigned n = s_listed;
    if (n <= kList && !isnan(log_all)) {
        for (unsigned i = tid; i < n; i += kThreads) {
            const unsigned long long key = s_list[i];
            int rank = 0;
            unsigned j = 0;
            for (; j + 4 <= n; j += 4) {
                const ulonglong2 p = *reinterpret_cast<const ulonglong2 *>(s_list + j), q = *reinterpret_cast<const ulonglong2 *>(s_list + j + 2);
                rank += (p.x > key) + (p.y > key) + (q.x > key) + (q.y > key);
            }
            for (; j < n; j++) rank += s_list[j] > key;
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
            logits_of<T>(r.load(i), v);
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

template <class T, int kThreads>
cudaError_t launch(const logprobs_args &a, void *stream) {
    hy3a_launch l(dim3((unsigned)a.rows * (kThreads == kShared ? a.cluster : 1)), dim3(kThreads), 0, stream);
    if (kThreads == kShared) l.cluster(a.cluster);
    return a.top_k ? cudaLaunchKernelEx(&l.cfg, hy3a_logprobs_kernel<T, true, kThreads>, a) : cudaLaunchKernelEx(&l.cfg, hy3a_logprobs_kernel<T, false, kThreads>, a);
}
template <class T>
cudaError_t launch_type(const logprobs_args &a, void *stream) { return a.cluster < 0 ? launch<T, kSmall>(a, stream) : (a.cluster ? launch<T, kShared>(a, stream) : launch<T, kAlone>(a, stream)); }

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
    /* Blocks of a row: none but one where there are more rows than SMs; else as many as fit on the device at once for all rows, up to a portable cluster, and with half a round of
     * loads for each at least. */
    int cluster = rows > sms ? 0 : kMaxCluster;
    /* Rows of one round of a small block's loads are its; of two rounds, where there are more rows than larger blocks fit at once (6171 rows of 2514 in bf16: 16.6 us and 52, 2692 of 5216 in fp16 26.7 and
     * 40; 300 rows of 4000 in fp32 8.1 and 7.4). */
    if ((long long)vocab * el <= (rows > sms * (1024 / kAlone) ? 2 : 1) * kSmall * 128) cluster = -1;
    while (cluster > 1 && (rows * cluster > sms || vocab < cluster * kShared * 16)) cluster >>= 1;
    const logprobs_args a = {logits, stride, tokens, asked_logp, entropy, top_logp, top_ids, rows, vocab, asked, top_k, cluster};
    const cudaError_t e = dtype == HY3A_F32 ? launch_type<float>(a, stream) : (dtype == HY3A_F16 ? launch_type<__half>(a, stream) : launch_type<__nv_bfloat16>(a, stream));
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "logprobs: %s", cudaGetErrorString(e));
    return HY3A_OK;
}

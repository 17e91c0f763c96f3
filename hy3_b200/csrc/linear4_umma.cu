/*
 * linear4_umma.cu -- rows through a matrix in 4 bits, many rows: on 5th-generation tensor cores (tcgen05 + TMEM + TMA).
 *
 * The weights are the M side of the product and the rows its N side (up to 256).  A pair of CTAs (cta_group::2) works on 256 outputs: each has 128 of them, and half of the
 * rows of x in shared memory.  Codes become weights on their way: a thread has an output, reads its codes of 64 k's from shared memory, and stores (code - 8) * scale
 * as the A operand into tensor memory, from where the product takes it; shared memory sees 4 bits a weight, and the tensor cores read only x from there.  Per CTA:
 *   16 warps   weights: each four of them (a lane quarter each) every fourth step of 64 k's; afterwards the results.  fp32 results: 12, every third step, and
 *              8 that add up sums;
 *   2          TMA producers: codes, 128 k's at a time, and x, 64 k's at a time;
 *   1          MMA issuer (of the leader): 4 x tcgen05.mma (K = 16) a step, fp32 results 8.
 *
 * Results of the rows' type: a weight, of up to 15 bits (fp16) or 11 (bf16), is rounded to that type once, which leaves an error like the result's own rounding.  Results that are not finite (of weights
 * rounded beyond the type's largest, of an infinite x that meets the rest) are computed again from the definition, by the warp that finds them, at a time when no bounded wait depends on it.
 *
 * Results in fp32: a weight enters as two numbers, the rounded one and the rest, which is exact, so that there are 8 products a step; and the tensor cores begin a new sum every 512 k's (bf16; fp16: 256), which warps of their own
 * add to results in registers: the tensor cores' sums are cut off and not rounded (one sum over 4096 k's left an error of 5.6e-6 of the result; sums of 512 leave 4.6e-7, of fp16 products, whose 22 bits lose more,
 * 1.1e-6, of 256 k's 6e-7 for 2% more time).  A = code - 8, with a sum for each group and its scale
 * at the end, is half as many products and rounds nothing, but reads sums 8 times as often: 64 rows on 10240 x 4096 took 26.8 us in an early form of this file, which had one tile a pair, and 26.4 as it is now; it has not been tried since.
 *
 * Where tiles are more than pairs of CTAs fit at once, a pair has several, and its warps go on to the next one each as far as it can.
 * Where tiles are few, the CTAs of a cluster share the k's of a tile; their sums meet in shared memory, and are added in the order of the k's.
 *
 * Every wait is bounded; one that runs out raises the CTA's abort flag and a code in the error word (hy3a_layer_sync), lets all warps fall through, and TMEM is always
 * released.
 */
#include <atomic>
#include <type_traits>

#include "linear4.h"
#include "linear4_plan.h"
#include "ring.cuh"

namespace {

using namespace hy3a_layer;
using namespace hy3a_ring;

constexpr int kUnit = 128 /* k's of a copy of codes */, kUnits = kLinear4Units /* in the ring */, kUnitBytes = 128 * kUnit / 2, kStepBytes = 128 * 128 /* x of 64 k's, at most 128 rows a CTA */;
constexpr int kMostSplits = kLinear4Splits, kMostSteps = kLinear4Steps, kXBytes = kLinear4XBytes, kOffX = kUnits * kUnitBytes, kOffBar = kOffX + kXBytes, kSmem = kOffBar + 512 + 1024;
enum { B_CODES = 0, B_CODES_FREE = kUnits, B_STEP = 2 * kUnits /* x and A of a step are there */, B_FREE = 2 * kUnits + kMostSteps, B_SUMS = 2 * kUnits + 2 * kMostSteps, B_RUN, B_RUN_FREE = B_RUN + 2, B_COUNT = B_RUN_FREE + 2 };
static_assert(8 * B_COUNT + 16 <= 512, "barriers");
static_assert(kXBytes == 8 * kStepBytes, "stages of 256 rows");
static_assert(128 * 256 * 4 <= kOffBar, "sums of a tile");

__device__ unsigned g_err[2];         /* {code, where} of the first wait that ran out, until hy3a_layer_sync reads it */

struct many_args {
    linear4_args a;
    int odd_out /* pairs of 16-bit results do not lie on 4-byte boundaries */, columns /* rows of a tile, a multiple of 32 */, m_tiles, tiles, units /* of 128 k's */, splits, steps /* stages of x and A */, a_column /* where those of A begin in tensor memory; the sums lie before, for fp32 results two of them */;
};

__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned cluster_addr(unsigned addr, unsigned rank) {
    unsigned r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
/* Relaxed: what it tells of lies in tensor memory, is waited for (tcgen05.wait::st) and ordered by tcgen05.fence::before_thread_sync.  A release in the cluster's scope would
 * wait for all else that the warp has under way, the scales asked for ahead among it (64 rows on 10240 x 4096: 49 us). */
__device__ __forceinline__ void mbar_arrive_cluster(unsigned bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void tma_codes(unsigned dst, const CUtensorMap *map, unsigned bar, int x, int y, unsigned long long policy, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %6, 0;\n"
                 " @e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;\n}"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "l"(policy), "r"(lead) : "memory");
}
__device__ __forceinline__ void tma_rows(unsigned dst, const CUtensorMap *map, unsigned bar, int x, int y, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %5, 0;\n"
                 " @e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];\n}"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(lead) : "memory");
}
/* K-major operand, 128-byte swizzle: 8-row groups 1024 B apart, descriptor version 1, layout 2 */
__device__ __forceinline__ unsigned long long make_desc(unsigned saddr) {
    return (unsigned long long)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
/* A in tensor memory */
__device__ __forceinline__ void umma_lead(unsigned d, unsigned a, unsigned long long b, unsigned idesc, unsigned accumulate, unsigned lead) {
    asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 e, %5, 0;\n setp.ne.b32 p, %4, 0;\n @e tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void umma_commit_lead(unsigned bar, unsigned short ctas, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n @e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n}"
                 ::"r"(bar), "r"(lead), "h"(ctas) : "memory");
}
__device__ __forceinline__ void tmem_st32(unsigned taddr, const unsigned (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
/* A wait's answer takes 100 clocks and more, also where nothing is waited for: the issuer looks at its barriers ahead of time, and waits only if that did not show them through.  What all_wait tells is the same
 * for all lanes, and the compiler knows (where it does not, each product that the warp issues behind it costs 100 clocks). */
__device__ __forceinline__ unsigned peek(unsigned bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
__device__ __forceinline__ bool all_wait(unsigned seen, unsigned bar, unsigned parity, volatile int *abort_flag, unsigned where) {
    return __all_sync(0xffffffffu, seen) || warp_wait(bar, parity, abort_flag, g_err, where);
}
template <class T> struct pair_of;
template <> struct pair_of<__nv_bfloat16> {
    static __device__ __forceinline__ unsigned mul(unsigned a, unsigned b) { unsigned r; asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ unsigned rest(unsigned a, unsigned b, unsigned hi) { unsigned r; asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(hi ^ 0x80008000u)); return r; }
};
template <> struct pair_of<__half> {
    static __device__ __forceinline__ unsigned mul(unsigned a, unsigned b) { unsigned r; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ unsigned rest(unsigned a, unsigned b, unsigned hi) { unsigned r; asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(hi ^ 0x80008000u)); return r; }
};

/* What is not finite among a lane's results y of output o and rows t, t + 1, .. t + n - 1 is NaN if x has one in its row (padding that nobody wrote may be such rows), and else computed again, by the whole
 * warp (rare: one piece of code, not unrolled) */
template <class T, int N> __device__ __forceinline__ void settle(const linear4_args &a, float (&y)[N], int n, int t, int o, bool mine) {
    bool odd = false;
#pragma unroll
    for (int j = 0; j < N; j++) odd |= j < n && !(fabsf(y[j]) < INFINITY);
    if (!__any_sync(0xffffffffu, odd && mine)) return;
#pragma unroll 1
    for (int j = 0; j < n; j++) {
        float now = y[0];
#pragma unroll
        for (int k = 1; k < N; k++) if (j == k) now = y[k];
        unsigned todo = __ballot_sync(0xffffffffu, mine && !(fabsf(now) < INFINITY));
        if (!todo) continue;
        if (has_nan<T>(a, t + j)) {
            if (!(fabsf(now) < INFINITY)) now = NAN;
            todo = 0u;
        }
#pragma unroll 1
        for (; todo; todo &= todo - 1) {
            const int l = __ffs(todo) - 1;
            const float again = plain<T>(a, t + j, __shfl_sync(0xffffffffu, o, l));
            if ((int)(threadIdx.x & 31) == l) now = again;
        }
#pragma unroll
        for (int k = 0; k < N; k++) if (j == k) y[k] = now;
    }
}
/* the same of results of type O that the warp has stored: rows t + c0 .. t + c0 + 15 of a tile's n, and those `step` further on and so forth.  Settling takes as long as it takes (up to a tenth of a second for a
 * tile of 256 rows of 65536): where a pair has several tiles, it comes when nothing in the pair waits for the warp any more, as waits are bounded. */
template <class T, class O> __device__ __noinline__ void settle_stored(const linear4_args &a, int t, int n, int c0, int step, int o, bool mine) {
#pragma unroll 1
    for (int c = c0; c < n; c += step) {
        O *const at = reinterpret_cast<O *>(a.out) + (size_t)(t + c) * a.out_stride + o;
        float y[16];
        unsigned odd = 0u;
#pragma unroll
        for (int j = 0; j < 16; j++) y[j] = mine && c + j < n ? type<O>::up(at[j * a.out_stride]) : 0.f;
#pragma unroll
        for (int j = 0; j < 16; j++) odd |= fabsf(y[j]) < INFINITY ? 0u : 1u << j;
        settle<T>(a, y, min(16, n - c), t + c, o, mine);
#pragma unroll
        for (int j = 0; j < 16; j++) if (odd >> j & 1) at[j * a.out_stride] = type<O>::down(y[j]);
    }
}
/* A lane's results of its output, row after row.  16-bit ones: neighbouring lanes exchange, so that one stores the even rows' two outputs and one the odd rows'. */
template <class T, bool WIDE, int N> __device__ __forceinline__ void store(const linear4_args &a, const float (&y)[N], int n, int t, int o, int odd_stride) {
    const bool mine = o < a.out_width;
    if (WIDE) {
#pragma unroll
        for (int j = 0; j < N; j++) if (j < n && mine) reinterpret_cast<float *>(a.out)[(size_t)(t + j) * a.out_stride + o] = y[j];
    } else if (odd_stride) {
#pragma unroll
        for (int j = 0; j < N; j++) if (j < n && mine) reinterpret_cast<T *>(a.out)[(size_t)(t + j) * a.out_stride + o] = type<T>::down(y[j]);
    } else {
        const int lane = threadIdx.x & 31, side = lane & 1;
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, side ? y[j] : y[j + 1], 1);
            T two[2] = {type<T>::down(side ? other : y[j]), type<T>::down(side ? y[j + 1] : other)};
            if (j + side < n && mine) *reinterpret_cast<unsigned *>(reinterpret_cast<T *>(a.out) + (size_t)(t + j + side) * a.out_stride + o - side) = *reinterpret_cast<const unsigned *>(two);
        }
    }
}

/* The warps of a CTA: teams of four that make A (a warp for each 32 outputs), those that add up groups, two producers, the issuer. */
template <bool WIDE> struct warps_of {
    static constexpr int kTeams = linear4_teams(WIDE), kAdders = WIDE ? 8 : 0, kWorkers = 4 * kTeams + kAdders, kCodes = kWorkers, kRowsOfX = kWorkers + 1, kIssuer = kWorkers + 2, kThreads = 32 * (kWorkers + 3);
};

/* WIDE: the result is fp32.  PER: scales of 64 k's (groups of 32: two).  MANY: more tiles than clusters, each cluster's one behind the other (then a cluster is a pair) */
template <class T, bool WIDE, int PER, bool MANY>
__global__ void __launch_bounds__(warps_of<WIDE>::kThreads, 1) hy3a_linear4_umma_kernel(const __grid_constant__ CUtensorMap tm_codes, const __grid_constant__ CUtensorMap tm_x, const many_args f) {
    extern __shared__ uint8_t s_raw[];
    using W = warps_of<WIDE>;
    constexpr int kAWide = WIDE ? 64 : 32 /* columns of a stage of A */, kTeams = W::kTeams, kCodes = W::kCodes, kRowsOfX = W::kRowsOfX, kIssuer = W::kIssuer, kRun = type<T>::code == HY3A_BF16 ? 8 : 4 /* WIDE: steps of a sum */;
    const int n_steps = f.steps;
    const unsigned x_bytes = f.columns * 64;          /* half the rows of 64 k's, a multiple of 1024 */
    const linear4_args &a = f.a;
    uint8_t *sm = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    const unsigned sbase = smem_u32(sm), bar0 = sbase + kOffBar;
    volatile unsigned *s_tmem = reinterpret_cast<volatile unsigned *>(sm + kOffBar + 8 * B_COUNT);
    volatile int *s_abort = reinterpret_cast<volatile int *>(sm + kOffBar + 8 * B_COUNT + 4);
#define BAR(i) (bar0 + 8u * (unsigned)(i))
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0) /* uniform for the compiler too */, lane = tid & 31;
    const unsigned me = cluster_rank(), leader = me & ~1u, rank = me & 1u;
    const int split = me >> 1, clusters = gridDim.x / 2, tile0 = blockIdx.x / (2 * f.splits);        /* MANY: a pair's tiles are tile0, tile0 + clusters, .. */
    const int u0 = (int)((long long)f.units * split / f.splits), u1 = (int)((long long)f.units * (split + 1) / f.splits), steps = 2 * (u1 - u0);
    const int N = f.columns, end = MANY ? f.tiles : tile0 + 1;
    const int m_first = tile0 % f.m_tiles * 256 + (int)rank * 128, row_first = tile0 / f.m_tiles * N;
    const auto m_of = [&](int tile) { return MANY && tile != tile0 ? tile % f.m_tiles * 256 + (int)rank * 128 : m_first; };        /* the tile's first output here, and its first row */
    const auto row_of = [&](int tile) { return MANY && tile != tile0 ? tile / f.m_tiles * N : row_first; };

    if (tid == 0) {
        *s_abort = 0;
        for (int i = 0; i < kUnits; i++) { mbar_init(BAR(B_CODES + i), 1); mbar_init(BAR(B_CODES_FREE + i), 8 /* two teams */); }
        for (int i = 0; i < n_steps; i++) { mbar_init(BAR(B_STEP + i), 9 /* a team of each CTA, and the bytes of x */); mbar_init(BAR(B_FREE + i), 1); }
        mbar_init(BAR(B_SUMS), 1);
        for (int i = 0; i < 2; i++) { mbar_init(BAR(B_RUN + i), 1); mbar_init(BAR(B_RUN_FREE + i), WIDE ? 16 : 32 /* those warps of each CTA that read sums */); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kCodes && lane < 2) {
        const CUtensorMap *m = lane == 0 ? &tm_codes : &tm_x;
        asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar0 + 8u * B_COUNT), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = *s_tmem;
    pdl_release();
    pdl_wait();

    /* a lane's sums of output o and the n rows from c0 on: stored, or left in shared memory where other CTAs have more of them */
    const auto put = [&](float (&y)[16], int c0, int n, int r, int o, int row0) {
        if (!MANY && f.splits > 1) {
#pragma unroll
            for (int j = 0; j < 16; j++) if (j < n) *reinterpret_cast<float *>(sm + ((c0 + j) * 128 + r) * 4) = y[j];
        } else {
            if (!MANY) settle<T>(a, y, n, row0 + c0, o, o < a.out_width);
            store<T, WIDE>(a, y, n, row0 + c0, o, f.odd_out);
        }
    };
    /* MANY: what a warp found not finite, if anything, once it has stored all of its results; odd: a bit for each tile that has some, the last one for all from the 32nd on */
    const auto settle_all = [&](unsigned odd, int c0, int step, int r) {
        odd = __reduce_or_sync(0xffffffffu, odd);
        if (!odd) return;
        __syncwarp();                /* (neighbours have stored for each other) */
#pragma unroll 1
        for (int tile = tile0, turn = 0; tile < end; tile += clusters, turn++)
            if (odd >> min(turn, 31) & 1) settle_stored<T, typename std::conditional<WIDE, float, T>::type>(a, row_of(tile), min(N, a.rows - row_of(tile)), c0, step, m_of(tile) + r, m_of(tile) + r < a.out_width);
    };
    if (warp == kCodes) {
        /* ===================== producer of codes ===================== */
        const unsigned lead = elect_one();
        unsigned long long policy;
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        int unit = 0;
        unsigned ph = 0;
        bool ok = true;
        for (int tile = tile0; tile < end && ok; tile = MANY ? tile + clusters : end) {
            const int m0 = m_of(tile);
#pragma unroll 1
            for (int u = u0; u < u1; u++) {
                if (!(ok = warp_wait(BAR(B_CODES_FREE + unit), ph ^ 1u, s_abort, g_err, 50u))) break;
                if (lead) mbar_expect_tx(BAR(B_CODES + unit), kUnitBytes);
                tma_codes(sbase + unit * kUnitBytes, &tm_codes, BAR(B_CODES + unit), u * (kUnit / 2), m0, policy, lead);
                if (++unit == kUnits) { unit = 0; ph ^= 1u; }
            }
        }
    } else if (warp == kRowsOfX) {
        /* ===================== producer of x ===================== */
        const unsigned lead = elect_one();
        int st = 0;
        unsigned ph = 0;
        bool ok = true;
        for (int tile = tile0; tile < end && ok; tile = MANY ? tile + clusters : end) {
            const int first = row_of(tile) + (int)rank * (N >> 1);
#pragma unroll 1
            for (int s = 0; s < steps; s++) {
                if (!(ok = warp_wait(BAR(B_FREE + st), ph ^ 1u, s_abort, g_err, 51u))) break;
                if (lead && rank == 0) mbar_expect_tx(BAR(B_STEP + st), N * 128);
                tma_rows(sbase + kOffX + st * x_bytes, &tm_x, cluster_addr(BAR(B_STEP + st), leader), u0 * kUnit + s * 64, first, lead);
                if (++st == n_steps) { st = 0; ph ^= 1u; }
            }
        }
        /* the last commits reach the barriers of both CTAs before either leaves */
        for (int i = 0; i < n_steps; i++) {
            if (!warp_wait(BAR(B_FREE + st), ph ^ 1u, s_abort, g_err, 52u)) break;
            if (++st == n_steps) { st = 0; ph ^= 1u; }
        }
    } else if (warp == kIssuer) {
        if (rank == 0) {
            /* ===================== MMA issuer: uniform control flow, one elected lane issues ===================== */
            const unsigned lead = elect_one();
            constexpr unsigned kType = type<T>::code == HY3A_BF16 ? (1u << 7) | (1u << 10) : 0u;
            const unsigned idesc = (1u << 4) | kType | (((unsigned)N >> 3) << 17) | ((256u >> 4) << 24);
            const unsigned short both = (unsigned short)(3u << leader);
            int st = 0, buf = 0;
            unsigned ph = 0, rph = 0, seen = 0;
            bool ok = true;
            int turn = 0;
            for (int tile = tile0; tile < end && ok; tile = MANY ? tile + clusters : end, turn++) {
            /* (the sums of the tile before have been read) */
            if (MANY && !WIDE && turn && !(ok = all_wait(0, BAR(B_RUN_FREE), (turn - 1) & 1, s_abort, 58u))) break;
            for (int s = 0; s < steps; s++) {
                if (!(ok = all_wait(seen, BAR(B_STEP + st), ph, s_abort, 53u))) break;
                const int next = st + 1 == n_steps ? 0 : st + 1;
                const unsigned next_ph = next ? ph : ph ^ 1u;
                seen = peek(BAR(B_STEP + next), next_ph);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned long long db = make_desc(sbase + kOffX + st * x_bytes);
                const unsigned da = tmem + f.a_column + st * kAWide;
                const bool begins = WIDE ? s % kRun == 0 : s == 0;
                if (WIDE && begins) {
                    if (!(ok = all_wait(0, BAR(B_RUN_FREE + buf), rph ^ 1u, s_abort, 59u))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                const unsigned d = tmem + (WIDE ? buf * N : 0);
#pragma unroll
                for (int k = 0; k < 4; k++) umma_lead(d, da + 8 * k, db + 2 * k, idesc, !begins || k > 0, lead);
                if (WIDE) {
#pragma unroll
                    for (int k = 0; k < 4; k++) umma_lead(d, da + 32 + 8 * k, db + 2 * k, idesc, 1, lead);
                    if (s % kRun == kRun - 1 || s == steps - 1) {
                        umma_commit_lead(BAR(B_RUN + buf), both, lead);
                        if (++buf == 2) { buf = 0; rph ^= 1u; }
                    }
                }
                umma_commit_lead(BAR(B_FREE + st), both, lead);
                st = next;
                ph = next_ph;
            }
            if (!WIDE && ok) umma_commit_lead(BAR(B_SUMS), both, lead);
            }
        }
    } else if (WIDE && warp >= 4 * kTeams) {
        /* ===================== sums of kRun steps: a lane has an output, the warp every other 16 rows ===================== */
        const int quarter = warp & 3, half = (warp >> 2) & 1, r = quarter * 32 + lane, runs = (steps + kRun - 1) / kRun;
        float acc[4][16];
        bool ok = true;
        unsigned odd = 0u, now = 1u;         /* bits of the tiles that have results that are not finite, and of this one */
        int buf = 0;
        unsigned rph = 0;
#pragma unroll 1
        for (int tile = tile0; tile < end && ok; tile = MANY ? tile + clusters : end) {
            const int row0 = row_of(tile), rows = min(N, a.rows - row0), o = m_of(tile) + r;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int k = 0; k < 16; k++) acc[i][k] = 0.f;
#pragma unroll 1
            for (int run = 0; run < runs; run++) {
                if (!(ok = warp_wait(BAR(B_RUN + buf), rph, s_abort, g_err, 60u))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int c0 = (2 * i + half) * 16;
                    if (c0 >= N) break;
                    unsigned v[16];
                    tmem_ld16(tmem + ((unsigned)(quarter * 32) << 16) + buf * N + c0, v);
#pragma unroll
                    for (int k = 0; k < 16; k++) acc[i][k] += __uint_as_float(v[k]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(cluster_addr(BAR(B_RUN_FREE + buf), leader));
                if (++buf == 2) { buf = 0; rph ^= 1u; }
            }
            if (!ok) break;
            if (!MANY) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int c0 = (2 * i + half) * 16;
#pragma unroll
                    for (int k = 0; k < 16; k++) if (c0 + k < rows) *reinterpret_cast<float *>(sm + ((c0 + k) * 128 + r) * 4) = acc[i][k];
                }
            } else {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    /* (code that is run once a tile: short) */
                    const int c0 = (2 * i + half) * 16, n = o < a.out_width ? rows - c0 : 0;
                    if (c0 >= rows) break;
                    float *to = reinterpret_cast<float *>(a.out) + (size_t)(row0 + c0) * a.out_stride + o;
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        sum = fmaf(acc[i][k], 0.f, sum);
                        if (k < n) *to = acc[i][k];
                        to += a.out_stride;
                    }
                }
                odd |= sum == 0.f ? 0u : now;
                now = now << 1 ? now << 1 : now;
            }
        }
        if (MANY && ok) settle_all(odd, half * 16, 32, r);
    } else {
        /* ===================== weights: a thread has an output; each team takes every third or fourth step, from tile to tile too ===================== */
        const int quarter = warp & 3, team = warp >> 2, r = quarter * 32 + lane;
        const unsigned short *scales = nullptr;
        const int shift = a.group == 128 ? 7 : (a.group == 64 ? 6 : 5);
        const unsigned to_a = tmem + f.a_column + ((unsigned)(quarter * 32) << 16), from = sbase + r * (kUnit / 2), turn = (unsigned)((r >> 1) & 3);
        unsigned short sc[3][PER];
        const auto fetch = [&](int s, unsigned short (&to)[PER]) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int j = (u0 * kUnit + s * 64 + 32 * i) >> shift;
                to[i] = 0;
                if (s < steps && j < a.groups) to[i] = scales[j];
            }
        };
        static_assert(kTeams + kMostSteps <= 2 * kUnits, "phases of the codes that a team does not wait for");
        int st = team, s0 = team /* the team's first step of the tile */, behind = 0;         /* units of the tiles before */
        unsigned ph = 0;
        const auto step = [&](int s, const unsigned short (&now)[PER], unsigned short (&ahead)[PER]) {
            fetch(s + 2 * kTeams, ahead);
            const int unit = (behind + (s >> 1)) % kUnits;
            if (!warp_wait(BAR(B_CODES + unit), (behind + (s >> 1)) / kUnits & 1, s_abort, g_err, 55u)) return false;
            uint4 c[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const unsigned at = from + unit * kUnitBytes + (((unsigned)((s & 1) * 2 + i) ^ turn) << 4);
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(c[i].x), "=r"(c[i].y), "=r"(c[i].z), "=r"(c[i].w) : "r"(at));
            }
            const unsigned w[8] = {c[0].x, c[0].y, c[0].z, c[0].w, c[1].x, c[1].y, c[1].z, c[1].w};
            unsigned weights[32], rest[WIDE ? 32 : 1];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                unsigned n[4];
                hy3a_layer::steps<T>::in_order(w[i], n);
                const unsigned s2 = __byte_perm(now[i * PER / 8], 0, 0x1010);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    weights[4 * i + j] = pair_of<T>::mul(n[j], s2);
                    if (WIDE) rest[WIDE ? 4 * i + j : 0] = pair_of<T>::rest(n[j], s2, weights[4 * i + j]);
                }
            }
            if (!warp_wait(BAR(B_FREE + st), ph ^ 1u, s_abort, g_err, 56u)) return false;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            tmem_st32(to_a + st * kAWide, weights);
            if constexpr (WIDE) tmem_st32(to_a + st * kAWide + 32, rest);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            /* (the codes are given back behind a store that needed them: an arrival does not wait for loads that are under way) */
            if (lane == 0) { mbar_arrive_cluster(cluster_addr(BAR(B_STEP + st), leader)); mbar_arrive(BAR(B_CODES_FREE + unit)); }
            st += kTeams;
            if (st >= n_steps) { st -= n_steps; ph ^= 1u; }
            return true;
        };
        const auto begin = [&](int tile) {
            scales = reinterpret_cast<const unsigned short *>(a.scales) + (size_t)min(m_of(tile) + r, a.out_width - 1) * a.groups;
            fetch(s0, sc[0]);
            fetch(s0 + kTeams, sc[1]);
        };
        begin(tile0);
        bool ok = true;
        unsigned parity = 0, odd = 0u, now = 1u;         /* (bits of tiles) */
#pragma unroll 1
        for (int tile = tile0; tile < end; tile = MANY ? tile + clusters : end) {
            for (int s = s0; s < steps && ok; s += 3 * kTeams) {
                ok = step(s, sc[0], sc[2]);
                if (ok && s + kTeams < steps) ok = step(s + kTeams, sc[1], sc[0]);
                if (ok && s + 2 * kTeams < steps) ok = step(s + 2 * kTeams, sc[2], sc[1]);
            }
            if (!ok) break;
            if (MANY && tile + clusters < end) {
                s0 = linear4_first_step(s0, steps, kTeams);
                begin(tile + clusters);
                behind += steps >> 1;
            }
            /* ===================== results: a lane has an output, the warp every fourth 16 rows ===================== */
            if (!WIDE) {
                const int row0 = row_of(tile), rows = min(N, a.rows - row0), o = m_of(tile) + r;
                if (!(ok = warp_wait(BAR(B_SUMS), parity, s_abort, g_err, 57u))) break;
                parity ^= 1u;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for (int c0 = team * 16; c0 < rows; c0 += 16 * kTeams) {
                    unsigned v[16];
                    tmem_ld16(tmem + ((unsigned)(quarter * 32) << 16) + c0, v);
                    float y[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        y[j] = __uint_as_float(v[j]);
                        if (MANY) odd |= fabsf(y[j]) < INFINITY ? 0u : now;
                    }
                    put(y, c0, min(16, rows - c0), r, o, row0);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (MANY && lane == 0) mbar_arrive_cluster(cluster_addr(BAR(B_RUN_FREE), leader));
                now = now << 1 ? now << 1 : now;
            }
        }
        if (MANY && !WIDE && ok) settle_all(odd, team * 16, 16 * kTeams, r);
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*s_abort) for (int i = 0; i < 10000; i++) __nanosleep(1000);      /* copies of the step that was given up are still on their way */
    /* what lies in shared memory: each CTA adds up the rows of its share, in the order of the k's */
    const auto add_up = [&](const auto &value) {
        if (warp >= 16 || *s_abort) return;
        constexpr int kAtOnce = 4;
        const int r = tid & 127, o = m_of(tile0) + r, row0 = row_of(tile0), rows = min(N, a.rows - row0), first = rows * split / f.splits, last = rows * (split + 1) / f.splits;        /* (such clusters have one tile) */
#pragma unroll 1
        for (int c = first + kAtOnce * (tid >> 7); c < last; c += kAtOnce * 4) {
            float y[kAtOnce] = {};
            const int n = min(kAtOnce, last - c);
#pragma unroll
            for (int i = 0; i < kMostSplits; i++) {
                if (i == f.splits) break;
                float v[kAtOnce];
#pragma unroll
                for (int j = 0; j < kAtOnce; j++) v[j] = value(i, ((c + j) * 128 + r) * 4);        /* (rows past the last lie in shared memory as well) */
#pragma unroll
                for (int j = 0; j < kAtOnce; j++) y[j] += v[j];
            }
            settle<T>(a, y, n, row0 + c, o, o < a.out_width);
            store<T, WIDE>(a, y, n, row0 + c, o, f.odd_out);
        }
        __syncwarp();
    };
    if (!MANY && WIDE && f.splits == 1) add_up([&](int, int at) { return *reinterpret_cast<const float *>(sm + at); });
    cluster_sync();
    if (!MANY && f.splits > 1) {
        add_up([&](int i, int at) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(sbase + at, 2 * i + rank)) : "memory");
            return v;
        });
        cluster_sync();
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == kIssuer) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
#undef BAR
}

template <class T, bool WIDE, int PER, bool MANY>
cudaError_t launch(const CUtensorMap &codes, const CUtensorMap &x, const many_args &f, int clusters, void *stream) {
    hy3a_launch l(dim3((unsigned)clusters * 2 * f.splits), dim3(warps_of<WIDE>::kThreads), kSmem, stream);
    l.cluster(2 * f.splits);
    return cudaLaunchKernelEx(&l.cfg, hy3a_linear4_umma_kernel<T, WIDE, PER, MANY>, codes, x, f);
}
/* Allows the shared memory, once per device, and tells how many clusters of 2 n CTAs fit on it at once, n = 1 .. kMostSplits (74, 33, 22 or so and 15: clusters stay within a part of the GPU). */
template <class T, bool WIDE, int PER>
cudaError_t ready(int device, int (&fit)[kMostSplits]) {
    static std::atomic<int> known[64][kMostSplits];
    for (int n = 0; n < kMostSplits; n++) {
        fit[n] = device < 64 ? known[device][n].load(std::memory_order_acquire) : 0;
        if (fit[n]) continue;
        cudaError_t e = cudaFuncSetAttribute(hy3a_linear4_umma_kernel<T, WIDE, PER, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(hy3a_linear4_umma_kernel<T, WIDE, PER, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return e;
        hy3a_launch l(dim3(2 * (n + 1)), dim3(warps_of<WIDE>::kThreads), kSmem, nullptr);
        l.cluster(2 * (n + 1));
        if ((e = cudaOccupancyMaxActiveClusters(&fit[n], hy3a_linear4_umma_kernel<T, WIDE, PER, false>, &l.cfg)) != cudaSuccess) return e;
        if (fit[n] < 1) fit[n] = 1;
        if (device < 64) known[device][n].store(fit[n], std::memory_order_release);
    }
    return cudaSuccess;
}

template <class T, bool WIDE, int PER>
cudaError_t run(const linear4_args &a, many_args &f, int device, void *stream, const char **what) {
    int fit[kMostSplits];
    cudaError_t e = ready<T, WIDE, PER>(device, fit);
    if (e != cudaSuccess) return e;
    const linear4_plan p = linear4_plan_of(a.rows, f.m_tiles, f.units, WIDE, fit);
    f.columns = p.columns; f.splits = p.splits; f.steps = p.steps; f.a_column = p.a_column;
    CUtensorMap codes, x;
    const encode_tiled_fn enc = encoder();
    const cuuint64_t dims[2] = {(cuuint64_t)(a.width / 2), (cuuint64_t)a.out_width}, strides[1] = {(cuuint64_t)(a.width / 2)};
    const cuuint32_t box[2] = {kUnit / 2, 128}, one[2] = {1, 1};
    const bool ok = enc && enc(&codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(a.codes), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS &&
                    encode(&x, 2, a.x, a.width, a.rows, 1, a.x_stride, 64, f.columns / 2);
    if (!ok) { *what = "no tensor map (cuTensorMapEncodeTiled)"; return cudaErrorInvalidValue; }
    if (p.tiles * 2 * f.splits > 0x7fffffffll) { *what = "too many tiles"; return cudaErrorInvalidValue; }
    f.tiles = (int)p.tiles;
    return f.splits == 1 && p.tiles > fit[0] ? launch<T, WIDE, PER, true>(codes, x, f, fit[0], stream) : launch<T, WIDE, PER, false>(codes, x, f, f.tiles, stream);
}
template <class T>
cudaError_t run_type(const linear4_args &a, many_args &f, int device, void *stream, const char **what) {
    if (a.group == 32) return a.wide ? run<T, true, 2>(a, f, device, stream, what) : run<T, false, 2>(a, f, device, stream, what);
    return a.wide ? run<T, true, 1>(a, f, device, stream, what) : run<T, false, 1>(a, f, device, stream, what);
}

} /* namespace */

cudaError_t hy3a_linear4_launch_many(const linear4_args &a, int dtype, int device, void *stream, const char **what) {
    many_args f = {a, ((uintptr_t)a.out & 3) || a.out_stride % 2 || a.out_width % 2, 0, (a.out_width + 255) / 256, 0, (a.width + kUnit - 1) / kUnit, 1, 0, 0};
    *what = NULL;
    return dtype == HY3A_BF16 ? run_type<__nv_bfloat16>(a, f, device, stream, what) : run_type<__half>(a, f, device, stream, what);
}

static __global__ void hy3a_linear4_many_wait_out_kernel() { wait_out(g_err, 69u); }
cudaError_t hy3a_linear4_many_wait_out(void *stream) {
    hy3a_linear4_many_wait_out_kernel<<<1, 32, 0, (cudaStream_t)stream>>>();
    return cudaGetLastError();
}
cudaError_t hy3a_linear4_many_words(unsigned **words) { return cudaGetSymbolAddress((void **)words, g_err); }

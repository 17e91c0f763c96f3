/*
 * experts_umma.cu -- the experts' two products on 5th-generation tensor cores (tcgen05 + TMEM + TMA).
 *
 * The weights are the M side of a product and the slots its N side: an expert has few or many slots, N takes any multiple of 16 up to 256, and
 * no rows are padded to 128.  A pair of CTAs (cta_group::2) works on 256 weight rows x up to 256 slots: each CTA holds its 128 weight
 * rows and half of the slots' rows in shared memory, and all slots of its weight rows in tensor memory (two accumulators of 256 columns, so that
 * one is stored while the next is computed).  Per CTA:
 *   warps 8-15 TMA producers: 64 k's a step into a ring of 6 stages; weight rows as boxes, rows of x gathered four at a time by row number
 *             (tile::gather4), rows of h, which lie in the order of the list, as boxes of 8, all with 128-byte swizzle; the byte counts of
 *             both CTAs go to the leader's barriers;
 *   warp 16   MMA issuer (of the leader): 4 x tcgen05.mma (K = 16) a step; commits reach both CTAs;
 *   warps 0-7 epilogue: tcgen05.ld, then h (of fp16 rows in fp32, for the launch that brings it into range) or y.
 * Gate / up: 16 gate rows and the 16 up rows of the same index alternate in the tile, so that a pair's halves lie 16 lanes apart in one
 * warp and meet in a shuffle.
 *
 * Pairs take tiles in turn: (slots' tile, 256 weight rows), the tiles of an expert's slots innermost, so that pairs that work on the same weights
 * at the same time find them in L2.
 *
 * With few slots an expert the kernels read weights (64 rows ask for 162 of 192 experts of 4096 x 1536: 6.1 GB in 928 us, 6.6 TB/s); with many, gate / up by itself
 * keeps the tensor pipe busy 78 % of the time, down 59 % (8192 slots on 24 experts; 1.07 PFLOP/s in gate / up from a cold start; passes for seconds run at
 * 1241 MHz, the median under the power limit, of 1965).  CTAs by themselves (cta_group::1, 128 weight rows) instead of pairs are 1 %
 * faster where weights are read and 30 % slower where products are computed: an SM's share of weights is the same.
 *
 * Every wait is bounded; one that runs out raises the CTA's abort flag and a code in the error word (hy3a_layer_sync), lets all warps fall
 * through, and TMEM is always released.
 */
#include <atomic>
#include <type_traits>

#include "experts.h"
#include "ring.cuh"

namespace {

using namespace hy3a_layer;
using namespace hy3a_ring;

constexpr int kStages = 6, kEpilogues = 8, kProducer = kEpilogues, kProducers = 8, kIssuer = kProducer + kProducers, kThreads = 32 * (kIssuer + 1);
constexpr int kABytes = 128 * 128, kBBytes = 128 * 128;      /* 128 rows of 64 k's, 2 bytes each */
constexpr int kPitch = 144, kPatch = 16 * kPitch;              /* an epilogue warp's patch: 16 slots of 32 fp32 values, rows 16 bytes apart in the banks */
constexpr int kOffPatch = kStages * (kABytes + kBBytes), kOffBar = kOffPatch + kEpilogues * kPatch, kSmem = kOffBar + 256 + 1024;
enum { B_FULL = 0, B_EMPTY = kStages, B_TFULL = 2 * kStages, B_TEMPTY = 2 * kStages + 2, B_COUNT = 2 * kStages + 4 };
static_assert(8 * B_COUNT + 16 <= 256, "barriers");

__device__ unsigned g_err[2];         /* {code, where} of the first wait that ran out, until hy3a_layer_sync reads it */

__device__ __forceinline__ void mbar_arrive_cluster(unsigned bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ unsigned cluster_addr(unsigned addr, unsigned rank) {
    unsigned r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
/* Copies are issued in uniform control flow by one elected lane (lead), so that their operands are computed in the uniform data path; both CTAs
 * count their bytes at the leader's barrier. */
__device__ __forceinline__ void tma_box(unsigned dst, const CUtensorMap *map, unsigned bar, int x, int y, int z, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %6, 0;\n"
                 " @e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];\n}"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(lead) : "memory");
}
__device__ __forceinline__ void tma_gather4(unsigned dst, const CUtensorMap *map, unsigned bar, int x, const int4 &row, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %8, 0;\n"
                 " @e cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n}"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(row.x), "r"(row.y), "r"(row.z), "r"(row.w), "r"(lead) : "memory");
}
/* K-major operand, 128-byte swizzle: 8-row groups 1024 B apart, descriptor version 1, layout 2 */
__device__ __forceinline__ unsigned long long make_desc(unsigned saddr) {
    return (unsigned long long)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void umma_lead(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate, unsigned lead) {
    asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 e, %5, 0;\n setp.ne.b32 p, %4, 0;\n @e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void umma_commit_lead(unsigned bar, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n @e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n}"
                 ::"r"(bar), "r"(lead), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ void tmem_ld16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
/* 32 bytes */
__device__ __forceinline__ void store32(void *p, const float4 &a, const float4 &b) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(a.x), "f"(a.y), "f"(a.z), "f"(a.w), "f"(b.x), "f"(b.y), "f"(b.z), "f"(b.w) : "memory");
}

/* what a tile is: its expert, weight rows from m0 (gate / up: pairs) and n of the listed slots from p0 */
struct where { int e, m0, p0, n; };
template <bool DOWN>
__device__ __forceinline__ where tile_of(const expert_tile &d, int t, int m_tiles) {
    const int in = t - d.first * m_tiles, m = in / d.tiles, j = in - m * d.tiles;
    const int width = ((d.count + d.tiles - 1) / d.tiles + 15) & ~15;       /* even, in the hardware's steps; at most 256, so no tile is empty */
    where w;
    w.e = d.expert; w.m0 = m * (DOWN ? 256 : 128); w.p0 = d.p0 + j * width; w.n = min(width, d.count - j * width);
    return w;
}
/* a warp's walk over the pair's tiles; the next one's line of the table is on its way while a tile is worked on */
template <bool DOWN>
struct tile_walk {
    const expert_args &a;
    const int step, m_tiles, total;
    int t;
    expert_tile next;
    __device__ __forceinline__ tile_walk(const expert_args &a_, int first, int step_, int m_tiles_, int total_) : a(a_), step(step_), m_tiles(m_tiles_), total(total_), t(first - step_) { fetch(); }
    __device__ __forceinline__ void fetch() { if (t + step < total) next = a.tiles[(t + step) / m_tiles]; }
    __device__ __forceinline__ bool take(where &w) {
        t += step;
        if (t >= total) return false;
        w = tile_of<DOWN>(next, t, m_tiles);
        fetch();
        return true;
    }
};

/* The steps of one tile for one producer warp: its weight box, and MINE of the tile's slot rows (gathers of 4, or boxes of 8), whose number is a
 * constant here so that the row numbers stay where the copy instruction reads them from: looked up in every step, a gather cost 52 clocks.
 * Each warp has a weight box in every step, so that no stage is filled, and none given back, before each has seen the stage's last phase end: one that
 * only waits may fall a ring behind, and a wait that has missed a phase ends with the next but one, or never. */
struct ring_state { unsigned st, ph; };
template <bool DOWN, int MINE>
__device__ __forceinline__ bool produce(ring_state &q, const CUtensorMap *tm_w, const CUtensorMap *tm_rows, unsigned sbase, unsigned bar0, volatile int *s_abort, int steps, int ahead /* steps whose weights are under way */, unsigned bytes /* 0: not the one that counts */,
                                        int part, int m, int e, const int4 (&row)[4], unsigned lead) {
    unsigned st = q.st, ph = q.ph;
    for (int s = 0; s < steps; s++) {
        /* (a stage whose weights are under way has not been used before) */
        if (s >= ahead && !warp_wait(bar0 + 8u * (B_EMPTY + st), ph ^ 1u, s_abort, g_err, 20u)) return false;
        const unsigned full = cluster_addr(bar0 + 8u * (B_FULL + st), 0), sa = sbase + st * (kABytes + kBBytes), sb = sa + kABytes;
        if (bytes && lead && s >= ahead) mbar_expect_tx(bar0 + 8u * (B_FULL + st), bytes);
        if (s >= ahead) tma_box(sa + part * 2048, tm_w, full, s * 64, m, e, lead);
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            if (DOWN) tma_box(sb + (part + kProducers * i) * 1024, tm_rows, full, s * 64, row[i].x, 0, lead);
            else tma_gather4(sb + (part + kProducers * i) * 512, tm_rows, full, s * 64, row[i], lead);
        }
        if (++st == kStages) { st = 0; ph ^= 1u; }
    }
    q.st = st; q.ph = ph;
    return true;
}

template <class T, bool DOWN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
hy3a_experts_umma_kernel(const __grid_constant__ CUtensorMap tm_w0, const __grid_constant__ CUtensorMap tm_w1, const __grid_constant__ CUtensorMap tm_rows, const expert_args a) {
    extern __shared__ uint8_t s_raw[];
    uint8_t *sm = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    const unsigned sbase = smem_u32(sm), bar0 = sbase + kOffBar;
    volatile unsigned *s_tmem = reinterpret_cast<volatile unsigned *>(sm + kOffBar + 8 * B_COUNT);
    volatile int *s_abort = reinterpret_cast<volatile int *>(sm + kOffBar + 8 * B_COUNT + 4);
#define BAR(i) (bar0 + 8u * (unsigned)(i))
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0) /* uniform for the compiler too */, lane = tid & 31;
    const unsigned rank = blockIdx.x & 1u;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int K = DOWN ? a.inter : a.hidden, steps = (K + 63) >> 6, m_tiles = DOWN ? (a.hidden + 255) >> 8 : (a.inter + 127) >> 7;

    if (tid == 0) {
        *s_abort = 0;
        for (int i = 0; i < kStages; i++) { mbar_init(BAR(B_FULL + i), 1); mbar_init(BAR(B_EMPTY + i), 1); }
        for (int i = 0; i < 2; i++) { mbar_init(BAR(B_TFULL + i), 1); mbar_init(BAR(B_TEMPTY + i), 2 * kEpilogues); }      /* empty: the epilogue warps of both CTAs */
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kProducer && lane < 3) {
        const CUtensorMap *m = lane == 0 ? &tm_w0 : (lane == 1 ? &tm_w1 : &tm_rows);
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
    /* Gate / up lets the next launch begin behind its own wait, and the one that fp16 rows have between the two lets `down` begin at once: `down` finds the plan
     * complete, and fetches its first weights before it waits for h. */
    if (!DOWN) pdl_wait();
    pdl_release();
    const int total = *a.n_tiles * m_tiles;
    if (DOWN && !(warp >= kProducer && warp < kProducer + kProducers)) pdl_wait();

    if (warp >= kProducer && warp < kProducer + kProducers) {
        /* ===================== producers: each an eighth of the weight boxes and of the slot rows ===================== */
        const int part = warp - kProducer;
        const unsigned lead = elect_one();
        ring_state q = {0, 0};
        tile_walk<DOWN> walk(a, pair, pairs, m_tiles, total);
        int ahead = 0;                  /* steps whose weights are under way */
        for (where w; walk.take(w);) {
            constexpr int kRows = DOWN ? 8 : 4;                                 /* of one copy */
            const int N = (w.n + 15) & ~15, half = N >> 1, first = w.p0 + (int)rank * half, last = w.p0 + w.n - 1;
            const int mine = (half / kRows - part + kProducers - 1) / kProducers;       /* (half is a multiple of 8) */
            int4 row[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = first + kRows * (part + kProducers * i);
                /* rows past the last are copies of it (gathered), or whatever lies behind: they are not stored */
                row[i] = make_int4(p, min(p + 1, last), min(p + 2, last), min(p + 3, last));
                if (!DOWN && i < mine) row[i] = make_int4(a.row[min(p, last)], a.row[row[i].y], a.row[row[i].z], a.row[row[i].w]);
            }
            const unsigned bytes = part == 0 && rank == 0 ? 2 * kABytes + N * 128 : 0;
            const CUtensorMap *tm = !DOWN && (part & 1) ? &tm_w1 : &tm_w0;
            const int m = w.m0 + (DOWN ? (int)rank * 128 + part * 16 : (int)rank * 64 + (part >> 1) * 16);
            if (DOWN && walk.t == pair) {
                ahead = min(steps, kStages);
                for (int s = 0; s < ahead; s++) {
                    const unsigned full = cluster_addr(BAR(B_FULL + s), 0);
                    if (bytes && lead) mbar_expect_tx(BAR(B_FULL + s), bytes);
                    tma_box(sbase + s * (kABytes + kBBytes) + part * 2048, tm, full, s * 64, m, w.e, lead);
                }
                pdl_wait();
            }
            bool ok;
            switch (mine) {
                case 4: ok = produce<DOWN, 4>(q, tm, &tm_rows, sbase, bar0, s_abort, steps, ahead, bytes, part, m, w.e, row, lead); break;
                case 3: ok = produce<DOWN, 3>(q, tm, &tm_rows, sbase, bar0, s_abort, steps, ahead, bytes, part, m, w.e, row, lead); break;
                case 2: ok = produce<DOWN, 2>(q, tm, &tm_rows, sbase, bar0, s_abort, steps, ahead, bytes, part, m, w.e, row, lead); break;
                case 1: ok = produce<DOWN, 1>(q, tm, &tm_rows, sbase, bar0, s_abort, steps, ahead, bytes, part, m, w.e, row, lead); break;
                default: ok = produce<DOWN, 0>(q, tm, &tm_rows, sbase, bar0, s_abort, steps, ahead, bytes, part, m, w.e, row, lead);
            }
            if (!ok) break;
            ahead = 0;
        }
        if (DOWN && pair >= total) pdl_wait();
        unsigned st = q.st, ph = q.ph;
        /* the last commits reach the barriers of both CTAs before either leaves */
        for (int i = 0; i < kStages; i++) {
            if (!warp_wait(BAR(B_EMPTY + st), ph ^ 1u, s_abort, g_err, 24u)) break;
            if (++st == kStages) { st = 0; ph ^= 1u; }
        }
    } else if (warp == kIssuer) {
        if (rank == 0) {
            /* ===================== MMA issuer: uniform control flow, one elected lane issues ===================== */
            const unsigned lead = elect_one();
            constexpr unsigned kType = type<T>::code == HY3A_BF16 ? (1u << 7) | (1u << 10) : 0u;
            unsigned st = 0, ph = 0, buf = 0, tph = 0;
            tile_walk<DOWN> walk(a, pair, pairs, m_tiles, total);
            for (where w; walk.take(w);) {
                const unsigned idesc = (1u << 4) | kType | (((unsigned)(w.n + 15) >> 4) << 18) | ((256u >> 4) << 24);
                if (!warp_wait(BAR(B_TEMPTY + buf), tph ^ 1u, s_abort, g_err, 21u)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                bool ok = true;
                for (int s = 0; s < steps; s++) {
                    if (!(ok = warp_wait(BAR(B_FULL + st), ph, s_abort, g_err, 22u))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned sa = sbase + st * (kABytes + kBBytes);
                    const unsigned long long da = make_desc(sa), db = make_desc(sa + kABytes);
#pragma unroll
                    for (int k = 0; k < 4; k++) umma_lead(tmem + buf * 256u, da + 2 * k, db + 2 * k, idesc, s + k > 0, lead);
                    umma_commit_lead(BAR(B_EMPTY + st), lead);
                    if (++st == kStages) { st = 0; ph ^= 1u; }
                }
                if (!ok) break;
                umma_commit_lead(BAR(B_TFULL + buf), lead);
                if (++buf == 2) { buf = 0; tph ^= 1u; }
            }
        }
    } else {
        /* ===================== epilogue: warp w has weight rows 32 (w % 4) .. + 31 of the CTA, and every other 16 slots =====================
         * A lane has a weight row, and what is stored is a slot's row: 16 slots at a time turn in a patch of shared memory, and leave as 32 bytes of y (or of h in fp32) or
         * 16 of h a lane (a store for each slot, of 32 neighbouring values, takes the warp 90 clocks beside the copies and products). */
        unsigned buf = 0, tph = 0;
        const int quarter = warp & 3, sl = lane & 15, half = lane >> 4;
        uint8_t *patch = sm + kOffPatch + warp * kPatch;
        tile_walk<DOWN> walk(a, pair, pairs, m_tiles, total);
        for (where w; walk.take(w);) {
            if (!warp_wait(BAR(B_TFULL + buf), tph, s_abort, g_err, 23u)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int m0 = DOWN ? w.m0 + (int)rank * 128 + quarter * 32 : w.m0 + (int)rank * 64 + quarter * 16;
            for (int c0 = (warp >> 2) * 16; c0 < w.n; c0 += 32) {
                unsigned v[16];
                tmem_ld16(tmem + ((unsigned)(quarter * 32) << 16) + buf * 256u + c0, v);
                if (DOWN) {
#pragma unroll
                    for (int j = 0; j < 16; j++) *reinterpret_cast<unsigned *>(patch + j * kPitch + lane * 4) = v[j];
                    __syncwarp();
                    /* four lanes a line of 128 bytes */
                    const int d = m0 + (lane & 3) * 8;
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int j = i * 8 + (lane >> 2);
                        const float4 *const from = reinterpret_cast<const float4 *>(patch + j * kPitch + (lane & 3) * 32);
                        if (c0 + j >= w.n || d >= a.hidden) continue;
                        float4 lo = from[0], hi = from[1];
                        if (type<T>::code == HY3A_F16) {
                            const float by = a.back[w.p0 + c0 + j];
                            lo.x *= by; lo.y *= by; lo.z *= by; lo.w *= by; hi.x *= by; hi.y *= by; hi.z *= by; hi.w *= by;
                        }
                        store32(a.y + (size_t)(w.p0 + c0 + j) * a.hidden + d, lo, hi);
                    }
                } else {
                    /* lanes below 16 have the gate, the others the up of one pair; of two slots each half finishes one */
                    using H = typename std::conditional<type<T>::code == HY3A_F16, float, T>::type;       /* what is stored */
                    constexpr int kPitchH = 16 * sizeof(H) + 16;
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float other = __shfl_xor_sync(0xffffffffu, __uint_as_float(half ? v[j] : v[j + 1]), 16);
                        const float g = half ? other : __uint_as_float(v[j]), u = half ? __uint_as_float(v[j + 1]) : other;
                        *reinterpret_cast<H *>(patch + (j + half) * kPitchH + sl * sizeof(H)) = type<H>::down(__fdividef(g, 1.f + __expf(-g)) * u);
                    }
                    __syncwarp();
                    if (c0 + sl < w.n && m0 + half * 8 < a.inter) {
                        const uint8_t *const from = patch + sl * kPitchH + half * 8 * sizeof(H);
                        const size_t at = (size_t)(w.p0 + c0 + sl) * a.inter + m0 + half * 8;
                        if (type<T>::code == HY3A_F16) store32(a.wide + at, *reinterpret_cast<const float4 *>(from), *reinterpret_cast<const float4 *>(from + 16));
                        else *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.h) + at) = *reinterpret_cast<const uint4 *>(from);
                    }
                }
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(cluster_addr(BAR(B_TEMPTY + buf), 0));
            if (++buf == 2) { buf = 0; tph ^= 1u; }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*s_abort) for (int i = 0; i < 10000; i++) __nanosleep(1000);      /* copies of the step that was given up are still on their way */
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == kIssuer) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
#undef BAR
}

struct maps { CUtensorMap gate, up, down, x, h; };
template <class T>
cudaError_t launch(const expert_args &a, const maps &m, int device, int sms, void *stream) {
    static std::atomic<bool> ready[64];       /* shared memory allowed, per device */
    cudaError_t e;
    if (device >= 64 || !ready[device].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(hy3a_experts_umma_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)) != cudaSuccess) return e;
        if ((e = cudaFuncSetAttribute(hy3a_experts_umma_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)) != cudaSuccess) return e;
        if (device < 64) ready[device].store(true, std::memory_order_release);
    }
    const dim3 grid(sms & ~1);
    {   hy3a_launch l(grid, dim3(kThreads), kSmem, stream);
        if ((e = cudaLaunchKernelEx(&l.cfg, hy3a_experts_umma_kernel<T, false>, m.gate, m.up, m.x, a)) != cudaSuccess) return e; }
    if (type<T>::code == HY3A_F16 && (e = hy3a_experts_launch_range(a, sms, stream)) != cudaSuccess) return e;
    hy3a_launch l(grid, dim3(kThreads), kSmem, stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_experts_umma_kernel<T, true>, m.down, m.down, m.h, a);
}

} /* namespace */

cudaError_t hy3a_experts_launch_umma(const expert_args &a, int dtype, int device, int sms, void *stream, const char **what) {
    *what = nullptr;
    maps m;
    const bool ok = encode(&m.gate, 3, a.gate, a.hidden, a.inter, a.held, a.hidden, 64, 16) && encode(&m.up, 3, a.up, a.hidden, a.inter, a.held, a.hidden, 64, 16) &&
                    encode(&m.down, 3, a.down, a.inter, a.hidden, a.held, a.inter, 64, 16) && encode(&m.x, 2, a.x, a.hidden, a.rows, 1, a.x_stride, 64, 1) &&
                    encode(&m.h, 3, a.h, a.inter, a.slots, 1, a.inter, 64, 8);
    if (!ok) { *what = "no tensor map (cuTensorMapEncodeTiled)"; return cudaErrorInvalidValue; }
    return dtype == HY3A_BF16 ? launch<__nv_bfloat16>(a, m, device, sms, stream) : launch<__half>(a, m, device, sms, stream);
}

static __global__ void hy3a_experts_wait_out_kernel() { wait_out(g_err, 29u); }
cudaError_t hy3a_experts_wait_out(void *stream) {
    hy3a_experts_wait_out_kernel<<<1, 32, 0, (cudaStream_t)stream>>>();
    return cudaGetLastError();
}
cudaError_t hy3a_experts_words(unsigned **words) { return cudaGetSymbolAddress((void **)words, g_err); }

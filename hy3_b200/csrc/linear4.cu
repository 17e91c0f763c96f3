/*
 * linear4.cu -- rows through a matrix of 4-bit codes with a scale for each group of neighbours in a row (hy3a_linear4), up to 16 rows:
 *
 *      y[t][o] = sum over groups j of scales[o][j] * sum over k of group j of (code[o][k] - 8) x[t][k]
 *
 * The inner sums are warp-level products of 16 outputs with 8 columns; the scale of a group multiplies its sum in fp32.  Nothing is rounded to fewer bits before the result.
 *   rows     the columns are rows: mma.m16n8k16 with fp32 sums; code - 8 is exact in the rows' type, and so are the products.  What makes numbers of codes bounds it, so a block has up to 16 rows for
 *            them, two products for each number, where registers have room for that much x (width 4096 at most), else 8 (16 rows on 10240 x 4096 in fp32: 12.0 us, by eights 15.7; on 120832 x 4096 85 and
 *            122).  More go to linear4_umma.cu, where 17 rows take 24.8 and 142 there (16-bit results 18 and 97, 10.6 on 4096 x 4096): 16 and 1 in calls of their own would take 21 and 130 for fp32 results, less,
 *            and more for 16-bit ones;
 *   digits   of one row, on large matrices, the columns are its digits: x = 2^E (d0 2^-7 + d1 2^-14 + .. + d7 2^-56), |d| < 128, with E from the largest |x| of the group, so that what is lost lies 2^-56
 *            below that (of 16-bit numbers: nothing, down to 2^-45 of it); mma.m16n8k32 of bytes with integer sums takes the codes as they are, two operations a word instead of 9, and
 *            -8 sum d comes in as the sum's first value.
 *
 * A block takes a contiguous part of the outputs (parts differ by four outputs at most), in tiles of 16, and streams their codes through a ring of shared memory: a
 * stage is a tile's codes for 4096 k's (or all, where there are fewer), copied as a box for each four outputs, and its scales, so that all blocks have 170 KB under way (one row on 120832 x 4096: 44 to 49 us, 5.4 to 6 TB/s).  (A bulk copy
 * for each output keeps the issuing lane busy for longer than its bytes take.)  The 16 warps share the k's; each keeps its part of x in registers for the whole launch.  Their
 * sums meet in shared memory, where a warp of their own adds them up.  Short launches wait for instructions as much as for codes: loops that are run a few times are not unrolled.
 *
 * mma wants of lane (g = lane / 4, t = lane % 4) four k's of outputs g and g + 8, and of column g; k's are renamed so that lane t has neighbouring ones, those of a word
 * (32 k's of 4 lanes) the least: a block of 32, 64 or 128 k's, one group's, is 1, 2 or 4 words a lane.
 */
#include <atomic>
#include <type_traits>

#include "linear4.h"
#include "ring.cuh"

namespace {

using namespace hy3a_layer;
using namespace hy3a_ring;

constexpr int kWarps = 16, kProducer = kWarps, kFinisher = kWarps + 1, kThreads = 32 * (kWarps + 2);
constexpr int kTile = 16 /* outputs */, kRows = 8 /* columns of a product */, kFewRows = 16, kStageK = 4096, kMaxStages = 16, kMaxWidth = 1 << 16, kMaxRows = 1 << 24, kMaxOut = 1 << 30 /* (numbers of outputs stay ints a tile past the last) */;
constexpr int kParts = 4 /* tiles of 8 rows whose parts may wait to be added up */, kPart = kTile * kRows /* values of a warp's part for 8 rows */;
constexpr int kBox = 4 /* outputs of a copy */, kLine = 128 /* its bytes of each, times the lines of a stage */;
constexpr int kRingBytes = 184 * 1024, kOffPart = kRingBytes, kOffBar = kOffPart + kParts * kWarps * kPart * 4, kSmem = kOffBar + 512 + 1024;
enum { B_FULL = 0, B_EMPTY = kMaxStages, B_READY = 2 * kMaxStages, B_TAKEN = 2 * kMaxStages + kParts, B_COUNT = 2 * kMaxStages + 2 * kParts };
static_assert(8 * B_COUNT + 8 <= 512, "barriers");
static_assert(kStageK / 8 * 8 * 8 <= kParts * kWarps * kPart * 4, "the digits of a stage's k's lie where the parts do later");

__device__ unsigned g_err[2];         /* {code, where} of the first wait that ran out, until hy3a_layer_sync reads it */

struct few_args {
    linear4_args a;
    int lines /* of 128 bytes, of an output's codes in a stage */, box_bytes /* of four outputs, with a line's more where lines is even: banks */, stage_bytes, stages, passes /* stages of a tile */;
    int in_stage /* groups of a stage */, per /* of a warp */;
    int boxed;                /* outputs whose lines of a stage are one copy: all where rows of codes are whole lines, else all but the last, as a row's last line ends in the next row (at k's whose x is 0) */
    int scale_pitch;          /* bytes of an output's scales in a stage; 0: rows of scales do not start on 16-byte boundaries, and are read where they lie */
    unsigned zero;            /* 0, which the compiler does not know */
};

/* Copies are issued in uniform control flow by one elected lane (lead): a lane's own operands cost each 50 clocks and more. */
__device__ __forceinline__ void copy_lines(unsigned dst, const CUtensorMap *map, unsigned bar, int x, int y, int z, unsigned long long policy, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %7, 0;\n"
                 " @e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;\n}"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(policy), "r"(lead) : "memory");
}
__device__ __forceinline__ void copy_scales(unsigned dst, const CUtensorMap *map, unsigned bar, int x, int y, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %5, 0;\n"
                 " @e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n}"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(lead) : "memory");
}
__device__ __forceinline__ void meet_workers() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }
template <class T> __device__ __forceinline__ float unpack(unsigned v, bool hi) {
    const unsigned short u = (unsigned short)(hi ? v >> 16 : v);
    return type<T>::up(*reinterpret_cast<const T *>(&u));
}
__device__ __forceinline__ unsigned scale_at(unsigned addr) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
    return v;
}
/* W words at an address of shared memory */
template <int W> __device__ __forceinline__ void load_words(unsigned addr, unsigned (&v)[W]) {
    if (W == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[W > 2 ? 2 : 0]), "=r"(v[W > 3 ? 3 : 0]) : "r"(addr));
    else if (W == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[W > 1 ? 1 : 0]) : "r"(addr));
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(addr));
}

/* ---- rows as columns: x of a lane for a group from k0 on, in the pairs' order; zeros past the width, and where the row is none ---- */
template <class T, int W> __device__ __forceinline__ void load_x(const T *row, bool there, int k0, int width, unsigned (&x)[4 * W]) {
    const int k = k0 + (threadIdx.x & 3) * 8 * W;
    there = there && k < width;        /* (all of the lane's or none: widths are multiples of 32) */
#pragma unroll
    for (int w = 0; w < W; w++) {
        uint4 v = zero16();
        if (there) v = load_row(row + k + 8 * w);
        x[4 * w + 0] = __byte_perm(v.x, v.z, 0x5410);
        x[4 * w + 1] = __byte_perm(v.x, v.z, 0x7632);
        x[4 * w + 2] = __byte_perm(v.y, v.w, 0x5410);
        x[4 * w + 3] = __byte_perm(v.y, v.w, 0x7632);
    }
}
/* type<T>::mma with sums from 0 */
template <class T> __device__ __forceinline__ void mma_first(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    if (type<T>::code == HY3A_BF16) asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                                        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
             : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <class T, int W, int C> struct row_columns {
    static constexpr bool kOne = C == 1;         /* (sums of one eight are multiplied in less time than numbers cost; 8 rows on 120832 x 4096: 59.9 us and 62.2, 16 rows: 82.3 and 80.5) */
    static constexpr float kPerStep = kOne ? steps<T>::kPerStep : 1.f;
    unsigned x[C][4 * W];
    __device__ __forceinline__ void sums(const unsigned (&wl)[W], const unsigned (&wh)[W], float (&d)[C][4]) const {
#pragma unroll
        for (int w = 0; w < W; w++) {
            unsigned vl[4], vh[4];
            if (kOne) { steps<T>::parts(wl[w], vl); steps<T>::parts(wh[w], vh); }
            else { steps<T>::of(wl[w], vl); steps<T>::of(wh[w], vh); }
#pragma unroll
            for (int c = 0; c < C; c++) {
                if (w == 0) mma_first<T>(d[c], vl[0], vh[0], vl[1], vh[1], x[c][0], x[c][1]);
                else type<T>::mma(d[c], vl[0], vh[0], vl[1], vh[1], x[c][4 * w], x[c][4 * w + 1]);
                type<T>::mma(d[c], vl[2], vh[2], vl[3], vh[3], x[c][4 * w + 2], x[c][4 * w + 3]);
            }
        }
    }
};

/* ---- digits as columns ---- */
constexpr unsigned kMostExponent = 127 + 100;
constexpr int kFirstSum = 0x4B400000;        /* 3 2^22 as a float: what is added to it as an integer, up to 2^22, is added to the float */
template <int W> struct digit_columns {
    static constexpr float kPerStep = 1.f;
    unsigned x[2 * W];                /* the column's digits of even and odd k's of each word */
    int first[2];                     /* kFirstSum - 8 sum of digits, of columns 2 t and 2 t + 1 */
    float unit;                       /* 2^(E - 7) */
    __device__ __forceinline__ void sums(const unsigned (&wl)[W], const unsigned (&wh)[W], float (&d)[1][4]) const {
        int n[4] = {first[0], first[1], first[0], first[1]};
#pragma unroll
        for (int w = 0; w < W; w++)
            asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                : "+r"(n[0]), "+r"(n[1]), "+r"(n[2]), "+r"(n[3])
                : "r"(wl[w] & 0x0f0f0f0fu), "r"(wh[w] & 0x0f0f0f0fu), "r"((wl[w] >> 4) & 0x0f0f0f0fu), "r"((wh[w] >> 4) & 0x0f0f0f0fu), "r"(x[2 * w]), "r"(x[2 * w + 1]));
#pragma unroll
        for (int i = 0; i < 4; i++) d[0][i] = fmaf(__int_as_float(n[i]), unit, -__int_as_float(kFirstSum) * unit);        /* exact, in the subnormal numbers too */
    }
};
__device__ __forceinline__ unsigned shift_left(unsigned v, int by) { unsigned r; asm("shl.b32 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(by)); return r; }        /* (0 by 32 and more, and by less than 0) */
__device__ __forceinline__ unsigned shift_right(unsigned v, int by) { unsigned r; asm("shr.u32 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(by)); return r; }

/* The digits of 8 k's from k on, a thread's share of a stage's: word `word` of the stage.  Row c = group * W + word of its lane holds the digits of four lanes, 8 bytes for
 * each column and lane, column j in place j ^ (c & 7): banks.  Sets *odd where x is not finite, or so large that its
 * unit times 2^24 might be infinite. */
template <class T, int W> __device__ __forceinline__ void store_digits(const T *row, int k, int width, int word, uint8_t *digits, float *units, int *odd) {
    uint4 raw = zero16();
    if (k < width) raw = load_row(row + k);
    const unsigned pairs[4] = {raw.x, raw.y, raw.z, raw.w};
    unsigned m[8], sign = 0;          /* |x| = m 2^(ex - 137), m < 2^11 */
    int ex[8], most = 1;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const unsigned u = __float_as_uint(unpack<T>(pairs[i / 2], i & 1)), e = (u >> 23) & 255u;
        m[i] = ((u >> 13) & 0x3ffu) | (e ? 0x400u : 0u);
        ex[i] = max((int)e, 1);
        most = max(most, ex[i]);
        sign |= (u >> 31) << i;
        if (e >= kMostExponent) *odd = 1;
    }
#pragma unroll
    for (int o = 1; o < 4 * W; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    /* (digits past the last bit of the warp's smallest x are 0) */
    int low = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) if (m[i]) low = max(low, most - ex[i]);
    const int digits_used = min(8, (__reduce_max_sync(0xffffffffu, low) + 11 + 6) / 7);
    const int c = word / (4 * W) * W + word % W, t = word / W & 3;
    if (word % (4 * W) == 0) units[word / (4 * W)] = most > 6 ? __int_as_float((most - 6) << 23) : __int_as_float(1 << (16 + most));
#pragma unroll 1
    for (int j = 0; j < 8; j++) {
        unsigned b[2] = {0, 0};
        if (j < digits_used)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int by = 7 * j - 4 + ex[i] - most;
            const unsigned d = (shift_left(m[i], by) | shift_right(m[i], -by)) & 127u, s = 0u - ((sign >> i) & 1u);
            b[i & 1] |= (((d ^ s) - s) & 255u) << (8 * (i >> 1));
        }
        *reinterpret_cast<uint2 *>(digits + c * 256 + ((j ^ (c & 7)) * 4 + t) * 8) = make_uint2(b[0], b[1]);
    }
}

/* W: words of a lane for a group; P: stages of a tile where x of all of them stays in registers, 0: x is read for each; ONE: one row; C: rows of a
 * block, in eights */
template <class T, int W, int P, bool ONE, int C>
__global__ void __launch_bounds__(kThreads, 1) hy3a_linear4_kernel(const __grid_constant__ CUtensorMap tm_codes, const __grid_constant__ CUtensorMap tm_line, const __grid_constant__ CUtensorMap tm_scales, const few_args f) {
    extern __shared__ uint8_t s_raw[];
    using columns = typename std::conditional<ONE, digit_columns<W>, row_columns<T, W, C>>::type;
    constexpr int kGroup = 32 * W, kMine = kStageK / kGroup / kWarps /* groups of a warp in a stage */, kSets = P ? P : 1, kPacks = (kMine + 3) / 4, kBufs = kParts / C;
    __shared__ float s_units[ONE ? kStageK / kGroup : 1];
    const linear4_args &a = f.a;
    uint8_t *sm = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    volatile int *s_abort = reinterpret_cast<volatile int *>(sm + kOffBar + 8 * B_COUNT);
    int *s_odd = reinterpret_cast<int *>(sm + kOffBar + 8 * B_COUNT + 4);
    const unsigned ring = smem_u32(sm), bar0 = ring + kOffBar;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0) /* uniform for the compiler too */, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int boxes = (a.out_width + kBox - 1) / kBox, first = kBox * (int)((long long)boxes * blockIdx.x / gridDim.x), last = min(a.out_width, kBox * (int)((long long)boxes * (blockIdx.x + 1) / gridDim.x));
    const int t0 = ONE ? 0 : blockIdx.y * (C * kRows), rows = ONE ? 1 : min(C * kRows, a.rows - t0);
    /* outputs g and g + 8 of the products are outputs mine and mine + 8 of the tile: such that lanes that read together find their words in different banks */
    const int mine_of = W == 4 ? (g & 1) * 4 + (g >> 1) : ((g >> 1) & 1) * 4 + (g & 1) * 2 + (g >> 2);
#define BAR(i) (bar0 + 8u * (unsigned)(i))
    if (tid == 0) {
        *s_abort = 0;
        *s_odd = 0;
        for (int i = 0; i < f.stages; i++) { mbar_init(BAR(B_FULL + i), 1); mbar_init(BAR(B_EMPTY + i), kWarps); }
        for (int i = 0; i < kParts; i++) { mbar_init(BAR(B_READY + i), kWarps); mbar_init(BAR(B_TAKEN + i), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kProducer && lane < 3) {
        const CUtensorMap *m = lane == 0 ? &tm_codes : lane == 1 ? &tm_scales : &tm_line;
        asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    __syncthreads();
    pdl_release();
    pdl_wait();
    int st = 0;
    unsigned ph = 0;
    if (warp == kProducer) {
        /* ===================== producer ===================== */
        const unsigned lead = elect_one();
        unsigned long long policy;
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        bool ok = true;
        for (int o0 = first; o0 < last && ok; o0 += kTile) {
            const int n = (min(kTile, last - o0) + kBox - 1) / kBox;
            for (int p = 0; p < f.passes; p++) {
                if (!(ok = warp_wait(BAR(B_EMPTY + st), ph ^ 1u, s_abort, g_err, 40u))) break;
                const unsigned to = ring + st * f.stage_bytes, full = BAR(B_FULL + st);
                /* (what lies past the matrix comes as zeros, and counts) */
                if (lead) mbar_expect_tx(full, n * f.lines * kBox * kLine + kTile * f.scale_pitch);
#pragma unroll 1
                for (int q = 0; q < n; q++) {
                    if (o0 + (q + 1) * kBox <= f.boxed || f.boxed == a.out_width) copy_lines(to + q * f.box_bytes, &tm_codes, full, 0, o0 + q * kBox, p * (kStageK / 2 / kLine), policy, lead);
                    else for (int c = 0; c < f.lines; c++) copy_lines(to + q * f.box_bytes + c * kBox * kLine, &tm_line, full, p * (kStageK / 2) + c * kLine, o0 + q * kBox, 0, policy, lead);
                }
                if (f.scale_pitch) copy_scales(to + (kTile / kBox) * f.box_bytes, &tm_scales, full, p * (kStageK / kGroup), o0, lead);
                if (++st == f.stages) { st = 0; ph ^= 1u; }
            }
        }
    } else if (warp == kFinisher) {
        /* ===================== the warps' parts, added up in the warps' order; a lane has an output and four columns ===================== */
        const int o = lane >> 1, r0 = (lane & 1) * 4;
        int turn = 0;
        unsigned skip = 0u;      /* rows with a NaN, whose results all are */
#pragma unroll 1
        for (int o0 = first; o0 < last; o0 += kTile, turn++) {
            const int buf = turn % kBufs;
            if (!warp_wait(BAR(B_READY + buf), (turn / kBufs) & 1, s_abort, g_err, 42u)) break;
            float v[4 * C];
            unsigned taken = 0u;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const float *part = reinterpret_cast<const float *>(sm + kOffPart) + (buf * kWarps * C + c) * kPart + lane * 4;
                float4 sum = *reinterpret_cast<const float4 *>(part);
#pragma unroll
                for (int w = 1; w < kWarps; w++) {
                    const float4 v = *reinterpret_cast<const float4 *>(part + w * C * kPart);
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                v[4 * c] = sum.x; v[4 * c + 1] = sum.y; v[4 * c + 2] = sum.z; v[4 * c + 3] = sum.w;
                taken |= __float_as_uint(sum.x);
            }
            __syncwarp();
            /* (an arrival does not wait for loads that are under way, so it takes something of the sums that they went into) */
            if (lane == 0) mbar_arrive(BAR(B_TAKEN + buf) + (taken & f.zero));
            const auto put = [&](int r, float y) {
                const size_t to = (size_t)(t0 + r) * a.out_stride + o0 + o;
                if (a.wide) reinterpret_cast<float *>(a.out)[to] = y;
                else reinterpret_cast<T *>(a.out)[to] = type<T>::down(y);
            };
            unsigned most = 0u;
            if (ONE) {
                /* digits: column c counts 2^-7c; an x that is not finite, or over 2^100, has none, and all results come from the definition */
                float y = (v[0] + v[1] * 0x1p-7f + (v[2] * 0x1p-14f + v[3] * 0x1p-21f)) * (r0 ? 0x1p-28f : 1.f);
                y += __shfl_xor_sync(0xffffffffu, y, 1);
                v[0] = *reinterpret_cast<volatile int *>(s_odd) ? NAN : y;
                if (r0 == 0 && o0 + o < last) {
                    put(0, v[0]);
                    most = skip ? 0u : __float_as_uint(v[0]) & 0x7fffffffu;
                }
            } else if (o0 + o < last) {
#pragma unroll
                for (int i = 0; i < 4 * C; i++) {
                    const int r = i / 4 * kRows + r0 + i % 4;
                    if (r < rows) {
                        put(r, v[i]);
                        most = max(most, skip >> r & 1 ? 0u : __float_as_uint(v[i]) & 0x7fffffffu);
                    }
                }
            }
            /* What is not finite (an infinite x or scale, a group's sum beyond fp32 whose product with its scale is not, digits that there are not) comes from the definition.  (256 results of 65536 products,
             * the most a tile has, take a small part of the half second that others wait for it.  Called functions cost each launch 0.4 to 2 us, also where they are not reached: these are in line.) */
            if (__any_sync(0xffffffffu, most >= 0x7f800000u)) {
#pragma unroll 1
                for (int r = 0; r < rows; r++) {
                    const int i = r / kRows * 4 + r % 4;
                    float y = v[0];
#pragma unroll
                    for (int k = 1; k < 4 * C; k++) if (i == k) y = v[k];
                    const bool mine = o0 + o < last && r0 == r % kRows / 4 * 4;
                    unsigned todo = __ballot_sync(0xffffffffu, mine && !(skip >> r & 1) && !(fabsf(y) < INFINITY));
                    if (!todo) continue;
                    if (has_nan<T>(a, t0 + r)) {
                        skip |= 1u << r;
                        continue;
                    }
#pragma unroll 1
                    for (; todo; todo &= todo - 1) {
                        const int l = __ffs(todo) - 1;
                        const float again = plain<T>(a, t0 + r, o0 + (l >> 1));
                        if (lane == l) put(r, again);
                    }
                }
            }
        }
    } else {
        /* ===================== products: a warp has `per` groups of a stage, one behind the other ===================== */
        columns x[kSets][kMine];
        const T *const rows_of_x = reinterpret_cast<const T *>(a.x) + (size_t)t0 * a.x_stride;
        const int g0 = warp * f.per;
        const auto load_columns = [&](columns (&to)[kMine], int p) {
            if constexpr (ONE) {
                uint8_t *const digits = sm + kOffPart;
                meet_workers();
                store_digits<T, W>(rows_of_x, p * kStageK + tid * 8, a.width, tid, digits, s_units, s_odd);
                meet_workers();
#pragma unroll
                for (int i = 0; i < kMine; i++) {
                    const bool there = i < f.per && g0 + i < kStageK / kGroup;
                    int sum = 0;
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        const int c = (g0 + i) * W + w;
                        const uint2 d = there ? *reinterpret_cast<const uint2 *>(digits + c * 256 + ((g ^ (c & 7)) * 4 + t) * 8) : make_uint2(0, 0);
                        to[i].x[2 * w] = d.x;
                        to[i].x[2 * w + 1] = d.y;
                        sum = __dp4a((int)d.x, 0x01010101, __dp4a((int)d.y, 0x01010101, sum));
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
                    for (int k = 0; k < 2; k++) to[i].first[k] = kFirstSum - 8 * __shfl_sync(0xffffffffu, sum, (2 * t + k) * 4);
                    to[i].unit = there ? s_units[g0 + i] : 0.f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kMine; i++)
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        const int r = c * kRows + g;
                        load_x<T, W>(rows_of_x + (size_t)min(r, rows - 1) * a.x_stride, r < rows && i < f.per, p * kStageK + (g0 + i) * kGroup, a.width, to[i].x[c]);
                    }
            }
        };
        if (P) {
#pragma unroll
            for (int p = 0; p < kSets; p++) load_columns(x[p], p);
            if (ONE) meet_workers();          /* (where the digits lay, parts come) */
        }
        /* where the lane's words are in a stage: line c of four outputs lies behind line c - 1, its 16-byte parts in an order that goes by their address (128-byte swizzle) */
        unsigned at[kMine];
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const unsigned in_row = (unsigned)((g0 + i) * 16 * W + t * 4 * W), line = (unsigned)(mine_of >> 2) * f.box_bytes + (in_row >> 7) * (kBox * kLine) + (unsigned)(mine_of & 3) * kLine;
            at[i] = ring + line + ((in_row & 127u) ^ ((line >> 3) & 0x70u));
        }
        const unsigned eight = 2 * f.box_bytes, scales_at = ring + (kTile / kBox) * f.box_bytes + mine_of * f.scale_pitch + (g0 + t) * 2;
        int turn = 0;
        const auto stage = [&](int o0, int p, const columns (&xs)[kMine], float (&acc)[C][4]) {
            const int mine = min(f.per, a.groups - p * (kStageK / kGroup) - g0);
            /* scales of the lane's two outputs, group 4 i + t of the warp's for i = 0 .. */
            unsigned both[kPacks];
            if (!f.scale_pitch) {
#pragma unroll
                for (int i = 0; i < kPacks; i++) {
                    const unsigned short *const s = reinterpret_cast<const unsigned short *>(a.scales) + (size_t)(o0 + mine_of) * a.groups + p * (kStageK / kGroup) + g0 + 4 * i + t;
                    both[i] = 0u;
                    if (4 * i + t < mine && o0 + mine_of < last) both[i] = s[0];
                    if (4 * i + t < mine && o0 + mine_of + 8 < last) both[i] |= (unsigned)s[(size_t)8 * a.groups] << 16;
                }
            }
            /* (polls of single lanes and one vote: one row on 120832 x 4096 45.0 us, 46.3 with votes on polls, 44.3 without any, which leaves it to chance that the lanes go on together) */
            if (__all_sync(0xffffffffu, mbar_wait(BAR(B_FULL + st), ph, s_abort, g_err, 41u))) {
                const unsigned by = st * f.stage_bytes;
                if (f.scale_pitch) {
#pragma unroll
                    for (int i = 0; i < kPacks; i++) both[i] = 4 * i + t < mine ? scale_at(scales_at + by + 8 * i) | scale_at(scales_at + by + 8 * i + 8 * f.scale_pitch) << 16 : 0u;
                }
                /* Groups that are not there have x and scales of 0, and codes of any value.  (Without branches between them the groups' chains overlap.) */
                constexpr int kHalf = kMine > 1 ? kMine / 2 : 1;
#pragma unroll
                for (int h = 0; h < kMine; h += kHalf) {
                    if (h >= mine) break;
#pragma unroll
                    for (int i = h; i < h + kHalf; i++) {
                        unsigned wl[W], wh[W];
                        load_words<W>(at[i] + by, wl);
                        load_words<W>(at[i] + by + eight, wh);
                        float d[C][4];
                        xs[i].sums(wl, wh, d);
                        const unsigned s = __shfl_sync(0xffffffffu, both[i / 4], (lane & 28) | (i & 3));
                        const float s0 = unpack<T>(s, false), s1 = unpack<T>(s, true);
#pragma unroll
                        for (int c = 0; c < C; c++) {
                            /* (the sum is what may be scaled: a scale times kPerStep need not be finite) */
#pragma unroll
                            for (int k = 0; k < 4; k++) d[c][k] *= columns::kPerStep;
                            acc[c][0] = fmaf(s0, d[c][0], acc[c][0]); acc[c][1] = fmaf(s0, d[c][1], acc[c][1]);
                            acc[c][2] = fmaf(s1, d[c][2], acc[c][2]); acc[c][3] = fmaf(s1, d[c][3], acc[c][3]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(B_EMPTY + st) + ((__float_as_uint(acc[0][0]) | __float_as_uint(acc[0][2])) & f.zero));
            if (++st == f.stages) { st = 0; ph ^= 1u; }
        };
#pragma unroll 1
        for (int o0 = first; o0 < last; o0 += kTile, turn++) {
            float acc[C][4] = {};
            if (P) {
#pragma unroll
                for (int p = 0; p < kSets; p++) stage(o0, p, x[p], acc);
            } else {
#pragma unroll 1
                for (int p = 0; p < f.passes; p++) {
                    load_columns(x[0], p);
                    stage(o0, p, x[0], acc);
                }
            }
            const int buf = turn % kBufs;
            if (turn >= kBufs && !warp_wait(BAR(B_TAKEN + buf), (turn / kBufs - 1) & 1, s_abort, g_err, 43u)) break;
            float *const part = reinterpret_cast<float *>(sm + kOffPart) + (buf * kWarps + warp) * C * kPart;       /* [eight rows][output][row] */
#pragma unroll
            for (int c = 0; c < C; c++) {
                *reinterpret_cast<float2 *>(part + c * kPart + mine_of * kRows + 2 * t) = make_float2(acc[c][0], acc[c][1]);
                *reinterpret_cast<float2 *>(part + c * kPart + (mine_of + 8) * kRows + 2 * t) = make_float2(acc[c][2], acc[c][3]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(B_READY + buf));
        }
    }
    if (*s_abort) for (int i = 0; i < 10000; i++) __nanosleep(1000);      /* copies of a stage that was given up are still on their way */
#undef BAR
}

template <class T, int W, int P, bool ONE, int C = 1>
cudaError_t launch(const CUtensorMap (&maps)[3], const few_args &f, int device, int sms, void *stream) {
    static std::atomic<bool> ready[64];       /* shared memory allowed, per device */
    cudaError_t e;
    if (device >= 64 || !ready[device].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(hy3a_linear4_kernel<T, W, P, ONE, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)) != cudaSuccess) return e;
        if (device < 64) ready[device].store(true, std::memory_order_release);
    }
    const int boxes = (f.a.out_width + kBox - 1) / kBox;
    hy3a_launch l(dim3(boxes < sms ? boxes : sms, (f.a.rows + C * kRows - 1) / (C * kRows)), dim3(kThreads), kSmem, stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_linear4_kernel<T, W, P, ONE, C>, maps[0], maps[1], maps[2], f);
}
template <class T, int W>
cudaError_t launch_group(const CUtensorMap (&maps)[3], const few_args &f, int device, int sms, void *stream) {
    constexpr bool kDigitsOfTwo = W > 1;       /* (short groups leave no registers for two stages' digits) */
    /* Digits save a third of a microsecond a tile and take two to make: for 6 tiles a block and more (one row on 4096 x 4096: 6.9 us with them, 5.0 without; on 120832 x 4096 50 and 63). */
    const bool digits = f.a.rows == 1 && f.a.out_width >= 6 * kTile * sms;
    if (f.passes == 1 && f.a.rows > kRows) return launch<T, W, 1, false, 2>(maps, f, device, sms, stream);
    if (f.passes == 1) return digits ? launch<T, W, 1, true>(maps, f, device, sms, stream) : launch<T, W, 1, false>(maps, f, device, sms, stream);
    if (f.passes == 2) return digits && kDigitsOfTwo ? launch<T, W, 2, kDigitsOfTwo>(maps, f, device, sms, stream) : launch<T, W, 2, false>(maps, f, device, sms, stream);
    return launch<T, W, 0, false>(maps, f, device, sms, stream);
}
template <class T>
cudaError_t launch_few(const linear4_args &a, int device, int sms, void *stream, const char **what) {
    const int k = a.width < kStageK ? a.width : kStageK, bytes = a.width / 2;
    few_args f = {a, (k / 2 + kLine - 1) / kLine, 0, 0, 0, (a.width + kStageK - 1) / kStageK, (k + a.group - 1) / a.group, 0, 0, 0, 0u};
    f.per = (f.in_stage + kWarps - 1) / kWarps;
    f.box_bytes = (f.lines | 1) * kBox * kLine;
    const bool boxed = a.groups % 8 == 0 && (uintptr_t)a.scales % 16 == 0;
    if (boxed) f.scale_pitch = 2 * (a.groups < kStageK / a.group ? a.groups : kStageK / a.group);
    f.stage_bytes = (kTile / kBox * f.box_bytes + kTile * f.scale_pitch + 1023) & ~1023;
    f.stages = kRingBytes / f.stage_bytes;
    if (f.stages > kMaxStages) f.stages = kMaxStages;
    /* [lines][outputs][128 bytes], all lines of a stage in a copy; and [outputs][bytes], a line in a copy */
    f.boxed = bytes % kLine == 0 ? a.out_width : bytes > kLine ? a.out_width - 1 : 0;
    CUtensorMap maps[3] = {};
    const encode_tiled_fn enc = encoder();
    const cuuint32_t one[3] = {1, 1, 1};
    const auto codes = [&](CUtensorMap *m, cuuint64_t inner, int outputs, int lines, cuuint64_t line_stride, int box_lines) {
        const cuuint64_t dims[3] = {inner, (cuuint64_t)outputs, (cuuint64_t)lines}, strides[2] = {(cuuint64_t)bytes, line_stride};
        const cuuint32_t box[3] = {kLine, kBox, (cuuint32_t)box_lines};
        return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(a.codes), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    bool ok = enc && (!f.boxed || codes(&maps[0], kLine, f.boxed, (bytes + kLine - 1) / kLine, kLine, f.lines)) && codes(&maps[1], bytes, a.out_width, 1, 16, 1);
    if (boxed && ok) {
        const cuuint64_t sdims[2] = {(cuuint64_t)a.groups, (cuuint64_t)a.out_width}, sstrides[1] = {2ull * a.groups};
        const cuuint32_t sbox[2] = {(cuuint32_t)f.scale_pitch / 2, kTile};
        ok = enc(&maps[2], CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(a.scales), sdims, sstrides, sbox, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                 CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    if (!f.boxed) maps[0] = maps[1];          /* (not used, but fetched) */
    if (!boxed) maps[2] = maps[1];
    if (!ok) {
        *what = "no tensor map (cuTensorMapEncodeTiled)";
        return cudaErrorInvalidValue;
    }
    if (a.group == 32) return launch_group<T, 1>(maps, f, device, sms, stream);
    if (a.group == 64) return launch_group<T, 2>(maps, f, device, sms, stream);
    return launch_group<T, 4>(maps, f, device, sms, stream);
}

} /* namespace */

int hy3a_quant4_sizes(const char *who, int out_width, int width, int group) {
    if (out_width < 0 || out_width > kMaxOut) return hy3a_fail(NULL, HY3A_EINVAL, "%s: out_width %d not in [0,%d]", who, out_width, kMaxOut);
    if (width < 32 || width > kMaxWidth || width % 32) return hy3a_fail(NULL, HY3A_EINVAL, "%s: width %d: a multiple of 32 in [32,%d]", who, width, kMaxWidth);
    if (group != 32 && group != 64 && group != 128) return hy3a_fail(NULL, HY3A_EINVAL, "%s: group %d not in {32,64,128}", who, group);
    return HY3A_OK;
}

extern "C" int hy3a_linear4(void *stream, int dtype, int rows, int width, int out_width, int group, const void *x, size_t x_stride, const void *codes, const void *scales,
                            int out_dtype, void *out, size_t out_stride) {
    if (dtype != HY3A_F16 && dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: dtype %d not in {1,2}", dtype);
    if (out_dtype != dtype && out_dtype != HY3A_F32) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: out_dtype %d is neither the rows' nor fp32", out_dtype);
    if (rows < 0 || rows > kMaxRows) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: rows %d not in [0,%d]", rows, kMaxRows);
    int rc = hy3a_quant4_sizes("linear4", out_width, width, group);
    if (rc) return rc;
    if (rows == 0 || out_width == 0) return HY3A_OK;
    if (!x || !codes || !scales || !out) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: NULL argument");
    if (((uintptr_t)x | (uintptr_t)codes) & 15) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: x and codes have to be 16-byte aligned");
    if (((uintptr_t)scales & 1) || ((uintptr_t)out & (out_dtype == HY3A_F32 ? 3 : 1))) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: a pointer is not aligned to its type");
    if (x_stride % 8) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: rows of x have to start on 16-byte boundaries");
    if (rows > 1 && out_stride < (size_t)out_width) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: rows of out overlap");
    int dev, sms;
    if ((rc = hy3a_layer_device("linear4", &dev, &sms))) return rc;
    const linear4_args a = {x, x_stride, (const uint8_t *)codes, scales, out, out_stride, rows, width, out_width, group, (width + group - 1) / group, out_dtype == HY3A_F32};
    const char *what = NULL;
    const cudaError_t e = rows > kFewRows ? hy3a_linear4_launch_many(a, dtype, dev, stream, &what)
                        : (dtype == HY3A_BF16 ? launch_few<__nv_bfloat16>(a, dev, sms, stream, &what) : launch_few<__half>(a, dev, sms, stream, &what));
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "linear4: %s", what ? what : cudaGetErrorString(e));
    return HY3A_OK;
}

static __global__ void hy3a_linear4_wait_out_kernel() { wait_out(g_err, 49u); }
cudaError_t hy3a_linear4_wait_out(void *stream) {
    hy3a_linear4_wait_out_kernel<<<1, 32, 0, (cudaStream_t)stream>>>();
    return cudaGetLastError();
}
cudaError_t hy3a_linear4_words(unsigned **words) { return cudaGetSymbolAddress((void **)words, g_err); }

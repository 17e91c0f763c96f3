/*
 * linear4.cu -- rows through a matrix of 4-bit codes with a scale for each group of neighbours in a row (hy3a_linear4), few rows:
 *
 *      y[t][o] = sum over groups j of scales[o][j] * sum over k of group j of (code[o][k] - 8) x[t][k]
 *
 * The inner sums are warp-level products (mma.m16n8k16, fp32 sums) of 16 outputs with 8 rows: the differences are exact in the rows' type and so are the
 * products; the scale of a group multiplies its sum in fp32.  Nothing is rounded to fewer bits before the result.
 *
 * A block takes a contiguous part of the outputs (parts differ by four outputs at most), in tiles of 16, and streams their codes through a ring of shared memory: a
 * stage is a tile's codes for 4096 k's (or all, where there are fewer), copied as a box for each four outputs, so that all blocks have 170 KB under way.  (A bulk copy for
 * each output keeps the issuing lane busy for longer than its bytes take.)  The 16 warps share the k's; each keeps its part of x in registers for the whole launch, and reads its scales two
 * stages ahead.  Their sums meet in shared memory, where a warp of their own adds them up.
 *
 * mma wants of lane (g = lane / 4, t = lane % 4) four k's of outputs g and g + 8, and of row g; k's are renamed so that lane t has neighbouring ones, those of a word
 * (32 k's of 4 lanes) the least: a block of 32, 64 or 128 k's, one group's, is 1, 2 or 4 words a lane.
 */
#include <atomic>

#include "linear4.h"
#include "ring.cuh"

namespace {

using namespace hy3a_layer;
using namespace hy3a_ring;

constexpr int kMostWarps = 16, kTile = 16 /* outputs */, kRows = 8, kStageK = 4096, kMaxStages = 16, kMaxWidth = 1 << 16;
constexpr int kParts = 4 /* tiles whose parts may wait to be added up */, kPart = kTile * kRows /* values of a warp's part */;
constexpr int kBox = 4 /* outputs of a copy */, kLine = 128 /* its bytes of each, times the lines of a stage */;
constexpr int kRingBytes = 180 * 1024, kOffPart = kRingBytes, kOffBar = kOffPart + kParts * kMostWarps * kPart * 4, kSmem = kOffBar + 512 + 1024;
enum { B_FULL = 0, B_EMPTY = kMaxStages, B_READY = 2 * kMaxStages, B_TAKEN = 2 * kMaxStages + kParts, B_COUNT = 2 * kMaxStages + 2 * kParts };
static_assert(8 * B_COUNT <= 512, "barriers");

__device__ unsigned g_err[2];         /* {code, where} of the first wait that ran out, until hy3a_layer_sync reads it */

struct few_args {
    linear4_args a;
    int lines /* of 128 bytes, of an output's codes in a stage */, box_bytes /* of four outputs, with a line's more where lines is even: banks */, stages, passes /* stages of a tile */, in_stage /* groups of a stage */, per /* of a warp */;
    int whole;                /* rows of codes are whole lines */
    unsigned zero;            /* 0, which the compiler does not know */
};

/* Copies are issued in uniform control flow by one elected lane (lead): a lane's own operands cost each 50 clocks and more. */
__device__ __forceinline__ void copy_lines(unsigned dst, const CUtensorMap *map, unsigned bar, int x, int y, int z, unsigned long long policy, unsigned lead) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %7, 0;\n"
                 " @e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;\n}"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(policy), "r"(lead) : "memory");
}
template <class T> __device__ __forceinline__ float unpack(unsigned v, bool hi) {
    const unsigned short u = (unsigned short)(hi ? v >> 16 : v);
    return type<T>::up(*reinterpret_cast<const T *>(&u));
}

/* x of a lane for a block of 32 W k's from k0 on, in the pairs' order; zeros past the width, and where the row is none */
template <class T, int W> __device__ __forceinline__ void load_x(const T *row, bool there, int k0, int width, unsigned (&x)[4 * W]) {
    const int k = k0 + (threadIdx.x & 3) * 8 * W;
#pragma unroll
    for (int w = 0; w < W; w++) {
        uint4 v = zero16();
        if (there && k + 8 * w < width) v = load_row(row + k + 8 * w);
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
/* W words at an address of shared memory */
template <int W> __device__ __forceinline__ void load_words(unsigned addr, unsigned (&v)[W]) {
    if (W == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[W > 2 ? 2 : 0]), "=r"(v[W > 3 ? 3 : 0]) : "r"(addr));
    else if (W == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[W > 1 ? 1 : 0]) : "r"(addr));
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(addr));
}

/* W: words of a lane for a group; P: stages of a tile where x of all of them stays in registers, 0: x is read for each */
template <class T, int W, int P, int kWarps>
__global__ void __launch_bounds__(32 * (kWarps + 2), 1) hy3a_linear4_kernel(const __grid_constant__ CUtensorMap tm, const few_args f) {
    extern __shared__ uint8_t s_raw[];
    constexpr int kProducer = kWarps, kFinisher = kWarps + 1, kGroup = 32 * W, kMine = kStageK / kGroup / kWarps /* groups of a warp in a stage */, kSets = P ? P : 1, kPacks = (kMine + 3) / 4, kAhead = P == 1 ? 2 : (P ? 1 : 0) /* tiles */;
    const linear4_args &a = f.a;
    uint8_t *sm = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    volatile int *s_abort = reinterpret_cast<volatile int *>(sm + kOffBar + 8 * B_COUNT);
    const unsigned ring = smem_u32(sm), bar0 = ring + kOffBar, stage_bytes = (kTile / kBox) * f.box_bytes;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0) /* uniform for the compiler too */, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int boxes = (a.out_width + kBox - 1) / kBox, first = kBox * (int)((long long)boxes * blockIdx.x / gridDim.x), last = min(a.out_width, kBox * (int)((long long)boxes * (blockIdx.x + 1) / gridDim.x));
    const int t0 = blockIdx.y * kRows, rows = min(kRows, a.rows - t0);
    /* outputs g and g + 8 of the products are outputs mine and mine + 8 of the tile: such that lanes that read together find their words in different banks */
    const int mine_of = W == 4 ? (g & 1) * 4 + (g >> 1) : ((g >> 1) & 1) * 4 + (g & 1) * 2 + (g >> 2);
#define BAR(i) (bar0 + 8u * (unsigned)(i))
    if (tid == 0) {
        *s_abort = 0;
        for (int i = 0; i < f.stages; i++) { mbar_init(BAR(B_FULL + i), 1); mbar_init(BAR(B_EMPTY + i), kWarps); }
        for (int i = 0; i < kParts; i++) { mbar_init(BAR(B_READY + i), kWarps); mbar_init(BAR(B_TAKEN + i), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kProducer && lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&tm) : "memory");
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
                if (!(ok = mbar_wait(BAR(B_EMPTY + st), ph ^ 1u, s_abort, g_err, 40u))) break;
                const unsigned to = ring + st * stage_bytes, full = BAR(B_FULL + st);
                /* (what lies past the matrix comes as zeros, and counts) */
                if (lead) mbar_expect_tx(full, n * f.lines * kBox * kLine);
                for (int q = 0; q < n; q++) {
                    if (f.whole) copy_lines(to + q * f.box_bytes, &tm, full, 0, o0 + q * kBox, p * (kStageK / 2 / kLine), policy, lead);
                    else for (int c = 0; c < f.lines; c++) copy_lines(to + q * f.box_bytes + c * kBox * kLine, &tm, full, p * (kStageK / 2) + c * kLine, o0 + q * kBox, 0, policy, lead);
                }
                if (++st == f.stages) { st = 0; ph ^= 1u; }
            }
        }
    } else if (warp == kFinisher) {
        /* ===================== the warps' parts, added up in the warps' order; a lane has an output and four rows ===================== */
        const int o = lane >> 1, r0 = (lane & 1) * 4;
        int turn = 0;
        for (int o0 = first; o0 < last; o0 += kTile, turn++) {
            const int buf = turn % kParts;
            if (!mbar_wait(BAR(B_READY + buf), (turn / kParts) & 1, s_abort, g_err, 42u)) break;
            const float *part = reinterpret_cast<const float *>(sm + kOffPart) + buf * kWarps * kPart + lane * 4;
            float4 sum = *reinterpret_cast<const float4 *>(part);
#pragma unroll
            for (int w = 1; w < kWarps; w++) {
                const float4 v = *reinterpret_cast<const float4 *>(part + w * kPart);
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(B_TAKEN + buf));
            if (o0 + o < last) {
                const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (r0 + r >= rows) break;
                    const size_t to = (size_t)(t0 + r0 + r) * a.out_stride + o0 + o;
                    if (a.wide) reinterpret_cast<float *>(a.out)[to] = v[r];
                    else reinterpret_cast<T *>(a.out)[to] = type<T>::down(v[r]);
                }
            }
        }
    } else {
        /* ===================== products: a warp has `mine` groups of a stage, one behind the other ===================== */
        unsigned x[kSets][kMine][4 * W];
        const T *row = reinterpret_cast<const T *>(a.x) + (size_t)(t0 + min(g, rows - 1)) * a.x_stride;
        const int g0 = warp * f.per;
        if (P) {
#pragma unroll
            for (int p = 0; p < kSets; p++)
#pragma unroll
                for (int i = 0; i < kMine; i++) load_x<T, W>(row, g < rows && i < f.per, p * kStageK + (g0 + i) * kGroup, a.width, x[p][i]);
        }
        /* where the lane's words are in a stage: line c of four outputs lies behind line c - 1, its 16-byte parts in an order that goes by their address (128-byte swizzle) */
        unsigned at[kMine];
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const unsigned in_row = (unsigned)((g0 + i) * 16 * W + t * 4 * W), line = (unsigned)(mine_of >> 2) * f.box_bytes + (in_row >> 7) * (kBox * kLine) + (unsigned)(mine_of & 3) * kLine;
            at[i] = ring + line + ((in_row & 127u) ^ ((line >> 3) & 0x70u));
        }
        const unsigned eight = 2 * f.box_bytes;
        /* Scales of the lane's two outputs, group 4 i + t of the warp's for i = 0 ..: those of a tile are asked for kAhead tiles before, into registers that nothing
         * touches until then. */
        unsigned short sc[kAhead + 1][kSets][kPacks][2];
        const auto fetch = [&](int o0, int p, unsigned short (&to)[kPacks][2]) {
#pragma unroll
            for (int i = 0; i < kPacks; i++) {
                const int j = p * (kStageK / kGroup) + g0 + 4 * i + t, o = o0 + mine_of;
                const unsigned short *const s = reinterpret_cast<const unsigned short *>(a.scales) + (size_t)o * a.groups + j;
                const bool there = 4 * i + t < f.per && j < a.groups;
                to[i][0] = to[i][1] = 0;
                if (there && o < last) to[i][0] = s[0];
                if (there && o + 8 < last) to[i][1] = s[(size_t)8 * a.groups];
            }
        };
        const auto stage = [&](int p, unsigned (&xs)[kMine][4 * W], const unsigned short (&scales)[kPacks][2], float (&acc)[4]) {
            const int mine = min(f.per, a.groups - p * (kStageK / kGroup) - g0);
            if (mbar_wait(BAR(B_FULL + st), ph, s_abort, g_err, 41u)) {
                const unsigned by = st * stage_bytes;
                unsigned both[kPacks];
#pragma unroll
                for (int i = 0; i < kPacks; i++) both[i] = (unsigned)scales[i][0] | (unsigned)scales[i][1] << 16;
                const auto group = [&](int i) {
                    unsigned wl[W], wh[W];
                    load_words<W>(at[i] + by, wl);
                    load_words<W>(at[i] + by + eight, wh);
                    float d[4];
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        unsigned vl[4], vh[4];
                        steps<T>::of(wl[w], vl);
                        steps<T>::of(wh[w], vh);
                        if (w == 0) mma_first<T>(d, vl[0], vh[0], vl[1], vh[1], xs[i][0], xs[i][1]);
                        else type<T>::mma(d, vl[0], vh[0], vl[1], vh[1], xs[i][4 * w], xs[i][4 * w + 1]);
                        type<T>::mma(d, vl[2], vh[2], vl[3], vh[3], xs[i][4 * w + 2], xs[i][4 * w + 3]);
                    }
                    const unsigned s = __shfl_sync(0xffffffffu, both[i / 4], (lane & 28) | (i & 3));
                    const float s0 = unpack<T>(s, false), s1 = unpack<T>(s, true);
                    acc[0] = fmaf(s0, d[0], acc[0]); acc[1] = fmaf(s0, d[1], acc[1]);
                    acc[2] = fmaf(s1, d[2], acc[2]); acc[3] = fmaf(s1, d[3], acc[3]);
                };
                /* (without branches between them the groups' chains overlap) */
                if (mine == kMine) {
#pragma unroll
                    for (int i = 0; i < kMine; i++) group(i);
                } else {
#pragma unroll
                    for (int i = 0; i < kMine; i++) if (i < mine) group(i);
                }
            }
            __syncwarp();
            /* (an arrival does not wait for loads that are under way, so it takes something of the sums that they went into) */
            if (lane == 0) mbar_arrive(BAR(B_EMPTY + st) + ((__float_as_uint(acc[0]) | __float_as_uint(acc[2])) & f.zero));
            if (++st == f.stages) { st = 0; ph ^= 1u; }
        };
        int turn = 0;
        /* a tile with its scales in set `now`, those of the tile kAhead further on to set `ahead`; false: given up */
        const auto tile = [&](int o0, unsigned short (&now)[kSets][kPacks][2], unsigned short (&ahead)[kSets][kPacks][2]) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            if (P) {
#pragma unroll
                for (int p = 0; p < kSets; p++) fetch(o0 + kAhead * kTile, p, ahead[p]);
#pragma unroll
                for (int p = 0; p < kSets; p++) stage(p, x[p], now[p], acc);
            } else {
                for (int p = 0; p < f.passes; p++) {
                    fetch(o0, p, now[0]);
#pragma unroll
                    for (int i = 0; i < kMine; i++) load_x<T, W>(row, g < rows && i < f.per, p * kStageK + (g0 + i) * kGroup, a.width, x[0][i]);
                    stage(p, x[0], now[0], acc);
                }
            }
            const int buf = turn % kParts;
            if (turn >= kParts && !mbar_wait(BAR(B_TAKEN + buf), (turn / kParts - 1) & 1, s_abort, g_err, 43u)) return false;
            float *const part = reinterpret_cast<float *>(sm + kOffPart) + (buf * kWarps + warp) * kPart;       /* [output][row] */
            *reinterpret_cast<float2 *>(part + mine_of * kRows + 2 * t) = make_float2(acc[0], acc[1]);
            *reinterpret_cast<float2 *>(part + (mine_of + 8) * kRows + 2 * t) = make_float2(acc[2], acc[3]);
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(B_READY + buf));
            turn++;
            return true;
        };
        if (P) {
#pragma unroll
            for (int i = 0; i < kAhead; i++)
#pragma unroll
                for (int p = 0; p < kSets; p++) fetch(first + i * kTile, p, sc[i][p]);
        }
        for (int o0 = first; o0 < last; o0 += (kAhead + 1) * kTile) {
            bool more = true;
#pragma unroll
            for (int i = 0; i <= kAhead; i++) more = more && o0 + i * kTile < last && tile(o0 + i * kTile, sc[i], sc[(i + kAhead) % (kAhead + 1)]);
            if (!more) break;
        }
    }
    if (*s_abort) for (int i = 0; i < 10000; i++) __nanosleep(1000);      /* copies of a stage that was given up are still on their way */
#undef BAR
}

template <class T, int W, int P>
cudaError_t launch(const CUtensorMap &tm, few_args f, int device, int sms, void *stream) {
    constexpr int kWarps = 16;
    static std::atomic<bool> ready[64];       /* shared memory allowed, per device */
    cudaError_t e;
    f.per = (f.in_stage + kWarps - 1) / kWarps;
    if (device >= 64 || !ready[device].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(hy3a_linear4_kernel<T, W, P, kWarps>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)) != cudaSuccess) return e;
        if (device < 64) ready[device].store(true, std::memory_order_release);
    }
    const int boxes = (f.a.out_width + kBox - 1) / kBox;
    hy3a_launch l(dim3(boxes < sms ? boxes : sms, (f.a.rows + kRows - 1) / kRows), dim3(32 * (kWarps + 2)), kSmem, stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_linear4_kernel<T, W, P, kWarps>, tm, f);
}
template <class T, int W>
cudaError_t launch_group(const CUtensorMap &tm, const few_args &f, int device, int sms, void *stream) {
    if (f.passes == 1) return launch<T, W, 1>(tm, f, device, sms, stream);
    constexpr int kTwo = W == 1 ? 0 : 2;       /* (short groups leave no registers) */
    return f.passes == 2 ? launch<T, W, kTwo>(tm, f, device, sms, stream) : launch<T, W, 0>(tm, f, device, sms, stream);
}
template <class T>
cudaError_t launch_few(const linear4_args &a, int device, int sms, void *stream, const char **what) {
    const int k = a.width < kStageK ? a.width : kStageK, bytes = a.width / 2;
    few_args f = {a, (k / 2 + kLine - 1) / kLine, 0, 0, (a.width + kStageK - 1) / kStageK, (k + a.group - 1) / a.group, 0, bytes % kLine == 0, 0u};
    f.box_bytes = (f.lines | 1) * kBox * kLine;
    f.stages = kRingBytes / (kTile / kBox * f.box_bytes);
    if (f.stages > kMaxStages) f.stages = kMaxStages;
    /* rows of whole lines: [lines][outputs][128 bytes], all lines of a stage in a copy; else [outputs][bytes], a line in a copy */
    CUtensorMap tm;
    const encode_tiled_fn enc = encoder();
    const cuuint64_t dims[3] = {(cuuint64_t)(f.whole ? kLine : bytes), (cuuint64_t)a.out_width, (cuuint64_t)(f.whole ? bytes / kLine : 1)}, strides[2] = {(cuuint64_t)bytes, (cuuint64_t)(f.whole ? kLine : 16)};
    const cuuint32_t box[3] = {kLine, kBox, (cuuint32_t)(f.whole ? f.lines : 1)}, one[3] = {1, 1, 1};
    if (!enc || enc(&tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(a.codes), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
        *what = "no tensor map (cuTensorMapEncodeTiled)";
        return cudaErrorInvalidValue;
    }
    if (a.group == 32) return launch_group<T, 1>(tm, f, device, sms, stream);
    if (a.group == 64) return launch_group<T, 2>(tm, f, device, sms, stream);
    return launch_group<T, 4>(tm, f, device, sms, stream);
}

} /* namespace */

int hy3a_quant4_sizes(const char *who, int out_width, int width, int group) {
    if (out_width < 0) return hy3a_fail(NULL, HY3A_EINVAL, "%s: out_width %d < 0", who, out_width);
    if (width < 32 || width > kMaxWidth || width % 32) return hy3a_fail(NULL, HY3A_EINVAL, "%s: width %d: a multiple of 32 in [32,%d]", who, width, kMaxWidth);
    if (group != 32 && group != 64 && group != 128) return hy3a_fail(NULL, HY3A_EINVAL, "%s: group %d not in {32,64,128}", who, group);
    return HY3A_OK;
}

extern "C" int hy3a_linear4(void *stream, int dtype, int rows, int width, int out_width, int group, const void *x, size_t x_stride, const void *codes, const void *scales,
                            int out_dtype, void *out, size_t out_stride) {
    if (dtype != HY3A_F16 && dtype != HY3A_BF16) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: dtype %d not in {1,2}", dtype);
    if (out_dtype != dtype && out_dtype != HY3A_F32) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: out_dtype %d is neither the rows' nor fp32", out_dtype);
    if (rows < 0) return hy3a_fail(NULL, HY3A_EINVAL, "linear4: rows %d < 0", rows);
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
    const cudaError_t e = rows > kRows ? hy3a_linear4_launch_many(a, dtype, dev, sms, stream, &what)
                        : (dtype == HY3A_BF16 ? launch_few<__nv_bfloat16>(a, dev, sms, stream, &what) : launch_few<__half>(a, dev, sms, stream, &what));
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "linear4: %s", what ? what : cudaGetErrorString(e));
    return HY3A_OK;
}

static __global__ void hy3a_linear4_wait_out_kernel() { wait_out(g_err, 49u); }
cudaError_t hy3a_linear4_wait_out(void *stream) {
    hy3a_linear4_wait_out_kernel<<<1, 1, 0, (cudaStream_t)stream>>>();
    return cudaGetLastError();
}
cudaError_t hy3a_linear4_error(unsigned *err) {
    const unsigned none[2] = {0, 0};
    cudaError_t e = cudaMemcpyFromSymbol(err, g_err, sizeof(none));
    if (e == cudaSuccess && err[0]) return cudaMemcpyToSymbol(g_err, none, sizeof(none));
    return e == cudaSuccess ? hy3a_linear4_many_error(err) : e;
}

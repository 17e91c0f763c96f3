/*
 * linear4.cu -- rows through a matrix of 4-bit codes with a scale for each group of neighbours in a row (hy3a_linear4), few rows:
 *
 *      y[t][o] = sum over groups j of scales[o][j] * sum over k of group j of (code[o][k] - 8) x[t][k]
 *
 * The inner sums are warp-level products (mma.m16n8k16, fp32 sums) of 16 outputs with 8 rows: the differences are exact in the rows' type and so are the
 * products; the scale of a group multiplies its sum in fp32.  Nothing is rounded to fewer bits before the result.
 *
 * A block takes a contiguous part of the outputs (all parts alike to one output), in tiles of 16, and streams their codes through a ring of shared memory: a
 * stage is a tile's codes for 4096 k's (or all, where there are fewer), each output's by a bulk copy of its own, so that all blocks have 100 KB and more under way, and its scales in words
 * (cp.async: their rows start anywhere).  The 16 warps share the k's; each keeps its part of x in registers for the whole launch.  Their sums meet in shared memory.
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

constexpr int kWarps = 16, kThreads = 32 * (kWarps + 1), kTile = 16 /* outputs */, kRows = 8, kStageK = 4096, kMaxStages = 16, kMaxWidth = 1 << 16;
constexpr int kRingBytes = 200 * 1024, kOffBar = 0, kOffPart = 512, kPartPitch = kTile * kRows, kOffRing = kOffPart + 2 * kWarps * kPartPitch * 4;

__device__ unsigned g_err[2];         /* {code, where} of the first wait that ran out, until hy3a_layer_sync reads it */

struct few_args {
    linear4_args a;
    int pitch /* bytes of an output's codes in a stage */, scale_pitch /* words of its scales */, stage_bytes, stages, passes /* stages of a tile */;
};

__device__ __forceinline__ void bulk_copy(unsigned dst, const void *src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(0x12F0000000000000ull) /* evict first */ : "memory");
}
__device__ __forceinline__ void copy_word(unsigned dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void arrive_behind_copies(unsigned bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
template <class T> __device__ __forceinline__ float scale_at(unsigned addr) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
    return type<T>::up(*reinterpret_cast<const T *>(&v));
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
/* W words at an address of shared memory */
template <int W> __device__ __forceinline__ void load_words(unsigned addr, unsigned (&v)[W]) {
    if (W == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[W > 2 ? 2 : 0]), "=r"(v[W > 3 ? 3 : 0]) : "r"(addr));
    else if (W == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[W > 1 ? 1 : 0]) : "r"(addr));
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(addr));
}

/* W: words of a lane for a group; P: stages of a tile where x of all of them stays in registers, 0: x is read for each */
template <class T, int W, int P>
__global__ void __launch_bounds__(kThreads, 1) hy3a_linear4_kernel(const few_args f) {
    extern __shared__ __align__(128) uint8_t s_raw[];
    constexpr int kGroup = 32 * W, kMine = kStageK / kGroup / kWarps /* groups of a warp in a stage */, kSets = P ? P : 1;
    const linear4_args &a = f.a;
    __shared__ int s_abort_flag;
    volatile int *s_abort = &s_abort_flag;
    const unsigned sbase = smem_u32(s_raw), bar0 = sbase + kOffBar, ring = sbase + kOffRing;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int first = (int)((long long)a.out_width * blockIdx.x / gridDim.x), last = (int)((long long)a.out_width * (blockIdx.x + 1) / gridDim.x);
    const int t0 = blockIdx.y * kRows, rows = min(kRows, a.rows - t0);
#define FULL(i) (bar0 + 8u * (unsigned)(i))
#define EMPTY(i) (bar0 + 8u * (unsigned)(kMaxStages + (i)))
    if (tid == 0) {
        s_abort_flag = 0;
        for (int i = 0; i < f.stages; i++) { mbar_init(FULL(i), 33); mbar_init(EMPTY(i), kWarps); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_release();
    pdl_wait();
    int st = 0;
    unsigned ph = 0;
    if (warp == kWarps) {
        /* ===================== producer ===================== */
        bool ok = true;
        const T *scales = reinterpret_cast<const T *>(a.scales);
        for (int o0 = first; o0 < last && ok; o0 += kTile) {
            const int n = min(kTile, last - o0);
            for (int p = 0; p < f.passes; p++) {
                if (!(ok = mbar_wait(EMPTY(st), ph ^ 1u, s_abort, g_err, 40u))) break;
                const unsigned to = ring + st * f.stage_bytes;
                const unsigned bytes = (unsigned)min(kStageK, a.width - p * kStageK) / 2;
                if (lane == 0) mbar_expect_tx(FULL(st), n * bytes);
                __syncwarp();
                if (lane < n) bulk_copy(to + lane * f.pitch, a.codes + (size_t)(o0 + lane) * (a.width / 2) + p * (kStageK / 2), bytes, FULL(st));
                const int j0 = p * (kStageK / kGroup), count = min(kStageK / kGroup, a.groups - j0);
                for (int r = 0; r < n; r++) {
                    const uintptr_t at = (uintptr_t)(scales + (size_t)(o0 + r) * a.groups + j0);
                    const int words = (int)(((at & 3) + 2 * count + 3) >> 2);
                    for (int i = lane; i < words; i += 32) copy_word(to + kTile * f.pitch + (r * f.scale_pitch + i) * 4, reinterpret_cast<const void *>((at & ~(uintptr_t)3) + 4 * i));
                }
                arrive_behind_copies(FULL(st));
                if (++st == f.stages) { st = 0; ph ^= 1u; }
            }
        }
    } else {
        /* ===================== products ===================== */
        unsigned x[kSets][kMine][4 * W];
        const T *row = reinterpret_cast<const T *>(a.x) + (size_t)(t0 + min(g, rows - 1)) * a.x_stride;
        if (P) {
#pragma unroll
            for (int p = 0; p < kSets; p++)
#pragma unroll
                for (int i = 0; i < kMine; i++) load_x<T, W>(row, g < rows, p * kStageK + (warp + kWarps * i) * kGroup, a.width, x[p][i]);
        }
        bool ok = true;
        int turn = 0;
        for (int o0 = first; o0 < last; o0 += kTile, turn++) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            const auto stage = [&](int p, unsigned (&xs)[kMine][4 * W]) {
                ok = ok && mbar_wait(FULL(st), ph, s_abort, g_err, 41u);
                if (ok) {
                    const unsigned at = ring + st * f.stage_bytes, lo = at + g * f.pitch + t * 4 * W;
                    const uintptr_t s_lo = (uintptr_t)(reinterpret_cast<const T *>(a.scales) + (size_t)(o0 + g) * a.groups + p * (kStageK / kGroup)), s_hi = s_lo + (size_t)8 * a.groups * 2;
                    const unsigned sc = at + kTile * f.pitch, sc_lo = sc + g * f.scale_pitch * 4 + (unsigned)(s_lo & 2), sc_hi = sc + (g + 8) * f.scale_pitch * 4 + (unsigned)(s_hi & 2);
#pragma unroll
                    for (int i = 0; i < kMine; i++) {
                        const int j = warp + kWarps * i;
                        if (p * kStageK + j * kGroup < a.width) {
                            unsigned wl[W], wh[W];
                            load_words<W>(lo + j * 16 * W, wl);
                            load_words<W>(lo + 8 * f.pitch + j * 16 * W, wh);
                            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int w = 0; w < W; w++) {
                                unsigned vl[4], vh[4];
                                steps<T>::of(wl[w], vl);
                                steps<T>::of(wh[w], vh);
                                type<T>::mma(d, vl[0], vh[0], vl[1], vh[1], xs[i][4 * w], xs[i][4 * w + 1]);
                                type<T>::mma(d, vl[2], vh[2], vl[3], vh[3], xs[i][4 * w + 2], xs[i][4 * w + 3]);
                            }
                            const float s0 = scale_at<T>(sc_lo + 2 * j), s1 = scale_at<T>(sc_hi + 2 * j);
                            acc[0] = fmaf(s0, d[0], acc[0]); acc[1] = fmaf(s0, d[1], acc[1]);
                            acc[2] = fmaf(s1, d[2], acc[2]); acc[3] = fmaf(s1, d[3], acc[3]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(EMPTY(st));
                if (++st == f.stages) { st = 0; ph ^= 1u; }
            };
            if (P) {
#pragma unroll
                for (int p = 0; p < kSets; p++) stage(p, x[p]);
            } else {
                for (int p = 0; p < f.passes; p++) {
#pragma unroll
                    for (int i = 0; i < kMine; i++) load_x<T, W>(row, g < rows, p * kStageK + (warp + kWarps * i) * kGroup, a.width, x[0][i]);
                    stage(p, x[0]);
                }
            }
            /* the warps' sums, [output][row], added up in the warps' order by four warps of them, others for each tile */
            float *const part = reinterpret_cast<float *>(s_raw + kOffPart) + (turn & 1) * kWarps * kPartPitch;
            *reinterpret_cast<float2 *>(part + warp * kPartPitch + g * kRows + 2 * t) = make_float2(acc[0], acc[1]);
            *reinterpret_cast<float2 *>(part + warp * kPartPitch + (g + 8) * kRows + 2 * t) = make_float2(acc[2], acc[3]);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
            if ((warp >> 2) == (turn & 3)) {
                const int q = (warp & 3) * 32 + lane, o = q & 15, r = q >> 4;
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) sum += part[w * kPartPitch + o * kRows + r];
                if (r < rows && o0 + o < last) {
                    const size_t to = (size_t)(t0 + r) * a.out_stride + o0 + o;
                    if (a.wide) reinterpret_cast<float *>(a.out)[to] = sum;
                    else reinterpret_cast<T *>(a.out)[to] = type<T>::down(sum);
                }
            }
        }
    }
    if (*s_abort) for (int i = 0; i < 10000; i++) __nanosleep(1000);      /* copies of a stage that was given up are still on their way */
#undef FULL
#undef EMPTY
}

template <class T, int W, int P>
cudaError_t launch(const few_args &f, int device, int sms, void *stream) {
    static std::atomic<bool> ready[64];       /* shared memory allowed, per device */
    const int smem = kOffRing + kRingBytes;
    cudaError_t e;
    if (device >= 64 || !ready[device].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(hy3a_linear4_kernel<T, W, P>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
        if (device < 64) ready[device].store(true, std::memory_order_release);
    }
    hy3a_launch l(dim3(f.a.out_width < sms ? f.a.out_width : sms, (f.a.rows + kRows - 1) / kRows), dim3(kThreads), smem, stream);
    return cudaLaunchKernelEx(&l.cfg, hy3a_linear4_kernel<T, W, P>, f);
}
template <class T, int W>
cudaError_t launch_passes(const few_args &f, int device, int sms, void *stream) {
    return f.passes == 1 ? launch<T, W, 1>(f, device, sms, stream) : (f.passes == 2 ? launch<T, W, 2>(f, device, sms, stream) : launch<T, W, 0>(f, device, sms, stream));
}
template <class T>
cudaError_t launch_few(const linear4_args &a, int device, int sms, void *stream) {
    const int words = a.group / 32, k = a.width < kStageK ? a.width : kStageK;
    few_args f = {a, ((k / 2 + 127) & ~127) + 16 * words, ((k + a.group - 1) / a.group / 2 + 1) | 1, 0, 0, (a.width + kStageK - 1) / kStageK};
    f.stage_bytes = kTile * (f.pitch + 4 * f.scale_pitch);
    f.stages = kRingBytes / f.stage_bytes < kMaxStages ? kRingBytes / f.stage_bytes : kMaxStages;
    if (words == 1) return launch_passes<T, 1>(f, device, sms, stream);
    if (words == 2) return launch_passes<T, 2>(f, device, sms, stream);
    return launch_passes<T, 4>(f, device, sms, stream);
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
    const cudaError_t e = dtype == HY3A_BF16 ? launch_few<__nv_bfloat16>(a, dev, sms, stream) : launch_few<__half>(a, dev, sms, stream);
    if (e != cudaSuccess) return hy3a_fail(NULL, HY3A_ECUDA, "linear4: %s", cudaGetErrorString(e));
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
    if (e == cudaSuccess && err[0]) e = cudaMemcpyToSymbol(g_err, none, sizeof(none));
    return e;
}

/*
 * grouping.cuh -- lists items by a key, on one block or a cluster of blocks: slots by their expert (experts.cu), rows by their adapter
 * (adapters.cu).
 *
 * Each block counts its part of the items, all read all counts, and each lists its part.  STABLE: items of a key keep their order (the warps of a
 * block take their places one after another).  Otherwise an item's place within its key's list comes from an atomic and may differ from run to run;
 * what the callers compute of an item does not depend on it.
 */
#ifndef HY3A_GROUPING_CUH
#define HY3A_GROUPING_CUH

#include "layer.h"

namespace hy3a_layer {

constexpr int kGroupThreads = 1024, kGroupCluster = 8, kGroupShared = 4096;      /* items from which blocks share them: 65 536 take 37 us with one block, 12 with 8 */

__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int peer_int(const int *p, unsigned rank) {
    unsigned a = (unsigned)__cvta_generic_to_shared(p);
    int v;
    asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(a) : "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

/* key(i): 0 .. bins - 1, or -1 (left out); tiles of `tile` items.  bin(key, first place, items, first tile, tiles) once for each key (a thread of the
 * first block), put(item, place) for each item; returns the number of tiles.  bins <= 1024 BPT.  Reads begin behind the wait for the launch before. */
template <int BLOCKS, int BPT, bool STABLE, class Key, class Bin, class Put>
__device__ __forceinline__ int group_items(int items, int bins, int tile, const Key &key, const Bin &bin, const Put &put) {
    __shared__ int s_count[kGroupThreads * BPT], s_next[kGroupThreads * BPT], s_warp[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned me = BLOCKS > 1 ? cluster_rank() : 0;
    const int per = (items + BLOCKS - 1) / BLOCKS, begin = min(items, (int)me * per), end = min(items, begin + per);
    for (int e = tid; e < bins; e += kGroupThreads) s_count[e] = 0;
    __syncthreads();
    pdl_wait();
#pragma unroll 4
    for (int i = begin + tid; i < end; i += kGroupThreads) {
        const int e = key(i);
        if (e >= 0) atomicAdd(&s_count[e], 1);
    }
    __syncthreads();
    if (BLOCKS > 1) { cluster_arrive(); cluster_wait(); }
    /* a thread has BPT neighbouring keys: their items, those of the blocks before this one, their tiles; exclusive sums over the keys */
    int n[BPT], earlier[BPT], sum[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < BPT; k++) {
        const int e = tid * BPT + k;
        n[k] = earlier[k] = 0;
        if (e < bins) {
            if (BLOCKS == 1) n[k] = s_count[e];
            else {
#pragma unroll
                for (int r = 0; r < BLOCKS; r++) {
                    const int c = peer_int(&s_count[e], r);
                    n[k] += c;
                    if (r < (int)me) earlier[k] += c;
                }
            }
        }
        sum[0] += n[k];
        sum[1] += (n[k] + tile - 1) / tile;
    }
    const int own[2] = {sum[0], sum[1]};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int u = __shfl_up_sync(0xffffffffu, sum[i], o);
            if (lane >= o) sum[i] += u;
        }
#pragma unroll
    for (int i = 0; i < 2; i++) if (lane == 31) s_warp[i][warp] = sum[i];
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        int w = s_warp[i][lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        if (i == 1) total = __shfl_sync(0xffffffffu, w, 31);
        const int before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
        sum[i] += (warp ? before : 0) - own[i];
    }
#pragma unroll
    for (int k = 0; k < BPT; k++) {
        const int e = tid * BPT + k, tiles = (n[k] + tile - 1) / tile;
        if (e < bins) {
            s_next[e] = sum[0] + earlier[k];          /* where the block's next item of the key goes */
            if (me == 0) bin(e, sum[0], n[k], sum[1], tiles);
        }
        sum[0] += n[k];
        sum[1] += tiles;
    }
    __syncthreads();
    if (STABLE) {
        for (int i0 = begin; i0 < end; i0 += kGroupThreads) {
            const int i = i0 + tid, e = i < end ? key(i) : -1, warps = min(kGroupThreads, end - i0 + 31) >> 5;
            const unsigned same = __match_any_sync(0xffffffffu, e);
            const int lead = __ffs(same) - 1;
            int p = 0;
            for (int w = 0; w < warps; w++) {
                if (w == warp && lane == lead && e >= 0) { p = s_next[e]; s_next[e] = p + __popc(same); }
                __syncthreads();
            }
            p = __shfl_sync(0xffffffffu, p, lead) + __popc(same & ((1u << lane) - 1u));
            if (e >= 0) put(i, p);
        }
    } else {
#pragma unroll 4
        for (int i = begin + tid; i < end; i += kGroupThreads) {
            const int e = key(i);
            if (e >= 0) put(i, atomicAdd(&s_next[e], 1));
        }
    }
    __syncthreads();
    if (BLOCKS > 1) { cluster_arrive(); cluster_wait(); }           /* nobody leaves while its counts are read */
    return total;
}

} /* namespace hy3a_layer */
#endif

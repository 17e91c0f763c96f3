/* experts.h -- what the kernels of hy3a_experts share: their arguments, and the table of slot tiles (experts.cu, experts_umma.cu). */
#ifndef HY3A_EXPERTS_H
#define HY3A_EXPERTS_H

#include "layer.h"

/* The tiles of one expert's slots stand one behind another in the table, with the same contents. */
struct expert_tile {
    int expert, first /* index of the expert's first tile */, tiles, p0 /* first listed slot */, count /* slots */;
};
constexpr int kTileSlots = 256;       /* most slots of a tile */

struct expert_args {
    const void *x;
    size_t x_stride;
    const int *ids;
    const float *weights;
    const void *gate, *up, *down;
    void *out;
    size_t out_stride;
    int rows, top_k, hidden, inter, held, first, slots;
    int *row, *place;   /* [slots] rows of the listed slots, expert by expert; where each slot is in that list (-1: not) */
    expert_tile *tiles; /* [*n_tiles] */
    int *n_tiles;
    void *h;            /* [slots][inter], in the order of the list (few slots: of the slots, and as much again, the rest) */
    short *q;           /* [slots][hidden], in the order of the list: y in 16 bits; with 2^e the power of two below the largest magnitude of 32 neighbours, multiples of 2^(e - 14) */
    float *q_scale;     /* [slots][hidden / 32, rounded up] that scale */
};
/* y is written and read once between two launches, and at many slots that is what these take: 8192 slots of 4096 are 134 MB in fp32.  16 bits of
 * fixed point leave at most 2^-15 of the largest neighbour, a hundredth of what the rounding of a bf16 result leaves and a tenth of an fp16
 * one's.  Neighbours that are not all finite are kept as bf16 instead (scale -1), so that infinities and NaN stay where they are; a largest
 * magnitude below 2^-100 counts as 0. */

/* Both products on tcgen05 (many slots per expert). */
cudaError_t hy3a_experts_launch_umma(const expert_args &a, int dtype, int device, int sms, void *stream, const char **what);

#endif

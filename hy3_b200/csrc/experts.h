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
    int *off;           /* [held + 1] first listed slot of each expert */
    int *active;        /* [0] number of experts with slots, [1..] which */
    int *slot, *row;    /* [slots] listed slots, expert by expert, and the rows that they belong to */
    expert_tile *tiles; /* [*n_tiles] */
    int *n_tiles;
    void *h;            /* [slots][inter], in the order of the list */
    float *y;           /* [slots][hidden], in the order of the slots */
};

/* Both products on tcgen05 (many slots per expert). */
cudaError_t hy3a_experts_launch_umma(const expert_args &a, int dtype, int device, int sms, void *stream, const char **what);

#endif

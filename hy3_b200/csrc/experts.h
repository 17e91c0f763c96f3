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
    void *h;            /* [slots][inter] of the rows' type, in the order of the list (few slots: of the slots, and as much again, the rest) */
    float *wide;        /* fp16: [slots][inter] h as it was computed (its room is y's, which comes later) */
    float *back;        /* fp16: [slots] what y is multiplied with */
    float *y;           /* [slots][hidden], in the order of the list */
};
/* y stays in fp32 between the launches.  It is written and read once, and at many slots that is what these take (8192 slots of 4096 are 134 MB), but fewer
 * bits lose what the result needs: 16 bits of fixed point on a scale that 32 neighbouring columns share gained 3 % (2048 rows of 192 experts, 8 each, in a
 * loop 1284 us instead of 1248; a share of 24 of them 347 to 365 instead of 340 to 359), and left a column beside one 1024 times as large eight bf16 roundings
 * short. */

/* Between gate / up and down of fp16 rows: h = wide * 2^n with a largest value in [2^14, 2^15) for each listed slot, back = 2^-n (experts.cu). */
cudaError_t hy3a_experts_launch_range(const expert_args &a, int sms, void *stream);
/* Both products on tcgen05 (many slots per expert). */
cudaError_t hy3a_experts_launch_umma(const expert_args &a, int dtype, int device, int sms, void *stream, const char **what);

#endif

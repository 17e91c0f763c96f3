/*
 * linear4_plan.h -- how linear4_umma.cu cuts rows and k's into tiles (host code, no CUDA).
 *
 * A pair of CTAs has tiles of 256 outputs with `columns` rows, the N of tcgen05.mma: from 32 in steps of 32, as a product of two CTAs with 256 outputs whose A lies in tensor memory has it. What is
 * rounded up are rows of zeros, and not stored.
 */
#ifndef HY3A_LINEAR4_PLAN_H
#define HY3A_LINEAR4_PLAN_H

#ifdef __CUDACC__
#define HY3A_ANYWHERE __host__ __device__
#else
#define HY3A_ANYWHERE
#endif

constexpr int kLinear4Splits = 4;                                            /* CTA pairs that share a tile's k's, at most */
constexpr int kLinear4Steps = 12;                                            /* stages of x and A, at most, */
constexpr int kLinear4Units = 8;                                             /* of 128 k's, two steps: codes in shared memory */
constexpr int kLinear4XBytes = 8 * 128 * 128;                                /* as shared memory has room for x */
constexpr int kLinear4Tmem = 512;                                            /* columns of tensor memory: sums (two of them for fp32 results), then the stages of A */

struct linear4_plan {
    int columns;              /* rows of a tile */
    long long tiles;
    int splits;               /* pairs of a tile */
    int steps;                /* stages of x (columns / 2 rows of 128 bytes a CTA) and of A */
    int a_column;             /* where those of A begin in tensor memory */
};
static inline int linear4_a_columns(bool wide) { return wide ? 64 : 32; }    /* of a stage of A: 64 k's, once or (wide: fp32 results) in two numbers */

/* Warps that make A work in teams, each of which takes every teams-th step of all that a pair has, through the ends of tiles: a team's first step in the tile after one of `steps` steps where its first was `before`
 * (it may lie past the tile's last).  A team does not see every phase of a barrier, and a wait for a phase's parity is also over two phases before it.  What rules that out: at step k, g = teams steps after the one
 * before, it has seen the product of step k - g - stages over; a stage of A and x is given back every `stages` steps, and a unit of codes comes every 2 kLinear4Units, so that the phases before those waited for are
 * over if g <= stages and g + stages <= 2 kLinear4Units.  (Teams that began each tile anew had steps up to 2 teams - 1 apart: 5 with 4 stages.) */
HY3A_ANYWHERE constexpr int linear4_teams(bool wide) { return wide ? 3 : 4; }
HY3A_ANYWHERE constexpr int linear4_first_step(int before, int steps, int teams) { return ((before - steps) % teams + teams) % teams; }

/* Rows of a tile and CTAs that share a tile's k's: what takes the least, in 10 ns, measured over 9 to 2048 rows: a step takes 160 + 0.6 N ns with N rows (fp32 results 220 + 0.9 N), a launch 6.5 us besides
 * (8.5; 1.5 more where CTAs share).  Pairs that have several tiles begin the next one's copies, and with fp32 results its products too, before the last one's results are stored: 2 us a tile (2698 rows on
 * 16942 x 448 in fp32 98 to 117 us, and 249 with a launch's start and end for each; 2048 on 4096 x 8192 in bf16 100 and 102).  units: of 128 k's; fit: clusters of 1 .. kLinear4Splits pairs at once. */
static inline linear4_plan linear4_plan_of(int rows, int m_tiles, int units, bool wide, const int (&fit)[kLinear4Splits]) {
    linear4_plan p = {};
    const int most = wide ? 128 : 256, least_tiles = (rows + most - 1) / most;
    double least = -1.;
    for (int n = least_tiles; n <= least_tiles + 4; n++) {
        const int columns = ((rows + n - 1) / n + 31) & ~31;
        const long long all = (long long)((rows + columns - 1) / columns) * m_tiles;
        for (int splits = 1; splits <= kLinear4Splits && splits <= units; splits++) {
            const int steps = 2 * ((units + splits - 1) / splits);
            const double rounds = (double)((all + fit[splits - 1] - 1) / fit[splits - 1]), once = wide ? 850. : 650., step = wide ? 22. + 0.09 * columns : 16. + 0.06 * columns;
            const double cost = splits == 1 ? rounds * (steps * step + 200.) + once - 200. : rounds * (steps * step + once + 150.);
            if (least < 0. || cost < least) { least = cost; p.tiles = all; p.columns = columns; p.splits = splits; }
        }
    }
    p.steps = (kLinear4Tmem - (wide ? 2 : 1) * p.columns) / linear4_a_columns(wide);
    const int room = kLinear4XBytes / (p.columns * 64);
    if (p.steps > room) p.steps = room;
    if (p.steps > kLinear4Steps) p.steps = kLinear4Steps;
    p.a_column = kLinear4Tmem - p.steps * linear4_a_columns(wide);
    return p;
}

#endif

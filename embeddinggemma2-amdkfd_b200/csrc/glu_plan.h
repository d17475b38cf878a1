// How the gated projection's launches share out their work, and what its
// gradient's workspace holds.  Plain host arithmetic on sizes, without CUDA.
#pragma once
#include <limits.h>
#include <stdint.h>

namespace eg2 {

static inline int glu_ceil(long long a, long long b) { return int((a + b - 1) / b); }
static inline int glu_tiles(unsigned rows, unsigned cols, int bn) { return glu_ceil(rows, 256) * glu_ceil(cols, bn); }

// What the choices below weigh, in hundredths of a K step of 64 with a 256-column
// tile (measured: 0.35 us): a step with tiles of 64, 128 and 256 columns (the
// tensor cores take nearly as long for the narrow ones), and a tile's epilogue
// (3.1 us at 256), which runs under the next tile's steps but for the last one's.
constexpr int GLU_STEP_COST[3] = {85, 90, 100}, GLU_EPI_COST[3] = {230, 450, 900};
static inline long long glu_cost(long long tiles, int steps, int width, int clusters) {
    const long long step = (long long)steps * GLU_STEP_COST[width], epi = GLU_EPI_COST[width];
    return tiles ? (tiles + clusters - 1) / clusters * (step > epi ? step : epi) + epi : 0;
}
// The projections' gradients are operands of the products that follow, rounded once to
// 16 bits; that adds as much error as the rounding of the results.  Over many
// elements the two add up to 1.41 times the latter, over few they need not: with few
// elements in dG and dU (n m), or few in dx (n k), whose own rounding then varies, a
// call could be up to 1.96 times as far from 64 bits as a form in fp32.  There each
// is two operands, the rounded value and what the rounding left, and the products' K
// is twice as long.  The borders: dw was more than 1.5 times as far in 6 of 1757 calls
// with n m in 4096 .. 5791 and in none of 13800 above, dx in 81 of 1711 with n k in
// 256 .. 1023, in 9 of 1622 in 1024 .. 2047 (up to 1.55) and in 2 of 13000 above.  At
// 2 x 80 x 392 two operands take 13.6 us where one took 13.1, at 1 x 512 x 2048 20.6
// and 17.3.
static inline int glu_halves(unsigned n, unsigned k, unsigned m) {
    return uint64_t(n) * m < 6144 || uint64_t(n) * k < 1024 ? 2 : 1;
}

// The backward products' plan: dx's K in `splits` parts, and `dxc` clusters for
// dx, so that the slowest cluster is done first.  Parts cost a launch that adds them.
struct GluPlan {
    int splits, dxc;  // dxc < 0: all clusters take dx's tiles and then the weights'
};
constexpr int GLU_PAIRS = 74;   // what workspaces are sized for: a whole device
constexpr int GLU_MOST = 8;     // parts
// For `pairs` clusters; `most` bounds the parts.  Fewer clusters can want more
// parts than a whole device does, so a launch passes what the workspace was
// sized for (glu_most_splits).
static inline GluPlan glu_plan(unsigned n, unsigned k, unsigned m, bool dx, int weights, int pairs, int most) {
    const long long td = dx ? glu_tiles(n, k, 256) : 0, tw = weights * (long long)glu_tiles(m, k, 256);
    const int sd = 2 * glu_ceil(m, 64) * glu_halves(n, k, m), sw = glu_ceil(n, 64) * glu_halves(n, k, m);
    if (td && tw && pairs < 2) return {1, -1};  // no cluster apiece
    GluPlan best{1, 0};
    long long least = LLONG_MAX;
    const int low = td ? 1 : 0, high = !td ? 0 : tw ? pairs - 1 : pairs;
    for (int splits = 1; splits <= (dx ? most : 1) && splits <= sd; splits *= 2) {
        // Parts: a launch to add them (900), and their floats written and read, 21000 bytes in a unit.
        const long long add = splits > 1 ? 900 + (long long)n * k * (8 * splits + 2) / 21000 : 0;
        int at = low;
        long long here = LLONG_MAX;
        const auto weigh = [&](int d) {
            if (d < low || d > high) return;
            const long long cd = td ? glu_cost(td * splits, glu_ceil(sd, splits), 2, d) : 0;
            const long long cw = tw ? glu_cost(tw, sw, 2, pairs - d) : 0, c = (cd > cw ? cd : cw) + add;
            if (c < here) here = c, at = d;
        };
        for (int d = low; d <= high; d += 4) weigh(d);  // coarsely, then around the best
        for (int d = at - 3, end = at + 3; d <= end; ++d) weigh(d);
        if (here < least) least = here, best = {splits, at};
    }
    // One after the other on all clusters, where the slowest is not later for it:
    // 8203 x 2048 x 8192 reads 1.1 GB from memory in that order (with tiles in bands of
    // 8 it was 1.6 GB, and 1.9 GB side by side).
    if (td && tw) {
        long long worst = 0;
        const long long cd = glu_cost(1, sd, 2, 1) - GLU_EPI_COST[2], cw = glu_cost(1, sw, 2, 1) - GLU_EPI_COST[2];
        for (int c = 0; c < pairs; ++c) {
            const long long mine = (td + tw - c + pairs - 1) / pairs, of_dx = c < td ? (td - c + pairs - 1) / pairs : 0;
            const long long t = of_dx * cd + (mine - of_dx) * cw + GLU_EPI_COST[2];
            if (t > worst) worst = t;
        }
        if (td + tw >= pairs && worst <= least + least / 50) best = {1, -1};
    }
    return best;
}
// The most parts that a whole device's plan takes for dx, alone or beside one or
// both weights' gradients.
static inline int glu_most_splits(unsigned n, unsigned k, unsigned m) {
    int most = 1;
    for (int w = 0; w <= 2; ++w) {
        const int s = glu_plan(n, k, m, true, w, GLU_PAIRS, GLU_MOST).splits;
        if (s > most) most = s;
    }
    return most;
}
// Workspace: dG and dU, what their roundings left where that is kept, then dx's parts.
static inline uint64_t glu_half(unsigned n, unsigned m) { return (uint64_t(n) * m * 2 + 255) / 256 * 256; }
static inline uint64_t glu_parts_at(unsigned n, unsigned k, unsigned m) { return 2 * glu_halves(n, k, m) * glu_half(n, m); }
static inline uint64_t glu_grad_bytes(unsigned n, unsigned k, unsigned m, int splits) {
    return glu_parts_at(n, k, m) + (splits > 1 ? uint64_t(splits) * n * k * 4 : 0);
}

}  // namespace eg2

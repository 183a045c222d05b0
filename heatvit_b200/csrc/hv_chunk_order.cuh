// hv_chunk_order.cuh — in which order chunk attention's copies fill its ring of tiles, and what a role may take as
// landed.  Plain constexpr functions, without CUDA, so that a host test can go through them.
#pragma once

#ifdef __CUDACC__
#define HV_ORDER __host__ __device__ constexpr
#else
#define HV_ORDER constexpr
#endif

namespace hv {
namespace chunk {

// Key (value) tiles of `parts` ring slots each, of `stages`; `row_tiles` in flight.  APART: a step's scores go ahead of the
// sums of the step before (they have tensor memory of their own), else behind them.
struct Order {
    bool apart;
    int parts, stages, row_tiles;

    // Which ring fill, from the segment's first, holds the keys (values) of its step j of n.  The keys of the first `lead`
    // steps come first, then those of step j + lead and the values of step j, in the order of their use: keys ahead
    // where scores go ahead of sums, else values.
    HV_ORDER static int lead_of(bool alt) { return alt ? 2 : 1; }
    HV_ORDER int k_fill(int j, int lead) const { return (j < lead ? j : 2 * j - lead + !apart) * parts; }
    HV_ORDER int v_fill(int j, int n, int lead) const { return (j + lead < n + !apart ? lead + 2 * j + apart : n + j) * parts; }

    // The products' warp takes units in turn: either row tile against each step's keys, or (alt) the one against the steps
    // in turn.  The scores of unit u are its turn 2 u, the sums of unit u stand `row_tiles` units behind them.
    HV_ORDER int scores_turn(int u) const { return 2 * u + !apart; }
    HV_ORDER int sums_turn(int u) const { return 2 * (u + row_tiles) + apart; }

    // A softmax warpgroup polls the barriers of a unit's value slots when it has seen that unit's scores and, with
    // `sums_ahead`, the sums of its row tile's unit before.  A barrier whose parity is polled has to be past the
    // slot's earlier fill, or the poll ends on the fill before that: is that fill landed, by the waits of the products'
    // warp up to there, in every step of segments of up to `most` steps?
    HV_ORDER bool values_may_be_polled(bool sums_ahead, int most) const {
        for (int alt = 0; alt < row_tiles; ++alt) {
            const bool pair = row_tiles == 2 && !alt;
            const int lead = lead_of(alt), per = pair ? 2 : 1;  // units of a step
            for (int n = 1; n <= most; ++n)
                for (int u = 0; u < n * per; ++u) {
                    int known = scores_turn(u);
                    if (sums_ahead && u >= row_tiles && sums_turn(u - row_tiles) > known) known = sums_turn(u - row_tiles);
                    for (int p = 0; p < parts; ++p) {
                        const int before = v_fill(u / per, n, lead) + p - stages;
                        if (before < 0) continue;  // of an earlier segment, which is through
                        bool landed = false;       // it has been waited for with the step that it belongs to
                        for (int j = 0; j < n; ++j) {
                            const int k = before - k_fill(j, lead), v = before - v_fill(j, n, lead);
                            landed = landed || (k >= 0 && k < parts && scores_turn(j * per) <= known) ||
                                     (v >= 0 && v < parts && sums_turn(j * per) <= known);
                        }
                        if (!landed) return false;
                    }
                }
        }
        return true;
    }
};

// Heads of D dimensions.
HV_ORDER int padded_dim(int d) { return (d + 63) / 64 * 64; }
HV_ORDER Order order_of(int d) {
    const int dp = padded_dim(d);
    return {d > 128 || dp == 64, dp <= 128 ? 1 : 2, dp == 64 ? 8 : dp == 128 ? 5 : dp == 192 ? 7 : 5, d <= 128 ? 2 : 1};
}

}  // namespace chunk
}  // namespace hv

// Which rows of a batch are a sequence's, and which positions a tile of them sees. Plain arithmetic, shared by the attention
// kernels and a host test: the starts and lengths are the caller's data, and whatever they hold, a row that comes out lies in
// the row arrays and no difference or product wraps.
#pragma once
#include <stdint.h>

#ifndef TLLM_HD
#if defined(__HIPCC__)
#define TLLM_HD __host__ __device__ __forceinline__
#else
#define TLLM_HD inline
#endif
#endif

namespace tllm {

TLLM_HD int lower_of(int a, int b) { return a < b ? a : b; }
TLLM_HD int higher_of(int a, int b) { return a > b ? a : b; }

struct SequenceRows {
    int row0, rows, pos0;  // first row, rows, position of the first row
};
// Rows s0 .. s1 - 1 of n_tokens, max_query of them at most; row s1 - 1 is position length - 1. Starts that do not rise inside
// the row arrays have no rows (decided before any difference is taken: s1 - s0 may be any 33-bit number).
TLLM_HD SequenceRows sequence_rows(int s0, int s1, int length, int n_tokens, int max_query) {
    if (s0 < 0 || s0 >= n_tokens || s1 <= s0) return SequenceRows{0, 0, 0};
    // (the last row's position is below `length`; rows are fewer than 2^24, so from -2^25 on none reaches position 0)
    const long long pos = (long long)length - s1 + s0;
    return SequenceRows{s0, lower_of(lower_of(s1, n_tokens) - s0, max_query), (int)(pos < -(1 << 25) ? -(1 << 25) : pos)};
}

// First position that a row at position pos (>= -1) sees.
TLLM_HD int window_begin(int window, int pos) { return window > 0 ? higher_of(0, pos - window + 1) : 0; }

struct TileSpan {
    int rows_left;          // rows of the sequence (times heads) from the tile's first on; <= 0: the tile has none
    int pos_low, pos_high;  // positions of its first and its last row (the first: -1 at least)
    int first_step, steps;  // steps of `step` positions that some row of it sees
};
// The tile of rows_per_tile rows (rows times the heads that share a kv head) from first_row on; none where the sequence has fewer
// than from_rows or at least to_rows. limit: positions that exist.
TLLM_HD TileSpan tile_span(const SequenceRows &s, int first_row, int heads, int rows_per_tile, int step, int window, int limit, int from_rows,
                           int to_rows) {
    const int rows = s.rows * heads, left = rows >= from_rows && rows < to_rows ? rows - first_row : 0;
    if (left <= 0) return TileSpan{0, -1, -1, 0, 0};
    TileSpan t;
    t.rows_left = left;
    t.pos_low = higher_of(s.pos0 + first_row / heads, -1);  // (rows before the first position see nothing; the largest window below -1 would wrap)
    t.pos_high = s.pos0 + (first_row + lower_of(left, rows_per_tile) - 1) / heads;
    const int lo = window_begin(window, t.pos_low), hi = lower_of(t.pos_high, limit - 1);  // the last
    t.first_step = lo / step;
    t.steps = hi >= lo ? hi / step - t.first_step + 1 : 0;
    return t;
}

}  // namespace tllm

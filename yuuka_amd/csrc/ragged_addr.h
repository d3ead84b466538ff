// ragged_addr.h — where the rows of a ragged batch are and which pages they
// take. Plain functions, so that a host compiler can check that no offset,
// position or count leads outside the arrays.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define YK_HD __host__ __device__ __forceinline__
#else
#define YK_HD inline
#endif

namespace yk {

YK_HD int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// Rows of request j, inside the row arrays whatever the offsets are: each is taken to be within them, and a
// request whose end lies before its start to be empty.
struct RowRange {
    int begin, end;
};
YK_HD RowRange row_range(const int32_t *offsets, int rows, int j) {
    const int begin = (int)clamp64(offsets[j], 0, rows), end = (int)clamp64(offsets[j + 1], 0, rows);
    return {begin, end > begin ? end : begin};
}

// What the convolution's wave with rows first .. last - 1 does with `row`, `r` being the first request that ends
// behind it. A request's first `early` rows need its window: they are the wave's that has the first of them, which goes
// past its own last row for these and for no others. Rows before a request are nobody's.
enum RowTurn { kRowDone, kRowSkipped, kRowTaken };
YK_HD RowTurn row_turn(RowRange r, int row, int first, int last, int early) {
    const bool begun = r.begin >= first && r.begin < last, needs_window = row - r.begin < early;
    if (row >= last && !(begun && needs_window)) return kRowDone;
    return row < r.begin || (needs_window && !begun) ? kRowSkipped : kRowTaken;
}

// The pages of a request at `position` that takes `count` rows, with `blocks`
// entries of its table in use: new ones are table entries first .. first + fresh - 1.
struct PageNeed {
    int first, fresh;
};
YK_HD PageNeed page_need(int64_t position, int64_t count, int64_t blocks, int block_size, int capacity) {
    const int64_t from = clamp64(position, 0, capacity), to = clamp64(position + count, 0, capacity);
    const int64_t entries = ((int64_t)capacity - 1) / block_size + 1;
    int64_t first = clamp64(blocks, 0, entries);
    if (from / block_size > first) first = from / block_size;
    const int64_t end = to > from ? (to - 1) / block_size + 1 : 0;
    return {(int)first, (int)(end > first ? end - first : 0)};
}

// Rows are worked on in chunks; those of request j, whose rows start at
// `begin`, are numbered from here on, and the numbers of two requests never meet where offsets ascend:
// (begin + n) / C - begin / C + 1 is n / C, rounded up, at the least.
template <int C> YK_HD int first_chunk(int begin, int j) { return begin / C + j; }
template <int C> YK_HD int chunk_numbers(int rows, int requests) { return rows / C + requests; }

}  // namespace yk

// kv_addr.h — where a token of the paged cache is. Plain functions, so that a
// host compiler can check that no table, position or page count leads outside
// the pool.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define YK_HD __host__ __device__ __forceinline__
#else
#define YK_HD inline
#endif

namespace yk {

// Pool formats. F32 and F16 pages are [block_size][kv_dim]. A Q8_0 page is
// [block_size][kv_dim] int8 digits, then [block_size][kv_dim / 32] F16 scales
// (the byte count of GGUF's 34-byte blocks, with the digits of a token in one
// aligned run instead of 32-byte pieces between the scales). Every 64 dims'
// digits are stored transposed, as a 16 x 4 matrix: byte 4 r + j of the 64
// holds dim 16 j + r. Lane r of a 16-wide output tile of the value product then
// has its column of four tiles in one dword, and the tiles 2 b and 2 b + 1
// have one scale each key; in the natural order the 16 columns of a tile
// would be spread over all the scales.
constexpr int kKvF32 = 0, kKvF16 = 1, kKvQ8 = 2;
// Rows and scales start at multiples of these bytes, whatever the shape: a Q8_0 page
// of one token of 64 dims is 68 bytes.
constexpr int kKvAlign = 4;

struct KvLayout {
    int fmt;
    int block_size, capacity;
    int kv_dim;
    int pages;  // pages of the pools; a table entry outside 0..pages-1 is an unmapped page
};

// Bytes of one token in one pool, and of one page.
YK_HD int64_t kv_token_bytes(int fmt, int64_t kv_dim) {
    return fmt == kKvF32 ? kv_dim * 4 : fmt == kKvF16 ? kv_dim * 2 : kv_dim + kv_dim / 32 * 2;
}
YK_HD int64_t kv_page_bytes(const KvLayout &a) { return kv_token_bytes(a.fmt, a.kv_dim) * a.block_size; }
YK_HD int kv_table_blocks(const KvLayout &a) { return (a.capacity - 1) / a.block_size + 1; }

// Byte offsets of the row of position p of request j in a pool, and of its
// Q8_0 scales; false when the position is outside the request's capacity or
// its page is unmapped.
YK_HD bool kv_slot(const KvLayout &a, const int32_t *table, int j, int64_t p, int64_t *row, int64_t *scales) {
    if (p < 0 || p >= a.capacity) return false;
    const int b = (int)p / a.block_size, t = (int)p % a.block_size;
    const int page = table[(int64_t)j * kv_table_blocks(a) + b];
    if ((uint32_t)page >= (uint32_t)a.pages) return false;
    const int64_t base = (int64_t)page * kv_page_bytes(a);
    if (a.fmt == kKvQ8) {
        *row = base + (int64_t)t * a.kv_dim;
        *scales = base + (int64_t)a.block_size * a.kv_dim + (int64_t)t * (a.kv_dim / 32) * 2;
    } else {
        *row = base + (int64_t)t * kv_token_bytes(a.fmt, a.kv_dim);
        *scales = 0;
    }
    return true;
}

}  // namespace yk

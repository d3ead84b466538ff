// k_batch.hip — where the rows of a ragged batch go: offsets, {request,
// position} and slot of every row, and pages from a free list into the block
// tables.
//
// Request j has p_j cached tokens, n_j new ones and blocks_j entries of its table
// in use:
//   offsets_j = sum of n_i before j        first_j = max(blocks_j, p_j / block)
//   new_j = ceil((p_j + n_j) / block) - first_j
//   entry first_j + i of its table = free[next + sum of new_i before j + i]
//   slot of position p = page * block + p % block
// Every block that gets a page holds a new row, so that the rows alone write the
// tables: the first of a block does.
//
// Bound by the launch: 16 requests of one row 6.4 us, 200 of 16300 rows (0.3 MB) 6.5; 4.8 to 7.9 in place, as a serving
// loop calls it. The sums are in 64 bits, so that no counts overflow them.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "internal.h"
#include "ragged.h"
#include "ragged_dev.h"

namespace yk {

yuuka_status batch_check(const BatchArgs &a) {
    constexpr int kBig = 1 << 30;
    if (a.block_size < 1 || a.block_size > (1 << 20) || a.capacity < 1 || a.capacity > kBig)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "batch plan: %d tokens in pages of %d", a.capacity, a.block_size);
    if (a.requests < 1 || a.requests > 65535 || a.rows < 1 || a.rows > kBig)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "batch plan: %d requests, %d rows", a.requests, a.rows);
    return YUUKA_OK;
}

namespace {

constexpr int kScan = 1024;

// What the scan leaves for the rows: {first, number in the free list of the request's first page} of
// every request, then the end of the free list. (The scan's outputs may be its inputs' own buffers.)
__device__ __forceinline__ int64_t scan_add(int64_t x, int64_t *sums, int64_t *total) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t y = __shfl_up(x, off);
        if (lane >= off) x += y;
    }
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    int64_t before = *total;
    for (int w = 0; w < kScan / 64; w++) {
        if (w < wave) before += sums[w];
        *total += sums[w];
    }
    __syncthreads();
    return before + x;
}

// The scan by one workgroup: sums of the requests' rows and pages, `put(j, end of its rows, {first, start})` for each;
// returned, the end of the free list. `write`: this workgroup leaves the outputs.
template <typename F>
__device__ __forceinline__ int scan_requests(const BatchBuffers &b, const BatchArgs &a, int64_t *sums, bool write, F &&put) {
    const int tid = threadIdx.x;
    const int64_t next = max(0, b.pool[0]), last = max(next, (int64_t)min(b.pool[1], b.free_entries));
    int64_t rows = 0, pages = 0;  // of the requests before this turn's
    for (int base = 0; base < a.requests; base += kScan) {
        const int j = base + tid;
        const bool live = j < a.requests;
        int64_t n = live ? max(0, b.counts[j]) : 0;
        const int blocks = live ? b.blocks[j] : 0;
        const int64_t position = live ? b.positions[2 * j + 1] : 0;
        const int64_t end = scan_add(n, sums, &rows);
        n = max((int64_t)0, min(end, (int64_t)a.rows) - (end - n));  // rows that the arrays hold
        const PageNeed need = live ? page_need(position, n, blocks, a.block_size, a.capacity) : PageNeed{0, 0};
        const int64_t start = next + scan_add(need.fresh, sums, &pages) - need.fresh;
        if (!live) continue;
        put(j, (int)min(end, (int64_t)a.rows), make_int2(need.first, (int)min(start, (int64_t)0x7fffffff)));
        const int64_t taken = clamp64(last - start, 0, need.fresh);
        if (write) b.blocks_out[j] = taken ? need.first + (int)taken : blocks;
    }
    if (write && tid == 0) {
        const int64_t taken = min(pages, last - next);
        b.pool_out[0] = (int)(next + taken);
        if (b.pool_out != b.pool) b.pool_out[1] = (int)min(pages - taken, (int64_t)0x7fffffff);  // else the count stays
    }
    return (int)last;
}

// One row: `offsets` and `plan` as the scan left them.
__device__ __forceinline__ void place_row(const BatchBuffers &b, const BatchArgs &a, int row, const int32_t *offsets,
                                          const int2 *plan, int last) {
    int lo = 0, hi = a.requests;  // the first request that ends behind the row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid + 1] > row) hi = mid;
        else lo = mid + 1;
    }
    if (lo == a.requests) {
        b.row_info[row] = make_int2(-1, -1);
        b.slots[row] = -1;
        return;
    }
    const int i = row - offsets[lo];
    const int64_t p = (int64_t)b.positions[2 * lo + 1] + i;
    b.row_info[row] = make_int2(lo, (int)min(p, (int64_t)0x7fffffff));
    int page = -1;
    if (p >= 0 && p < a.capacity) {
        const int2 mine = plan[lo];
        const int block = (int)p / a.block_size;
        int32_t *const entry = b.table + (int64_t)lo * ((a.capacity - 1) / a.block_size + 1) + block;
        if (block < mine.x) {
            page = *entry;
        } else {
            const int64_t at = (int64_t)mine.y + (block - mine.x);
            if (at < last) page = b.free_pages[at];
            if (i == 0 || (int)p % a.block_size == 0) *entry = page;
        }
    }
    b.slots[row] = page < 0 ? -1 : (int64_t)page * a.block_size + (int)p % a.block_size;
}

__global__ __launch_bounds__(kScan) void batch_scan_kernel(BatchBuffers b, BatchArgs a, int2 *__restrict__ plan) {
    __shared__ int64_t sums[kScan / 64];
    const int last = scan_requests(b, a, sums, true, [&](int j, int end, int2 mine) {
        b.offsets[j + 1] = end;
        plan[j] = mine;
    });
    if (threadIdx.x == 0) {
        b.offsets[0] = 0;
        plan[a.requests] = make_int2(last, 0);
    }
}

__global__ __launch_bounds__(256) void batch_rows_kernel(BatchBuffers b, BatchArgs a, const int2 *__restrict__ plan) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row < a.rows) place_row(b, a, row, b.offsets, plan, plan[a.requests].x);
}

// Both for up to kScan requests: every workgroup scans for itself, the first leaves the outputs.
__global__ __launch_bounds__(kScan) void batch_plan_kernel(BatchBuffers b, BatchArgs a) {
    __shared__ int64_t sums[kScan / 64];
    __shared__ int32_t offsets[kScan + 1];
    __shared__ int2 plan[kScan];
    const bool write = blockIdx.x == 0;
    if (threadIdx.x == 0) {
        offsets[0] = 0;
        if (write) b.offsets[0] = 0;
    }
    const int last = scan_requests(b, a, sums, write, [&](int j, int end, int2 mine) {
        offsets[j + 1] = end;
        plan[j] = mine;
        if (write) b.offsets[j + 1] = end;
    });
    __syncthreads();
    for (int64_t row = (int64_t)blockIdx.x * kScan + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * kScan)
        place_row(b, a, (int)row, offsets, plan, last);
}

}  // namespace

uint64_t batch_plan_scratch_bytes(const BatchArgs &a) { return ((uint64_t)a.requests + 1) * sizeof(int2); }

hipError_t launch_batch_plan(const BatchBuffers &b, const BatchArgs &a, void *scratch, hipStream_t s) {
    // One launch where a workgroup scans the requests in one turn and none reads what another overwrites: 16 requests
    // of one row 10.5 -> 6.8 us, 200 of 16300 rows 10.5 -> 6.9. In place a workgroup alone takes 1024, 2048 and 4096 rows of
    // 200 requests in 5.6, 6.7 and 9.0 us (host loop), two launches take 7.9, also for 16300.
    const bool in_place = b.blocks_out == b.blocks || b.pool_out == b.pool;
    if (a.requests <= kScan && (!in_place || a.rows <= 2048)) {
        batch_plan_kernel<<<in_place ? 1 : (uint32_t)((a.rows + kScan - 1) / kScan), kScan, 0, s>>>(b, a);
        return hipGetLastError();
    }
    int2 *const plan = static_cast<int2 *>(scratch);
    batch_scan_kernel<<<1, kScan, 0, s>>>(b, a, plan);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    batch_rows_kernel<<<(uint32_t)((a.rows + 255) / 256), 256, 0, s>>>(b, a, plan);
    return hipGetLastError();
}

}  // namespace yk

// ragged_dev.h — the requests of a ragged batch's rows on the device.
#pragma once

#include "ragged.h"
#include "ragged_addr.h"

namespace yk {

// The first of 0..n-1 (n if none) for which `after` holds, and it holds for all behind
// it: a wave looks at 64 places at once.
template <typename F>
__device__ __forceinline__ int wave_first(int n, F &&after) {
    int lo = 0, hi = n;  // the answer is in lo..hi
    const int lane = threadIdx.x & 63;
    while (lo < hi) {
        const int step = (hi - lo + 63) >> 6;
        const int at = (int)min((int64_t)lo + (int64_t)step * (lane + 1) - 1, (int64_t)hi - 1);
        const uint64_t past = __ballot(after(at));
        if (!past) return hi;  // (the last lane looked at hi - 1)
        const int k = __ffsll((unsigned long long)past) - 1;
        const int first = (int)min((int64_t)lo + (int64_t)step * (k + 1) - 1, (int64_t)hi - 1);
        if (step == 1) return first;
        lo += step * k;
        hi = first;
    }
    return lo;
}

// Request of a row, or `requests` for one behind the last. (Whatever the offsets hold, it is one of these.)
__device__ __forceinline__ int wave_request_of_row(const int32_t *offsets, int requests, int row) {
    return __builtin_amdgcn_readfirstlane(wave_first(requests, [&](int j) { return offsets[j + 1] > row; }));
}

}  // namespace yk

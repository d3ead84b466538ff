// kv_dev.h — positions of the paged cache's rows on the device.
#pragma once

#include "kv.h"

namespace yk {

// Position of row r of request j (64 bits: a device position is any int32).
__device__ __forceinline__ int64_t kv_position(const KvArgs &a, const ModelDyn &dyn, int j, int r) {
    const int base = dyn.pos_dev ? dyn.pos_dev[2 * j] : dyn.pos;
    return (int64_t)base + a.displacement + r;
}

}  // namespace yk

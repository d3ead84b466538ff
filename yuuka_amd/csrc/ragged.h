// ragged.h — batches of requests with different numbers of new rows, laid one
// after another without padding: argument blocks and launchers of k_batch.hip
// (tables and slots), k_gdnrow.hip (convolution, one token) and k_gdnchunk.hip
// (prompts).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/yuuka_hip.h"

namespace yk {

struct BatchArgs {
    int requests, rows, block_size, capacity;
};

struct RaggedArgs {
    int requests, rows;
    int groups, heads, head_dim, channels;  // channels = (2 groups + heads) head_dim
    int stride;                             // elements between rows of x / qkv
    int kernel;                             // convolution: taps
    int log_decay;
    int states;                             // slots of the state pool; one outside 0..states-1 is none
    float scale, eps;
};

// Checks the argument blocks (without buffers).
yuuka_status batch_check(const BatchArgs &a);
// `conv`: of the convolution, whose states are windows of `kernel` - 1 inputs.
yuuka_status ragged_check(RaggedArgs *a, uint32_t dtype, bool conv);
inline uint64_t ragged_state_bytes(const RaggedArgs &a, bool conv) {
    return 4ull * (conv ? (uint64_t)a.channels * (a.kernel - 1) : (uint64_t)a.heads * a.head_dim * a.head_dim);
}
inline uint64_t ragged_element_bytes(uint32_t dtype) { return dtype == YUUKA_DTYPE_F32 ? 4 : 2; }

struct BatchBuffers {
    const int32_t *positions, *counts, *blocks;
    int32_t *table;
    const int32_t *free_pages, *pool;
    int free_entries;  // of the list; pool's count is taken to be no more
    int32_t *offsets;
    int2 *row_info;
    int64_t *slots;
    int32_t *blocks_out, *pool_out;
};
uint64_t batch_plan_scratch_bytes(const BatchArgs &a);
hipError_t launch_batch_plan(const BatchBuffers &b, const BatchArgs &a, void *scratch, hipStream_t s);

hipError_t launch_gdn_ragged_conv(void *out, const void *x, uint32_t dtype, const float *weight, float *state,
                                  const int32_t *offsets, const int2 *slots, const RaggedArgs &a, hipStream_t s);

struct GdnRows {
    void *out;
    const void *qkv;
    const float *alpha, *beta, *dt, *a;
    float *state;
    const int32_t *offsets;  // (not of a step: row j is request j's)
    const int2 *slots;
};
hipError_t launch_gdn_step(const GdnRows &b, uint32_t dtype, const RaggedArgs &a, hipStream_t s);
uint64_t gdn_prompt_scratch_bytes(const RaggedArgs &a);
hipError_t launch_gdn_prompt(const GdnRows &b, uint32_t dtype, const RaggedArgs &a, void *scratch, hipStream_t s);

}  // namespace yk

// kv.h — the paged key/value cache of a batch of requests: argument block and
// launchers of k_kv.hip (append, read back) and
// k_kvattn.hip (attention of the newest rows).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kv_addr.h"
#include "model_kernels.h"

namespace yk {

struct KvArgs : KvLayout {
    int requests, rows;
    int rq_rows;            // rows between consecutive requests
    int heads, kv_heads, head_dim;
    int rope_dim;           // append: rotated dimensions of a key (0: none)
    int gated;              // attention: query rows are [q | gate] per head
    int displacement;       // row r of request j is at position_j + displacement + r
    float scale, eps;
};

inline int kv_fmt_of(uint32_t dtype) {
    return dtype == YUUKA_DTYPE_F32 ? kKvF32 : dtype == YUUKA_DTYPE_F16 ? kKvF16 : dtype == YUUKA_DTYPE_Q8_0 ? kKvQ8 : -1;
}

// Checks the argument block and sets kv_dim and rq_rows; `attention` checks
// the query heads too.
yuuka_status kv_check(KvArgs *a, uint32_t dtype, bool attention);
// Pages of two pools of these sizes (at most INT32_MAX).
int kv_pages(const KvArgs &a, uint64_t kbytes, uint64_t vbytes);
inline uint64_t kv_table_entries(const KvArgs &a) {
    return (uint64_t)a.requests * kv_table_blocks(a);
}
inline uint64_t kv_span_rows(const KvArgs &a) { return (uint64_t)(a.requests - 1) * a.rq_rows + a.rows; }

// Rounds the rows' keys and values into the pools. k_norm (per-head RMSNorm
// of the keys) and rope ({cos, sin} of a.rope_dim / 2 pairs a row) may be
// null. With q, the query rows are normalised by q_norm and rotated like the
// keys into q_out [rows][heads][head_dim] (q rows [q | gate] when a.gated).
hipError_t launch_kv_append(const float *k, const float *v, void *kpool, void *vpool, const int32_t *table,
                            const float *k_norm, const float2 *rope, const float *q, const float *q_norm,
                            float *q_out, const KvArgs &a, const ModelDyn &dyn, hipStream_t s);
// Positions base + displacement + r of every request as float32 rows; a null
// pool or output leaves that side out.
hipError_t launch_kv_read(const void *kpool, const void *vpool, const int32_t *table, float *k_out, float *v_out,
                          const KvArgs &a, const ModelDyn &dyn, hipStream_t s);
// Attention of the rows' queries over their request's pages. q rows are
// [heads][q_stride] floats, the gate (a.gated) `gate` [heads][gate_stride].
uint64_t kv_attention_scratch_bytes(const KvArgs &a);
hipError_t launch_kv_attention(const float *q, int q_stride, const float *gate, int gate_stride, const void *kpool,
                               const void *vpool, const int32_t *table, float *out, const KvArgs &a, void *scratch,
                               const ModelDyn &dyn, hipStream_t s);

}  // namespace yk

// k_kvattn.hip — attention of the newest rows of a batch of requests over
// their paged cache (F16 or Q8_0 pages), each request at its own length: the
// decode step of engine/gpu's session (one row) and the verify rows.
//
//   out = sum_t softmax_t(scale q . k_t) v_t,  t = 0 .. position of the row
//
// A request's keys are cut into `splits` ranges; a workgroup keeps the running
// maximum m, sum l and unnormalised output o of its range, and the merge
// kernel joins the ranges' records with weights exp(m - max m).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "internal.h"
#include "kv_dev.h"
#include "refmath.h"

namespace yk {
namespace {

constexpr int kChunk = 64;

// Keys a row sees: those at positions up to its own, within the capacity.
__device__ __forceinline__ int row_keys(const KvArgs &a, const ModelDyn &dyn, int j, int r) {
    const int64_t p = kv_position(a, dyn, j, r);
    return p < 0 ? 0 : (int)min(p + 1, (int64_t)a.capacity);
}

// Value of dim d of head h of a token.
template <int FMT>
__device__ __forceinline__ float kv_value(const KvArgs &a, const uint8_t *pool, int64_t at, int64_t sc, int h, int d) {
    const int D = a.head_dim;
    if constexpr (FMT == kKvF16) return h2f(reinterpret_cast<const uint16_t *>(pool + at)[h * D + d]);
    return (float)(int8_t)pool[at + h * D + (d & ~63) + 4 * (d & 15) + ((d >> 4) & 3)] *
           h2f(reinterpret_cast<const uint16_t *>(pool + sc)[h * (D / 32) + (d >> 5)]);
}

// One workgroup per (range, query head, request), the rows in turn.
template <int FMT>
__global__ __launch_bounds__(256) void kv_attention_kernel(const float *__restrict__ q, int q_stride,
                                                           const uint8_t *__restrict__ kpool,
                                                           const uint8_t *__restrict__ vpool,
                                                           const int32_t *__restrict__ table, KvArgs a, int splits,
                                                           float *__restrict__ part, ModelDyn dyn) {
    __shared__ float qs[256], ps[kChunk], stat[2];
    __shared__ int64_t at[kChunk], sc[kChunk];
    const int split = blockIdx.x, h = blockIdx.y, j = blockIdx.z, D = a.head_dim, tid = threadIdx.x;
    const int kvh = h / (a.heads / a.kv_heads);
    for (int r = 0; r < a.rows; r++) {
        const int n = row_keys(a, dyn, j, r);
        const int chunks = (n + kChunk - 1) / kChunk, per = (chunks + splits - 1) / splits;
        const int c0 = split * per, c1 = min(chunks, c0 + per);
        const float *qr = q + (((int64_t)j * a.rq_rows + r) * a.heads + h) * q_stride;
        __syncthreads();
        if (tid < D) qs[tid] = qr[tid];
        float m = -INFINITY, l = 0.0f, o = 0.0f;
        for (int c = c0; c < c1; c++) {
            __syncthreads();
            if (tid < kChunk) {
                const int t = c * kChunk + tid;
                if (t >= n || !kv_slot(a, table, j, t, &at[tid], &sc[tid])) at[tid] = -1;
            }
            __syncthreads();
            {
                const int kk = tid >> 2, quarter = tid & 3;
                float s = 0.0f;
                if (at[kk] >= 0)
                    for (int d = quarter; d < D; d += 4) s = fmaf(qs[d], kv_value<FMT>(a, kpool, at[kk], sc[kk], kvh, d), s);
                s += __shfl_xor(s, 1);
                s += __shfl_xor(s, 2);
                if (quarter == 0) ps[kk] = at[kk] >= 0 ? s * a.scale : -INFINITY;
            }
            __syncthreads();
            float mn = m;
            for (int kk = 0; kk < kChunk; kk++) mn = fmaxf(mn, ps[kk]);
            __syncthreads();
            const float shrink = m == mn ? 1.0f : expf(m - mn);
            if (tid < kChunk) ps[tid] = at[tid] >= 0 ? expf(ps[tid] - mn) : 0.0f;
            __syncthreads();
            l *= shrink;
            o *= shrink;
            for (int kk = 0; kk < kChunk; kk++) {
                if (at[kk] < 0) continue;
                l += ps[kk];
                if (tid < D) o = fmaf(ps[kk], kv_value<FMT>(a, vpool, at[kk], sc[kk], kvh, tid), o);
            }
            m = mn;
        }
        float *rec = part + ((((int64_t)j * a.rows + r) * a.heads + h) * splits + split) * (D + 2);
        if (tid < D) rec[tid] = o;
        if (tid == 0) {
            rec[D] = m;
            rec[D + 1] = l;
        }
    }
}

// One workgroup per (row, head, request): joins the ranges' records.
__global__ __launch_bounds__(256) void kv_attention_merge_kernel(const float *__restrict__ part, int splits,
                                                                 const float *__restrict__ gate, int gate_stride,
                                                                 float *__restrict__ out, KvArgs a) {
    const int r = blockIdx.x, h = blockIdx.y, j = blockIdx.z, D = a.head_dim, d = threadIdx.x;
    if (d >= D) return;
    const float *rec = part + (((int64_t)j * a.rows + r) * a.heads + h) * splits * (int64_t)(D + 2);
    float m = -INFINITY;
    for (int s = 0; s < splits; s++) m = fmaxf(m, rec[(int64_t)s * (D + 2) + D]);
    float l = 0.0f, o = 0.0f;
    for (int s = 0; s < splits; s++) {
        const float *p = rec + (int64_t)s * (D + 2);
        if (p[D + 1] == 0.0f) continue;  // a range without keys
        const float w = p[D] == m ? 1.0f : expf(p[D] - m);
        l = fmaf(w, p[D + 1], l);
        o = fmaf(w, p[d], o);
    }
    float y = l == 0.0f ? 0.0f : o / l;  // a row that sees no key
    const int64_t row = (int64_t)j * a.rq_rows + r;
    if (gate) y *= sigmoid_ref(gate[(row * a.heads + h) * gate_stride + d]);
    out[(row * a.heads + h) * D + d] = y;
}

int kv_splits(const KvArgs &a) {
    const int64_t work = (int64_t)a.heads * a.requests;
    const int64_t want = (2048 + work - 1) / work, most = (a.capacity + 4 * kChunk - 1) / (4 * kChunk);
    return (int)std::max<int64_t>(1, std::min(want, most));
}

}  // namespace

uint64_t kv_attention_scratch_bytes(const KvArgs &a) {
    return (uint64_t)a.requests * a.rows * a.heads * kv_splits(a) * (a.head_dim + 2) * 4;
}

hipError_t launch_kv_attention(const float *q, int q_stride, const float *gate, int gate_stride, const void *kpool,
                               const void *vpool, const int32_t *table, float *out, const KvArgs &a, void *scratch,
                               const ModelDyn &dyn, hipStream_t s) {
    const int splits = kv_splits(a);
    auto *kernel = a.fmt == kKvF16 ? kv_attention_kernel<kKvF16> : kv_attention_kernel<kKvQ8>;
    float *part = static_cast<float *>(scratch);
    kernel<<<dim3(splits, a.heads, a.requests), 256, 0, s>>>(q, q_stride, static_cast<const uint8_t *>(kpool),
                                                             static_cast<const uint8_t *>(vpool), table, a, splits,
                                                             part, dyn);
    kv_attention_merge_kernel<<<dim3(a.rows, a.heads, a.requests), 256, 0, s>>>(part, splits, gate, gate_stride, out, a);
    return hipGetLastError();
}

}  // namespace yk

// k_kv.hip — writing the paged key/value cache of a batch of requests and
// reading it back (the reference's row codec model/qwen35/kv_format.go:93-168
// behind kv_pool.go:131-170, on the device).
//
// Q8_0 rounding of a block of 32 values x, every step in float32:
//   scale = max|x| * (1 / 127), stored as F16 (half up, as every F16 of the cache)
//   digit = x / scale to the nearest, halves away from zero; 0 where scale is 0
//   value = digit * F16 scale (exact in float32: 7 + 11 significant bits)
// The reference's EncodeRow (kv_format.go:93-137) divides max|x| by 127: the
// product's last bit differs in one block of 22, which moves one digit in a
// million by a step. A value is off by at most half a step, scale / 2, and by
// |x| 2^-11 for the scale's own rounding.
// A block that holds a NaN has a NaN scale (the reference leaves that case
// undefined), so that it reads back as NaN instead of as finite values.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "internal.h"
#include "kv_dev.h"
#include "refmath.h"

namespace yk {

yuuka_status kv_check(KvArgs *a, uint32_t dtype, bool attention) {
    a->fmt = kv_fmt_of(dtype);
    if (a->fmt < 0) return fail(YUUKA_ERR_UNSUPPORTED, "KV pool dtype %u (F32, F16 and Q8_0 are served)", dtype);
    if (attention && a->fmt == kKvF32)
        return fail(YUUKA_ERR_UNSUPPORTED, "decode attention over an F32 pool (F16 and Q8_0 are served)");
    constexpr int kBig = 1 << 30;
    if (a->block_size < 1 || a->block_size > (1 << 20) || a->capacity < 1 || a->capacity > kBig)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV cache of %d tokens in pages of %d", a->capacity, a->block_size);
    if (a->requests < 1 || a->requests > 65535 || a->rows < 1 || a->rows > kBig || a->displacement < -kBig ||
        a->displacement > kBig)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV cache: %d requests of %d rows at displacement %d", a->requests,
                    a->rows, a->displacement);
    if (a->rq_rows < a->rows) a->rq_rows = a->rows;
    if (a->kv_heads < 1 || a->kv_heads > 4096)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV cache of %d heads", a->kv_heads);
    if (a->head_dim < 64 || a->head_dim % 64 || a->head_dim > 256)
        return fail(YUUKA_ERR_UNSUPPORTED, "KV cache head dimension %d (64, 128, 192 and 256 are served)", a->head_dim);
    a->kv_dim = a->kv_heads * a->head_dim;
    if (a->rope_dim < 0 || a->rope_dim % 2 || a->rope_dim > a->head_dim || a->rope_dim > 128)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV cache rotation of %d dimensions", a->rope_dim);
    if ((int64_t)a->rows * (2 * a->kv_heads + a->heads) > (1 << 25))  // vectors of one launch
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV cache: %d rows of %d heads in one call", a->rows, a->kv_heads);
    if (attention && (a->heads < 1 || a->heads % a->kv_heads || a->heads > 65535 ||
                      a->heads / a->kv_heads > 256 || a->rows > 4096))
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "decode attention of %d rows, %d heads over %d KV heads", a->rows,
                    a->heads, a->kv_heads);
    if (attention && (int64_t)a->requests * a->kv_heads * ((a->heads / a->kv_heads * (int64_t)a->rows + 7) / 8) > (1 << 23))
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "decode attention: %d requests of %d rows, %d heads in one call",
                    a->requests, a->rows, a->heads);  // (workgroups of one launch)
    if (attention && kv_page_bytes(*a) > 0x7fffffff)
        return fail(YUUKA_ERR_UNSUPPORTED, "decode attention over pages of %lld bytes (below 2 GiB are served)",
                    (long long)kv_page_bytes(*a));
    return YUUKA_OK;
}

int kv_pages(const KvArgs &a, uint64_t kbytes, uint64_t vbytes) {
    return (int)std::min<uint64_t>(std::min(kbytes, vbytes) / (uint64_t)kv_page_bytes(a), 0x7fffffff);
}

namespace {

// A wave takes 256 dims of whole heads: a 16-lane row has 64 dims, a lane four
// of them. D = 64 and 128 put four and two heads in a wave, D = 192 leaves the
// last row idle.
struct LaneDims {
    int head, first;  // head of the wave's, and the dim of value 0 (value i: first + i * step)
    bool live;
};
template <int FMT, int GROUPS>
__device__ __forceinline__ LaneDims lane_dims(int lane) {
    const int g = lane >> 4, r = lane & 15;
    return {g / GROUPS, 64 * (g % GROUPS) + (FMT == kKvQ8 ? r : 4 * r), GROUPS != 3 || g < 3};
}
constexpr int dim_step(int fmt) { return fmt == kKvQ8 ? 16 : 1; }
constexpr int heads_per_wave(int groups) { return groups == 1 ? 4 : groups == 2 ? 2 : 1; }

// Largest of two, NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); }

// One wave per 256 dims: a row's keys, then its values, then its queries
// (those only with q). Bound by the float32 rows it reads.
constexpr int kAppendWaves = 4;

template <int FMT, int GROUPS>
__global__ __launch_bounds__(64 * kAppendWaves) void kv_append_kernel(
    const float *__restrict__ k, const float *__restrict__ v, uint8_t *__restrict__ kpool, uint8_t *__restrict__ vpool,
    const int32_t *__restrict__ table, const float *__restrict__ k_norm, const float2 *__restrict__ rope,
    const float *__restrict__ q, const float *__restrict__ q_norm, float *__restrict__ q_out, KvArgs a, ModelDyn dyn) {
    constexpr int D = 64 * GROUPS, HPW = heads_per_wave(GROUPS), STEP = dim_step(FMT);
    __shared__ float swap[kAppendWaves][256];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int kv_waves = (a.kv_heads + HPW - 1) / HPW;
    const int per_row = 2 * kv_waves + (q ? (a.heads + HPW - 1) / HPW : 0);
    const int64_t item = (int64_t)blockIdx.x * kAppendWaves + wave;
    const int64_t r64 = item / per_row;
    if (r64 >= a.rows) return;  // whole waves: no barrier below
    const int r = (int)r64, part = (int)(item % per_row), j = blockIdx.y;
    const bool query = part >= 2 * kv_waves, value = !query && part >= kv_waves;
    int64_t at = 0, sc = 0;
    if (!query && !kv_slot(a, table, j, kv_position(a, dyn, j, r), &at, &sc)) return;
    const LaneDims ld = lane_dims<FMT, GROUPS>(lane);
    const int h = (query ? part - 2 * kv_waves : value ? part - kv_waves : part) * HPW + ld.head;
    const bool live = ld.live && h < (query ? a.heads : a.kv_heads);
    const int64_t row = (int64_t)j * a.rq_rows + r;
    const float *src = query   ? q + (row * a.heads + h) * (int64_t)(a.gated ? 2 * D : D)
                       : value ? v + row * a.kv_dim + (int64_t)h * D
                               : k + row * a.kv_dim + (int64_t)h * D;
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = live ? src[ld.first + i * STEP] : 0.0f;
    const float *norm = query ? q_norm : value ? nullptr : k_norm;
    if (norm) {  // x * (1 / rms * w), forward.go:472-482
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 4; i++) ss += (double)x[i] * (double)x[i];
#pragma unroll
        for (int off = 1; off < 16 * (GROUPS == 3 ? 4 : GROUPS); off <<= 1) ss += __shfl_xor(ss, off);
        const float mean = (float)(ss / (double)D);
        const float scale = (float)(1.0 / sqrt((double)(mean + a.eps)));
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = __fmul_rn(x[i], __fmul_rn(scale, norm[ld.first + i * STEP]));
    }
    if (rope && !value) {  // pairs (i, i + half), forward.go:495-514: partners meet in LDS
        const int half = a.rope_dim / 2;
        const float2 *cs = rope + row * half;
        float *mine = &swap[wave][ld.head * D];
        if (ld.live) {
#pragma unroll
            for (int i = 0; i < 4; i++) mine[ld.first + i * STEP] = x[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma clang fp contract(off)  // products and sums rounded separately, as the reference
            const int d = ld.first + i * STEP;
            if (ld.live && d < a.rope_dim) {
                const bool first = d < half;
                const float o = mine[first ? d + half : d - half];
                const float2 c = cs[first ? d : d - half];
                x[i] = first ? x[i] * c.x - o * c.y : o * c.y + x[i] * c.x;
            }
        }
    }
    if (query) {
        if (live)
#pragma unroll
            for (int i = 0; i < 4; i++) q_out[(row * a.heads + h) * (int64_t)D + ld.first + i * STEP] = x[i];
        return;
    }
    uint8_t *pool = value ? vpool : kpool;
    if constexpr (FMT == kKvF32) {
        if (live)
#pragma unroll
            for (int i = 0; i < 4; i++) reinterpret_cast<float *>(pool + at)[h * D + ld.first + i] = x[i];
    } else if constexpr (FMT == kKvF16) {
        if (live)
#pragma unroll
            for (int i = 0; i < 4; i++)
                reinterpret_cast<uint16_t *>(pool + at)[h * D + ld.first + i] = ref_f32_to_f16(x[i]);
    } else {
        // a lane's values 0, 1 and 2, 3 are in the two blocks of its 16-lane row
        float m[2] = {max_nan(fabsf(x[0]), fabsf(x[1])), max_nan(fabsf(x[2]), fabsf(x[3]))};
        uint16_t d16[2];
        uint32_t digits = 0;
#pragma unroll
        for (int b = 0; b < 2; b++) {
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) m[b] = max_nan(m[b], __shfl_xor(m[b], off));
            const float scale = __fmul_rn(m[b], 1.0f / 127.0f);
            d16[b] = ref_f32_to_f16(scale);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float t = scale > 0.0f ? roundf(__fdiv_rn(x[2 * b + i], scale)) : 0.0f;
                // inf / inf and finite / inf: 0 (the value is then 0 * inf)
                const int digit = fabsf(t) <= 127.0f ? (int)t : 0;
                digits |= (uint32_t)(uint8_t)(int8_t)digit << (8 * (2 * b + i));
            }
        }
        if (!live) return;
        const int group = h * GROUPS + (lane >> 4) % GROUPS;  // 64 dims: 16 dwords, two scales
        reinterpret_cast<uint32_t *>(pool + at)[group * 16 + (lane & 15)] = digits;
        if (!(lane & 15)) reinterpret_cast<uint32_t *>(pool + sc)[group] = (uint32_t)d16[0] | ((uint32_t)d16[1] << 16);
    }
}

// One wave per 256 dims of a token's keys or values; unmapped positions read
// as zeros.
template <int FMT, int GROUPS>
__global__ __launch_bounds__(256) void kv_read_kernel(const uint8_t *__restrict__ kpool, const uint8_t *__restrict__ vpool,
                                                      const int32_t *__restrict__ table, float *__restrict__ k_out,
                                                      float *__restrict__ v_out, KvArgs a, ModelDyn dyn) {
    constexpr int D = 64 * GROUPS, HPW = heads_per_wave(GROUPS), STEP = dim_step(FMT);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int kv_waves = (a.kv_heads + HPW - 1) / HPW;
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int64_t r64 = item / kv_waves;
    if (r64 >= a.rows) return;
    const int r = (int)r64, j = blockIdx.y;
    const LaneDims ld = lane_dims<FMT, GROUPS>(lane);
    const int h = (int)(item % kv_waves) * HPW + ld.head;
    const uint8_t *pool = blockIdx.z ? vpool : kpool;
    float *out = blockIdx.z ? v_out : k_out;
    if (!pool || !out || !ld.live || h >= a.kv_heads) return;
    int64_t at = 0, sc = 0;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (kv_slot(a, table, j, kv_position(a, dyn, j, r), &at, &sc)) {
        const int e = h * D + ld.first;
        if constexpr (FMT == kKvQ8) {
            const int group = h * GROUPS + (lane >> 4) % GROUPS;
            const uint32_t digits = reinterpret_cast<const uint32_t *>(pool + at)[group * 16 + (lane & 15)];
            const uint32_t d = reinterpret_cast<const uint32_t *>(pool + sc)[group];
#pragma unroll
            for (int i = 0; i < 4; i++)
                x[i] = (float)(int8_t)(uint8_t)(digits >> (8 * i)) * h2f((uint16_t)(d >> (16 * (i >> 1))));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                x[i] = FMT == kKvF32 ? reinterpret_cast<const float *>(pool + at)[e + i]
                                     : h2f(reinterpret_cast<const uint16_t *>(pool + at)[e + i]);
        }
    }
    float *dst = out + ((int64_t)j * a.rq_rows + r) * a.kv_dim + (int64_t)h * D + ld.first;
#pragma unroll
    for (int i = 0; i < 4; i++) dst[i * STEP] = x[i];
}

template <typename F>
hipError_t by_format(const KvArgs &a, F &&f) {
    auto width = [&](auto fmt) {
        switch (a.head_dim / 64) {
        case 1: f(fmt, std::integral_constant<int, 1>{}); break;
        case 2: f(fmt, std::integral_constant<int, 2>{}); break;
        case 3: f(fmt, std::integral_constant<int, 3>{}); break;
        default: f(fmt, std::integral_constant<int, 4>{}); break;
        }
    };
    switch (a.fmt) {
    case kKvF32: width(std::integral_constant<int, kKvF32>{}); break;
    case kKvF16: width(std::integral_constant<int, kKvF16>{}); break;
    default: width(std::integral_constant<int, kKvQ8>{}); break;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append(const float *k, const float *v, void *kpool, void *vpool, const int32_t *table,
                            const float *k_norm, const float2 *rope, const float *q, const float *q_norm,
                            float *q_out, const KvArgs &a, const ModelDyn &dyn, hipStream_t s) {
    const int hpw = heads_per_wave(a.head_dim / 64);
    const int64_t items = (int64_t)a.rows * (2 * ((a.kv_heads + hpw - 1) / hpw) + (q ? (a.heads + hpw - 1) / hpw : 0));
    const int64_t blocks = (items + kAppendWaves - 1) / kAppendWaves;
    return by_format(a, [&](auto fmt, auto n) {
        kv_append_kernel<fmt(), n()><<<dim3((uint32_t)blocks, (uint32_t)a.requests), 64 * kAppendWaves, 0, s>>>(
            k, v, static_cast<uint8_t *>(kpool), static_cast<uint8_t *>(vpool), table, k_norm,
            a.rope_dim ? rope : nullptr, q, q_norm, q_out, a, dyn);
    });
}

hipError_t launch_kv_read(const void *kpool, const void *vpool, const int32_t *table, float *k_out, float *v_out,
                          const KvArgs &a, const ModelDyn &dyn, hipStream_t s) {
    const int hpw = heads_per_wave(a.head_dim / 64);
    const int64_t blocks = ((int64_t)a.rows * ((a.kv_heads + hpw - 1) / hpw) + 3) / 4;
    return by_format(a, [&](auto fmt, auto n) {
        kv_read_kernel<fmt(), n()><<<dim3((uint32_t)blocks, (uint32_t)a.requests, 2), 256, 0, s>>>(
            static_cast<const uint8_t *>(kpool), static_cast<const uint8_t *>(vpool), table, k_out, v_out, a, dyn);
    });
}

}  // namespace yk

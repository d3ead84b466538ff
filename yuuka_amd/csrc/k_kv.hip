// k_kv.hip — writing the paged key/value cache of a batch of requests and
// reading it back (the reference's row codec model/qwen35/kv_format.go:93-168
// behind kv_pool.go:131-170, on the device).
//
// Q8_0 rounding of a block of 32 values x, every step in float32:
//   scale = max|x| * (1 / 127), stored as F16 (half up, as every F16 of the cache)
//   digit = x / scale to the nearest, halves away from zero; 0 where scale is 0
//   value = digit * F16 scale (exact in float32: 7 + 11 significant bits)
// The reference's EncodeRow (kv_format.go:93-137) divides max|x| by 127. The product is what
// torch computes for that division on the GPU (a constant divisor is inverted first), so that
// pages written from there and from here hold the same bytes, and costs less (8191 rows of 8
// heads of 128: 27.9 us, with the quotient 28.6). Over normal values its last bit differs from
// the quotient's in one block of 23, a stored scale in one block of 2.5 million and a digit, by
// one, in one value of 7 million, only where x / scale is within 5 * 2^-17 of a half. A value is
// off by at most half a step, scale / 2, and by |x| 2^-11 for the scale's own rounding.
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
    if (!a->rq_rows) a->rq_rows = a->rows;
    if (a->rq_rows < a->rows)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV cache: %d rows between requests of %d", a->rq_rows, a->rows);
    if (a->kv_heads < 1 || a->kv_heads > 4096)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV cache of %d heads", a->kv_heads);
    if (a->head_dim < 64 || a->head_dim % 64 || a->head_dim > 256)
        return fail(YUUKA_ERR_UNSUPPORTED, "KV cache head dimension %d (64, 128, 192 and 256 are served)", a->head_dim);
    a->kv_dim = a->kv_heads * a->head_dim;
    // 2^36 rows of 64 dims are 16 TiB, more than any buffer: below that a row's bytes
    // (2^27 at the most: 2^16 heads of 256 and their gates) times the rows stay under 2^63
    if (kv_span_rows(*a) > 1ull << 36)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV cache: %d requests of %d rows, %d rows apart", a->requests, a->rows,
                    a->rq_rows);
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
// consecutive ones (16 bytes of the float32 side, so that a wave's access is one
// run). D = 64 and 128 put four and two heads in a wave, D = 192 leaves the
// last row idle.
struct LaneDims {
    int head, first;  // head of the wave's, and the first dim
    bool live;
};
template <int GROUPS>
__device__ __forceinline__ LaneDims lane_dims(int lane) {
    const int g = lane >> 4, r = lane & 15;
    return {g / GROUPS, 64 * (g % GROUPS) + 4 * r, GROUPS != 3 || g < 3};
}
constexpr int heads_per_wave(int groups) { return groups == 1 ? 4 : groups == 2 ? 2 : 1; }

typedef float floats4 __attribute__((ext_vector_type(4), aligned(4)));  // rows are 4-byte aligned
typedef uint32_t dwords4 __attribute__((ext_vector_type(4), aligned(4)));  // Q8_0 pages start at any dword
static_assert(alignof(dwords4) <= kKvAlign, "a row's loads need more than a row has");

// ref_f32_to_f16, short for what becomes a normal half.
__device__ __forceinline__ uint32_t f32_to_f16(float f) {
    const uint32_t u = __float_as_uint(f) & 0x7fffffffu;
    if (u - 0x38800000u < 0x0f000000u)  // 2^-14 .. 2^16: the carry of the rounding goes into the exponent
        return ((u + 0x1000u - 0x38000000u) >> 13) | ((__float_as_uint(f) >> 16) & 0x8000u);
    return ref_f32_to_f16(f);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(dpp<CTRL>(__float_as_uint(x)));
}
template <int CTRL>
__device__ __forceinline__ double add_dpp(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return x + __builtin_bit_cast(double, (uint64_t)dpp<CTRL>((uint32_t)(u >> 32)) << 32 | dpp<CTRL>((uint32_t)u));
}
// Sum over the lanes of a head: 16, 32 or 64.
template <int GROUPS>
__device__ __forceinline__ double head_sum(double x) {
    x = add_dpp<0xb1>(x);   // lanes l ^ 1 and l ^ 2, then the 16-lane row rotated by 4 and 8
    x = add_dpp<0x4e>(x);
    x = add_dpp<0x124>(x);
    x = add_dpp<0x128>(x);
    for (int off = 16; off < 16 * (GROUPS == 3 ? 4 : GROUPS); off <<= 1) x += __shfl_xor(x, off);
    return x;
}

// The digits of a 64-dim group from a lane's four consecutive dims (byte i: dim
// 4 r + i) to the pages' 16 x 4 order: lane r = 4 e + i ends with row 4 i + e of
// the matrix (dims 16 j + 4 i + e, from byte e of the lanes 4 j + i).
__device__ __forceinline__ uint32_t transpose_digits(uint32_t mine, int r) {
    const uint32_t e = r >> 2;
    // of the lanes e, e + 1, e + 2, e + 3 (times 4, modulo 16): byte e of each
    const uint32_t d1 = dpp<0x12c>(mine), d2 = dpp<0x128>(mine), d3 = dpp<0x124>(mine);  // rotated by 12, 8, 4
    const uint32_t sel = e | (4 + e) << 8;
    const uint32_t lo = __builtin_amdgcn_perm(d1, mine, sel), hi = __builtin_amdgcn_perm(d3, d2, sel);
    const uint32_t all = __builtin_amdgcn_perm(hi, lo, 0x05040100u);  // byte b: lane e + b
    return __builtin_amdgcn_alignbit(all, all, 32 - 8 * e);           // byte j: lane j
}

// One wave per 256 dims of kAppendRows rows: keys, values, or queries (those
// only with q). Bound by the float32 rows it reads once (past the caches), those of all the
// wave's rows asked for before any is used, and by vector instructions (49 % of a SIMD's cycles):
// 8191 rows of 8 heads of 128 to Q8_0 (85 MB) 28 us, 3.0 TB/s; with the key norm and 64 dims
// rotated (87 MB) 34 us, 64 %. To F16 28 and 33, to F32 26 and 31. Two rows a wave: with the
// read back 45.8 us, one 51.2, four 48.4.
constexpr int kAppendWaves = 4, kAppendRows = 2;

// SLOTS: `slots` says where each row goes, instead of the table and the position: 8191 rows of 8 heads of 128
// to F32 (134 MB) 25.3 us, 5.3 TB/s; to F16 24.1 (101 MB) and Q8_0 24.6 (85 MB), with a rotation 27.5 either.
template <int FMT, int GROUPS, bool SLOTS>
__global__ __launch_bounds__(64 * kAppendWaves) void kv_append_kernel(
    const float *__restrict__ k, const float *__restrict__ v, uint8_t *__restrict__ kpool, uint8_t *__restrict__ vpool,
    const int32_t *__restrict__ table, const float *__restrict__ k_norm, const float2 *__restrict__ rope,
    const float *__restrict__ q, const float *__restrict__ q_norm, float *__restrict__ q_out, KvArgs a, ModelDyn dyn,
    const int64_t *__restrict__ slots) {
    constexpr int D = 64 * GROUPS, HPW = heads_per_wave(GROUPS);
    __shared__ float swap[kAppendWaves][256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int kv_waves = (a.kv_heads + HPW - 1) / HPW;
    const uint32_t per_row = 2 * kv_waves + (q ? (a.heads + HPW - 1) / HPW : 0);
    const uint32_t item = blockIdx.x * kAppendWaves + wave;  // (below 2^26)
    const int first_row = (int)(item / per_row) * kAppendRows, part = (int)(item % per_row), j = blockIdx.y;
    if (first_row >= a.rows) return;  // whole waves: no barrier below
    const bool query = part >= 2 * kv_waves, value = !query && part >= kv_waves;
    const LaneDims ld = lane_dims<GROUPS>(lane);
    const int h = (query ? part - 2 * kv_waves : value ? part - kv_waves : part) * HPW + ld.head;
    const bool live = ld.live && h < (query ? a.heads : a.kv_heads);
    const int64_t row0 = (int64_t)j * a.rq_rows + first_row;
    const int64_t stride = query ? (int64_t)a.heads * (a.gated ? 2 * D : D) : a.kv_dim;
    const float *src = (query   ? q + (int64_t)h * (a.gated ? 2 * D : D)
                        : value ? v + (int64_t)h * D
                                : k + (int64_t)h * D) + row0 * stride + ld.first;
    const floats4 none = {0.f, 0.f, 0.f, 0.f};
    floats4 rows[kAppendRows];
#pragma unroll
    for (int n = 0; n < kAppendRows; n++)
        rows[n] = live && first_row + n < a.rows ? __builtin_nontemporal_load(reinterpret_cast<const floats4 *>(src + n * stride)) : none;
    const float *norm = query ? q_norm : value ? nullptr : k_norm;
    const floats4 weight = norm && ld.live ? *reinterpret_cast<const floats4 *>(norm + ld.first) : none;
    const int64_t p0 = query || SLOTS ? 0 : kv_position(a, dyn, j, first_row);
#pragma unroll
    for (int n = 0; n < kAppendRows; n++) {
        if (first_row + n >= a.rows) return;
        int64_t at = 0, sc = 0;
        if constexpr (SLOTS) {
            if (!kv_row_of_slot(a, slots[first_row + n], &at, &sc)) continue;
        } else {
            if (!query && !kv_slot(a, table, j, p0 + n, &at, &sc)) continue;
        }
        const int64_t row = row0 + n;
        float x[4] = {rows[n][0], rows[n][1], rows[n][2], rows[n][3]};
        if (norm) {  // x * (1 / rms * w), forward.go:472-482
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 4; i++) ss += (double)x[i] * (double)x[i];
            ss = head_sum<GROUPS>(ss);
            const float mean = (float)(ss / (double)D);
            const float scale = (float)(1.0 / sqrt((double)(mean + a.eps)));
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = __fmul_rn(x[i], __fmul_rn(scale, weight[i]));
        }
        if (rope && !value) {  // pairs (i, i + half), forward.go:495-514: partners meet in LDS
            const int half = a.rope_dim / 2;
            const float2 *cs = rope + row * half;
            float *mine = &swap[wave][ld.head * D];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (ld.live) {
#pragma unroll
                for (int i = 0; i < 4; i++) mine[ld.first + i] = x[i];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int d = ld.first;
            if (half % 4 == 0) {  // a lane's four are on one side, their partners in a row
                if (ld.live && d < a.rope_dim) {
                    const bool first = d < half;
                    const floats4 o = *reinterpret_cast<const floats4 *>(mine + (first ? d + half : d - half));
                    const floats4 *c = reinterpret_cast<const floats4 *>(cs + (first ? d : d - half));
                    const floats4 c01 = c[0], c23 = c[1];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
#pragma clang fp contract(off)  // products and sums rounded separately, as the reference
                        const float turned = o[i] * (i < 2 ? c01 : c23)[2 * (i & 1) + 1];
                        x[i] = x[i] * (i < 2 ? c01 : c23)[2 * (i & 1)] + (first ? -turned : turned);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
#pragma clang fp contract(off)
                    if (ld.live && d + i < a.rope_dim) {
                        const bool first = d + i < half;
                        const float o = mine[first ? d + i + half : d + i - half];
                        const float2 c = cs[first ? d + i : d + i - half];
                        x[i] = first ? x[i] * c.x - o * c.y : o * c.y + x[i] * c.x;
                    }
                }
            }
        }
        const floats4 done = {x[0], x[1], x[2], x[3]};
        if (query) {
            if (live) *reinterpret_cast<floats4 *>(q_out + (row * a.heads + h) * (int64_t)D + ld.first) = done;
            continue;
        }
        uint8_t *pool = value ? vpool : kpool;
        if constexpr (FMT == kKvF32) {
            if (live) *reinterpret_cast<floats4 *>(reinterpret_cast<float *>(pool + at) + h * D + ld.first) = done;
        } else if constexpr (FMT == kKvF16) {
            if (live)
                *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(pool + at) + h * D + ld.first) =
                    make_uint2(f32_to_f16(x[0]) | f32_to_f16(x[1]) << 16, f32_to_f16(x[2]) | f32_to_f16(x[3]) << 16);
        } else {
            // a block of 32 dims is eight lanes; as integers, NaN is above infinity
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
            m = max(m, dpp<0xb1>(m));   // lanes l ^ 1, l ^ 2 and 7 - l of the eight
            m = max(m, dpp<0x4e>(m));
            m = max(m, dpp<0x141>(m));
            const float scale = __fmul_rn(__uint_as_float(m), 1.0f / 127.0f);
            const uint32_t d16 = f32_to_f16(scale);
            // Digits are x / scale rounded to the nearest, halves away from zero. The
            // product with the reciprocal is within 2^-15 of the quotient: it decides
            // the digit unless it is that close to a half. (With a division for every
            // digit, 8191 rows of 8 heads of 128 took 31.9 us instead of 27.4.)
            uint32_t digits = 0;
            const float inverse = __builtin_amdgcn_rcpf(scale);
            float close = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float y = x[i] * inverse, up = fabsf(y) + 0.5f;
                close = fmaxf(close, fabsf(__builtin_amdgcn_fractf(up) - 0.5f));  // up to 0.5 at a half
                digits |= ((uint32_t)(int)copysignf(up, y) & 0xffu) << (8 * i);
            }
            const bool plain = m - 0x0d800000u < 0x65000000u;  // 2^-100 .. 2^102: no end of the range near
            if (!plain || close > 0.5f - 0x1p-13f) {
                digits = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float t = scale > 0.0f ? roundf(__fdiv_rn(x[i], scale)) : 0.0f;
                    // inf / inf and finite / inf: 0 (the value is then 0 * inf)
                    const int digit = fabsf(t) <= 127.0f ? (int)t : 0;
                    digits |= (uint32_t)(uint8_t)(int8_t)digit << (8 * i);
                }
            }
            const int r = lane & 15;
            digits = transpose_digits(digits, r);
            const uint32_t d16_other = dpp<0x128>(d16);  // of lane (r + 8) % 16
            if (live) {
                const int group = h * GROUPS + (lane >> 4) % GROUPS;  // 64 dims: 16 dwords, two scales
                reinterpret_cast<uint32_t *>(pool + at)[group * 16 + 4 * (r & 3) + (r >> 2)] = digits;
                if (!r) reinterpret_cast<uint32_t *>(pool + sc)[group] = d16 | d16_other << 16;
            }
        }
    }
}

// One wave per 256 dims of kReadRows tokens' keys or values, all loads before the
// first store; unmapped positions read as zeros. Bound by the float32 rows it writes,
// past the caches: 16 requests of 4000 tokens of 4 heads of 256 from Q8_0 (664 MB): 117 us,
// 5.7 TB/s (132 at the clock that many passes in a row leave); through the caches 127; with one
// token a wave 189, two 141, eight 129. 8191 tokens of 8 heads of 128 from Q8_0 and F16 18 us,
// from F32 22.
constexpr int kReadRows = 4;

template <int FMT, int GROUPS>
__global__ __launch_bounds__(256) void kv_read_kernel(const uint8_t *__restrict__ kpool, const uint8_t *__restrict__ vpool,
                                                      const int32_t *__restrict__ table, float *__restrict__ k_out,
                                                      float *__restrict__ v_out, KvArgs a, ModelDyn dyn) {
    constexpr int D = 64 * GROUPS, HPW = heads_per_wave(GROUPS);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t kv_waves = (a.kv_heads + HPW - 1) / HPW;
    const uint32_t item = blockIdx.x * 4 + wave;  // (below 2^26)
    const int first_row = (int)(item / kv_waves) * kReadRows, j = blockIdx.y;
    if (first_row >= a.rows) return;
    const LaneDims ld = lane_dims<GROUPS>(lane);
    const int h = (int)(item % kv_waves) * HPW + ld.head;
    const uint8_t *pool = blockIdx.z ? vpool : kpool;
    float *out = blockIdx.z ? v_out : k_out;
    if (!pool || !out || !ld.live || h >= a.kv_heads) return;
    const int64_t p0 = kv_position(a, dyn, j, first_row);
    const int e = h * D + ld.first, group = h * GROUPS + (lane >> 4) % GROUPS, r = lane & 15;
    int64_t at[kReadRows], sc[kReadRows];
    bool there[kReadRows];
#pragma unroll
    for (int n = 0; n < kReadRows; n++) {
        at[n] = sc[n] = 0;
        there[n] = first_row + n < a.rows && kv_slot(a, table, j, p0 + n, &at[n], &sc[n]);
    }
    dwords4 raw[kReadRows];
    uint32_t scale[kReadRows];
#pragma unroll
    for (int n = 0; n < kReadRows; n++) {
        raw[n] = dwords4{0, 0, 0, 0};
        scale[n] = 0;
        if (!there[n]) continue;
        if constexpr (FMT == kKvQ8) {  // rows 4 (r & 3) .. + 3 of the 16 x 4 matrix: column r >> 2 is the lane's
            raw[n] = *reinterpret_cast<const dwords4 *>(pool + at[n] + group * 64 + 16 * (r & 3));
            scale[n] = reinterpret_cast<const uint32_t *>(pool + sc[n])[group];
        } else if constexpr (FMT == kKvF32) {
            raw[n] = *reinterpret_cast<const dwords4 *>(pool + at[n] + (int64_t)e * 4);
        } else {
            const uint2 w = *reinterpret_cast<const uint2 *>(pool + at[n] + (int64_t)e * 2);
            raw[n][0] = w.x;
            raw[n][1] = w.y;
        }
    }
#pragma unroll
    for (int n = 0; n < kReadRows; n++) {
        if (first_row + n >= a.rows) return;
        floats4 x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (FMT == kKvQ8)
                x[i] = (float)(int8_t)(uint8_t)(raw[n][i] >> (8 * (r >> 2))) * h2f((uint16_t)(scale[n] >> (16 * (r >> 3))));
            else if constexpr (FMT == kKvF32)
                x[i] = __uint_as_float(raw[n][i]);
            else
                x[i] = h2f((uint16_t)(raw[n][i >> 1] >> (16 * (i & 1))));
        }
        __builtin_nontemporal_store(x, reinterpret_cast<floats4 *>(out + ((int64_t)j * a.rq_rows + first_row + n) * a.kv_dim + e));
    }
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
    const int64_t items = ((int64_t)a.rows + kAppendRows - 1) / kAppendRows * (2 * ((a.kv_heads + hpw - 1) / hpw) + (q ? (a.heads + hpw - 1) / hpw : 0));
    const int64_t blocks = (items + kAppendWaves - 1) / kAppendWaves;
    return by_format(a, [&](auto fmt, auto n) {
        kv_append_kernel<fmt(), n(), false><<<dim3((uint32_t)blocks, (uint32_t)a.requests), 64 * kAppendWaves, 0, s>>>(
            k, v, static_cast<uint8_t *>(kpool), static_cast<uint8_t *>(vpool), table, k_norm,
            a.rope_dim ? rope : nullptr, q, q_norm, q_out, a, dyn, nullptr);
    });
}

hipError_t launch_kv_append_slots(const float *k, const float *v, void *kpool, void *vpool, const int64_t *slots,
                                  const float *k_norm, const float2 *rope, const KvArgs &a, hipStream_t s) {
    const int hpw = heads_per_wave(a.head_dim / 64);
    const int64_t items = ((int64_t)a.rows + kAppendRows - 1) / kAppendRows * (2 * ((a.kv_heads + hpw - 1) / hpw));
    const int64_t blocks = (items + kAppendWaves - 1) / kAppendWaves;
    return by_format(a, [&](auto fmt, auto n) {
        kv_append_kernel<fmt(), n(), true><<<(uint32_t)blocks, 64 * kAppendWaves, 0, s>>>(
            k, v, static_cast<uint8_t *>(kpool), static_cast<uint8_t *>(vpool), nullptr, k_norm,
            a.rope_dim ? rope : nullptr, nullptr, nullptr, nullptr, a, ModelDyn{}, slots);
    });
}

hipError_t launch_kv_read(const void *kpool, const void *vpool, const int32_t *table, float *k_out, float *v_out,
                          const KvArgs &a, const ModelDyn &dyn, hipStream_t s) {
    const int hpw = heads_per_wave(a.head_dim / 64);
    const int64_t blocks = (((int64_t)a.rows + kReadRows - 1) / kReadRows * ((a.kv_heads + hpw - 1) / hpw) + 3) / 4;
    return by_format(a, [&](auto fmt, auto n) {
        kv_read_kernel<fmt(), n()><<<dim3((uint32_t)blocks, (uint32_t)a.requests, 2), 256, 0, s>>>(
            static_cast<const uint8_t *>(kpool), static_cast<const uint8_t *>(vpool), table, k_out, v_out, a, dyn);
    });
}

}  // namespace yk

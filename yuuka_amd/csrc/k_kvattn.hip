// k_kvattn.hip — attention of the newest rows of a batch of requests over
// their paged cache (F16 or Q8_0 pages), each request at its own length: the
// decode step of engine/gpu's session (one row) and the verify rows.
//
//   out = sum_t softmax_t(scale q . k_t) v_t,  t = 0 .. position of the row
//
// A workgroup takes one kv head of one request, up to 16 of its (row, query
// head) pairs and a range of the keys; its eight waves walk the range's
// 32-key tiles, each with a running reference, sum and output of its own, and
// are joined at the end. With more ranges than one the records {o, m, l} of
// the ranges are joined by a second kernel.
//
// Both products run on v_mfma_f32_16x16x32_f16 straight from the pages:
//  * scores = K Q^T (keys are the rows of the tile, so that a lane ends with
//    the scores of one query row and the keys 4 g .. 4 g + 3 of both 16-key
//    halves), P V with those very keys as lane g's eight: probabilities go from
//    the first product's result to the second's operand without leaving the lane;
//  * int8 digits are exact halves. A query is two halves (scaled by a power of
//    two to below 2^14), a probability times its key's scale too: products are good
//    to 2^-22, sums are float32. Key scales multiply the scores block by block
//    (an MFMA covers one block of 32 dims), value scales the probabilities.
//  * up to eight pairs ("stacked") put both halves in one 16-wide operand, as rows
//    n and n + 8; more take two MFMAs.
//  * p = 2^(s - m') with the reference m' = running max + E - 10, E the
//    exponent of the largest value scale so far: p times a scale stays below 2^14
//    and the halves' 39 octaves are used; m' moves (and the accumulators are
//    rescaled) when a tile passes it by 4.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <mutex>

#include "internal.h"
#include "kv_dev.h"
#include "refmath.h"

namespace yk {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int N> struct Dwords {  // N dwords at dword alignment
    typedef uint32_t V __attribute__((ext_vector_type(N), aligned(4)));
};
template <> struct Dwords<1> { typedef uint32_t V; };
template <int N> __device__ __forceinline__ uint32_t dword(const typename Dwords<N>::V &v, int i) { return v[i]; }
template <> __device__ __forceinline__ uint32_t dword<1>(const uint32_t &v, int) { return v; }

constexpr int kWaves = 8, kTile = 32;
constexpr float kHeadroom = 10.0f, kSlack = 4.0f;

__device__ __forceinline__ float max_rows(float x) {  // over the four 16-lane rows
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_halves(float x) {  // lane l and l ^ 32
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float sum_rows(float x) {
    x = sum_halves(x);
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float ror8(float x) {  // lane (l + 8) % 16 of the row
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, true));
}
__device__ __forceinline__ half2v to_half2(float a, float b) {
    return __builtin_convertvector((float2v){a, b}, half2v);
}
__device__ __forceinline__ half8 join(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ void wave_lds_fence() {  // the wave's LDS writes are in order before its reads
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Two digits of a dword of keys as halves: 0x6400 | u is 1024 + u.
template <int H>
__device__ __forceinline__ half2v key_digits(uint32_t biased) {
    const uint32_t u = __builtin_amdgcn_perm(0x64646464u, biased, H ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(half2v, u) + half2v{(_Float16)-1152.0f, (_Float16)-1152.0f};
}
// Digit J of two keys' dwords, times 2^-9: u as a subnormal half is u 2^-24.
template <int J>
__device__ __forceinline__ half2v value_digits(uint32_t x, uint32_t y) {
    const uint32_t u = __builtin_amdgcn_perm(y, x, 0x0c000c00u | ((4u + J) << 16) | J);
    return __builtin_elementwise_fma(__builtin_bit_cast(half2v, u), half2v{(_Float16)32768.0f, (_Float16)32768.0f},
                                     half2v{(_Float16)-0.25f, (_Float16)-0.25f});
}
// Half J of two keys' four values.
template <int J>
__device__ __forceinline__ half2v value_halves(u32x2 x, u32x2 y) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(y[J >> 1], x[J >> 1], J & 1 ? 0x07060302u : 0x05040100u));
}

template <int FMT, int GROUPS, bool STACK, bool PAGED> struct Layout {
    static constexpr bool Q8 = FMT == kKvQ8;
    static constexpr int D = 64 * GROUPS, NB = 2 * GROUPS, ROWS = STACK ? 8 : 16;
    static constexpr uint32_t plane = NB * 1024;                              // query operands, one half
    static constexpr uint32_t scales = STACK ? plane : 2 * plane;             // [wave][key, value][GROUPS][32] dwords
    static constexpr uint32_t addr = scales + (Q8 ? kWaves * 256 * GROUPS : 0);  // [wave][32] row offsets
    static constexpr uint32_t loop = addr + (PAGED ? 0 : kWaves * 256);
    static constexpr int slot_row = D + 4;                                    // floats; rows 4 g land 16 banks apart
    static constexpr uint32_t slots = kWaves * ROWS * slot_row * 4;           // over the loop's areas, after it
    static constexpr uint32_t stats = loop > slots ? loop : slots;            // m[8][16], l[8][16], factor[16]
    static constexpr uint32_t total = stats + (2 * kWaves + 1) * 16 * 4;
};

struct AttnSplit {
    int splits, row_blocks;
    int page_shift;  // PAGED: log2(block_size / 16)
};

// 512 threads. PAGED: pages are 16 << page_shift tokens, so that a 16-key half
// of a tile lies in one page, found by scalar loads and read through a
// buffer resource of that page's bytes (none for an unmapped page or past the end:
// such loads cost nothing and give zeros).
template <int FMT, int GROUPS, bool STACK, bool PAGED>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void kv_attention_kernel(
    const float *__restrict__ q, int q_stride, const float *__restrict__ gate, int gate_stride,
    const uint8_t *__restrict__ kpool, const uint8_t *__restrict__ vpool, const int32_t *__restrict__ table, KvArgs a,
    AttnSplit sp, float *__restrict__ part, float2 *__restrict__ stats, float *__restrict__ out, ModelDyn dyn) {
    using L = Layout<FMT, GROUPS, STACK, PAGED>;
    constexpr bool Q8 = L::Q8;
    constexpr int D = L::D, NB = L::NB, ROWS = L::ROWS;
    constexpr int KP = Q8 ? GROUPS : 2 * GROUPS;  // 16-byte pieces of a key per lane
    extern __shared__ __align__(16) uint8_t lds[];
    float *const st_m = reinterpret_cast<float *>(lds + L::stats), *const st_l = st_m + kWaves * 16;
    float *const row_factor = st_l + kWaves * 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int r16 = lane & 15, g4 = lane >> 4;
    int bx = blockIdx.x;
    const int rb = bx % sp.row_blocks;
    bx /= sp.row_blocks;
    const int split = bx % sp.splits, kvh = bx / sp.splits, j = blockIdx.y;
    const int G = a.heads / a.kv_heads;
    const int n0 = rb * ROWS, nr = min(ROWS, G * a.rows - n0);  // pairs n = row * G + head of the group
    const int64_t p0 = kv_position(a, dyn, j, 0);
    // last key a row sees, -1 for none
    auto limit = [&](int n) { return (int)max((int64_t)-1, min(p0 + n / G, (int64_t)a.capacity - 1)); };
    const int len = __builtin_amdgcn_readfirstlane(limit(n0 + nr - 1) + 1);
    const int least = __builtin_amdgcn_readfirstlane(limit(n0));
    const int tiles = (len + kTile - 1) / kTile;
    const int per = max((tiles + sp.splits - 1) / sp.splits, kWaves);
    const int c0 = split * per, c1 = min(tiles, c0 + per);
    const int64_t out_row = (int64_t)j * a.rq_rows;
    if (c0 >= c1 && sp.splits > 1) {  // nothing here: an empty record
        if (threadIdx.x < (uint32_t)nr) {
            const int n = n0 + threadIdx.x, r = n / G, h = kvh * G + n % G;
            stats[(((int64_t)j * a.rows + r) * a.heads + h) * sp.splits + split] = make_float2(-INFINITY, 0.0f);
        }
        return;
    }

    // the query rows that this wave prepares: loaded before the first tile, since
    // loads return in order
    float queries[ROWS / kWaves][GROUPS];
#pragma unroll
    for (int half = 0; half < ROWS / kWaves; half++) {
        const int n = min(wave + kWaves * half, nr - 1), r = (n0 + n) / G, h = kvh * G + (n0 + n) % G;
#pragma unroll
        for (int s = 0; s < GROUPS; s++) {
            const float x = q[((out_row + r) * a.heads + h) * q_stride + 64 * s + lane];
            queries[half][s] = wave + kWaves * half < nr ? x : 0.0f;
        }
    }

    // ---- pages of a tile's halves, and which of its keys there are
    const int32_t *const table_j = table + (int64_t)j * kv_table_blocks(a);
    const uint32_t page_bytes = (uint32_t)kv_page_bytes(a);
    const uint32_t row_bytes = Q8 ? a.kv_dim : a.kv_dim * 2;
    // (PAGED: everything uniform, made scalar by hand; a buffer resource out of
    // vector registers costs every load a loop over the lanes)
    struct Tile {
        uint64_t row[2], scales[2];  // offsets in the pools: first token of each half, and its scales
        uint32_t bytes[2];           // from there to the end of the page; 0: unmapped or past the end
        uint32_t keys;               // bit k: key k of the tile is there
    };
    auto scalar64 = [](uint64_t x) {  // (the builtin's result is a signed int)
        const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
        const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
        return (uint64_t)hi << 32 | lo;
    };
    auto pages_of = [&](int c) {
        Tile t{};
        if constexpr (PAGED) {
#pragma unroll
            for (int T = 0; T < 2; T++) {
                const int tok = kTile * c + 16 * T;
                int page = -1;
                if (c < c1 && tok < len) page = __builtin_amdgcn_readfirstlane(table_j[tok >> (4 + sp.page_shift)]);
                const bool mapped = (uint32_t)page < (uint32_t)a.pages;
                const uint32_t in = tok & ((16u << sp.page_shift) - 1);  // tokens before the half in its page
                const uint64_t at = (uint64_t)(mapped ? (uint32_t)page : 0u) * page_bytes;
                t.row[T] = scalar64(at + in * row_bytes);
                t.scales[T] = scalar64(at + a.block_size * row_bytes + in * (a.kv_dim / 16));
                t.bytes[T] = __builtin_amdgcn_readfirstlane(mapped ? page_bytes - in * row_bytes : 0u);
                if (mapped) t.keys |= (0xffffu >> max(0, tok + 16 - len)) << (16 * T);
            }
            t.keys = __builtin_amdgcn_readfirstlane(t.keys);
        }
        return t;
    };
    // ---- loads of one tile
    u32x4 kreg[2][KP];
    uint32_t vdig[Q8 ? 8 : 1][GROUPS];
    u32x2 vhalf[Q8 ? 1 : 8][GROUPS];
    typename Dwords<GROUPS>::V sreg;  // lanes 0..31: scales of key `lane`, 32..63: of value `lane - 32`
    const uint8_t *krow[PAGED ? 1 : 2], *vrow[PAGED ? 1 : 8];  // rows of the tile to be loaded
    uint32_t koff = r16 * row_bytes + kvh * D * (Q8 ? 1 : 2) + 16 * g4;
    const uint32_t voff = 4 * g4 * row_bytes + kvh * D * (Q8 ? 1 : 2) + r16 * (Q8 ? 4 : 8);
    uint32_t voff_row[4] = {voff, voff + row_bytes, voff + 2 * row_bytes, voff + 3 * row_bytes};
    auto resource = [&](const uint8_t *pool, const Tile &t, int T) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(pool) + (PAGED ? t.row[T] : 0), (short)0,
                                                 PAGED ? (int)t.bytes[T] : 0, 0x00020000);
    };
    // LDS offsets of the wave's scales: where the lane's key goes, and keys 4 g4 .. + 3
    uint32_t scale_write = L::scales + wave * 256 * GROUPS + (lane >> 5) * 128 * GROUPS + (lane & 31) * 4;
    uint32_t scale_read = L::scales + wave * 256 * GROUPS + g4 * 16;
    uint32_t query_read = lane * 16;  // of the lane's operands
    int64_t *const my_addr = reinterpret_cast<int64_t *>(lds + L::addr) + wave * 32;
    const uint32_t soff = (lane & 15) * (a.kv_dim / 16) + kvh * NB * 2;
    auto load_scales = [&](const Tile &t) {  // (an unmapped half reads page 0's: not used)
        if constexpr (Q8 && PAGED) {
            const uint8_t *k0 = kpool + t.scales[0], *k1 = kpool + t.scales[1];
            const uint8_t *v0 = vpool + t.scales[0], *v1 = vpool + t.scales[1];
            const uint8_t *at = (lane < 32 ? (lane & 16 ? k1 : k0) : (lane & 16 ? v1 : v0)) + soff;
            sreg = *reinterpret_cast<const typename Dwords<GROUPS>::V *>(at);
        }
    };
    // !PAGED: every lane finds the row (and the scales) of key `lane & 31`
    auto find_rows = [&](int c) {
        Tile t{};
        if constexpr (!PAGED) {
            const int key = kTile * c + (lane & 31);
            int64_t row = 0, sc = 0;
            const bool there = c < c1 && key < len && kv_slot(a, table, j, key, &row, &sc);
            t.keys = (uint32_t)__builtin_amdgcn_ballot_w64(there);
            wave_lds_fence();
            if (lane < 32) my_addr[lane] = there ? row : 0;
            wave_lds_fence();
#pragma unroll
            for (int T = 0; T < 2; T++) krow[T] = kpool + my_addr[16 * T + r16] + (koff - r16 * row_bytes);
#pragma unroll
            for (int i = 0; i < 8; i++)
                vrow[i] = vpool + my_addr[16 * (i >> 2) + 4 * g4 + (i & 3)] + (voff - 4 * g4 * row_bytes);
            if constexpr (Q8)
                sreg = *reinterpret_cast<const typename Dwords<GROUPS>::V *>((lane < 32 ? kpool : vpool) +
                                                                             (there ? sc + kvh * NB * 2 : 0));
        }
        return t;
    };
    auto load_key = [&](__amdgpu_buffer_rsrc_t rs, int T, int p) {
        if constexpr (PAGED)
            kreg[T][p] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, koff + 64 * p, 0, 0));
        else
            kreg[T][p] = *reinterpret_cast<const typename Dwords<4>::V *>(krow[T] + 64 * p);
    };
    auto load_value = [&](__amdgpu_buffer_rsrc_t rs, int i, int s) {
        const uint32_t off = voff_row[i & 3];
        if constexpr (Q8 && PAGED) vdig[i][s] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, off + 64 * s, 0, 0);
        else if constexpr (Q8) vdig[i][s] = *reinterpret_cast<const uint32_t *>(vrow[i] + 64 * s);
        else if constexpr (PAGED)
            vhalf[i][s] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, off + 128 * s, 0, 0));
        else
            vhalf[i][s] = *reinterpret_cast<const typename Dwords<2>::V *>(vrow[i] + 128 * s);
    };
    int c = c0 + wave;
    Tile cur = PAGED ? pages_of(c) : find_rows(c);
    load_scales(cur);
    {
        const auto k0 = resource(kpool, cur, 0), k1 = resource(kpool, cur, 1);
        const auto v0 = resource(vpool, cur, 0), v1 = resource(vpool, cur, 1);
#pragma unroll
        for (int p = 0; p < KP; p++) {
            load_key(k0, 0, p);
            load_key(k1, 1, p);
        }
#pragma unroll
        for (int s = 0; s < GROUPS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) load_value(i < 4 ? v0 : v1, i, s);
    }

    // ---- queries as MFMA operands in LDS: wave w prepares rows w and w + 8
#pragma unroll
    for (int half = 0; half < ROWS / kWaves; half++) {
        const int n = wave + kWaves * half;
        const float(&x)[GROUPS] = queries[half];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < GROUPS; s++) top = fmaxf(top, fabsf(x[s]));
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
        int e = 14;
        if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e);  // top < 2^e
        const int in = Q8 ? lane : 0;
        // dim 64 s + lane: block 2 s + h, lane group g, place k of the operand's eight
        const int hb = Q8 ? in >> 5 : lane >> 5;
        const int g = Q8 ? (lane & 15) >> 2 : (lane & 31) >> 3;
        const int k = Q8 ? 2 * (lane & 3) + ((lane >> 4) & 1) : lane & 7;
#pragma unroll
        for (int s = 0; s < GROUPS; s++) {
            const float y = ldexpf(x[s], 14 - e);
            const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
            const uint32_t at = ((2 * s + hb) * 64 + 16 * g + n) * 16 + 2 * k;
            *reinterpret_cast<_Float16 *>(lds + at) = hi;
            *reinterpret_cast<_Float16 *>(lds + at + (STACK ? 8 * 16 : L::plane)) = lo;
        }
        // scores in units of log2: factor * (operand product)
        if (lane == 0) row_factor[n] = ldexpf(a.scale * 1.44269504088896341f, e - 14);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");

    const int my_n = STACK ? r16 & 7 : r16;
    const float factor = row_factor[my_n];
    const int my_limit = my_n < nr ? limit(n0 + my_n) : -1;
    const bool low_half = STACK && r16 >= 8;  // this lane's probabilities are the remainders
    f32x4 acc[GROUPS][4];
#pragma unroll
    for (int s = 0; s < GROUPS; s++)
#pragma unroll
        for (int t = 0; t < 4; t++) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref = -INFINITY, l = 0.0f;

    Tile next{};
    if constexpr (PAGED) next = pages_of(c + kWaves);
    for (; c < c1; c += kWaves) {
        // Opaque in every turn: the constant steps from these addresses then stay
        // in the instructions' immediate offsets. Hoisted out of the loop they take a
        // register each, loaded values spill, and every spill waits for all loads.
        asm volatile("" : "+v"(koff), "+v"(voff_row[0]), "+v"(voff_row[1]), "+v"(voff_row[2]), "+v"(voff_row[3]));
        asm volatile("" : "+v"(scale_write), "+v"(scale_read), "+v"(query_read));
        // every row sees every key of the tile
        const bool whole = cur.keys == ~0u && kTile * c + kTile - 1 <= least;
        float E = 0.0f;
        uint32_t poison = 0;  // keys with a non-finite value that not every row sees: left out, their rows made NaN
        if constexpr (Q8) {
            // scales to LDS (those of missing keys as zeros), and the largest finite value scale's exponent
            wave_lds_fence();
            const bool there = (cur.keys >> (lane & 31)) & 1;
            uint32_t d[GROUPS], most = 0, over = 0;
#pragma unroll
            for (int s = 0; s < GROUPS; s++) {
                d[s] = there ? dword<GROUPS>(sreg, s) : 0u;
                const uint32_t lo = d[s] & 0x7fffu, hi = (d[s] >> 16) & 0x7fffu;
                most = max(most, max(lo < 0x7c00u ? lo : 0u, hi < 0x7c00u ? hi : 0u));
                over |= ((d[s] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
            }
            if (!whole) {
                const uint64_t b = __builtin_amdgcn_ballot_w64(over != 0 && kTile * c + (lane & 31) > least);
                poison = (uint32_t)(b >> 32);
                if (lane >= 32 && (poison >> (lane & 31)) & 1) {
#pragma unroll
                    for (int s = 0; s < GROUPS; s++) d[s] = 0;
                }
            }
#pragma unroll
            for (int s = 0; s < GROUPS; s++) *reinterpret_cast<uint32_t *>(lds + scale_write + 128 * s) = d[s];
            float m = __uint_as_float(lane < 32 ? 0u : most);  // non-negative: ordered as floats
            m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0xb1, 0xf, 0xf, true)));
            m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x4e, 0xf, 0xf, true)));
            m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x124, 0xf, 0xf, true)));
            m = fmaxf(m, ror8(m));
            m = max_rows(m);
            E = (float)((int)(__float_as_uint(m) >> 10) - 14);  // scale < 2^E
            wave_lds_fence();
        }
        Tile after{};
        if constexpr (!PAGED) next = find_rows(c + kWaves);
        // ---- scores: keys 4 g + e of half T against query row r16
        float s[2][4] = {};
        {
            u32x4 ks[2];  // two blocks' scales of the lane's keys
            const auto k0 = resource(kpool, next, 0), k1 = resource(kpool, next, 1);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if constexpr (Q8) {
                    if (!(b & 1))
#pragma unroll
                        for (int T = 0; T < 2; T++)
                            ks[T] = *reinterpret_cast<const u32x4 *>(lds + scale_read + (b >> 1) * 128 + 64 * T);
                }
                const half8 qh = *reinterpret_cast<const half8 *>(lds + query_read + b * 1024);
                half8 ql{};
                if constexpr (!STACK) ql = *reinterpret_cast<const half8 *>(lds + query_read + L::plane + b * 1024);
#pragma unroll
                for (int T = 0; T < 2; T++) {
                    half8 kk;
                    if constexpr (Q8) {
                        const u32x4 w = kreg[T][b >> 1] ^ 0x80808080u;
                        kk = b & 1 ? join(key_digits<1>(w[0]), key_digits<1>(w[1]), key_digits<1>(w[2]), key_digits<1>(w[3]))
                                   : join(key_digits<0>(w[0]), key_digits<0>(w[1]), key_digits<0>(w[2]), key_digits<0>(w[3]));
                    } else {
                        kk = __builtin_bit_cast(half8, kreg[T][b]);
                    }
                    f32x4 d = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (!Q8) d = f32x4{s[T][0], s[T][1], s[T][2], s[T][3]};
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qh, d, 0, 0, 0);
                    if constexpr (!STACK) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, ql, d, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (Q8)
                            s[T][e] = fmaf(d[e], (float)__builtin_bit_cast(half2v, (uint32_t)ks[T][e])[b & 1], s[T][e]);
                        else
                            s[T][e] = d[e];
                    }
                }
                if (!Q8 || (b & 1)) {
                    load_key(k0, 0, Q8 ? b >> 1 : b);
                    load_key(k1, 1, Q8 ? b >> 1 : b);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        load_scales(next);
        if constexpr (PAGED) after = pages_of(c + 2 * kWaves);
        // ---- softmax of the lane's row over its eight keys
        float top = -INFINITY;
#pragma unroll
        for (int T = 0; T < 2; T++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (STACK) s[T][e] += ror8(s[T][e]);
                s[T][e] *= factor;
            }
        if (!whole) {
            int first = 4 * g4;  // opaque: what follows is not kept in registers for every tile
            asm volatile("" : "+v"(first));
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int kk = first + 16 * (i >> 2) + (i & 3);
                bool there = (cur.keys >> kk) & 1, bad = (poison >> kk) & 1;
                if constexpr (!Q8) {  // values that not every row sees must be finite for those that do not
                    uint32_t over = 0;
#pragma unroll
                    for (int u = 0; u < GROUPS; u++)
#pragma unroll
                        for (int w = 0; w < 2; w++) over |= (vhalf[i][u][w] & 0x7fff7fffu) + 0x04000400u;
                    const uint64_t b = __builtin_amdgcn_ballot_w64((over & 0x80008000u) != 0);
                    bad = ((b >> (4 * first)) & 0xffffu) != 0 && kTile * c + kk > least;
                    if (!there || bad) {
#pragma unroll
                        for (int u = 0; u < GROUPS; u++) vhalf[i][u] = u32x2{0, 0};
                    }
                }
                const bool seen = there && kTile * c + kk <= my_limit;
                s[i >> 2][i & 3] = !seen ? -INFINITY : bad ? NAN : s[i >> 2][i & 3];
            }
        }
#pragma unroll
        for (int T = 0; T < 2; T++)
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, s[T][e]);
        top = max_rows(top) + (E - kHeadroom);
        if (__any(top > ref + kSlack)) {
            const float moved = fmaxf(ref, top);
            const float shrink = moved == ref ? 1.0f : __builtin_amdgcn_exp2f(ref - moved);
            ref = moved;
            l *= shrink;
            float row_shrink[4];
#pragma unroll
            for (int e = 0; e < 4; e++) row_shrink[e] = __shfl(shrink, 4 * g4 + e);
#pragma unroll
            for (int u = 0; u < GROUPS; u++)
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[u][t][e] *= row_shrink[e];
        }
        float p[8];
        {
            const float base = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                p[i] = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] - base);
                l += p[i];
            }
        }
        // ---- value product: keys 4 g + e of both halves are the lane's eight
        {
            u32x4 vs[2];  // two blocks' scales of the lane's keys
            const auto v0 = resource(vpool, next, 0), v1 = resource(vpool, next, 1);
            half8 ph, pl;
            // p[i] * d(i) as two halves (stacked: the one that the lane's row is)
            auto halves = [&](auto d) {
                half2v h[4], o[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = d(2 * i), y = d(2 * i + 1);
                    h[i] = half2v{(_Float16)fmaf(p[2 * i], x, 0.0f), (_Float16)fmaf(p[2 * i + 1], y, 0.0f)};
                    o[i] = half2v{(_Float16)fmaf(p[2 * i], x, -(float)h[i][0]), (_Float16)fmaf(p[2 * i + 1], y, -(float)h[i][1])};
                    // one value h in every lane: rounded twice by different
                    // instructions, the two rows' halves need not be each other's
                    if constexpr (STACK) o[i] = low_half ? o[i] : h[i];
                }
                ph = join(h[0], h[1], h[2], h[3]);
                pl = join(o[0], o[1], o[2], o[3]);
            };
            if constexpr (!Q8) halves([](int) { return 1.0f; });
#pragma unroll
            for (int u = 0; u < GROUPS; u++) {
                uint32_t w[8];
                if constexpr (Q8) {
#pragma unroll
                    for (int T = 0; T < 2; T++)
                        vs[T] = *reinterpret_cast<const u32x4 *>(lds + scale_read + (GROUPS + u) * 128 + 64 * T);
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = vdig[i][u] ^ 0x80808080u;
                }
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    half8 vv;
                    if constexpr (Q8) {
                        if (!(t & 1))  // block 2 u + t / 2
                            halves([&](int i) {
                                return (float)__builtin_bit_cast(half2v, (uint32_t)vs[i >> 2][i & 3])[t >> 1];
                            });
                        vv = t == 0   ? join(value_digits<0>(w[0], w[1]), value_digits<0>(w[2], w[3]), value_digits<0>(w[4], w[5]), value_digits<0>(w[6], w[7]))
                             : t == 1 ? join(value_digits<1>(w[0], w[1]), value_digits<1>(w[2], w[3]), value_digits<1>(w[4], w[5]), value_digits<1>(w[6], w[7]))
                             : t == 2 ? join(value_digits<2>(w[0], w[1]), value_digits<2>(w[2], w[3]), value_digits<2>(w[4], w[5]), value_digits<2>(w[6], w[7]))
                                      : join(value_digits<3>(w[0], w[1]), value_digits<3>(w[2], w[3]), value_digits<3>(w[4], w[5]), value_digits<3>(w[6], w[7]));
                    } else {
                        auto pairs = [&](auto J) {
                            return join(value_halves<J()>(vhalf[0][u], vhalf[1][u]), value_halves<J()>(vhalf[2][u], vhalf[3][u]),
                                        value_halves<J()>(vhalf[4][u], vhalf[5][u]), value_halves<J()>(vhalf[6][u], vhalf[7][u]));
                        };
                        vv = t == 0   ? pairs(std::integral_constant<int, 0>{})
                             : t == 1 ? pairs(std::integral_constant<int, 1>{})
                             : t == 2 ? pairs(std::integral_constant<int, 2>{})
                                      : pairs(std::integral_constant<int, 3>{});
                    }
                    if constexpr (!STACK) acc[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, vv, acc[u][t], 0, 0, 0);
                    acc[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, vv, acc[u][t], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) load_value(i < 4 ? v0 : v1, i, u);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        cur = next;
        if constexpr (PAGED) next = after;
    }

    // ---- the waves' outputs joined: o = sum_w 2^(ref_w - max ref) o_w
    l = sum_rows(l);
    __syncthreads();  // every wave is done with the operands the slots lie over
    {
        float *const slot = reinterpret_cast<float *>(lds) + wave * ROWS * L::slot_row;
        const float unit = Q8 ? 512.0f : 1.0f;  // the digits were times 2^-9
#pragma unroll
        for (int u = 0; u < GROUPS; u++)
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float x = acc[u][t][e] * unit;
                    if constexpr (STACK) x = sum_halves(x);  // rows n and n + 8
                    if (!STACK || g4 < 2)
                        slot[(4 * g4 + e) * L::slot_row + 64 * u + (Q8 ? 16 * t + r16 : 4 * r16 + t)] = x;
                }
        if (lane < ROWS) {
            st_m[wave * 16 + lane] = ref;
            st_l[wave * 16 + lane] = l;
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < nr * (D / 4); idx += 64 * kWaves) {
        const int n = idx / (D / 4), d = 4 * (idx % (D / 4));
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; w++) m = fmaxf(m, st_m[w * 16 + n]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float mw = st_m[w * 16 + n];
            const float f = mw == m ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
            const f32x4 x = *reinterpret_cast<const f32x4 *>(lds + ((w * ROWS + n) * L::slot_row + d) * 4);
            o += f * x;
            total = fmaf(f, st_l[w * 16 + n], total);
        }
        const int r = (n0 + n) / G, h = kvh * G + (n0 + n) % G;
        if (sp.splits == 1) {
            const int64_t at = (out_row + r) * a.heads + h;
            const float inv = 1.0f / total;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float y = total == 0.0f ? 0.0f : o[i] * inv;  // a row that sees no key
                if (gate) y *= sigmoid_ref(gate[at * gate_stride + d + i]);
                out[at * D + d + i] = y;
            }
        } else {
            const int64_t rec = (((int64_t)j * a.rows + r) * a.heads + h) * sp.splits + split;
            *reinterpret_cast<f32x4 *>(part + rec * D + d) = o;
            if (d == 0) stats[rec] = make_float2(m, total);
        }
    }
}

// One workgroup of four waves per (row, head, request): joins the ranges'
// records. The weights come first, a range a thread; then wave w adds the
// ranges w, w + 4, ... with four loads in flight, a lane four dims (or two, or
// one: D / 64).
constexpr int kMaxSplits = 256;

template <int GROUPS>
__global__ __launch_bounds__(256) void kv_attention_merge_kernel(const float *__restrict__ part,
                                                                 const float2 *__restrict__ stats, int splits,
                                                                 const float *__restrict__ gate, int gate_stride,
                                                                 float *__restrict__ out, KvArgs a) {
    constexpr int D = 64 * GROUPS;
    __shared__ float weight[kMaxSplits], red[2][4];
    __shared__ float sum[4][D];
    const int r = blockIdx.x, h = blockIdx.y, j = blockIdx.z, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t rec = (((int64_t)j * a.rows + r) * a.heads + h) * splits;
    const int64_t row = ((int64_t)j * a.rq_rows + r) * a.heads + h;
    const float2 ml = tid < splits ? stats[rec + tid] : make_float2(-INFINITY, 0.0f);
    float g = 0.0f;
    if (gate && tid < D) g = gate[row * gate_stride + tid];
    float m = ml.x;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    // a range without keys (no sum) weighs nothing, whatever its output holds
    const float w = ml.y == 0.0f ? 0.0f : ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m);
    weight[tid] = ml.y == 0.0f ? -1.0f : w;
    float l = w * ml.y;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off);
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    float o[GROUPS] = {};
    for (int s0 = wave; s0 < splits; s0 += 16) {
        float x[4][GROUPS], f[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int s = s0 + 4 * u;
            f[u] = s < splits ? weight[s] : -1.0f;
#pragma unroll
            for (int i = 0; i < GROUPS; i++) x[u][i] = f[u] >= 0.0f ? part[(rec + s) * D + 64 * i + lane] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < GROUPS; i++)
                if (f[u] >= 0.0f) o[i] = fmaf(f[u], x[u][i], o[i]);
    }
#pragma unroll
    for (int i = 0; i < GROUPS; i++) sum[wave][64 * i + lane] = o[i];
    __syncthreads();
    if (tid < D) {
        float y = (sum[0][tid] + sum[1][tid]) + (sum[2][tid] + sum[3][tid]);
        y = l == 0.0f ? 0.0f : y / l;  // a row that sees no key
        if (gate) y *= sigmoid_ref(g);
        out[row * D + tid] = y;
    }
}

bool stacked(const KvArgs &a) { return a.heads / a.kv_heads * a.rows <= 8; }
int row_blocks(const KvArgs &a) {
    const int pairs = a.heads / a.kv_heads * a.rows, per = stacked(a) ? 8 : 16;
    return (pairs + per - 1) / per;
}

int kv_splits(const KvArgs &a) {
    const int64_t work = (int64_t)a.kv_heads * a.requests * row_blocks(a);
    const int64_t want = (kMaxSplits + work - 1) / work, most = (a.capacity + kWaves * kTile - 1) / (kWaves * kTile);
    return (int)std::max<int64_t>(1, std::min(want, most));
}

uint64_t kv_records(const KvArgs &a) { return (uint64_t)a.requests * a.rows * a.heads * kv_splits(a); }

}  // namespace

uint64_t kv_attention_scratch_bytes(const KvArgs &a) {
    const int splits = kv_splits(a);
    return splits == 1 ? 0 : kv_records(a) * (a.head_dim + 2) * 4;  // outputs, then {m, l}
}

hipError_t launch_kv_attention(const float *q, int q_stride, const float *gate, int gate_stride, const void *kpool,
                               const void *vpool, const int32_t *table, float *out, const KvArgs &a, void *scratch,
                               const ModelDyn &dyn, hipStream_t s) {
    AttnSplit sp{kv_splits(a), row_blocks(a), 0};
    while ((16 << sp.page_shift) < a.block_size) sp.page_shift++;
    const bool paged = (16 << sp.page_shift) == a.block_size;
    float *part = static_cast<float *>(scratch);
    float2 *stats = part ? reinterpret_cast<float2 *>(part + kv_records(a) * a.head_dim) : nullptr;
    hipError_t err = hipSuccess;
    auto launch = [&](auto fmt, auto groups, auto stack, auto pages) {
        constexpr auto kernel = kv_attention_kernel<fmt(), groups(), stack(), pages()>;
        constexpr uint32_t bytes = Layout<fmt(), groups(), stack(), pages()>::total;
        static std::once_flag once;
        std::call_once(once, [&] {
            (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)bytes);
        });
        kernel<<<dim3((uint32_t)((int64_t)sp.splits * sp.row_blocks * a.kv_heads), a.requests), 64 * kWaves, bytes, s>>>(
            q, q_stride, gate, gate_stride, static_cast<const uint8_t *>(kpool), static_cast<const uint8_t *>(vpool), table,
            a, sp, part, stats, out, dyn);
        err = hipGetLastError();
    };
    auto by_pages = [&](auto fmt, auto groups) {
        if (!paged) launch(fmt, groups, std::false_type{}, std::false_type{});
        else if (stacked(a)) launch(fmt, groups, std::true_type{}, std::true_type{});
        else launch(fmt, groups, std::false_type{}, std::true_type{});
    };
    auto by_width = [&](auto fmt) {
        switch (a.head_dim / 64) {
        case 1: by_pages(fmt, std::integral_constant<int, 1>{}); break;
        case 2: by_pages(fmt, std::integral_constant<int, 2>{}); break;
        case 3: by_pages(fmt, std::integral_constant<int, 3>{}); break;
        default: by_pages(fmt, std::integral_constant<int, 4>{}); break;
        }
    };
    if (a.fmt == kKvF16) by_width(std::integral_constant<int, kKvF16>{});
    else by_width(std::integral_constant<int, kKvQ8>{});
    if (err != hipSuccess || sp.splits == 1) return err;
    auto merge = a.head_dim == 64    ? kv_attention_merge_kernel<1>
                 : a.head_dim == 128 ? kv_attention_merge_kernel<2>
                 : a.head_dim == 192 ? kv_attention_merge_kernel<3>
                                     : kv_attention_merge_kernel<4>;
    merge<<<dim3(a.rows, a.heads, a.requests), 256, 0, s>>>(part, stats, sp.splits, gate, gate_stride, out, a);
    return hipGetLastError();
}

}  // namespace yk

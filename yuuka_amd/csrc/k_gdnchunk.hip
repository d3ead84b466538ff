// k_gdnchunk.hip — the gated delta rule over whole prompts (recurrent.go:56-105),
// 64 rows at a time.
//
// With c_i the sum of the log decays of a chunk's rows up to i, and S the state before it,
//   A_ij = beta_i (k_i . k_j) e^(c_i - c_j)  for i > j,    T = (I + A)^-1
//   V' = T (beta V - beta e^c (K S))             the rows' corrections, d_i in the rule
//   out = e^c (Q S) + P V',     P_ij = (q_i . k_j) e^(c_i - c_j)  for i >= j
//   S <- e^(c_last) S + K^T diag(e^(c_last - c)) V'
// The first kernel makes T and P of every chunk and head, all chunks at once; the second
// walks the chunks of a request with S in registers. Row after row, with two sums over the workgroup each, 8191 rows
// of 16 heads of 128 in F32 take 17.7 ms; 64 at a time 0.43.
//
// The bytes that cannot be done without are 0.27 GB there, 56 us at the rate of a large copy, and the products 0.1 TFLOP of
// bf16. Neither binds: the second kernel's chain does, 2.7 us a chunk (2.0 with nothing loaded from memory), of three
// phases that each write LDS, wait for a barrier, read LDS and run a chain of matrix instructions. Matrix
// instructions are busy 24 % of the cycles of the 128 CUs that have a workgroup, vector ones issue in 57 %.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "gdn_ragged_dev.h"
#include "internal.h"

namespace yk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kC = 64;             // rows of a chunk
constexpr int kRowPitch = kC + 4;  // floats of a row of A in LDS
constexpr float kLeast = -200.0f;  // e^-200 is zero in float32, and the sums of 64 stay exact to 1e-12 in float64
constexpr f32x4 kZero = {0.f, 0.f, 0.f, 0.f};

// Products on v_mfma_f32_16x16x4_f32. Lane l has row (A) or column (B) l % 16 and, of 16 terms of
// the sum, 4 (l / 16) + e in the e-th of four instructions; the result's lane has column l % 16 and
// rows 4 (l / 16) + e. A result is thus the next product's B operand, or the A operand of its
// transpose, in the registers that it is in.
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// The same for 32 terms on v_mfma_f32_16x16x32_bf16, lane l with terms 4 (l / 16) + e of two tiles of 16:
// a float32 is the sum of three bf16 (8 bits each, cut off), a half of two. Of the products of parts those
// below 2^-23 of the whole are left out: six instructions of 16 cycles for eight of 32.
// The first part's product with the first is summed apart from the small ones.
struct Sum {
    f32x4 big, small;
    __device__ __forceinline__ f32x4 all() const { return big + small; }
};
template <int NA, int NB>
__device__ __forceinline__ void mma32(const u32x4 (&a)[NA], const u32x4 (&b)[NB], Sum &c) {
#pragma unroll
    for (int order = 2; order >= 0; order--)
#pragma unroll
        for (int i = 0; i < NA; i++)
#pragma unroll
            for (int k = 0; k < NB; k++) {
                if (i + k != order) continue;
                f32x4 &to = order ? c.small : c.big;
                to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[i]), __builtin_bit_cast(bf16x8, b[k]),
                                                             to, 0, 0, 0);
            }
}
// The first N parts of two values, one dword each.
template <int N> __device__ __forceinline__ void split(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
        p[i] = __builtin_amdgcn_perm(v, u, 0x07060302u);
        if (i == N - 1) break;
        x -= __uint_as_float(u & 0xffff0000u);
        y -= __uint_as_float(v & 0xffff0000u);
    }
}
template <int N> __device__ __forceinline__ void split(f32x4 x, u32x2 (&p)[N]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t d[N];
        split(x[2 * i], x[2 * i + 1], d);
#pragma unroll
        for (int k = 0; k < N; k++) p[k][i] = d[k];
    }
}
template <int N> __device__ __forceinline__ void split(f32x4 x, f32x4 y, u32x4 (&p)[N]) {
    u32x2 a[N], b[N];
    split(x, a);
    split(y, b);
#pragma unroll
    for (int k = 0; k < N; k++) p[k] = u32x4{a[k][0], a[k][1], b[k][0], b[k][1]};
}
// bf16 parts that hold a row's element exactly.
template <typename E> constexpr int kParts = std::is_same<E, RowF32>::value ? 3 : std::is_same<E, RowF16>::value ? 2 : 1;

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
// Whether any value of a wave is not finite: zero times such a value is NaN, and so is a sum with it.
template <int N> __device__ __forceinline__ bool any_not_finite(const f32x4 (&x)[N]) {
    float zero = 0.0f;
#pragma unroll
    for (int c = 0; c < N; c++)
#pragma unroll
        for (int e = 0; e < 4; e++) zero = fmaf(x[c][e], 0.0f, zero);
    return __builtin_amdgcn_ballot_w64(zero != 0.0f) != 0;
}
// Of two bf16 first parts, all bits of those that are finite (a part has the value's exponent).
__device__ __forceinline__ uint32_t finite_halves(uint32_t u) {
    return ((u & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((u & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
}

// A barrier for what is in LDS: loads from memory stay under way.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// 16 lanes give the addresses of four rows of 16 elements, four elements each; a lane gets a column.
__device__ __forceinline__ u32x2 columns_of(const uint8_t *at) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4 *)(const_cast<uint8_t *>(at))));
}

// Loads stay where they stand: the compiler would move those of a next turn down to it.
__device__ __forceinline__ void pin_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// What the first kernel leaves for a chunk and head: operands as the second loads them, 64 lanes
// of 16 bytes each (256 dwords).
namespace left {
constexpr int t = 0;              // [step][tile] of T, float32
constexpr int p = 6 * 2 * 256;    // [step][tile] of P
constexpr int v = 2 * p;          // float32: beta, beta e^c, scale e^c, e^(c_last - c) of every row, e^c_last 64 times
constexpr int dwords = v + 5 * kC;
// Row tile i against rows 32 s .. (those up to its own are there).
constexpr int step(int i, int s) { return i < 2 ? i : 2 * i - 2 + s; }
}  // namespace left

// Rows as operands of products over their dims, zeros for one that is not there.
template <typename E, int D> struct RowOperand {  // 16-bit: products are exact
    u32x4 x[D / 32];
    __device__ __forceinline__ void load(const typename E::T *row, int g4, bool there) {
#pragma unroll
        for (int s = 0; s < D / 32; s++)
            x[s] = there ? *reinterpret_cast<const u32x4 *>(row + 32 * s + 8 * g4) : u32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ f32x4 times(const RowOperand &o) const {
        f32x4 c = kZero;
#pragma unroll
        for (int s = 0; s < D / 32; s++) {
            if constexpr (std::is_same<E, RowF16>::value)
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x[s]),
                                                           __builtin_bit_cast(f16x8, o.x[s]), c, 0, 0, 0);
            else
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[s]),
                                                            __builtin_bit_cast(bf16x8, o.x[s]), c, 0, 0, 0);
        }
        return c;
    }
};
template <int D> struct RowOperand<RowF32, D> {
    f32x4 x[D / 16];
    __device__ __forceinline__ void load(const float *row, int g4, bool there) {
#pragma unroll
        for (int s = 0; s < D / 16; s++) x[s] = there ? *reinterpret_cast<const f32x4 *>(row + 16 * s + 4 * g4) : kZero;
    }
    __device__ __forceinline__ f32x4 times(const RowOperand &o) const {
        f32x4 c = kZero;
#pragma unroll
        for (int s = 0; s < D / 16; s++) c = mma(x[s], o.x[s], c);
        return c;
    }
};

// Sums of the lanes up to and with each.
template <int CTRL, int ROWS> __device__ __forceinline__ double add_shifted(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
    return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lanes_scan(double x) {
    x = add_shifted<0x111, 0xf>(x);  // by 1, 2, 4 and 8 lanes of a row of 16
    x = add_shifted<0x112, 0xf>(x);
    x = add_shifted<0x114, 0xf>(x);
    x = add_shifted<0x118, 0xf>(x);
    x = add_shifted<0x142, 0xa>(x);  // the last lane of row 0 to row 1 and of row 2 to row 3
    return add_shifted<0x143, 0xc>(x);  // lane 31 to rows 2 and 3
}

// A request of one or two rows, row after row by the first kernel: S = e^g S;  d = beta (v - S^T k);  S += k d^T;
// o = S^T q. A workgroup has a head's state, a thread four columns of every (2048 / D)th row. 200 requests of 16
// heads of 128 in BF16 of one, two and four rows each 236, 237 and 238 us in chunks, 88, 96 and 117 (then by four
// rows) this way; with four, a batch of 96 requests of unequal lengths, 6000 rows of 16 heads of 64 in F16, took 102 us
// for 97.
constexpr int kFew = 2;
template <typename E, int D>
__device__ __forceinline__ void few_rows(const GdnRows &b, const RaggedArgs &a, RowRange r, int j, int h, float *lds) {
    typedef typename E::T T;
    constexpr int C4 = D / 4, RG = 512 / C4, NR = D / RG;
    float *const qkv = lds;  // q, k and v of the row
    float4 *const part = reinterpret_cast<float4 *>(lds + 3 * D);  // [2][8][C4]
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, c4 = t % C4, rg = t / C4, group = h % a.groups;
    const int64_t size = (int64_t)a.heads * D * D, mine = (int64_t)h * D * D + 4 * c4;
    const int2 slot = b.slots[j];
    float4 s[NR];
#pragma unroll
    for (int m = 0; m < NR; m++)
        s[m] = (uint32_t)slot.x < (uint32_t)a.states
                   ? *reinterpret_cast<const float4 *>(b.state + slot.x * size + mine + (int64_t)(rg + RG * m) * D)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    // sum over the row groups of every column, in every thread
    auto total = [&](float4 x, int which) {
#pragma unroll
        for (int off = C4; off < 64; off <<= 1) {
            x.x += __shfl_xor(x.x, off);
            x.y += __shfl_xor(x.y, off);
            x.z += __shfl_xor(x.z, off);
            x.w += __shfl_xor(x.w, off);
        }
        if (lane < C4) part[(which * 8 + wave) * C4 + c4] = x;
        lds_barrier();
        float4 sum = part[which * 8 * C4 + c4];
#pragma unroll
        for (int w = 1; w < 8; w++) {
            const float4 y = part[(which * 8 + w) * C4 + c4];
            sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
        }
        return sum;
    };
    for (int row = r.begin; row < r.end; row++) {
        const T *const x = static_cast<const T *>(b.qkv) + (int64_t)row * a.stride;
        if (t < 3 * D) {
            const int part_of = t / D;
            const float y = (float)x[(part_of == 0 ? group : part_of == 1 ? a.groups + group : 2 * a.groups + h) * D + t % D];
            qkv[t] = part_of == 0 ? y * a.scale : y;
        }
        const float decay = expf(log_decay_of(b, a, (int64_t)row * a.heads + h, h));
        const float beta = beta_of(b, a, (int64_t)row * a.heads + h);
        lds_barrier();
        float4 seen = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int m = 0; m < NR; m++) {
            const float k = qkv[D + rg + RG * m];
            s[m].x *= decay; s[m].y *= decay; s[m].z *= decay; s[m].w *= decay;
            seen.x = fmaf(s[m].x, k, seen.x);
            seen.y = fmaf(s[m].y, k, seen.y);
            seen.z = fmaf(s[m].z, k, seen.z);
            seen.w = fmaf(s[m].w, k, seen.w);
        }
        seen = total(seen, 0);
        const float4 v = *reinterpret_cast<const float4 *>(qkv + 2 * D + 4 * c4);
        const float4 d = make_float4((v.x - seen.x) * beta, (v.y - seen.y) * beta, (v.z - seen.z) * beta, (v.w - seen.w) * beta);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int m = 0; m < NR; m++) {
            const float q = qkv[rg + RG * m], k = qkv[D + rg + RG * m];
            s[m].x = fmaf(k, d.x, s[m].x);
            s[m].y = fmaf(k, d.y, s[m].y);
            s[m].z = fmaf(k, d.z, s[m].z);
            s[m].w = fmaf(k, d.w, s[m].w);
            o.x = fmaf(s[m].x, q, o.x);
            o.y = fmaf(s[m].y, q, o.y);
            o.z = fmaf(s[m].z, q, o.z);
            o.w = fmaf(s[m].w, q, o.w);
        }
        o = total(o, 1);
        if (t < C4) {
            T *const to = static_cast<T *>(b.out) + ((int64_t)row * a.heads + h) * D + 4 * t;
            to[0] = (T)o.x;
            to[1] = (T)o.y;
            to[2] = (T)o.z;
            to[3] = (T)o.w;
        }
    }
    if ((uint32_t)slot.y < (uint32_t)a.states) {
#pragma unroll
        for (int m = 0; m < NR; m++)
            *reinterpret_cast<float4 *>(b.state + slot.y * size + mine + (int64_t)(rg + RG * m) * D) = s[m];
    }
}

// Eight waves: four for k_i . k_j, four for q_i . k_j, then four for the T of every head. HH heads of a group share
// the products. Small dependent phases: waves wait in 63 % of their cycles, vector instructions issue in 39 % (BF16;
// in F32 57 and 21 %, the matrix units busy in 26 %). 81 us for 8191 rows of 16 heads of 128 in F32 (0.12 GB moved), 62
// for 8192 rows of 16 prompts and 32 heads in BF16 (0.15 GB).
// (Six waves a SIMD for 16-bit rows: the registers of few_rows would leave five, 62 -> 70 us.)
template <typename E, int D, int HH>
__global__ __launch_bounds__(512, (kParts<E> == 3 ? 1 : 6)) void chunk_prepare_kernel(GdnRows b, RaggedArgs a,
                                                                                     uint32_t *__restrict__ left_all) {
    typedef typename E::T T;
    __shared__ double sum[HH][kC];  // of the log decays, base 2
    __shared__ __align__(16) float beta[HH][kC];
    __shared__ __align__(16) float at_all[HH][kC][kRowPitch];  // A^T, its diagonal blocks later those of T^T
    __shared__ int lost[HH][kC];  // rows of A with a value that is not finite
    const int number = blockIdx.x, group = blockIdx.y % a.groups;
    auto head = [&](int u) { return group + a.groups * (HH * (int)(blockIdx.y / a.groups) + u); };
    // the request whose chunk this is
    const int after = wave_first(a.requests, [&](int j) {
        return first_chunk<kC>(row_range(b.offsets, a.rows, j).begin, j) > number;
    });
    const int j = __builtin_amdgcn_readfirstlane(after) - 1;
    if (j < 0) return;
    const RowRange r = row_range(b.offsets, a.rows, j);
    const int row0 = r.begin + (number - first_chunk<kC>(r.begin, j)) * kC, n = min(kC, r.end - row0);
    if (n <= 0) return;
    if (r.end - r.begin <= kFew) {  // (the second kernel leaves them out)
        for (int u = 0; u < HH; u++) few_rows<E, D>(b, a, r, j, head(u), &at_all[0][0][0]);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
    // the waves' parts differ in length: turned from chunk to chunk, so that no SIMD has the longest each time
    const int role = (__builtin_amdgcn_readfirstlane(tid >> 6) + number + blockIdx.y) & 7, wave = role & 3;
    const bool keys = role < 4;
    const T *const rows = static_cast<const T *>(b.qkv) + (int64_t)row0 * a.stride;
    const T *const k = rows + (a.groups + group) * D, *const mine = keys ? k : rows + group * D;
    auto left_here = [&](int u) { return left_all + ((int64_t)number * a.heads + head(u)) * left::dwords; };

    if (role >= 8 - HH) {  // a row a lane
        const int u = 7 - role, h = head(u);
        float *const factors = reinterpret_cast<float *>(left_here(u) + left::v);
        const bool there = lane < n;
        const int64_t from = (int64_t)(row0 + (there ? lane : 0)) * a.heads + h;
        const float g = there ? log_decay_of(b, a, from, h) : 0.0f, step = there ? beta_of(b, a, from) : 0.0f;
        const double c = lanes_scan(1.4426950408889634 * (g < kLeast ? kLeast : g));
        const uint64_t bits = __builtin_bit_cast(uint64_t, c);
        const double last = __builtin_bit_cast(
            double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(bits >> 32), 63) << 32 |
                        (uint32_t)__builtin_amdgcn_readlane((int)bits, 63));
        sum[u][lane] = c;
        beta[u][lane] = step;
        lost[u][lane] = 0;
        const float grown = __builtin_amdgcn_exp2f((float)c);
        factors[lane] = step;
        factors[kC + lane] = step * grown;
        factors[2 * kC + lane] = grown * a.scale;
        factors[3 * kC + lane] = __builtin_amdgcn_exp2f((float)(last - c));
        factors[4 * kC + lane] = __builtin_amdgcn_exp2f((float)last);
    }
    // ---- products of rows by tiles of 16 x 16 on and below the diagonal, i the columns of a result:
    // wave 0 has (0,0) (1,0) (1,1), 1 (2,0..2), 2 (3,0) (3,1), 3 (3,2) (3,3)
    const int tiles = wave < 2 ? 3 : 2;
    auto tile_of = [&](int m, int *i, int *jt) {
        *i = wave == 0 ? (m == 0 ? 0 : 1) : wave == 1 ? 2 : 3;
        *jt = wave == 0 ? (m == 2 ? 1 : 0) : wave == 3 ? m + 2 : m;
    };
    typedef RowOperand<E, D> Rows;
    auto row_operand = [&](const T *x, int tile, Rows &o) {
        o.load(x + (int64_t)(16 * tile + r16) * a.stride, g4, 16 * tile + r16 < n);
    };
    f32x4 dot[3];
    {  // (all rows asked for before the first product take 148 registers for 84, and a fifth longer)
        Rows xi, kj;
#pragma unroll
        for (int m = 0; m < 3; m++) {
            if (m >= tiles) break;
            int i, jt;
            tile_of(m, &i, &jt);
            if (m == 0 || (wave == 0 && m == 1)) row_operand(mine, i, xi);
            row_operand(k, jt, kj);
            dot[m] = kj.times(xi);
        }
    }
    // four terms of a row tile's sum over rows: half a step of 32
    auto put = [&](uint32_t *area, int i, int jt, f32x4 x) {
        uint32_t *const to = area + (left::step(i, jt >> 1) * 2 * 64 + lane) * 4;
        *reinterpret_cast<f32x4 *>(to + 256 * (jt & 1)) = x;
        if (i == jt && !(i & 1)) *reinterpret_cast<f32x4 *>(to + 256) = kZero;  // above the diagonal
    };
    lds_barrier();
#pragma unroll
    for (int m = 0; m < 3; m++) {
        if (m >= tiles) break;
        int it, jt;
        tile_of(m, &it, &jt);
        const int i = 16 * it + r16, j0 = 16 * jt + 4 * g4;
#pragma unroll
        for (int u = 0; u < HH; u++) {
            const double sum_i = sum[u][i];
            const float factor = keys ? beta[u][i] : a.scale;
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool low = keys ? j0 + e < i : j0 + e <= i;
                const float fall = low ? __builtin_amdgcn_exp2f((float)(sum_i - sum[u][j0 + e])) : 0.0f;
                x[e] = low ? dot[m][e] * fall * factor : 0.0f;
            }
            if (keys) {
                // What is not finite in A would make NaN of rows of T before its own, where it meets their zeros: it is
                // taken as zero, and its row's T_ii becomes NaN below.
                const f32x4 all[1] = {x};
                if (__builtin_expect(any_not_finite(all), false)) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (finite(x[e])) continue;
                        x[e] = 0.0f;
                        lost[u][i] = 1;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) at_all[u][j0 + e][i] = x[e];
            } else {
                put(left_here(u) + left::p, it, jt, x);
            }
        }
    }
    lds_barrier();
    // ---- T: a wave inverts a diagonal block, from T (I + A) = I, a row a lane
    const int diag = 16 * wave, which = HH == 2 ? role >> 2 : 0;
    const bool inverts = HH == 2 || keys;
    auto &at = at_all[which];
    if (inverts) {
        float t[16];
#pragma unroll
        for (int c = 15; c >= 0; c--) {
            float x = c == r16 ? 1.0f : 0.0f;
#pragma unroll
            for (int m4 = c / 4; m4 < 4; m4++) {
                const f32x4 y = *reinterpret_cast<const f32x4 *>(&at[diag + c][diag + 4 * m4]);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * m4 + e > c) x = fmaf(-y[e], t[4 * m4 + e], x);
            }
            t[c] = x;
        }
        if (g4 == 0) {
#pragma unroll
            for (int c = 0; c < 16; c++) at[diag + c][diag + r16] = t[c];
        }
    }
    lds_barrier();
    if (!inverts) return;
    // then its row of blocks: T_ij^T = -T_jj^T sum_m A_mj^T T_im^T
    auto block = [&](int jt, int m) { return *reinterpret_cast<const f32x4 *>(&at[16 * jt + r16][16 * m + 4 * g4]); };
    f32x4 t[4];
#pragma unroll
    for (int jt = 3; jt >= 0; jt--) {
        if (jt > wave) {
            t[jt] = kZero;
            continue;
        }
        if (jt == wave) {
#pragma unroll
            for (int e = 0; e < 4; e++) t[jt][e] = at[diag + 4 * g4 + e][diag + r16];
            if (lost[which][diag + r16]) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * g4 + e == r16) t[jt][e] = __builtin_nanf("");
            }
        } else {
            f32x4 x = kZero;
#pragma unroll
            for (int m = jt + 1; m < 4; m++)
                if (m <= wave) x = mma(block(jt, m), t[m], x);
            t[jt] = mma(block(jt, jt), -x, kZero);
        }
        put(left_here(which) + left::t, wave, jt, t[jt]);
    }
}

// The longest requests go first, so that none of them is left alone at the end: request number `rank` by its
// rows. (More than 64 are taken as they come.)
__device__ __forceinline__ int by_length(const int32_t *offsets, const RaggedArgs &a, int rank) {
    if (a.requests == 1 || a.requests > 64) return rank;
    const int lane = threadIdx.x & 63;
    const RowRange r = row_range(offsets, a.rows, min(lane, a.requests - 1));
    const int mine = lane < a.requests ? r.end - r.begin : -1;
    int before = 0;
    for (int i = 0; i < a.requests; i++) {
        const int other = __builtin_amdgcn_readlane(mine, i);
        before += other > mine || (other == mine && i < lane);
    }
    return __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(before == rank)) - 1;
}

template <typename E, int D, int CT> struct ScanLds {
    static constexpr int KS = D / 32, NP = kParts<E>;
    static constexpr uint32_t state = 0;                             // S, [32 dims of k][tile][part]
    static constexpr uint32_t r = state + KS * CT * 3 * 1024;        // beta V - beta e^c K S, [32 rows][tile][part]
    static constexpr uint32_t v = r + 2 * CT * 3 * 1024;             // V'
    static constexpr uint32_t tail = v + 2 * CT * 3 * 1024;          // e^(c_last - c) V'
    static constexpr uint32_t keys = tail + 2 * CT * 3 * 1024;       // [chunk & 1][part][row]
    // Rows of K, a plane a part, 16 bytes apart where LDS holds that. Without them, piece x of 8 bytes of a row is
    // at x ^ turn(row), so that 16 rows of a piece and four rows of four lie in different banks: float32 keys of 128
    // dims then leave room for two tiles (16 prompts of 8000 rows in all, 32 heads, 526 -> 410 us); with one tile the turn
    // takes longer than the space (1 prompt of 8191 rows, the second kernel, 352 -> 362).
    static constexpr bool turned = keys + 2 * NP * kC * (2 * D + 16) > 160 * 1024;
    static constexpr uint32_t pitch = 2 * D + (turned ? 0 : 16), key_part = kC * pitch, key_buffer = NP * key_part;
    static constexpr uint32_t lost = keys + 2 * key_buffer;  // the first row of every column that is not finite
    static constexpr uint32_t total = lost + 64 * CT;
    static __device__ __forceinline__ int at(int row, int piece) {
        return row * pitch + 8 * (turned ? piece ^ ((row & 3) << 2 | (row >> 2 & 3)) : piece);
    }
};

// A workgroup has CT tiles of 16 columns of one head's state. Four waves walk the state, wave w with the rows
// D / 4 w .. of it and the chunk's rows 16 w .. + 15; four make the outputs of 16 rows each, and those, or four
// more where a key has several parts (float32 keys split by the waves of the outputs: a fifth longer), bring the keys to
// LDS, a chunk ahead. Three barriers a chunk:
//   S and K there | K S -> R; Q S | T R -> V' | S; P V'
// What is not finite in R or V' would make NaN of rows before its own, where it meets the zeros of T and P. A wave whose
// V' has such a value works it out again with zeros for those of R, and leaves zeros for its own; the column's outputs
// from that row on and its state are replaced by NaN behind the loop. us of this kernel without any of it and so: 8191
// rows of 16 heads of 128 in F32 340, 342; 16 prompts of 8192 rows, 32 heads in BF16 217, 210; 96 of 6000 rows, 16 heads
// of 64 in F16 65, 66. (With R looked at as well, before it is stored, and the outputs replaced in their turn: 366, 217, 68.)
// What a chunk needs from memory is asked for one chunk ahead; two ahead, or W = T (beta e^c K) from the
// first kernel for one phase less, took more registers than there are and were slower.
template <typename E> constexpr int kScanWaves = kParts<E> == 3 ? 12 : 8;
template <typename E, int D, int CT>
__global__ __launch_bounds__(64 * kScanWaves<E>) void chunk_scan_kernel(GdnRows b, RaggedArgs a, const uint32_t *left_all) {
    typedef typename E::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int KT = D / 16, KS = D / 32, ST = D / 64, NP = kParts<E>;
    constexpr bool kApart = kScanWaves<E> == 12;
    using L = ScanLds<E, D, CT>;
    extern __shared__ __align__(16) uint8_t lds[];
    const int h = blockIdx.x, col0 = blockIdx.y * 16 * CT, j = by_length(b.offsets, a, blockIdx.z);
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
    const int role = __builtin_amdgcn_readfirstlane(tid >> 6), wave = role & 3;
    const RowRange r = row_range(b.offsets, a.rows, j);
    if (r.end > r.begin && r.end - r.begin <= kFew) return;  // done by the first kernel
    const int group = h % a.groups;
    const int number0 = first_chunk<kC>(r.begin, j), last = (r.end - r.begin + kC - 1) / kC - 1;
    int *const lost = reinterpret_cast<int *>(lds + L::lost);  // (rows are counted from the request's first)
    if (tid < 16 * CT) lost[tid] = 0x7fffffff;
    auto any_lost = [&]() -> bool {  // behind the last chunk
        if (last < 0) return false;
        int from = 0x7fffffff;
        if (lane < 16 * CT) from = lost[lane];
        return __builtin_expect(__builtin_amdgcn_ballot_w64(from < r.end - r.begin) != 0, false);
    };
    const T *const qkv = static_cast<const T *>(b.qkv);
    auto chunk_at = [&](int i) { return left_all + ((int64_t)(number0 + min(i, last)) * a.heads + h) * left::dwords; };
    auto factors_at = [&](int i, int which) {  // of the lane's four rows
        return *reinterpret_cast<const f32x4 *>(chunk_at(i) + left::v + which * kC + 16 * wave + 4 * g4);
    };
    // an operand's parts in LDS: of a tile of 16 columns, 32 terms in a step
    auto operand = [&](uint32_t area, int step, int c, u32x4 (&x)[3]) {
#pragma unroll
        for (int m = 0; m < 3; m++)
            x[m] = *reinterpret_cast<const u32x4 *>(lds + area + ((step * CT + c) * 3 + m) * 1024 + lane * 16);
    };
    auto store_half = [&](uint32_t area, int tile, int c, f32x4 x) {
        u32x2 part[3];
        split(x, part);
#pragma unroll
        for (int m = 0; m < 3; m++)
            *reinterpret_cast<u32x2 *>(lds + area + (((tile >> 1) * CT + c) * 3 + m) * 1024 + lane * 16 + 8 * (tile & 1)) = part[m];
    };
    // the lane's four terms of tile t of its key, of 16
    auto key_at = [&](int t) { return L::at(r16, 4 * t + g4); };
    // (No branches among the loads and stores of a turn: a wait counts the least that may have been issued since, and
    // would be one for what was asked for last.)
    auto load_step = [&](int i, int what, int s, f32x4 (&x)[2][2]) {
        const int step = left::step(wave, min(s, wave >> 1));
#pragma unroll
        for (int m = 0; m < 2; m++)
            x[s][m] = *reinterpret_cast<const f32x4 *>(chunk_at(i) + what + ((step * 2 + m) * 64 + lane) * 4);
    };

    if (role >= 4) {  // ---- keys and outputs
        auto load_rows = [&](int i, int head, T4 (&x)[KT]) {
            const int row = min(r.begin + i * kC + 16 * wave + r16, r.end - 1);
            const T *const from = qkv + (int64_t)row * a.stride + head * D + 4 * g4;
#pragma unroll
            for (int t = 0; t < KT; t++) x[t] = *reinterpret_cast<const T4 *>(from + 16 * t);
        };
        auto parts = [&](const T4 &x, const T4 &y, u32x4 (&o)[NP]) {
            if constexpr (NP == 1) {
                const T4 both[2] = {x, y};
                __builtin_memcpy(&o[0], both, 16);
            } else {
                split(f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]},
                      f32x4{(float)y[0], (float)y[1], (float)y[2], (float)y[3]}, o);
            }
        };
        T4 k[KT];
        auto keys_to_lds = [&](int i) {
            uint8_t *const to = lds + L::keys + (i & 1) * L::key_buffer + 16 * wave * L::pitch;
            const bool there = r.begin + i * kC + 16 * wave + r16 < r.end;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                u32x4 x[NP];
                parts(k[2 * s], k[2 * s + 1], x);
#pragma unroll
                for (int m = 0; m < NP; m++) {  // (rows behind the end are zeros: they meet zeros of V')
                    *reinterpret_cast<u32x2 *>(to + m * L::key_part + key_at(2 * s)) =
                        there ? u32x2{x[m][0], x[m][1]} : u32x2{0, 0};
                    *reinterpret_cast<u32x2 *>(to + m * L::key_part + key_at(2 * s + 1)) =
                        there ? u32x2{x[m][2], x[m][3]} : u32x2{0, 0};
                }
            }
        };
        if (last >= 0 && (!kApart || role >= 8)) {
            load_rows(0, a.groups + group, k);
            keys_to_lds(0);
            if constexpr (kApart) load_rows(1, a.groups + group, k);
        }
        if (kApart && role >= 8) {
            for (int i = 0; i <= last; i++) {
                lds_barrier();
                keys_to_lds(i + 1);
                load_rows(i + 2, a.groups + group, k);
                pin_loads();
                lds_barrier();
                lds_barrier();
            }
            return;
        }
        T4 q[KT];
        f32x4 p[2][2];
        f32x4 front;
        if (last >= 0) {
            load_rows(0, group, q);
            front = factors_at(0, 2);
            if constexpr (!kApart) load_rows(1, a.groups + group, k);
            load_step(0, left::p, 0, p);
            load_step(0, left::p, 1, p);
        }
        for (int i = 0; i <= last; i++) {
            const int row0 = r.begin + i * kC, n = min(kC, r.end - row0);
            lds_barrier();
            Sum o[CT];
#pragma unroll
            for (int c = 0; c < CT; c++) o[c] = Sum{kZero, kZero};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                u32x4 x[NP];
                parts(q[2 * s], q[2 * s + 1], x);
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    u32x4 y[3];
                    operand(L::state, s, c, y);
                    mma32(x, y, o[c]);
                }
            }
            load_rows(i + 1, group, q);
            pin_loads();
#pragma unroll
            for (int c = 0; c < CT; c++) {
                o[c].big *= front;
                o[c].small *= front;
            }
            front = factors_at(i + 1, 2);
            pin_loads();
            lds_barrier();
            if constexpr (!kApart) {
                keys_to_lds(i + 1);
                load_rows(i + 2, a.groups + group, k);
                pin_loads();
            }
            lds_barrier();
#pragma unroll
            for (int s = 0; s < 2; s++) {
                if (s > wave / 2) break;
                u32x4 x[3];
                split(p[s][0], p[s][1], x);
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    u32x4 y[3];
                    operand(L::v, s, c, y);
                    mma32(x, y, o[c]);
                }
            }
            load_step(i + 1, left::p, 0, p);
            load_step(i + 1, left::p, 1, p);
            pin_loads();
            // rows behind the end lie behind the buffer, and are not written
            const uint32_t pitch = a.heads * D * sizeof(T);
            const uint64_t base = reinterpret_cast<uint64_t>(b.out) + (uint64_t)row0 * pitch;
            void *const first = reinterpret_cast<void *>((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32)) << 32 |
                                                         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base));
            const auto rows = __builtin_amdgcn_make_buffer_rsrc(first, (short)0, __builtin_amdgcn_readfirstlane(n * pitch),
                                                                0x00020000);
            const uint32_t at = (16 * wave + 4 * g4) * pitch + (h * D + col0 + r16) * sizeof(T);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    const T y = (T)(o[c].big[e] + o[c].small[e]);
                    const uint32_t to = at + e * pitch + 16 * c * sizeof(T);
                    if constexpr (sizeof(T) == 4)
                        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, y), rows, to, 0, 0);
                    else
                        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, y), rows, to, 0, 0);
                }
        }
        if (!any_lost()) return;
#pragma unroll 1
        for (int c = 0; c < CT; c++) {  // (each wave the rows that it has stored, so that its stores are in order)
            T *const column = static_cast<T *>(b.out) + ((int64_t)r.begin * a.heads + h) * D + col0 + 16 * c + r16;
            const int from = lost[16 * c + r16];
            if (from >= r.end - r.begin) continue;
            for (int row = from / kC * kC + 16 * wave; row < r.end - r.begin; row += kC)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int mine = row + 4 * g4 + e;
                    if (mine >= from && mine < r.end - r.begin) column[(int64_t)mine * a.heads * D] = (T)__builtin_nanf("");
                }
        }
        return;
    }

    // ---- the state
    const int2 slot = b.slots[j];
    const int64_t size = (int64_t)a.heads * D * D, at0 = (int64_t)h * D * D + col0 + r16;
    f32x4 s[ST][CT];
#pragma unroll
    for (int t = 0; t < ST; t++)
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                s[t][c][e] = (uint32_t)slot.x < (uint32_t)a.states
                                 ? b.state[slot.x * size + at0 + (int64_t)(16 * (wave * ST + t) + 4 * g4 + e) * D + 16 * c]
                                 : 0.0f;
    f32x4 t[2][2];
    T v[CT][4];
    f32x4 beta, grown, tail;
    float fall;
    auto load_values = [&](int i) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int row = min(r.begin + i * kC + 16 * wave + 4 * g4 + e, r.end - 1);
#pragma unroll
            for (int c = 0; c < CT; c++)
                v[c][e] = qkv[(int64_t)row * a.stride + (2 * a.groups + h) * D + col0 + 16 * c + r16];
        }
        beta = factors_at(i, 0);
        grown = factors_at(i, 1);
    };
    auto load_tail = [&](int i) {
        tail = factors_at(i, 3);
        // (a scalar load would make every wait for LDS one for memory)
        fall = *reinterpret_cast<const float *>(chunk_at(i) + left::v + 4 * kC + lane);
    };
    if (last >= 0) {
        load_values(0);
        load_step(0, left::t, 0, t);
        load_step(0, left::t, 1, t);
        load_tail(0);
    }
    // V' again without what is not finite, whose columns are lost from there on
    auto again = [&](int i) {
        f32x4 tt[2][2];
        load_step(i, left::t, 0, tt);
        load_step(i, left::t, 1, tt);
#pragma unroll 1
        for (int c = 0; c < CT; c++) {
            Sum w = {kZero, kZero};
#pragma unroll
            for (int d = 0; d < 2; d++) {
                if (d > wave / 2) break;
                u32x4 z[3], x[3];
                split(tt[d][0], tt[d][1], z);
                operand(L::r, d, c, x);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t keep = finite_halves(x[0][k]);
#pragma unroll
                    for (int m = 0; m < 3; m++) x[m][k] &= keep;
                }
                mma32(z, x, w);
            }
            f32x4 y = w.all();
            const u32x2 own = *reinterpret_cast<const u32x2 *>(lds + L::r + ((wave >> 1) * CT + c) * 3 * 1024 + lane * 16 +
                                                               8 * (wave & 1));  // R as `store_half` left it
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if ((finite_halves(own[e >> 1]) >> 16 * (e & 1) & 1) && finite(y[e])) continue;
                y[e] = 0.0f;
                atomicMin(lost + 16 * c + r16, i * kC + 16 * wave + 4 * g4 + e);
            }
            store_half(L::tail, wave, c, y * tail);
            store_half(L::v, wave, c, y);
        }
    };
    for (int i = 0; i <= last; i++) {
        const uint32_t keys = L::keys + (i & 1) * L::key_buffer;
#pragma unroll
        for (int c = 0; c < CT; c++) {
            if constexpr (ST == 2) {
                u32x4 part[3];
                split(s[0][c], s[1][c], part);
#pragma unroll
                for (int m = 0; m < 3; m++)
                    *reinterpret_cast<u32x4 *>(lds + L::state + ((wave * CT + c) * 3 + m) * 1024 + lane * 16) = part[m];
            } else {
                store_half(L::state, wave, c, s[0][c]);
            }
        }
        lds_barrier();
        Sum x[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) x[c] = Sum{kZero, kZero};
#pragma unroll
        for (int d = 0; d < KS; d++) {
            const uint8_t *const from = lds + keys + 16 * wave * L::pitch;
            u32x4 k[NP];
#pragma unroll
            for (int m = 0; m < NP; m++) {
                const u32x2 lo = *reinterpret_cast<const u32x2 *>(from + m * L::key_part + key_at(2 * d));
                const u32x2 hi = *reinterpret_cast<const u32x2 *>(from + m * L::key_part + key_at(2 * d + 1));
                k[m] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
#pragma unroll
            for (int c = 0; c < CT; c++) {
                u32x4 y[3];
                operand(L::state, d, c, y);
                mma32(k, y, x[c]);
            }
        }
        const int n = r.end - (r.begin + i * kC) - 16 * wave - 4 * g4;  // rows from the lane's first on
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const f32x4 ks = x[c].all();
            f32x4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = e < n ? beta[e] * (float)v[c][e] - grown[e] * ks[e] : 0.0f;
            store_half(L::r, wave, c, y);
        }
        load_values(i + 1);
        pin_loads();
        lds_barrier();
        Sum w[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) w[c] = Sum{kZero, kZero};
#pragma unroll
        for (int d = 0; d < 2; d++) {
            if (d > wave / 2) break;
            u32x4 z[3];
            split(t[d][0], t[d][1], z);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                u32x4 y[3];
                operand(L::r, d, c, y);
                mma32(z, y, w[c]);
            }
        }
        load_step(i + 1, left::t, 0, t);
        load_step(i + 1, left::t, 1, t);
        pin_loads();
        f32x4 y[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) y[c] = w[c].all();
#pragma unroll
        for (int c = 0; c < CT; c++) {
            store_half(L::tail, wave, c, y[c] * tail);
            store_half(L::v, wave, c, y[c]);
        }
        if (__builtin_expect(any_not_finite(y), false)) again(i);
        lds_barrier();
        Sum next[ST][CT];
#pragma unroll
        for (int u = 0; u < ST; u++)
#pragma unroll
            for (int c = 0; c < CT; c++) next[u][c] = Sum{s[u][c] * fall, kZero};
        load_tail(i + 1);
        pin_loads();
#pragma unroll
        for (int d = 0; d < 2; d++) {
            // K^T: a lane's eight rows of one column, four rows of 16 columns turned over at a time
            u32x4 k[ST][NP];
#pragma unroll
            for (int u = 0; u < ST; u++)
#pragma unroll
                for (int m = 0; m < NP; m++) {
                    const uint32_t from = keys + m * L::key_part + 32 * d * L::pitch +
                                          L::at(4 * g4 + (r16 >> 2), 4 * (wave * ST + u) + (r16 & 3));
                    const u32x2 lo = columns_of(lds + from), hi = columns_of(lds + from + 16 * L::pitch);
                    k[u][m] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                }
#pragma unroll
            for (int c = 0; c < CT; c++) {
                u32x4 y[3];
                operand(L::tail, d, c, y);
#pragma unroll
                for (int u = 0; u < ST; u++) mma32(k[u], y, next[u][c]);
            }
        }
#pragma unroll
        for (int u = 0; u < ST; u++)
#pragma unroll
            for (int c = 0; c < CT; c++) s[u][c] = next[u][c].all();
    }
    if ((uint32_t)slot.y < (uint32_t)a.states) {
        if (any_lost()) {
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const bool mine = lost[16 * c + r16] < r.end - r.begin;
#pragma unroll
                for (int t = 0; t < ST; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[t][c][e] = mine ? __builtin_nanf("") : s[t][c][e];
            }
        }
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    b.state[slot.y * size + at0 + (int64_t)(16 * (wave * ST + t) + 4 * g4 + e) * D + 16 * c] = s[t][c][e];
    }
}

template <typename F> hipError_t by_kind(uint32_t dtype, int head_dim, F &&f) {
    auto by_dim = [&](auto e) {
        return head_dim == 128 ? f(e, std::integral_constant<int, 128>{}) : f(e, std::integral_constant<int, 64>{});
    };
    return dtype == YUUKA_DTYPE_F32 ? by_dim(RowF32{}) : dtype == YUUKA_DTYPE_F16 ? by_dim(RowF16{}) : by_dim(RowBF16{});
}

}  // namespace

uint64_t gdn_prompt_scratch_bytes(const RaggedArgs &a) {
    return (uint64_t)chunk_numbers<kC>(a.rows, a.requests) * a.heads * left::dwords * 4;
}

hipError_t launch_gdn_prompt(const GdnRows &b, uint32_t dtype, const RaggedArgs &a, void *scratch, hipStream_t s) {
    const uint32_t numbers = chunk_numbers<kC>(a.rows, a.requests);
    return by_kind(dtype, a.head_dim, [&](auto e, auto d) {
        using E = decltype(e);
        constexpr int D = d();
        uint32_t *const left_all = static_cast<uint32_t *>(scratch);
        // Two heads a workgroup where that leaves every CU one. us of the whole call with one and with two: 32 heads of 16
        // groups, 2000 rows in F32 126 and 112, 16 prompts of 8192 rows in all in BF16 267 and 245; 500 rows in BF16 33 and
        // 35, which stay at one.
        if (a.heads / a.groups % 2 == 0 && (int64_t)numbers * a.heads >= 2 * 256)
            chunk_prepare_kernel<E, D, 2><<<dim3(numbers, a.heads / 2), 512, 0, s>>>(b, a, left_all);
        else chunk_prepare_kernel<E, D, 1><<<dim3(numbers, a.heads), 512, 0, s>>>(b, a, left_all);
        hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
        auto go = [&](auto tiles) {
            constexpr int CT = tiles();
            constexpr uint32_t bytes = ScanLds<E, D, CT>::total;
            if constexpr (bytes <= 160 * 1024) {  // (more are not asked for)
                constexpr auto scan = chunk_scan_kernel<E, D, CT>;
                if constexpr (bytes > 64 * 1024) {  // (a device's own setting)
                    static std::once_flag once[64];
                    int device = 0;
                    (void)hipGetDevice(&device);
                    std::call_once(once[device & 63], [] {
                        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(scan),
                                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
                    });
                }
                scan<<<dim3(a.heads, D / 16 / CT, a.requests), 64 * kScanWaves<E>, bytes, s>>>(b, a, left_all);
                err = hipGetLastError();
            }
        };
        // The most columns that LDS holds and that leave every CU a workgroup: what is loaded for a chunk serves more of
        // them. us with 1, 2 and 4 tiles, BF16: 1 prompt of 2000 rows, 16 heads of 128 (128 workgroups at one tile) 88, 120,
        // 167; 4 of 1000 (512) 101, 82, 105; 4 of 1000, 32 heads (1024) 182, 138, 114; 16 of 8192 rows in all (4096)
        // 388, 305, 244. F32, 16 heads: 4 of 1000 rows 137, 110, 64 of 300 in all 282, 184.
        const int64_t columns = (int64_t)a.requests * a.heads * (D / 16);
        if (columns >= 4 * 256 && ScanLds<E, D, 4>::total <= 160 * 1024) go(std::integral_constant<int, 4>{});
        else if (columns >= 2 * 256 && ScanLds<E, D, 2>::total <= 160 * 1024) go(std::integral_constant<int, 2>{});
        else go(std::integral_constant<int, 1>{});
        return err;
    });
}

}  // namespace yk

// k_gdnchunk.hip — the gated delta rule over whole prompts (recurrent.go:56-105),
// 64 rows at a time.
//
// With c_i the sum of the log decays of a chunk's rows up to i, and S the state before it,
//   A_ij = beta_i (k_i . k_j) e^(c_i - c_j)  for i > j
//   (I + A) U = diag(beta) V,   (I + A) W = diag(beta e^c) K
//   V' = U - W S                                 the rows' corrections, d_i in the rule
//   out = e^c (Q S) + P V',     P_ij = (q_i . k_j) e^(c_i - c_j)  for i >= j
//   S <- e^(c_last) S + K^T diag(e^(c_last - c)) V'
// The first kernel makes U, W and P of every chunk and head, all chunks at once; the second
// walks the chunks of a request with S in registers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gdn_ragged_dev.h"
#include "internal.h"

namespace yk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kC = 64;           // rows of a chunk
constexpr int kRowPitch = kC + 4;  // floats of a row of A in LDS
constexpr float kLeast = -200.0f;  // e^-200 is zero in float32, and the sums of 64 stay exact to 1e-12 in float64

// Products on v_mfma_f32_16x16x4_f32. Lane l has row (A) or column (B) l % 16 and, of 16 terms of
// the sum, 4 (l / 16) + e in the e-th of four instructions; the result's lane has column l % 16 and
// rows 4 (l / 16) + e. A result is thus the next product's B operand, or the A operand of its
// transpose, in the registers that it is in.
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
constexpr f32x4 kZero = {0.f, 0.f, 0.f, 0.f};

// A barrier for what is in LDS: loads from memory stay under way.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// What the first kernel leaves for a chunk and head: operands as the second loads them, 64 lanes
// of 16 bytes each.
template <int D> struct Left {
    static constexpr int kTiles = D / 16;
    static constexpr int w = 0;                      // [row tile][tile of k's dims]: A of W S
    static constexpr int u = w + 4 * kTiles * 256;   // [row tile][tile of v's dims]: C layout
    static constexpr int p = u + 4 * kTiles * 256;   // [row tile i, tile j <= i]: A of P V'
    static constexpr int v = p + 10 * 256;           // scale e^c of every row, e^(c_last - c), e^c_last
    static constexpr int floats = v + 2 * kC + 64;
    static constexpr int keys = 4 * kTiles * 256;    // of a group: [row tile][tile of k's dims], A of K^T V'
};
constexpr int p_tile(int i, int j) { return i * (i + 1) / 2 + j; }

// Four consecutive elements of a row, zeros for a row that is not there.
template <typename E> __device__ __forceinline__ f32x4 four(const typename E::T *at, bool there) {
    typedef typename E::T T4 __attribute__((ext_vector_type(4)));
    T4 x = {0, 0, 0, 0};
    if (there) x = *reinterpret_cast<const T4 *>(at);
    return f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}

template <typename E, int D>
__global__ __launch_bounds__(256) void chunk_prepare_kernel(GdnRows b, RaggedArgs a, float *__restrict__ left,
                                                            float *__restrict__ keys) {
    typedef typename E::T T;
    constexpr int KT = D / 16;
    using L = Left<D>;
    __shared__ double sum[kC];
    __shared__ __align__(16) float beta[kC], grown[kC];  // e^c
    __shared__ __align__(16) float am[kC][kRowPitch], tm[kC][kRowPitch];  // A with its diagonal blocks' inverses; T diag(beta)
    const int number = blockIdx.x, h = blockIdx.y;
    // the request whose chunk this is
    const int after = wave_first(a.requests, [&](int j) {
        return first_chunk<kC>(row_range(b.offsets, a.rows, j).begin, j) > number;
    });
    const int j = __builtin_amdgcn_readfirstlane(after) - 1;
    if (j < 0) return;
    const RowRange r = row_range(b.offsets, a.rows, j);
    const int row0 = r.begin + (number - first_chunk<kC>(r.begin, j)) * kC, n = min(kC, r.end - row0);
    if (n <= 0) return;
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
    // the waves' parts differ in length: turned from chunk to chunk, so that no SIMD has the longest each time
    const int wave = (__builtin_amdgcn_readfirstlane(tid >> 6) + number + h) & 3;
    const T *const rows = static_cast<const T *>(b.qkv) + (int64_t)row0 * a.stride;
    const int group = h % a.groups;
    const T *const q = rows + group * D, *const k = rows + (a.groups + group) * D, *const v = rows + (2 * a.groups + h) * D;
    float *const mine = left + ((int64_t)number * a.heads + h) * L::floats;

    if (wave == 0) {  // a row a lane
        const bool there = lane < n;
        const int64_t at = (int64_t)(row0 + (there ? lane : 0)) * a.heads + h;
        const float g = there ? log_decay_of(b, a, at, h) : 0.0f;
        double c = g < kLeast ? kLeast : g;
        for (int off = 1; off < 64; off <<= 1) {
            const double x = __shfl_up(c, off);
            if (lane >= off) c += x;
        }
        const double last = __shfl(c, 63);
        sum[lane] = c;
        beta[lane] = there ? beta_of(b, a, at) : 0.0f;
        grown[lane] = expf((float)c);
        mine[L::v + lane] = expf((float)c) * a.scale;
        mine[L::v + kC + lane] = expf((float)(last - c));
        if (lane == 0) mine[L::v + 2 * kC] = expf((float)last);
    }
    // ---- k_i . k_j and q_i . k_j by tiles of 16 x 16 on and below the diagonal, i the columns of a result
    auto row_operand = [&](const T *x, int tile, f32x4 (&o)[KT]) {
        const int row = 16 * tile + r16;
#pragma unroll
        for (int s = 0; s < KT; s++) o[s] = four<E>(x + (int64_t)row * a.stride + 16 * s + 4 * g4, row < n);
    };
    const int it0 = wave == 0 ? 0 : wave == 1 ? 2 : 3, it1 = wave == 0 ? 1 : it0;
    f32x4 kk[3], qk[3];  // wave 0: (0,0) (1,0) (1,1); 1: (2,0..2); 2: (3,0) (3,1); 3: (3,2) (3,3)
    auto tile_of = [&](int m, int *i, int *jt) {
        *i = wave == 0 && m == 0 ? 0 : it1;
        *jt = wave == 0 ? (m == 2 ? 1 : 0) : wave == 3 ? m + 2 : m;
    };
    const int tiles = wave < 2 ? 3 : 2;
    {
        f32x4 ki[KT], qi[KT], kj[KT];
#pragma unroll
        for (int m = 0; m < 3; m++) {
            if (m >= tiles) break;
            int i, jt;
            tile_of(m, &i, &jt);
            if (m == 0 || (wave == 0 && m == 1)) {
                row_operand(k, i, ki);
                row_operand(q, i, qi);
            }
            row_operand(k, jt, kj);
            kk[m] = qk[m] = kZero;
#pragma unroll
            for (int s = 0; s < KT; s++) {
                kk[m] = mma(kj[s], ki[s], kk[m]);
                qk[m] = mma(kj[s], qi[s], qk[m]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 3; m++) {
        if (m >= tiles) break;
        int it, jt;
        tile_of(m, &it, &jt);
        const int i = 16 * it + r16, j0 = 16 * jt + 4 * g4;
        f32x4 x, p;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool low = j0 + e <= i;
            const float fall = low ? expf((float)(sum[i] - sum[j0 + e])) : 0.0f;
            x[e] = j0 + e < i ? kk[m][e] * fall * beta[i] : 0.0f;
            p[e] = low ? qk[m][e] * fall * a.scale : 0.0f;
        }
        *reinterpret_cast<f32x4 *>(&am[i][j0]) = x;
        *reinterpret_cast<f32x4 *>(mine + L::p + (p_tile(it, jt) * 64 + lane) * 4) = p;
    }
    __syncthreads();
    // ---- T = (I + A)^-1: a wave inverts a diagonal block by substitution, a column a lane
    const int diag = 16 * wave;
    {
        float t[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float x = i == r16 ? 1.0f : 0.0f;
#pragma unroll
            for (int m4 = 0; m4 < (i + 3) / 4; m4++) {
                const f32x4 y = *reinterpret_cast<const f32x4 *>(&am[diag + i][diag + 4 * m4]);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * m4 + e < i) x = fmaf(-y[e], t[4 * m4 + e], x);
            }
            t[i] = x;
        }
        if (g4 == 0) {
#pragma unroll
            for (int i = 0; i < 16; i++) am[diag + i][diag + r16] = t[i];
        }
    }
    __syncthreads();
    // then the column of blocks below it: T_ij = -T_ii sum_m A_im T_mj
    auto block_rows = [&](int i, int jt) { return *reinterpret_cast<const f32x4 *>(&am[16 * i + r16][16 * jt + 4 * g4]); };
    {
        f32x4 t[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i < wave) {
                t[i] = kZero;
            } else if (i == wave) {
#pragma unroll
                for (int e = 0; e < 4; e++) t[i][e] = am[diag + 4 * g4 + e][diag + r16];
            } else {
                f32x4 x = kZero;
#pragma unroll
                for (int m = 0; m < i; m++)
                    if (m >= wave) x = mma(block_rows(i, m), t[m], x);
                t[i] = mma(block_rows(i, i), -x, kZero);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) tm[16 * i + 4 * g4 + e][diag + r16] = t[i][e] * beta[diag + r16];
        }
    }
    __syncthreads();
    // ---- U = T diag(beta) V and W^T = K^T (T diag(beta e^c))^T, a tile of 16 columns at a time
    f32x4 tv[10], tk[10];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t <= i; t++) {
            tv[p_tile(i, t)] = *reinterpret_cast<const f32x4 *>(&tm[16 * i + r16][16 * t + 4 * g4]);
            tk[p_tile(i, t)] = tv[p_tile(i, t)] * *reinterpret_cast<const f32x4 *>(&grown[16 * t + 4 * g4]);
        }
    auto column_operand = [&](const T *x, int tile, f32x4 (&o)[4]) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = 16 * t + 4 * g4 + e;
                o[t][e] = row < n ? (float)x[(int64_t)row * a.stride + 16 * tile + r16] : 0.0f;
            }
    };
    float *const group_keys = keys + ((int64_t)number * a.groups + group) * L::keys;
#pragma unroll
    for (int c = wave; c < KT; c += 4) {
        f32x4 x[4];
        column_operand(k, c, x);
        if (h < a.groups) {
#pragma unroll
            for (int t = 0; t < 4; t++) *reinterpret_cast<f32x4 *>(group_keys + ((t * KT + c) * 64 + lane) * 4) = x[t];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f32x4 y = kZero;
#pragma unroll
            for (int t = 0; t <= i; t++) y = mma(x[t], tk[p_tile(i, t)], y);
            *reinterpret_cast<f32x4 *>(mine + L::w + ((i * KT + c) * 64 + lane) * 4) = y;
        }
        column_operand(v, c, x);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f32x4 y = kZero;
#pragma unroll
            for (int t = 0; t <= i; t++) y = mma(tv[p_tile(i, t)], x[t], y);
            *reinterpret_cast<f32x4 *>(mine + L::u + ((i * KT + c) * 64 + lane) * 4) = y;
        }
    }
}

// A workgroup has CT tiles of 16 columns of one head's state; wave w the state's rows D / 4 w .. and the
// chunk's rows 16 w .. + 15.
template <typename E, int D, int CT>
__global__ __launch_bounds__(256, 1) void chunk_scan_kernel(GdnRows b, RaggedArgs a, const float *__restrict__ left,
                                                         const float *__restrict__ keys) {
    typedef typename E::T T;
    constexpr int KT = D / 16, ST = D / 64;
    using L = Left<D>;
    __shared__ f32x4 ls[KT][CT][64], lv[4][CT][64], lt[4][CT][64];  // S, V' and e^(c_last - c) V' as B operands
    const int h = blockIdx.x, col0 = blockIdx.y * 16 * CT, j = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const RowRange r = row_range(b.offsets, a.rows, j);
    const int2 slot = b.slots[j];
    const int64_t size = (int64_t)a.heads * D * D, at0 = (int64_t)h * D * D + col0 + r16;
    const int group = h % a.groups;
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
    // A chunk's operands are loaded while the one before it is worked on, each as soon as its registers are free.
    typedef T T4 __attribute__((ext_vector_type(4)));
    f32x4 w[KT], u[CT], p[4], k[ST][4], front, tail;
    T4 q[KT];
    float fall;
    const int number0 = first_chunk<kC>(r.begin, j), last = (r.end - r.begin + kC - 1) / kC - 1;
    auto chunk_at = [&](int i) { return left + ((int64_t)(number0 + min(i, last)) * a.heads + h) * L::floats; };
    auto load_row = [&](int i, int t) {
        const int row = r.begin + i * kC + 16 * wave + r16;
        q[t] = T4{0, 0, 0, 0};
        if (row < r.end)
            q[t] = *reinterpret_cast<const T4 *>(static_cast<const T *>(b.qkv) + (int64_t)row * a.stride + group * D + 16 * t + 4 * g4);
        w[t] = *reinterpret_cast<const f32x4 *>(chunk_at(i) + L::w + ((wave * KT + t) * 64 + lane) * 4);
    };
    auto load_rest = [&](int i) {
        const float *const mine = chunk_at(i);
#pragma unroll
        for (int c = 0; c < CT; c++)
            u[c] = *reinterpret_cast<const f32x4 *>(mine + L::u + ((wave * KT + col0 / 16 + c) * 64 + lane) * 4);
        front = *reinterpret_cast<const f32x4 *>(mine + L::v + 16 * wave + 4 * g4);
        tail = *reinterpret_cast<const f32x4 *>(mine + L::v + kC + 16 * wave + 4 * g4);
        fall = mine[L::v + 2 * kC];
    };
    auto load_p = [&](int i, int t) {
        if (t <= wave) p[t] = *reinterpret_cast<const f32x4 *>(chunk_at(i) + L::p + (p_tile(wave, t) * 64 + lane) * 4);
    };
    auto load_k = [&](int i, int x, int t) {
        k[x][t] = *reinterpret_cast<const f32x4 *>(keys + ((int64_t)(number0 + min(i, last)) * a.groups + group) * L::keys +
                                                   ((t * KT + wave * ST + x) * 64 + lane) * 4);
    };
    if (last >= 0) {
#pragma unroll
        for (int t = 0; t < KT; t++) load_row(0, t);
        load_rest(0);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            load_p(0, t);
#pragma unroll
            for (int x = 0; x < ST; x++) load_k(0, x, t);
        }
    }
    for (int i = 0; i <= last; i++) {
        const int row0 = r.begin + i * kC, n = min(kC, r.end - row0);
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int c = 0; c < CT; c++) ls[wave * ST + t][c][lane] = s[t][c];
        lds_barrier();
        f32x4 ws[CT], o[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) ws[c] = o[c] = kZero;
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const f32x4 x = {(float)q[t][0], (float)q[t][1], (float)q[t][2], (float)q[t][3]};
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const f32x4 y = ls[t][c][lane];
                ws[c] = mma(w[t], y, ws[c]);
                o[c] = mma(x, y, o[c]);
            }
            load_row(i + 1, t);
        }
        const float before = fall;
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const f32x4 x = u[c] - ws[c];
            lv[wave][c][lane] = x;
            lt[wave][c][lane] = x * tail;
            o[c] *= front;
        }
        load_rest(i + 1);
        lds_barrier();
#pragma unroll
        for (int x = 0; x < ST; x++)
#pragma unroll
            for (int c = 0; c < CT; c++) s[x][c] *= before;
#pragma unroll
        for (int t = 0; t < 4; t++) {
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const f32x4 y = lt[t][c][lane];
#pragma unroll
                for (int x = 0; x < ST; x++) s[x][c] = mma(k[x][t], y, s[x][c]);
                if (t <= wave) o[c] = mma(p[t], lv[t][c][lane], o[c]);
            }
#pragma unroll
            for (int x = 0; x < ST; x++) load_k(i + 1, x, t);
            load_p(i + 1, t);
        }
        T *const out = static_cast<T *>(b.out) + ((int64_t)(row0 + 16 * wave + 4 * g4) * a.heads + h) * D + col0 + r16;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (16 * wave + 4 * g4 + e < n) {
#pragma unroll
                for (int c = 0; c < CT; c++) out[(int64_t)e * a.heads * D + 16 * c] = (T)o[c][e];
            }
    }
    if ((uint32_t)slot.y < (uint32_t)a.states) {
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    b.state[slot.y * size + at0 + (int64_t)(16 * (wave * ST + t) + 4 * g4 + e) * D + 16 * c] = s[t][c][e];
    }
}

uint64_t left_floats(const RaggedArgs &a) { return a.head_dim == 128 ? Left<128>::floats : Left<64>::floats; }
uint64_t keys_floats(const RaggedArgs &a) { return a.head_dim == 128 ? Left<128>::keys : Left<64>::keys; }

}  // namespace

uint64_t gdn_prompt_scratch_bytes(const RaggedArgs &a) {
    const uint64_t numbers = chunk_numbers<kC>(a.rows, a.requests);
    return numbers * (a.heads * left_floats(a) + a.groups * keys_floats(a)) * 4;
}

hipError_t launch_gdn_prompt(const GdnRows &b, uint32_t dtype, const RaggedArgs &a, void *scratch, hipStream_t s) {
    const uint32_t numbers = chunk_numbers<kC>(a.rows, a.requests);
    float *const left = static_cast<float *>(scratch), *const keys = left + (uint64_t)numbers * a.heads * left_floats(a);
    hipError_t err = hipSuccess;
    auto go = [&](auto e, auto d) {
        using E = decltype(e);
        constexpr int D = d();
        chunk_prepare_kernel<E, D><<<dim3(numbers, a.heads), 256, 0, s>>>(b, a, left, keys);
        err = hipGetLastError();
        if (err != hipSuccess) return;
        chunk_scan_kernel<E, D, 1><<<dim3(a.heads, D / 16, a.requests), 256, 0, s>>>(b, a, left, keys);
        err = hipGetLastError();
    };
    auto by_dim = [&](auto e) {
        if (a.head_dim == 128) go(e, std::integral_constant<int, 128>{});
        else go(e, std::integral_constant<int, 64>{});
    };
    if (dtype == YUUKA_DTYPE_F32) by_dim(RowF32{});
    else if (dtype == YUUKA_DTYPE_F16) by_dim(RowF16{});
    else by_dim(RowBF16{});
    return err;
}

}  // namespace yk

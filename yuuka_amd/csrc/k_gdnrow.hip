// k_gdnrow.hip — Gated DeltaNet layers over ragged rows: the causal
// convolution with SiLU and the q / k norm (forward.go:248-268, 484-493), and the
// delta rule for one row of every request (recurrent.go:56-105).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gdn_ragged_dev.h"
#include "internal.h"

namespace yk {

yuuka_status ragged_check(RaggedArgs *a, uint32_t dtype, bool conv) {
    constexpr int kBig = 1 << 30;
    if (dtype != YUUKA_DTYPE_F32 && dtype != YUUKA_DTYPE_F16 && dtype != YUUKA_DTYPE_BF16)
        return fail(YUUKA_ERR_UNSUPPORTED, "GDN rows of dtype %u (F32, F16 and BF16 are served)", dtype);
    if (a->requests < 1 || a->requests > 65535 || a->rows < 1 || a->rows > kBig)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "GDN rows: %d requests, %d rows", a->requests, a->rows);
    if (a->groups < 1 || a->heads < 1 || a->heads > 1024 || a->heads % a->groups)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "GDN rows: %d heads of %d groups", a->heads, a->groups);
    if (a->head_dim != 64 && a->head_dim != 128)
        return fail(YUUKA_ERR_UNSUPPORTED, "GDN head dimension %d (64 and 128 are served)", a->head_dim);
    a->channels = (2 * a->groups + a->heads) * a->head_dim;
    if (!a->stride) a->stride = a->channels;
    if (a->stride < a->channels || a->stride % 8 || a->stride > kBig)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "GDN rows of %d channels, %d elements apart (a multiple of 8)",
                    a->channels, a->stride);
    if (conv && (a->kernel < 2 || a->kernel > 8))
        return fail(YUUKA_ERR_UNSUPPORTED, "GDN convolution of %d taps (2 to 8 are served)", a->kernel);
    return YUUKA_OK;
}

namespace {

// Sum over aligned groups of N lanes, in every lane.
template <int CTRL> __device__ __forceinline__ float add_dpp(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int N> __device__ __forceinline__ float lanes_sum(float x) {
    x = add_dpp<0xb1>(x);   // lanes l ^ 1, l ^ 2, 7 - l of eight
    x = add_dpp<0x4e>(x);
    x = add_dpp<0x141>(x);
    if constexpr (N >= 16) x = add_dpp<0x128>(x);  // rotated by 8
    if constexpr (N >= 32) {
        const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(y[0]) + __uint_as_float(y[1]);
    }
    return x;
}

// Convolution: y_t = SiLU(sum_i w_i x_{t - K + 1 + i}), then q and k over their head's
// norm, q times `scale`. A wave takes 64 x 16 bytes of channels (whole heads) of `run`
// rows and keeps the last KT - 1 of them in registers; the wave with a request's first
// row reads its window and leaves its new one, which may be in the same slot.
// Requests without rows have their window moved by waves of their own.
// 8191 rows of 8192 channels in BF16, 0.27 GB, 71 us, 3.8 TB/s (a large copy reaches 4.7 to 5.1): vector
// instructions issue in 74 % of the SIMDs' cycles, and waves, four a SIMD, wait in 53 % of theirs.
template <typename E, int KT, int D>
__global__ __launch_bounds__(256) void ragged_conv_kernel(typename E::T *__restrict__ out,
                                                          const typename E::T *__restrict__ x,
                                                          const float *__restrict__ weight, float *__restrict__ state,
                                                          const int32_t *__restrict__ offsets,
                                                          const int2 *__restrict__ slots, RaggedArgs a, int run,
                                                          int row_blocks, int columns) {
    constexpr int V = E::kWide;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool moves = (int)blockIdx.y >= columns;  // windows of requests without rows
    const int item = moves ? ((int)blockIdx.y - columns) * (int)gridDim.x + (int)blockIdx.x : 0;
    const int column = moves ? item % columns : (int)blockIdx.y;
    if (!moves && (int)blockIdx.x >= row_blocks) return;
    const int c = (column * 64 + lane) * V;
    const bool live = c < a.channels;
    // The taps of the workgroup's channels, a channel's four in a place whose low bits are turned by the reading lane's,
    // so that lanes, whose channels are V apart, meet few banks. Read from memory by every lane for itself, 128 bytes
    // apart, they took 9 of 80 us.
    __shared__ float4 taps[KT == 4 ? 64 * V : 1];
    if constexpr (KT == 4) {
        const int c0 = column * 64 * V;
#pragma unroll
        for (int u = 0; u < V / 4; u++) {
            const int n = u * 256 + threadIdx.x;
            taps[n ^ (V == 8 ? n >> 3 & 7 : n >> 2 & 3)] = reinterpret_cast<const float4 *>(weight)[min(c0 + n, a.channels - 1)];
        }
        __syncthreads();
    }
    const int K1 = KT == 4 ? 3 : a.kernel - 1;  // (four taps are four; other numbers are the last of eight)
    const int64_t window = (int64_t)a.channels * K1;
    // the request's window before its rows, oldest first, zeros in front where K < KT
    float past[KT - 1][V] = {};
    auto load_window = [&](int j) {
        const int from = slots[j].x;
        const bool there = live && (uint32_t)from < (uint32_t)a.states;
        const float *const at = state + (there ? from * window + (int64_t)c * K1 : 0);
        if constexpr (KT == 4) {  // V channels of three inputs, side by side
            float4 y[3 * V / 4];
#pragma unroll
            for (int i = 0; i < 3 * V / 4; i++)
                y[i] = there ? reinterpret_cast<const float4 *>(at)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
            const float *const flat = reinterpret_cast<const float *>(y);
#pragma unroll
            for (int i = 0; i < V; i++)
#pragma unroll
                for (int t = 0; t < 3; t++) past[t][i] = flat[3 * i + t];
        } else {
#pragma unroll
            for (int t = 0; t < KT - 1; t++)
#pragma unroll
                for (int i = 0; i < V; i++)
                    past[t][i] = there && t >= KT - 1 - K1 ? at[i * K1 + t - (KT - 1 - K1)] : 0.0f;
        }
    };
    auto load_row = [&](int row, float (&y)[V]) {
        const Bytes16 none = {0, 0, 0, 0};
        unpack<E>(live ? *reinterpret_cast<const Bytes16 *>(x + (int64_t)row * a.stride + c) : none, y);
    };
    // The window after the request's rows: the last K - 1 of [window, rows].
    auto store_window = [&](int j, RowRange r) {
        const int to = slots[j].y, n = r.end - r.begin;
        if ((uint32_t)to >= (uint32_t)a.states) return;
        float next[KT - 1][V];
#pragma unroll
        for (int t = 0; t < KT - 1; t++) {
            const int back = KT - 1 - t;  // of the newest row: 1
            if (back <= n) {
                load_row(r.end - back, next[t]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) next[t][i] = 0.0f;
#pragma unroll
                for (int u = 0; u < KT - 1; u++)
                    if (u == t + n)
#pragma unroll
                        for (int i = 0; i < V; i++) next[t][i] = past[u][i];
            }
        }
        float *const at = state + to * window + (int64_t)c * K1;
        if (!live) return;
        if constexpr (KT == 4) {
            float4 y[3 * V / 4];
            float *const flat = reinterpret_cast<float *>(y);
#pragma unroll
            for (int i = 0; i < V; i++)
#pragma unroll
                for (int t = 0; t < 3; t++) flat[3 * i + t] = next[t][i];
#pragma unroll
            for (int i = 0; i < 3 * V / 4; i++) reinterpret_cast<float4 *>(at)[i] = y[i];
        } else {
#pragma unroll
            for (int t = 0; t < KT - 1; t++)
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (t >= KT - 1 - K1) at[i * K1 + t - (KT - 1 - K1)] = next[t][i];
        }
    };
    if (moves) {
        const int j = item / columns * 4 + wave;
        if (j >= a.requests) return;
        const RowRange r = row_range(offsets, a.rows, j);
        if (r.end > r.begin) return;
        load_window(j);
        store_window(j, r);
        return;
    }
    const int64_t first = ((int64_t)blockIdx.x * 4 + wave) * run;
    if (first >= a.rows) return;
    int row = (int)first;
    const int last = (int)min(first + run, (int64_t)a.rows);
    int j = wave_request_of_row(offsets, a.requests, row);
    if (j >= a.requests) return;
    float w[KT][V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        if constexpr (KT == 4) {
            const int n = lane * V + i;
            const float4 y = taps[n ^ (V == 8 ? n >> 3 & 7 : n >> 2 & 3)];
            w[0][i] = y.x, w[1][i] = y.y, w[2][i] = y.z, w[3][i] = y.w;
        } else {
#pragma unroll
            for (int t = 0; t < KT; t++) {
                const int at = t - (KT - 1 - K1);
                w[t][i] = live && at >= 0 ? weight[(int64_t)(c + i) * (K1 + 1) + at] : 0.0f;
            }
        }
    }
    const int keys = a.groups * D;
    RowRange r = row_range(offsets, a.rows, j);
    bool fresh = true;  // the window is not in the registers
    // Rows of the run that are on their way while one is worked on: three, since the window of four taps then moves by
    // names alone and the registers hold four waves a SIMD (8191 rows in BF16: two 81 us, three 78, four 111).
    constexpr int kAhead = 3;
    Bytes16 ahead[kAhead];
    auto load_raw = [&](int at) {
        const Bytes16 none = {0, 0, 0, 0};
        return live ? *reinterpret_cast<const Bytes16 *>(x + (int64_t)at * a.stride + c) : none;
    };
#pragma unroll
    for (int u = 0; u < kAhead; u++) ahead[u] = load_raw(min(row + u, last - 1));
    // A request's window is the wave's that has its first row: nobody else reads the slot that it may write. False when
    // the wave is done.
    auto step = [&](Bytes16 &slot) {
        while (row >= r.end) {
            if (row >= last || ++j >= a.requests) return false;
            r = row_range(offsets, a.rows, j);
            fresh = true;
        }
        const RowTurn turn = row_turn(r, row, (int)first, last, K1);
        if (turn == kRowDone) return false;
        const Bytes16 raw = row < last ? slot : load_raw(row);
        slot = load_raw(min(row + kAhead, last - 1));
        if (turn == kRowSkipped) return true;
        if (fresh) {
            if (row == r.begin) {
                load_window(j);
                store_window(j, r);
            } else {  // K - 1 rows of the request, or more, are before this one
#pragma unroll
                for (int t = 0; t < KT - 1; t++)
                    if (t >= KT - 1 - K1) load_row(max(row - (KT - 1 - t), r.begin), past[t]);
            }
            fresh = false;
        }
        float now[V], y[V], squares = 0.0f;
        unpack<E>(raw, now);
#pragma unroll
        for (int i = 0; i < V; i++) {
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < KT - 1; t++)
                if (t >= KT - 1 - K1) sum = fmaf(w[t][i], past[t][i], sum);
            sum = fmaf(w[KT - 1][i], now[i], sum);
            // SiLU by the hardware's exponential and reciprocal, a unit in the last place each
            y[i] = sum * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sum * -1.44269504088896341f));
            squares = fmaf(y[i], y[i], squares);
        }
        if (c < 2 * keys) {  // whole heads: a group of lanes takes one way
            const float norm = (c < keys ? a.scale : 1.0f) / sqrtf(lanes_sum<D / V>(squares) + a.eps);
#pragma unroll
            for (int i = 0; i < V; i++) y[i] *= norm;
        }
        if (live) *reinterpret_cast<Bytes16 *>(out + (int64_t)row * a.channels + c) = pack<E>(y);
#pragma unroll
        for (int t = 0; t < KT - 2; t++)
#pragma unroll
            for (int i = 0; i < V; i++) past[t][i] = past[t + 1][i];
#pragma unroll
        for (int i = 0; i < V; i++) past[KT - 2][i] = now[i];
        return true;
    };
    for (;;) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (!step(ahead[u])) return;
            row++;
        }
    }
}

// One row of every request:
//   S = e^g S;  d = beta (v - S^T k);  S += k d^T;  o = S^T q
// A workgroup holds COLS columns of one head's state, a thread four of them in every
// (256 / (COLS / 4))th row: the state is read and written once, in registers between, and is all the
// traffic there is to speak of. The row's own values are asked for before it (after it: 145 us for 141).
// 200 requests of 32 heads of 128 move 0.84 GB in 141 us, 6.0 TB/s; with 16, 64 and 128 columns a
// workgroup 154, 146, 146.
template <typename E, int D, int COLS>
__global__ __launch_bounds__(256) void ragged_step_kernel(GdnRows b, RaggedArgs a) {
    constexpr int C4 = COLS / 4, RG = 256 / C4, NR = D / RG, SPAN = C4 < 64 ? C4 : 64;
    static_assert(D % RG == 0, "whole rows");
    __shared__ float qk[2][D], vs[COLS];
    __shared__ float4 part[2][4][C4];
    typedef typename E::T T;
    const int h = blockIdx.x, col0 = blockIdx.y * COLS, j = blockIdx.z;  // (row j is request j's)
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, c4 = t % C4, rg = t / C4;
    const int2 slot = b.slots[j];
    const int64_t size = (int64_t)a.heads * D * D, mine = (int64_t)h * D * D + col0 + 4 * c4;
    const T *const x = static_cast<const T *>(b.qkv) + (int64_t)j * a.stride;
    const int group = h % a.groups;
    // sum over the row groups of every column, in every thread
    auto total = [&](float4 x, int which) {
#pragma unroll
        for (int off = C4; off < 64; off <<= 1) {
            x.x += __shfl_xor(x.x, off);
            x.y += __shfl_xor(x.y, off);
            x.z += __shfl_xor(x.z, off);
            x.w += __shfl_xor(x.w, off);
        }
        if (lane < SPAN) part[which][wave][c4] = x;
        __syncthreads();
        float4 sum = part[which][0][c4];
#pragma unroll
        for (int w = 1; w < 4; w++) {
            const float4 y = part[which][w][c4];
            sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
        }
        return sum;
    };
    const float own = t < 2 * D ? (float)x[(t < D ? group : a.groups + group) * D + (t & (D - 1))] : 0.0f;
    const float own_v = t < COLS ? (float)x[(2 * a.groups + h) * D + col0 + t] : 0.0f;
    const float decay = expf(log_decay_of(b, a, (int64_t)j * a.heads + h, h));
    const float beta = beta_of(b, a, (int64_t)j * a.heads + h);
    float4 s[NR];
#pragma unroll
    for (int m = 0; m < NR; m++)
        s[m] = (uint32_t)slot.x < (uint32_t)a.states
                   ? *reinterpret_cast<const float4 *>(b.state + slot.x * size + mine + (int64_t)(rg + RG * m) * D)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    if (t < 2 * D) qk[t / D][t & (D - 1)] = t < D ? own * a.scale : own;
    if (t < COLS) vs[t] = own_v;
    __syncthreads();
    float4 seen = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int m = 0; m < NR; m++) {
        const float k = qk[1][rg + RG * m];
        s[m].x *= decay; s[m].y *= decay; s[m].z *= decay; s[m].w *= decay;
        seen.x = fmaf(s[m].x, k, seen.x);
        seen.y = fmaf(s[m].y, k, seen.y);
        seen.z = fmaf(s[m].z, k, seen.z);
        seen.w = fmaf(s[m].w, k, seen.w);
    }
    seen = total(seen, 0);
    const float4 d = make_float4((vs[4 * c4] - seen.x) * beta, (vs[4 * c4 + 1] - seen.y) * beta,
                                 (vs[4 * c4 + 2] - seen.z) * beta, (vs[4 * c4 + 3] - seen.w) * beta);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int m = 0; m < NR; m++) {
        const float k = qk[1][rg + RG * m], q = qk[0][rg + RG * m];
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
        T *const to = static_cast<T *>(b.out) + ((int64_t)j * a.heads + h) * D + col0 + 4 * t;
        to[0] = (T)o.x;
        to[1] = (T)o.y;
        to[2] = (T)o.z;
        to[3] = (T)o.w;
    }
    if ((uint32_t)slot.y < (uint32_t)a.states) {
#pragma unroll
        for (int m = 0; m < NR; m++)
            *reinterpret_cast<float4 *>(b.state + slot.y * size + mine + (int64_t)(rg + RG * m) * D) = s[m];
    }
}

template <typename F> void by_type(uint32_t dtype, F &&f) {
    if (dtype == YUUKA_DTYPE_F32) f(RowF32{});
    else if (dtype == YUUKA_DTYPE_F16) f(RowF16{});
    else f(RowBF16{});
}

}  // namespace

hipError_t launch_gdn_ragged_conv(void *out, const void *x, uint32_t dtype, const float *weight, float *state,
                                  const int32_t *offsets, const int2 *slots, const RaggedArgs &a, hipStream_t s) {
    by_type(dtype, [&](auto e) {
        using E = decltype(e);
        typedef typename E::T T;
        // A wave's rows: as few as leave every CU the same number of workgroups, four or a multiple, and about 32 at most (16
        // in F32, of half the channels; a row or two more where the columns do not divide the workgroups, and more for
        // hundreds of columns and few rows). A wave's start, with request, taps and K - 1 rows more, is what fewer cost: 7 prompts of
        // 8191 rows, 32 heads in BF16, 8, 16 and 32 rows a wave 84, 77 and 71 us, 31 (a fifth workgroup on some CUs) 91;
        // 16 of 8000 rows, 32 heads in F32, 120, 115 and 127.
        constexpr int kRows = 4 * E::kWide;
        const int columns = (a.channels + 64 * E::kWide - 1) / (64 * E::kWide);
        const int64_t turns = ((int64_t)a.rows * columns + kRows * 4096 - 1) / (kRows * 4096);
        const int64_t runs = 4 * std::max<int64_t>(1024 * turns / columns, 1);
        const int run = (int)((a.rows + runs - 1) / runs);
        const int row_blocks = (int)(((int64_t)a.rows + 4 * run - 1) / (4 * run));
        // Windows that only move come after the rows, which are thus spread evenly: 16 prompts of 8000 rows, 16 heads in
        // F16, 74 -> 57 us.
        const int fours = (a.requests + 3) / 4, width = std::max(row_blocks, (fours + 7) / 8);
        const dim3 grid(width, columns + (int)(((int64_t)fours * columns + width - 1) / width));
        auto go = [&](auto taps, auto d) {
            ragged_conv_kernel<E, taps(), d()><<<grid, 256, 0, s>>>(static_cast<T *>(out), static_cast<const T *>(x), weight,
                                                                    state, offsets, slots, a, run, row_blocks, columns);
        };
        auto by_dim = [&](auto taps) {
            if (a.head_dim == 128) go(taps, std::integral_constant<int, 128>{});
            else go(taps, std::integral_constant<int, 64>{});
        };
        if (a.kernel == 4) by_dim(std::integral_constant<int, 4>{});
        else by_dim(std::integral_constant<int, 8>{});
    });
    return hipGetLastError();
}

hipError_t launch_gdn_step(const GdnRows &b, uint32_t dtype, const RaggedArgs &a, hipStream_t s) {
    by_type(dtype, [&](auto e) {
        using E = decltype(e);
        const dim3 grid(a.heads, a.head_dim / 32, a.requests);
        if (a.head_dim == 128) ragged_step_kernel<E, 128, 32><<<grid, 256, 0, s>>>(b, a);
        else ragged_step_kernel<E, 64, 32><<<grid, 256, 0, s>>>(b, a);
    });
    return hipGetLastError();
}

}  // namespace yk

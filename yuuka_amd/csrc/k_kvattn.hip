// k_kvattn.hip — attention of the newest rows of a batch of requests over
// their paged cache (F16 or Q8_0 pages), each request at its own length: the
// decode step of engine/gpu's session (one row) and the verify rows.
//
//   out = sum_t softmax_t(scale q . k_t) v_t,  t = 0 .. position of the row
//
// A workgroup takes one kv head of one request, up to 16 of its (row, query
// head) pairs and a part of the keys; its four waves walk the part's
// 32-key tiles, each with a running reference, sum and output of its own, and
// are joined at the end. With more parts than one the records {o, m, l} of
// the parts are joined by a second kernel. Keys and values of a wave's next tile
// are on their way while it works on one: a register is loaded again as soon as
// it has been used.
//
// Both products run on v_mfma_f32_16x16x32_f16 straight from the pages:
//  * scores = K Q^T (keys are the rows of the tile, so that a lane ends with
//    the scores of one query row and the keys 4 g .. 4 g + 3 of both 16-key
//    halves), P V with those very keys as lane g's eight: probabilities go from
//    the first product's result to the second's operand without leaving the lane;
//  * int8 digits are exact halves. A query is two halves (scaled by a power of
//    two to below 2^14), 22 bits of its largest element; a probability times its value
//    scale too, 22 bits in steps of 2^-24 at the least. The largest weight times the largest
//    scale is 2^9 or more in these units, so that blocks of values whose scale is more than 12
//    octaves below the largest lose precision by so much. Subnormal F16 values are summed to
//    2^-36 (an MFMA aligns them as if they were 2^-14). Sums are float32. Key scales
//    multiply the scores block by block (an MFMA covers one block of 32 dims).
//  * up to eight pairs ("stacked") put both halves in one 16-wide operand, as rows
//    n and n + 8; more take two MFMAs.
//  * p = 2^(s - m') with the reference m' = running max + E - 10, E the
//    exponent of the largest value scale so far: p times a scale stays below 2^14
//    and the halves' 39 octaves are used; m' moves (and the accumulators are
//    rescaled) when a tile passes it by 4.
//
// Measured, with the join: one row of one request over 120001 keys of 4 heads of 256, 16 query
// heads (261 MB of Q8_0) 62 us, 4.2 TB/s, of which some 12 before the first tile, after the
// last and for the join; 16 requests of 4096 such keys 40 us; 16 of 4096 keys of 8 heads of 128
// in F16 (269 MB) 58 us, 4.6 TB/s. Vector instructions issue in 52 % of a SIMD's cycles at
// 256 dims (700 a tile in the loop, 800 to 900 with what a wave does once), 61 % at 128, 17 %
// over F16: bound by the reads and, from Q8_0, by two waves a SIMD (256 registers) that wait
// for them in turn. 4 requests of 17 rows over 16384 keys of 4 heads of 256 take 101 us, and 114
// at the clock that a profiled run leaves: instructions (71 %), for every 16-row block turns
// each tile's digits to halves again.
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
typedef float Floats4 __attribute__((ext_vector_type(4), aligned(4)));  // at float alignment
typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int N> struct Dwords {  // N dwords at dword alignment
    typedef uint32_t V __attribute__((ext_vector_type(N), aligned(4)));
};
template <> struct Dwords<1> { typedef uint32_t V; };
template <int N> __device__ __forceinline__ uint32_t dword(const typename Dwords<N>::V &v, int i) { return v[i]; }
template <> __device__ __forceinline__ uint32_t dword<1>(const uint32_t &v, int) { return v; }

constexpr int kWaves = 4, kTile = 32;
constexpr float kHeadroom = 10.0f, kSlack = 4.0f;
// Waves of a SIMD, and workgroups of a CU, by the registers: a tile and accumulators of 64 dims are 32.
constexpr int waves_held(int groups, int blocks) {
    const int n = groups == 1 ? 4 : groups == 2 ? 3 : 2;
    return blocks == 1 ? n : n - 1;
}

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
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float max_wave(float x) {  // non-negative or not, no NaN kept
    x = fmaxf(x, dpp<0xb1>(x));   // lanes l ^ 1, l ^ 2, then rotated by 4 and 8
    x = fmaxf(x, dpp<0x4e>(x));
    x = fmaxf(x, dpp<0x124>(x));
    x = fmaxf(x, dpp<0x128>(x));
    return max_rows(x);
}
__device__ __forceinline__ uint32_t max_wave(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true));
    auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(a[0], a[1]);
    a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return max(a[0], a[1]);
}
__device__ __forceinline__ float sum_wave(float x) {
    x += dpp<0xb1>(x);
    x += dpp<0x4e>(x);
    x += dpp<0x124>(x);
    x += dpp<0x128>(x);
    return sum_rows(x);
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

// The lane's number, worked out where it stands. What is rarely used and kept over the loop is spilled,
// and a reload waits for all loads in flight.
__device__ __forceinline__ int lane_anew() {
    int zero = 0;
    asm volatile("" : "+v"(zero));
    return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
}
// Two halves, zeros in the place of infinities and NaN.
__device__ __forceinline__ uint32_t finite_halves(uint32_t x) {
    return ((x & 0x7c00u) == 0x7c00u ? 0u : x & 0xffffu) | ((x & 0x7c000000u) == 0x7c000000u ? 0u : x & 0xffff0000u);
}

template <int FMT, int GROUPS, bool STACK, bool PAGED, int RB> struct Layout {
    static constexpr bool Q8 = FMT == kKvQ8;
    static constexpr int D = 64 * GROUPS, NB = 2 * GROUPS, PER = STACK ? 8 : 16, ROWS = PER * RB;
    static constexpr uint32_t plane = NB * 1024;                              // query operands, one half
    static constexpr uint32_t scales = STACK ? plane : 2 * plane * RB;        // [wave][key, value][GROUPS][32] dwords
    static constexpr uint32_t addr = scales + (Q8 ? kWaves * 256 * GROUPS : 0);  // [wave][32] row offsets
    static constexpr uint32_t loop = addr + (PAGED ? 0 : kWaves * 256);
    static constexpr int slot_row = D + 4;                                    // floats; rows 4 g land 16 banks apart
    static constexpr uint32_t slots = kWaves * PER * slot_row * 4;            // over the loop's areas, after it
    static constexpr uint32_t stats = loop > slots ? loop : slots;            // m and l [wave][16], factor[ROWS], late[wave]
    static constexpr uint32_t late = stats + (2 * kWaves + RB) * 16 * 4;
    static constexpr uint32_t total = late + kWaves * 4;
};

// How the work is cut. A "column" is one (row block, kv head) of a request; a
// request's keys are cut into parts of at most `chunk` tiles, the same for all
// requests. W = all columns' tiles over `target`, the workgroups that the GPU
// holds at once. The smallest chunk of W .. 1.5 W (in four steps) whose parts are
// one round is taken; where there is none (more columns than workgroups, or
// very different lengths), W / 2, so that the last workgroups are short ones. The
// lengths are on the device: every wave works the cut out for itself, a
// request a lane (2700 cycles for one request, 3800 for 16).
struct AttnSplit {
    int row_blocks, columns;  // columns = row_blocks * kv_heads
    int group;                // query heads of a kv head
    uint32_t group_inverse;   // ceil(2^32 / group): n / group = high word of the product, n < 2^24 (group 1: 0)
    int target;
    float share;              // columns / target
    // 1: every request is one part, from twice as many columns as workgroups on. Nothing is worked out or
    // joined then, which is faster where the lengths are alike and far slower where one stands out: requests of
    // one row, 4 heads of 256 a KV head and 4 KV heads, 500 keys each: 255 (cut) 66.5 us, 256 (whole) 60.7; with
    // 120001 keys in one of them 158 and 2155 us.
    int whole;
    int page_shift;           // PAGED: log2(block_size / 16)
};
constexpr int kMaxParts = 256;

__device__ __forceinline__ int wave_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true);
    return __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) +
           __builtin_amdgcn_readlane(x, 48);
}
__device__ __forceinline__ int wave_max(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, true));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, true));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, true));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true));
    return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
               max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}

// Sums of the lanes up to and with each.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 into rows 2 and 3
    return x;
}

constexpr int kSegments = 4;  // of 64 requests, whose tiles stay in registers
struct Cut {
    int chunk, total;       // tiles of a part at most; parts of all requests
    float inverse;          // (just below) 1 / chunk
    int tiles[kSegments];   // the lane's requests'
    int64_t position;       // of the lane's request of the first 64: its first row's
};
// (requests that are cut are at most 2^11)
__device__ __forceinline__ int cut_tiles(const KvArgs &a, int64_t position) {
    const int len = (int)max((int64_t)1, min(position + a.rows, (int64_t)a.capacity));
    return min((len - 1) / kTile + 1, 1 << 19);
}
__device__ __forceinline__ int cut_tiles(const KvArgs &a, const ModelDyn &dyn, int base) {
    const int j = base + (threadIdx.x & 63);
    return j < a.requests ? cut_tiles(a, kv_position(a, dyn, j, 0)) : 0;
}
// ceil(tiles / chunk), or now and then one less (chunks of thousands of tiles): never more
__device__ __forceinline__ int cut_parts(int tiles, float inverse) {
    return tiles ? (int)(((float)tiles - 0.5f) * inverse) + 1 : 0;
}
// f(segment's tiles, its first request) for all of them
template <typename F>
__device__ __forceinline__ void each_segment(const KvArgs &a, const ModelDyn &dyn, const Cut &cut, F &&f) {
    f(cut.tiles[0], 0);
    if (a.requests <= 64) return;
#pragma unroll
    for (int i = 1; i < kSegments; i++) f(cut.tiles[i], 64 * i);
    for (int base = 64 * kSegments; base < a.requests; base += 64) f(cut_tiles(a, dyn, base), base);
}

__device__ __forceinline__ Cut cut_work(const KvArgs &a, const ModelDyn &dyn, const AttnSplit &sp) {
    Cut cut{0, a.requests, 0.0f, {}, 0};
    if (sp.whole) return cut;
    const int lane = threadIdx.x & 63;
    cut.position = kv_position(a, dyn, min(lane, a.requests - 1), 0);
    cut.tiles[0] = lane < a.requests ? cut_tiles(a, cut.position) : 0;
    if (a.requests > 64) {
#pragma unroll
        for (int i = 1; i < kSegments; i++) cut.tiles[i] = cut_tiles(a, dyn, 64 * i);
    }
    int sum = 0, top = 0;
    each_segment(a, dyn, cut, [&](int t, int) {
        sum += t;
        top = max(top, t);
    });
    if (a.requests > 1) {
        sum = wave_sum(sum);
        top = wave_max(top);
    }
    sum = __builtin_amdgcn_readfirstlane(sum);
    top = __builtin_amdgcn_readfirstlane(top);
    const int least = max(kWaves, (top + kMaxParts - 1) / kMaxParts);
    const int even = (int)ceilf((float)sum * sp.share);  // W: below 2^21, for at most 2 target columns are cut
    auto count = [&](Cut &cut) {
        cut.inverse = __builtin_amdgcn_rcpf((float)cut.chunk) * (1.0f - 0x1p-21f);
        int n = 0;
        each_segment(a, dyn, cut, [&](int t, int) { n += cut_parts(t, cut.inverse); });
        return a.requests > 1 ? wave_sum(n) : __builtin_amdgcn_readfirstlane(n);
    };
    for (int turn = 0; turn < 5; turn++) {  // W, then 1.5 W: if that is more than one round, nothing between is less
        const int eighths = turn == 0 ? 8 : turn == 2 ? 9 : turn == 3 ? 10 : 12;
        cut.chunk = max(least, (even * eighths + 7) / 8);
        cut.total = count(cut);
        const bool fits = cut.total * sp.columns <= sp.target;
        if (fits && turn != 1) break;
        if (!fits && turn == 1) {
            cut.chunk = max(least, (even + 1) / 2);
            cut.total = count(cut);
            break;
        }
    }
    return cut;
}

struct Part {
    int j, index, parts;  // request, part of it, its number of parts
    int record;           // parts before it of the requests with several
};

// Part number `item` of all.
__device__ __forceinline__ Part find_part(const KvArgs &a, const ModelDyn &dyn, const AttnSplit &sp, const Cut &cut,
                                          int item) {
    if (sp.whole) return {item, 0, 1, 0};
    if (a.requests == 1) return {0, item, cut.total, 0};
    Part part{};
    int before = 0, records_before = 0;
    each_segment(a, dyn, cut, [&](int t, int base) {
        const int n = cut_parts(t, cut.inverse);
        // parts, and parts of requests with several, summed as one (64 * 256 of each at most)
        const int own = n | (n > 1 ? n << 16 : 0), upto = wave_scan(own);
        const int here = __builtin_amdgcn_readlane(upto, 63);
        if (item >= before && item < before + (here & 0xffff)) {
            const int at = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(before + (upto & 0xffff) > item)) - 1;
            const int past = __builtin_amdgcn_readlane(upto - own, at);
            part = {base + at, item - before - (past & 0xffff), __builtin_amdgcn_readlane(n, at), records_before + (past >> 16)};
        }
        before += here & 0xffff;
        records_before += here >> 16;
    });
    return part;
}

// PAGED: pages are 16 << page_shift tokens, so that a 16-key half
// of a tile lies in one page, found by scalar loads and read through a
// buffer resource of that page's bytes (none for an unmapped page or past the end:
// such loads cost nothing and give zeros).
template <int FMT, int GROUPS, bool STACK, bool PAGED, int RB>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(waves_held(GROUPS, RB)))) void kv_attention_kernel(
    const float *__restrict__ q, int q_stride, const float *__restrict__ gate, int gate_stride,
    const uint8_t *__restrict__ kpool, const uint8_t *__restrict__ vpool, const int32_t *__restrict__ table, KvArgs a,
    AttnSplit sp, float *__restrict__ part, float2 *__restrict__ stats, int2 *__restrict__ plan, float *__restrict__ out,
    ModelDyn dyn) {
    using L = Layout<FMT, GROUPS, STACK, PAGED, RB>;
    constexpr bool Q8 = L::Q8;
    constexpr int D = L::D, NB = L::NB, PER = L::PER, ROWS = L::ROWS;
    constexpr int KP = Q8 ? GROUPS : 2 * GROUPS;  // 16-byte pieces of a key per lane
    extern __shared__ __align__(16) uint8_t lds[];
    float *const st_m = reinterpret_cast<float *>(lds + L::stats), *const st_l = st_m + kWaves * 16;
    float *const row_factor = st_l + kWaves * 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    // the wave's values that are not finite, and that not every row sees, were taken as zeros (in LDS, which
    // costs the loop no register)
    auto late = [&]() -> int & { return *reinterpret_cast<int *>(lds + L::late + 4 * wave); };
    const int r16 = lane & 15, g4 = lane >> 4;
    // Workgroups go to the eight XCDs in turn. Each XCD gets one run of the work
    // items in the order (row block, kv head, part, request), so that what
    // reads one run of tokens, all heads' scales in one line, shares an L2.
    const Cut cut = cut_work(a, dyn, sp);
    int item = blockIdx.x;
    {
        const int n = __builtin_amdgcn_readfirstlane(cut.total) * sp.columns, x = item & 7;
        if (item >= n) return;
        item = x * (n >> 3) + min(x, n & 7) + (item >> 3);
    }
    const int turn_of = (uint32_t)item / (uint32_t)sp.columns, column = item - turn_of * sp.columns;
    const int kvh = sp.row_blocks == 1 ? column : (uint32_t)column / (uint32_t)sp.row_blocks;
    const int rb = column - kvh * sp.row_blocks;
    const Part pt = find_part(a, dyn, sp, cut, turn_of);
    const int j = __builtin_amdgcn_readfirstlane(pt.j), split = __builtin_amdgcn_readfirstlane(pt.index);
    const int parts = __builtin_amdgcn_readfirstlane(pt.parts);
    const int G = sp.group;
    auto row_of = [&](int n) { return sp.group_inverse ? (int)__umulhi((uint32_t)n, sp.group_inverse) : n; };
    const int n0 = rb * ROWS, nr = min(ROWS, G * a.rows - n0);  // pairs n = row * G + head of the group
    int64_t p0;
    if (sp.whole || j >= 64) p0 = kv_position(a, dyn, j, 0);
    else p0 = (int64_t)__builtin_amdgcn_readlane((int)(cut.position >> 32), j) << 32 |
              (uint32_t)__builtin_amdgcn_readlane((int)cut.position, j);
    // last key a row sees, -1 for none
    auto limit = [&](int n) { return (int)max((int64_t)-1, min(p0 + row_of(n), (int64_t)a.capacity - 1)); };
    const int len = __builtin_amdgcn_readfirstlane(limit(n0 + nr - 1) + 1);
    const int least = __builtin_amdgcn_readfirstlane(limit(n0));
    // (the parts are of the last row block's tiles; an earlier one may need fewer)
    const int tiles = (len + kTile - 1) / kTile;
    int c0 = 0, c1 = tiles;
    if (parts > 1) {
        const int last = (int)max((int64_t)1, min(p0 + a.rows, (int64_t)a.capacity));
        const uint32_t all = (uint32_t)((last - 1) / kTile + 1), each = all / (uint32_t)parts, more = all - each * parts;
        c0 = split * each + min(split, (int)more);
        c1 = min(tiles, c0 + (int)each + (split < (int)more));
    }
    c0 = __builtin_amdgcn_readfirstlane(c0);
    c1 = __builtin_amdgcn_readfirstlane(c1);
    const int64_t record = ((int64_t)(__builtin_amdgcn_readfirstlane(pt.record) + split) * sp.columns + column) * ROWS;
    const int64_t out_row = (int64_t)j * a.rq_rows;
    if (plan && split == 0 && column == 0 && threadIdx.x == 0) plan[j] = make_int2(parts, pt.record);
    if (c0 >= c1 && parts > 1) {  // nothing here: empty records
        const int tid = 64 * wave + lane_anew();
        if (tid < nr) stats[record + tid] = make_float2(-INFINITY, 0.0f);
        return;
    }

    // the query rows that this wave prepares: loaded before the first tile, since
    // loads return in order
    float queries[ROWS / kWaves][GROUPS];
#pragma unroll
    for (int half = 0; half < ROWS / kWaves; half++) {
        const int n = min(wave + kWaves * half, nr - 1), r = row_of(n0 + n), h = kvh * G + n0 + n - r * G;
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
    // The pages of the wave's next 32 tiles, two a tile, a half a lane: one load in
    // 32 turns. (A scalar load a turn stalls it: any wait for LDS is one for that load too.)
    int page_queue = -1;
    auto pages_of = [&](int turn) {
        Tile t{};
        if constexpr (PAGED) {
            if ((turn & 31) == 0) {
                int at = lane;  // opaque: nothing of this is kept in registers over the loop
                asm volatile("" : "+v"(at));
                const int mine = c0 + wave + kWaves * (turn + (at >> 1)), tok = kTile * mine + 16 * (at & 1);
                const bool in = mine < c1 && tok < len;
                const int page = table_j[(uint32_t)(in ? tok >> (4 + sp.page_shift) : 0)];
                page_queue = in ? page : -1;
            }
            const int c = c0 + wave + kWaves * turn;
#pragma unroll
            for (int T = 0; T < 2; T++) {
                const int tok = kTile * c + 16 * T;
                const int page = __builtin_amdgcn_readlane(page_queue, 2 * (turn & 31) + T);
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
    uint32_t soff = (lane & 15) * (a.kv_dim / 16) + kvh * NB * 2;
    auto load_scales = [&](const Tile &t) {  // (an unmapped half reads page 0's: not used)
        if constexpr (Q8 && PAGED) {
            uint64_t k0 = (uint64_t)kpool + t.scales[0], k1 = (uint64_t)kpool + t.scales[1];
            uint64_t v0 = (uint64_t)vpool + t.scales[0], v1 = (uint64_t)vpool + t.scales[1];
            asm volatile("" : "+s"(k0), "+s"(k1), "+s"(v0), "+s"(v1));  // (no lane's pool kept in registers)
            const uint64_t at = (lane < 32 ? (lane & 16 ? k1 : k0) : (lane & 16 ? v1 : v0)) + soff;
            sreg = *reinterpret_cast<const __attribute__((address_space(1))) typename Dwords<GROUPS>::V *>(at);
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
    // 64-byte pieces p - 1 and p of the keys (the last may be alone), and 64-dim groups of
    // the values: what shares a line is asked for together.
    auto load_keys = [&](__amdgpu_buffer_rsrc_t rs, int T, int p) {
        if (p & 1) load_key(rs, T, p - 1);
        load_key(rs, T, p);
    };
    auto load_values = [&](__amdgpu_buffer_rsrc_t v0, __amdgpu_buffer_rsrc_t v1, int u) {
        if (Q8 && !(u & 1) && u < GROUPS - 1) return;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (Q8 && (u & 1)) load_value(i < 4 ? v0 : v1, i, u - 1);
            load_value(i < 4 ? v0 : v1, i, u);
        }
    };
    int c = c0 + wave;
    Tile cur = PAGED ? pages_of(0) : find_rows(c);
    // (in the loop's order: its waits count the loads issued since, on either way into it)
    load_scales(cur);
    __builtin_amdgcn_sched_barrier(0);
    {
        const auto k0 = resource(kpool, cur, 0), k1 = resource(kpool, cur, 1);
        const auto v0 = resource(vpool, cur, 0), v1 = resource(vpool, cur, 1);
#pragma unroll
        for (int p = 0; p < KP; p++)
            if ((p & 1) || p == KP - 1) {
                load_keys(k0, 0, p);
                load_keys(k1, 1, p);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
        for (int u = 0; u < GROUPS; u++) {
            load_values(v0, v1, u);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : a.scale;
    // ---- queries as MFMA operands in LDS: wave w prepares rows w, w + kWaves, ...
#pragma unroll
    for (int half = 0; half < ROWS / kWaves; half++) {
        const int n = wave + kWaves * half;
        const float(&x)[GROUPS] = queries[half];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < GROUPS; s++) top = fmaxf(top, fabsf(x[s]));
        top = max_wave(top);
        int e = 14;
        if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e);  // top < 2^e
        const int in = Q8 ? lane : 0;
        // dim 64 s + lane: block 2 s + h, lane group g, place k of the operand's eight
        const int hb = Q8 ? in >> 5 : lane >> 5;
        const int g = Q8 ? (lane & 15) >> 2 : (lane & 31) >> 3;
        const int k = Q8 ? 2 * (lane & 3) + ((lane >> 4) & 1) : lane & 7;
#pragma unroll
        for (int s = 0; s < GROUPS; s++) {
            const float y = ldexpf(x[s] * sign, 14 - e);
            const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
            const uint32_t at = n / PER * 2 * L::plane + ((2 * s + hb) * 64 + 16 * g + n % PER) * 16 + 2 * k;
            *reinterpret_cast<_Float16 *>(lds + at) = hi;
            *reinterpret_cast<_Float16 *>(lds + at + (STACK ? 8 * 16 : L::plane)) = lo;
        }
        // scores in units of log2: factor * (operand product). The factor is above zero (a key left
        // out has -infinity times it): the sign, or the whole of a scale of zero, goes to the
        // query. (Products are below 2^45: times 2^-126 they are nothing to the exponential.)
        if (lane == 0) row_factor[n] = fmaxf(ldexpf(fabsf(a.scale) * 1.44269504088896341f, e - 14), 0x1p-126f);
    }
    late() = 0;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");

    const int my_n = STACK ? r16 & 7 : r16;
    const bool low_half = STACK && r16 >= 8;  // this lane's probabilities are the remainders
    float factor[RB];
    int my_limit[RB];
    f32x4 acc[RB][GROUPS][4];
    float ref[RB], l[RB];
#pragma unroll
    for (int b = 0; b < RB; b++) {
        const int n = PER * b + my_n;
        factor[b] = row_factor[n];
        my_limit[b] = n < nr ? limit(n0 + n) : -1;
        ref[b] = -INFINITY;
        l[b] = 0.0f;
#pragma unroll
        for (int s = 0; s < GROUPS; s++)
#pragma unroll
            for (int t = 0; t < 4; t++) acc[b][s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    Tile next{};
    if constexpr (PAGED) next = pages_of(1);
    for (int turn = 0; c < c1; c += kWaves, turn++) {
        // Opaque in every turn: the constant steps from these addresses then stay
        // in the instructions' immediate offsets. Hoisted out of the loop they take a
        // register each, loaded values spill, and every spill waits for all loads.
        asm volatile("" : "+v"(koff), "+v"(voff_row[0]), "+v"(voff_row[1]), "+v"(voff_row[2]), "+v"(voff_row[3]));
        asm volatile("" : "+v"(scale_write), "+v"(scale_read), "+v"(query_read), "+v"(soff));
        // every row sees every key of the tile
        const bool whole = cur.keys == ~0u && kTile * c + kTile - 1 <= least;
        float E = 0.0f;
        if constexpr (Q8) {
            // scales to LDS (those of missing keys as zeros), and the largest finite value scale's exponent
            wave_lds_fence();
            const bool there = __builtin_amdgcn_inverse_ballot_w64((uint64_t)cur.keys << 32 | cur.keys);
            uint32_t d[GROUPS];
            ushort2v two = {0, 0};  // largest of each half, as integers
#pragma unroll
            for (int s = 0; s < GROUPS; s++) {
                d[s] = there ? dword<GROUPS>(sreg, s) : 0u;
                two = __builtin_elementwise_max(two, __builtin_bit_cast(ushort2v, d[s] & 0x7fff7fffu));
            }
            uint32_t most = max((uint32_t)two[0], (uint32_t)two[1]);
            const bool over = most >= 0x7c00u;  // an infinity or a NaN
            if (__any(over)) {
                most = 0;
#pragma unroll
                for (int s = 0; s < GROUPS; s++) {
                    const uint32_t lo = d[s] & 0x7fffu, hi = (d[s] >> 16) & 0x7fffu;
                    most = max(most, max(lo < 0x7c00u ? lo : 0u, hi < 0x7c00u ? hi : 0u));
                    // infinities become NaN: with one, a score could be -infinity and leave its key out
                    d[s] |= (lo < 0x7c00u ? 0u : 0x200u) | (hi < 0x7c00u ? 0u : 0x2000000u);
                }
            }
            if (!whole && __any(over)) {  // a value's scale that not every row sees
                const bool put_off = over && lane_anew() >= 32 && kTile * c + (lane_anew() & 31) > least;
                if (__any(put_off)) late() = 1;
                if (put_off) {
#pragma unroll
                    for (int s = 0; s < GROUPS; s++) d[s] = finite_halves(d[s]);
                }
            }
#pragma unroll
            for (int s = 0; s < GROUPS; s++) *reinterpret_cast<uint32_t *>(lds + scale_write + 128 * s) = d[s];
            E = (float)((int)(max_wave(lane < 32 ? 0u : most) >> 10) - 14);  // scale < 2^E
            wave_lds_fence();
        }
        Tile after{};
        if constexpr (!PAGED) next = find_rows(c + kWaves);
        // ---- scores: keys 4 g + e of half T against query row r16
        float s[RB][2][4] = {};
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
                half8 kk[2];
#pragma unroll
                for (int T = 0; T < 2; T++) {
                    if constexpr (Q8) {
                        const u32x4 w = kreg[T][b >> 1] ^ 0x80808080u;
                        kk[T] = b & 1 ? join(key_digits<1>(w[0]), key_digits<1>(w[1]), key_digits<1>(w[2]), key_digits<1>(w[3]))
                                      : join(key_digits<0>(w[0]), key_digits<0>(w[1]), key_digits<0>(w[2]), key_digits<0>(w[3]));
                    } else {
                        kk[T] = __builtin_bit_cast(half8, kreg[T][b]);
                    }
                }
#pragma unroll
                for (int n = 0; n < RB; n++) {
                    const uint8_t *const operand = lds + query_read + (2 * n * L::plane + b * 1024);
                    const half8 qh = *reinterpret_cast<const half8 *>(operand);
                    half8 ql{};
                    if constexpr (!STACK) ql = *reinterpret_cast<const half8 *>(operand + L::plane);
#pragma unroll
                    for (int T = 0; T < 2; T++) {
                        f32x4 d = {0.f, 0.f, 0.f, 0.f};
                        if constexpr (!Q8) d = f32x4{s[n][T][0], s[n][T][1], s[n][T][2], s[n][T][3]};
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[T], qh, d, 0, 0, 0);
                        if constexpr (!STACK) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[T], ql, d, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if constexpr (Q8)
                                s[n][T][e] = fmaf(d[e], (float)__builtin_bit_cast(half2v, (uint32_t)ks[T][e])[b & 1], s[n][T][e]);
                            else
                                s[n][T][e] = d[e];
                        }
                    }
                }
                const int p = Q8 ? b >> 1 : b;  // the piece that this block was in
                if ((!Q8 || (b & 1)) && ((p & 1) || p == KP - 1)) {
                    load_keys(k0, 0, p);
                    load_keys(k1, 1, p);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        load_scales(next);
        if constexpr (PAGED) after = pages_of(turn + 2);
        // ---- softmax of the lane's rows over its eight keys
#pragma unroll
        for (int n = 0; n < RB; n++)
#pragma unroll
            for (int T = 0; T < 2; T++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (STACK) s[n][T][e] += ror8(s[n][T][e]);
                    // An infinite score, of a key that holds one (others are below 2^45), becomes NaN:
                    // one of -infinity would leave its key out.
                    if constexpr (!Q8) s[n][T][e] = fmaf(s[n][T][e], 0.0f, s[n][T][e]);
                }
        if (!whole) {
            const int first = 4 * (lane_anew() >> 4);  // (what follows is not kept in registers for every tile)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int kk = first + 16 * (i >> 2) + (i & 3);
                const bool there = (cur.keys >> kk) & 1;
                if constexpr (!Q8) {  // values that not every row sees must be finite for those that do not
                    uint32_t over = 0;
#pragma unroll
                    for (int u = 0; u < GROUPS; u++)
#pragma unroll
                        for (int w = 0; w < 2; w++) over |= (vhalf[i][u][w] & 0x7fff7fffu) + 0x04000400u;
                    const bool put_off = there && (over & 0x80008000u) != 0 && kTile * c + kk > least;
                    if (__any(put_off)) {
                        late() = 1;
                        if (put_off) {
#pragma unroll
                            for (int u = 0; u < GROUPS; u++)
#pragma unroll
                                for (int w = 0; w < 2; w++) vhalf[i][u][w] = finite_halves(vhalf[i][u][w]);
                        }
                    }
                    if (!there) {
#pragma unroll
                        for (int u = 0; u < GROUPS; u++) vhalf[i][u] = u32x2{0, 0};
                    }
                }
#pragma unroll
                for (int n = 0; n < RB; n++) {
                    const bool seen = there && kTile * c + kk <= my_limit[n];
                    s[n][i >> 2][i & 3] = seen ? s[n][i >> 2][i & 3] : -INFINITY;
                }
            }
        }
        float p[RB][8];
        float top[RB];
        bool move = false;
#pragma unroll
        for (int n = 0; n < RB; n++) {
            top[n] = -INFINITY;
#pragma unroll
            for (int T = 0; T < 2; T++)
#pragma unroll
                for (int e = 0; e < 4; e++) top[n] = fmaxf(top[n], s[n][T][e]);
            top[n] = fmaf(max_rows(top[n]), factor[n], E - kHeadroom);
            move = move || top[n] > ref[n] + kSlack;
        }
        if (__any(move)) {
#pragma unroll
            for (int n = 0; n < RB; n++) {
                const bool filled = __any(ref[n] != -INFINITY);  // not in the wave's first tile
                const float moved = fmaxf(ref[n], top[n]);
                const float shrink = moved == ref[n] ? 1.0f : __builtin_amdgcn_exp2f(ref[n] - moved);
                ref[n] = moved;
                if (filled) {
                    l[n] *= shrink;
                    float row_shrink[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) row_shrink[e] = __shfl(shrink, 4 * g4 + e);
#pragma unroll
                    for (int u = 0; u < GROUPS; u++)
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[n][u][t][e] *= row_shrink[e];
                }
            }
        }
#pragma unroll
        for (int n = 0; n < RB; n++) {
            const float base = ref[n] == -INFINITY ? 0.0f : ref[n];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                p[n][i] = __builtin_amdgcn_exp2f(fmaf(s[n][i >> 2][i & 3], factor[n], -base));
                l[n] += p[n][i];
            }
        }
        // ---- value product: keys 4 g + e of both halves are the lane's eight
        {
            u32x4 vs[2];  // two blocks' scales of the lane's keys
            const auto v0 = resource(vpool, next, 0), v1 = resource(vpool, next, 1);
            half8 ph[RB], pl[RB];
            // p[i] * d(i) as two halves (stacked: the one that the lane's row is)
            auto halves = [&](int n, auto d) {
                half2v h[4], o[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = d(2 * i), y = d(2 * i + 1), px = p[n][2 * i], py = p[n][2 * i + 1];
                    h[i] = half2v{(_Float16)fmaf(px, x, 0.0f), (_Float16)fmaf(py, y, 0.0f)};
                    o[i] = half2v{(_Float16)fmaf(px, x, -(float)h[i][0]), (_Float16)fmaf(py, y, -(float)h[i][1])};
                    // one value h in every lane: rounded twice by different
                    // instructions, the two rows' halves need not be each other's
                    if constexpr (STACK) o[i] = low_half ? o[i] : h[i];
                }
                ph[n] = join(h[0], h[1], h[2], h[3]);
                pl[n] = join(o[0], o[1], o[2], o[3]);
            };
            if constexpr (!Q8) {
#pragma unroll
                for (int n = 0; n < RB; n++) halves(n, [](int) { return 1.0f; });
            }
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
                        if (!(t & 1)) {  // block 2 u + t / 2
#pragma unroll
                            for (int n = 0; n < RB; n++)
                                halves(n, [&](int i) {
                                    return (float)__builtin_bit_cast(half2v, (uint32_t)vs[i >> 2][i & 3])[t >> 1];
                                });
                        }
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
#pragma unroll
                    for (int n = 0; n < RB; n++) {
                        if constexpr (!STACK) acc[n][u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[n], vv, acc[n][u][t], 0, 0, 0);
                        acc[n][u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[n], vv, acc[n][u][t], 0, 0, 0);
                    }
                }
                load_values(v0, v1, u);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        cur = next;
        if constexpr (PAGED) next = after;
    }

    {
        const int lane = lane_anew(), r16 = lane & 15, g4 = lane >> 4, tid = 64 * wave + lane;
        // ---- the values put off: their dims of the rows that see them are not finite, as where every row does
        if (least + 1 < len && __builtin_amdgcn_readfirstlane(late())) {
            KvLayout cache = a;
            asm volatile("" : "+s"(cache.block_size));  // (its reciprocal is not kept over the loop either)
            for (int key = max(least + 1, kTile * c0); key < min(len, kTile * c1); key++) {
                int64_t row, sc;
                if ((key / kTile - c0) % kWaves != wave || !kv_slot(cache, table, j, key, &row, &sc)) continue;
                const uint16_t *const halves = reinterpret_cast<const uint16_t *>(vpool + (Q8 ? sc : row)) + kvh * (Q8 ? NB : D);
#pragma unroll
                for (int u = 0; u < GROUPS; u++)
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const bool bad = (halves[Q8 ? 2 * u + (t >> 1) : 64 * u + 4 * r16 + t] & 0x7c00u) == 0x7c00u;
#pragma unroll
                        for (int b = 0; b < RB; b++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (__shfl(my_limit[b], 4 * g4 + e) >= key && bad) acc[b][u][t][e] = NAN;
                    }
            }
        }

        // ---- the waves' outputs joined: o = sum_w 2^(ref_w - max ref) o_w
#pragma unroll
        for (int b = 0; b < RB; b++) {
            if (b * PER >= nr) break;
            l[b] = sum_rows(l[b]);
            __syncthreads();  // every wave is done with what the slots lie over
            float *const slot = reinterpret_cast<float *>(lds) + wave * PER * L::slot_row;
            const float unit = Q8 ? 512.0f : 1.0f;  // the digits were times 2^-9
            auto dim = [&](int u, int t) { return 64 * u + (Q8 ? 16 * t + r16 : 4 * r16 + t); };
#pragma unroll
            for (int u = 0; u < GROUPS; u++)
#pragma unroll
                for (int t = 0; t < 4; t += STACK ? 2 : 1)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (STACK) {
                            // rows n and n + 8, 32 lanes apart: one swap puts t's two halves and t + 1's
                            // side by side, their sums in the lower and the upper lanes
                            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[b][u][t][e]),
                                                                            __float_as_uint(acc[b][u][t + 1][e]), false, false);
                            slot[(4 * (g4 & 1) + e) * L::slot_row + dim(u, t) + (Q8 ? 16 : 1) * (g4 >> 1)] =
                                (__uint_as_float(x[0]) + __uint_as_float(x[1])) * unit;
                        } else {
                            slot[(4 * g4 + e) * L::slot_row + dim(u, t)] = acc[b][u][t][e] * unit;
                        }
                    }
            if (lane < PER) {
                st_m[wave * 16 + lane] = ref[b];
                st_l[wave * 16 + lane] = l[b];
            }
            __syncthreads();
            for (int idx = tid; idx < min(PER, nr - b * PER) * (D / 4); idx += 64 * kWaves) {
                const int m16 = idx / (D / 4), n = b * PER + m16, d = 4 * (idx % (D / 4));
                float m = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWaves; w++) m = fmaxf(m, st_m[w * 16 + m16]);
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
                float total = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float mw = st_m[w * 16 + m16];
                    const float f = mw == m ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
                    const f32x4 x = *reinterpret_cast<const f32x4 *>(lds + ((w * PER + m16) * L::slot_row + d) * 4);
                    o += f * x;
                    total = fmaf(f, st_l[w * 16 + m16], total);
                }
                const int r = row_of(n0 + n), h = kvh * G + n0 + n - r * G;
                if (parts == 1) {
                    const int64_t at = (out_row + r) * a.heads + h;
                    const float inv = 1.0f / total;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float y = total == 0.0f ? 0.0f : o[i] * inv;  // a row that sees no key
                        if (gate) y *= sigmoid_ref(gate[at * gate_stride + d + i]);
                        out[at * D + d + i] = y;
                    }
                } else {
                    *reinterpret_cast<f32x4 *>(part + (record + n) * D + d) = o;
                    if (d == 0) stats[record + n] = make_float2(m, total);
                }
            }
        }
    }
}

// Where the records of one (row, head) of a request are: part s's at first + s * step.
struct Records {
    int parts;
    int64_t first, step;
};
__device__ __forceinline__ Records records_of(const int2 *plan, const KvArgs &a, int row_blocks, int pairs_per_block, int j,
                                              int r, int h) {
    const int2 mine = plan[j];
    const int G = a.heads / a.kv_heads, kvh = h / G, pair = r * G + h - kvh * G, columns = row_blocks * a.kv_heads;
    const int column = kvh * row_blocks + pair / pairs_per_block;
    return {mine.x, ((int64_t)mine.y * columns + column) * pairs_per_block + pair % pairs_per_block,
            (int64_t)columns * pairs_per_block};
}

// Joins a request's parts, few of them: one wave per (row, head, request), a part a lane for the
// weights, four dims a lane for the outputs, with kDeep records in flight from before the
// weights are known.
template <int GROUPS>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(const float *__restrict__ part,
                                                                const float2 *__restrict__ stats,
                                                                const int2 *__restrict__ plan,
                                                                const float *__restrict__ gate, int gate_stride,
                                                                float *__restrict__ out, KvArgs a, int row_blocks,
                                                                int pairs_per_block) {
    constexpr int D = 64 * GROUPS, kQuads = D / 4, kWide = 64 / kQuads, kDeep = 8;  // kWide records side by side
    const int lane = threadIdx.x & 63, j = blockIdx.y;
    const int item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= a.rows * a.heads) return;  // whole waves: no barrier below
    const int r = item / a.heads, h = item - r * a.heads;
    const Records rec = records_of(plan, a, row_blocks, pairs_per_block, j, r, h);
    if (rec.parts == 1) return;  // written by its workgroup
    const int64_t row = ((int64_t)j * a.rq_rows + r) * a.heads + h;
    const int sub = lane / kQuads, d = 4 * (lane % kQuads);
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    f32x4 x[kDeep], o = none, g = none;
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < kDeep; u++) {
            const int s = min(s0 + kWide * u + sub, rec.parts - 1);  // (no branches between the loads)
            x[u] = *reinterpret_cast<const f32x4 *>(part + (rec.first + s * rec.step) * D + d);
        }
    };
    // weights of the parts base + lane; 64 of them at a time, the maximum over all first
    auto stat = [&](int base) {
        return base + lane < rec.parts ? stats[rec.first + (base + lane) * rec.step] : make_float2(-INFINITY, 0.0f);
    };
    float2 ml = stat(0);
    load(0);
    if (gate && lane < kQuads) g = *reinterpret_cast<const Floats4 *>(gate + row * gate_stride + d);
    float m = ml.x;
    for (int base = 64; base < rec.parts; base += 64) m = fmaxf(m, stat(base).x);
    m = max_wave(m);
    float l = 0.0f;
    for (int base = 0;;) {
        // a part without keys (no sum) weighs nothing, whatever its output holds
        const float w = ml.y == 0.0f ? 0.0f : ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m);
        const float weight = ml.y == 0.0f ? -1.0f : w;
        l += w * ml.y;
        const int upto = min(64, rec.parts - base);
        for (int s0 = 0;;) {
#pragma unroll
            for (int u = 0; u < kDeep; u++) {
                const int s = s0 + kWide * u + sub;
                const float f = __shfl(weight, s & 63);
                if (s < upto && f >= 0.0f) o += f * x[u];
            }
            s0 += kWide * kDeep;
            if (s0 >= upto) break;
            load(base + s0);
        }
        base += 64;
        if (base >= rec.parts) break;
        ml = stat(base);
        load(base);
    }
    l = sum_wave(l);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = kWide == 4 ? sum_rows(o[i]) : kWide == 2 ? sum_halves(o[i]) : o[i];
    if (lane < kQuads) {
        const float inv = 1.0f / l;
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y[i] = l == 0.0f ? 0.0f : o[i] * inv;  // a row that sees no key
            if (gate) y[i] *= sigmoid_ref(g[i]);
        }
        *reinterpret_cast<Floats4 *>(out + row * D + d) = y;
    }
}

// The same for many parts: one workgroup per (row, head, request) and 64 dims. A thread has
// four dims of every 16th record, eight of them loaded while the weights are worked
// out, a part a thread.
__global__ __launch_bounds__(256) void kv_attention_merge_kernel(const float *__restrict__ part,
                                                                 const float2 *__restrict__ stats,
                                                                 const int2 *__restrict__ plan,
                                                                 const float *__restrict__ gate, int gate_stride,
                                                                 float *__restrict__ out, KvArgs a, int row_blocks,
                                                                 int pairs_per_block) {
    static_assert(kMaxParts <= 256, "a part a thread");
    constexpr int kDeep = 8;
    __shared__ float weight[256], red[2][4];
    __shared__ f32x4 sum[4][16];
    const int h = blockIdx.y, j = blockIdx.z, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int slices = a.head_dim / 64, r = blockIdx.x / slices, d0 = 64 * (blockIdx.x % slices);
    const Records recs = records_of(plan, a, row_blocks, pairs_per_block, j, r, h);
    const int parts = recs.parts;
    if (parts == 1) return;  // written by its workgroup
    const int64_t row = ((int64_t)j * a.rq_rows + r) * a.heads + h;
    const float2 ml = tid < parts ? stats[recs.first + tid * recs.step] : make_float2(-INFINITY, 0.0f);
    const int rec = tid >> 4, d = d0 + 4 * (tid & 15);
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    f32x4 x[kDeep], o = none;
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < kDeep; u++) {
            const int s = s0 + 16 * u;
            x[u] = s < parts ? *reinterpret_cast<const f32x4 *>(part + (recs.first + s * recs.step) * a.head_dim + d) : none;
        }
    };
    load(rec);
    float g = 0.0f;
    if (gate && tid < 64) g = gate[row * gate_stride + d0 + tid];
    float m = max_wave(ml.x);
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    // a part without keys (no sum) weighs nothing, whatever its output holds
    const float w = ml.y == 0.0f ? 0.0f : ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m);
    weight[tid] = ml.y == 0.0f ? -1.0f : w;
    float l = sum_wave(w * ml.y);
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    for (int s0 = rec;;) {
#pragma unroll
        for (int u = 0; u < kDeep; u++) {
            const float f = weight[(s0 + 16 * u) & 255];
            if (s0 + 16 * u < parts && f >= 0.0f) o += f * x[u];
        }
        s0 += 16 * kDeep;
        if (s0 - rec >= parts) break;
        load(s0);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = sum_rows(o[i]);
    if (lane < 16) sum[wave][lane] = o;
    __syncthreads();
    if (tid < 64) {
        const float *const t = reinterpret_cast<const float *>(sum);
        float y = (t[tid] + t[64 + tid]) + (t[128 + tid] + t[192 + tid]);
        y = l == 0.0f ? 0.0f : y / l;  // a row that sees no key
        if (gate) y *= sigmoid_ref(g);
        out[row * a.head_dim + d0 + tid] = y;
    }
}

// A 16-key half of a tile lies in one page. Other page sizes have the rows of every tile found a lane a key,
// and never share an operand between a query's halves: 16 requests of 4096 keys, pages of 16, 48 and 64 tokens, 16
// query heads: Q8_0, 4 heads of 256 37.5, 38.9 and 37.2 us for one row, 84.7, 93.6 and 84.9 for nine; F16 58.4, 60.9 and
// 58.1, 111.8, 116.7 and 112.0.
bool paged(const KvArgs &a) { return a.block_size % 16 == 0 && (a.block_size & (a.block_size - 1)) == 0; }
bool stacked(const KvArgs &a) { return paged(a) && a.heads / a.kv_heads * a.rows <= 8; }
// 16-row blocks of a wave. Two share each tile's way to halves, at two waves a SIMD for
// three: 16 requests of 8 rows, 4 heads of 128 a kv head, over 4096 keys 64.3 -> 55.4 us
// (two blocks), 4 of 17 rows over 16384 117.9 -> 109.8 (five blocks, one half idle); with
// three blocks it does not pay (70.7 -> 75.0), nor from 192 dims, where one wave a SIMD is
// left (256 dims, five blocks: 114 -> 136).
int blocks_of_wave(const KvArgs &a) {
    const int blocks = (a.heads / a.kv_heads * a.rows + 15) / 16;
    return a.fmt == kKvQ8 && paged(a) && a.head_dim <= 128 && blocks != 1 && blocks != 3 ? 2 : 1;
}
int pairs_of(const KvArgs &a) { return stacked(a) ? 8 : 16 * blocks_of_wave(a); }
int row_blocks(const KvArgs &a) {
    const int pairs = a.heads / a.kv_heads * a.rows, per = pairs_of(a);
    return (pairs + per - 1) / per;
}

AttnSplit attn_split(const KvArgs &a) {
    AttnSplit sp{};
    sp.row_blocks = row_blocks(a);
    sp.columns = sp.row_blocks * a.kv_heads;
    sp.group = a.heads / a.kv_heads;
    sp.group_inverse = sp.group == 1 ? 0 : (uint32_t)(((1ull << 32) + sp.group - 1) / sp.group);
    sp.target = 256 * waves_held(a.head_dim / 64, blocks_of_wave(a));
    sp.share = (float)sp.columns / (float)sp.target;
    sp.whole = (int64_t)sp.columns * a.requests >= 2 * sp.target;
    if (paged(a)) while ((16 << sp.page_shift) < a.block_size) sp.page_shift++;
    return sp;
}
// Most parts of a request, by its capacity.
int64_t most_parts(const KvArgs &a) {
    const int64_t tiles = ((int64_t)a.capacity - 1) / kTile + 1;
    return std::min<int64_t>(kMaxParts, (tiles - 1) / kWaves + 1);
}
// Workgroups, and records of requests in several parts: a part has more than half a
// chunk of tiles there, and a chunk is 1 / (2 target) of all tiles at the least.
int64_t most_items(const KvArgs &a, const AttnSplit &sp) {
    const int64_t columns = (int64_t)sp.columns * a.requests;
    return sp.whole ? columns : std::min(columns * most_parts(a), columns + 2 * sp.target);
}
int64_t most_records(const KvArgs &a, const AttnSplit &sp) {
    if (sp.whole || most_parts(a) == 1) return 0;
    const int64_t items = std::min((int64_t)sp.columns * a.requests * most_parts(a), (int64_t)4 * sp.target);
    return items * pairs_of(a);
}

}  // namespace

uint64_t kv_attention_scratch_bytes(const KvArgs &a) {
    const int64_t records = most_records(a, attn_split(a));  // outputs, {m, l}, then {parts, first record} of the requests
    return records ? (uint64_t)records * (a.head_dim + 2) * 4 + (uint64_t)a.requests * 8 : 0;
}

hipError_t launch_kv_attention(const float *q, int q_stride, const float *gate, int gate_stride, const void *kpool,
                               const void *vpool, const int32_t *table, float *out, const KvArgs &a, void *scratch,
                               const ModelDyn &dyn, hipStream_t s) {
    const AttnSplit sp = attn_split(a);
    const int64_t records = most_records(a, sp);
    float *part = static_cast<float *>(scratch);
    float2 *stats = records ? reinterpret_cast<float2 *>(part + records * a.head_dim) : nullptr;
    int2 *plan = records ? reinterpret_cast<int2 *>(stats + records) : nullptr;
    hipError_t err = hipSuccess;
    auto launch = [&](auto fmt, auto groups, auto stack, auto pages, auto blocks) {
        constexpr auto kernel = kv_attention_kernel<fmt(), groups(), stack(), pages(), blocks()>;
        constexpr uint32_t bytes = Layout<fmt(), groups(), stack(), pages(), blocks()>::total;
        if constexpr (bytes > 64 * 1024) {  // (a device's own setting)
            static std::once_flag once[64];
            int device = 0;
            (void)hipGetDevice(&device);
            std::call_once(once[device & 63], [] {
                (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                          (int)bytes);
            });
        }
        kernel<<<(uint32_t)most_items(a, sp), 64 * kWaves, bytes, s>>>(
            q, q_stride, gate, gate_stride, static_cast<const uint8_t *>(kpool), static_cast<const uint8_t *>(vpool), table,
            a, sp, part, stats, plan, out, dyn);
        err = hipGetLastError();
    };
    auto by_pages = [&](auto fmt, auto groups) {
        const std::true_type yes;
        const std::false_type no;
        const std::integral_constant<int, 1> one;
        if (!paged(a)) return launch(fmt, groups, no, no, one);
        if (stacked(a)) return launch(fmt, groups, yes, yes, one);
        if constexpr (fmt() == kKvQ8 && groups() <= 2) {
            if (blocks_of_wave(a) == 2) return launch(fmt, groups, no, yes, std::integral_constant<int, 2>{});
        }
        launch(fmt, groups, no, yes, one);
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
    if (err != hipSuccess || !records) return err;
    // A wave a row, or where a request can have many parts a workgroup each 64 dims: then what counts
    // is the records in flight. (us with the attention, a wave a row and a workgroup a row: 96 requests of
    // up to 6 parts, 8 heads of 128 a KV head, 91.5 and 94.5; 16 of 8 parts 42.1 and 42.3; 5 rows of 9
    // parts 14.6 and 13.8. 125 parts: a workgroup a row 69.3, each 64 dims 64.6.
    // The estimate goes by the tables' length: 517 and 1029 keys in tables of 131072 tokens take 12.6 and 14.3, in
    // tables that they fill 12.3 and 14.8.)
    const int64_t parts = std::min<int64_t>(most_parts(a), sp.target / ((int64_t)sp.columns * a.requests));
    if (parts > 32) {
        kv_attention_merge_kernel<<<dim3(a.rows * (a.head_dim / 64), a.heads, a.requests), 256, 0, s>>>(
            part, stats, plan, gate, gate_stride, out, a, sp.row_blocks, pairs_of(a));
        return hipGetLastError();
    }
    auto join = a.head_dim == 64    ? kv_attention_join_kernel<1>
                : a.head_dim == 128 ? kv_attention_join_kernel<2>
                : a.head_dim == 192 ? kv_attention_join_kernel<3>
                                    : kv_attention_join_kernel<4>;
    join<<<dim3((a.rows * a.heads + 3) / 4, a.requests), 256, 0, s>>>(part, stats, plan, gate, gate_stride, out, a,
                                                                      sp.row_blocks, pairs_of(a));
    return hipGetLastError();
}

}  // namespace yk

// ops_ragged.cpp — validation and dispatch of the ops over ragged batches
// (BATCH_PLAN, KV_APPEND_SLOTS, GDN_CONV, GDN_PROMPT, GDN_STEP), for plans and for
// the direct calls alike. Layouts: include/yuuka_hip.h.
#include <algorithm>
#include <initializer_list>

#include "kv.h"
#include "ops.h"
#include "ragged.h"

namespace yk {

namespace {

template <typename T>
T *at(const yuuka_op &op, int i) {
    return op.buf[i] ? reinterpret_cast<T *>(static_cast<uint8_t *>(op.buf[i]->ptr) + op.off[i]) : nullptr;
}

int clip(uint64_t v) { return (int)std::min<uint64_t>(v, 0x7fffffff); }
// A count as the direct calls' int32 gives it: what is negative there is refused as such.
int count(uint64_t v) { return (int64_t)v < 0 ? -1 : clip(v); }

// Buffer `buf` of an op, of which the call uses `bytes` (the whole of it: 0) and writes them or not.
struct Area {
    int buf;
    uint64_t bytes;
    bool written;
};

// Every area is there, aligned, and no written one overlaps another; `same` lists pairs that may be one
// buffer (and then start together).
yuuka_status check_areas(const yuuka_op &op, const char *what, std::initializer_list<Area> areas,
                         std::initializer_list<std::pair<int, int>> same = {}) {
    struct Span {
        uint64_t begin, end;
    };
    auto span = [&](const Area &a) {
        const uint64_t begin = reinterpret_cast<uint64_t>(op.buf[a.buf]->ptr) + op.off[a.buf];
        return Span{begin, begin + (a.bytes ? a.bytes : op.buf[a.buf]->bytes - op.off[a.buf])};
    };
    for (const Area &a : areas) {
        const yuuka_buffer *const b = op.buf[a.buf];
        if (!b || !b->ptr) return fail(YUUKA_ERR_INVALID_ARGUMENT, "%s: buffer %d is null", what, a.buf);
        if (op.off[a.buf] % 16 || op.off[a.buf] > b->bytes || a.bytes > b->bytes - op.off[a.buf])
            return fail(YUUKA_ERR_INVALID_ARGUMENT, "%s: buffer %d is too small, or its offset no multiple of 16", what,
                        a.buf);
    }
    for (const Area &a : areas)
        for (const Area &b : areas) {
            if (!a.written || a.buf == b.buf) continue;
            const Span x = span(a), y = span(b);
            if (x.begin >= y.end || y.begin >= x.end) continue;
            bool fine = false;
            for (const auto &p : same)
                fine = fine || (x.begin == y.begin && ((p.first == a.buf && p.second == b.buf) ||
                                                      (p.first == b.buf && p.second == a.buf)));
            if (!fine)
                return fail(YUUKA_ERR_INVALID_ARGUMENT, "%s: output buffer %d overlaps buffer %d", what, a.buf, b.buf);
        }
    return YUUKA_OK;
}

BatchArgs batch_args(const yuuka_op &op) {
    return BatchArgs{count(op.n[0]), count(op.n[1]), (int)op.u[0], (int)op.u[1]};
}

yuuka_status validate_batch_plan(const yuuka_op &op, uint64_t *ws) {
    const BatchArgs a = batch_args(op);
    yuuka_status st = batch_check(a);
    if (st != YUUKA_OK) return st;
    const uint64_t n = a.requests, rows = a.rows, entries = (a.capacity - 1) / a.block_size + 1;
    *ws = batch_plan_scratch_bytes(a);
    return check_areas(op, "batch plan",
                       {{0, 8 * n, false},
                        {1, 4 * n, false},
                        {2, 4 * n, false},
                        {3, 4 * n * entries, true},
                        {4, 0, false},
                        {5, 8, false},
                        {6, 4 * (n + 1), true},
                        {7, 8 * rows, true},
                        {8, 8 * rows, true},
                        {9, 4 * n, true},
                        {10, 8, true}},
                       {{2, 9}, {5, 10}});
}

yuuka_status slots_args(const yuuka_op &op, KvArgs *a) {
    *a = KvArgs{};
    a->kv_heads = count(op.n[0]);
    a->head_dim = count(op.n[2]);
    a->rows = count(op.n[4]);
    a->block_size = (int)op.u[0];
    a->capacity = a->requests = 1;
    a->rope_dim = (int)op.u[3];
    a->eps = op.f[1];
    const yuuka_status st = kv_check(a, op.u[2], false);
    if (st != YUUKA_OK) return st;
    uint64_t bytes[2] = {0, 0};
    for (int i = 0; i < 2; i++)
        if (op.buf[2 + i] && op.off[2 + i] <= op.buf[2 + i]->bytes) bytes[i] = op.buf[2 + i]->bytes - op.off[2 + i];
    a->pages = kv_pages(*a, bytes[0], bytes[1]);
    return YUUKA_OK;
}

yuuka_status validate_append_slots(const yuuka_op &op) {
    KvArgs a;
    yuuka_status st = slots_args(op, &a);
    if (st != YUUKA_OK) return st;
    if (op.n[3] != (uint64_t)a.kv_dim) return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV append by slot: row width");
    if ((a.rope_dim != 0) != (op.buf[6] != nullptr))
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV append by slot: a rotation needs its dimensions and its table");
    if (!a.pages) return fail(YUUKA_ERR_INVALID_ARGUMENT, "KV append by slot: pools of no page");
    const uint64_t bytes = (uint64_t)a.rows * a.kv_dim * 4;
    st = check_areas(op, "KV append by slot",
                     {{0, bytes, false}, {1, bytes, false}, {2, 0, true}, {3, 0, true}, {4, 8ull * a.rows, false}});
    if (st == YUUKA_OK && op.buf[5])
        st = check_areas(op, "KV append by slot", {{5, 4ull * a.head_dim, false}, {2, 0, true}, {3, 0, true}});
    if (st == YUUKA_OK && op.buf[6])
        st = check_areas(op, "KV append by slot",
                         {{6, (uint64_t)a.rows * (a.rope_dim / 2) * 8, false}, {2, 0, true}, {3, 0, true}});
    return st;
}

// The arguments of the three ops over recurrent states, whose pool is buffer `pool`.
yuuka_status ragged_args(const yuuka_op &op, bool conv, int pool, RaggedArgs *a) {
    *a = RaggedArgs{};
    a->requests = count(op.n[0]);
    a->rows = count(op.n[1]);
    a->groups = count(op.n[2]);
    a->heads = count(op.n[3]);
    a->head_dim = count(op.n[4]);
    a->stride = count(op.n[5]);
    a->kernel = (int)op.u[1];
    a->log_decay = op.u[2] != 0;
    a->scale = op.f[0];
    a->eps = op.f[1];
    const yuuka_status st = ragged_check(a, op.u[0], conv);
    if (st != YUUKA_OK) return st;
    if (!op.buf[pool] || op.off[pool] > op.buf[pool]->bytes)
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "GDN rows: the pool of states is null");
    a->states = clip((op.buf[pool]->bytes - op.off[pool]) / ragged_state_bytes(*a, conv));
    return YUUKA_OK;
}

uint64_t input_bytes(const RaggedArgs &a, uint64_t size) {
    return ((uint64_t)(a.rows - 1) * a.stride + a.channels) * size;
}

yuuka_status validate_conv(const yuuka_op &op) {
    RaggedArgs a;
    const yuuka_status st = ragged_args(op, true, 3, &a);
    if (st != YUUKA_OK) return st;
    const uint64_t size = ragged_element_bytes(op.u[0]);
    return check_areas(op, "GDN convolution",
                       {{0, (uint64_t)a.rows * a.channels * size, true},
                        {1, input_bytes(a, size), false},
                        {2, (uint64_t)a.channels * a.kernel * 4, false},
                        {3, 0, true},
                        {4, 4ull * (a.requests + 1), false},
                        {5, 8ull * a.requests, false}});
}

yuuka_status validate_delta(const yuuka_op &op, uint64_t *ws) {
    const bool step = op.code == YUUKA_EXT_OP_GDN_STEP;
    const char *const what = step ? "GDN step" : "GDN prompt";
    RaggedArgs a;
    yuuka_status st = ragged_args(op, false, 4, &a);
    if (st != YUUKA_OK) return st;
    if (step && (a.rows < a.requests || op.buf[5]))
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "GDN step: %d rows of %d requests, without offsets", a.rows, a.requests);
    if (a.log_decay ? op.buf[7] || op.buf[8] : !op.buf[7] || !op.buf[8])
        return fail(YUUKA_ERR_INVALID_ARGUMENT, "%s: dt and a come with alpha and beta of the projections, and only then", what);
    const uint64_t size = ragged_element_bytes(op.u[0]), out = (uint64_t)a.rows * a.heads * a.head_dim * size;
    const uint64_t coefficients = (uint64_t)a.rows * a.heads * 4;
    st = check_areas(op, what,
                     {{0, out, true},
                      {1, input_bytes(a, size), false},
                      {2, coefficients, false},
                      {3, coefficients, false},
                      {4, 0, true},
                      {6, 8ull * a.requests, false}});
    if (st == YUUKA_OK && !step)
        st = check_areas(op, what, {{0, out, true}, {4, 0, true}, {5, 4ull * (a.requests + 1), false}});
    if (st == YUUKA_OK && !a.log_decay)
        st = check_areas(op, what, {{0, out, true}, {4, 0, true}, {7, 4ull * a.heads, false}, {8, 4ull * a.heads, false}});
    if (st == YUUKA_OK && !step) *ws = gdn_prompt_scratch_bytes(a);
    return st;
}

}  // namespace

bool ragged_op(const yuuka_op &op) {
    return op.code >= YUUKA_EXT_OP_BATCH_PLAN && op.code <= YUUKA_EXT_OP_GDN_STEP;
}

yuuka_status validate_ragged_op(const yuuka_op &op, uint64_t *ws) {
    *ws = 0;
    switch (op.code) {
    case YUUKA_EXT_OP_BATCH_PLAN: return validate_batch_plan(op, ws);
    case YUUKA_EXT_OP_KV_APPEND_SLOTS: return validate_append_slots(op);
    case YUUKA_EXT_OP_GDN_CONV: return validate_conv(op);
    default: return validate_delta(op, ws);
    }
}

yuuka_status execute_ragged_op(const yuuka_op &op, const ExecCtx &ctx) {
    hipError_t err = hipSuccess;
    switch (op.code) {
    case YUUKA_EXT_OP_BATCH_PLAN: {
        const BatchBuffers b{at<const int32_t>(op, 0), at<const int32_t>(op, 1), at<const int32_t>(op, 2),
                             at<int32_t>(op, 3), at<const int32_t>(op, 4), at<const int32_t>(op, 5),
                             clip((op.buf[4]->bytes - op.off[4]) / 4), at<int32_t>(op, 6), at<int2>(op, 7),
                             at<int64_t>(op, 8), at<int32_t>(op, 9), at<int32_t>(op, 10)};
        err = launch_batch_plan(b, batch_args(op), ctx.ws, ctx.stream);
        break;
    }
    case YUUKA_EXT_OP_KV_APPEND_SLOTS: {
        KvArgs a;
        const yuuka_status st = slots_args(op, &a);
        if (st != YUUKA_OK) return st;
        err = launch_kv_append_slots(at<const float>(op, 0), at<const float>(op, 1), at<void>(op, 2), at<void>(op, 3),
                                     at<const int64_t>(op, 4), at<const float>(op, 5), at<const float2>(op, 6), a,
                                     ctx.stream);
        break;
    }
    case YUUKA_EXT_OP_GDN_CONV: {
        RaggedArgs a;
        const yuuka_status st = ragged_args(op, true, 3, &a);
        if (st != YUUKA_OK) return st;
        err = launch_gdn_ragged_conv(at<void>(op, 0), at<const void>(op, 1), op.u[0], at<const float>(op, 2),
                                     at<float>(op, 3), at<const int32_t>(op, 4), at<const int2>(op, 5), a, ctx.stream);
        break;
    }
    default: {
        RaggedArgs a;
        const yuuka_status st = ragged_args(op, false, 4, &a);
        if (st != YUUKA_OK) return st;
        const GdnRows b{at<void>(op, 0), at<const void>(op, 1), at<const float>(op, 2), at<const float>(op, 3),
                        at<const float>(op, 7), at<const float>(op, 8), at<float>(op, 4), at<const int32_t>(op, 5),
                        at<const int2>(op, 6)};
        err = op.code == YUUKA_EXT_OP_GDN_STEP ? launch_gdn_step(b, op.u[0], a, ctx.stream)
                                               : launch_gdn_prompt(b, op.u[0], a, ctx.ws, ctx.stream);
    }
    }
    if (err != hipSuccess) return fail(YUUKA_ERR_DEVICE, "op %u launch: %s", op.code, hip_error(err));
    return YUUKA_OK;
}

}  // namespace yk

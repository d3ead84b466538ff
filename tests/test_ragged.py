"""CPU checks of the calls over ragged batches: where rows and pages are
(ragged_addr.h and kv_addr.h compiled for the host), and the refusals of the
direct calls and plan ops, which are decided before anything is launched."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from yuuka_amd import hip

CSRC = Path(__file__).resolve().parent.parent / "yuuka_amd" / "csrc"

PROGRAM = r"""
#include "kv_addr.h"
#include "ragged_addr.h"
#include <cstdio>
#include <random>
#include <set>
#include <vector>

using namespace yk;

int main() {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    long bad = 0, fresh = 0;
    const int32_t edge[] = {INT32_MIN, -1, 0, 1, INT32_MAX, 1000000};
    for (int trial = 0; trial < 20000; trial++) {
        // whatever the offsets are, rows lie inside the arrays
        const int rows = pick(1, 300), n = pick(1, 9);
        std::vector<int32_t> off(n + 1);
        for (auto &o : off) o = pick(0, 3) ? pick(0, rows) : edge[pick(0, 5)];
        for (int j = 0; j < n; j++) {
            const RowRange r = row_range(off.data(), rows, j);
            if (r.begin < 0 || r.end < r.begin || r.end > rows) bad++;
        }
        // ascending ones: every row of a request, and chunk numbers that never meet
        off[0] = 0;
        for (int j = 0; j < n; j++) off[j + 1] = off[j] + (pick(0, 2) ? pick(0, 90) : 0);
        const int total = off[n] + pick(0, 5) + 1;
        std::set<int> seen;
        for (int j = 0; j < n; j++) {
            const RowRange r = row_range(off.data(), total, j);
            if (r.begin != off[j] || r.end != off[j + 1]) bad++;
            for (int c = 0; c < (r.end - r.begin + 15) / 16; c++) {
                const int number = first_chunk<16>(r.begin, j) + c;
                if (number < 0 || number >= chunk_numbers<16>(total, n) || !seen.insert(number).second) bad++;
                if (j + 1 < n && number >= first_chunk<16>(off[j + 1], j + 1)) bad++;
            }
        }
        // new pages: entries inside the table, each with a new row in it, none of them in use
        const int block = pick(1, 40), cap = pick(1, 400), entries = (cap - 1) / block + 1;
        const int64_t p = pick(0, 3) ? pick(0, cap) : edge[pick(0, 5)], count = pick(0, 3) ? pick(0, 200) : pick(0, 1) * 0x40000000;
        const int64_t blocks = pick(0, 3) ? pick(0, entries) : edge[pick(0, 5)];
        const PageNeed need = page_need(p, count, blocks, block, cap);
        if (need.fresh < 0 || need.first < 0 || (need.fresh && need.first + need.fresh > entries)) bad++;
        std::set<int> want;
        for (int64_t q = p < 0 ? 0 : p; q < cap && q < p + count; q++)
            if (q / block >= blocks) want.insert((int)(q / block));
        if ((int)want.size() != need.fresh) bad++;
        for (int i = 0; i < need.fresh; i++) bad += !want.count(need.first + i);
        fresh += need.fresh;
        // slots: inside the pool, or none
        KvLayout a;
        a.fmt = pick(0, 2);
        a.block_size = pick(1, 40);
        a.capacity = 1;
        a.kv_dim = 64 * pick(1, 16);
        a.pages = pick(1, 40);
        const int64_t tokens = (int64_t)a.pages * a.block_size, pool = kv_page_bytes(a) * a.pages;
        const int64_t far[] = {-1, tokens, tokens - 1, INT64_MIN, INT64_MAX, (int64_t)1 << 32, -((int64_t)1 << 32)};
        const int64_t slot = pick(0, 1) ? pick(0, (int)tokens - 1) : far[pick(0, 6)];
        int64_t row = -1, scales = -1, row2 = -2, scales2 = -2;
        const bool ok = kv_row_of_slot(a, slot, &row, &scales);
        if (ok != (slot >= 0 && slot < tokens)) bad++;
        if (!ok) continue;
        if (row < 0 || row + (a.fmt == kKvQ8 ? a.kv_dim : kv_token_bytes(a.fmt, a.kv_dim)) > pool) bad++;
        if (a.fmt == kKvQ8 && scales + a.kv_dim / 16 > pool) bad++;
        // the place that a table with that page gives
        a.capacity = a.block_size;
        const int32_t table[1] = {(int32_t)(slot / a.block_size)};
        if (!kv_slot(a, table, 0, slot % a.block_size, &row2, &scales2) || row2 != row || scales2 != scales) bad++;
    }
    KvLayout a{kKvF16, 16, 1, 1024, 1 << 20};  // past 32 bits
    int64_t row, scales;
    if (!kv_row_of_slot(a, ((int64_t)1 << 24) - 1, &row, &scales) || row + 2048 != kv_page_bytes(a) << 20) bad++;
    a.pages = INT32_MAX;
    if (!kv_row_of_slot(a, ((int64_t)INT32_MAX - 1) * 16 + 3, &row, &scales) || row != kv_page_bytes(a) * ((int64_t)INT32_MAX - 1) + 3 * 2048) bad++;
    printf("%d %ld\n", fresh > 10000, bad);
}
"""


def test_no_offset_or_slot_leads_outside(tmp_path):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "ragged.cpp"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(src), "-o", str(tmp_path / "ragged")], check=True)
    out = subprocess.run([str(tmp_path / "ragged")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["1", "0"]


WALK = r"""
#include "ragged_addr.h"
#include <cstdio>
#include <random>
#include <vector>

using namespace yk;

// The convolution's walk over the rows, wave by wave, as k_gdnrow.hip has it.
int main() {
    std::mt19937 rng(11);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    long bad = 0, front = 0;
    for (int trial = 0; trial < 20000; trial++) {
        const int n = pick(1, 8), early = pick(1, 7), run = pick(1, 33);
        std::vector<int32_t> off(n + 1);
        off[0] = pick(0, 1) ? 0 : pick(1, 120);  // a part of a batch: rows in front of it are nobody's
        for (int j = 0; j < n; j++) off[j + 1] = off[j] + (pick(0, 3) ? pick(0, 1) ? pick(0, 4) : pick(0, 90) : 0);
        const int rows = off[n] + pick(0, 40) + 1;
        std::vector<int> outs(rows, 0), windows(n, 0);
        for (int first = 0; first < rows; first += run) {
            const int last = first + run < rows ? first + run : rows;
            int row = first, j = 0, steps = 0;
            while (j < n && off[j + 1] <= row) j++;
            if (j == n) continue;
            RowRange r = row_range(off.data(), rows, j);
            bool fresh = true;
            for (;; row++) {
                if (++steps > run + early + 1) { bad++; break; }  // no further than the rows that it has
                bool end = false;
                while (row >= r.end) {
                    if (row >= last || ++j >= n) { end = true; break; }
                    r = row_range(off.data(), rows, j);
                    fresh = true;
                }
                if (end) break;
                const RowTurn turn = row_turn(r, row, first, last, early);
                if (turn == kRowDone) break;
                if (turn == kRowSkipped) continue;
                if (row < r.begin || row >= rows) { bad++; break; }
                if (fresh && row == r.begin) windows[j]++;
                else if (fresh && row - r.begin < early) bad++;  // needs inputs of the window
                fresh = false;
                outs[row]++;
            }
        }
        for (int row = 0; row < rows; row++) bad += outs[row] != (row >= off[0] && row < off[n]);
        for (int j = 0; j < n; j++) bad += windows[j] != (off[j + 1] > off[j]);
        front += off[0] > run;
    }
    printf("%d %ld\n", front > 5000, bad);
}
"""


def test_every_row_and_window_of_a_convolution_is_one_waves(tmp_path):
    """Whatever row a batch starts with: each of its rows is computed once, and each window read and written by one wave."""
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "walk.cpp"
    src.write_text(WALK)
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(src), "-o", str(tmp_path / "walk")], check=True)
    out = subprocess.run([str(tmp_path / "walk")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["1", "0"]


DISORDER = r"""
#include "ragged_addr.h"
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

using namespace yk;

// The 64-fold search of ragged_dev.h, all lanes at once.
template <typename F> int wave_first(int n, F &&after) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        int k = 0;
        while (k < 64 && !after((int)std::min<int64_t>(lo + (int64_t)step * (k + 1) - 1, hi - 1))) k++;
        if (k == 64) return hi;
        const int first = (int)std::min<int64_t>(lo + (int64_t)step * (k + 1) - 1, hi - 1);
        if (step == 1) return first;
        lo += step * k;
        hi = first;
    }
    return lo;
}

int main() {
    std::mt19937 rng(5);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    const int32_t edge[] = {INT32_MIN, -1, 0, 1, INT32_MAX, 1000000};
    long bad = 0, taken = 0;
    for (int trial = 0; trial < 20000; trial++) {
        const int n = pick(0, 9) ? pick(1, 9) : pick(60, 300), rows = pick(1, 300), early = pick(1, 7), run = pick(1, 33);
        std::vector<int32_t> off(n + 1);
        for (auto &o : off) o = pick(0, 5) ? pick(0, rows) : edge[pick(0, 5)];
        // the convolution: every wave ends, and takes rows of the arrays alone
        for (int first = 0; first < rows; first += run) {
            const int last = std::min(first + run, rows);
            int row = first, j = wave_first(n, [&](int i) { return off[i + 1] > row; });
            if (j >= n) continue;
            RowRange r = row_range(off.data(), rows, j);
            for (int steps = 0;; row++) {
                if (++steps > run + early + 1) { bad++; break; }
                bool end = false;
                while (row >= r.end) {
                    if (row >= last || ++j >= n) { end = true; break; }
                    r = row_range(off.data(), rows, j);
                }
                if (end) break;
                const RowTurn turn = row_turn(r, row, first, last, early);
                if (turn == kRowDone) break;
                if (turn == kRowSkipped) continue;
                if (row < 0 || row >= rows || row < r.begin) bad++;
                taken++;
            }
        }
        // the delta rule: chunks of rows of the arrays, whose places in the workspace are there
        const int numbers = chunk_numbers<64>(rows, n);
        for (int number = 0; number < numbers; number++) {
            const int j = wave_first(n, [&](int i) { return first_chunk<64>(row_range(off.data(), rows, i).begin, i) > number; }) - 1;
            if (j < 0) continue;
            const RowRange r = row_range(off.data(), rows, j);
            const int row0 = r.begin + (number - first_chunk<64>(r.begin, j)) * 64, some = std::min(64, r.end - row0);
            if (j >= n || row0 < 0 || (some > 0 && row0 + some > rows)) bad++;
        }
        for (int j = 0; j < n; j++) {
            const RowRange r = row_range(off.data(), rows, j);
            const int last = (r.end - r.begin + 63) / 64 - 1;
            if (last >= 0 && first_chunk<64>(r.begin, j) + last >= numbers) bad++;
        }
    }
    printf("%d %ld\n", taken > 100000, bad);
}
"""


def test_offsets_out_of_order_stay_inside(tmp_path):
    """Where offsets do not ascend results are undefined; every wave ends, and nothing outside the arrays is touched."""
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "disorder.cpp"
    src.write_text(DISORDER)
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(src), "-o", str(tmp_path / "disorder")], check=True)
    out = subprocess.run([str(tmp_path / "disorder")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["1", "0"]


# ------------------------------------------------------------- refusals
# Handles as internal.h lays them out, over memory that nothing reads: a refused call
# launches nothing.

class _Handle(C.Structure):
    _fields_ = [("dev", C.c_void_p), ("ptr", C.c_void_p), ("bytes", C.c_uint64)]


class _Stream(C.Structure):
    _fields_ = [("dev", C.c_void_p), ("stream", C.c_void_p), ("areas", C.c_uint64 * 4)]


class _Mem:
    made = 0

    def __init__(self, nbytes):
        _Mem.made += 1
        self.handle = _Handle(None, _Mem.made << 40, nbytes)  # apart from every other
        self.ptr = C.c_void_p(C.addressof(self.handle))


# 2 requests of 5 rows in all; 2 groups, 4 heads of 64: 512 channels
ROWS, CH, HEADS, DIM = 5, 512, 4, 64
KVD = 256
BUFFERS = {
    "batch_plan": [("positions", 16), ("counts", 8), ("blocks", 8), ("table", 2 * 7 * 4), ("free_pages", 4), ("pool", 8),
                   ("offsets", 12), ("row_info", 8 * ROWS), ("slots", 8 * ROWS), ("blocks_out", 8), ("pool_out", 8)],
    "kv_append_slots": [("k", ROWS * KVD * 4), ("v", ROWS * KVD * 4), ("kpool", 16 * KVD * 2), ("vpool", 16 * KVD * 2),
                        ("slots", 8 * ROWS), ("k_norm", 128 * 4), ("rope", ROWS * 32 * 8)],
    "gdn_conv": [("out", ROWS * CH * 2), ("x", ROWS * CH * 2), ("weight", CH * 4 * 4), ("windows", CH * 3 * 4),
                 ("offsets", 12), ("slots", 16)],
    "gdn_prompt": [("out", ROWS * HEADS * DIM * 2), ("qkv", ROWS * CH * 2), ("alpha", ROWS * HEADS * 4),
                   ("beta", ROWS * HEADS * 4), ("dt", HEADS * 4), ("a", HEADS * 4), ("states", HEADS * DIM * DIM * 4),
                   ("offsets", 12), ("slots", 16)],
    "gdn_step": [("out", ROWS * HEADS * DIM * 2), ("qkv", ROWS * CH * 2), ("alpha", ROWS * HEADS * 4),
                 ("beta", ROWS * HEADS * 4), ("dt", HEADS * 4), ("a", HEADS * 4), ("states", HEADS * DIM * DIM * 4),
                 ("slots", 16)],
}
OUTPUTS = dict(batch_plan=("table", "offsets", "row_info", "slots", "blocks_out", "pool_out"),
               kv_append_slots=("kpool", "vpool"), gdn_conv=("out", "windows"), gdn_prompt=("out", "states"),
               gdn_step=("out", "states"))
# buffers that may hold less (pools of states: then no slot is inside) or nothing
OPTIONAL = {("batch_plan", "free_pages"), ("gdn_conv", "windows"), ("gdn_prompt", "states"), ("gdn_step", "states")}
GDN = dict(dtype=hip.F16, requests=2, rows=ROWS, groups=2, heads=HEADS, head_dim=DIM)


def _params(name, **change):
    if name == "batch_plan":
        return hip.batch_params(**{**dict(requests=2, rows=ROWS, block_size=16, capacity=100), **change})
    if name == "kv_append_slots":
        return hip.kv_params(**{**dict(dtype=hip.F16, block_size=16, capacity=0, kv_heads=2, head_dim=128, rows=ROWS,
                                       requests=0, rope_dim=64), **change})
    return hip.gdn_params(**{**GDN, **change})


def _memory(name):
    return {b: _Mem(n) for b, n in BUFFERS[name]}


def _call(name, m, p, stream=None):
    raw = stream or _Stream()
    bufs = [m[b].ptr if m.get(b) is not None else None for b, _ in BUFFERS[name]]
    return getattr(hip.lib(), f"yuuka_{name}")(C.c_void_p(C.addressof(raw)), *bufs, C.byref(p), None)


SHAPES = [("batch_plan", c, hip.INVALID_ARGUMENT) for c in (
    dict(requests=0), dict(requests=-1), dict(requests=65536), dict(rows=0), dict(rows=-4), dict(rows=(1 << 30) + 1),
    dict(block_size=0), dict(block_size=-16), dict(block_size=(1 << 20) + 1), dict(capacity=0), dict(capacity=-1))]
SHAPES += [("kv_append_slots", c, s) for c, s in (
    (dict(dtype=hip.Q4_K), hip.UNSUPPORTED), (dict(dtype=hip.BF16), hip.UNSUPPORTED), (dict(head_dim=96), hip.UNSUPPORTED),
    (dict(block_size=0), hip.INVALID_ARGUMENT), (dict(rows=0), hip.INVALID_ARGUMENT), (dict(rows=-1), hip.INVALID_ARGUMENT),
    (dict(rows=1 << 29), hip.INVALID_ARGUMENT), (dict(kv_heads=0), hip.INVALID_ARGUMENT),
    (dict(kv_heads=-2), hip.INVALID_ARGUMENT), (dict(rope_dim=-2), hip.INVALID_ARGUMENT),
    (dict(rope_dim=3), hip.INVALID_ARGUMENT), (dict(rope_dim=130), hip.INVALID_ARGUMENT),
    (dict(rope_dim=0), hip.INVALID_ARGUMENT))]
SHAPES += [(name, c, s) for name in ("gdn_conv", "gdn_prompt", "gdn_step") for c, s in (
    (dict(dtype=hip.Q8_0), hip.UNSUPPORTED), (dict(dtype=99), hip.UNSUPPORTED), (dict(head_dim=32), hip.UNSUPPORTED),
    (dict(head_dim=256), hip.UNSUPPORTED), (dict(head_dim=-64), hip.UNSUPPORTED), (dict(requests=0), hip.INVALID_ARGUMENT),
    (dict(requests=-2), hip.INVALID_ARGUMENT), (dict(requests=65536), hip.INVALID_ARGUMENT),
    (dict(rows=0), hip.INVALID_ARGUMENT), (dict(rows=-1), hip.INVALID_ARGUMENT), (dict(rows=(1 << 30) + 1), hip.INVALID_ARGUMENT),
    (dict(groups=0), hip.INVALID_ARGUMENT), (dict(groups=3), hip.INVALID_ARGUMENT), (dict(heads=0), hip.INVALID_ARGUMENT),
    (dict(heads=5), hip.INVALID_ARGUMENT), (dict(heads=1026), hip.INVALID_ARGUMENT),
    (dict(row_stride=CH - 8), hip.INVALID_ARGUMENT), (dict(row_stride=CH + 4), hip.INVALID_ARGUMENT),
    (dict(row_stride=-CH), hip.INVALID_ARGUMENT))]
SHAPES += [("gdn_conv", dict(kernel=k), hip.UNSUPPORTED) for k in (1, 0, -4, 9)]
SHAPES += [("gdn_step", dict(rows=1), hip.INVALID_ARGUMENT)]
SHAPES += [(n, dict(log_decay=True), hip.INVALID_ARGUMENT) for n in ("gdn_prompt", "gdn_step")]  # with dt and a


@pytest.mark.parametrize("name,change,status", SHAPES)
def test_direct_calls_refuse_shapes(name, change, status):
    assert _call(name, _memory(name), _params(name, **change)) == status
    assert hip.lib().yuuka_last_error()


@pytest.mark.parametrize("name,buf", [(n, b) for n in BUFFERS for b, _ in BUFFERS[n]])
def test_direct_calls_refuse_missing_and_short_buffers(name, buf):
    m = _memory(name)
    if (name, buf) not in OPTIONAL:
        m[buf].handle.bytes -= 1
        assert _call(name, m, _params(name)) == hip.INVALID_ARGUMENT
    m = _memory(name)
    m[buf] = None
    if buf != "k_norm":
        assert _call(name, m, _params(name)) == hip.INVALID_ARGUMENT
        m[buf] = _Mem(1 << 20)
        m[buf].handle.ptr = None  # freed
        assert _call(name, m, _params(name)) == hip.INVALID_ARGUMENT


@pytest.mark.parametrize("name", sorted(BUFFERS))
def test_null_streams_and_parameters(name):
    L, m = hip.lib(), _memory(name)
    bufs = [m[b].ptr for b, _ in BUFFERS[name]]
    fn = getattr(L, f"yuuka_{name}")
    assert fn(None, *bufs, C.byref(_params(name)), None) == hip.INVALID_ARGUMENT
    assert fn(C.c_void_p(C.addressof(_Stream())), *bufs, None, None) == hip.INVALID_ARGUMENT


@pytest.mark.parametrize("name,out,other", [(n, o, b) for n in BUFFERS for o in OUTPUTS[n] for b, _ in BUFFERS[n] if b != o])
def test_outputs_may_not_overlap(name, out, other):
    m = _memory(name)
    for shift in (0, -4) if (out, other) not in (("blocks_out", "blocks"), ("pool_out", "pool")) else (-4,):
        m[out].handle.ptr = m[other].handle.ptr + shift
        assert _call(name, m, _params(name)) == hip.INVALID_ARGUMENT
        assert b"overlaps" in hip.lib().yuuka_last_error()


@pytest.mark.parametrize("name", sorted(BUFFERS))
def test_buffers_of_another_device_are_refused(name):
    one, two = C.c_int32(0), C.c_int32(1)  # yuuka_device starts with its index
    for moved, _ in BUFFERS[name]:
        m = _memory(name)
        for b in m.values():
            b.handle.dev = C.addressof(one)
        m[moved].handle.dev = C.addressof(two)
        assert _call(name, m, _params(name), _Stream(dev=C.addressof(one))) == hip.INVALID_ARGUMENT
        assert b"device 1" in hip.lib().yuuka_last_error()


# -------------------------------------------------------------- plan ops

class _Plan:
    """A plan that only records: it is never executed."""

    def __init__(self):
        p = C.c_void_p()
        self.dev = C.create_string_buffer(8192)
        hip.check(hip.lib().yuuka_plan_create(C.addressof(self.dev), C.byref(p)), "plan_create")
        self.ptr = p

    def add(self, name, bufs, n, u, f=(), offs=None):
        op = hip.yuuka_op()
        op.code = hip.OP[name]
        for i, b in enumerate(bufs):
            op.buf[i] = None if b is None else b.ptr.value
        for i, v in (offs or {}).items():
            op.off[i] = v
        for what, values in ((op.n, n), (op.u, u), (op.f, f)):
            for i, v in enumerate(values):
                what[i] = v
        return hip.lib().yuuka_plan_add(self.ptr, C.byref(op))


def _op(name):
    """A plan op as it is accepted: buffers, n, u."""
    direct = name.lower()
    m = _memory(direct)
    b = [m[x] for x, _ in BUFFERS[direct]]
    if name == "BATCH_PLAN":
        return b, [2, ROWS], [16, 100]
    if name == "KV_APPEND_SLOTS":
        return b, [2, 0, 128, KVD, ROWS], [16, 0, hip.F16, 64]
    n = [2, ROWS, 2, HEADS, DIM, 0]
    if name == "GDN_CONV":
        return b, n, [hip.F16, 4]
    b = [m["out"], m["qkv"], m["alpha"], m["beta"], m["states"], m.get("offsets"), m["slots"], m["dt"], m["a"]]
    return b, n, [hip.F16, 0, 0]


NAMES = ["BATCH_PLAN", "KV_APPEND_SLOTS", "GDN_CONV", "GDN_PROMPT", "GDN_STEP"]


@pytest.mark.parametrize("name", NAMES)
def test_plan_ops(name):
    plan = _Plan()
    bufs, n, u = _op(name)
    assert plan.add(name, bufs, n, u, f=[1.0, 1e-6]) == hip.OK
    for i, b in enumerate(bufs):
        if b is None or (name, i) in (("KV_APPEND_SLOTS", 5),):
            continue
        gone = list(bufs)
        gone[i] = None
        assert plan.add(name, gone, n, u) == hip.INVALID_ARGUMENT, i
        # an offset takes from the buffer's end, and is a multiple of 16
        assert plan.add(name, bufs, n, u, offs={i: 8}) == hip.INVALID_ARGUMENT, i
        assert plan.add(name, bufs, n, u, offs={i: 1 << 40}) == hip.INVALID_ARGUMENT, i
        b.handle.bytes += 32
        assert plan.add(name, bufs, n, u, offs={i: 32}) == hip.OK, i
    for i in (0, 1) if name != "KV_APPEND_SLOTS" else (0, 4):  # counts that do not fit 32 bits
        assert plan.add(name, bufs, [(1 << 40) if k == i else v for k, v in enumerate(n)], u) != hip.OK
        assert plan.add(name, bufs, [(1 << 64) - 5 if k == i else v for k, v in enumerate(n)], u) != hip.OK


def test_a_step_takes_no_offsets():
    bufs, n, u = _op("GDN_STEP")
    bufs[5] = _Mem(12)
    assert _Plan().add("GDN_STEP", bufs, n, u) == hip.INVALID_ARGUMENT


def test_the_key_rows_width():
    bufs, n, u = _op("KV_APPEND_SLOTS")
    n[3] += 1
    assert _Plan().add("KV_APPEND_SLOTS", bufs, n, u) == hip.INVALID_ARGUMENT

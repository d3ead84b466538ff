"""CPU checks of the paged key/value cache: page addressing (kv_addr.h compiled
for the host) and the refusals of the direct calls and plan ops, which are
decided before anything is launched."""
import ctypes as C
import gc
import shutil
import subprocess
import weakref
from dataclasses import replace
from pathlib import Path
from types import SimpleNamespace

import pytest

from yuuka_amd import hip
from yuuka_amd import model as Mdl

CSRC = Path(__file__).resolve().parent.parent / "yuuka_amd" / "csrc"

PROGRAM = r"""
#include "kv_addr.h"
#include <cstdio>
#include <map>
#include <random>
#include <vector>

using namespace yk;

int main() {
    std::mt19937 rng(5);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    long inside = 0, dropped = 0, bad = 0;
    for (int trial = 0; trial < 4000; trial++) {
        KvLayout a;
        a.fmt = pick(0, 2);
        a.block_size = pick(1, 40);
        a.capacity = trial % 7 ? pick(1, 300) : pick(1, 5);
        a.kv_dim = 64 * pick(1, 16);
        a.pages = pick(1, 40);
        const int requests = pick(1, 3), blocks = kv_table_blocks(a);
        if ((int64_t)blocks * a.block_size < a.capacity || (int64_t)(blocks - 1) * a.block_size >= a.capacity) bad++;
        // entries inside, on and outside the pool's borders; canaries around the table
        std::vector<int32_t> table(requests * blocks + 2, 0x7eadbeef);
        for (int i = 0; i < requests * blocks; i++) {
            const int edge[] = {-1, a.pages, a.pages - 1, 0, INT32_MIN, INT32_MAX};
            table[i + 1] = pick(0, 2) ? pick(0, a.pages - 1) : edge[pick(0, 5)];
        }
        const int64_t pool = kv_page_bytes(a) * a.pages, row_bytes = a.fmt == kKvQ8 ? a.kv_dim : kv_token_bytes(a.fmt, a.kv_dim);
        std::map<int64_t, int64_t> taken;  // byte runs by start, of distinct (page, token) pairs
        for (int j = 0; j < requests; j++)
            for (int64_t p : {(int64_t)-1, (int64_t)INT32_MIN - 5, (int64_t)0, (int64_t)a.capacity - 1, (int64_t)a.capacity,
                              (int64_t)INT32_MAX + 9, (int64_t)pick(0, a.capacity - 1)}) {
                int64_t row = -1, scales = -1;
                const bool ok = kv_slot(a, table.data() + 1, j, p, &row, &scales);
                const bool within = p >= 0 && p < a.capacity;
                const int page = within ? table[1 + j * blocks + (int)(p / a.block_size)] : -1;
                if (ok != (within && page >= 0 && page < a.pages)) bad++;
                if (!ok) { dropped++; continue; }
                inside++;
                if (row < 0 || row + row_bytes > pool || row % 4) bad++;
                if (a.fmt == kKvQ8 && (scales < row || scales + a.kv_dim / 16 > pool || scales % 4)) bad++;
                if (row / kv_page_bytes(a) != page) bad++;
                if (a.fmt == kKvQ8 && (scales + a.kv_dim / 16 - 1) / kv_page_bytes(a) != page) bad++;
            }
    }
    // a page's rows and scales cover it once
    for (int fmt = 0; fmt < 3; fmt++) {
        KvLayout a{fmt, 7, 21, 192, 3};
        int32_t table[3] = {2, 0, 1};
        std::vector<int> hits(kv_page_bytes(a) * 3);
        for (int p = 0; p < 21; p++) {
            int64_t row, scales;
            if (!kv_slot(a, table, 0, p, &row, &scales)) bad++;
            for (int64_t i = 0; i < (fmt == kKvQ8 ? 192 : kv_token_bytes(fmt, 192)); i++) hits[row + i]++;
            if (fmt == kKvQ8) for (int i = 0; i < 12; i++) hits[scales + i]++;
        }
        for (int h : hits) bad += h != 1;
    }
    // offsets past 32 bits
    KvLayout a{kKvQ8, 16, 1 << 24, 1024, 1 << 20};
    std::vector<int32_t> table(kv_table_blocks(a), (1 << 20) - 1);
    int64_t row, scales;
    if (!kv_slot(a, table.data(), 0, (1 << 24) - 1, &row, &scales) || scales + 64 != kv_page_bytes(a) << 20) bad++;
    printf("%ld %ld %ld\n", inside > 5000, dropped > 5000, bad);
}
"""


def test_no_table_or_position_leads_outside_the_pool(tmp_path):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "addr.cpp"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(src), "-o", str(tmp_path / "addr")], check=True)
    out = subprocess.run([str(tmp_path / "addr")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["1", "1", "0"]


ALIGNMENT = r"""
#include "kv_addr.h"
#include <cstdio>
#include <initializer_list>

using namespace yk;

int main() {
    int64_t common = 0;  // of all rows' and scales' offsets
    auto fold = [&](int64_t x) {
        for (int64_t y = common; y;) { const int64_t r = x % y; x = y; y = r; }
        common = x;
    };
    const int32_t table[] = {1, 2, 3, 4};
    for (int fmt : {kKvF32, kKvF16, kKvQ8})
        for (int kv_dim = 64; kv_dim <= 512; kv_dim += 64)
            for (int block = 1; block <= 17; block++) {
                KvLayout a{fmt, block, 4 * block, kv_dim, 5};
                for (int p = 0; p < a.capacity; p++) {
                    int64_t row, scales;
                    if (!kv_slot(a, table, 0, p, &row, &scales)) return 1;
                    fold(row);
                    if (fmt == kKvQ8) fold(scales);
                }
            }
    printf("%lld %d\n", (long long)common, kKvAlign);
}
"""


def test_the_alignment_of_rows(tmp_path):
    """What the read back's loads may ask for is what every row has, and no more."""
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "align.cpp"
    src.write_text(ALIGNMENT)
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", f"-I{CSRC}", str(src), "-o", str(tmp_path / "align")], check=True)
    out = subprocess.run([str(tmp_path / "align")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["4", "4"]


# Handles as the library lays them out (internal.h), over no device memory: a
# call that gets past its checks would be refused by the missing device, with
# another status than the ones asked for here.

class _Handle(C.Structure):
    _fields_ = [("dev", C.c_void_p), ("ptr", C.c_void_p), ("bytes", C.c_uint64)]


class _Stream(C.Structure):
    _fields_ = [("dev", C.c_void_p), ("stream", C.c_void_p), ("areas", C.c_uint64 * 4)]


class _Mem:
    def __init__(self, nbytes):
        self.handle = _Handle(None, 4096, nbytes)
        self.ptr = C.c_void_p(C.addressof(self.handle))


GOOD = dict(dtype=hip.Q8_0, block_size=16, capacity=100, kv_heads=2, head_dim=128, rows=3, requests=2)
KVD, PAGES = 256, 14


def _memory(dtype=hip.Q8_0, heads=4, gated=False):
    token = {hip.F32: 4 * KVD, hip.F16: 2 * KVD, hip.Q8_0: KVD * 34 // 32}[dtype]
    return dict(k=_Mem(6 * KVD * 4), v=_Mem(6 * KVD * 4), kpool=_Mem(PAGES * 16 * token), vpool=_Mem(PAGES * 16 * token),
                table=_Mem(2 * 7 * 4), positions=_Mem(16), norm=_Mem(128 * 4), rope=_Mem(6 * 32 * 8),
                q=_Mem(6 * heads * 128 * 4 * (2 if gated else 1)), out=_Mem(6 * heads * 128 * 4))


def _call(name, m, p):
    """The status of a direct call on a stream without a device."""
    raw = _Stream()
    s = C.c_void_p(C.addressof(raw))
    g = lambda n: m[n].ptr if m.get(n) is not None else None  # noqa: E731
    L = hip.lib()
    if name == "append":
        return L.yuuka_kv_append(s, g("k"), g("v"), g("kpool"), g("vpool"), g("table"), g("positions"), g("norm"),
                                 g("rope"), C.byref(p), None)
    if name == "read":
        return L.yuuka_kv_read(s, g("k"), g("v"), g("kpool"), g("vpool"), g("table"), g("positions"), C.byref(p), None)
    return L.yuuka_attn_decode(s, g("out"), g("q"), g("kpool"), g("vpool"), g("table"), g("positions"), C.byref(p), None)


SHAPES = [
    (dict(dtype=hip.Q4_K), hip.UNSUPPORTED), (dict(dtype=99), hip.UNSUPPORTED),
    (dict(head_dim=32), hip.UNSUPPORTED), (dict(head_dim=96), hip.UNSUPPORTED), (dict(head_dim=320), hip.UNSUPPORTED),
    (dict(head_dim=0), hip.UNSUPPORTED), (dict(head_dim=-64), hip.UNSUPPORTED),
    (dict(block_size=0), hip.INVALID_ARGUMENT), (dict(block_size=-16), hip.INVALID_ARGUMENT),
    (dict(capacity=0), hip.INVALID_ARGUMENT), (dict(capacity=-5), hip.INVALID_ARGUMENT),
    (dict(requests=0), hip.INVALID_ARGUMENT), (dict(requests=65536), hip.INVALID_ARGUMENT),
    (dict(rows=0), hip.INVALID_ARGUMENT), (dict(rows=-1), hip.INVALID_ARGUMENT),
    (dict(rows=1 << 29), hip.INVALID_ARGUMENT), (dict(request_rows=-3), hip.INVALID_ARGUMENT),
    (dict(kv_heads=0), hip.INVALID_ARGUMENT), (dict(kv_heads=5000), hip.INVALID_ARGUMENT),
    (dict(displacement=-(1 << 31)), hip.INVALID_ARGUMENT), (dict(displacement=(1 << 31) - 1), hip.INVALID_ARGUMENT),
]


@pytest.mark.parametrize("name", ["append", "read", "attn"])
@pytest.mark.parametrize("change,status", SHAPES)
def test_direct_calls_refuse_shapes(name, change, status):
    extra = dict(heads=4) if name == "attn" else {}
    m = _memory()
    m.update(norm=None, rope=None)
    assert _call(name, m, hip.kv_params(**{**GOOD, **extra, **change})) == status
    assert hip.lib().yuuka_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(dtype=hip.F32), hip.UNSUPPORTED), (dict(heads=0), hip.INVALID_ARGUMENT), (dict(heads=3), hip.INVALID_ARGUMENT),
    (dict(heads=-4), hip.INVALID_ARGUMENT), (dict(heads=65538), hip.INVALID_ARGUMENT),
    (dict(rows=4097), hip.INVALID_ARGUMENT)])
def test_attention_refuses_heads_and_rows(change, status):
    assert _call("attn", _memory(), hip.kv_params(**{**GOOD, "heads": 4, **change})) == status


@pytest.mark.parametrize("change,words", [
    (dict(heads=2 * 257), b"514 heads over 2 KV heads"),
    (dict(requests=65535, rows=4096, heads=64), b"in one call"),        # 65535 * 2 * 4096 * 32 / 8 workgroups
    (dict(requests=4097, rows=512, heads=32), b"in one call")])         # 2^23 and 2048 more
def test_attention_refuses_more_than_one_launch(change, words):
    m = _memory()
    for b in m.values():  # no buffer is too small
        b.handle.bytes = 1 << 60
    assert _call("attn", m, hip.kv_params(**{**GOOD, **change})) == hip.INVALID_ARGUMENT
    assert words in hip.lib().yuuka_last_error()


@pytest.mark.parametrize("name,small", [(n, b) for n, bs in dict(
    append=("k", "v", "kpool", "vpool", "table", "positions", "norm", "rope"),
    read=("k", "v", "kpool", "vpool", "table", "positions"),
    attn=("q", "out", "kpool", "vpool", "table", "positions")).items() for b in bs])
def test_direct_calls_refuse_missing_and_short_buffers(name, small):
    p = hip.kv_params(**GOOD, heads=4, rope_dim=64)
    m = _memory()
    # a pool may hold fewer pages than the tables could name, but not less than one
    m[small].handle.bytes = 16 * (KVD * 34 // 32) - 1 if small in ("kpool", "vpool") else m[small].handle.bytes - 1
    assert _call(name, m, p) == hip.INVALID_ARGUMENT
    m = _memory()
    m[small] = None
    if (name, small) not in (("append", "norm"), ("read", "positions")):
        assert _call(name, m, p) == hip.INVALID_ARGUMENT


def test_a_rotation_needs_its_table_and_its_width():
    m = _memory()
    assert _call("append", m, hip.kv_params(**GOOD, rope_dim=0)) == hip.INVALID_ARGUMENT   # a table, no width
    for width in (-2, 3, 130, 256):
        assert _call("append", m, hip.kv_params(**GOOD, rope_dim=width)) == hip.INVALID_ARGUMENT
    m["rope"] = None
    assert _call("append", m, hip.kv_params(**GOOD, rope_dim=64)) == hip.INVALID_ARGUMENT  # a width, no table


def test_the_gate_doubles_the_query_rows():
    assert _call("attn", _memory(), hip.kv_params(**GOOD, heads=4, gated=True)) == hip.INVALID_ARGUMENT


def test_buffers_of_another_device_are_refused():
    # yuuka_device starts with its index
    one, two = C.c_int32(0), C.c_int32(1)
    for name, moved in (("append", "vpool"), ("read", "table"), ("attn", "positions")):
        m = _memory()
        m.update(norm=None, rope=None)
        raw = _Stream(dev=C.addressof(one))
        for b in m.values():
            if b is not None:
                b.handle.dev = C.addressof(one)
        m[moved].handle.dev = C.addressof(two)
        s, p = C.c_void_p(C.addressof(raw)), hip.kv_params(**GOOD, heads=4)
        g = lambda n: m[n].ptr  # noqa: E731
        L = hip.lib()
        st = (L.yuuka_kv_append(s, g("k"), g("v"), g("kpool"), g("vpool"), g("table"), g("positions"), None, None,
                                C.byref(p), None) if name == "append" else
              L.yuuka_kv_read(s, g("k"), g("v"), g("kpool"), g("vpool"), g("table"), g("positions"), C.byref(p), None)
              if name == "read" else
              L.yuuka_attn_decode(s, g("out"), g("q"), g("kpool"), g("vpool"), g("table"), g("positions"), C.byref(p),
                                  None))
        assert st == hip.INVALID_ARGUMENT
        assert b"device 1" in L.yuuka_last_error()


@pytest.mark.parametrize("dtype,token", [(hip.F32, 1024), (hip.F16, 512), (hip.Q8_0, 272)])
def test_page_bytes(dtype, token):
    assert hip.kv_page_bytes(hip.kv_params(**{**GOOD, "dtype": dtype})) == 16 * token
    assert hip.kv_page_bytes(hip.kv_params(**{**GOOD, "dtype": dtype, "head_dim": 80})) == 0
    assert hip.kv_page_bytes(hip.kv_params(**{**GOOD, "dtype": hip.Q6_K})) == 0


# ---------------------------------------------------------------- plan ops

class _Plan:
    """A plan that only records: it is never executed."""

    def __init__(self):
        p = C.c_void_p()
        self.dev = C.create_string_buffer(8192)
        hip.check(hip.lib().yuuka_plan_create(C.addressof(self.dev), C.byref(p)), "plan_create")
        self.ptr = p

    def add(self, name, bufs, n, u, f=(), offs=(), flags=0):
        op = hip.yuuka_op()
        op.code, op.flags = OPS[name], flags
        for i, b in enumerate(bufs):
            op.buf[i] = None if b is None else b.ptr.value
        for i, v in enumerate(offs):
            op.off[i] = v
        for i, v in enumerate(n):
            op.n[i] = v
        for i, v in enumerate(u):
            op.u[i] = v
        for i, v in enumerate(f):
            op.f[i] = v
        return hip.lib().yuuka_plan_add(self.ptr, C.byref(op))


OPS = dict(hip.OP, KV_WRITE_PAGED=26, ATTENTION_PAGED=27)
_U = lambda low=0, requests=2, stride=0: low | requests << 8 | stride << 20  # noqa: E731


def _ops(m):
    """The ops over Q8_0 pools, each as it is accepted: (name, buffers, n, u, flags)."""
    pos = m["positions"]

    def bufs(*b):
        return list(b) + [None] * (15 - len(b)) + [pos]

    n, au = [2, 4, 128, KVD, 3, 0], [16, 100, hip.Q8_0]
    return {
        "KV_APPEND": (bufs(m["k"], m["v"], m["kpool"], m["vpool"], m["table"], m["norm"], m["rope"]),
                      [2, 0, 128, KVD, 3, 0], au + [_U(64)], hip.FLAG_OWN_POS),
        "KV_READ": (bufs(m["kpool"], m["vpool"], m["k"], m["v"], m["table"]), [2, 0, 128, KVD, 3, 0], au + [_U()], 0),
        "ATTN_DECODE": (bufs(m["q"], m["kpool"], m["vpool"], m["out"], m["table"]), n, au + [_U(0)], hip.FLAG_OWN_POS),
        "ATTN_VERIFY": (bufs(_Mem(6 * 4 * 256 * 4), m["k"], m["v"], m["kpool"], m["vpool"], m["out"], m["table"],
                             m["norm"], m["norm"], m["rope"]), n, au + [_U(64)], hip.FLAG_OWN_POS),
        "KV_WRITE_PAGED": ([m["k"], m["v"], m["kpool"], m["vpool"], m["table"]], [KVD], au, 0),
        "KV_WRITE_BATCH_PAGED": ([m["k"], m["v"], m["kpool"], m["vpool"], m["table"]], [KVD, 6], au, 0),
        "ATTENTION_PAGED": ([m["q"], m["kpool"], m["vpool"], m["out"], None, m["table"]], [2, 4, 128, KVD, 100],
                            au + [1], 0),
        "ATTENTION_PREFILL_PAGED": ([m["q"], m["kpool"], m["vpool"], m["out"], m["table"]], [2, 4, 128, KVD, 6, 0],
                                    au + [1], 0),
    }


@pytest.mark.parametrize("name", sorted(_ops(_memory())))
def test_plan_ops_over_q8_0_pools(name):
    plan = _Plan()
    bufs, n, u, flags = _ops(_memory())[name]
    assert plan.add(name, bufs, n, u, flags=flags) == hip.OK, hip.lib().yuuka_last_error()
    # a width that is not the heads', an unknown dtype, no capacity
    wrong = list(n)
    wrong[0 if "WRITE" in name else 3] += 32
    assert plan.add(name, bufs, wrong, u, flags=flags) == hip.INVALID_ARGUMENT
    assert plan.add(name, bufs, n, [16, 100, 77] + list(u[3:]), flags=flags) == hip.UNSUPPORTED
    assert plan.add(name, bufs, n, [16, 0, hip.Q8_0] + list(u[3:]), flags=flags) == hip.INVALID_ARGUMENT
    assert plan.add(name, bufs, n, [0, 100, hip.Q8_0] + list(u[3:]), flags=flags) == hip.INVALID_ARGUMENT
    # each buffer: missing, too short, and at an offset that leaves too little or is misaligned
    for i, b in enumerate(bufs):
        if b is None or (b is bufs[-1] and not flags):
            continue
        if (name, i) not in (("KV_APPEND", 5),):
            less = list(bufs)
            less[i] = None
            assert plan.add(name, less, n, u, flags=flags) == hip.INVALID_ARGUMENT, (name, i, "missing")
        offs = [0] * 16
        offs[i] = b.handle.bytes
        assert plan.add(name, bufs, n, u, offs=offs, flags=flags) == hip.INVALID_ARGUMENT, (name, i, "offset")
        offs[i] = 2
        assert plan.add(name, bufs, n, u, offs=offs, flags=flags) == hip.INVALID_ARGUMENT, (name, i, "aligned")


@pytest.mark.parametrize("name", ["KV_APPEND", "ATTN_DECODE", "ATTN_VERIFY"])
def test_several_requests_need_their_own_positions(name):
    plan = _Plan()
    bufs, n, u, _ = _ops(_memory())[name]
    assert plan.add(name, bufs, n, u, flags=0) == hip.INVALID_ARGUMENT


@pytest.mark.parametrize("disp,status", [(2 ** 64 - 3, hip.OK), (5, hip.OK), (2 ** 40, hip.INVALID_ARGUMENT),
                                         (2 ** 63, hip.INVALID_ARGUMENT), (2 ** 31, hip.INVALID_ARGUMENT)])
def test_displacements_are_signed(disp, status):
    plan = _Plan()
    bufs, n, u, flags = _ops(_memory())["KV_READ"]
    assert plan.add("KV_READ", bufs, n[:5] + [disp], u, flags=flags) == status


def test_prefill_attention_takes_16_rows():
    plan = _Plan()
    m = _memory()
    m["q"], m["out"] = _Mem(17 * 4 * 128 * 4), _Mem(17 * 4 * 128 * 4)
    bufs, n, u, flags = _ops(m)["ATTENTION_PREFILL_PAGED"]
    for rows, status in ((16, hip.OK), (17, hip.INVALID_ARGUMENT)):
        assert plan.add("ATTENTION_PREFILL_PAGED", bufs, n[:4] + [rows, 0], u, flags=flags) == status


# ------------------------------------------------------- rows between requests

WRAP = [  # the rows' bytes are 2^64 and a little: requests, rows between them, heads, kv heads
    ("append", 4097, 1 << 30, 0, 4096),            # 4096 2^30 rows of 2^22 bytes
    ("read", 4097, 1 << 30, 0, 4096),
    ("append", 16385, 1 << 28, 0, 4096),
    ("attn", 513, 1 << 30, 32768, 128),            # 512 2^30 rows of 2^25 bytes
    ("attn", 1025, 1 << 29, 32768, 128),
]


@pytest.mark.parametrize("name,requests,stride,heads,kv_heads", WRAP)
def test_rows_that_wrap_around_64_bits_are_refused(name, requests, stride, heads, kv_heads):
    """Buffers of one request's size do not pass for those of thousands."""
    m = _memory()
    m.update(norm=None, rope=None)
    row = 4 * 256 * (heads or kv_heads)
    assert (requests - 1) * stride * row % 2 ** 64 == 0
    for b in m.values():
        if b is not None:
            b.handle.bytes = 1 << 26
    for b in ("k", "v", "q", "out"):
        m[b].handle.bytes = row
    for b in ("kpool", "vpool"):
        m[b].handle.bytes = 1 << 40
    p = hip.kv_params(hip.Q8_0, 16, 100, kv_heads, 256, 1, requests, heads=heads, request_rows=stride)
    assert _call(name, m, p) == hip.INVALID_ARGUMENT
    assert b"rows" in hip.lib().yuuka_last_error()


@pytest.mark.parametrize("name", ["append", "read", "attn"])
def test_requests_do_not_overlap(name):
    """Rows between requests are none (the rows themselves) or at least the rows: 3 here."""
    m = _memory()
    m.update(norm=None, rope=None)
    for stride in (1, 2):
        assert _call(name, m, hip.kv_params(**GOOD, heads=4, request_rows=stride)) == hip.INVALID_ARGUMENT
        assert b"rows between requests of 3" in hip.lib().yuuka_last_error()
    assert hip.kv_page_bytes(hip.kv_params(**GOOD, request_rows=2)) == 0
    for stride in (0, 3):
        assert hip.kv_page_bytes(hip.kv_params(**GOOD, request_rows=stride)) > 0


@pytest.mark.parametrize("name", ["KV_APPEND", "KV_READ", "ATTN_DECODE", "ATTN_VERIFY"])
def test_requests_of_an_op_do_not_overlap(name):
    """ATTN_VERIFY takes fewer rows between requests as the rows, over pools of every format."""
    plan = _Plan()
    bufs, n, u, flags = _ops(_memory())[name]
    low = u[3] & 0xff
    less = hip.OK if name == "ATTN_VERIFY" else hip.INVALID_ARGUMENT
    for stride, status in ((0, hip.OK), (1, less), (2, less), (3, hip.OK)):
        assert plan.add(name, bufs, n, list(u[:3]) + [_U(low, 2, stride)], flags=flags) == status, stride
    if name == "ATTN_VERIFY":
        m = _memory(hip.F16)
        m["kpool"], m["vpool"] = _Mem(7 * 16 * 2 * KVD), _Mem(7 * 16 * 2 * KVD)
        bufs, n, u, flags = _ops(m)[name]
        for stride in range(4):
            assert plan.add(name, bufs, n, [16, 100, hip.F16, _U(low, 2, stride)], flags=flags) == hip.OK


# ------------------------------------------------------------------ the engine

def _create(**change):
    """The status of an engine creation on a device that there is not."""
    cfg = replace(Mdl.TINY, kv_dtype=hip.Q8_0, batch=2, **change)
    if not hasattr(hip.lib(), "_q35_declared"):
        Mdl._declare(hip.lib())
        hip.lib()._q35_declared = True
    cs, ws, layers = Mdl.config_struct(cfg), Mdl.yuuka_q35_weights(), (Mdl.yuuka_q35_layer_weights * cfg.n_layers)()
    ws.layers = C.cast(layers, C.POINTER(Mdl.yuuka_q35_layer_weights))
    dev, out = C.c_int32(1 << 20), C.c_void_p()  # yuuka_device starts with its index
    return hip.lib().yuuka_q35_create(C.addressof(dev), C.byref(cs), C.byref(ws), C.byref(out))


@pytest.mark.parametrize("change,status", [
    (dict(head_dim=96), hip.UNSUPPORTED), (dict(head_dim=320), hip.UNSUPPORTED), (dict(head_dim=32), hip.UNSUPPORTED),
    (dict(rope_dim=0), hip.INVALID_ARGUMENT), (dict(rope_dim=130), hip.INVALID_ARGUMENT),
    (dict(rope_dim=31), hip.INVALID_ARGUMENT), (dict(heads=514, kv_heads=2), hip.INVALID_ARGUMENT),
    (dict(block_size=1 << 21), hip.INVALID_ARGUMENT)])
def test_an_engine_over_q8_0_pages_refuses_what_its_attention_does(change, status):
    """At its creation, before a weight is uploaded, not in its first step; what is served gets as far as the device."""
    assert _create(**change) == status
    assert _create() == hip.DEVICE
    # without a layer of attention there is no cache
    assert _create(**change, full_interval=Mdl.TINY.n_layers + 1) == hip.DEVICE


# ------------------------------------------------------------------- the binding

def test_a_graph_keeps_the_buffers_it_was_captured_over(monkeypatch):
    """It holds their addresses, and may outlive its plan."""
    class Owner:
        pass

    plan, dynamic, buffers = Owner(), Owner(), [Owner() for _ in range(3)]
    plan.ptr, plan.keep, dynamic.ptr = None, list(buffers), None
    calls = []
    monkeypatch.setattr(hip, "lib", lambda: SimpleNamespace(yuuka_graph_create=lambda *a: calls.append(a) or hip.OK,
                                                            yuuka_graph_destroy=lambda p: calls.append(p)))
    graph = hip.Graph(plan, SimpleNamespace(ptr=None), dynamic)
    graph.ptr = 1
    alive = [weakref.ref(b) for b in buffers + [dynamic]]
    later = Owner()
    plan.keep.append(later)       # of an op that is not in the graph
    alive_later = weakref.ref(later)
    del plan, dynamic, buffers, later
    gc.collect()
    assert all(a() is not None for a in alive) and alive_later() is None
    graph.destroy()
    gc.collect()
    assert len(calls) == 2 and all(a() is None for a in alive)

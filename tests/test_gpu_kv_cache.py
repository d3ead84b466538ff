"""The paged key/value cache on the GPU (yuuka_kv_append, yuuka_kv_read,
yuuka_attn_decode, their plan ops, the v10 cache ops and the engine over Q8_0
pools) against plain NumPy: the Q8_0 rounding bit for bit, attention in
float64.

Attention's tolerance, relative to the output's 2-norm: a query is split into
two halves of 11 bits (2^-23 of its largest element), products are exact and
summed in float32, the weights' exponential is within 2^-22, and a value's
weight is again two halves (2^-22). A score of magnitude s is then off by about
s 2^-23 sqrt(4): with |s| up to 16 in these inputs, 2^-18 of a weight at the
most, and far less in the norm. 2^-18 in the norm, with nothing hidden by it:
rounding a value or a weight to one half alone would be 2^-12."""
from __future__ import annotations

import math
from dataclasses import replace

import numpy as np
import pytest

from oracle import oracle as O
from yuuka_amd import hip
from yuuka_amd import model as Mdl

pytestmark = pytest.mark.gpu

F32, F16, Q8 = hip.F32, hip.F16, hip.Q8_0
TOL = 2.0 ** -18


# ------------------------------------------------------------------ reference

def half_up(x):
    """float32 -> half bits, halves upwards in magnitude and what is below 2^-24 to zero (the reference's
    Float32ToFloat16)."""
    x = np.ascontiguousarray(x, np.float32)
    a = np.abs(x)
    with np.errstate(all="ignore"):
        normal = ((a.view(np.uint32) + np.uint32(0x1000)) & ~np.uint32(0x1FFF)).view(np.float32)
        small = np.where(a < 2.0 ** -24, 0, np.floor(a.astype(np.float64) * 2.0 ** 24 + 0.5)) * 2.0 ** -24
        return np.copysign(np.where(a < 2.0 ** -14, small, normal), x).astype(np.float16).view(np.uint16)


def encode(x):
    """float32 [..., kv_dim] -> (int8 digits in storage order, half scales' bits)."""
    x = np.asarray(x, np.float32)
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        top = np.abs(b).max(-1, keepdims=True)  # NaN where the block holds one
        s = (top * (np.float32(1) / np.float32(127))).astype(np.float32)
        t = np.where(s > 0, b / s, np.float32(0)).astype(np.float64)
        d = np.copysign(np.floor(np.abs(t) + 0.5), t)
        d = np.where(np.isfinite(t) & (np.abs(d) <= 127), d, 0).astype(np.int8)
    d = d.reshape(*x.shape[:-1], -1, 4, 16).swapaxes(-1, -2)  # 64 dims as 16 x 4
    return d.reshape(x.shape), half_up(s[..., 0])


def decode(digits, scales):
    v = digits.reshape(*digits.shape[:-1], -1, 16, 4).swapaxes(-1, -2).reshape(*digits.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore"):  # 0 * inf
        return (v.astype(np.float32) * scales.view(np.float16).astype(np.float32)[..., None]).reshape(digits.shape)


class Cache:
    """Pools, tables and positions on the host, and their device copies."""

    def __init__(self, dev, dtype, bs, cap, nk, D, requests, positions, seed=0, pages=None, shared=False, fill=None):
        rng = np.random.default_rng(seed)
        self.dev, self.dtype, self.bs, self.cap, self.nk, self.D = dev, dtype, bs, cap, nk, D
        self.kvd, self.requests = nk * D, requests
        self.blocks = -(-cap // bs)
        self.pages = pages or requests * self.blocks + 2
        self.token = {F32: 4 * self.kvd, F16: 2 * self.kvd, Q8: self.kvd * 34 // 32}[dtype]
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.tile(order[: self.blocks], (requests, 1)) if shared else \
            order[: requests * self.blocks].reshape(requests, self.blocks).copy()
        self.pool = [np.full((self.pages, bs * self.token), 0xA5, np.uint8) for _ in range(2)]
        if fill is not None:
            for p in self.pool:
                fill(rng, p)
        self.positions = np.zeros((requests, 2), np.int32)
        self.positions[:, 1] = positions
        self.b_pool = [dev.upload(p) for p in self.pool]
        self.b_table, self.b_pos = dev.upload(self.table), dev.upload(self.positions)

    def upload(self):
        for b, p in zip(self.b_pool, self.pool):
            b.write(p)
        self.b_table.write(self.table)
        self.b_pos.write(self.positions)

    def params(self, rows, **kw):
        return hip.kv_params(self.dtype, self.bs, self.cap, self.nk, self.D, rows, self.requests, **kw)

    def at(self, j, p):
        """(page, slot) of a position, None where there is none."""
        if p < 0 or p >= self.cap:
            return None
        page = self.table[j, p // self.bs]
        return (page, p % self.bs) if 0 <= page < self.pages else None

    def put(self, side, j, p, row):
        """What an append leaves in the pool."""
        at = self.at(j, p)
        if at is None:
            return
        page, t = at
        pool, n = self.pool[side][page], self.kvd
        if self.dtype == Q8:
            d, s = encode(row)
            pool[t * n:(t + 1) * n] = d.view(np.uint8)
            o = self.bs * n + t * n // 16
            pool[o:o + n // 16] = s.view(np.uint8)
        else:
            raw = half_up(row) if self.dtype == F16 else np.asarray(row, np.float32)
            pool[t * self.token:(t + 1) * self.token] = raw.view(np.uint8)

    def row(self, side, j, p):
        """A cached row as float32; zeros where there is none."""
        at = self.at(j, p)
        if at is None:
            return np.zeros(self.kvd, np.float32)
        page, t = at
        pool, n = self.pool[side][page], self.kvd
        if self.dtype == Q8:
            o = self.bs * n + t * n // 16
            return decode(pool[t * n:(t + 1) * n].view(np.int8), pool[o:o + n // 16].copy().view(np.uint16))
        raw = pool[t * self.token:(t + 1) * self.token].copy()
        return raw.view(np.float16).astype(np.float32) if self.dtype == F16 else raw.view(np.float32)

    def read_pool(self, side):
        return self.b_pool[side].read(np.uint8).reshape(self.pages, -1)


def q8_fill(scale=0.03):
    """Random digits and scales."""
    def fill(rng, pool):
        n = pool.shape[1] * 32 // 34
        pool[:, :n] = rng.normal(0, 42, (pool.shape[0], n)).clip(-127, 127).astype(np.int8).view(np.uint8)
        s = (scale * rng.uniform(0.5, 1.5, (pool.shape[0], n // 32))).astype(np.float16)
        pool[:, n:] = s.view(np.uint8)
    return fill


def f16_fill(rng, pool):
    pool[:] = rng.normal(0, 1, (pool.shape[0], pool.shape[1] // 2)).astype(np.float16).view(np.uint8)


def attention(c, q, rows, heads, scale, gated, request_rows=None, displacement=0):
    """float64 [requests * request_rows][heads][D]; rows in between are NaN."""
    rr, D, G = request_rows or rows, c.D, heads // c.nk
    q = q.astype(np.float64)
    out = np.full((c.requests * rr, heads, D), np.nan)
    for j in range(c.requests):
        first = int(c.positions[j, 1]) + displacement
        n = max(0, min(first + rows, c.cap))
        seen = [p for p in range(n) if c.at(j, p) is not None]
        K = np.array([c.row(0, j, p) for p in seen], np.float64).reshape(len(seen), c.nk, D)
        V = np.array([c.row(1, j, p) for p in seen], np.float64).reshape(len(seen), c.nk, D)
        for r in range(rows):
            m = sum(p <= first + r for p in seen)
            for h in range(heads):
                if m == 0:
                    out[j * rr + r, h] = 0
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    s = K[:m, h // G] @ q[j * rr + r, h, :D] * scale
                    w = np.exp(s - s.max())
                    o = w @ V[:m, h // G] / w.sum()
                    if gated:
                        o = o / (1 + np.exp(-q[j * rr + r, h, D:]))
                out[j * rr + r, h] = o
    return out


def close(got, want, tol=TOL, floor=0.0):
    """Equal up to tol of the norm, and `floor` an element."""
    got, want = got.astype(np.float64), np.asarray(want, np.float64)
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    ok = np.isfinite(want)
    d = np.linalg.norm(got[ok] - want[ok])
    assert d <= tol * np.linalg.norm(want[ok]) + floor * math.sqrt(ok.sum()), d / np.linalg.norm(want[ok])


# --------------------------------------------------------- append and read back

SHAPES = [  # kv heads, head width, page, capacity, rows, row stride, positions, displacement
    (1, 64, 1, 5, 1, 0, [0], 0),
    (3, 64, 3, 40, 2, 5, [7, 0, 38], 0),
    (5, 64, 16, 48, 3, 0, [0, 31], 1),
    (16, 64, 64, 130, 1, 0, [129, 0, 64], 0),
    (1, 128, 16, 33, 4, 0, [14, 29], 0),
    (3, 128, 5, 60, 7, 9, [3, 50], -2),
    (8, 128, 32, 64, 2, 0, [31], 0),
    (1, 192, 7, 30, 3, 0, [5, 26], 0),
    (2, 192, 16, 64, 5, 6, [13, 0], 0),
    (1, 256, 16, 64, 1, 0, [17], 0),
    (4, 256, 16, 600, 9, 0, [517, 0, 15], 0),
    (2, 256, 100, 300, 120, 130, [0, 90], 0),
]


@pytest.mark.parametrize("dtype", [Q8, F16, F32])
@pytest.mark.parametrize("nk,D,bs,cap,rows,stride,positions,disp", SHAPES)
def test_append_and_read(dev, stream, dtype, nk, D, bs, cap, rows, stride, positions, disp):
    """The whole pool after an append is the reference's, bytes that are no new row's as they were; the rows read back
    are the values those bytes stand for."""
    n = len(positions)
    c = Cache(dev, dtype, bs, cap, nk, D, n, positions, seed=nk * D + rows)
    rr = max(stride, rows)
    rng = np.random.default_rng(rows)
    x = (rng.normal(0, 1, (2, n * rr, c.kvd)) * np.exp(rng.normal(0, 1, (2, n * rr, 1)))).astype(np.float32)
    x[:, :, :32] *= 0                     # a block of zeros
    x[0, 0, -1] = -np.abs(x).max() * 3    # a lone large value
    bufs = [dev.upload(x[0]), dev.upload(x[1])]
    p = c.params(rows, request_rows=stride, displacement=disp)
    hip.kv_append(stream, *bufs, *c.b_pool, c.b_table, c.b_pos, p)
    stream.sync()
    for j in range(n):
        for r in range(rows):
            for side in range(2):
                c.put(side, j, positions[j] + disp + r, x[side, j * rr + r])
    for side in range(2):
        assert np.array_equal(c.read_pool(side), c.pool[side])
    out = [dev.upload(np.full((n * rr, c.kvd), 7.25, np.float32)) for _ in range(2)]
    hip.kv_read(stream, *out, *c.b_pool, c.b_table, p, positions=c.b_pos)
    stream.sync()
    for side in range(2):
        got = out[side].read(np.float32).reshape(n, rr, c.kvd)
        for j in range(n):
            for r in range(rr):
                want = c.row(side, j, positions[j] + disp + r) if r < rows else np.full(c.kvd, 7.25, np.float32)
                assert np.array_equal(got[j, r].view(np.uint32), want.view(np.uint32)), (side, j, r)


def test_read_one_side_and_absolute_positions(dev, stream):
    c = Cache(dev, Q8, 16, 50, 2, 128, 3, [0, 9, 20], fill=q8_fill())
    out = dev.upload(np.full((3 * 50, c.kvd), 7.25, np.float32))
    for side in range(2):
        hip.kv_read(stream, out if side == 0 else None, out if side else None, c.b_pool[0] if side == 0 else None,
                    c.b_pool[1] if side else None, c.b_table, c.params(50))
        stream.sync()
        got = out.read(np.float32).reshape(3, 50, c.kvd)
        assert np.array_equal(got, [[c.row(side, j, p) for p in range(50)] for j in range(3)])


def test_the_references_half():
    """half_up here is the oracle's conversion."""
    x = np.concatenate([np.float32([0, -0.0, 1e-8, 2.0 ** -25, 2.0 ** -25.5, 3e-6, 6.1e-5, 65504, 65519, 65520, -7e4, np.inf]),
                        np.random.default_rng(0).normal(0, 1, 2000).astype(np.float32) ** 9])
    assert [O.f32_to_f16(float(v)) for v in x] == half_up(x).tolist()


def _special_blocks():
    f = np.float32
    rng = np.random.default_rng(3)
    rows = [np.zeros(32)]
    for top in (1e-45, 1e-40, 3e-38, 1e-12, 127 * 2.0 ** -26, 127 * 2.0 ** -25, 127 * 2.0 ** -24.5, 127 * 2.0 ** -24,
                127 * 2.0 ** -14, 1.0, 127 * 65504.0, 127 * 65519.0, 127 * 65520.0, 1e10, 3e38):
        b = rng.uniform(-1, 1, 32)
        b[5] = -1
        rows.append(f(top) * b.astype(f))
    for m in range(40):  # scales half way between two halves, and next to that
        mid = (2048 + 2 * (m * 25 % 1024) + 1) * 2.0 ** -12
        for step in (-1, 0, 1):
            b = rng.normal(0, 20, 32).clip(-60, 60)
            b[31] = (f(127 * mid).view(np.int32) + step).view(f)
            rows.append(b)
    ties = np.arange(32) - 15.5  # digits half way, of both signs, at scale 1
    ties[0] = 127
    rows += [ties, -ties, np.nextafter(ties.astype(f), f(0)), np.nextafter(ties.astype(f), f(1e9))]
    for bad in (np.nan, np.inf, -np.inf):
        b = rng.normal(0, 1, 32)
        b[11] = bad
        rows.append(b)
    b = rng.normal(0, 1, 32)
    b[3], b[4] = np.inf, np.nan
    rows.append(b)
    n = len(rows)
    return np.array(rows + [np.ones(32)] * (-n % 8), f)


@pytest.mark.parametrize("nk,D", [(4, 64), (2, 128), (1, 256)])
def test_append_rounding_at_the_borders(dev, stream, nk, D):
    """Subnormal, tied, overflowing and non-finite scales and digits."""
    x = _special_blocks().reshape(-1, 256)
    c = Cache(dev, Q8, 16, len(x), nk, D, 1, [0])
    with np.errstate(all="ignore"):
        hip.kv_append(stream, dev.upload(x), dev.upload(x[::-1].copy()), *c.b_pool, c.b_table, c.b_pos, c.params(len(x)))
        stream.sync()
        for p, row in enumerate(x):
            c.put(0, 0, p, row)
            c.put(1, 0, len(x) - 1 - p, row)
        for side in range(2):
            got, want = c.read_pool(side), c.pool[side]
            n = 16 * 256
            assert np.array_equal(got[:, :n], want[:, :n])
            s, t = got[:, n:].copy().view(np.float16), want[:, n:].copy().view(np.float16)
            assert np.array_equal(s, t, equal_nan=True)
        out = [dev.alloc(x.nbytes) for _ in range(2)]
        hip.kv_read(stream, *out, *c.b_pool, c.b_table, c.params(len(x)))
        stream.sync()
        got = out[0].read(np.float32).reshape(x.shape)
        assert np.array_equal(got, [c.row(0, 0, p) for p in range(len(x))], equal_nan=True)
        # a block that holds a NaN or an infinity, or values past the scale's range, does not read back as finite
        past = ~(np.abs(x.reshape(-1, 32)) < 127 * 65521).all(1)
        assert past.sum() == 6 and not np.isfinite(got.reshape(-1, 32)).all(1)[past].any()
        assert np.isnan(got.reshape(-1, 32)[np.isnan(x.reshape(-1, 32)).any(1)]).all()


@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_append_over_the_whole_float_range(dev, stream, D):
    """Blocks from the smallest subnormal to the largest float, and with infinities: bit for bit."""
    tops = [1e-45, 1e-42, 1e-38, 3e-32, 1e-30, 7e-31, 1e-20, 6e-6, 7.5e-6, 1e-3, 1.0, 127.0, 8.3e6, 8.4e6, 1e20, 5e30, 2e31,
            1e37, 3.4e38, 0.0]
    rng = np.random.default_rng(D)
    x = rng.uniform(-1, 1, (2, len(tops), 4 * D))
    x = (x * np.array(tops)[:, None]).astype(np.float32)
    x[0, 3, 5], x[1, 9, D], x[0, 12, 2 * D + 1] = np.inf, -np.inf, np.nan
    c = Cache(dev, Q8, 16, 64, 4, D, 1, [10])
    hip.kv_append(stream, dev.upload(x[0]), dev.upload(x[1]), *c.b_pool, c.b_table, c.b_pos, c.params(len(tops)))
    stream.sync()
    for side in range(2):
        for r in range(len(tops)):
            c.put(side, 0, 10 + r, x[side, r])
        got, want = c.read_pool(side), c.pool[side]
        nan = np.isnan(x[side]).any()
        if nan:  # the scale of a block with a NaN is a NaN, of whichever payload
            page, t = c.at(0, 22)
            o = 16 * c.kvd + t * c.kvd // 16 + (2 * D // 32) * 2
            assert np.isnan(got[page, o:o + 2].copy().view(np.float16)).all()
            got[page, o:o + 2] = want[page, o:o + 2]
        assert np.array_equal(got, want)


@pytest.mark.parametrize("dtype", [Q8, F16, F32])
@pytest.mark.parametrize("nk,D,rot", [(3, 64, 64), (3, 128, 20), (2, 192, 128), (4, 256, 64), (1, 256, 2)])
def test_append_with_norm_and_rotation(dev, stream, dtype, nk, D, rot):
    """The key norm and rotation inside the append are the separate ops'."""
    rows, positions = 5, [3, 40]
    c = Cache(dev, dtype, 16, 64, nk, D, 2, positions, seed=D)
    rng = np.random.default_rng(rot)
    k, v = (rng.normal(0, 2, (2 * rows, c.kvd)).astype(np.float32) for _ in range(2))
    w = (1 + 0.1 * rng.normal(0, 1, D)).astype(np.float32)
    rope = dev.alloc(2 * rows * rot // 2 * 8)
    kb, vb, wb, knb = dev.upload(k), dev.upload(v), dev.upload(w), dev.alloc(k.nbytes)
    plan = hip.Plan(dev)
    plan.add(hip.OP["ROPE_TABLE"], [rope] + [None] * 14 + [c.b_pos], n=[rows, rot, 0, 2, rows], f=[1e4],
             flags=hip.FLAG_OWN_POS)
    plan.add(hip.OP["RMSNORM_HEADS_BATCH"], [kb, wb, knb], n=[D, nk, D, 2 * rows], f=[1e-6])
    plan.execute(stream)
    stream.sync()
    kn = knb.read(np.float32).reshape(2 * rows, nk, D)
    cs = rope.read(np.float32).reshape(2 * rows, 1, rot // 2, 2)
    a, b = kn[..., :rot // 2].copy(), kn[..., rot // 2:rot].copy()
    kn[..., :rot // 2] = a * cs[..., 0] - b * cs[..., 1]
    kn[..., rot // 2:rot] = a * cs[..., 1] + b * cs[..., 0]
    hip.kv_append(stream, kb, vb, *c.b_pool, c.b_table, c.b_pos, c.params(rows, rope_dim=rot), k_norm=wb, rope=rope)
    stream.sync()
    for j in range(2):
        for r in range(rows):
            c.put(0, j, positions[j] + r, kn[j * rows + r].reshape(-1))
            c.put(1, j, positions[j] + r, v[j * rows + r])
    for side in range(2):
        assert np.array_equal(c.read_pool(side), c.pool[side])
    plan.destroy()


@pytest.mark.parametrize("dtype", [Q8, F16])
def test_unmapped_pages_and_positions_outside(dev, stream, dtype):
    """Writes to unmapped pages and positions outside the capacity are dropped, such rows read as zeros, and attention
    leaves their tokens out; a row that sees nothing is zero."""
    D, nk, heads, rows = 128, 2, 4, 4
    fill = q8_fill() if dtype == Q8 else f16_fill
    positions = [37, -2, 60, -9, 2 ** 31 - 2, 5, -(2 ** 31)]
    c = Cache(dev, dtype, 16, 62, nk, D, len(positions), positions, fill=fill)
    c.table[0, 1] = -1
    c.table[0, 2] = c.pages
    c.table[2, 3] = 2 ** 31 - 1
    c.table[5, :] = -7
    c.upload()
    rng = np.random.default_rng(8)
    n = len(positions) * rows
    x = rng.normal(0, 1, (2, n, c.kvd)).astype(np.float32)
    p = c.params(rows, heads=heads, gated=True, scale=D ** -0.5)
    hip.kv_append(stream, dev.upload(x[0]), dev.upload(x[1]), *c.b_pool, c.b_table, c.b_pos, p)
    stream.sync()
    for j, pos in enumerate(positions):
        for r in range(rows):
            for side in range(2):
                c.put(side, j, pos + r, x[side, j * rows + r])
    for side in range(2):
        assert np.array_equal(c.read_pool(side), c.pool[side])
    out = [dev.alloc(n * c.kvd * 4) for _ in range(2)]
    hip.kv_read(stream, *out, *c.b_pool, c.b_table, p, positions=c.b_pos)
    q = rng.normal(0, 1, (n, heads, 2 * D)).astype(np.float32)
    o = dev.upload(np.full((n, heads, D), 3.5, np.float32))
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, p)
    stream.sync()
    for side in range(2):
        want = [c.row(side, j, pos + r) for j, pos in enumerate(positions) for r in range(rows)]
        assert np.array_equal(out[side].read(np.float32).reshape(n, -1), want)
    got, want = o.read(np.float32).reshape(n, heads, D), attention(c, q, rows, heads, D ** -0.5, True)
    close(got, want)
    empty = (want == 0).all((1, 2))
    assert empty.sum() >= 4 + 4 + 4 + 2 and (got[empty] == 0).all()


# ------------------------------------------------------------------- attention

ATTN = [  # heads, kv heads, head width, page, rows, positions, gated
    (1, 1, 64, 1, 1, [0, 1, 2, 14, 15, 16], False),
    (4, 4, 64, 16, 1, [31, 32, 33, 63, 64, 65], True),
    (16, 1, 64, 16, 1, [200, 7], False),
    (40, 2, 64, 5, 2, [100, 18], False),
    (32, 8, 128, 16, 1, [127, 128, 129, 300], False),
    (8, 2, 128, 64, 5, [0, 40, 511], True),
    (6, 2, 192, 16, 1, [90, 0, 255], False),
    (6, 1, 192, 7, 3, [90, 3], True),
    (16, 4, 256, 16, 1, [517, 0, 1030], True),
    (8, 2, 256, 16, 4, [0, 61, 62, 63, 64], True),
    (16, 2, 256, 32, 1, [400], False),
    (16, 4, 256, 16, 5, [517, 28], True),
    (16, 4, 256, 16, 9, [250, 1], True),
    (16, 4, 256, 16, 17, [333], True),
    (8, 2, 256, 16, 32, [0, 100], False),
    (2, 2, 256, 16, 70, [40], False),
    (12, 4, 128, 16, 3, [2049], False),
    (7, 7, 64, 16, 11, [13], False),
]


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("heads,nk,D,bs,rows,positions,gated", ATTN)
def test_attention(dev, stream, dtype, heads, nk, D, bs, rows, positions, gated):
    cap = max(positions) + rows + 3
    c = Cache(dev, dtype, bs, cap, nk, D, len(positions), positions, seed=heads + rows,
              fill=q8_fill() if dtype == Q8 else f16_fill)
    rng = np.random.default_rng(D + rows)
    n = len(positions) * rows
    q = rng.normal(0, 1, (n, heads, 2 * D if gated else D)).astype(np.float32)
    o = dev.alloc(n * heads * D * 4)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos,
                    c.params(rows, heads=heads, gated=gated, scale=D ** -0.5))
    stream.sync()
    close(o.read(np.float32).reshape(n, heads, D), attention(c, q, rows, heads, D ** -0.5, gated))


def test_attention_row_stride_and_displacement(dev, stream):
    """Rows between the requests' are neither read nor written."""
    heads, nk, D, rows, rr = 8, 2, 128, 3, 5
    c = Cache(dev, Q8, 16, 90, nk, D, 3, [20, 50, 4], fill=q8_fill())
    rng = np.random.default_rng(4)
    q = rng.normal(0, 1, (3 * rr, heads, D)).astype(np.float32)
    want = attention(c, q, rows, heads, 0.1, False, request_rows=rr, displacement=-5)
    q[np.isnan(want[:, 0, 0])] = np.nan
    o = dev.upload(np.full((3 * rr, heads, D), np.nan, np.float32))
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos,
                    c.params(rows, heads=heads, scale=0.1, request_rows=rr, displacement=-5))
    stream.sync()
    close(o.read(np.float32).reshape(want.shape), want)


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("rows", [1, 6])
def test_what_is_past_a_row_does_not_reach_it(dev, stream, dtype, rows):
    """Every byte of the pools that no row sees is 0xFF: NaN halves, NaN scales."""
    heads, nk, D = 8, 2, 256
    c = Cache(dev, dtype, 16, 300, nk, D, 4, [0, 15, 70, 250], fill=q8_fill() if dtype == Q8 else f16_fill)
    keep = [np.full_like(p, 0xFF) for p in c.pool]
    n = c.kvd
    for j in range(4):
        for p in range(int(c.positions[j, 1]) + rows):
            page, t = c.at(j, p)
            for side in range(2):
                runs = [(t * c.token, (t + 1) * c.token)] if dtype == F16 else \
                    [(t * n, (t + 1) * n), (16 * n + t * n // 16, 16 * n + (t + 1) * n // 16)]
                for lo, hi in runs:
                    keep[side][page, lo:hi] = c.pool[side][page, lo:hi]
    c.pool = keep
    c.upload()
    q = np.random.default_rng(1).normal(0, 1, (4 * rows, heads, D)).astype(np.float32)
    o = dev.alloc(q.nbytes)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=D ** -0.5))
    stream.sync()
    close(o.read(np.float32).reshape(q.shape), attention(c, q, rows, heads, D ** -0.5, False))


@pytest.mark.parametrize("dtype", [Q8, F16])
def test_a_nan_reaches_the_rows_that_see_it(dev, stream, dtype):
    heads, nk, D, rows = 8, 2, 128, 3
    c = Cache(dev, dtype, 16, 100, nk, D, 3, [60, 60, 60], fill=q8_fill() if dtype == Q8 else f16_fill)
    nan = np.ones(c.kvd, np.float32)
    nan[D + 40] = np.nan       # the second kv head's key
    c.put(0, 0, 61, nan)       # seen by rows 1 and 2 of request 0
    c.put(1, 1, 5, nan)        # a value that every row of request 1 sees
    c.upload()
    q = np.random.default_rng(1).normal(0, 1, (9, heads, D)).astype(np.float32)
    q[7, 3, 17] = np.nan       # one query of request 2
    o = dev.alloc(q.nbytes)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=D ** -0.5))
    stream.sync()
    got = np.isnan(o.read(np.float32).reshape(q.shape))
    want = np.zeros_like(got)
    want[1:3, 4:] = True
    block = slice(32, 64) if dtype == Q8 else slice(40, 41)
    want[3:6, 4:, block] = True
    want[7, 3] = True
    assert np.array_equal(got, want)


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("qs,ks,vs", [(1e-12, 1e-3, 1e-6), (3e4, 1e-4, 100.0), (1e-3, 30.0, 1e-4), (1e15, 1e-5, 1.0)])
def test_magnitudes(dev, stream, dtype, qs, ks, vs):
    """Queries and values from tiny to large, and a value block a thousand times the next: nothing is lost to the range
    of a half. The scale puts the scores at a few units."""
    heads, nk, D, rows = 8, 2, 256, 2
    c = Cache(dev, dtype, 16, 200, nk, D, 2, [150, 30], fill=None)
    rng = np.random.default_rng(2)
    size = np.where(np.arange(c.kvd) // 32 % 2, 1.0, 1e-3)
    for j in range(2):
        for p in range(200):
            grow = 10.0 ** (p // 40 - 3)  # later tokens' values are larger
            c.put(0, j, p, (rng.normal(0, ks, c.kvd)).astype(np.float32))
            c.put(1, j, p, (rng.normal(0, vs, c.kvd) * size * grow).astype(np.float32))
    c.upload()
    q = rng.normal(0, qs, (4, heads, D)).astype(np.float32)
    scale = 2.0 / (qs * ks * 16)
    want = attention(c, q, rows, heads, np.float32(scale), False)
    o = dev.alloc(q.nbytes)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=scale))
    stream.sync()
    got = o.read(np.float32).reshape(q.shape)
    for odd in range(2):  # the small blocks on their own
        dims = np.arange(D) // 32 % 2 == odd
        # An MFMA aligns the products it sums by their exponent fields, and a subnormal half has that of 2^-14: with
        # weights that sum to one, such values (steps of 2^-24) are summed to 2^-14 2^-24 = 2^-38. Q8_0 digits are
        # normal halves; the last bits of 2^-38 a term, over the terms' 2^4 spread of weights, are 2^-36 at the most.
        close(got[..., dims], want[..., dims], floor=2.0 ** -36 if dtype == F16 else 0.0)


@pytest.mark.parametrize("dtype", [Q8, F16])
def test_scores_far_apart(dev, stream, dtype):
    """One key far above the others, first, in the middle and last: the running maximum moves by hundreds."""
    heads, nk, D = 4, 1, 64
    c = Cache(dev, dtype, 16, 700, nk, D, 4, [599] * 4, fill=q8_fill() if dtype == Q8 else f16_fill)
    rng = np.random.default_rng(6)
    q = rng.normal(0, 1, (4, heads, D)).astype(np.float32)
    for j, p in enumerate([0, 300, 599]):
        c.put(0, j, p, q[j, 1] * 30)
    c.upload()
    o = dev.alloc(q.nbytes)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(1, heads=heads, scale=1.0))
    stream.sync()
    # scores up to 2000: their float32 rounding alone is 2000 * 2^-24, a few times that after 64 terms
    close(o.read(np.float32).reshape(q.shape), attention(c, q, 1, heads, 1.0, False), tol=2000 * 2.0 ** -22)


@pytest.mark.parametrize("dtype", [Q8, F16])
def test_long_contexts_and_shared_pages(dev, stream, dtype):
    """A context of many splits, and requests that share the prefix's pages."""
    heads, nk, D = 8, 2, 128
    positions = [9000, 8191, 8192, 4095, 33]
    c = Cache(dev, dtype, 64, 9001, nk, D, 5, positions, shared=True, pages=150,
              fill=q8_fill() if dtype == Q8 else f16_fill)
    q = np.random.default_rng(1).normal(0, 1.5, (5, heads, D)).astype(np.float32)
    o = dev.alloc(q.nbytes)
    p = c.params(1, heads=heads, scale=D ** -0.5)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, p)
    stream.sync()
    first = o.read(np.float32)
    close(first.reshape(q.shape), attention(c, q, 1, heads, D ** -0.5, False))
    for _ in range(3):  # the same bits every time
        hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, p)
        stream.sync()
        assert np.array_equal(o.read(np.uint32), first.view(np.uint32))


MANY = [  # requests, heads, kv heads, head width, page, rows, longest
    (17, 8, 2, 256, 16, 1, 700),    # a round of workgroups holds every part
    (70, 2, 1, 256, 16, 1, 900),    # more requests than lanes; joined by whole rows
    (70, 6, 2, 192, 16, 1, 500),
    (65, 12, 3, 128, 16, 3, 300),
    (300, 4, 1, 128, 16, 1, 260),   # more requests than are kept in registers
    (300, 4, 2, 64, 16, 1, 150),
    (260, 4, 4, 64, 6, 2, 100),     # pages of no power of two
    (200, 16, 8, 128, 32, 1, 400),  # more columns than two rounds: no request is cut
    (33, 8, 2, 128, 16, 9, 600),    # 36 pairs of a kv head: three blocks of 16, each a wave's
    (21, 16, 4, 128, 16, 8, 500),   # two blocks a wave
    (9, 16, 4, 64, 16, 17, 400),    # five, in pairs
]


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("requests,heads,nk,D,bs,rows,longest", MANY)
def test_batches_of_ragged_requests(dev, stream, dtype, requests, heads, nk, D, bs, rows, longest):
    """Every way that the work of a batch is cut: lengths from none to the longest, which one request has alone."""
    rng = np.random.default_rng(requests + D)
    positions = rng.integers(-rows - 1, longest // 3, requests)
    positions[0], positions[-1], positions[requests // 2] = 0, -rows - 3, longest
    c = Cache(dev, dtype, bs, longest + rows, nk, D, requests, positions, seed=rows, shared=True,
              pages=-(-(longest + rows) // bs) + 3, fill=q8_fill() if dtype == Q8 else f16_fill)
    n = requests * rows
    q = rng.normal(0, 1, (n, heads, D)).astype(np.float32)
    o = dev.upload(np.full(n * heads * D, 7.5, np.float32))
    p = c.params(rows, heads=heads, scale=D ** -0.5)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, p)
    stream.sync()
    got, want = o.read(np.float32).reshape(q.shape), attention(c, q, rows, heads, D ** -0.5, False)
    close(got, want)
    for j in range(requests):  # no request hides in the others' norm
        close(got[j * rows:(j + 1) * rows], want[j * rows:(j + 1) * rows])
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, p)
    stream.sync()
    assert np.array_equal(o.read(np.uint32), got.reshape(-1).view(np.uint32))


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("requests,heads,nk,D,rows", [(17, 8, 2, 256, 1), (18, 4, 2, 192, 2), (13, 6, 3, 128, 1), (37, 2, 1, 64, 3)])
def test_one_long_request_among_short_ones(dev, stream, dtype, requests, heads, nk, D, rows):
    """The long one is cut into more parts than a wave has lanes, though a request of the batch has few on average."""
    longest = 9000
    positions = np.random.default_rng(D).integers(0, 60, requests)
    positions[requests // 3] = longest
    c = Cache(dev, dtype, 64, longest + rows, nk, D, requests, positions, seed=rows, shared=True,
              pages=-(-(longest + rows) // 64) + 2, fill=q8_fill() if dtype == Q8 else f16_fill)
    q = np.random.default_rng(2).normal(0, 1, (requests * rows, heads, 2 * D)).astype(np.float32)
    o = dev.alloc(requests * rows * heads * D * 4)
    p = c.params(rows, heads=heads, gated=True, scale=D ** -0.5)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, p)
    stream.sync()
    got = o.read(np.float32).reshape(requests * rows, heads, D)
    want = attention(c, q, rows, heads, D ** -0.5, True)
    for j in range(requests):
        close(got[j * rows:(j + 1) * rows], want[j * rows:(j + 1) * rows])


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("scale,size", [(0.0, 1.0), (-0.0, 1.0), (-0.09, 1.0), (1e-25, 1e-25), (-1e-30, 1e-15), (1e-40, 1.0)])
def test_scales_of_zero_below_and_next_to_nothing(dev, stream, dtype, scale, size):
    """The mean of the values, or the signed scores; keys a row does not see stay out."""
    heads, nk, D, rows = 8, 2, 128, 3
    c = Cache(dev, dtype, 16, 200, nk, D, 3, [130, 0, -2], fill=q8_fill() if dtype == Q8 else f16_fill)
    q = (size * np.random.default_rng(3).normal(0, 1, (3 * rows, heads, D))).astype(np.float32)
    o = dev.upload(np.full(q.shape, 2.5, np.float32))
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=scale))
    stream.sync()
    want = attention(c, q, rows, heads, scale, False)
    assert (want[6:8] == 0).all() and (want[8] != 0).any()
    close(o.read(np.float32).reshape(q.shape), want)


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("heads,nk,D,rows", [(8, 2, 128, 8), (8, 2, 64, 5), (8, 2, 256, 6), (4, 2, 128, 3)])
def test_an_infinity_that_only_later_rows_see(dev, stream, dtype, heads, nk, D, rows):
    """A value that is not finite, at the position of a row in the middle: the earlier rows keep theirs."""
    c = Cache(dev, dtype, 16, 300, nk, D, 2, [250, 31], fill=q8_fill() if dtype == Q8 else f16_fill)
    q = np.random.default_rng(2).normal(0, 1, (2 * rows, heads, D)).astype(np.float32)
    mid = rows // 2
    bad = np.ones(c.kvd, np.float32)
    bad[:D] = np.inf           # the first kv head's
    for j in range(2):
        c.put(1, j, int(c.positions[j, 1]) + mid, bad)
    c.upload()
    want = attention(c, q, rows, heads, D ** -0.5, False)
    o = dev.alloc(q.nbytes)
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=D ** -0.5))
    stream.sync()
    got = o.read(np.float32).reshape(q.shape)
    assert np.isfinite(want[:mid]).all() and not np.isfinite(want[mid:rows, : heads // nk]).any()
    close(got, want)


@pytest.mark.parametrize("dtype", [Q8, F16])
def test_pools_past_four_gigabytes(dev, stream, dtype):
    """Pages whose byte offsets pass 32 bits, signed and unsigned."""
    nk, D, heads, bs = 8, 128, 8, 16
    token = {F16: 2048, Q8: 1088}[dtype]
    per_page = bs * token
    pages = (9 << 29) // per_page + 8  # 4.5 GiB
    table = np.array([[(1 << 31) // per_page + 1, pages - 1, (1 << 32) // per_page + 1, 3]], np.int32)
    pools = [dev.alloc(pages * per_page) for _ in range(2)]
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (2, 64, nk * D)).astype(np.float32)
    p = hip.kv_params(dtype, bs, 64, nk, D, 64)
    tb, pos = dev.upload(table), dev.upload(np.zeros(2, np.int32))
    hip.kv_append(stream, dev.upload(x[0]), dev.upload(x[1]), *pools, tb, pos, p)
    out = [dev.alloc(x[0].nbytes) for _ in range(2)]
    hip.kv_read(stream, *out, *pools, tb, p)
    q = rng.normal(0, 1, (1, heads, D)).astype(np.float32)
    o = dev.alloc(q.nbytes)
    hip.attn_decode(stream, o, dev.upload(q), *pools, tb, dev.upload(np.array([0, 63], np.int32)),
                    hip.kv_params(dtype, bs, 64, nk, D, 1, heads=heads, scale=D ** -0.5))
    stream.sync()
    small = Cache(dev, dtype, bs, 64, nk, D, 1, [63])
    for t in range(64):
        for side in range(2):
            small.put(side, 0, t, x[side, t])
    for side in range(2):
        got = out[side].read(np.float32).reshape(64, -1)
        assert np.array_equal(got, [small.row(side, 0, t) for t in range(64)])
    close(o.read(np.float32).reshape(q.shape), attention(small, q, 1, heads, D ** -0.5, False))
    for b in pools:
        b.free()


# --------------------------------------------------------------- runs together

def test_decode_steps_append_attend_read(dev, stream):
    """Decode steps as a server runs them, the device's positions moved by ADVANCE: captured once, replayed, with eager
    work between, against the host's own cache."""
    heads, nk, D, bs, cap = 8, 2, 128, 16, 120
    start = [0, 15, 63]
    c = Cache(dev, Q8, bs, cap, nk, D, 3, start, fill=q8_fill())
    rng = np.random.default_rng(5)
    kb, vb, qb = dev.alloc(3 * c.kvd * 4), dev.alloc(3 * c.kvd * 4), dev.alloc(3 * heads * D * 4)
    ob, rb = dev.alloc(3 * heads * D * 4), dev.alloc(3 * c.kvd * 4)
    result = dev.upload(np.zeros((3, 4), np.int32))  # nothing accepted beyond the row itself
    own = lambda *b: list(b) + [None] * (15 - len(b)) + [c.b_pos]  # noqa: E731
    u, n = [bs, cap, Q8, 3 << 8], [nk, heads, D, c.kvd, 1, 0]
    plan = hip.Plan(dev)
    plan.add(hip.OP["KV_APPEND"], own(kb, vb, *c.b_pool, c.b_table), n=n, u=u, flags=hip.FLAG_OWN_POS)
    plan.add(hip.OP["ATTN_DECODE"], own(qb, *c.b_pool, ob, c.b_table), n=n, u=u, f=[D ** -0.5], flags=hip.FLAG_OWN_POS)
    plan.add(hip.OP["KV_READ"], own(c.b_pool[0], None, rb, None, c.b_table), n=n, u=u, flags=hip.FLAG_OWN_POS)
    plan.add(hip.OP["ADVANCE"], [c.b_pos, result], n=[1], u=[3])
    graph = hip.Graph(plan, stream, None)
    other = dev.alloc(3 * heads * D * 4)
    for step in range(12):
        k, v = rng.normal(0, 1, (2, 3, c.kvd)).astype(np.float32)
        q = rng.normal(0, 1, (3, heads, D)).astype(np.float32)
        for b, x in ((kb, k), (vb, v), (qb, q)):
            b.write(x)
        (graph.replay if step % 3 else plan.execute)(stream)
        # eager work that uses the stream's own workspace, between the replays
        hip.attn_decode(stream, other, qb, *c.b_pool, c.b_table, c.b_pos,
                        c.params(1, heads=heads, scale=D ** -0.5, displacement=-1))
        stream.sync()
        for j in range(3):
            c.put(0, j, start[j] + step, k[j])
            c.put(1, j, start[j] + step, v[j])
        assert np.array_equal(c.read_pool(0), c.pool[0]) and np.array_equal(c.read_pool(1), c.pool[1])
        want = attention(c, q, 1, heads, D ** -0.5, False)
        got = ob.read(np.float32).reshape(q.shape)
        close(got, want)
        assert np.array_equal(other.read(np.uint32), got.reshape(-1).view(np.uint32))
        assert np.array_equal(rb.read(np.float32).reshape(3, -1), [c.row(0, j, start[j] + step) for j in range(3)])
        c.positions[:, 1] += 1
        assert np.array_equal(c.b_pos.read(np.int32).reshape(3, 2), c.positions)
    graph.destroy()
    plan.destroy()


def test_two_streams_at_once(dev, stream):
    """Calls that overlap on two streams have workspaces of their own."""
    heads, nk, D = 16, 4, 256
    s2 = hip.Stream(dev)
    caches = [Cache(dev, Q8, 16, 1500, nk, D, 2, [1400, 900], seed=s, fill=q8_fill()) for s in range(2)]
    q = np.random.default_rng(1).normal(0, 1, (2, heads, D)).astype(np.float32)
    qb, outs = dev.upload(q), [dev.alloc(q.nbytes) for _ in range(2)]
    for _ in range(20):
        for s, c, o in zip((stream, s2), caches, outs):
            hip.attn_decode(s, o, qb, *c.b_pool, c.b_table, c.b_pos, c.params(1, heads=heads, scale=D ** -0.5))
    stream.sync()
    s2.sync()
    for c, o in zip(caches, outs):
        close(o.read(np.float32).reshape(q.shape), attention(c, q, 1, heads, D ** -0.5, False))
    s2.destroy()


def test_graphs_of_one_plan_and_of_two(dev, stream):
    """Two captures replayed on two streams at once, of one plan and of two: no workspace is shared between them; a
    graph outlives a plan that grew, and the plan itself."""
    heads, nk, D = 8, 2, 128
    s2 = hip.Stream(dev)
    q = np.random.default_rng(1).normal(0, 1, (1, heads, D)).astype(np.float32)
    dyn = [dev.upload(np.array([0, p], np.int32)) for p in (700, 333)]
    c = Cache(dev, Q8, 16, 800, nk, D, 1, [700], fill=q8_fill())
    qb, ob = dev.upload(q), dev.alloc(q.nbytes)
    args = dict(n=[nk, heads, D, c.kvd, 1, 0], u=[16, 800, Q8, 0], f=[D ** -0.5])
    plan = hip.Plan(dev)
    plan.add(hip.OP["ATTN_DECODE"], [qb, *c.b_pool, ob, c.b_table], **args)
    wants = []
    for p in (700, 333):
        c.positions[:, 1] = p
        wants.append(attention(c, q, 1, heads, D ** -0.5, False))
    # the same plan captured for two positions: only the output is shared
    graphs = [hip.Graph(plan, s, d) for s, d in zip((stream, s2), dyn)]
    for g, s, w in zip(graphs, (stream, s2), wants):
        for _ in range(3):
            g.replay(s)
            s.sync()
            close(ob.read(np.float32).reshape(q.shape), w)
    # the plan grows a larger workspace and runs; the first captures still replay, and do so after its end
    wide = Cache(dev, Q8, 16, 9000, nk, D, 1, [8000], fill=q8_fill())
    big = dev.upload(np.random.default_rng(2).normal(0, 1, (64, heads, D)).astype(np.float32))
    bo = dev.alloc(64 * heads * D * 4)
    plan.add(hip.OP["ATTN_DECODE"], [big, *wide.b_pool, bo, wide.b_table], n=[nk, heads, D, c.kvd, 64, 0],
             u=[16, 9000, Q8, 0], f=[D ** -0.5])
    plan.execute(stream, position=690)
    stream.sync()
    for _ in range(2):
        graphs[0].replay(stream)
        stream.sync()
        close(ob.read(np.float32).reshape(q.shape), wants[0])
    plan.destroy()
    for _ in range(2):
        graphs[1].replay(s2)
        s2.sync()
        close(ob.read(np.float32).reshape(q.shape), wants[1])
    for g in graphs:
        g.destroy()
    # two plans, overlapping
    outs, plans, graphs = [dev.alloc(q.nbytes) for _ in range(2)], [], []
    for o, d, s in zip(outs, dyn, (stream, s2)):
        plans.append(hip.Plan(dev))
        plans[-1].add(hip.OP["ATTN_DECODE"], [qb, *c.b_pool, o, c.b_table], **args)
        graphs.append(hip.Graph(plans[-1], s, d))
    for _ in range(20):
        for g, s in zip(graphs, (stream, s2)):
            g.replay(s)
    stream.sync()
    s2.sync()
    for o, w in zip(outs, wants):
        close(o.read(np.float32).reshape(q.shape), w)
    for g in graphs:
        g.destroy()
    for p in plans:
        p.destroy()
    s2.destroy()


# ------------------------------------------- the v10 cache ops and ATTN_VERIFY

@pytest.mark.parametrize("heads,nk,D,gated", [(8, 2, 256, True), (12, 4, 64, False), (6, 2, 192, True)])
def test_v10_cache_ops_over_q8_0(dev, stream, heads, nk, D, gated):
    """KV_WRITE_BATCH_PAGED and ATTENTION_PREFILL_PAGED for a chunk, then KV_WRITE_PAGED and ATTENTION_PAGED token by
    token, the position the plan's."""
    bs, cap, rows = 16, 80, 11
    c = Cache(dev, Q8, bs, cap, nk, D, 1, [0], fill=q8_fill())
    rng = np.random.default_rng(5)
    width = 2 * D if gated else D
    kb, vb, qb = dev.alloc(rows * c.kvd * 4), dev.alloc(rows * c.kvd * 4), dev.alloc(rows * heads * width * 4)
    ob = dev.alloc(rows * heads * D * 4)
    gate = 0 if gated else 1
    chunk, token = hip.Plan(dev), hip.Plan(dev)
    chunk.add(hip.OP["KV_WRITE_BATCH_PAGED"], [kb, vb, *c.b_pool, c.b_table], n=[c.kvd, rows], u=[bs, cap, Q8])
    chunk.add(hip.OP["ATTENTION_PREFILL_PAGED"], [qb, *c.b_pool, ob, c.b_table], n=[nk, heads, D, c.kvd, rows, 0],
              u=[bs, cap, Q8, gate], f=[D ** -0.5])
    token.add(26, [kb, vb, *c.b_pool, c.b_table], n=[c.kvd], u=[bs, cap, Q8])
    token.add(27, [qb, *c.b_pool, ob, None, c.b_table], n=[nk, heads, D, c.kvd, cap], u=[bs, cap, Q8, gate],
              f=[D ** -0.5])
    pos = 0
    for plan, n in ((chunk, rows), (chunk, rows), (token, 1), (token, 1), (token, 1)):
        k, v = rng.normal(0, 1, (2, n, c.kvd)).astype(np.float32)
        q = rng.normal(0, 1, (n, heads, width)).astype(np.float32)
        for b, x in ((kb, k), (vb, v), (qb, q)):
            b.write(x)
        plan.execute(stream, position=pos)
        stream.sync()
        for r in range(n):
            c.put(0, 0, pos + r, k[r])
            c.put(1, 0, pos + r, v[r])
        c.positions[0, 1] = pos
        for side in range(2):
            assert np.array_equal(c.read_pool(side), c.pool[side])
        close(ob.read(np.float32)[:n * heads * D].reshape(n, heads, D), attention(c, q, n, heads, D ** -0.5, gated))
        pos += n
    chunk.destroy()
    token.destroy()


@pytest.mark.parametrize("heads,nk,D,rot,rows", [(8, 2, 256, 64, 5), (6, 2, 128, 128, 3), (4, 4, 64, 20, 1),
                                                 (16, 4, 256, 64, 17)])
def test_attn_verify_over_q8_0(dev, stream, heads, nk, D, rot, rows):
    """ATTN_VERIFY's norms, rotations, write and attention are those of the separate ops."""
    bs, cap, positions = 16, 300, [200, 0, 77]
    a = Cache(dev, Q8, bs, cap, nk, D, 3, positions, fill=q8_fill())
    b = Cache(dev, Q8, bs, cap, nk, D, 3, positions, fill=q8_fill())
    rng = np.random.default_rng(rot)
    n = 3 * rows
    q = rng.normal(0, 2, (n, heads, 2 * D)).astype(np.float32)
    kb, vb = (dev.upload(rng.normal(0, 2, (n, a.kvd)).astype(np.float32)) for _ in range(2))
    qn, kn = (dev.upload((1 + 0.1 * rng.normal(0, 1, D)).astype(np.float32)) for _ in range(2))
    qb, rope = dev.upload(q), dev.alloc(n * rot // 2 * 8)
    out, out2 = dev.alloc(n * heads * D * 4), dev.alloc(n * heads * D * 4)
    plan = hip.Plan(dev)
    own = lambda c, *bufs: list(bufs) + [None] * (15 - len(bufs)) + [c.b_pos]  # noqa: E731
    u = rot | 3 << 8 | rows << 20
    plan.add(hip.OP["ROPE_TABLE"], own(a, rope), n=[rows, rot, 0, 3, rows], f=[1e4], flags=hip.FLAG_OWN_POS)
    plan.add(hip.OP["ATTN_VERIFY"], own(a, qb, kb, vb, *a.b_pool, out, a.b_table, qn, kn, rope),
             n=[nk, heads, D, a.kvd, rows, 0], u=[bs, cap, Q8, u], f=[D ** -0.5, 1e-6], flags=hip.FLAG_OWN_POS)
    plan.execute(stream)
    stream.sync()
    # the queries' norm in place of their q half, their rotation on the host, the gate as it is
    qd = dev.upload(np.ascontiguousarray(q[..., :D]))
    norm = hip.Plan(dev)
    norm.add(hip.OP["RMSNORM_HEADS_BATCH"], [qd, qn, qd], n=[D, heads, D, n], f=[1e-6])
    norm.execute(stream)
    hip.kv_append(stream, kb, vb, *b.b_pool, b.b_table, b.b_pos, b.params(rows, rope_dim=rot), k_norm=kn, rope=rope)
    stream.sync()
    for side in range(2):
        assert np.array_equal(a.read_pool(side), b.read_pool(side))
    y = qd.read(np.float32).reshape(n, heads, D)
    cs = rope.read(np.float32).reshape(n, 1, rot // 2, 2)
    lo, hi = y[..., :rot // 2].copy(), y[..., rot // 2:rot].copy()
    y[..., :rot // 2] = lo * cs[..., 0] - hi * cs[..., 1]
    y[..., rot // 2:rot] = lo * cs[..., 1] + hi * cs[..., 0]
    hip.attn_decode(stream, out2, dev.upload(np.concatenate([y, q[..., D:]], 2)), *b.b_pool, b.b_table, b.b_pos,
                    b.params(rows, heads=heads, gated=True, scale=D ** -0.5))
    stream.sync()
    assert np.array_equal(out.read(np.uint32), out2.read(np.uint32))
    plan.destroy()
    norm.destroy()


# ------------------------------------------------------------------- the engine

def _logits_close(got, want, what):
    """The bar of the other cache formats: 1e-2 of a logit, or of the row's rms."""
    got, want = np.atleast_2d(got), np.atleast_2d(want)
    for r in range(want.shape[0]):
        rms = math.sqrt(float(np.mean(want[r].astype(np.float64) ** 2)))
        err = np.abs(got[r].astype(np.float64) - want[r])
        assert np.all(err <= 1e-2 * (np.abs(want[r]) + rms)), (what, r, float(err.max()), rms)


def test_engine_over_a_q8_0_cache(dev):
    """Prefill, verify steps and a forked request with kv_dtype Q8_0 against the CPU decoder with its Q8_0 cache."""
    cfg = replace(Mdl.TINY, kv_dtype=Q8, batch=2)
    w = Mdl.make_weights(cfg, seed=11)
    eng, orc = Mdl.Engine(dev, cfg, w), O.Q35(cfg, w, kv_format=2)
    rng = np.random.default_rng(2)
    prompt = rng.integers(0, cfg.vocab, 53).astype(np.int32)
    _logits_close(eng.prefill(prompt[:-1]), orc.forward(prompt[:-1]), "prefill")
    pending = int(prompt[-1])
    for step, k in enumerate((4, 0, 7)):
        rows = np.concatenate([[pending], rng.integers(0, cfg.vocab, k)]).astype(np.int32)
        res = eng.verify(rows)
        snap, pos = orc.snapshot()
        want = orc.forward(rows, all_logits=True)
        _logits_close(eng.logits(k + 1), want, f"verify {step}")
        orc.restore(snap, pos)
        orc.forward(rows[:int(res[0]) + 1])
        assert eng.position == orc.position
        pending = int(res[1])
    # a second request takes the first one's pages (the partial last one is copied), both go on alike
    eng.fork(0, 1)
    rows = np.concatenate([[pending], rng.integers(0, cfg.vocab, 3)]).astype(np.int32)
    eng.step_batch(np.stack([rows, rows]), accept=Mdl.accept_struct())
    got = eng.logits(8)
    want = orc.forward(rows, all_logits=True)
    _logits_close(got[:4], want, "after the fork")
    assert np.array_equal(got[:4], got[4:])
    eng.close()
    orc.close()


# ----------------------------------------------- keys and values that are not finite

ODD = [  # heads, kv heads, head width, page, rows, context: one operand for both halves, one and two blocks a wave, ...
    (4, 2, 128, 16, 3, 90),
    (8, 2, 128, 16, 3, 90),
    (16, 4, 128, 16, 8, 500),
    (8, 2, 64, 64, 9, 40),
    (6, 2, 192, 16, 4, 200),
    (8, 2, 256, 16, 6, 1500),   # several parts
    (8, 2, 256, 16, 2, 64),
    (8, 2, 128, 48, 5, 300),    # pages of no power of two
]


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan, 1e10])
@pytest.mark.parametrize("heads,nk,D,bs,rows,context", ODD)
def test_a_value_that_is_not_finite_keeps_to_its_dims(dev, stream, dtype, bad, heads, nk, D, bs, rows, context):
    """In the rows that see it, its dim (F16) or its block of 32 dims (Q8_0), wherever its token lies: among the newest
    rows, where some see it and some do not, before them, and long before."""
    ends = [context + rows // 2, context + rows - 1, context, context - 1, context // 2, 0]
    c = Cache(dev, dtype, bs, context + rows + 2, nk, D, len(ends), [context] * len(ends), seed=D,
              fill=q8_fill() if dtype == Q8 else f16_fill)
    for j, p in enumerate(ends):
        row = c.row(1, j, p).copy()
        row[D + 40] = bad   # of the second kv head
        c.put(1, j, p, row)
    c.upload()
    q = np.random.default_rng(rows).normal(0, 1, (len(ends) * rows, heads, D)).astype(np.float32)
    o = dev.upload(np.full(q.shape, 2.5, np.float32))
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=D ** -0.5))
    stream.sync()
    got, want = o.read(np.float32).reshape(q.shape), attention(c, q, rows, heads, D ** -0.5, False)
    width = 32 if dtype == Q8 else 1
    for j, p in enumerate(ends):
        seen = sum(context + r >= p for r in range(rows))
        assert (~np.isfinite(want[j * rows:(j + 1) * rows])).sum() == seen * heads // nk * width
        close(got[j * rows:(j + 1) * rows], want[j * rows:(j + 1) * rows])


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("heads,nk,D,bs,rows,context", ODD)
def test_a_key_that_is_not_finite_makes_its_rows_nan(dev, stream, dtype, heads, nk, D, bs, rows, context):
    """Whether its score would be an infinity of either sign or a NaN: the rows that see it, of its kv head."""
    rng = np.random.default_rng(rows)
    ends = [context + rows // 2, context + rows - 1, context - 1, context // 2, 0, None]
    c = Cache(dev, dtype, bs, context + rows + 2, nk, D, len(ends), [context] * len(ends), seed=D,
              fill=q8_fill() if dtype == Q8 else f16_fill)
    q = rng.normal(0, 1, (len(ends) * rows, heads, D)).astype(np.float32)
    # dim 17: both halves of the query are of one sign, which differs between the heads
    q[..., 17] = np.where(np.arange(heads) % 2, 1, -1) * np.float32(1 + 2.0 ** -12)
    scale = np.float32(D ** -0.5)
    for j, p in enumerate(ends):
        for t in range(context + rows) if p is None else [p]:  # the last request: every key
            row = c.row(0, j, t).copy()
            if dtype == Q8:
                row[D:D + 32] *= 1e12   # an infinite scale, digits of both signs
            else:
                row[D + 17] = -np.inf
            c.put(0, j, t, row)
    c.upload()
    want = attention(c, q, rows, heads, scale, False)
    for j, p in enumerate(ends):
        for r in range(rows):
            if p is None or context + r >= p:
                want[j * rows + r, heads // nk:2 * heads // nk] = np.nan
    o = dev.upload(np.full(q.shape, 2.5, np.float32))
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=scale))
    stream.sync()
    got = o.read(np.float32).reshape(q.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    close(got, want)


# ----------------------------------------------------------- the reference's codec

def test_append_next_to_the_references_quotient(dev, stream):
    """The cached bytes are those of the reference's codec, which takes s as max / 127 where the append takes max * (1 / 127),
    but for what the last bits of s decide. Each s is within 2^-24 (the quotient) and 2 * 2^-24 (the constant and the
    product) of max / 127, so that they differ by at most 3 * 2^-24 of it: the stored halves differ only where max / 127 is
    that close to the middle of two. x / s is rounded to 2^-24 again, twice 2^-24 for the pair: two digits differ, by one,
    only where x / s, up to 128, is within 5 * 128 * 2^-24 of a half."""
    rng = np.random.default_rng(9)
    x = rng.normal(0, 1, (600, 2, 256)) * np.exp(rng.normal(0, 2, (600, 2, 1)))
    special = _special_blocks()
    special = special[np.isfinite(special).all(1) & (np.abs(special).max(1) > 2.0 ** -100)]
    special = special[:len(special) // 8 * 8].reshape(-1, 256)
    x[0, 0, :32] = 0
    x = np.concatenate([x.reshape(-1, 256).astype(np.float32), special])
    c = Cache(dev, Q8, 16, len(x), 2, 128, 1, [0])
    hip.kv_append(stream, dev.upload(x), dev.upload(x), *c.b_pool, c.b_table, c.b_pos, c.params(len(x)))
    stream.sync()
    c.pool = [c.read_pool(0), c.read_pool(1)]
    assert np.array_equal(*c.pool)
    n = c.kvd
    digits, scales = np.zeros(x.shape, np.int8), np.zeros((len(x), n // 32), np.uint16)
    for p in range(len(x)):
        page, t = c.at(0, p)
        stored = c.pool[0][page, t * n:(t + 1) * n].view(np.int8)
        digits[p] = stored.reshape(-1, 16, 4).swapaxes(1, 2).reshape(-1)
        scales[p] = c.pool[0][page, 16 * n + t * n // 16:16 * n + (t + 1) * n // 16].copy().view(np.uint16)
    want_digits, want_scales = O.kv_encode_rows(x)
    s = np.abs(x.astype(np.float64)).reshape(len(x), -1, 32).max(2) / 127
    other = scales != want_scales
    low = np.minimum(scales, want_scales)
    assert (np.maximum(scales, want_scales) - low)[other].max(initial=0) <= 1
    with np.errstate(over="ignore", invalid="ignore"):
        middle = (low.view(np.float16).astype(np.float64) + (low + 1).astype(np.uint16).view(np.float16)) / 2
    assert (np.abs(s - middle)[other] <= 3 * 2.0 ** -24 * s[other]).all()
    with np.errstate(invalid="ignore"):
        t = np.abs(x.astype(np.float64)).reshape(*s.shape, 32) / s[..., None]
    other = (digits != want_digits).reshape(t.shape)
    assert np.abs(digits.astype(int) - want_digits).max() <= 1
    assert (np.abs(t - np.floor(t) - 0.5)[other] <= 5 * 128 * 2.0 ** -24).all()
    ordinary = np.arange(len(x)) < 1200
    assert (digits == want_digits)[ordinary].mean() > 0.99999 and (scales == want_scales)[ordinary].mean() > 0.999


def test_two_captures_of_one_plan_at_once(dev, stream):
    """The second capture, of the plan after it grew, runs what the first does and more; both fill the shared output with
    the same values, so that only a workspace in common could make them wrong."""
    heads, nk, D, rounds = 8, 2, 128, 12
    s2 = hip.Stream(dev)
    rng = np.random.default_rng(1)
    plan, caches, outs, wants = hip.Plan(dev), [], [], []
    streams, graphs = (stream, s2), []
    for positions, s in zip(([2900, 1500], [700, 2600]), streams):
        c = Cache(dev, Q8, 16, 3000, nk, D, 2, positions, seed=positions[0], fill=q8_fill())
        q = rng.normal(0, 1, (2, heads, D)).astype(np.float32)
        o = dev.upload(np.zeros(q.shape, np.float32))
        plan.add(hip.OP["ATTN_DECODE"], [dev.upload(q), *c.b_pool, o, c.b_table] + [None] * 10 + [c.b_pos],
                 n=[nk, heads, D, c.kvd, 1, 0], u=[16, 3000, Q8, 2 << 8], f=[D ** -0.5], flags=hip.FLAG_OWN_POS)
        graphs.append(hip.Graph(plan, s, None))
        caches.append(c)
        outs.append(o)
        wants.append(attention(c, q, 1, heads, D ** -0.5, False))
    for _ in range(rounds):
        for o in outs:
            o.write(np.full(wants[0].shape, np.nan, np.float32))
        for _ in range(8):
            for g, s in zip(graphs, streams):
                g.replay(s)
        stream.sync()
        s2.sync()
        for o, w in zip(outs, wants):
            close(o.read(np.float32).reshape(w.shape), w)
    for g in graphs:
        g.destroy()
    plan.destroy()
    s2.destroy()


@pytest.mark.parametrize("dtype", [Q8, F16])
@pytest.mark.parametrize("requests,heads,nk,D,rows", [(260, 16, 4, 256, 1), (52, 16, 4, 256, 17), (520, 8, 4, 64, 1)])
def test_one_long_request_among_more_than_are_cut(dev, stream, dtype, requests, heads, nk, D, rows):
    """So many requests that each is one part, whatever its length."""
    longest = 2500
    positions = np.random.default_rng(D).integers(0, 30, requests)
    positions[requests // 3] = longest
    c = Cache(dev, dtype, 64, longest + rows, nk, D, requests, positions, seed=rows, shared=True,
              pages=-(-(longest + rows) // 64) + 2, fill=q8_fill() if dtype == Q8 else f16_fill)
    q = np.random.default_rng(2).normal(0, 1, (requests * rows, heads, D)).astype(np.float32)
    o = dev.upload(np.full(q.shape, 7.5, np.float32))
    hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=D ** -0.5))
    stream.sync()
    got, want = o.read(np.float32).reshape(q.shape), attention(c, q, rows, heads, D ** -0.5, False)
    for j in range(requests):
        close(got[j * rows:(j + 1) * rows], want[j * rows:(j + 1) * rows])


@pytest.mark.parametrize("heads,nk,D,rows", [(8, 2, 128, 1), (8, 2, 256, 5), (16, 4, 64, 8)])
@pytest.mark.parametrize("octaves", [6, 13, 20, 27])
def test_value_scales_octaves_apart(dev, stream, octaves, heads, nk, D, rows):
    """What the header states of blocks next to much larger ones. A weight times a value scale is two halves: off by 2^-22
    of itself, or by half a step of 2^-24. Weights are in units in which the largest, 1, times the power of two above the
    largest scale S is 2^10 at the least: half a step is at most 2^-25 2^-10 2 S = 2^-34 S there. So an output, sum of
    w_k s_k digit_k over sum of w_k, is off by 2^-34 S sum |digit_k| / sum w_k beside the relative 2^-18 of every term."""
    c = Cache(dev, Q8, 16, 400, nk, D, 2, [350, 33], fill=q8_fill())
    rng = np.random.default_rng(octaves)
    n = 16 * c.kvd
    s = rng.uniform(1, 2, (c.pages, 16, c.kvd // 32)) * 2.0 ** 10
    s[..., ::2] *= 2.0 ** -octaves
    c.pool[1][:, n:] = s.astype(np.float16).reshape(c.pages, -1).view(np.uint8)
    c.upload()
    q = rng.normal(0, 1, (2 * rows, heads, D)).astype(np.float32)
    o = dev.alloc(q.nbytes)
    for scale in (0.0, D ** -0.5):
        hip.attn_decode(stream, o, dev.upload(q), *c.b_pool, c.b_table, c.b_pos, c.params(rows, heads=heads, scale=scale))
        stream.sync()
        got, want = o.read(np.float32).reshape(q.shape), attention(c, q, rows, heads, scale, False)
        for j in range(2):
            K, V = (np.array([c.row(side, j, p) for p in range(c.positions[j, 1] + rows)], np.float64).reshape(-1, nk, D)
                    for side in range(2))
            steps = np.array([s[c.at(j, p)].repeat(32) for p in range(len(V))]).reshape(V.shape)  # a digit's
            for r in range(rows):
                m = c.positions[j, 1] + r + 1
                for h in range(heads):
                    g = h // (heads // nk)
                    t = K[:m, g] @ q[j * rows + r, h].astype(np.float64) * scale
                    w = np.exp(t - t.max())
                    off = 2.0 ** -34 * steps.max() * (np.abs(V[:m, g]) / steps[:m, g]).sum(0) + TOL * (w @ np.abs(V[:m, g]))
                    d = np.abs(got[j * rows + r, h] - want[j * rows + r, h])
                    assert (d <= off / w.sum()).all(), (j, r, h, scale, (d * w.sum() / off).max())


@pytest.mark.parametrize("dtype", [Q8, F16])
def test_v10_single_token_ops_refuse_positions_past_the_capacity(dev, stream, dtype):
    """In every format; the last position is served, and a refused write leaves the pools as they were."""
    heads, nk, D, bs, cap = 8, 2, 128, 16, 70
    c = Cache(dev, dtype, bs, cap, nk, D, 1, [cap - 1], fill=q8_fill() if dtype == Q8 else f16_fill)
    rng = np.random.default_rng(3)
    k, v = rng.normal(0, 1, (2, 1, c.kvd)).astype(np.float32)
    q = rng.normal(0, 1, (1, heads, D)).astype(np.float32)
    o = dev.upload(np.zeros(q.shape, np.float32))
    scores = dev.alloc(heads * cap * 4)
    write, attend = hip.Plan(dev), hip.Plan(dev)
    write.add(26, [dev.upload(k), dev.upload(v), *c.b_pool, c.b_table], n=[c.kvd], u=[bs, cap, dtype])
    attend.add(27, [dev.upload(q), *c.b_pool, o, scores, c.b_table], n=[nk, heads, D, c.kvd, cap], u=[bs, cap, dtype, 1],
               f=[D ** -0.5])
    for plan in (write, attend):
        for position in (cap, cap + 9, 2 ** 31 - 1):
            with pytest.raises(hip.HipError, match="capacity"):
                plan.execute(stream, position=position)
    stream.sync()
    for side in range(2):
        assert np.array_equal(c.read_pool(side), c.pool[side])
    write.execute(stream, position=cap - 1)
    attend.execute(stream, position=cap - 1)
    stream.sync()
    c.put(0, 0, cap - 1, k[0])
    c.put(1, 0, cap - 1, v[0])
    for side in range(2):
        assert np.array_equal(c.read_pool(side), c.pool[side])
    close(o.read(np.float32).reshape(q.shape), attention(c, q, 1, heads, D ** -0.5, False))
    write.destroy()
    attend.destroy()

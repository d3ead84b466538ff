"""GPU checks of ragged batches against plain implementations in 64 bits: tables
and slots, append by slot, the convolution and the gated delta rule over rows
without padding, single tokens, and the path through all of them.

Tolerances. u = 2^-24 is half a step of float32. A dot product of D float32 terms is
off by at most D u of the sum of its terms' sizes; a 16-bit output by half a step of
its own more. For the delta rule see `_bounds`."""
from __future__ import annotations

import math

import numpy as np
import pytest

from yuuka_amd import hip

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {hip.F32: U, hip.F16: 2.0 ** -11, hip.BF16: 2.0 ** -8}
TYPES = [hip.F32, hip.F16, hip.BF16]


def to_bits(x, dtype):
    """Float32 values as the type's bytes, to the nearest, ties to even."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == hip.F32:
        return x
    if dtype == hip.F16:
        return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    up = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), up).astype(np.uint16)


def from_bits(b, dtype):
    if dtype == hip.BF16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


def np_type(dtype):
    return {hip.F32: np.float32, hip.F16: np.float16, hip.BF16: np.uint16}[dtype]


def i32(*v):
    return np.array(v, np.int32)


def offsets_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


# ----------------------------------------------------------- tables and slots

def plan_reference(positions, counts, blocks, table, free, pool, rows, block, capacity):
    table, blocks_out = table.copy(), blocks.copy()
    entries = table.shape[1]
    offsets, info, slots = [0], np.full((rows, 2), -1, np.int64), np.full(rows, -1, np.int64)
    nxt, last = max(0, int(pool[0])), min(int(pool[1]), len(free))
    first_free, missing = nxt, 0
    for j, (p, n) in enumerate(zip(positions.tolist(), counts.tolist())):
        n = max(0, min(n, rows - offsets[-1]))
        used = min(max(int(blocks[j]), 0), entries)
        for i in range(n):
            row, at = offsets[-1] + i, p + i
            info[row] = j, min(at, 2 ** 31 - 1)
            if not 0 <= at < capacity:
                continue
            b = at // block
            if b >= used and (i == 0 or at % block == 0):  # the first new row of a block without a page
                if first_free < last:
                    table[j, b] = free[first_free]
                    first_free += 1
                    blocks_out[j] = b + 1
                else:
                    table[j, b] = -1
                    missing += 1
            if table[j, b] >= 0:
                slots[row] = int(table[j, b]) * block + at % block
        offsets.append(offsets[-1] + n)
    return np.array(offsets), info, slots, blocks_out, np.array([first_free, missing]), table


def run_plan(dev, stream, positions, counts, blocks, table, free, pool, rows, block, capacity, in_place=False):
    n = len(counts)
    pairs = np.stack([np.full(n, 77, np.int32), positions.astype(np.int32)], 1)
    b = [dev.upload(x.astype(np.int32)) for x in (pairs, counts, blocks, table, free, pool)]
    out = [dev.alloc(4 * (n + 1)), dev.alloc(8 * rows), dev.alloc(8 * rows)]
    out += [b[2], b[5]] if in_place else [dev.alloc(4 * n), dev.alloc(8)]
    hip.batch_plan(stream, *b, *out, hip.batch_params(n, rows, block, capacity))
    stream.sync()
    got = [out[0].read(np.int32), out[1].read(np.int32).reshape(rows, 2), out[2].read(np.int64),
           out[3].read(np.int32), out[4].read(np.int32), b[3].read(np.int32).reshape(table.shape)]
    assert np.array_equal(b[0].read(np.int32).reshape(n, 2), pairs)
    return got


PLANS = [  # requests, rows, block, capacity, most new rows, free pages, first free
    (1, 1, 16, 64, 1, 9, 0), (1, 700, 16, 1000, 700, 99, 3), (3, 5, 1, 9, 4, 40, 0), (16, 16, 16, 4096, 1, 64, 5),
    (200, 3000, 48, 500, 30, 4000, 1), (200, 300, 7, 500, 30, 500, 1), (64, 400, 16, 100, 40, 25, 10),
    (1500, 2500, 16, 200, 3, 3000, 0), (9, 100, 16, 100, 20, 0, 0), (5, 64, 1 << 20, 1 << 22, 20, 5, 0),
    (3000, 1, 16, 64, 1, 100, 0),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,rows,block,capacity,most,frees,first", PLANS)
def test_batch_plan(dev, stream, n, rows, block, capacity, most, frees, first, in_place):
    rng = np.random.default_rng(n + rows + block)
    entries = -(-capacity // block)
    positions = rng.integers(0, capacity, n)
    counts = rng.integers(0, most + 1, n)
    blocks = -(-positions // block)
    if n > 4:
        positions[::7] = -3            # rows before the start
        blocks[::7] = 0
        positions[3] = capacity        # full
        counts[4] = -9
        blocks[1] = min(entries, blocks[1] + 2)  # pages ahead of the tokens
        positions[2] = 2 ** 31 - 2     # rows past every capacity
        blocks[2] = entries + 5
    table = rng.integers(-1, 10 ** 6, (n, entries)).astype(np.int32)
    free = np.arange(frees, dtype=np.int32) + 10 ** 7
    if frees > 8:
        free[first + 2] = -1           # a bad page: no slot
    pool = i32(first, frees)
    args = (positions, counts, blocks, table, free if frees else i32(5), pool, rows, block, capacity)
    want = plan_reference(*args)
    if in_place:
        want[4][1] = pool[1]  # the list goes on: only its start moves
    got = run_plan(dev, stream, *args, in_place=in_place)
    for name, w, g in zip(("offsets", "rows", "slots", "blocks", "pool", "table"), want, got):
        assert np.array_equal(w, g), name


@pytest.mark.parametrize("n,rows", [(200, 1024), (200, 1025), (90, 2047), (1024, 2048), (200, 2049), (1025, 2048), (7, 5000)])
def test_batch_plan_in_place(dev, stream, n, rows):
    """By one workgroup in a few turns, and by two launches."""
    test_batch_plan(dev, stream, n, rows, 16, 4000, max(2, 2 * rows // n), n + rows // 16 + 100, 3, True)


@pytest.mark.parametrize("pool", [(-5, 3), (0, 1000), (7, 5), (2 ** 31 - 1, 2 ** 31 - 1), (2, -8)])
def test_free_lists_that_lie(dev, stream, pool):
    """Bounds of the list that lie outside of it: no page from there."""
    free = np.arange(6, dtype=np.int32) + 50
    args = (i32(0, 20), i32(40, 100), i32(0, 2), np.full((2, 20), 9, np.int32), free, i32(*pool), 140, 16, 320)
    want = plan_reference(*args)
    got = run_plan(dev, stream, *args)
    for name, w, g in zip(("offsets", "rows", "slots", "blocks"), want, got):
        assert np.array_equal(w, g), name
    assert np.array_equal(want[5], got[5])
    assert got[4][1] == want[4][1]


# ------------------------------------------------------------ append by slot

@pytest.mark.parametrize("dtype", [hip.F32, hip.F16, hip.Q8_0])
@pytest.mark.parametrize("nk,D,bs,rows,norm,rot", [(2, 128, 16, 1, False, 0), (3, 64, 7, 37, True, 20),
                                                  (4, 256, 48, 150, False, 64), (1, 192, 16, 65, True, 0)])
def test_append_by_slot(dev, stream, dtype, nk, D, bs, rows, norm, rot):
    """The bytes that yuuka_kv_append writes, wherever the slots are; rows without one write nothing."""
    rng = np.random.default_rng(rows + D)
    pages = -(-rows // bs) + 2
    table = rng.permutation(pages)[:-(-rows // bs)].astype(np.int32)
    p = hip.kv_params(dtype, bs, -(-rows // bs) * bs, nk, D, rows, rope_dim=rot)
    fill = rng.integers(0, 255, pages * hip.kv_page_bytes(p)).astype(np.uint8)
    k, v = rng.normal(0, 1, (2, rows, nk * D)).astype(np.float32)
    kb, vb, gain = dev.upload(k), dev.upload(v), dev.upload(rng.normal(1, 0.1, D).astype(np.float32)) if norm else None
    rope = dev.upload(rng.normal(0, 1, (rows, rot)).astype(np.float32)) if rot else None
    want = [dev.upload(fill), dev.upload(fill)]
    hip.kv_append(stream, kb, vb, *want, dev.upload(table), dev.upload(i32(0, 0)), p, k_norm=gain, rope=rope)
    row = np.arange(rows)
    slots = table[row // bs].astype(np.int64) * bs + row % bs
    got = [dev.upload(fill), dev.upload(fill)]
    hip.kv_append_slots(stream, kb, vb, *got, dev.upload(slots), p, k_norm=gain, rope=rope)
    stream.sync()
    for w, g in zip(want, got):
        assert np.array_equal(w.read(np.uint8), g.read(np.uint8))
    # slots outside the pool: those rows are dropped, the others written as before
    outside = [-1, pages * bs, 2 ** 40, -2 ** 63, 2 ** 63 - 1, -(2 ** 32)]
    gone = np.arange(rows) % 3 == 1
    slots[gone] = [outside[i % 6] for i in range(gone.sum())]
    some = [dev.upload(fill), dev.upload(fill)]
    hip.kv_append_slots(stream, kb, vb, *some, dev.upload(slots), p, k_norm=gain, rope=rope)
    full, rest = dev.upload(fill), [x.read(np.uint8) for x in some]
    outs = [dev.alloc(rows * nk * D * 4) for _ in range(4)]
    hip.kv_read(stream, *outs[:2], *some, dev.upload(table), p)
    hip.kv_read(stream, *outs[2:], *want, dev.upload(table), p)
    stream.sync()
    some_k, some_v, all_k, all_v = (o.read(np.float32).reshape(rows, -1) for o in outs)
    assert np.array_equal(some_k[~gone], all_k[~gone]) and np.array_equal(some_v[~gone], all_v[~gone])
    if gone.all() or rows == 1:
        return
    changed = rest[1] != full.read(np.uint8)
    page = np.arange(len(fill)) // hip.kv_page_bytes(p)
    assert not changed[~np.isin(page, table)].any()


@pytest.mark.parametrize("dtype", [hip.F32, hip.Q8_0])
def test_append_by_slot_rotated_by_the_plans_positions(dev, stream, dtype):
    """Rotations of rows at the positions that the plan works out, more rows than one op takes, captured and replayed."""
    rng = np.random.default_rng(31)
    n, rows, nk, D, rot, block, capacity, base = 5, 5000, 2, 64, 32, 16, 4096, 1e4
    entries = capacity // block
    up, alloc = dev.upload, dev.alloc
    b = dict(positions=alloc(8 * n), counts=alloc(4 * n), blocks=up(np.zeros(n, np.int32)),
             table=up(np.full((n, entries), -1, np.int32)), free=up(rng.permutation(n * entries).astype(np.int32)),
             pool=up(i32(0, n * entries)), offsets=alloc(4 * (n + 1)), info=alloc(8 * rows), slots=alloc(8 * rows),
             k=alloc(4 * rows * nk * D), v=alloc(4 * rows * nk * D), rope=alloc(4 * rows * rot))
    p = hip.kv_params(dtype, block, capacity, nk, D, rows, rope_dim=rot)
    pools = [alloc(n * entries * hip.kv_page_bytes(p)) for _ in range(2)]
    plan = hip.Plan(dev)
    plan.add(hip.OP["BATCH_PLAN"], [b[k] for k in ("positions", "counts", "blocks", "table", "free", "pool", "offsets", "info",
                                                   "slots", "blocks", "pool")], n=[n, rows], u=[block, capacity])
    for first in range(0, rows, 4096):
        offs = [first * rot * 4] + [0] * 14 + [first * 8]
        plan.add(hip.OP["ROPE_TABLE"], [b["rope"]] + [None] * 14 + [b["info"]], offs=offs,
                 n=[1, rot, 0, min(4096, rows - first)], f=[base], flags=hip.FLAG_OWN_POS)
    plan.add(hip.OP["KV_APPEND_SLOTS"], [b["k"], b["v"], *pools, b["slots"], None, b["rope"]], n=[nk, 0, D, nk * D, rows],
             u=[block, 0, dtype, rot], f=[0, 1e-6])
    graph = hip.Graph(plan, stream, None)
    position, cached = np.zeros(n, np.int64), [np.zeros((0, nk, D)) for _ in range(n)]
    for counts in ([700, 0, 1, 2900, 30], [1, 1, 1, 1, 1], [0, 3000, 90, 2, 1]):
        k, v = rng.normal(0, 1, (2, rows, nk, D)).astype(np.float32)
        for name, x in (("k", k), ("v", v), ("counts", i32(*counts)),
                        ("positions", np.stack([np.full(n, 9), position], 1).astype(np.int32))):
            b[name].write(x)
        graph.replay(stream)
        stream.sync()
        off = offsets_of(counts)
        for j, c in enumerate(counts):
            own = k[off[j]:off[j + 1]].astype(np.float64)
            angle = (position[j] + np.arange(c))[:, None] * base ** (-np.arange(0, rot, 2) / rot)
            x, y, cos, sin = own[..., :rot // 2], own[..., rot // 2:rot], np.cos(angle)[:, None], np.sin(angle)[:, None]
            turned = np.concatenate([x * cos - y * sin, x * sin + y * cos, own[..., rot:]], 2)
            cached[j] = np.concatenate([cached[j], turned])
        position += np.array(counts)
    most = int(position.max())
    out = [alloc(n * most * nk * D * 4) for _ in range(2)]
    hip.kv_read(stream, *out, *pools, b["table"], hip.kv_params(dtype, block, capacity, nk, D, most, n))
    stream.sync()
    got = out[0].read(np.float32).reshape(n, most, nk, D)
    for j in range(n):
        want = cached[j]
        # u each for the table, the product and the sum, of |x| + |y| <= 2 sqrt(2) times the larger of the turned two
        tol = 9 * U * np.abs(want).max(2, initial=1, keepdims=True)
        if dtype == hip.Q8_0:  # half a step of the 32 values' largest by 127, and the scale's own rounding to half
            most_of = np.repeat(np.abs(want).reshape(len(want), nk, D // 32, 32).max(3), 32, 2)
            tol = tol + most_of * (0.5 / 127 + 2.0 ** -11 + 2.0 ** -12)
        assert np.all(np.abs(got[j, :len(want)] - want) <= tol)
    graph.destroy()
    plan.destroy()


# ----------------------------------------------------------------- convolution

def conv_reference(x, w, windows, offsets, slots, groups, D, scale, eps):
    rows, channels = x.shape
    K = w.shape[1]
    out, new = np.full(x.shape, np.nan), windows.copy()
    size = np.full(x.shape, np.nan)
    for j in range(len(slots)):
        src, dst = slots[j]
        past = windows[src].T if 0 <= src < len(windows) else np.zeros((K - 1, channels))
        line = np.concatenate([past, x[offsets[j]:offsets[j + 1]]])
        for r in range(offsets[j], offsets[j + 1]):
            part = line[r - offsets[j]:r - offsets[j] + K] * w.T
            out[r], size[r] = part.sum(0), np.abs(part).sum(0)
        if 0 <= dst < len(windows):
            new[dst] = line[len(line) - K + 1:].T
    # |silu'| <= 1.1, so that an error of the sum comes through no larger
    y = out / (1 + np.exp(-out))
    error = 1.1 * K * U * size + 8 * U * np.abs(y)
    keys = groups * D
    qk = y[:, :2 * keys].reshape(rows, 2 * groups, D)
    norm = np.sqrt((qk * qk).sum(2, keepdims=True) + eps)
    # a head's norm is off by no more than its elements together, and D u for the sum
    e = error[:, :2 * keys].reshape(rows, 2 * groups, D)
    off = np.sqrt((e * e).sum(2, keepdims=True)) / norm + D * U
    y[:, :2 * keys] = (qk / norm).reshape(rows, 2 * keys)
    error[:, :2 * keys] = (e / norm + np.abs(qk / norm) * off).reshape(rows, 2 * keys)
    y[:, :keys] *= scale
    error[:, :keys] *= abs(scale)
    return y, error + 4 * U * np.abs(y), new


CONVS = [  # counts, groups, heads, D, taps
    ([1], 1, 1, 64, 4), ([7, 0, 1, 2, 3, 5, 0, 0, 100, 4], 2, 4, 64, 4), ([130, 1, 1, 1, 65], 1, 2, 128, 4),
    ([9, 2, 1, 30], 1, 3, 128, 2), ([1, 1, 2, 50, 3, 8, 7, 6, 0], 2, 2, 64, 8), ([1] * 70, 1, 1, 128, 3),
    ([5, 0, 33], 3, 3, 128, 5), ([0, 0], 1, 1, 64, 4),
    # several rows a wave, with requests that start, end and lie within
    ([1] * 9 + [0, 2, 3, 0, 5, 40, 1, 900, 0, 0, 1500, 33, 2, 2, 2], 4, 12, 128, 4),
    ([1] * 9 + [0, 2, 3, 0, 5, 40, 1, 1900, 0, 0, 2500, 33, 2, 2, 2], 4, 8, 64, 3),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,groups,heads,D,K", CONVS)
def test_conv(dev, stream, dtype, counts, groups, heads, D, K, in_place):
    rng = np.random.default_rng(sum(counts) + D + K)
    n, behind, channels = len(counts), 3, (2 * groups + heads) * D
    rows, stride = sum(counts) + behind, channels + 8
    offsets = offsets_of(counts)
    x = to_bits(rng.normal(0, 1, (rows, stride)), dtype)
    x[:, channels:] = to_bits(np.full((rows, 8), np.nan), dtype)   # between the rows: not read
    x[sum(counts):] = to_bits(np.full((behind, stride), np.nan), dtype)
    w = rng.normal(0, 0.5, (channels, K)).astype(np.float32)
    windows = rng.normal(0, 1, (2 * n + 1, channels, K - 1)).astype(np.float32)
    order = rng.permutation(2 * n)
    slots = np.stack([order[:n], order[:n] if in_place else order[n:]], 1).astype(np.int32)
    if n > 2:
        slots[1] = (-1, slots[1, 1])        # starts from zeros
        slots[2, 1] = 10 ** 9               # not kept
    ob = dev.upload(to_bits(np.full((rows, channels), 7.0), dtype))
    wb = dev.upload(windows)
    scale, eps = D ** -0.5, 1e-6
    p = hip.gdn_params(dtype, n, rows, groups, heads, D, kernel=K, row_stride=stride, scale=scale, eps=eps)
    hip.gdn_conv(stream, ob, dev.upload(x), dev.upload(w), wb, dev.upload(offsets), dev.upload(slots), p)
    stream.sync()
    live = sum(counts)
    want, error, new = conv_reference(from_bits(x[:, :channels], dtype), w.astype(np.float64), windows.astype(np.float64),
                                      offsets, slots, groups, D, scale, eps)
    got = from_bits(ob.read(np_type(dtype)).reshape(rows, channels), dtype)
    assert np.all(got[live:] == 7.0)
    if live:
        tol = error[:live] + HALF[dtype] * np.abs(want[:live]) + (2.0 ** -25 if dtype == hip.F16 else 0)
        assert np.all(np.abs(got[:live] - want[:live]) <= tol)
    assert np.array_equal(wb.read(np.float32).reshape(windows.shape), new.astype(np.float32))


PARTS = [  # rows in front of the first request, counts, groups, heads, D, taps
    (1, [1], 1, 1, 64, 4), (8, [8], 1, 1, 128, 4), (70, [1, 2, 3, 0, 40, 1], 2, 4, 64, 4),
    (900, [2, 1, 0, 3, 1, 1, 1500, 5], 4, 8, 128, 4), (2000, [1] * 20 + [0, 700, 2], 4, 12, 128, 4),
    (130, [3, 9, 1, 0, 2], 1, 2, 128, 8), (33, [1, 50], 2, 2, 64, 2),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("front,counts,groups,heads,D,K", PARTS)
def test_conv_of_a_part_of_a_batch(dev, stream, dtype, front, counts, groups, heads, D, K):
    """A batch whose first request does not start with the first row, every window left where it was read."""
    rng = np.random.default_rng(front + D + K)
    n, behind, channels = len(counts), 3, (2 * groups + heads) * D
    live = sum(counts)
    rows, offsets = front + live + behind, offsets_of(counts) + front
    x = to_bits(rng.normal(0, 1, (rows, channels)), dtype)
    x[:front] = x[front + live:] = to_bits(np.full(channels, np.nan), dtype)
    w = rng.normal(0, 0.5, (channels, K)).astype(np.float32)
    windows = rng.normal(0, 1, (n, channels, K - 1)).astype(np.float32)
    slots = np.stack([rng.permutation(n)] * 2, 1).astype(np.int32)
    ob, wb = dev.upload(to_bits(np.full((rows, channels), 7.0), dtype)), dev.upload(windows)
    scale = D ** -0.5
    p = hip.gdn_params(dtype, n, rows, groups, heads, D, kernel=K, scale=scale, eps=1e-6)
    hip.gdn_conv(stream, ob, dev.upload(x), dev.upload(w), wb, dev.upload(offsets), dev.upload(slots), p)
    stream.sync()
    own = slice(front, front + live)
    want, error, new = conv_reference(from_bits(x[own], dtype), w.astype(np.float64), windows.astype(np.float64),
                                      offsets - front, slots, groups, D, scale, 1e-6)
    got = from_bits(ob.read(np_type(dtype)).reshape(rows, channels), dtype)
    assert np.all(got[:front] == 7.0) and np.all(got[front + live:] == 7.0)
    assert np.all(np.abs(got[own] - want) <= error + HALF[dtype] * np.abs(want) + (2.0 ** -25 if dtype == hip.F16 else 0))
    assert np.array_equal(wb.read(np.float32).reshape(windows.shape), new.astype(np.float32))


# ------------------------------------------------------------- the delta rule

def delta_reference(qkv, g, beta, states, offsets, slots, groups, heads, D, scale):
    """Outputs and new states in float64, and bounds of what float32 may be off by."""
    rows = len(qkv)
    x = qkv.reshape(rows, 2 * groups + heads, D)
    group = np.arange(heads) % groups
    q, k, v = x[:, group] * scale, x[:, groups + group], x[:, 2 * groups:]
    out, off = np.full((rows, heads, D), np.nan), np.zeros((rows, heads, D))
    new, new_off = states.copy(), np.zeros(states.shape)
    for j in range(len(slots)):
        src, dst = slots[j]
        S = states[src].copy() if 0 <= src < len(states) else np.zeros((heads, D, D))
        n = offsets[j + 1] - offsets[j]
        most = np.sqrt((S * S).sum(1))  # largest norm so far of every column
        c = _bounds(n, D)
        for r in range(offsets[j], offsets[j + 1]):
            S *= np.exp(g[r])[:, None, None]
            d = (v[r] - np.einsum("hij,hi->hj", S, k[r])) * beta[r][:, None]
            S += k[r][:, :, None] * d[:, None]
            out[r] = np.einsum("hij,hi->hj", S, q[r])
            most = np.maximum(most, np.maximum(np.sqrt((S * S).sum(1)), np.abs(v[r])))
            off[r] = c * most * np.sqrt((q[r] ** 2).sum(1))[:, None]
        if 0 <= dst < len(states):
            new[dst], new_off[dst] = S, (c * most)[:, None]
    return out, off, new, new_off


def _bounds(n, D):
    """Of a column of the state after n rows, relative to its largest norm.

    A row turns a column S into e^g (S - beta k (k.S)) + beta k v, which for |k| <= 1, beta in 0..1 and
    g <= 0 makes no error larger. What it adds: the dot product k.S is off by at most D u |k| |S|, the
    decay by a few u of itself for the rounding of its own exponent (|g| u, with e^g |g| <= 0.4), the
    product and the sum by 2 u: (D + 4) u of the column, of either sign, so that n rows add up as sqrt(n).
    A chunk of rows solved at once replaces its dot products by sums of the same products over 64 rows."""
    return (D + 64 + 4) * U * math.sqrt(max(n, 1))


def gates(rng, rows, heads, raw, slow=0.02):
    """alpha, beta, dt, a, and what they stand for."""
    alpha, beta = rng.normal(0, 1, (2, rows, heads)).astype(np.float32)
    dt, a = rng.normal(0, 0.5, heads).astype(np.float32), (-np.exp(rng.uniform(math.log(slow), math.log(2), heads))).astype(np.float32)
    if not raw:
        alpha = (np.log1p(np.exp(alpha + dt)) * a).astype(np.float32)
        beta = (1 / (1 + np.exp(-beta))).astype(np.float32)
        return alpha, beta, None, None, alpha.astype(np.float64), beta.astype(np.float64)
    g = np.logaddexp(0, alpha.astype(np.float64) + dt) * a.astype(np.float64)
    return alpha, beta, dt, a, g, 1 / (1 + np.exp(-beta.astype(np.float64)))


def unit_rows(rng, rows, groups, heads, D, dtype, stride=0):
    """Rows [q | k | v] as the convolution leaves them, keys and queries of norm up to 1."""
    x = rng.normal(0, 1, (rows, 2 * groups + heads, D))
    x[:, :2 * groups] /= 1.005 * np.sqrt((x[:, :2 * groups] ** 2).sum(2, keepdims=True))
    full = np.full((rows, stride or x[0].size), np.nan)
    full[:, :x[0].size] = x.reshape(rows, -1)
    return to_bits(full, dtype)


def run_delta(dev, stream, dtype, qkv, alpha, beta, dt, a, states, counts, slots, groups, heads, D, scale=1.0, step=False,
              stride=0, offsets=None):
    rows = len(qkv)
    ob, sb = dev.upload(to_bits(np.full((rows, heads, D), 7.0), dtype)), dev.upload(states)
    p = hip.gdn_params(dtype, len(slots), rows, groups, heads, D, row_stride=stride, log_decay=dt is None, scale=scale)
    more = {} if dt is None else dict(dt=dev.upload(dt), a=dev.upload(a))
    bufs = [ob, dev.upload(qkv), dev.upload(alpha), dev.upload(beta), sb]
    if step:
        hip.gdn_step(stream, *bufs, dev.upload(np.asarray(slots, np.int32)), p, **more)
    else:
        hip.gdn_prompt(stream, *bufs, dev.upload(offsets_of(counts) if offsets is None else offsets),
                       dev.upload(np.asarray(slots, np.int32)), p, **more)
    stream.sync()
    return from_bits(ob.read(np_type(dtype)).reshape(rows, heads, D), dtype), sb.read(np.float32).reshape(states.shape)


def check_delta(got, want, dtype, live):
    (o, s), (wo, off, ws, s_off) = got, want
    assert np.all(o[live:] == 7.0)
    tol = off[:live] + HALF[dtype] * np.abs(wo[:live]) + (2.0 ** -25 if dtype == hip.F16 else 0)
    worst = np.max(np.abs(o[:live] - wo[:live]) / tol, initial=0)
    assert np.all(np.abs(o[:live] - wo[:live]) <= tol), worst
    assert np.all(np.abs(s - ws) <= s_off + U * np.abs(ws)), np.max(np.abs(s - ws))


DELTAS = [  # counts, groups, heads, D
    ([1], 1, 1, 64), ([1], 1, 2, 128), ([3, 0, 1, 2], 2, 4, 64), ([15, 16, 17, 31, 32, 33], 1, 2, 128),
    ([63, 64, 65], 1, 1, 64), ([63, 64, 65, 0], 2, 2, 128), ([130, 1, 0, 0, 200, 7], 1, 3, 128), ([300], 2, 4, 64),
    ([127, 128, 129], 1, 1, 128), ([5] * 40, 1, 2, 64), ([0], 1, 1, 128), ([1, 2, 0] * 25, 2, 8, 64), ([2, 1] * 40, 1, 8, 128),
    ([1] * 70, 1, 1, 128),
]


@pytest.mark.parametrize("raw", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,groups,heads,D", DELTAS)
def test_prompt(dev, stream, dtype, counts, groups, heads, D, raw):
    rng = np.random.default_rng(sum(counts) + D + heads)
    n, live = len(counts), sum(counts)
    rows, stride = live + 2, (2 * groups + heads) * D + 16
    qkv = unit_rows(rng, rows, groups, heads, D, dtype, stride)
    qkv[live:] = to_bits(np.full((2, stride), np.nan), dtype)
    alpha, beta, dt, a, g, b = gates(rng, rows, heads, raw)
    states = rng.normal(0, 0.3, (2 * n + 1, heads, D, D)).astype(np.float32)
    order = rng.permutation(2 * n)
    slots = np.stack([order[:n], order[n:]], 1)
    if n > 2:
        slots[0] = slots[0, 0], slots[0, 0]   # in place
        slots[1, 0] = -1                      # from zeros
        slots[2, 1] = 2 * n + 1               # not kept
    if n > 3:
        slots[3, 0] = slots[0, 0] if slots[0, 0] != slots[0, 1] else 2 * n
    got = run_delta(dev, stream, dtype, qkv, alpha, beta, dt, a, states, counts, slots, groups, heads, D, D ** -0.5,
                    stride=stride)
    x = from_bits(qkv[:, :(2 * groups + heads) * D], dtype)
    want = delta_reference(x[:live], g, b, states.astype(np.float64), offsets_of(counts), slots, groups, heads, D, D ** -0.5)
    pad = [np.concatenate([w, np.zeros((2, heads, D))]) for w in want[:2]]
    check_delta(got, (*pad, *want[2:]), dtype, live)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,groups,heads,D", [(40, 1, 2, 128), (60, 2, 4, 128), (80, 1, 2, 64), (70, 2, 4, 64), (60, 2, 8, 128),
                                              (70, 1, 8, 64), (90, 2, 6, 64)])
def test_prompts_of_many_requests(dev, stream, dtype, n, groups, heads, D):
    """Workgroups of two and four tiles of columns and of two heads, and more requests than are put in order."""
    rng = np.random.default_rng(n + D)
    counts = [int(x) for x in rng.permutation([0, 1, 64, 65, 130, 200] + [int(x) for x in rng.integers(0, 20, n - 6)])]
    rows = sum(counts)
    qkv = unit_rows(rng, rows, groups, heads, D, dtype)
    alpha, beta, _, _, g, b = gates(rng, rows, heads, False)
    states = rng.normal(0, 0.3, (n, heads, D, D)).astype(np.float32)
    slots = np.stack([rng.permutation(n)] * 2, 1)
    got = run_delta(dev, stream, dtype, qkv, alpha, beta, None, None, states, counts, slots, groups, heads, D)
    want = delta_reference(from_bits(qkv, dtype), g, b, states.astype(np.float64), offsets_of(counts), slots, groups, heads,
                           D, 1.0)
    check_delta(got, want, dtype, rows)


@pytest.mark.parametrize("raw", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,groups,heads,D", [(1, 1, 1, 64), (1, 16, 16, 128), (5, 2, 4, 128), (9, 1, 3, 64), (70, 1, 2, 128)])
def test_step(dev, stream, dtype, n, groups, heads, D, raw):
    rng = np.random.default_rng(n + D + heads)
    rows, stride = n + 3, (2 * groups + heads) * D + 8
    qkv = unit_rows(rng, rows, groups, heads, D, dtype, stride)
    qkv[n:] = to_bits(np.full((3, stride), np.nan), dtype)
    alpha, beta, dt, a, g, b = gates(rng, rows, heads, raw)
    states = rng.normal(0, 0.3, (2 * n + 1, heads, D, D)).astype(np.float32)
    order = rng.permutation(2 * n)
    slots = np.stack([order[:n], order[n:]], 1)
    if n > 2:
        slots[0, 0] = slots[0, 1]
        slots[1, 0] = -7
        slots[2, 1] = -1
    got = run_delta(dev, stream, dtype, qkv, alpha, beta, dt, a, states, None, slots, groups, heads, D, 0.25, step=True,
                    stride=stride)
    x = from_bits(qkv[:, :(2 * groups + heads) * D], dtype)
    want = delta_reference(x[:n], g, b, states.astype(np.float64), np.arange(n + 1), slots, groups, heads, D, 0.25)
    pad = [np.concatenate([w, np.zeros((3, heads, D))]) for w in want[:2]]
    check_delta(got, (*pad, *want[2:]), dtype, n)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["no decay", "forgets", "forgets now and then", "one key", "no step", "full step", "huge",
                                  "tiny", "overwhelmed"])
def test_prompt_extremes(dev, stream, what, D):
    rng = np.random.default_rng(len(what) + D)
    counts, groups, heads = [150, 70], 1, 2
    rows = sum(counts)
    qkv = unit_rows(rng, rows, groups, heads, D, hip.F32).reshape(rows, -1, D)
    alpha, beta, _, _, _, _ = gates(rng, rows, heads, False)
    states = rng.normal(0, 0.3, (2, heads, D, D)).astype(np.float32)
    if what == "no decay":
        alpha[:] = 0
    elif what == "forgets":
        alpha[:] = -60
        alpha[::3] = -1e30
    elif what == "forgets now and then":
        alpha[:] = -0.01
        alpha[40], alpha[64], alpha[100] = -np.inf, -np.inf, -500.0
    elif what == "one key":
        qkv[:, 1] = qkv[0, 1]
        alpha[:] = -0.001
    elif what == "no step":
        beta[:] = 0
    elif what == "full step":
        beta[:] = 1
        alpha[:] = -1e-4
    elif what == "huge":
        states *= 1e30
        qkv[:, 2:] *= 1e30
    elif what == "tiny":
        states *= 1e-25
        qkv[:, 2:] *= 1e-25
    elif what == "overwhelmed":  # values of very different sizes, side by side
        qkv[::5, 2:] *= 1e6
        qkv[2::5, 2:] *= 1e-6
        alpha[:] = -3.0
    slots = np.array([[0, 0], [1, 1]])
    qkv = qkv.reshape(rows, -1)
    got = run_delta(dev, stream, hip.F32, qkv, alpha, beta, None, None, states, counts, slots, groups, heads, D)
    want = delta_reference(qkv.astype(np.float64), alpha.astype(np.float64), beta.astype(np.float64),
                           states.astype(np.float64), offsets_of(counts), slots, groups, heads, D, 1.0)
    check_delta(got, want, hip.F32, rows)


def test_a_nan_stays_with_its_request(dev, stream):
    """Values that are not finite in one request's rows or state reach no other request, and in a head no other head."""
    rng = np.random.default_rng(3)
    counts, groups, heads, D = [70, 70, 70], 2, 4, 64
    rows = sum(counts)
    qkv = unit_rows(rng, rows, groups, heads, D, hip.F32).reshape(rows, -1, D)
    alpha, beta, _, _, g, b = gates(rng, rows, heads, False)
    states = rng.normal(0, 0.3, (3, heads, D, D)).astype(np.float32)
    clean = delta_reference(qkv.reshape(rows, -1).astype(np.float64), g, b, states.astype(np.float64), offsets_of(counts),
                            np.array([[0, 0], [1, 1], [2, 2]]), groups, heads, D, 1.0)
    qkv[100, 2 * groups + 1, 5] = np.nan   # a value of head 1
    states[1, 2, 3, 9] = np.inf            # head 2
    out, new = run_delta(dev, stream, hip.F32, qkv.reshape(rows, -1), alpha, beta, None, None, states, counts,
                         [[0, 0], [1, 1], [2, 2]], groups, heads, D)
    other = np.ones((rows, heads), bool)
    other[70:140, 1:3] = False
    assert np.all(np.abs(out - clean[0])[other] <= (clean[1] + U * np.abs(clean[0]))[other])
    assert np.isnan(out[100:140, 1, 5]).all()
    assert not np.isfinite(out[70:140, 2, 9]).any()
    assert np.isfinite(new[[0, 2]]).all() and np.isfinite(new[1, [0, 3]]).all()


@pytest.mark.parametrize("what", ["key", "query", "value", "infinite value", "decay", "growth", "step", "state", "huge keys"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,groups,heads,D", [(7, 1, 3, 64), (20, 2, 4, 128), (70, 1, 2, 128), (70, 2, 4, 64)])
def test_rows_before_one_that_is_not_finite(dev, stream, dtype, n, groups, heads, D, what):
    """As the rule goes row by row: what is not finite reaches its own row and those after it, and of another head or column none."""
    rng = np.random.default_rng(n + D + len(what))
    counts = ([130, 3, 64, 65, 1, 17, 2] * n)[:n] if n < 40 else [int(x) for x in rng.permutation([130, 64, 65, 1, 2, 0] + [
        int(x) for x in rng.integers(1, 40, n - 6)])]
    rows, off = sum(counts), offsets_of(counts)
    qkv = unit_rows(rng, rows, groups, heads, D, dtype).reshape(rows, -1, D)
    alpha, beta, _, _, _, _ = gates(rng, rows, heads, False)
    states = rng.normal(0, 0.3, (n, heads, D, D)).astype(np.float32)
    slots = np.stack([rng.permutation(n)] * 2, 1)
    bad = to_bits(np.array([np.nan, np.inf]), dtype)
    at = np.array([off[j] + rng.integers(0, c) if c else -1 for j, c in enumerate(counts)])
    for j in range(0, n, 2):
        if at[j] < 0:
            continue
        if counts[j] == 130:
            at[j] = off[j] + 64 + 20
        if what == "key":
            qkv[at[j], groups + groups - 1, 7] = bad[j // 2 % 2]
        elif what == "query":
            qkv[at[j], 0, D - 1] = bad[j // 2 % 2]
        elif what in ("value", "infinite value"):
            qkv[at[j], 2 * groups + heads - 1, 21] = bad[int(what == "infinite value")]
        elif what in ("decay", "growth"):
            alpha[at[j], heads - 1] = np.nan if what == "decay" else np.inf
        elif what == "step":
            beta[at[j], 0] = (np.nan, np.inf)[j // 2 % 2]
        elif what == "state":
            states[slots[j, 0], 0, 3, D - 2] = (np.nan, np.inf)[j // 2 % 2]
        else:  # their products with one another pass the type's largest value (F16: their sum of squares does not)
            big = 6e4 if dtype == hip.F16 else 1e20
            qkv[at[j]:off[j + 1], groups] = to_bits(np.full(D, big), dtype)
    qkv = qkv.reshape(rows, -1)
    got = run_delta(dev, stream, dtype, qkv, alpha, beta, None, None, states, counts, slots, groups, heads, D)
    with np.errstate(all="ignore"):
        want = delta_reference(from_bits(qkv, dtype), alpha.astype(np.float64), beta.astype(np.float64),
                               states.astype(np.float64), off, slots, groups, heads, D, 1.0)
    (o, s), (wo, o_off, ws, s_off) = got, want
    fine, fine_s = np.isfinite(wo), np.isfinite(ws)
    if what == "huge keys":  # (64 bits hold what float32 does not; keys beyond norm 1 have no bound)
        for j in range(0, n, 2):
            fine[at[j]:off[j + 1]] = False
            fine_s[slots[j, 1]] = False
    else:
        assert not np.isfinite(o[~fine]).any() and not np.isfinite(s[~fine_s]).any()
        assert not fine.all()
    with np.errstate(all="ignore"):
        tol = o_off + HALF[dtype] * np.abs(wo) + (2.0 ** -25 if dtype == hip.F16 else 0)
        assert np.all((np.abs(o - wo) <= tol)[fine])
        assert np.all((np.abs(s - ws) <= s_off + U * np.abs(ws))[fine_s])


def test_offsets_that_lie(dev, stream):
    """Offsets outside the arrays are taken as their ends; a request that ends before it starts is empty."""
    rng = np.random.default_rng(8)
    groups, heads, D, rows = 1, 2, 64, 100
    qkv = unit_rows(rng, rows, groups, heads, D, hip.F32)
    alpha, beta, _, _, g, b = gates(rng, rows, heads, False)
    states = rng.normal(0, 0.3, (3, heads, D, D)).astype(np.float32)
    slots = np.array([[0, 0], [1, 1], [2, 2]])
    got = run_delta(dev, stream, hip.F32, qkv, alpha, beta, None, None, states, None, slots, groups, heads, D,
                    offsets=i32(-50, 60, 40, 2 ** 31 - 1))
    # request 0 has rows 0..59, request 1 none, request 2 rows 40..99: rows 40..59 hold either's outputs
    for j, (lo, hi) in ((0, (0, 60)), (2, (40, 100))):
        w = delta_reference(qkv.astype(np.float64)[lo:hi], g[lo:hi], b[lo:hi], states.astype(np.float64),
                            np.array([0, hi - lo]), slots[j:j + 1], groups, heads, D, 1.0)
        assert np.all(np.abs(got[1][j] - w[2][j]) <= w[3][j] + U * np.abs(w[2][j]))
        keep = slice(0, 40) if j == 0 else slice(20, 60)
        assert np.all(np.abs(got[0][lo:hi][keep] - w[0][keep]) <= w[1][keep] + U * np.abs(w[0][keep]))
    assert np.array_equal(got[1][1], states[1])


@pytest.mark.parametrize("offsets", [(200, 0, 100), (50, 20, 60), (150, -5, 120, 7, 7, 200), (2 ** 31 - 1, 0, 64, -2 ** 31, 130)])
def test_offsets_out_of_order(dev, stream, offsets):
    """Results are undefined there, but nothing outside the rows and the slots is touched, and the next call is sound."""
    rng = np.random.default_rng(len(offsets))
    groups, heads, D, rows, n = 1, 2, 64, 200, len(offsets) - 1
    qkv = unit_rows(rng, rows, groups, heads, D, hip.F32)
    alpha, beta, _, _, g, b = gates(rng, rows, heads, False)
    states = rng.normal(0, 0.3, (n + 1, heads, D, D)).astype(np.float32)
    windows = rng.normal(0, 1, (n + 1, qkv.shape[1], 3)).astype(np.float32)
    slots = np.stack([np.arange(n)] * 2, 1).astype(np.int32)
    p = hip.gdn_params(hip.F32, n, rows, groups, heads, D, log_decay=True)
    ends = dev.upload(i32(*offsets))
    y, o = dev.upload(np.full((rows + 70, qkv.shape[1]), 7, np.float32)), dev.upload(np.full((rows + 70, heads, D), 7, np.float32))
    wb, sb = dev.upload(windows), dev.upload(states)
    where, weight = dev.upload(slots), dev.upload(rng.normal(0, 0.5, (qkv.shape[1], 4)).astype(np.float32))
    hip.gdn_conv(stream, y, dev.upload(qkv), weight, wb, ends, where, p)
    hip.gdn_prompt(stream, o, dev.upload(qkv), dev.upload(alpha), dev.upload(beta), sb, ends, where, p)
    stream.sync()
    for buf in (y, o):
        assert np.all(buf.read(np.float32).reshape(rows + 70, -1)[rows:] == 7)
    assert np.array_equal(wb.read(np.float32).reshape(windows.shape)[n], windows[n])
    assert np.array_equal(sb.read(np.float32).reshape(states.shape)[n], states[n])
    got = run_delta(dev, stream, hip.F32, qkv, alpha, beta, None, None, states, [rows - 90, 90], [[0, 0], [1, 1]], groups, heads, D)
    want = delta_reference(qkv.astype(np.float64), g, b, states.astype(np.float64), i32(0, rows - 90, rows),
                           np.array([[0, 0], [1, 1]]), groups, heads, D, 1.0)
    check_delta(got, want, hip.F32, rows)


@pytest.mark.parametrize("front", [1, 70, 200])
@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_of_a_part_of_a_batch(dev, stream, dtype, front):
    """Requests that start behind the first row, with as many of one and two rows: the rows in front are left alone."""
    rng = np.random.default_rng(front)
    groups, heads, D, counts = 1, 2, 64, [1, 90, 0, 2, 3, 130]
    n, live = len(counts), sum(counts)
    qkv = unit_rows(rng, front + live, groups, heads, D, dtype)
    qkv[:front] = to_bits(np.full(qkv.shape[1], np.nan), dtype)
    alpha, beta, _, _, g, b = gates(rng, front + live, heads, False)
    states = rng.normal(0, 0.3, (n, heads, D, D)).astype(np.float32)
    slots = np.stack([rng.permutation(n)] * 2, 1)
    out, new = run_delta(dev, stream, dtype, qkv, alpha, beta, None, None, states, None, slots, groups, heads, D,
                         offsets=offsets_of(counts) + i32(front))
    want = delta_reference(from_bits(qkv[front:], dtype), g[front:], b[front:], states.astype(np.float64), offsets_of(counts),
                           slots, groups, heads, D, 1.0)
    assert np.all(out[:front] == 7.0)
    check_delta((out[front:], new), want, dtype, live)


@pytest.mark.parametrize("D", [64, 128])
def test_a_prompt_in_pieces(dev, stream, D):
    """A prompt in one call, in three, and token by token."""
    rng = np.random.default_rng(D)
    groups, heads, rows = 2, 4, 150
    qkv = unit_rows(rng, rows, groups, heads, D, hip.F32)
    alpha, beta, dt, a, g, b = gates(rng, rows, heads, True)
    state = rng.normal(0, 0.3, (1, heads, D, D)).astype(np.float32)
    want = delta_reference(qkv.astype(np.float64), g, b, state.astype(np.float64), i32(0, rows), np.array([[0, 0]]), groups,
                           heads, D, 1.0)
    for pieces in ([rows], [1, 70, 79], [1] * rows):
        s, outs, at = state, [], 0
        for n in pieces:
            cut = slice(at, at + n)
            o, s = run_delta(dev, stream, hip.F32, qkv[cut], alpha[cut], beta[cut], dt, a, s, [n], [[0, 0]], groups, heads,
                             D, step=n == 1)
            outs.append(o)
            at += n
        check_delta((np.concatenate(outs), s), want, hip.F32, rows)


# --------------------------------------------------- all of them, one behind the other

class Batch:
    """A ragged batch through one recurrent and one attention layer: a plan's buffers, and the same in float64."""

    def __init__(self, dev, requests, rows, seed, groups=2, heads=4, D=64, nk=2, KD=64, block=16, capacity=256):
        rng = self.rng = np.random.default_rng(seed)
        self.n, self.rows, self.block, self.capacity = requests, rows, block, capacity
        self.groups, self.heads, self.D, self.nk, self.KD = groups, heads, D, nk, KD
        self.channels, self.kvd = (2 * groups + heads) * D, nk * KD
        entries, self.pages = capacity // block, requests * (capacity // block)
        up = dev.upload
        self.position = np.zeros(requests, np.int64)
        self.weight = rng.normal(0, 0.5, (self.channels, 4)).astype(np.float32)
        self.dt, self.a = rng.normal(0, 0.5, heads).astype(np.float32), -rng.uniform(0.05, 2, heads).astype(np.float32)
        self.windows, self.states = np.zeros((requests, self.channels, 3)), np.zeros((requests, heads, D, D))
        self.keys = [[np.zeros((0, self.kvd))] * 2 for _ in range(requests)]
        self.b = dict(
            positions=up(np.zeros((requests, 2), np.int32)), counts=up(np.zeros(requests, np.int32)),
            blocks=up(np.zeros(requests, np.int32)), table=up(np.full((requests, entries), -1, np.int32)),
            free=up(rng.permutation(self.pages).astype(np.int32)), pool=up(i32(0, self.pages)),
            offsets=dev.alloc(4 * (requests + 1)), info=dev.alloc(8 * rows), slots=dev.alloc(8 * rows),
            x=dev.alloc(rows * self.channels * 4), y=dev.alloc(rows * self.channels * 4), weight=up(self.weight),
            windows=up(self.windows.astype(np.float32)), states=up(self.states.astype(np.float32)),
            alpha=dev.alloc(rows * heads * 4), beta=dev.alloc(rows * heads * 4), dt=up(self.dt), a=up(self.a),
            where=up(np.stack([np.arange(requests)] * 2, 1).astype(np.int32)), out=dev.alloc(rows * heads * D * 4),
            k=dev.alloc(rows * self.kvd * 4), v=dev.alloc(rows * self.kvd * 4),
            kpool=dev.alloc(self.pages * block * self.kvd * 2), vpool=dev.alloc(self.pages * block * self.kvd * 2))

    def plan(self, dev):
        b, p = self.b, hip.Plan(dev)
        n = [self.n, self.rows, self.groups, self.heads, self.D, 0]
        p.add(hip.OP["BATCH_PLAN"], [b["positions"], b["counts"], b["blocks"], b["table"], b["free"], b["pool"], b["offsets"],
                                     b["info"], b["slots"], b["blocks"], b["pool"]], n=n[:2], u=[self.block, self.capacity])
        p.add(hip.OP["KV_APPEND_SLOTS"], [b["k"], b["v"], b["kpool"], b["vpool"], b["slots"]],
              n=[self.nk, 0, self.KD, self.kvd, self.rows], u=[self.block, 0, hip.F16, 0], f=[0, 1e-6])
        p.add(hip.OP["GDN_CONV"], [b["y"], b["x"], b["weight"], b["windows"], b["offsets"], b["where"]], n=n,
              u=[hip.F32, 4], f=[self.D ** -0.5, 1e-6])
        p.add(hip.OP["GDN_PROMPT"], [b["out"], b["y"], b["alpha"], b["beta"], b["states"], b["offsets"], b["where"], b["dt"],
                                     b["a"]], n=n, u=[hip.F32, 0, 0], f=[1.0])
        return p

    def fill(self, counts):
        """New rows in the buffers; the outputs that are due, and their bounds."""
        rng, rows = self.rng, self.rows
        live, off = sum(counts), offsets_of(counts)
        data = dict(x=rng.normal(0, 1, (rows, self.channels)), alpha=rng.normal(0, 1, (rows, self.heads)),
                    beta=rng.normal(0, 1, (rows, self.heads)), k=rng.normal(0, 1, (rows, self.kvd)),
                    v=rng.normal(0, 1, (rows, self.kvd)))
        data = {name: v.astype(np.float32) for name, v in data.items()}
        for name, v in data.items():
            self.b[name].write(v)
        self.b["counts"].write(np.array(counts, np.int32))
        self.b["positions"].write(np.stack([np.zeros(self.n), self.position], 1).astype(np.int32))
        where = np.stack([np.arange(self.n)] * 2, 1)
        y, y_off, self.windows = conv_reference(data["x"][:live].astype(np.float64), self.weight.astype(np.float64),
                                                self.windows, off, where, self.groups, self.D, self.D ** -0.5, 1e-6)
        g = np.logaddexp(0, data["alpha"].astype(np.float64) + self.dt) * self.a.astype(np.float64)
        beta = 1 / (1 + np.exp(-data["beta"].astype(np.float64)))
        out, o_off, self.states, _ = delta_reference(y, g, beta, self.states, off, where, self.groups, self.heads, self.D, 1.0)
        for j in range(self.n):
            self.keys[j] = [np.concatenate([old, data[s][off[j]:off[j + 1]].astype(np.float16).astype(np.float64)])
                            for old, s in zip(self.keys[j], "kv")]
        self.position += np.array(counts)
        # rows that are off by y_off change a column of the state by as much, row after row
        return out, o_off + 64 * np.max(y_off, initial=0) * max(1, np.max(np.abs(out), initial=0)), live

    def check(self, dev, stream, due):
        out, tol, live = due
        got = self.b["out"].read(np.float32).reshape(self.rows, self.heads, self.D)[:live]
        assert np.all(np.abs(got - out) <= tol + U * np.abs(out))
        most = int(max(self.position.max(), 1))
        ko, vo = (dev.alloc(self.n * most * self.kvd * 4) for _ in range(2))
        hip.kv_read(stream, ko, vo, self.b["kpool"], self.b["vpool"], self.b["table"],
                    hip.kv_params(hip.F16, self.block, self.capacity, self.nk, self.KD, most, self.n))
        stream.sync()
        for buf, side in ((ko, 0), (vo, 1)):
            rows = buf.read(np.float32).reshape(self.n, most, -1)
            for j in range(self.n):
                want = self.keys[j][side]
                assert np.all(np.abs(rows[j, :len(want)] - want) <= 2.0 ** -10 * np.abs(want))  # one half step apart


SERIES = [[5, 70, 0, 17], [1, 1, 1, 1], [0, 40, 33, 2], [1, 1, 1, 1], [30, 0, 0, 0]]


def test_a_ragged_batch_step_by_step(dev, stream):
    batch = Batch(dev, 4, 96, 5)
    plan = batch.plan(dev)
    for counts in SERIES:
        due = batch.fill(counts)
        plan.execute(stream)
        stream.sync()
        batch.check(dev, stream, due)
    plan.destroy()


def test_a_ragged_batch_captured(dev, stream):
    """One graph replayed at other lengths, with eager work between; a second one of the same plan has a workspace of its own."""
    batch = Batch(dev, 4, 96, 6)
    plan = batch.plan(dev)
    s2 = hip.Stream(dev)
    graphs = [hip.Graph(plan, stream, None), hip.Graph(plan, s2, None)]
    plan.destroy()
    other = Batch(dev, 3, 200, 9)
    for i, counts in enumerate(SERIES):
        due = batch.fill(counts)
        theirs = other.fill([3 + i, 50, 11 * i])
        graphs[i % 2].replay((stream, s2)[i % 2])
        p = other.plan(dev)
        p.execute(stream)
        stream.sync()
        s2.sync()
        batch.check(dev, stream, due)
        other.check(dev, stream, theirs)
        p.destroy()
    for g in graphs:
        g.destroy()
    s2.destroy()


def test_tokens_captured(dev, stream):
    """A token of every request, pages and all, as one graph replayed: 1100 requests of which some take none."""
    rng = np.random.default_rng(21)
    n, groups, heads, D, block, capacity = 1100, 1, 1, 64, 16, 64
    channels, entries = 3 * D, capacity // block
    weight = rng.normal(0, 0.5, (channels, 4)).astype(np.float32)
    windows, states = np.zeros((n, channels, 3)), np.zeros((n, heads, D, D))
    where = np.stack([np.arange(n)] * 2, 1).astype(np.int32)
    up, alloc = dev.upload, dev.alloc
    b = dict(positions=alloc(8 * n), counts=alloc(4 * n), blocks=up(np.zeros(n, np.int32)),
             table=up(np.full((n, entries), -1, np.int32)), free=up(rng.permutation(n * entries).astype(np.int32)),
             pool=up(i32(0, n * entries)), offsets=alloc(4 * (n + 1)), info=alloc(8 * n), slots=alloc(8 * n),
             x=alloc(4 * n * channels), y=alloc(4 * n * channels), weight=up(weight), where=up(where),
             windows=up(windows.astype(np.float32)), states=up(states.astype(np.float32)), alpha=alloc(4 * n), beta=alloc(4 * n),
             out=alloc(4 * n * D))
    plan = hip.Plan(dev)
    plan.add(hip.OP["BATCH_PLAN"], [b[k] for k in ("positions", "counts", "blocks", "table", "free", "pool", "offsets", "info",
                                                   "slots", "blocks", "pool")], n=[n, n], u=[block, capacity])
    plan.add(hip.OP["GDN_CONV"], [b[k] for k in ("y", "x", "weight", "windows", "offsets", "where")],
             n=[n, n, groups, heads, D, 0], u=[hip.F32, 4], f=[1.0, 1e-6])
    plan.add(hip.OP["GDN_STEP"], [b[k] for k in ("out", "y", "alpha", "beta", "states")] + [None, b["where"]],
             n=[n, n, groups, heads, D, 0], u=[hip.F32, 0, 1], f=[1.0])
    graph = hip.Graph(plan, stream, None)
    position, used, blocks = np.zeros(n, np.int64), 0, np.zeros(n, np.int64)
    free = b["free"].read(np.int32)
    for turn in range(4):
        x = rng.normal(0, 1, (n, channels)).astype(np.float32)
        alpha = -rng.uniform(0, 1, (n, 1)).astype(np.float32)
        beta = rng.uniform(0, 1, (n, 1)).astype(np.float32)
        for name, v in (("x", x), ("alpha", alpha), ("beta", beta), ("counts", np.ones(n, np.int32)),
                        ("positions", np.stack([np.zeros(n), position], 1).astype(np.int32))):
            b[name].write(v)
        graph.replay(stream)
        stream.sync()
        offsets = np.arange(n + 1)
        assert np.array_equal(b["offsets"].read(np.int32), offsets)
        fresh = position // block >= blocks
        slots = b["slots"].read(np.int64)
        assert np.array_equal(slots[fresh] // block, free[used:used + fresh.sum()])
        used += int(fresh.sum())
        blocks = np.maximum(blocks, position // block + 1)
        assert np.array_equal(slots % block, position % block) and len(set(slots.tolist())) == n
        y, y_off, windows = conv_reference(x.astype(np.float64), weight.astype(np.float64), windows, offsets, where, groups, D,
                                           1.0, 1e-6)
        out, off, states, _ = delta_reference(y, alpha.astype(np.float64), beta.astype(np.float64), states, offsets, where,
                                              groups, heads, D, 1.0)
        tol = off + 64 * np.max(y_off) * max(1, np.max(np.abs(out))) + U * np.abs(out)
        assert np.all(np.abs(b["out"].read(np.float32).reshape(out.shape) - out) <= tol)
        position += np.where(np.arange(n) % 3 == turn % 3, 15, 1)
    graph.destroy()
    plan.destroy()


def test_attention_over_planned_pages(dev, stream):
    """Decode attention over what the plan and the append by slot left."""
    batch = Batch(dev, 3, 64, 12, KD=64)
    plan = batch.plan(dev)
    for counts in ([20, 33, 1], [1, 1, 1]):
        batch.fill(counts)
        plan.execute(stream)
    stream.sync()
    heads = 4
    q = np.random.default_rng(1).normal(0, 1, (3, heads, 64)).astype(np.float32)
    ob = dev.alloc(q.nbytes)
    p = hip.kv_params(hip.F16, batch.block, batch.capacity, batch.nk, 64, 1, 3, heads=heads, scale=0.125)
    hip.attn_decode(stream, ob, dev.upload(q), batch.b["kpool"], batch.b["vpool"], batch.b["table"], batch.b["positions"], p)
    stream.sync()
    got = ob.read(np.float32).reshape(q.shape)
    for j in range(3):
        k, v = (x.reshape(len(x), batch.nk, 64) for x in batch.keys[j])
        for h in range(heads):
            s = k[:, h // 2] @ q[j, h].astype(np.float64) * 0.125
            w = np.exp(s - s.max())
            want = (w / w.sum()) @ v[:, h // 2]
            # keys and values within a half step of 2^-10: a score by 2^-10 of its terms' sizes
            e = 2.0 ** -10 * (np.abs(k[:, h // 2]) @ np.abs(q[j, h]) * 0.125).max()
            assert np.all(np.abs(got[j, h] - want) <= (2 * e + 2.0 ** -9) * np.abs(v[:, h // 2]).max())
    plan.destroy()


@pytest.mark.parametrize("dtype,groups,heads,D", [(hip.F32, 1024, 1024, 128), (hip.BF16, 1, 1024, 64), (hip.F16, 512, 1024, 64)])
def test_as_many_heads_as_are_served(dev, stream, dtype, groups, heads, D):
    """1024 heads: more columns of channels than the convolution has workgroups to spread, and a workgroup's rule for few rows."""
    rng = np.random.default_rng(groups + D)
    counts, channels = [1, 0, 70, 2, 6], (2 * groups + heads) * D
    n, rows = len(counts), sum(counts)
    offsets, slots = offsets_of(counts), np.stack([rng.permutation(n)] * 2, 1).astype(np.int32)
    x = to_bits(rng.normal(0, 1, (rows, channels)), dtype)
    w = rng.normal(0, 0.5, (channels, 4)).astype(np.float32)
    windows = rng.normal(0, 1, (n, channels, 3)).astype(np.float32)
    ob, wb = dev.alloc(x.nbytes), dev.upload(windows)
    p = hip.gdn_params(dtype, n, rows, groups, heads, D, scale=D ** -0.5, eps=1e-6)
    hip.gdn_conv(stream, ob, dev.upload(x), dev.upload(w), wb, dev.upload(offsets), dev.upload(slots), p)
    stream.sync()
    want, error, new = conv_reference(from_bits(x, dtype), w.astype(np.float64), windows.astype(np.float64), offsets, slots,
                                      groups, D, D ** -0.5, 1e-6)
    got = from_bits(ob.read(np_type(dtype)).reshape(rows, channels), dtype)
    assert np.all(np.abs(got - want) <= error + HALF[dtype] * np.abs(want) + (2.0 ** -25 if dtype == hip.F16 else 0))
    assert np.array_equal(wb.read(np.float32).reshape(windows.shape), new.astype(np.float32))
    qkv = unit_rows(rng, rows, groups, heads, D, dtype)
    alpha, beta, dt, a, g, b = gates(rng, rows, heads, True)
    states = rng.normal(0, 0.3, (n, heads, D, D)).astype(np.float32)
    got = run_delta(dev, stream, dtype, qkv, alpha, beta, dt, a, states, counts, slots, groups, heads, D)
    check_delta(got, delta_reference(from_bits(qkv, dtype), g, b, states.astype(np.float64), offsets, slots, groups, heads, D, 1.0),
                dtype, rows)
    got = run_delta(dev, stream, dtype, qkv, alpha, beta, dt, a, states, None, slots, groups, heads, D, step=True)
    first = slice(0, n)
    (out, new), want = got, delta_reference(from_bits(qkv[first], dtype), g[first], b[first], states.astype(np.float64),
                                            np.arange(n + 1), slots, groups, heads, D, 1.0)
    assert np.all(out[n:] == 7.0)
    check_delta((out[first], new), want, dtype, n)


def test_a_refused_workspace_leaves_no_error(dev, stream):
    """A call whose workspace no card has (1.7 TB), and a buffer of a petabyte, are refused; the next call is sound."""
    n, heads, D = 65535, 1024, 64
    small = [dev.alloc(4 * (2 + heads) * D) for _ in range(2)] + [dev.alloc(4 * heads) for _ in range(2)]
    for refused in (lambda: hip.gdn_prompt(stream, *small, dev.alloc(4 * heads * D * D), dev.upload(np.zeros(n + 1, np.int32)),
                                           dev.upload(np.full((n, 2), -1, np.int32)),
                                           hip.gdn_params(hip.F32, n, 1, 1, heads, D, log_decay=True)),
                    lambda: dev.alloc(1 << 50)):
        with pytest.raises(hip.HipError) as e:
            refused()
        assert e.value.status == hip.ALLOCATION
        args = (i32(0, 20), i32(40, 100), i32(0, 2), np.full((2, 20), 9, np.int32), np.arange(60, dtype=np.int32), i32(0, 60), 140, 16, 320)
        for w, g in zip(plan_reference(*args), run_plan(dev, stream, *args)):
            assert np.array_equal(w, g)
        test_a_prompt_in_pieces(dev, stream, 64)


def test_two_streams_at_once(dev, stream):
    s2 = hip.Stream(dev)
    rng = np.random.default_rng(2)
    groups, heads, D, counts = 2, 4, 128, [200, 90]
    cases = []
    for s in (stream, s2):
        qkv = unit_rows(rng, 290, groups, heads, D, hip.F32)
        alpha, beta, _, _, g, b = gates(rng, 290, heads, False)
        states = rng.normal(0, 0.3, (4, heads, D, D)).astype(np.float32)
        bufs = [dev.alloc(290 * heads * D * 4), dev.upload(qkv), dev.upload(alpha), dev.upload(beta), dev.upload(states),
                dev.upload(offsets_of(counts)), dev.upload(i32(0, 2, 1, 3))]
        cases.append((s, bufs, delta_reference(qkv.astype(np.float64), g, b, states.astype(np.float64), offsets_of(counts),
                                               np.array([[0, 2], [1, 3]]), groups, heads, D, 1.0)))
    p = hip.gdn_params(hip.F32, 2, 290, groups, heads, D, log_decay=True)
    for _ in range(20):
        for s, bufs, _ in cases:
            hip.gdn_prompt(s, *bufs, p)
    stream.sync()
    s2.sync()
    for _, bufs, want in cases:
        got = bufs[0].read(np.float32).reshape(290, heads, D), bufs[4].read(np.float32).reshape(4, heads, D, D)
        check_delta(got, want, hip.F32, 290)
    s2.destroy()


def test_states_past_four_gigabytes(dev, stream):
    """Slots whose states lie behind 2^32 bytes, for the delta rule, a token and the convolution."""
    rng = np.random.default_rng(4)
    groups, heads, D = 16, 16, 128
    size, far = heads * D * D * 4, 4300
    pool = dev.alloc((far + 2) * size)
    state = rng.normal(0, 0.3, (1, heads, D, D)).astype(np.float32)
    src = dev.upload(state)
    hip.check(hip.lib().yuuka_buffer_copy(stream.ptr, pool.ptr, far * size, src.ptr, 0, size, None), "copy")
    rows = 66
    qkv = unit_rows(rng, rows, groups, heads, D, hip.F32)
    alpha, beta, _, _, g, b = gates(rng, rows, heads, False)
    want = delta_reference(qkv.astype(np.float64), g, b, state.astype(np.float64), i32(0, rows), np.array([[0, 0]]), groups,
                           heads, D, 1.0)
    ob = dev.alloc(rows * heads * D * 4)
    bufs = [ob, dev.upload(qkv), dev.upload(alpha), dev.upload(beta), pool]
    hip.gdn_prompt(stream, *bufs, dev.upload(i32(0, rows - 1)), dev.upload(i32(far, far + 1)),
                   hip.gdn_params(hip.F32, 1, rows, groups, heads, D, log_decay=True))
    first = ob.read(np.float32).reshape(rows, heads, D)[:rows - 1] if stream.sync() is None else None
    last = [dev.upload(x[rows - 1:]) for x in (qkv, alpha, beta)]
    ob2 = dev.alloc(heads * D * 4)
    hip.gdn_step(stream, ob2, *last, pool, dev.upload(i32(far + 1, far + 1)),
                 hip.gdn_params(hip.F32, 1, 1, groups, heads, D, log_decay=True))
    stream.sync()
    out = np.concatenate([first, ob2.read(np.float32).reshape(1, heads, D)])
    got = pool.read(np.float32, heads * D * D, (far + 1) * size).reshape(1, heads, D, D)
    check_delta((out, got), want, hip.F32, rows)
    pool.free()


def test_windows_and_rows_past_four_gigabytes(dev, stream):
    """Windows in slots and rows that lie behind 2^32 bytes: the convolution, and the delta rule over the same rows."""
    rng = np.random.default_rng(14)
    groups, heads, D, rows, far = 16, 16, 128, 180000, 59000
    channels, counts = (2 * groups + heads) * D, [2, 70]
    front, live = rows - sum(counts), sum(counts)
    x, y, pool = dev.alloc(rows * channels * 4), dev.alloc(rows * channels * 4), dev.alloc((far + 4) * channels * 3 * 4)
    copy = hip.lib().yuuka_buffer_copy

    def put(buf, at, data):
        src = dev.upload(data)
        hip.check(copy(stream.ptr, buf.ptr, at, src.ptr, 0, data.nbytes, None), "copy")
        stream.sync()

    data = rng.normal(0, 1, (live, channels)).astype(np.float32)
    windows = rng.normal(0, 1, (4, channels, 3)).astype(np.float32)
    w = rng.normal(0, 0.5, (channels, 4)).astype(np.float32)
    put(x, front * channels * 4, data)
    put(pool, far * channels * 12, windows)
    offsets, slots = offsets_of(counts), np.array([[0, 2], [1, 1]])
    ends, where = dev.upload(offsets + i32(front)), dev.upload((slots + far).astype(np.int32))
    p = hip.gdn_params(hip.F32, 2, rows, groups, heads, D, scale=D ** -0.5, eps=1e-6)
    hip.gdn_conv(stream, y, x, dev.upload(w), pool, ends, where, p)
    stream.sync()
    want, error, new = conv_reference(data.astype(np.float64), w.astype(np.float64), windows.astype(np.float64), offsets, slots,
                                      groups, D, D ** -0.5, 1e-6)
    got = y.read(np.float32, live * channels, front * channels * 4).reshape(live, channels)
    assert np.all(np.abs(got - want) <= error + U * np.abs(want))
    assert np.array_equal(pool.read(np.float32, 4 * channels * 3, far * channels * 12).reshape(windows.shape), new.astype(np.float32))
    qkv = unit_rows(rng, live, groups, heads, D, hip.F32)
    put(x, front * channels * 4, qkv)
    alpha, beta, _, _, g, b = gates(rng, live, heads, False)
    states = rng.normal(0, 0.3, (3, heads, D, D)).astype(np.float32)
    gap = np.zeros((front, heads), np.float32)
    ob, sb = dev.alloc(rows * heads * D * 4), dev.upload(states)
    p.log_decay = 1
    p.scale = 1.0
    hip.gdn_prompt(stream, ob, x, dev.upload(np.concatenate([gap, alpha])), dev.upload(np.concatenate([gap, beta])), sb, ends,
                   dev.upload(slots.astype(np.int32)), p)
    stream.sync()
    got = ob.read(np.float32, live * heads * D, front * heads * D * 4).reshape(live, heads, D), sb.read(np.float32).reshape(states.shape)
    want = delta_reference(qkv.astype(np.float64), g, b, states.astype(np.float64), offsets, slots, groups, heads, D, 1.0)
    check_delta(got, want, hip.F32, live)
    for buf in (x, y, pool, ob):
        buf.free()

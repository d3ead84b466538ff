"""How exact the gated delta rule over ragged rows is: root mean squares of the errors
of outputs and states, against a bound that float32 sums keep and factors cut to 16 bits
do not. The worst-case bounds of test_gpu_ragged.py, which hold for every element, are
a hundred times wider.

The bound. u = 2^-24 is half a step of float32; over many values a rounding's error has
the root mean square u / sqrt(3) of the value at most. What a row adds to a column of the
state, relative to the column's norm: one rounding of the product with the decay, two of
the decay itself (its exponent and the exponential), one of the sum with k d, and one for
k.S, whose partial sums are no larger than |k| |S| (the value d beside it is counted in
the column's largest norm): sqrt(1 + 4 + 1 + 1) u / sqrt(3) = 1.5 u. A later row shrinks
it by its decay, and for |k| <= 1 and beta in 0..1 nothing enlarges it; independent errors
add as squares. With m the largest sum, over the rows, of the squared decays since each
row before, the column is off by 1.5 u sqrt(m). An output is the product with a query
whose direction the errors do not know: of |q| times the column's norm 1 / sqrt(D) of
that, and u more for its own sum."""
from __future__ import annotations

import math

import numpy as np
import pytest

from test_gpu_ragged import U, _bounds, delta_reference, from_bits, gates, i32, offsets_of, run_delta, unit_rows
from yuuka_amd import hip


def inputs(seed, rows, requests, groups, heads, D, dtype=hip.F32):
    """Rows of a few heads that remember 10 to 250 rows, and states."""
    rng = np.random.default_rng(seed)
    qkv = unit_rows(rng, rows, groups, heads, D, dtype)
    _, beta, _, _, _, b = gates(rng, rows, heads, False)
    alpha = (-np.exp(rng.uniform(math.log(0.002), math.log(0.05), (rows, heads)))).astype(np.float32)
    states = rng.normal(0, 0.3, (requests, heads, D, D)).astype(np.float32)
    return qkv, alpha, beta, states


def errors(got, want, counts, D):
    """Root mean squares in u: of the outputs relative to |q| times the largest norm so far of their column, of the states
    relative to that of the column (an error of its norm)."""
    (out, new), (w_out, off, w_new, new_off) = got, want
    c = np.repeat([_bounds(n, D) for n in counts], counts)[:, None, None]
    most = np.stack([new_off[j] / _bounds(n, D) for j, n in enumerate(counts)])
    return (float(np.sqrt(np.mean(((out - w_out) / (off / c)) ** 2)) / U),
            float(np.sqrt(np.mean(((new - w_new) / most) ** 2) * D) / U))


def bounds(g, counts, D):
    offsets, most = offsets_of(counts), []
    for j in range(len(counts)):
        m = np.zeros(g.shape[1])
        best = m
        for r in range(offsets[j], offsets[j + 1]):
            m = m * np.exp(2 * g[r]) + 1
            best = np.maximum(best, m)
        most.append(best)
    state = 1.5 * math.sqrt(np.mean(most))
    return state / math.sqrt(D) + 1, state


# ------------------------------------------- the chunked rule with factors cut on purpose

def parts(x, n):
    """A float32 as the sum of n bf16, each cut off."""
    out, x = [], np.ascontiguousarray(x, np.float32)
    for _ in range(n):
        out.append((x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32))
        x = np.ascontiguousarray(x - out[-1])
    return out


def product(a, b, a_parts, b_parts, small=True):
    a, b = parts(a, a_parts), parts(b, b_parts)
    low = np.zeros(1, np.float32)
    for order in (2, 1):
        for i in range(order + 1):
            if i < a_parts and order - i < b_parts:
                low = low + np.matmul(a[i], b[order - i])
    return np.matmul(a[0], b[0]) + (low if small else 0)


def by_chunks(qkv, g, beta, state, groups, heads, D, cut=None):
    """64 rows at a time in float32, every factor as three bf16 parts; `cut` names one with two, or the product whose small
    part is lost."""
    n = {name: 2 if name == cut else 3 for name in ("K", "S", "T", "R", "Q", "P", "V", "tail")}
    rows = len(qkv)
    x, group = qkv.reshape(rows, -1, D).astype(np.float32), np.arange(heads) % groups
    q, k, v = (np.ascontiguousarray(y.transpose(1, 0, 2)) for y in (x[:, group], x[:, groups + group], x[:, 2 * groups:]))
    g, beta, S = g.T.astype(np.float64), beta.T.astype(np.float32), state.astype(np.float32)
    out = np.zeros((heads, rows, D), np.float32)
    for first in range(0, rows, 64):
        these = slice(first, min(first + 64, rows))
        c = np.cumsum(g[:, these], 1)
        low = np.tril(np.ones((c.shape[1],) * 2, bool))
        fall = np.exp(np.where(low, c[:, :, None] - c[:, None], -np.inf)).astype(np.float32)
        K, Q, V, b = k[:, these], q[:, these], v[:, these], beta[:, these, None]
        turned = K.transpose(0, 2, 1)
        T = np.linalg.inv(np.eye(c.shape[1]) + np.tril(np.matmul(K, turned) * fall * b, -1).astype(np.float64)).astype(np.float32)
        P = np.matmul(Q, turned) * fall
        since, tail = np.exp(c).astype(np.float32)[:, :, None], np.exp(c[:, -1:] - c).astype(np.float32)[:, :, None]
        R = b * V - b * since * product(K, S, n["K"], n["S"], cut != "K S")
        new = product(T, R, n["T"], n["R"], cut != "T R")
        out[:, these] = since * product(Q, S, n["Q"], n["S"], cut != "Q S") + product(P, new, n["P"], n["V"], cut != "P V")
        S = S * since[:, -1:] + product(turned, new * tail, n["K"], n["tail"], cut != "K V")
    return out.transpose(1, 0, 2), S


CUTS = ["K", "S", "T", "R", "Q", "P", "V", "tail", "K S", "T R", "Q S", "P V", "K V"]


@pytest.mark.parametrize("rows,D", [(130, 64), (300, 64), (130, 128), (300, 128)])
def test_the_bound_knows_a_lost_part(rows, D):
    """On the CPU: float32 as three parts keeps the bound with room, and every factor or sum that loses one breaks it."""
    groups, heads = 2, 4
    qkv, alpha, beta, states = inputs(rows + D, rows, 1, groups, heads, D)
    g, b = alpha.astype(np.float64), beta.astype(np.float64)
    want = delta_reference(qkv.astype(np.float64), g, b, states.astype(np.float64), i32(0, rows), np.array([[0, 0]]), groups,
                           heads, D, 1.0)
    limit = bounds(g, [rows], D)

    def found(cut):
        out, new = by_chunks(qkv, g, b, states[0], groups, heads, D, cut)
        return errors((out, new[None]), want, [rows], D)

    assert all(2 * e < most for e, most in zip(found(None), limit)), (found(None), limit)
    for cut in CUTS:
        assert any(e > most for e, most in zip(found(cut), limit)), (cut, found(cut), limit)


# ----------------------------------------------------------------------- the kernels

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [hip.F32, hip.F16, hip.BF16])
@pytest.mark.parametrize("counts,groups,heads,D", [([130], 2, 4, 64), ([300], 2, 4, 128), ([100] * 16, 4, 4, 128),
                                                   ([90] * 32, 2, 4, 64), ([80] * 33, 2, 4, 128), ([70] * 64, 2, 4, 64)])
def test_prompt_is_as_exact_as_float32(dev, stream, dtype, counts, groups, heads, D):
    """One, two and four tiles of columns a workgroup. (16-bit outputs are rounded, the states are not.)"""
    n, rows = len(counts), sum(counts)
    qkv, alpha, beta, states = inputs(rows + D, rows, n, groups, heads, D, dtype)
    g, b = alpha.astype(np.float64), beta.astype(np.float64)
    slots = np.stack([np.arange(n)] * 2, 1)
    got = run_delta(dev, stream, dtype, qkv, alpha, beta, None, None, states, counts, slots, groups, heads, D)
    want = delta_reference(from_bits(qkv, dtype), g, b, states.astype(np.float64), offsets_of(counts), slots, groups, heads, D, 1.0)
    (out, state), limit = errors(got, want, counts, D), bounds(g, counts, D)
    assert state <= limit[1], (state, limit)
    if dtype == hip.F32:
        assert out <= limit[0], (out, limit)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("piece", [0, 1, 2])
def test_tokens_are_as_exact_as_float32(dev, stream, D, piece):
    """Row by row: by the step (0), and by prompts of one and two rows."""
    groups, heads, rows = 2, 4, 64
    qkv, alpha, beta, states = inputs(D + piece, rows, 1, groups, heads, D)
    g, b = alpha.astype(np.float64), beta.astype(np.float64)
    want = delta_reference(qkv.astype(np.float64), g, b, states.astype(np.float64), i32(0, rows), np.array([[0, 0]]), groups,
                           heads, D, 1.0)
    outs, state = [], states
    for at in range(0, rows, max(piece, 1)):
        cut = slice(at, at + max(piece, 1))
        o, state = run_delta(dev, stream, hip.F32, qkv[cut], alpha[cut], beta[cut], None, None, state, [max(piece, 1)], [[0, 0]],
                             groups, heads, D, step=piece == 0)
        outs.append(o)
    for e, most in zip(errors((np.concatenate(outs), state), want, [rows], D), bounds(g, [rows], D)):
        assert e <= most, (e, most)

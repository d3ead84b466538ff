"""Performance cases of the quantised key/value cache: what a serving program
has it compute, at the sizes it is used at.

A case is a dict; "kind" names the operator:

  append  new key and value rows of a batch of requests, rounded into the
          paged Q8_0 pools (yuuka_kv_append) and read back as the values the
          pools then stand for (yuuka_kv_read of the same rows)
  read    the first `context` tokens of every request back to float32
          (yuuka_kv_read)
  attn    attention of the requests' newest rows over their paged cache, each
          request at its own length (yuuka_attn_decode): one row is a decode
          step, more are the rows of a speculative verify step

Q8_0 page of `block` tokens: block x kv_dim int8 digits, then block x
kv_dim / 32 half scales; dim i of a token is digit * scale of its block of 32.
Every 64 dims' digits are stored as a 16 x 4 matrix: byte 4 r + j of the 64
holds dim 16 j + r.
"""
from __future__ import annotations

import math

import torch

own = False

# heads, key/value heads, head width: the decoder's own shapes, then generic ones
SHAPES = [(16, 4, 256), (8, 2, 256), (16, 2, 256), (32, 8, 128), (16, 16, 64)]


def listed():
    return [
        # one decoded token of one request, one layer: launch latency
        dict(name="append_token", kind="append", requests=1, rows=1, context=517, block=16, kv_heads=4, head_dim=256),
        # a verify step of sixteen requests, k = 8
        dict(name="append_batch16", kind="append", requests=16, rows=9, context=4096, block=16, kv_heads=4,
             head_dim=256),
        # a whole prompt at once, eight 128-wide heads
        dict(name="append_prompt", kind="append", requests=1, rows=8191, context=0, block=16, kv_heads=8,
             head_dim=128),
        # one request's cache read back, a partial last page
        dict(name="read_request", kind="read", requests=1, context=517, block=16, kv_heads=4, head_dim=256),
        # sixteen requests' prefixes read back
        dict(name="read_batch16", kind="read", requests=16, context=4000, block=16, kv_heads=4, head_dim=256),
        # a decode step early in a conversation
        dict(name="decode_short", kind="attn", requests=1, rows=1, context=517, spread=0, block=16, heads=16,
             kv_heads=4, head_dim=256, gated=True, kv="q8_0"),
        # a decode step of one request far into a long document
        dict(name="decode_long", kind="attn", requests=1, rows=1, context=120001, spread=0, block=16, heads=16,
             kv_heads=4, head_dim=256, gated=True, kv="q8_0"),
        # a decode step of sixteen requests with 4k contexts
        dict(name="decode_batch16", kind="attn", requests=16, rows=1, context=4096, spread=0, block=16, heads=16,
             kv_heads=4, head_dim=256, gated=True, kv="q8_0"),
        # a decode step of many requests of very different lengths, generic widths
        dict(name="decode_ragged96", kind="attn", requests=96, rows=1, context=3001, spread=1, block=64, heads=32,
             kv_heads=8, head_dim=128, gated=False, kv="q8_0"),
        # the same step over a half-precision cache
        dict(name="decode_batch16_f16", kind="attn", requests=16, rows=1, context=4096, spread=0, block=16, heads=32,
             kv_heads=8, head_dim=128, gated=False, kv="f16"),
        # a verify step of one request, k = 4
        dict(name="verify_short", kind="attn", requests=1, rows=5, context=1029, spread=0, block=16, heads=16,
             kv_heads=4, head_dim=256, gated=True, kv="q8_0"),
        # a verify step of four requests with 16k contexts, k = 16
        dict(name="verify_batch4", kind="attn", requests=4, rows=17, context=16384, spread=0, block=16, heads=16,
             kv_heads=4, head_dim=256, gated=True, kv="q8_0"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "attn", "attn", "attn"])
    heads, kv_heads, head_dim = rng.choice(SHAPES)
    block = rng.choice([16, 16, 32, 64])
    requests = _log_int(rng, 1, 96)
    kv_dim = kv_heads * head_dim
    if kind == "append":
        return dict(kind=kind, requests=requests, rows=_log_int(rng, 1, 8191 // requests),
                    context=rng.randint(0, 4096), block=block, kv_heads=kv_heads, head_dim=head_dim)
    if kind == "read":
        return dict(kind=kind, requests=requests, context=_log_int(rng, 1, 64000 * 1024 // kv_dim // requests),
                    block=block, kv_heads=kv_heads, head_dim=head_dim)
    rows = rng.choice([1, 1, rng.randint(2, 17)])
    tokens = 120000 * 1024 // kv_dim if rows == 1 else 65536 * 1024 // max(kv_dim, heads * head_dim // 4)
    return dict(kind=kind, requests=requests, rows=rows,
                context=_log_int(rng, rows, max(rows, min(120001, tokens // requests))),
                spread=rng.choice([0, 1]), block=block, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                gated=rng.choice([True, False]), kv=rng.choice(["q8_0", "q8_0", "f16"]))


def _lengths(case):
    """Tokens cached before the new rows, by request: all `context`, or spread evenly from an eighth of it up to it."""
    n, ctx = case["requests"], case["context"]
    if not case.get("spread"):
        return [ctx] * n
    return [max(1, ctx * (n + 7 * (j + 1)) // (8 * n)) for j in range(n)]


def work(case):
    kv_dim = case["kv_heads"] * case["head_dim"]
    quantised = kv_dim * 34 / 32
    if case["kind"] == "append":
        n = 2 * case["requests"] * case["rows"]
        # float32 rows in, packed rows out and in again, float32 values out
        return {"bytes": n * (8 * kv_dim + 2 * quantised), "flops": n * kv_dim * 4}
    if case["kind"] == "read":
        n = 2 * case["requests"] * case["context"]
        return {"bytes": n * (4 * kv_dim + quantised), "flops": n * kv_dim}
    rows, width = case["rows"], case["heads"] * case["head_dim"]
    tokens = sum(_lengths(case)) + case["requests"] * rows
    pairs = sum(rows * ctx + rows * (rows + 1) // 2 for ctx in _lengths(case))
    per_token = 2 * (quantised if case["kv"] == "q8_0" else 2 * kv_dim)
    io = case["requests"] * rows * width * 4 * (3 if case["gated"] else 2)
    return {"bytes": tokens * per_token + io, "flops": 4 * pairs * width}


# ------------------------------------------------------------ device memory

_device = _stream = None


def _open():
    """The library's device and the stream that every call runs on."""
    global _device, _stream
    from yuuka_amd import hip
    if _device is None:
        torch.cuda.init()
        _device = hip.Device(0)
        _stream = hip.Stream(_device)
    return hip, _device, _stream


class _Shared:
    """A library buffer as torch sees it."""

    def __init__(self, buf, shape, typestr):
        self.buf = buf
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr=typestr, data=(buf.device_ptr, False),
                                             version=2)


_TYPESTR = {torch.float32: "<f4", torch.int32: "<i4", torch.uint8: "|u1"}


def _put(state, name, t):
    """Where a program keeps t: device memory, which is a library buffer (name + "_buf") for the library's calls."""
    if own:
        _, dev, _ = _open()
        buf = dev.alloc(max(16, t.numel() * t.element_size()))
        state[name + "_buf"] = buf
        shared = torch.as_tensor(_Shared(buf, t.shape, _TYPESTR[t.dtype]), device="cuda")
        shared.copy_(t)
        t = shared
    state[name] = t


# ------------------------------------------------------------------- inputs

def _packed_pool(g, pages, block, kv_dim):
    """Pages of random digits and scales, as rows of spread about one leave them."""
    digits = torch.randn(pages, block * kv_dim, generator=g, device="cuda").mul_(42).round_().clamp_(-127, 127)
    scales = 0.015 + 0.02 * torch.rand(pages, block * kv_dim // 32, generator=g, device="cuda")
    return torch.cat([digits.to(torch.int8).view(torch.uint8), scales.to(torch.float16).view(torch.uint8)], 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 % (1 << 62) + 29)
    c, n = case, case["requests"]
    kv_dim = c["kv_heads"] * c["head_dim"]
    rows = c.get("rows", 0)
    blocks = -(-(c["context"] + rows) // c["block"])  # pages of one request
    pages = n * blocks
    s = {"case": c}
    position = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32)
    position = position[torch.randperm(n, generator=g, device="cuda")]
    s["position"] = position.to(torch.int64)
    _put(s, "positions", torch.stack([torch.zeros_like(position), position], 1).contiguous())
    _put(s, "table", torch.randperm(pages, generator=g, device="cuda").to(torch.int32).reshape(n, blocks))
    for name in ("kpool", "vpool"):
        if c.get("kv") == "f16":
            pool = torch.randn(pages, c["block"] * kv_dim, generator=g, device="cuda").to(torch.float16)
            pool = pool.view(torch.uint8)
        else:
            pool = _packed_pool(g, pages, c["block"], kv_dim)
        _put(s, name, pool)
    if c["kind"] == "append":
        for name in ("k", "v"):
            _put(s, name, torch.randn(n, rows, kv_dim, generator=g, device="cuda"))
    if c["kind"] == "attn":
        width = c["head_dim"] * (2 if c["gated"] else 1)
        _put(s, "q", torch.randn(n, rows, c["heads"], width, generator=g, device="cuda"))
        _put(s, "out", torch.zeros(n, rows, c["heads"], c["head_dim"], device="cuda"))
    else:
        for name in ("k_out", "v_out"):
            _put(s, name, torch.zeros(n, rows or c["context"], kv_dim, device="cuda"))
    return s


# ---------------------------------------------------------------------- run

def run(state):
    if own:
        return _run_library(state)
    c = state["case"]
    if c["kind"] == "append":
        at = state["position"][:, None] + torch.arange(c["rows"], device="cuda")
        return [_append(state, "kpool", state["k"], at), _append(state, "vpool", state["v"], at)]
    if c["kind"] == "read":
        at = torch.arange(c["context"], device="cuda").expand(c["requests"], -1)
        return [_values(state, "kpool", at).flatten(2), _values(state, "vpool", at).flatten(2)]
    return _attention(state)


def _run_library(state):
    hip, _, stream = _open()
    c = state["case"]
    b = {name: state.get(name + "_buf") for name in ("k", "v", "kpool", "vpool", "table", "positions", "q")}
    capacity = state["table"].shape[1] * c["block"]
    rows = c.get("rows") or c["context"]
    dtype = hip.F16 if c.get("kv") == "f16" else hip.Q8_0
    p = hip.kv_params(dtype, c["block"], capacity, c["kv_heads"], c["head_dim"], rows, c["requests"],
                      heads=c.get("heads", 0), gated=c.get("gated", False), scale=c["head_dim"] ** -0.5)
    if c["kind"] == "attn":
        hip.attn_decode(stream, state["out_buf"], b["q"], b["kpool"], b["vpool"], b["table"], b["positions"], p)
        return state["out"]
    if c["kind"] == "append":
        hip.kv_append(stream, b["k"], b["v"], b["kpool"], b["vpool"], b["table"], b["positions"], p)
    hip.kv_read(stream, state["k_out_buf"], state["v_out_buf"], b["kpool"], b["vpool"], b["table"], p,
                positions=b["positions"] if c["kind"] == "append" else None)
    return [state["k_out"], state["v_out"]]


def _slots(state, at):
    """(page, slot in the page) of positions at [requests][n]."""
    block = state["case"]["block"]
    at = at.clamp(max=state["table"].shape[1] * block - 1)
    return torch.gather(state["table"].to(torch.int64), 1, at // block), at % block


def _planes(state, pool):
    """A packed pool's digits [pages][block][kv_dim] and scales [pages][block][kv_dim / 32]."""
    c = state["case"]
    n = c["block"] * c["kv_heads"] * c["head_dim"]
    return (state[pool][:, :n].view(torch.int8).unflatten(1, (c["block"], -1)),
            state[pool][:, n:].view(torch.float16).unflatten(1, (c["block"], -1)))


def _values(state, pool, at):
    """What the pool holds at positions at [requests][n], float32 [requests][n][kv_heads][head_dim]."""
    c = state["case"]
    page, slot = _slots(state, at)
    if c.get("kv") == "f16":
        rows = state[pool].view(torch.float16).unflatten(1, (c["block"], -1))[page, slot]
        return rows.to(torch.float32).unflatten(2, (c["kv_heads"], c["head_dim"]))
    digits, scales = _planes(state, pool)
    digits = digits[page, slot].unflatten(2, (-1, 16, 4)).transpose(3, 4).to(torch.float32)
    scales = scales[page, slot].to(torch.float32)
    values = digits.flatten(2).unflatten(2, (-1, 32)) * scales.unsqueeze(3)
    return values.flatten(2).unflatten(2, (c["kv_heads"], c["head_dim"]))


def _half_up(x):
    """Positive float32 values in the range of normal and subnormal halves, to the nearest half, ties upwards."""
    normal = ((x.view(torch.int32) + 0x1000) & ~0x1FFF).view(torch.float32)
    small = torch.floor(x * 2.0 ** 24 + 0.5) * 2.0 ** -24
    return torch.where(x >= 2.0 ** -14, normal, small).to(torch.float16)


def _append(state, pool, x, at):
    x = x.unflatten(2, (-1, 32))
    scale = x.abs().amax(3, keepdim=True) / 127
    steps = torch.where(scale > 0, x / scale, 0).to(torch.float64)  # in 64 bits from here: halves round away from zero
    digits = (torch.floor(steps.abs() + 0.5) * torch.sign(steps)).to(torch.int8)
    page, slot = _slots(state, at)
    to_digits, to_scales = _planes(state, pool)
    to_digits[page, slot] = digits.flatten(2).unflatten(2, (-1, 4, 16)).transpose(3, 4).flatten(2)
    to_scales[page, slot] = _half_up(scale.squeeze(3))
    return _values(state, pool, at).flatten(2)


def _attention(state):
    c = state["case"]
    n, rows, kv_heads, d = c["requests"], c["rows"], c["kv_heads"], c["head_dim"]
    q, gate = state["q"][..., :d], state["q"][..., d:]
    at = torch.arange(c["context"] + rows, device="cuda").expand(n, -1)
    keys = _values(state, "kpool", at).transpose(1, 2).contiguous()  # [requests][kv_heads][tokens][d]
    values = _values(state, "vpool", at).transpose(1, 2).contiguous()
    group = c["heads"] // kv_heads
    q = q.unflatten(2, (kv_heads, group)).permute(0, 2, 1, 3, 4).reshape(n, kv_heads, rows * group, d)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()) * d ** -0.5
    last = state["position"][:, None] + torch.arange(rows, device="cuda")
    seen = at[:, None, :] <= last[:, :, None]  # [requests][rows][tokens]
    scores = scores.unflatten(2, (rows, group)).masked_fill(~seen[:, None, :, None], -math.inf)
    weights = torch.exp(scores - scores.amax(4, keepdim=True))
    weights = (weights / weights.sum(4, keepdim=True)).flatten(2, 3)
    out = torch.matmul(weights, values).unflatten(2, (rows, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out / (1 + torch.exp(-gate)) if c["gated"] else out.contiguous()


# -------------------------------------------------------------------- exact

def _stored(rows):
    """Float64 rows [..., kv_dim] after the Q8_0 rounding: blocks of 32, s = max|x| / 127 and x / s rounded to float32,
    the scale s to the nearest half (ties upwards), the digit x / s to the nearest integer (halves away from zero)."""
    x = rows.unflatten(-1, (-1, 32))
    s = (x.abs().amax(-1, keepdim=True) / 127).to(torch.float32).to(torch.float64)
    step = torch.exp2((torch.frexp(s)[1] - 11).clamp(min=-24).to(torch.float64))
    digits = (x / s).to(torch.float32).to(torch.float64)
    digits = digits.trunc() + digits.frac().mul(2).trunc()
    return (digits.nan_to_num() * torch.floor(s / step + 0.5) * step).flatten(-2)


def _exact_rows(c, s, pool, j, n):
    """Request j's first n tokens in float64 [n][kv_heads][head_dim], page by page."""
    kv_heads, d, block = c["kv_heads"], c["head_dim"], c["block"]
    pages = s[pool][s["table"][j, : -(-n // block)].to(torch.int64)]
    if c.get("kv") == "f16":
        return pages.view(torch.float16).to(torch.float64).reshape(-1, kv_heads, d)[:n]
    split = block * kv_heads * d
    digits = pages[:, :split].contiguous().view(torch.int8).reshape(-1, kv_heads, d // 64, 16, 4)[:n].to(torch.float64)
    scales = pages[:, split:].contiguous().view(torch.float16).reshape(-1, kv_heads, d // 32)[:n].to(torch.float64)
    dim = torch.arange(d, device="cuda")
    return digits[:, :, dim // 64, dim % 16, dim % 64 // 16] * scales[:, :, dim // 32]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "append":
        return [_stored(s["k"].to(torch.float64)), _stored(s["v"].to(torch.float64))]
    if c["kind"] == "read":
        return [torch.stack([_exact_rows(c, s, pool, j, c["context"]).flatten(1) for j in range(c["requests"])])
                for pool in ("kpool", "vpool")]
    d, group, outs = c["head_dim"], c["heads"] // c["kv_heads"], []
    for j in range(c["requests"]):
        first = int(s["position"][j])
        n = first + c["rows"]
        keys, values = (_exact_rows(c, s, pool, j, n).transpose(0, 1).contiguous() for pool in ("kpool", "vpool"))
        q = s["q"][j].to(torch.float64)
        query = q[..., :d].reshape(c["rows"], c["kv_heads"], group, d)
        after = torch.arange(n, device="cuda") > torch.arange(first, n, device="cuda")[:, None]
        for_head = []
        for h in range(c["kv_heads"]):
            scores = (query[:, h].flatten(0, 1) @ keys[h].t()).unflatten(0, (c["rows"], group)) / math.sqrt(d)
            scores = scores.masked_fill(after[:, None], -math.inf)
            for_head.append(torch.softmax(scores, 2).flatten(0, 1) @ values[h])
        out = torch.stack([o.unflatten(0, (c["rows"], group)) for o in for_head], 1).flatten(1, 2)
        outs.append(out * torch.sigmoid(q[..., d:]) if c["gated"] else out)
    return torch.stack(outs)

"""Performance cases of a ragged batch: requests with different numbers of new
rows, laid one after another without padding, on their way into the two kinds of
state that the decoder keeps of its context, pages and recurrent states.

A case is a dict; "kind" names the operator:

  plan    where the batch's rows go: row offsets, {request, position} and the slot
          of every row, pages from a free list into the block tables
          (yuuka_batch_plan)
  append  the rows' keys and values into the paged pools by their slots
          (yuuka_kv_append_slots)
  conv    causal convolution, SiLU and the q / k norm of the rows, with the
          requests' windows (yuuka_gdn_conv)
  gdn     the gated delta rule over the rows, with the requests' states
          (yuuka_gdn_prompt)
  step    the same for one token of every request (yuuka_gdn_step)

The rows of request j are offsets[j] .. offsets[j + 1] - 1. A row of the last three
is [q | k | v]: q and k of `groups` heads, v of `heads` heads, head h with the q and k
of group h % groups. Head h of a request has a state [head_dim][head_dim] (rows: k's
dims, columns: v's), read from the request's slot `from` (none: zeros) and left in
its slot `to`. alpha and beta are the projections' outputs: the log of a row's decay
is softplus(alpha + dt) * a, its step sigmoid(beta); or, with "coef" = "log", they
are those two themselves.
"""
from __future__ import annotations

import math

import torch

own = False

KERNEL, EPS = 4, 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the tables of a decode step of sixteen requests: launch latency
        dict(name="plan_decode16", kind="plan", requests=16, rows=16, spread=0, context=4096, block=16, capacity=16384),
        # those of 200 requests, prompts and decode steps mixed
        dict(name="plan_prompts", kind="plan", requests=200, rows=16300, spread=1, context=8000, block=16,
             capacity=32768),
        # their keys and values, one token of sixteen requests
        dict(name="append_decode16", kind="append", rows=16, block=16, kv_heads=4, head_dim=256, kv="f16", norm=True),
        # the prompts of a batch into float32 pages, eight 128-wide heads
        dict(name="append_prompts", kind="append", rows=8191, block=16, kv_heads=8, head_dim=128, kv="f32", norm=False),
        # one token of sixteen requests through the convolution
        dict(name="conv_decode16", kind="conv", requests=16, rows=16, spread=0, groups=16, heads=16, head_dim=128,
             dtype="f32"),
        # seven prompts of different lengths
        dict(name="conv_prompts", kind="conv", requests=7, rows=8191, spread=1, groups=16, heads=32, head_dim=128,
             dtype="bf16"),
        # a short prompt on the 4B-like decoder
        dict(name="gdn_short", kind="gdn", requests=1, rows=77, spread=0, groups=16, heads=16, head_dim=128,
             dtype="f32", coef="raw"),
        # a long prompt
        dict(name="gdn_prompt", kind="gdn", requests=1, rows=8191, spread=0, groups=16, heads=16, head_dim=128,
             dtype="f32", coef="raw"),
        # sixteen prompts of different lengths, twice as many value heads as groups
        dict(name="gdn_ragged16", kind="gdn", requests=16, rows=8192, spread=1, groups=16, heads=32, head_dim=128,
             dtype="bf16", coef="raw"),
        # many short prompts, narrow heads
        dict(name="gdn_ragged96", kind="gdn", requests=96, rows=6000, spread=1, groups=8, heads=16, head_dim=64,
             dtype="f16", coef="log"),
        # one token of one request
        dict(name="step_token", kind="step", requests=1, groups=16, heads=16, head_dim=128, dtype="f32", coef="raw"),
        # one token of 200 requests
        dict(name="step_batch200", kind="step", requests=200, groups=16, heads=32, head_dim=128, dtype="bf16",
             coef="raw"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "conv", "gdn", "gdn", "gdn", "step"])
    if kind == "plan":
        requests = _log_int(rng, 1, 200)
        return dict(kind=kind, requests=requests, rows=_log_int(rng, requests, 16300), spread=rng.choice([0, 1]),
                    context=_log_int(rng, 1, 8000), block=rng.choice([16, 16, 32, 48]), capacity=32768)
    if kind == "append":
        kv_heads, head_dim = rng.choice([(4, 256), (2, 256), (8, 128), (16, 64)])
        return dict(kind=kind, rows=_log_int(rng, 1, 8191), block=rng.choice([16, 16, 32, 48]), kv_heads=kv_heads,
                    head_dim=head_dim, kv=rng.choice(["f16", "f32"]), norm=rng.choice([True, False]))
    groups, heads, head_dim = rng.choice([(16, 16, 128), (16, 16, 128), (16, 32, 128), (8, 16, 128), (16, 32, 64),
                                          (8, 16, 64)])
    c = dict(kind=kind, requests=_log_int(rng, 1, 96), groups=groups, heads=heads, head_dim=head_dim,
             dtype=rng.choice(["f32", "f32", "f16", "bf16"]))
    if kind != "step":
        c.update(rows=_log_int(rng, c["requests"], 6000), spread=rng.choice([0, 1]))
    if kind != "conv":
        c.update(coef=rng.choice(["raw", "log"]))
    return c


def _counts(case):
    """New rows by request: alike, or from none or one up to a few times the mean."""
    n, rows = case["requests"], case["rows"]
    if not case["spread"]:
        return [rows // n + (j < rows % n) for j in range(n)]
    weights = [(j + 1) ** 2 for j in range(n)]
    counts = [rows * w // sum(weights) for w in weights]
    counts[-1] += rows - sum(counts)
    return counts


def _channels(case):
    return (2 * case["groups"] + case["heads"]) * case["head_dim"]


def work(case):
    c = case
    if c["kind"] == "plan":
        pages = sum(-(-n // c["block"]) for n in _counts(c))
        return {"bytes": c["requests"] * 24 + pages * 8 + c["rows"] * 16, "flops": c["rows"] * 8}
    if c["kind"] == "append":
        values = 2 * c["rows"] * c["kv_heads"] * c["head_dim"]
        return {"bytes": values * (4 + (2 if c["kv"] == "f16" else 4)) + 8 * c["rows"], "flops": values * 2}
    size = torch.empty((), dtype=DTYPES[c["dtype"]]).element_size()
    if c["kind"] == "conv":
        windows = 2 * c["requests"] * _channels(c) * (KERNEL - 1) * 4
        values = c["rows"] * _channels(c)
        return {"bytes": 2 * values * size + windows + _channels(c) * KERNEL * 4, "flops": values * (2 * KERNEL + 6)}
    rows = c.get("rows", c["requests"])
    state = c["heads"] * c["head_dim"] ** 2
    return {"bytes": rows * (size * (_channels(c) + c["heads"] * c["head_dim"]) + 8 * c["heads"])
            + 2 * c["requests"] * state * 4, "flops": 7 * rows * state}


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


_TYPESTR = {torch.float32: "<f4", torch.float16: "<f2", torch.bfloat16: "<i2", torch.int32: "<i4", torch.int64: "<i8"}


def _put(state, name, t):
    """Where a program keeps t: device memory, which is a library buffer (name + "_buf") for the library's calls."""
    if own:
        _, dev, _ = _open()
        buf = dev.alloc(max(16, t.numel() * t.element_size()))
        state[name + "_buf"] = buf
        shared = torch.as_tensor(_Shared(buf, t.shape, _TYPESTR[t.dtype]), device="cuda").view(t.dtype)
        shared.copy_(t)
        t = shared
    state[name] = t


# ------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 % (1 << 62) + 41)
    s = {"case": case}
    {"plan": _prepare_plan, "append": _prepare_append}.get(case["kind"], _prepare_recurrent)(case, s, g)
    return s


def _order(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def _prepare_plan(c, s, g):
    n, rows, block = c["requests"], c["rows"], c["block"]
    counts = torch.tensor(_counts(c), device="cuda")[_order(g, n)]
    room = torch.clamp(c["capacity"] - counts, min=0)
    # a fifth of the requests start here, the others hold up to `context` tokens
    position = (torch.rand(n, generator=g, device="cuda") * 1.25 - 0.25).clamp(min=0) * c["context"]
    position = torch.minimum(position.to(torch.int64), room)
    blocks = -(-position // block)
    width = -(-c["capacity"] // block)
    pages = n * width
    order = _order(g, pages).to(torch.int32)
    table = order.reshape(n, width).clone()
    held = torch.arange(width, device="cuda") < blocks[:, None]
    _put(s, "table", torch.where(held, table, -1).to(torch.int32))
    # the free list: pages that no table holds, after some that earlier steps took
    free = torch.cat([order.flip(0)[:5], table.flatten()[torch.argsort(held.flatten().to(torch.int32), stable=True)]])
    free = free[:5 + rows + n]
    _put(s, "free", free.contiguous())
    _put(s, "pool", torch.tensor([5, free.numel()], device="cuda", dtype=torch.int32))
    _put(s, "positions", torch.stack([torch.full_like(position, 11), position], 1).to(torch.int32).contiguous())
    _put(s, "counts", counts.to(torch.int32))
    _put(s, "blocks", blocks.to(torch.int32))
    _put(s, "offsets", torch.zeros(n + 1, device="cuda", dtype=torch.int32))
    _put(s, "row_info", torch.zeros(rows, 2, device="cuda", dtype=torch.int32))
    _put(s, "slots", torch.zeros(rows, device="cuda", dtype=torch.int64))
    _put(s, "blocks_out", torch.zeros(n, device="cuda", dtype=torch.int32))
    _put(s, "pool_out", torch.zeros(2, device="cuda", dtype=torch.int32))


def _prepare_append(c, s, g):
    rows, block, kv_dim = c["rows"], c["block"], c["kv_heads"] * c["head_dim"]
    pages = -(-rows // block) + 3
    row = torch.arange(rows, device="cuda")
    slots = _order(g, pages)[row // block] * block + row % block
    _put(s, "slots", torch.where(row >= rows - rows // 50, -1, slots))  # the last rows of a padded batch go nowhere
    for name in ("k", "v"):
        _put(s, name, torch.randn(rows, kv_dim, generator=g, device="cuda"))
    for name in ("kpool", "vpool"):
        _put(s, name, torch.randn(pages, block, kv_dim, generator=g, device="cuda").to(DTYPES[c["kv"]]))
    if c["norm"]:
        _put(s, "k_norm", 1 + 0.1 * torch.randn(c["head_dim"], generator=g, device="cuda"))


def _prepare_recurrent(c, s, g):
    n, heads, d, channels = c["requests"], c["heads"], c["head_dim"], _channels(c)
    rows, dtype = c.get("rows", n), DTYPES[c["dtype"]]
    counts = torch.tensor(_counts(c) if "rows" in c else [1] * n, device="cuda")[_order(g, n)]
    _put(s, "offsets", torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32))
    # every request's state moves from one slot to another; a few requests are new
    at = _order(g, 2 * n)
    fresh = torch.rand(n, generator=g, device="cuda") < 0.2
    _put(s, "slots", torch.stack([torch.where(fresh, -1, at[:n]), at[n:]], 1).to(torch.int32).contiguous())
    if c["kind"] == "conv":
        _put(s, "x", torch.randn(rows, channels, generator=g, device="cuda").to(dtype))
        _put(s, "weight", 0.5 * torch.randn(channels, KERNEL, generator=g, device="cuda"))
        _put(s, "state", torch.randn(2 * n, channels, KERNEL - 1, generator=g, device="cuda"))
        _put(s, "out", torch.zeros(rows, channels, device="cuda", dtype=dtype))
        return
    x = torch.randn(rows, channels, generator=g, device="cuda")
    qk = x[:, :2 * c["groups"] * d].unflatten(1, (-1, d))  # as the convolution leaves them
    qk /= torch.sqrt((qk * qk).sum(2, keepdim=True) + EPS)
    x[:, :c["groups"] * d] *= d ** -0.5
    x[:, 2 * c["groups"] * d:] *= 0.5
    _put(s, "x", x.to(dtype))
    alpha, beta = (torch.randn(rows, heads, generator=g, device="cuda") for _ in range(2))
    dt = 0.5 * torch.randn(heads, generator=g, device="cuda")
    a = -torch.exp(math.log(0.02) + math.log(100) * torch.rand(heads, generator=g, device="cuda"))
    if c["coef"] == "log":
        alpha, beta = torch.log1p(torch.exp(alpha + dt)) * a, 1 / (1 + torch.exp(-beta))
    for name, t in (("alpha", alpha), ("beta", beta), ("dt", dt), ("a", a)):
        _put(s, name, t)
    _put(s, "state", 0.2 * torch.randn(2 * n, heads, d, d, generator=g, device="cuda"))
    _put(s, "out", torch.zeros(rows, heads, d, device="cuda", dtype=dtype))


# ---------------------------------------------------------------------- run

def run(state):
    if own:
        return _run_library(state)
    return {"plan": _plan, "append": _append, "conv": _conv, "gdn": _gdn, "step": _step}[state["case"]["kind"]](state)


_PLAN = ("offsets", "row_info", "slots", "blocks_out", "pool_out", "table")


def _run_library(state):
    hip, _, stream = _open()
    c = state["case"]
    b = {name[:-4]: buf for name, buf in state.items() if name.endswith("_buf")}
    if c["kind"] == "plan":
        hip.batch_plan(stream, b["positions"], b["counts"], b["blocks"], b["table"], b["free"], b["pool"], b["offsets"],
                       b["row_info"], b["slots"], b["blocks_out"], b["pool_out"],
                       hip.batch_params(c["requests"], c["rows"], c["block"], c["capacity"]))
        return [state[name] for name in _PLAN]
    if c["kind"] == "append":
        p = hip.kv_params(hip.F16 if c["kv"] == "f16" else hip.F32, c["block"], c["block"], c["kv_heads"],
                          c["head_dim"], c["rows"], eps=EPS)
        hip.kv_append_slots(stream, b["k"], b["v"], b["kpool"], b["vpool"], b["slots"], p, k_norm=b.get("k_norm"))
        return [state["kpool"], state["vpool"]]
    dtype = {"f32": hip.F32, "f16": hip.F16, "bf16": hip.BF16}[c["dtype"]]
    p = hip.gdn_params(dtype, c["requests"], c.get("rows", c["requests"]), c["groups"], c["heads"], c["head_dim"],
                       kernel=KERNEL, scale=c["head_dim"] ** -0.5 if c["kind"] == "conv" else 1.0, eps=EPS,
                       log_decay=c.get("coef") == "log")
    if c["kind"] == "conv":
        hip.gdn_conv(stream, b["out"], b["x"], b["weight"], b["state"], b["offsets"], b["slots"], p)
        return [state["out"], state["state"]]
    gate = dict(dt=b["dt"], a=b["a"]) if c["coef"] == "raw" else {}
    if c["kind"] == "gdn":
        hip.gdn_prompt(stream, b["out"], b["x"], b["alpha"], b["beta"], b["state"], b["offsets"], b["slots"], p, **gate)
    else:
        hip.gdn_step(stream, b["out"], b["x"], b["alpha"], b["beta"], b["state"], b["slots"], p, **gate)
    return [state["out"], state["state"]]


def _row_requests(s, rows):
    """Request of every row and the row's number in it."""
    row = torch.arange(rows, device="cuda")
    request = torch.searchsorted(s["offsets"][1:], row.to(torch.int32), right=True)
    return request, row - s["offsets"][request]


def _plan(s):
    c = s["case"]
    rows, block = c["rows"], c["block"]
    position, counts, blocks = (t.to(torch.int64) for t in (s["positions"][:, 1], s["counts"], s["blocks"]))
    s["offsets"][1:] = counts.cumsum(0)
    request, i = _row_requests(s, rows)
    at = position[request] + i
    # pages from the first new row's block, or the first that the table lacks, to the last row's
    first = torch.maximum(blocks, position // block)
    new = torch.where(counts > 0, (-(-(position + counts) // block) - first).clamp(min=0), 0)
    base = s["pool"][0] + new.cumsum(0) - new
    taken = (s["pool"][1] - base).clamp(min=0).minimum(new)
    number = at // block - first[request]  # of the row's page among its request's new ones
    free = (base[request] + number).clamp(0, s["free"].numel() - 1)
    page = torch.where(number < 0, s["table"][request, at // block],
                       torch.where(number < taken[request], s["free"][free], -1))
    s["table"][request, at // block] = page
    s["row_info"][:, 0] = request
    s["row_info"][:, 1] = at
    s["slots"].copy_(torch.where(page < 0, -1, page.to(torch.int64) * block + at % block))
    s["blocks_out"].copy_(torch.where(taken > 0, first + taken, blocks))
    s["pool_out"].copy_(torch.stack([s["pool"][0] + taken.sum(), (new - taken).sum()]))
    return [s[name] for name in _PLAN]


def _append(s):
    c = s["case"]
    slot = s["slots"]
    k = s["k"].unflatten(1, (-1, c["head_dim"]))
    if c["norm"]:
        k = k * (s["k_norm"] / torch.sqrt((k * k).mean(2, keepdim=True) + EPS))
    # rows that go nowhere are written as the first row once more, which has a slot in every case
    row = torch.where(slot >= 0, torch.arange(c["rows"], device="cuda"), 0)
    for pool, x in ((s["kpool"], k.flatten(1)), (s["vpool"], s["v"])):
        pool.flatten(0, 1)[slot[row]] = x[row].to(pool.dtype)
    return [s["kpool"], s["vpool"]]


def _conv(s):
    c = s["case"]
    x, w = s["x"].to(torch.float32), s["weight"]
    request, i = _row_requests(s, c["rows"])
    start = s["slots"][:, 0].to(torch.int64)
    old = torch.where((start >= 0)[:, None, None], s["state"][start.clamp(min=0)], 0.0)  # [requests][channels][3]
    row = torch.arange(c["rows"], device="cuda")

    def before(back, request, i, row):  # the inputs `back` rows before
        past = old[request, :, (i - back + KERNEL - 1).clamp(0, KERNEL - 2)]
        return torch.where((i >= back)[:, None], x[(row - back).clamp(min=0)], past)

    y = sum(before(back, request, i, row) * w[:, KERNEL - 1 - back] for back in range(KERNEL - 1, 0, -1))
    y = y + x * w[:, KERNEL - 1]
    y = y / (1 + torch.exp(-y))
    keys = c["groups"] * c["head_dim"]
    qk = y[:, :2 * keys].unflatten(1, (-1, c["head_dim"]))
    y[:, :2 * keys] = (qk / torch.sqrt((qk * qk).sum(2, keepdim=True) + EPS)).flatten(1)
    y[:, :keys] *= c["head_dim"] ** -0.5
    s["out"].copy_(y)
    counts = s["offsets"].diff()
    each, end = torch.arange(c["requests"], device="cuda"), s["offsets"][1:].to(torch.int64)
    window = [before(back, each, counts, end) for back in range(KERNEL - 1, 0, -1)]
    s["state"][s["slots"][:, 1].to(torch.int64)] = torch.stack(window, 2)
    return [s["out"], s["state"]]


def _coefficients(s):
    """Log decay and step size of every row and head."""
    if s["case"]["coef"] == "log":
        return s["alpha"], s["beta"]
    return torch.log1p(torch.exp(s["alpha"] + s["dt"])) * s["a"], 1 / (1 + torch.exp(-s["beta"]))


def _rows(s):
    """q, k and v of every row and head in float32 [rows][heads][head_dim]."""
    c = s["case"]
    x = s["x"].to(torch.float32).unflatten(1, (-1, c["head_dim"]))
    group = torch.arange(c["heads"], device="cuda") % c["groups"]
    return x[:, group], x[:, c["groups"] + group], x[:, 2 * c["groups"]:]


def _first_states(s):
    start = s["slots"][:, 0].to(torch.int64)
    return torch.where((start >= 0)[:, None, None, None], s["state"][start.clamp(min=0)], 0.0)


def _step(s):
    q, k, v = _rows(s)
    g, beta = _coefficients(s)
    state = _first_states(s) * torch.exp(g)[:, :, None, None]
    delta = (v - (state * k[:, :, :, None]).sum(2)) * beta[:, :, None]
    state = state + k[:, :, :, None] * delta[:, :, None]
    s["out"].copy_((state * q[:, :, :, None]).sum(2))
    s["state"][s["slots"][:, 1].to(torch.int64)] = state
    return [s["out"], s["state"]]


def _gdn(s):
    """By chunks of 64 rows: within one, the rows' corrections solve a triangular system; between them, the state."""
    c, C = s["case"], 64
    n, heads, d, rows = c["requests"], c["heads"], c["head_dim"], c["rows"]
    chunks = max(1, -(-max(_counts(c)) // C))
    request, i = _row_requests(s, rows)
    to = request * (chunks * C) + i

    def padded(x):  # [requests][heads][chunks][C][...]
        full = x.new_zeros(n * chunks * C, *x.shape[1:])
        full[to] = x
        return full.unflatten(0, (n, chunks, C)).movedim(3, 1).contiguous()

    q, k, v = (padded(x) for x in _rows(s))
    g, beta = (padded(x) for x in _coefficients(s))
    fall = g.to(torch.float64).cumsum(3)  # small differences of long sums
    low = torch.ones(C, C, device="cuda", dtype=torch.bool).tril()
    between = torch.where(low, fall[..., :, None] - fall[..., None, :], -math.inf).exp().to(torch.float32)
    since, until = fall.exp().to(torch.float32), (fall[..., -1:] - fall).exp().to(torch.float32)
    kt = k.transpose(3, 4).contiguous()
    solve = -(torch.matmul(k, kt) * between * beta[..., None]).tril(-1)
    for r in range(2, C):
        solve[..., r, :r] += (solve[..., r, :r, None] * solve[..., :r, :r]).sum(3)
    solve = solve + torch.eye(C, device="cuda")
    u = torch.matmul(solve, v * beta[..., None])
    w = torch.matmul(solve, k * (beta * since)[..., None])
    scores = torch.matmul(q, kt) * between
    q = q * since[..., None]
    kt = kt * until[..., None, :]
    state = _first_states(s)
    out = torch.empty_like(v)
    for t in range(chunks):
        new = u[:, :, t] - torch.matmul(w[:, :, t], state)
        out[:, :, t] = torch.matmul(q[:, :, t], state) + torch.matmul(scores[:, :, t], new)
        state = state * since[:, :, t, -1, None, None] + torch.matmul(kt[:, :, t], new)
    s["out"].copy_(out.movedim(1, 3).flatten(0, 2)[to])
    s["state"][s["slots"][:, 1].to(torch.int64)] = state
    return [s["out"], s["state"]]


# -------------------------------------------------------------------- exact

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "plan":
        return None
    if c["kind"] == "append":
        k = s["k"].to(torch.float64).reshape(c["rows"], -1, c["head_dim"])
        if c["norm"]:
            k = k * torch.rsqrt(k.square().mean(2, keepdim=True) + EPS) * s["k_norm"].to(torch.float64)
        outs, there = [], s["slots"] >= 0
        for pool, x in ((s["kpool"], k.reshape(c["rows"], -1)), (s["vpool"], s["v"].to(torch.float64))):
            full = pool.to(torch.float64).reshape(-1, pool.shape[2])
            full[s["slots"][there]] = x[there]
            outs.append(full.reshape(pool.shape))
        return outs
    states = s["state"].to(torch.float64)
    ends = s["offsets"].tolist()
    x = s["x"].to(torch.float64)
    if c["kind"] == "conv":
        keys, out = c["groups"] * c["head_dim"], torch.empty_like(x)
        w = s["weight"].to(torch.float64)
        new = states.clone()
        for j, (start, to) in enumerate(s["slots"].tolist()):
            past = states[start].t() if start >= 0 else x.new_zeros(KERNEL - 1, x.shape[1])
            line = torch.cat([past, x[ends[j]:ends[j + 1]]])
            out[ends[j]:ends[j + 1]] = (line.unfold(0, KERNEL, 1) * w).sum(2) if len(line) >= KERNEL else 0.0
            new[to] = line[len(line) - KERNEL + 1:].t()
        out = out * torch.sigmoid(out)
        qk = out[:, :2 * keys].reshape(len(out), -1, c["head_dim"])
        out[:, :2 * keys] = (qk * torch.rsqrt(qk.square().sum(2, keepdim=True) + EPS)).reshape(len(out), -1)
        out[:, :keys] *= 1 / math.sqrt(c["head_dim"])
        return [out, new]
    # token by token, the requests side by side, the longest first
    G, H, d = c["groups"], c["heads"], c["head_dim"]
    alpha, beta = s["alpha"].to(torch.float64), s["beta"].to(torch.float64)
    if c["coef"] == "raw":
        alpha = torch.nn.functional.softplus(alpha + s["dt"].to(torch.float64)) * s["a"].to(torch.float64)
        beta = torch.sigmoid(beta)
    lengths = [ends[j + 1] - ends[j] for j in range(c["requests"])]
    order = sorted(range(c["requests"]), key=lambda j: -lengths[j])
    starts = s["slots"][:, 0].tolist()
    state = torch.stack([states[starts[j]] if starts[j] >= 0 else torch.zeros_like(states[0]) for j in order])
    first = torch.tensor([ends[j] for j in order], device="cuda")
    heads = torch.arange(H, device="cuda") % G
    x = x.reshape(len(x), -1, d)
    out = x.new_zeros(len(x), H, d)
    for t in range(max(lengths)):
        live = sum(length > t for length in lengths)
        at = first[:live] + t
        row = x[at]
        q, k, v = row[:, heads], row[:, G + heads], row[:, 2 * G:]
        state[:live] *= torch.exp(alpha[at])[:, :, None, None]
        seen = torch.matmul(k[:, :, None], state[:live])[:, :, 0]
        state[:live] += k[:, :, :, None] * ((v - seen) * beta[at][:, :, None])[:, :, None]
        out[at] = torch.matmul(q[:, :, None], state[:live])[:, :, 0]
    states[s["slots"][:, 1].to(torch.int64)[order]] = state
    return [out, states]

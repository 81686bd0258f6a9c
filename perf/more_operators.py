"""The operators of a decoder layer served in 8 bits, as measured cases: the residual's addition with the
root-mean-square norm and codes of 8 bits, rows to codes of 8 bits, the product of such codes, and the rotation of
queries and keys on their way into the paged cache.

Codes: a row x has the scale s = max|x| / 127 and the codes rint(127 x / max|x|), halves to even, as exact arithmetic
gives them; a row of zeros (or of nothing above 127 * 2^-126) has s = 0 and codes 0.  It stands for the values code * s.

  norm     h = x + delta, y = h / sqrt(mean(h^2) + eps) * w, then the codes and the scale of every row of y; h is
           written too, as the next residual.  The norm cancels in the codes: they are those of g = h w.  h and g are
           fp32 numbers by definition, as the residual stream is.
  quant    the codes and the scale of every row of a matrix.
  linear   out[t, f] = s_x[t] s_w[f] sum_j w[f, j] x[t, j], then STORE (+ bias), RESID (+ a residual) or SWIGLU
           (rows of w interleaved, 16 gate and 16 up: up * gate / (1 + exp(-gate))).
  append   rows of new tokens (q, k, v side by side or apart): norms of q and k (none, over the whole vector, per
           head), rotation by their position (split halves), queries out, keys and values into their pages.
           Row i of a sequence's n new rows is at position kv_len - n + i.

Cache layout (one layer): [page][kv_head][page_size][head_dim]; page_table[slot][i] is the page that holds
positions [i * page_size, (i + 1) * page_size) of a slot, -1 where it has none.
"""
import math
import random

import torch

own = False
DEV = "cuda"
ROPE_THETA = 1e6
EPS = 1e-6
TINY = 127 * 2.0 ** -126  # rows whose largest magnitude is below this count as zero


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def _norm(rows, dim, x="f32", delta="f32", idle=0):
    """`rows` rows of the residual stream (x: its type; delta: the type of what is added, or "none"); the last `idle`
    rows are unused places of a batch and hold zeros."""
    return dict(op="norm", rows=rows, dim=dim, x=x, delta=delta, idle=idle)


def _quant(rows, dim, x="bf16", idle=0):
    return dict(op="quant", rows=rows, dim=dim, x=x, idle=idle)


def _linear(t, n_out, k, epi, out="f32", bias=False):
    """epi: store, resid (fp32) or swiglu (bf16)."""
    return dict(op="linear", t=t, n_out=n_out, k=k, epi=epi, out=out, bias=bias)


def _append(batch, chunks, new, ctx, heads, kv_heads, qk_norm, head_dim=128, page=64, x="f32", fp32=False, fused=True,
            idle=0, mix=1):
    """`chunks` of the batch's sequences bring new[0]..new[1] new tokens, the others one, onto ctx[0]..ctx[1] cached
    positions; the last `idle` sequences are unused places of the batch (one row, nothing cached)."""
    return dict(op="append", batch=batch, chunks=chunks, new_lo=new[0], new_hi=new[1], ctx_lo=ctx[0], ctx_hi=ctx[1],
                heads=heads, kv_heads=kv_heads, qk_norm=qk_norm, head_dim=head_dim, page=page, x=x, fp32=fp32,
                fused=fused, idle=idle, mix=mix)


def listed():
    return [
        # one user's next token through a small model (0.6B width): launch latency
        dict(_norm(1, 1024), name="norm-one-token"),
        # one step of a large batch at the 8B width, four places of it unused; the projection left bf16 sums
        dict(_norm(64, 4096, "f32", "bf16", idle=4), name="norm-decode-64"),
        # the prompts of a batch at the 8B width: the memory's bandwidth
        dict(_norm(8192, 4096), name="norm-prefill"),
        # the SwiGLU products of a decode step at the 8B width
        dict(_quant(64, 12288, idle=4), name="quant-decode-64"),
        # the same of a batch of prompts
        dict(_quant(8192, 12288), name="quant-prefill"),
        # the fused q, k and v projection of one token at the 8B width: the weights' bandwidth
        dict(_linear(1, 6144, 4096, "store"), name="linear-one-token"),
        # the down projection of a decode step of 64 sequences, added to the residual
        dict(_linear(64, 4096, 12288, "resid"), name="linear-decode-64"),
        # ragged turns through a model of width 896 (14 / 2 heads of 64) with biases, to bf16
        dict(_linear(333, 1152, 896, "store", "bf16", True), name="linear-turns"),
        # gate and up of a batch of prompts at the 8B width: the largest
        dict(_linear(8192, 24576, 4096, "swiglu", "bf16"), name="linear-prefill"),
        # one token onto a short prompt (16 / 8 heads): launch latency
        dict(_append(1, 0, (1, 1), (300, 300), 16, 8, "head"), name="append-one-token"),
        # a decode step of 64 sequences at the 8B geometry, norms over whole vectors, three places unused
        dict(_append(64, 0, (1, 1), (100, 700), 32, 8, "vector", idle=3, mix=2), name="append-decode-64"),
        # eight ragged prompts at the 8B geometry
        dict(_append(8, 8, (1400, 2048), (0, 0), 32, 8, "head", x="bf16", mix=3), name="append-prefill"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["norm", "quant", "linear", "linear", "append"])
    wide = rng.choice([896, 1024, 1536, 2048, 3584, 4096, 5120, 8192, _log(rng, 33, 16384), _log(rng, 33, 16384)])
    if op == "norm":
        rows = _log(rng, 1, 16384)
        x, delta = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "none"),
                               ("bf16", "none")])
        return _norm(rows, wide, x, delta, rng.randint(0, rows // 4))
    if op == "quant":
        rows = _log(rng, 1, 16384)
        return _quant(rows, rng.choice([4864, 6144, 12288, wide]), rng.choice(["bf16", "bf16", "f32"]),
                      rng.randint(0, rows // 4))
    if op == "linear":
        epi, out = rng.choice([("store", "f32"), ("store", "bf16"), ("resid", "f32"), ("swiglu", "bf16")])
        n_out = rng.choice([1152, 4096, 6144, 9728, 24576, _log(rng, 40, 25600), _log(rng, 40, 25600)])
        return _linear(_log(rng, 1, 8192), max(32, n_out // 32 * 32) if epi == "swiglu" else n_out,
                       rng.choice([wide, 4864, 12288]), epi, out, epi == "store" and rng.random() < 0.5)
    heads, kv_heads, head_dim = rng.choice([(16, 8, 128), (32, 8, 128), (64, 8, 128), (8, 8, 128), (12, 2, 128),
                                            (28, 4, 128), (14, 2, 64), (16, 4, 64), (8, 1, 64)])
    kind = rng.choice(["step", "chunk", "mixed"])
    batch, new = _log(rng, 1, 64), _log(rng, 2, 2048)
    hi = _log(rng, 40, 8192)
    chunks = 0 if kind == "step" else batch if kind == "chunk" else max(1, batch // 8)
    return _append(batch, chunks, (1, 1) if kind == "step" else (max(1, new // 4), new), (hi // 2, hi), heads, kv_heads,
                   rng.choice(["none", "vector", "head"]), head_dim, rng.choice([16, 32, 64, 128, 256]),
                   rng.choice(["f32", "bf16"]), rng.random() < 0.25, rng.random() < 0.5, rng.randint(0, batch // 4),
                   rng.randrange(1 << 20))


def draw(rng):
    """A case of the listed ranges that moves and computes no more than the largest ones."""
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] > 1.65e12 or w["bytes"] > 1e9:
            continue
        if c["op"] == "append":
            new, kv = _lengths(c)
            if sum(new) > 16384 or sum(kv) > 65536:
                continue
        return c


# ---------------------------------------------------------------------------------------------------------------
# lengths: a property of the case, the same for every seed
# ---------------------------------------------------------------------------------------------------------------
def _lengths(c):
    """(new rows, cache length with them) of every sequence of an append case."""
    r = random.Random(c["mix"])
    new, kv = [], []
    for b in range(c["batch"]):
        idle = b >= c["batch"] - c["idle"] and b >= c["chunks"]
        n = r.randint(c["new_lo"], c["new_hi"]) if b < c["chunks"] else 1
        p = r.randint(c["ctx_lo"], c["ctx_hi"])
        new.append(n)
        kv.append(0 if idle else p + n)
    return new, kv


def _size(t):
    return {"f32": 4, "bf16": 2, "none": 0}[t]


def work(case):
    c = case
    if c["op"] == "norm":
        cells = c["rows"] * c["dim"]
        return {"bytes": cells * (2 * _size(c["x"]) + _size(c["delta"]) + 1) + 4 * c["dim"] + 4 * c["rows"],
                "flops": 6 * cells}
    if c["op"] == "quant":
        cells = c["rows"] * c["dim"]
        return {"bytes": cells * (_size(c["x"]) + 1) + 4 * c["rows"], "flops": 2 * cells}
    if c["op"] == "linear":
        t, n, k = c["t"], c["n_out"], c["k"]
        out = t * n // 2 * 2 if c["epi"] == "swiglu" else t * n * _size(c["out"]) * (2 if c["epi"] == "resid" else 1)
        return {"bytes": n * k + t * k + 4 * (n + t) + (4 * n if c["bias"] else 0) + out, "flops": 2 * t * n * k}
    new, kv = _lengths(c)
    live = sum(min(n, m) for n, m in zip(new, kv))
    d, rows, esz = c["head_dim"], sum(new), 4 if c["fp32"] else 2
    width = (c["heads"] + 2 * c["kv_heads"]) * d
    return {"bytes": rows * width * _size(c["x"]) + (rows * c["heads"] + 2 * live * c["kv_heads"]) * d * esz + live * 4 * d,
            "flops": 6 * rows * width}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
class State:
    pass


def _type(t):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[t]


def _native_type(t):
    from common_b200 import native
    return {"f32": native.DTYPE_F32, "bf16": native.DTYPE_BF16}[t]


def _stream(rows, dim, g):
    """Rows of a residual stream: every channel has a size of its own, some are far larger than the rest."""
    gain = torch.randn(dim, device=DEV, generator=g).mul_(0.7).exp_()
    return torch.randn((rows, dim), device=DEV, generator=g).mul_(gain)


def _codes_for(values, ld, g):
    """(codes, scale) of a weight matrix or of activations that a program has in 8 bits, rows `ld` codes apart."""
    top = values.abs().amax(1)
    # behind the rows: anything
    codes = torch.randint(-127, 128, (values.shape[0], ld), device=DEV, dtype=torch.int8, generator=g)
    codes[:, : values.shape[1]] = (values * (127.0 / top)[:, None]).round_().to(torch.int8)
    return codes, top / 127.0


def _prepare_norm(c, g):
    s = State()
    rows, dim = c["rows"], c["dim"]
    live = torch.arange(rows, device=DEV) < rows - c["idle"]
    s.x = (_stream(rows, dim, g) * live[:, None]).to(_type(c["x"]))
    s.delta = None
    if c["delta"] != "none":
        s.delta = (torch.randn((rows, dim), device=DEV, generator=g) * 0.5 * live[:, None]).to(_type(c["delta"]))
    s.w = 1.0 + 0.2 * torch.randn(dim, device=DEV, generator=g)
    s.sum = torch.empty_like(s.x)
    s.ld = -(-dim // 16) * 16
    s.q = torch.empty((rows, s.ld), dtype=torch.int8, device=DEV)
    s.scale = torch.empty(rows, device=DEV)
    if own:
        from common_b200 import native
        s.norm = native.NormQ8(dim, s.w.data_ptr(), EPS, x_dtype=_native_type(c["x"]),
                               delta_dtype=_native_type(c["delta"] if s.delta is not None else "f32"))
    return s


def _prepare_quant(c, g):
    s = State()
    rows, dim = c["rows"], c["dim"]
    live = torch.arange(rows, device=DEV) < rows - c["idle"]
    # products of an activation: many near zero, a few large
    x = _stream(rows, dim, g)
    s.x = (x * torch.sigmoid(2 * x) * live[:, None]).to(_type(c["x"]))
    s.ld = -(-dim // 16) * 16
    s.q = torch.empty((rows, s.ld), dtype=torch.int8, device=DEV)
    s.scale = torch.empty(rows, device=DEV)
    return s


def _prepare_linear(c, g):
    s = State()
    t, n, k = c["t"], c["n_out"], c["k"]
    ld = -(-k // 16) * 16
    # weights whose sums have about the size of one
    s.w, s.w_scale = _codes_for(torch.randn((n, k), device=DEV, generator=g).mul_(1.0 / math.sqrt(k)), ld, g)
    s.x, s.x_scale = _codes_for(_stream(t, k, g), ld, g)
    s.bias = torch.randn(n, device=DEV, generator=g) if c["bias"] else None
    s.resid = torch.randn((t, n), device=DEV, generator=g) if c["epi"] == "resid" else None
    s.out = torch.empty((t, n // 2 if c["epi"] == "swiglu" else n), device=DEV, dtype=_type(c["out"]))
    s.ld = ld
    if own:
        from common_b200 import native
        epi = {"store": native.LINEAR_STORE, "resid": native.LINEAR_RESID, "swiglu": native.LINEAR_SWIGLU}[c["epi"]]
        s.linear = native.LinearQ8(s.w.data_ptr(), s.w_scale.data_ptr(), n, k, ld_w=ld, epi=epi,
                                   bias=s.bias.data_ptr() if c["bias"] else 0, out_dtype=_native_type(c["out"]))
    return s


def _prepare_append(c, g):
    s = State()
    page, H, Hkv, d = c["page"], c["heads"], c["kv_heads"], c["head_dim"]
    new, kv = _lengths(c)
    batch = c["batch"]
    need = [-(-m // page) for m in kv]
    s.num_pages = sum(need) + 3
    s.max_pages = max(need + [1])
    order = torch.randperm(s.num_pages, device=DEV, generator=g).to(torch.int32)
    s.table = torch.full((batch, s.max_pages), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b in range(batch):
        s.table[b, : need[b]] = order[at : at + need[b]]
        at += need[b]
    dt = torch.float32 if c["fp32"] else torch.bfloat16
    shape = (s.num_pages, Hkv, page, d)
    s.k_cache = torch.randn(shape, device=DEV, dtype=dt, generator=g)
    s.v_cache = torch.randn(shape, device=DEV, dtype=dt, generator=g)
    s.row_start = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    s.kv_len = torch.tensor(kv, dtype=torch.int32, device=DEV)
    s.rows, s.max_new = sum(new), max(new)
    if c["fused"]:  # as the fused projection leaves them
        qkv = torch.randn((s.rows, (H + 2 * Hkv) * d), device=DEV, generator=g).mul_(1.5).to(_type(c["x"]))
        s.q, s.k, s.v = qkv.split([H * d, Hkv * d, Hkv * d], 1)
    else:
        s.q, s.k, s.v = (torch.randn((s.rows, h * d), device=DEV, generator=g).mul_(1.5).to(_type(c["x"]))
                         for h in (H, Hkv, Hkv))
    s.q_norm = s.k_norm = None
    if c["qk_norm"] != "none":
        wide = c["qk_norm"] == "vector"
        s.q_norm = 1.0 + 0.2 * torch.randn(H * d if wide else d, device=DEV, generator=g)
        s.k_norm = 1.0 + 0.2 * torch.randn(Hkv * d if wide else d, device=DEV, generator=g)
    s.rope_len = max(kv + [1])
    angle = torch.arange(s.rope_len, dtype=torch.float64, device=DEV)[:, None] * \
        ROPE_THETA ** (-torch.arange(d // 2, dtype=torch.float64, device=DEV) * 2 / d)
    s.rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    s.q_out = torch.empty((s.rows, H, d), device=DEV, dtype=dt)
    if own:
        from common_b200 import native
        s.append = native.KvAppend(
            H, Hkv, d, page, s.num_pages, s.max_pages, rope=s.rope.data_ptr(), rope_len=s.rope_len,
            qk_norm={"none": native.QKNORM_NONE, "vector": native.QKNORM_VECTOR, "head": native.QKNORM_HEAD}[c["qk_norm"]],
            q_norm=s.q_norm.data_ptr() if s.q_norm is not None else 0,
            k_norm=s.k_norm.data_ptr() if s.k_norm is not None else 0, eps=EPS, in_dtype=_native_type(c["x"]),
            dtype=_native_type("f32" if c["fp32"] else "bf16"))
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"norm": _prepare_norm, "quant": _prepare_quant, "linear": _prepare_linear,
         "append": _prepare_append}[case["op"]](case, g)
    s.c = case
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _as_codes(y):
    """(codes as fp32, max|y|) of every row of y in fp32; next to a half of a code only 64 bits tell the sides apart."""
    top = y.abs().amax(1, keepdim=True)
    top = torch.where(top < TINY, 0.0, top)
    return torch.where(top > 0, y.double().mul_(127.0).div_(top).round_(), 0.0).float(), top


def _plain_norm(s):
    h = s.x.float()
    if s.delta is not None:
        h = h + s.delta.float()
    s.sum.copy_(h)
    rms = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    codes, top = _as_codes(h * s.w)
    scale = top * rms / 127.0
    return {"sum": s.sum, "values": codes * scale, "scale": scale.squeeze(1)}


def _plain_quant(s):
    codes, top = _as_codes(s.x.float())
    scale = top / 127.0
    return {"values": codes * scale, "scale": scale.squeeze(1)}


def _plain_linear(s):
    c = s.c
    y = s.x[:, : c["k"]].float() @ s.w[:, : c["k"]].float().T
    y = y * s.w_scale * s.x_scale[:, None]
    if c["epi"] == "swiglu":
        gate, up = y.view(c["t"], -1, 2, 16).unbind(2)
        y = (up * (gate / (1.0 + torch.exp(-gate)))).reshape(c["t"], -1)
    elif c["epi"] == "resid":
        y = s.resid + y
    elif c["bias"]:
        y = y + s.bias
    s.out.copy_(y)
    return s.out


def _plain_append(s):
    c = s.c
    H, Hkv, d, page, half = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["head_dim"] // 2
    r = torch.arange(s.rows, device=DEV)
    b = torch.searchsorted(s.row_start[1:].long().contiguous(), r, right=True)
    pos = s.kv_len.long()[b] - s.row_start.long()[b + 1] + r
    live = pos >= 0
    cos, sin = s.rope[pos.clamp(min=0)].unsqueeze(1).unbind(-1)

    def turned(x, heads, w):
        x = x.float()
        if c["qk_norm"] == "vector":
            x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * w
        x = x.view(-1, heads, d)
        if c["qk_norm"] == "head":
            x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS) * w
        lo, hi = x[..., :half], x[..., half:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    s.q_out.copy_(torch.where(live[:, None, None], turned(s.q, H, s.q_norm), 0.0))
    p = pos[live]
    pg, row = s.table.long()[b[live], p // page], p % page
    s.k_cache[pg, :, row] = turned(s.k, Hkv, s.k_norm)[live].to(s.k_cache.dtype)
    s.v_cache[pg, :, row] = s.v.reshape(-1, Hkv, d)[live].to(s.v_cache.dtype)
    return {"q": s.q_out, "k_cache": s.k_cache, "v_cache": s.v_cache}


def run(state):
    s = state
    c = s.c
    if not own:
        return {"norm": _plain_norm, "quant": _plain_quant, "linear": _plain_linear, "append": _plain_append}[c["op"]](s)
    from common_b200 import native
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "norm":
        s.norm(s.x.data_ptr(), s.q.data_ptr(), s.scale.data_ptr(), c["rows"],
               delta=s.delta.data_ptr() if s.delta is not None else 0, sum_out=s.sum.data_ptr(), ld_q=s.ld, stream=stream)
        # what the codes stand for, for a reader of the outputs
        return {"sum": s.sum, "values": s.q[:, : c["dim"]] * s.scale[:, None], "scale": s.scale}
    if c["op"] == "quant":
        native.op_quant_q8(s.x.data_ptr(), _native_type(c["x"]), c["rows"], c["dim"], s.q.data_ptr(), s.scale.data_ptr(),
                           ld_q=s.ld, stream=stream)
        return {"values": s.q[:, : c["dim"]] * s.scale[:, None], "scale": s.scale}
    if c["op"] == "linear":
        s.linear(s.x.data_ptr(), s.x_scale.data_ptr(), c["t"], s.out.data_ptr(),
                 resid=s.resid.data_ptr() if s.resid is not None else 0, ld_x=s.ld, stream=stream)
        return s.out
    s.append(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.q_out.data_ptr(), s.k_cache.data_ptr(),
             s.v_cache.data_ptr(), s.table.data_ptr(), s.row_start.data_ptr(), s.kv_len.data_ptr(), c["batch"], s.rows,
             ld_q=s.q.stride(0), ld_k=s.k.stride(0), ld_v=s.v.stride(0), stream=stream)
    return {"q": s.q_out, "k_cache": s.k_cache, "v_cache": s.v_cache}


# ---------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_steps(y):
    """(codes, largest magnitude) of y's rows: 254 |y| against the odd multiples of the largest magnitude, all whole in
    64 bits, so that halves are halves."""
    top = torch.linalg.vector_norm(y, math.inf, 1)[:, None]
    twice = 254 * y.abs()
    low = torch.nan_to_num(torch.floor(twice / (2 * top)))
    low = low - (twice < 2 * low * top).double() + (twice >= 2 * (low + 1) * top).double() * (top > 0)
    half = (2 * low + 1) * top
    up = (twice > half) | ((twice == half) & (low % 2 == 1) & (top > 0))
    return (low + up.double()) * torch.sign(y), top.squeeze(1)


def _exact_norm(s):
    h = s.x.double() if s.delta is None else s.x.double() + s.delta.double()
    held = h.float().double()
    length = torch.linalg.vector_norm(held, 2, 1)
    codes, top = _exact_steps((held * s.w.double()).float().double())
    scale = top / 127 / torch.sqrt(length * length / h.shape[1] + EPS)
    return {"sum": h, "values": codes * scale[:, None], "scale": scale}


def _exact_quant(s):
    codes, top = _exact_steps(s.x.double())
    return {"values": codes * (top / 127)[:, None], "scale": top / 127}


def _exact_linear(s):
    c = s.c
    w = s.w[:, : c["k"]].double() * s.w_scale.double()[:, None]
    out = torch.empty(s.out.shape, dtype=torch.float64, device=DEV)
    for a in range(0, c["t"], 1024):
        e = min(a + 1024, c["t"])
        y = torch.einsum("tk,fk->tf", s.x[a:e, : c["k"]].double() * s.x_scale[a:e].double()[:, None], w)
        if c["epi"] == "swiglu":
            f = torch.arange(c["n_out"], device=DEV)
            gate, up = y[:, f % 32 < 16], y[:, f % 32 >= 16]
            out[a:e] = up * gate * torch.sigmoid(gate)
        else:
            out[a:e] = y + (s.bias.double() if c["bias"] else s.resid[a:e].double() if c["epi"] == "resid" else 0.0)
    return out


def _exact_append(s):
    c = s.c
    H, Hkv, d, page, half = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["head_dim"] // 2
    new, kv = _lengths(c)
    k_cache, v_cache = s.k_cache.double(), s.v_cache.double()
    q_out = torch.zeros((s.rows, H, d), dtype=torch.float64, device=DEV)
    turn = torch.view_as_complex(s.rope.double())
    at = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        if m >= n:
            p = torch.arange(m - n, m, device=DEV)
            z = turn[p][:, None, :]

            def rotated(x, heads, w):
                x = x[at : at + n].double().reshape(n, heads, d)
                if c["qk_norm"] != "none":
                    axes = (1, 2) if c["qk_norm"] == "vector" else (2,)
                    x = x / torch.sqrt((x * x).mean(axes, keepdim=True) + EPS)
                    x = x * (w.double().view(heads, d) if c["qk_norm"] == "vector" else w.double())
                y = torch.complex(x[..., :half], x[..., half:]) * z
                return torch.cat([y.real, y.imag], -1)

            pages = s.table[b].long()[p // page]
            q_out[at : at + n] = rotated(s.q, H, s.q_norm)
            k_cache[pages, :, p % page] = rotated(s.k, Hkv, s.k_norm)
            v_cache[pages, :, p % page] = s.v[at : at + n].double().reshape(n, Hkv, d)
        at += n
    return {"q": q_out, "k_cache": k_cache, "v_cache": v_cache}


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    return {"norm": _exact_norm, "quant": _exact_quant, "linear": _exact_linear, "append": _exact_append}[case["op"]](s)

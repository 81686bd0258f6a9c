"""The operators of a shared paged KV cache, as measured cases: attention of ragged chunks of new tokens over the
cache, copying (forking) its pages, and compacting sequences within it.

Cache layout (one layer): [page][kv_head][page_size][head_dim]; page_table[slot][i] is the page that holds
positions [i * page_size, (i + 1) * page_size) of a slot, -1 where it has none.

  attn     out[r] = sum_j softmax_j(q[r] . k[j] / sqrt(d)) v[j] for every row r of a batch of sequences with
           different numbers of new tokens and of cached positions; row i of a sequence's n new rows is at position
           p = kv_len - n + i and sees positions max(0, p - window + 1) .. p (window 0: all up to p).  Also the
           natural log of the softmax sum (lse).  A row that sees nothing gives zeros and -inf.
  copy     rows [0, rows[i]) of page src[i] -> page dst[i], every KV head of every layer, keys and values.
  compact  position i of sequence b's new pages <- its cached position keep[keep_start[b] + i]; keys are turned back
           by the rotary angle of the distance they move (split-half pairs, cos / sin table).
"""
import math
import random

import torch

own = False
DEV = "cuda"
ROPE_THETA = 1e6


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def _attn(batch, chunks, new, ctx, heads, kv_heads, head_dim=128, page=64, window=0, idle=0, fused=False, mix=1):
    """`chunks` of the batch's sequences bring new[0]..new[1] new tokens, the others one; all stand on ctx[0]..ctx[1]
    cached positions; the last `idle` sequences are unused places of the batch (one row, nothing cached).  fused: the
    queries lie in rows that hold q, k and v side by side, as the fused projection leaves them."""
    return dict(op="attn", batch=batch, chunks=chunks, new_lo=new[0], new_hi=new[1], ctx_lo=ctx[0], ctx_hi=ctx[1],
                heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, window=window, idle=idle, fused=fused,
                mix=mix)


def _copy(parents, children, rows, layers, kv_heads, head_dim=128, page=64, fp32=False):
    """Each of `parents` pages goes to `children` new pages: its first `rows` rows."""
    return dict(op="copy", parents=parents, children=children, rows=rows, layers=layers, kv_heads=kv_heads,
                head_dim=head_dim, page=page, fp32=fp32)


def _compact(batch, ctx, keep, scattered, layers, kv_heads, head_dim=128, page=64, fp32=False, mix=1):
    """Sequences of ctx[0]..ctx[1] positions keep the share `keep`: all but one gap in the middle, or scattered ones."""
    return dict(op="compact", batch=batch, ctx_lo=ctx[0], ctx_hi=ctx[1], keep=keep, scattered=scattered, layers=layers,
                kv_heads=kv_heads, head_dim=head_dim, page=page, fp32=fp32, mix=mix)


def listed():
    return [
        # one user's next token after a short prompt (0.6B / 1.7B geometry): launch latency
        dict(_attn(1, 0, (1, 1), (300, 300), 16, 8), name="attn-one-token"),
        # one step of a large batch at the 8B geometry and 4096-token contexts: the cache's bandwidth
        dict(_attn(64, 0, (1, 1), (3900, 4250), 32, 8, fused=True), name="attn-decode-64"),
        # one token on one very long document: a single sequence over the whole GPU
        dict(_attn(1, 0, (1, 1), (120001, 120001), 32, 8), name="attn-long-one"),
        # the next turns of eight conversations: short ragged chunks on kept histories
        dict(_attn(8, 8, (17, 300), (2500, 7000), 32, 8, mix=2), name="attn-turns"),
        # serving mix: one new chunk rides with 32 running generations, three places of the batch unused
        dict(_attn(36, 1, (512, 512), (900, 3500), 32, 8, idle=3, fused=True, mix=3), name="attn-mixed"),
        # the prompts of a batch, nothing cached: the ordinary prefill, ragged
        dict(_attn(8, 8, (1400, 2048), (0, 0), 32, 8, mix=4), name="attn-prefill"),
        # a further chunk of a long prompt: the largest
        dict(_attn(1, 1, (4096, 4096), (16000, 16000), 32, 8), name="attn-long-chunk"),
        # seven query heads per KV head at head size 64, small pages, a sliding window whose old pages are released
        dict(_attn(6, 6, (100, 700), (1000, 4000), 14, 2, 64, 16, 1024, mix=5), name="attn-window-64"),
        # forking four ways from one prompt: the last, partly filled page of the 0.6B cache
        dict(_copy(1, 4, 37, 28, 8), name="copy-fork"),
        # duplicating the caches of a few sequences at the 8B geometry
        dict(_copy(160, 1, 64, 36, 8), name="copy-pages"),
        # dropping an old turn from the middle of one conversation
        dict(_compact(1, (2100, 2100), 0.7, False, 28, 8), name="compact-gap"),
        # evicting scattered tokens from long sequences
        dict(_compact(4, (6500, 8192), 0.6, True, 28, 8, mix=2), name="compact-evict"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    heads, kv_heads, head_dim = rng.choice([(16, 8, 128), (32, 8, 128), (64, 8, 128), (8, 8, 128), (12, 2, 128),
                                            (28, 4, 128), (14, 2, 64), (16, 4, 64), (8, 1, 64)])
    page = rng.choice([16, 32, 64, 128, 256])
    kind = rng.choice(["step", "chunk", "mixed", "copy", "compact"])
    mix = rng.randrange(1 << 20)
    if kind == "copy":
        return _copy(_log(rng, 1, 160), _log(rng, 1, 8), rng.randint(1, page), _log(rng, 1, 36), kv_heads, head_dim,
                     page, rng.random() < 0.25)
    if kind == "compact":
        hi = _log(rng, 30, 8192)
        return _compact(_log(rng, 1, 8), (max(1, hi // 2), hi), round(rng.uniform(0.2, 0.95), 2), rng.random() < 0.5,
                        _log(rng, 1, 36), kv_heads, head_dim, page, rng.random() < 0.25, mix)
    batch = _log(rng, 1, 64)
    hi = _log(rng, 40, 120000 if kind == "step" else 16000)
    new = _log(rng, 2, 4096)
    window = rng.choice([0, 0, 0, 128, _log(rng, 50, 5000)])
    chunks = 0 if kind == "step" else batch if kind == "chunk" else max(1, batch // 8)
    return _attn(batch, chunks, (1, 1) if kind == "step" else (max(1, new // 4), new), (hi // 2, hi), heads, kv_heads,
                 head_dim, page, window, rng.randint(0, batch // 4), rng.random() < 0.5, mix)


def draw(rng):
    """A case of the listed ranges whose work and whose plain form's score matrix are no larger than the largest's."""
    while True:
        c = _draw(rng)
        w = work(c)
        if c["op"] == "attn":
            new = c["new_hi"] if c["chunks"] else 1
            scores = c["batch"] * c["heads"] * new * (c["ctx_hi"] + new)
            cells = c["batch"] * c["kv_heads"] * c["head_dim"] * (c["ctx_hi"] + new)
            if scores > 2.5e9 or cells > 6e8 or w["flops"] > 1.2e12:
                continue
        if w["bytes"] <= 3e9:
            return c


# ---------------------------------------------------------------------------------------------------------------
# lengths: a property of the case, the same for every seed
# ---------------------------------------------------------------------------------------------------------------
def _lengths(c):
    """(new rows, cache length with them) of every sequence of an attention case."""
    r = random.Random(c["mix"])
    new, kv = [], []
    for b in range(c["batch"]):
        idle = b >= c["batch"] - c["idle"] and b >= c["chunks"]
        n = r.randint(c["new_lo"], c["new_hi"]) if b < c["chunks"] else 1
        p = r.randint(c["ctx_lo"], c["ctx_hi"])
        new.append(n)
        kv.append(0 if idle else p + n)
    return new, kv


def _contexts(c):
    r = random.Random(c["mix"])
    ctx = [r.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["batch"])]
    return ctx, [max(1, int(n * c["keep"])) for n in ctx]


def _first_seen(c, n, kv):
    """The first position that any of a sequence's new rows sees."""
    return max(0, kv - n - c["window"] + 1) if c["window"] else 0


def work(case):
    c = case
    esz = 4 if c.get("fp32") else 2
    if c["op"] == "copy":
        cell = c["layers"] * 2 * c["kv_heads"] * c["head_dim"] * esz
        return {"bytes": cell * c["rows"] * c["parents"] * (1 + c["children"]) + 12 * c["parents"] * c["children"],
                "flops": 0}
    if c["op"] == "compact":
        cell = c["layers"] * 2 * c["kv_heads"] * c["head_dim"]
        rows = sum(_contexts(c)[1])
        return {"bytes": rows * (2 * cell * esz + 4), "flops": rows * cell // 2 * 3}
    new, kv = _lengths(c)
    pairs = seen = 0
    for n, k in zip(new, kv):
        lo = _first_seen(c, n, k)
        seen += max(0, k - lo)
        a, b = max(0, k - n), k  # positions of the rows that see something
        w = c["window"] or (1 << 40)
        full = max(0, min(b, w) - min(a, w))  # rows whose window is not yet full: p + 1 positions each
        pairs += (min(a, w) + 1 + min(a, w) + full) * full // 2 + (b - a - full) * w
    d, rows = c["head_dim"], sum(new)
    return {"bytes": 2 * seen * c["kv_heads"] * d * 2 + rows * c["heads"] * (4 * d + 4) + 4 * (seen // c["page"] + 1),
            "flops": 4 * d * c["heads"] * pairs}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
class State:
    pass


def _rows_of(table, start, length, page):
    """(page, row in page) of positions start .. start + length - 1 of one sequence."""
    p = torch.arange(start, start + length, device=DEV)
    return table[p // page], p % page


def _prepare_attn(c, g):
    s = State()
    page, H, Hkv, d = c["page"], c["heads"], c["kv_heads"], c["head_dim"]
    new, kv = _lengths(c)
    batch = c["batch"]
    need = [-(-k // page) for k in kv]
    s.num_pages = sum(need) + 8
    s.max_pages = max(need + [1])
    # pages lie in the order in which a long-running pool hands them out: none
    order = torch.randperm(s.num_pages, device=DEV, generator=g).to(torch.int32)
    table = torch.full((batch, s.max_pages), -1, dtype=torch.int32, device=DEV)
    shape = (s.num_pages, Hkv, page, d)
    s.k = torch.randn(shape, device=DEV, dtype=torch.bfloat16, generator=g)
    s.v = torch.randn(shape, device=DEV, dtype=torch.bfloat16, generator=g)
    written = torch.zeros((s.num_pages, page), dtype=torch.bool, device=DEV)
    at = 0
    for b in range(batch):
        table[b, : need[b]] = order[at : at + need[b]]
        at += need[b]
        lo = _first_seen(c, new[b], kv[b])
        table[b, : lo // page] = -1  # pages that no row's window reaches have been released
        if kv[b] > lo:
            pg, row = _rows_of(table[b].long(), lo, kv[b] - lo, page)
            written[pg, row] = True
    # what no position of any sequence has written (or sees any more) holds what the last owner left there
    s.k.masked_fill_(~written[:, None, :, None], float("nan"))
    s.v.masked_fill_(~written[:, None, :, None], float("nan"))
    s.table = table
    s.row_start = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    s.kv_len = torch.tensor(kv, dtype=torch.int32, device=DEV)
    s.rows, s.max_new, s.max_kv = sum(new), max(new), max(max(kv), 1)
    # queries of normalised heads with a learned gain: scores q . k / sqrt(d) spread by about 1.5
    wide = (H + 2 * Hkv) * d if c["fused"] else H * d
    s.qkv = torch.randn((s.rows, wide), device=DEV, generator=g).mul_(1.5).to(torch.bfloat16)
    s.q = s.qkv[:, : H * d].view(s.rows, H, d)
    s.out = torch.empty((s.rows, H, d), device=DEV, dtype=torch.bfloat16)
    s.lse = torch.empty((s.rows, H), device=DEV, dtype=torch.float32)
    s.c = c
    if own:
        from common_b200 import native
        n = native.chunk_attn_workspace(H, Hkv, d)
        s.workspace = torch.zeros(n, dtype=torch.uint8, device=DEV)
        s.attn = native.ChunkAttention(H, Hkv, d, page, s.num_pages, s.max_pages, s.workspace.data_ptr(), n,
                                       window=c["window"])
    return s


def _pools(c, num_pages, g):
    shape = (c["layers"], num_pages, c["kv_heads"], c["page"], c["head_dim"])
    dt = torch.float32 if c["fp32"] else torch.bfloat16
    return torch.randn(shape, device=DEV, dtype=dt, generator=g), torch.randn(shape, device=DEV, dtype=dt, generator=g)


def _native_pool(s, c, num_pages):
    from common_b200 import native
    return native.KvPool(s.k.data_ptr(), s.v.data_ptr(), c["layers"], num_pages, c["kv_heads"], c["page"],
                         c["head_dim"], native.DTYPE_F32 if c["fp32"] else native.DTYPE_BF16)


def _prepare_copy(c, g):
    s = State()
    n = c["parents"] * c["children"]
    num_pages = c["parents"] + n + 3
    order = torch.randperm(num_pages, device=DEV, generator=g).to(torch.int32)
    s.src = order[: c["parents"]].repeat_interleave(c["children"]).contiguous()
    s.dst = order[c["parents"] : c["parents"] + n].contiguous()
    s.n_rows = torch.full((n,), c["rows"], dtype=torch.int32, device=DEV)
    s.k, s.v = _pools(c, num_pages, g)
    s.n, s.c = n, c
    if own:
        s.pool = _native_pool(s, c, num_pages)
    return s


def _prepare_compact(c, g):
    s = State()
    page, d = c["page"], c["head_dim"]
    ctx, kept = _contexts(c)
    old, new = [-(-n // page) for n in ctx], [-(-n // page) for n in kept]
    num_pages = sum(old) + sum(new)
    s.max_pages = max(old)
    order = torch.randperm(num_pages, device=DEV, generator=g).to(torch.int32)
    s.src_table = torch.full((c["batch"], s.max_pages), -1, dtype=torch.int32, device=DEV)
    s.dst_table = s.src_table.clone()
    keep, at = [], 0
    for b in range(c["batch"]):
        s.src_table[b, : old[b]] = order[at : at + old[b]]
        at += old[b]
        s.dst_table[b, : new[b]] = order[at : at + new[b]]
        at += new[b]
        if c["scattered"]:
            keep.append(torch.randperm(ctx[b], device=DEV, generator=g)[: kept[b]].sort().values)
        else:
            p = torch.arange(kept[b], device=DEV)
            cut = int(torch.randint(0, kept[b] + 1, (1,), device=DEV, generator=g))
            keep.append(torch.where(p < cut, p, p + ctx[b] - kept[b]))
    s.keep = torch.cat(keep).to(torch.int32)
    s.keep_start = torch.tensor([0] + kept, device=DEV).cumsum(0).to(torch.int32)
    s.rows = sum(kept)
    s.k, s.v = _pools(c, num_pages, g)
    s.rope_len = max(ctx)
    angle = torch.arange(s.rope_len, dtype=torch.float64, device=DEV)[:, None] * \
        ROPE_THETA ** (-torch.arange(d // 2, dtype=torch.float64, device=DEV) * 2 / d)
    s.rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    s.c = c
    if own:
        s.pool = _native_pool(s, c, num_pages)
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"attn": _prepare_attn, "copy": _prepare_copy, "compact": _prepare_compact}[case["op"]](case, g)


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _plain_attn(s):
    c = s.c
    B, N, L, page = c["batch"], s.max_new, s.max_kv, c["page"]
    H, Hkv, d = c["heads"], c["kv_heads"], c["head_dim"]
    n = (s.row_start[1:] - s.row_start[:-1]).long()
    row = s.row_start[:-1].long()[:, None] + torch.arange(N, device=DEV)
    mine = torch.arange(N, device=DEV) < n[:, None]
    pos = s.kv_len.long()[:, None] - n[:, None] + torch.arange(N, device=DEV)
    key = torch.arange(L, device=DEV)
    first = (s.kv_len.long() - n - c["window"] + 1 if c["window"] else torch.zeros_like(n))[:, None]
    held = (key < s.kv_len[:, None]) & (key >= first)
    pg = torch.where(held, s.table.long()[:, key // page], 0)
    k = torch.where(held[:, :, None, None], s.k[pg, :, key % page].float(), 0.0)  # (B, L, Hkv, d)
    v = torch.where(held[:, :, None, None], s.v[pg, :, key % page].float(), 0.0)
    q = s.q.float()[row.clamp(max=s.rows - 1)].view(B, N, Hkv, H // Hkv, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(B, Hkv, H // Hkv * N, d)
    x = q @ k.permute(0, 2, 3, 1) * (1.0 / math.sqrt(d))
    sees = key <= pos[:, :, None]
    if c["window"]:
        sees &= key > pos[:, :, None] - c["window"]
    x = x.view(B, Hkv, H // Hkv, N, L).masked_fill_(~sees[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(B, Hkv, -1, L) @ v.transpose(1, 2)).view(B, Hkv, H // Hkv, N, d) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    s.out.copy_(o.permute(0, 3, 1, 2, 4).reshape(B, N, H, d)[mine])
    s.lse.copy_(lse.permute(0, 3, 1, 2).reshape(B, N, H)[mine])
    return {"out": s.out, "lse": s.lse}


def _plain_copy(s):
    row = torch.arange(s.c["page"], device=DEV)
    pair, row = (row < s.n_rows[:, None]).nonzero(as_tuple=True)
    src, dst = s.src.long()[pair], s.dst.long()[pair]
    s.k[:, dst, :, row] = s.k[:, src, :, row]
    s.v[:, dst, :, row] = s.v[:, src, :, row]
    return {"k": s.k, "v": s.v}


def _plain_compact(s):
    c = s.c
    page, half = c["page"], c["head_dim"] // 2
    r = torch.arange(s.rows, device=DEV)
    b = torch.searchsorted(s.keep_start[1:].long().contiguous(), r, right=True)
    to, come = r - s.keep_start.long()[b], s.keep.long()
    src, dst = s.src_table.long()[b, come // page], s.dst_table.long()[b, to // page]
    k = s.k[:, src, :, come % page].float()  # (rows, layers, Hkv, d): the indices lie apart, so rows come first
    cos, sin = s.rope[come - to].unbind(-1)
    cos, sin = cos[:, None, None], sin[:, None, None]
    lo, hi = k[..., :half], k[..., half:]
    k = torch.cat([lo * cos + hi * sin, hi * cos - lo * sin], -1)
    s.k[:, dst, :, to % page] = k.to(s.k.dtype)
    s.v[:, dst, :, to % page] = s.v[:, src, :, come % page]
    return {"k": s.k, "v": s.v}


def run(state):
    s = state
    op = s.c["op"]
    if not own:
        return {"attn": _plain_attn, "copy": _plain_copy, "compact": _plain_compact}[op](s)
    from common_b200 import native
    stream = torch.cuda.current_stream().cuda_stream
    if op == "attn":
        s.attn(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.table.data_ptr(), s.row_start.data_ptr(),
               s.kv_len.data_ptr(), s.c["batch"], s.rows, s.out.data_ptr(), lse=s.lse.data_ptr(), ld_q=s.q.stride(0),
               stream=stream)
        return {"out": s.out, "lse": s.lse}
    if op == "copy":
        native.op_kv_copy_pages(s.pool, s.src.data_ptr(), s.dst.data_ptr(), s.n_rows.data_ptr(), s.n, stream)
    else:
        native.op_kv_compact(s.pool, s.src_table.data_ptr(), s.dst_table.data_ptr(), s.max_pages, s.keep.data_ptr(),
                             s.keep_start.data_ptr(), s.c["batch"], s.rows, rope=s.rope.data_ptr(),
                             rope_len=s.rope_len, stream=stream)
    return {"k": s.k, "v": s.v}


# ---------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits, sequence by sequence and head by head
# ---------------------------------------------------------------------------------------------------------------
def _exact_attn(s):
    c = s.c
    d, group = c["head_dim"], c["heads"] // c["kv_heads"]
    new, kv = _lengths(c)
    out = torch.zeros((s.rows, c["heads"], d), dtype=torch.float64, device=DEV)
    lse = torch.full((s.rows, c["heads"]), -math.inf, dtype=torch.float64, device=DEV)
    r0 = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        lo = _first_seen(c, n, m)
        skip = max(0, n - m)  # rows at positions before the first
        if m > lo and n > skip:
            pg, row = _rows_of(s.table[b].long(), lo, m - lo, c["page"])
            p = torch.arange(m - n + skip, m, device=DEV)[:, None]
            j = torch.arange(lo, m, device=DEV)[None, :]
            hidden = (j > p) | ((j <= p - c["window"]) if c["window"] else False)
            for h in range(c["heads"]):
                k, v = s.k[pg, h // group, row].double(), s.v[pg, h // group, row].double()
                x = s.q[r0 + skip : r0 + n, h].double() @ k.T / math.sqrt(d)
                x[hidden] = -math.inf
                lse[r0 + skip : r0 + n, h] = torch.logsumexp(x, 1)
                out[r0 + skip : r0 + n, h] = torch.softmax(x, 1) @ v
        r0 += n
    return {"out": out, "lse": lse}


def _exact_copy(s):
    k, v = s.k.double(), s.v.double()
    for a, b, n in zip(s.src.tolist(), s.dst.tolist(), s.n_rows.tolist()):
        k[:, b, :, :n] = k[:, a, :, :n]
        v[:, b, :, :n] = v[:, a, :, :n]
    return {"k": k, "v": v}


def _exact_compact(s):
    c = s.c
    page, half = c["page"], c["head_dim"] // 2
    k, v = s.k.double(), s.v.double()
    for b in range(c["batch"]):
        a, e = int(s.keep_start[b]), int(s.keep_start[b + 1])
        come, to = s.keep[a:e].long(), torch.arange(e - a, device=DEV)
        z = torch.view_as_complex(s.rope.double())[come - to].conj()  # turning back is the conjugate angle
        sp, dp = s.src_table[b].long()[come // page], s.dst_table[b].long()[to // page]
        for l in range(c["layers"]):
            x = k[l][sp, :, come % page]
            y = torch.complex(x[..., :half], x[..., half:]) * z[:, None, :]
            k[l][dp, :, to % page] = torch.cat([y.real, y.imag], -1)
            v[l][dp, :, to % page] = v[l][sp, :, come % page]
    return {"k": k, "v": v}


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    return {"attn": _exact_attn, "copy": _exact_copy, "compact": _exact_compact}[case["op"]](s)

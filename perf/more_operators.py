"""Cases, plain forms and 64-bit definitions of the operators around the 4-bit paged KV cache:

  append   new K and V rows (K rotated) into a paged cache of 4-bit codes with a (low, step) pair for each row and head
  attend   attention of the step's query rows over that cache: one-token decode, a few tokens at a time, ragged
           prompts, with optional tanh score cap, distance bias, document mask and prefix mask

With `own` False, `run` computes them from elementary torch operations in 32 bits (64 for the rotation's angles); with
`own` True it makes the framework's calls. Layouts: pools uint8 [n_pages, kv_heads, page, dim / 2], ranges fp16
[n_pages, kv_heads, page, 2] of (low, step), block table int32 [batch, max_pages]; row t of sequence b is row t % page of
page block_table[b, t // page]. A code c stands for low + step * c. Four bytes hold elements e0 .. e7 as the nibbles
e0 e2, e4 e6, e1 e3, e5 e7 (the lower one first).
"""
import math
import random

import numpy as np
import torch

own = False

THETA = 500000.0  # rotary base of the batched-decode and long-prompt configurations
TINY = 2.0 ** -24  # the least step


# --------------------------------------------------------------------------------------------- the cases

def _case(name, op, **kw):
    c = dict(op=op, batch=1, q_heads=32, kv_heads=8, dim=128, page=64, cached_lo=0, cached_hi=0, new_lo=1, new_hi=1,
             mix=1, io="f16", rope=0, cap=0.0, bias=False, prefix=False, docs=False)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the rows of one decode step of a full batch, rotated and stored
        _case("append decode", "append", batch=64, cached_lo=256, cached_hi=8192, rope=1, mix=3),
        # four prompt chunks of uneven length, half-split rotation
        _case("append prompts", "append", batch=4, cached_lo=0, cached_hi=3000, new_lo=900, new_hi=3100, rope=2, mix=7),
        # a small model in 32 bits on small pages, odd lengths
        _case("append f32", "append", batch=5, q_heads=32, kv_heads=4, dim=64, page=16, cached_lo=3, cached_hi=700,
              new_lo=1, new_hi=77, io="f32", rope=1, mix=2),
        # one user's next token on a small model: latency
        _case("decode one", "attend", q_heads=14, kv_heads=2, dim=64, page=16, cached_lo=513, cached_hi=513, rope=1),
        # one user's next token far into a long document: the cache split over the whole GPU
        _case("decode far", "attend", cached_lo=130001, cached_hi=130001, rope=2),
        # the batched-decode configuration's lengths
        _case("decode batch", "attend", batch=64, cached_lo=256, cached_hi=8192, rope=1, mix=3),
        # the largest decode: 64 query heads, caches twice as long as 8 bits would allow, capped scores
        _case("decode long", "attend", batch=32, q_heads=64, page=128, cached_lo=32768, cached_hi=32768, cap=30.0),
        # 32-bit tensors of a small model, distance bias
        _case("decode f32", "attend", batch=7, q_heads=32, kv_heads=4, dim=64, page=32, cached_lo=37, cached_hi=3001,
              io="f32", bias=True, mix=4),
        # a few drafted tokens a request, checked in one step
        _case("decode drafts", "attend", batch=24, page=32, cached_lo=1000, cached_hi=9000, new_lo=2, new_hi=5, rope=1, mix=9),
        # short continuations of running chats, prompt prefixes visible both ways, capped scores
        _case("prompt ragged", "attend", batch=6, q_heads=14, kv_heads=2, dim=64, page=16, cached_lo=0, cached_hi=2111,
              new_lo=3, new_hi=611, rope=2, prefix=True, cap=50.0, mix=6),
        # several documents packed in one prompt, attending within their own document
        _case("prompt docs", "attend", batch=2, page=64, new_lo=3900, new_hi=4096, rope=1, docs=True, mix=8),
        # a long prompt's later chunk
        _case("prompt long", "attend", page=128, cached_lo=14336, cached_hi=14336, new_lo=2048, new_hi=2048, rope=1),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "append", "attend", "attend", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    heads, kv, dim = rng.choice([(32, 8, 128), (64, 8, 128), (14, 2, 64), (32, 4, 64), (12, 4, 128), (8, 8, 64)])
    io = rng.choice(["f16", "f16", "f32"])
    base = dict(q_heads=heads, kv_heads=kv, dim=dim, page=page, mix=rng.randrange(1, 1 << 20), rope=rng.choice([0, 1, 2]))
    if op == "append":
        if rng.random() < 0.5:  # a decode step
            hi = _spread(rng, 1, 8192)
            return _case(None, op, batch=_spread(rng, 1, 128), cached_lo=rng.randrange(0, hi + 1), cached_hi=hi, io=io, **base)
        batch = _spread(rng, 1, 16)
        new = _spread(rng, 2, 10000 // batch)
        return _case(None, op, batch=batch, cached_hi=_spread(rng, 1, 3000), new_lo=rng.randrange(1, new + 1), new_hi=new,
                     io=io, **base)
    if rng.random() < 0.65:  # one token per sequence, or a few
        batch = _spread(rng, 1, 64)
        hi = _spread(rng, 1, min(131072, 500000 // batch))
        few = rng.choice([1, 1, 1, rng.randrange(2, 9)])
        return _case(None, op, batch=batch, cached_lo=rng.randrange(0, hi + 1), cached_hi=hi, new_hi=few, io=io,
                     cap=rng.choice([0.0, 0.0, 30.0]), bias=rng.random() < 0.25, **base)
    batch = _spread(rng, 1, 8)
    new = _spread(rng, 2, 2048 // batch)
    hi = _spread(rng, 1, 6144 // batch)
    docs = rng.random() < 0.3
    return _case(None, op, batch=batch, cached_lo=rng.randrange(0, hi + 1), cached_hi=hi, new_lo=rng.randrange(1, new + 1),
                 new_hi=new, cap=rng.choice([0.0, 0.0, 50.0]), bias=rng.random() < 0.25, docs=docs,
                 prefix=not docs and rng.random() < 0.4, **base)


def _lengths(case):
    """Cached and new rows of every sequence: part of the case, not of the data's seed."""
    r = random.Random(case["mix"])
    n = case["batch"]
    return ([r.randint(case["cached_lo"], case["cached_hi"]) for _ in range(n)],
            [r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)])


def _prefix(case, b, cached, new):
    """A prompt's two-way prefix: it may end among the cached rows, the new ones, or be absent."""
    return random.Random(case["mix"] * 1000 + b).choice([0, cached // 2, cached + new // 2, cached + new])


def _first_rows(case, cached, new):
    """First visible cache row of every new row: the start of its document (documents of 100 to 900 rows)."""
    first = []
    for b, (c, n) in enumerate(zip(cached, new)):
        r, start, row = random.Random(case["mix"] * 1000 + b), 0, []
        end = r.randint(100, 900)
        for p in range(c + n):
            if p == end:
                start, end = p, p + r.randint(100, 900)
            if p >= c:
                row.append(start)
        first += row
    return first


def _pairs(case):
    """(query row, visible cache row) pairs of one query head."""
    cached, new = _lengths(case)
    if case["docs"]:
        first, at, total = _first_rows(case, cached, new), 0, 0
        for c, n in zip(cached, new):
            total += sum(c + i + 1 - first[at + i] for i in range(n))
            at += n
        return total
    total = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        pre = _prefix(case, b, c, n) if case["prefix"] else 0
        total += sum(max(c + i + 1, pre) for i in range(n))
    return total


def work(case):
    cached, new = _lengths(case)
    T, H, D, P, B = sum(new), case["kv_heads"], case["dim"], case["page"], case["batch"]
    io = 2 if case["io"] == "f16" else 4
    row = 2 * H * (D // 2 + 4)  # a row of the cache: K and V codes and ranges
    if case["op"] == "append":
        # rows, slots and positions in, codes and ranges out; then the new rows out as the values they stand for
        return {"bytes": T * (2 * H * D * io + 20 + row) + T * 2 * H * D * io, "flops": 2 * H * D * T * 6}
    rows = 0  # cache rows that some query row sees
    first, at = (_first_rows(case, cached, new) if case["docs"] else None), 0
    for c, n in zip(cached, new):
        rows += c + n - (first[at] if first else 0)
        at += n
    return {"bytes": rows * row + 4 * (rows // P + 3 * B) + 2 * T * case["q_heads"] * D * io,
            "flops": 4 * case["q_heads"] * D * _pairs(case)}


# --------------------------------------------------------------------------------------------- inputs

def _dtype(case):
    return torch.float16 if case["io"] == "f16" else torch.float32


def _fill(g, n_pages, H, P, D, dev):
    """Pages as a running server holds them: rows of normal values about a mean of their own, in 4 bits."""
    pool = torch.empty(n_pages, H, P, D // 2, dtype=torch.uint8, device=dev)
    rng = torch.empty(n_pages, H, P, 2, dtype=torch.float16, device=dev)
    step = max(1, (1 << 27) // (H * P * D))
    for a in range(0, n_pages, step):
        x = torch.randn(min(step, n_pages - a), H, P, D, generator=g, device=dev)
        x += 0.5 * torch.randn(x.shape[0], H, P, 1, generator=g, device=dev)
        pool[a:a + step], rng[a:a + step] = _quantise(x)
    return pool, rng


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    cached, new = _lengths(case)
    B, P, H, D, Hq = case["batch"], case["page"], case["kv_heads"], case["dim"], case["q_heads"]
    T = sum(new)
    i32 = dict(dtype=torch.int32, device=dev)
    s = dict(case=case, tokens=T, max_new=max(new), max_kv=max(c + n for c, n in zip(cached, new)))
    s["max_pages"] = -(-s["max_kv"] // P) + 2
    held = [-(-(c + n) // P) for c, n in zip(cached, new)]
    s["n_pages"] = n_pages = sum(held) + 5
    # the pages of every sequence, scattered over the pool
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = np.full((B, s["max_pages"]), -1, dtype=np.int64)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = np.arange(at, at + n)
        at += n
    t = torch.from_numpy(table).to(dev)
    s["block_table"] = torch.where(t >= 0, order[t.clamp(min=0)], -1).to(torch.int32)
    s["row_start"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), **i32)
    s["kv_len"] = torch.tensor([c + n for c, n in zip(cached, new)], **i32)
    pos = np.concatenate([np.arange(c, c + n) for c, n in zip(cached, new)])
    seq = np.repeat(np.arange(B), new)
    s["positions"] = torch.tensor(pos, **i32)
    q, p = torch.from_numpy(seq).to(dev), torch.from_numpy(pos).to(dev)
    s["slots"] = s["block_table"].to(torch.int64)[q, p // P] * P + p % P
    for n in ("k", "v"):
        s[n + "_pool"], s[n + "_range"] = _fill(g, n_pages, H, P, D, dev)
    dt = _dtype(case)
    if case["op"] == "append":
        # rows of a fused projection's output: K and V beside each other
        kv = torch.randn(T, 2, H, D, generator=g, device=dev).to(dt)
        s["k_new"], s["v_new"] = kv[:, 0], kv[:, 1]
        return s
    s["q"] = (torch.randn(T, Hq, D, generator=g, device=dev) * (2.0 if case["cap"] else 1.0)).to(dt)
    s["prefix"] = s["first"] = s["slopes"] = None
    if case["prefix"]:
        s["prefix"] = torch.tensor([_prefix(case, b, c, n) for b, (c, n) in enumerate(zip(cached, new))], **i32)
    if case["docs"]:
        s["first"] = torch.tensor(_first_rows(case, cached, new), **i32)
    if case["bias"]:  # the usual geometric slopes
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=dev)
    return s


# --------------------------------------------------------------------------------------------- plain forms

def _quantise(x):
    """Rows x [..., D] (32 bits) as codes [..., D / 2] and ranges [..., 2]; every operation is rounded to 32 bits."""
    low = x.amin(-1).to(torch.float16)
    step = ((x.amax(-1) - low.to(torch.float32)) * (1.0 / 15.0)).to(torch.float16).clamp(min=TINY)
    inv = 1.0 / step.to(torch.float32)
    c = torch.round((x - low.to(torch.float32)[..., None]) * inv[..., None]).clamp(0, 15).to(torch.uint8)
    c = c.unflatten(-1, (-1, 8))
    c = c[..., [0, 4, 1, 5]] | c[..., [2, 6, 3, 7]] << 4
    return c.flatten(-2), torch.stack([low, step], dim=-1)


def _values(pool, rng):
    """The 32-bit values [..., D] that codes [..., D / 2] with ranges [..., 2] stand for."""
    c = pool.unflatten(-1, (-1, 4))
    c = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2)[..., [0, 4, 1, 5, 2, 6, 3, 7]].flatten(-2)
    r = rng.to(torch.float32)
    return r[..., 0:1] + r[..., 1:2] * c.to(torch.float32)


def _freqs(D):
    """Rotary frequencies 1 / theta^(2i/D), every step rounded to 32 bits."""
    f = np.float32
    return [float(f(1) / f(THETA ** float(f(2 * i) / f(D)))) for i in range(D // 2)]


def _rotate(x, pos, mode):
    """x [n, heads, D] (32 bits) rotated at pos [n] (mode 1: pairs (2i, 2i+1); 2: pairs (i, i + D/2)). The angle is the
    32-bit product of position and frequency, as everywhere in the framework; its cosine and sine come from 64 bits."""
    if mode == 0:
        return x
    D = x.shape[-1]
    ang = pos.to(torch.float32)[:, None] * torch.tensor(_freqs(D), dtype=torch.float32, device=x.device)
    ang = ang.double()[:, None, :]
    c, s = torch.cos(ang).to(torch.float32), torch.sin(ang).to(torch.float32)
    if mode == 1:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1)


def _plain_append(s):
    P, slots, dt = s["case"]["page"], s["slots"], _dtype(s["case"])
    page, row = slots // P, slots % P
    k = _rotate(s["k_new"].to(torch.float32), s["positions"], s["case"]["rope"])
    s["k_pool"][page, :, row], s["k_range"][page, :, row] = _quantise(k)
    s["v_pool"][page, :, row], s["v_range"][page, :, row] = _quantise(s["v_new"].to(torch.float32))
    return [_values(s["k_pool"][page, :, row], s["k_range"][page, :, row]).to(dt),
            _values(s["v_pool"][page, :, row], s["v_range"][page, :, row]).to(dt), s["k_range"], s["v_range"]]


def _plain_attend(s):
    case, T, S, L = s["case"], s["tokens"], s["max_new"], s["max_kv"]
    B, P, H, D, Hq = case["batch"], case["page"], case["kv_heads"], case["dim"], case["q_heads"]
    dev = s["q"].device
    start, kv_len = s["row_start"].to(torch.int64), s["kv_len"].to(torch.int64)
    t = torch.arange(T, device=dev)
    tb = torch.searchsorted(start, t, right=True) - 1
    c = kv_len - (start[1:] - start[:-1])
    q = _rotate(s["q"].to(torch.float32), c[tb] + t - start[tb], case["rope"])
    # sequences side by side, padded to the longest
    i, j = torch.arange(S, device=dev), torch.arange(L, device=dev)
    tok = (start[:-1, None] + i).clamp(max=T - 1)
    q = q[tok].reshape(B, S, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, Hq // H * S, D)
    page = s["block_table"].to(torch.int64).clamp(min=0)[:, j // P]
    k = _values(s["k_pool"][page, :, j % P], s["k_range"][page, :, j % P])
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))
    del k
    x = x.reshape(B, H, Hq // H, S, L)
    if case["cap"]:
        x = torch.tanh(x / case["cap"]) * case["cap"]
    pos = c[:, None] + i
    if s["slopes"] is not None:
        far = (pos[:, :, None] - j).abs().to(torch.float32)
        x = x - s["slopes"].reshape(1, H, Hq // H, 1, 1) * far[:, None, None]
    end = pos + 1 if s["prefix"] is None else torch.maximum(pos + 1, torch.minimum(s["prefix"], kv_len)[:, None])
    seen = j < torch.minimum(end, kv_len[:, None])[..., None]
    if s["first"] is not None:
        seen = seen & (j >= s["first"][tok][..., None])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    total = x.sum(-1, keepdim=True)
    x = x / torch.where(total > 0, total, 1.0)
    v = _values(s["v_pool"][page, :, j % P], s["v_range"][page, :, j % P])
    o = torch.matmul(x.reshape(B, H, Hq // H * S, L), v.permute(0, 2, 1, 3))
    o = o.reshape(B, H, Hq // H, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, Hq, D)
    return o[tb, t - start[tb]].to(s["q"].dtype)


# --------------------------------------------------------------------------------------------- one pass

_context = []


def _ops(s):
    """The handle that a user's program keeps: one context, one description of the layer."""
    from aihost_b200 import F16, F32, ROPE_INTERLEAVED, ROPE_NEOX, ROPE_NONE
    from aihost_b200.kv4 import Kv4Ops, Kv4Spec
    from aihost_b200.ops import Context

    if not _context:
        _context.append(Context(0))
    case = s["case"]
    code = F16 if case["io"] == "f16" else F32
    spec = Kv4Spec(case["q_heads"], case["kv_heads"], case["dim"], page_rows=case["page"], n_pages=s["n_pages"],
                   max_pages=s["max_pages"], io_dtype=code, out_dtype=code, score_cap=case["cap"], rope_theta=THETA,
                   rope_mode=(ROPE_NONE, ROPE_INTERLEAVED, ROPE_NEOX)[case["rope"]])
    s["ops"] = Kv4Ops(_context[0], spec)
    return s["ops"]


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return (_plain_append if op == "append" else _plain_attend)(s)
    ops = s.get("ops") or _ops(s)
    if op == "append":
        ops.append(s["k_new"], s["v_new"], s["slots"], s["positions"], s["k_pool"], s["v_pool"], s["k_range"], s["v_range"])
        dt = s["k_new"].dtype
        return [ops.read(s["k_pool"], s["k_range"], s["slots"], dt), ops.read(s["v_pool"], s["v_range"], s["slots"], dt),
                s["k_range"], s["v_range"]]
    return ops.attend(s["q"], s["row_start"], s["kv_len"], s["block_table"], s["k_pool"], s["v_pool"], s["k_range"],
                      s["v_range"], max_new=s["max_new"], max_kv=s["max_kv"], prefix_len=s["prefix"],
                      row_first=s["first"], alibi_slopes=s["slopes"])


# --------------------------------------------------------------------------------------------- the definitions, in 64 bits

def _turn(x, pos, mode):
    """x [n, heads, D] in 64 bits, as complex numbers times exp(i angle)."""
    if mode == 0:
        return x
    n, h, D = x.shape
    z = x.reshape(n, h, D // 2, 2) if mode == 1 else x.reshape(n, h, 2, D // 2).transpose(2, 3)
    ang = pos.to(torch.float32)[:, None] * torch.tensor(_freqs(D), dtype=torch.float32, device=x.device)
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(ang, dtype=torch.float64), ang.double())[:, None, :]
    z = torch.view_as_real(z)
    return (z if mode == 1 else z.transpose(2, 3)).reshape(n, h, D)


def _nibble(e):
    """Byte and shift of element e of a row."""
    n = (e % 8) // 2 + 4 * (e % 2)
    return e // 8 * 4 + n // 2, n % 2 * 4


def _decode(pool, rng, D):
    """Rows in 64 bits, element by element."""
    at = [_nibble(e) for e in range(D)]
    where = torch.tensor([a for a, _ in at], device=pool.device)
    shift = torch.tensor([b for _, b in at], dtype=torch.uint8, device=pool.device)
    return rng[..., 0:1].double() + ((pool[..., where] >> shift) & 15).double() * rng[..., 1:2].double()


def _exact_append(s):
    case, P = s["case"], s["case"]["page"]
    out, ranges = [], []
    for x, name in ((_turn(s["k_new"].double(), s["positions"], case["rope"]), "k"), (s["v_new"].double(), "v")):
        low = x.amin(-1, keepdim=True).to(torch.float16).double()
        step = ((x.amax(-1, keepdim=True) - low) / 15).to(torch.float16).double().clamp(min=TINY)
        out.append(low + step * torch.round((x - low) / step).clamp(0, 15))
        r = s[name + "_range"].double()
        r[s["slots"] // P, :, s["slots"] % P] = torch.cat([low, step], dim=-1)
        ranges.append(r)
    return out + ranges


def _exact_attend(s):
    case, P, D = s["case"], s["case"]["page"], s["case"]["dim"]
    H, G = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    cached, new = _lengths(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        j = torch.arange(c + n, device=out.device)
        pages = s["block_table"][b, :-(-(c + n) // P)].long()
        i = torch.arange(c, c + n, device=out.device)
        q = _turn(s["q"][at:at + n].double(), i, case["rope"])
        end = (i + 1).clamp(min=_prefix(case, b, c, n) if case["prefix"] else 0)
        hidden = j[None, :] >= end[:, None]
        if case["docs"]:
            hidden |= j[None, :] < s["first"][at:at + n, None]
        for h in range(H):
            k = _decode(s["k_pool"][pages, h], s["k_range"][pages, h], D).reshape(-1, D)[:c + n]
            v = _decode(s["v_pool"][pages, h], s["v_range"][pages, h], D).reshape(-1, D)[:c + n]
            for g in range(h * G, h * G + G):
                x = (q[:, g] @ k.T) / math.sqrt(D)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["bias"]:
                    x -= 2.0 ** (-8.0 * (g + 1) / case["q_heads"]) * (i[:, None] - j[None, :]).abs()
                out[at:at + n, g] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v
        at += n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)

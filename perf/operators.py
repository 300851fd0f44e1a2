"""Timed cases of the operators around the KV cache: norm and rotation of heads, the rotated append,
the cache read back as values, and attention of a chunk of new tokens over the cache.

Every case is a dict of plain values. `prepare` makes what a serving program holds before the call,
`run` makes one pass, in plain torch where `own` is false and through kvforge_b200.api where it is true.

    op      rope, append, gather or attend
    B, T    sequences and new tokens per sequence (gather: tokens read back)
    H, Hkv  query heads and KV heads;  d  channels of a head
    n       tokens a sequence's cache holds;  fmt, group, order, page  its format and placement
    dtype   type of the model's activations
    ragged  sequences of unequal lengths (a ramp, in an order that the seed gives)
    norm    RMS norm of each head before the rotation;  rot  rotated channels;  inter  adjacent pairs
    causal  new token j sees the cache up to itself (else the whole sequence)
"""
import math

import torch

own = False

F16, INT8, INT4 = 0, 1, 2
HEAD, TOKEN = 0, 1
EPS = 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
FMTS = {"f16": F16, "int8": INT8, "int4": INT4}


def listed():
    return [
        # one decode step of a batch of 64 with the query heads of the 70B serving shape
        dict(name="rope_step_b64", op="rope", B=64, T=1, H=64, Hkv=8, d=128, dtype="bf16", ragged=False, norm=True,
             rot=128, inter=False, positions=16384),
        # a batch of four prompt chunks of odd length, the same heads
        dict(name="rope_chunk_b4", op="rope", B=4, T=4001, H=64, Hkv=8, d=128, dtype="bf16", ragged=False, norm=True,
             rot=128, inter=False, positions=32768),
        # the same decode step's keys and values (and queries) on their way into an int8 paged cache
        dict(name="append_step_b64_int8", op="append", B=64, T=1, H=64, Hkv=8, d=128, n=16384, fmt="int8", group=64,
             order="token", page=16, dtype="bf16", ragged=False, norm=True, rot=128, inter=False),
        # prompt chunks of unequal lengths into an int8 paged cache
        dict(name="append_chunk_b8_int8", op="append", B=8, T=2048, H=32, Hkv=8, d=128, n=8192, fmt="int8", group=64,
             order="token", page=16, dtype="bf16", ragged=True, norm=False, rot=128, inter=False),
        # a model with narrow heads, partial rotation of adjacent pairs, f16 head-major cache, odd sizes
        dict(name="append_odd_f16_d64", op="append", B=3, T=333, H=20, Hkv=5, d=64, n=1000, fmt="f16", group=0,
             order="head", page=0, dtype="f16", ragged=True, norm=False, rot=32, inter=True),
        # the ragged paged f16 batch read back, as when sequences move to another pool
        dict(name="gather_b8_f16_p16", op="gather", B=8, T=8192, H=32, Hkv=8, d=128, n=8192, fmt="f16", group=0,
             order="token", page=16, dtype="f16", ragged=True),
        # one long int4 sequence read back as values
        dict(name="gather_b1_n65536_int4", op="gather", B=1, T=65536, H=32, Hkv=8, d=128, n=65536, fmt="int4",
             group=32, order="head", page=0, dtype="bf16", ragged=False),
        # four drafted tokens per sequence verified against the 70B serving batch's cache
        dict(name="attend_verify_b64_int8", op="attend", B=64, T=4, H=64, Hkv=8, d=128, n=16384, fmt="int8", group=64,
             order="token", page=16, dtype="bf16", ragged=False, causal=True),
        # a chunk of a long prompt against all that came before it, the 8B shape
        dict(name="attend_chunk_n32768_int8", op="attend", B=1, T=4096, H=32, Hkv=8, d=128, n=32768, fmt="int8",
             group=64, order="token", page=0, dtype="bf16", ragged=False, causal=True),
        # a whole prompt at once, one KV head per query head
        dict(name="attend_prompt_mha_f16", op="attend", B=1, T=4096, H=32, Hkv=32, d=128, n=4096, fmt="f16", group=0,
             order="head", page=0, dtype="f16", ragged=False, causal=True),
        # chunks of unequal lengths over a ragged paged f16 batch
        dict(name="attend_ragged_b8_f16_p16", op="attend", B=8, T=512, H=32, Hkv=8, d=128, n=8192, fmt="f16", group=0,
             order="token", page=16, dtype="bf16", ragged=True, causal=True),
        # cross attention to an encoder's states of odd length, fp32 queries, narrow heads
        dict(name="attend_cross_f32_d64", op="attend", B=4, T=100, H=16, Hkv=16, d=64, n=1500, fmt="int4", group=32,
             order="head", page=0, dtype="f32", ragged=False, causal=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "append", "gather", "attend"))
    d = rng.choice((64, 128, 128))
    g = rng.choice((1, 2, 4, 5, 7, 8))
    Hkv = rng.choice((1, 2, 4, 5, 8, 8, 16))
    c = dict(op=op, B=_log(rng, 1, 64), T=_log(rng, 1, 4096), H=g * Hkv, Hkv=Hkv, d=d,
             dtype=rng.choice(("bf16", "bf16", "f16", "f32")), ragged=rng.random() < 0.5)
    if op in ("rope", "append"):
        c.update(norm=rng.random() < 0.5, rot=rng.choice((d, d, d // 2)), inter=rng.random() < 0.3)
    if op == "rope":
        while c["B"] * c["T"] * (c["H"] + 2 * Hkv) * d > 80_000_000:
            c["T"] = (c["T"] + 1) // 2
        c["positions"] = _log(rng, c["T"] + 1, 65536)
        return c
    fmt = rng.choice(("f16", "int8", "int8", "int4"))
    c.update(fmt=fmt, group=0 if fmt == "f16" else rng.choice([x for x in (32, 64, 128) if x <= d and (x > 32 or fmt == "int4")]),
             order=rng.choice(("head", "token")), page=rng.choice((0, 16, 32, 64, 128)))
    if op == "attend":
        c["causal"] = rng.random() < 0.75
    n = _log(rng, 16, 32768)
    # bounds on the cache and on the scores, which the plain form holds whole
    while c["B"] * Hkv * n * d > 60_000_000:
        if c["B"] > 1:
            c["B"] = (c["B"] + 1) // 2
        else:
            n = (n + 1) // 2
    c["n"] = n
    c["T"] = n if op == "gather" else min(c["T"], n)
    if op == "attend":
        while c["B"] * c["H"] * c["T"] * n > 2_000_000_000:
            c["T"] = (c["T"] + 1) // 2
    return c


# ------------------------------------------------------------------ inputs
def _ramp(lo, hi, B):
    """B lengths from lo to hi: their sum is the case's, whatever order the seed gives."""
    return [lo + (hi - lo) * (i + 1) // B for i in range(B)] if B > 1 else [(lo + hi + 1) // 2]


def _lengths(case):
    """(new tokens, stored tokens) of each sequence, before the seed's order."""
    B, T, n = case["B"], case["T"], case.get("n", 0)
    if not case["ragged"]:
        return [T] * B, [n] * B
    if case["op"] == "gather":
        kv = _ramp(max(1, n // 4), n, B)
        return kv, kv
    new = _ramp(max(1, T // 4), T, B)
    if case["op"] == "attend":
        return new, [max(t, x) for t, x in zip(new, _ramp(max(1, n // 4), n, B))]
    return new, [n] * B


def _table(g, B, n, page):
    """Pages of every sequence in an order that the seed gives."""
    blocks = (n + page - 1) // page
    return torch.randperm(B * blocks, generator=g, device="cuda").to(torch.int32).reshape(B, blocks), B * blocks


def _rows(case, table, b, h, t):
    """Physical cache row of (sequence, KV head, token), broadcast over the three."""
    n, Hkv, page = case["n"], case["Hkv"], case["page"]
    if not page:
        return (b * Hkv + h) * n + t if case["order"] == "head" else (b * n + t) * Hkv + h
    base = table.long()[b, t // page] * (Hkv * page)
    return base + (h * page + t % page if case["order"] == "head" else (t % page) * Hkv + h)


def _quantize(x, fmt, group):
    """Rows of fp32 channels as the cache stores them: (payload, words of scale and zero or None)."""
    if fmt == "f16":
        return x.half().view(torch.uint8), None
    levels = 255 if fmt == "int8" else 15
    y = x.reshape(*x.shape[:-1], -1, group)
    lo, hi = y.amin(-1), y.amax(-1)
    scale = (hi - lo) / levels
    scale_h, zero_h = torch.where(scale <= 0, 1.0, scale).half(), lo.half()
    t = (y - zero_h.float()[..., None]) / scale_h.float()[..., None]
    code = torch.where(t - t.floor() < 0.5, t.floor(), t.floor() + 1).clamp(0, levels).to(torch.uint8).reshape(x.shape)
    word = torch.stack((scale_h, zero_h), -1).view(torch.int32)[..., 0]
    return (code if fmt == "int8" else code[..., 0::2] | (code[..., 1::2] << 4)), word


def _values(data, word, fmt, group):
    """fp32 values of stored rows."""
    if fmt == "f16":
        return data.view(torch.float16).float()
    if fmt == "int4":
        data = torch.stack((data & 15, data >> 4), -1).flatten(-2)
    s = word[..., None].contiguous().view(torch.float16).float()
    y = data.float().reshape(*data.shape[:-1], -1, group)
    return (y * s[..., 0:1] + s[..., 1:2]).reshape(data.shape)


def _cache(case, g):
    """A filled cache: keys and values of normal channels, one channel in a hundred eight times as large."""
    B, Hkv, n, d, fmt, group = (case[k] for k in ("B", "Hkv", "n", "d", "fmt", "group"))
    table, pages = _table(g, B, n, case["page"]) if case["page"] else (None, 0)
    rows = pages * Hkv * case["page"] if case["page"] else B * Hkv * n
    c = {"table": table}
    loud = torch.where(torch.rand((Hkv, d), generator=g, device="cuda") < 0.01, 8.0, 1.0)
    channels = torch.arange(rows, device="cuda")
    head = (channels % Hkv if case["order"] == "token" else channels // (case["page"] or n) % Hkv)
    for name in ("k", "v"):
        x = torch.randn((rows, d), generator=g, device="cuda") * loud[head]
        c[name], c[name + "_meta"] = _quantize(x, fmt, group)
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    B, T, H, Hkv, d, op = (case[k] for k in ("B", "T", "H", "Hkv", "d", "op"))
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    order = torch.randperm(B, generator=g, device="cuda")
    new, kv = (torch.tensor(x, dtype=torch.int32, device="cuda")[order] for x in _lengths(case))
    st["lens"] = new if case["ragged"] else None
    # activations as one projection leaves them: query, key and value heads side by side
    if op in ("rope", "append", "attend"):
        st["qkv"] = torch.randn((B, T, (H + 2 * Hkv), d), generator=g, device="cuda", dtype=torch.float32).to(dt)
        st["q"], st["k_new"], st["v_new"] = st["qkv"].split((H, Hkv, Hkv), 2)
        st["out"] = torch.zeros((B, T, H, d), dtype=dt, device="cuda")
    if op in ("rope", "append"):
        size = case["positions"] if op == "rope" else case["n"]
        angle = torch.arange(size, dtype=torch.float64, device="cuda")[:, None] * \
            10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        st["wq"], st["wk"] = ((1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt) if case["norm"] else None
                              for _ in range(2))
        st["pos"] = torch.randint(0, size - T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    if op != "rope":
        st.update(_cache(case, g))
    if op in ("gather", "attend"):
        st["seq_lens"] = kv if case["ragged"] else None
        st["kv"] = kv
    if op in ("append", "gather"):
        # read back in 16 bits: which of two neighbouring codes a value on their border gets is a matter of rounding
        st["values"] = [torch.zeros((B, T, Hkv, d), dtype=torch.float16 if dt == torch.float32 and op == "append" else dt,
                                    device="cuda") for _ in range(2)]
    if own:
        from kvforge_b200 import api
        from kvforge_b200.layout import Placement

        if op != "rope":
            st["cache"] = api.KVCache(
                fmt=FMTS[case["fmt"]], d=d, group=case["group"],
                place=Placement(HEAD if case["order"] == "head" else TOKEN, case["page"] > 0, case["page"]), B=B,
                Hkv=Hkv, n=case["n"], k=st["k"], v=st["v"], k_meta=st["k_meta"], v_meta=st["v_meta"],
                block_table=st["table"], max_blocks=st["table"].shape[1] if st["table"] is not None else 0,
                seq_lens=st.get("seq_lens"))
        if op in ("rope", "append"):
            st["rope"] = api.Rope(st["cos"], st["sin"], interleaved=case["inter"])
        if op == "attend":
            st["ws"] = api.ChunkWorkspace.allocate(st["cache"], T, H, dt)
    return st


# ------------------------------------------------------------------ plain forms
def _norm_rope(x, st, weight):
    """Heads in fp32: x * (1 / sqrt(mean(x^2) + eps)) * weight, then the rotation of its first `rot` channels."""
    case = st["case"]
    x = x.float()
    if weight is not None:
        s = x * x
        # the squares added in pairs of neighbours, so that the order of the sum is a given one
        s = s.unflatten(-1, (-1, 2)).sum(-1).unflatten(-1, (-1, 2)).sum(-1).unflatten(-1, (-1, 2)).sum(-1)
        s = s.unflatten(-1, (-1, 2)).sum(-1).unflatten(-1, (-1, 2)).sum(-1).unflatten(-1, (-1, 2)).sum(-1)
        s = s.unflatten(-1, (-1, 2)).sum(-1) if s.shape[-1] == 2 else s
        x = x * (1.0 / torch.sqrt(s / case["d"] + EPS)) * weight.float()
    at = (st["pos"][:, None] + torch.arange(case["T"], device="cuda")).long()
    c, s = st["cos"][at][:, :, None], st["sin"][at][:, :, None]
    r = case["rot"]
    if case["inter"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((y, x[..., r:]), -1)


def _live(st, T):
    """[B][T]: the new tokens that are there."""
    B = st["case"]["B"]
    if st["lens"] is None:
        return torch.ones((B, T), dtype=torch.bool, device="cuda")
    return torch.arange(T, device="cuda") < st["lens"][:, None]


def _token_rows(case, table, first):
    """[B][T][Hkv] physical rows of T tokens from `first` on (the last token's where there are no more)."""
    b = torch.arange(case["B"], device="cuda")[:, None, None]
    t = first.long()[:, None, None] + torch.arange(case["T"], device="cuda")[:, None]
    return _rows(case, table, b, torch.arange(case["Hkv"], device="cuda"), t.clamp(max=case["n"] - 1))


def _plain_rope(st):
    return torch.where(_live(st, st["case"]["T"])[..., None, None], _norm_rope(st["q"], st, st["wq"]), 0.0).to(st["out"].dtype)


def _plain_append(st):
    case = st["case"]
    live = _live(st, case["T"])
    q = torch.where(live[..., None, None], _norm_rope(st["q"], st, st["wq"]), 0.0).to(st["out"].dtype)
    k, v = _norm_rope(st["k_new"], st, st["wk"]), st["v_new"].float()
    rows = _token_rows(case, st["table"], st["pos"])[live].flatten()
    back = []
    for name, x in (("k", k), ("v", v)):
        data, word = _quantize(x[live].flatten(0, 1), case["fmt"], case["group"])
        st[name][rows] = data
        if word is not None:
            st[name + "_meta"][rows] = word
            values = _values(data, word, case["fmt"], case["group"])
            out = torch.zeros_like(x)
            out[live] = values.unflatten(0, (-1, case["Hkv"]))
            back.append(out.to(st["values"][0].dtype))
        else:
            back.append(st[name].view(torch.float16))
    return [q] + back


def _plain_gather(st):
    case = st["case"]
    rows = _token_rows(case, st["table"], torch.zeros(case["B"], device="cuda"))
    live = _live(st, case["T"])[..., None, None]
    back = []
    for name in ("k", "v"):
        word = st[name + "_meta"]
        x = _values(st[name][rows], None if word is None else word[rows], case["fmt"], case["group"])
        back.append(torch.where(live, x, 0.0).to(st["values"][0].dtype))
    return back


def _plain_attend(st):
    case = st["case"]
    B, T, H, Hkv, d, n = (case[k] for k in ("B", "T", "H", "Hkv", "d", "n"))
    b, h = torch.arange(B, device="cuda")[:, None, None], torch.arange(Hkv, device="cuda")[:, None]
    t = torch.arange(n, device="cuda")
    rows = _rows(case, st["table"], b, h, t)
    k, v = (_values(st[x][rows], None if st[x + "_meta"] is None else st[x + "_meta"][rows], case["fmt"], case["group"])
            for x in ("k", "v"))
    kv = st["kv"].long()[:, None, None, None]
    v = torch.where(t[:, None] < kv, v, 0.0)
    q = st["q"].float().unflatten(2, (Hkv, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [B][Hkv][T * g][d]
    live = _live(st, T)
    seen = kv.expand(B, 1, T, 1)
    if case["causal"]:
        seen = seen - live.sum(1)[:, None, None, None] + torch.arange(T, device="cuda")[:, None] + 1
    seen = seen.repeat_interleave(H // Hkv, 2)
    s = (q @ k.transpose(-1, -2)).mul_(d ** -0.5)
    s.masked_fill_(t >= seen, -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_min_(-3e38)).exp_()
    o = (s @ v) / s.sum(-1, keepdim=True).clamp_min_(1e-38)
    o = o.unflatten(2, (T, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return torch.where(live[..., None, None], o, 0.0).to(st["out"].dtype)


def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return {"rope": _plain_rope, "append": _plain_append, "gather": _plain_gather, "attend": _plain_attend}[op](st)
    from kvforge_b200 import api

    if op == "rope":
        return api.norm_rope(st["q"], st["pos"], st["rope"], weight=st["wq"], eps=EPS, lens=st["lens"], out=st["out"])
    if op == "append":
        q = api.append_rope(st["cache"], st["k_new"], st["v_new"], st["rope"], pos=st["pos"], lens=st["lens"],
                            k_weight=st["wk"], q=st["q"], q_weight=st["wq"], q_out=st["out"], eps=EPS)
        if case["fmt"] == "f16":
            return [q, st["k"].view(torch.float16), st["v"].view(torch.float16)]
        return [q] + list(api.gather(st["cache"], case["T"], pos=st["pos"], lens=st["lens"], out=st["values"]))
    if op == "gather":
        return list(api.gather(st["cache"], case["T"], lens=st["lens"], out=st["values"]))
    return api.chunk_attention(st["q"], st["cache"], q_lens=st["lens"], causal=case["causal"], out=st["out"],
                               workspace=st["ws"])


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    B, T, H, Hkv, d, op = (case[k] for k in ("B", "T", "H", "Hkv", "d", "op"))
    new, kv = _lengths(case)
    e = SIZE[case["dtype"]]
    row = 0
    if op != "rope":
        row = {"f16": 2 * d, "int8": d, "int4": d // 2}[case["fmt"]] + (4 * d // case["group"] if case["group"] else 0)
    tables = sum(new) * 4 * case.get("rot", 0)
    if op == "rope":
        return {"bytes": 2 * sum(new) * H * d * e + tables, "flops": sum(new) * H * d * (7 if case["norm"] else 3)}
    if op == "append":
        values = 2 * sum(new) * Hkv * (d * e + row)  # the rows as they come and as they are stored
        back = 2 * sum(new) * Hkv * d * 2 if case["fmt"] != "f16" else 0  # the values of what was stored
        return {"bytes": 2 * sum(new) * H * d * e + values + back + tables, "flops": 10 * sum(new) * (H + 2 * Hkv) * d}
    if op == "gather":
        return {"bytes": 2 * sum(new) * Hkv * (row + d * e), "flops": 2 * sum(new) * Hkv * d * 2}
    pairs = sum(t * x - (t * (t - 1) // 2 if case["causal"] else 0) for t, x in zip(new, kv))
    return {"bytes": 2 * sum(new) * H * d * e + 2 * sum(kv) * Hkv * row, "flops": 4 * pairs * H * d}


# ------------------------------------------------------------------ 64 bits, from the definitions
def _exact_heads(x, st, weight):
    case = st["case"]
    x, r = x.double(), case["rot"]
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    at = st["pos"].long()[:, None] + torch.arange(case["T"], device="cuda")
    turn = torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, :, None]
    head = x[..., :r].unflatten(-1, (r // 2, 2) if case["inter"] else (2, r // 2))
    if not case["inter"]:
        head = head.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
    z = z.flatten(-2) if case["inter"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., r:]), -1)


def _exact_stored(data, word, fmt, group):
    if fmt == "f16":
        return data.view(torch.float16).double()
    if fmt == "int4":
        both = torch.empty((*data.shape[:-1], 2 * data.shape[-1]), dtype=torch.uint8, device="cuda")
        both[..., 0::2], both[..., 1::2] = data % 16, data // 16
        data = both
    pair = word.contiguous().view(torch.float16).double()
    return data.double() * pair[..., 0::2].repeat_interleave(group, -1) + pair[..., 1::2].repeat_interleave(group, -1)


def _exact_quantized(x, fmt, group):
    """The values that the nearest codes of each group's range stand for."""
    top = {"int8": 255, "int4": 15}[fmt]
    y = x.unflatten(-1, (-1, group))
    low, high = y.aminmax(dim=-1, keepdim=True)
    zero, step = low.half().double(), (high - low) / top
    step = torch.where(step > 0, step, 1.0).half().double()
    return (((y - zero) / step + 0.5).floor().clamp(0, top) * step + zero).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    B, T, H, Hkv, n, op = (case[k] for k in ("B", "T", "H", "Hkv", "n", "op")) if "n" in case else \
        (*(case[k] for k in ("B", "T", "H", "Hkv")), 0, "rope")
    lens = st["lens"].tolist() if st["lens"] is not None else [T] * B
    if op in ("rope", "append"):
        q = _exact_heads(st["q"], st, st["wq"])
        for b, m in enumerate(lens):
            q[b, m:] = 0
        if op == "rope":
            return q
        k, v = _exact_heads(st["k_new"], st, st["wk"]), st["v_new"].double()
        if case["fmt"] != "f16":
            back = [_exact_quantized(x, case["fmt"], case["group"]) for x in (k, v)]
            for x in back:
                for b, m in enumerate(lens):
                    x[b, m:] = 0
            return [q] + back
        back = [st[x].view(torch.float16).double() for x in ("k", "v")]
        heads = torch.arange(Hkv, device="cuda")
        for b, m in enumerate(lens):
            t = int(st["pos"][b]) + torch.arange(m, device="cuda")[:, None]
            rows = _rows(case, st["table"], torch.full_like(t, b), heads, t)
            for x, y in zip(back, (k, v)):
                x[rows] = y[b, :m]
        return [q] + back
    if op == "gather":
        back = [torch.zeros((B, T, Hkv, case["d"]), dtype=torch.float64, device="cuda") for _ in range(2)]
    else:
        out = torch.zeros((B, T, H, case["d"]), dtype=torch.float64, device="cuda")
    kv = st["kv"].tolist()
    g = H // Hkv
    for b in range(B):
        t = torch.arange(kv[b], device="cuda")
        for h in range(Hkv):
            rows = _rows(case, st["table"], torch.full_like(t, b), h, t)
            k, v = (_exact_stored(st[x][rows], st[x + "_meta"][rows] if st[x + "_meta"] is not None else None,
                                  case["fmt"], case["group"]) for x in ("k", "v"))
            if op == "gather":
                for x, y in zip(back, (k, v)):
                    x[b, : lens[b], h] = y[: lens[b]]
                continue
            s = st["q"][b, : lens[b], h * g: h * g + g].double() @ k.T / math.sqrt(case["d"])
            if case["causal"]:
                last = kv[b] - lens[b] + torch.arange(lens[b], device="cuda")
                s.masked_fill_(t > last[:, None, None], -math.inf)
            out[b, : lens[b], h * g: h * g + g] = torch.softmax(s, -1) @ v
    return back if op == "gather" else out

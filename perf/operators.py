"""The paged key-value cache: appending new tokens (position rotation applied on the way) and the attention of one new token
per sequence over it, or of a few (drafted tokens that are checked in one pass), as cases that a serving program makes.

A case is a dict of plain values; its `kind` names the calls of one pass:

  append         PagedAttnKernel.append         FixedI8 rows into int8 pages, queries rotated too
  append_scaled  PagedAttnKernel.append_scaled  bf16 rows, rotated, then quantised with one scale per token and head
  decode         PagedAttnKernel.decode         attention over FixedI8 pages, bf16 out and L
  decode_scaled  PagedAttnKernel.decode_scaled  the same over codes with a scale per token and head
  step           append, then decode            what one layer of a decode step does, FixedI8 out

With `own` false `run` computes the same in elementary torch operations. The cache's codes are whole numbers by definition (the
FixedI8 rotation is integer arithmetic; the scaled form's code is a rounded f32 product of defined operations), so they are
returned as they lie in the pages and have to be equal; FixedI8 attention output is returned as the values it stands for.
"""
import math

import torch

own = False

SINK_SCALE = 0.125        # FixedI8: value = code / 8
ROPE_ONE = 1 << 14        # cos and sin are int16 in units of 2^-14
TINY = 2.0 ** -100        # a head whose largest value is no larger is stored as zeros

_STREAM = None


def _stream():
    """The program's one stream, opened at first use: torch work on it is ordered with the framework's."""
    global _STREAM
    if _STREAM is None:
        from x17ai_b200 import device
        s = torch.cuda.Stream()
        _STREAM = (s, device.TorchStream(s))
    return _STREAM


def listed():
    return [
        # one user's decode step: a single token goes into the cache of the benchmark's heads; bound by the launch
        dict(name="append_one_user", kind="append", heads=32, kv_heads=32, head_dim=128, page=64, rotary=128, adjacent=False,
             seqs=1, tokens=1, start=1500, padding=0, kv_out=False),
        # continuous batching: one token for each of 121 sequences at different lengths, and 7 rows of padding
        dict(name="append_step_scaled", kind="append_scaled", heads=32, kv_heads=8, head_dim=128, page=32, rotary=128,
             adjacent=False, seqs=121, tokens=121, start=3000, padding=7),
        # a long prompt of the benchmark's size; its prefill attention reads the rotated rows too
        dict(name="append_prompt", kind="append", heads=32, kv_heads=32, head_dim=128, page=64, rotary=128, adjacent=False,
             seqs=1, tokens=8192, start=0, padding=0, kv_out=True),
        # three prompts of odd lengths behind cached prefixes, narrower heads of which half is rotated, adjacent pairs
        dict(name="append_prompts_scaled", kind="append_scaled", heads=64, kv_heads=8, head_dim=64, page=16, rotary=32,
             adjacent=True, seqs=3, tokens=13001, start=777, padding=0),
        # a single user's decode: few keys, one sequence
        dict(name="decode_one_user", kind="decode", heads=32, kv_heads=32, head_dim=128, page=64, seqs=1, length=1500, new=1,
             window=0, ragged=False),
        # the reference harness's narrow heads, three short sequences with five drafted tokens each, the smallest page
        dict(name="decode_narrow_heads", kind="decode", heads=64, kv_heads=64, head_dim=32, page=16, seqs=3, length=701,
             new=5, window=0, ragged=True),
        # continuous batching with a window: 48 sequences at different lengths, four query heads a key head
        dict(name="decode_ragged_window", kind="decode", heads=32, kv_heads=8, head_dim=128, page=32, seqs=48, length=4096,
             new=1, window=1024, ragged=True),
        # a large ragged batch, eight query heads a key head
        dict(name="decode_grouped_batch", kind="decode", heads=32, kv_heads=4, head_dim=128, page=64, seqs=128, length=8192,
             new=1, window=0, ragged=True),
        # the most cache a pass reads: 64 full sequences of the benchmark's heads, 2.1 GB
        dict(name="decode_full_batch", kind="decode", heads=32, kv_heads=32, head_dim=128, page=128, seqs=64, length=4096,
             new=1, window=0, ragged=False),
        # one user with a very long context: the work has to be split over its length
        dict(name="decode_scaled_long", kind="decode_scaled", heads=32, kv_heads=8, head_dim=128, page=64, seqs=1,
             length=131072, new=1, window=0, ragged=False),
        # ragged batch of narrower heads with scales, three drafted tokens a sequence
        dict(name="decode_scaled_ragged", kind="decode_scaled", heads=16, kv_heads=2, head_dim=64, page=16, seqs=24,
             length=16001, new=3, window=0, ragged=True),
        # one layer's cache work in a decode step of 16 sequences
        dict(name="step_16", kind="step", heads=32, kv_heads=32, head_dim=128, page=64, rotary=128, adjacent=False, seqs=16,
             length=1800, new=1, window=0, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (heads, kv_heads): the benchmark's, the reference harness's, and grouped ones, odd groups and a single key head among them
_HEADS = ((32, 32), (64, 64), (32, 8), (32, 4), (16, 2), (20, 4), (12, 4), (56, 8), (64, 4), (16, 1), (8, 8), (7, 7))


def draw(rng):
    kind = rng.choice(("append", "append", "append_scaled", "append_scaled", "decode", "decode", "decode", "decode_scaled",
                       "decode_scaled", "decode_scaled", "step"))
    heads, kv_heads = rng.choice(_HEADS)
    d = rng.choice((32, 64, 128, 128))
    page = rng.choice((16, 32, 64, 128))
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, head_dim=d, page=page)
    if kind.startswith("append") or kind == "step":
        c.update(rotary=rng.choice((d, d, 32, 0) if d > 32 else (32, 32, 0)), adjacent=rng.random() < 0.4)
    if kind.startswith("append"):
        tokens = _log(rng, 1, 16384)
        while tokens * (heads + 2 * kv_heads) * d > 2.2e8:
            tokens = tokens * 2 // 3
        seqs = tokens if rng.random() < 0.4 else _log(rng, 1, tokens)
        c.update(seqs=min(seqs, 512), tokens=tokens, start=_log(rng, 1, 30000), padding=rng.choice((0, 0, 1, 13)))
        if kind == "append":
            c["kv_out"] = rng.random() < 0.5
        # the pool holds the cached prefixes as well: keep it to a size that is made quickly
        while (c["start"] + 1) * c["seqs"] * kv_heads * 2 * d > 4e8:
            c["start"] = c["start"] * 2 // 3
        return c
    length = _log(rng, 1, 100000) if kind != "step" else _log(rng, 16, 8192)
    seqs = _log(rng, 1, 256)
    while seqs > 1 and seqs * length * kv_heads * 2 * d > 1.5e9:
        seqs -= max(1, seqs // 8)
    while seqs * length * kv_heads * 2 * d > 1.5e9:
        length = length * 2 // 3
    new = rng.choice((1, 1, 1, 2, 4, 7)) if kind != "step" else 1
    c.update(seqs=seqs, length=length, new=new, window=rng.choice((0, 0, 16 * rng.randint(1, 64), 1024, 4096)), ragged=rng.random() < 0.6)
    return c


# ---- inputs ------------------------------------------------------------------------------------------

def _lens(c):
    """Keys in front of each sequence's first new token (spread evenly up to `length` where ragged; the same for every seed, so the work is too)."""
    n, b = c["length"], c["seqs"]
    return [max(1, n * (1 + (7 * i + 3) % b) // b) if c["ragged"] else n for i in range(b)]


def _tokens(c):
    """(first position, new tokens) of each sequence of an append."""
    b, t = c["seqs"], c["tokens"]
    return [(c["start"] * (1 + (5 * i + 2) % b) // b, t * (i + 1) // b - t * i // b) for i in range(b)]


def _unit_heads(x):
    """Heads scaled to unit mean square over their last dimension, as the K projection leaves them."""
    return x.div_(x.square().mean(-1, keepdim=True).sqrt_())


def _codes(x):
    return x.mul_(8.0).round_().clamp_(-127, 127).to(torch.int8)


def _kv_values(g, rows, heads, d):
    """K | V rows: K of unit mean square per head, V a little wider."""
    x = torch.randn(rows, heads, 2, d, generator=g, device="cuda")
    _unit_heads(x[:, :, 0])
    x[:, :, 1] *= 1.3
    return x


def _page_table(g, page, ends):
    """A page for every 16 to 128 tokens up to each sequence's end, in no order; -1 behind the last one."""
    need = [-(-e // page) for e in ends]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(ends), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, n_pages


def _pool(c, g, n_pages):
    """Pages filled with keys and values of earlier tokens (and their scales)."""
    h, page, d = c["kv_heads"], c["page"], c["head_dim"]
    pages = torch.empty((n_pages, h, page, 2 * d), dtype=torch.int8, device="cuda")
    scales = torch.empty((n_pages, h, page, 2), device="cuda") if c["kind"].endswith("scaled") else None
    chunk = max(1, (1 << 26) // (h * page * 2 * d))
    for i in range(0, n_pages, chunk):
        n = min(chunk, n_pages - i)
        x = _kv_values(g, n * page, h, d).view(n, page, h, 2, d).transpose(1, 2)
        if scales is None:
            pages[i:i + n] = _codes(x).reshape(n, h, page, 2 * d)
        else:
            s = x.abs().amax(-1).div_(127.0)
            scales[i:i + n] = s
            pages[i:i + n] = x.div(s.unsqueeze(-1)).round_().to(torch.int8).reshape(n, h, page, 2 * d)
    return pages, scales


def _rope(n, rotary):
    """cos and sin of position * 10000^(-2i / rotary), angles in 64 bits, int16 in units of 2^-14."""
    f = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    a = torch.arange(n, dtype=torch.float64, device="cuda").unsqueeze(1) * f
    return torch.stack((a.cos(), a.sin()), dim=-1).mul_(ROPE_ONE).round_().to(torch.int16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _new(dtype, *shape):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _prepare_append(c, g, st, runs):
    """`runs`: (first position, new tokens) of each sequence."""
    h, hk, d, scaled = c["heads"], c["kv_heads"], c["head_dim"], c["kind"] == "append_scaled"
    seqs = [i for i, (_, n) in enumerate(runs) for _ in range(n)]
    positions = [p + j for p, n in runs for j in range(n)]
    pad = c.get("padding", 0)
    t = len(seqs) + pad
    st["token_seqs"], st["positions"] = _i32(seqs + [-1] * pad), _i32(positions + [0] * pad)
    st["rope"] = _rope(max(positions) + 1, c["rotary"]) if c["rotary"] else None
    q, kv = torch.randn(t, h, d, generator=g, device="cuda"), _kv_values(g, t, hk, d)
    if scaled:
        st.update(q_in=q.to(torch.bfloat16).view(t, h * d), kv=kv.to(torch.bfloat16).view(t, hk * 2 * d), q_scale=_new(torch.float32, t, h))
    else:
        st.update(q_in=_codes(q).view(t, h * d), kv=_codes(kv).view(t, hk * 2 * d))
    st["q"] = _new(torch.int8, t, h * d)
    st["kv_out"] = _new(torch.int8, t, hk * 2 * d) if c.get("kv_out") else None


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    kind, b, h, hk, d = c["kind"], c["seqs"], c["heads"], c["kv_heads"], c["head_dim"]
    st = dict(case=dict(c))
    if kind.startswith("append"):
        runs = _tokens(c)
        ends = [p + n for p, n in runs]
    else:
        lens = _lens(c)
        runs, ends = [(n, 1) for n in lens], [n + c["new"] for n in lens]   # the new tokens' keys are in the cache
        st["kv_lens"] = _i32(lens)
    st["table"], n_pages = _page_table(g, c["page"], ends)
    st["pages"], st["scales"] = _pool(c, g, n_pages)
    if kind.startswith("append") or kind == "step":
        _prepare_append(c, g, st, runs)
    if not kind.startswith("append"):
        rows = b * c["new"]
        if kind == "decode_scaled":
            x = torch.randn(rows, h, d, generator=g, device="cuda")
            st["q_scale"] = x.abs().amax(-1).div_(127.0)
            st["q"] = x.div_(st["q_scale"].unsqueeze(-1)).round_().to(torch.int8).view(rows, h * d)
        elif kind == "decode":
            st["q"] = _codes(torch.randn(rows, h * d, generator=g, device="cuda"))
        st["sink_k"] = _codes(_unit_heads(torch.randn(h, d, generator=g, device="cuda")))
        st["sink_v"] = _codes(torch.randn(h, d, generator=g, device="cuda").mul_(1.3))
        st["temp"] = (0.5 + torch.rand(h, generator=g, device="cuda")).float()
        st["out"] = _new(torch.int8 if kind == "step" else torch.bfloat16, rows, h * d)
        st["l"] = _new(torch.float32, rows, h)
    if own:
        from x17ai_b200 import kernels as K
        st["kern"] = K.PagedAttnKernel(K.PagedConfig(h, hk, d, c["page"], h * d, 2 * hk * d, h * d, c.get("rotary", 0), c.get("adjacent", False)))
        _stream()
    torch.cuda.synchronize()   # torch made the inputs on its default stream
    return st


# ---- one pass ----------------------------------------------------------------------------------------

def run(st):
    kind = st["case"]["kind"]
    if own:
        return _run_own(st, kind)
    if kind == "append":
        return _plain_append(st)
    if kind == "append_scaled":
        return _plain_append_scaled(st)
    if kind == "step":
        new = _plain_append(st)
        out, l = _plain_attention(st, new["q"])
        return {**new, "out": out.mul(8.0).round().clamp(-127, 127).mul(SINK_SCALE).to(torch.bfloat16), "l": l}
    out, l = _plain_attention(st, st["q"])
    return {"out": out.to(torch.bfloat16), "l": l}


def _run_own(st, kind):
    c, kern, (torch_stream, s) = st["case"], st["kern"], _stream()
    if kind == "append":
        kern.append(s, st["q_in"], st["kv"], st["token_seqs"], st["positions"], st["table"], st["pages"], st["q"], st["rope"], st["kv_out"])
        return {"pages": st["pages"], "q": st["q"], "kv_out": st["kv_out"]}
    if kind == "append_scaled":
        kern.append_scaled(s, st["q_in"], st["kv"], st["token_seqs"], st["positions"], st["table"], st["pages"], st["scales"], st["q"],
                           st["q_scale"], st["rope"])
        return {"pages": st["pages"], "scales": st["scales"], "q": st["q"], "q_scale": st["q_scale"]}
    if kind == "step":
        kern.append(s, st["q_in"], st["kv"], st["token_seqs"], st["positions"], st["table"], st["pages"], st["q"], st["rope"])
        kern.decode(s, st["q"], st["pages"], st["table"], st["kv_lens"], st["sink_k"], st["sink_v"], st["temp"], st["out"], st["l"],
                    c["window"])
        with torch.cuda.stream(torch_stream):
            values = st["out"].to(torch.bfloat16).mul_(SINK_SCALE)
        return {"pages": st["pages"], "q": st["q"], "out": values, "l": st["l"], "kv_out": None}
    if kind == "decode_scaled":
        kern.decode_scaled(s, st["q"], st["q_scale"], st["pages"], st["scales"], st["table"], st["kv_lens"], st["sink_k"], st["sink_v"],
                           st["temp"], st["out"], st["l"], c["window"])
    else:
        kern.decode(s, st["q"], st["pages"], st["table"], st["kv_lens"], st["sink_k"], st["sink_v"], st["temp"], st["out"], st["l"],
                    c["window"])
    return {"out": st["out"], "l": st["l"]}


def _rows(st):
    """(tokens that are no padding, their pages, their places in them)"""
    t = (st["token_seqs"] >= 0).nonzero().squeeze(1)
    seq, pos, page = st["token_seqs"][t].long(), st["positions"][t].long(), st["case"]["page"]
    return t, st["table"][seq, pos // page].long(), pos % page


def _pairs(x, rotary, adjacent):
    """The rotated part of heads [.., D] as (x, y), and the rest."""
    r, rest = x[..., :rotary], x[..., rotary:]
    return (r[..., 0::2], r[..., 1::2], rest) if adjacent else (r[..., :rotary // 2], r[..., rotary // 2:], rest)


def _unpair(x, y, rest, adjacent):
    r = torch.stack((x, y), dim=-1).flatten(-2) if adjacent else torch.cat((x, y), dim=-1)
    return torch.cat((r, rest), dim=-1)


def _rotated_codes(c, rope, x):
    """int8 heads [T, H, D] at their table rows [T, R / 2, 2]: products and sums in 32-bit integers."""
    if rope is None:
        return x
    a, b, rest = _pairs(x, c["rotary"], c["adjacent"])
    a, b, cs = a.int(), b.int(), rope.int().unsqueeze(1)
    cos, sin = cs[..., 0], cs[..., 1]
    turn = lambda v: ((v + ROPE_ONE // 2) >> 14).clamp(-127, 127).to(torch.int8)
    return _unpair(turn(a * cos - b * sin), turn(a * sin + b * cos), rest, c["adjacent"])


def _plain_append(st):
    c = st["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    t, page, slot = _rows(st)
    rope = None if st["rope"] is None else st["rope"][st["positions"][t].long()]
    st["q"][t] = _rotated_codes(c, rope, st["q_in"][t].view(-1, h, d)).flatten(1)
    kv = st["kv"][t].view(-1, hk, 2, d)
    kv = torch.stack((_rotated_codes(c, rope, kv[:, :, 0]), kv[:, :, 1]), dim=2)
    st["pages"][page, :, slot] = kv.flatten(2)
    if st["kv_out"] is not None:
        st["kv_out"][t] = kv.flatten(1)
    return {"pages": st["pages"], "q": st["q"], "kv_out": st["kv_out"]}


def _quantised(x):
    """Heads [.., D] in f32 as codes and scales: scale = absmax / 127, code = x * (127 / absmax)."""
    top = x.abs().amax(-1, keepdim=True)
    live = top > TINY
    inv = torch.where(live, torch.full_like(top, 127.0) / top, 0.0)
    return x.mul(inv).round().clamp(-127, 127).to(torch.int8), torch.where(live, top * (1.0 / 127.0), 0.0).squeeze(-1)


def _rotated_values(c, rope, x):
    if rope is None:
        return x
    a, b, rest = _pairs(x, c["rotary"], c["adjacent"])
    cs = rope.float().mul(1.0 / ROPE_ONE).unsqueeze(1)
    cos, sin = cs[..., 0], cs[..., 1]
    return _unpair(a * cos - b * sin, a * sin + b * cos, rest, c["adjacent"])


def _plain_append_scaled(st):
    c = st["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    t, page, slot = _rows(st)
    rope = None if st["rope"] is None else st["rope"][st["positions"][t].long()]
    q, q_scale = _quantised(_rotated_values(c, rope, st["q_in"][t].float().view(-1, h, d)))
    st["q"][t], st["q_scale"][t] = q.flatten(1), q_scale
    kv = st["kv"][t].float().view(-1, hk, 2, d)
    kv, scale = _quantised(torch.stack((_rotated_values(c, rope, kv[:, :, 0]), kv[:, :, 1]), dim=2))
    st["pages"][page, :, slot] = kv.flatten(2)
    st["scales"][page, :, slot] = scale
    return {"pages": st["pages"], "scales": st["scales"], "q": st["q"], "q_scale": st["q_scale"]}


def _plain_attention(st, q):
    """Values in f32 [B new, H D] and L; a row of the products is one query head of one new token."""
    c = st["case"]
    b, new, h, hk, d, page = c["seqs"], c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    g, n = h // hk, st["table"].shape[1] * page
    by_key_head = lambda t: t.view(b, new, hk, g, -1).transpose(1, 2).reshape(b, hk, new * g, -1)
    at = st["table"].clamp(min=0).long()
    kv = st["pages"][at].transpose(1, 2).reshape(b, hk, n, 2 * d).float()
    q = by_key_head(q.float())
    if st["scales"] is None:
        q_scale, k_scale, v_scale = SINK_SCALE, SINK_SCALE, SINK_SCALE
    else:
        scales = st["scales"][at].transpose(1, 2).reshape(b, hk, 1, n, 2)
        q_scale, k_scale, v_scale = by_key_head(st["q_scale"]), scales[..., 0], scales[..., 1]
    lens = (st["kv_lens"].view(b, 1) + torch.arange(new, device=q.device)).repeat_interleave(g, 1).view(b, 1, new * g, 1)
    seen = lens if c["window"] == 0 else lens.clamp(max=c["window"])
    head = lambda t: t.view(1, hk, 1, g, -1).expand(b, hk, new, g, -1).reshape(b, hk, new * g, -1)
    temp = (seen.double() + 4).log2().mul(d ** -0.5).float() * head(st["temp"])
    x = (q @ kv[..., :d].transpose(2, 3)) * (q_scale * k_scale) * temp
    key = torch.arange(n, device=x.device)
    x = torch.where((key < lens) & (key >= lens - seen), x, -math.inf)
    sink = (q * head(st["sink_k"].float())).sum(-1, keepdim=True) * (q_scale * SINK_SCALE) * temp
    top = torch.maximum(x.amax(-1, keepdim=True), sink)
    p, p_sink = torch.exp2(x - top), torch.exp2(sink - top)
    total = p.sum(-1, keepdim=True) + p_sink
    weight = torch.where(p > 0, p * v_scale, 0.0)
    out = (weight @ kv[..., d:] + p_sink * (head(st["sink_v"].float()) * SINK_SCALE)) / total
    by_token = lambda t: t.view(b, hk, new, g, -1).transpose(1, 2).reshape(b * new, -1)
    return by_token(out), by_token(total.mul(255.0).log2() + top)


# ---- the definition in 64 bits -------------------------------------------------------------------------

def _exact_attention(st, q):
    c = st["case"]
    h, hk, d, page, w = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["window"]
    outs, ls = [], []
    for i in range(c["seqs"] * c["new"]):
        seq = i // c["new"]
        n = _lens(c)[seq] + i % c["new"]
        first = max(0, n - w) if w else 0
        j = torch.arange(first, n, device="cuda")
        where, slot = st["table"][seq, j // page].long(), j % page
        rows = st["pages"][where, :, slot].double().view(-1, hk, 2, d)
        if st["scales"] is None:
            rows, qs = rows / 8, torch.full((h,), 0.125, dtype=torch.float64, device="cuda")
        else:
            rows, qs = rows * st["scales"][where, :, slot].double().unsqueeze(-1), st["q_scale"][i].double()
        factor = qs * st["temp"].double() * math.log2(n - first + 4) / math.sqrt(d)
        query = q[i].double().view(h, d) * factor.unsqueeze(1)
        outs.append([])
        for k in range(hk):
            mine = slice(k * (h // hk), (k + 1) * (h // hk))
            scores = torch.cat((rows[:, k, 0] @ query[mine].t(), (query[mine] * st["sink_k"][mine].double() / 8).sum(1).unsqueeze(0)))
            lse = torch.logsumexp(scores * math.log(2.0), 0)
            p = torch.exp(scores * math.log(2.0) - lse)
            outs[-1].append(p[:-1].t() @ rows[:, k, 1] + p[-1].unsqueeze(1) * st["sink_v"][mine].double() / 8)
            ls.append(lse / math.log(2.0) + math.log2(255.0))
        outs[-1] = torch.cat(outs[-1]).flatten()
    return torch.stack(outs), torch.cat(ls).view(-1, h)


def _turned(c, rope, x):
    """x [T, H, D] in 64 bits as complex numbers times the table's."""
    r = c["rotary"]
    if r == 0:
        return x
    z = torch.view_as_complex(x[..., :r].unflatten(-1, (r // 2, 2) if c["adjacent"] else (2, r // 2)).movedim(-1 if c["adjacent"] else -2, -1)
                              .contiguous())
    z = torch.view_as_real(z * torch.view_as_complex(rope.double() / ROPE_ONE).unsqueeze(1))
    return torch.cat((z.flatten(-2) if c["adjacent"] else z.transpose(-1, -2).flatten(-2), x[..., r:]), dim=-1)


def exact(case, seed):
    c, st = case, prepare(case, seed)
    kind, h, hk, d = c["kind"], c["heads"], c["kv_heads"], c["head_dim"]
    if kind.startswith("decode"):
        out, l = _exact_attention(st, st["q"])
        return {"out": out, "l": l}
    rope = None if st["rope"] is None else st["rope"][st["positions"].long()]
    if kind == "append":
        return None   # whole numbers only
    if kind == "step":
        q = torch.floor(_turned(c, rope, st["q_in"].view(-1, h, d).double()) + 0.5).clamp(-127, 127)
        if c["rotary"] == 0:
            q = st["q_in"].view(-1, h, d).double()
        else:
            q[..., c["rotary"]:] = st["q_in"].view(-1, h, d)[..., c["rotary"]:].double()
        out, l = _exact_attention(st, q.flatten(1))   # the new token's own key is not among those it sees
        return {"pages": None, "q": None, "kv_out": None, "out": (out * 8).round().clamp(-127, 127) / 8, "l": l}
    scales, q_scale = st["scales"].double(), st["q_scale"].double()
    top_q = _turned(c, rope, st["q_in"].double().view(-1, h, d)).abs().amax(-1) / 127
    kv = st["kv"].double().view(-1, hk, 2, d)
    top_kv = torch.stack((_turned(c, rope, kv[:, :, 0]).abs().amax(-1), kv[:, :, 1].abs().amax(-1)), dim=-1) / 127
    for i, (s, p) in enumerate(zip(st["token_seqs"].tolist(), st["positions"].tolist())):
        if s < 0:
            break   # padding comes last
    else:
        i += 1
    seq, pos = st["token_seqs"][:i].long(), st["positions"][:i].long()
    scales[st["table"][seq, pos // c["page"]].long(), :, pos % c["page"]] = top_kv[:i]
    q_scale[:i] = top_q[:i]
    return {"pages": None, "scales": scales, "q": None, "q_scale": q_scale}


# ---- what a pass cannot do without ---------------------------------------------------------------------

def work(case):
    c = case
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    scaled = c["kind"].endswith("scaled")
    nbytes, flops = 0.0, 0.0
    if c["kind"].startswith("append") or c["kind"] == "step":
        t = c["tokens"] if "tokens" in c else c["seqs"]
        values = t * (h + 2 * hk) * d
        nbytes += values * (3 if scaled else 2) + (4 * t * (h + 2 * hk) if scaled else 0) + (t * 2 * hk * d if c.get("kv_out") else 0)
        nbytes += t * (12 + 2 * c["rotary"])            # sequence, position, page, and the table's row
        flops += 3.0 * t * (h + hk) * c["rotary"] + (2.0 * values if scaled else 0.0)
    if not c["kind"].startswith("append"):
        lens = _lens(c)
        # all new tokens of a sequence read the same keys, each but the first a few more
        seen = [[n + i if c["window"] == 0 else min(n + i, c["window"]) for i in range(c["new"])] for n in lens]
        keys, rows = sum(s[-1] for s in seen), c["seqs"] * c["new"]
        nbytes += keys * hk * (2 * d + (8 if scaled else 0)) + rows * h * (3 * d + 4 + (4 if scaled else 0)) + 4 * keys // c["page"]
        flops += 4.0 * d * h * (sum(map(sum, seen)) + rows)
    return {"bytes": float(nbytes), "flops": flops}

"""Measured cases of the 8-bit block-scaled cache and of the operators around it.

Four operators, the way a decoder layer uses them:

    norm_rope  q and k of a batch of tokens: RMS norm of every head, rotation at the token's position     er_qk_norm_rope
    append     k (normed, rotated) and v of new tokens into 8-bit pages with one scale per block          er_kv8_append
    decode     attention of one or a few new tokens per sequence over such pages                          er_kv8_attention_decode
    prefill    attention of a ragged batch of prompts or prompt chunks over such pages                    er_kv8_attention_prefill

`run` computes them with elementary torch operations, or (`own`) with the framework's kernels; `exact` is the definition in 64 bits.
"""
import math
import random

import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one token of a small model (16 query heads, 8 kv heads), activations in float32 as the step calls take them: latency
        dict(name="norm_rope_1", op="norm_rope", tokens=1, heads=16, kv_heads=8, dim=128, partial=1.0, dtype="float32", norm=True, theta=1e6, packed=False, far=4096),
        # an odd number of tokens, half-rotated heads of 64, rows cut out of one packed projection
        dict(name="norm_rope_777_packed", op="norm_rope", tokens=777, heads=12, kv_heads=4, dim=64, partial=0.5, dtype="float16", norm=True, theta=1e4, packed=True, far=131072),
        # a prompt step of 16 sequences x 2048 tokens (32 query heads, 8 kv heads)
        dict(name="norm_rope_32768", op="norm_rope", tokens=32768, heads=32, kv_heads=8, dim=128, partial=1.0, dtype="bfloat16", norm=True, theta=5e5, packed=True, far=131072),
        # a decode step of one sequence: one row into a block that holds rows already
        dict(name="append_1", op="append", seqs=1, new_lo=1, new_hi=1, old_lo=4090, old_hi=4090, kv_heads=8, dim=128, page=16, block=16, format="e4m3", dtype="float32", norm=True, theta=1e6, lens=3),
        # a decode step of 64 sequences
        dict(name="append_64", op="append", seqs=64, new_lo=1, new_hi=1, old_lo=1024, old_hi=2048, kv_heads=8, dim=128, page=16, block=16, format="e4m3", dtype="bfloat16", norm=False, theta=5e5, lens=2),
        # a prompt step of 16 sequences x 2048 tokens, each behind an odd number of earlier rows
        dict(name="append_16x2048", op="append", seqs=16, new_lo=2048, new_hi=2048, old_lo=0, old_hi=300, kv_heads=8, dim=128, page=64, block=32, format="e4m3", dtype="bfloat16", norm=True, theta=1e6, lens=4),
        # one sequence, short context, float32 activations: latency
        dict(name="decode_1x4097", op="decode", seqs=1, q_len=1, old_lo=4096, old_hi=4096, heads=16, kv_heads=8, dim=128, page=16, block=16, format="e4m3", dtype="float32", window=0, lens=5),
        # batched serving: 64 sequences of 1024 to 16384 rows
        dict(name="decode_64_ragged", op="decode", seqs=64, q_len=1, old_lo=1024, old_hi=16384, heads=32, kv_heads=8, dim=128, page=16, block=16, format="e4m3", dtype="bfloat16", window=0, lens=2),
        # one long context, the work of a row split over the whole GPU
        dict(name="decode_1x131072", op="decode", seqs=1, q_len=1, old_lo=131071, old_hi=131071, heads=32, kv_heads=8, dim=128, page=64, block=64, format="int8", dtype="float16", window=0, lens=6),
        # one short prompt: latency
        dict(name="prefill_100", op="prefill", seqs=1, new_lo=100, new_hi=100, old_lo=0, old_hi=0, heads=16, kv_heads=8, dim=128, page=16, block=16, format="e4m3", dtype="bfloat16", window=0, lens=7),
        # eight prompts of different odd lengths in one call
        dict(name="prefill_8_ragged", op="prefill", seqs=8, new_lo=17, new_hi=2048, old_lo=0, old_hi=0, heads=32, kv_heads=8, dim=128, page=16, block=16, format="e4m3", dtype="bfloat16", window=0, lens=8),
        # a chunk of 2048 tokens of a long prompt
        dict(name="prefill_2048_at_32768", op="prefill", seqs=1, new_lo=2048, new_hi=2048, old_lo=30720, old_hi=30720, heads=32, kv_heads=8, dim=128, page=64, block=64, format="int8", dtype="float16", window=0, lens=9),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "decode", "prefill"])
    kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16]), rng.choice([64, 128, 128])
    kv_heads = min(kv_heads, 32 // group if group <= 8 else 2)
    page = rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64, 128) if page % b == 0])
    cache = dict(kv_heads=kv_heads, dim=dim, page=page, block=block, format=rng.choice(["e4m3", "int8"]), lens=rng.randrange(1 << 20))
    theta = rng.choice([1e4, 5e5, 1e6])
    if op == "norm_rope":
        return dict(op=op, tokens=_log_int(rng, 1, 16384), heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice([64, 80, 128, 256]), partial=rng.choice([1.0, 1.0, 0.5, 0.25]),
                    dtype=rng.choice(list(_TYPES)), norm=rng.random() < 0.75, theta=theta, packed=rng.random() < 0.5, far=_log_int(rng, 64, 1 << 20))
    if op == "append":
        new = _log_int(rng, 1, 8192)
        seqs = _log_int(rng, 1, max(1, min(64, 16384 // new)))
        old = _log_int(rng, 1, 1000)
        return dict(op=op, seqs=seqs, new_lo=max(1, new // 3), new_hi=new, old_lo=0, old_hi=old, dtype=rng.choice(list(_TYPES)), norm=rng.random() < 0.5, theta=theta, **cache)
    if op == "decode":
        old = _log_int(rng, 1, 65536)
        seqs = _log_int(rng, 1, max(1, min(64, (64 * 8192) // old)))
        return dict(op=op, seqs=seqs, q_len=rng.choice([1, 1, 1, 2, 4]), old_lo=old // 4, old_hi=old, heads=kv_heads * group, dtype=rng.choice(list(_TYPES)),
                    window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]), **cache)
    new = _log_int(rng, 1, 2048)
    seqs = _log_int(rng, 1, max(1, min(16, 4096 // new)))
    old = _log_int(rng, 1, 8192)
    return dict(op=op, seqs=seqs, new_lo=max(1, new // 4), new_hi=new, old_lo=0, old_hi=rng.choice([0, old]), heads=kv_heads * group, dtype=rng.choice(["float16", "bfloat16"]),
                window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]), **cache)


def _lengths(case):
    """(rows that each sequence holds before the call, new tokens of each), from the case alone."""
    rng = random.Random(case["lens"])
    n = case["seqs"]
    old = [rng.randint(case["old_lo"], case["old_hi"]) for _ in range(n)]
    new = [case["q_len"]] * n if case["op"] == "decode" else [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
    return old, new


def work(case):
    es = 4 if case["dtype"] == "float32" else 2
    d, hk = case["dim"], case["kv_heads"]
    if case["op"] == "norm_rope":
        rows = case["tokens"] * (case["heads"] + hk)
        return {"bytes": 2 * rows * d * es + 4 * case["tokens"] + 8 * d, "flops": 8 * rows * d}
    old, new = _lengths(case)
    if case["op"] == "append":
        rows = sum(new) * hk
        blocks = sum(-(-(o + n) // case["block"]) - o // case["block"] for o, n in zip(old, new)) * hk
        return {"bytes": 2 * rows * d * (es + 1) + 8 * blocks, "flops": 12 * rows * d}
    seen, pairs = 0, 0   # rows that some query sees, (query, row) pairs
    for o, n in zip(old, new):
        w = case["window"] or (o + n)
        seen += min(o + n, n - 1 + w)
        pairs += sum(min(o + i + 1, w) for i in range(n))
    h = case["heads"]
    return {"bytes": 2 * seen * hk * (d + 4 / case["block"]) + 2 * sum(new) * h * d * es, "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _quantise_blocks(x, fmt):
    """[..., block, dim] float32 -> (codes as uint8, scales [...])."""
    amax = x.abs().amax(dim=(-1, -2))
    s = _need(amax, fmt)
    inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))[..., None, None]
    return _encode(x * inv, fmt), s


def _need(amax, fmt):
    """The scale of a block whose largest magnitude is amax: e4m3 the smallest power of two with amax / scale <= 448, int8 amax / 127."""
    if fmt == "int8":
        return amax / 127.0
    m, e = torch.frexp(amax)   # 448 = 0.875 * 2^9; a division by 448 would round magnitudes that need no rounding
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), torch.where(m > 0.875, e - 8, e - 9)), torch.zeros_like(amax))


def _encode(x, fmt):
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _decode(codes, fmt, dtype=torch.float32):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).to(dtype)


def _pages(case, g, total_pages):
    """Pages of rows as earlier steps left them: N(0, 1) rows with a few strong channels in the keys."""
    hk, d, page, block = case["kv_heads"], case["dim"], case["page"], case["block"]
    out = []
    for side in range(2):
        codes = torch.empty(total_pages, hk, page, d, dtype=torch.uint8, device="cuda")
        scales = torch.empty(total_pages, hk, page // block, device="cuda")
        loud = torch.where(torch.rand(d, generator=g, device="cuda") < 0.03, 8.0, 1.0) if side == 0 else torch.ones(d, device="cuda")
        step = max(1, (64 << 20) // (hk * page * d))
        for p in range(0, total_pages, step):
            n = min(step, total_pages - p)
            c, s = _quantise_blocks(torch.randn(n, hk, page // block, block, d, generator=g, device="cuda") * loud, case["format"])
            codes[p:p + n] = c.view(n, hk, page, d)
            scales[p:p + n] = s
        out += [codes, scales]
    return out


def prepare(case, seed):
    g = _gen(seed)
    dt, d, hk = _TYPES[case["dtype"]], case["dim"], case["kv_heads"]
    st = {"case": case}
    if case["op"] == "norm_rope":
        t, h = case["tokens"], case["heads"]
        if case["packed"]:   # q and k are parts of one projection's rows, with the values behind them
            rows = torch.randn(t, h + 2 * hk, d, generator=g, device="cuda").mul_(1.5).to(dt)
            st["q"], st["k"] = rows[:, :h], rows[:, h:h + hk]
        else:
            st["q"], st["k"] = (torch.randn(t, n, d, generator=g, device="cuda").mul_(1.5).to(dt) for n in (h, hk))
        st["pos"] = torch.randint(0, case["far"], (t,), generator=g, device="cuda", dtype=torch.int32)
        st["qw"], st["kw"] = (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda") for _ in range(2)) if case["norm"] else (None, None)
        st["q_out"], st["k_out"] = (torch.empty(t, n, d, device="cuda", dtype=dt) for n in (h, hk))
        return st
    old, new = _lengths(case)
    page = case["page"]
    need = [-(-(o + n) // page) for o, n in zip(old, new)]
    total = sum(need)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((case["seqs"], max(need)), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    st["table"] = table.cuda()
    st["lens"] = torch.tensor([o + n for o, n in zip(old, new)], dtype=torch.int32, device="cuda")
    st["starts"] = torch.tensor([sum(new[:s]) for s in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    st["new"], st["old"] = new, old
    st["keys"], st["key_scales"], st["values"], st["value_scales"] = _pages(case, g, total)
    t = sum(new)
    if case["op"] == "append":
        rows = torch.randn(t, 2 * hk, d, generator=g, device="cuda").mul_(1.2).to(dt)
        st["k"], st["v"] = rows[:, :hk], rows[:, hk:]
        st["kw"] = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda") if case["norm"] else None
    else:
        st["q"] = torch.randn(t, case["heads"], d, generator=g, device="cuda").to(dt)
        st["out"] = torch.empty(t, case["heads"], d, device="cuda", dtype=dt)
    if own:   # the handle that a program keeps over its pages
        import edgerunner_b200 as er
        st["cache"] = er.BlockScaledKVCache.from_tensors(st["keys"], st["values"], st["key_scales"], st["value_scales"], er.BlockScaledFormat[case["format"]])
    return st


# ------------------------------------------------------------------------------------------------------------- plain forms

def _norm_rope(x, weight, pos, theta, partial):
    """x [tokens, heads, dim] in float32; pairs (i, i + dim / 2), the first dim / 2 * partial of them rotated."""
    half = x.shape[-1] // 2
    n = int(half * partial)
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + _EPS) * weight
    angle = pos.double()[:, None] * torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device), -torch.arange(n, device=x.device, dtype=torch.float64) / half)
    c, s = (f.to(x.dtype)[:, None, :] for f in (angle.cos(), angle.sin()))
    a, b = x[..., :n], x[..., half:half + n]
    return torch.cat([a * c - b * s, x[..., n:half], a * s + b * c, x[..., half + n:]], dim=-1)


def _plain_append(st):
    case = st["case"]
    page, block, fmt, hk, d = case["page"], case["block"], case["format"], case["kv_heads"], case["dim"]
    t, per = st["k"].shape[0], page // block
    seq = torch.searchsorted(st["starts"][1:], torch.arange(t, device="cuda", dtype=torch.int32), right=True)
    count = st["starts"][1:] - st["starts"][:-1]
    first = st["lens"] - count                                           # first new position of each sequence
    pos = first[seq] + torch.arange(t, device="cuda", dtype=torch.int32) - st["starts"][:-1][seq]
    row_page, slot = st["table"][seq, pos // page].long(), (pos % page).long()
    blk = row_page * per + slot // block                                 # block of each new row
    part_page = st["table"][torch.arange(len(first), device="cuda"), first // page].long()
    part = part_page * per + (first % page) // block                     # the block that each sequence's first new row falls into
    partial = (first % block) != 0                                       # ... and whether it holds earlier rows
    heads = torch.arange(hk, device="cuda")
    k = _norm_rope(st["k"].float(), st["kw"], pos, case["theta"], 1.0)
    out = []
    for x, codes, scales in ((k, st["keys"], st["key_scales"]), (st["v"].float(), st["values"], st["value_scales"])):
        amax = torch.full((codes.shape[0] * per, hk), -1.0, device="cuda")
        amax.scatter_reduce_(0, blk[:, None].expand(-1, hk), x.abs().amax(dim=-1), "amax")
        s_old = scales.transpose(1, 2).reshape(-1, hk)                   # [page * per, heads]
        s_new = torch.where(amax >= 0, _need(amax.clamp(min=0), fmt), s_old)
        kept = torch.where(partial[:, None], s_old[part], torch.zeros_like(s_old[part]))
        s_new[part] = torch.maximum(s_new[part], kept)
        ratio = torch.where(partial[:, None] & (s_new[part] > 0), s_old[part] / s_new[part], torch.ones_like(kept))
        blocks = codes.view(codes.shape[0], hk, per, block, d)
        at = (part_page[:, None], heads[None], ((first % page) // block).long()[:, None])
        earlier = (torch.arange(block, device="cuda") < (first % block)[:, None])[:, None, :, None]
        blocks[at] = torch.where((ratio < 1)[..., None, None] & earlier, _encode(_decode(blocks[at], fmt) * ratio[..., None, None], fmt), blocks[at])
        inv = torch.where(s_new > 0, 1.0 / s_new, torch.zeros_like(s_new))[blk]
        codes[row_page[:, None], heads[None], slot[:, None]] = _encode(x * inv[..., None], fmt)
        scales.copy_(s_new.view(-1, per, hk).transpose(1, 2))
        out += [_values(codes, fmt), scales]
    return dict(zip(("keys", "key_scales", "values", "value_scales"), out))


def _values(codes, fmt):
    """Codes as the numbers that they stand for, before the block's scale."""
    return codes.view(torch.int8).to(torch.float16) if fmt == "int8" else codes.view(torch.float8_e4m3fn)


def _plain_attention(st):
    case = st["case"]
    block, fmt, hk, d, h = case["block"], case["format"], case["kv_heads"], case["dim"], case["heads"]
    table, n = st["table"].clamp(min=0).long(), case["seqs"]
    side = lambda codes, scales: (_decode(codes[table], fmt).view(n, table.shape[1], hk, -1, block, d) * scales[table][..., None, None]).transpose(1, 2).reshape(n, hk, -1, d)  # noqa: E731
    k, v = side(st["keys"], st["key_scales"]), side(st["values"], st["value_scales"])
    rows = max(st["new"])                                                # queries of each sequence, padded to the longest
    i = torch.arange(rows, device="cuda")
    count = (st["starts"][1:] - st["starts"][:-1])[:, None]
    q = st["q"].float()[(st["starts"][:-1][:, None] + i).clamp(max=st["q"].shape[0] - 1).long()]
    q = q.view(n, rows, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    s = torch.matmul(q, k.transpose(-1, -2)).div_(math.sqrt(d)).view(n, hk, h // hk, rows, -1)
    pos = (st["lens"][:, None] - count + i)[:, None, None, :, None]
    at = torch.arange(k.shape[2], device="cuda")
    hidden = (at > pos) | (at >= st["lens"][:, None, None, None, None])
    if case["window"]:
        hidden = hidden | (at <= pos - case["window"])
    s.masked_fill_(hidden, -math.inf)
    s.sub_(s.amax(dim=-1, keepdim=True).clamp(min=-1e30)).exp_()
    s.div_(s.sum(dim=-1, keepdim=True).clamp(min=1e-30))
    o = torch.matmul(s.view(n, hk, -1, s.shape[-1]), v).view(n, h, rows, d).transpose(1, 2)
    return o[(i < count)].to(st["q"].dtype)


def run(state):
    case = state["case"]
    if case["op"] == "norm_rope":
        if own:
            import edgerunner_b200 as er
            er.QKNormRopeKernel().encode(state["q"], state["q_out"], state["pos"], k=state["k"], k_out=state["k_out"], q_norm_weight=state["qw"], k_norm_weight=state["kw"],
                                         rms_eps=_EPS, rope_theta=case["theta"], partial_rotary_factor=case["partial"])
            return {"q": state["q_out"], "k": state["k_out"]}
        return {n: _norm_rope(state[n].float(), state[n + "w"], state["pos"], case["theta"], case["partial"]).to(state[n].dtype) for n in ("q", "k")}
    if case["op"] == "append":
        if not own:
            return _plain_append(state)
        cache, fmt = state["cache"], case["format"]
        cache.append(state["k"], state["v"], state["table"], state["lens"], state["starts"], k_norm_weight=state["kw"], rms_eps=_EPS, rope_theta=case["theta"])
        return {"keys": _values(state["keys"], fmt), "key_scales": state["key_scales"], "values": _values(state["values"], fmt), "value_scales": state["value_scales"]}
    if not own:
        return _plain_attention(state)
    if case["op"] == "decode":
        return state["cache"].attention_decode(state["q"], state["table"], state["lens"], out=state["out"], query_len=case["q_len"], sliding_window=case["window"])
    return state["cache"].attention_prefill(state["q"], state["starts"], state["table"], state["lens"], out=state["out"], max_query_len=max(state["new"]), sliding_window=case["window"])


# ------------------------------------------------------------------------------------------------------------------- exact

def _exact_rotated(x, weight, pos, theta, partial):
    x = x.double()
    half = x.shape[-1] // 2
    if weight is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + _EPS) ** 0.5 * weight.double()
    for i in range(int(half * partial)):
        a = pos.double() * (1.0 / theta ** (i / half))
        turn = torch.polar(torch.ones_like(a), a)[:, None] * torch.complex(x[..., i], x[..., i + half])
        x[..., i], x[..., i + half] = turn.real, turn.imag
    return x


def _exact_append(st):
    case, out = st["case"], {}
    page, block, fmt = case["page"], case["block"], case["format"]
    pos = torch.cat([torch.arange(o, o + n) for o, n in zip(st["old"], st["new"])]).cuda()
    sides = {"key": _exact_rotated(st["k"], st["kw"], pos, case["theta"], 1.0), "value": st["v"].double()}
    bound = 448.0 if fmt == "e4m3" else 127.0
    for name, x in sides.items():
        codes, scales = _decode(st[name + "s"], fmt, torch.float64), st[name + "_scales"].double()
        for s, (o, n) in enumerate(zip(st["old"], st["new"])):
            rows = x[sum(st["new"][:s]):sum(st["new"][:s + 1])].transpose(0, 1)             # [heads, n, dim]
            lead = o % block                                                                # earlier rows of the first block
            count = -(-(lead + n) // block)
            full = torch.zeros(rows.shape[0], count * block, rows.shape[2], dtype=torch.float64, device="cuda")
            full[:, lead:lead + n] = rows
            full = full.view(rows.shape[0], count, block, -1)
            need = full.abs().amax(dim=(2, 3)) / torch.full((), bound, dtype=torch.float64, device="cuda")   # by a tensor: a true quotient
            if fmt == "e4m3":                                                                # the next power of two, itself where it is one
                mantissa, e = torch.frexp(need)
                need = torch.where(need > 0, torch.ldexp(torch.ones_like(need), torch.where(mantissa > 0.5, e, e - 1)), need)
            g = o // block + torch.arange(count, device="cuda")                              # block numbers along the sequence
            pg, b = st["table"][s].long()[g * block // page], g % (page // block)
            if lead:
                before = scales[pg[0], :, b[0]]
                need[:, 0] = torch.maximum(need[:, 0], before)
                view = codes.view(codes.shape[0], codes.shape[1], page // block, block, -1)
                full[:, 0, :lead] = view[pg[0], :, b[0], :lead] * before[:, None, None]
            y = full / torch.where(need > 0, need, torch.ones_like(need))[..., None, None]
            y = _decode(_encode(y.float(), fmt), fmt, torch.float64)
            stay = slice(0, lead + n - (count - 1) * block)                                  # rows behind the last one stay as they were
            view = codes.view(codes.shape[0], codes.shape[1], page // block, block, -1)
            for j in range(count):
                if j + 1 < count:
                    view[pg[j], :, b[j]] = y[:, j]
                else:
                    view[pg[j], :, b[j], stay] = y[:, j, stay]
            scales[pg, :, b] = need.transpose(0, 1)
        out[name + "s"], out[name + "_scales"] = codes, scales
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm_rope":
        return {n: _exact_rotated(st[n], st[n + "w"], st["pos"], case["theta"], case["partial"]) for n in ("q", "k")}
    if case["op"] == "append":
        return _exact_append(st)
    fmt, page, block, hk, d = case["format"], case["page"], case["block"], case["kv_heads"], case["dim"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s, (o, n) in enumerate(zip(st["old"], st["new"])):
        t = torch.arange(o + n, device="cuda")
        pg = st["table"][s].long()[t // page]
        at = sum(st["new"][:s])
        p = o + torch.arange(n, device="cuda")
        seen = t[None] <= p[:, None]
        if case["window"]:
            seen &= t[None] > p[:, None] - case["window"]
        for j in range(hk):
            k = _decode(st["keys"][pg, j, t % page], fmt, torch.float64) * st["key_scales"].double()[pg, j, t % page // block, None]
            v = _decode(st["values"][pg, j, t % page], fmt, torch.float64) * st["value_scales"].double()[pg, j, t % page // block, None]
            for i in range(j * (case["heads"] // hk), (j + 1) * (case["heads"] // hk)):
                w = (st["q"][at:at + n, i].double() @ k.T / d ** 0.5).masked_fill(~seen, -math.inf)
                out[at:at + n, i] = torch.softmax(w, dim=-1) @ v
    return out

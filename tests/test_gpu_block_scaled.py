"""The 8-bit block-scaled paged cache (append, decode and prefill attention) and the head norms with rotation, against 64-bit references.

Tolerances.  u(t) = finfo(t).eps / 2 is half a step of type t, relative to the value.
  norm + rotation: one rounding to t, plus float32 arithmetic on values up to the row's largest magnitude A: the norm factor (sum of squares,
    rsqrt: 4 steps), weight, sin / cos (2 steps each) and the turn (3 steps) stay under 16 u(float32) A.
  codes: half a step of the code, max(|x| 2^-4, 2^-10 scale) for E4M3, scale / 2 for int8, on values that are off by 16 u(float32) A themselves.
  attention, V = largest |value| that a query sees: float32 carries 22 bits of q and of the weights; a score of magnitude S is off by 2^-21 S' with S' =
    |q| |k| softmax_scale <= 40 here (2e-5), and the weights with it: 6e-5 V.  16-bit types round each weight to 11 bits, relative error 2^-11 of each
    and so of the mean, numerator only: 2^-11 V, plus u(t) of the output and the float32 terms above.
"""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def er():
    import edgerunner_b200 as er
    assert er.lib().er_device_count() > 0
    return er


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def dtype(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def half_step(torch, t):
    return torch.finfo(t).eps / 2


U32 = 2.0 ** -24


def gen(torch, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ref_norm_rope(torch, x, pos, weight, theta, scaling=1.0, partial=1.0, eps=1e-6):
    x = x.double()
    half = x.shape[-1] // 2
    n = int(half * partial)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    f = theta ** (-torch.arange(n, device=x.device, dtype=torch.float64) / half) / scaling
    ang = pos.double()[:, None] * f
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    y = x.clone()
    y[..., :n] = x[..., :n] * c - x[..., half:half + n] * s
    y[..., half:half + n] = x[..., :n] * s + x[..., half:half + n] * c
    return y


# ------------------------------------------------------------------------------------------------- head norms and rotation

@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens, heads, kv_heads, dim, partial, norm", [
    (1, 16, 8, 128, 1.0, True), (3, 5, 2, 64, 0.5, True), (37, 32, 8, 128, 1.0, False), (38, 1, 1, 256, 0.25, True), (129, 7, 1, 80, 1.0, True),
    (2049, 12, 4, 64, 1.0, True), (5, 3, 0, 16, 1.0, True), (2, 130, 2, 240, 0.3, True), (4, 4, 4, 48, 0.0, True)])
def test_norm_rope(er, torch, t, tokens, heads, kv_heads, dim, partial, norm):
    dt, g = dtype(torch, t), gen(torch, tokens + heads)
    rows = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g, device="cuda").mul(2).to(dt)     # q, k and v of one projection
    q, k = rows[:, :heads], rows[:, heads:heads + kv_heads] if kv_heads else None
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    qw, kw = (torch.randn(dim, generator=g, device="cuda") for _ in range(2)) if norm else (None, None)
    if heads == 5:
        qw = None                     # a norm for the keys only
    before = rows.clone()
    qo, ko = torch.empty(tokens, heads, dim, device="cuda", dtype=dt), torch.empty(tokens, kv_heads, dim, device="cuda", dtype=dt) if kv_heads else None
    er.QKNormRopeKernel().encode(q, qo, pos if partial > 0 else None, k=k, k_out=ko, q_norm_weight=qw, k_norm_weight=kw, rope_theta=5e5, rope_scaling=2.0,
                                 partial_rotary_factor=partial)
    assert torch.equal(rows, before)
    for x, y, w in ((q, qo, qw), (k, ko, kw)):
        if x is None:
            continue
        want = ref_norm_rope(torch, x, pos, w, 5e5, 2.0, partial)
        bound = half_step(torch, dt) * want.abs() + 16 * U32 * want.abs().amax(-1, keepdim=True) + (2.0 ** -25 if t == "f16" else 0)   # half a step of a float16 subnormal
        assert bool(((y.double() - want).abs() <= bound).all())
    # in place on the packed rows: the same bits, the values behind them untouched
    er.QKNormRopeKernel().encode(q, q, pos if partial > 0 else None, k=k, k_out=k, q_norm_weight=qw, k_norm_weight=kw, rope_theta=5e5, rope_scaling=2.0,
                                 partial_rotary_factor=partial)
    assert torch.equal(q, qo) and (k is None or torch.equal(k, ko)) and torch.equal(rows[:, heads + kv_heads:], before[:, heads + kv_heads:])


def test_norm_rope_rows_of_zeros_and_infinities(er, torch):
    x = torch.zeros(3, 2, 128, device="cuda")
    x[1, 1, 5] = math.inf
    y = torch.empty_like(x)
    er.QKNormRopeKernel().encode(x, y, torch.arange(3, device="cuda", dtype=torch.int32), q_norm_weight=torch.ones(128, device="cuda"))
    assert bool((y[0] == 0).all()) and bool((y[2] == 0).all()) and bool((y[1, 0] == 0).all()) and bool(torch.isnan(y[1, 1]).any())
    er.QKNormRopeKernel().encode(x[:0], y[:0], torch.arange(0, device="cuda", dtype=torch.int32))      # no tokens


# ------------------------------------------------------------------------------------------------------------------ append

def codes_of(torch, c, fmt):
    return c.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).to(torch.float64)


def make_cache(er, torch, fmt, pages, page, heads, dim, block, seed=1):
    """Pages full of bytes that are nobody's rows yet, the codes of E4M3's NaN among them, with scales to match."""
    g = gen(torch, seed)
    bytes_ = [torch.randint(0, 256, (pages, heads, page, dim), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    scales = [torch.rand(pages, heads, page // block, generator=g, device="cuda") for _ in range(2)]
    return er.BlockScaledKVCache.from_tensors(*bytes_, *scales, er.BlockScaledFormat[fmt])


def tables(torch, lens, page, pages, seed=3, extra=1):
    """A random page for every `page` rows; -1 behind them."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    out, at = torch.full((len(lens), max(need + [1]) + extra), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        out[s, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return out.cuda()


def ints(torch, x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def needed(torch, amax, fmt):
    if fmt == "int8":
        return amax / 127.0
    m, e = torch.frexp(amax)          # 448 = 0.875 * 2^9
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), torch.where(m > 0.875, e - 8, e - 9)), torch.zeros_like(amax))


def quantum(torch, x, scale, fmt):
    """Half a step of the code that stands for x."""
    return (scale / 2).expand_as(x) if fmt == "int8" else torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("t, dim, heads, page, block, old, new", [
    ("f32", 128, 8, 16, 16, [0], [1]), ("bf16", 128, 3, 32, 32, [5, 0, 31, 64], [1, 1, 1, 1]), ("f16", 64, 2, 64, 16, [0, 7, 100], [130, 1, 29]),
    ("f32", 64, 1, 128, 128, [3, 128, 250], [127, 300, 6]), ("bf16", 128, 5, 64, 64, [0, 63, 10, 200], [17, 2, 0, 64]),
    ("f16", 128, 8, 128, 32, [1000, 0], [1, 333]), ("bf16", 64, 9, 16, 16, [15, 16, 17], [2, 15, 1])])
def test_append(er, torch, fmt, t, dim, heads, page, block, old, new):
    dt, g = dtype(torch, t), gen(torch, 11)
    lens = [o + n for o, n in zip(old, new)]
    cache = make_cache(er, torch, fmt, sum(-(-n // page) for n in lens) + 2, page, heads, dim, block)
    table = tables(torch, lens, page, cache.num_pages)
    starts = ints(torch, [sum(new[:i]) for i in range(len(new) + 1)])
    rows = torch.randn(sum(new) + 3, 2 * heads, dim, generator=g, device="cuda").mul(3).to(dt)            # three tokens behind the last sequence
    rows[0, 0] = 0
    kw = 1 + 0.3 * torch.randn(dim, generator=g, device="cuda")
    for x, n in ((cache.key_scales, 0.02), (cache.value_scales, 0.02)):                                    # some blocks have to grow, some do not
        x.mul_(n * 2 if fmt == "int8" else n).add_(1e-4)
        if fmt == "e4m3":
            x.copy_(torch.exp2(torch.round(torch.log2(x))))
    before = [x.clone() for x in (cache.keys, cache.values, cache.key_scales, cache.value_scales)]
    one = all(n == 1 for n in new)
    k, v = rows[:sum(new) if one else None, :heads], rows[:sum(new) if one else None, heads:]
    cache.append(k, v, table, ints(torch, lens), None if one else starts, k_norm_weight=kw, rope_theta=1e6)
    assert cache.device_status() == 0
    pos = torch.cat([torch.arange(o, o + n) for o, n in zip(old, new)]).cuda()
    side = ((ref_norm_rope(torch, k[:sum(new)], pos, kw, 1e6), cache.keys, cache.key_scales, before[0], before[2], 16 * U32),
            (v[:sum(new)].double(), cache.values, cache.value_scales, before[1], before[3], 0.0))
    for x, codes, scales, codes0, scales0, off in side:
        got, was = codes_of(torch, codes, fmt), codes_of(torch, codes0, fmt)
        touched = torch.zeros(codes.shape[:3], dtype=torch.bool, device="cuda")                            # rows that may change
        fresh = torch.zeros_like(scales, dtype=torch.bool)
        for s, (o, n) in enumerate(zip(old, new)):
            first = sum(new[:s])
            for b in range(o // block, -(-(o + n) // block) if n else 0):
                lo, hi = max(o, b * block), min(o + n, (b + 1) * block)
                pg, at = int(table[s, b * block // page]), b * block % page
                mine = x[first + lo - o:first + hi - o].transpose(0, 1)                                    # [heads, rows, dim]
                amax = mine.abs().amax(dim=(1, 2))
                lead = lo - b * block
                need = needed(torch, amax, fmt)
                want = torch.maximum(need, scales0[pg, :, at // block].double()) if lead else need
                sc = scales[pg, :, at // block].double()
                assert bool(((sc - want).abs() <= 64 * U32 * want).all()), (s, b)
                fresh[pg, :, at // block] = True
                touched[pg, :, at:at + hi - b * block] = True
                err = (got[pg, :, at + lead:at + hi - b * block] * sc[:, None, None] - mine).abs()
                slack = off * amax[:, None, None]
                assert bool((err <= (quantum(torch, mine, sc[:, None, None], fmt) + slack) * (1 + 1e-5)).all()), (s, b)
                if lead:       # earlier rows: the same codes where the scale stayed, else re-encoded
                    then, now = was[pg, :, at:at + lead], got[pg, :, at:at + lead]
                    s0 = scales0[pg, :, at // block].double()
                    for h in range(heads):
                        if float(sc[h]) == float(s0[h]):
                            assert torch.equal(codes[pg, h, at:at + lead], codes0[pg, h, at:at + lead])
                        else:
                            fine = torch.isfinite(then[h])
                            e = (now[h] * sc[h] - then[h] * s0[h]).abs()[fine]
                            assert bool((e <= quantum(torch, then[h] * s0[h], sc[h], fmt)[fine] * (1 + 1e-5)).all())
        assert torch.equal(codes[~touched], codes0[~touched]) and torch.equal(scales[~fresh], scales0[~fresh])


def test_append_token_by_token_is_append_at_once_for_e4m3(er, torch):
    """Power-of-two scales: a block that grows step by step ends with the codes of one append, except codes that fell below the smallest step on the way."""
    g = gen(torch, 5)
    k, v = (torch.randn(40, 2, 128, generator=g, device="cuda") * torch.linspace(0.1, 30, 40, device="cuda")[:, None, None] for _ in range(2))
    a, b = (er.BlockScaledKVCache(3, 16, 2, 128) for _ in range(2))
    table = ints(torch, [[2, 0, 1]])
    a.append(k, v, table, ints(torch, [40]), ints(torch, [0, 40]))
    for i in range(40):
        b.append(k[i:i + 1], v[i:i + 1], table, ints(torch, [i + 1]))
    assert torch.equal(a.key_scales, b.key_scales) and torch.equal(a.value_scales, b.value_scales)
    for x, y, s in zip(a.decoded_rows([2, 0, 1], 40), b.decoded_rows([2, 0, 1], 40), (a.key_scales, a.value_scales)):
        smallest = s.repeat_interleave(16, dim=2)[[2, 0, 1]].transpose(1, 2).reshape(48, 2)[:40, :, None] * 2.0 ** -9
        assert bool(((x == y) | ((x - y).abs() <= smallest)).all())
        assert float((x == y).float().mean()) > 0.9


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_of_values_that_are_not_finite(er, torch, fmt):
    cache = er.BlockScaledKVCache(2, 32, 1, 64, er.BlockScaledFormat[fmt])
    k, v = torch.ones(32, 1, 64, device="cuda"), torch.ones(32, 1, 64, device="cuda")
    k[3, 0, 7], v[20, 0, 0] = math.nan, -math.inf
    v[:16] = 0
    cache.append(k, v, ints(torch, [[1]]), ints(torch, [32]), ints(torch, [0, 32]), partial_rotary_factor=0.0)
    dk, dv = cache.decoded_rows([1], 32)
    assert bool(torch.isnan(dk[:16]).all()) and bool((dk[16:] == 1).all())
    assert bool((dv[:16] == 0).all()) and float(cache.value_scales[1, 0, 0]) == 0.0 and bool(torch.isnan(dv[16:]).all())


def test_append_skips_what_has_no_page_and_says_so(er, torch):
    cache = make_cache(er, torch, "e4m3", 4, 16, 2, 128, 16)
    before = [x.clone() for x in (cache.keys, cache.values, cache.key_scales, cache.value_scales)]
    k = torch.randn(3, 2, 128, device="cuda")
    cache.append(k, k, ints(torch, [[-1], [99], [0]]), ints(torch, [1, 1, 17]))        # no page, a page that does not exist, behind the table
    assert cache.device_status() == -10
    cache.clear_device_status()
    cache.append(k, k, ints(torch, [[0], [1], [2]]), ints(torch, [0, 16, 3]), ints(torch, [0, 1, 5, 3]))   # before row 0; beyond the tokens; backwards
    assert cache.device_status() == -7
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.keys, cache.values, cache.key_scales, cache.value_scales)))


# --------------------------------------------------------------------------------------------------------------- attention

def fill(er, torch, fmt, lens, page, heads, dim, block, seed=2):
    """A cache whose sequences hold quantised rows, all other bytes being noise; its table, and the rows as float64."""
    g = gen(torch, seed)
    cache = make_cache(er, torch, fmt, sum(-(-n // page) for n in lens) + 2, page, heads, dim, block, seed)
    table = tables(torch, lens, page, cache.num_pages)
    total = sum(lens)
    k, v = (torch.randn(total, heads, dim, generator=g, device="cuda") * (0.2 + 4 * torch.rand(total, 1, 1, generator=g, device="cuda")) for _ in range(2))
    cache.append(k, v, table, ints(torch, lens), ints(torch, [sum(lens[:i]) for i in range(len(lens) + 1)]), partial_rotary_factor=0.0)
    rows = [tuple(x.double() for x in cache.decoded_rows([p for p in table[s].tolist() if p >= 0], n)) for s, n in enumerate(lens)]
    assert cache.device_status() == 0
    return cache, table, rows


def ref_attention(torch, q, k, v, len_, scale, window=0, hidden=None):
    """q [n, heads, dim] the newest n positions of len_ rows -> [n, heads, dim], and the largest |value| each query sees."""
    n, h, d = q.shape
    hk = k.shape[1]
    at, pos = torch.arange(len_, device="cuda"), torch.arange(len_ - n, len_, device="cuda")
    see = at[None] <= pos[:, None]
    if window:
        see &= at[None] > pos[:, None] - window
    if hidden is not None:
        see &= ~hidden[None]
    kk, vv = (x.repeat_interleave(h // hk, dim=1) for x in (k, v))
    s = torch.einsum("nhd,thd->hnt", q.double(), kk) * scale
    s = s.masked_fill(~see, -math.inf)
    w = torch.where(see, torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)), torch.zeros_like(s))
    out = torch.einsum("hnt,thd->nhd", w / w.sum(-1, keepdim=True).clamp(min=1e-300), vv)
    seen = torch.where(see.any(1), torch.where(see[:, :, None], v.abs().amax(-1)[None], 0).amax(dim=(1, 2)) if len_ else 0, 0) if len_ else torch.zeros(n, device="cuda")
    return out, seen.double()[:, None, None]


def check_attention(torch, got, want, big, t):
    dt = dtype(torch, t)
    bound = 6e-5 * big + (2.0 ** -11 * big + half_step(torch, dt) * want.abs() if t != "f32" else 0) + (2.0 ** -25 if t == "f16" else 0)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-30)).max())


SHAPES = [   # lens, heads, kv heads, dim, page, block
    ([1], 1, 1, 128, 16, 16), ([513], 16, 8, 128, 16, 16), ([0, 1, 16, 17, 300], 8, 2, 128, 32, 16), ([5, 64, 65], 14, 2, 64, 64, 32),
    ([700, 33], 32, 2, 128, 128, 128), ([129, 1000, 31], 6, 6, 64, 16, 16), ([4000], 3, 1, 128, 64, 64), ([77, 78], 34, 2, 128, 32, 32)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_decode(er, torch, fmt, t, shape):
    lens, heads, kv_heads, dim, page, block = SHAPES[shape]
    cache, table, rows = fill(er, torch, fmt, lens, page, kv_heads, dim, block, 20 + shape)
    g = gen(torch, shape)
    for query_len, window, scale in ((1, 0, 0.0), (3, 0, 0.05), (2, 33, 0.0), (16, 1, 0.0)):
        q = torch.randn(len(lens) * query_len, heads, dim, generator=g, device="cuda").to(dtype(torch, t))
        got = cache.attention_decode(q, table, ints(torch, lens), query_len=query_len, sliding_window=window, softmax_scale=scale)
        for s, n in enumerate(lens):
            mine = slice(s * query_len, (s + 1) * query_len)
            if n < query_len:        # queries before the first row see nothing
                assert bool((got[mine][:query_len - n] == 0).all())
            m = min(n, query_len)
            if m:
                want, big = ref_attention(torch, q[mine][query_len - m:], *rows[s], n, scale or dim ** -0.5, window)
                check_attention(torch, got[mine][query_len - m:], want, big, t)
    assert cache.device_status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens, new, heads, kv_heads, dim, page, block", [
    ([100], [100], 16, 8, 128, 16, 16), ([1, 17, 0, 40, 130], [1, 17, 0, 3, 129], 8, 2, 128, 32, 32), ([257, 700], [257, 5], 14, 2, 64, 16, 16),
    ([1500], [300], 3, 1, 128, 64, 64), ([640, 1025], [128, 640], 4, 4, 64, 128, 128), ([90, 500], [90, 500], 34, 2, 128, 32, 16),
    ([2100], [1031], 4, 1, 128, 128, 32)])
def test_prefill(er, torch, fmt, t, lens, new, heads, kv_heads, dim, page, block):
    cache, table, rows = fill(er, torch, fmt, lens, page, kv_heads, dim, block, 40 + len(lens))
    g = gen(torch, 9)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    q = torch.randn(starts[-1] + 2, heads + 1, dim, generator=g, device="cuda").to(dtype(torch, t))[:, :heads]     # strides; two tokens of nobody
    for window, scale in ((0, 0.0), (65, 0.1)):
        out = torch.full((q.shape[0], 2 * heads, dim), 7.0, device="cuda", dtype=q.dtype)[:, heads:]
        cache.attention_prefill(q, ints(torch, starts), table, ints(torch, lens), out=out, max_query_len=max(new), sliding_window=window, softmax_scale=scale)
        assert bool((out[starts[-1]:] == 7).all())
        for s, (n, m) in enumerate(zip(lens, new)):
            if m:
                want, big = ref_attention(torch, q[starts[s]:starts[s + 1]], *rows[s], n, scale or dim ** -0.5, window)
                check_attention(torch, out[starts[s]:starts[s + 1]], want, big, t)
    assert cache.device_status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_pages_that_are_missing_are_hidden(er, torch, fmt, t):
    """Rows in a page that the table does not name are not seen, whatever the bytes are; the status word tells."""
    lens = [200, 90]
    cache, table, rows = fill(er, torch, fmt, lens, 32, 2, 128, 16)
    bad = table.clone()
    bad[0, 2], bad[1, 0] = -1, 1 << 20
    hidden = [torch.zeros(n, dtype=torch.bool, device="cuda") for n in lens]
    hidden[0][64:96] = True
    hidden[1][:32] = True
    q = torch.randn(2, 8, 128, generator=gen(torch, 1), device="cuda").to(dtype(torch, t))
    for fn in (lambda: cache.attention_decode(q, bad, ints(torch, lens)), lambda: cache.attention_prefill(q, ints(torch, [0, 1, 2]), bad, ints(torch, lens))):
        cache.clear_device_status()
        got = fn()
        assert cache.device_status() == -10
        for s in range(2):
            want, big = ref_attention(torch, q[s:s + 1], *rows[s], lens[s], 128 ** -0.5, 0, hidden[s])
            check_attention(torch, got[s:s + 1], want, big, t)
    none = torch.full_like(table, -1)                                       # nothing to see at all
    assert bool((cache.attention_decode(q, none, ints(torch, lens)) == 0).all())
    long = 40 + 300 * 2                                                     # a prompt whose middle is missing
    q = torch.randn(long, 4, 128, generator=gen(torch, 1), device="cuda").to(dtype(torch, t))
    cache, table, rows = fill(er, torch, fmt, [long], 32, 2, 128, 16)
    table[0, 3:5] = -1
    hidden = torch.zeros(long, dtype=torch.bool, device="cuda")
    hidden[96:160] = True
    want, big = ref_attention(torch, q, *rows[0], long, 128 ** -0.5, 0, hidden)
    check_attention(torch, cache.attention_prefill(q, ints(torch, [0, long]), table, ints(torch, [long])), want, big, t)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_pages_in_front_of_the_window_may_be_gone(er, torch, t):
    """A sliding window that begins in the second page of 16 rows of a larger unit of work: freed pages before it are no mistake."""
    lens, window = [16 * 23 + 5, 700], 100
    cache, table, rows = fill(er, torch, "e4m3", lens, 16, 2, 128, 16)
    q = torch.randn(2 * 70, 4, 128, generator=gen(torch, 3), device="cuda").to(dtype(torch, t))
    for n in (1, 70):
        freed = table.clone()
        for s in range(2):
            freed[s, :(lens[s] - n - window + 1) // 16] = -1
        mine = torch.cat([q[:n], q[70:70 + n]])
        got = cache.attention_decode(mine, freed, ints(torch, lens), sliding_window=window) if n == 1 else cache.attention_prefill(
            mine, ints(torch, [0, n, 2 * n]), freed, ints(torch, lens), sliding_window=window)
        assert cache.device_status() == 0
        for s in range(2):
            want, big = ref_attention(torch, mine[s * n:(s + 1) * n], *rows[s], lens[s], 128 ** -0.5, window)
            check_attention(torch, got[s * n:(s + 1) * n], want, big, t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_values_that_are_not_finite_reach_only_those_who_see_them(er, torch, t):
    """A NaN among the newest rows: earlier queries of the same call, and other sequences, stay finite; later ones are NaN."""
    lens = [180, 64]
    cache, table, rows = fill(er, torch, "e4m3", lens, 16, 1, 128, 16)
    page = int(table[0, 170 // 16])
    q = torch.randn(60, 4, 128, generator=gen(torch, 1), device="cuda").to(dtype(torch, t))
    for side in (cache.key_scales, cache.value_scales):
        kept = side.clone()
        side[page] = math.nan                                              # rows 160 .. 175 of sequence 0
        out = cache.attention_prefill(q, ints(torch, [0, 50, 60]), table, ints(torch, lens))
        assert bool(torch.isfinite(out[:30]).all()) and bool(torch.isnan(out[30:50]).all()) and bool(torch.isfinite(out[50:]).all())
        dec = cache.attention_decode(q[:2], table, ints(torch, lens))
        assert bool(torch.isnan(dec[0]).all()) and bool(torch.isfinite(dec[1]).all())
        dec = cache.attention_decode(q[:2], table, ints(torch, [160, 64]))
        assert bool(torch.isfinite(dec).all())
        side.copy_(kept)
    q[0, 0, 0] = math.inf                                                  # a query that is not finite spoils its own row only
    out = cache.attention_decode(q[:2], table, ints(torch, lens))
    assert bool(torch.isnan(out[0, 0]).any()) and bool(torch.isfinite(out[0, 1:]).all()) and bool(torch.isfinite(out[1]).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_scales_of_very_different_blocks(er, torch, t):
    """Value scales from 2^-40 to 2^30 in one row of blocks, key scales that make one token win, queries of large and small magnitude."""
    lens = [256, 256]
    cache, table, _ = fill(er, torch, "e4m3", lens, 16, 2, 64, 16)
    g = gen(torch, 4)
    cache.value_scales.copy_(torch.exp2(torch.randint(-40, 31, cache.value_scales.shape, generator=g, device="cuda").float()))
    rows = [tuple(x.double() for x in cache.decoded_rows([p for p in table[s].tolist() if p >= 0], 256)) for s in range(2)]
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(dtype(torch, t))
    q[1] *= 1e-3
    got = cache.attention_decode(q, table, ints(torch, lens))
    if t != "f16":       # its range ends at 65504
        for s in range(2):
            want, big = ref_attention(torch, q[s:s + 1], *rows[s], 256, 64 ** -0.5)
            check_attention(torch, got[s:s + 1], want, big, t)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_prefill_with_wrong_hints_and_short_caches(er, torch, t):
    """max_query_len is a hint: too small a one loses no rows.  Queries in front of row 0 (more queries than rows) see nothing."""
    lens, new = [300, 40, 9], [120, 40, 1]
    cache, table, rows = fill(er, torch, "e4m3", lens, 16, 2, 64, 16)
    starts = ints(torch, [0, 120, 160, 161])
    q = torch.randn(161, 8, 64, generator=gen(torch, 3), device="cuda").to(dtype(torch, t))
    for hint in (0, 1, 120, 10000):
        got = cache.attention_prefill(q, starts, table, ints(torch, lens), max_query_len=hint)
        for s, at in enumerate((0, 120, 160)):
            want, big = ref_attention(torch, q[at:at + new[s]], *rows[s], lens[s], 64 ** -0.5)
            check_attention(torch, got[at:at + new[s]], want, big, t)
    got = cache.attention_prefill(q, starts, table, ints(torch, [50, 40, 0]))
    assert bool((got[:70] == 0).all()) and bool((got[160:] == 0).all())
    want, big = ref_attention(torch, q[70:120], rows[0][0][:50], rows[0][1][:50], 50, 64 ** -0.5)
    check_attention(torch, got[70:120], want, big, t)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_a_cache_beyond_four_gigabytes(er, torch, t):
    """Pages whose bytes lie behind the first 2^32 of a side."""
    pages, page, heads, dim = 34000, 128, 8, 128                     # 4.46 GB of codes a side
    codes = [torch.empty(pages, heads, page, dim, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, heads, 1, device="cuda") for _ in range(2)]
    cache = er.BlockScaledKVCache.from_tensors(*codes, *scales)
    ids, n = [pages - 1, 0, pages - 2], 300
    g = gen(torch, 6)
    k, v = (torch.randn(n, heads, dim, generator=g, device="cuda").to(dtype(torch, t)) for _ in range(2))
    table = ints(torch, [ids])
    cache.append(k, v, table, ints(torch, [n]), ints(torch, [0, n]), partial_rotary_factor=0.0)
    dk, dv = (x.double() for x in cache.decoded_rows(ids, n))
    assert bool(((dv - v.double()).abs() <= v.double().abs() * 2.0 ** -4 + 2.0 ** -14).all())
    q = torch.randn(n, 16, dim, generator=g, device="cuda").to(dtype(torch, t))
    want, big = ref_attention(torch, q, dk, dv, n, dim ** -0.5)
    check_attention(torch, cache.attention_prefill(q, ints(torch, [0, n]), table, ints(torch, [n])), want, big, t)
    check_attention(torch, cache.attention_decode(q[-1:], table, ints(torch, [n])), want[-1:], big[-1:], t)
    assert cache.device_status() == 0


def test_outputs_that_overlap_are_refused(er, torch):
    cache, table, rows = fill(er, torch, "e4m3", [40], 16, 2, 128, 16)
    q = torch.randn(1, 4, 128, device="cuda")
    with pytest.raises(er.EdgeRunnerCUDAError) as e:
        cache.attention_decode(q, table, ints(torch, [40]), out=torch.empty(1, 1, 128, device="cuda").expand(1, 4, 128))
    assert e.value.name == "shape"
    with pytest.raises(er.EdgeRunnerCUDAError) as e:
        er.QKNormRopeKernel().encode(q, torch.empty(1, 1, 128, device="cuda").expand(1, 4, 128), ints(torch, [3]))
    assert e.value.name == "shape"
    out = torch.empty(4, 1, 128, device="cuda").transpose(0, 1)       # heads far apart, tokens inside
    assert torch.equal(cache.attention_decode(q, table, ints(torch, [40]), out=out), cache.attention_decode(q, table, ints(torch, [40])))


def test_many_sequences(er, torch):
    """More sequences than a CTA has threads, empty ones and ones without queries among them."""
    n = 700
    lens = [(7 * s) % 50 for s in range(n)]
    new = [min(lens[s], s % 4) for s in range(n)]
    cache, table, rows = fill(er, torch, "int8", lens, 16, 1, 64, 16)
    starts = [sum(new[:s]) for s in range(n + 1)]
    q = torch.randn(starts[-1], 4, 64, generator=gen(torch, 2), device="cuda").bfloat16()
    got = cache.attention_prefill(q, ints(torch, starts), table, ints(torch, lens), max_query_len=3)
    dec = cache.attention_decode(q[:n], table, ints(torch, lens))
    for s in range(n):
        if new[s]:
            want, big = ref_attention(torch, q[starts[s]:starts[s + 1]], *rows[s], lens[s], 64 ** -0.5)
            check_attention(torch, got[starts[s]:starts[s + 1]], want, big, "bf16")
        if lens[s]:
            want, big = ref_attention(torch, q[s:s + 1], *rows[s], lens[s], 64 ** -0.5)
            check_attention(torch, dec[s:s + 1], want, big, "bf16")
        else:
            assert bool((dec[s] == 0).all())
    assert cache.device_status() == 0


def test_two_streams_and_a_graph(er, torch):
    """Calls on two streams do not share a workspace; captured calls follow the lengths and queries of their buffers at replay."""
    lens = [3000, 2500]
    cache, table, rows = fill(er, torch, "e4m3", lens, 16, 2, 128, 16)
    g = gen(torch, 2)
    qs = [torch.randn(2, 8, 128, generator=g, device="cuda") for _ in range(2)]
    want = [cache.attention_decode(q, table, ints(torch, lens)).clone() for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ln = ints(torch, lens)
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attention_decode(qs[i], table, ln))
    explicit = cache.attention_decode(qs[0], table, ln, stream=streams[1])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])                 # the same bits each time
    assert torch.equal(explicit, want[0])
    q, n, out = qs[0].clone(), ints(torch, lens), torch.empty(2, 8, 128, device="cuda")
    p, pout, starts = torch.randn(40, 8, 128, generator=g, device="cuda").bfloat16(), torch.empty(40, 8, 128, device="cuda", dtype=torch.bfloat16), ints(torch, [0, 30, 40])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention_decode(q, table, n, out=out)
        cache.attention_prefill(p, starts, table, n, out=pout)
    for step in range(3):
        n.copy_(ints(torch, [lens[0] - 700 * step, lens[1] - 3 * step]))
        q.copy_(qs[step % 2])
        graph.replay()
        assert torch.equal(out, cache.attention_decode(q, table, n)) and torch.equal(pout, cache.attention_prefill(p, starts, table, n))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_prompt_and_decode_steps_together(er, torch, fmt):
    """The four operators as a decoder layer uses them, pages from the allocator: every step's output against attention over the rows that the
    cache holds then, computed in 64 bits from the step's own (normed, rotated) queries."""
    heads, kv_heads, dim, page, theta = 8, 2, 128, 32, 1e6
    g, dt = gen(torch, 8), torch.bfloat16
    prompts = [45, 1, 130]
    alloc = er.BlockTableAllocator(32, page)
    cache = er.BlockScaledKVCache(32, page, kv_heads, dim, er.BlockScaledFormat[fmt], scale_block=32)
    qw, kw = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda") for _ in range(2))
    table = torch.full((3, 8), -1, dtype=torch.int32)
    lens = [0, 0, 0]
    for step in range(6):
        new = prompts if step == 0 else [1, 1, 1]
        lens = [a + b for a, b in zip(lens, new)]
        for s in range(3):
            ids = alloc.ensure(s, lens[s])
            table[s, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        dev = table.cuda()
        rows = torch.randn(sum(new), heads + 2 * kv_heads, dim, generator=g, device="cuda").to(dt)
        pos = torch.cat([torch.arange(n - m, n, dtype=torch.int32) for n, m in zip(lens, new)]).cuda()
        q = torch.empty(sum(new), heads, dim, device="cuda", dtype=dt)
        er.QKNormRopeKernel().encode(rows[:, :heads], q, pos, q_norm_weight=qw, rope_theta=theta)
        starts = ints(torch, [sum(new[:i]) for i in range(4)])
        cache.append(rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:], dev, ints(torch, lens), starts if step == 0 else None, k_norm_weight=kw, rope_theta=theta)
        out = cache.attention_prefill(q, starts, dev, ints(torch, lens), max_query_len=max(new)) if step == 0 else cache.attention_decode(q, dev, ints(torch, lens))
        at = 0
        for s in range(3):
            k, v = (x.double() for x in cache.decoded_rows(alloc.block_table(s), lens[s]))
            want, big = ref_attention(torch, q[at:at + new[s]], k, v, lens[s], dim ** -0.5)
            check_attention(torch, out[at:at + new[s]], want, big, "bf16")
            # ... and the cache holds the rows it was given: normed and rotated keys, values as they came
            wk = ref_norm_rope(torch, rows[at:at + new[s], heads:heads + kv_heads], pos[at:at + new[s]], kw, theta)
            wv = rows[at:at + new[s], heads + kv_heads:].double()
            for x, y in ((k[-new[s]:], wk), (v[-new[s]:], wv)):      # 4 re-roundings of a block at most since it was written: none here, it is the newest
                amax = max(float(x.abs().amax()), float(y.abs().amax()), 8.0)
                assert bool(((x - y).abs() <= (amax / 127 / 2 if fmt == "int8" else y.abs() * 2.0 ** -4 + amax * 2.0 ** -17) * (1 + 1e-4) + 16 * U32 * amax).all())
            at += new[s]
    assert cache.device_status() == 0

"""The 8-bit block-scaled cache where its ranges end: long runs of keys, scales far apart, extreme windows, epsilons and magnitudes, streams.

Tolerances are those of test_gpu_block_scaled.py (derived there), with one more term where keys run long: each product of 16 keys that the tensor cores add
to a running sum truncates it, by less than one unit in the last place, 2^-23 relative; a run of n keys adds n / 16 of them at most.
"""
import math

import pytest

from test_gpu_block_scaled import check_attention, dtype, er, fill, gen, half_step, ints, ref_attention, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def far_apart(torch, cache, seed, key_bits=4, value_bits=6):
    """Block scales that differ by powers of two from block to block: keys down to 2^-key_bits, values 2^-value_bits .. 2^value_bits of what they were."""
    g = gen(torch, seed)
    cache.key_scales.mul_(torch.exp2(-torch.randint(0, key_bits + 1, cache.key_scales.shape, generator=g, device="cuda").float()))
    cache.value_scales.mul_(torch.exp2(torch.randint(-value_bits, value_bits + 1, cache.value_scales.shape, generator=g, device="cuda").float()))


def rows_of(cache, table, length):
    return tuple(x.double() for x in cache.decoded_rows([p for p in table.tolist() if p >= 0], length))


def check_long(torch, got, want, big, t, keys):
    bound = (6e-5 + 2.0 ** -11 + keys / 16 * 2.0 ** -23) * big + half_step(torch, dtype(torch, t)) * want.abs() + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("dim, seqs, n, longest, block", [
    (64, 32, 10, 8000, 16), (64, 23, 40, 4100, 16), (64, 23, 40, 2500, 128), (128, 32, 10, 4000, 16), (128, 23, 40, 2300, 32)])
def test_prefill_over_many_key_tiles(er, torch, fmt, t, dim, seqs, n, longest, block):  # noqa: F811
    """18 to 63 key tiles to a CTA: 4 kv heads times 37 slots of 256 query rows make 148 tile pairs, which are not cut along the keys.  One row tile a CTA
    (10 queries of 4 heads) and two (40 of them).  The sequences read the same pages, at lengths of their own."""
    heads, kv_heads = 16, 4
    cache, table, _ = fill(er, torch, fmt, [longest], 128, kv_heads, dim, block, seed=dim + block)
    far_apart(torch, cache, 5)
    k, v = rows_of(cache, table[0], longest)
    lens = [longest - 37 * s for s in range(seqs)]
    starts = ints(torch, [n * s for s in range(seqs + 1)])
    q = torch.randn(n * seqs, heads, dim, generator=gen(torch, 7), device="cuda").to(dtype(torch, t))
    many = table.expand(seqs, -1).contiguous()
    got = [cache.attention_prefill(q, starts, many, ints(torch, lens), max_query_len=n) for _ in range(3)]
    assert cache.device_status() == 0
    assert all(torch.equal(x, got[0]) for x in got[1:])
    for s, length in enumerate(lens):
        mine = slice(n * s, n * (s + 1))
        want, big = ref_attention(torch, q[mine], k[:length], v[:length], length, dim ** -0.5)
        check_long(torch, got[0][mine], want, big, t, length)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_append_without_an_epsilon(er, torch, fmt, t):  # noqa: F811
    """rms_eps 0: rows of the block that the call does not write have no norm, and must not decide its scale."""
    g = gen(torch, 3)
    cache = er.BlockScaledKVCache(4, 32, 2, 128, er.BlockScaledFormat[fmt])
    table, kw = ints(torch, [[2, 0], [1, 3]]), 1 + 0.1 * torch.randn(128, generator=g, device="cuda")
    lens, new = [0, 0], [[5, 1], [1, 1], [14, 1], [13, 33]]
    kept = [[], []]
    for step in new:
        lens = [a + b for a, b in zip(lens, step)]
        k, v = (torch.randn(sum(step), 2, 128, generator=g, device="cuda").to(dtype(torch, t)) for _ in range(2))
        cache.append(k, v, table, ints(torch, lens), ints(torch, [0, step[0], sum(step)]), k_norm_weight=kw, rms_eps=0.0, partial_rotary_factor=0.0)
        for s, part in enumerate(k.split(step)):
            x = part.double()
            kept[s].append(x / x.square().mean(-1, keepdim=True).sqrt() * kw.double())
    assert bool(torch.isfinite(cache.key_scales).all()) and bool(torch.isfinite(cache.value_scales).all())
    for s in range(2):
        want, (k, _) = torch.cat(kept[s]), cache.decoded_rows(table[s], lens[s])
        # a code is written once and rounded again when its block's scale grows, on each of 3 later calls at most: half a step each, of a block whose
        # magnitudes stay below 8; E4M3's smallest codes 2^-10 of a scale of at most 2^-5
        bound = 4 * 8 / 127 / 2 if fmt == "int8" else want.abs() * 2.0 ** -4 * (1 + 1e-4) + 4 * 2.0 ** -15
        assert bool(((k.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_append_of_tiny_rows(er, torch, fmt, t):  # noqa: F811
    """Keys of 1e-37 under an epsilon of 1e-6: what turns them into codes, the norm factor (1000) over the scale, is beyond float32's range."""
    g = gen(torch, 4)
    cache = er.BlockScaledKVCache(2, 32, 1, 64, er.BlockScaledFormat[fmt])
    k = (torch.randn(20, 1, 64, generator=g, device="cuda") * 1e-37).to(dtype(torch, t))
    k[3] = 0
    k[:, :, ::7] = 0
    cache.append(k, k, ints(torch, [[1]]), ints(torch, [20]), ints(torch, [0, 20]), k_norm_weight=torch.ones(64, device="cuda"), partial_rotary_factor=0.0)
    want = k.double() / math.sqrt(1e-6)
    got = cache.decoded_rows([1], 20)[0].double()
    scale = cache.key_scales[1, 0].double().repeat_interleave(16)[:20, None, None]
    step = scale / 2 if fmt == "int8" else torch.maximum(want.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    # the norm factor is off by a few steps of float32; a decoded value below 2^-126 may be flushed
    assert bool(((got - want).abs() <= step * (1 + 1e-4) + want.abs() * 2.0 ** -20 + 2.0 ** -126).all())


def test_the_output_of_a_call_on_another_stream_is_that_streams_memory(er, torch):  # noqa: F811
    """Without `out` the output comes from the memory of the stream that the kernel runs on: a block of the current stream's may still be in use there."""
    cache, table, rows = fill(er, torch, "e4m3", [40], 16, 2, 64, 16)
    other = torch.cuda.Stream()
    q, starts, lens = torch.randn(1, 4, 64, device="cuda"), ints(torch, [0, 1]), ints(torch, [40])
    torch.cuda.synchronize()
    for stream in (other, other.cuda_stream):
        for out in (cache.attention_decode(q, table, lens, stream=stream), cache.attention_prefill(q, starts, table, lens, stream=stream)):
            at = out.data_ptr()
            owner = [s["stream"] for s in torch.cuda.memory_snapshot() if s["address"] <= at < s["address"] + s["total_size"]]
            assert owner == [other.cuda_stream]
            other.synchronize()
            want, big = ref_attention(torch, q, *rows[0], 40, 64 ** -0.5)
            check_attention(torch, out, want, big, "f32")


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0x7FFFFFFF, 0x7FFFFFFF - 40, 1 << 30])
def test_windows_wider_than_any_sequence(er, torch, t, window):  # noqa: F811
    """The same as no window, also for queries in front of row 0."""
    cache, table, rows = fill(er, torch, "int8", [70, 300], 16, 2, 64, 16)
    q = torch.randn(120, 4, 64, generator=gen(torch, 2), device="cuda").to(dtype(torch, t))
    for lens in ([70, 300], [9, 20], [0, 300]):
        args = (table, ints(torch, lens))
        starts = ints(torch, [0, 100, 120])
        assert torch.equal(cache.attention_prefill(q, starts, *args, sliding_window=window), cache.attention_prefill(q, starts, *args))
        assert torch.equal(cache.attention_decode(q[:32], *args, query_len=16, sliding_window=window), cache.attention_decode(q[:32], *args, query_len=16))
    got = cache.attention_prefill(q, starts, table, ints(torch, [9, 20]), sliding_window=window)
    want, big = ref_attention(torch, q[91:100], rows[0][0][:9], rows[0][1][:9], 9, 64 ** -0.5)
    check_attention(torch, got[91:100], want, big, t)
    assert bool((got[:91] == 0).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("where", ["later", "left"])
def test_hidden_blocks_with_large_values(er, torch, t, op, dim, where):  # noqa: F811
    """A block whose value scale is 2^40 times the others' costs those queries nothing that do not see it: those in front of it, or (`left`) those whose
    window has left it behind."""
    if op == "decode":
        length, n, block, window = (100, 8, 96, 0) if where == "later" else (100, 8, 64, 20)
    else:
        length, n, block, window = (300, 200, 272, 0) if where == "later" else (200, 200, 16, 50)
    cache, table, _ = fill(er, torch, "e4m3", [length], 16, 2, dim, 16)
    cache.value_scales[int(table[0, block // 16])] *= 2.0 ** 40
    k, v = rows_of(cache, table[0], length)
    q = torch.randn(n, 8, dim, generator=gen(torch, 2), device="cuda").to(dtype(torch, t))
    pos = torch.arange(length - n, length, device="cuda")
    sees = (pos >= block) & ((pos - window + 1 <= block + 15) if window else True)
    assert bool(sees.any()) and bool((~sees).any())
    got = (cache.attention_decode(q, table, ints(torch, [length]), query_len=n, sliding_window=window) if op == "decode" else
           cache.attention_prefill(q, ints(torch, [0, n]), table, ints(torch, [length]), sliding_window=window))
    want, big = ref_attention(torch, q, k, v, length, dim ** -0.5, window)
    check_attention(torch, got[~sees], want[~sees], big[~sees], t)
    if t != "f16":          # beyond its range
        check_attention(torch, got[sees], want[sees], big[sees], t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_value_scales_over_forty_powers_of_two(er, torch, t, op, fmt):  # noqa: F811
    """Within float16's range of outputs; the bound is relative to the largest value that the query sees."""
    length, n = 700, 8 if op == "decode" else 150
    cache, table, _ = fill(er, torch, fmt, [length], 16, 2, 64, 16)
    g = gen(torch, 4)
    cache.value_scales.copy_(torch.exp2(torch.randint(-40, 1, cache.value_scales.shape, generator=g, device="cuda").float()))
    k, v = rows_of(cache, table[0], length)
    q = torch.randn(n, 8, 64, generator=g, device="cuda").to(dtype(torch, t))
    for window in (0, 70):
        got = (cache.attention_decode(q, table, ints(torch, [length]), query_len=n, sliding_window=window) if op == "decode" else
               cache.attention_prefill(q, ints(torch, [0, n]), table, ints(torch, [length]), sliding_window=window))
        want, big = ref_attention(torch, q, k, v, length, 64 ** -0.5, window)
        assert float(want.abs().max()) < 60000
        check_attention(torch, got, want, big, t)


def mean_of_roundings(torch, t, n):
    """What the roundings of weights and of `n` outputs may add to the mean relative error, in all but one of a million cases.  The outputs here are means of
    65536 or more values between 0.5 and 1.5 under nearly equal weights: 1 with a deviation of sqrt(1 / 12) / 256 = 0.0011.  float16's steps there are
    2^-10 and 2^-11, no wider than that, so its roundings have either sign: 5 deviations of a mean of n uniform errors.  A step of bfloat16 is 2^-7 or
    2^-8, wider than the outputs' spread: all of them may round the same way, and the mean of their errors is bounded by half a step alone."""
    u = half_step(torch, dtype(torch, t))
    return 5 * (u + 2.0 ** -11) / math.sqrt(3 * n) if t == "f16" else u + 5 * 2.0 ** -11 / math.sqrt(3 * n)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_sums_over_a_long_context_are_not_biased(er, torch, t, dim):  # noqa: F811
    """Half a million keys and values around 1: what truncation takes from a running sum would add up.  128 sequences of 10 queries of 4 heads
    over the same pages are 148 tile pairs, which are not cut along the keys."""
    length, seqs, n = 500000, 128, 10
    cache, table, _ = fill(er, torch, "e4m3", [16], 128, 1, dim, 16)
    g = gen(torch, 6)
    pages = -(-length // 128)
    codes = [torch.randn(pages, 1, 128, dim, generator=g, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8),
             (torch.rand(pages, 1, 128, dim, generator=g, device="cuda") + 0.5).to(torch.float8_e4m3fn).view(torch.uint8)]
    cache = er.BlockScaledKVCache.from_tensors(*codes, *(torch.full((pages, 1, 8), s, device="cuda") for s in (0.125, 1.0)))
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None]
    k, v = rows_of(cache, table[0], length)
    q = torch.randn(seqs * n, 4, dim, generator=g, device="cuda").to(dtype(torch, t))
    starts = ints(torch, [n * s for s in range(seqs + 1)])
    got = cache.attention_prefill(q, starts, table.expand(seqs, -1).contiguous(), ints(torch, [length] * seqs), max_query_len=n)
    for s in (0, 77):
        want, big = ref_attention(torch, q[n * s:n * (s + 1)], k, v, length, dim ** -0.5)
        check_attention(torch, got[n * s:n * (s + 1)], want, big, t)
        # a chain of 16384 keys between sums kept in float32 is truncated by at most 1024 * 2^-23
        mean = float(((got[n * s:n * (s + 1)].double() - want) / want).mean())
        assert abs(mean) <= mean_of_roundings(torch, t, 40 * dim) + 1024 * 2.0 ** -23, mean


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("t, dim, seqs, lengths", [("f16", 128, 23, (40000, 16384, 16385, 5000)), ("bf16", 64, 23, (33000, 16513, 100)), ("bf16", 128, 1, (150000,)),
                                                   ("f16", 64, 1, (280000,))])
def test_sums_joined_over_a_long_context(er, torch, fmt, t, dim, seqs, lengths):  # noqa: F811
    """Contexts of several stretches of 16384 keys, on either side of one, and cut along the keys as well (one sequence); maxima that rise and scales
    that differ from stretch to stretch; windows longer and shorter than one.  Calls on two streams at a time give the bits of calls one by one."""
    kv_heads, n = (4, 40) if seqs > 1 else (1, 70)
    heads, longest = 4 * kv_heads, max(lengths)
    cache, table, _ = fill(er, torch, fmt, [longest], 128, kv_heads, dim, 16, seed=dim)
    far_apart(torch, cache, 5)
    order = torch.arange(table.shape[1], device="cuda").float()      # later stretches of 64 pages: larger keys, smaller values
    at = table[0].clamp(min=0).long()
    cache.key_scales[at] *= torch.exp2(-3 + 3 * torch.floor(order / 64) / max(1, table.shape[1] // 64))[:, None, None]
    cache.value_scales[at] *= torch.exp2(-torch.floor(order / 64).clamp(max=10))[:, None, None]
    k, v = rows_of(cache, table[0], longest)
    lens = [lengths[s % len(lengths)] for s in range(seqs)]
    q = torch.randn(n * seqs, heads, dim, generator=gen(torch, 7), device="cuda").to(dtype(torch, t))
    args = (q, ints(torch, [n * s for s in range(seqs + 1)]), table.expand(seqs, -1).contiguous(), ints(torch, lens))
    got = {w: cache.attention_prefill(*args, max_query_len=n, sliding_window=w) for w in (0, 3000, 20001)}
    for w, out in got.items():
        for s in range(min(seqs, len(lengths))):
            mine, length = slice(n * s, n * (s + 1)), lens[s]
            want, big = ref_attention(torch, q[mine], k[:length], v[:length], length, dim ** -0.5, w)
            check_long(torch, out[mine], want, big, t, 16384)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(cache.attention_prefill(*args, max_query_len=n, sliding_window=(0, 20001)[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, got[0]) for x in outs[0]) and all(torch.equal(x, got[20001]) for x in outs[1])
    assert cache.device_status() == 0


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("dim, heads", [(64, 8), (128, 8), (128, 16)])
def test_decode_sums_over_millions_of_rows_are_not_biased(er, torch, t, dim, heads):  # noqa: F811
    """Four million rows a sequence, the same 65536 over and over: their mean is that of the 65536.  148 sequences, so that a CTA walks whole ones."""
    base, times, seqs = 65536, 64, 148
    g = gen(torch, 6)
    pages = base // 128
    codes = [torch.randn(pages, 1, 128, dim, generator=g, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8),
             (torch.rand(pages, 1, 128, dim, generator=g, device="cuda") + 0.5).to(torch.float8_e4m3fn).view(torch.uint8)]
    cache = er.BlockScaledKVCache.from_tensors(*codes, *(torch.full((pages, 1, 8), s, device="cuda") for s in (0.125, 1.0)))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    q = torch.randn(seqs, heads, dim, generator=g, device="cuda").to(dtype(torch, t))
    got = cache.attention_decode(q, order.repeat(times)[None].expand(seqs, -1).contiguous(), ints(torch, [base * times] * seqs))
    k, v = rows_of(cache, order, base)
    want, big = (torch.cat(x) for x in zip(*(ref_attention(torch, q[s:s + 1], k, v, base, dim ** -0.5) for s in range(8))))
    check_attention(torch, got[:8], want, big, t)
    # 512 units of 32 rows between sums kept in float32 are 1024 products of 16, each of which takes less than 2^-23
    mean = float(((got[:8].double() - want) / want).mean())
    assert abs(mean) <= mean_of_roundings(torch, t, 8 * heads * dim) + 1024 * 2.0 ** -23, mean
    assert cache.device_status() == 0


def test_the_status_waits_for_every_stream(er, torch):  # noqa: F811
    """device_status() tells what a call on any stream has met, also one that is still running when it is asked."""
    cache = er.BlockScaledKVCache(2, 16, 1, 64)
    k = torch.ones(1, 1, 64, device="cuda")
    table, lens, other = ints(torch, [[-1]]), ints(torch, [1]), torch.cuda.Stream()
    cache.append(k, k, table, lens, partial_rotary_factor=0.0)
    assert cache.device_status() == -10
    cache.clear_device_status()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        torch.cuda._sleep(200_000_000)          # 0.1 s
        cache.append(k, k, table, lens, partial_rotary_factor=0.0)
    assert cache.device_status() == -10


def test_tables_without_pages(er, torch):  # noqa: F811
    """A batch of empty sequences whose table has no column yet: nothing to see, and nowhere to write."""
    cache = er.BlockScaledKVCache(2, 16, 1, 64)
    q = torch.randn(2, 2, 64, device="cuda")
    table, lens = torch.empty(2, 0, dtype=torch.int32, device="cuda"), ints(torch, [0, 0])
    assert bool((cache.attention_decode(q, table, lens) == 0).all())
    assert bool((cache.attention_prefill(q, ints(torch, [0, 1, 2]), table, lens) == 0).all())
    assert cache.device_status() == 0
    cache.append(q[:, :1], q[:, :1], table, ints(torch, [1, 1]), partial_rotary_factor=0.0)
    assert cache.device_status() == -10


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim, heads, kv_heads, query_len", [(128, 4, 1, 1), (64, 6, 2, 1), (128, 8, 1, 1), (64, 2, 2, 4), (128, 16, 1, 1), (128, 14, 2, 2), (64, 32, 4, 3), (128, 3, 1, 1)])
def test_float16_decode_is_as_exact_as_its_outputs(er, torch, fmt, dim, heads, kv_heads, query_len):  # noqa: F811
    """What is left against 64 bits is the rounding of the outputs to float16.  With y = want + d before it, |round(y) - want| <= |round(want) - want| + 2 |d|
    (round(y) is no farther from y than round(want) is), and so are the norms.  d is float32's share: 22 bits of the weights, scores of exact products,
    sums of some thousand terms, less than 2^-17 = 7.6e-6 of the output all together."""
    lens = [9000, 20001]
    cache, table, rows = fill(er, torch, fmt, lens, 128, kv_heads, dim, 16)
    q = (0.3 * torch.randn(2 * query_len, heads, dim, generator=gen(torch, 2), device="cuda")).half()
    got = cache.attention_decode(q, table, ints(torch, lens), query_len=query_len)
    for s, n in enumerate(lens):
        mine = slice(s * query_len, (s + 1) * query_len)
        want, _ = ref_attention(torch, q[mine], *rows[s], n, dim ** -0.5)
        best = float((want.half().double() - want).norm())
        assert float((got[mine].double() - want).norm()) <= best + 2 * 2.0 ** -17 * float(want.norm())


@pytest.mark.parametrize("theta, scaling", [(1e4, 1.0), (5e5, 8.0)])
def test_turns_are_right_where_they_are_small(er, torch, theta, scaling):  # noqa: F811
    """Pairs (1, 0) come out as (cos, sin).  Each is off by one step of the function, half a step of the correction's addition (2^-23 and 2^-24 of itself) and the angle:
    64 bits over up to 2^20 / (2 pi) turns, 3 roundings, 4e-10 radians.  An angle rounded to 32 bits alone would be off by up to 9e-8."""
    g = gen(torch, 2)
    pos = torch.randint(0, 1 << 20, (4096,), generator=g, device="cuda", dtype=torch.int32)
    x = torch.zeros(4096, 1, 128, device="cuda")
    x[..., :64] = 1
    y = torch.empty_like(x)
    er.QKNormRopeKernel().encode(x, y, pos, rope_theta=theta, rope_scaling=scaling)
    angle = pos.double()[:, None] * (theta ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64) / scaling)
    want = torch.cat([angle.cos(), angle.sin()], dim=-1)[:, None]
    assert bool(((y.double() - want).abs() <= want.abs() * 1.5 * 2.0 ** -23 + 1e-9).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_pages_in_front_of_the_window_may_be_somebody_elses(er, torch, t, dim):  # noqa: F811
    """A freed page whose id is still in the table: whatever lies there now, bytes that are codes of NaN and scales that are not finite among it, is not read
    as anything."""
    lens, window = [16 * 23 + 5, 700], 100
    cache, table, rows = fill(er, torch, "e4m3", lens, 16, 2, dim, 16)
    other = int(torch.arange(cache.num_pages, device="cuda")[~torch.isin(torch.arange(cache.num_pages, device="cuda"), table)][0])
    cache.keys[other], cache.values[other] = 0x7F, 0xFF                    # NaN in every row
    cache.key_scales[other], cache.value_scales[other] = math.nan, math.inf
    q = torch.randn(2 * 70, 4, dim, generator=gen(torch, 3), device="cuda").to(dtype(torch, t))
    for n in (1, 3, 70):
        stale = table.clone()
        for s in range(2):
            stale[s, :(lens[s] - n - window + 1) // 16] = other
        mine = torch.cat([q[:n], q[70:70 + n]])
        got = [cache.attention_prefill(mine, ints(torch, [0, n, 2 * n]), stale, ints(torch, lens), sliding_window=window)]
        if n <= 16:
            got.append(cache.attention_decode(mine, stale, ints(torch, lens), query_len=n, sliding_window=window))
        for out in got:
            for s in range(2):
                want, big = ref_attention(torch, mine[s * n:(s + 1) * n], *rows[s], lens[s], dim ** -0.5, window)
                check_attention(torch, out[s * n:(s + 1) * n], want, big, t)
    assert cache.device_status() == 0


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("columns", [100, 2100, 17000])
def test_tables_wider_than_the_sequences(er, torch, t, columns):  # noqa: F811
    """A server's tables have a fixed width: 1600, 33600 and 272000 rows here, beyond what either kernel keeps in its accumulators.  Prompts beside single tokens,
    eager and as a captured graph that sees other lengths at its replay."""
    lens, new = [400, 90, 0, 1030], [400, 1, 0, 130]
    cache, table, rows = fill(er, torch, "e4m3", lens, 16, 2, 128, 16)
    wide = torch.full((4, columns), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    starts = [sum(new[:s]) for s in range(5)]
    q = torch.randn(starts[-1], 8, 128, generator=gen(torch, 3), device="cuda").to(dtype(torch, t))
    one = q[:4].contiguous()
    n, st = ints(torch, lens), ints(torch, starts)

    def check(out, dec, now):
        for s in range(4):
            if new[s]:
                want, big = ref_attention(torch, q[starts[s]:starts[s + 1]], rows[s][0][:now[s]], rows[s][1][:now[s]], now[s], 128 ** -0.5)
                check_attention(torch, out[starts[s]:starts[s + 1]], want, big, t)
            if now[s]:
                want, big = ref_attention(torch, one[s:s + 1], rows[s][0][:now[s]], rows[s][1][:now[s]], now[s], 128 ** -0.5)
                check_attention(torch, dec[s:s + 1], want, big, t)

    check(cache.attention_prefill(q, st, wide, n, max_query_len=400), cache.attention_decode(one, wide, n), lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dec = cache.attention_prefill(q, st, wide, n, max_query_len=400), cache.attention_decode(one, wide, n)
    for now in (lens, [400, 60, 0, 500]):
        n.copy_(ints(torch, now))
        graph.replay()
        check(out, dec, now)
    assert cache.device_status() == 0

"""Refusals of the 8-bit block-scaled cache and of the head-norm operator that need no device: the C entry points check their
arguments before anything touches the GPU, the Python layer checks its tensors before it calls them."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def er():
    import edgerunner_b200 as er
    from edgerunner_b200 import build
    build.build()
    return er


BASE = 1 << 20   # an aligned address that is never followed


def cache(**kw):
    from edgerunner_b200 import _lib
    v = _lib.er_kv8_cache()
    for n in ("keys", "values", "key_scales", "value_scales", "block_tables", "kv_lens"):
        setattr(v, n, BASE)
    v.num_pages, v.page_size, v.scale_block, v.num_kv_heads, v.head_dim, v.format = 4, 32, 16, 2, 128, 0
    v.num_seqs, v.block_table_width, v.block_table_stride = 2, 3, 3
    for n, x in kw.items():
        setattr(v, n, x)
    return v


def attention(**kw):
    from edgerunner_b200 import _lib
    p = _lib.er_kv8_attention_params()
    p.q, p.out, p.q_token_stride, p.q_head_stride, p.out_token_stride, p.out_head_stride = BASE, BASE, 512, 128, 512, 128
    p.query_starts, p.num_tokens, p.num_heads, p.query_len, p.type = BASE, 2, 4, 1, 1
    p.workspace, p.workspace_bytes = BASE, 1 << 30
    for n, x in kw.items():
        setattr(p, n, x)
    return p


def append(**kw):
    from edgerunner_b200 import _lib
    p = _lib.er_kv8_append_params()
    p.k, p.v, p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride = BASE, BASE, 256, 128, 256, 128
    p.num_tokens, p.type, p.rope_theta, p.rope_scaling, p.partial_rotary_factor = 2, 2, 1e4, 1.0, 1.0
    for n, x in kw.items():
        setattr(p, n, x)
    return p


def norm(**kw):
    from edgerunner_b200 import _lib
    p = _lib.er_qk_norm_rope_params()
    p.q = p.q_out = p.positions = BASE
    p.q_token_stride, p.q_head_stride, p.q_out_token_stride, p.q_out_head_stride = 512, 128, 512, 128
    p.num_tokens, p.num_heads, p.head_dim, p.type = 3, 4, 128, 0
    p.rope_theta, p.rope_scaling, p.partial_rotary_factor = 1e4, 1.0, 1.0
    for n, x in kw.items():
        setattr(p, n, x)
    return p


SHAPE, INVALID, UNSUPPORTED = -7, -9, -11


@pytest.mark.parametrize("change, code", [
    (dict(keys=0), INVALID), (dict(kv_lens=0), INVALID), (dict(block_tables=0), INVALID), (dict(value_scales=0), INVALID),
    (dict(format=2), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED), (dict(scale_block=8), UNSUPPORTED),
    (dict(scale_block=48), UNSUPPORTED), (dict(page_size=24), SHAPE), (dict(page_size=0), SHAPE), (dict(num_pages=0), SHAPE),
    (dict(num_kv_heads=0), SHAPE), (dict(num_seqs=65537), UNSUPPORTED), (dict(block_table_width=4), SHAPE),
    (dict(block_table_width=1 << 27, block_table_stride=1 << 27), UNSUPPORTED), (dict(values=BASE + 8), INVALID)])
def test_cache_refusals(er, change, code):
    L = er.lib()
    if code == SHAPE and change == dict(num_kv_heads=0):
        assert L.er_kv8_decode_workspace_bytes(C.byref(cache(**change)), C.byref(attention())) == INVALID
    assert L.er_kv8_append(C.byref(cache(**change)), C.byref(append()), None) == code
    assert L.er_kv8_attention_decode(C.byref(cache(**change)), C.byref(attention()), None) == code
    assert L.er_kv8_attention_prefill(C.byref(cache(**change)), C.byref(attention()), None) == code


@pytest.mark.parametrize("change, code", [
    (dict(k=0), INVALID), (dict(v=0), INVALID), (dict(type=3), INVALID), (dict(k=BASE + 2), INVALID), (dict(k_token_stride=130), INVALID),
    (dict(v_head_stride=-128), INVALID), (dict(partial_rotary_factor=1.5), INVALID), (dict(partial_rotary_factor=float("nan")), INVALID),
    (dict(rope_theta=0.0), INVALID), (dict(rope_scaling=-1.0), INVALID), (dict(rope_theta=float("inf")), INVALID), (dict(rms_eps=-1.0), INVALID),
    (dict(num_tokens=3), SHAPE), (dict(num_tokens=0xFFFFFFFF), UNSUPPORTED)])
def test_append_refusals(er, change, code):
    assert er.lib().er_kv8_append(C.byref(cache()), C.byref(append(**change)), None) == code


@pytest.mark.parametrize("change, code", [
    (dict(q=0), INVALID), (dict(q_out=0), INVALID), (dict(k=BASE), INVALID), (dict(type=7), INVALID), (dict(head_dim=120), UNSUPPORTED),
    (dict(head_dim=272), UNSUPPORTED), (dict(num_heads=0), SHAPE), (dict(positions=0), INVALID), (dict(q_token_stride=514), INVALID),
    (dict(q=BASE + 4), INVALID), (dict(num_tokens=0xFFFFFFFF), UNSUPPORTED), (dict(k=BASE, k_out=BASE), SHAPE), (dict(rms_eps=float("nan")), INVALID)])
def test_norm_refusals(er, change, code):
    assert er.lib().er_qk_norm_rope(C.byref(norm(**change)), None) == code


@pytest.mark.parametrize("change, code", [
    (dict(q=0), INVALID), (dict(out=0), INVALID), (dict(type=3), INVALID), (dict(num_heads=3), SHAPE), (dict(num_heads=0), SHAPE), (dict(q=BASE + 8), INVALID),
    (dict(q_head_stride=4), INVALID), (dict(softmax_scale=-1.0), INVALID), (dict(softmax_scale=float("inf")), INVALID), (dict(sliding_window=0xFFFFFFFF), UNSUPPORTED),
    (dict(out_head_stride=64), SHAPE), (dict(out_token_stride=128), SHAPE), (dict(num_tokens=1 << 30), UNSUPPORTED)])
def test_attention_refusals(er, change, code):
    L = er.lib()
    assert L.er_kv8_attention_decode(C.byref(cache()), C.byref(attention(**change)), None) == code
    assert L.er_kv8_attention_prefill(C.byref(cache()), C.byref(attention(**change)), None) == code


def test_decode_and_prefill_refusals(er):
    L = er.lib()
    for change, code in ((dict(query_len=0), UNSUPPORTED), (dict(query_len=17, num_tokens=34), UNSUPPORTED), (dict(num_tokens=3), SHAPE)):
        assert L.er_kv8_attention_decode(C.byref(cache()), C.byref(attention(**change)), None) == code
    assert L.er_kv8_attention_prefill(C.byref(cache()), C.byref(attention(query_starts=0)), None) == INVALID
    assert L.er_qk_norm_rope(C.byref(norm(q_out_head_stride=0)), None) == SHAPE
    assert L.er_kv8_attention_decode(None, C.byref(attention()), None) == INVALID
    assert L.er_kv8_append(C.byref(cache()), None, None) == INVALID


def test_attention_needs_a_device(er):
    """What passes every check of arguments reaches the device check and, without one, fails loudly."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    for fn in (er.lib().er_kv8_attention_decode, er.lib().er_kv8_attention_prefill):
        assert fn(C.byref(cache()), C.byref(attention()), None) == -8
    assert er.lib().er_kv8_append(C.byref(cache()), C.byref(append()), None) == -8
    assert er.lib().er_qk_norm_rope(C.byref(norm(num_tokens=0)), None) == 0     # nothing to do is not an error


def test_python_layer_refuses_host_tensors(er):
    import torch
    x = torch.zeros(2, 3, 128)
    with pytest.raises(ValueError, match="CUDA"):
        er.QKNormRopeKernel().encode(x, x, torch.zeros(2, dtype=torch.int32))
    codes, scales = torch.zeros(2, 1, 16, 128, dtype=torch.uint8), torch.zeros(2, 1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        er.BlockScaledKVCache.from_tensors(codes, codes, scales, scales)
    with pytest.raises(ValueError, match="multiple of scale_block"):
        er.BlockScaledKVCache(4, 24, 1, 128)
    assert [f.name for f in er.BlockScaledFormat] == ["e4m3", "int8"]


def test_struct_layouts(er):
    """The ctypes structures against the sizes that the C compiler gives the header's."""
    import os
    import subprocess
    import tempfile
    from edgerunner_b200 import _lib
    names = ["er_qk_norm_rope_params", "er_kv8_cache", "er_kv8_append_params", "er_kv8_attention_params"]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "s.c")
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include "er_kv.h"\nint main(void) { %s return 0; }\n' % "".join('printf("%%zu ", sizeof(%s));' % n for n in names))
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), src, "-o", os.path.join(d, "s")], check=True)
        got = subprocess.run([os.path.join(d, "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == [C.sizeof(getattr(_lib, n)) for n in names]

"""Refusals of the 8-bit block-scaled cache and of the head-norm operator that keep kernels inside their buffers; nothing here needs a device."""
import ctypes as C

import pytest

from test_block_scaled_cpu import BASE, INVALID, UNSUPPORTED, append, attention, cache, er, norm  # noqa: F401


@pytest.mark.parametrize("change", [dict(q_norm_weight=BASE + 4), dict(k=BASE, k_out=BASE, num_kv_heads=2, k_token_stride=256, k_head_stride=128, k_out_token_stride=256,
                                                                       k_out_head_stride=128, k_norm_weight=BASE + 12), dict(positions=BASE + 2)])
def test_norm_refuses_misaligned_buffers(er, change):  # noqa: F811
    """Weights are read as pairs of floats: a view at an odd offset would be a misaligned load."""
    assert er.lib().er_qk_norm_rope(C.byref(norm(**change)), None) == INVALID


@pytest.mark.parametrize("change", [dict(k_norm_weight=BASE + 4), dict(query_starts=BASE + 1)])
def test_append_refuses_misaligned_buffers(er, change):  # noqa: F811
    assert er.lib().er_kv8_append(C.byref(cache()), C.byref(append(**change)), None) == INVALID


@pytest.mark.parametrize("field", ["key_scales", "value_scales", "block_tables", "kv_lens", "status"])
def test_cache_refuses_misaligned_words(er, field):  # noqa: F811
    L, c = er.lib(), cache(**{field: BASE + 2})
    assert L.er_kv8_append(C.byref(c), C.byref(append()), None) == INVALID
    assert L.er_kv8_attention_decode(C.byref(c), C.byref(attention()), None) == INVALID
    assert L.er_kv8_attention_prefill(C.byref(c), C.byref(attention()), None) == INVALID


def test_prefill_refuses_misaligned_starts(er):  # noqa: F811
    assert er.lib().er_kv8_attention_prefill(C.byref(cache()), C.byref(attention(query_starts=BASE + 2)), None) == INVALID


def test_python_layer_refuses_misaligned_weights(er):  # noqa: F811
    """The check itself, on a stand-in with the address of a view that starts one float into an aligned buffer."""
    import torch
    from edgerunner_b200 import block_scaled_cache as b

    class View:
        dtype, shape = torch.float32, (128,)

        def __init__(self, at):
            self.at = at

        def is_contiguous(self):
            return True

        def get_device(self):
            return 0

        def data_ptr(self):
            return self.at

    b._types()
    assert b._weight(View(BASE + 8), "w", 128, 0) == BASE + 8
    with pytest.raises(ValueError, match="8-byte"):
        b._weight(View(BASE + 4), "w", 128, 0)


def test_norm_refuses_more_tokens_than_its_counter_holds(er):  # noqa: F811
    """A warp steps by the slots of the whole grid (148 * 4 * 8 at most) from token to token: the number behind the last one has to stay an int."""
    for tokens in (0x7FFFFF00, 0x7FFF0001):
        assert er.lib().er_qk_norm_rope(C.byref(norm(num_tokens=tokens)), None) == UNSUPPORTED
    import torch
    if not torch.cuda.is_available():
        assert er.lib().er_qk_norm_rope(C.byref(norm(num_tokens=0x7FFF0000)), None) == -8      # past the checks of arguments: no device


def test_attention_refuses_windows_whose_arithmetic_leaves_an_int(er):  # noqa: F811
    """Positions go down to -num_tokens (more queries than rows), and the window is subtracted from them."""
    wide = dict(block_table_width=0x7FFFFF00 // 32, block_table_stride=0x7FFFFF00 // 32, num_seqs=1)
    fn = er.lib().er_kv8_attention_prefill
    assert fn(C.byref(cache(**wide)), C.byref(attention(num_tokens=512, sliding_window=0x7FFFFEFF)), None) == UNSUPPORTED
    assert fn(C.byref(cache(**wide)), C.byref(attention(num_tokens=512, sliding_window=5)), None) == UNSUPPORTED
    import torch
    if not torch.cuda.is_available():       # past the checks of arguments: no device
        for tokens, window in ((512, 0), (512, 0x7FFFFFFF), (255, 0x7FFFFEFF)):
            assert fn(C.byref(cache(**wide)), C.byref(attention(num_tokens=tokens, sliding_window=window)), None) == -8


def test_tables_without_columns_need_no_buffer(er):  # noqa: F811
    """No pages yet: an empty table has no address.  With columns it needs one."""
    import torch
    none = dict(block_tables=0, block_table_width=0, block_table_stride=0)
    for fn, p in ((er.lib().er_kv8_attention_decode, attention()), (er.lib().er_kv8_attention_prefill, attention()), (er.lib().er_kv8_append, append())):
        assert fn(C.byref(cache(block_tables=0)), C.byref(p), None) == INVALID
        if not torch.cuda.is_available():       # past the checks of arguments: no device
            assert fn(C.byref(cache(**none)), C.byref(p), None) == -8


def test_packed_structures_are_the_headers(er):  # noqa: F811
    """The calls hand their structures over as packed bytes: size and every field's place against the C compiler's layout of the header."""
    import os
    import subprocess
    import tempfile
    from edgerunner_b200 import _lib
    from edgerunner_b200 import block_scaled_cache as b
    pairs = [("er_qk_norm_rope_params", b._NORM_ROPE), ("er_kv8_cache", b._CACHE), ("er_kv8_append_params", b._APPEND), ("er_kv8_attention_params", b._ATTENTION)]
    prints = ["printf(\"%%zu \", sizeof(%s));" % n + "".join("printf(\"%%zu \", offsetof(%s, %s));" % (n, f[0]) for f in getattr(_lib, n)._fields_) for n, _ in pairs]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "s.c")
        with open(src, "w") as f:
            f.write("#include <stddef.h>\n#include <stdio.h>\n#include \"er_kv.h\"\nint main(void) { %s return 0; }\n" % " ".join(prints))
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), src, "-o", os.path.join(d, "s")], check=True)
        got = [int(x) for x in subprocess.run([os.path.join(d, "s")], capture_output=True, text=True, check=True).stdout.split()]
    for name, packed in pairs:
        kind = getattr(_lib, name)
        fields = [f[0] for f in kind._fields_]
        size, offsets, got = got[0], got[1:1 + len(fields)], got[1 + len(fields):]
        assert size == packed.size == C.sizeof(kind)
        assert offsets == [getattr(kind, f).offset for f in fields]
        values = list(range(1, len(fields) + 1))          # a value of its own for each field, in the header's order
        back = kind.from_buffer_copy(packed.pack(*values))
        assert [getattr(back, f) for f in fields] == values, name
    assert got == []


def test_python_layer_refuses_negative_counts(er):  # noqa: F811
    """A window or a hint below zero is a ValueError that names it, like every other argument the layer refuses."""
    import torch
    cache_ = object.__new__(er.BlockScaledKVCache)
    q, n = torch.zeros(1, 2, 128), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="sliding_window"):
        cache_.attention_decode(q, n[None], n, sliding_window=-1)
    with pytest.raises(ValueError, match="sliding_window"):
        cache_.attention_prefill(q, n, n[None], n, sliding_window=-1)
    with pytest.raises(ValueError, match="max_query_len"):
        cache_.attention_prefill(q, n, n[None], n, max_query_len=-2)

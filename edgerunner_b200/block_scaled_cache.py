"""An 8-bit paged KV cache with one scale per (page, kv head, block of tokens), the operators over it, and head norms with the rotation
as an operator of its own (er_kv8_*, er_qk_norm_rope in include/er_kv.h).  No counterpart in the reference.

Inputs are torch CUDA tensors in float32, float16 or bfloat16: [tokens, heads, head_dim], the last dimension contiguous, any 16-byte
aligned strides before it (so slices of one projection's output go in as they are).  Work is enqueued on `stream`, by default the current
torch stream of the tensors' device; nothing waits, and every call may be captured into a CUDA graph.  A step over a batch:

    QKNormRopeKernel().encode(q, q, positions, q_norm_weight=qw, rope_theta=theta)       # queries, in place
    cache.append(k, v, block_tables, kv_lens, query_starts, k_norm_weight=kw, rope_theta=theta)
    out = cache.attention_prefill(q, query_starts, block_tables, kv_lens)                 # or attention_decode for single tokens
"""
import ctypes as C
import enum

from ._lib import (check, er_kv8_append_params, er_kv8_attention_params, er_kv8_cache, er_qk_norm_rope_params, lib, stream_ptr)

_TYPE = {}


def _types():
    if not _TYPE:
        import torch
        _TYPE.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    return _TYPE


def _stream(stream, device):
    if stream is not None:
        return stream_ptr(stream)
    import torch
    return torch.cuda.current_stream(device).cuda_stream


def _call(fn, device, *args):
    """fn(*args) with the tensors' device current (the C ABI wants it to be)."""
    import torch
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return check(fn(*args))
    return check(fn(*args))


def _rows(x, name, device=None, dtype=None, dim=None):
    if x.dim() != 3 or x.stride(2) != 1:
        raise ValueError("%s must be [tokens, heads, head_dim] with a contiguous last dimension" % name)
    if x.dtype not in _types():
        raise ValueError("%s must be float32, float16 or bfloat16" % name)
    if not x.is_cuda or (device is not None and x.device != device):
        raise ValueError("%s must be a CUDA tensor on the device of the others" % name)
    if dtype is not None and x.dtype != dtype:
        raise ValueError("%s must have the type of the other rows" % name)
    if dim is not None and x.shape[2] != dim:
        raise ValueError("%s must have %d elements a head" % (name, dim))
    return x


def _ints(x, name, shape, device):
    if x.dtype.is_floating_point or x.element_size() != 4 or tuple(x.shape) != shape or x.device != device or x.stride(-1) != 1:
        raise ValueError("%s must be int32 %r, contiguous, on %s" % (name, list(shape), device))
    return x.data_ptr()


def _weight(w, name, dim, device):
    if w is None:
        return None
    if str(w.dtype) != "torch.float32" or tuple(w.shape) != (dim,) or not w.is_contiguous() or w.device != device:
        raise ValueError("%s must be float32 [%d] on %s" % (name, dim, device))
    return w.data_ptr()


class QKNormRopeKernel:
    def encode(self, q, q_out, positions, *, k=None, k_out=None, q_norm_weight=None, k_norm_weight=None, rms_eps=1e-6, rope_theta=10000.0,
               rope_scaling=1.0, partial_rotary_factor=1.0, stream=None):
        """er_qk_norm_rope: every head of q (and k) normed by its root mean square (weight None: not) and rotated at its token's
        position.  An output may be its own input.  positions: int32 [tokens] (None with partial_rotary_factor 0)."""
        _rows(q, "q")
        dev, (tokens, heads, dim) = q.device, q.shape
        p = er_qk_norm_rope_params()
        p.num_tokens, p.num_heads, p.head_dim, p.type = tokens, heads, dim, _types()[q.dtype]
        for name, x, y, at in (("q", q, q_out, 0), ("k", k, k_out, 1)):
            if x is None and y is None and at == 1:
                break
            if x is None or y is None:
                raise ValueError("%s and %s_out come together" % (name, name))
            _rows(x, name, dev, q.dtype, dim)
            _rows(y, name + "_out", dev, q.dtype, dim)
            if x.shape[0] != tokens or y.shape != x.shape:
                raise ValueError("%s_out must have the shape of %s, with as many tokens as q" % (name, name))
            if at == 0:
                p.q, p.q_out = x.data_ptr(), y.data_ptr()
                p.q_token_stride, p.q_head_stride, _ = x.stride()
                p.q_out_token_stride, p.q_out_head_stride, _ = y.stride()
            else:
                p.k, p.k_out, p.num_kv_heads = x.data_ptr(), y.data_ptr(), x.shape[1]
                p.k_token_stride, p.k_head_stride, _ = x.stride()
                p.k_out_token_stride, p.k_out_head_stride, _ = y.stride()
        if positions is not None:
            p.positions = _ints(positions, "positions", (tokens,), dev)
        p.q_norm_weight = _weight(q_norm_weight, "q_norm_weight", dim, dev)
        p.k_norm_weight = _weight(k_norm_weight, "k_norm_weight", dim, dev)
        p.rms_eps, p.rope_theta, p.rope_scaling, p.partial_rotary_factor = rms_eps, rope_theta, rope_scaling, partial_rotary_factor
        if tokens:
            _call(lib().er_qk_norm_rope, dev, C.byref(p), _stream(stream, dev))


class BlockScaledFormat(enum.IntEnum):
    e4m3 = 0    # 8-bit floats, power-of-two scales
    int8 = 1    # integers, scales amax / 127


class BlockScaledKVCache:
    """The pages of one layer.  Which pages belong to a sequence is the caller's (BlockTableAllocator hands them out): every call takes
    block_tables, int32 [sequences, pages], -1 for none, and kv_lens, int32 [sequences]: the rows of each sequence with the call's own
    tokens included, which are its newest ones.  Element = code * scale of (page, kv head, slot // scale_block)."""

    def __init__(self, num_pages, page_size, num_kv_heads, head_dim, format=BlockScaledFormat.e4m3, scale_block=16, device="cuda"):
        import torch
        if page_size <= 0 or scale_block <= 0 or page_size % scale_block:
            raise ValueError("page_size must be a positive multiple of scale_block")
        shape = (num_pages, num_kv_heads, page_size)
        codes = [torch.zeros(*shape, head_dim, dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.zeros(num_pages, num_kv_heads, page_size // scale_block, device=device) for _ in range(2)]
        self._take(codes[0], codes[1], scales[0], scales[1], format)

    @classmethod
    def from_tensors(cls, keys, values, key_scales, value_scales, format=BlockScaledFormat.e4m3):
        """Over buffers that exist: codes uint8 [pages, kv_heads, page_size, head_dim], scales float32 [pages, kv_heads, blocks of a page]."""
        self = cls.__new__(cls)
        self._take(keys, values, key_scales, value_scales, format)
        return self

    def _take(self, keys, values, key_scales, value_scales, format):
        import torch
        if keys.dim() != 4 or keys.dtype != torch.uint8 or not keys.is_cuda or not keys.is_contiguous():
            raise ValueError("keys must be contiguous uint8 [pages, kv_heads, page_size, head_dim] on a CUDA device")
        if values.shape != keys.shape or values.dtype != keys.dtype or values.device != keys.device or not values.is_contiguous():
            raise ValueError("values must be like keys")
        pages, heads, page_size, dim = keys.shape
        for s in (key_scales, value_scales):
            if (s.dim() != 3 or s.shape[:2] != keys.shape[:2] or s.shape[2] == 0 or page_size % s.shape[2] or s.dtype != torch.float32 or
                    s.device != keys.device or not s.is_contiguous() or s.shape != key_scales.shape):
                raise ValueError("scales must be contiguous float32 [pages, kv_heads, page_size / scale_block] beside the codes")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.format = BlockScaledFormat(format)
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = pages, heads, page_size, dim
        self.scale_block = page_size // key_scales.shape[2]
        self.device = keys.device
        self._status = torch.zeros(1, dtype=torch.int32, device=keys.device)

    def _view(self, block_tables, kv_lens):
        n = kv_lens.shape[0]
        if block_tables.dim() != 2 or block_tables.shape[0] != n:
            raise ValueError("block_tables must be [sequences, pages], kv_lens [sequences]")
        v = er_kv8_cache()
        v.keys, v.values, v.key_scales, v.value_scales = (x.data_ptr() for x in (self.keys, self.values, self.key_scales, self.value_scales))
        v.block_tables = _ints(block_tables, "block_tables", tuple(block_tables.shape), self.device)
        v.kv_lens = _ints(kv_lens, "kv_lens", (n,), self.device)
        v.status = self._status.data_ptr()
        v.num_pages, v.page_size, v.scale_block, v.num_kv_heads, v.head_dim = self.num_pages, self.page_size, self.scale_block, self.num_kv_heads, self.head_dim
        v.format, v.num_seqs, v.block_table_width = int(self.format), n, block_tables.shape[1]
        v.block_table_stride = max(block_tables.stride(0), block_tables.shape[1])
        if n > 1 and block_tables.stride(0) < block_tables.shape[1]:
            raise ValueError("rows of block_tables overlap")
        return v

    def append(self, k, v, block_tables, kv_lens, query_starts=None, *, k_norm_weight=None, rms_eps=1e-6, rope_theta=10000.0, rope_scaling=1.0,
               partial_rotary_factor=1.0, stream=None):
        """er_kv8_append: the call's tokens as the newest rows of their sequences.  query_starts: int32 [sequences + 1], the tokens of
        each sequence; None: one each.  partial_rotary_factor 0: keys come rotated already."""
        _rows(k, "k", self.device, None, self.head_dim)
        _rows(v, "v", self.device, k.dtype, self.head_dim)
        if v.shape != k.shape or k.shape[1] != self.num_kv_heads:
            raise ValueError("k and v must be [tokens, %d, %d]" % (self.num_kv_heads, self.head_dim))
        view = self._view(block_tables, kv_lens)
        p = er_kv8_append_params()
        p.k, p.v = k.data_ptr(), v.data_ptr()
        p.k_token_stride, p.k_head_stride, _ = k.stride()
        p.v_token_stride, p.v_head_stride, _ = v.stride()
        if query_starts is not None:
            p.query_starts = _ints(query_starts, "query_starts", (view.num_seqs + 1,), self.device)
        p.k_norm_weight = _weight(k_norm_weight, "k_norm_weight", self.head_dim, self.device)
        p.num_tokens, p.type = k.shape[0], _types()[k.dtype]
        p.rms_eps, p.rope_theta, p.rope_scaling, p.partial_rotary_factor = rms_eps, rope_theta, rope_scaling, partial_rotary_factor
        if k.shape[0]:
            _call(lib().er_kv8_append, self.device, C.byref(view), C.byref(p), _stream(stream, self.device))

    def _attention(self, fn, size_fn, q, out, block_tables, kv_lens, query_starts, query_len, max_query_len, softmax_scale, sliding_window, stream):
        import torch
        _rows(q, "q", self.device, None, self.head_dim)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _rows(out, "out", self.device, q.dtype, self.head_dim)
        if out.shape != q.shape:
            raise ValueError("out must have the shape of q")
        view = self._view(block_tables, kv_lens)
        p = er_kv8_attention_params()
        p.q, p.out = q.data_ptr(), out.data_ptr()
        p.q_token_stride, p.q_head_stride, _ = q.stride()
        p.out_token_stride, p.out_head_stride, _ = out.stride()
        if query_starts is not None:
            p.query_starts = _ints(query_starts, "query_starts", (view.num_seqs + 1,), self.device)
        p.num_tokens, p.num_heads, p.query_len, p.max_query_len, p.type = q.shape[0], q.shape[1], query_len, max_query_len, _types()[q.dtype]
        p.softmax_scale, p.sliding_window = softmax_scale, sliding_window
        if q.shape[0] == 0:
            return out
        size = _call(size_fn, self.device, C.byref(view), C.byref(p))
        # a fresh block of the caching allocator for each call: calls on different streams never share one, and a captured call keeps its own
        if stream is None:
            work = torch.empty(size, dtype=torch.uint8, device=self.device)
        else:
            with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=self.device) if isinstance(stream, int) else stream):
                work = torch.empty(size, dtype=torch.uint8, device=self.device)
        p.workspace, p.workspace_bytes = work.data_ptr(), size
        _call(fn, self.device, C.byref(view), C.byref(p), _stream(stream, self.device))
        return out

    def attention_decode(self, q, block_tables, kv_lens, out=None, query_len=1, softmax_scale=0.0, sliding_window=0, stream=None):
        """er_kv8_attention_decode: query_len tokens for every sequence (q: [sequences * query_len, heads, head_dim])."""
        if query_len < 1 or q.shape[0] != kv_lens.shape[0] * query_len:
            raise ValueError("q must hold query_len tokens for every sequence")
        return self._attention(lib().er_kv8_attention_decode, lib().er_kv8_decode_workspace_bytes, q, out, block_tables, kv_lens, None, query_len, 0,
                               softmax_scale, sliding_window, stream)

    def attention_prefill(self, q, query_starts, block_tables, kv_lens, out=None, max_query_len=0, softmax_scale=0.0, sliding_window=0, stream=None):
        """er_kv8_attention_prefill: a ragged batch, sequence s has the tokens query_starts[s] .. query_starts[s + 1).  max_query_len: no
        sequence has more (0: not known)."""
        return self._attention(lib().er_kv8_attention_prefill, lib().er_kv8_prefill_workspace_bytes, q, out, block_tables, kv_lens, query_starts, 0,
                               max_query_len, softmax_scale, sliding_window, stream)

    def decoded_rows(self, block_table, length):
        """(keys, values) of one sequence, float32 [length, kv_heads, head_dim].  block_table: page ids that cover `length` rows."""
        import torch
        ids = torch.as_tensor(block_table, dtype=torch.int64, device=self.device)[: -(-int(length) // self.page_size)]
        if ids.numel() * self.page_size < length or (ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= self.num_pages)):
            raise ValueError("block_table does not cover %d rows" % length)
        out = []
        for codes, scales in ((self.keys, self.key_scales), (self.values, self.value_scales)):
            x = codes[ids].view(torch.int8 if self.format == BlockScaledFormat.int8 else torch.float8_e4m3fn).to(torch.float32)
            x = x * scales[ids].repeat_interleave(self.scale_block, dim=2)[..., None]
            out.append(x.transpose(1, 2).reshape(-1, self.num_kv_heads, self.head_dim)[:length].contiguous())
        return tuple(out)

    def device_status(self):
        """The sticky status word as an ER_ERR_* code, 0 when nothing was skipped (waits for the device); clear_device_status() resets it."""
        return int(self._status.item())

    def clear_device_status(self):
        self._status.zero_()

"""An 8-bit paged KV cache with one scale per (page, kv head, block of tokens), the operators over it, and head norms with the rotation
as an operator of its own (er_kv8_*, er_qk_norm_rope in include/er_kv.h).  No counterpart in the reference.

Inputs are torch CUDA tensors in float32, float16 or bfloat16: [tokens, heads, head_dim], the last dimension contiguous, any 16-byte
aligned strides before it (so slices of one projection's output go in as they are).  Work is enqueued on `stream`, by default the current
torch stream of the tensors' device; nothing waits, and every call may be captured into a CUDA graph.  With an explicit `stream` the inputs have
to be ready on it; an output that the call allocates is that stream's memory, kept until the current stream is done with it too.  A step over a batch:

    QKNormRopeKernel().encode(q, q, positions, q_norm_weight=qw, rope_theta=theta)       # queries, in place
    cache.append(k, v, block_tables, kv_lens, query_starts, k_norm_weight=kw, rope_theta=theta)
    out = cache.attention_prefill(q, query_starts, block_tables, kv_lens)                 # or attention_decode for single tokens
"""
import enum
import struct

from ._lib import check, lib, stream_ptr

# The parameter structures of include/er_kv.h as packed bytes: one call instead of some thirty attribute writes, which cost more than a
# small kernel runs for.  Field order as in the header (a test compares sizes and every field's place with the compiler's).
_NORM_ROPE = struct.Struct("@4P8q3P5I4f4x")
_CACHE = struct.Struct("@7P9I4x")
_APPEND = struct.Struct("@2P4q2P2I4f")
_ATTENTION = struct.Struct("@2P4qP5IfIPQ")

_TYPE = {}
_torch = None    # imported with the first tensor, like everywhere in this package


def _types():
    global _torch
    if _torch is None:
        import torch
        _TYPE.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        _torch = torch
    return _TYPE


def _stream(stream, index):
    if stream is not None:
        return stream_ptr(stream)
    raw = getattr(_torch._C, "_cuda_getCurrentRawStream", None)      # the same without a Stream object
    return raw(index) if raw is not None else _torch.cuda.current_stream(index).cuda_stream


def _call(fn, index, *args):
    """fn(*args) with the tensors' device current (the C ABI wants it to be)."""
    if _torch.cuda.current_device() != index:
        with _torch.cuda.device(index):
            return check(fn(*args))
    rc = fn(*args)
    return rc if rc >= 0 else check(rc)


def _rows(x, name, index=None, dtype=None, dim=None):
    """(address, token stride, head stride, tokens, heads) of [tokens, heads, head_dim] rows."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or (stride[2] != 1 and shape[2] != 1):
        raise ValueError("%s must be [tokens, heads, head_dim] with a contiguous last dimension" % name)
    at = x.get_device()
    if at < 0 or (index is not None and at != index):
        raise ValueError("%s must be a CUDA tensor on the device of the others" % name)
    if dtype is not None and x.dtype is not dtype:
        raise ValueError("%s must have the type of the other rows" % name)
    if dim is not None and shape[2] != dim:
        raise ValueError("%s must have %d elements a head" % (name, dim))
    return x.data_ptr(), stride[0], stride[1], shape[0], shape[1]


def _type(x, name):
    t = _types().get(x.dtype)
    if t is None:
        raise ValueError("%s must be float32, float16 or bfloat16" % name)
    return t


def _ints(x, name, shape, index):
    if x.dtype is not _torch.int32 or x.shape != shape or x.get_device() != index or (x.stride(-1) != 1 and shape[-1] > 1):
        raise ValueError("%s must be int32 %r, contiguous, on CUDA device %d" % (name, list(shape), index))
    return x.data_ptr()


def _weight(w, name, dim, index):
    if w is None:
        return 0
    if w.dtype is not _torch.float32 or w.shape != (dim,) or not w.is_contiguous() or w.get_device() != index:
        raise ValueError("%s must be float32 [%d] on CUDA device %d" % (name, dim, index))
    p = w.data_ptr()
    if p & 7:
        raise ValueError("%s must start on an 8-byte boundary (a view at an odd offset of a larger buffer does not)" % name)
    return p


class QKNormRopeKernel:
    def encode(self, q, q_out, positions, *, k=None, k_out=None, q_norm_weight=None, k_norm_weight=None, rms_eps=1e-6, rope_theta=10000.0,
               rope_scaling=1.0, partial_rotary_factor=1.0, stream=None):
        """er_qk_norm_rope: every head of q (and k) normed by its root mean square (weight None: not) and rotated at its token's
        position.  An output may be its own input.  positions: int32 [tokens] (None with partial_rotary_factor 0)."""
        kind = _type(q, "q")
        dt, index, dim = q.dtype, q.get_device(), q.shape[-1]
        qp, qt, qh, tokens, heads = _rows(q, "q")
        op, ot, oh, *shape = _rows(q_out, "q_out", index, dt, dim)
        if shape != [tokens, heads]:
            raise ValueError("q_out must have the shape of q")
        kp = kt = kh = kop = kot = koh = kv_heads = 0
        if k is not None or k_out is not None:
            if k is None or k_out is None:
                raise ValueError("k and k_out come together")
            kp, kt, kh, *shape = _rows(k, "k", index, dt, dim)
            kop, kot, koh, *out_shape = _rows(k_out, "k_out", index, dt, dim)
            kv_heads = shape[1]
            if shape != out_shape or shape[0] != tokens:
                raise ValueError("k_out must have the shape of k, with as many tokens as q")
        pos = 0 if positions is None else _ints(positions, "positions", (tokens,), index)
        if tokens:
            _call(lib().er_qk_norm_rope, index, _NORM_ROPE.pack(
                qp, op, kp, kop, qt, qh, ot, oh, kt, kh, kot, koh, pos, _weight(q_norm_weight, "q_norm_weight", dim, index),
                _weight(k_norm_weight, "k_norm_weight", dim, index), tokens, heads, kv_heads, dim, kind, rms_eps, rope_theta, rope_scaling,
                partial_rotary_factor), _stream(stream, index))


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
        self._index = keys.get_device()
        self._buffers = tuple(x.data_ptr() for x in (keys, values, key_scales, value_scales))
        self._status_ptr = self._status.data_ptr()
        self._shape = (pages, page_size, self.scale_block, heads, dim, int(self.format))
        self._workspace_bytes = {}     # by the shape of a call

    def _view(self, block_tables, kv_lens):
        """(er_kv8_cache bytes, sequences)"""
        n, index = kv_lens.shape[0], self._index
        shape, stride = block_tables.shape, block_tables.stride()
        if len(shape) != 2 or shape[0] != n:
            raise ValueError("block_tables must be [sequences, pages], kv_lens [sequences]")
        if n > 1 and stride[0] < shape[1]:
            raise ValueError("rows of block_tables overlap")
        return _CACHE.pack(*self._buffers, _ints(block_tables, "block_tables", shape, index), _ints(kv_lens, "kv_lens", (n,), index), self._status_ptr,
                           *self._shape, n, shape[1], max(stride[0], shape[1])), n

    def append(self, k, v, block_tables, kv_lens, query_starts=None, *, k_norm_weight=None, rms_eps=1e-6, rope_theta=10000.0, rope_scaling=1.0,
               partial_rotary_factor=1.0, stream=None):
        """er_kv8_append: the call's tokens as the newest rows of their sequences.  query_starts: int32 [sequences + 1], the tokens of
        each sequence; None: one each.  partial_rotary_factor 0: keys come rotated already."""
        index = self._index
        kind = _type(k, "k")
        kp, kt, kh, tokens, heads = _rows(k, "k", index, None, self.head_dim)
        vp, vt, vh, *shape = _rows(v, "v", index, k.dtype, self.head_dim)
        if shape != [tokens, heads] or heads != self.num_kv_heads:
            raise ValueError("k and v must be [tokens, %d, %d]" % (self.num_kv_heads, self.head_dim))
        view, n = self._view(block_tables, kv_lens)
        starts = 0 if query_starts is None else _ints(query_starts, "query_starts", (n + 1,), index)
        if tokens:
            _call(lib().er_kv8_append, index, view, _APPEND.pack(
                kp, vp, kt, kh, vt, vh, starts, _weight(k_norm_weight, "k_norm_weight", self.head_dim, index), tokens, kind, rms_eps, rope_theta,
                rope_scaling, partial_rotary_factor), _stream(stream, index))

    def _empty(self, shape, dtype, stream):
        """Memory of the stream that the kernel runs on: another stream's block of the caching allocator may still be in use there."""
        if stream is None:
            return _torch.empty(shape, dtype=dtype, device=self.device)
        with _torch.cuda.stream(_torch.cuda.ExternalStream(stream, device=self.device) if isinstance(stream, int) else stream):
            return _torch.empty(shape, dtype=dtype, device=self.device)

    def _attention(self, fn, size_fn, q, out, block_tables, kv_lens, query_starts, query_len, max_query_len, softmax_scale, sliding_window, stream):
        if sliding_window < 0 or max_query_len < 0:
            raise ValueError("sliding_window and max_query_len must not be negative (0: none, not known)")
        index = self._index
        kind = _type(q, "q")
        if out is None:
            out = self._empty(q.shape, q.dtype, stream)
            if stream is not None:       # the caller's stream will read it
                out.record_stream(_torch.cuda.current_stream(index))
        qp, qt, qh, tokens, heads = _rows(q, "q", index, None, self.head_dim)
        op, ot, oh, *shape = _rows(out, "out", index, q.dtype, self.head_dim)
        if shape != [tokens, heads]:
            raise ValueError("out must have the shape of q")
        view, n = self._view(block_tables, kv_lens)
        starts = 0 if query_starts is None else _ints(query_starts, "query_starts", (n + 1,), index)
        if tokens == 0:
            return out
        # a fresh block of the caching allocator for each call: calls on different streams never share one, and a captured call keeps its own
        key = (n, block_tables.shape[1], tokens, heads, query_len, max_query_len, kind, sliding_window)
        size = self._workspace_bytes.get(key)
        if size is None:
            if len(self._workspace_bytes) > 256:
                self._workspace_bytes.clear()
            size = self._workspace_bytes[key] = _call(size_fn, index, view, _ATTENTION.pack(
                qp, op, qt, qh, ot, oh, starts, tokens, heads, query_len, max_query_len, kind, softmax_scale, sliding_window, 0, 0))
        work = None
        if size:
            work = _torch.empty(size, dtype=_torch.uint8, device=self.device) if stream is None else self._empty((size,), _torch.uint8, stream)
        _call(fn, index, view, _ATTENTION.pack(qp, op, qt, qh, ot, oh, starts, tokens, heads, query_len, max_query_len, kind, softmax_scale, sliding_window,
                                               work.data_ptr() if size else 0, size), _stream(stream, index))
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
        """The sticky status word as an ER_ERR_* code, 0 when nothing was skipped (waits for the device, calls on every stream); clear_device_status()
        resets it, in the order of the current stream."""
        import torch
        torch.cuda.synchronize(self.device)
        return int(self._status.item())

    def clear_device_status(self):
        self._status.zero_()

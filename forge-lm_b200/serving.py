"""Serving operators on torch CUDA tensors (include/forge_b200.h, "serving
operators"): a paged K/V cache that is quantised as it is written, attention
of single tokens or drafted trees over it, linear layers with 4-bit weights,
and penalties, biases and grammar masks on logits.

Every call runs the library's kernels on torch's current stream of the
tensors' device and returns without waiting.  Results and workspaces come from
torch's allocator.  Nothing here records gradients.  Wrong shapes, types or
devices raise ArgumentError before anything is launched.
"""
from __future__ import annotations

import ctypes as C
import math
import struct

from . import _native as N
from ._native import ArgumentError

__all__ = ["QuantKvCache", "W4Linear", "logit_controls"]

_FORMATS = {"int8": N.FB2_KVQ_INT8, "int4": N.FB2_KVQ_INT4}
_CACHE = struct.Struct("=QQ6i")
_ATTENTION = struct.Struct("=8Q4q8ifi")
_LINEAR = struct.Struct("=QQQ4i")
_CONTROL = struct.Struct("=12Q4q6i")

_torch = None
_codes: dict = {}
_stream = _device = None


def _t():
    """torch, imported at the first use: the rest of the package does without it."""
    global _torch, _stream, _device
    if _torch is None:
        import torch
        _codes.update({torch.float32: N.FB2_F32, torch.bfloat16: N.FB2_BF16, torch.float16: N.FB2_F16})
        # the handle itself: a Stream object costs more than a small kernel
        _stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _device = torch.cuda.current_device
        _torch = torch
    return _torch


def _refuse(message: str):
    raise ArgumentError(N.FB2_INVALID_ARG, message)


def _need(ok: bool, message: str) -> None:
    if not ok:
        _refuse(message)


def _code(dtype) -> int:
    code = _codes.get(dtype)
    if code is None:
        _refuse(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    return code


def _plain(t, name: str, dtype, index: int) -> int:
    """Address of a contiguous tensor of `dtype` on CUDA device `index`; 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous {dtype} tensor on cuda:{index}")
    return t.data_ptr()


def _run(index: int, fn, *args) -> None:
    """fn(*args, stream) on device `index`'s current stream."""
    if _device() == index:
        status = fn(*args, _stream(index))
    else:
        with _torch.cuda.device(index):
            status = fn(*args, _stream(index))
    if status:
        N.check(status)


class _Workspace:
    """Scratch memory of a handle, one buffer for each stream that uses it:
    calls of one stream run one after the other.  A call that is captured in a
    graph gets a buffer of the graph's own, as its replays run elsewhere."""

    def __init__(self):
        self.buffers: dict = {}

    def address(self, index: int, size: int) -> int:
        if _torch.cuda.is_current_stream_capturing():
            return _torch.empty(size, dtype=_torch.uint8, device=f"cuda:{index}").data_ptr()
        stream = _stream(index)
        held = self.buffers.get(stream)
        if held is None or held[1] < size:
            buffer = _torch.empty(size, dtype=_torch.uint8, device=f"cuda:{index}")
            held = self.buffers[stream] = (buffer, size, buffer.data_ptr())
        return held[2]


class QuantKvCache:
    """One layer's paged, quantised K/V cache over two buffers:

      codes uint8 [pages][kv heads][2: K, V][page size][row bytes]
      meta  int32 [pages][kv heads][2][page size]

    fmt "int8": row bytes = head_dim, byte = code + 128, meta = bits of the
    fp32 scale, value = code * scale; "int4": row bytes = head_dim / 2, low
    nibble first, meta = bf16 bits of scale | minimum << 16, value = minimum +
    scale * code.  A slot is page * page_size + offset.  The object holds the
    buffers; `empty` makes new ones."""

    def __init__(self, codes, meta, head_dim: int, fmt: str = "int8"):
        torch = _t()
        _need(fmt in _FORMATS, "fmt must be 'int8' or 'int4'")
        _need(codes.dim() == 5 and codes.shape[2] == 2 and codes.dtype is torch.uint8 and codes.is_cuda,
              "codes must be a CUDA uint8 tensor [pages, kv heads, 2, page size, row bytes]")
        _need(head_dim == codes.shape[4] * (1 if fmt == "int8" else 2), f"row bytes do not fit head_dim {head_dim}")
        _need(tuple(meta.shape) == tuple(codes.shape[:4]), "meta must be [pages, kv heads, 2, page size]")
        self.device, self._index = codes.device, codes.get_device()
        p_codes = _plain(codes, "codes", torch.uint8, self._index)
        p_meta = _plain(meta, "meta", torch.int32, self._index)
        self.codes, self.meta = codes, meta
        self.n_pages, self.n_kv_heads, _, self.page_size, _ = codes.shape
        self.head_dim, self.fmt = int(head_dim), fmt
        _need(self.n_pages * self.page_size <= 2 ** 31 - 1, "the cache must have at most 2^31 - 1 slots")
        self._desc = _CACHE.pack(p_codes, p_meta, self.n_pages, self.page_size, self.n_kv_heads, self.head_dim,
                                 _FORMATS[fmt], 0)
        size = C.c_int64()
        L = N.load()
        N.check(L.fb2_kvq_sizes(self._desc, C.byref(size), C.byref(C.c_int64())))
        self._write, self._read, self._attend = L.fb2_kvq_write, L.fb2_kvq_read, L.fb2_kvq_attend
        self._attend_workspace = L.fb2_kvq_attend_workspace
        self._workspace, self._sizes = _Workspace(), {}
        self._scale = 1.0 / math.sqrt(self.head_dim)

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, fmt: str = "int8",
              device="cuda") -> "QuantKvCache":
        """A cache of new buffers whose rows all stand for zeros."""
        torch = _t()
        _need(fmt in _FORMATS, "fmt must be 'int8' or 'int4'")
        row = head_dim if fmt == "int8" else head_dim // 2
        codes = torch.full((n_pages, n_kv_heads, 2, page_size, row), 128 if fmt == "int8" else 0, dtype=torch.uint8,
                           device=device)
        meta = torch.zeros((n_pages, n_kv_heads, 2, page_size), dtype=torch.int32, device=device)
        return cls(codes, meta, head_dim, fmt)

    def _rows(self, t, name: str, rows: int, heads: int):
        if tuple(t.shape) != (rows, heads, self.head_dim):
            _refuse(f"{name} must be [{rows}, {heads}, {self.head_dim}]")
        stride = t.stride()
        if stride[2] != 1 or t.get_device() != self._index:
            _refuse(f"{name} must be on {self.device} with a contiguous last dimension")
        return stride

    def write(self, k, v, slots) -> None:
        """Quantises rows k, v [rows, kv heads, head_dim] (any row and head
        strides) into the slots (int32, one per row, distinct; a negative one
        skips its row)."""
        rows, heads = slots.numel(), self.n_kv_heads
        ks, vs = self._rows(k, "k", rows, heads), self._rows(v, "v", rows, heads)
        dtype = k.dtype
        if v.dtype is not dtype:
            _refuse("k and v must have the same dtype")
        _run(self._index, self._write, self._desc, rows, k.data_ptr(), v.data_ptr(), _code(dtype), ks[0], ks[1], vs[0], vs[1],
             _plain(slots, "slots", _torch.int32, self._index))

    def read(self, slots, dtype=None):
        """(k, v) [rows, kv heads, head_dim] of the slots as `dtype` (default
        float32); a slot outside the cache reads as zeros."""
        dtype = dtype or _torch.float32
        code, rows = _code(dtype), slots.numel()
        where = _plain(slots, "slots", _torch.int32, self._index)
        shape = (rows, self.n_kv_heads, self.head_dim)
        k = _torch.empty(shape, dtype=dtype, device=self.device)
        v = _torch.empty(shape, dtype=dtype, device=self.device)
        _run(self._index, self._read, self._desc, rows, where, k.data_ptr(), v.data_ptr(), code)
        return k, v

    def attend(self, q, page_table, prefix_lens, starts=None, mask=None, scale: float | None = None,
               max_nodes: int | None = None, max_len: int | None = None):
        """(out, lse) of rows q [rows, heads, head_dim] over the cache.

        Sequence b's rows are q[starts[b]:starts[b+1]] (starts None: one row
        per sequence); its row i is the token at position prefix_lens[b] + i,
        already written to the cache, whose pages page_table[b] lists.  A row
        sees every position before prefix_lens[b] and, of its sequence's own
        rows, those whose bit its mask words [rows, words] int32 set (mask
        None: itself and the earlier ones).  scale defaults to
        1 / sqrt(head_dim).  max_nodes and max_len are host bounds of a
        sequence's rows and of prefix + rows (default: all rows, the page
        table's width): the tighter, the better the work is split.  out has
        q's dtype, lse [rows, heads] is float32; a row that sees nothing
        gives zeros and -inf."""
        torch, index = _torch, self._index
        _need(q.dim() == 3, "q must be [rows, heads, head_dim]")
        rows, heads, dim = q.shape
        qs = self._rows(q, "q", rows, heads)
        dtype = q.dtype
        code, i32 = _code(dtype), torch.int32
        if page_table.dim() != 2 or page_table.dtype is not i32 or page_table.get_device() != index:
            _refuse(f"page_table must be an int32 tensor [sequences, pages] on {self.device}")
        seqs, pages = page_table.shape
        row, step = page_table.stride()
        if step != 1 and pages > 1:
            _refuse("page_table must have contiguous rows")
        if prefix_lens.numel() != seqs:
            _refuse("prefix_lens must have one entry per sequence")
        words = 0
        if mask is not None:
            _need(mask.dim() == 2 and mask.shape[0] == rows and mask.shape[1] > 0, "mask must be [rows, words]")
            words = mask.shape[1]
        if starts is None:
            _need(max_nodes is None or max_nodes == 1, "starts is needed for more than one row per sequence")
            max_nodes = 1
        else:
            _need(starts.numel() == seqs + 1, "starts must have one entry more than there are sequences")
            if max_nodes is None:
                max_nodes = max(rows, 1)
        p_prefix = _plain(prefix_lens, "prefix_lens", i32, index)
        p_starts, p_mask = _plain(starts, "starts", i32, index), _plain(mask, "mask", i32, index)
        out = torch.empty((rows, heads, dim), dtype=dtype, device=self.device)
        lse = torch.empty((rows, heads), dtype=torch.float32, device=self.device)
        if rows == 0:
            return out, lse
        sizes = (seqs, rows, heads, code, pages, max_nodes, max_len or 0, words,
                 self._scale if scale is None else scale, 0)
        head = (q.data_ptr(), out.data_ptr(), lse.data_ptr(), page_table.data_ptr(), p_prefix, p_starts, p_mask)
        strides = (qs[0], qs[1], row if row > pages else pages)
        # the workspace's size goes by these numbers alone
        bound = (seqs, rows, heads, pages, max_nodes, max_len)
        size = self._sizes.get(bound)
        if size is None:
            got = C.c_int64()
            N.check(self._attend_workspace(self._desc, _ATTENTION.pack(*head, 0, 0, *strides, *sizes), C.byref(got)))
            if len(self._sizes) >= 1024:
                self._sizes.clear()
            size = self._sizes[bound] = got.value
        work = self._workspace.address(index, size) if size else 0
        _run(index, self._attend, self._desc, _ATTENTION.pack(*head, work, size, *strides, *sizes))
        return out, lse


class W4Linear:
    """y = x W + bias with W [in][out] in 4-bit codes and, for each output
    and group of 32, 64 or 128 inputs, a bf16 scale and minimum: blocks of 16
    outputs x 64 inputs, padded up.

      codes int32 [ceil(out/16)][ceil(in/64)][32][4]
      meta  int32 [ceil(out/16)][ceil(in/group)][16]

    (the bits' places: include/forge_b200.h, fb2_w4_linear)."""

    def __init__(self, codes, meta, in_features: int, out_features: int, group: int, bias=None):
        torch = _t()
        _need(codes.is_cuda, "codes must be a CUDA tensor")
        self.device, self._index = codes.device, codes.get_device()
        p_codes = _plain(codes, "codes", torch.int32, self._index)
        p_meta = _plain(meta, "meta", torch.int32, self._index)
        p_bias = _plain(bias, "bias", torch.float32, self._index)
        _need(bias is None or bias.numel() == out_features, "bias must have out_features entries")
        self.codes, self.meta, self.bias = codes, meta, bias
        self.in_features, self.out_features, self.group = int(in_features), int(out_features), int(group)
        self._desc = _LINEAR.pack(p_codes, p_meta, p_bias, self.in_features, self.out_features, self.group, 0)
        L = N.load()
        n_codes, n_meta = C.c_int64(), C.c_int64()
        N.check(L.fb2_w4_sizes(self._desc, C.byref(n_codes), C.byref(n_meta)))
        _need(codes.numel() * 4 == n_codes.value and meta.numel() * 4 == n_meta.value,
              f"codes and meta must have {n_codes.value} and {n_meta.value} bytes")
        self._matvec, self._matvec_workspace = L.fb2_w4_matvec, L.fb2_w4_matvec_workspace
        self._workspace, self._sizes = _Workspace(), {}

    @classmethod
    def pack(cls, w, group: int = 64, bias=None) -> "W4Linear":
        """Quantises W [in, out] (the layout of the model's projections)."""
        torch = _t()
        _need(w.dim() == 2 and w.is_cuda and (w.stride(1) == 1 or w.shape[1] == 1),
              "w must be a CUDA tensor [in, out] with contiguous rows")
        _need(group in (32, 64, 128), "group must be 32, 64 or 128")
        k, n = w.shape
        blocks = -(-n // 16)
        codes = torch.zeros((blocks, -(-k // 64), 32, 4), dtype=torch.int32, device=w.device)
        meta = torch.zeros((blocks, -(-k // group), 16), dtype=torch.int32, device=w.device)
        self = cls(codes, meta, k, n, group, bias)
        _run(self._index, N.load().fb2_w4_pack, self._desc, w.data_ptr(), _code(w.dtype), max(w.stride(0), n))
        return self

    def __call__(self, x):
        """x [..., in] -> [..., out] in x's dtype; sums in fp32."""
        k, n, index, shape = self.in_features, self.out_features, self._index, x.shape
        if len(shape) == 0 or shape[-1] != k or x.get_device() != index:
            _refuse(f"x must be [..., {k}] on {self.device}")
        dtype = x.dtype
        code = _code(dtype)
        flat = x if len(shape) == 2 else x.reshape(-1, k)
        row, step = flat.stride()
        if step != 1 and k != 1:
            _refuse("x must have a contiguous last dimension")
        rows = flat.shape[0]
        y = _torch.empty((*shape[:-1], n), dtype=dtype, device=self.device)
        if rows == 0:
            return y
        size = self._sizes.get((rows, code))
        if size is None:
            got = C.c_int64()
            N.check(self._matvec_workspace(self._desc, rows, code, C.byref(got)))
            if len(self._sizes) >= 1024:
                self._sizes.clear()
            size = self._sizes[(rows, code)] = got.value
        work = self._workspace.address(index, size) if size else None
        _run(index, self._matvec, self._desc, rows, flat.data_ptr(), row, y.data_ptr(), n, code, work, size)
        return y


def logit_controls(logits, *, tokens=None, token_starts=None, repetition=None, presence=None, frequency=None,
                   bias_ids=None, bias_values=None, bias_starts=None, allowed=None, mask_rows=None, out=None):
    """Penalties, biases and grammar masks on logit rows [rows, vocab].

    tokens int32 holds the rows' windows back to back, row r's from
    token_starts[r] to token_starts[r + 1]; repetition, presence and frequency
    are float32 [rows].  bias_ids / bias_values (float32) / bias_starts list
    each row's biases; allowed int32 [masks, words] are grammar masks (bit
    v % 32 of word v / 32 allows id v) and mask_rows int32 [rows] each row's
    mask (outside the masks: none; None: mask r).  For an id that the row's
    window holds c > 0 times: l * repetition where l < 0, else l / repetition;
    then - presence - frequency * c.  Then the bias is added and what the mask
    does not allow becomes -inf.  Computed in fp32; the result has the logits'
    dtype and goes to `out` (which may be `logits`) or a new tensor."""
    torch = _t()
    if logits.dim() != 2 or not logits.is_cuda:
        _refuse("logits must be a CUDA tensor [rows, vocab]")
    rows, vocab = logits.shape
    row, step = logits.stride()
    index, dtype = logits.get_device(), logits.dtype
    code = _code(dtype)
    if step != 1 and vocab > 1:
        _refuse("logits must have contiguous rows")
    if out is None:
        out = torch.empty((rows, vocab), dtype=dtype, device=logits.device)
        out_row = vocab
    else:
        _need(out.shape == logits.shape and out.dtype is dtype and out.get_device() == index and
              (out.stride(1) == 1 or vocab <= 1), "out must have the logits' shape, dtype, device and contiguous rows")
        out_row = out.stride(0)
    i32, f32 = torch.int32, torch.float32
    _need((tokens is None) == (token_starts is None), "tokens and token_starts go together")
    _need(tokens is not None or (repetition is None and presence is None and frequency is None),
          "penalties need tokens")
    _need(token_starts is None or token_starts.numel() == rows + 1, "token_starts must have rows + 1 entries")
    _need((bias_ids is None) == (bias_values is None) == (bias_starts is None),
          "bias_ids, bias_values and bias_starts go together")
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency), ("mask_rows", mask_rows)):
        if t is not None and t.numel() != rows:
            raise ArgumentError(N.FB2_INVALID_ARG, f"{name} must have one entry per row")
    n_biases = 0
    if bias_ids is not None:
        _need(bias_starts.numel() == rows + 1, "bias_starts must have rows + 1 entries")
        n_biases = bias_ids.numel()
        _need(bias_values.numel() == n_biases, "bias_values must have one entry per id")
    n_masks = words = 0
    if allowed is not None:
        _need(allowed.dim() == 2, "allowed must be [masks, words]")
        n_masks, words = allowed.shape
        _need(mask_rows is not None or n_masks == rows, "allowed must have one mask per row without mask_rows")
    else:
        _need(mask_rows is None, "mask_rows needs allowed")
    args = _CONTROL.pack(
        logits.data_ptr(), out.data_ptr(), _plain(tokens, "tokens", i32, index),
        _plain(token_starts, "token_starts", i32, index), _plain(repetition, "repetition", f32, index),
        _plain(presence, "presence", f32, index), _plain(frequency, "frequency", f32, index),
        _plain(bias_ids, "bias_ids", i32, index), _plain(bias_values, "bias_values", f32, index),
        _plain(bias_starts, "bias_starts", i32, index), _plain(allowed, "allowed", i32, index),
        _plain(mask_rows, "mask_rows", i32, index), row, out_row,
        tokens.numel() if tokens is not None else 0, n_biases, rows, vocab, code, n_masks, words, 0)
    if rows and vocab:
        _run(index, N.load().fb2_logit_controls, args)
    return out

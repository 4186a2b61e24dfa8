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


def _t():
    """torch, imported at the first use: the rest of the package does without it."""
    global _torch
    if _torch is None:
        import torch
        _codes.update({torch.float32: N.FB2_F32, torch.bfloat16: N.FB2_BF16, torch.float16: N.FB2_F16})
        _torch = torch
    return _torch


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ArgumentError(N.FB2_INVALID_ARG, message)


def _code(dtype) -> int:
    code = _codes.get(dtype)
    if code is None:
        raise ArgumentError(N.FB2_INVALID_ARG, f"dtype must be float32, bfloat16 or float16, not {dtype}")
    return code


def _plain(t, name: str, dtype, device) -> int:
    """Address of a contiguous tensor of `dtype` on `device`; 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.device != device or not t.is_contiguous():
        raise ArgumentError(N.FB2_INVALID_ARG, f"{name} must be a contiguous {dtype} tensor on {device}")
    return t.data_ptr()


def _run(device, fn, *args) -> None:
    """fn(*args, stream) on `device`'s current stream."""
    torch = _torch
    if torch.cuda.current_device() == device.index:
        N.check(fn(*args, torch.cuda.current_stream().cuda_stream))
    else:
        with torch.cuda.device(device):
            N.check(fn(*args, torch.cuda.current_stream().cuda_stream))


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
        self.device = codes.device
        p_codes = _plain(codes, "codes", torch.uint8, self.device)
        p_meta = _plain(meta, "meta", torch.int32, self.device)
        self.codes, self.meta = codes, meta
        self.n_pages, self.n_kv_heads, _, self.page_size, _ = codes.shape
        self.head_dim, self.fmt = int(head_dim), fmt
        _need(self.n_pages * self.page_size <= 2 ** 31 - 1, "the cache must have at most 2^31 - 1 slots")
        self._desc = _CACHE.pack(p_codes, p_meta, self.n_pages, self.page_size, self.n_kv_heads, self.head_dim,
                                 _FORMATS[fmt], 0)
        size = C.c_int64()
        self._lib = N.load()
        N.check(self._lib.fb2_kvq_sizes(self._desc, C.byref(size), C.byref(C.c_int64())))

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
        if t.dim() != 3 or t.shape[0] != rows or t.shape[1] != heads or t.shape[2] != self.head_dim:
            raise ArgumentError(N.FB2_INVALID_ARG, f"{name} must be [{rows}, {heads}, {self.head_dim}]")
        stride = t.stride()
        if stride[2] != 1 or t.device != self.device:
            raise ArgumentError(N.FB2_INVALID_ARG, f"{name} must be on {self.device} with a contiguous last dimension")
        return stride

    def write(self, k, v, slots) -> None:
        """Quantises rows k, v [rows, kv heads, head_dim] (any row and head
        strides) into the slots (int32, one per row, distinct; a negative one
        skips its row)."""
        torch = _torch
        rows = slots.numel()
        ks, vs = self._rows(k, "k", rows, self.n_kv_heads), self._rows(v, "v", rows, self.n_kv_heads)
        _need(v.dtype is k.dtype, "k and v must have the same dtype")
        _run(self.device, self._lib.fb2_kvq_write, self._desc, rows, k.data_ptr(), v.data_ptr(), _code(k.dtype), ks[0],
             ks[1], vs[0], vs[1], _plain(slots, "slots", torch.int32, self.device))

    def read(self, slots, dtype=None):
        """(k, v) [rows, kv heads, head_dim] of the slots as `dtype` (default
        float32); a slot outside the cache reads as zeros."""
        torch = _torch
        dtype = dtype or torch.float32
        code = _code(dtype)
        both = torch.empty((2, slots.numel(), self.n_kv_heads, self.head_dim), dtype=dtype, device=self.device)
        k, v = both.unbind(0)
        _run(self.device, self._lib.fb2_kvq_read, self._desc, slots.numel(),
             _plain(slots, "slots", torch.int32, self.device), k.data_ptr(), v.data_ptr(), code)
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
        torch = _torch
        device = self.device
        _need(q.dim() == 3, "q must be [rows, heads, head_dim]")
        rows, heads, _ = q.shape
        qs = self._rows(q, "q", rows, heads)
        code = _code(q.dtype)
        _need(page_table.dim() == 2 and page_table.dtype is torch.int32 and page_table.device == device and
              (page_table.stride(1) == 1 or page_table.shape[1] <= 1),
              f"page_table must be an int32 tensor [sequences, pages] on {device} with contiguous rows")
        seqs, pages = page_table.shape
        _need(prefix_lens.numel() == seqs, "prefix_lens must have one entry per sequence")
        words = 0
        if mask is not None:
            _need(mask.dim() == 2 and mask.shape[0] == rows, "mask must be [rows, words]")
            words = mask.shape[1]
            _need(words > 0, "mask must have words")
        if starts is None:
            _need(max_nodes is None or max_nodes == 1, "starts is needed for more than one row per sequence")
            max_nodes = 1
        else:
            _need(starts.numel() == seqs + 1, "starts must have one entry more than there are sequences")
            if max_nodes is None:
                max_nodes = max(rows, 1)
        out = torch.empty((rows, heads, self.head_dim), dtype=q.dtype, device=device)
        lse = torch.empty((rows, heads), dtype=torch.float32, device=device)
        if rows == 0:
            return out, lse
        fields = [q.data_ptr(), out.data_ptr(), lse.data_ptr(), page_table.data_ptr(),
                  _plain(prefix_lens, "prefix_lens", torch.int32, device),
                  _plain(starts, "starts", torch.int32, device), _plain(mask, "mask", torch.int32, device), 0, 0, qs[0],
                  qs[1], max(page_table.stride(0), pages), seqs, rows, heads, code, pages, max_nodes, max_len or 0, words,
                  1.0 / math.sqrt(self.head_dim) if scale is None else scale, 0]
        size = C.c_int64()
        N.check(self._lib.fb2_kvq_attend_workspace(self._desc, _ATTENTION.pack(*fields), C.byref(size)))
        if size.value:
            workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
            fields[7], fields[8] = workspace.data_ptr(), size.value
        _run(device, self._lib.fb2_kvq_attend, self._desc, _ATTENTION.pack(*fields))
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
        self.device = codes.device
        _need(codes.is_cuda, "codes must be a CUDA tensor")
        p_codes, p_meta = _plain(codes, "codes", torch.int32, self.device), _plain(meta, "meta", torch.int32, self.device)
        p_bias = _plain(bias, "bias", torch.float32, self.device)
        _need(bias is None or bias.numel() == out_features, "bias must have out_features entries")
        self.codes, self.meta, self.bias = codes, meta, bias
        self.in_features, self.out_features, self.group = int(in_features), int(out_features), int(group)
        self._desc = _LINEAR.pack(p_codes, p_meta, p_bias, self.in_features, self.out_features, self.group, 0)
        self._lib = N.load()
        n_codes, n_meta = C.c_int64(), C.c_int64()
        N.check(self._lib.fb2_w4_sizes(self._desc, C.byref(n_codes), C.byref(n_meta)))
        _need(codes.numel() * 4 == n_codes.value and meta.numel() * 4 == n_meta.value,
              f"codes and meta must have {n_codes.value} and {n_meta.value} bytes")

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
        _run(w.device, self._lib.fb2_w4_pack, self._desc, w.data_ptr(), _code(w.dtype), max(w.stride(0), n))
        return self

    def __call__(self, x):
        """x [..., in] -> [..., out] in x's dtype; sums in fp32."""
        torch = _torch
        k, n = self.in_features, self.out_features
        _need(x.dim() >= 1 and x.shape[-1] == k and x.device == self.device, f"x must be [..., {k}] on {self.device}")
        code = _code(x.dtype)
        flat = x if x.dim() == 2 else x.reshape(-1, k)
        _need(flat.stride(1) == 1 or k == 1, "x must have a contiguous last dimension")
        rows = flat.shape[0]
        y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=self.device)
        if rows == 0:
            return y
        size = C.c_int64()
        N.check(self._lib.fb2_w4_matvec_workspace(self._desc, rows, code, C.byref(size)))
        workspace = torch.empty(size.value, dtype=torch.uint8, device=self.device) if size.value else None
        _run(self.device, self._lib.fb2_w4_matvec, self._desc, rows, flat.data_ptr(), flat.stride(0), y.data_ptr(), n, code,
             workspace.data_ptr() if size.value else None, size.value)
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
    device = logits.device
    _need(logits.dim() == 2 and logits.is_cuda and (logits.stride(1) == 1 or logits.shape[1] <= 1),
          "logits must be a CUDA tensor [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    code = _code(logits.dtype)
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=device)
    else:
        _need(out.shape == logits.shape and out.dtype is logits.dtype and out.device == device and
              (out.stride(1) == 1 or vocab <= 1), "out must have the logits' shape, dtype, device and contiguous rows")
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
        logits.data_ptr(), out.data_ptr(), _plain(tokens, "tokens", i32, device),
        _plain(token_starts, "token_starts", i32, device), _plain(repetition, "repetition", f32, device),
        _plain(presence, "presence", f32, device), _plain(frequency, "frequency", f32, device),
        _plain(bias_ids, "bias_ids", i32, device), _plain(bias_values, "bias_values", f32, device),
        _plain(bias_starts, "bias_starts", i32, device), _plain(allowed, "allowed", i32, device),
        _plain(mask_rows, "mask_rows", i32, device), logits.stride(0), out.stride(0),
        tokens.numel() if tokens is not None else 0, n_biases, rows, vocab, code, n_masks, words, 0)
    if rows and vocab:
        _run(device, N.load().fb2_logit_controls, args)
    return out

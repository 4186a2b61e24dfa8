"""Serving operators on torch CUDA tensors (include/forge_b200.h, "serving
operators"): a paged K/V cache that is quantised as it is written, attention
of single tokens or drafted trees over it, linear layers with 4-bit weights,
and penalties, biases and grammar masks on logits.

Every call runs the library's kernels on torch's current stream of the
tensors' device and returns without waiting.  Results and workspaces come from
torch's allocator.  Nothing here computes gradients: a backward pass that comes
to the result of an input that requires one raises (out= refuses such inputs;
what is written to a cache or packed is its values).  Wrong shapes, types or
devices raise ArgumentError before anything is launched.  The checks and calls
are compiled (csrc/serving_binding.cpp).
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import json
import os

from . import _native as N
from ._native import ArgumentError

__all__ = ["QuantKvCache", "W4Linear", "logit_controls"]

_FORMATS = {"int8": N.FB2_KVQ_INT8, "int4": N.FB2_KVQ_INT4}
_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_serving.so")
_calls = None


def _load():
    """The extension module, loaded at the first use: the rest of the package
    does without torch."""
    global _calls
    if _calls is None:
        import torch  # noqa: F401  its libraries have to be there

        N.load()
        if not os.path.exists(_PATH):
            raise OSError(f"_serving.so not built at {_PATH}; run __graft_entry__.build()")
        try:  # what it was built for (build.py)
            with open(_PATH + ".flags") as f:
                built = json.load(f)["torch"]
        except (OSError, ValueError, KeyError):
            built = None  # not known
        if built not in (None, importlib.metadata.version("torch")):
            raise OSError(f"_serving.so was built for torch {built}, not the installed one; run __graft_entry__.build()")
        spec = importlib.util.spec_from_file_location("_serving", _PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.setup(ArgumentError, N.check)
        _calls = module
    return _calls


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ArgumentError(N.FB2_INVALID_ARG, message)


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
        _need(fmt in _FORMATS, "fmt must be 'int8' or 'int4'")
        self._calls = _load()
        self._handle = self._calls.cache_new(codes, meta, head_dim, _FORMATS[fmt])
        self.codes, self.meta, self.device = codes, meta, codes.device
        self.n_pages, self.n_kv_heads, _, self.page_size, _ = codes.shape
        self.head_dim, self.fmt = int(head_dim), fmt

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, fmt: str = "int8",
              device="cuda") -> "QuantKvCache":
        """A cache of new buffers whose rows all stand for zeros."""
        import torch
        _need(fmt in _FORMATS, "fmt must be 'int8' or 'int4'")
        row = head_dim if fmt == "int8" else head_dim // 2
        codes = torch.full((n_pages, n_kv_heads, 2, page_size, row), 128 if fmt == "int8" else 0, dtype=torch.uint8,
                           device=device)
        meta = torch.zeros((n_pages, n_kv_heads, 2, page_size), dtype=torch.int32, device=device)
        return cls(codes, meta, head_dim, fmt)

    def write(self, k, v, slots) -> None:
        """Quantises rows k, v [rows, kv heads, head_dim] (any row and head
        strides) into the slots (int32, one per row, distinct; a negative one
        skips its row)."""
        self._calls.cache_write(self._handle, k, v, slots)

    def read(self, slots, dtype=None):
        """(k, v) [rows, kv heads, head_dim] of the slots as `dtype` (default
        float32); a slot outside the cache reads as zeros."""
        return self._calls.cache_read(self._handle, slots, dtype)

    def attend(self, q, page_table, prefix_lens, starts=None, mask=None, scale: float | None = None,
               max_nodes: int | None = None, max_len: int | None = None):
        """(out, lse) of rows q [rows, heads, head_dim] over the cache.

        Sequence b's rows are q[starts[b]:starts[b+1]] (starts None: one row
        per sequence); its row i is the token at position prefix_lens[b] + i,
        already written to the cache, whose pages page_table[b] lists (an
        expanded table gives all sequences the same pages).  A row
        sees every position before prefix_lens[b] and, of its sequence's own
        rows, those whose bit its mask words [rows, words] int32 set (mask
        None: itself and the earlier ones).  scale defaults to
        1 / sqrt(head_dim).  max_nodes and max_len are host bounds of a
        sequence's rows and of prefix + rows (default: all rows, or as many as
        the mask has bits; the page table's width): the tighter, the better the
        work is split, and several sequences without max_nodes are planned as
        if each had all of the rows.  out has
        q's dtype, lse [rows, heads] is float32; a row that sees nothing, is
        in no sequence or lies past max_nodes of its own gives zeros and -inf."""
        return self._calls.cache_attend(self._handle, q, page_table, prefix_lens, starts, mask, scale, max_nodes, max_len)


class W4Linear:
    """y = x W + bias with W [in][out] in 4-bit codes and, for each output
    and group of 32, 64 or 128 inputs, a bf16 scale and minimum: blocks of 16
    outputs x 64 inputs, padded up.

      codes int32 [ceil(out/16)][ceil(in/64)][32][4]
      meta  int32 [ceil(out/16)][ceil(in/group)][16]

    (the bits' places: include/forge_b200.h, fb2_w4_linear)."""

    def __init__(self, codes, meta, in_features: int, out_features: int, group: int, bias=None):
        self._calls = _load()
        self._handle = self._calls.linear_new(codes, meta, bias, in_features, out_features, group)
        self.codes, self.meta, self.bias, self.device = codes, meta, bias, codes.device
        self.in_features, self.out_features, self.group = int(in_features), int(out_features), int(group)

    @classmethod
    def pack(cls, w, group: int = 64, bias=None) -> "W4Linear":
        """Quantises W [in, out] (the layout of the model's projections)."""
        import torch
        _need(w.dim() == 2 and w.is_cuda, "w must be a CUDA tensor [in, out]")
        _need(group in (32, 64, 128), "group must be 32, 64 or 128")
        k, n = w.shape
        blocks = -(-n // 16)
        codes = torch.zeros((blocks, -(-k // 64), 32, 4), dtype=torch.int32, device=w.device)
        meta = torch.zeros((blocks, -(-k // group), 16), dtype=torch.int32, device=w.device)
        self = cls(codes, meta, k, n, group, bias)
        self._calls.linear_pack(self._handle, w)
        return self

    def __call__(self, x):
        """x [..., in] -> [..., out] in x's dtype; sums in fp32."""
        return self._calls.linear_call(self._handle, x)


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
    dtype and goes to `out` (which may be `logits`, but not overlap it in any
    other way) or a new tensor."""
    return (_calls or _load()).controls(logits, tokens, token_starts, repetition, presence, frequency, bias_ids, bias_values,
                                        bias_starts, allowed, mask_rows, out)

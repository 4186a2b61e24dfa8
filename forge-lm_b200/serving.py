"""Serving operators on torch CUDA tensors (include/forge_b200.h, "serving
operators"): pages of sequences, a paged K/V cache that is quantised as it is
written, attention of single tokens or drafted trees over it, the residual stream
with its norms, linear layers with 4-bit weights or in 8-bit integers, penalties,
biases and grammar masks on logits, and the verification of drafted tokens.

Every call runs the library's kernels on torch's current stream of the
tensors' device and returns without waiting.  Results and workspaces come from
torch's allocator (small results of one call may share an allocation).
Nothing here computes gradients: a backward pass that comes to the result of an
input that requires one raises (out= refuses such inputs), an input with a
forward-mode tangent is refused; what is written to a cache or packed, and
whole-number results, are of the values.  Wrong shapes, types or devices raise
ArgumentError before anything is launched.  The checks and calls are compiled
(csrc/serving_binding.cpp).
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import json
import os

from . import _native as N
from ._native import ArgumentError

__all__ = ["QuantKvCache", "W4Linear", "logit_controls", "PageTable", "W8Linear", "quantise_rows", "residual_norm", "verify_drafts"]

_NORMS = {"layer": N.FB2_NORM_LAYER, "rms": N.FB2_NORM_RMS}
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


class PageTable:
    """Pages of a cache for a number of sequences, kept on the device:

      table  int32 [sequences, pages]  the pages of each, -1 behind them
      lens   int32 [sequences]         tokens of each
      free   int32 [all pages]         free pages, the first n_free entries
      n_free int32 [1]

    (QuantKvCache.attend's page_table is `table`.)  A page belongs to one
    sequence or to the list.  The object holds the buffers; `empty` makes new
    ones."""

    def __init__(self, table, lens, free, n_free, page_size: int):
        self._calls = _load()
        self._handle = self._calls.pages_new(table, lens, free, n_free, page_size)
        self.table, self.lens, self.free, self.n_free = table, lens, free, n_free
        self.page_size, self.device = int(page_size), table.device
        self.n_seqs, self.max_pages = table.shape

    @classmethod
    def empty(cls, n_seqs: int, max_pages: int, n_pages: int, page_size: int, device="cuda") -> "PageTable":
        """Sequences without tokens and all pages free (page 0 is taken first)."""
        import torch

        def ints(shape, value):
            return torch.full(shape, value, dtype=torch.int32, device=device)

        free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(ints((n_seqs, max_pages), -1), ints((n_seqs,), 0), free, ints((1,), n_pages), page_size)

    def extend(self, counts, max_rows: int):
        """(starts, prefix_lens, slots, positions) for counts [sequences] int32
        more tokens of each sequence.

        Sequence b's rows are starts[b]:starts[b+1] of slots and positions
        [max_rows], its length before is prefix_lens[b]; rows behind the last
        have slot -1 and position 0.  These are what QuantKvCache.write and
        .attend take.  Sequences are served in their order: one whose tokens
        would not fit its row of the table (or whose count is negative) asks
        for nothing; of the others one is served if the tokens asked for up to
        it are at most max_rows and, where it needs pages, the pages asked for
        at most the free ones.  What is not served stays as it is and has no
        rows."""
        return self._calls.pages_extend(self._handle, counts, max_rows)

    def truncate(self, lens) -> None:
        """Shortens the sequences to lens [sequences] int32 tokens (one that is
        not longer stays as it is); pages that they no longer need are free.
        A sequence's first tokens stay: the rows of others that are to stay (a
        tree's accepted ones) have to be moved in the cache first."""
        self._calls.pages_truncate(self._handle, lens)


def residual_norm(h, x, weight, bias=None, *, post_weight=None, post_bias=None, gate=None, scale: float = 1.0, kind: str = "layer",
                  eps: float = 1e-5, quantise: bool = False, dtype=None):
    """(s, y) with s = x + scale * gate * post(h) and y = norm(s), over rows
    [rows, dim] with contiguous last dimension; with quantise (s, codes, scales),
    y's rows as quantise_rows makes them.

    kind "layer": (v - mean) / sqrt(variance + eps) * weight + bias, "rms":
    v / sqrt(mean of squares + eps) * weight + bias; weights and biases are
    float32 [dim].  post_weight norms h first; gate [dim] or [rows, dim] has h's
    dtype.  x, the stream, has h's dtype or is float32.  h None: s is x, and y
    has x's dtype or `dtype`.  Computed in fp32, y from s before s is rounded; s
    has x's dtype, y has h's.  A row's sums may be in another order in a call of
    more (over 592) or fewer rows: the last bit, or a code, may differ."""
    _need(kind in _NORMS, "kind must be 'layer' or 'rms'")
    return (_calls or _load()).norm(h, x, weight, bias, post_weight, post_bias, gate, scale, _NORMS[kind], eps, quantise, dtype)


def quantise_rows(x):
    """(codes int8 [rows, columns], scales float32 [rows]) of x [rows, columns]:
    scale = max|x| / 127, code = round(x * (127 / max|x|)).  Rows of codes begin on
    16 bytes.  A row with a non-finite element has scale NaN."""
    return (_calls or _load()).quantise_rows(x)


class W8Linear:
    """y = x W + bias in 8-bit integers: codes int8 [out, in] (rows a multiple of
    16 bytes apart) with a float32 scale for each output, W[i][o] =
    codes[o][i] * scales[o], and rows of x as quantise_rows makes them.  Sums of
    products are exact; scales and bias are applied in fp32."""

    def __init__(self, codes, scales, bias=None):
        self._calls = _load()
        self._handle = self._calls.linear8_new(codes, scales, bias)
        self.codes, self.scales, self.bias, self.device = codes, scales, bias, codes.device
        self.out_features, self.in_features = codes.shape

    @classmethod
    def pack(cls, w, bias=None) -> "W8Linear":
        """Quantises W [in, out] (the layout of the model's projections)."""
        import torch
        _need(w.dim() == 2 and w.is_cuda, "w must be a CUDA tensor [in, out]")
        k, n = w.shape
        codes = torch.zeros((n, -(-k // 16) * 16), dtype=torch.int8, device=w.device)[:, :k]
        self = cls(codes, torch.zeros(n, dtype=torch.float32, device=w.device), bias)
        self._calls.linear8_pack(self._handle, w)
        return self

    def __call__(self, x, scales=None, dtype=None):
        """x [..., in] -> [..., out] in x's dtype (or `dtype`), its rows quantised
        first; or codes int8 x [..., in] with scales, one per row, -> `dtype`
        (default float32).  Codes whose rows do not begin on 16 bytes are copied
        first."""
        return self._calls.linear8_call(self._handle, x, scales, dtype)


def verify_drafts(logits, drafts, uniforms, *, starts=None, parents=None, draft_probs=None, temperature=None, max_nodes: int | None = None):
    """(tokens, nodes, counts): which drafted tokens the target accepts, and the
    token that follows them.

    Sequence b's rows are starts[b]:starts[b+1] (None: one each): its last token,
    then drafts [rows] int32 below it.  parents [rows] int32 counts a row's parent
    from the sequence's first (earlier) row; None: a chain.  logits [rows, vocab]
    are what the target says follows each row, p = softmax(logits / temperature[b])
    (float32; None: 1; 0: all of it on the largest logit).  From the first row on,
    drafts c below a row are tried in order, each with uniforms[c] (float64 in
    [0, 1)).  With draft_probs [rows, vocab] float32 (chains): accepted where
    uniforms[c] * q(c) < p(c), and what may follow a rejected one is max(p - q, 0).
    Without: accepted where uniforms[c] * (1 - p of siblings rejected) < p(c), and
    what may follow is p without the rejected ones.  The last token is the lowest id
    at which the running sum of that passes uniforms[starts[b]] times its total.

    counts [sequences] int32: tokens gained, accepted ones and the last; tokens
    [sequences, max_nodes] int32: these; nodes [sequences, max_nodes] int32: the
    row, counted from the sequence's first, that each of them follows, so the rows
    that stay in the cache; -1 behind them.  Of a chain these are the first rows, and
    PageTable.truncate(prefix_lens + counts) drops the others; of a tree they may lie
    apart, and the cache's rows nodes[b, j] have to be moved to places j before.
    max_nodes (up to 1024) is a host bound of a sequence's rows; later ones are not looked
    at.  A row of logits with a NaN, a +inf or nothing above -inf accepts nothing and
    draws -1."""
    return (_calls or _load()).verify(logits, drafts, uniforms, starts, parents, draft_probs, temperature, max_nodes)

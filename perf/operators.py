"""The serving operators of a compressed decode step, as measured cases.

Four operators that one step of drafting and verifying tokens runs after each
other: projections with 4-bit weights, a paged K/V cache that is quantised as
it is written (and read back), attention for a tree of drafted tokens over
that cache, and the controls (penalties, biases, grammar masks) on the logits
it ends in.  `run` computes each either in elementary torch operations in 32
bits (`own` false) or through the library's public calls (`own` true); both
work on the same device buffers in the documented layouts.

Cache (all integers little endian, C order):
  codes u8  [pages][kv heads][2: K, V][page size][row bytes]
  meta  i32 [pages][kv heads][2: K, V][page size]
  int8: row bytes = head_dim, byte = code + 128, meta = the fp32 scale's bits,
        value = code * scale, scale = max|x| / 127;
  int4: row bytes = head_dim / 2, dimension 2i in the low nibble of byte i and
        2i + 1 in the high one, meta = bf16 bits of (scale | minimum << 16),
        value = minimum + scale * code.
4-bit weights of y = x W (W [in][out]), in blocks of 16 outputs x 64 inputs:
  codes i32 [out/16][in/64][lane 4g+t][word j]; nibble p of a word is output
        8 (p & 1) + g and input 16 t + 4 j + (p & 2) + (p >> 2) of its block;
  meta  i32 [out/16][groups of inputs][16], bf16 (scale | minimum << 16).
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TINY = 1e-35  # a row whose range is below this is stored as a constant


def _package():
    """The library's package (its folder's name is no identifier)."""
    if "forge_lm_b200" not in sys.modules:
        folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forge-lm_b200")
        if os.path.isdir("forge-lm_b200"):
            folder = os.path.abspath("forge-lm_b200")
        spec = importlib.util.spec_from_file_location("forge_lm_b200", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["forge_lm_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["forge_lm_b200"]


# ---- cases --------------------------------------------------------------------

def listed():
    return [
        # one decode step of one sequence of the 98M model: its K and V go into the cache
        {"name": "append-step", "op": "store", "rows": 1, "kv_heads": 12, "head_dim": 64, "page": 16,
         "fmt": "int8", "dtype": "fp32"},
        # a long prompt's chunk goes into a 4-bit cache and comes back as the values attention will see
        {"name": "append-chunk", "op": "store", "rows": 32785, "kv_heads": 8, "head_dim": 128, "page": 32,
         "fmt": "int4", "dtype": "bf16"},
        # a shared prefix of many sequences is read back densely for a prefill over it
        {"name": "read-prefix", "op": "read", "rows": 131072, "kv_heads": 8, "head_dim": 128, "page": 16,
         "fmt": "int8", "dtype": "bf16"},
        # plain decoding: one sequence of the 98M model in the middle of its context (latency)
        {"name": "attend-one", "op": "attend", "seqs": 1, "len_lo": 576, "len_hi": 576, "nodes_lo": 1,
         "nodes_hi": 1, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "fmt": "int8", "dtype": "fp32"},
        # plain decoding: a ragged batch of the 98M model
        {"name": "attend-batch", "op": "attend", "seqs": 32, "len_lo": 64, "len_hi": 1023, "nodes_lo": 1,
         "nodes_hi": 1, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "fmt": "int8", "dtype": "fp32"},
        # plain decoding over long contexts with shared K/V heads, 4-bit cache
        {"name": "attend-long", "op": "attend", "seqs": 16, "len_lo": 40000, "len_hi": 65535, "nodes_lo": 1,
         "nodes_hi": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "fmt": "int4", "dtype": "fp16"},
        # verification of drafted trees over long contexts with shared K/V heads
        {"name": "attend-tree", "op": "attend", "seqs": 4, "len_lo": 9001, "len_hi": 32768, "nodes_lo": 23,
         "nodes_hi": 64, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "fmt": "int8", "dtype": "bf16"},
        # the fused q/k/v projection of the 98M model, one row (latency)
        {"name": "project-step", "op": "project", "rows": 1, "k": 768, "n": 2304, "group": 64, "dtype": "fp32"},
        # one row through a large model's projection
        {"name": "project-large", "op": "project", "rows": 1, "k": 16384, "n": 16384, "group": 128, "dtype": "bf16"},
        # a drafted tree's rows through the tied head of the 220M model
        {"name": "project-tree", "op": "project", "rows": 61, "k": 1024, "n": 16384, "group": 32, "dtype": "fp16"},
        # one sampled token of the 98M model (latency)
        {"name": "control-step", "op": "control", "rows": 1, "vocab": 16384, "window": 576, "biases": 8,
         "masks": 1, "dtype": "fp32"},
        # the rows of several drafted trees over a large vocabulary, each in its grammar's state
        {"name": "control-tree", "op": "control", "rows": 256, "vocab": 131071, "window": 4096, "biases": 300,
         "masks": 40, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "read", "attend", "attend", "attend", "project", "project", "control"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    fmt = rng.choice(["int8", "int4"])
    page = rng.choice([8, 16, 32, 64, 128])
    kv_heads, share = rng.choice([(12, 1), (16, 1), (8, 4), (1, 8), (2, 7), (5, 3), (4, 2)])
    head_dim = rng.choice([32, 64, 64, 80, 128, 128, 256])
    if op in ("store", "read"):
        most = max(1, min(131072, 16000000 // (kv_heads * head_dim)))
        return {"op": op, "rows": _log_int(rng, 1, most), "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
                "fmt": fmt, "dtype": dtype}
    if op == "attend":
        nodes_hi = _log_int(rng, 1, 64) if rng.random() < 0.6 else 1
        nodes_lo = _log_int(rng, 1, nodes_hi)
        seqs = _log_int(rng, 1, 64)
        # tokens over all sequences: by the cache's size, and by the products of wide trees
        most = min(100000000 // (kv_heads * head_dim),
                   int(6e10 / (4.0 * nodes_hi * kv_heads * share * head_dim)))
        len_hi = _log_int(rng, nodes_hi, max(nodes_hi + 1, min(65536, most // seqs)))
        len_lo = _log_int(rng, nodes_hi, len_hi)
        return {"op": op, "seqs": seqs, "len_lo": len_lo, "len_hi": len_hi, "nodes_lo": nodes_lo,
                "nodes_hi": nodes_hi, "heads": kv_heads * share, "kv_heads": kv_heads, "head_dim": head_dim,
                "page": page, "fmt": fmt, "dtype": dtype}
    if op == "project":
        k = _log_int(rng, 64, 16384)
        n = _log_int(rng, 64, min(16384, 100000000 // k))
        rows = _log_int(rng, 1, 64) if rng.random() < 0.6 else 1
        return {"op": op, "rows": rows, "k": k, "n": n, "group": rng.choice([32, 64, 128]), "dtype": dtype}
    vocab = _log_int(rng, 1000, 200000)
    rows = _log_int(rng, 1, min(256, 30000000 // vocab))
    return {"op": op, "rows": rows, "vocab": vocab, "window": _log_int(rng, 1, 8192),
            "biases": min(_log_int(rng, 1, 1000), vocab), "masks": _log_int(rng, 1, rows), "dtype": dtype}


def _spread(lo, hi, count):
    """`count` whole numbers over lo..hi in no order, both ends among them where they fit."""
    if count == 1:
        return [hi]
    step = 7 if count % 7 else 11
    return [lo + (hi - lo) * ((i * step + 3) % count) // (count - 1) for i in range(count)]


def _lens(case):
    """Cached tokens (drafted ones included) and drafted tokens of each sequence."""
    lens = _spread(case["len_lo"], case["len_hi"], case["seqs"])
    nodes = _spread(case["nodes_lo"], case["nodes_hi"], case["seqs"])[::-1]
    return lens, [min(a, b) for a, b in zip(nodes, lens)]


def _row_bytes(case):
    return case["head_dim"] if case["fmt"] == "int8" else case["head_dim"] // 2


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] in ("store", "read"):
        each = 2 * case["kv_heads"]
        dense = case["rows"] * each * case["head_dim"] * size
        coded = case["rows"] * each * (_row_bytes(case) + 4)
        if case["op"] == "store":  # rows in, codes out, codes' values out
            return {"bytes": 2 * dense + coded + 4 * case["rows"], "flops": 0}
        return {"bytes": dense + coded + 4 * case["rows"], "flops": 0}
    if case["op"] == "attend":
        lens, nodes = _lens(case)
        rows, d = sum(nodes), case["head_dim"]
        cached = sum(lens) * case["kv_heads"] * 2 * (_row_bytes(case) + 4)
        words = (case["nodes_hi"] + 31) // 32
        pages = sum(-(-n // case["page"]) for n in lens)
        flops = sum(4 * t * (n - t) + 4 * t for n, t in zip(lens, nodes)) * case["heads"] * d
        return {"bytes": cached + rows * (case["heads"] * (2 * d * size + 4) + 4 * words) + 4 * pages, "flops": flops}
    if case["op"] == "project":
        k, n, rows = case["k"], case["n"], case["rows"]
        groups = -(-k // case["group"])
        return {"bytes": k * n // 2 + groups * n * 4 + rows * (k + n) * size + 4 * n, "flops": 2 * rows * k * n}
    v, rows = case["vocab"], case["rows"]
    return {"bytes": rows * (2 * v * size + 4 * case["window"] + 8 * case["biases"] + 16) + case["masks"] * v // 8,
            "flops": 0}


# ---- inputs ---------------------------------------------------------------------

def _bits(x):
    return x.to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xFFFF


def _from_bits(word):
    """bf16 (low half, high half) of 32-bit words, as fp32."""
    return (word << 16).view(torch.float32), (word & -65536).view(torch.float32)


def _quantise(x, fmt):
    """(bytes, meta) of fp32 rows over the last dimension, by the cache's format."""
    finite = torch.isfinite(x).all(-1, keepdim=True)
    nan = torch.full((), math.nan, device=x.device)
    if fmt == "int8":
        top = x.abs().amax(-1, keepdim=True)
        live = finite & (top >= TINY)
        inv = torch.full((), 127.0, device=x.device) / torch.where(live, top, 1.0)
        code = torch.where(live, torch.round(x * inv).clamp(-127, 127), 0.0)
        scale = torch.where(finite, torch.where(live, top / torch.full((), 127.0, device=x.device), 0.0), nan)
        return (code + 128).to(torch.uint8), scale.squeeze(-1).contiguous().view(torch.int32)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / torch.full((), 15.0, device=x.device)).to(torch.bfloat16).float()
    least = low.to(torch.bfloat16).float()
    finite = finite & torch.isfinite(scale) & torch.isfinite(least)
    live = finite & (scale >= TINY)
    scale = torch.where(live, scale, 0.0)
    inv = 1.0 / torch.where(live, scale, 1.0)
    code = torch.where(live, torch.round((x - least) * inv).clamp(0, 15), 0.0).to(torch.uint8)
    meta = _bits(torch.where(finite, scale, nan)) | (_bits(torch.where(finite, least, nan)) << 16)
    return code[..., 0::2] | (code[..., 1::2] << 4), meta.squeeze(-1)


def _values(codes, meta, fmt):
    """The fp32 values that bytes and meta stand for."""
    if fmt == "int8":
        return (codes.float() - 128.0) * meta.contiguous().view(torch.float32)[..., None]
    scale, least = _from_bits(meta.contiguous())
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return code * scale[..., None] + least[..., None]


def _filled(case, pages, gen):
    """Cache buffers that hold quantised normal values."""
    shape = (pages, case["kv_heads"], 2, case["page"])
    codes = torch.empty(shape + (_row_bytes(case),), dtype=torch.uint8, device=DEV)
    meta = torch.empty(shape, dtype=torch.int32, device=DEV)
    step = max(1, (1 << 27) // (shape[1] * shape[2] * shape[3] * case["head_dim"]))
    for at in range(0, pages, step):
        x = torch.randn((min(step, pages - at),) + shape[1:] + (case["head_dim"],), device=DEV, generator=gen)
        codes[at:at + step], meta[at:at + step] = _quantise(x, case["fmt"])
    return codes, meta


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case, "dtype": dtype}

    def normal(*shape):
        return torch.randn(shape, device=DEV, generator=gen)

    if case["op"] in ("store", "read"):
        rows, heads, dim = case["rows"], case["kv_heads"], case["head_dim"]
        pages = -(-rows * 5 // (4 * case["page"])) + 1
        s["slots"] = torch.randperm(pages * case["page"], device=DEV, generator=gen)[:rows].to(torch.int32)
        if case["op"] == "store":
            # K and V as the fused projection leaves them: [rows][q | k | v]
            qkv = normal(rows, 3 * heads * dim).to(dtype)
            s["k"] = qkv[:, heads * dim:2 * heads * dim].unflatten(1, (heads, dim))
            s["v"] = qkv[:, 2 * heads * dim:].unflatten(1, (heads, dim))
            s["codes"] = torch.full((pages, heads, 2, case["page"], _row_bytes(case)), 128, dtype=torch.uint8, device=DEV)
            s["meta"] = torch.zeros((pages, heads, 2, case["page"]), dtype=torch.int32, device=DEV)
        else:
            s["slots"] = s["slots"].sort().values
            s["codes"], s["meta"] = _filled(case, pages, gen)
    elif case["op"] == "attend":
        lens, nodes = _lens(case)
        pages = [-(-n // case["page"]) for n in lens]
        s["codes"], s["meta"] = _filled(case, sum(pages), gen)
        order = torch.randperm(sum(pages), device=DEV, generator=gen).to(torch.int32)
        s["table"] = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(pages):
            s["table"][i, :n] = order[at:at + n]
            at += n
        starts = [0]
        for t in nodes:
            starts.append(starts[-1] + t)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["prefix"] = torch.tensor([n - t for n, t in zip(lens, nodes)], dtype=torch.int32, device=DEV)
        s["q"] = (2.0 * normal(starts[-1], case["heads"], case["head_dim"])).to(dtype)
        s["mask"] = None
        if case["nodes_hi"] > 1:
            # each drafted token hangs below a random earlier one and sees its ancestors and itself
            words = (case["nodes_hi"] + 31) // 32
            pick = torch.rand(starts[-1], generator=torch.Generator().manual_seed(seed)).tolist()
            rows = []
            for a, b in zip(starts, starts[1:]):
                seen = []
                for i in range(b - a):
                    seen.append((seen[int(pick[a + i] * i)] if i else 0) | 1 << i)
                rows += seen
            flat = [[(r >> 32 * w) & 0xFFFFFFFF for w in range(words)] for r in rows]
            s["mask"] = torch.tensor(flat, dtype=torch.int64, device=DEV).to(torch.int32)
        s["max_len"], s["max_nodes"] = max(lens), max(nodes)
    elif case["op"] == "project":
        k, n, group = case["k"], case["n"], case["group"]
        blocks, deep, groups = -(-n // 16), -(-k // 64), -(-k // group)
        s["codes"] = torch.randint(-2 ** 31, 2 ** 31, (blocks, deep, 32, 4), device=DEV, generator=gen).to(torch.int32)
        scale = 0.003 + 0.004 * torch.rand((blocks, groups, 16), device=DEV, generator=gen)
        least = -7.5 * scale * (1 + 0.1 * normal(blocks, groups, 16))
        s["meta"] = _bits(scale) | (_bits(least) << 16)
        s["bias"] = 0.1 * normal(n)
        s["x"] = normal(case["rows"], k).to(dtype)
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = (4.0 * normal(rows, vocab)).to(dtype)
        # tokens as text repeats them: half of them from few ids
        often = torch.randint(0, max(1, vocab // 50), (rows, case["window"]), device=DEV, generator=gen)
        any_ = torch.randint(0, vocab, (rows, case["window"]), device=DEV, generator=gen)
        half = torch.rand((rows, case["window"]), device=DEV, generator=gen) < 0.5
        s["tokens"] = torch.where(half, often, any_).to(torch.int32).flatten()
        s["token_starts"] = torch.arange(rows + 1, device=DEV, dtype=torch.int32) * case["window"]
        ids = torch.rand((rows, vocab), device=DEV, generator=gen).argsort(1)[:, :case["biases"]]
        s["bias_ids"] = ids.to(torch.int32).flatten()
        s["bias_values"] = 2.0 * normal(rows * case["biases"])
        s["bias_starts"] = torch.arange(rows + 1, device=DEV, dtype=torch.int32) * case["biases"]
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (case["masks"], (vocab + 31) // 32), device=DEV,
                                     generator=gen).to(torch.int32)
        s["mask_rows"] = torch.randint(-1, case["masks"], (rows,), device=DEV, generator=gen).to(torch.int32)
        s["repetition"] = 1.0 + 0.5 * torch.rand(rows, device=DEV, generator=gen)
        s["presence"] = torch.rand(rows, device=DEV, generator=gen) - 0.2
        s["frequency"] = torch.rand(rows, device=DEV, generator=gen) * 0.3
    if own:  # the handles that a program keeps: they hold the same buffers
        pkg = _package()
        if "codes" in s and case["op"] != "project":
            s["cache"] = pkg.QuantKvCache(s["codes"], s["meta"], case["head_dim"], case["fmt"])
        elif case["op"] == "project":
            s["linear"] = pkg.W4Linear(s["codes"], s["meta"], case["k"], case["n"], case["group"], bias=s["bias"])
    return s


# ---- one pass ---------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        if op == "store":
            s["cache"].write(s["k"], s["v"], s["slots"])
            return s["cache"].read(s["slots"], s["dtype"])
        if op == "read":
            return s["cache"].read(s["slots"], s["dtype"])
        if op == "attend":
            return s["cache"].attend(s["q"], s["table"], s["prefix"], starts=s["starts"], mask=s["mask"],
                                     max_nodes=s["max_nodes"], max_len=s["max_len"])
        if op == "project":
            return s["linear"](s["x"])
        return _package().logit_controls(
            s["logits"], tokens=s["tokens"], token_starts=s["token_starts"], repetition=s["repetition"],
            presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
            bias_starts=s["bias_starts"], allowed=s["allowed"], mask_rows=s["mask_rows"])
    return {"store": _store, "read": _read, "attend": _attend, "project": _project, "control": _control}[op](s)


def _store(s):
    case = s["case"]
    page, at = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    for_k, k_meta = _quantise(s["k"].float(), case["fmt"])
    for_v, v_meta = _quantise(s["v"].float(), case["fmt"])
    s["codes"][page, :, 0, at], s["codes"][page, :, 1, at] = for_k, for_v
    s["meta"][page, :, 0, at], s["meta"][page, :, 1, at] = k_meta, v_meta
    return _read(s)


def _read(s):
    case = s["case"]
    page, at = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    k = _values(s["codes"][page, :, 0, at], s["meta"][page, :, 0, at], case["fmt"])
    v = _values(s["codes"][page, :, 1, at], s["meta"][page, :, 1, at], case["fmt"])
    return k.to(s["dtype"]), v.to(s["dtype"])


def _attend(s):
    case = s["case"]
    seqs, kv, dim = case["seqs"], case["kv_heads"], case["head_dim"]
    share, most, wide = case["heads"] // kv, s["max_len"], s["max_nodes"]
    place = torch.arange(most, device=DEV)
    page = s["table"][:, place // case["page"]].long().clamp(min=0)
    at = (place % case["page"]).expand(seqs, most)
    k = _values(s["codes"][page, :, 0, at], s["meta"][page, :, 0, at], case["fmt"])  # [seqs, most, kv, dim]
    v = _values(s["codes"][page, :, 1, at], s["meta"][page, :, 1, at], case["fmt"])
    first, last = s["starts"][:-1].long(), s["starts"][1:].long()
    node = torch.arange(wide, device=DEV)
    live = node < (last - first)[:, None]                                            # [seqs, wide]
    row = torch.where(live, first[:, None] + node, 0)
    q = s["q"].float()[row].unflatten(2, (kv, share)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [seqs, kv, wide*share, dim]
    scores = (q @ k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(dim))
    drafted = place - s["prefix"].long()[:, None]                                     # [seqs, most]
    sees = (drafted[:, None] < 0).expand(seqs, wide, most)
    inside = (drafted >= 0) & (drafted < (last - first)[:, None])
    if s["mask"] is None:
        bit = drafted[:, None] <= node[:, None]
    else:
        j = torch.where(inside, drafted, 0)
        word = s["mask"].long()[row].gather(2, (j >> 5)[:, None].expand(seqs, wide, most))
        bit = ((word >> (j & 31)[:, None]) & 1).bool()
    sees = sees | (inside[:, None] & bit)
    sees = sees.repeat_interleave(share, 1)[:, None]
    scores = scores.masked_fill(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    lse = top + torch.log(total)
    where = live.flatten().nonzero().squeeze(1)
    out = out.unflatten(2, (wide, share)).permute(0, 2, 1, 3, 4).flatten(2, 3).flatten(0, 1)[where]
    lse = lse.squeeze(-1).unflatten(2, (wide, share)).permute(0, 2, 1, 3).flatten(2, 3).flatten(0, 1)[where]
    return out.to(s["dtype"]), lse


def _weights(s):
    """W^T [out][in] in fp32 of the packed codes."""
    case = s["case"]
    k, n, blocks, deep = case["k"], case["n"], s["codes"].shape[0], s["codes"].shape[1]
    nibble = (s["codes"][..., None] >> (4 * torch.arange(8, device=DEV))) & 15
    # lane (g, t), word j, nibble (second of its pair, which pair, which half of the outputs)
    code = nibble.to(torch.uint8).reshape(blocks, deep, 8, 4, 4, 2, 2, 2).permute(0, 7, 2, 1, 3, 4, 6, 5)
    code = code.reshape(blocks * 16, deep * 64)[:n, :k].float()
    scale, least = _from_bits(s["meta"].permute(0, 2, 1).reshape(blocks * 16, -1)[:n].contiguous())
    group = torch.arange(k, device=DEV) // case["group"]
    return code * scale[:, group] + least[:, group]


def _project(s):
    return (s["x"].float() @ _weights(s).T + s["bias"]).to(s["dtype"])


def _control(s):
    case = s["case"]
    rows, vocab = case["rows"], case["vocab"]
    x = s["logits"].float()
    owner = torch.arange(rows, device=DEV)
    token = owner.repeat_interleave(case["window"]) * vocab + s["tokens"]
    count = torch.zeros(rows * vocab, device=DEV).index_add_(0, token, torch.ones_like(token, dtype=torch.float32))
    count = count.view(rows, vocab)
    penalty = s["repetition"][:, None]
    x = torch.where(count > 0, torch.where(x < 0, x * penalty, x / penalty), x)
    x = x - torch.where(count > 0, s["presence"][:, None], 0.0) - s["frequency"][:, None] * count
    bias = torch.zeros(rows * vocab, device=DEV)
    bias[owner.repeat_interleave(case["biases"]) * vocab + s["bias_ids"]] = s["bias_values"]
    x = x + bias.view(rows, vocab)
    column = torch.arange(vocab, device=DEV)
    free = s["mask_rows"] < 0
    words = s["allowed"][s["mask_rows"].long().clamp(min=0)][:, column >> 5]
    allowed = ((words >> (column & 31).to(torch.int32)) & 1).bool() | free[:, None]
    return x.masked_fill(~allowed, -math.inf).to(s["dtype"])


# ---- the definitions in 64 bits -----------------------------------------------------

def _cached(codes, meta, fmt):
    if fmt == "int8":
        return (codes.double() - 128) * meta.contiguous().view(torch.float32).double()[..., None]
    wide = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device=codes.device)
    wide[..., 0::2] = (codes % 16).double()
    wide[..., 1::2] = (codes // 16).double()
    halves = meta.contiguous().view(torch.bfloat16).unflatten(-1, (-1, 2)).double()
    return halves[..., 1:] + halves[..., :1] * wide


def _rounded(x, fmt):
    """What the cache holds of fp64 rows: the format's definition."""
    if fmt == "int8":
        top = x.abs().amax(-1, keepdim=True)
        return torch.round(127 * x / top) * (top / 127)
    low = x.amin(-1, keepdim=True)
    step = ((x.amax(-1, keepdim=True) - low) / 15).float().bfloat16().double()
    low = low.bfloat16().double()
    return low + step * torch.round((x - low) / step).clamp(0, 15)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return _rounded(s["k"].double(), case["fmt"]), _rounded(s["v"].double(), case["fmt"])
    if case["op"] == "read":
        flat = s["slots"].long()
        both = []
        for kind in (0, 1):
            codes = s["codes"][:, :, kind].transpose(1, 2).flatten(0, 1)[flat]
            meta = s["meta"][:, :, kind].transpose(1, 2).flatten(0, 1)[flat]
            both.append(_cached(codes, meta, case["fmt"]))
        return tuple(both)
    if case["op"] == "attend":
        lens, nodes = _lens(case)
        share = case["heads"] // case["kv_heads"]
        outs, sums, at = [], [], 0
        for i, (n, t) in enumerate(zip(lens, nodes)):
            pages = s["table"][i, :-(-n // case["page"])].long()
            sees = torch.ones((t, n), dtype=torch.bool, device=DEV)
            if s["mask"] is None:
                sees[:, n - t:] = torch.ones((t, t), dtype=torch.bool, device=DEV).tril()
            else:
                bits = s["mask"][at:at + t].cpu().tolist()
                sees[:, n - t:] = torch.tensor([[(r[j >> 5] >> (j & 31)) & 1 for j in range(t)] for r in bits],
                                               device=DEV).bool()
            head_out, head_sum = [], []
            for h in range(case["heads"]):
                g = h // share
                k = _cached(s["codes"][pages, g, 0].flatten(0, 1)[:n], s["meta"][pages, g, 0].flatten()[:n], case["fmt"])
                v = _cached(s["codes"][pages, g, 1].flatten(0, 1)[:n], s["meta"][pages, g, 1].flatten()[:n], case["fmt"])
                score = torch.einsum("td,nd->tn", s["q"][at:at + t, h].double(), k) / math.sqrt(case["head_dim"])
                score[~sees] = -math.inf
                head_sum.append(torch.logsumexp(score, 1))
                head_out.append(torch.softmax(score, 1) @ v)
            outs.append(torch.stack(head_out, 1))
            sums.append(torch.stack(head_sum, 1))
            at += t
        return torch.cat(outs), torch.cat(sums)
    if case["op"] == "project":
        k, n = case["k"], case["n"]
        out = torch.empty((case["rows"], n), dtype=torch.float64, device=DEV)
        x = s["x"].double()
        i, lane = torch.arange(k, device=DEV), torch.arange(16, device=DEV)
        # where output o of a block and input i lie: lane, word, nibble
        o = lane[:, None]
        inner = i % 64
        which = (o % 8) * 4 + inner // 16
        word = (inner % 16 // 4).expand(16, k)
        nib = o // 8 + (inner & 2) + 4 * (inner & 1)
        for b in range(s["codes"].shape[0]):
            code = (s["codes"][b][(i // 64).expand(16, k), which, word].long() >> (4 * nib)) & 15
            halves = s["meta"][b].T.contiguous().view(torch.bfloat16).unflatten(-1, (-1, 2)).double()
            halves = halves[:, i // case["group"]]
            w = halves[..., 1] + halves[..., 0] * code.double()
            m = min(16, n - 16 * b)
            out[:, 16 * b:16 * b + m] = x @ w[:m].T + s["bias"][16 * b:16 * b + m].double()
        return out
    rows, vocab, window = case["rows"], case["vocab"], case["window"]
    out = s["logits"].double()
    for r in range(rows):
        ids, count = torch.unique(s["tokens"][r * window:(r + 1) * window].long(), return_counts=True)
        x = out[r, ids]
        rep = s["repetition"][r].double()
        x = torch.where(x < 0, x * rep, x / rep) - s["presence"][r].double() - s["frequency"][r].double() * count
        out[r, ids] = x
        part = slice(r * case["biases"], (r + 1) * case["biases"])
        out[r, s["bias_ids"][part].long()] += s["bias_values"][part].double()
        m = int(s["mask_rows"][r])
        if m >= 0:
            bits = (s["allowed"][m][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
            out[r, bits.flatten()[:vocab] == 0] = -math.inf
    return out

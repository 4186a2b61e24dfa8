"""The serving operators (quantised K/V cache, attention over it, 4-bit linear
layers, logit controls) against plain 64-bit implementations, at the sizes and
masks where they can go wrong, and their refusals."""
from __future__ import annotations

import math
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def within(got, want, tol):
    """Whether every value is the rounding, in its own type, of something at
    most tol from want (fp64): rounding is monotonic, so it lies between the
    roundings of the ends."""
    got, want = got.cpu(), want.cpu()
    low, high = (want - tol).to(got.dtype), (want + tol).to(got.dtype)
    return bool(((got >= low) & (got <= high)).all())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def decode(cache):
    """fp64 (k, v) [slots, kv heads, head_dim] that the buffers stand for."""
    codes, meta = cache.codes.cpu().numpy(), cache.meta.cpu().numpy()
    if cache.fmt == "int8":
        scale = meta.view(np.float32).astype(np.float64)
        x = (codes.astype(np.float64) - 128) * scale[..., None]
    else:
        code = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1,)).astype(np.float64)
        scale = (meta << 16).view(np.float32).astype(np.float64)
        least = (meta & -65536).view(np.float32).astype(np.float64)
        x = least[..., None] + scale[..., None] * code
    both = torch.from_numpy(x).permute(2, 0, 3, 1, 4).flatten(1, 2)  # [2][pages*size][heads][dim]
    return both[0], both[1]


def filled(pkg, g, pages, page, heads, dim, fmt):
    cache = pkg.QuantKvCache.empty(pages, page, heads, dim, fmt)
    slots = torch.arange(pages * page, dtype=torch.int32, device="cuda")
    cache.write(normal(g, pages * page, heads, dim), normal(g, pages * page, heads, dim), slots)
    return cache


# ---- the cache ------------------------------------------------------------------

def check_rows(fmt, x, codes, meta):
    """One side's stored rows against the formats' definition in 64 bits:
    x fp64 [rows, heads, dim], codes and meta as stored."""
    if fmt == "int8":
        scale = meta.view(np.float32).astype(np.float64)
        top = np.abs(x).max(-1)
        # one fp32 division
        assert (np.abs(scale - top / 127) <= 2.0 ** -23 * top / 127).all()
        want = 127 * x / top[..., None]
        # the factor and the product are rounded once each: below 2 * 127 * 2^-24 off a code
        assert (np.abs(codes.astype(np.float64) - 128 - want) <= 0.5 + 2e-5).all()
    else:
        scale = (meta << 16).view(np.float32).astype(np.float64)
        least = (meta & -65536).view(np.float32).astype(np.float64)
        low, span = x.min(-1), x.max(-1) - x.min(-1)
        assert (np.abs(least - low) <= 2.0 ** -8 * np.abs(low)).all()
        assert (np.abs(scale - span / 15) <= 2.0 ** -8 * span / 15).all()
        code = np.stack([codes & 15, codes >> 4], -1).reshape(x.shape).astype(np.float64)
        want = np.clip((x - least[..., None]) / scale[..., None], 0, 15)
        assert (np.abs(code - want) <= 0.5 + 2e-5).all()


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,heads,dim,page", [(1, 1, 16, 8), (3, 12, 64, 16), (37, 5, 80, 32), (130, 8, 128, 64),
                                                  (17, 2, 256, 1024), (9, 3, 48, 8)])
def test_write_stores_the_rows_and_nothing_else(pkg, fmt, dtype, rows, heads, dim, page):
    g = gen(rows + dim)
    pages = -(-2 * rows // page) + 1
    cache = pkg.QuantKvCache.empty(pages, page, heads, dim, fmt)
    cache.codes.random_(0, 256, generator=g)
    cache.meta.random_(0, 1 << 30, generator=g)
    before = cache.codes.clone(), cache.meta.clone()
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:rows].to(torch.int32)
    k, v = normal(g, rows, heads, dim, dtype=DTYPES[dtype]), 3 * normal(g, rows, heads, dim, dtype=DTYPES[dtype])
    cache.write(k, v, slots)
    at = slots.long()
    codes = cache.codes.permute(2, 0, 3, 1, 4).flatten(1, 2)
    meta = cache.meta.permute(2, 0, 3, 1).flatten(1, 2)
    for kind, x in enumerate((k, v)):
        check_rows(fmt, x.double().cpu().numpy(), codes[kind][at].cpu().numpy(), meta[kind][at].cpu().numpy())
    others = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    others[at] = False
    assert torch.equal(codes[:, others], before[0].permute(2, 0, 3, 1, 4).flatten(1, 2)[:, others])
    assert torch.equal(meta[:, others], before[1].permute(2, 0, 3, 1).flatten(1, 2)[:, others])


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 208])
def test_written_codes_are_those_of_the_formula_in_fp32(pkg, fmt, dtype, dim):
    """Bit for bit, where values lie halfway between two codes too: multiples of
    a power of two, as values of 16-bit types are."""
    g = gen(dim)
    rows = 64
    x = normal(g, rows, 2, dim)
    x[::2] = torch.round(x[::2] * 8) / 8
    x[1::4] += 300  # a minimum that is rounded by more than a code
    x = x.to(DTYPES[dtype])
    cache = pkg.QuantKvCache.empty(4, 16, 2, dim, fmt)
    cache.write(x, x, torch.arange(rows, dtype=torch.int32, device="cuda"))
    f = x.float().cpu()
    codes = cache.codes.permute(2, 0, 3, 1, 4).flatten(1, 2).cpu()
    if fmt == "int8":
        want = torch.round(f * torch.div(torch.tensor(127.0), f.abs().amax(-1, keepdim=True))) + 128  # number / tensor is two roundings
    else:
        low, high = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
        scale, least = ((high - low) / 15).bfloat16().float(), low.bfloat16().float()
        want = torch.round((f - least) * (1 / scale)).clamp(0, 15)
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    assert torch.equal(codes[0].float(), want) and torch.equal(codes[1].float(), want)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,heads,dim,page", [(1, 1, 16, 8), (5, 12, 64, 16), (131, 5, 80, 32), (40, 8, 128, 64),
                                                  (17, 2, 256, 1024)])
def test_read_gives_the_stored_values(pkg, fmt, dtype, rows, heads, dim, page):
    g = gen(7)
    pages = -(-rows // page) + 2
    cache = filled(pkg, g, pages, page, heads, dim, fmt)
    slots = torch.randint(0, pages * page, (rows,), device="cuda", generator=g).to(torch.int32)
    slots[rows // 2] = -1 if rows > 1 else slots[0]
    if rows > 4:
        slots[3] = pages * page
    k, v = cache.read(slots, DTYPES[dtype])
    wk, wv = decode(cache)
    for got, want in ((k, wk), (v, wv)):
        want = want[slots.long().cpu().clamp(0, pages * page - 1)]
        want[(slots.cpu() < 0) | (slots.cpu() >= pages * page)] = 0
        # one fp32 rounding, then the type's
        assert got.dtype == DTYPES[dtype] and torch.equal(got.cpu(), want.float().to(DTYPES[dtype]))


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_write_of_strided_unaligned_and_skipped_rows(pkg, fmt):
    g = gen(3)
    heads, dim, rows = 4, 32, 21
    cache = pkg.QuantKvCache.empty(4, 16, heads, dim, fmt)
    dense = pkg.QuantKvCache.empty(4, 16, heads, dim, fmt)
    base = normal(g, rows, 3 * heads * dim + 1)
    k = base[:, 1:1 + heads * dim].unflatten(1, (heads, dim))                    # not 16-byte aligned
    v = base[:, 1 + heads * dim:1 + 2 * heads * dim].unflatten(1, (dim, heads)).transpose(1, 2)  # wrong last stride
    slots = torch.arange(rows, dtype=torch.int32, device="cuda") * 3
    slots[4], slots[9], slots[20] = -1, 64, 2 ** 31 - 1
    with pytest.raises(pkg.ArgumentError):
        cache.write(k, v, slots)
    v = base[:, :heads * dim].unflatten(1, (heads, dim)).flip(0)
    cache.write(k, v, slots)
    keep = (slots >= 0) & (slots < 64)
    dense.write(k.contiguous()[keep], v.contiguous()[keep], slots[keep].contiguous())
    assert torch.equal(cache.codes, dense.codes) and torch.equal(cache.meta, dense.meta)
    one = normal(g, 1, 1, dim).expand(rows, heads, dim)  # one row for every head and token
    cache.write(one, one, slots)
    k2, _ = cache.read(slots[:1].contiguous())
    assert torch.equal(k2[0, 0], k2[0, 3])


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dim", [16, 80, 128])
def test_write_of_special_rows(pkg, fmt, dim):
    inf, nan = math.inf, math.nan
    rows = torch.randn((9, dim), generator=torch.Generator().manual_seed(1))
    rows[0] = 0.0
    rows[1] = 2.5                  # a constant
    rows[2, dim - 1] = inf
    rows[3, 3] = -inf
    rows[4, 0] = nan
    rows[5] *= 1e-40               # below every scale that can be held
    rows[6] *= 1e30
    rows[7] = -0.0
    rows[8] = nan
    x = rows[:, None].cuda()
    cache = pkg.QuantKvCache.empty(2, 8, 1, dim, fmt)
    slots = torch.arange(9, dtype=torch.int32, device="cuda")
    cache.write(x, x.flip(2).contiguous(), slots)
    k, v = (t[:, 0].double().cpu() for t in cache.read(slots))
    for t in (k, v):
        assert (t[0] == 0).all() and (t[7] == 0).all()
        assert (t[1] == 2.5).all()
        assert t[2].isnan().all() and t[3].isnan().all() and t[4].isnan().all() and t[8].isnan().all()
        assert (t[5].abs() <= 1e-35).all()
    span = rows[6].double().max() - rows[6].double().min()
    step = rows[6].double().abs().max() / 127 if fmt == "int8" else span / 15
    # half a step, and for int4 the bf16 roundings of scale (15 codes) and minimum
    more = 0 if fmt == "int8" else (15 * step + rows[6].double().abs().max()) * 2.0 ** -8
    assert ((k[6] - rows[6].double()).abs() <= 0.501 * step + more).all()


def test_more_rows_than_the_cache_takes(pkg):
    """The last blocks' row numbers stay within 32 bits."""
    import struct
    from forge_lm_b200 import _native as N
    L = N.load()
    c = struct.Struct("=QQ6i").pack(4096, 4096, 10, 16, 3, 64, 0, 0)
    for rows in (2 ** 31 - 128, 2 ** 31 - 1):
        assert L.fb2_kvq_write(c, rows, 4096, 4096, 0, 192, 64, 192, 64, 4096, None) == N.FB2_INVALID_ARG
        assert L.fb2_kvq_read(c, rows, 4096, 4096, 4096, 0, None) == N.FB2_INVALID_ARG


# ---- attention --------------------------------------------------------------------

def plain_attention(cache, q, table, prefix, starts, bits, scale, max_len=None):
    """fp64 (out, lse) by the definition; bits: per row the set of drafted
    tokens it sees, or None for the causal order."""
    k, v = decode(cache)
    q = q.double().cpu()
    rows, heads, dim = q.shape
    out = torch.zeros((rows, heads, dim), dtype=torch.float64)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    share = heads // cache.n_kv_heads
    table = table.cpu()
    cap = table.shape[1] * cache.page_size
    for b in range(len(prefix)):
        for r in range(starts[b], starts[b + 1]):
            i = r - starts[b]
            seen = list(range(prefix[b])) + [prefix[b] + j for j in range(starts[b + 1] - starts[b])
                                             if (j <= i if bits is None else j in bits[r])]
            seen = [p for p in seen if p < cap and (max_len is None or p < max_len)]
            pages = [int(table[b, p // cache.page_size]) for p in seen]
            slots = [pg * cache.page_size + p % cache.page_size for pg, p in zip(pages, seen)
                     if 0 <= pg < cache.n_pages]
            if not slots:
                continue
            for h in range(heads):
                s = (k[slots, h // share] @ q[r, h]) * scale
                lse[r, h] = torch.logsumexp(s, 0)
                out[r, h] = torch.softmax(s, 0) @ v[slots, h // share]
    return out, lse


def check_attention(dtype, got, want, big, scores):
    """big: largest |v|; scores: largest |score|.  fp32: a score is off by a few
    roundings of its size (sums of up to 256 products, the scale's and the
    exponential's), which moves out by that times the values' spread; every
    product and sum after it by 2^-24 and the accumulations by less than
    2^-20 of the largest value.  The type's rounding comes on top."""
    out, lse = got
    tol = (8 * 2.0 ** -23 * (scores + 4) + 2.0 ** -20) * big
    if dtype != "fp32":
        tol += 2.0 ** -11 * big  # probabilities may be carried in 11 bits
    assert torch.isfinite(out).all()
    assert within(out, want[0], tol), float((out.double().cpu() - want[0]).abs().max())
    empty = want[1] == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    assert (out.cpu()[empty] == 0).all()
    off = (lse.double().cpu() - want[1])[~empty].abs()
    assert off.numel() == 0 or float(off.max()) <= 8 * 2.0 ** -23 * (scores + 16)


def attention_case(pkg, seed, fmt, dtype, prefix, nodes, heads, kv_heads, dim, page, tree, spare=3, scale=None,
                   wide_table=0, max_len=None):
    g, rnd = gen(seed), random.Random(seed)
    lens = [p + t for p, t in zip(prefix, nodes)]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    cache = filled(pkg, g, pages, page, kv_heads, dim, fmt)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need + [1]) + wide_table), -1, dtype=torch.int32)
    used = torch.zeros(pages * page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(need):
        mine = order[at:at + n]
        table[b, :n] = torch.tensor(mine, dtype=torch.int32)
        for p in range(lens[b]):
            used[mine[p // page] * page + p % page] = True
        at += n
    # what no row sees must not count: NaN scales and other codes there
    hidden = ~used.view(pages, page).cuda()
    meta = cache.meta.permute(0, 3, 1, 2)
    meta[hidden] = torch.tensor(0x7FC07FC0, dtype=torch.int32, device="cuda")
    cache.codes.permute(0, 3, 1, 2, 4)[hidden] = 255
    clean = pkg.QuantKvCache(cache.codes, cache.meta, dim, fmt)
    starts = [0]
    for t in nodes:
        starts.append(starts[-1] + t)
    q = (2 * normal(g, starts[-1], heads, dim)).to(DTYPES[dtype])
    bits = mask = None
    if tree:
        words = (max(nodes) + 31) // 32
        bits, flat = [], []
        for b, t in enumerate(nodes):
            seen = []
            for i in range(t):
                up = seen[rnd.randrange(i)] if i and rnd.random() < 0.9 else set()
                seen.append(up | {i})
            if t > 2:
                seen[t - 1] = set()  # sees nothing drafted, not even itself
            bits += seen
        for s in bits:
            flat.append([sum(1 << (j - 32 * w) for j in s if 32 * w <= j < 32 * w + 32) for w in range(words)])
        mask = torch.tensor(flat, dtype=torch.int64).reshape(-1, words).to(torch.int32).cuda()
    got = clean.attend(q, table.cuda(), torch.tensor(prefix, dtype=torch.int32, device="cuda"),
                       starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), mask=mask, scale=scale,
                       max_nodes=max(nodes), max_len=max_len)
    s = scale if scale is not None else 1 / math.sqrt(dim)
    want = plain_attention(clean, q, table, prefix, starts, bits, s, max_len)
    k, v = cache.read(torch.arange(pages * page, dtype=torch.int32, device="cuda")[used.cuda()])
    top = float(v.abs().max()) if v.numel() else 1.0
    scores = float(q.float().norm(dim=2).max() * k.norm(dim=2).max() * abs(s)) if k.numel() else 1.0
    check_attention(dtype, got, want, top, scores)
    return got


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(1, 1, 16, 8), (12, 12, 64, 16), (8, 1, 64, 32), (14, 2, 80, 8),
                                                      (32, 8, 128, 64), (4, 4, 256, 16), (15, 5, 32, 1024),
                                                      (3, 1, 112, 16), (17, 1, 192, 8)])
def test_attention_of_single_tokens(pkg, fmt, dtype, heads, kv_heads, dim, page):
    prefix = [0, 1, 7, 15, 16, 31, 32, 33, 63, 64, 100, 257]
    attention_case(pkg, dim, fmt, dtype, prefix, [1] * len(prefix), heads, kv_heads, dim, page, tree=False)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(2, 2, 16, 8), (12, 12, 64, 16), (8, 2, 128, 32), (7, 1, 64, 64),
                                                      (5, 5, 80, 8), (4, 1, 256, 16)])
def test_attention_of_drafted_trees(pkg, fmt, dtype, heads, kv_heads, dim, page):
    attention_case(pkg, dim + 1, fmt, dtype, [0, 5, 64, 200, 31, 0], [9, 64, 1, 33, 17, 3], heads, kv_heads, dim, page,
                   tree=True)


@gpu
@pytest.mark.parametrize("fmt,dtype", [("int8", "fp32"), ("int4", "bf16"), ("int8", "bf16"), ("int4", "fp32")])
def test_attention_of_long_rows_in_causal_order(pkg, fmt, dtype):
    attention_case(pkg, 11, fmt, dtype, [0, 130, 3], [75, 1, 130], 6, 2, 64, 16, tree=False)


@gpu
@pytest.mark.parametrize("fmt,dtype", [("int8", "fp32"), ("int4", "fp16"), ("int8", "bf16")])
@pytest.mark.parametrize("nodes", [1, 40])
def test_attention_over_long_caches(pkg, fmt, dtype, nodes):
    """Lengths at which one sequence is split over many blocks."""
    attention_case(pkg, 5, fmt, dtype, [9000, 2047, 4500], [nodes, max(1, nodes // 3), nodes], 4, 2, 64, 32,
                   tree=nodes > 1, wide_table=700)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_with_more_mask_words_than_one(pkg, dtype):
    attention_case(pkg, 21, "int8", dtype, [70, 0], [100, 129], 4, 4, 64, 16, tree=True)


@gpu
def test_attention_rows_that_see_nothing(pkg):
    g = gen(1)
    cache = filled(pkg, g, 4, 16, 2, 64, "int8")
    q = normal(g, 3, 4, 64)
    table = torch.tensor([[0, 1], [-1, -1], [7, 3]], dtype=torch.int32, device="cuda")
    prefix = torch.tensor([0, 20, 16], dtype=torch.int32, device="cuda")
    starts = torch.arange(4, dtype=torch.int32, device="cuda")
    mask = torch.zeros((3, 1), dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, table, prefix, starts=starts, mask=mask, max_nodes=1)
    # row 0: an empty mask and no prefix; row 1: no pages; row 2: its prefix's page is not in the cache
    assert (out == 0).all() and (lse == -math.inf).all()
    mask[2] = 1
    out, lse = cache.attend(q, table, prefix, starts=starts, mask=mask, max_nodes=1)
    _, v = cache.read(torch.tensor([48], dtype=torch.int32, device="cuda"))
    assert (out[:2] == 0).all()
    want = v[0].repeat_interleave(2, 0)
    assert ((out[2] - want).abs() <= 2.0 ** -21 * want.abs().max()).all() and torch.isfinite(lse[2]).all()


@gpu
def test_attention_of_masked_and_seen_nan(pkg):
    """A NaN row of the cache reaches the rows that see it and no others."""
    g = gen(2)
    heads, dim = 2, 64
    for fmt in ("int8", "int4"):
        for dtype in (torch.float32, torch.bfloat16):
            for kind in (0, 1):
                cache = filled(pkg, g, 4, 16, heads, dim, fmt)
                table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
                x = normal(g, 1, heads, dim)
                bad = x.clone()
                bad[:, 1] = math.nan
                cache.write(bad if kind == 0 else x, bad if kind == 1 else x,
                            torch.tensor([2 * 16 + 11], dtype=torch.int32, device="cuda"))
                mask = torch.tensor([[1], [0b10], [0b101]], dtype=torch.int32, device="cuda")
                out, _ = cache.attend(normal(g, 3, heads, dim, dtype=dtype), table,
                                      torch.tensor([10], dtype=torch.int32, device="cuda"),
                                      starts=torch.tensor([0, 3], dtype=torch.int32, device="cuda"), mask=mask, max_nodes=3)
                assert torch.isfinite(out[[0, 2]]).all() and torch.isfinite(out[1, 0]).all()
                assert out[1, 1].isnan().all()


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("nodes", [1, 40])
@pytest.mark.parametrize("at", [3, 70, 300, 303])
def test_attention_of_seen_nan_with_no_weight(pkg, fmt, dtype, nodes, at):
    """A NaN V row that a row sees reaches it however small its probability, in a whole
    tile of positions (3, 70) as in the last one (300, 303)."""
    g = gen(53)
    prefix, dim = 304, 64
    cache = filled(pkg, g, 24, 16, 2, dim, fmt)
    k, v = torch.zeros((1, 2, dim), device="cuda"), torch.full((1, 2, dim), math.nan, device="cuda")
    k[..., 0] = -400.0  # a score some 400 below the others
    v[:, 0] = 1.0       # the first head's row is not NaN
    cache.write(k, v, _i32([at]))
    q = normal(g, nodes, 4, dim, dtype=DTYPES[dtype])
    q[..., 0] = 8
    out, lse = cache.attend(q, torch.arange(24, dtype=torch.int32, device="cuda")[None], _i32([prefix]),
                            starts=_i32([0, nodes]), max_nodes=nodes)
    assert torch.isfinite(out[:, :2]).all() and out[:, 2:].isnan().all() and torch.isfinite(lse).all()


@gpu
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e30])
def test_attention_of_large_and_small_values(pkg, size):
    g = gen(4)
    cache = pkg.QuantKvCache.empty(8, 16, 2, 64, "int8")
    slots = torch.arange(128, dtype=torch.int32, device="cuda")
    spread = torch.logspace(-3, 0, 128, device="cuda")[:, None, None]
    cache.write(normal(g, 128, 2, 64) / size, normal(g, 128, 2, 64) * size * spread, slots)
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    q = normal(g, 1, 4, 64) * size
    prefix = torch.tensor([121], dtype=torch.int32, device="cuda")
    got = cache.attend(q, table, prefix)
    want = plain_attention(cache, q, table, [121], [0, 1], None, 0.125)
    k, v = decode(cache)
    check_attention("fp32", (got[0] / size, got[1]), (want[0] / size, want[1]), float(v.abs().max()) / size,
                    float(q.double().norm(dim=2).max().cpu() * k.norm(dim=2).max()) / 8)


def plain_of_one_sequence(cache, q, slots, prefix, bits, scale):
    """fp64 (out, lse) of one sequence's rows by the definition, its positions in
    `slots`, and for each row and head sum_p softmax_p max|v_p|; bits as for
    plain_attention."""
    k, v = (x[slots.long().cpu()].repeat_interleave(q.shape[1] // cache.n_kv_heads, 1) for x in decode(cache))
    rows, total = q.shape[0], len(slots)
    sees = torch.zeros((rows, total), dtype=torch.bool)
    sees[:, :prefix] = True
    for r in range(rows):
        sees[r, [prefix + j for j in (range(r + 1) if bits is None else bits[r])]] = True
    s = torch.einsum("rhd,phd->rhp", q.double().cpu(), k) * scale
    s[~sees[:, None].expand_as(s)] = -math.inf
    p = torch.softmax(s, 2)
    return ((torch.einsum("rhp,phd->rhd", p, v), torch.logsumexp(s, 2)),
            torch.einsum("rhp,ph->rh", p, v.abs().amax(2)))


def check_own_size(fmt, dtype, got, want, own, scores, rows):
    """As check_attention, for each row by what the row itself weighs: the
    weights' errors are relative to the row's largest weight, whatever other
    rows or masked positions hold.  int4 values are summed in two parts (the
    row's middle and codes - 8), each up to about as large as the values."""
    tol = 8 * 2.0 ** -23 * (scores + 4) + 2.0 ** -20
    if dtype != "fp32":
        tol += 2.0 ** -11
    tol *= 2 if fmt == "int4" else 1
    out, lse = got
    assert torch.isfinite(out[rows]).all()
    assert within(out[rows], want[0][rows], tol * own[rows][:, :, None]), \
        float(((out.double().cpu() - want[0]).abs() / own[:, :, None])[rows].max())
    assert float((lse.double().cpu() - want[1])[rows].abs().max()) <= 8 * 2.0 ** -23 * (scores + 16)


def large_value_case(pkg, fmt, dtype, nodes, dim, big, far, late):
    """One V row 2^big times the others: a drafted node that some rows do not
    see (far 0), or a cached position that all see with a score about `far`
    below the others (at the end or the start of the prefix)."""
    g = gen(51)
    prefix, heads = 300, 4
    cache = pkg.QuantKvCache.empty(24, 16, 2, dim, fmt)
    order = torch.randperm(24, generator=torch.Generator().manual_seed(6)).to(torch.int32)
    total = prefix + nodes
    k, v = normal(g, total, 2, dim), normal(g, total, 2, dim)
    q = (2 * normal(g, nodes, heads, dim)).to(DTYPES[dtype])
    scale = 1 / math.sqrt(dim)
    k[:, :, 0] = 0
    q[:, :, 0] = 8
    which = prefix + 1 if not far else prefix - 3 if late else 2
    if far:
        k[which, :, 0] = -far / 8 / scale
    v[which] *= 2.0 ** big
    slots = torch.tensor([int(order[p // 16]) * 16 + p % 16 for p in range(total)], dtype=torch.int32, device="cuda")
    cache.write(k, v, slots)
    bits = [{0, i} | ({1} if i % 2 else set()) for i in range(nodes)]
    words = (nodes + 31) // 32
    flat = [[sum(1 << (j - 32 * w) for j in s if 32 * w <= j < 32 * w + 32) for w in range(words)] for s in bits]
    mask = torch.tensor(flat, dtype=torch.int64).to(torch.int32).cuda()
    got = cache.attend(q, order[None].cuda(), _i32([prefix]), starts=_i32([0, nodes]), mask=mask, max_nodes=nodes)
    want, own = plain_of_one_sequence(cache, q, slots, prefix, bits, scale)
    ks, _ = decode(cache)
    scores = float(q.double().cpu().norm(dim=2).max() * ks.norm(dim=2).max() * scale)
    # what fp16 cannot hold is no result to compare
    rows = torch.tensor([i for i in range(nodes) if far or i % 2 == 0 or dtype != "fp16"])
    check_own_size(fmt, dtype, got, want, own, scores, rows)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("nodes,dim", [(4, 64), (40, 64), (34, 128), (8, 256)])
@pytest.mark.parametrize("big", [20, 40, 100])
def test_attention_beside_large_masked_values(pkg, fmt, dtype, nodes, dim, big):
    """What a row does not see does not cost it bits, however large."""
    large_value_case(pkg, fmt, dtype, nodes, dim, big, 0, False)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("nodes,dim", [(4, 64), (40, 64), (34, 128), (8, 256)])
@pytest.mark.parametrize("late", [False, True])
def test_attention_with_large_values_of_no_weight(pkg, fmt, dtype, nodes, dim, late):
    """Nor does what it sees with a score 100 below its others, first or last."""
    large_value_case(pkg, fmt, dtype, nodes, dim, 60, 100, late)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("nodes", [2, 40])
@pytest.mark.parametrize("step", [12, -12])
def test_attention_over_values_that_grow(pkg, fmt, dtype, nodes, step):
    """V rows 2^12 larger (or smaller) every 128 positions, all of them seen."""
    g = gen(52)
    prefix, dim = 900, 64
    total = prefix + nodes
    cache = pkg.QuantKvCache.empty(60, 16, 2, dim, fmt)
    order = torch.randperm(60, generator=torch.Generator().manual_seed(7)).to(torch.int32)
    v = normal(g, total, 2, dim) * 2.0 ** (step * (torch.arange(total, device="cuda") // 128).float())[:, None, None]
    slots = torch.tensor([int(order[p // 16]) * 16 + p % 16 for p in range(total)], dtype=torch.int32, device="cuda")
    cache.write(normal(g, total, 2, dim), v, slots)
    q = (2 * normal(g, nodes, 4, dim)).to(DTYPES[dtype])
    got = cache.attend(q, order[None].cuda(), _i32([prefix]), starts=_i32([0, nodes]), max_nodes=nodes)
    want, own = plain_of_one_sequence(cache, q, slots, prefix, None, 0.125)
    ks, _ = decode(cache)
    scores = float(q.double().cpu().norm(dim=2).max() * ks.norm(dim=2).max() * 0.125)
    check_own_size(fmt, dtype, got, want, own, scores, torch.arange(nodes))


@gpu
def test_attention_of_strided_queries_on_another_stream(pkg):
    g = gen(6)
    heads, dim = 6, 64
    cache = filled(pkg, g, 12, 16, 2, dim, "int8")
    table = torch.randperm(12, device="cuda", generator=g)[None].to(torch.int32)
    qkv = normal(g, 5, heads * dim * 3 + 3)
    q = qkv[:, 3:3 + heads * dim].unflatten(1, (heads, dim))
    prefix = torch.tensor([150], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    want = cache.attend(q.contiguous(), table, prefix, starts=starts, max_nodes=5)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(q, table, prefix, starts=starts, max_nodes=5)
        other = cache.attend(turned, table.expand(1, 12), prefix, starts=starts, max_nodes=5, max_len=155)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert ((other[0] - want[0]).abs() <= 2.0 ** -20 * want[0].abs().max()).all()
    again = cache.attend(q.contiguous(), table, prefix, starts=starts, max_nodes=5)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])  # the same bits each time


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("nodes", [1, 12])
def test_attention_of_sequences_that_share_a_page_table(pkg, dtype, nodes):
    """A table expanded over the sequences, or with rows apart: the values of a dense copy."""
    g = gen(41)
    cache = filled(pkg, g, 24, 16, 2, 64, "int8")
    q = normal(g, 3 * nodes, 8, 64, dtype=DTYPES[dtype])
    prefix, starts = _i32([150, 0, 77]), _i32([0, nodes, 2 * nodes, 3 * nodes])
    row = torch.randperm(24, generator=torch.Generator().manual_seed(4))[:11].to(torch.int32).cuda()
    wide = torch.randint(0, 24, (3, 20), device="cuda", generator=g).to(torch.int32)
    for table in (row[None].expand(3, 11), row[:1, None].expand(3, 1), wide[:, 3:14]):
        want = cache.attend(q, table.contiguous(), prefix, starts=starts, max_nodes=nodes)
        got = cache.attend(q, table, prefix, starts=starts, max_nodes=nodes)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one sequence's row may have any stride; rows that overlap in part are refused
    one = cache.attend(q[:nodes], row.as_strided((1, 11), (3, 1)), prefix[:1], starts=starts[:2], max_nodes=nodes)
    want = cache.attend(q[:nodes], row[None].contiguous(), prefix[:1], starts=starts[:2], max_nodes=nodes)
    assert torch.equal(one[0], want[0])
    with pytest.raises(pkg.ArgumentError):
        cache.attend(q, row.as_strided((3, 7), (2, 1)), prefix, starts=starts, max_nodes=nodes)


def test_stride_of_a_shared_page_table(pkg):
    """The C entry takes a row stride of 0 as it is and refuses rows that overlap in part."""
    import ctypes as C
    import struct
    from forge_lm_b200 import _native as N
    L, size = N.load(), C.c_int64()
    cache = struct.Struct("=QQ6i").pack(4096, 4096, 10, 16, 3, 64, 0, 0)
    for stride, status in ((0, N.FB2_OK), (4, N.FB2_OK), (9, N.FB2_OK), (1, N.FB2_INVALID_ARG), (3, N.FB2_INVALID_ARG),
                           (-4, N.FB2_INVALID_ARG)):
        a = struct.Struct("=8Q4q8ifi").pack(*[4096] * 5, 0, 0, 0, 0, 64, 64, stride, 2, 2, 6, 0, 4, 1, 0, 0, 0.125, 0)
        assert L.fb2_kvq_attend_workspace(cache, a, C.byref(size)) == status, stride


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_without_max_nodes(pkg, dtype):
    """Several trees whose mask has fewer bits than the call has rows; more rows than 2^16."""
    g, rnd = gen(61), random.Random(61)
    cache = filled(pkg, g, 24, 16, 2, 64, "int8")
    table = torch.arange(24, dtype=torch.int32, device="cuda").view(3, 8)
    q = normal(g, 60, 4, 64, dtype=DTYPES[dtype])
    mask = _i32([[rnd.randrange(1 << (i % 20 + 1)) | 1 << i % 20] for i in range(60)])
    args = (q, table, _i32([90, 0, 31]))
    kw = dict(starts=_i32([0, 20, 40, 60]), mask=mask)
    got, want = cache.attend(*args, **kw), cache.attend(*args, **kw, max_nodes=20)
    assert ((got[0].double() - want[0].double()).abs() <= (2.0 ** -20 if dtype == "fp32" else 2.0 ** -7) * 5).all()
    assert ((got[1] - want[1]).abs() <= 8 * 2.0 ** -23 * 40).all()
    rows = 70000  # with the page table's width, each sees at most 16 positions
    q = normal(g, rows, 2, 64, dtype=DTYPES[dtype])
    args = (q, table[:2, :1].contiguous(), _i32([3, 11]))
    kw = dict(starts=_i32([0, rows // 2, rows]))
    got, want = cache.attend(*args, **kw), cache.attend(*args, **kw, max_nodes=rows // 2)
    assert ((got[0].double() - want[0].double()).abs() <= (2.0 ** -20 if dtype == "fp32" else 2.0 ** -7) * 5).all()
    assert torch.isfinite(got[1]).all()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads", [2, 8])
@pytest.mark.parametrize("pages", [8, 300])
def test_attention_rows_outside_every_sequence(pkg, dtype, heads, pages):
    """They, and rows past max_nodes, give zeros and -inf from Python; the C call leaves
    them alone unless it is asked to fill them."""
    import ctypes as C
    import struct
    from forge_lm_b200 import _native as N
    g = gen(62)
    cache = filled(pkg, g, 24, 16, 2, 64, "int8")
    table = torch.full((3, pages), -1, dtype=torch.int32, device="cuda")  # a wide one: several blocks and their merge
    table[:, :8] = torch.arange(24, dtype=torch.int32, device="cuda").view(3, 8)
    q = normal(g, 50, heads, 64, dtype=DTYPES[dtype])
    prefix, starts = _i32([90, 0, 31]), _i32([3, 10, 30, 44])
    rest = torch.ones(50, dtype=torch.bool, device="cuda")
    for a, b in ((3, 10), (10, 22), (30, 42)):
        rest[a:b] = False

    def poison():
        for shape, kind in ((q.shape, q.dtype), (q.shape[:2], torch.float32)):
            x = torch.full(shape, 7.0, dtype=kind, device="cuda")
            del x  # what the call gets next

    poison()
    out, lse = cache.attend(q, table, prefix, starts=starts, max_nodes=12)
    assert (out[rest] == 0).all() and (lse[rest] == -math.inf).all()
    assert (out[~rest] != 0).any(-1).all() and torch.isfinite(lse[~rest]).all()
    out2, lse2 = cache.attend(q, table, prefix, starts=_i32([3, 3, 50, 50]), max_nodes=12)  # sequences without rows
    assert (out2[:3] == 0).all() and (out2[15:] == 0).all() and torch.isfinite(lse2[3:15]).all() and (lse2[15:] == -math.inf).all()
    for kw in (dict(), dict(max_nodes=5)):  # no sequence at all
        poison()
        none, no_lse = cache.attend(q, table[:0], prefix[:0], starts=starts[:1], **kw)
        assert (none == 0).all() and (no_lse == -math.inf).all()
    L, size = N.load(), C.c_int64()
    c = struct.Struct("=QQ6i").pack(cache.codes.data_ptr(), cache.meta.data_ptr(), 24, 16, 2, 64, 0, 0)
    for fill in (0, 1):
        got, got_lse = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
        work = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
        a = struct.Struct("=8Q4q8ifi").pack(
            q.data_ptr(), got.data_ptr(), got_lse.data_ptr(), table.data_ptr(), prefix.data_ptr(), starts.data_ptr(), 0,
            work.data_ptr(), work.numel(), heads * 64, 64, pages, 3, 50, heads, 0 if dtype == "fp32" else 1, pages, 12, 0, 0, 0.125, fill)
        assert L.fb2_kvq_attend_workspace(c, a, C.byref(size)) == N.FB2_OK and size.value <= work.numel()
        assert L.fb2_kvq_attend(c, a, torch.cuda.current_stream().cuda_stream) == N.FB2_OK
        torch.cuda.synchronize()
        assert torch.equal(got[~rest], out[~rest]) and torch.equal(got_lse[~rest], lse[~rest])
        assert (got[rest] == (0 if fill else 7)).all() and (got_lse[rest] == (-math.inf if fill else 7)).all()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads", [2, 8])
def test_attention_of_malformed_starts(pkg, dtype, heads):
    """Row starts at the ends of 32 bits reach nothing outside the tensors, and the
    rows that they do name are right."""
    g = gen(63)
    cache = filled(pkg, g, 24, 16, 2, 64, "int8")
    table = torch.arange(24, dtype=torch.int32, device="cuda").view(3, 8)
    q = normal(g, 50, heads, 64, dtype=DTYPES[dtype])
    got = cache.attend(q, table, _i32([90, 70, 31]), starts=_i32([5, -2 ** 31, 2 ** 31 - 1, 50]), max_nodes=50)
    want = cache.attend(q, table, _i32([90, 70, 31]), starts=_i32([0, 0, 50, 50]), max_nodes=50)
    assert torch.equal(got[0][5:], want[0][5:]) and torch.equal(got[1][5:], want[1][5:])
    got = cache.attend(q, table, _i32([90, 70, 31]), starts=_i32([2 ** 31 - 1, -2 ** 31, -2 ** 31, -2 ** 31]), max_nodes=50)
    assert (got[0] == 0).all() and (got[1] == -math.inf).all()


@gpu
@pytest.mark.parametrize("dtype,heads", [("fp32", 1), ("bf16", 1), ("bf16", 40)])
def test_attention_over_two_billion_positions(pkg, dtype, heads):
    """As many positions as are counted, most of them in one page: what counts is the last page."""
    g = gen(64)
    pages, page, dim = (2 ** 31 - 65536) // 1024, 1024, 16
    cache = filled(pkg, g, 2, page, 1, dim, "int4")
    k = normal(g, page, 1, dim)
    k[..., 0] = 30.0
    v = normal(g, page, 1, dim)
    cache.write(k, v, torch.arange(page, 2 * page, dtype=torch.int32, device="cuda"))
    table = torch.zeros((1, pages), dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    q = normal(g, 1, heads, dim, dtype=DTYPES[dtype])
    q[..., 0] = 12  # scores some 80 above the other page's: together they weigh 2^31 exp(-80)
    got = cache.attend(q, table, _i32([pages * page - 1]))
    want = plain_attention(cache, q, torch.tensor([[1]]), [page - 1], [0, 1], None, 0.25)
    _, vs = decode(cache)
    ks, _ = decode(cache)
    check_attention(dtype, got, want, float(vs.abs().max()), float(q.double().cpu().norm(dim=2).max() * ks.norm(dim=2).max() * 0.25))


def test_longest_page_table(pkg):
    """The host refuses more positions than the kernels count, by the table's width or by max_len."""
    import ctypes as C
    import struct
    from forge_lm_b200 import _native as N
    L, size = N.load(), C.c_int64()
    cache = struct.Struct("=QQ6i").pack(4096, 4096, 10, 1024, 3, 64, 0, 0)
    for pages, max_len, status in ((2097088, 0, N.FB2_OK), (2097089, 0, N.FB2_INVALID_ARG), (2097089, 1000, N.FB2_OK),
                                   (2097151, 2 ** 31 - 65536, N.FB2_OK), (2097151, 2 ** 31 - 65535, N.FB2_INVALID_ARG)):
        a = struct.Struct("=8Q4q8ifi").pack(*[4096] * 5, 0, 0, 0, 0, 64, 64, pages, 2, 2, 6, 0, pages, 1, max_len, 0, 0.125, 0)
        assert L.fb2_kvq_attend_workspace(cache, a, C.byref(size)) == status, (pages, max_len)


@gpu
@pytest.mark.parametrize("dtype,heads", [("fp32", 2), ("bf16", 80)])
def test_cache_without_pages(pkg, dtype, heads):
    """Its buffers are empty: nothing is written, zeros are read, no row sees anything."""
    cache = pkg.QuantKvCache.empty(0, 16, 2, 64)
    k = torch.ones((3, 2, 64), device="cuda")
    cache.write(k, k, _i32([0, 1, -1]))
    assert all((t == 0).all() for t in cache.read(_i32([0, 1, -1])))
    q = torch.ones((3, heads, 64), dtype=DTYPES[dtype], device="cuda")
    for table in (torch.zeros((3, 40), dtype=torch.int32, device="cuda"), torch.zeros((3, 0), dtype=torch.int32, device="cuda")):
        out, lse = cache.attend(q, table, _i32([600, 0, 5]))
        assert (out == 0).all() and (lse == -math.inf).all()
    from forge_lm_b200 import _native as N
    import ctypes as C
    import struct
    size = C.c_int64()
    a = struct.Struct("=8Q4q8ifi").pack(*[4096] * 5, 0, 0, 0, 0, 64, 64, 4000, 2, 2, 6, 0, 4000, 1, 0, 0, 0.125, 0)
    assert N.load().fb2_kvq_attend_workspace(struct.Struct("=QQ6i").pack(0, 0, 0, 16, 3, 64, 0, 0), a, C.byref(size)) == N.FB2_OK
    assert size.value == 0  # nothing to split


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype,power", [("fp32", 90), ("bf16", 90), ("fp16", 10)])
@pytest.mark.parametrize("nodes", [2, 30])
def test_attention_of_large_and_small_queries(pkg, fmt, dtype, power, nodes):
    """q times a power of two with a scale that takes it back: the same bits; rows of q
    that are not finite give NaN and leave the others alone."""
    g = gen(65)
    cache = filled(pkg, g, 24, 16, 2, 64, fmt)
    table = torch.arange(24, dtype=torch.int32, device="cuda")[None]
    q = normal(g, nodes, 4, 64, dtype=DTYPES[dtype])
    if dtype == "fp16":  # where 2^-10 does not make subnormal numbers of them
        q = torch.where(q.abs() < 2.0 ** -3, torch.zeros_like(q), q)
    kw = dict(starts=_i32([0, nodes]), max_nodes=nodes)
    want = cache.attend(q, table, _i32([200]), scale=0.125, **kw)
    for p in (power, -power):
        got = cache.attend(q * 2.0 ** p, table, _i32([200]), scale=0.125 * 2.0 ** -p, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q[1, 2, 7], q[0, 0, 63] = math.inf, math.nan
    got = cache.attend(q, table, _i32([200]), scale=0.125, **kw)
    bad = torch.zeros((nodes, 4), dtype=torch.bool, device="cuda")
    bad[1, 2] = bad[0, 0] = True
    assert got[0][bad].isnan().all() and got[1][bad].isnan().all()
    assert torch.equal(got[0][~bad], want[0][~bad]) and torch.equal(got[1][~bad], want[1][~bad])


@gpu
def test_attention_bounds_that_cut(pkg):
    """max_len and the page table's width cut what is seen; max_nodes which rows are written."""
    attention_case(pkg, 31, "int8", "fp32", [100, 40], [1, 1], 4, 2, 64, 16, tree=False, max_len=77)
    g = gen(8)
    cache = filled(pkg, g, 8, 16, 2, 64, "int8")
    table = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    q = normal(g, 1, 4, 64)
    got = cache.attend(q, table, torch.tensor([500], dtype=torch.int32, device="cuda"))
    want = plain_attention(cache, q, table, [500], [0, 1], None, 0.125)
    check_attention("fp32", got, want, 5.0, 20.0)
    low = cache.attend(q, table, torch.tensor([-5], dtype=torch.int32, device="cuda"))
    none = cache.attend(q, table, torch.tensor([0], dtype=torch.int32, device="cuda"))
    assert torch.equal(low[0], none[0])


@gpu
def test_cache_past_32_bit_offsets(pkg):
    """5 GB of codes: byte and row offsets past 2^32."""
    pages, page, dim = 10000, 1024, 256
    codes = torch.empty((pages, 1, 2, page, dim), dtype=torch.uint8, device="cuda")
    meta = torch.zeros((pages, 1, 2, page), dtype=torch.int32, device="cuda")
    cache = pkg.QuantKvCache(codes, meta, dim, "int8")
    g = gen(9)
    slots = torch.arange((pages - 1) * page - 40, (pages - 1) * page + 60, dtype=torch.int32, device="cuda")
    k, v = normal(g, 100, 1, dim), normal(g, 100, 1, dim)
    small = pkg.QuantKvCache.empty(2, page, 1, dim)
    cache.write(k, v, slots)
    small.write(k, v, torch.arange(page - 40, page + 60, dtype=torch.int32, device="cuda"))
    for a, b in zip(cache.read(slots), small.read(torch.arange(page - 40, page + 60, dtype=torch.int32, device="cuda"))):
        assert torch.equal(a, b)
    codes[pages - 2, :, :, :page - 40] = 128
    small.codes[0, :, :, :page - 40] = 128
    q = normal(g, 1, 2, dim)
    prefix = torch.tensor([page + 59], dtype=torch.int32, device="cuda")
    got = cache.attend(q, torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device="cuda"), prefix)
    want = small.attend(q, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), prefix)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- 4-bit linear layers --------------------------------------------------------------

def unpack(linear):
    """fp64 W [in][out] that the packed buffers stand for."""
    k, n, group = linear.in_features, linear.out_features, linear.group
    codes, meta = linear.codes.cpu().numpy(), linear.meta.cpu().numpy()
    w = np.empty((k, n))
    i, o = np.meshgrid(np.arange(k), np.arange(n), indexing="ij")
    lane = 4 * (o % 8) + i % 64 // 16
    nibble = (o % 16) // 8 + (i & 2) + 4 * (i & 1)
    code = (codes[o // 16, i // 64, lane, i % 16 // 4] >> (4 * nibble)) & 15
    m = meta[o // 16, i // group, o % 16]
    return (m & -65536).view(np.float32).astype(np.float64) + (m << 16).view(np.float32).astype(np.float64) * code


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("k,n,group", [(64, 16, 64), (100, 77, 32), (32, 1, 32), (1, 40, 128), (300, 130, 128), (256, 64, 64)])
def test_pack_of_weights(pkg, dtype, k, n, group):
    g = gen(k)
    w = (0.02 * normal(g, k, n)).to(DTYPES[dtype])
    w[0, 0] = 0.5
    linear = pkg.W4Linear.pack(w, group)
    got, want = unpack(linear), w.double().cpu().numpy()
    for a in range(0, k, group):
        part = want[a:a + group]
        span = part.max(0) - part.min(0)
        # half a step, plus the bf16 roundings of scale (over 15 codes) and minimum
        most = span / 15 * (0.5 + 1e-3) + 2.0 ** -8 * (span + np.abs(part.min(0)))
        assert (np.abs(got[a:a + group] - part) <= most).all()


@gpu
def test_pack_of_special_weights(pkg):
    w = torch.randn((64, 20), generator=torch.Generator().manual_seed(5)).cuda()
    w[:, 3] = 0.25
    w[7, 5] = math.nan
    w[9, 6] = math.inf
    w[:, 8] = 1e-40
    wide = torch.zeros((64, 33), device="cuda")
    wide[:, 5:25] = w
    linear = pkg.W4Linear.pack(wide[:, 5:25], 32)
    got = unpack(linear)
    assert (got[:, 3] == 0.25).all() and np.isnan(got[:32, 5]).all() and np.isnan(got[:32, 6]).all()
    assert np.isfinite(got[32:, 5]).all() and (np.abs(got[:, 8]) < 1e-35).all()
    y = linear(torch.randn((3, 64), device="cuda"))
    assert y[:, [5, 6]].isnan().all() and torch.isfinite(y[:, [i for i in range(20) if i not in (5, 6)]]).all()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_pack_of_broadcast_and_single_rows(pkg, dtype):
    """W with every row the same (stride 0) or one row of any stride: as its dense copy."""
    g = gen(43)
    row = normal(g, 1, 50, dtype=DTYPES[dtype])
    for w in (row.expand(100, 50), row[0].as_strided((1, 50), (3, 1)), normal(g, 70, 1, dtype=DTYPES[dtype])[:1].expand(70, 1)):
        got, want = pkg.W4Linear.pack(w, 32), pkg.W4Linear.pack(w.contiguous(), 32)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.meta, want.meta)
    with pytest.raises(pkg.ArgumentError):
        pkg.W4Linear.pack(normal(g, 90, dtype=DTYPES[dtype]).as_strided((20, 50), (2, 1)), 32)


def test_stride_of_weights_to_pack(pkg):
    """The C entry refuses rows that overlap in part."""
    import struct
    from forge_lm_b200 import _native as N
    L = N.load()
    w = struct.Struct("=QQQ4i").pack(4096, 4096, 0, 100, 33, 32, 0)
    for stride in (1, 32, -33):
        assert L.fb2_w4_pack(w, 4096, 0, stride, None) == N.FB2_INVALID_ARG
        assert b"w_row_stride" in L.fb2_last_error()


def random_linear(pkg, g, k, n, group, bias):
    blocks, groups = -(-n // 16), -(-k // group)
    codes = torch.randint(-2 ** 31, 2 ** 31, (blocks, -(-k // 64), 32, 4), device="cuda", generator=g).to(torch.int32)
    scale = 0.01 + 0.02 * torch.rand((blocks, groups, 16), device="cuda", generator=g)
    least = -7.0 * scale + 0.02 * torch.randn((blocks, groups, 16), device="cuda", generator=g)
    pair = torch.stack((scale, least), -1).to(torch.bfloat16).view(torch.int32).squeeze(-1).contiguous()
    # padded outputs' scales are not looked at
    pad = torch.arange(blocks * 16, device="cuda").view(blocks, 1, 16) >= n
    pair[pad.expand_as(pair)] = 0x7FC07FC0
    return pkg.W4Linear(codes, pair, k, n, group, bias=normal(g, n) if bias else None)


def check_product(pkg, dtype, rows, k, n, group, bias=True, strided=False):
    g = gen(rows * 7 + k + n)
    linear = random_linear(pkg, g, k, n, group, bias)
    x = normal(g, rows, k + (5 if strided else 0), dtype=DTYPES[dtype])
    if strided:
        x = x[:, 5:]
    y = linear(x)
    w, xd = unpack(linear), x.double().cpu().numpy()
    want = xd @ w + (linear.bias.double().cpu().numpy() if bias else 0)
    # fp32 sums of code * x and of x: their terms' sizes bound the roundings
    # (pairwise over at least 16, at most k / 16 + 16 in a row)
    m = linear.meta.cpu().numpy()
    step = (m << 16).view(np.float32).astype(np.float64)[:, :, :].transpose(0, 2, 1).reshape(-1, m.shape[1])[:n]
    low = np.abs((m & -65536).view(np.float32).astype(np.float64)).transpose(0, 2, 1).reshape(-1, m.shape[1])[:n]
    grp = np.arange(k) // group
    size = np.abs(xd) @ (15 * step + low)[:, grp].T + np.abs(want)
    tol = 2.0 ** -24 * (k / 16 + 16) ** 0.5 * 4 * size
    assert y.dtype == DTYPES[dtype] and within(y, torch.from_numpy(want), torch.from_numpy(tol))


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 16), (1, 768, 2304), (1, 1, 1), (2, 100, 77), (3, 300, 130), (8, 1000, 33),
                                       (5, 2000, 50), (9, 192, 100), (17, 640, 48), (33, 96, 200), (64, 1024, 70),
                                       (100, 130, 40), (1, 5000, 16)])
def test_products_with_4_bit_weights(pkg, dtype, group, rows, k, n):
    check_product(pkg, dtype, rows, k, n, group)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,k,n", [(1, 333, 64), (7, 128, 48), (40, 515, 19)])
def test_products_of_unaligned_rows(pkg, dtype, rows, k, n):
    check_product(pkg, dtype, rows, k, n, 64, bias=False, strided=True)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,k,n,group", [(129, 200, 50, 32), (513, 320, 77, 64), (2050, 130, 33, 128)])
def test_products_of_a_prompt(pkg, dtype, rows, k, n, group):
    """Hundreds of rows: many chunks of columns, the last of them not full."""
    check_product(pkg, dtype, rows, k, n, group)


@gpu
def test_products_of_special_rows_and_shapes(pkg):
    g = gen(12)
    linear = random_linear(pkg, g, 200, 40, 32, True)
    x = normal(g, 6, 200)
    want = linear(x)
    x[1, 7], x[2, 199], x[4] = math.inf, math.nan, 0.0
    got = linear(x)
    assert torch.equal(got[[0, 3, 5]], want[[0, 3, 5]]) and not torch.isfinite(got[[1, 2]]).any()
    assert torch.equal(got[4], linear.bias)
    assert linear(x[:0]).shape == (0, 40)
    assert torch.equal(linear(x.view(2, 3, 200)).nan_to_num(), got.view(2, 3, 40).nan_to_num())
    assert torch.equal(linear(x[0]), linear(x[:1])[0])
    assert torch.equal(linear(x[[0, 3]]), linear(x[[0, 3]]))  # the same bits each time
    plain = pkg.W4Linear(linear.codes, linear.meta, 200, 40, 32)
    small, large = plain(x[[0, 3]] * 2.0 ** -80), plain(x[[0, 3]] * 2.0 ** 80)
    base = plain(x[[0, 3]])
    assert torch.equal(small * 2.0 ** 80, base) and torch.equal(large * 2.0 ** -80, base)


def test_more_rows_than_a_product_takes(pkg):
    """Sizes are computed in 64 bits: no number of rows is taken for a few."""
    import ctypes as C
    import struct
    from forge_lm_b200 import _native as N
    L, size = N.load(), C.c_int64()
    w = struct.Struct("=QQQ4i").pack(4096, 4096, 0, 1, 1, 32, 0)
    for dtype in (0, 1, 2):
        last = 0
        for rows in (100, 10 ** 6, 2 ** 29, 2 ** 30, 715827883, 1431655766, 2 ** 31 - 1):
            assert L.fb2_w4_matvec_workspace(w, rows, dtype, C.byref(size)) == N.FB2_OK
            assert (size.value > last) if rows < 2 ** 29 else size.value >= rows * 2048 // 16
            last = size.value
            assert L.fb2_w4_matvec(w, rows, 4096, 1, 4096, 1, dtype, None, 0, None) == N.FB2_INVALID_ARG


# ---- logit controls -----------------------------------------------------------------------

def plain_controls(logits, windows=None, rep=None, pres=None, freq=None, biases=None, allowed=None, mask_rows=None):
    out = logits.double().cpu().clone()
    rows, vocab = out.shape
    for r in range(rows):
        if windows is not None:
            for t in set(windows[r]):
                if not 0 <= t < vocab:
                    continue
                x = float(out[r, t])
                if rep is not None:
                    x = x * float(rep[r]) if x < 0 else x / float(rep[r])
                x -= (float(pres[r]) if pres is not None else 0) + (float(freq[r]) if freq is not None else 0) * windows[r].count(t)
                out[r, t] = x
        if biases is not None:
            for t, b in dict(biases[r]).items():
                if 0 <= t < vocab:
                    out[r, t] += b
        if allowed is not None:
            m = r if mask_rows is None else mask_rows[r]
            if 0 <= m < len(allowed):
                bits = (allowed[m].cpu().long()[:, None] >> torch.arange(32)) & 1
                out[r, bits.flatten()[:vocab] == 0] = -math.inf
    return out


def lists(rows, kind):
    flat = [x for r in rows for x in r]
    starts = np.concatenate([[0], np.cumsum([len(r) for r in rows])])
    return torch.tensor(flat, dtype=kind, device="cuda"), torch.tensor(starts, dtype=torch.int32, device="cuda")


def check_controls(got, want):
    # four fp32 operations on values below `size`, then the type's rounding
    assert torch.equal(torch.isfinite(got.cpu()), torch.isfinite(want))
    fine = torch.isfinite(want)
    assert (got.cpu()[~fine] == -math.inf).all()
    assert within(got.cpu()[fine], want[fine], 2.0 ** -22 * (want[fine].abs() + 40))


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 16384), (3, 1003), (2, 4096), (4, 4097), (2, 131071), (5, 33)])
def test_controls_on_logits(pkg, dtype, rows, vocab):
    rnd = random.Random(vocab)
    g = gen(vocab)
    logits = (5 * normal(g, rows, vocab)).to(DTYPES[dtype])
    windows = [[rnd.randrange(-2, min(vocab + 3, 300)) for _ in range(rnd.randrange(0, 700))] + [vocab - 1, vocab, 2 ** 31 - 1]
               for _ in range(rows)]
    windows[0] = windows[0] * 2
    if rows > 2:
        windows[2] = []
    biases = [[(rnd.randrange(-1, vocab + 1), rnd.uniform(-3, 3)) for _ in range(rnd.randrange(0, 50))] for _ in range(rows)]
    biases[0] = biases[0] + [(0, 1.5), (0, -2.5)]  # the last of an id's biases counts
    biases = [[(t, float(np.float32(b))) for t, b in r] for r in biases]
    tokens, token_starts = lists(windows, torch.int32)
    ids, bias_starts = lists([[t for t, _ in r] for r in biases], torch.int32)
    values, _ = lists([[b for _, b in r] for r in biases], torch.float32)
    rep = (1 + torch.rand(rows, device="cuda", generator=g))
    pres, freq = torch.rand(rows, device="cuda", generator=g), torch.rand(rows, device="cuda", generator=g) - 0.5
    allowed = torch.randint(-2 ** 31, 2 ** 31, (3, (vocab + 31) // 32 + 1), device="cuda", generator=g).to(torch.int32)
    allowed[1] = 0
    which = [rnd.randrange(-1, 4) for _ in range(rows)]
    mask_rows = torch.tensor(which, dtype=torch.int32, device="cuda")
    every = dict(tokens=tokens, token_starts=token_starts, repetition=rep, presence=pres, frequency=freq, bias_ids=ids,
                 bias_values=values, bias_starts=bias_starts, allowed=allowed, mask_rows=mask_rows)
    want = plain_controls(logits, windows, rep, pres, freq, biases, allowed, which)
    got = pkg.logit_controls(logits, **every)
    assert got.dtype == logits.dtype and got.data_ptr() != logits.data_ptr()
    check_controls(got, want)
    # rows apart and unaligned, in place
    wide = torch.zeros((rows, vocab + 3), dtype=logits.dtype, device="cuda")
    wide[:, 1:1 + vocab] = logits
    view = wide[:, 1:1 + vocab]
    assert pkg.logit_controls(view, out=view, **every) is view
    assert torch.equal(view, got) and (wide[:, 0] == 0).all() and (wide[:, 1 + vocab:] == 0).all()
    # each control alone
    check_controls(pkg.logit_controls(logits, tokens=tokens, token_starts=token_starts, repetition=rep),
                   plain_controls(logits, windows, rep))
    check_controls(pkg.logit_controls(logits, tokens=tokens, token_starts=token_starts, frequency=freq),
                   plain_controls(logits, windows, freq=freq))
    check_controls(pkg.logit_controls(logits, bias_ids=ids, bias_values=values, bias_starts=bias_starts),
                   plain_controls(logits, biases=biases))
    check_controls(pkg.logit_controls(logits, allowed=allowed, mask_rows=mask_rows),
                   plain_controls(logits, allowed=allowed, mask_rows=which))
    assert torch.equal(pkg.logit_controls(logits), logits)


@gpu
def test_controls_on_special_logits(pkg):
    logits = torch.tensor([[math.inf, -math.inf, math.nan, 1.0, torch.finfo(torch.float32).min]], device="cuda")
    allowed = torch.tensor([[0b11000]], dtype=torch.int32, device="cuda")
    got = pkg.logit_controls(logits, allowed=allowed)
    assert (got[0, :3] == -math.inf).all() and torch.equal(got[0, 3:], logits[0, 3:])  # masked whatever they were
    tokens = torch.tensor([0, 1, 4], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    got = pkg.logit_controls(logits, tokens=tokens, token_starts=starts, repetition=torch.tensor([2.0], device="cuda"))
    assert got[0, 0] == math.inf and got[0, 1] == -math.inf and got[0, 2].isnan() and got[0, 4] == -math.inf


@gpu
def test_controls_of_long_windows(pkg):
    """More tokens in a window than a block has threads many times over; one id thousands of times."""
    g = gen(14)
    vocab = 50000
    logits = normal(g, 2, vocab)
    windows = [torch.randint(0, vocab, (40000,), generator=torch.Generator().manual_seed(1)).tolist(), [77] * 30000]
    tokens, starts = lists(windows, torch.int32)
    freq = torch.tensor([0.25, 0.125], device="cuda")
    got = pkg.logit_controls(logits, tokens=tokens, token_starts=starts, frequency=freq).double().cpu()
    count = torch.stack([torch.bincount(torch.tensor(w), minlength=vocab) for w in windows]).double()
    want = logits.double().cpu() - freq.double().cpu()[:, None] * count
    assert ((got - want).abs() <= 2.0 ** -22 * (want.abs() + 10)).all()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("ids", [511, 768, 769, 4096, 6143, 6145, 9000])
def test_controls_of_lists_of_many_different_ids(pkg, dtype, ids):
    """One row's lists alone are long: what it keeps of them outgrows one size after another."""
    rnd = random.Random(ids)
    vocab = 20001
    logits = (3 * normal(gen(ids), 3, vocab)).to(DTYPES[dtype])
    windows = [[5, 5, 20000], rnd.sample(range(vocab), ids - 200) + [19999] * 40, []]
    some = rnd.sample(range(vocab), 159)
    biases = [[], [(t, float(np.float32(rnd.uniform(-2, 2)))) for t in some + some[:1]], [(7, 1.25)]]
    tokens, token_starts = lists(windows, torch.int32)
    bias_ids, bias_starts = lists([[t for t, _ in r] for r in biases], torch.int32)
    values, _ = lists([[b for _, b in r] for r in biases], torch.float32)
    rep, pres = torch.tensor([1.5, 1.25, 2.0], device="cuda"), torch.tensor([0.5, -0.25, 1.0], device="cuda")
    freq = torch.tensor([0.125, 0.0625, 1.0], device="cuda")
    every = dict(tokens=tokens, token_starts=token_starts, repetition=rep, presence=pres, frequency=freq,
                 bias_ids=bias_ids, bias_values=values, bias_starts=bias_starts)
    got = pkg.logit_controls(logits, **every)
    check_controls(got, plain_controls(logits, windows, rep, pres, freq, biases))
    pkg.logit_controls(logits, out=logits, **every)
    assert torch.equal(logits, got)


def test_controls_refuse_rows_that_overlap(pkg):
    """out in place of the logits, beside them or between them, but not across them."""
    import struct
    from forge_lm_b200 import _native as N
    L, con = N.load(), struct.Struct("=12Q4q6i")

    def status(logits, out, in_row, out_row, rows, vocab=100):
        s = L.fb2_logit_controls(con.pack(logits, out, *[0] * 10, in_row, out_row, 0, 0, rows, vocab, 0, 0, 0, 0), None)
        return s == N.FB2_INVALID_ARG and b"overlap" in L.fb2_last_error()

    at = 1 << 20
    for logits, out, in_row, out_row, rows in ((at, at, 100, 120, 3), (at, at, 0, 100, 3), (at, at + 4, 100, 100, 1),
                                               (at, at + 4, 120, 120, 3), (at, at + 400, 100, 100, 3), (at + 400, at, 100, 100, 3),
                                               (at, at + 440, 220, 200, 9), (at, at + 396, 300, 300, 2), (at + 1000, at, 0, 200, 4)):
        assert status(logits, out, in_row, out_row, rows)


@gpu
def test_controls_between_rows_of_the_logits(pkg):
    g = gen(71)
    both = normal(g, 5, 300)
    keep = both[:, :100].clone()
    allowed = torch.randint(-2 ** 31, 2 ** 31, (5, 4), device="cuda", generator=g).to(torch.int32)
    want = pkg.logit_controls(keep, allowed=allowed)
    pkg.logit_controls(both[:, :100], allowed=allowed, out=both[:, 100:200])
    assert torch.equal(both[:, 100:200], want) and torch.equal(both[:, :100], keep)
    pkg.logit_controls(both[:, :100], allowed=allowed, out=both[:, :100])
    assert torch.equal(both[:, :100], want)
    with pytest.raises(pkg.ArgumentError):
        pkg.logit_controls(both[:, :100], out=both[:, 50:150])


# ---- together -------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_operators_in_a_graph(pkg, dtype):
    """Captured once, replayed with other contents of the same tensors."""
    g = gen(77)
    cache = filled(pkg, g, 12, 16, 2, 64, "int8")
    linear = random_linear(pkg, g, 512, 96, 64, True)
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
    prefix, starts = _i32([40, 90]), _i32([0, 3, 5])
    slots, mask = _i32([40, 41, 42, 186, 187]), _i32([[1], [3], [5], [1], [3]])
    tokens, token_starts = _i32([1, 2, 2, 7, 9]), _i32([0, 3, 4, 4, 5, 5])
    rep = torch.full((5,), 1.5, device="cuda")

    def step(k, v, q):
        cache.write(k, v, slots)
        out, lse = cache.attend(q, table, prefix, starts=starts, mask=mask, max_nodes=3, max_len=96)
        y = linear(out.reshape(5, 512))
        return out, lse, y, pkg.logit_controls(y, tokens=tokens, token_starts=token_starts, repetition=rep)

    def inputs():
        return [normal(g, 5, h, 64).to(DTYPES[dtype]) for h in (2, 2, 8)]

    held = inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*held)
    for _ in range(3):
        for t, new in zip(held, inputs()):
            t.copy_(new)
        want = [t.clone() for t in step(*held)]
        for t in outs:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype,nodes", [("fp32", 3), ("bf16", 3), ("bf16", 40), ("fp16", 40)])
def test_split_attention_in_a_graph(pkg, fmt, dtype, nodes):
    """Chunks, their merge and the tcgen05 blocks captured once; replayed over another
    prefix, other pages and other rows."""
    g = gen(78)
    cache = filled(pkg, g, 200, 16, 2, 64, fmt)
    held = [normal(g, 2 * nodes, 4, 64, dtype=DTYPES[dtype]), _i32([1500, 700]),
            torch.randperm(200, generator=torch.Generator().manual_seed(9))[:200].to(torch.int32).cuda().view(2, 100)]
    starts = _i32([0, nodes, 2 * nodes])

    def step(q, prefix, table):
        return cache.attend(q, table, prefix, starts=starts, max_nodes=nodes, max_len=1600)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*held)
    for lens in ([1500, 700], [3, 1555], [640, 0]):
        held[0].copy_(normal(g, 2 * nodes, 4, 64, dtype=DTYPES[dtype]))
        held[1].copy_(_i32(lens))
        held[2].copy_(held[2].flip(1).clone())
        want = [t.clone() for t in step(*held)]
        for t in outs:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.isfinite(want[1]).all()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@gpu
@pytest.mark.parametrize("fmt,dtype", [("int8", "fp32"), ("int4", "fp32"), ("int8", "bf16"), ("int4", "fp16")])
@pytest.mark.parametrize("scale", [0.0, -0.07, 1e-6])
def test_attention_with_any_scale(pkg, fmt, dtype, scale):
    """No weighting, the smallest scores first, and nearly none; few rows and many."""
    attention_case(pkg, 91, fmt, dtype, [70, 0, 33], [1, 1, 1], 4, 2, 64, 16, False, scale=scale)
    attention_case(pkg, 92, fmt, dtype, [150, 9], [20, 40], 4, 1, 64, 16, True, scale=scale)
    attention_case(pkg, 93, fmt, dtype, [150, 9], [20, 40], 4, 2, 80, 16, True, scale=scale)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim,share", [(48, 6), (80, 3), (128, 8)])
def test_attention_of_many_unaligned_rows(pkg, fmt, dtype, dim, share):
    """The same rows at an odd element and in one piece: the same values."""
    g = gen(dim)
    cache = filled(pkg, g, 40, 16, 2, dim, fmt)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(3)).to(torch.int32).cuda().view(2, 20)
    rows, heads = 33, 2 * share
    flat = normal(g, rows * heads * dim + 1).to(DTYPES[dtype])
    q = flat[1:].view(rows, heads, dim)
    args = (table, _i32([281, 130]))
    kw = dict(starts=_i32([0, 20, 33]), max_nodes=20)
    out, lse = cache.attend(q, *args, **kw)
    again, lse2 = cache.attend(q.clone(), *args, **kw)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    bits = [set(range(i + 1)) for t in (20, 13) for i in range(t)]
    want = plain_attention(cache, q, table.cpu(), [281, 130], [0, 20, 33], bits, 1 / math.sqrt(dim))
    k, v = cache.read(torch.arange(640, dtype=torch.int32, device="cuda"))
    check_attention(dtype, (out, lse), want, float(v.abs().max()),
                    float(q.float().norm(dim=2).max() * k.norm(dim=2).max()) / math.sqrt(dim))


@gpu
@pytest.mark.parametrize("cache", ["int8", "int4"])
def test_example_of_a_decoder(pkg, cache):
    """Drafted generation gives greedy tokens: each is the largest controlled
    logit of a run of the whole text in one piece, up to the difference that
    a stored code one step off makes (a score moves by 1 / 127 or 1 / 15 of
    its key's range at most where sums of another order round another way)."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "quantised_decode.py")
    spec = importlib.util.spec_from_file_location("quantised_decode", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    cfg = pkg.ModelConfig(512, 128, 128, 3, 4)
    params = pkg.init_params(cfg, 5)
    prompts = [[1, 2, 3, 1, 2, 3, 1, 2], [7], [9, 8] * 20]
    words = torch.full((1, 16), -1, dtype=torch.int32, device="cuda")
    words[0, 1], words[0, 15] = 0, 0  # neither 32..63 nor 480..511

    def model():
        return ex.QuantisedGpt(cfg, params, 3, cache, dtype=torch.float32)

    out, steps = ex.generate(model(), prompts, 24, draft=4, repetition=0.8, allowed=words)
    assert [len(t) for t in out] == [24] * 3 and 1 <= steps <= 24
    once, single = ex.generate(model(), prompts, 24, draft=0, repetition=0.8, allowed=words)
    assert single == 24 and steps < 24  # a repetition "penalty" below one repeats itself: drafts are kept
    text = [p + t for p, t in zip(prompts, out)]
    whole = model()
    starts, slots = [0], []
    for s, t in enumerate(text):
        starts.append(starts[-1] + len(t))
        slots += whole.slots(s, range(len(t)))
    logits = whole.logits([x for t in text for x in t], [i for t in text for i in range(len(t))], slots, [0, 0, 0],
                          starts, max_nodes=max(map(len, text)))
    step = 1 / 127 if cache == "int8" else 1 / 15
    for s, (p, t) in enumerate(zip(prompts, text)):
        for i in range(len(p), len(t)):
            assert not (32 <= t[i] < 64 or t[i] >= 480)
            row = logits[starts[s] + i - 1:starts[s] + i]
            want = plain_controls(row, [t[:i]], [0.8], allowed=words, mask_rows=[0])[0]
            assert float(want[t[i]]) >= float(want.max()) - step * float(row.abs().max())


@gpu
def test_buffers_that_are_replaced(pkg):
    """Calls use the held tensors' memory as it is at the call; ones of another size are refused."""
    g = gen(81)
    cache = filled(pkg, g, 4, 16, 2, 64, "int8")
    slots = torch.arange(64, dtype=torch.int32, device="cuda")
    k, v = cache.read(slots)
    codes, meta = cache.codes, cache.meta
    old = codes.data_ptr()
    codes.data, meta.data = codes.clone(), meta.clone()
    codes.data[0], meta.data[0] = 128, 0
    assert codes.data_ptr() != old
    k2, v2 = cache.read(slots)
    assert (k2[:16] == 0).all() and torch.equal(k2[16:], k[16:]) and torch.equal(v2[16:], v[16:])
    linear = random_linear(pkg, g, 128, 48, 64, True)
    x = normal(g, 2, 128)
    y = linear(x)
    linear.codes.data = torch.zeros_like(linear.codes)
    linear.meta.data = torch.zeros_like(linear.meta)
    assert torch.equal(linear(x), linear.bias.expand(2, 48))
    linear.bias.data = linear.bias + 1
    assert torch.equal(linear(x), linear.bias.expand(2, 48)) and not torch.equal(y, linear(x))
    for tensor, change in ((codes, lambda: codes.resize_(1, 2, 2, 16, 64)), (meta, lambda: meta.set_(torch.zeros(3, dtype=torch.int32, device="cuda"))),
                           (linear.bias, lambda: linear.bias.resize_(47)), (linear.codes, lambda: setattr(linear.codes, "data", linear.codes[:1]))):
        keep = tensor.data
        change()
        with pytest.raises(pkg.ArgumentError):
            cache.read(slots) if tensor is codes or tensor is meta else linear(x)
        with pytest.raises(pkg.ArgumentError):
            cache.write(k, v, slots) if tensor is codes or tensor is meta else linear(x)
        tensor.data = keep.clone()
        if tensor is codes:
            codes.resize_(4, 2, 2, 16, 64)


@gpu
def test_gradients_are_not_cut_in_silence(pkg):
    """A backward pass through a result of an input that requires a gradient raises."""
    g = gen(83)
    cache = filled(pkg, g, 4, 16, 2, 64, "int8")
    linear = random_linear(pkg, g, 64, 48, 64, True)
    x, q, logits = normal(g, 2, 64), normal(g, 1, 4, 64), normal(g, 2, 32)
    calls = ((x, lambda t: linear(t)), (x, lambda t: linear(t.view(1, 2, 64))), (logits, lambda t: pkg.logit_controls(t)),
             (q, lambda t: cache.attend(t, _i32([[0, 1]]), _i32([20]))[0]), (q, lambda t: cache.attend(t, _i32([[0, 1]]), _i32([20]))[1]))
    for value, call in calls:
        plain = call(value)
        assert not plain.requires_grad
        tracked = value.clone().requires_grad_()
        with torch.no_grad():
            assert not call(tracked).requires_grad
        got = call(tracked)
        assert torch.equal(got, plain)
        other = torch.ones((), device="cuda", requires_grad=True)
        with pytest.raises(RuntimeError, match="computes no gradient"):
            (got.sum() * other).backward()
        assert tracked.grad is None
    tracked = logits.clone().requires_grad_()
    with pytest.raises(pkg.ArgumentError):
        pkg.logit_controls(tracked, out=torch.empty_like(logits))
    with torch.no_grad():
        pkg.logit_controls(tracked, out=torch.empty_like(logits))
    # values are stored and packed whether they require a gradient or not
    k = normal(g, 1, 2, 64).requires_grad_()
    cache.write(k, k, _i32([5]))
    pkg.W4Linear.pack(torch.nn.Parameter(normal(g, 64, 16)), 32)


@gpu
def test_changed_tensors_are_counted(pkg):
    """What a call writes into has a new version: autograd refuses to use a stale value."""
    cache = pkg.QuantKvCache.empty(2, 16, 1, 32)
    k = torch.ones((1, 1, 32), device="cuda")
    before = cache.codes._version, cache.meta._version
    cache.write(k, k, _i32([3]))
    assert cache.codes._version > before[0] and cache.meta._version > before[1]
    before = cache.codes._version
    cache.read(_i32([3]))
    assert cache.codes._version == before
    logits = torch.randn((2, 64), device="cuda")
    weight = torch.ones((2, 64), device="cuda", requires_grad=True)
    loss = (weight * logits).sum()  # keeps logits for weight's gradient
    before = logits._version
    pkg.logit_controls(logits, allowed=torch.zeros((2, 2), dtype=torch.int32, device="cuda"), out=logits)
    assert logits._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # has no versions
        out = torch.zeros((2, 64), device="cuda")
        assert pkg.logit_controls(torch.ones((2, 64), device="cuda"), out=out) is out and (out == 1).all()
        other = pkg.QuantKvCache.empty(2, 16, 1, 32)
        other.write(k, k, _i32([3]))
    other.write(k, k, _i32([4]))
    assert all((t == 1).all() for t in other.read(_i32([3, 4])))


# ---- refusals -------------------------------------------------------------------------------

@gpu
def test_negated_views_are_refused(pkg):
    """Their memory holds the values with the other sign."""
    g = gen(82)
    cache = pkg.QuantKvCache.empty(2, 16, 1, 32)
    k, slots = normal(g, 1, 1, 32), _i32([3])
    neg = torch._neg_view(k)
    assert neg.is_neg() and torch.equal(neg, -k)
    w = normal(g, 32, 16)
    linear = pkg.W4Linear.pack(w, 32)
    logits = normal(g, 1, 32)
    for call in (lambda: cache.write(neg, k, slots), lambda: cache.write(k, neg, slots),
                 lambda: cache.attend(neg, _i32([[0, 1]]), _i32([4])), lambda: linear(neg),
                 lambda: pkg.W4Linear.pack(torch._neg_view(w), 32), lambda: pkg.logit_controls(torch._neg_view(logits)),
                 lambda: pkg.logit_controls(logits, out=torch._neg_view(logits.clone()))):
        with pytest.raises(pkg.ArgumentError, match="negated"):
            call()
    cache.write(neg.resolve_neg(), k, slots)
    got, _ = cache.read(slots)
    assert ((got + k).abs() <= k.abs().max() / 250).all()


@gpu
def test_refusals_on_the_device(pkg):
    E = pkg.ArgumentError
    cache = pkg.QuantKvCache.empty(4, 16, 2, 64)
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")
    k = torch.zeros((3, 2, 64), device="cuda")
    for bad in (dict(page_size=12), dict(page_size=4), dict(page_size=2048), dict(head_dim=24), dict(head_dim=272),
                dict(fmt="fp8")):
        with pytest.raises(E):
            pkg.QuantKvCache.empty(**{**dict(n_pages=2, page_size=16, n_kv_heads=2, head_dim=64), **bad})
    for args in ((k[:2], k, slots), (k, k.half(), slots), (k.cpu(), k, slots), (k, k, slots.long()), (k, k, slots.cpu()),
                 (k.double(), k.double(), slots), (k[:, :1], k, slots), (k[..., :32], k, slots)):
        with pytest.raises(E):
            cache.write(*args)
    with pytest.raises(E):
        cache.read(slots, torch.float64)
    with pytest.raises(E):
        cache.read(slots.view(3, 1).expand(3, 2))
    table = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    prefix, starts = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    good = dict(q=torch.zeros((3, 4, 64), device="cuda"), page_table=table, prefix_lens=prefix)
    cache.attend(**good)
    for bad in (dict(q=good["q"][:, :3]), dict(q=good["q"][..., :32]), dict(q=good["q"].double()), dict(q=good["q"][:2]),
                dict(page_table=table.long()), dict(page_table=table.t()), dict(prefix_lens=prefix[:2]),
                dict(prefix_lens=prefix.float()), dict(starts=starts[:3]), dict(max_nodes=2),
                dict(mask=torch.zeros((3, 0), dtype=torch.int32, device="cuda")), dict(scale=math.nan), dict(scale=math.inf),
                dict(starts=starts, max_nodes=40, mask=torch.zeros((3, 1), dtype=torch.int32, device="cuda")),
                dict(starts=starts, max_nodes=0), dict(max_len=-1)):
        with pytest.raises(E):
            cache.attend(**{**good, **bad})
    w = torch.zeros((64, 32), device="cuda")
    linear = pkg.W4Linear.pack(w, 32)
    for call in (lambda: pkg.W4Linear.pack(w, 16), lambda: pkg.W4Linear.pack(w.double()), lambda: pkg.W4Linear.pack(w.t()),
                 lambda: linear(torch.zeros((2, 63), device="cuda")), lambda: linear(torch.zeros((2, 64))),
                 lambda: linear(torch.zeros((2, 64), device="cuda", dtype=torch.float64)),
                 lambda: linear(torch.zeros((64, 2), device="cuda").t()),
                 lambda: pkg.W4Linear(linear.codes, linear.meta, 64, 48, 32),
                 lambda: pkg.W4Linear(linear.codes, linear.meta, 64, 32, 32, bias=torch.zeros(31, device="cuda"))):
        with pytest.raises(E):
            call()
    logits = torch.zeros((2, 100), device="cuda")
    t32 = torch.zeros(4, dtype=torch.int32, device="cuda")
    s3 = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    row = torch.ones(2, device="cuda")
    for bad in (dict(tokens=t32), dict(repetition=row), dict(tokens=t32, token_starts=s3[:2]),
                dict(tokens=t32.long(), token_starts=s3), dict(tokens=t32, token_starts=s3, repetition=row[:1]),
                dict(bias_ids=t32, bias_starts=s3), dict(bias_ids=t32, bias_values=row, bias_starts=s3),
                dict(allowed=torch.zeros((2, 3), dtype=torch.int32, device="cuda")),
                dict(allowed=torch.zeros((1, 4), dtype=torch.int32, device="cuda")), dict(mask_rows=t32[:2]),
                dict(out=torch.zeros((2, 99), device="cuda")), dict(out=logits.half())):
        with pytest.raises(E):
            pkg.logit_controls(logits, **bad)
    with pytest.raises(E):
        pkg.logit_controls(logits.t())
    with pytest.raises(E):
        pkg.logit_controls(logits.double())


def test_refusals_of_the_c_entries(pkg):
    """What the C entry points refuse before any device work."""
    import ctypes as C
    import struct
    from forge_lm_b200 import _native as N
    L = N.load()
    cache = struct.Struct("=QQ6i")
    a, b = C.c_int64(), C.c_int64()
    assert L.fb2_kvq_sizes(cache.pack(0, 0, 10, 16, 3, 64, 0, 0), C.byref(a), C.byref(b)) == N.FB2_OK
    assert (a.value, b.value) == (10 * 16 * 3 * 2 * 64, 10 * 16 * 3 * 2 * 4)
    assert L.fb2_kvq_sizes(cache.pack(0, 0, 10, 16, 3, 64, 1, 0), C.byref(a), C.byref(b)) == N.FB2_OK
    assert a.value == 10 * 16 * 3 * 2 * 32
    for bad in ((-1, 16, 3, 64, 0), (10, 17, 3, 64, 0), (10, 16, 0, 64, 0), (10, 16, 3, 8, 0), (10, 16, 3, 64, 2),
                (2 ** 31 - 1, 16, 3, 64, 0)):
        assert L.fb2_kvq_sizes(cache.pack(0, 0, *bad, 0), C.byref(a), C.byref(b)) == N.FB2_INVALID_ARG
    assert L.fb2_kvq_sizes(None, C.byref(a), C.byref(b)) == N.FB2_INVALID_ARG
    ok = cache.pack(4096, 4096, 10, 16, 3, 64, 0, 0)
    args = (1, 1, 1, 1)
    assert L.fb2_kvq_write(ok, 1, None, None, 0, *args, None, None) == N.FB2_INVALID_ARG
    assert L.fb2_kvq_write(ok, -1, 4096, 4096, 0, *args, 4096, None) == N.FB2_INVALID_ARG
    assert L.fb2_kvq_write(ok, 1, 4096, 4096, 7, *args, 4096, None) == N.FB2_INVALID_ARG
    assert L.fb2_kvq_write(ok, 1, 4098, 4096, 0, *args, 4096, None) == N.FB2_INVALID_ARG
    assert L.fb2_kvq_write(ok, 0, None, None, 0, *args, None, None) == N.FB2_OK
    assert L.fb2_kvq_write(cache.pack(4097, 4096, 10, 16, 3, 64, 0, 0), 1, 4096, 4096, 0, *args, 4096, None) == N.FB2_INVALID_ARG
    assert L.fb2_kvq_read(ok, 1, 4096, 4100, 4096, 0, None) == N.FB2_INVALID_ARG
    assert L.fb2_kvq_read(ok, 0, None, None, None, 0, None) == N.FB2_OK
    att = struct.Struct("=8Q4q8ifi")
    base = [4096] * 3 + [4096, 4096, 0, 0, 0] + [0, 64, 64, 4] + [2, 2, 6, 0, 4, 1, 0, 0] + [0.125, 0]
    assert L.fb2_kvq_attend_workspace(ok, att.pack(*base), C.byref(a)) == N.FB2_OK and a.value >= 0
    for where, value in ((12, -1), (13, 3), (14, 7), (14, 0), (15, 3), (16, -1), (17, 0), (17, 2), (18, -1), (11, 3),
                         (20, math.nan)):
        bad = list(base)
        bad[where] = value
        assert L.fb2_kvq_attend_workspace(ok, att.pack(*bad), C.byref(a)) == N.FB2_INVALID_ARG, where
        assert L.fb2_kvq_attend(ok, att.pack(*bad), None) == N.FB2_INVALID_ARG, where
    assert b"" != L.fb2_last_error()
    lin = struct.Struct("=QQQ4i")
    assert L.fb2_w4_sizes(lin.pack(0, 0, 0, 100, 33, 32, 0), C.byref(a), C.byref(b)) == N.FB2_OK
    assert (a.value, b.value) == (3 * 2 * 512, 3 * 4 * 64)
    for bad in ((0, 33, 32), (100, 0, 32), (100, 33, 48), (2 ** 31 - 1, 33, 32)):
        assert L.fb2_w4_sizes(lin.pack(0, 0, 0, *bad, 0), C.byref(a), C.byref(b)) == N.FB2_INVALID_ARG
    w = lin.pack(4096, 4096, 0, 100, 33, 32, 0)
    assert L.fb2_w4_pack(w, 4096, 0, 32, None) == N.FB2_INVALID_ARG
    assert L.fb2_w4_pack(w, None, 0, 33, None) == N.FB2_INVALID_ARG
    assert L.fb2_w4_matvec(w, 2, 4096, 100, 4096, 32, 0, None, 0, None) == N.FB2_INVALID_ARG
    assert L.fb2_w4_matvec(w, -1, 4096, 100, 4096, 33, 0, None, 0, None) == N.FB2_INVALID_ARG
    assert L.fb2_w4_matvec(w, 0, None, 0, None, 0, 0, None, 0, None) == N.FB2_OK
    con = struct.Struct("=12Q4q6i")
    base = [4096, 4096] + [0] * 10 + [100, 100, 0, 0] + [2, 100, 0, 0, 0, 0]
    for where, value in ((0, 0), (1, 0), (0, 4097), (13, 99), (2, 4096), (7, 4096), (10, 4096), (16, -1),
                         (16, 70000), (17, -1), (18, 5)):
        bad = list(base)
        bad[where] = value
        assert L.fb2_logit_controls(con.pack(*bad), None) == N.FB2_INVALID_ARG, where
    assert L.fb2_logit_controls(None, None) == N.FB2_INVALID_ARG
    base[16] = 0
    assert L.fb2_logit_controls(con.pack(*base), None) == N.FB2_OK

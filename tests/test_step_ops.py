"""The serving operators around attention and 4-bit layers (pages of sequences,
residual stream and norms, 8-bit linear layers, verification of drafts) against
plain implementations in whole numbers or 64 bits, at the sizes and values where
they can go wrong, and their refusals."""
from __future__ import annotations

import itertools
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
    tol = tol.cpu() if torch.is_tensor(tol) else tol
    low, high = (want - tol).to(got.dtype), (want + tol).to(got.dtype)
    return bool(((got >= low) & (got <= high)).all())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- pages of sequences ------------------------------------------------------------

class Pages:
    """The rules in Python lists."""

    def __init__(self, seqs, width, pages, page):
        self.page, self.width = page, width
        self.table = [[-1] * width for _ in range(seqs)]
        self.lens = [0] * seqs
        self.free = list(range(pages - 1, -1, -1))

    def need(self, n):
        return -(-n // self.page)

    def extend(self, counts, most):
        starts, prefix, slots, positions = [0], list(self.lens), [], []
        asked = wanted = 0
        had = len(self.free)
        for b, count in enumerate(counts):
            n = self.lens[b]
            if count < 0 or n < 0 or n + count > self.width * self.page:
                count = 0
            need = self.need(n + count) - self.need(n) if count else 0
            asked, wanted = asked + count, wanted + need
            if asked <= most and (need == 0 or wanted <= had):
                for i in range(need):
                    self.table[b][self.need(n) + i] = self.free.pop()
                for p in range(n, n + count):
                    slots.append(self.table[b][p // self.page] * self.page + p % self.page)
                    positions.append(p)
                self.lens[b] = n + count
            starts.append(len(slots))
        return starts, prefix, slots + [-1] * (most - len(slots)), positions + [0] * (most - len(positions))

    def truncate(self, lens):
        dropped = []
        for b, want in enumerate(lens):
            want = max(want, 0)
            if want < self.lens[b]:
                for i in range(self.need(want), self.need(self.lens[b])):
                    dropped.append(self.table[b][i])
                    self.table[b][i] = -1
                self.lens[b] = want
        self.free += dropped[::-1]

    def same(self, pages):
        n = int(pages.n_free)
        return (n == len(self.free) and pages.free[:n].tolist() == self.free and pages.lens.tolist() == self.lens
                and pages.table.tolist() == self.table)


@gpu
@pytest.mark.parametrize("seqs,width,pages,page,most", [(1, 1, 1, 8, 8), (1, 40, 50, 16, 300), (3, 7, 12, 8, 40), (33, 5, 100, 16, 200),
                                                         (1024, 3, 2000, 8, 9000), (1500, 2, 900, 32, 4000), (16384, 1, 9000, 8, 30000), (40, 400, 12000, 8, 90000),
                                                         (2, 9000, 17000, 8, 140001)])
def test_pages_come_and_go(pkg, seqs, width, pages, page, most):
    rng = random.Random(seqs)
    own, want = pkg.PageTable.empty(seqs, width, pages, page), Pages(seqs, width, pages, page)
    assert want.same(own)
    for step in range(6):
        counts = [rng.choice([0, 1, 1, 2, page, rng.randint(0, width * page)]) for _ in range(seqs)]
        if step == 3:
            counts = [-c if i % 5 == 2 else c for i, c in enumerate(counts)]  # refused one by one
        got = own.extend(ints(counts), most)
        for g, w in zip(got, want.extend(counts, most)):
            assert g.dtype == torch.int32 and g.tolist() == w
        assert want.same(own)
        to = [rng.choice([n, n + 3, n - 1, n // 2, 0, -1]) for n in want.lens]
        own.truncate(ints(to))
        want.truncate(to)
        assert want.same(own)


@gpu
def test_pages_that_were_dropped_come_back(pkg):
    own = pkg.PageTable.empty(4, 8, 20, 8)
    own.extend(ints([5, 17, 0, 30]), 64)
    before = [t.clone() for t in (own.table, own.lens, own.free[:int(own.n_free)])]
    first = own.extend(ints([9, 1, 8, 12]), 64)
    own.truncate(first[1])
    assert all(torch.equal(a, b) for a, b in zip(before, (own.table, own.lens, own.free[:int(own.n_free)])))
    again = own.extend(ints([9, 1, 8, 12]), 64)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@gpu
def test_pages_without_room(pkg):
    own = pkg.PageTable.empty(3, 4, 5, 8)
    # 3 pages, then 3 of the 2 that are left, then none
    starts, prefix, slots, positions = own.extend(ints([20, 17, 0]), 100)
    assert starts.tolist() == [0, 20, 20, 20] and own.lens.tolist() == [20, 0, 0] and int(own.n_free) == 2
    assert slots[20:].eq(-1).all() and positions[20:].eq(0).all()
    # a sequence that needs no page is served behind one that gets none
    starts, *_ = own.extend(ints([0, 32, 0]), 100)
    assert starts.tolist() == [0, 0, 0, 0]
    starts, *_ = own.extend(ints([4, 0, 8]), 100)
    assert starts.tolist() == [0, 4, 4, 12] and own.lens.tolist() == [24, 0, 8]
    # rows: the second would pass them, the third with it
    own.truncate(ints([0, 0, 0]))
    starts, *_ = own.extend(ints([3, 6, 2]), 8)
    assert starts.tolist() == [0, 3, 3, 3]
    starts, _, slots, _ = own.extend(ints([0, 0, 0]), 0)
    assert starts.tolist() == [0, 0, 0, 0] and slots.numel() == 0
    # 33 tokens do not fit 4 pages of 8, whatever the others ask
    starts, *_ = own.extend(ints([0, 33, 8]), 100)
    assert starts.tolist() == [0, 0, 0, 8]


@gpu
def test_pages_of_malformed_state(pkg):
    """Lengths, lists and counts that no sequence of calls makes: nothing outside the buffers is touched."""
    own = pkg.PageTable.empty(4, 4, 6, 8)
    own.lens.copy_(ints([-3, 2 ** 31 - 1, 33, 5]))
    own.table[3, 0] = 5
    own.free.copy_(ints([0, 9, -7, 2 ** 31 - 1, 1, 5]))
    own.n_free.fill_(2 ** 31 - 1)  # read as 6
    starts, prefix, slots, _ = own.extend(ints([2 ** 31 - 1, 1, 1, 20]), 50)
    assert starts.tolist() == [0, 0, 0, 0, 20] and prefix.tolist() == [-3, 2 ** 31 - 1, 33, 5]
    # pages 5 (its own), 5, 1 and what no page is
    assert slots[:20].tolist() == [45, 46, 47] + list(range(40, 48)) + list(range(8, 16)) + [-1]
    own.n_free.fill_(6)
    own.truncate(ints([0, 0, 0, 0]))
    assert own.lens.tolist() == [0 if n == 25 else n for n in (-3, 2 ** 31 - 1, 33, 25)]
    assert int(own.n_free) == 6 and own.table[3].tolist() == [-1] * 4
    own.n_free.fill_(-5)
    starts, *_ = own.extend(ints([0, 0, 0, 1]), 8)
    assert starts.tolist() == [0] * 5


# ---- residual stream and norms ---------------------------------------------------------

def plain_norm(v, w, b, kind, eps):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    out = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * w.double()
    return out if b is None else out + b.double()


def norm_case(g, rows, dim, dtype, stream, post, gate, bias=True, strided=False):
    def make(n, t):
        wide = normal(g, n, dim + (5 if strided else 0)).to(t)
        return wide[:, 3:3 + dim] if strided else wide
    c = dict(h=make(rows, dtype), x=2 * make(rows, stream) + 0.5, weight=1 + 0.2 * normal(g, dim),
             bias=0.2 * normal(g, dim) if bias else None)
    if post:
        c.update(post_weight=1 + 0.2 * normal(g, dim), post_bias=0.2 * normal(g, dim) if bias else None)
    if gate:
        c["gate"] = make(rows, dtype) if gate == "rows" else normal(g, dim).to(dtype)
    return c


def plain_residual_norm(c, scale, kind, eps):
    h = c["h"].double()
    if c.get("post_weight") is not None:
        h = plain_norm(h, c["post_weight"], c["post_bias"], kind, eps)
    if c.get("gate") is not None:
        h = h * c["gate"].double()
    s = c["x"].double() + scale * h
    return s, plain_norm(s, c["weight"], c["bias"], kind, eps)


# A row's sums of up to 32768 terms: at most 32 in a thread, 5 steps over lanes, 32 warps, so
# fewer than 80 roundings on one path: 2^-24 * 80 < 2^-17 relative in a mean or variance.
SUMS = 2.0 ** -17


def check_norm(c, got, scale, kind, eps):
    s, y = plain_residual_norm(c, scale, kind, eps)
    # post(h): a relative SUMS of its size (values of some units), then three roundings
    big = s.abs().amax(1, keepdim=True).clamp(min=1) + 8
    off = 2.0 ** -22 * big + (SUMS * 8 if c.get("post_weight") is not None else 0)
    assert got[0].dtype == c["x"].dtype and within(got[0], s, off)
    # y: an error of s as itself, in its mean and in its variance, over the row's spread; sums as said
    v = s - s.mean(1, keepdim=True) if kind == "layer" else s
    spread = torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    off = (4 * off / spread + 2 * SUMS * (1 + v.abs() / spread + s.abs().mean(1, keepdim=True) / spread)) * 2 + 2.0 ** -22
    assert within(got[1], y, off * (1 + v.abs() / spread))


@gpu
@pytest.mark.parametrize("dtype,stream", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,dim", [(1, 768), (5, 64), (3, 1), (7, 257), (9, 1000), (2, 1025), (4, 4096), (3, 5001), (2, 16384), (2, 32767), (2, 32768)])
def test_residual_and_norm(pkg, dtype, stream, kind, rows, dim):
    g = gen(rows * dim)
    for post, gate, strided in ((False, None, False), (True, "rows", False), (True, "all", True), (False, "rows", True)):
        c = norm_case(g, rows, dim, DTYPES[dtype], DTYPES[stream], post, gate, bias=kind == "layer", strided=strided)
        got = pkg.residual_norm(c["h"], c["x"], c["weight"], c["bias"], post_weight=c.get("post_weight"),
                                post_bias=c.get("post_bias"), gate=c.get("gate"), scale=0.7, kind=kind, eps=1e-5)
        assert got[1].dtype == DTYPES[dtype]
        check_norm(c, got, 0.7, kind, 1e-5)


@gpu
@pytest.mark.parametrize("stream", ["fp32", "bf16"])
def test_norm_alone(pkg, stream):
    g = gen(1)
    c = norm_case(g, 6, 333, torch.bfloat16, DTYPES[stream], False, None)
    c["h"] = torch.zeros_like(c["h"])
    got = pkg.residual_norm(None, c["x"], c["weight"], c["bias"], dtype=torch.bfloat16)
    assert got[0] is c["x"] and got[1].dtype == torch.bfloat16
    check_norm(c, got, 1.0, "layer", 1e-5)
    assert pkg.residual_norm(None, c["x"], c["weight"])[1].dtype == DTYPES[stream]


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,dim", [(1, 768), (11, 33), (4, 1024), (5, 4099)])
def test_norm_into_codes(pkg, dtype, kind, rows, dim):
    """The codes stand for y to half a step of its row, and the error that y itself may have."""
    g = gen(dim)
    c = norm_case(g, rows, dim, DTYPES[dtype], torch.float32, True, "rows")
    args = dict(post_weight=c["post_weight"], post_bias=c["post_bias"], gate=c["gate"], scale=1.3, kind=kind)
    s, codes, scales = pkg.residual_norm(c["h"], c["x"], c["weight"], c["bias"], quantise=True, **args)
    dense = pkg.residual_norm(c["h"], c["x"], c["weight"], c["bias"], **args)
    assert torch.equal(s, dense[0]) and codes.dtype == torch.int8 and scales.dtype == torch.float32
    assert codes.shape == (rows, dim) and codes.stride(0) % 16 == 0
    _, y = plain_residual_norm(c, 1.3, kind, 1e-5)
    top = y.abs().amax(1)
    assert ((scales.double() - top / 127).abs() <= 1e-4 * top / 127).all()
    step = scales.double()[:, None]
    assert ((codes.double() * step - y).abs() <= 0.5 * step * (1 + 1e-4) + 1e-4 * (1 + y.abs())).all()
    if dtype == "fp32":  # y in hand: the codes are its own
        again, its = pkg.quantise_rows(dense[1])
        assert torch.equal(again, codes) and torch.equal(its, scales)


@gpu
def test_norm_of_special_rows(pkg):
    x = torch.randn((6, 100), generator=torch.Generator().manual_seed(2))
    x[1] = 3.0                    # no variance
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4] = 0.0
    x = x.cuda()
    h = torch.zeros_like(x)
    w, b = torch.ones(100, device="cuda"), torch.full((100,), 0.25, device="cuda")
    for kind in ("layer", "rms"):
        s, y = pkg.residual_norm(h, x, w, b, kind=kind)
        assert torch.equal(s.nan_to_num(9), x.nan_to_num(9)) and y[2].isnan().all() and y[0].isfinite().all() and y[5].isfinite().all()
        assert not y[3].isfinite().all() and y[4].eq(0.25).all()
        assert y[1].sub(0.25 if kind == "layer" else 1.25).abs().max() < 1e-5
        _, codes, scales = pkg.residual_norm(h, x, w, b, kind=kind, quantise=True)
        assert scales[2].isnan() and scales[3].isnan() and codes[2].eq(0).all() and scales[[0, 1, 4, 5]].isfinite().all()


# ---- rows as codes, 8-bit products ---------------------------------------------------------

def plain_codes(x):
    """The formula, with its roundings to fp32."""
    x = x.float().cpu()
    top = x.abs().amax(-1, keepdim=True)
    live = top >= 1e-35
    inv = torch.div(torch.tensor(127.0), torch.where(live, top, 1.0))
    codes = torch.where(live, torch.round(x * inv), 0.0)
    return codes, torch.where(live, top / torch.tensor(127.0), 0.0).squeeze(-1)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 16), (5, 77), (2, 768), (9, 2056), (2, 40001)])
def test_rows_as_codes(pkg, dtype, rows, dim):
    g = gen(dim)
    x = normal(g, rows, dim)
    x[::2] = torch.round(x[::2] * 8) / 8  # many values halfway
    for x in (x.to(DTYPES[dtype]), normal(g, rows, dim + 3, dtype=DTYPES[dtype])[:, 1:1 + dim]):
        codes, scales = pkg.quantise_rows(x)
        want, its = plain_codes(x)
        assert torch.equal(codes.cpu().float(), want) and torch.equal(scales.cpu(), its)
        assert codes.data_ptr() % 16 == 0 and (rows == 1 or codes.stride(0) % 16 == 0)


@gpu
def test_codes_of_special_rows(pkg):
    x = torch.randn((7, 50), generator=torch.Generator().manual_seed(3))
    x[0] = 0.0
    x[1, 4], x[2, 49], x[3, 0] = math.nan, math.inf, -math.inf
    x[4] *= 1e-38
    x[5] *= 1e37
    codes, scales = pkg.quantise_rows(x.cuda())
    codes, scales = codes.cpu(), scales.cpu()
    assert scales[1:4].isnan().all() and codes[:5].eq(0).all() and scales[0] == 0 and scales[4] == 0
    for r in (5, 6):
        want, its = plain_codes(x[r:r + 1])
        assert torch.equal(codes[r:r + 1].float(), want) and scales[r] == its[0]


def w8_case(pkg, g, k, n, bias=True, pad=0):
    codes = torch.full((n, -(-k // 16) * 16 + pad), 99, dtype=torch.int8, device="cuda")[:, :k]  # what is behind a row does not count
    codes.copy_(torch.randint(-128, 128, (n, k), device="cuda", generator=g))
    return pkg.W8Linear(codes, torch.rand(n, device="cuda", generator=g) + 0.1, normal(g, n) if bias else None)


def check_w8(linear, codes, scales, got):
    """Exact sums; a fp32 rounding of the sum, two products and an addition."""
    sums = codes.double().cpu() @ linear.codes.double().cpu().T
    part = sums * linear.scales.double().cpu() * scales.double().cpu()[:, None]
    bias = 0.0 if linear.bias is None else linear.bias.double().cpu()
    assert within(got, part + bias, 2.0 ** -24 * (3 * part.abs() + (part + bias).abs()) * 1.01)


ROWS = [1, 2, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 200, 300]


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("k,n", [(1, 1), (16, 7), (100, 130), (128, 128), (768, 257), (1000, 33), (2064, 400)])
def test_products_of_codes(pkg, dtype, k, n):
    g = gen(k + n)
    linear = w8_case(pkg, g, k, n, bias=n % 2 == 1, pad=16 * (k % 3))
    for rows in ROWS:
        x = torch.randint(-128, 128, (rows, -(-k // 16) * 16 + 16), device="cuda", generator=g).to(torch.int8)[:, :k]
        scales = torch.rand(rows, device="cuda", generator=g) + 0.1
        y = linear(x, scales=scales, dtype=DTYPES[dtype])
        assert y.shape == (rows, n) and y.dtype == DTYPES[dtype]
        check_w8(linear, x, scales, y)


@gpu
@pytest.mark.parametrize("rows,k,n", [(1, 131072, 40), (3, 40000, 300), (20, 16384, 128), (1, 8192, 9000), (700, 520, 1100),
                                      (1500, 4096, 520), (4100, 256, 700)])
def test_products_of_codes_at_length(pkg, rows, k, n):
    g = gen(k + n)
    linear = w8_case(pkg, g, k, n)
    linear.codes[: n // 2].fill_(-128)  # the largest sums there are
    x = torch.randint(-128, 128, (rows, k), device="cuda", generator=g).to(torch.int8)
    x[0] = 127
    scales = torch.rand(rows, device="cuda", generator=g) + 0.1
    check_w8(linear, x, scales, linear(x, scales=scales))


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,k,n", [(1, 768, 2304), (1, 77, 50), (4, 1000, 60), (13, 512, 1000), (150, 640, 96), (1, 8200, 64)])
def test_products_of_values(pkg, dtype, rows, k, n):
    g = gen(k)
    linear = w8_case(pkg, g, k, n)
    x = normal(g, rows, k + 2, dtype=DTYPES[dtype])
    for x in (x[:, 1:1 + k], x[:, :k].contiguous()):
        y = linear(x)
        assert y.dtype == DTYPES[dtype]
        codes, scales = plain_codes(x)
        check_w8(linear, codes, scales, y)
        assert torch.equal(y, linear(*pkg.quantise_rows(x), dtype=DTYPES[dtype]))
    assert torch.equal(linear(x.view(1, rows, 1, k))[0, :, 0], y)
    assert linear(x, dtype=torch.float32).dtype == torch.float32


@gpu
@pytest.mark.parametrize("rows", [1, 3, 140])
def test_products_of_special_rows(pkg, rows):
    g = gen(9)
    linear = w8_case(pkg, g, 300, 150)
    x = normal(g, rows, 300)
    x[rows // 2, 17] = math.nan
    y = linear(x)
    assert y[rows // 2].isnan().all()
    keep = [r for r in range(rows) if r != rows // 2]
    assert y[keep].isfinite().all()
    assert torch.equal(linear(torch.zeros_like(x)), linear.bias.expand(rows, 150))
    assert linear(x[:0]).shape == (0, 150)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("k,n", [(64, 16), (100, 77), (1, 40), (300, 130), (513, 32)])
def test_pack_of_8_bit_weights(pkg, dtype, k, n):
    g = gen(n)
    for w in (normal(g, k, n, dtype=DTYPES[dtype]), normal(g, k, n + 3, dtype=DTYPES[dtype])[:, 2:2 + n], normal(g, 1, n, dtype=DTYPES[dtype]).expand(k, n)):
        linear = pkg.W8Linear.pack(w)
        codes, scales = plain_codes(w.T)
        assert torch.equal(linear.codes.cpu().float(), codes) and torch.equal(linear.scales.cpu(), scales)
        assert linear.in_features == k and linear.out_features == n
    w[0, n // 2:] = math.inf
    y = pkg.W8Linear.pack(w.clone())(torch.ones((2, k), device="cuda"))
    assert y[:, n // 2:].isnan().all() and y[:, :n // 2].isfinite().all()


# ---- verification of drafts -----------------------------------------------------------------

def plain_verify(logits, drafts, uniforms, starts, parents=None, probs=None, heat=None, wide=None):
    """The rules in fp64, one row after another."""
    logits, uniforms = logits.double().cpu(), uniforms.cpu()
    probs = None if probs is None else probs.double().cpu()
    tokens, nodes, counts = [], [], []
    for b in range(len(starts) - 1):
        a, n = starts[b], min(starts[b + 1] - starts[b], wide)
        t = 1.0 if heat is None else float(heat[b])
        if n == 0:
            tokens.append([-1] * wide), nodes.append([-1] * wide), counts.append(0)
            continue

        def target(i):
            x = logits[a + i]
            if x.isnan().any() or x.max() == math.inf or x.max() == -math.inf:
                return None
            if t > 0:
                e = torch.exp((x - x.max()) / t)
                return torch.where(x == -math.inf, 0.0, e / e.sum()) if math.isinf(t) is False else (x > -math.inf).double() / (x > -math.inf).sum()
            return torch.zeros_like(x).index_fill_(0, (x == x.max()).nonzero()[0], 1.0)

        at, said, path = 0, [], [0]
        while True:
            p = target(at)
            left, gone = (p, set())
            taken = None
            for i in range(at + 1, n):
                if (i - 1 if parents is None else parents[a + i]) != at or p is None:
                    continue
                x, u = int(drafts[a + i]), float(uniforms[a + i])
                here = float(left[x]) if 0 <= x < len(left) else 0.0
                if probs is not None:
                    q = float(probs[a + i, x]) if 0 <= x < len(p) else math.nan
                    if u * q < float(p[x] if 0 <= x < len(p) else 0):
                        taken = i
                        break
                    left = (p - probs[a + i]).clamp(min=0)
                    left = p if float(left.sum()) == 0 else left
                else:
                    if u * float(left.sum()) < here:
                        taken = i
                        break
                    if 0 <= x < len(left):
                        left = left.clone()
                        left[x] = 0
            if taken is None:
                break
            said.append(int(drafts[a + taken]))
            path.append(taken)
            at = taken
        if p is None:
            said.append(-1)
        else:
            left = p if float(left.sum()) == 0 else left
            run = torch.cumsum(left, 0)
            past = (run > float(uniforms[a]) * float(run[-1])).nonzero()
            said.append(int(past[0]) if len(past) else int(left.nonzero()[-1]))
        tokens.append(said + [-1] * (wide - len(said)))
        nodes.append(path + [-1] * (wide - len(path)))
        counts.append(len(said))
    return tokens, nodes, counts


def check_verify(pkg, logits, drafts, uniforms, starts, parents=None, probs=None, heat=None, wide=None, **more):
    wide = wide or max(1, max(b - a for a, b in zip(starts, starts[1:])))
    got = pkg.verify_drafts(logits, drafts, uniforms, starts=ints(starts), parents=None if parents is None else ints(parents),
                            draft_probs=probs, temperature=None if heat is None else torch.tensor(heat, device="cuda"),
                            max_nodes=wide, **more)
    want = plain_verify(logits, drafts.tolist(), uniforms, starts, parents, probs,
                        None if heat is None else torch.tensor(heat).tolist(), wide)
    for g, w in zip(got, want):
        assert g.dtype == torch.int32 and g.tolist() == w
    return got


def verify_case(g, rng, nodes, vocab, dtype, tree, peak=8.0):
    rows = sum(nodes)
    logits = normal(g, rows, vocab)
    logits += peak * (torch.rand((rows, vocab), device="cuda", generator=g) < 4 / vocab)
    starts, parents = [0], []
    for n in nodes:
        parents += [rng.randrange(i) if i and tree else i - 1 for i in range(n)]
        starts.append(starts[-1] + n)
    first = [s for s, n in zip(starts, nodes) for _ in range(n)]
    above = [max(f + p, 0) for f, p in zip(first, parents)]
    logits = logits.to(dtype)
    best = logits.float().topk(min(vocab, 3), 1).indices
    drafts = ints([int(best[a, rng.randrange(best.shape[1])]) for a in above])
    uniforms = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
    return logits, drafts, uniforms, starts, parents, above


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [1, 2, 17, 1000, 4099, 16384, 50257])
def test_verification_of_trees(pkg, dtype, vocab):
    g, rng = gen(vocab), random.Random(vocab)
    for turn in range(4):
        nodes = [1, 2, 9, rng.randint(1, 40), 0, 5]
        logits, drafts, uniforms, starts, parents, _ = verify_case(g, rng, nodes, vocab, DTYPES[dtype], True)
        check_verify(pkg, logits, drafts, uniforms, starts, parents, heat=[0.7, 1.0, 0.0, 1.3, 1.0, 0.8])
        check_verify(pkg, logits, drafts, uniforms, starts)  # as chains


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [1, 2, 17, 1000, 4099, 16384, 50257])
def test_verification_of_drawn_chains(pkg, dtype, vocab):
    g, rng = gen(vocab), random.Random(vocab)
    for turn in range(4):
        nodes = [3, 1, 6, 2, 12]
        logits, _, uniforms, starts, _, above = verify_case(g, rng, nodes, vocab, DTYPES[dtype], False)
        probs = torch.softmax(logits.float()[above] + normal(g, len(above), vocab), 1)
        drafts = torch.multinomial(probs, 1, generator=g).squeeze(1).to(torch.int32)
        check_verify(pkg, logits, drafts, uniforms, starts, probs=probs, heat=[1.0, 0.9, 0.0, 1.2, 0.8])
        wide = torch.zeros((len(above), vocab + 5), device="cuda")  # rows that begin anywhere
        wide[:, 3:3 + vocab] = probs
        logits2 = torch.zeros((len(above), vocab + 3), device="cuda", dtype=DTYPES[dtype])
        logits2[:, 1:1 + vocab] = logits
        check_verify(pkg, logits2[:, 1:1 + vocab], drafts, uniforms, starts, probs=wide[:, 3:3 + vocab])


@gpu
def test_verification_of_one_row_each(pkg):
    g = gen(4)
    logits = normal(g, 300, 5000, dtype=torch.bfloat16)
    uniforms = torch.rand(300, device="cuda", generator=g, dtype=torch.float64)
    drafts = torch.zeros(300, dtype=torch.int32, device="cuda")
    tokens, nodes, counts = pkg.verify_drafts(logits, drafts, uniforms)
    want = plain_verify(logits, drafts.tolist(), uniforms, list(range(301)), wide=1)
    assert tokens.tolist() == want[0] and nodes.eq(0).all() and counts.eq(1).all()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_verification_next_to_borders(pkg, dtype):
    """Draws just inside both ends of tokens' intervals, the narrowest of them 2^-30 of the widest.
    Uniforms and running sums up to total < 2.1 are fp64: 8 of each are off by less than 2^-49 total together, so
    that a draw as far inside is the token's (2^-30 * 1e-9 inside would round to the end itself)."""
    vocab = 64
    powers = [0, 3, 1, 2, 5, 4, 8, 30]
    x = torch.full((1, vocab), -math.inf)
    for i, k in enumerate(powers):
        x[0, 5 * i + 1] = -k * math.log(2.0)
    heat = 1.0
    weights = [math.exp(float(x[0, 5 * i + 1].to(DTYPES[dtype]).double())) for i in range(len(powers))]
    total = math.fsum(weights)
    draws, want, run = [], [], 0.0
    for i, w in enumerate(weights):
        inside = max(w * 1e-9, 2.0 ** -49 * total)
        for u in ((run + inside) / total, (run + w - inside) / total):
            draws.append(u), want.append(5 * i + 1)
        run += w
    rows = len(draws)
    logits = x.to(DTYPES[dtype]).cuda().expand(rows, vocab).contiguous()
    uniforms = torch.tensor(draws, dtype=torch.float64, device="cuda")
    tokens, _, _ = pkg.verify_drafts(logits, torch.zeros(rows, dtype=torch.int32, device="cuda"), uniforms,
                                     temperature=torch.full((rows,), heat, device="cuda"))
    assert tokens[:, 0].tolist() == want
    # the ends of the uniforms, and what is none
    ends = torch.tensor([0.0, 1 - 2.0 ** -53, 1.0, -1.0, math.nan], dtype=torch.float64, device="cuda")
    tokens, _, _ = pkg.verify_drafts(logits[:5], torch.zeros(5, dtype=torch.int32, device="cuda"), ends)
    assert tokens[:, 0].tolist() == [1, 36, 36, 1, 36]


@gpu
def test_verification_of_rows_without_probabilities(pkg):
    g = gen(6)
    logits = normal(g, 12, 3000)
    logits[1] = -math.inf
    logits[3, 7] = math.nan
    logits[5, 2999] = math.inf
    logits[7] = -math.inf
    logits[7, 11] = -5.0       # one that is left
    logits[9, ::2] = -math.inf
    drafts = logits.nan_to_num(0).argmax(1).to(torch.int32)
    drafts[0] = -1
    drafts = drafts.roll(1)
    uniforms = torch.rand(12, device="cuda", generator=g, dtype=torch.float64)
    for heat in ([1.0] * 6, [0.0] * 6, [-1.0] * 6, [math.inf] * 6, [1e-30] * 6, [1e-38] * 6, [3e38] * 6):
        check_verify(pkg, logits, drafts, uniforms, list(range(0, 13, 2)), heat=heat)
        check_verify(pkg, logits, drafts, uniforms * 0, [0, 4, 8, 12], heat=heat[:3])


@gpu
def test_verification_of_same_and_unknown_drafts(pkg):
    """Siblings with the same token, tokens outside the vocabulary, parents that are none."""
    g = gen(8)
    vocab = 40
    logits = normal(g, 14, vocab)
    top = int(logits[0].argmax())
    drafts = ints([0, top, top, 999, -5, vocab, top, 3, 3, 4, 5, 6, 7, 2 ** 31 - 1])
    parents = [0] * 14
    for u in (0.0, 0.3, 0.6, 0.999999):
        uniforms = torch.full((14,), u, device="cuda", dtype=torch.float64)
        check_verify(pkg, logits, drafts, uniforms, [0, 14], parents, heat=[1.0])
    odd = [5, 7, -1, 2 ** 31 - 1, 4, 0, 99, 0, 0, 9, 1, 0, 2, 0]
    uniforms = torch.rand(14, device="cuda", generator=g, dtype=torch.float64)
    seen = [p if 0 <= p < i else -1 for i, p in enumerate(odd)]
    want = plain_verify(logits, drafts.tolist(), uniforms, [0, 14], seen, wide=14)
    got = pkg.verify_drafts(logits, drafts, uniforms, starts=ints([0, 14]), parents=ints(odd))
    assert [t.tolist() for t in got] == list(want)
    # every token of the vocabulary rejected, one after another
    logits = torch.zeros((vocab + 1, vocab), device="cuda")
    drafts = ints([0] + list(range(vocab)))
    uniforms = torch.full((vocab + 1,), 2.0, device="cuda", dtype=torch.float64)
    got = pkg.verify_drafts(logits, drafts, uniforms, starts=ints([0, vocab + 1]), parents=ints([0] * (vocab + 1)))
    assert got[2].tolist() == [1] and got[0][0, 0] == vocab - 1


@gpu
def test_verification_cuts_nodes(pkg):
    g, rng = gen(5), random.Random(5)
    logits, drafts, uniforms, starts, parents, _ = verify_case(g, rng, [20, 3, 1024], 300, torch.float32, True, peak=2.0)
    check_verify(pkg, logits, drafts, uniforms, starts, parents, wide=6)
    check_verify(pkg, logits, drafts, uniforms, starts, parents)


@gpu
def test_verification_of_malformed_starts(pkg):
    """Starts that descend or lie outside: nothing outside the tensors is touched; sequences in order come out right."""
    g, rng = gen(5), random.Random(5)
    logits, drafts, uniforms, _, _, _ = verify_case(g, rng, [4, 4], 500, torch.float32, False)
    for starts in ([0, 4, 4, 8], [-7, 4, 100, 300], [8, 0, 8], [5, 3, 8], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
        tokens, nodes, counts = pkg.verify_drafts(logits, drafts, uniforms, starts=ints(starts), max_nodes=8)
        assert counts.ge(0).all() and counts.le(8).all()
    want = plain_verify(logits, drafts.tolist(), uniforms, [0, 4, 8, 8], wide=8)
    tokens, nodes, counts = pkg.verify_drafts(logits, drafts, uniforms, starts=ints([-7, 4, 100, 300]), max_nodes=8)
    assert tokens.tolist() == want[0] and counts.tolist() == want[2]


@gpu
@pytest.mark.parametrize("drawn", [False, True])
def test_accepted_tokens_are_distributed_as_the_target(pkg, drawn):
    """The first token of many sequences against p: 40000 of them, so that a count's deviation is
    sqrt(n p (1 - p)) and 6 of them hold for all 12 tokens but once in some 10^8 runs."""
    g = gen(11)
    n, vocab = 40000, 12
    one, other = normal(g, vocab), normal(g, vocab)
    p, q = torch.softmax(one.double(), 0), torch.softmax(other, 0)
    logits = one.expand(2 * n, vocab).contiguous()
    starts = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
    uniforms = torch.rand(2 * n, device="cuda", generator=g, dtype=torch.float64)
    drafts = torch.multinomial(q, 2 * n, replacement=True, generator=g).to(torch.int32)
    probs = q.expand(2 * n, vocab).contiguous() if drawn else None
    if not drawn:
        drafts = torch.full_like(drafts, 3)
    tokens, _, _ = pkg.verify_drafts(logits, drafts, uniforms, starts=starts, draft_probs=probs, max_nodes=2)
    counts = torch.bincount(tokens[:, 0].long(), minlength=vocab).double()
    assert ((counts - n * p).abs() <= 6 * torch.sqrt(n * p * (1 - p))).all()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("heat", [0.0, 0.8])
def test_verification_under_masks_of_the_lowest_value(pkg, dtype, heat):
    """Masked by the type's lowest value, in part and in whole (then all are alike)."""
    g, rng = gen(3), random.Random(3)
    logits, drafts, uniforms, starts, parents, _ = verify_case(g, rng, [5, 9, 2], 3001, DTYPES[dtype], True)
    low = torch.finfo(DTYPES[dtype]).min
    logits[torch.rand(logits.shape, device="cuda", generator=g) < 0.6] = low
    check_verify(pkg, logits, drafts, uniforms, starts, parents, heat=[heat] * 3)
    logits[starts[1]:] = low
    logits[starts[2], :7] = -math.inf
    check_verify(pkg, logits, drafts, uniforms, starts, parents, heat=[heat] * 3)


@gpu
def test_verification_decides_close_tests_in_64_bits(pkg):
    """Uniforms a part in 10^12 to either side of a draft's probability: sums from 32-bit
    exponentials cannot tell them apart."""
    g = gen(21)
    vocab, n = 5000, 12
    logits = normal(g, 2 * n, vocab)
    drafts = torch.randint(0, vocab, (2 * n,), device="cuda", generator=g).to(torch.int32)
    uniforms = torch.rand(2 * n, device="cuda", generator=g, dtype=torch.float64)
    starts, heat = list(range(0, 2 * n + 1, 2)), [0.5 + 0.1 * i for i in range(n)]
    p = torch.stack([torch.softmax(logits[2 * i].double() / float(torch.tensor(heat[i])), 0) for i in range(n)])
    at = p[torch.arange(n), drafts[1::2].long()]
    probs = torch.softmax(normal(g, 2 * n, vocab), 1)
    q = probs[torch.arange(1, 2 * n, 2), drafts[1::2].long()].double()
    for side, count in ((1 - 1e-12, 2), (1 + 1e-12, 1)):
        uniforms[1::2] = at * side
        _, _, counts = check_verify(pkg, logits, drafts, uniforms, starts, heat=heat)
        assert counts.eq(count).all()
        uniforms[1::2] = at / q * side  # (past 1 for some: as good a number to compare)
        _, _, counts = check_verify(pkg, logits, drafts, uniforms, starts, heat=heat, probs=probs)
        assert counts.eq(count).all()
    # siblings: the second is held against what the first has left, and a chain goes on behind a close test
    wide = logits[:1].expand(4, vocab).contiguous()
    p = torch.softmax(wide[0].double(), 0)
    a, b = int(p.argmax()), int(p.argmin())
    for side, want in ((1 - 1e-12, 2), (1 + 1e-12, 1)):
        u = torch.tensor([0.5, float(p[a]) * (1 + 1e-12), float(p[b] / (1 - p[a])) * side, 0.0], dtype=torch.float64, device="cuda")
        _, _, counts = check_verify(pkg, wide, ints([0, a, b, 7]), u, [0, 4], parents=[0, 0, 0, 1])
        assert counts.tolist() == [want]


@gpu
def test_verification_of_many_rows_and_far_ones(pkg):
    """More rows than 16 bits count, and logits and probabilities past 2^32 bytes."""
    g = gen(2)
    n, vocab = 70000, 64
    logits = normal(g, n, vocab, dtype=torch.bfloat16)
    uniforms = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    starts = torch.arange(0, n + 1, 2, dtype=torch.int32, device="cuda")
    drafts = torch.randint(0, vocab, (n,), device="cuda", generator=g).to(torch.int32)
    tokens, nodes, counts = pkg.verify_drafts(logits, drafts, uniforms, starts=starts, max_nodes=2)
    want = plain_verify(logits[-200:], drafts[-200:].tolist(), uniforms[-200:], list(range(0, 201, 2)), wide=2)
    assert tokens[-100:].tolist() == want[0] and counts[-100:].tolist() == want[2]
    rows, vocab = 3, 1 << 20
    flat = torch.zeros(rows * 1200000000 // 2, dtype=torch.bfloat16, device="cuda")  # 3.6 GB
    far = flat.as_strided((rows, vocab), (600000000, 1))
    far.copy_(normal(g, rows, vocab))
    q = torch.zeros(2 * 1200000000 // 2 + vocab, device="cuda").as_strided((rows, vocab), (600000000, 1))  # 4.8 GB
    q.copy_(torch.softmax(normal(g, rows, vocab), 1))
    drafts = torch.multinomial(q, 1, generator=g).squeeze(1).to(torch.int32)
    uniforms = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
    check_verify(pkg, far, drafts, uniforms, [0, 3], probs=q)


@gpu
@pytest.mark.parametrize("rows,k", [(1, 32768), (1, 20000), (2, 16384), (2, 9000), (3, 8192), (4, 8192), (4, 8191), (3, 10000), (1, 32769)])
def test_products_at_the_ends_of_few_rows(pkg, rows, k):
    """The sizes at which lanes hold their last piece of inputs, and those past them."""
    g = gen(k)
    for n in (5, 1203):
        linear = w8_case(pkg, g, k, n)
        x = normal(g, rows, k, dtype=torch.bfloat16)
        codes, scales = plain_codes(x)
        check_w8(linear, codes, scales, linear(x))
        check_w8(linear, codes, scales, linear(codes.to(torch.int8).cuda(), scales=scales.cuda()))


@gpu
def test_products_read_nothing_behind_the_last_row(pkg):
    """Buffers that end with the last row's last code: what is behind is another tensor's NaN, and stays."""
    g = gen(5)
    for k, n, rows in ((77, 9, 2), (100, 40, 6), (1000, 130, 40), (300, 257, 200)):
        row = -(-k // 16) * 16
        flat = torch.randint(-127, 128, ((n - 1) * row + k,), device="cuda", generator=g).to(torch.int8)
        linear = pkg.W8Linear(flat.as_strided((n, k), (row, 1)), torch.rand(n, device="cuda", generator=g) + 0.1)
        x = torch.randint(-127, 128, ((rows - 1) * row + k,), device="cuda", generator=g).to(torch.int8).as_strided((rows, k), (row, 1))
        scales = torch.rand(rows, device="cuda", generator=g)
        check_w8(linear, x, scales, linear(x, scales=scales))


@gpu
def test_product_past_32_bit_offsets(pkg):
    g = gen(6)
    k, n = 48, 100_000_000  # 4.8 GB of codes
    codes = torch.zeros((n, k), dtype=torch.int8, device="cuda")
    codes[-1000:] = torch.randint(-127, 128, (1000, k), device="cuda", generator=g).to(torch.int8)
    scales = torch.ones(n, device="cuda")
    linear = pkg.W8Linear(codes, scales)
    for rows in (1, 5, 130):
        x = torch.randint(-127, 128, (rows, k), device="cuda", generator=g).to(torch.int8)
        y = linear(x, scales=torch.ones(rows, device="cuda"), dtype=torch.bfloat16)
        want = x.double() @ codes[-1000:].double().T
        assert torch.equal(y[:, -1000:], want.to(torch.bfloat16)) and y[:, :-1000:4099].eq(0).all()


@gpu
def test_norm_of_rows_past_32_bit_offsets(pkg):
    g = gen(7)
    rows, dim = 600_000, 4096  # 4.9 GB of h
    h = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")
    h[-50:] = normal(g, 50, dim)
    x = torch.zeros(1, dim, device="cuda").expand(rows, dim)  # one row for all
    w = 1 + 0.1 * normal(g, dim)
    s, codes, scales = pkg.residual_norm(h, x, w, quantise=True, kind="rms")
    few = pkg.residual_norm(h[-50:], x[-50:], w, quantise=True, kind="rms")
    assert torch.equal(s[-50:], few[0]) and torch.equal(scales[:-50], torch.zeros_like(scales[:-50]))
    # (other threads hold a row's parts where rows are few: sums differ in their last bits)
    assert (codes[-50:].int() - few[1].int()).abs().max() <= 1 and torch.allclose(scales[-50:], few[2], rtol=1e-5, atol=0)


# ---- calls as a program makes them -----------------------------------------------------------

@gpu
def test_operators_on_another_stream(pkg):
    g = gen(12)
    x, w = normal(g, 40, 512, dtype=torch.bfloat16), normal(g, 512, 300)
    linear, weight = pkg.W8Linear.pack(w), torch.ones(512, device="cuda")
    logits, uniforms = normal(g, 6, 9000), torch.rand(6, device="cuda", generator=g, dtype=torch.float64)
    drafts, starts = ints([1, 2, 3, 4, 5, 6]), ints([0, 3, 6])

    def calls(x, logits):
        s, codes, scales = pkg.residual_norm(x, x, weight, quantise=True)
        return s, linear(codes, scales=scales), linear(x[:2]), *pkg.verify_drafts(logits, drafts, uniforms, starts=starts)

    want = calls(x, logits)
    side = torch.cuda.Stream()
    busy = torch.zeros(1 << 28, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):
            busy.add_(1.0)
        a, b = x * busy[0] / 4, logits * busy[0] / 4  # made behind the stream's long work
        got = calls(a, b)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


class Step:
    """One layer of a decoder that drafts and verifies, on the operators."""

    def __init__(self, pkg, g, seqs, dim, heads, vocab, drafts, page):
        self.pkg, self.heads, self.dim, self.vocab, self.most = pkg, heads, dim, vocab, seqs * (drafts + 1)
        self.pages = pkg.PageTable.empty(seqs, 6, seqs * 5, page)
        self.cache = pkg.QuantKvCache.empty(seqs * 5, page, heads, dim // heads, "int8")
        self.emb = normal(g, vocab, dim, dtype=torch.bfloat16)
        self.qkv, self.out, self.head = (pkg.W8Linear.pack(normal(g, dim, n) / dim ** 0.5) for n in (3 * dim, dim, vocab))
        self.w, self.b = 1 + 0.1 * normal(g, dim), 0.1 * normal(g, dim)

    def run(self, tokens, counts, uniforms):
        """tokens [most] of the served rows in order; returns everything that the step makes."""
        pkg, n = self.pkg, self.most
        starts, prefix, slots, positions = self.pages.extend(counts, n)
        x = self.emb[tokens.long()] + 0.01 * positions[:, None]
        _, codes, scales = pkg.residual_norm(None, x, self.w, self.b, quantise=True)
        qkv = self.qkv(codes, scales=scales, dtype=torch.bfloat16).view(n, 3, self.heads, -1)
        self.cache.write(qkv[:, 1], qkv[:, 2], slots)
        a, _ = self.cache.attend(qkv[:, 0], self.pages.table, prefix, starts=starts, max_nodes=8)
        x, h = pkg.residual_norm(self.out(a.reshape(n, -1)), x, self.w, self.b)
        logits = pkg.logit_controls(self.head(h))
        kept, nodes, gained = pkg.verify_drafts(logits, tokens, uniforms, starts=starts, max_nodes=8)
        self.pages.truncate(prefix + gained)
        return starts, prefix, slots, positions, logits, kept, nodes, gained, self.pages.lens.clone(), self.pages.table.clone()


@gpu
def test_a_step_of_all_operators(pkg):
    """A sequence of steps: pages and verification as their rules say of what the step made, and the
    logits as a plain computation of the same layer over everything kept so far."""
    g = gen(31)
    seqs, dim, heads, vocab, page = 5, 128, 4, 500, 8
    step = Step(pkg, g, seqs, dim, heads, vocab, 5, page)
    want = Pages(seqs, 6, seqs * 5, page)
    text = [[] for _ in range(seqs)]  # tokens in the cache
    rng = random.Random(4)
    last = [rng.randrange(vocab) for _ in range(seqs)]
    scale = [l.scales.double() for l in (step.qkv, step.out, step.head)]
    dense = [(l.codes.double() * s[:, None]).T for l, s in zip((step.qkv, step.out, step.head), scale)]
    for turn in range(5):
        news = [[last[b]] + [rng.randrange(vocab) for _ in range(rng.randint(0, 5))] for b in range(seqs)]
        counts = [len(t) for t in news]
        tokens = [t for n in news for t in n]
        uniforms = torch.rand(step.most, device="cuda", generator=g, dtype=torch.float64)
        made = step.run(ints(tokens + [0] * (step.most - len(tokens))), ints(counts), uniforms)
        starts, prefix, slots, positions, logits, kept, nodes, gained = made[:8]
        assert [t.tolist() for t in made[:4]] == list(want.extend(counts, step.most))
        plain = plain_verify(logits, tokens, uniforms, starts.tolist(), wide=8)
        assert (kept.tolist(), nodes.tolist(), gained.tolist()) == plain
        want.truncate([n + c for n, c in zip(prefix.tolist(), plain[2])])
        assert want.same(step.pages)
        for b in range(seqs):
            ids = torch.tensor(text[b] + news[b], device="cuda")
            x = step.emb[ids].double() + 0.01 * torch.arange(len(ids), device="cuda")[:, None]
            qkv = (plain_norm(x, step.w, step.b, "layer", 1e-5) @ dense[0]).view(-1, 3, heads, dim // heads)
            s = torch.einsum("qhd,khd->hqk", qkv[:, 0], qkv[:, 1]) / math.sqrt(dim // heads)
            s = s.masked_fill(~torch.ones(len(ids), len(ids), device="cuda").tril().bool(), -math.inf)
            a = torch.einsum("hqk,khd->qhd", torch.softmax(s, 2), qkv[:, 2]).flatten(1)
            ref = plain_norm(x + a @ dense[1], step.w, step.b, "layer", 1e-5) @ dense[2]
            got = logits[int(starts[b]):int(starts[b + 1])].double()
            ref = ref[-len(news[b]):]
            # three products of 8-bit rows (a row's half step is 1/254 of its largest, some 3 deviations: 1 % of a
            # deviation, over sums of independent terms), an 8-bit cache as much, bf16 in between: 4 % at most
            assert ((got - ref).square().mean() / ref.square().mean()).sqrt() < 0.04
            text[b] += [news[b][i] for i in plain[1][b] if i >= 0]
            last[b] = plain[0][b][plain[2][b] - 1]


@gpu
def test_a_step_in_a_graph(pkg):
    """Captured once, replayed with other inputs in the same places: as without the graph."""
    def steps(g):
        return Step(pkg, g, 5, 128, 4, 500, 5, 8)
    plain, own = steps(gen(8)), steps(gen(8))
    g = gen(9)
    tokens, counts = torch.zeros(own.most, dtype=torch.int32, device="cuda"), ints([0] * 5)
    uniforms = torch.zeros(own.most, dtype=torch.float64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own.run(tokens, counts, uniforms)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = own.run(tokens, counts, uniforms)
    torch.cuda.synchronize()
    for turn in range(6):
        tokens.copy_(torch.randint(0, 500, (own.most,), device="cuda", generator=g))
        counts.copy_(torch.randint(0, 7, (5,), device="cuda", generator=g))
        uniforms.copy_(torch.rand(own.most, device="cuda", generator=g, dtype=torch.float64))
        graph.replay()
        want = plain.run(tokens, counts, uniforms)
        n = int(want[0][-1])
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a[:n] if i == 4 else a, b[:n] if i == 4 else b), i  # (logits of rows that are there)


@gpu
def test_two_calls_give_the_same_bits(pkg):
    g = gen(17)
    x = normal(g, 300, 1500, dtype=torch.bfloat16)
    linear = pkg.W8Linear.pack(normal(g, 1500, 700))
    logits, uniforms = normal(g, 30, 30000), torch.rand(30, device="cuda", generator=g, dtype=torch.float64)
    probs = torch.softmax(normal(g, 30, 30000), 1)
    drafts, starts = torch.multinomial(probs, 1, generator=g).squeeze(1).to(torch.int32), ints(list(range(0, 31, 6)))
    calls = [lambda: pkg.residual_norm(x, x, torch.ones(1500, device="cuda")), lambda: (linear(x), linear(x[:3]), linear(x[:50])),
             lambda: pkg.verify_drafts(logits, drafts, uniforms, starts=starts, draft_probs=probs)]
    for call in calls:
        first = call()
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(first, call()))


@gpu
def test_step_operators_cut_no_gradient_in_silence(pkg):
    x = torch.randn((3, 64), device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    linear = pkg.W8Linear.pack(torch.randn(64, 20, device="cuda"))
    plain = x.detach()
    results = [pkg.residual_norm(x, plain, w.detach())[0], pkg.residual_norm(plain, x, w.detach())[1],
               pkg.residual_norm(plain, plain, w)[1], pkg.residual_norm(plain, plain, w, quantise=True)[2], linear(x),
               pkg.quantise_rows(x)[1], linear(x, dtype=torch.bfloat16)]
    for r in results:
        assert r.requires_grad
        with pytest.raises(RuntimeError, match="computes no gradient"):
            r.sum().backward()
    assert not pkg.residual_norm(plain, plain, w)[0].requires_grad  # the stream does not depend on the norm's weight
    with torch.no_grad():
        assert not linear(x).requires_grad


@gpu
def test_step_operators_count_what_they_change(pkg):
    pages = pkg.PageTable.empty(2, 3, 6, 8)
    before = [t._version for t in (pages.table, pages.lens, pages.free, pages.n_free)]
    pages.extend(ints([3, 4]), 10)
    after = [t._version for t in (pages.table, pages.lens, pages.free, pages.n_free)]
    assert [b - a for a, b in zip(before, after)] == [1, 1, 0, 1]
    pages.truncate(ints([0, 0]))
    assert [t._version - a for t, a in zip((pages.table, pages.lens, pages.free, pages.n_free), after)] == [1, 1, 1, 1]


@gpu
def test_step_operators_refuse_replaced_buffers(pkg):
    pages = pkg.PageTable.empty(2, 3, 6, 8)
    pages.lens.resize_(3)
    with pytest.raises(pkg.ArgumentError):
        pages.extend(ints([1, 1]), 4)
    linear = pkg.W8Linear.pack(torch.ones(32, 16, device="cuda"))
    x = torch.ones((2, 32), device="cuda")
    before = linear(x)
    linear.codes.data = torch.zeros((16, 48), dtype=torch.int8, device="cuda")
    with pytest.raises(pkg.ArgumentError):
        linear(x)
    linear.codes.data = torch.zeros((16, 32), dtype=torch.int8, device="cuda")
    assert linear(x).eq(0).all() and before.gt(0).all()


@gpu
@pytest.mark.parametrize("rows,k,n,lost_rows,lost_outputs", [(40, 1024, 1024, 40, 128), (300, 1024, 1024, 128, 128), (300, 512, 9000, 256, 256)])
def test_a_wait_of_the_products_that_runs_out(pkg, rows, k, n, lost_rows, lost_outputs):
    """A copy that never comes: that block's rows are NaN, the call returns, the next one is right."""
    from forge_lm_b200 import _native as N
    g = gen(1)
    linear = w8_case(pkg, g, k, n)
    x = torch.randint(-127, 128, (rows, k), device="cuda", generator=g).to(torch.int8)
    scales = torch.ones(rows, device="cuda")
    want = linear(x, scales=scales)
    N.check(N.load().fb2_test_w8_withhold(1, 200_000_000))
    y = linear(x, scales=scales)
    torch.cuda.synchronize()
    lost = y.isnan()
    assert lost[:lost_rows, :lost_outputs].all() and int(lost.sum()) == lost_rows * lost_outputs
    assert torch.equal(y[~lost], want[~lost])
    assert torch.equal(linear(x, scales=scales), want)


@gpu
def test_step_refusals_on_the_device(pkg):
    E = pkg.ArgumentError
    f, h = torch.ones((3, 64), device="cuda"), torch.ones((3, 64), device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda")
    pages = pkg.PageTable.empty(2, 3, 6, 8)
    linear = pkg.W8Linear.pack(torch.ones(64, 32, device="cuda"))
    codes, scales = pkg.quantise_rows(f)
    u = torch.zeros(3, device="cuda", dtype=torch.float64)
    d = ints([0, 0, 0])
    neg = torch.complex(f, f).conj().imag
    for call in (
            lambda: pages.extend(ints([1, 1, 1]), 4), lambda: pages.extend(ints([1, 1]).long(), 4), lambda: pages.extend(ints([1, 1]), -1),
            lambda: pages.extend(ints([1, 1]).cpu(), 4), lambda: pages.extend(ints([1, 1]), 2 ** 31), lambda: pages.extend(None, 4),
            lambda: pages.truncate(ints([1])), lambda: pages.truncate([1, 1]),
            lambda: pkg.PageTable(pages.table, pages.lens, pages.free, pages.n_free, 12),
            lambda: pkg.PageTable(pages.table.t(), pages.lens, pages.free, pages.n_free, 8),
            lambda: pkg.PageTable(pages.table, pages.lens[:1], pages.free, pages.n_free, 8),
            lambda: pkg.PageTable(pages.table, pages.lens, pages.free, pages.lens, 8),
            lambda: pkg.PageTable(pages.table, pages.lens, None, pages.n_free, 8),
            lambda: pkg.PageTable.empty(20000, 1, 1, 8),
            lambda: pkg.residual_norm(f, h, w), lambda: pkg.residual_norm(f, f[:2], w), lambda: pkg.residual_norm(f, f, w[:5]),
            lambda: pkg.residual_norm(f, f, w.half()), lambda: pkg.residual_norm(f, f, None), lambda: pkg.residual_norm(f, f.t(), w),
            lambda: pkg.residual_norm(f.double(), f, w), lambda: pkg.residual_norm(f, f, w, kind="other"),
            lambda: pkg.residual_norm(f, f, w, scale=math.inf), lambda: pkg.residual_norm(f, f, w, eps=-1.0),
            lambda: pkg.residual_norm(None, f, w, gate=f), lambda: pkg.residual_norm(None, f, w, post_weight=w),
            lambda: pkg.residual_norm(f, f, w, gate=h), lambda: pkg.residual_norm(f, f, w, gate=w[:3]),
            lambda: pkg.residual_norm(f, f, w, post_bias=w), lambda: pkg.residual_norm(f, f.cpu(), w),
            lambda: pkg.residual_norm(f, neg, w), lambda: pkg.residual_norm(f, f, w, dtype=torch.bfloat16),
            lambda: pkg.residual_norm(torch.ones((1, 40000), device="cuda"), torch.ones((1, 40000), device="cuda"), torch.ones(40000, device="cuda")),
            lambda: pkg.quantise_rows(f.t()), lambda: pkg.quantise_rows(f.double()), lambda: pkg.quantise_rows(f[0]), lambda: pkg.quantise_rows(f.cpu()),
            lambda: linear(f[:, :63]), lambda: linear(f.cpu()), lambda: linear(f.double()), lambda: linear(codes), lambda: linear(f, scales=scales),
            lambda: linear(codes, scales=scales[:2]), lambda: linear(codes, scales=scales.half()), lambda: linear(torch.ones((64, 3), device="cuda").t()),
            lambda: linear(f, dtype=torch.float64), lambda: linear(neg),
            lambda: pkg.W8Linear(codes.float(), scales), lambda: pkg.W8Linear(codes, scales[:2]), lambda: pkg.W8Linear(codes, scales, bias=scales[:1]),
            lambda: pkg.W8Linear(codes[:, 1:], scales), lambda: pkg.W8Linear(codes[:1].expand(3, 64), scales),
            lambda: pkg.W8Linear(torch.zeros((2, 131073 + 15), dtype=torch.int8, device="cuda")[:, :131073], scales[:2]),
            lambda: pkg.W8Linear.pack(f.double()), lambda: pkg.W8Linear.pack(f.t()), lambda: pkg.W8Linear.pack(f[0]),
            lambda: pkg.verify_drafts(f, d, u.float()), lambda: pkg.verify_drafts(f, d.long(), u), lambda: pkg.verify_drafts(f, d[:2], u),
            lambda: pkg.verify_drafts(f.t(), d, u), lambda: pkg.verify_drafts(f.double(), d, u), lambda: pkg.verify_drafts(f, d, u[:2]),
            lambda: pkg.verify_drafts(f, d, u, parents=d, draft_probs=f), lambda: pkg.verify_drafts(f, d, u, draft_probs=h),
            lambda: pkg.verify_drafts(f, d, u, draft_probs=f[:2]), lambda: pkg.verify_drafts(f, d, u, max_nodes=0),
            lambda: pkg.verify_drafts(f, d, u, max_nodes=1025), lambda: pkg.verify_drafts(f, d, u, temperature=w[:2]),
            lambda: pkg.verify_drafts(f, d, u, starts=ints([])), lambda: pkg.verify_drafts(f, d, u, starts=ints([0, 3]), temperature=w[:2]),
            lambda: pkg.verify_drafts(f[:, :0], d, u), lambda: pkg.verify_drafts(f.cpu(), d, u)):
        with pytest.raises(E):
            call()
    many = torch.zeros((1025, 4), device="cuda")
    with pytest.raises(E):  # a bound of a sequence's rows is needed
        pkg.verify_drafts(many, ints([0] * 1025), torch.zeros(1025, device="cuda", dtype=torch.float64), starts=ints([0, 1025]))


def test_step_refusals_of_the_c_entries(pkg):
    """What the C entry points refuse before any device work."""
    import ctypes as C
    import struct
    from forge_lm_b200 import _native as N
    L = N.load()
    bad, ok, p = N.FB2_INVALID_ARG, N.FB2_OK, 4096
    pages = struct.Struct("=4Qq4i")
    base = [p, p, p, p, 10, 4, 10, 100, 16]
    assert L.fb2_pages_check(pages.pack(*base)) == ok
    for where, value in ((0, 0), (1, 0), (2, 0), (3, 0), (0, 4098), (1, 4097), (2, 4098), (3, 4097), (4, 9), (5, -1), (5, 16385), (6, -1),
                         (7, -1), (8, 12), (8, 4), (8, 2048), (7, 2 ** 31 - 1)):
        wrong = list(base)
        wrong[where] = value
        s = pages.pack(*wrong)
        assert L.fb2_pages_check(s) == bad, (where, value)
        assert L.fb2_pages_extend(s, p, 10, p, p, p, p, None) == bad and L.fb2_pages_truncate(s, p, None) == bad
    assert L.fb2_pages_check(None) == bad
    good = pages.pack(*base)
    for args in ((0, 10, p, p, p, p), (p, 10, 0, p, p, p), (p, 10, p, 0, p, p), (p, 10, p, p, 0, p), (p, 10, p, p, p, 0), (p, -1, p, p, p, p),
                 (p, 2 ** 31 - 1, p, p, p, p), (4098, 10, p, p, p, p), (p, 10, p, p, 4097, p)):
        assert L.fb2_pages_extend(good, *args, None) == bad, args
    assert L.fb2_pages_truncate(good, None, None) == bad and L.fb2_pages_truncate(good, 4098, None) == bad

    norm = struct.Struct("=11Q6q5i2fi")
    base = [p, p, 0, p, 0, 0, 0, p, p, 0, 0] + [64] * 5 + [64] + [2, 64, 1, 1, 0, 1.0, 1e-5, 0]
    for where, value in ((1, 0), (3, 0), (7, 0), (8, 0), (9, p), (10, p), (0, 4097), (1, 4097), (8, 4097), (3, 4098), (6, p), (14, 63), (15, 63),
                         (17, -1), (18, 0), (18, 32769), (19, 3), (20, 2), (21, 2), (22, math.nan), (23, -1.0), (23, math.inf)):
        wrong = list(base)
        wrong[where] = value
        assert L.fb2_residual_norm(norm.pack(*wrong), None) == bad, (where, value)
    coded = list(base)
    coded[8], coded[9], coded[10] = 0, p, p
    for where, value in ((9, 4100), (16, 60), (16, 72), (10, 4098)):
        wrong = list(coded)
        wrong[where] = value
        assert L.fb2_residual_norm(norm.pack(*wrong), None) == bad, (where, value)
    alone = list(base)
    alone[0], alone[2] = 0, p
    assert L.fb2_residual_norm(norm.pack(*alone), None) == bad and L.fb2_residual_norm(None, None) == bad
    base[17] = 0
    assert L.fb2_residual_norm(norm.pack(*base), None) == ok

    for args in ((-1, 8, p, 0, 8, p, 16, p), (1, 0, p, 0, 8, p, 16, p), (1, 8, 0, 0, 8, p, 16, p), (1, 8, p, 3, 8, p, 16, p), (1, 8, p, 0, 8, 4100, 16, p),
                 (2, 8, p, 0, 8, p, 8, p), (2, 32, p, 0, 32, p, 16, p), (1, 8, 4098, 0, 8, p, 16, p), (1, 8, p, 0, 8, p, 16, 4098)):
        assert L.fb2_quantise_rows(*args, None) == bad, args
    assert L.fb2_quantise_rows(0, 8, None, 0, 8, None, 16, None, None) == ok

    lin = struct.Struct("=QQQq2i")
    base = [p, p, 0, 112, 100, 33]
    n = C.c_int64()
    for where, value in ((0, 0), (1, 0), (0, 4104), (1, 4098), (2, 4098), (3, 96), (3, 104), (4, 0), (4, 131073), (5, 0), (5, 2 ** 31 - 1)):
        wrong = list(base)
        wrong[where] = value
        w = lin.pack(*wrong)
        assert L.fb2_w8_check(w) == bad, (where, value)
        assert L.fb2_w8_pack(w, p, 0, 33, None) == bad and L.fb2_w8_matmul(w, 1, p, 112, p, p, 33, 0, None) == bad
        assert L.fb2_w8_forward(w, 1, p, 100, p, 33, 0, p, 1 << 20, None) == bad and L.fb2_w8_forward_workspace(w, 1, C.byref(n)) == bad
    w = lin.pack(*base)
    assert L.fb2_w8_check(w) == ok and L.fb2_w8_check(None) == bad
    assert L.fb2_w8_pack(w, None, 0, 33, None) == bad and L.fb2_w8_pack(w, p, 0, 32, None) == bad and L.fb2_w8_pack(w, 4098, 0, 33, None) == bad
    for args in ((-1, p, 112, p, p, 33, 0), (1, 0, 112, p, p, 33, 0), (1, p, 112, 0, p, 33, 0), (1, p, 112, p, 0, 33, 0), (1, p, 112, p, p, 33, 5),
                 (1, 4104, 112, p, p, 33, 0), (2, p, 96, p, p, 33, 0), (2, p, 104, p, p, 33, 0), (2, p, 112, p, p, 32, 0), (1, p, 112, 4098, p, 33, 0),
                 (1, p, 112, p, 4097, 33, 1)):
        assert L.fb2_w8_matmul(w, *args, None) == bad, args
    assert L.fb2_w8_matmul(w, 0, None, 0, None, None, 0, 0, None) == ok
    assert L.fb2_w8_forward_workspace(w, 9, C.byref(n)) == ok and n.value == 9 * (112 + 4)
    assert L.fb2_w8_forward_workspace(w, -1, C.byref(n)) == bad and L.fb2_w8_forward_workspace(w, 9, None) == bad
    for args in ((9, p, 100, p, 33, 0, p, 9 * 116 - 1), (9, p, 100, p, 33, 0, 0, 0), (9, p, 100, p, 33, 0, 4100, 9 * 116), (9, 0, 100, p, 33, 0, p, 9 * 116),
                 (9, p, 100, p, 32, 0, p, 9 * 116), (9, 4098, 100, p, 33, 0, p, 9 * 116), (-1, p, 100, p, 33, 0, p, 9 * 116)):
        assert L.fb2_w8_forward(w, *args, None) == bad, args
    assert L.fb2_w8_forward(w, 0, None, 0, None, 0, 0, None, 0, None) == ok

    ver = struct.Struct("=11Q3q6i")
    base = [p, 0, p, p, 0, p, 0, p, p, p, p] + [6 * 16, 50, 50] + [2, 6, 50, 0, 4, 0]
    assert L.fb2_verify_workspace(ver.pack(*base), C.byref(n)) == ok and n.value == 6 * 16
    for where, value in ((0, 0), (2, 0), (5, 0), (7, 0), (8, 0), (9, 0), (10, 0), (0, 4098), (1, 4098), (2, 4097), (3, 4097), (4, 4097), (5, 4100), (6, 4097),
                         (7, 4097), (8, 4098), (9, 4098), (10, 4104), (11, 95), (14, -1), (15, -1), (16, 0), (16, 2 ** 31 - 1), (17, 4), (18, 0), (18, 1025)):
        wrong = list(base)
        wrong[where] = value
        assert L.fb2_verify_drafts(ver.pack(*wrong), None) == bad, (where, value)
    chain = list(base)
    chain[1] = chain[4] = p
    assert L.fb2_verify_drafts(ver.pack(*chain), None) == bad
    alone = list(base)
    alone[3] = 0
    assert L.fb2_verify_drafts(ver.pack(*alone), None) == bad  # 6 rows, 2 sequences
    base[14] = 0
    assert L.fb2_verify_drafts(ver.pack(*base), None) == ok
    assert L.fb2_verify_drafts(None, None) == bad and L.fb2_verify_workspace(ver.pack(*base), None) == bad
    assert L.fb2_test_w8_withhold(-1, 5) == bad and L.fb2_test_w8_withhold(0, 0) == bad and L.fb2_test_w8_withhold(0, 3_000_000_000) == bad
    assert L.fb2_last_error() != b""


@gpu
def test_calls_of_two_streams_at_once(pkg):
    """Nothing that one call writes is another's: the same calls on two streams, begun together again and again."""
    g = gen(14)
    linear = pkg.W8Linear.pack(normal(g, 700, 900))
    weight = torch.ones(700, device="cuda")
    logits, probs = normal(g, 40, 20000, dtype=torch.bfloat16), torch.softmax(normal(g, 40, 20000), 1)
    drafts = torch.multinomial(probs, 1, generator=g).squeeze(1).to(torch.int32)
    starts, uniforms = ints(list(range(0, 41, 5))), torch.rand(40, device="cuda", generator=g, dtype=torch.float64)
    xs = [normal(g, n, 700, dtype=torch.float16) for n in (2, 60, 700)]

    def calls():
        made = []
        for x in xs:
            s, codes, scales = pkg.residual_norm(x, x, weight, quantise=True)
            made += [s, linear(codes, scales=scales, dtype=torch.float16), linear(x)]
        return made + list(pkg.verify_drafts(logits, drafts, uniforms, starts=starts, draft_probs=probs, max_nodes=5))

    want = calls()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls())
    torch.cuda.synchronize()
    for rounds in got:
        for made in rounds:
            assert all(torch.equal(a, b) for a, b in zip(want, made))


@gpu
@pytest.mark.parametrize("vocab", [300001, 3000000])
def test_verification_over_very_large_vocabularies(pkg, vocab):
    """More ids than the parts of one pass have batches for, in rows of every alignment."""
    g = gen(vocab)
    logits = normal(g, 6, vocab + 7, dtype=torch.bfloat16)[:, 3:3 + vocab]
    probs = torch.softmax(logits.float().roll(1, 0) + 0.5 * normal(g, 6, vocab), 1)
    drafts = torch.multinomial(probs, 1, generator=g).squeeze(1).to(torch.int32)
    uniforms = torch.rand(6, device="cuda", generator=g, dtype=torch.float64)
    check_verify(pkg, logits, drafts, uniforms, [0, 3, 6], probs=probs, heat=[1.0, 0.7])
    check_verify(pkg, logits, drafts, uniforms, [0, 3, 6], parents=[0, 0, 0, 0, 0, 1], heat=[1.5, 0.7])


@gpu
def test_results_are_apart(pkg):
    """Small results come from one allocation: none overlaps another, and what is written into one
    changes nothing else and only its own version."""
    g = gen(3)
    x, w = normal(g, 3, 100, dtype=torch.bfloat16), torch.ones(100, device="cuda")
    pages = pkg.PageTable.empty(3, 4, 12, 8)
    u = torch.rand(3, device="cuda", generator=g, dtype=torch.float64)
    made = [pkg.residual_norm(x, x, w), pkg.residual_norm(x, x, w, quantise=True), pages.extend(ints([3, 9, 1]), 20),
            pkg.verify_drafts(normal(g, 3, 500), ints([1, 2, 3]), u, starts=ints([0, 2, 3]))]
    for results in made:
        before = [t.clone() for t in results]
        spans = sorted((t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t[0].numel()) * t.element_size()) for t in results)
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and all(t.data_ptr() % 16 == 0 for t in results)
        for i, t in enumerate(results):
            versions = [r._version for r in results]
            t.add_(1)
            assert [r._version - v for r, v in zip(results, versions)] == [int(i == k) for k in range(len(results))]
            assert all(torch.equal(r, b) for k, (r, b) in enumerate(zip(results, before)) if k > i)


@gpu
@pytest.mark.parametrize("cache", ["int8", "int4"])
def test_example_of_a_decoder_in_8_bit_integers(pkg, cache):
    """It runs, keeps to the grammar, and its logits are finite and do not hang on rows of other sequences."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "quantised_decode.py")
    spec = importlib.util.spec_from_file_location("quantised_decode", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    cfg = pkg.ModelConfig(512, 128, 128, 3, 4)
    params = pkg.init_params(cfg, 5)

    def model():
        return ex.QuantisedGpt(cfg, params, 3, cache, products="int8")

    words = torch.full((1, 16), -1, dtype=torch.int32, device="cuda")
    words[0, 1] = 0  # not 32..63
    out, steps = ex.generate(model(), [[1, 2, 3, 1, 2, 3], [7], [9, 8] * 20], 20, draft=4, allowed=words)
    assert [len(t) for t in out] == [20] * 3 and 1 <= steps <= 20
    assert all(0 <= x < 512 and not 32 <= x < 64 for t in out for x in t)
    both, one = model(), model()
    tokens = [5, 6, 7, 8, 9, 10]
    logits = both.logits(tokens, [0, 1, 2, 0, 1, 2], both.slots(0, range(3)) + both.slots(1, range(3)), [0, 0, 0], [0, 3, 6, 6], max_nodes=3)
    first = one.logits(tokens[:3], [0, 1, 2], one.slots(0, range(3)), [0, 0, 0], [0, 3, 3, 3], max_nodes=3)
    assert logits.isfinite().all() and torch.equal(logits[:3], first)


@gpu
@pytest.mark.parametrize("drawn", [False, True])
def test_verification_asks_for_sums_all_along_a_path(pkg, drawn):
    """Chains whose every test is next to equal, so that the walk goes on after each row's sum of 64 bits: to the
    last node, or to a rejected one; in clusters of every size, with more CTAs than the GPU holds at once."""
    g = gen(31)
    for vocab, n, seqs in ((1000, 6, 300), (6000, 5, 40), (40000, 4, 12)):
        logits = normal(g, seqs * n, vocab, dtype=torch.bfloat16)
        drafts = torch.randint(0, vocab, (seqs * n,), device="cuda", generator=g).to(torch.int32)
        p = torch.softmax(logits.double(), 1)
        at = p[:-1].gather(1, drafts[1:].long().unsqueeze(1)).squeeze(1)
        probs = None
        if drawn:
            probs = torch.softmax(normal(g, seqs * n, vocab), 1)
            at = at / probs[1:].gather(1, drafts[1:].long().unsqueeze(1)).squeeze(1).double()
        side = torch.full((seqs, n), 1 - 1e-12, dtype=torch.float64, device="cuda")
        want = [n if b % 3 == 0 else 1 + b % (n - 1) for b in range(seqs)]  # tokens of each sequence
        for b, w in enumerate(want):
            if w < n:
                side[b, w] = 1 + 1e-12
        uniforms = torch.rand(seqs * n, device="cuda", generator=g, dtype=torch.float64)
        uniforms[1:] = torch.where(torch.arange(1, seqs * n, device="cuda") % n == 0, uniforms[1:], at * side.flatten()[1:])
        args = dict(starts=ints(list(range(0, seqs * n + 1, n))), draft_probs=probs, max_nodes=n)
        first = pkg.verify_drafts(logits, drafts, uniforms, **args)
        assert first[2].tolist() == want
        some = 4 * n
        check_verify(pkg, logits[:some], drafts[:some], uniforms[:some], list(range(0, some + 1, n)),
                     probs=None if probs is None else probs[:some])
        for _ in range(20):
            assert all(torch.equal(a, b) for a, b in zip(first, pkg.verify_drafts(logits, drafts, uniforms, **args)))


@gpu
def test_verification_asks_for_sums_at_the_lowest_temperatures(pkg):
    """Below 1e-30 every test asks for its row's sum: p is shared by the largest logits."""
    g, rng = gen(32), random.Random(32)
    logits, drafts, uniforms, starts, parents, _ = verify_case(g, rng, [9, 1, 17, 6], 5000, torch.float32, True)
    logits = (logits * 0.5).round()
    drafts = ints([int(r[0]) for r in logits.topk(1, 1).indices[[max(p, 0) + starts[sum(s <= i for s in starts) - 1] for i, p in enumerate(parents)]]])
    for heat in (1e-31, 1e-36):
        check_verify(pkg, logits, drafts, uniforms, starts, parents, heat=[heat] * 4)
        check_verify(pkg, logits, drafts, uniforms, starts, heat=[heat] * 4)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_verification_of_temperatures_next_to_a_logits_step(pkg, dtype):
    """Temperatures down to far below the step between neighbouring logits: weights fall from 1 to
    nothing (below 2^-1000) within a few steps, and none lies beyond."""
    g, rng = gen(33), random.Random(33)
    vocab, nodes, cases = 2500, 3, []
    steps = torch.finfo(DTYPES[dtype]).eps
    for top in (1500.0, 30.0, 10.0, 1.0, -40.0):
        for heat in (1e-3, 1e-5, 1e-6, 1e-7, 1e-8, 1e-9, 3e-12):
            cases.append((top, heat))
    rows = nodes * len(cases)
    logits = torch.empty((rows, vocab), dtype=torch.float64, device="cuda")
    for i, (top, _) in enumerate(cases):
        step = 2.0 ** math.floor(math.log2(abs(top))) * steps  # of the type at the largest logit
        down = torch.randint(0, 13, (nodes, vocab), device="cuda", generator=g)
        logits[nodes * i:nodes * (i + 1)] = top - step * down
    logits = logits.to(DTYPES[dtype])
    drafts = torch.randint(0, vocab, (rows,), device="cuda", generator=g).to(torch.int32)
    drafts[1:] = torch.where(torch.rand(rows - 1, device="cuda", generator=g) < 0.7, logits[:-1].argmax(1), drafts[1:]).to(torch.int32)
    starts, heats = list(range(0, rows + 1, nodes)), [h for _, h in cases]
    parents = [i - 1 if rng.random() < 0.5 else 0 for _ in cases for i in range(nodes)]
    for _ in range(3):
        uniforms = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
        check_verify(pkg, logits, drafts, uniforms, starts, heat=heats)
        check_verify(pkg, logits, drafts, uniforms, starts, parents=parents, heat=heats)
        probs = torch.softmax(normal(g, rows, vocab), 1)
        check_verify(pkg, logits, drafts, uniforms, starts, probs=probs, heat=heats)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_verification_of_tiny_logits_at_tiny_temperatures(pkg, dtype):
    """Zeros of both signs and logits below the normal numbers, at temperatures about as small: as in fp64."""
    g = gen(34)
    vocab, nodes = 1500, 3
    least = 2.0 ** -149 if dtype == "fp32" else 2.0 ** -133  # of the type
    heats = [least, 3 * least, 1e-38, 3e-37, 1e-31, 1e-24, 1e-21, 1e-3]
    rows = nodes * len(heats)
    for step in (least, 1e-38, 1e-24):
        logits = -step * torch.randint(0, 9, (rows, vocab), device="cuda", generator=g).double()
        logits = logits.to(DTYPES[dtype])  # -0 among them
        logits[:, ::7] = logits[:, ::7].abs() * 0
        logits[:, 5::11] = -1e30
        drafts = logits.argmax(1).roll(1).to(torch.int32)
        for _ in range(3):
            uniforms = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
            check_verify(pkg, logits, drafts, uniforms, list(range(0, rows + 1, nodes)), heat=heats)
            check_verify(pkg, logits, drafts, uniforms, list(range(0, rows + 1, nodes)), parents=[-1, 0, 0] * len(heats), heat=heats)
            check_verify(pkg, logits, drafts, uniforms, list(range(0, rows + 1, nodes)), heat=heats,
                         probs=torch.softmax(normal(g, rows, vocab), 1))


@gpu
def test_products_read_what_the_launch_before_has_just_written(pkg):
    """Rows and weights that are made again and again in the same memory by the launch before a product,
    which begins under it: nothing of the round before is read."""
    g = gen(35)
    k, n = 1040, 600
    weight = torch.ones(k, device="cuda")
    sources = [normal(g, n, k), 3 * normal(g, n, k)]

    def round_of(x, w):
        codes, scales = pkg.quantise_rows(w)
        linear = pkg.W8Linear(codes, scales)
        y = linear(x)  # begins under the rows' codes
        _, c, s = pkg.residual_norm(x, x, weight, quantise=True)
        made = [y, linear(c, scales=s)]
        codes.copy_(pkg.quantise_rows(-w)[0])  # the same memory, for a product right behind
        return made + [pkg.W8Linear(*pkg.quantise_rows(w[:, :256]))(c[:, :256], scales=s), linear(c, scales=s)]

    for rows in (1, 2, 4, 40, 100, 300, 600):
        xs = [normal(g, rows, k, dtype=torch.bfloat16), 5 * normal(g, rows, k, dtype=torch.bfloat16)]
        want = []
        for x, w in zip(xs, sources):
            want.append([t.clone() for t in round_of(x, w)])
            torch.cuda.synchronize()
        got = [round_of(xs[i % 2], sources[i % 2]) for i in range(12)]
        for i, made in enumerate(got):
            assert all(torch.equal(a, b) for a, b in zip(want[i % 2], made))
        for i in range(12):  # memory of the round before, freed
            made = round_of(xs[i % 2], sources[i % 2])
            assert all(torch.equal(a, b) for a, b in zip(want[i % 2], made))
            del made


@gpu
def test_serving_operators_refuse_tangents(pkg):
    """Forward-mode derivatives are not computed either, and do not vanish in silence."""
    from torch.autograd import forward_ad
    w = torch.ones(64, device="cuda")
    plain = torch.randn((3, 64), device="cuda")
    linear, four = pkg.W8Linear.pack(torch.randn(64, 20, device="cuda")), pkg.W4Linear.pack(torch.randn(64, 20, device="cuda"))
    cache = pkg.QuantKvCache.empty(2, 16, 1, 64)
    table, lens = ints([[0], [1], [1]]), ints([0, 0, 0])
    codes, scales = pkg.quantise_rows(plain)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        x = dual(plain)
        calls = [lambda: pkg.residual_norm(x, plain, w), lambda: pkg.residual_norm(plain, x, w), lambda: pkg.residual_norm(None, x, w),
                 lambda: pkg.residual_norm(plain, plain, dual(w), quantise=True), lambda: pkg.residual_norm(plain, plain, w, dual(w)),
                 lambda: pkg.residual_norm(plain, plain, w, gate=x), lambda: pkg.residual_norm(plain, plain, w, post_weight=dual(w)),
                 lambda: linear(x), lambda: linear(codes, scales=dual(scales)),
                 lambda: pkg.W8Linear(linear.codes, dual(linear.scales))(plain),
                 lambda: pkg.W8Linear(linear.codes, linear.scales, dual(w[:20]))(plain), lambda: pkg.quantise_rows(x),
                 lambda: four(x), lambda: pkg.logit_controls(x), lambda: pkg.logit_controls(x, out=plain.clone()),
                 lambda: pkg.logit_controls(plain, out=dual(plain.clone())),
                 lambda: cache.attend(x.view(3, 1, 64), table, lens)]
        for call in calls:
            with torch.no_grad(), pytest.raises(pkg.ArgumentError, match="computes no gradient"):
                call()
            with pytest.raises(pkg.ArgumentError, match="computes no gradient"):
                call()
        assert pkg.residual_norm(plain, plain, w)[1].shape == plain.shape  # none here
        cache.write(x.view(3, 1, 64), x.view(3, 1, 64), ints([0, 1, 2]))  # (its values)


@gpu
def test_verification_over_the_largest_vocabulary(pkg):
    """2^31 - 65537 ids: ends of parts come near 2^31.  Four of them have a weight, in the first and last parts."""
    vocab = 2**31 - 1 - 65536
    ids = [5, vocab // 2, vocab - 200000, vocab - 1]
    row = torch.full((1, vocab), -math.inf, dtype=torch.bfloat16, device="cuda")
    row[0, ids] = 0.0
    with pytest.raises(pkg.ArgumentError):
        pkg.verify_drafts(torch.empty((1, vocab + 1), dtype=torch.bfloat16, device="cuda"), ints([0]),
                          torch.zeros(1, dtype=torch.float64, device="cuda"))
    uniforms = torch.tensor([0.1, 0.3, 0.6, 0.9], dtype=torch.float64, device="cuda")
    for heat in (None, torch.full((4,), 1e-20, device="cuda")):
        tokens, _, counts = pkg.verify_drafts(row.expand(4, vocab), ints([0] * 4), uniforms, temperature=heat)
        assert tokens.flatten().tolist() == ids and counts.eq(1).all()
    tokens, _, _ = pkg.verify_drafts(row, ints([0]), uniforms[:1], temperature=torch.zeros(1, device="cuda"))
    assert tokens.tolist() == [[5]]
    drafts, starts = ints([0, ids[3], 0, ids[2]]), ints([0, 2, 4])
    uniforms = torch.tensor([0.9, 0.2, 0.7, 0.3], dtype=torch.float64, device="cuda")
    tokens, nodes, counts = pkg.verify_drafts(row.expand(4, vocab), drafts, uniforms, starts=starts, max_nodes=2)
    assert counts.tolist() == [2, 1] and tokens.tolist() == [[ids[3], ids[3]], [ids[3], -1]] and nodes.tolist() == [[0, 1], [0, -1]]

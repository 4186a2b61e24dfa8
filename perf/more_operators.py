"""The operators around attention in a serving step, as measured cases.

A step that drafts tokens and verifies them runs, besides projections and
attention over its paged cache:

  pages    pages for the new tokens of every sequence and the tables and slots
           that the cache's write and its attention take; pages of dropped
           tokens go back
  norm     a block's output onto the residual stream (normed itself, gated and
           scaled, each optional) and the norm before the next block
  project  products in 8-bit integers with a scale for each token and output
  enter    norm and project together, as a block begins: the norm's result
           leaves as 8-bit codes and scales
  verify   drafted tokens against the target's probabilities, and the token
           that follows the accepted ones

`run` computes each either in elementary torch operations (`own` false) or
through the library's public calls (`own` true).

Formulas.  Rows of codes: top = max|x|, code = round(x * (127 / top)) to the
nearest even, each step rounded to fp32, scale = top / 127.
Norm: s = x + scale * gate * post(h), y = pre(s), with post and pre either
(v - mean) / sqrt(var + eps) * w + b or v / sqrt(mean of squares + eps) * w.
Verify: rows of a sequence are its last token and the drafts below it, parents
before children.  At a node with p = softmax(logits / temperature), its drafts
c are tried in order: with draft probabilities q (one draft to a node) c is
accepted where u[c] q(c) < p(c), and what may follow a rejected one is
max(p - q, 0); without, where u[c] (1 - p of rejected siblings) < p(c), and
what may follow rejected ones is p without them.  An accepted draft is the next
node.  Where none is, the last token is the lowest id at which the running sum
of what may follow passes u[first row] times its total.  Temperature 0: p is 1
at the (lowest) largest logit.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5


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
        # one decode step of a batch: a token and up to 7 drafts of each sequence (latency)
        {"name": "pages-step", "op": "pages", "seqs": 32, "len_hi": 1000, "new_lo": 1, "new_hi": 8, "page": 16, "short": False},
        # a step that takes in many prompts, or parts of them
        {"name": "pages-prompts", "op": "pages", "seqs": 512, "len_hi": 4000, "new_lo": 1, "new_hi": 511, "page": 32,
         "short": False},
        # between two blocks of the 98M model, one token (latency)
        {"name": "norm-step", "op": "norm", "rows": 1, "dim": 768, "dtype": "fp32", "stream": "fp32", "kind": "layer",
         "post": False, "gate": "none", "scale": 1.0},
        # between two blocks of a large model with norms on both sides and gates, a prompt
        {"name": "norm-prompt", "op": "norm", "rows": 16383, "dim": 4096, "dtype": "bf16", "stream": "fp32", "kind": "rms",
         "post": True, "gate": "all", "scale": 0.7},
        # one token through the fused q/k/v projection of the 98M model (latency)
        {"name": "int8-step", "op": "project", "rows": 1, "k": 768, "n": 2304, "dtype": "fp32"},
        # one token through a large model's widest projection
        {"name": "int8-large", "op": "project", "rows": 1, "k": 8192, "n": 28672, "dtype": "bf16"},
        # a long prompt through a large model's widest projection
        {"name": "int8-prompt", "op": "project", "rows": 8192, "k": 4096, "n": 14336, "dtype": "bf16"},
        # the rows of a drafted tree into the first MLP projection of the 220M model
        {"name": "enter-tree", "op": "enter", "rows": 61, "dim": 1024, "n": 4096, "dtype": "fp16", "stream": "fp16",
         "kind": "layer", "post": False, "gate": "none", "scale": 1.0},
        # a prompt into a large model's projection
        {"name": "enter-prompt", "op": "enter", "rows": 4095, "dim": 4096, "n": 11008, "dtype": "bf16", "stream": "bf16",
         "kind": "rms", "post": False, "gate": "rows", "scale": 1.0},
        # one sequence of the 98M model with 4 drafts of a smaller model (latency)
        {"name": "verify-chain", "op": "verify", "seqs": 1, "nodes_lo": 5, "nodes_hi": 5, "vocab": 16384, "probs": True,
         "masked": False, "dtype": "fp32"},
        # a batch with up to 7 drafts each over a large vocabulary
        {"name": "verify-batch", "op": "verify", "seqs": 32, "nodes_lo": 3, "nodes_hi": 8, "vocab": 131071, "probs": True,
         "masked": False, "dtype": "bf16"},
        # trees of drafts taken from the text itself, under a grammar's mask
        {"name": "verify-tree", "op": "verify", "seqs": 8, "nodes_lo": 9, "nodes_hi": 64, "vocab": 50257, "probs": False,
         "masked": True, "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pages", "norm", "norm", "project", "project", "enter", "verify", "verify"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "pages":
        seqs = _log_int(rng, 1, 1024)
        new_hi = _log_int(rng, 1, max(1, min(4096, 130000 // seqs)))
        return {"op": op, "seqs": seqs, "len_hi": _log_int(rng, 16, 8000), "new_lo": rng.randint(0, new_hi), "new_hi": new_hi,
                "page": rng.choice([8, 16, 32, 64, 128]), "short": rng.random() < 0.3}
    if op == "norm":
        dim = _log_int(rng, 33, 16384)
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        return {"op": op, "rows": _log_int(rng, 1, min(65536, 60000000 // dim)), "dim": dim, "dtype": dtype,
                "stream": rng.choice([dtype, "fp32"]), "kind": rng.choice(["layer", "rms"]), "post": rng.random() < 0.5,
                "gate": rng.choice(["none", "all", "rows"]), "scale": rng.choice([1.0, 0.5, 0.22])}
    if op == "verify":
        probs = rng.random() < 0.5
        vocab = _log_int(rng, 1000, 200000)
        nodes_hi = _log_int(rng, 1, 12 if probs else 64)
        seqs = _log_int(rng, 1, max(1, min(64, 24000000 // (vocab * nodes_hi))))
        return {"op": op, "seqs": seqs, "nodes_lo": rng.randint(1, nodes_hi), "nodes_hi": nodes_hi, "vocab": vocab,
                "probs": probs, "masked": rng.random() < 0.4, "dtype": dtype}
    k = _log_int(rng, 64, 16384)
    if rng.random() < 0.5:
        k = k // 64 * 64
    n = _log_int(rng, 64, min(16384, 200000000 // k))
    rows = _log_int(rng, 1, min(8192, 400000000000 // (k * n))) if rng.random() < 0.7 else rng.randint(1, 8)
    if op == "project":
        return {"op": op, "rows": rows, "k": k, "n": n, "dtype": dtype}
    # codes of values that were computed in fp32 may fall to either side of a half, which fp32 results would show
    dtype = rng.choice(["bf16", "fp16"])
    return {"op": op, "rows": rows, "dim": k, "n": n, "dtype": dtype, "stream": rng.choice([dtype, "fp32"]),
            "kind": rng.choice(["layer", "rms"]), "post": rng.random() < 0.5, "gate": rng.choice(["none", "all", "rows"]),
            "scale": rng.choice([1.0, 0.5])}


def _spread(lo, hi, count):
    """`count` whole numbers over lo..hi in no order, both ends among them where they fit."""
    if count == 1:
        return [hi]
    step = 7 if count % 7 else 11
    return [lo + (hi - lo) * ((i * step + 3) % count) // (count - 1) for i in range(count)]


def _requests(case):
    """Cached and new tokens of each sequence, pages held and pages wanted."""
    lens = _spread(0, case["len_hi"], case["seqs"])
    news = _spread(case["new_lo"], case["new_hi"], case["seqs"])[::-1]
    page = case["page"]
    held = [-(-n // page) for n in lens]
    want = [-(-(n + c) // page) - h for n, c, h in zip(lens, news, held)]
    return lens, news, held, want


def _norm_work(case, out_size):
    """Bytes of the norm's inputs and of the stream that it writes, and of its result."""
    size, wide = (4 if case[t] == "fp32" else 2 for t in ("dtype", "stream"))
    rows, dim = case["rows"], case["dim"]
    gate = {"none": 0, "all": dim * size, "rows": rows * dim * size}[case["gate"]]
    weights = 4 * dim * (1 + (case["kind"] == "layer")) * (1 + case["post"])
    return rows * dim * (size + 2 * wide + out_size) + gate + weights


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "pages":
        lens, news, held, want = _requests(case)
        # counts and lengths in, starts, prefixes and lengths out, twice; slots and positions; pages off the list and back
        return {"bytes": 4 * (8 * case["seqs"] + 2 * case["seqs"] * case["new_hi"] + 4 * sum(want)), "flops": 0}
    if case["op"] == "norm":
        return {"bytes": _norm_work(case, size), "flops": 0}
    if case["op"] == "project":
        k, n, rows = case["k"], case["n"], case["rows"]
        return {"bytes": k * n + 8 * n + rows * (k + n) * size, "flops": 2 * rows * k * n}
    if case["op"] == "enter":
        k, n, rows = case["dim"], case["n"], case["rows"]
        return {"bytes": _norm_work(case, 0) + k * n + 8 * n + rows * n * size, "flops": 2 * rows * k * n}
    rows = sum(_spread(case["nodes_lo"], case["nodes_hi"], case["seqs"]))
    probs = case["seqs"] * case["vocab"] * 4 if case["probs"] else 0
    return {"bytes": rows * (case["vocab"] * size + 16) + probs, "flops": 0}


# ---- inputs ---------------------------------------------------------------------

def _codes(x):
    """(codes, scales) of fp32 rows, by the formula."""
    top = x.abs().amax(-1, keepdim=True)
    live = top >= 1e-35
    full = torch.full((), 127.0, device=x.device)
    inv = full / torch.where(live, top, 1.0)
    code = torch.where(live, torch.round(x * inv).clamp(-127, 127), 0.0)
    return code.to(torch.int8), torch.where(live, top / full, 0.0).squeeze(-1)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    dtype = s["dtype"] = DTYPES.get(case.get("dtype"))

    def normal(*shape):
        return torch.randn(shape, device=DEV, generator=gen)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    if case["op"] == "pages":
        lens, news, held, want = _requests(case)
        page, seqs = case["page"], case["seqs"]
        spare = sum(want) * 2 // 3 if case["short"] else sum(want) + 5
        width = -(-(case["len_hi"] + case["new_hi"]) // page)
        pages = sum(held) + spare
        order = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
        at = torch.arange(width, device=DEV)
        first = ints(held).cumsum(0) - ints(held)
        taken = at < ints(held)[:, None]
        s["table"] = torch.where(taken, order[torch.where(taken, first[:, None] + at, 0)], -1).to(torch.int32).contiguous()
        s["free"] = torch.zeros(pages, dtype=torch.int32, device=DEV)
        s["free"][:spare] = order[sum(held):]
        s["n_free"], s["lens"], s["counts"] = ints([spare]), ints(lens), ints(news)
        s["most"] = max(1, seqs * case["new_hi"] * 7 // 8 if case["short"] else sum(news))
        if own:
            s["pages"] = _package().PageTable(s["table"], s["lens"], s["free"], s["n_free"], page)
    if case["op"] in ("norm", "enter"):
        rows, dim = case["rows"], case["dim"]
        s["h"] = normal(rows, dim).to(dtype)
        s["x"] = (3.0 * normal(rows, dim) + 0.3).to(DTYPES[case["stream"]])
        bias = case["kind"] == "layer"
        s["w"], s["b"] = 1.0 + 0.2 * normal(dim), 0.2 * normal(dim) if bias else None
        s["post_w"] = 1.0 + 0.2 * normal(dim) if case["post"] else None
        s["post_b"] = 0.2 * normal(dim) if case["post"] and bias else None
        shape = {"none": None, "all": (dim,), "rows": (rows, dim)}[case["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(normal(*shape)).to(dtype)
    if case["op"] in ("project", "enter"):
        k, n = case["k"] if case["op"] == "project" else case["dim"], case["n"]
        s["codes"] = torch.zeros((n, -(-k // 16) * 16), dtype=torch.int8, device=DEV)[:, :k]
        s["codes"].copy_((40.0 * normal(n, k)).round().clamp(-127, 127))
        s["scales"] = (0.5 + torch.rand(n, device=DEV, generator=gen)) / (40.0 * math.sqrt(k))
        s["bias"] = 0.1 * normal(n)
        if case["op"] == "project":
            s["a"] = normal(case["rows"], k).to(dtype)
        if own:
            s["linear"] = _package().W8Linear(s["codes"], s["scales"], s["bias"])
    if case["op"] == "verify":
        seqs, vocab = case["seqs"], case["vocab"]
        nodes = _spread(case["nodes_lo"], case["nodes_hi"], seqs)
        starts, parents = [0], []
        pick = torch.rand(sum(nodes), generator=torch.Generator().manual_seed(seed)).tolist()
        nth = []  # which child of its parent a row is
        for t in nodes:
            kids = [0] * t
            for i in range(t):
                parent = i - 1 if case["probs"] or not i else int(pick[starts[-1] + i] ** 0.5 * i)
                parents.append(parent)
                nth.append(kids[parent] if i else 0)
                if i:
                    kids[parent] += 1
            starts.append(starts[-1] + t)
        rows = starts[-1]
        # a few tokens that stand out over a long tail, as language has it
        x = 1.5 * normal(rows, vocab)
        band = vocab // 24
        high = torch.randint(0, band, (rows, 24), device=DEV, generator=gen) + band * torch.arange(24, device=DEV)
        x.scatter_add_(1, high, 12.0 * torch.rand((rows, 24), device=DEV, generator=gen))
        s["logits"] = x.to(dtype)
        first = ints(starts[:-1]).long().repeat_interleave(ints(nodes).long())
        above = (first + ints(parents).long()).clamp(min=0)  # the row of a draft's parent
        temperature = [0.0 if i % 4 == 3 else 0.6 + 0.1 * (i % 7) for i in range(seqs)]
        s["temperature"] = torch.tensor(temperature, device=DEV)
        heat = s["temperature"].clamp(min=0.1).repeat_interleave(ints(nodes).long())[:, None]
        if case["probs"]:
            s["probs"] = torch.softmax((s["logits"].float()[above] + 0.7 * normal(rows, vocab)) / heat, 1)
            s["drafts"] = torch.multinomial(s["probs"], 1, generator=gen).squeeze(1).to(torch.int32)
            s["parents"] = None
        else:
            s["probs"] = None
            best = x.topk(64, 1).indices[above]
            s["drafts"] = best.gather(1, ints(nth).long()[:, None]).squeeze(1).to(torch.int32)
            s["parents"] = ints(parents)
        if case["masked"]:
            s["logits"].masked_fill_(torch.rand((rows, vocab), device=DEV, generator=gen) < 0.3, -math.inf)
        s["uniforms"] = torch.rand(rows, device=DEV, generator=gen, dtype=torch.float64)
        s["starts"], s["max_nodes"] = ints(starts), max(nodes)
    return s


# ---- one pass ---------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if not own:
        return {"pages": _pages, "norm": _norm, "project": _project, "enter": _enter, "verify": _verify}[op](s)
    pkg = _package()
    if op == "pages":
        # pages for the step's tokens; then, as after a step whose tokens were all dropped, all of them back
        starts, prefix, slots, positions = s["pages"].extend(s["counts"], s["most"])
        s["pages"].truncate(prefix)
        return starts, prefix, slots, positions, s["table"], s["lens"], s["free"], s["n_free"]
    if op == "project":
        return s["linear"](s["a"])
    if op in ("norm", "enter"):
        c = s["case"]
        made = pkg.residual_norm(s["h"], s["x"], s["w"], s["b"], post_weight=s["post_w"], post_bias=s["post_b"], gate=s["gate"],
                                 scale=c["scale"], kind=c["kind"], eps=EPS, quantise=op == "enter")
        if op == "norm":
            return made
        return made[0], s["linear"](made[1], scales=made[2], dtype=s["dtype"])
    return pkg.verify_drafts(s["logits"], s["drafts"], s["uniforms"], starts=s["starts"], parents=s["parents"],
                             draft_probs=s["probs"], temperature=s["temperature"], max_nodes=s["max_nodes"])


def _before(x):
    return x.cumsum(0) - x


def _pages(s):
    page, most = s["case"]["page"], s["most"]
    table, lens, free, n_free = s["table"].clone(), s["lens"].long(), s["free"].clone(), s["n_free"].long()
    count = s["counts"].long()
    held = (lens + page - 1) // page
    fits = lens + count <= table.shape[1] * page
    count = torch.where(fits, count, 0)
    need = torch.where(fits, (lens + count + page - 1) // page - held, 0)
    served = (count.cumsum(0) <= most) & ((need == 0) | (need.cumsum(0) <= n_free))
    count, need = torch.where(served, count, 0), torch.where(served, need, 0)
    ends, wanted = count.cumsum(0), need.cumsum(0)
    # pages from the end of the list, in the sequences' order
    j = torch.arange(free.shape[0], device=DEV)
    seq = torch.searchsorted(wanted, j, right=True)
    inside = seq < len(lens)
    seq = torch.where(inside, seq, 0)
    place = torch.where(inside, held[seq] + j - _before(need)[seq], 0)
    taken = free[torch.where(inside, n_free - 1 - j, 0)]
    wide = torch.cat((table, torch.zeros_like(table[:, :1])), 1)  # what is outside goes into one more column
    wide[seq, torch.where(inside, place, table.shape[1])] = taken
    table = wide[:, :-1].contiguous()
    row = torch.arange(most, device=DEV)
    seq = torch.searchsorted(ends, row, right=True)
    live = seq < len(lens)
    seq = torch.where(live, seq, 0)
    position = torch.where(live, lens[seq] + row - _before(count)[seq], 0)
    slots = torch.where(live, table[seq, position // page].long() * page + position % page, -1).to(torch.int32)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends)).to(torch.int32)
    # back to the lengths before
    n_free, now = n_free - wanted[-1:], (lens + count + page - 1) // page
    j = torch.arange(free.shape[0], device=DEV)
    drop = now - held
    dropped = drop.cumsum(0)
    seq = torch.searchsorted(dropped, j, right=True)
    inside = seq < len(lens)
    seq = torch.where(inside, seq, 0)
    place = torch.where(inside, held[seq] + j - _before(drop)[seq], 0)
    to = torch.where(inside, n_free + dropped[-1:] - 1 - j, free.shape[0])
    longer = torch.cat((free, free[:1]))
    longer[to] = table[seq, place]
    free = longer[:-1].contiguous()
    table = torch.where(torch.arange(table.shape[1], device=DEV) >= held[:, None], -1, table)
    return (starts, s["lens"].clone(), slots, position.to(torch.int32), table, s["lens"].clone(), free,
            (n_free + dropped[-1:]).to(torch.int32))


def _normed(v, w, b, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w
    return v if b is None else v + b


def _stream(s):
    c = s["case"]
    h = s["h"].float()
    if s["post_w"] is not None:
        h = _normed(h, s["post_w"], s["post_b"], c["kind"])
    if s["gate"] is not None:
        h = h * s["gate"].float()
    return s["x"].float() + c["scale"] * h


def _norm(s):
    x = _stream(s)
    return x.to(s["x"].dtype), _normed(x, s["w"], s["b"], s["case"]["kind"]).to(s["dtype"])


def _product(s, codes, scales):
    return ((codes.float() @ s["codes"].float().T) * s["scales"] * scales[:, None] + s["bias"]).to(s["dtype"])


def _project(s):
    return _product(s, *_codes(s["a"].float()))


def _enter(s):
    x = _stream(s)
    return x.to(s["x"].dtype), _product(s, *_codes(_normed(x, s["w"], s["b"], s["case"]["kind"])))


def _verify(s):
    seqs, wide = s["case"]["seqs"], s["max_nodes"]
    first, last = s["starts"][:-1].long(), s["starts"][1:].long()
    owner = torch.arange(seqs, device=DEV).repeat_interleave(last - first)
    heat = s["temperature"].double()[owner][:, None]
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    # running sums next to a border need 64 bits
    e = torch.exp((x - top) / torch.where(heat > 0, heat, 1.0))
    column = torch.arange(x.shape[1], device=DEV)
    best = (column == torch.where(x == top, column, x.shape[1]).amin(1, keepdim=True)).double()  # the lowest of equal ones
    e = torch.where(heat > 0, e, best)
    total = e.sum(1)
    parent = torch.arange(len(e), device=DEV) - 1 - first[owner] if s["parents"] is None else s["parents"].long()
    at = torch.zeros(seqs, dtype=torch.long, device=DEV)          # the node that was come to, counted from the first
    gone = torch.zeros((seqs, x.shape[1]), dtype=torch.bool, device=DEV)
    rejected = torch.full((seqs,), -1, dtype=torch.long, device=DEV)
    nodes = torch.full((seqs, wide), -1, dtype=torch.long, device=DEV)
    tokens = nodes.clone()
    nodes[:, 0] = 0
    count = torch.ones(seqs, dtype=torch.long, device=DEV)
    every = torch.arange(seqs, device=DEV)
    for i in range(1, wide):
        row = torch.where(first + i < last, first + i, first)
        tried = (first + i < last) & (parent[row] == at)
        node = first + at
        token = s["drafts"].long()[row]
        mass = torch.where(gone[every, token], 0.0, e[node, token])
        if s["probs"] is None:
            # u (total - rejected ones) < p
            left = total[node] - torch.where(gone, e[node], 0.0).sum(1)
            good = s["uniforms"][row] * left < mass
        else:
            good = s["uniforms"][row] * s["probs"].double()[row, token] * total[node] < mass
        yes, no = tried & good, tried & ~good
        where = torch.where(yes, count, 0)
        nodes[every, where] = torch.where(yes, i, nodes[every, where])
        where = torch.where(yes, count - 1, wide - 1)
        tokens[every, where] = torch.where(yes, token, tokens[every, where])
        count = count + yes
        at = torch.where(yes, i, at)
        gone = gone & ~yes[:, None]
        rejected = torch.where(no, first + i, torch.where(yes, -1, rejected))
        gone[every, token] = gone[every, token] | no
    node = first + at
    rest = torch.where(gone, 0.0, e[node])
    if s["probs"] is not None:
        q = s["probs"].double()[rejected.clamp(min=0)]
        rest = torch.where(rejected[:, None] >= 0, (e[node] / total[node][:, None] - q).clamp(min=0), e[node])
    run_sum = rest.cumsum(1)
    target = s["uniforms"][first] * run_sum[:, -1]
    token = torch.searchsorted(run_sum, target[:, None], right=True).squeeze(1)
    tokens[every, count - 1] = token
    return tokens.to(torch.int32), nodes.to(torch.int32), count.to(torch.int32)


# ---- the definitions in 64 bits -----------------------------------------------------

def _exact_norm(v, w, b, kind):
    centre = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    spread = (v - centre).square().mean(1, keepdim=True)
    out = (v - centre) * torch.rsqrt(spread + EPS) * w.double()
    return out if b is None else out + b.double()


def _exact_stream(s):
    c = s["case"]
    h = s["h"].double() if s["post_w"] is None else _exact_norm(s["h"].double(), s["post_w"], s["post_b"], c["kind"])
    return torch.addcmul(s["x"].double(), h, torch.ones_like(h) if s["gate"] is None else s["gate"].double().expand_as(h),
                         value=c["scale"])


def _exact_product(s, y):
    """y's codes (the formula's roundings are part of it) times the weights."""
    y = y.float()
    top = y.abs().max(1, keepdim=True).values
    code = torch.round(y * (torch.full_like(top, 127.0) / top)).double()
    out = torch.empty((y.shape[0], s["case"]["n"]), dtype=torch.float64, device=DEV)
    for at in range(0, s["case"]["n"], 2048):
        part = slice(at, at + 2048)
        out[:, part] = code @ s["codes"][part].double().T * s["scales"][part].double()
    return out * (top.double() / 127) + s["bias"].double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        page, most = case["page"], s["most"]
        table, lens, free = s["table"].tolist(), s["lens"].tolist(), s["free"].tolist()
        n_free, rows, new_pages = int(s["n_free"]), 0, 0
        starts, slots, positions = [0], [], []
        asked = wanted = 0  # by the sequences up to here, served or not
        before = [list(t) for t in table]
        for b, count in enumerate(s["counts"].tolist()):
            if lens[b] + count > len(table[b]) * page:
                count = 0
            need = -(-(lens[b] + count) // page) - -(-lens[b] // page)
            asked, wanted = asked + count, wanted + need
            if asked > most or (need and wanted > n_free):
                count = need = 0
            for p in range(lens[b], lens[b] + count):
                if table[b][p // page] < 0:
                    new_pages += 1
                    table[b][p // page] = free[n_free - new_pages]
                slots.append(table[b][p // page] * page + p % page)
                positions.append(p)
            starts.append(len(slots))
        rows = len(slots)
        slots += [-1] * (most - rows)
        positions += [0] * (most - rows)
        lists = (starts, lens, slots, positions, before, lens, free, [n_free])
        return tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in lists)
    if case["op"] == "norm":
        x = _exact_stream(s)
        return x, _exact_norm(x, s["w"], s["b"], case["kind"])
    if case["op"] == "project":
        return _exact_product(s, s["a"])
    if case["op"] == "enter":
        x = _exact_stream(s)
        return x, _exact_product(s, _exact_norm(x, s["w"], s["b"], case["kind"]))
    wide, starts = s["max_nodes"], s["starts"].tolist()
    drafts, uniforms = s["drafts"].tolist(), s["uniforms"].tolist()
    tokens, nodes, counts = [], [], []
    for b in range(case["seqs"]):
        a, rows = starts[b], starts[b + 1] - starts[b]
        heat = float(s["temperature"][b])

        def target(i):
            x = s["logits"][a + i].double()
            if heat > 0:
                return torch.softmax(x / heat, 0)
            p = torch.zeros_like(x)
            p[int((x == x.max()).nonzero()[0])] = 1.0
            return p

        kids = [[] for _ in range(rows)]
        for i in range(1, rows):
            kids[i - 1 if s["parents"] is None else int(s["parents"][a + i])].append(i)
        path, said, node = [0], [], 0
        while node is not None:
            p = target(node)
            node = None
            for c in kids[path[-1]]:
                token, u = drafts[a + c], uniforms[a + c]
                if s["probs"] is not None:
                    q = s["probs"][a + c].double()
                    if u * float(q[token]) < float(p[token]):
                        node = c
                    else:
                        p = torch.clamp(p - q, min=0)
                elif u * float(p.sum()) < float(p[token]):
                    node = c
                else:
                    p[token] = 0
                if node is not None:
                    break
            if node is not None:
                said.append(drafts[a + node])
                path.append(node)
        sums = torch.cumsum(p, 0)
        said.append(int((sums <= uniforms[a] * float(sums[-1])).sum()))
        tokens.append(said + [-1] * (wide - len(said)))
        nodes.append(path + [-1] * (wide - len(path)))
        counts.append(len(said))
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (tokens, nodes, counts))

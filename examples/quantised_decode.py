"""Greedy generation with the serving operators: 4-bit projections, a paged
K/V cache that is quantised as it is written, attention of drafted trees over
it, and penalties and a grammar's mask on the logits.

    python examples/quantised_decode.py [--cache int4] [--draft 0] ...

Weights are the seeded initialisation of a GPT of the given size.  Each step
runs the last token of every sequence and two drafted continuations, taken
from where the sequence had the same token before; the greedy path through
them is kept.  torch computes the embeddings, norms and GELU around the
operators.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import __graft_entry__ as graft  # noqa: E402

forge = graft.load_package()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class QuantisedGpt:
    """The GPT of a ModelConfig with W4Linear projections and one QuantKvCache
    per layer; sequence s owns pages s * pages_per_seq onwards."""

    def __init__(self, cfg, params, seqs: int, cache: str = "int8", group: int = 64, page: int = 32,
                 dtype=torch.bfloat16, spare: int = 16):
        self.cfg, self.dtype, self.page = cfg, dtype, page
        p = {n: torch.from_numpy(a).cuda() for n, a in zip(forge.param_names(cfg), params)}
        self.norms = {n: t.to(dtype) for n, t in p.items() if ".ln" in n or n.startswith("ln_f")}
        self.tok, self.pos = p["tok_emb"].to(dtype), p["pos_emb"].to(dtype)
        self.layers = [{n: forge.W4Linear.pack(p[f"blocks.{i}.{n}.w"], group, p[f"blocks.{i}.{n}.b"])
                        for n in ("attn.qkv", "attn.proj", "mlp.fc", "mlp.proj")} for i in range(cfg.n_layers)]
        self.head = forge.W4Linear.pack(p["tok_emb"].t().contiguous(), group)
        pages = -(-(cfg.context_length + spare) // page)  # a step's drafted rows may pass the last position
        self.table = torch.arange(seqs * pages, dtype=torch.int32, device="cuda").view(seqs, pages)
        self.caches = [forge.QuantKvCache.empty(seqs * pages, page, cfg.n_heads, cfg.head_dim, cache)
                       for _ in range(cfg.n_layers)]

    def slots(self, seq: int, places) -> list[int]:
        first = seq * self.table.shape[1] * self.page
        return [first + at for at in places]

    def _norm(self, x, name):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], self.norms[name + ".w"], self.norms[name + ".b"], 1e-5)

    def logits(self, tokens, positions, slots, prefix, starts, mask=None, max_nodes=None):
        """Logits [rows, vocab] of rows that are written to `slots`; the rest
        as in QuantKvCache.attend.  tokens and positions: [rows] on the host."""
        cfg, rows = self.cfg, len(tokens)
        slots, prefix, starts = _ints(slots), _ints(prefix), _ints(starts)
        x = self.tok[_ints(tokens).long()] + self.pos[_ints(positions).long()]
        for i, layer in enumerate(self.layers):
            qkv = layer["attn.qkv"](self._norm(x, f"blocks.{i}.ln1")).view(rows, 3, cfg.n_heads, cfg.head_dim)
            self.caches[i].write(qkv[:, 1], qkv[:, 2], slots)
            out, _ = self.caches[i].attend(qkv[:, 0], self.table, prefix, starts=starts, mask=mask, max_nodes=max_nodes)
            x = x + layer["attn.proj"](out.reshape(rows, -1))
            h = layer["mlp.fc"](self._norm(x, f"blocks.{i}.ln2"))
            x = x + layer["mlp.proj"](torch.nn.functional.gelu(h, approximate="tanh"))
        return self.head(self._norm(x, "ln_f"))

    def move(self, seq: int, sources: list[int], targets: list[int]) -> None:
        """Copies cache rows as they are (the kept drafted rows to their places)."""
        a, b = (torch.tensor(self.slots(seq, s), device="cuda") for s in (sources, targets))
        for c in self.caches:
            for t in (c.codes, c.meta):
                t[b // self.page, :, :, b % self.page] = t[a // self.page, :, :, a % self.page]


def draft_tree(history: list[int], depth: int, room: int) -> list[tuple[int, int]]:
    """Nodes (token, parent) below node 0, the last token: up to two chains of
    what followed earlier occurrences of that token."""
    nodes: list[tuple[int, int]] = []
    firsts = set()
    for at in range(len(history) - 2, -1, -1):
        if len(firsts) == 2:
            break
        if history[at] == history[-1] and history[at + 1] not in firsts:
            firsts.add(history[at + 1])
            parent = 0
            for token in history[at + 1:at + 1 + min(depth, room)]:
                nodes.append((token, parent))
                parent = len(nodes)
    return nodes


def generate(model: QuantisedGpt, prompts: list[list[int]], new: int, draft: int = 4, repetition: float = 1.2,
             frequency: float = 0.0, allowed=None) -> tuple[list[list[int]], int]:
    """(new tokens of each prompt, steps taken).  allowed: None or mask words
    [1, ceil(vocab / 32)] of what may be generated at all."""
    limit = model.cfg.context_length
    if any(not p or len(p) + new > limit for p in prompts):
        raise ValueError(f"a prompt has 1 to {limit} - new tokens")
    text = [list(p) for p in prompts]
    done = [0] * len(text)  # tokens of each sequence in the cache

    def run(trees, mask, max_nodes):
        """Logits of the sequences' rows; tree: (token, position, place) each."""
        starts = [0]
        for t in trees:
            starts.append(starts[-1] + len(t))
        rows = [r for t in trees for r in t]
        slots = [s for i, t in enumerate(trees) for s in model.slots(i, [r[2] for r in t])]
        return model.logits([r[0] for r in rows], [r[1] for r in rows], slots, done, starts, mask, max_nodes)

    # all but the prompts' last tokens: rows in causal order
    ahead = [[(t, i, i) for i, t in enumerate(p[:-1])] for p in text]
    if any(ahead):
        run(ahead, None, max(len(t) for t in ahead))
        done = [len(t) for t in ahead]
    steps = 0
    while any(len(t) - len(p) < new for t, p in zip(text, prompts)):
        trees, masks, windows, parents = [], [], [], []
        for t, p, at in zip(text, prompts, done):
            left = new - (len(t) - len(p))
            nodes = [(t[-1], -1)] + (draft_tree(t, draft, left - 1) if left > 1 else [])
            tree, bits, window, depth = [], [], [], []
            for i, (token, parent) in enumerate(nodes):
                depth.append(depth[parent] + 1 if i else 0)
                bits.append((bits[parent] if i else 0) | 1 << i)
                window.append(window[parent] + [token] if i else list(t))
                tree.append((token, at + depth[i], at + i))
            trees.append(tree), masks.extend(bits), windows.extend(window), parents.append([n[1] for n in nodes])
        signed = [b - (1 << 32) if b >> 31 else b for b in masks]
        raw = run(trees, _ints(signed).view(-1, 1), max(len(t) for t in trees))
        ends = [0]
        for w in windows:
            ends.append(ends[-1] + len(w))
        rows = len(windows)
        each = torch.ones(rows, device="cuda")
        controlled = forge.logit_controls(
            raw, tokens=_ints([x for w in windows for x in w]), token_starts=_ints(ends), repetition=each * repetition,
            frequency=each * frequency, allowed=allowed,
            mask_rows=None if allowed is None else torch.zeros(rows, dtype=torch.int32, device="cuda"))
        best = controlled.argmax(dim=1).tolist()
        steps += 1
        row = 0
        for s, tree in enumerate(trees):
            if len(text[s]) - len(prompts[s]) < new:
                path = [0]
                while True:  # down the tree as long as a child is the greedy token
                    token = best[row + path[-1]]
                    text[s].append(token)
                    below = [i for i, parent in enumerate(parents[s]) if parent == path[-1] and tree[i][0] == token]
                    if not below or len(text[s]) - len(prompts[s]) == new:
                        break
                    path.append(below[0])
                if path != list(range(len(path))):
                    model.move(s, [done[s] + i for i in path], [done[s] + i for i in range(len(path))])
                done[s] += len(path)
            row += len(tree)
    return [t[len(p):] for t, p in zip(text, prompts)], steps


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--layers", type=int, default=12)
    ap.add_argument("--d-model", type=int, default=768)
    ap.add_argument("--heads", type=int, default=12)
    ap.add_argument("--vocab", type=int, default=16384)
    ap.add_argument("--context", type=int, default=1024)
    ap.add_argument("--cache", choices=("int8", "int4"), default="int8")
    ap.add_argument("--group", type=int, choices=(32, 64, 128), default=64)
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=64, help="tokens of a prompt")
    ap.add_argument("--new", type=int, default=48, help="tokens to generate")
    ap.add_argument("--draft", type=int, default=4, help="drafted tokens in a chain, at most 7")
    ap.add_argument("--seed", type=int, default=7)
    args = ap.parse_args(argv)
    if not 0 <= args.draft <= 7:
        ap.error("--draft must be 0 to 7")
    cfg = forge.ModelConfig(args.vocab, args.context, args.d_model, args.layers, args.heads)
    model = QuantisedGpt(cfg, forge.init_params(cfg, args.seed), args.seqs, args.cache, args.group)
    gen = torch.Generator().manual_seed(args.seed)
    prompts = torch.randint(0, args.vocab, (args.seqs, args.prompt), generator=gen).tolist()
    out, steps = generate(model, prompts, args.new, args.draft)
    for s, tokens in enumerate(out):
        print(f"{s}: {' '.join(map(str, tokens))}")
    print(f"{args.new} tokens of {args.seqs} sequences in {steps} steps")


if __name__ == "__main__":
    main()

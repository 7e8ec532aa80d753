"""Speculative decoding with one progressive matrix as its own draft: a small decoder, end to end.

Every projection is a progressive int2 matrix.  Its prefix 1 (a quarter of the bytes) drafts a tree
of tokens, its full prefix verifies the whole tree at once, and the path that the full prefix
agrees with is kept.  Around the projections stand the serving operators:

    PagePlan         per step: token positions and tree masks from lengths and parents; after the
                     verification, pages and slots for the tokens that are kept
    LoraSet          each request's own adapter beside the shared query/key/value projection
    TreeAttention    the drafted nodes over the paged cache
    PagedCache       the kept nodes' keys and values, picked out of the step's

Weights are random, so the draft agrees with the verifier only sometimes; what is checked is that
every kept token is the one plain decoding (one token a step, the same full prefix) gives.

    python examples/draft_tree_decode.py [--tokens 24] [--requests 3]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "harp-q_b200"))
import harpq_b200 as hqb  # noqa: E402

HEADS, KV_HEADS, DIM, LAYERS, VOCAB, PAGE = 8, 2, 64, 2, 512, 16
HIDDEN, FULL, DRAFT = HEADS * DIM, 4, 1
BRANCH, DEPTH = 2, 3  # children of a node, levels of a tree


def progressive(rows: int, cols: int, g: torch.Generator) -> "hqb.PlaneMatrix":
    """A random progressive matrix: stage s is 4^-s of the first."""
    codes = [torch.randint(0, 256, (-(-rows // 128) * 128 * -(-cols // 128) * 32,), generator=g, device="cuda",
                           dtype=torch.uint8) for _ in range(FULL)]
    count = -(-rows // 128) * 128 * -(-cols // 128)
    scales = [torch.full((count,), cols ** -0.5 * 4.0 ** -s, device="cuda").half().view(torch.int16) for s in range(FULL)]
    return hqb.PlaneMatrix.from_stages(rows, cols, codes, scales)


class Decoder:
    """Attention layers between an embedding and its transpose; sizes fixed above."""

    def __init__(self, requests: int, capacity: int, seed: int = 0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.requests = requests
        self.embed = torch.randn(VOCAB, HIDDEN, generator=g, device="cuda")
        self.qkv = [progressive((HEADS + 2 * KV_HEADS) * DIM, HIDDEN, g) for _ in range(LAYERS)]
        self.out = [progressive(HIDDEN, HIDDEN, g) for _ in range(LAYERS)]
        self.head = progressive(VOCAB, HIDDEN, g)
        rows, rank = (HEADS + 2 * KV_HEADS) * DIM, 8
        self.lora = [hqb.LoraSet(torch.randn(requests, rank, HIDDEN, generator=g, device="cuda").mul(HIDDEN ** -0.5).half(),
                                 torch.randn(requests, rows, rank, generator=g, device="cuda").mul(0.1).half(), max_tokens=0)
                     for _ in range(LAYERS)]
        pages = requests * -(-capacity // PAGE)
        self.caches = [hqb.PagedCache(*(torch.zeros(pages, PAGE, KV_HEADS, DIM, dtype=torch.float16, device="cuda")
                                        for _ in range(2))) for _ in range(LAYERS)]
        self.nodes = sum(BRANCH ** level for level in range(DEPTH))
        tokens = requests * self.nodes
        # the layers follow one another, so one workspace of each kind serves them all
        scratch: list = []

        def shared(need: int) -> "hqb.Workspace":
            if not scratch or scratch[-1].nbytes < need:
                scratch.append(hqb.Workspace(need, clear=256))
            return scratch[-1]

        self.attend = [hqb.TreeAttention(c, HEADS, requests, tokens, self.nodes, capacity, workspace=shared) for c in self.caches]
        self.lora_scratch = hqb.Workspace(max(s.workspace_bytes(tokens) for s in self.lora), clear=256)
        self.tree = hqb.PagePlan(requests, tokens, PAGE, pages, max_new=self.nodes)
        self.keep = hqb.PagePlan(requests, tokens, PAGE, pages)
        self.tables = torch.full((requests, -(-capacity // PAGE)), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.held = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.taken = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def project(self, m: "hqb.PlaneMatrix", x: torch.Tensor, prefix: int) -> torch.Tensor:
        """Rows of x through a matrix; a decode step's GEMV takes up to 16 at a time."""
        return torch.cat([m.gemv(part, prefix=prefix, flags=hqb.FLAG_F16MMA) for part in x.split(hqb.MAX_BATCH)])

    def forward(self, tokens: torch.Tensor, counts: torch.Tensor, parents: torch.Tensor, prefix: int):
        """Logits [tokens, vocab] and each layer's (k, v) of a step of trees."""
        plan = self.tree.build(self.lengths, counts, parents=parents)
        n = len(tokens)
        angle = plan.positions[:n, None] * torch.logspace(0, -3, HIDDEN // 2, device="cuda")
        hidden = (self.embed[tokens] + torch.cat([angle.sin(), angle.cos()], 1)).half()
        ids, kept = plan.requests[:n].contiguous(), []
        for layer in range(LAYERS):
            y = self.project(self.qkv[layer], hidden, prefix)
            self.lora[layer].apply(hidden, ids, base=y, out=y, workspace=self.lora_scratch)
            q, k, v = (t.view(n, -1, DIM) for t in y.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], 1))
            mixed = self.attend[layer](q, k, v, self.tables, self.lengths, plan.starts, plan.mask)
            mixed = self.project(self.out[layer], mixed.view(n, HIDDEN), prefix)
            hidden = torch.nn.functional.layer_norm(hidden.float() + mixed.float(), (HIDDEN,)).half()
            kept.append((k, v))
        return self.project(self.head, hidden, prefix).float(), kept

    def commit(self, kept, rows: torch.Tensor, counts: torch.Tensor) -> None:
        """Gives the kept tokens (rows of the step, request after request) pages and writes their keys and values."""
        plan = self.keep.build(self.lengths, counts, held=self.held, tables=self.tables, free_pages=self.free,
                               free_head=self.taken)
        slots = plan.slots[:len(rows)].contiguous()
        for cache, (k, v) in zip(self.caches, kept):
            cache.append(k, v, slots, rows=rows)
        self.held, self.taken = plan.held.clone(), plan.free_head.clone()
        self.lengths = self.lengths + counts


def decode_plain(model: Decoder, first: torch.Tensor, steps: int) -> torch.Tensor:
    """[requests, steps + 1] tokens, one a step at the full prefix."""
    tokens, ones = [first], torch.ones_like(model.lengths)
    roots = torch.full_like(model.lengths, -1)
    for _ in range(steps):
        logits, kept = model.forward(tokens[-1], ones, roots, FULL)
        model.commit(kept, torch.arange(len(first), device="cuda", dtype=torch.int32), ones)
        tokens.append(logits.argmax(1))
    return torch.stack(tokens, 1)


def decode_trees(model: Decoder, first: torch.Tensor, steps: int) -> tuple[list[list[int]], int]:
    """At least `steps` more tokens a request, and the verifications that took."""
    requests = len(first)
    done, rounds = [[t] for t in first.tolist()], 0
    while min(map(len, done)) <= steps:
        # ---- draft: levels of the tree at the first prefix, the most likely children of each node
        trees = [[d[-1]] for d in done]
        parents = [[-1] for _ in done]
        level = [[0] for _ in done]
        for _ in range(DEPTH - 1):
            logits, _ = model.forward(torch.tensor(sum(trees, []), device="cuda"),
                                      torch.full((requests,), len(trees[0]), dtype=torch.int32, device="cuda"),
                                      torch.tensor(sum(parents, []), dtype=torch.int32, device="cuda"), DRAFT)
            children = logits.topk(BRANCH, 1).indices.view(requests, -1, BRANCH).tolist()
            for r in range(requests):
                grown = []
                for node in level[r]:
                    for token in children[r][node]:
                        grown.append(len(trees[r]))
                        trees[r].append(token)
                        parents[r].append(node)
                level[r] = grown
        # ---- verify the whole trees at the full prefix, keep the path that it agrees with
        size = len(trees[0])
        logits, kept = model.forward(torch.tensor(sum(trees, []), device="cuda"),
                                     torch.full((requests,), size, dtype=torch.int32, device="cuda"),
                                     torch.tensor(sum(parents, []), dtype=torch.int32, device="cuda"), FULL)
        best = logits.argmax(1).view(requests, size).tolist()
        rows, counts = [], []
        for r in range(requests):
            node, path = 0, [0]
            while True:
                done[r].append(best[r][node])
                child = [i for i in range(size) if parents[r][i] == node and trees[r][i] == best[r][node]]
                if not child:
                    break
                node = child[0]
                path.append(node)
            rows += [r * size + i for i in path]
            counts.append(len(path))
        model.commit(kept, torch.tensor(rows, dtype=torch.int32, device="cuda"),
                     torch.tensor(counts, dtype=torch.int32, device="cuda"))
        rounds += 1
    return done, rounds


def main(requests: int = 3, steps: int = 24, seed: int = 0) -> tuple[bool, float]:
    """Whether both ways of decoding give the same tokens, and the tokens kept a verification."""
    capacity = steps + 2 + sum(BRANCH ** level for level in range(DEPTH))
    first = torch.arange(1, requests + 1, device="cuda") * 7
    plain = decode_plain(Decoder(requests, capacity, seed), first, steps).tolist()
    trees, rounds = decode_trees(Decoder(requests, capacity, seed), first, steps)
    same = all(t[:steps + 1] == p for t, p in zip(trees, plain))
    return same, sum(len(t) - 1 for t in trees) / (rounds * requests)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--requests", type=int, default=3)
    a = ap.parse_args()
    same, rate = main(a.requests, a.tokens)
    print(f"same tokens as plain decoding: {same}; {rate:.2f} tokens a verification")
    sys.exit(0 if same else 1)

"""Speculative decoding within a budget of cached keys, on the device from end to end.

A step verifies a tree of drafted tokens for every sequence in one pass over its cache
(dvattn_tree_sdpa), appends the tokens that the model itself would have chosen
(dvattn_tree_append), adds what attention they paid to the cached keys, their own ones among
them (dvattn_paged_mass), and, once a sequence holds more keys than its budget, lets each KV head
drop its least attended ones (dvattn_paged_evict).  Nothing in a step waits for the host.

The model is a toy, one attention layer with random weights: its logits are those of the draft
(a table by token) plus a projection of the attention output.

    python examples/speculative_decode.py --sequences 32 --steps 200 --budget 1024
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import dvattn_b200  # noqa: E402

# the drafted tree: the token chosen last, its two likeliest successors, theirs
PARENTS = [-1, 0, 0, 1, 1, 2, 2]
DEPTH = [0, 1, 1, 2, 2, 2, 2]
LEVELS = max(DEPTH)


class Toy:
    def __init__(self, Hq, Hkv, E, R, vocab, dtype, device, seed=0):
        g = torch.Generator().manual_seed(seed)
        D = 64

        def weight(*shape):
            return (torch.randn(shape, generator=g) / shape[0] ** 0.5).to(device)

        self.Hq, self.Hkv, self.E, self.R, self.dtype, self.device = Hq, Hkv, E, R, dtype, device
        self.scale = E ** -0.5
        self.emb = torch.randn((vocab, D), generator=g).to(device)
        self.wq, self.wk, self.wv = weight(D, Hq * E), weight(D, Hkv * E), weight(D, Hkv * E)
        self.wo = 8 * weight(Hq * E, vocab)
        self.draft_logits = 4 * torch.randn((vocab, vocab), generator=g).to(device)
        self.successors = self.draft_logits.topk(2, dim=1).indices

    def qkv(self, tokens):
        """tokens [W,S] -> q [W,Hq,S,E], k and v [W,Hkv,S,E]"""
        W, S = tokens.shape
        x = self.emb[tokens]
        return [(x @ w).view(W, S, -1, self.E).transpose(1, 2).to(self.dtype).contiguous() for w in (self.wq, self.wk, self.wv)]

    def choose(self, tokens, out):
        """The model's next token after each of tokens [W,S], with attention output [W,Hq,S,E]."""
        W, S = tokens.shape
        return (self.draft_logits[tokens] + out.float().transpose(1, 2).reshape(W, S, -1) @ self.wo).argmax(-1)

    def angles(self, positions):
        """positions [W,S] -> full-width cos and sin rows [W,S,R]"""
        inv = 10000.0 ** (-torch.arange(0, self.R, 2, device=self.device, dtype=torch.float32) / self.R)
        a = positions[..., None].float() * inv
        return torch.cat([a.cos()] * 2, -1), torch.cat([a.sin()] * 2, -1)


class Decoder:
    """The paged caches of W sequences and one decode step over them."""

    def __init__(self, model, prompt, capacity, block_size=16):
        m, (W, n) = model, prompt.shape
        dev, pages = m.device, -(-capacity // block_size)
        self.model, self.W = m, W
        self.k = torch.zeros((W * pages, block_size, m.Hkv, m.E), dtype=m.dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        self.tables = torch.randperm(W * pages, generator=torch.Generator().manual_seed(1)).to(dev).int().view(W, pages)
        self.turns = torch.tensor([pages * block_size], dtype=torch.int32, device=dev)  # one turn, as long as the table
        self.cached = torch.zeros(W, dtype=torch.int32, device=dev)  # keys in the cache
        self.seen = torch.zeros(W, dtype=torch.int32, device=dev)    # tokens so far: the position of the next
        self.mass = torch.zeros((W, m.Hkv, pages * block_size), device=dev)
        self.parents = torch.tensor(PARENTS, dtype=torch.int32, device=dev).repeat(W, 1)
        self.depth = torch.tensor(DEPTH, dtype=torch.int32, device=dev)
        # the prompt's keys; its last token is the first to be attended from
        _, k, v = m.qkv(prompt[:, :-1])
        cos, sin = m.angles(torch.arange(n - 1, device=dev).repeat(W, 1))
        dvattn_b200.dvattn_paged_append(self.k, self.v, k, v, cos, sin, self.tables, self.cached)
        self.cached += n - 1
        self.seen += n - 1
        self.pending = prompt[:, -1].clone()

    def step(self, budget=None, sink=4, recent=64):
        """One verification: the tokens [W, LEVELS + 1] that each sequence gained (-1: none)."""
        m = self.model
        tokens = torch.empty((self.W, len(PARENTS)), dtype=torch.long, device=m.device)
        tokens[:, 0] = self.pending
        for s in range(1, len(PARENTS)):
            tokens[:, s] = m.successors[tokens[:, PARENTS[s]], (s - 1) % 2]
        q, k, v = m.qkv(tokens)
        cos, sin = m.angles(self.seen[:, None] + self.depth)
        loc = (self.cached - 1)[None, :, None].expand(1, self.W, len(PARENTS)).contiguous()
        lse = torch.empty(q.shape[:3], device=m.device)
        out = dvattn_b200.dvattn_tree_sdpa(q, self.parents, loc, cos[None], sin[None], self.turns, self.k, self.v, self.tables,
                                           k, v, m.scale, lse=lse)
        # from the root on, the child that is the model's own choice
        best = m.choose(tokens, out)
        node = torch.zeros((self.W, 1), dtype=torch.long, device=m.device)
        path, counts = [node], torch.ones(self.W, dtype=torch.int32, device=m.device)
        going = torch.ones((self.W, 1), dtype=torch.bool, device=m.device)
        for _ in range(LEVELS):
            child = (self.parents == node) & (tokens == best.gather(1, node))
            going = going & child.any(1, keepdim=True)
            node = torch.where(going, child.int().argmax(1, keepdim=True), node)
            path.append(node)
            counts += going[:, 0]
        path = torch.cat(path, 1).int()
        dvattn_b200.dvattn_tree_append(self.k, self.v, k, v, cos, sin, self.tables, self.cached, path, counts)
        # only accepted tokens count as queries; their own keys are cached by now, one a level of the tree
        taken = torch.zeros(tokens.shape, dtype=torch.bool, device=m.device).scatter(1, path.long(), True)
        lse.masked_fill_(~taken[:, None], -float("inf"))
        seen = (self.cached[:, None] + self.depth)[None].contiguous()
        dvattn_b200.dvattn_paged_mass(self.mass, q, lse, seen, cos[None], sin[None], self.turns, self.k, self.tables, m.scale)
        self.cached += counts
        self.seen += counts
        gained = torch.where(torch.arange(LEVELS + 1, device=m.device) < counts[:, None], best.gather(1, path.long()), -1)
        self.pending = best.gather(1, node)[:, 0]
        if budget is not None:
            keep = self.cached.clamp(max=budget)
            dvattn_b200.dvattn_paged_evict(self.k, self.v, self.mass, self.tables, torch.zeros_like(keep), self.cached, keep,
                                           sink=sink, recent=recent)
            self.cached = keep
        return gained


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--sequences", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=1500)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--budget", type=int, default=1024)
    a = ap.parse_args()
    model = Toy(Hq=64, Hkv=4, E=128, R=64, vocab=512, dtype=torch.bfloat16, device="cuda:0")
    prompt = torch.randint(0, 512, (a.sequences, a.prompt), generator=torch.Generator().manual_seed(2)).to("cuda:0")
    decoder = Decoder(model, prompt, capacity=max(a.prompt, a.budget) + LEVELS + 1)
    decoder.step(a.budget)  # the prompt is thinned out here
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    gained = torch.stack([decoder.step(a.budget) for _ in range(a.steps)])
    end.record()
    torch.cuda.synchronize()
    n = int((gained >= 0).sum())
    print(f"{n} tokens of {a.sequences} sequences in {a.steps} steps ({n / a.steps / a.sequences:.2f} a step), "
          f"{start.elapsed_time(end) / a.steps:.3f} ms a step, {int(decoder.cached.max())} keys cached for {int(decoder.seen.max())} tokens")


if __name__ == "__main__":
    main()

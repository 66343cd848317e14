"""Generation with a hybrid decoder: gated delta layers, attention over an 8-bit cache, rules on the logits.

A small model of random weights (every fourth layer attends, the others carry a gated delta state) reads prompts
of different lengths in one packed call and then writes a token per sequence and step:

    python examples/hybrid_generate.py --prompts 700 65 1 --tokens 32
"""
from __future__ import annotations

import argparse
import os
import sys
import time
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import decisive_b200 as db  # noqa: E402


@dataclass
class Sizes:
    layers: int = 8
    hidden: int = 512
    k_heads: int = 4   # of a delta layer; 128 wide, like every head here
    v_heads: int = 8
    q_heads: int = 8   # of an attention layer
    kv_heads: int = 2
    vocab: int = 8192

    def attends(self, layer: int) -> bool:
        return layer % 4 == 3


class Hybrid:
    """The model's weights and what its sequences keep: a delta state or a cache per layer, and their lengths."""

    def __init__(self, s: Sizes, sequences: int, max_tokens: int, seed: int = 0, dtype=torch.bfloat16):
        rng = torch.Generator("cuda").manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=rng, device="cuda") * cols ** -0.5).to(dtype)

        self.s, self.sequences = s, sequences
        self.embed, self.layers, self.states = weight(s.vocab, s.hidden), [], []
        width = (max_tokens + db.KvCache8.BLOCK - 1) // db.KvCache8.BLOCK
        for i in range(s.layers):
            if s.attends(i):
                rows, out = (s.q_heads + 2 * s.kv_heads) * 128, s.q_heads * 128
                self.states.append(db.KvCache8.allocate(sequences, sequences * width, width, s.kv_heads, dtype))
            else:
                rows, out = (2 * s.k_heads + s.v_heads) * 128 + 2 * s.v_heads, s.v_heads * 128
                self.states.append(torch.zeros(sequences, s.v_heads, 128, 128, device="cuda"))
            self.layers.append((weight(rows, s.hidden), weight(s.hidden, out)))
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device="cuda")

    def _delta(self, x, state, packed):
        s, h, kv = self.s, self.s.v_heads, (2 * self.s.k_heads + self.s.v_heads) * 128
        q, k, v = x[:, :kv].view(len(x), -1, 128).split([s.k_heads, s.k_heads, h], 1)  # views: no copies are made
        g = -torch.nn.functional.softplus(x[:, kv:kv + h].float())
        beta = torch.sigmoid(x[:, kv + h:].float())
        return db.gated_delta(q, k, v, g, beta, items=self.sequences, state=state, state_out=state, **packed)[0]

    def _attend(self, x, cache, packed, max_keys):
        s = self.s
        q, k, v = x.view(len(x), -1, 128).split([s.q_heads, s.kv_heads, s.kv_heads], 1)
        rows = {"cu_seqlens": packed["cu_seqlens"], "max_rows": packed["max_len"]} if packed else {}
        db.kv8_append(cache, k, v, self.lengths, **rows)
        return db.kv8_attention(cache, q, self.lengths, max_keys=max_keys, **rows)

    def forward(self, tokens, max_keys: int, cu_seqlens=None, max_len: int | None = None):
        """Logits f32 of each sequence's last new token.  tokens: the sequences' new tokens one after another, bounded by
        cu_seqlens; without it one per sequence.  max_keys: the longest sequence's tokens, these among them."""
        packed = {} if cu_seqlens is None else {"cu_seqlens": cu_seqlens, "max_len": max_len}
        x = self.embed[tokens]
        for i, (project, back) in enumerate(self.layers):
            y = torch.nn.functional.rms_norm(x, x.shape[-1:]) @ project.T
            state = self.states[i]
            y = self._attend(y, state, packed, max_keys) if self.s.attends(i) else self._delta(y, state, packed)
            x = x + y.flatten(1) @ back.T
        self.lengths += 1 if cu_seqlens is None else cu_seqlens.diff()
        if cu_seqlens is not None:
            x = x[cu_seqlens[1:].long() - 1]
        return torch.nn.functional.rms_norm(x, x.shape[-1:]).float() @ self.embed.float().T


def generate(model: Hybrid, prompts, tokens: int, mask=None, repetition: float = 1.1, presence: float = 0.2,
             frequency: float = 0.1):
    """Greedy continuation of the prompts (lists of ids) under the rules -> (ids [sequences, tokens] int32, their
    log-probabilities)."""
    n, lengths = len(prompts), [len(p) for p in prompts]
    device = model.embed.device
    most = max(lengths)
    history = torch.zeros(n, most + tokens, dtype=torch.int32, device=device)
    for i, p in enumerate(prompts):
        history[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    filled = torch.tensor(lengths, dtype=torch.int32, device=device)
    cu = torch.zeros(n + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lengths).cumsum(0)
    flat = torch.tensor([t for p in prompts for t in p], device=device)
    rule = {k: torch.full((n,), v, device=device) for k, v in
            (("repetition", repetition), ("presence", presence), ("frequency", frequency))}
    logits = model.forward(flat, most, cu.to(device), most)
    ids, logs = [], []
    for step in range(tokens):
        _, best, lse = db.logit_rules(logits, history, filled, mask=mask, out=logits, **rule)
        ids.append(best)
        logs.append(logits.gather(1, best.long()[:, None])[:, 0] - lse)
        if step + 1 < tokens:
            history.scatter_(1, filled.long()[:, None], best[:, None])
            filled += 1
            logits = model.forward(best, most + step + 1)
    return torch.stack(ids, 1), torch.stack(logs, 1)


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--prompts", type=int, nargs="+", default=[700, 65, 1], help="their lengths, in tokens")
    p.add_argument("--tokens", type=int, default=32)
    a = p.parse_args()
    s, rng = Sizes(), torch.Generator().manual_seed(1)
    prompts = [torch.randint(s.vocab, (n,), generator=rng).tolist() for n in a.prompts]
    # the grammar here: even ids only
    mask = torch.full((len(prompts), s.vocab // 32), 0x55555555, dtype=torch.int32, device="cuda")
    for run in ("first run", "again"):
        model = Hybrid(s, len(prompts), max(a.prompts) + a.tokens)
        torch.cuda.synchronize()
        start = time.perf_counter()
        ids, logs = generate(model, prompts, a.tokens, mask)
        torch.cuda.synchronize()
        ms = (time.perf_counter() - start) * 1e3
        print(f"{run}: {sum(a.prompts)} prompt tokens and {a.tokens} steps of {len(prompts)} sequences in {ms:.1f} ms")
    for i in range(len(prompts)):
        print(f"sequence {i}: {ids[i, :8].tolist()} ... log-probability {logs[i].sum().item():.2f}")


if __name__ == "__main__":
    main()

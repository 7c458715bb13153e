"""A small decoder with a paged cache and MoE layers, as a server would run it:  python examples/decode.py

Random weights.  A prompt goes in at once, three samples fork from it and share its pages, each grows token by token,
a draft of several tokens is checked in one step and its rejected end rolled back, finished sequences free their pages
and the pool is compacted.  Projections, norms of the residual stream and sampling are torch's; cache, attention and
experts are the library's.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from xcalibur_b200 import PagedKVCache, PreparedMoE, Rope  # noqa: E402
from xcalibur_b200.synth import make_weights  # noqa: E402


class Decoder:
    """``layers`` x (attention, MoE) over one ``PagedKVCache``."""

    def __init__(self, *, layers=2, hidden=512, q_heads=8, kv_heads=2, head_dim=64, experts=8, inter=256, top_k=2,
                 vocab=1000, pages=64, page_size=16, max_seqs=8, max_pages=32, window=0, kv_dtype=torch.bfloat16,
                 device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape, std=0.02):
            return (torch.randn(shape, generator=g, device=device) * std).bfloat16()

        self.heads, self.kv_heads, self.head_dim, self.top_k, self.window = q_heads, kv_heads, head_dim, top_k, window
        self.embed = weight(vocab, hidden, std=1.0)
        self.blocks = [dict(qkv=weight((q_heads + 2 * kv_heads) * head_dim, hidden), o=weight(hidden, q_heads * head_dim),
                            q_norm=1 + weight(head_dim), k_norm=1 + weight(head_dim), router=weight(experts, hidden),
                            moe=PreparedMoE(**make_weights(experts, hidden, inter, seed=seed + i, device=device)))
                       for i in range(layers)]
        self.rope = Rope(head_dim, base=1e6, device=device)
        self.cache = PagedKVCache(layers, pages, kv_heads, page_size, head_dim, max_seqs=max_seqs, max_pages=max_pages,
                                  dtype=kv_dtype, device=device)

    def step(self, tokens: torch.Tensor, seqs: torch.Tensor) -> torch.Tensor:
        """Logits [B, L, vocab] of ``tokens`` [B, L], which follow what sequences ``seqs`` (int32 [B]) hold."""
        B, L = tokens.shape
        H, K, D = self.heads, self.kv_heads, self.head_dim
        cache = self.cache
        cache.extend(seqs, torch.full_like(seqs, L))
        first = cache.seq_lens[seqs.long()] - L
        positions = (first[:, None] + torch.arange(L, dtype=torch.int32, device=first.device)).flatten()
        owners = seqs[:, None].expand(B, L).flatten()
        x = self.embed[tokens.flatten()]
        for i, w in enumerate(self.blocks):
            qkv = (_norm(x) @ w["qkv"].T).view(B * L, H + 2 * K, D)
            q, k, v = qkv.split([H, K, K], dim=1)  # strided views: read in place
            q = cache.append(i, q, k, v, positions, owners, self.rope, q_weight=w["q_norm"], k_weight=w["k_norm"])
            a = cache.attend(i, q.view(B, L, H, D), seqs=seqs, window=self.window)
            x = x + a.view(B * L, H * D) @ w["o"].T
            h = _norm(x)
            x = x + w["moe"].forward(h, (h @ w["router"].T).float(), self.top_k)
        return (_norm(x) @ self.embed.T).float().view(B, L, -1)


def _norm(x: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.rms_norm(x, x.shape[-1:])


def ints(*values: int, device="cuda") -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=device)


def main() -> None:
    model = Decoder()
    cache = model.cache
    g = torch.Generator(device="cuda").manual_seed(1)
    prompt = torch.randint(0, 1000, (1, 37), generator=g, device="cuda")
    logits = model.step(prompt, ints(0))[:, -1]

    cache.fork(ints(0, 0), ints(1, 2))  # three samples of one prompt: its full pages are stored once
    seqs = ints(0, 1, 2)
    tokens = torch.multinomial(torch.softmax(logits.expand(3, -1), -1), 1, generator=g)
    for _ in range(20):
        logits = model.step(tokens, seqs)[:, -1]
        tokens = torch.multinomial(torch.softmax(logits, -1), 1, generator=g)
    print("lengths", cache.seq_lens[:3].tolist(), "pages in use", int((cache.refcounts > 0).sum()))

    draft = torch.randint(0, 1000, (3, 3), generator=g, device="cuda")  # a guess of the next three tokens of each
    before = cache.seq_lens[:3].clone()
    best = model.step(torch.cat([tokens, draft], 1), seqs).argmax(-1)
    kept = (best[:, :-1] == draft).long().cumprod(1).sum(1)
    cache.truncate(seqs, (before + 1 + kept).int())
    print("draft tokens kept", kept.tolist(), "lengths", cache.seq_lens[:3].tolist())

    cache.free(ints(0, 1))
    cache.compact()
    held = cache.page_table[2][cache.page_table[2] >= 0]
    print("after free and compact: pages in use", int((cache.refcounts > 0).sum()), "highest id", int(held.max()))
    best = model.step(tokens[2:], ints(2)).argmax(-1)
    print("next token of the last sequence", int(best), "status", cache.check_device_status())


if __name__ == "__main__":
    main()

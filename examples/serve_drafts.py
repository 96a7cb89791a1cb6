"""A serving loop over a paged 4-bit cache: draft, attend, verify, append.

A small random model stands in for a real one: tokens are embedded, a few attention layers add
to the embedding, and a head gives the logits. The drafter is the same model without its
attention (next-token logits from the embedding alone), so that it agrees with the target often
but not always. Every step

  1. drafts `drafts` tokens per request from the drafter,
  2. runs the target over [last token | drafts]: per layer PagedCache.attend, the rows of a draft
     seeing the cache and the drafted tokens before them,
  3. accepts drafts and draws the next token (verify_drafts),
  4. plans the slots of the kept tokens (TokenPlan.build: one plan for all layers, which share
     the page table) and appends their K/V rows to every layer's pool (PagedCache.append).

    python examples/serve_drafts.py --batch 32 --steps 50
"""

from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from maskahead_b200.serving import PagedCache, TokenPlan, verify_drafts  # noqa: E402


@dataclass
class Layer:
    wq: torch.Tensor
    wk: torch.Tensor
    wv: torch.Tensor
    wo: torch.Tensor
    cache: PagedCache


class Server:
    """Requests of a random model, decoded in steps of up to `drafts` + 1 tokens each."""

    def __init__(self, *, batch=8, layers=2, q_heads=28, heads=4, head_dim=128, width=512, vocab=2048, drafts=4,
                 page_size=64, max_len=2048, device="cuda", seed=0):
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.batch, self.drafts, self.vocab, self.heads, self.head_dim, self.q_heads = batch, drafts, vocab, heads, head_dim, q_heads
        self.device = device
        self.embed = self._normal(vocab, width)
        self.head = self._normal(width, vocab) * 0.15
        max_pages = (max_len + page_size - 1) // page_size
        num_pages = batch * max_pages
        self.layers: list[Layer] = []
        tables = None
        for _ in range(layers):
            kchan = torch.full((batch, heads, head_dim), 2.0, device=device)
            cache = PagedCache.allocate(batch=batch, heads=heads, head_dim=head_dim, num_pages=num_pages, page_size=page_size,
                                        max_pages=max_pages, kchan=kchan, device=device)
            if tables is not None:     # every layer reads the same page table and lengths
                cache = PagedCache(kq=cache.kq, ks=cache.ks, kz=cache.kz, vq=cache.vq, vs=cache.vs, vz=cache.vz,
                                   kchan=kchan, pages=tables.pages, lens=tables.lens)
            else:
                tables = cache
            scale = width ** -0.5
            self.layers.append(Layer(self._normal(width, q_heads * head_dim) * scale, self._normal(width, heads * head_dim) * scale,
                                     self._normal(width, heads * head_dim) * scale,
                                     self._normal(q_heads * head_dim, width) * 0.3 * (q_heads * head_dim) ** -0.5, cache))
        self.tables = tables
        self.plan: TokenPlan = tables.plan(max_tokens=batch * (drafts + 1))
        self.last = torch.randint(0, vocab, (batch,), generator=self.gen, device=device, dtype=torch.int32)

    def _normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=self.device).to(torch.bfloat16)

    def _draft(self):
        """(tokens [B, K] int32, the distributions they were drawn from [B, K, V] fp32)."""
        tokens, rows, at = [], [], self.last
        for _ in range(self.drafts):
            q = torch.softmax((self.embed[at.long()] @ self.head).float(), -1)
            at = torch.multinomial(q, 1, generator=self.gen)[:, 0].to(torch.int32)
            tokens.append(at)
            rows.append(q)
        return torch.stack(tokens, 1), torch.stack(rows, 1)

    def step(self):
        """One step; returns (accepted [B], tokens [B, K + 1]) as verify_drafts does."""
        B, T = self.batch, self.drafts + 1
        drafts, q_rows = self._draft()
        x = self.embed[torch.cat([self.last[:, None], drafts], 1).long()]                     # [B, T, width]
        kept = []
        for layer in self.layers:
            q = (x @ layer.wq).view(B, T, self.q_heads, self.head_dim).transpose(1, 2)
            k = (x @ layer.wk).view(B, T, self.heads, self.head_dim)
            v = (x @ layer.wv).view(B, T, self.heads, self.head_dim)
            a = layer.cache.attend(q, k.transpose(1, 2), v.transpose(1, 2))
            x = x + a.transpose(1, 2).reshape(B, T, -1) @ layer.wo
            kept.append((k.reshape(B * T, self.heads, self.head_dim), v.reshape(B * T, self.heads, self.head_dim)))
        target = torch.softmax((x @ self.head).float(), -1)
        uniforms = torch.rand(B, T, generator=self.gen, device=self.device)
        accepted, tokens = verify_drafts(target, q_rows, drafts, None, uniforms)
        # the last token and the accepted drafts stay: their rows go into the cache
        before = self.tables.lens.clone()
        plan = self.plan.build(before + accepted + 1)
        owner = plan.seqs.long().clamp(min=0)
        row = (owner * T + plan.positions.long() - before[owner].long()).clamp(0, B * T - 1)
        for layer, (k, v) in zip(self.layers, kept):
            layer.cache.append(k[row], v[row], plan.slots, plan.seqs)
        self.last = tokens.gather(1, accepted.long()[:, None])[:, 0].contiguous()
        return accepted, tokens


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--steps", type=int, default=20)
    args = ap.parse_args()
    server = Server(batch=args.batch, drafts=args.drafts)
    total = torch.zeros((), device="cuda", dtype=torch.int64)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    server.step()
    start.record()
    for _ in range(args.steps):
        accepted, _ = server.step()
        total += accepted.sum() + args.batch
    end.record()
    torch.cuda.synchronize()
    steps = args.steps * args.batch
    print(f"{args.batch} requests, {args.steps} steps: {total.item() / steps:.2f} tokens a step and request, "
          f"{total.item() / start.elapsed_time(end) * 1e3:.0f} tokens/s, longest {int(server.tables.lens.max())}")


if __name__ == "__main__":
    main()

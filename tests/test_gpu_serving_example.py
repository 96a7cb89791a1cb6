"""The serving operators together, as examples/serve_drafts.py runs them."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu


def test_steps_keep_the_books():
    """Lengths grow by the accepted drafts and one, pages are held once, every kept token's row is
    where the page table says, and the emitted tokens are the drafts up to the first refusal."""
    from serve_drafts import Server

    B, K, steps, page = 5, 3, 6, 16
    server = Server(batch=B, drafts=K, layers=2, page_size=page, max_len=64, vocab=256, seed=3)
    seen = torch.zeros(B, dtype=torch.int64)
    for _ in range(steps):
        accepted, tokens = server.step()
        a, t = accepted.cpu(), tokens.cpu()
        seen += a + 1
        assert server.tables.lens.cpu().tolist() == seen.tolist()
        for b in range(B):
            n = int(a[b])
            assert 0 <= n <= K and (t[b, :n + 1] >= 0).all() and (t[b, n + 1:] == -1).all()
            assert int(server.last[b]) == int(t[b, n])
        lens, table = server.tables.lens.tolist(), server.tables.pages.tolist()
        held = [table[b][j] for b in range(B) for j in range((lens[b] + page - 1) // page)]
        free = server.tables.free.tolist()[:int(server.tables.free_count)]
        assert sorted(held + free) == list(range(server.tables.num_pages))
    # a stored slot has a value scale (an empty one none): exactly the live slots are written
    for layer in server.layers:
        c = layer.cache
        for b in range(B):
            for j in range(lens[b]):
                assert (c.vs[table[b][j // page], :, j % page] > 0).all()
        assert int((c.vs[:, 0, :, 0] > 0).sum()) == sum(lens)


def test_full_pages_refuse_in_order():
    """A pool too small for the batch: requests that do not fit keep their length."""
    from serve_drafts import Server

    server = Server(batch=3, drafts=2, layers=1, page_size=4, max_len=8, vocab=64, seed=1)
    for _ in range(12):
        server.step()
        assert int(server.tables.lens.max()) <= 8

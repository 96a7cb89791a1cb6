"""The serving entry points without a GPU: rejected arguments return before the device is touched."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from maskahead_b200.build import build

    build()
    import maskahead_b200

    return maskahead_b200.load_library()


def test_rejected_arguments(lib):
    from maskahead_b200._lib import MaBlock, MaKV, MaPagePlan, MaRows, i64

    s2, s3 = i64(0, 0), i64(0, 0, 0)
    assert lib.ma_page_plan(MaPagePlan(), None, None, 0, None) == -1
    assert lib.ma_page_plan(None, 16, None, 0, None) == -1
    assert lib.ma_append_tokens(MaKV(), 1, 1, 128, None, None, 1, 1, s2, s2, None, None, None, None, None) == -2     # not packed
    assert lib.ma_append_tokens(None, 1, 1, 128, None, None, 1, 1, s2, s2, None, None, None, None, None) == -1
    assert lib.ma_append_tokens(MaKV(), 1, 1, 96, None, None, 1, 1, s2, s2, None, None, None, None, None) == -2
    assert lib.ma_decode_attention(MaRows(), MaKV(), 1, MaBlock(), 1.0, 1, None, s3, None, 0, None) == -1
    assert lib.ma_verify_drafts(None, None, 0, 1, 1, 8, s2, s2, None, None, None, None, None, None, 0, None) == -1
    # addresses that are never read: the vocabulary and the workspace are looked at first
    assert lib.ma_verify_drafts(16, 16, 0, 1, 1, (1 << 20) + 1, s2, s2, 16, None, 16, 16, 16, None, 0, None) == -2
    assert lib.ma_verify_drafts(16, 16, 0, 1, 1, 8, s2, s2, 16, None, 16, 16, 16, None, 0, None) == -3
    assert lib.ma_verify_drafts(17, 16, 0, 1, 1, 8, s2, s2, 16, None, 16, 16, 16, None, 0, None) == -1


def test_page_plan_struct_matches_the_header(lib):
    """The ctypes mirror's layout: four pointers, five int32 (and padding), two int64, eight pointers."""
    from maskahead_b200._lib import MaPagePlan

    assert ctypes.sizeof(MaPagePlan) == 4 * 8 + 5 * 4 + 4 + 2 * 8 + 8 * 8
    assert MaPagePlan.spg.offset == 56 and MaPagePlan.lens_out.offset == 72


def test_workspace_sizes(lib):
    assert lib.ma_page_plan_workspace() >= 512
    assert lib.ma_decode_attention_workspace(0, 1, 1, 128, 0) == 0
    assert lib.ma_verify_drafts_workspace(0, 10) == 0
    # at most three CTAs an SM with two partials of 32 rows each, or one such CTA per head and row tile
    for h, r, d in ((4, 7, 128), (4, 64, 128), (1, 1, 64), (8, 500, 128)):
        heads = h * ((r + 7) // 8)
        most = max(3 * 256, heads) * 2 * 32 * (4 * d + 8)
        assert 0 < lib.ma_decode_attention_workspace(1, h, r, d, 1) <= (1 << 20) + most
    # a row's partial sums: at most 2048 spans of 8 bytes a request beside the fixed part
    fixed = lib.ma_verify_drafts_workspace(1, 1)
    for b, v in ((1, 1 << 20), (7, 100003), (5000, 50021)):
        assert lib.ma_verify_drafts_workspace(b, v) <= fixed + b * 2048 * 8


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_no_cpu_path():
    from maskahead_b200 import KernelUnavailableError
    from maskahead_b200.serving import TokenPlan, verify_drafts

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(KernelUnavailableError):
        TokenPlan(lens=i32(2), pages=i32(2, 2), free=i32(4), free_count=i32(1), page_size=16, num_pages=4, max_tokens=4)
    with pytest.raises(KernelUnavailableError):
        verify_drafts(torch.zeros(1, 2, 8), None, i32(1, 1), None, torch.zeros(1, 2))

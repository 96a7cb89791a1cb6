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


def _append(pool=None, k=0, n=1, dtype=1, d=128):
    from maskahead_b200._lib import APPEND_ARGS

    return APPEND_ARGS.pack(k, k, k, k, 0, 0, 128, 128, 128, 128, n, dtype, 0 if pool is None else ctypes.addressof(pool), 1, 1, d, 0)


def _verify(target=16, vocab=8, dtype=0, ws=0, nbytes=0):
    from maskahead_b200._lib import VERIFY_HEAD, VERIFY_TAIL

    return VERIFY_HEAD.pack(target, 16, 16, 0, 16, 16, 16, ws, nbytes) + VERIFY_TAIL.pack(0, 0, 0, 0, dtype, 1, 1, vocab)


def test_rejected_arguments(lib):
    from maskahead_b200._lib import DECODE_HEAD, DECODE_TAIL, MaKV, MaPagePlan

    kv = MaKV()
    assert lib.ma_page_plan(MaPagePlan(), None, None, 0, None) == -1
    assert lib.ma_page_plan(None, 16, None, 0, None) == -1
    assert lib.ma_append_tokens(None, None) == -1
    assert lib.ma_append_tokens(_append(), None) == -1
    assert lib.ma_append_tokens(_append(kv), None) == -2              # a dense cache
    assert lib.ma_append_tokens(_append(kv, d=96), None) == -2
    assert lib.ma_append_tokens(_append(kv, dtype=2), None) == -1
    assert lib.ma_decode_attention(None, None) == -1
    assert lib.ma_decode_attention(DECODE_HEAD.pack(0, 0, 0, 0, 0, 0) + DECODE_TAIL.pack(*[0] * 12, ctypes.addressof(kv), *[1] * 8, 1.0, 0),
                                   None) == -1
    # addresses that are never read: sizes, alignment and the workspace are looked at first
    assert lib.ma_verify_drafts(None, None) == -1
    assert lib.ma_verify_drafts(_verify(target=0), None) == -1
    assert lib.ma_verify_drafts(_verify(dtype=7), None) == -1
    assert lib.ma_verify_drafts(_verify(target=17), None) == -1
    assert lib.ma_verify_drafts(_verify(vocab=(1 << 20) + 1), None) == -2
    assert lib.ma_verify_drafts(_verify(), None) == -3
    assert lib.ma_verify_drafts(_verify(ws=4096, nbytes=1000), None) == -3


def test_live_pages_rejects_what_has_no_table(lib):
    from maskahead_b200._lib import MaKV

    assert lib.ma_live_pages(None, 1, 16, 16, None) == -1
    kv = MaKV()
    kv.nq = 32
    assert lib.ma_live_pages(kv, 1, 16, 16, None) == -1               # not paged
    kv.pages, kv.page_size, kv.num_pages = 16, 16, 4
    for b, out, lens in ((0, 16, 16), (1, None, 16), (1, 16, None)):
        assert lib.ma_live_pages(kv, b, out, lens, None) == -1
    kv.nf = 1
    assert lib.ma_live_pages(kv, 1, 16, 16, None) == -1               # a tail behind the table


def test_packed_structs_match_the_header(tmp_path):
    """The packed argument structs have the sizes and offsets that a C compiler gives the header's."""
    import shutil
    import subprocess
    from pathlib import Path

    from maskahead_b200._lib import APPEND_ARGS, DECODE_HEAD, DECODE_TAIL, VERIFY_HEAD, VERIFY_TAIL

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src, exe = tmp_path / "sizes.c", tmp_path / "sizes"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "maskahead_b200.h"\nint main(void) {\n'
                   'printf("%zu %zu %zu %zu %zu %zu %zu", sizeof(ma_append_args), offsetof(ma_append_args, pool), '
                   'sizeof(ma_decode_args), offsetof(ma_decode_args, sq), offsetof(ma_decode_args, scale), '
                   'sizeof(ma_verify_args), offsetof(ma_verify_args, st)); return 0; }\n')
    root = Path(__file__).resolve().parents[1]
    subprocess.run([cc, "-I", str(root / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    head, tail = DECODE_HEAD.size, DECODE_TAIL.size
    assert got == [APPEND_ARGS.size, 88, head + tail, head, head + 12 * 8 + 8 + 8 * 4, VERIFY_HEAD.size + VERIFY_TAIL.size, VERIFY_HEAD.size]


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


def test_workspace_of_the_general_route(lib):
    """It holds an in-place call's part, the split attention's scratch and both unpacked copies."""
    from maskahead_b200.serving import _SPLITK_HEAD, decode_workspace_bytes

    for b, h, r, d, tc, n in ((1, 1, 1, 64, 0, 1), (2, 2, 104, 128, 2, 576), (32, 4, 224, 128, 32, 8192)):
        here, split = lib.ma_decode_attention_workspace(b, h, r, d, tc), lib.ma_prefix_attention_workspace(b, h, r, n, d, tc)
        assert decode_workspace_bytes(b, h, r, d, tc) == here
        assert decode_workspace_bytes(b, h, r, d, tc, capacity=n) >= here + split + 4 * b * h * n * d
    # a call of one row and no key: little but the fixed words at the front
    assert lib.ma_prefix_attention_workspace(1, 1, 1, 0, 128, 0) <= _SPLITK_HEAD


def test_launches_for_another_device_are_refused(monkeypatch):
    """A default stream's handle is 0 on every device: the current device decides where a launch goes."""
    from maskahead_b200 import _lib

    monkeypatch.setattr(_lib, "current_device", lambda: 0)
    monkeypatch.setattr(_lib, "_raw_stream", lambda index: 100 + index)
    assert _lib.stream_handle(torch.device("cuda", 0)) == 100
    with pytest.raises(RuntimeError, match="cuda:1"):
        _lib.stream_handle(torch.device("cuda", 1))


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_no_cpu_path():
    from maskahead_b200 import KernelUnavailableError
    from maskahead_b200.serving import TokenPlan, verify_drafts

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(KernelUnavailableError):
        TokenPlan(lens=i32(2), pages=i32(2, 2), free=i32(4), free_count=i32(1), page_size=16, num_pages=4, max_tokens=4)
    with pytest.raises(KernelUnavailableError):
        verify_drafts(torch.zeros(1, 2, 8), None, i32(1, 1), None, torch.zeros(1, 2))

"""The paged serving operators against plain implementations in 64 bits.

decode attention: float64 softmax over the dequantized cache. The kernel rounds q * kchan to
fp16 (relative 2^-11 per product, so a score is off by at most 2^-11 sum_d |q_d k_d|), p and
p * scale to fp16 (2^-11 each), and the output to bf16 (8 significant bits: 2^-8). With d_j the score's bound that
gives, per element and before any run,
    sum_j p_j (d_j + dbar) |v_j - o| + 2^-10 sum_j p_j (|c s| + |z|) + 2^-8 |o|
(dbar = sum_j p_j d_j), the derivative of a softmax average times the perturbations; `_attend_ref`
returns it beside the values, with a factor 1.25 for the second order and the fp32 sums. The
rounding errors are independent, so the error's 2-norm stays far below: bf16's own is at most
2^-9 / sqrt(3) = 1.13e-3 of an element plus at most as much again: 3e-3 of the norm.

page plans, appends and verification give whole numbers (or exactly defined roundings): equal.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


# ------------------------------------------------------------------------- attention
def _packed_rows(x):
    """[..., D] float -> codes, payload, fp16 scale and zero per 32 channels (any 4-bit code is
    as good as another here: the reference dequantizes what is stored)."""
    g = x.unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).clamp_min(1e-8)
    c = ((g - lo) / s).round().clamp(0, 15).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), s.squeeze(-1).to(torch.float16), lo.squeeze(-1).to(torch.float16)


def _cache_tensors(B, H, D, lens, page, seed, vscale=1.0, fill_nan=True):
    """A shuffled pool holding lens[b] slots per request; unused positions hold NaN parameters."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    P = sum(need) + 2
    order = torch.randperm(P, generator=g).tolist()
    width = max(max(need), 1)
    pages = torch.full((B, width), -1, dtype=torch.int32)
    G = D // 32
    pool = {n: torch.full((P, H, page, G), float("nan") if fill_nan else 0.0, dtype=torch.float16)
            for n in ("ks", "kz", "vs", "vz")}
    pool.update({n: torch.full((P, H, page, G, 16), 0x5A, dtype=torch.uint8) for n in ("kq", "vq")})
    at = 0
    for b in range(B):
        k = torch.randn(H, lens[b], D, generator=g)
        k[:, :, torch.randperm(D, generator=g)[:2]] *= 4.0
        v = torch.randn(H, lens[b], D, generator=g) * vscale
        pk, sk, zk = _packed_rows(k)
        pv, sv, zv = _packed_rows(v)
        for i in range(need[b]):
            pg = order[at]
            at += 1
            pages[b, i] = pg
            lo, hi = i * page, min(lens[b], (i + 1) * page)
            for name, t in (("kq", pk), ("ks", sk), ("kz", zk), ("vq", pv), ("vs", sv), ("vz", zv)):
                pool[name][pg, :, :hi - lo] = t[:, lo:hi]
    kchan = 0.5 + 1.5 * torch.rand(B, H, D, generator=g)
    return pool, pages, torch.tensor(lens, dtype=torch.int32), kchan


def _make(B, H, D, lens, page, seed, **kw):
    from maskahead_b200.serving import PagedCache

    pool, pages, ln, kchan = _cache_tensors(B, H, D, lens, page, seed, **kw)
    return PagedCache(**{k: t.to(DEV) for k, t in pool.items()}, kchan=kchan.to(DEV), pages=pages.to(DEV), lens=ln.to(DEV))


def _inputs(B, Hq, H, T, D, Tc, seed):
    g = torch.Generator().manual_seed(seed + 999)
    q = torch.randn(B, Hq, T, D, generator=g).to(torch.bfloat16).to(DEV)
    kc = torch.randn(B, H, Tc, D, generator=g).to(torch.bfloat16).to(DEV) if Tc else None
    vc = torch.randn(B, H, Tc, D, generator=g).to(torch.bfloat16).to(DEV) if Tc else None
    return q, kc, vc


def _dequant(payload, s, z):
    c = torch.stack([payload & 15, payload >> 4], -1).flatten(-2).double()
    return (c * s.double()[..., None]).flatten(-2), z.double()[..., None].expand(*z.shape, 32).flatten(-2)


def _slots(prefix, b, h):
    """(k, code part of v, zero part of v, live) of request b, head h in float64."""
    n = prefix.nq
    lens = n if prefix.lens is None else min(int(prefix.lens[b]), n)
    j = torch.arange(n, device=DEV)
    live = j < lens
    if prefix.pages is not None:
        pg = prefix.pages[b].long()[j // prefix.page_size]
        live &= (pg >= 0) & (pg < prefix.kq.shape[0])
        pg, pos = pg.clamp(0, prefix.kq.shape[0] - 1), j % prefix.page_size
    else:
        pg, pos = torch.full_like(j, b), j
    if prefix.mask is not None:
        live &= prefix.mask[b, h].bool()
    pg, pos = pg[live], pos[live]
    kc, kz = _dequant(prefix.kq[pg, h, pos], prefix.ks[pg, h, pos], prefix.kz[pg, h, pos])
    vc, vz = _dequant(prefix.vq[pg, h, pos], prefix.vs[pg, h, pos], prefix.vz[pg, h, pos])
    return (kc + kz) * prefix.kch[b, h].double(), vc, vz


def _attend_ref(q, prefix, kc, vc, scaling=None, causal=True):
    B, Hq, T, D = q.shape
    H = prefix.vq.shape[1]
    G = Hq // H
    scale = D ** -0.5 if scaling is None else scaling
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    for b in range(B):
        for h in range(H):
            k, cv, zv = _slots(prefix, b, h)
            n = k.shape[0]
            if kc is not None:
                k = torch.cat([k, kc[b, h].double()])
                cv = torch.cat([cv, vc[b, h].double()])
                zv = torch.cat([zv, torch.zeros_like(vc[b, h].double())])
            tc = k.shape[0] - n
            v = cv + zv
            for t in range(T):
                seen = torch.ones(k.shape[0], dtype=torch.bool, device=DEV)
                if tc and causal:
                    seen[n:] = torch.arange(tc, device=DEV) <= t + tc - T
                if not bool(seen.any()):
                    continue
                for g in range(G):
                    x = q[b, h * G + g, t].double()
                    s = (k[seen] @ x) * scale
                    p = torch.softmax(s, 0)
                    o = p @ v[seen]
                    d = (k[seen].abs() @ x.abs()) * abs(scale) * 2.0 ** -11
                    w = p * (d + (p * d).sum())
                    e = (w[:, None] * (v[seen] - o).abs()).sum(0)
                    e += 2.0 ** -10 * (p @ (cv[seen].abs() + zv[seen].abs()))
                    out[b, h * G + g, t] = o
                    tol[b, h * G + g, t] = 1.25 * e + 2.0 ** -8 * o.abs() + 1e-6
    return out, tol


def _close(got, ref, tol):
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    worst = (err / tol.clamp_min(1e-30)).max().item()
    assert worst <= 1.0, f"error {worst} times its bound"
    norm = ref.norm().item()
    if norm > 0 and ref.numel() >= 1024:
        assert err.norm().item() <= 3e-3 * norm, f"2-norm error {err.norm().item() / norm}"


SHAPES = [
    # B, Hq, H, D, T, lens, page
    (1, 28, 4, 128, 1, [1], 64),
    (1, 28, 4, 128, 1, [4097], 64),
    (3, 8, 8, 128, 1, [31, 32, 33], 16),
    (4, 7, 1, 128, 1, [127, 128, 129, 0], 48),
    (2, 16, 2, 128, 1, [1000, 5], 100),
    (2, 9, 1, 128, 1, [700, 257], 5),
    (2, 16, 1, 128, 1, [640, 63], 64),
    (2, 17, 1, 128, 1, [300, 511], 64),
    (2, 28, 4, 128, 5, [600, 1025], 64),
    (1, 28, 4, 128, 8, [2000], 64),
    (1, 64, 1, 128, 1, [333], 32),
    (5, 32, 8, 64, 3, [1, 47, 48, 49, 961], 48),
    (2, 8, 8, 64, 1, [130, 2049], 64),
    (1, 12, 1, 64, 4, [515], 7),
    (40, 4, 2, 128, 1, [(i * 37) % 300 for i in range(40)], 16),
]


@pytest.mark.parametrize("B,Hq,H,D,T,lens,page", SHAPES)
@pytest.mark.parametrize("block", [True, False])
def test_decode_attention_matches_float64(B, Hq, H, D, T, lens, page, block):
    cache = _make(B, H, D, lens, page, seed=B * 100 + Hq)
    q, kc, vc = _inputs(B, Hq, H, T, D, T if block else 0, seed=Hq)
    out = cache.attend(q, kc, vc)
    ref, tol = _attend_ref(q, cache.prefix(), kc, vc)
    _close(out, ref, tol)
    assert torch.equal(out, cache.attend(q, kc, vc)), "two runs differ"


@pytest.mark.parametrize("Tc,T,causal", [(1, 1, False), (4, 2, True), (40, 3, True), (70, 2, False), (33, 33, True)])
def test_decode_attention_blocks(Tc, T, causal):
    cache = _make(2, 2, 128, [70, 0], 32, seed=5)
    q, kc, vc = _inputs(2, 2, 2, T, 128, Tc, seed=Tc)
    out = cache.attend(q, kc, vc, causal=causal)
    ref, tol = _attend_ref(q, cache.prefix(), kc, vc, causal=causal)
    _close(out, ref, tol)


@pytest.mark.parametrize("D,G,T,Tc", [(128, 7, 2, 2), (128, 3, 5, 40), (64, 8, 4, 4), (128, 1, 1, 1)])
def test_block_keys_a_row_does_not_see(D, G, T, Tc):
    """Later keys of the block may hold anything, NaN included."""
    cache = _make(2, 2, D, [70, 0], 32, seed=40)
    q, kc, vc = _inputs(2, 2 * G, 2, T, D, Tc, seed=41)
    for t in range(T):
        k, v = kc.clone(), vc.clone()
        k[:, :, t + Tc - T + 1:], v[:, :, t + Tc - T + 1:] = float("nan"), float("nan")
        out = cache.attend(q, k, v)
        ref, tol = _attend_ref(q[:, :, :t + 1], cache.prefix(), kc[:, :, :t + Tc - T + 1], vc[:, :, :t + Tc - T + 1])
        _close(out[:, :, :t + 1], ref, tol)


def test_rows_without_a_key_are_zero():
    cache = _make(3, 2, 128, [0, 5, 0], 16, seed=6)
    q, _, _ = _inputs(3, 14, 2, 1, 128, 0, seed=6)
    out = cache.attend(q)
    assert torch.count_nonzero(out[0]) == 0 and torch.count_nonzero(out[2]) == 0
    ref, tol = _attend_ref(q, cache.prefix(), None, None)
    _close(out, ref, tol)


@pytest.mark.parametrize("paged", [True, False])
def test_masks(paged):
    """Masked slots hold NaN parameters; one head has no live slot, one a single one."""
    from maskahead_b200.layouts import Prefix
    from maskahead_b200.serving import decode_attention

    B, Hq, H, D, n = 2, 6, 3, 128, 333
    g = torch.Generator().manual_seed(8)
    if paged:
        pre = _make(B, H, D, [n, n - 40], 64, seed=8).prefix()
    else:
        pk, sk, zk = _packed_rows(torch.randn(B, H, n, D, generator=g))
        pv, sv, zv = _packed_rows(torch.randn(B, H, n, D, generator=g))
        pre = Prefix(kq=pk.to(DEV), ks=sk.to(DEV), kz=zk.to(DEV), vq=pv.to(DEV), vs=sv.to(DEV), vz=zv.to(DEV), nq=n,
                     kb=4, vb=4, kmode=1, kch=(0.5 + torch.rand(B, H, D, generator=g)).to(DEV))
    mask = (torch.rand(B, H, pre.nq, generator=g) < 0.5)
    mask[0, 1] = False
    mask[1, 2] = False
    mask[1, 2, 77] = True
    pre.mask = mask.to(DEV)
    if not paged:       # poison what is masked
        dead = ~pre.mask.bool()
        for t in (pre.ks, pre.kz, pre.vs, pre.vz):
            t[dead] = float("nan")
    q, kc, vc = _inputs(B, Hq, H, 2, D, 2, seed=9)
    for args in ((None, None), (kc, vc)):
        out = decode_attention(q, pre, *args)
        ref, tol = _attend_ref(q, pre, *args)
        _close(out, ref, tol)
        if args[0] is None:
            assert torch.count_nonzero(out[0, 2:4]) == 0


@pytest.mark.parametrize("B,Hq,H,D,T", [(2, 14, 2, 128, 3), (400, 3, 1, 64, 1)])
def test_a_cache_without_slots_needs_no_arrays(B, Hq, H, D, T):
    """nq = 0 and null pointers, as the other C entries take an empty cache: the block's keys alone.
    (Both launch forms: few sequences, and more of them than SMs.)"""
    import ctypes

    from maskahead_b200._lib import DECODE_HEAD, DECODE_TAIL, MA_BF16, MA_KV_PACKED_TOKEN, MaKV, lib
    from maskahead_b200.serving import decode_workspace_bytes

    q, kc, vc = _inputs(B, Hq, H, T, D, T, seed=61)
    kv = MaKV()
    kv.layout, kv.dtype = MA_KV_PACKED_TOKEN, MA_BF16
    out = torch.empty_like(q)
    ws = torch.zeros(decode_workspace_bytes(B, H, Hq // H * T, D, T), dtype=torch.uint8, device=DEV)
    rc = lib().ma_decode_attention(
        DECODE_HEAD.pack(q.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel())
        + DECODE_TAIL.pack(*q.stride()[:3], *kc.stride()[:3], *vc.stride()[:3], *out.stride()[:3], ctypes.addressof(kv),
                           MA_BF16, B, Hq, H, T, D, T, 1, D ** -0.5, 0), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    # the same requests in a cache whose lengths are 0
    assert torch.equal(out, _make(B, H, D, [0] * B, 32, seed=62).attend(q, kc, vc))


def test_bad_pages_read_as_dead():
    cache = _make(2, 2, 128, [200, 200], 32, seed=10)
    cache.pages[0, 1] = -1
    cache.pages[1, 0] = cache.num_pages
    cache.pages[1, 3] = 2 ** 30
    q, kc, vc = _inputs(2, 14, 2, 1, 128, 1, seed=10)
    ref, tol = _attend_ref(q, cache.prefix(), kc, vc)
    _close(cache.attend(q, kc, vc), ref, tol)


@pytest.mark.parametrize("vscale", [1e-6, 1e-3, 50.0, 4000.0])
def test_value_ranges(vscale):
    """Value scales from fp16's subnormals to its top, growing along the sequence."""
    B, H, D, n = 1, 2, 128, 700
    cache = _make(B, H, D, [n], 64, seed=11, vscale=vscale)
    ramp = torch.linspace(0.01, 1.0, cache.page_size, device=DEV)
    for t in (cache.vs, cache.vz):
        t.copy_((t.float() * ramp[None, None, :, None]).to(torch.float16))
    q, _, _ = _inputs(B, 14, H, 1, D, 0, seed=12)
    ref, tol = _attend_ref(q, cache.prefix(), None, None)
    _close(cache.attend(q), ref, tol)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("small,large", [(1e-4, 1e3), (1e-2, 1e4), (1e-3, 1e-1)])
@pytest.mark.parametrize("late", [False, True])
def test_value_groups_of_different_sizes(D, small, large, late):
    """A channel group of large values (from the start, or from the middle on) leaves the others exact to
    the same relative bounds."""
    n = 600
    cache = _make(1, 1, D, [n], 64, seed=93)
    g = torch.Generator().manual_seed(94)
    v = torch.randn(1, n, D, generator=g) * small
    v[:, n // 2 if late else 0:, 32:64] *= large / small
    pv, sv, zv = _packed_rows(v)
    for i, page in enumerate(cache.pages[0].tolist()):
        lo, hi = i * 64, min(n, i * 64 + 64)
        for t, x in ((cache.vq, pv), (cache.vs, sv), (cache.vz, zv)):
            t[page, :, :hi - lo] = x[:, lo:hi].to(DEV)
    q, _, _ = _inputs(1, 16, 1, 1, D, 0, seed=95)
    ref, tol = _attend_ref(q, cache.prefix(), None, None)
    out = cache.attend(q)
    _close(out, ref, tol)
    for first in range(0, D, 32):
        part = slice(first, first + 32)
        assert (out[..., part].double() - ref[..., part]).norm() <= 3e-3 * ref[..., part].norm()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("ratio", [10.0, 100.0, 1000.0])
def test_query_and_key_groups_of_opposite_sizes(D, ratio):
    """Channels whose queries are as much smaller as their keys (with large zeros) are larger give their
    whole part of a score."""
    n = 600
    cache = _make(1, 1, D, [n], 64, seed=96)
    g = torch.Generator().manual_seed(97)
    size = torch.full((D,), 1 / ratio)
    size[32:64] = ratio
    pk, sk, zk = _packed_rows((torch.randn(1, n, D, generator=g) + 2) * size)
    for i, page in enumerate(cache.pages[0].tolist()):
        lo, hi = i * 64, min(n, i * 64 + 64)
        for t, x in ((cache.kq, pk), (cache.ks, sk), (cache.kz, zk)):
            t[page, :, :hi - lo] = x[:, lo:hi].to(DEV)
    cache.kchan.fill_(1.0)
    q, _, _ = _inputs(1, 16, 1, 1, D, 0, seed=98)
    q = (q.float() / size.to(DEV)).to(torch.bfloat16)
    ref, tol = _attend_ref(q, cache.prefix(), None, None)
    _close(cache.attend(q), ref, tol)


def test_zero_value_scales():
    """A group of equal values has scale 1e-8, which fp16 rounds to 0."""
    cache = _make(1, 1, 128, [100], 16, seed=13)
    cache.vs.zero_()
    cache.ks.zero_()
    cache.kz.zero_()
    cache.vz.nan_to_num_(0.0)
    q, _, _ = _inputs(1, 3, 1, 1, 128, 0, seed=13)
    ref, tol = _attend_ref(q, cache.prefix(), None, None)
    _close(cache.attend(q), ref, tol)


@pytest.mark.parametrize("scaling", [0.0, 1e-3, 1.0, -0.5])
def test_peaked_and_flat_scores(scaling):
    """From a flat softmax to one whose mass is a single key; the running maximum moves."""
    cache = _make(2, 2, 128, [1500, 777], 64, seed=14)
    q, kc, vc = _inputs(2, 14, 2, 2, 128, 2, seed=14)
    ref, tol = _attend_ref(q, cache.prefix(), kc, vc, scaling=scaling)
    _close(cache.attend(q, kc, vc, scaling=scaling), ref, tol)


def test_scaling_is_read_anew_each_call():
    """A scale (or the causal switch) given as a tensor that is written between the calls."""
    cache = _make(2, 2, 128, [120, 45], 64, seed=81)
    q, kc, vc = _inputs(2, 8, 2, 2, 128, 2, seed=82)
    scale, causal = torch.tensor(0.1), torch.tensor(True)
    for s, c in ((0.1, True), (0.02, True), (0.02, False), (1, 1)):
        scale.fill_(s)
        causal.fill_(c)
        assert torch.equal(cache.attend(q, kc, vc, scaling=scale, causal=causal),
                           cache.attend(q, kc, vc, scaling=float(scale), causal=bool(c)))
    assert torch.equal(cache.attend(q, kc, vc, scaling=1), cache.attend(q, kc, vc, scaling=1.0))


def test_query_magnitudes_per_row():
    """Rows from 2^-60 to 2^30: each is scaled by its own power of two (q'.k stays finite)."""
    cache = _make(1, 1, 128, [300], 64, seed=15)
    q, _, _ = _inputs(1, 8, 1, 1, 128, 0, seed=15)
    q = q * (2.0 ** torch.tensor([-60, -30, -10, 0, 1, 2, -3, 0.0], device=DEV))[None, :, None, None].to(torch.bfloat16)
    q[0, 7] = 0
    ref, tol = _attend_ref(q, cache.prefix(), None, None)
    _close(cache.attend(q), ref, tol)


def test_strides_and_out():
    cache = _make(2, 2, 128, [90, 140], 64, seed=16)
    base, kc, vc = _inputs(2, 6, 2, 3, 128, 3, seed=16)
    want = cache.attend(base, kc, vc)
    q = base.transpose(1, 2).contiguous().transpose(1, 2)             # [B, T, Hq, D] storage
    k2 = kc.transpose(1, 2).contiguous().transpose(1, 2)
    buf = torch.full((2, 3, 6, 256), float("nan"), device=DEV, dtype=torch.bfloat16)
    out = buf[..., :128].transpose(1, 2)
    got = cache.attend(q, k2, vc, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    assert torch.isnan(buf[..., 128:]).all()
    # a query whose rows are not 16-byte aligned is copied
    odd = torch.empty(2, 6, 3, 129, device=DEV, dtype=torch.bfloat16)[..., 1:]
    odd.copy_(base)
    assert torch.equal(cache.attend(odd, kc, vc), want)


def test_out_axes_of_length_one_have_any_stride():
    """One request's rows inside a padded buffer: aligned rows, whatever the stride of the axes of length one."""
    cache = _make(1, 2, 128, [90], 64, seed=83)
    q, kc, vc = _inputs(1, 6, 2, 1, 128, 1, seed=84)
    want = cache.attend(q, kc, vc)
    buf = torch.full((6 * 128 + 1,), float("nan"), device=DEV, dtype=torch.bfloat16)
    out = buf.as_strided((1, 6, 1, 128), (769, 128, 7, 1))
    got = cache.attend(q, kc, vc, out=out)
    assert got is out and torch.equal(out, want) and torch.isnan(buf[-1])


def test_tensors_are_written_into_not_replaced():
    """The calls keep the tensors' addresses: a new tensor in their place would not be read."""
    cache = _make(1, 1, 64, [10], 16, seed=60)
    plan = cache.plan(max_tokens=4) if cache.free is not None else None
    for name in ("kq", "lens", "pages", "kchan"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name).clone())
    q, _, _ = _inputs(1, 1, 1, 1, 64, 0, seed=60)
    before = cache.attend(q)
    cache.lens.fill_(3)
    assert not torch.equal(cache.attend(q), before)
    if plan is not None:
        with pytest.raises(AttributeError):
            plan.slots = plan.slots.clone()


def test_sliced_pool():
    """A layer's slice of a stacked pool: the page stride is not the page's size."""
    from maskahead_b200.serving import PagedCache

    pool, pages, lens, kchan = _cache_tensors(2, 2, 128, [150, 65], 64, seed=17)
    stacked = {k: torch.stack([torch.zeros_like(t), t], 1).to(DEV) for k, t in pool.items()}       # [P, layers, H, ...]
    a = PagedCache(**{k: t[:, 1] for k, t in stacked.items()}, kchan=kchan.to(DEV), pages=pages.to(DEV), lens=lens.to(DEV))
    b = PagedCache(**{k: t.to(DEV) for k, t in pool.items()}, kchan=kchan.to(DEV), pages=pages.to(DEV), lens=lens.to(DEV))
    q, kc, vc = _inputs(2, 14, 2, 1, 128, 1, seed=17)
    assert torch.equal(a.attend(q, kc, vc), b.attend(q, kc, vc))


def test_offsets_past_32_bits():
    """Pages whose payload lies more than 2^31 bytes into the pool."""
    from maskahead_b200.serving import PagedCache

    P, page = 70000, 512
    small, _, lens, kchan = _cache_tensors(1, 1, 128, [1300], page, seed=18)
    q8 = torch.zeros(P, 1, page, 4, 16, device=DEV, dtype=torch.uint8)
    sc = torch.zeros(P, 1, page, 4, device=DEV, dtype=torch.float16)
    far = [P - 1, P - 3, 2]
    pages = torch.tensor([far], dtype=torch.int32, device=DEV)
    near = PagedCache(**{k: t.to(DEV) for k, t in small.items()}, kchan=kchan.to(DEV),
                      pages=torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV), lens=lens.to(DEV))
    for i, pg in enumerate(far):
        q8[pg], sc[pg] = near.kq[i], near.ks[i]
    far_cache = PagedCache(kq=q8, ks=sc, kz=sc, vq=q8, vs=sc, vz=sc, kchan=kchan.to(DEV), pages=pages, lens=lens.to(DEV))
    same = PagedCache(kq=near.kq, ks=near.ks, kz=near.ks, vq=near.kq, vs=near.ks, vz=near.ks, kchan=kchan.to(DEV),
                      pages=near.pages, lens=lens.to(DEV))
    same.ks.nan_to_num_(0.0)
    sc.nan_to_num_(0.0)
    q, kc, vc = _inputs(1, 7, 1, 1, 128, 1, seed=18)
    assert torch.equal(far_cache.attend(q, kc, vc), same.attend(q, kc, vc))
    # and the append writes there
    g = torch.Generator().manual_seed(1)
    k = torch.randn(2, 1, 128, generator=g).to(torch.bfloat16).to(DEV)
    slots = torch.tensor([(P - 1) * page + 500, (P - 5) * page + 3], device=DEV)
    seqs = torch.zeros(2, dtype=torch.int32, device=DEV)
    far_cache.vq = far_cache.kq
    before = int(q8[P - 5].sum())
    far_cache.append(k, k, slots, seqs)
    assert int(q8[P - 5].sum()) != before and int(q8[P - 5, 0, 3].sum()) > 0


@pytest.mark.parametrize("kind", ["dense", "channel", "tail", "rows", "float32"])
def test_other_prefixes_take_the_general_route(kind):
    """What is not read in place runs as splitk_attention (K and V rounded to bf16: 2e-2)."""
    from maskahead_b200.layouts import Prefix, pack_prefix
    from maskahead_b200.serving import decode_attention

    B, H, D, n, T = 2, 2, 128, 160, 2
    Hq = 100 if kind == "rows" else 8
    g = torch.Generator().manual_seed(20)
    k = torch.randn(B, H, n, D, generator=g).to(torch.bfloat16).to(DEV)
    v = torch.randn(B, H, n, D, generator=g).to(torch.bfloat16).to(DEV)
    q, kc, vc = _inputs(B, Hq, H, T, D, T, seed=21)
    if kind == "dense":
        pre = Prefix.dense(k, v)
    elif kind == "float32":
        q, kc, vc, pre = q.float(), kc.float(), vc.float(), Prefix.dense(k.float(), v.float())
    else:
        m = 128 if kind == "tail" else n
        pre = pack_prefix(k[:, :, :m].contiguous(), v[:, :, :m].contiguous(), key_mode="channel" if kind == "channel" else "token")
        if kind == "tail":
            pre.kf, pre.vf, pre.nf = k[:, :, m:].contiguous(), v[:, :, m:].contiguous(), n - m
    out = torch.empty_like(q)
    got = decode_attention(q, pre, kc, vc, out=out)
    assert got.data_ptr() == out.data_ptr()
    G = Hq // H
    kk, vv = torch.cat([k, kc], 2).double().cpu(), torch.cat([v, vc], 2).double().cpu()
    ref = torch.empty(B, Hq, T, D, dtype=torch.float64)
    for t in range(T):
        s = torch.einsum("bhgd,bhnd->bhgn", q[:, :, t].double().cpu().view(B, H, G, D), kk[:, :, :n + t + 1]) * D ** -0.5
        ref[:, :, t] = torch.einsum("bhgn,bhnd->bhgd", torch.softmax(s, -1), vv[:, :, :n + t + 1]).reshape(B, Hq, D)
    # 4-bit storage is off by half a step of about 5/15 per element of k and v: compare loosely
    limit = 2e-2 if kind in ("dense", "float32") else 0.2
    assert (got.double().cpu() - ref).norm() / ref.norm() < limit


@pytest.mark.parametrize("D,page", [(128, 64), (128, 16), (64, 48)])
@pytest.mark.parametrize("kind", ["plain", "no lens", "mask", "tail"])
def test_bad_pages_read_as_dead_on_the_general_route(kind, D, page):
    """More rows than are read in place: page numbers outside the pool stay dead in the unpacked copy too."""
    from maskahead_b200.serving import decode_attention

    B, H, T = 4, 2, 2
    lens = [300, 223, 0, 1500]
    cache = _make(B, H, D, lens, page, seed=89)
    pre = cache.prefix()
    cache.pages[0, 2] = -1
    cache.pages[0, (lens[0] - 1) // page] = cache.num_pages            # the last, partial page
    cache.pages[1, 0] = 2 ** 30
    cache.pages[3, 5:23:3] = -7
    q, kc, vc = _inputs(B, 104, H, T, D, T, seed=90)
    if kind == "no lens":                                             # every slot of the table
        pre.lens = None
        cache.ks.nan_to_num_(0.0), cache.kz.nan_to_num_(0.0), cache.vs.nan_to_num_(0.0), cache.vz.nan_to_num_(0.0)
    if kind == "mask":
        g = torch.Generator().manual_seed(91)
        pre.mask = (torch.rand(B, H, pre.nq, generator=g) < 0.7).to(DEV)
    if kind == "tail":                                                # bf16 rows behind the paged part: full tables
        pre.lens, m = None, 33
        cache.ks.nan_to_num_(0.0), cache.kz.nan_to_num_(0.0), cache.vs.nan_to_num_(0.0), cache.vz.nan_to_num_(0.0)
        tk, tv = _inputs(B, H, H, 1, D, m, seed=92)[1:]
        ref, _ = _attend_ref(q, pre, torch.cat([tk, kc], 2), torch.cat([tv, vc], 2))
        pre.kf, pre.vf, pre.nf = tk, tv, m
    else:
        ref, _ = _attend_ref(q, pre, kc, vc)
    out = decode_attention(q, pre, kc, vc)
    assert torch.isfinite(out).all()
    assert (out.double() - ref).norm() <= 2e-2 * ref.norm()           # as test_many_rows
    if kind == "plain":
        assert torch.equal(cache.attend(q, kc, vc), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_general_route_copies_rows_off_a_boundary(dtype):
    """Contiguous tensors that start between 16-byte boundaries, or whose axes of length one have odd strides."""
    from maskahead_b200.kernels import splitk_attention

    cache = _make(1, 2, 128, [90], 32, seed=87)
    q, kc, vc = (x.to(dtype) for x in _inputs(1, 104, 2, 1, 128, 1, seed=88))
    want = cache.attend(q, kc, vc)
    pre = cache.prefix()
    whole, _ = splitk_attention(q, pre, kc, vc)

    def shifted(x):
        return torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape)

    def strided(x):
        return x.clone().as_strided(x.shape, (x.stride(0) + 1, 128, 1, 1))

    for form in (shifted, strided):
        assert form(q).is_contiguous() and torch.equal(form(q), q)
        assert torch.equal(cache.attend(form(q), form(kc), form(vc)), want)
        assert torch.equal(splitk_attention(form(q), pre, form(kc), form(vc))[0], whole)


def test_a_cache_takes_the_general_route_too():
    """float32 queries, and more rows than are read in place, over a paged cache."""
    cache = _make(2, 2, 128, [200, 90], 32, seed=30)
    for hq, t, dtype in ((8, 2, torch.float32), (80, 2, torch.bfloat16)):
        q, kc, vc = _inputs(2, hq, 2, t, 128, t, seed=31)
        ref, _ = _attend_ref(q, cache.prefix(), kc, vc)
        out = cache.attend(q.to(dtype), kc.to(dtype), vc.to(dtype))
        assert out.dtype == dtype
        # k and v rounded to bf16 on this route: 2^-8 of each, as test_packed_fa's 2e-2
        assert (out.double() - ref).norm() <= 2e-2 * ref.norm()


@pytest.mark.parametrize("Hq,H,T,D,lens,page", [(12, 1, 8, 128, [300, 0, 5000], 64), (13, 1, 5, 64, [1, 700], 48),
                                                (56, 4, 6, 128, [2500] * 9, 64), (52, 1, 2, 128, [260, 90], 32)])
def test_many_rows(Hq, H, T, D, lens, page):
    """65 to 96 rows a KV head in place, 104 through the unpacked prefix (k and v rounded to bf16 there)."""
    from maskahead_b200.serving import MAX_DECODE_ROWS

    B = len(lens)
    cache = _make(B, H, D, lens, page, seed=50)
    q, kc, vc = _inputs(B, Hq, H, T, D, T, seed=51)
    out = cache.attend(q, kc, vc)
    ref, tol = _attend_ref(q, cache.prefix(), kc, vc)
    if Hq // H * T <= MAX_DECODE_ROWS:
        _close(out, ref, tol)
    else:
        assert (out.double() - ref).norm() <= 2e-2 * ref.norm()


@pytest.mark.parametrize("Hq,H,T,lens,page", [(13, 1, 8, [300, 0, 5000], 64), (56, 4, 8, [2500] * 3, 64), (104, 2, 2, [260, 90], 32)])
def test_general_route_scratch_past_the_lengths(Hq, H, T, lens, page):
    """What an earlier call left in the unpacked copy behind the lengths, NaN included, is not read."""
    from maskahead_b200 import _lib

    B = len(lens)
    cache = _make(B, H, 128, lens, page, seed=63)
    q, kc, vc = _inputs(B, Hq, H, T, 128, T, seed=64)
    cache.attend(q, kc, vc)
    for purpose in ("unpack_k", "unpack_v"):
        _lib.workspace(q.device, purpose, 1).fill_(0xFF)          # bf16 NaN
    out = cache.attend(q, kc, vc)
    ref, _ = _attend_ref(q, cache.prefix(), kc, vc)
    assert torch.isfinite(out).all()
    assert (out.double() - ref).norm() <= 2e-2 * ref.norm()       # as test_many_rows


@pytest.mark.parametrize("Hq,T", [(28, 1), (28, 32), (8, 32)])
def test_dense_ragged_caches_hold_anything_past_the_lengths(Hq, T):
    from maskahead_b200.layouts import Prefix
    from maskahead_b200.serving import decode_attention

    B, H, n, D = 3, 4, 700, 128
    g = torch.Generator().manual_seed(65)
    k = torch.randn(B, H, n, D, generator=g).to(torch.bfloat16).to(DEV)
    v = torch.randn(B, H, n, D, generator=g).to(torch.bfloat16).to(DEV)
    q, kc, vc = _inputs(B, Hq, H, T, D, T, seed=66)
    lens = torch.tensor([238, 17, 697], dtype=torch.int32, device=DEV)
    outs = []
    for rest in (0.0, float("nan"), float("inf")):
        for b in range(B):
            k[b, :, int(lens[b]):] = rest
            v[b, :, int(lens[b]):] = rest
        pre = Prefix.dense(k, v)
        pre.lens = lens
        outs.append(decode_attention(q, pre, kc, vc))
    assert torch.isfinite(outs[0]).all()
    assert torch.equal(outs[1], outs[0]) and torch.equal(outs[2], outs[0])


def test_a_capture_needs_the_workspace_first(monkeypatch):
    import maskahead_b200.serving as serving

    cache = _make(1, 1, 64, [10], 16, seed=32)
    q, _, _ = _inputs(1, 1, 1, 1, 64, 0, seed=32)
    monkeypatch.setattr(serving, "_SHARED", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError):
        cache.attend(q)


def test_streams_graphs_and_own_workspace():
    from maskahead_b200.serving import decode_workspace_bytes

    cache = _make(3, 4, 128, [400, 1200, 30], 64, seed=22)
    q, kc, vc = _inputs(3, 28, 4, 1, 128, 1, seed=22)
    want = cache.attend(q, kc, vc)
    ws = torch.zeros(decode_workspace_bytes(3, 4, 7, 128, 1), dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cache.attend(q, kc, vc, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(q)
    with torch.cuda.graph(graph):
        cache.attend(q, kc, vc, out=out)
    cache.lens[1] = 333                     # the lengths are read on the device
    graph.replay()
    graph.replay()
    assert torch.equal(out, cache.attend(q, kc, vc))
    assert not torch.equal(out, want)


@pytest.mark.parametrize("kind", ["rows", "float32", "channel"])
def test_general_route_stays_in_its_own_workspace(kind):
    """With a workspace given, the route through splitk_attention touches no shared scratch, so calls on
    two streams do not meet; too small a workspace is refused."""
    from maskahead_b200 import _lib
    from maskahead_b200.layouts import pack_prefix
    from maskahead_b200.serving import decode_attention, decode_workspace_bytes

    B, H, D, T, n = 2, 2, 128, 2, 576
    Hq = 104 if kind == "rows" else 8
    dtype = torch.float32 if kind == "float32" else torch.bfloat16
    sources, inputs = [], []
    for seed in (70, 71):
        if kind == "channel":
            g = torch.Generator().manual_seed(seed)
            k, v = (torch.randn(B, H, n, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
            sources.append(pack_prefix(k, v, key_mode="channel"))
        else:
            sources.append(_make(B, H, D, [n, 90], 32, seed=seed))
        inputs.append([x.to(dtype) for x in _inputs(B, Hq, H, T, D, T, seed=seed)])
    want = [decode_attention(q, s, k, v) for s, (q, k, v) in zip(sources, inputs)]
    shared = [b for (_, _, purpose), b in _lib._WORKSPACES.items() if purpose in ("attention", "unpack_k", "unpack_v", "decode")]
    assert shared
    nbytes = decode_workspace_bytes(B, H, Hq // H * T, D, T, capacity=n)
    room = [torch.zeros(nbytes + 8, dtype=torch.uint8, device=DEV)[i:nbytes + i] for i in (0, 3)]       # any alignment
    before = [b.clone() for b in shared]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                q, k, v = inputs[i]
                got[i].append(decode_attention(q, sources[i], k, v, workspace=room[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    assert all(torch.equal(a, b) for a, b in zip(shared, before))
    with pytest.raises(ValueError):
        q, k, v = inputs[0]
        decode_attention(q, sources[0], k, v, workspace=room[0][:1 << 16])


def test_one_workspace_serves_both_routes():
    from maskahead_b200.serving import decode_workspace_bytes

    cache = _make(2, 2, 128, [576, 90], 32, seed=72)
    few, many = _inputs(2, 14, 2, 2, 128, 2, seed=73), _inputs(2, 104, 2, 2, 128, 2, seed=74)
    want = [cache.attend(*few), cache.attend(*many)]
    nbytes = max(decode_workspace_bytes(2, 2, r, 128, 2, capacity=576) for r in (14, 104))
    ws = torch.zeros(nbytes, dtype=torch.uint8, device=DEV)
    for _ in range(3):
        assert torch.equal(cache.attend(*few, workspace=ws), want[0])
        assert torch.equal(cache.attend(*many, workspace=ws), want[1])


def test_calls_make_the_tensors_device_current(monkeypatch):
    """With another device current every call enters the tensors' own (the query of the current device
    stands in for a second GPU); the operators that do not enter it refuse."""
    from maskahead_b200 import _lib
    from maskahead_b200.kernels import splitk_attention
    from maskahead_b200.layouts import Prefix
    from maskahead_b200.serving import PagedCache, decode_attention, verify_drafts

    def calls():
        cache = PagedCache.allocate(batch=2, heads=2, head_dim=64, num_pages=4, page_size=32, max_pages=2,
                                    kchan=torch.ones(2, 2, 64, device=DEV))
        q, k, v = _inputs(2, 4, 2, 2, 64, 2, seed=75)
        plan = cache.plan(64)
        yield lambda: plan.build(torch.tensor([20, 33], dtype=torch.int32, device=DEV)).slots
        rows = torch.randn(64, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
        yield lambda: cache.append(rows, rows, plan.slots, plan.seqs, return_rows=True)[0]
        yield lambda: cache.attend(q, k, v)
        yield lambda: decode_attention(q, cache, k, v)
        yield lambda: decode_attention(q, Prefix.dense(k, v), k, v)
        yield lambda: verify_drafts(*_verify_inputs(2, 2, 50, torch.float32, seed=1))[1]

    want = [f().clone() for f in calls()]
    now, entered = [7], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)
            self.before, now[0] = now[0], self.index

        def __exit__(self, *exc):
            now[0] = self.before

    with monkeypatch.context() as m:
        m.setattr(_lib, "current_device", lambda: now[0])
        m.setattr(torch.cuda, "device", Device)
        got = [f().clone() for f in calls()]
        assert entered == [0] * len(want) and now == [7]
        q, k, v = _inputs(2, 4, 2, 2, 64, 2, seed=75)
        with pytest.raises(RuntimeError):
            splitk_attention(q, Prefix.dense(k, v), k, v)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_keys_of_another_rank_are_refused(dtype):
    cache = _make(2, 2, 128, [50, 60], 16, seed=85)
    q, kc, vc = (x.to(dtype) for x in _inputs(2, 4, 2, 2, 128, 2, seed=86))
    for bad in (lambda x: x[0, 0], lambda x: x[0], lambda x: x[None]):
        with pytest.raises(ValueError):
            cache.attend(q, bad(kc), bad(vc))


def test_attention_refusals():
    import ctypes

    from maskahead_b200 import KernelUnavailableError
    from maskahead_b200._lib import DECODE_HEAD, DECODE_TAIL, lib
    from maskahead_b200.serving import PagedCache, decode_attention

    cache = _make(2, 2, 128, [50, 60], 16, seed=23)
    q, kc, vc = _inputs(2, 4, 2, 2, 128, 2, seed=23)
    with pytest.raises(ValueError):
        cache.attend(q[0])
    with pytest.raises(ValueError):
        cache.attend(q[:1])
    with pytest.raises(ValueError):
        cache.attend(q[:, :3])
    with pytest.raises(ValueError):
        cache.attend(q[..., :64])
    with pytest.raises(ValueError):
        cache.attend(q, kc[:, :, :1], vc[:, :, :1])             # causal rows without their own key
    with pytest.raises(ValueError):
        cache.attend(q, kc, vc[:, :1])
    with pytest.raises(ValueError):
        cache.attend(q, kc, vc, out=torch.empty_like(q, dtype=torch.float32))
    with pytest.raises(ValueError):
        cache.attend(q, kc, vc, workspace=torch.zeros(1024, dtype=torch.uint8, device=DEV))
    with pytest.raises(KernelUnavailableError):
        cache.attend(q.cpu(), None, None)
    with pytest.raises(ValueError):
        PagedCache(kq=cache.kq, ks=cache.ks[:, :1], kz=cache.kz, vq=cache.vq, vs=cache.vs, vz=cache.vz,
                   kchan=cache.kchan, pages=cache.pages, lens=cache.lens)
    with pytest.raises(ValueError):
        PagedCache(kq=cache.kq, ks=cache.ks, kz=cache.kz, vq=cache.vq, vs=cache.vs, vz=cache.vz, kchan=cache.kchan,
                   pages=cache.pages.long(), lens=cache.lens)
    with pytest.raises(ValueError):
        decode_attention(q, type("Empty", (), {"nq": 0, "kf": None, "nf": 0})())
    # the C entry itself
    L, o = lib(), torch.empty_like(q)

    def call(dtype=1, heads=2, tc=0, ptr=q.data_ptr(), ws=0, nbytes=0):
        st = q.stride()[:3]
        return L.ma_decode_attention(
            DECODE_HEAD.pack(ptr, 0, 0, o.data_ptr(), ws, nbytes)
            + DECODE_TAIL.pack(*st, *st, *st, *st, ctypes.addressof(cache._desc.kv), dtype, 2, 4, heads, 2, 128, tc, 1, 1.0, 0), None)

    assert call() == -3 and call(heads=3) == -1 and call(dtype=0) == -2 and call(tc=2) == -1 and call(ptr=q.data_ptr() + 2) == -1
    assert L.ma_decode_attention(None, None) == -1
    assert L.ma_decode_attention_workspace(0, 1, 1, 128, 0) == 0


# ------------------------------------------------------------------------- page plans
def _plan_ref(lens, new, pages, free, count, page, pool, most):
    B, width = len(lens), len(pages[0])
    up = lambda n: (n + page - 1) // page  # noqa: E731
    want = [max(n, 0) for n in new]
    want = [lens[b] if up(want[b]) > width else want[b] for b in range(B)]
    stack = list(free[:count])
    for b in range(B):
        for j in range(up(want[b]), up(lens[b])):
            stack.append(pages[b][j])
    out = [list(p) for p in pages]
    tokens, used, ok = [], 0, True
    starts = [0]
    for b in range(B):
        if want[b] > lens[b]:
            need, grow = up(want[b]) - up(lens[b]), want[b] - lens[b]
            if ok and need <= len(stack) and used + grow <= most:
                for j in range(up(lens[b]), up(want[b])):
                    out[b][j] = stack.pop()
                for x in range(lens[b], want[b]):
                    pg = out[b][x // page]
                    tokens.append((pg * page + x % page if 0 <= pg < pool else -1, b, x))
                used += grow
            else:
                ok = False
                want[b] = lens[b]
        starts.append(used)
    left = len(stack)
    free_out = list(free)
    for i in range(count, left):
        free_out[i] = stack[i]
    pad = most - len(tokens)
    return (want, out, free_out, left, starts, [t[0] for t in tokens] + [-1] * pad, [t[1] for t in tokens] + [-1] * pad,
            [t[2] for t in tokens] + [-1] * pad)


def _plan_state(B, width, page, lens, spare, seed):
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    P = sum(need) + spare
    order = torch.randperm(max(P, 1), generator=g).tolist()
    pages = [[-1] * width for _ in range(B)]
    at = 0
    for b in range(B):
        for j in range(need[b]):
            pages[b][j] = order[at]
            at += 1
    free = order[at:P] + [-7] * at
    return pages, free[:P], P - at, P


def _run_plan(lens, new, pages, free, count, page, pool, most, in_place):
    from maskahead_b200.serving import TokenPlan

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    plan = TokenPlan(lens=i32(lens), pages=i32(pages), free=i32(free), free_count=i32([count]), page_size=page,
                     num_pages=pool, max_tokens=most, in_place=in_place)
    plan.build(i32(new))
    return plan, (plan.lens.tolist(), plan.pages.tolist(), plan.free.tolist(), int(plan.free_count), plan.starts.tolist(),
                  plan.slots.tolist(), plan.seqs.tolist(), plan.positions.tolist())


PLANS = [
    # B, width, page, spare pages, max_tokens, seed, kind
    (1, 4, 16, 3, 5, 0, "grow"),
    (1, 1, 1, 0, 1, 1, "shrink"),
    (7, 9, 5, 20, 40, 2, "mixed"),
    (33, 12, 48, 50, 3000, 3, "mixed"),
    (64, 20, 64, 10, 4001, 4, "mixed"),        # too few pages
    (64, 20, 64, 200, 77, 5, "mixed"),         # too small a slot map
    (257, 6, 16, 300, 9000, 6, "mixed"),
    (520, 4, 7, 900, 8191, 7, "mixed"),        # more requests than a scan's threads
    (1100, 3, 16, 100, 600, 8, "mixed"),
    (12, 8, 16, 60, 0, 9, "mixed"),            # no room for any token: only shrinking
    (300, 40, 64, 13000, 300000, 10, "prompts"),
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("B,width,page,spare,most,seed,kind", PLANS)
def test_page_plan(B, width, page, spare, most, seed, kind, in_place):
    r = np.random.RandomState(seed)
    cap = width * page
    if kind == "grow":
        lens, new = [3], [8]
    elif kind == "shrink":
        lens, new = [1], [0]
    elif kind == "prompts":
        lens = [0] * B
        new = r.randint(0, cap + 1, B).tolist()
    else:
        lens = r.randint(0, cap + 1, B).tolist()
        new = [max(0, x) for x in (np.array(lens) + r.randint(-2 * page, 2 * page, B)).tolist()]
        for b in range(0, B, 5):
            new[b] = [0, lens[b], -3, cap + 1 + b, lens[b] + 1][b // 5 % 5]
    pages, free, count, pool = _plan_state(B, width, page, lens, spare, seed)
    want = _plan_ref(lens, new, pages, free, count, page, pool, most)
    _, got = _run_plan(lens, new, pages, free, count, page, pool, most, in_place)
    for name, a, b in zip(("lens", "pages", "free", "count", "starts", "slots", "seqs", "positions"), got, want):
        assert a == b, f"{name} differs"


def test_page_plan_keeps_pages_apart():
    """Steps of growing, ending and trimmed requests: no page is held twice or lost."""
    from maskahead_b200.serving import PagedCache

    B, width, page, P = 9, 6, 16, 31
    cache = PagedCache.allocate(batch=B, heads=1, head_dim=64, num_pages=P, page_size=page, max_pages=width,
                                kchan=torch.ones(B, 1, 64, device=DEV))
    plan = cache.plan(200)
    r = np.random.RandomState(3)
    for _ in range(60):
        new = (cache.lens.cpu().numpy() + r.randint(-30, 40, B)).clip(0, width * page)
        plan.build(torch.tensor(new, dtype=torch.int32, device=DEV))
        lens, table = cache.lens.tolist(), cache.pages.tolist()
        held = [table[b][j] for b in range(B) for j in range((lens[b] + page - 1) // page)]
        free = cache.free.tolist()[:int(cache.free_count)]
        assert sorted(held + free) == list(range(P))
        slots = [s for s in plan.slots.tolist() if s >= 0]
        assert len(set(slots)) == len(slots) == plan.starts.tolist()[-1]


def test_page_plan_inconsistent_state_stays_in_bounds():
    """Lengths past the table, a free count past the pool and bad page numbers are clamped."""
    _, got = _run_plan([1000, 40], [2000, 41], [[5, 99], [1, -4]], [3, 2, 0, 0], 9, 16, 4, 8, True)
    assert got[0] == [32, 32] and got[5] == [-1] * 8    # a table of two pages holds 32 tokens
    _, got = _run_plan([20, 20], [21, 21], [[0, 99], [1, -4]], [3, 2, 0, 0], 2, 16, 4, 8, True)
    assert got[0] == [21, 21] and got[5] == [-1] * 8 and got[6] == [0, 1] + [-1] * 6


def test_page_plan_many_requests_and_refusals():
    from maskahead_b200._lib import MaError
    from maskahead_b200.serving import TokenPlan

    B = 8192
    lens, new = [0] * B, [1] * B
    pages, free, count, pool = _plan_state(B, 1, 16, lens, B, 1)
    want = _plan_ref(lens, new, pages, free, count, 16, pool, B)
    _, got = _run_plan(lens, new, pages, free, count, 16, pool, B, True)
    assert got == want
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    good = dict(lens=i32(4), pages=i32(4, 2), free=i32(8), free_count=i32(1), page_size=16, num_pages=8, max_tokens=4)
    for bad in (dict(lens=i32(3)), dict(lens=i32(4).long()), dict(free=i32(7)), dict(page_size=0), dict(max_tokens=-1),
                dict(pages=i32(4, 4)[:, ::2]), dict(free_count=i32(2))):
        with pytest.raises(ValueError):
            TokenPlan(**{**good, **bad})
    plan = TokenPlan(**good)
    with pytest.raises(ValueError):
        plan.build(i32(5))
    with pytest.raises(ValueError):
        plan.build(i32(4).long())
    many = TokenPlan(**{**good, "lens": i32(8193), "pages": i32(8193, 1)})
    with pytest.raises(MaError):
        many.build(i32(8193))


def test_page_plan_around_the_default_shared_memory_limit():
    """Request counts whose arrays end just below 48 KB, the kernel's static bytes above it, in a process
    that has planned nothing larger."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from maskahead_b200.serving import TokenPlan
i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
for B in (2446, 2447, 2452, 2457, 2458):
    plan = TokenPlan(lens=i32(B), pages=i32(B, 1), free=torch.arange(B, dtype=torch.int32, device="cuda"),
                     free_count=i32(1) + B, page_size=16, num_pages=B, max_tokens=B)
    plan.build(i32(B) + 1)
    assert plan.lens.eq(1).all() and int(plan.free_count) == 0 and plan.seqs.tolist() == list(range(B))
    assert sorted(plan.slots.tolist()) == [16 * p for p in range(B)]
"""
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# ------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,H,D,page", [(1, 1, 128, 16), (5, 3, 64, 7), (33, 4, 128, 64), (300, 2, 128, 48), (4097, 1, 64, 32)])
def test_append_stores_what_the_quantizer_gives(N, H, D, page, dtype):
    from maskahead_b200.layouts import quantize_tokens
    from maskahead_b200.serving import PagedCache

    g = torch.Generator().manual_seed(N)
    B = 3
    P = (N + N // 4) // page + 2
    kchan = 0.3 + 2 * torch.rand(B, H, D, generator=g)
    cache = PagedCache.allocate(batch=B, heads=H, head_dim=D, num_pages=P, page_size=page, max_pages=P, kchan=kchan.to(DEV))
    for t in (cache.kq, cache.vq):
        t.fill_(0xAB)
    k = torch.randn(N, H, D, generator=g).to(dtype).to(DEV)
    v = (torch.randn(N, H, D, generator=g) * 3 + 1).to(dtype).to(DEV)
    v[0, 0, :32] = 2.0                                   # a group of equal values
    slots = torch.randperm(P * page, generator=g)[:N].to(DEV)
    seqs = torch.randint(0, B, (N,), generator=g).to(torch.int32).to(DEV)
    skip = [(i, w) for i, w in enumerate(["slot", "slot", "seq", "seq"]) if N > 8]
    for i, w in skip:
        if w == "slot":
            slots[i] = [-1, P * page][i]
        else:
            seqs[i] = [-1, B][i - 2]
    before = [t.clone() for t in (cache.kq, cache.ks, cache.kz, cache.vq, cache.vs, cache.vz)]
    rows_k, rows_v = cache.append(k, v, slots, seqs, return_rows=True)
    owned = (seqs >= 0) & (seqs < B)
    kc = cache.kchan[seqs.clamp(0, B - 1).long()]                                     # [N, H, D]
    # a token a sequence of its own: [N, H, 1, D] rows with their divisors
    kq, ks, kz = quantize_tokens(k[:, :, None].contiguous(), kc.contiguous())
    vq, vs, vz = quantize_tokens(v[:, :, None].contiguous())
    want = before
    for i in range(N):
        s = int(slots[i])
        if not bool(owned[i]) or not 0 <= s < P * page:
            continue
        for t, x in zip(want, (kq, ks, kz, vq, vs, vz)):
            t[s // page, :, s % page] = x[i, :, 0]
    for t, x in zip((cache.kq, cache.ks, cache.kz, cache.vq, cache.vs, cache.vz), want):
        assert torch.equal(t, x)
    for rows, (q, s, z), mult in ((rows_k, (kq, ks, kz), kc), (rows_v, (vq, vs, vz), None)):
        c, zz = _dequant(q[:, :, 0], s[:, :, 0], z[:, :, 0])
        ref = (c + zz) * (1.0 if mult is None else mult.double())
        ref = torch.where(owned[:, None, None], ref, torch.zeros_like(ref))
        # one fp32 fma, for keys one fp32 product, one rounding to the type
        eps = (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22)
        assert ((rows.double() - ref).abs() <= eps * ref.abs() + 2.0 ** -22 * (c.abs() + zz.abs()) * 4).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_extreme_rows(dtype):
    """Non-finite, huge, tiny, equal and signed-zero rows, and divisors of every size, give the
    quantizer's bytes: the short cuts for bf16 rows hold or step aside."""
    from maskahead_b200.layouts import quantize_tokens
    from maskahead_b200.serving import PagedCache

    H, D = 2, 128
    g = torch.Generator().manual_seed(12)
    rows = [torch.randn(H, D, generator=g) * s for s in (1e-40, 1e-30, 1e-9, 1e-4, 1.0, 300.0, 1e10, 1e30, 3e38)]
    mixed = torch.randn(H, D, generator=g)
    for value, where in ((float("nan"), 3), (float("inf"), 40), (float("-inf"), 70), (1e38, 100)):
        x = mixed.clone()
        x[:, where] = value
        rows.append(x)
    both = mixed.clone()
    both[:, 5], both[:, 6] = float("inf"), float("-inf")
    zeros = torch.zeros(H, D)
    zeros[:, ::2] = -0.0
    steps = torch.arange(D).float().expand(H, D) % 16                     # codes that fall on whole numbers
    halves = (torch.arange(D).float().expand(H, D) % 31) * 0.5            # and between them
    rows += [both, zeros, torch.full((H, D), float("nan")), torch.full((H, D), 7.0), steps, halves, -steps, halves * 3e-3]
    x = torch.stack(rows).to(dtype).to(DEV)
    n = x.shape[0]
    divisors = [1.0, 2.0, 3.0, 1e-20, 1e20, 1e-35, 1e35, 0.0, 1.9999999]
    for d in divisors:
        kchan = torch.full((1, H, D), d, device=DEV)
        if d == 3.0:
            kchan += torch.rand(1, H, D, generator=g).to(DEV)
        cache = PagedCache.allocate(batch=1, heads=H, head_dim=D, num_pages=2, page_size=32, max_pages=2, kchan=kchan)
        cache.append(x, x, torch.arange(n, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV))
        kc = kchan.expand(n, H, D).contiguous()
        want_k, want_v = quantize_tokens(x[:, :, None].contiguous(), kc), quantize_tokens(x[:, :, None].contiguous())
        for got, want in zip((cache.kq, cache.ks, cache.kz, cache.vq, cache.vs, cache.vz), want_k + want_v):
            a, b = got[0, :, :n].transpose(0, 1), want[:, :, 0]
            same = (a.view(torch.int16) == b.view(torch.int16)) if a.dtype == torch.float16 else a == b
            assert same.all(), f"divisor {d}: rows {sorted(set(torch.nonzero(~same)[:, 0].tolist()))}"


def test_append_32_bit_rows_between_codes():
    """Elements a few units in the last place from the middle between two codes get the quantizer's."""
    from maskahead_b200.layouts import quantize_tokens
    from maskahead_b200.serving import PagedCache

    H, D, N = 2, 128, 4096
    g = torch.Generator().manual_seed(21)
    low, step = torch.randn(N, H, 4, 1, generator=g), 10.0 ** (3 * torch.rand(N, H, 4, 1, generator=g) - 2)
    x = low + step * (torch.randint(0, 15, (N, H, 4, 32), generator=g) + 0.5)
    x = x * (1 + torch.randint(-3, 4, x.shape, generator=g) * 2.0 ** -23)
    x[..., 0], x[..., 1] = low[..., 0], (low + 15 * step)[..., 0]
    x = x.reshape(N, H, D).to(DEV)
    cache = PagedCache.allocate(batch=1, heads=H, head_dim=D, num_pages=N // 64, page_size=64, max_pages=N // 64,
                                kchan=torch.ones(1, H, D, device=DEV))
    cache.append(x, x, torch.arange(N, device=DEV), torch.zeros(N, dtype=torch.int32, device=DEV))
    want = quantize_tokens(x[:, :, None].contiguous())
    for got in ((cache.kq, cache.ks, cache.kz), (cache.vq, cache.vs, cache.vz)):
        for a, b in zip(got, want):
            assert torch.equal(a.transpose(1, 2).reshape(b[:, :, 0].shape), b[:, :, 0])


def test_append_strides_empty_and_refusals():
    from maskahead_b200.serving import PagedCache

    g = torch.Generator().manual_seed(2)
    H, D, N = 2, 128, 6
    make = lambda: PagedCache.allocate(batch=1, heads=H, head_dim=D, num_pages=2, page_size=16, max_pages=2,  # noqa: E731
                                       kchan=torch.full((1, H, D), 1.5, device=DEV))
    k = torch.randn(N, H, D, generator=g).to(torch.bfloat16).to(DEV)
    slots, seqs = torch.arange(N, device=DEV) * 3, torch.zeros(N, dtype=torch.int32, device=DEV)
    a, b, c = make(), make(), make()
    a.append(k, k, slots, seqs)
    swapped = k.transpose(0, 1).contiguous().transpose(0, 1)
    b.append(swapped, swapped, slots, seqs)
    odd = torch.empty(N, H, D + 1, device=DEV, dtype=torch.bfloat16)[..., 1:]
    odd.copy_(k)
    c.append(odd, k, slots, seqs)
    for x in (b, c):
        assert torch.equal(a.kq, x.kq) and torch.equal(a.vq, x.vq) and torch.equal(a.ks, x.ks) and torch.equal(a.vz, x.vz)
    a.append(k[:0], k[:0], slots[:0], seqs[:0])
    for bad in ((k[:, :1], k[:, :1], slots, seqs), (k, k.float(), slots, seqs), (k, k, slots[:3], seqs),
                (k, k, slots.int(), seqs), (k, k, slots, seqs.long()), (k.half(), k.half(), slots, seqs)):
        with pytest.raises(ValueError):
            a.append(*bad)


@pytest.mark.parametrize("H,n", [(4, 1), (1, 3), (1, 1)])
def test_append_axes_of_length_one_have_any_stride(H, n):
    """A single token cut from a padded buffer, and the rows of a single head: contiguous, whatever the
    stride of the axis of length one."""
    from maskahead_b200.serving import PagedCache

    D = 128
    g = torch.Generator().manual_seed(80)
    make = lambda: PagedCache.allocate(batch=1, heads=H, head_dim=D, num_pages=1, page_size=16, max_pages=1,  # noqa: E731
                                       kchan=torch.full((1, H, D), 1.5, device=DEV))
    if H > 1:
        k = torch.randn(2, H * D + 1, generator=g).to(torch.bfloat16).to(DEV)[:, :H * D].unflatten(1, (H, D))[:n]
    else:
        k = torch.randn(n, D, generator=g).to(torch.bfloat16).to(DEV).as_strided((n, 1, D), (D, 7, 1))
    assert k.is_contiguous() and any(s % 8 for s in k.stride()[:2])
    slots, seqs = torch.arange(n, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    a, b = make(), make()
    rows = a.append(k, k, slots, seqs, return_rows=True)
    want = b.append(k.clone(memory_format=torch.contiguous_format), k.clone(memory_format=torch.contiguous_format), slots, seqs,
                    return_rows=True)
    assert torch.equal(a.kq, b.kq) and torch.equal(a.vz, b.vz) and torch.equal(rows[0], want[0]) and torch.equal(rows[1], want[1])


def test_appended_tokens_are_attended():
    """Plan, append and attend agree on where a token lies."""
    from maskahead_b200.serving import PagedCache

    B, H, D, page = 3, 2, 128, 16
    g = torch.Generator().manual_seed(4)
    cache = PagedCache.allocate(batch=B, heads=H, head_dim=D, num_pages=40, page_size=page, max_pages=8,
                                kchan=(0.5 + torch.rand(B, H, D, generator=g)).to(DEV))
    plan = cache.plan(200)
    kept = [[] for _ in range(B)]
    for grow in ([40, 0, 7], [1, 17, 30], [3, 1, 1]):
        old = cache.lens.clone()
        plan.build(old + torch.tensor(grow, dtype=torch.int32, device=DEV))
        n = sum(grow)
        k = torch.randn(200, H, D, generator=g).to(torch.bfloat16).to(DEV)
        v = torch.randn(200, H, D, generator=g).to(torch.bfloat16).to(DEV)
        rk, rv = cache.append(k, v, plan.slots, plan.seqs, return_rows=True)
        at = plan.starts.tolist()
        for b in range(B):
            kept[b].append((rk[at[b]:at[b + 1]], rv[at[b]:at[b + 1]]))
        assert torch.count_nonzero(rk[n:]) == 0
    q, _, _ = _inputs(B, 8, H, 1, D, 0, seed=3)
    out = cache.attend(q)
    for b in range(B):
        k = torch.cat([x[0] for x in kept[b]]).double()
        v = torch.cat([x[1] for x in kept[b]]).double()
        assert k.shape[0] == int(cache.lens[b])
        s = torch.einsum("hgd,nhd->hgn", q[b, :, 0].double().view(H, 4, D), k) * D ** -0.5
        ref = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(8, D)
        # the rows returned are rounded to bf16 once more than what the cache holds: 2^-9 of a
        # key's and a value's elements, so 2^-9 (1 + sum |q k| scale) <= 2^-9 * 30 of |v| ~ 3
        assert (out[b, :, 0].double() - ref).abs().max() < 0.1


# -------------------------------------------------------------------------- verification
def _verify_ref(target, draft, tokens, counts, u):
    target = target.float().cpu().numpy().astype(np.float32)
    draft = None if draft is None else draft.float().cpu().numpy().astype(np.float32)
    tokens, u = tokens.cpu().numpy(), u.cpu().numpy().astype(np.float32)
    B, K1, V = target.shape
    K = K1 - 1
    acc, out = [], []
    for b in range(B):
        n = K if counts is None else min(max(int(counts[b]), 0), K)
        a = 0
        while a < n:
            x = int(tokens[b, a])
            if not 0 <= x < V:
                break
            q = np.float32(1.0) if draft is None else draft[b, a, x]
            if not (np.float32(u[b, a] * q) < target[b, a, x]):
                break
            a += 1

        def weights(r):
            with np.errstate(invalid="ignore"):
                r = np.where(r > 0, np.minimum(r, np.float32(1)), np.float32(0)).astype(np.float64)
            return np.floor(r * 2.0 ** 40).astype(np.int64)

        p = target[b, a]
        r = p
        if a < n and draft is not None:
            with np.errstate(invalid="ignore"):
                r = (p - draft[b, a]).astype(np.float32)
        w = weights(r)
        if a < n and draft is None and 0 <= tokens[b, a] < V:
            w[tokens[b, a]] = 0
        if w.sum() == 0:
            w = weights(p)
        total = int(w.sum())
        mark = total * min(max(int(float(u[b, K]) * 2 ** 24), 0), 2 ** 24 - 1)
        hi = (total >> 24) * min(max(int(float(u[b, K]) * 2 ** 24), 0), 2 ** 24 - 1)
        lo = ((total & (2 ** 24 - 1)) * min(max(int(float(u[b, K]) * 2 ** 24), 0), 2 ** 24 - 1)) >> 24
        mark = hi + lo
        tok = int(np.searchsorted(np.cumsum(w), mark, side="right")) if total else -1
        acc.append(a)
        out.append(tokens[b, :a].tolist() + [tok] + [-1] * (K - a))
    return acc, out


def _verify_inputs(B, K, V, dtype, seed, noise=0.5):
    g = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn(B, K + 1, V, generator=g)
    target = torch.softmax(logits, -1).to(dtype).to(DEV)
    q = torch.softmax(logits[:, :K] + noise * torch.randn(B, K, V, generator=g), -1)
    tokens = torch.multinomial(q.reshape(-1, V).clamp_min(1e-9), 1, generator=g).reshape(B, K) if K else torch.zeros(B, 0)
    u = torch.rand(B, K + 1, generator=g)
    counts = torch.randint(0, K + 1, (B,), generator=g)
    return (target, q.to(dtype).to(DEV), tokens.to(torch.int32).to(DEV), counts.to(torch.int32).to(DEV), u.to(DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 0, 17), (5, 4, 1000), (2, 40, 333), (64, 3, 1023), (9, 2, 1025),
                                   (2, 3, 50021), (300, 1, 4099)])
def test_verify_matches_whole_number_reference(B, K, V, dtype):
    from maskahead_b200.serving import verify_drafts

    target, draft, tokens, counts, u = _verify_inputs(B, K, V, dtype, seed=B * 7 + K)
    for d, c in ((draft, counts), (draft, None), (None, counts)):
        acc, out = verify_drafts(target, d, tokens, c, u)
        ra, ro = _verify_ref(target, d, tokens, c, u)
        assert acc.tolist() == ra
        assert out.tolist() == ro


def test_verify_edges():
    from maskahead_b200.serving import verify_drafts

    V, K = 2500, 2
    target, draft, tokens, _, u = _verify_inputs(8, K, V, torch.float32, seed=3)
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24                   # always accepted / accepted where q <= p
    tokens[2, 0], tokens[3, 0] = -1, V                   # outside the vocabulary: refused
    target[4, 0] = 0.0                                   # no mass at all: refused, nothing to draw
    draft[5, 0], target[5, 0] = 1.0, 0.5                 # p <= q everywhere: the residual is empty
    u[5, 0] = 0.75
    target[6, 0, 100:200] = float("nan")                 # a broken row: NaN weighs nothing
    u[6, 0] = 0.999
    tokens[6, 0] = 150
    target[7, 0] = 3.0                                   # above 1 counts as 1
    acc, out = verify_drafts(target, draft, tokens, None, u)
    ra, ro = _verify_ref(target, draft, tokens, None, u)
    assert acc.tolist() == ra and out.tolist() == ro
    assert ra[0] == 2 and ra[2] == ra[3] == ra[4] == ra[5] == ra[6] == 0
    assert ro[4][0] == -1 and ro[5][0] >= 0


def test_verify_strides_and_determinism():
    from maskahead_b200.serving import verify_drafts, verify_workspace_bytes

    B, K, V = 6, 3, 3001
    target, draft, tokens, counts, u = _verify_inputs(B, K, V, torch.bfloat16, seed=5)
    want = verify_drafts(target, draft, tokens, counts, u)
    wide = torch.empty(B, K + 1, V + 5, device=DEV, dtype=torch.bfloat16)
    wide[..., 1:V + 1] = target
    flipped = draft.transpose(0, 1).contiguous().transpose(0, 1)
    ws = torch.zeros(verify_workspace_bytes(B, V), dtype=torch.uint8, device=DEV)
    for _ in range(3):
        got = verify_drafts(wide[..., 1:V + 1], flipped, tokens, counts, u, workspace=ws)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_verify_rows_at_every_offset(dtype):
    """Rows that begin at any element of 16 bytes, p's and q's apart, their mass where the summed
    pieces begin and end (multiples of 512 elements and their neighbours)."""
    from maskahead_b200.serving import verify_drafts

    B, K, V = 24, 1, 4601
    g = torch.Generator().manual_seed(31)
    edge = torch.arange(V) % 512
    heavy = (edge <= 1) | (edge >= 510) | (torch.arange(V) == V - 1)
    p = (torch.rand(B, K + 1, V, generator=g) * torch.where(heavy, 0.05, 1e-6)).to(dtype).to(DEV)
    q = (torch.rand(B, K, V, generator=g) * torch.where(heavy, 0.03, 1e-6)).to(dtype).to(DEV)
    tokens = torch.randint(0, V, (B, K), generator=g).to(torch.int32).to(DEV)
    u = torch.rand(B, K + 1, generator=g).to(DEV)
    u[::2, 0] = 1.0 - 2.0 ** -24                          # every second draft refused, the others mostly accepted
    u[1::2, 0] = 0.0
    want = {}
    for po in range(8):
        for qo in range(8):
            if po and qo and (po + 3 * qo) % 5:           # all pairs of parities, each offset at least twice
                continue
            wp = torch.full((B, K + 1, V + 15), float("nan"), device=DEV, dtype=dtype)
            wq = torch.full((B, K, V + 15), float("nan"), device=DEV, dtype=dtype)
            wp[..., po:po + V], wq[..., qo:qo + V] = p, q
            for d in (wq[..., qo:qo + V], None):
                if (d is None) not in want:
                    want[d is None] = _verify_ref(p, None if d is None else q, tokens, None, u)
                acc, out = verify_drafts(wp[..., po:po + V], d, tokens, None, u)
                assert acc.tolist() == want[d is None][0] and out.tolist() == want[d is None][1], (po, qo)


def test_verify_leaves_the_target_distribution():
    """Emitted first tokens are distributed as the target's row, whatever the drafter: 40000
    independent requests, each token's frequency within 5 standard deviations."""
    from maskahead_b200.serving import verify_drafts

    B, V = 40000, 6
    g = torch.Generator().manual_seed(9)
    p = torch.tensor([0.35, 0.05, 0.2, 0.1, 0.0, 0.3])
    q = torch.tensor([0.1, 0.4, 0.1, 0.1, 0.2, 0.1])
    tokens = torch.multinomial(q, B, replacement=True, generator=g).to(torch.int32)[:, None].to(DEV)
    target = p.expand(B, 2, V).contiguous().to(DEV)
    draft = q.expand(B, 1, V).contiguous().to(DEV)
    u = torch.rand(B, 2, generator=g).to(DEV)
    acc, out = verify_drafts(target, draft, tokens, None, u)
    freq = torch.bincount(out[:, 0].cpu().long(), minlength=V).double() / B
    sd = (p.double() * (1 - p.double()) / B).sqrt()
    assert ((freq - p.double()).abs() <= 5 * sd + 1e-12).all()
    share = acc.double().mean().item()
    expect = torch.minimum(p, q).sum().item()
    assert abs(share - expect) <= 5 * (expect * (1 - expect) / B) ** 0.5


def test_verify_refusals():
    from maskahead_b200 import KernelUnavailableError, MaError
    from maskahead_b200.serving import verify_drafts

    target, draft, tokens, counts, u = _verify_inputs(2, 2, 50, torch.float32, seed=1)
    for bad in ((target[0], draft, tokens, counts, u), (target.double(), draft, tokens, counts, u),
                (target, draft.half(), tokens, counts, u), (target, draft[:, :1], tokens, counts, u),
                (target, draft, tokens.long(), counts, u), (target, draft, tokens, counts.long(), u),
                (target, draft, tokens, counts, u[:, :2]), (target.transpose(1, 2), draft, tokens, counts, u)):
        with pytest.raises(ValueError):
            verify_drafts(*bad)
    with pytest.raises(KernelUnavailableError):
        verify_drafts(*(x.cpu() for x in (target, draft, tokens, counts, u)))
    big = torch.empty(1, 1, (1 << 20) + 1, device=DEV)
    with pytest.raises(MaError):
        verify_drafts(big, None, tokens[:1, :0], None, u[:1, :1])

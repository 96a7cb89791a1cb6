"""The serving operators over the paged 4-bit cache: their cases, plain forms and work.

Four operators that one decoding step of a serving program runs in turn:

  plan     page tables and slot maps from the requests' old and new lengths
  append   K/V rows quantized into the pool's slots (4-bit codes, fp16 scale and zero)
  attend   attention of one token or a short draft per request over the 4-bit pool, read in
           place, and over the draft itself (token-causal)
  verify   drafted tokens accepted or refused against the target's probabilities with given
           uniforms, and the next token drawn

`run` computes the plain forms in elementary torch operations where `own` is false, and
makes the calls of maskahead_b200.serving where it is true.
"""

import math

import torch

own = False

GROUP = 32          # channels per quantization group
DEV = "cuda"


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token more for each of a few chats
        {"name": "plan 8 tokens", "op": "plan", "batch": 8, "low": 100, "high": 4000, "page": 64, "kind": "token", "grow": 1},
        # a serving batch's drafts; some requests end and hand their pages back; odd page size
        {"name": "plan 256 drafts", "op": "plan", "batch": 256, "low": 4096, "high": 16384, "page": 48, "kind": "draft", "grow": 5},
        # a burst of prompts beside running requests: every prompt token needs its slot
        {"name": "plan 600 prompts", "op": "plan", "batch": 600, "low": 1, "high": 16384, "page": 64, "kind": "prompt", "grow": 0},
        # the accepted tokens of a small batch
        {"name": "append 13 tokens", "op": "append", "tokens": 13, "batch": 4, "heads": 4, "dim": 128, "page": 64, "dtype": "bf16"},
        # accepted drafts of a large batch, 32-bit rows of 64 channels
        {"name": "append 1283 f32 d64", "op": "append", "tokens": 1283, "batch": 256, "heads": 8, "dim": 64, "page": 48, "dtype": "f32"},
        # prompts of a burst
        {"name": "append 131000 prompt", "op": "append", "tokens": 131000, "batch": 9, "heads": 4, "dim": 128, "page": 64, "dtype": "bf16"},
        # one chat, one token, a medium prefix: latency counts
        {"name": "attend 1x1 8192", "op": "attend", "batch": 1, "q_heads": 28, "heads": 4, "dim": 128, "tokens": 1, "low": 8192, "high": 8192, "page": 64},
        # odd lengths, 64 channels, a page size that ends inside a tile, three drafted rows
        {"name": "attend 7x3 ragged d64", "op": "attend", "batch": 7, "q_heads": 32, "heads": 8, "dim": 64, "tokens": 3, "low": 1, "high": 3001, "page": 48},
        # drafts of a serving batch
        {"name": "attend 32x5 drafts", "op": "attend", "batch": 32, "q_heads": 28, "heads": 4, "dim": 128, "tokens": 5, "low": 4096, "high": 16384, "page": 64},
        # single tokens of the serving batch
        {"name": "attend 64x1 serving", "op": "attend", "batch": 64, "q_heads": 28, "heads": 4, "dim": 128, "tokens": 1, "low": 4096, "high": 16384, "page": 64},
        # one chat's four drafts
        {"name": "verify 1x4 32000", "op": "verify", "batch": 1, "drafts": 4, "vocab": 32000, "dtype": "f32"},
        # a serving batch's drafts over an odd, large vocabulary in 16 bits
        {"name": "verify 200x5 100003", "op": "verify", "batch": 200, "drafts": 5, "vocab": 100003, "dtype": "bf16"},
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm, odd more often than not."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))
    n = min(max(n, low), high)
    if rng.random() < 0.5 and n % 2 == 0 and n > low:
        n -= 1
    return n if n != 3 * 1024 else n - 1


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "verify"])
    if op == "plan":
        kind = rng.choice(["token", "draft", "prompt"])
        high = _between(rng, 64, 16384)
        return {"op": op, "batch": _between(rng, 1, 600), "low": _between(rng, 1, high), "high": high,
                "page": rng.choice([16, 32, 48, 64, 100, 128]), "kind": kind,
                "grow": 1 if kind == "token" else rng.randint(2, 16) if kind == "draft" else 0}
    if op == "append":
        return {"op": op, "tokens": _between(rng, 1, 60000), "batch": _between(rng, 1, 256), "heads": rng.choice([1, 2, 4, 8]),
                "dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 48, 64, 100]), "dtype": rng.choice(["bf16", "f32"])}
    if op == "attend":
        heads, group = rng.choice([(4, 7), (8, 4), (2, 8), (1, 12), (8, 1)])
        high = _between(rng, 33, 16384)
        batch = _between(rng, 1, max(1, min(64, 600000 // (high * heads))))
        return {"op": op, "batch": batch, "q_heads": heads * group, "heads": heads, "dim": rng.choice([64, 128, 128]),
                "tokens": rng.choice([1, 1, 1, 2, 3, 4, 6, 8]), "low": _between(rng, 1, high), "high": high,
                "page": rng.choice([16, 32, 48, 64, 64, 100, 128])}
    return {"op": op, "batch": _between(rng, 1, 128), "drafts": rng.randint(1, 5), "vocab": _between(rng, 1000, 100003),
            "dtype": rng.choice(["f32", "bf16", "bf16"])}


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _lengths(case):
    """Request lengths evenly spaced over [low, high]: their sum is the case's, their order the seed's."""
    at = (torch.arange(case["batch"], dtype=torch.float64) + 0.5) / case["batch"]
    return case["low"] + torch.floor(at * (case["high"] - case["low"] + 1)).to(torch.int64)


def _shuffled(count, seed):
    g = torch.Generator()
    g.manual_seed(int(seed) * 7919 + 3)
    return torch.randperm(count, generator=g)


def _table(lens, page, width, pool, seed):
    """A page table of the requests' pages, taken in a shuffled order, and the pages left over."""
    g = torch.Generator()
    g.manual_seed(int(seed) * 104729 + 11)
    order = torch.randperm(pool, generator=g).to(torch.int32)
    need = (lens + page - 1) // page
    ends = torch.cumsum(need, 0)
    first = ends - need
    j = torch.arange(width)
    held = j[None, :] < need[:, None]
    at = (first[:, None] + j[None, :]).clamp(max=max(pool - 1, 0))
    pages = torch.where(held, order[at], torch.full((1, 1), -1, dtype=torch.int32))
    used = int(ends[-1])
    return pages, order[used:].contiguous(), used


def _group_codes(x):
    """4-bit codes, fp16 scale and zero of x [..., D] over groups of 32 channels, each
    operation rounded to x's type as the cache's quantizer does."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    # by a tensor: torch multiplies by a rounded 1/15 where the divisor is a number
    step = ((high - low) / torch.full_like(high, 15.0)).clamp_min(1e-8)
    codes = ((g - low) / step).round().clamp(0, 15).to(torch.uint8)
    payload = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return codes, payload, step.squeeze(-1).to(torch.float16), low.squeeze(-1).to(torch.float16)


def _pool(seed, pages, heads, page, dim):
    """A pool's six arrays, filled with quantized K and V ~ N(0, 1)."""
    gen = _gen(seed)
    made = {"kq": torch.empty(pages, heads, page, dim // GROUP, GROUP // 2, dtype=torch.uint8, device=DEV)}
    made["ks"] = torch.empty(pages, heads, page, dim // GROUP, dtype=torch.float16, device=DEV)
    made["kz"], made["vq"] = torch.empty_like(made["ks"]), torch.empty_like(made["kq"])
    made["vs"], made["vz"] = torch.empty_like(made["ks"]), torch.empty_like(made["ks"])
    step = max(1, (1 << 26) // (heads * page * dim))
    for at in range(0, pages, step):
        for which in ("k", "v"):
            n = min(step, pages - at)
            x = torch.randn(n, heads, page, dim, generator=gen, device=DEV).to(torch.bfloat16)
            _, payload, scale, zero = _group_codes(x)
            made[which + "q"][at:at + n], made[which + "s"][at:at + n], made[which + "z"][at:at + n] = payload, scale, zero
    return made


def _divisor(seed, batch, heads, dim):
    """The per-channel key divisor sqrt(max |K|): about 2 for keys ~ N(0, 1), more for the
    1% of channels that are outliers."""
    gen = _gen(seed + 5)
    base = 3.0 + 1.5 * torch.rand(batch, heads, dim, generator=gen, device=DEV)
    outlier = torch.rand(batch, heads, dim, generator=gen, device=DEV) < 0.01
    return (base * torch.where(outlier, 8.0, 1.0)).sqrt()


def _bf16(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV).to(torch.bfloat16)


def prepare(case, seed):
    op, gen = case["op"], _gen(seed)
    if op == "plan":
        B, page = case["batch"], case["page"]
        if case["kind"] == "prompt":      # nine requests in ten are new prompts, the others run on
            new = _lengths(case)
            old = torch.where(torch.arange(B) % 10 == 3, new, torch.zeros_like(new))
            new = torch.where(old > 0, old + 1, new)
        else:
            old = _lengths(case)
            new = old + case["grow"]
            if case["kind"] == "draft":   # one in sixteen ends, one in sixteen gives drafted tokens back
                at = torch.arange(B) % 16
                new = torch.where(at == 5, torch.zeros_like(new), torch.where(at == 11, (old - case["grow"]).clamp(min=0), new))
        order = _shuffled(B, seed)
        old, new = old[order], new[order]
        width = (case["high"] + 16 + page - 1) // page + 1
        held = int(((torch.maximum(old, new) + page - 1) // page).sum())
        pool = held + B + 7
        pages, free, used = _table(old, page, width, pool, seed)
        stack = torch.full((pool,), -1, dtype=torch.int32)
        stack[:pool - used] = free
        most = int((new - old).clamp(min=0).sum())
        return {"case": case, "page": page, "most": max(1, most + most // 50), "pool": pool,
                "lens": old.to(torch.int32).to(DEV), "new": new.to(torch.int32).to(DEV), "pages": pages.to(DEV),
                "free": stack.to(DEV), "count": torch.tensor([pool - used], dtype=torch.int32, device=DEV)}
    if op == "append":
        N, B, H, D, page = case["tokens"], case["batch"], case["heads"], case["dim"], case["page"]
        slots_in_use = N + N // 8 + page
        pages = (slots_in_use + page - 1) // page
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        state = {"case": case, "page": page, "count": pages}
        for name, inner, kind in (("kq", (D // GROUP, GROUP // 2), torch.uint8), ("ks", (D // GROUP,), torch.float16),
                                  ("kz", (D // GROUP,), torch.float16), ("vq", (D // GROUP, GROUP // 2), torch.uint8),
                                  ("vs", (D // GROUP,), torch.float16), ("vz", (D // GROUP,), torch.float16)):
            # one page more than the pool has: where the plain form puts the rows of padded slots
            state[name] = torch.zeros(pages + 1, H, page, *inner, dtype=kind, device=DEV)
        slots = torch.randperm(pages * page, generator=gen, device=DEV)[:N]
        padded = torch.rand(N, generator=gen, device=DEV) < 0.02     # a slot map is padded with -1
        state["slots"] = torch.where(padded, -1, slots)
        state["seqs"] = torch.randint(0, B, (N,), generator=gen, device=DEV).sort().values.to(torch.int32)
        state["kchan"] = _divisor(seed, B, H, D)
        state["pages"] = torch.full((B, 1), -1, dtype=torch.int32, device=DEV)    # the append reads the slot map alone
        state["lens"] = torch.zeros(B, dtype=torch.int32, device=DEV)
        state["key"] = torch.randn(N, H, D, generator=gen, device=DEV).to(dtype)
        state["value"] = torch.randn(N, H, D, generator=gen, device=DEV).to(dtype)
        return state
    if op == "attend":
        B, H, D, T, page = case["batch"], case["heads"], case["dim"], case["tokens"], case["page"]
        lens = _lengths(case)[_shuffled(B, seed)]
        need = int(((lens + page - 1) // page).sum())
        width = (case["high"] + page - 1) // page
        pages, _, _ = _table(lens, page, width, need + 3, seed)
        state = {"case": case, "page": page, "pages": pages.to(DEV), "lens": lens.to(torch.int32).to(DEV)}
        state.update(_pool(seed, need + 3, H, page, D))
        state["kchan"] = _divisor(seed, B, H, D)
        state["query"] = _bf16(gen, B, case["q_heads"], T, D)
        state["key"], state["value"] = _bf16(gen, B, H, T, D), _bf16(gen, B, H, T, D)
        return state
    B, K, V = case["batch"], case["drafts"], case["vocab"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    # drafter and target see nearly the same logits: most drafts are accepted
    target = torch.empty(B, K + 1, V, dtype=dtype, device=DEV)
    draft = torch.empty(B, K, V, dtype=dtype, device=DEV)
    tokens = torch.empty(B, K, dtype=torch.int32, device=DEV)
    for i in range(K + 1):
        logits = 3.0 * torch.randn(B, V, generator=gen, device=DEV)
        target[:, i] = torch.softmax(logits, -1).to(dtype)
        if i < K:
            q = torch.softmax(logits + 0.4 * torch.randn(B, V, generator=gen, device=DEV), -1)
            draft[:, i] = q.to(dtype)
            noise = torch.empty(B, V, device=DEV).exponential_(generator=gen)
            tokens[:, i] = (q / noise).argmax(-1).to(torch.int32)
    counts = torch.randint(max(0, K - 1), K + 1, (B,), generator=gen, device=DEV).to(torch.int32)
    return {"case": case, "target": target, "draft": draft, "tokens": tokens, "counts": counts,
            "uniforms": torch.rand(B, K + 1, generator=gen, device=DEV)}


# ------------------------------------------------------------------------- plain forms
def _plain_plan(s):
    page, most = s["page"], s["most"]
    lens, new, pages, free = s["lens"].long(), s["new"].long(), s["pages"].long(), s["free"].long()
    count = s["count"].long()
    B, width = pages.shape
    pool = free.shape[0]
    want = new.clamp(min=0)
    want = torch.where((want + page - 1) // page > width, lens, want)
    had, get = (lens + page - 1) // page, (want + page - 1) // page
    lost = (had - get).clamp(min=0)
    handed = lost.sum()
    need, more = (get - had).clamp(min=0), (want - lens).clamp(min=0)
    fits = (need.cumsum(0) <= count + handed) & (more.cumsum(0) <= most)
    need, more = need * fits, more * fits
    lens_out = torch.where((want > lens) & ~fits, lens, want)
    j = torch.arange(width, device=pages.device)[None, :]
    goes = (j >= get[:, None]) & (j < had[:, None])
    rank = (lost.cumsum(0) - lost)[:, None] + j - get[:, None]
    stack = torch.cat([free, free.new_zeros(1)])
    stack = stack.scatter(0, torch.where(goes, count + rank, pool).clamp(0, pool).reshape(-1), pages.reshape(-1))
    taken = need.sum()
    comes = (j >= had[:, None]) & (j < (had + need)[:, None])
    at = count + handed - 1 - ((need.cumsum(0) - need)[:, None] + j - had[:, None])
    pages_out = torch.where(comes, stack[at.clamp(0, pool)], pages)
    left = count + handed - taken
    i = torch.arange(pool, device=pages.device)
    free_out = torch.where((i >= count) & (i < left), stack[:pool], free)
    ends = more.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends])
    i = torch.arange(most, device=pages.device)
    real = i < ends[-1]
    owner = (torch.searchsorted(ends, i, right=True)).clamp(max=B - 1)
    at = lens[owner] + i - starts[owner]
    home = pages_out[owner, (at // page).clamp(0, width - 1)]
    slot = torch.where(real & (home >= 0) & (home < s["pool"]), home * page + at % page, -1)
    return {"lens": lens_out.to(torch.int32), "pages": pages_out.to(torch.int32), "free": free_out.to(torch.int32),
            "count": left.to(torch.int32), "starts": starts.to(torch.int32), "slots": slot,
            "seqs": torch.where(real, owner, -1).to(torch.int32), "positions": torch.where(real, at, -1).to(torch.int32)}


def _plain_append(s):
    page, pool = s["page"], s["count"]
    slots = torch.where(s["slots"] >= 0, s["slots"], pool * page)
    home, at = slots // page, slots % page
    kchan = s["kchan"][s["seqs"].long()]
    out = {}
    for which, x, divisor in (("k", s["key"], kchan), ("v", s["value"], None)):
        y = x if divisor is None else (x.float() / divisor).to(x.dtype)
        codes, payload, scale, zero = _group_codes(y)
        s[which + "q"][home, :, at], s[which + "s"][home, :, at], s[which + "z"][home, :, at] = payload, scale, zero
        back = (codes.float() * scale.float()[..., None] + zero.float()[..., None]).flatten(-2)
        out[which + "_rows"] = (back if divisor is None else back * divisor).to(x.dtype)
        out.update({which + c: s[which + c][:pool] for c in "qsz"})
    return out


def _unpacked(payload, scale, zero, dtype):
    """codes * scale + zero of [..., D/32, 16] bytes as [..., D]."""
    codes = torch.stack([payload & 15, payload >> 4], -1).flatten(-2)
    return (codes.to(dtype) * scale.to(dtype)[..., None] + zero.to(dtype)[..., None]).flatten(-2)


def _plain_attend(s):
    c, page = s["case"], s["page"]
    B, H, T, D = c["batch"], c["heads"], c["tokens"], c["dim"]
    G = c["q_heads"] // H
    home = s["pages"].long().clamp(min=0)
    n = home.shape[1] * page

    def gathered(q, scale, zero):      # [B, pages, H, page, ...] -> [B, H, n, D]
        return _unpacked(q[home], scale[home], zero[home], torch.float32).transpose(1, 2).reshape(B, H, n, D)

    q = s["query"].float().reshape(B, H, G * T, D) * D ** -0.5
    k = gathered(s["kq"], s["ks"], s["kz"]) * s["kchan"][:, :, None]
    a = q @ k.transpose(-1, -2)
    del k
    dead = torch.arange(n, device=q.device)[None, :] >= s["lens"][:, None]
    a = a.masked_fill(dead[:, None, None], -math.inf)
    b = q @ s["key"].float().transpose(-1, -2)
    t = torch.arange(T, device=q.device)
    ahead = (t[None, :] > t[:, None]).repeat(G, 1)
    b = b.masked_fill(ahead, -math.inf)
    top = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
    a, b = torch.exp(a - top), torch.exp(b - top)
    total = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
    o = a @ gathered(s["vq"], s["vs"], s["vz"]) + b @ s["value"].float()
    return (o / total).reshape(B, H * G, T, D).to(torch.bfloat16)


def _plain_verify(s):
    target, draft, tokens, u = s["target"], s["draft"], s["tokens"].long(), s["uniforms"]
    B, K = tokens.shape
    p = target[:, :K].gather(-1, tokens[..., None]).squeeze(-1).float()
    q = draft.gather(-1, tokens[..., None]).squeeze(-1).float()
    i = torch.arange(K, device=tokens.device)[None, :]
    good = (u[:, :K] * q < p) & (i < s["counts"][:, None])
    run_ = good.long().cumprod(-1).sum(-1)
    b = torch.arange(B, device=tokens.device)
    row = target[b, run_].float()
    other = draft[b, run_.clamp(max=K - 1)].float()
    other = torch.where((run_ < s["counts"])[:, None], other, torch.zeros_like(other))

    def weights(x):
        return (torch.where(x > 0, x, torch.zeros_like(x)).clamp(max=1.0) * 2.0 ** 40).to(torch.int64)

    w = weights(row - other)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, weights(row))
    total = w.sum(-1)
    pick = (u[:, K] * 2.0 ** 24).to(torch.int64).clamp(0, (1 << 24) - 1)
    mark = (total >> 24) * pick + (((total & ((1 << 24) - 1)) * pick) >> 24)
    token = (w.cumsum(-1) <= mark[:, None]).sum(-1)
    token = torch.where(total > 0, token, -1)
    j = torch.arange(K + 1, device=tokens.device)[None, :]
    kept = torch.cat([tokens, tokens.new_full((B, 1), -1)], -1)
    out = torch.where(j < run_[:, None], kept, torch.where(j == run_[:, None], token[:, None], -1))
    return {"accepted": run_.to(torch.int32), "tokens": out.to(torch.int32)}


# --------------------------------------------------------------------- the framework's
def _cache(s):
    """The cache object that a serving program keeps; made once for a state."""
    if "cache" not in s:
        from maskahead_b200.serving import PagedCache

        pool = s["count"] if s["case"]["op"] == "append" else s["kq"].shape[0]
        s["cache"] = PagedCache(kq=s["kq"][:pool], ks=s["ks"][:pool], kz=s["kz"][:pool], vq=s["vq"][:pool],
                                vs=s["vs"][:pool], vz=s["vz"][:pool], kchan=s["kchan"], pages=s["pages"], lens=s["lens"])
    return s["cache"]


def _own_plan(s):
    if "plan" not in s:
        from maskahead_b200.serving import TokenPlan

        s["plan"] = TokenPlan(lens=s["lens"], pages=s["pages"], free=s["free"], free_count=s["count"], page_size=s["page"],
                              num_pages=s["pool"], max_tokens=s["most"], in_place=False)
    plan = s["plan"]
    plan.build(s["new"])
    return {"lens": plan.lens, "pages": plan.pages, "free": plan.free, "count": plan.free_count, "starts": plan.starts,
            "slots": plan.slots, "seqs": plan.seqs, "positions": plan.positions}


def _own_append(s):
    cache = _cache(s)
    k, v = cache.append(s["key"], s["value"], s["slots"], s["seqs"], return_rows=True)
    out = {"k_rows": k, "v_rows": v}
    out.update({c: getattr(cache, c) for c in ("kq", "ks", "kz", "vq", "vs", "vz")})
    return out


def _own_verify(s):
    from maskahead_b200.serving import verify_drafts

    accepted, tokens = verify_drafts(s["target"], s["draft"], s["tokens"], s["counts"], s["uniforms"])
    return {"accepted": accepted, "tokens": tokens}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "verify": _plain_verify}[op](state)
    if op == "plan":
        return _own_plan(state)
    if op == "append":
        return _own_append(state)
    if op == "attend":
        return _cache(state).attend(state["query"], state["key"], state["value"])
    return _own_verify(state)


# -------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "plan":
        B, page, mean = case["batch"], case["page"], (case["low"] + case["high"]) / 2
        width = (case["high"] + 16 + page - 1) // page + 1
        tokens = {"token": B, "draft": B * case["grow"] * 14 / 16, "prompt": B * 0.9 * mean}[case["kind"]]
        table, stack = B * width, B * mean / page + B
        return {"bytes": 16 * B + 8 * table + 8 * stack + 16 * tokens * 1.02, "flops": 0}
    if op == "append":
        N, H, D = case["tokens"], case["heads"], case["dim"]
        e = 2 if case["dtype"] == "bf16" else 4
        divisors = 4 * min(N, case["batch"]) * H * D
        return {"bytes": N * (H * (4 * D * e + 2 * (D // 2 + D // 8)) + 12) + divisors, "flops": 10 * N * H * D}
    if op == "attend":
        B, H, D, T = case["batch"], case["heads"], case["dim"], case["tokens"]
        slots = B * (case["low"] + case["high"]) / 2
        rows = B * case["q_heads"] * T
        io = 2 * rows * D * 2 + 2 * B * H * T * D * 2 + 4 * B * H * D + 4 * slots / case["page"]
        return {"bytes": slots * H * 2 * (D // 2 + D // 8) + io, "flops": 4 * D * (slots * case["q_heads"] * T + rows * (T + 1) / 2)}
    B, V, e = case["batch"], case["vocab"], 2 if case["dtype"] == "bf16" else 4
    refused = 1 - 0.85 ** case["drafts"]      # measured: about 0.85 of these drafts are accepted
    return {"bytes": B * (V * e * (1 + refused) + case["drafts"] * (2 * e + 8) + 16), "flops": 2 * B * V}


# ------------------------------------------------------------------------------- exact
def _near_bf16(x):
    """float64 values rounded to the nearest bfloat16, ties to even."""
    return x.to(torch.float32).to(torch.bfloat16).to(torch.float64)


def _exact_append(s):
    out = {}
    narrow = s["key"].dtype == torch.bfloat16
    near = _near_bf16 if narrow else (lambda x: x.to(torch.float32).to(torch.float64))
    for which in ("k", "v"):
        x = (s["key"] if which == "k" else s["value"]).to(torch.float64)
        if which == "k":
            divisor = s["kchan"].to(torch.float64)[s["seqs"].long()]
            x = near(x / divisor)
        N, H, D = x.shape
        x = x.view(N, H, D // GROUP, GROUP)
        low = x.min(-1, keepdim=True).values
        step = near(near(x.max(-1, keepdim=True).values - low) / 15)
        step = torch.maximum(step, near(torch.tensor(1e-8, dtype=torch.float64, device=x.device)))
        codes = torch.round(near(near(x - low) / step)).clamp(0, 15)
        y = (codes * step.to(torch.float16).to(torch.float64) + low.to(torch.float16).to(torch.float64)).view(N, H, D)
        out[which + "_rows"] = y * divisor if which == "k" else y
        out.update({which + c: None for c in "qsz"})
    return out


def _exact_attend(s):
    c, page = s["case"], s["page"]
    B, H, T, D = c["batch"], c["heads"], c["tokens"], c["dim"]
    G = c["q_heads"] // H
    out = torch.empty(B, c["q_heads"], T, D, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist()
    for b in range(B):
        mine = s["pages"][b, :(lens[b] + page - 1) // page].long()

        def rows(name):
            x = _unpacked(s[name + "q"][mine], s[name + "s"][mine], s[name + "z"][mine], torch.float64)
            return x.transpose(0, 1).reshape(H, -1, D)[:, :lens[b]]

        k = torch.cat([rows("k") * s["kchan"][b].double()[:, None], s["key"][b].double()], 1)
        v = torch.cat([rows("v"), s["value"][b].double()], 1)
        for t in range(T):
            seen = lens[b] + t + 1
            q = s["query"][b, :, t].double().view(H, G, D)
            p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k[:, :seen]) / math.sqrt(D), -1)
            out[b, :, t] = torch.einsum("hgn,hnd->hgd", p, v[:, :seen]).reshape(-1, D)
    return out


def exact(case, seed):
    if case["op"] in ("plan", "verify"):
        return None            # whole numbers
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)

"""One decoding step of a serving loop over a paged k4v4 cache.

The select + attend path (hotpath.py) reads a paged cache; this module keeps one. Per step
and layer a serving program

  1. plans the step's slots from the requests' lengths (TokenPlan.build: page tables, free
     stack, slot map, all on the device),
  2. attends with few rows -- one token, or a short draft whose rows see each other causally --
     over the packed pool read in place (PagedCache.attend, decode_attention),
  3. verifies drafted tokens against the target's probabilities (verify_drafts),
  4. appends the kept tokens' K/V rows through the slot map (PagedCache.append).

The reference has no counterpart (its cache is contiguous, its sessions run one batch);
the pool's arrays are its token-mode k4v4 layout (cache.py:142-189) with the page as the
first axis. Everything runs on the current stream of the pool's device (made current for the
call if another one is) without waiting for it, and can be captured in a CUDA graph (run once before the capture, so that the shared
workspace exists). Calls share one workspace per device and purpose, like the other
operators: calls that can overlap on the GPU pass their own (`workspace`, a zeroed uint8
tensor of decode_workspace_bytes / verify_workspace_bytes / PLAN_WORKSPACE_BYTES; attention
that is not read in place needs decode_workspace_bytes with its `capacity`).
"""

from __future__ import annotations

import copy
import ctypes

import torch

from . import _lib
from ._lib import APPEND_ARGS, DECODE_HEAD, DECODE_TAIL, VERIFY_HEAD, VERIFY_TAIL
from .layouts import Prefix, as_prefix, kv_descriptor

__all__ = ["PagedCache", "TokenPlan", "decode_attention", "verify_drafts", "decode_workspace_bytes",
           "verify_workspace_bytes", "PLAN_WORKSPACE_BYTES", "MAX_DECODE_ROWS"]

PLAN_WORKSPACE_BYTES = 512

# Rows per KV head (query heads of the group x tokens) up to which attention reads the packed
# cache in place; beyond, a prefix is unpacked once and the 128-row tensor-core tiles run. In
# place against unpacked, device us: 32 requests x 8192 slots, 4 KV heads, 35 rows 134 / 563, 63
# rows 186 / 565, 84 rows 288 / 567, 112 rows 371 / 334; 30 x 16000, 1 head, 96 rows 135 / 161; 4 x 8192, 4
# heads, 84 rows 48 / 86, 112 rows 72 / 60; 1 x 8192, 84 rows 19 / 37, 112 rows 22 / 29, 224 rows 47 / 29; 1 x 300,
# 112 rows 12 / 17, 224 rows 19 / 17. The unpacked route's host time is 122 against 8, so a short call just
# past the constant is the slower one: it is one number for all sizes.
MAX_DECODE_ROWS = 96

_GROUP = 32


_SHARED: dict[tuple, tuple] = {}     # (device index, purpose) -> (the shared workspace, its address, its bytes)


def _scratch(device: torch.device, purpose: str, nbytes: int, given: torch.Tensor | None) -> tuple[int, int]:
    """(address, bytes) of a call's workspace: the caller's, or the shared one of the device."""
    if given is None:
        held = _SHARED.get((device.index, purpose))
        if held is None or held[2] < nbytes:       # (the shared workspace of a purpose only ever grows, and only here)
            if torch.cuda.is_current_stream_capturing():     # its zero fill would be a node of the graph
                raise RuntimeError(f"run the largest call once before capturing a graph: the shared '{purpose}' "
                                   "workspace must exist")
            ws = _lib.workspace(device, purpose, nbytes)
            held = _SHARED[(device.index, purpose)] = (ws, ws.data_ptr(), ws.numel())
        return held[1], held[2]
    if (given.dtype != torch.uint8 or not given.is_contiguous() or given.device != device or given.numel() < nbytes):
        raise ValueError(f"workspace: need a contiguous uint8 tensor of at least {nbytes} bytes on {device}")
    return given.data_ptr(), given.numel()


def decode_workspace_bytes(batch: int, heads: int, rows: int, head_dim: int, block_tokens: int = 0, *,
                           capacity: int = 0) -> int:
    """Workspace of decode_attention: rows = query heads per KV head x tokens. With capacity =
    the prefix's slots per sequence (max_pages * page_size of a paged cache), also of calls that
    are not read in place: those keep the unpacked prefix and splitk_attention's scratch in it
    (device_status looks at the shared workspaces only: a wait that gave up in a caller's shows as
    rows of NaN)."""
    nbytes = int(_lib.load_library().ma_decode_attention_workspace(batch, heads, rows, head_dim, block_tokens))
    if nbytes == 0 or capacity <= 0:
        return nbytes
    return _general_layout(batch, heads, rows, head_dim, block_tokens, capacity, True)[2]


# splitk_attention's error word and merge counters lie in the first bytes of its scratch
_SPLITK_HEAD = 1 << 17


def _general_layout(batch, heads, rows, head_dim, block_tokens, slots, unpack) -> tuple[int, int, int]:
    """A caller's workspace on the general route: (offset and bytes of splitk_attention's scratch, end),
    from its first 256-byte boundary, the unpacked K and V behind the scratch. All of it lies behind
    what an in-place call of these sizes uses, whose counters are zero between calls."""
    lib, up = _lib.load_library(), lambda x: (x + 255) & ~255  # noqa: E731
    at = up(int(lib.ma_decode_attention_workspace(batch, heads, rows, head_dim, block_tokens)))
    scratch = up(int(lib.ma_prefix_attention_workspace(batch, heads, rows, slots, head_dim, block_tokens))) + 256
    return at, scratch, at + scratch + (2 * up(2 * batch * heads * slots * head_dim) if unpack else 0) + 256


def verify_workspace_bytes(batch: int, vocab: int) -> int:
    return int(_lib.load_library().ma_verify_drafts_workspace(batch, vocab))


def _check(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")


class _FixedTensors:
    """The kernels are given the addresses of these objects' tensors once: a tensor is written
    into, not replaced."""

    def __setattr__(self, name: str, value) -> None:
        held = self.__dict__.get(name)
        if isinstance(held, torch.Tensor) and value is not held:
            raise AttributeError(f"{type(self).__name__}.{name} is fixed for the object's life: write into the tensor")
        super().__setattr__(name, value)


# --------------------------------------------------------------------------- slot planning
class TokenPlan(_FixedTensors):
    """The slots of a step's new tokens, planned on the device from the requests' lengths.

    lens [B] int32 and pages [B, width] int32 describe the requests now (request b holds
    ceil(lens[b] / page_size) pages), free [num_pages] int32 is a stack of free_count [1]
    unused pages. build(new_lens) plans the step: shorter requests hand pages back, longer
    ones take pages from the stack in request order while pages and max_tokens last (from the
    first that does not fit on, none grows: lens then differs from new_lens there).

    After build the attributes hold: lens, pages, free, free_count (the new state; the tensors
    given when in_place, else tensors of the plan's own), starts [B + 1] int32, and per new
    token slots [max_tokens] int64 (page * page_size + offset), seqs and positions
    [max_tokens] int32, -1 past the last token. They are the plan's buffers: the next build
    overwrites them.
    """

    def __init__(self, *, lens: torch.Tensor, pages: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor,
                 page_size: int, num_pages: int, max_tokens: int, in_place: bool = True):
        dev = lens.device
        if dev.type != "cuda":
            raise _lib.KernelUnavailableError("maskahead_b200 kernels need CUDA tensors")
        if lens.ndim != 1 or pages.ndim != 2 or pages.shape[0] != lens.shape[0]:
            raise ValueError("lens must be [B] and pages [B, width]")
        b, width = pages.shape
        if pages.dtype != torch.int32 or pages.device != dev or (pages.stride(1) != 1 and width > 1):
            raise ValueError(f"pages must be int32 on {dev} with a contiguous page axis")
        _check("lens", lens, torch.int32, (b,), dev)
        _check("free", free, torch.int32, (num_pages,), dev)
        _check("free_count", free_count, torch.int32, (1,), dev)
        if page_size <= 0 or max_tokens < 0 or b == 0:
            raise ValueError("need at least one request, page_size > 0 and max_tokens >= 0")
        self.device, self.batch, self.width = dev, b, width
        self.page_size, self.num_pages, self.max_tokens = int(page_size), int(num_pages), int(max_tokens)
        self._in = (lens, pages, free, free_count)
        if in_place:
            self.lens, self.pages, self.free, self.free_count = self._in
        else:
            self.lens, self.free = torch.empty_like(lens), torch.empty_like(free)
            self.pages = torch.empty((b, width), device=dev, dtype=torch.int32)
            self.free_count = torch.empty_like(free_count)
        self.starts = torch.empty(b + 1, device=dev, dtype=torch.int32)
        self.slots = torch.empty(max_tokens, device=dev, dtype=torch.int64)
        self.seqs = torch.empty(max_tokens, device=dev, dtype=torch.int32)
        self.positions = torch.empty(max_tokens, device=dev, dtype=torch.int32)
        self._call = _lib.lib().ma_page_plan
        self._index = lens.get_device()
        self._args = _lib.MaPagePlan(
            lens.data_ptr(), pages.data_ptr(), free.data_ptr(), free_count.data_ptr(), b, width, self.num_pages,
            self.page_size, self.max_tokens, pages.stride(0) if b > 1 else width,
            self.pages.stride(0) if b > 1 else width, self.lens.data_ptr(), self.pages.data_ptr(), self.free.data_ptr(),
            self.free_count.data_ptr(), self.starts.data_ptr(), self.slots.data_ptr(), self.seqs.data_ptr(),
            self.positions.data_ptr())

    def build(self, new_lens: torch.Tensor, *, workspace: torch.Tensor | None = None) -> "TokenPlan":
        """Plan the step whose requests shall have new_lens [B] int32 tokens; returns self."""
        if self._index != _lib.current_device():
            with torch.cuda.device(self._index):
                return self.build(new_lens, workspace=workspace)
        if (new_lens.dtype is not torch.int32 or new_lens.get_device() != self._index or new_lens.dim() != 1
                or new_lens.size(0) != self.batch or not new_lens.is_contiguous()):
            _check("new_lens", new_lens, torch.int32, (self.batch,), self.device)
        ws = _scratch(self.device, "page_plan", PLAN_WORKSPACE_BYTES, workspace)
        rc = self._call(self._args, new_lens.data_ptr(), *ws, _lib.stream_handle(self.device))
        if rc:
            _lib.check("ma_page_plan", rc)
        return self


# ----------------------------------------------------------------------------- the cache
class PagedCache(_FixedTensors):
    """A pool of token-mode k4v4 pages with its requests' tables.

    kq, vq [P, H, page_size, D/32, 16] uint8 codes, ks, kz, vs, vz [P, H, page_size, D/32]
    float16, kchan [B, H, D] float32 key divisors, pages [B, max_pages] int32, lens [B]
    int32; free [P] int32 and free_count [1] int32 (optional) the stack of unused pages. The
    cache addresses these tensors for its life (they are written into, not replaced); lens and
    pages are read on the device by every call.
    """

    def __init__(self, *, kq, ks, kz, vq, vs, vz, kchan, pages, lens, free=None, free_count=None):
        self.kq, self.ks, self.kz, self.vq, self.vs, self.vz = kq, ks, kz, vq, vs, vz
        self.kchan, self.pages, self.lens, self.free, self.free_count = kchan, pages, lens, free, free_count
        if kq.ndim != 5 or not kq.is_cuda:
            raise ValueError("kq must be a rank-5 CUDA tensor [P, H, page_size, D/32, 16]")
        self.num_pages, self.heads, self.page_size = kq.shape[0], kq.shape[1], kq.shape[2]
        self.head_dim = kq.shape[3] * _GROUP
        for name, t in (("ks", ks), ("kz", kz), ("vs", vs), ("vz", vz)):
            if tuple(t.shape) != tuple(kq.shape[:4]):
                raise ValueError(f"{name} must be [P, H, page_size, D/32] = {tuple(kq.shape[:4])}")
        if tuple(vq.shape) != tuple(kq.shape) or kq.shape[4] != _GROUP // 2:
            raise ValueError("kq and vq must be [P, H, page_size, D/32, 16]")
        self.batch = pages.shape[0]
        if tuple(kchan.shape) != (self.batch, self.heads, self.head_dim):
            raise ValueError(f"kchan must be [B, H, D] = {(self.batch, self.heads, self.head_dim)}")
        self.device = kq.device
        self._index = kq.get_device()
        for t in (ks, kz, vq, vs, vz, kchan, pages, lens):
            if t.device != self.device:
                raise ValueError("a cache's tensors must lie on one device")
        self._desc = kv_descriptor(self.prefix())       # checks types and strides
        self._kv = ctypes.addressof(self._desc.kv)
        self._lib = _lib.lib()
        self._forms: dict[tuple, _Call] = {}            # attention calls' forms that passed their checks

    @classmethod
    def allocate(cls, *, batch: int, heads: int, head_dim: int, num_pages: int, page_size: int, max_pages: int,
                 kchan: torch.Tensor, device="cuda") -> "PagedCache":
        """An empty cache: every page on the free stack, every request of length 0."""
        groups = head_dim // _GROUP
        q = [torch.zeros((num_pages, heads, page_size, groups, _GROUP // 2), device=device, dtype=torch.uint8)
             for _ in range(2)]
        s = [torch.zeros((num_pages, heads, page_size, groups), device=device, dtype=torch.float16) for _ in range(4)]
        return cls(kq=q[0], ks=s[0], kz=s[1], vq=q[1], vs=s[2], vz=s[3], kchan=kchan,
                   pages=torch.full((batch, max_pages), -1, device=device, dtype=torch.int32),
                   lens=torch.zeros(batch, device=device, dtype=torch.int32),
                   free=torch.arange(num_pages - 1, -1, -1, device=device, dtype=torch.int32),
                   free_count=torch.full((1,), num_pages, device=device, dtype=torch.int32))

    def prefix(self) -> Prefix:
        """The cache as the prefix of the other operators (every live slot)."""
        return Prefix(kq=self.kq, ks=self.ks, kz=self.kz, vq=self.vq, vs=self.vs, vz=self.vz,
                      nq=self.pages.shape[1] * self.page_size, kb=4, vb=4, kg=_GROUP, vg=_GROUP, kmode=1,
                      kch=self.kchan, pages=self.pages, page_size=self.page_size, lens=self.lens)

    def plan(self, max_tokens: int) -> TokenPlan:
        """A TokenPlan over this cache's tables, updated in place by its build."""
        if self.free is None or self.free_count is None:
            raise ValueError("the cache was made without its free stack (free, free_count)")
        return TokenPlan(lens=self.lens, pages=self.pages, free=self.free, free_count=self.free_count,
                         page_size=self.page_size, num_pages=self.num_pages, max_tokens=max_tokens)

    def append(self, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor, seqs: torch.Tensor, *,
               return_rows: bool = False):
        """Quantize the tokens' K/V rows [N, H, D] (bfloat16 or float32) into the pool: token i
        into slots[i] (int64, as TokenPlan gives them; outside the pool: not stored), its keys
        divided by the divisor of request seqs[i] (int32). The bytes are those of
        layouts.quantize_tokens. return_rows: also the values the slots now stand for, (k, v)
        [N, H, D] in the rows' type."""
        shape, index, dev = key.shape, self._index, self.device
        if index != _lib.current_device():
            with torch.cuda.device(index):
                return self.append(key, value, slots, seqs, return_rows=return_rows)
        n = shape[0] if len(shape) == 3 else -1
        if (n < 0 or value.shape != shape or value.dtype is not key.dtype or shape[1] != self.heads
                or shape[2] != self.head_dim or key.get_device() != index or value.get_device() != index
                or slots.dtype is not torch.int64 or slots.shape != (n,) or slots.get_device() != index
                or seqs.dtype is not torch.int32 or seqs.shape != (n,) or seqs.get_device() != index
                or not slots.is_contiguous() or not seqs.is_contiguous()):
            self._refuse_append(key, value, slots, seqs)
        code = _lib.dtype_code(key.dtype)
        k, v = key, value
        if not (k.is_contiguous() and v.is_contiguous()) or (k.data_ptr() | v.data_ptr()) & 15:
            k, v = _aligned(k), _aligned(v)
        rows_k = rows_v = None
        if return_rows:
            rows_k = torch.empty_like(k) if k.is_contiguous() else k.new_empty(shape)
            rows_v = torch.empty_like(rows_k)
        dense = (self.heads * self.head_dim, self.head_dim)     # (a contiguous tensor's axis of length one has any stride)
        sk, sv = dense if k.is_contiguous() else k.stride(), dense if v.is_contiguous() else v.stride()
        rc = self._lib.ma_append_tokens(APPEND_ARGS.pack(
            k.data_ptr(), v.data_ptr(), slots.data_ptr(), seqs.data_ptr(), rows_k.data_ptr() if return_rows else 0,
            rows_v.data_ptr() if return_rows else 0, sk[0], sk[1], sv[0], sv[1], n, code, self._kv, self.batch,
            self.heads, self.head_dim, 0), _lib.stream_handle(dev))
        if rc:
            _lib.check("ma_append_tokens", rc)
        return (rows_k, rows_v) if return_rows else None

    def _refuse_append(self, key, value, slots, seqs) -> None:
        if key.ndim != 3 or key.shape != value.shape or key.dtype != value.dtype:
            raise ValueError("key and value must be [N, H, D] tensors of one shape and type")
        if tuple(key.shape[1:]) != (self.heads, self.head_dim):
            raise ValueError(f"rows must be [N, {self.heads}, {self.head_dim}]")
        if key.device != self.device or value.device != self.device:
            raise ValueError(f"rows must lie on {self.device}")
        _check("slots", slots, torch.int64, (key.shape[0],), self.device)
        _check("seqs", seqs, torch.int32, (key.shape[0],), self.device)
        raise ValueError("key, value, slots and seqs do not belong to this cache")

    def attend(self, query: torch.Tensor, current_key: torch.Tensor | None = None,
               current_value: torch.Tensor | None = None, *, scaling: float | None = None, causal: bool = True,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """decode_attention over this cache."""
        if self._index != _lib.current_device():
            with torch.cuda.device(self._index):
                return self.attend(query, current_key, current_value, scaling=scaling, causal=causal, out=out,
                                   workspace=workspace)
        return _attend(query, self, self._desc, current_key, current_value, scaling, causal, out, workspace)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t with a contiguous last axis and every row on a 16-byte boundary, copied if it is not."""
    es = t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * es % 16 == 0 for s in t.stride()[:-1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _row_strides(t: torch.Tensor) -> tuple:
    """Strides over (b, h, t); an axis of length one is not stepped along and may have any."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape))


# ----------------------------------------------------------------------------- attention
def decode_attention(query: torch.Tensor, prefix, current_key: torch.Tensor | None = None,
                     current_value: torch.Tensor | None = None, *, scaling: float | None = None, causal: bool = True,
                     out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a few rows per request, query [B, Hq, T, D], over [live prefix | the step's
    own keys current_key / current_value [B, Hkv, Tc, D]]; returns [B, Hq, T, D].

    causal: row t sees the step's key j iff j <= t + Tc - T (Tc >= T; a draft's tokens see the
    ones before them), else all of them. prefix: a PagedCache, a Prefix or a cache view.
    Token-mode k4v4 storage without a dense tail (contiguous or paged, ragged, masked) is read
    in place when the query is bfloat16 and a KV head has at most MAX_DECODE_ROWS rows; its
    elements are then not rounded to bfloat16. Everything else runs as splitk_attention,
    over a bfloat16 copy of a packed prefix. A row that sees no key is zero. workspace: see
    decode_workspace_bytes; one too small for the route of the call is refused.
    """
    if isinstance(prefix, PagedCache):
        return prefix.attend(query, current_key, current_value, scaling=scaling, causal=causal, out=out,
                             workspace=workspace)
    index = query.get_device()
    if index >= 0 and index != _lib.current_device():
        with torch.cuda.device(index):
            return decode_attention(query, prefix, current_key, current_value, scaling=scaling, causal=causal, out=out,
                                    workspace=workspace)
    pre = as_prefix(prefix)
    return _attend(query, pre, None, current_key, current_value, scaling, causal, out, workspace)


class _Call:
    """What one form of an in-place attention call (its tensors' shapes, strides and types)
    passes besides the pointers."""

    __slots__ = ("run", "device", "block", "tail", "keep", "shape", "packed", "nbytes")


_MAX_FORMS = 256     # remembered forms per cache; a loop has a few


def _attend(query, source, desc, current_key, current_value, scaling, causal, out, workspace):
    """decode_attention. The checks below depend on shapes, strides, types and devices alone, so
    a PagedCache remembers the forms that passed them (the checks and descriptors took 28 us
    of host time a call, the kernel of a single token over 8192 slots a third of that)."""
    forms = form = call = None
    # plain values in the remembered forms: a tensor would be found again by its identity, whatever it holds by then
    if scaling is not None and type(scaling) is not float:
        scaling = float(scaling)
    causal = bool(causal)
    if isinstance(source, PagedCache):
        forms = source._forms
        form = (query.shape, query.stride(), query.dtype, query.get_device(), scaling, causal,
                None if current_key is None else (current_key.shape, current_key.stride(), current_key.dtype,
                                                  current_key.get_device()),
                None if current_value is None else (current_value.shape, current_value.stride(), current_value.dtype,
                                                    current_value.get_device()),
                None if out is None else (out.shape, out.stride(), out.dtype, out.get_device()))
        call = forms.get(form)
    if call is None:
        if query.dtype == torch.bfloat16 and current_value is not None and current_key is not None:
            k2, v2 = _aligned(current_key.to(query.dtype)), _aligned(current_value.to(query.dtype))
        else:
            k2, v2 = current_key, current_value
        q2 = _aligned(query)
        if q2 is not query or k2 is not current_key or v2 is not current_value:
            return _attend(q2, source, desc, k2, v2, scaling, causal, out, workspace)
        call = _attend_form(query, source, desc, current_key, current_value, scaling, causal, out)
        if call is None:
            return _attend_general(query, source, current_key, current_value, scaling, causal, out, workspace)
        if forms is not None:
            if len(forms) >= _MAX_FORMS:
                forms.clear()
            forms[form] = call
    q = query.data_ptr()
    k = v = 0
    if call.block:
        k, v = current_key.data_ptr(), current_value.data_ptr()
    if (q | k | v) & 15:       # strides that can be read, but a start between 16-byte boundaries
        if k | v:
            current_key, current_value = _aligned(current_key), _aligned(current_value)
        return _attend(_aligned(query), source, desc, current_key, current_value, scaling, causal, out, workspace)
    if out is not None and out.data_ptr() & 15:
        raise ValueError("out must start on a 16-byte boundary")
    o = out if out is not None else torch.empty_like(query) if call.packed else query.new_empty(call.shape)
    dev = call.device
    ws, nbytes = _scratch(dev, "decode", call.nbytes, workspace)
    rc = call.run(DECODE_HEAD.pack(q, k, v, o.data_ptr(), ws, nbytes) + call.tail, _lib.stream_handle(dev))
    if rc == _lib.MA_ERR_UNSUPPORTED:
        return _attend_general(query, source, current_key, current_value, scaling, causal, out, workspace)
    if rc:
        _lib.check("ma_decode_attention", rc)
    return o


def _attend_form(query, source, desc, current_key, current_value, scaling, causal, out) -> _Call | None:
    """Check a call; its _Call when it is read in place, None for the general route."""
    if query.ndim != 4:
        raise ValueError("query must have shape [B, Hq, T, D]")
    if not query.is_cuda:
        raise _lib.KernelUnavailableError("maskahead_b200 kernels need CUDA tensors")
    b, hq, t, d = query.shape
    if (current_key is None) != (current_value is None) or current_key is not None and (
            current_key.shape != current_value.shape or current_key.ndim != 4):
        raise ValueError("current K and V must be [B, Hkv, Tc, D] tensors of one shape")
    tc = 0 if current_key is None else current_key.shape[2]
    if causal and 0 < tc < t:
        raise ValueError(f"causal rows need at least as many current keys as rows: Tc={tc} < T={t}")
    cached = isinstance(source, PagedCache)
    if cached:
        heads = source.heads
        if b != source.batch or d != source.head_dim or query.device != source.device:
            raise ValueError(f"query must be [{source.batch}, Hq, T, {source.head_dim}] on {source.device}")
    else:
        stored = source.kf if source.kf is not None else source.vq
        if stored is None and current_key is None:
            raise ValueError("nothing to attend: an empty prefix and no current keys")
        heads = current_key.shape[1] if stored is None else stored.shape[1]
    if hq % heads:
        raise ValueError("Hq must be divisible by Hkv")
    if current_key is not None and (tuple(current_key.shape) != (b, heads, tc, d) or current_key.device != query.device
                                    or current_value.device != query.device):
        raise ValueError(f"current K and V must be [{b}, {heads}, Tc, {d}] on {query.device}")
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype or out.device != query.device
                            or out.stride(-1) != 1 or any(s * out.element_size() % 16 for s in _row_strides(out))):
        raise ValueError("out must match the query's shape, type and device, with contiguous rows on 16-byte boundaries")
    rows = hq // heads * t
    if query.dtype != torch.bfloat16 or rows > MAX_DECODE_ROWS or not (
            cached or (source.nq > 0 and source.nf == 0 and source.kmode == 1)):
        return None
    if desc is None:
        desc = kv_descriptor(source, batch=b, heads=heads, head_dim=d)
    call = _Call()
    call.run, call.device, call.block, call.keep = _lib.lib().ma_decode_attention, query.device, tc > 0, desc
    call.shape, call.packed = (b, hq, t, d), query.is_contiguous()
    none = (0, 0, 0)
    call.tail = DECODE_TAIL.pack(
        *query.stride()[:3], *(current_key.stride()[:3] if tc else none), *(current_value.stride()[:3] if tc else none),
        *((hq * t * d, t * d, d) if out is None else _row_strides(out)), ctypes.addressof(desc.kv), _lib.MA_BF16, b, hq,
        heads, t, d, tc, 1 if causal else 0, d ** -0.5 if scaling is None else float(scaling), 0)
    call.nbytes = int(_lib.lib().ma_decode_attention_workspace(b, heads, rows, d, tc))
    return call


def _without_dead_pages(prefix: Prefix, batch: int, heads: int, head_dim: int, desc) -> Prefix:
    """The paged prefix as the unpacked copy may hold it: that copy has no page table, so slots on
    page numbers outside the pool would come back as keys of zeros. Their pages are left out (the
    order of slots does not matter to attention), or, where slots are named by a mask or a tail's
    place behind them, masked."""
    own, nq, dev = copy.copy(prefix), prefix.nq, prefix.vq.device
    if prefix.mask is None and prefix.nf == 0:
        width = -(-nq // prefix.page_size)
        words = torch.empty(batch * (width + 1), device=dev, dtype=torch.int32)
        own.pages, own.lens = words[batch:].view(batch, width), words[:batch]
        if desc is None:
            desc = kv_descriptor(prefix, batch=batch, heads=heads, head_dim=head_dim)
        _lib.check("ma_live_pages", _lib.lib().ma_live_pages(desc.kv, batch, own.pages.data_ptr(), own.lens.data_ptr(),
                                                             _lib.stream_handle(dev)))
        return own
    live = (prefix.pages >= 0) & (prefix.pages < prefix.vq.shape[0])
    live = live[:, torch.arange(nq, device=dev) // prefix.page_size]
    live = torch.cat([live, live.new_ones(batch, prefix.nf)], 1)[:, None].expand(batch, heads, prefix.n)
    own.mask = live.contiguous() if prefix.mask is None else live & prefix.mask.bool()
    return own


def _attend_general(query, source, current_key, current_value, scaling, causal, out, workspace):
    from .hotpath import unpacked_prefix
    from .kernels.splitk import splitk_attention

    prefix = source.prefix() if isinstance(source, PagedCache) else source
    b, hq, t, d = query.shape
    tc = 0 if current_key is None else current_key.shape[2]
    stored = prefix.kf if prefix.kf is not None else prefix.vq
    heads = stored.shape[1] if current_key is None else current_key.shape[1]
    unpack = query.dtype == torch.bfloat16 and prefix.nq > 0
    scratch = unpacked = None
    if workspace is not None:      # nothing shared: the call's scratch and copies lie in what it was given
        at, nbytes, end = _general_layout(b, heads, hq // heads * t, d, tc, prefix.n, unpack)
        base = -_scratch(query.device, "decode", end, workspace)[0] % 256 + at
        scratch = workspace[base:base + nbytes]
        scratch[:_SPLITK_HEAD].zero_()       # (in-place calls leave partials here)
        if unpack:
            size, shape = 2 * b * heads * prefix.n * d, (b, heads, prefix.n, d)
            at_k = base + nbytes
            at_v = at_k + ((size + 255) & ~255)
            unpacked = tuple(workspace[x:x + size].view(torch.bfloat16).view(shape) for x in (at_k, at_v))
    if unpack:
        if prefix.pages is not None:
            prefix = _without_dead_pages(prefix, b, heads, d, source._desc if isinstance(source, PagedCache) else None)
        prefix = unpacked_prefix(prefix, b, heads, d, out=unpacked)
    res, _ = splitk_attention(query, prefix, current_key, current_value, scaling=scaling,
                              causal_block=1 if causal and tc else 0, q_pos0=tc - t, c_pos0=0, workspace=scratch)
    if out is None:
        return res
    out.copy_(res)
    return out


# -------------------------------------------------------------------------- verification
def verify_drafts(target: torch.Tensor, draft: torch.Tensor | None, tokens: torch.Tensor,
                  counts: torch.Tensor | None, uniforms: torch.Tensor, *, workspace: torch.Tensor | None = None):
    """Accept or refuse drafted tokens against the target's probabilities and draw the next.

    target [B, K + 1, V] (float32, bfloat16 or float16): the target's probabilities after the
    context and after each draft; draft [B, K, V] of the same type: the distributions the
    drafts were drawn from (None: each draft was certain, e.g. greedy or looked up); tokens
    [B, K] int32; counts [B] int32 drafts in use (None: K); uniforms [B, K + 1] float32 in
    [0, 1). Draft i is accepted while u_i q_i(x_i) < p_i(x_i); after a accepted drafts the next
    token is drawn from max(p_a - q_a, 0), or from p_a when all were accepted, with the last
    uniform: every emitted token is then distributed as the target's own. The drawing sums
    whole numbers (floor(r 2^40)), so the same inputs give the same token on any GPU.

    Returns (accepted [B] int32, tokens [B, K + 1] int32: the accepted drafts, the next token,
    then -1); tokens[b, accepted[b]] is -1 only when p_a has no mass.
    """
    index = target.get_device()
    if index >= 0 and index != _lib.current_device():
        with torch.cuda.device(index):
            return verify_drafts(target, draft, tokens, counts, uniforms, workspace=workspace)
    form = (target.shape, target.stride(), target.dtype, index, tokens.shape, tokens.stride(), tokens.dtype,
            tokens.get_device(), uniforms.shape, uniforms.stride(), uniforms.dtype, uniforms.get_device(),
            None if draft is None else (draft.shape, draft.stride(), draft.dtype, draft.get_device()),
            None if counts is None else (counts.shape, counts.stride(), counts.dtype, counts.get_device()))
    tail = _verify_forms.get(form)
    if tail is None:
        tail = _verify_form(target, draft, tokens, counts, uniforms)
        if len(_verify_forms) >= _MAX_FORMS:
            _verify_forms.clear()
        _verify_forms[form] = tail
    accepted = uniforms.new_empty(tail[0], dtype=torch.int32) if counts is None else torch.empty_like(counts)
    out = torch.empty_like(uniforms, dtype=torch.int32)
    dev = target.device
    ws, nbytes = _scratch(dev, "verify", tail[1], workspace)
    rc = _lib.lib().ma_verify_drafts(VERIFY_HEAD.pack(
        target.data_ptr(), 0 if draft is None else draft.data_ptr(), tokens.data_ptr(),
        0 if counts is None else counts.data_ptr(), uniforms.data_ptr(), accepted.data_ptr(), out.data_ptr(), ws, nbytes)
        + tail[2], _lib.stream_handle(dev))
    if rc:
        _lib.check("ma_verify_drafts", rc)
    return accepted, out


# Forms of call (shapes, strides, types, devices) that passed the checks: (requests, workspace bytes, the
# packed end of ma_verify_args). The checks took a third of a small call's host time.
_verify_forms: dict[tuple, tuple[int, int, bytes]] = {}


def _verify_form(target, draft, tokens, counts, uniforms) -> tuple[int, int, bytes]:
    shape, index = target.shape, target.get_device()
    b, k1, v = shape if len(shape) == 3 else (0, 0, 0)
    k = k1 - 1
    code = _PROBABILITIES.get(target.dtype)
    if (code is None or index < 0 or b < 1 or k < 0 or v < 1 or tokens.dtype is not torch.int32
            or tokens.shape != (b, k) or tokens.get_device() != index or not tokens.is_contiguous()
            or uniforms.dtype is not torch.float32 or uniforms.shape != (b, k1) or uniforms.get_device() != index
            or not uniforms.is_contiguous() or (target.stride(2) != 1 and v > 1)
            or (counts is not None and (counts.dtype is not torch.int32 or counts.shape != (b,)
                                        or counts.get_device() != index or not counts.is_contiguous()))
            or (draft is not None and (draft.dtype is not target.dtype or draft.shape != (b, k, v)
                                       or draft.get_device() != index or (draft.stride(2) != 1 and v > 1)))):
        _refuse_verify(target, draft, tokens, counts, uniforms)
    st, sd = target.stride(), (0, 0) if draft is None else draft.stride()
    return b, verify_workspace_bytes(b, v), VERIFY_TAIL.pack(st[0], st[1], sd[0], sd[1], code, b, k, v)


_PROBABILITIES = {torch.float32: _lib.MA_F32, torch.bfloat16: _lib.MA_BF16, torch.float16: _lib.MA_F16}


def _refuse_verify(target, draft, tokens, counts, uniforms) -> None:
    if target.ndim != 3 or target.dtype not in _PROBABILITIES:
        raise ValueError("target must be a float32, bfloat16 or float16 tensor [B, K + 1, V]")
    b, k1, v = target.shape
    k, dev = k1 - 1, target.device
    if dev.type != "cuda":
        raise _lib.KernelUnavailableError("maskahead_b200 kernels need CUDA tensors")
    if k < 0 or b == 0 or v == 0:
        raise ValueError("target must be [B, K + 1, V] with B, V >= 1 and K >= 0")
    if target.stride(2) != 1 and v > 1:
        raise ValueError("target must have a contiguous vocabulary axis")
    if draft is not None and (draft.dtype != target.dtype or tuple(draft.shape) != (b, k, v) or draft.device != dev
                              or (draft.stride(2) != 1 and v > 1)):
        raise ValueError(f"draft must be a {target.dtype} tensor {(b, k, v)} on {dev} with a contiguous vocabulary axis")
    _check("tokens", tokens, torch.int32, (b, k), dev)
    _check("uniforms", uniforms, torch.float32, (b, k1), dev)
    if counts is not None:
        _check("counts", counts, torch.int32, (b,), dev)
    raise ValueError("the tensors do not belong together")

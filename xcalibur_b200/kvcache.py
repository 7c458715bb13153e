"""The attention side of a decoder layer: a paged key-value cache and the operators on it.

``PagedKVCache`` holds keys and values of all layers in pages, with the tables that say which pages a sequence has.
A decode step of one layer is ``append`` (norms of queries and keys, position rotation, store of keys and values) and
``attend`` (attention of the new tokens over the pages), around which a model's projections and its MoE layer
(``PreparedMoE``) stand; once per step ``extend`` makes room for the new tokens.  ``fork``, ``truncate``, ``free`` and
``compact`` serve parallel sampling, rolled-back drafts, finished sequences and a pool that is to shrink.

PyTorch supplies device memory and the current stream; all work runs in the sm_100a kernels of the library, on the
current stream, without host synchronisation (``check_device_status`` excepted).  Argument errors raise before a
launch; what only the device can see (a page id out of range, a sequence that cannot grow) sets bits of the cache's
status word, read by ``check_device_status``.  The reference has no attention operator.
"""
from __future__ import annotations

import ctypes
import math
import struct
from operator import index
from typing import Optional

import torch

from . import _lib
from ._lib import XcbAttnArgs, XcbKvCache, XcbRopeArgs, check

_CACHE_DTYPES = {torch.bfloat16: _lib.XCB_DTYPE_BF16, torch.float16: _lib.XCB_DTYPE_F16,
                 torch.float8_e4m3fn: _lib.XCB_DTYPE_E4M3}
_Q_DTYPES = {torch.bfloat16: _lib.XCB_DTYPE_BF16, torch.float16: _lib.XCB_DTYPE_F16}


# The C structures of a call, packed in one go (a call's cost on the host is a good part of a short kernel's).
_ROPE_ARGS = struct.Struct("8i3fi3P10q7P")
_ATTN_ARGS = struct.Struct("6ifP3q3P")
assert _ROPE_ARGS.size == ctypes.sizeof(XcbRopeArgs) and _ATTN_ARGS.size == ctypes.sizeof(XcbAttnArgs)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _check_ints(t: torch.Tensor, n: Optional[int], device: torch.device, what: str) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != 1 or (n is not None and t.shape[0] != n) or t.device != device:
        raise ValueError(f"{what} must be int32 [{'n' if n is None else n}] on {device}")
    return t if t.is_contiguous() else t.contiguous()


class Rope:
    """Rotation frequencies of a model: f_i = base^(-2 i / rotary_dim), changed by ``scaling`` for long contexts.

    ``interleaved``: pairs are (2i, 2i + 1), else (i, i + rotary_dim / 2).  ``rotary_dim`` values of each head turn,
    the rest pass.  ``scaling``: None, or a dict with ``type``

    * ``"linear"``: positions are divided by ``factor``;
    * ``"ntk"``: the base grows by ``factor^(rotary_dim / (rotary_dim - 2))``;
    * ``"yarn"``: frequencies that turn more than ``beta_fast`` (32) times within the ``original`` context stay, those
      that turn less than ``beta_slow`` (1) times are divided by ``factor``, a ramp between; cos and sin are
      multiplied by ``mscale`` (0.1 ln(factor) + 1).

    Frequencies are kept as 64-bit fractions of a turn, so angles are exact at any position."""

    def __init__(self, rotary_dim: int, *, base: float = 10000.0, interleaved: bool = False,
                 scaling: Optional[dict] = None, device="cuda"):
        if rotary_dim < 0 or rotary_dim % 2 or rotary_dim > 256:
            raise ValueError("rotary_dim must be even, 0 to 256")
        if not base > 0:
            raise ValueError("base must be positive")
        self.rotary_dim, self.base, self.interleaved = int(rotary_dim), float(base), bool(interleaved)
        self.frequencies, self.mscale = self._frequencies(dict(scaling) if scaling else {})
        if any(not 0 <= f < 2 * math.pi for f in self.frequencies):
            raise ValueError("a rotation frequency is not below a full turn per position")
        words = [min((1 << 64) - 1, int(f / (2 * math.pi) * 2.0 ** 64)) for f in self.frequencies]
        self.turns = torch.tensor([w - (1 << 64) if w >= 1 << 63 else w for w in words], dtype=torch.int64,
                                  device=device)

    def _frequencies(self, scaling: dict):
        rot, base = self.rotary_dim, self.base
        if scaling and scaling.get("type") is None:
            raise ValueError("scaling needs a type")
        kind = scaling.pop("type", None)
        if kind == "yarn" and "original" not in scaling:
            raise ValueError("yarn needs the original context")
        factor = float(scaling.pop("factor", 1.0))
        if not (0 < factor < math.inf):
            raise ValueError("the scaling factor must be positive")
        mscale = 1.0
        if kind == "ntk":
            base *= factor ** (rot / max(rot - 2, 1))
        freqs = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
        if kind == "linear":
            freqs = [f / factor for f in freqs]
        elif kind == "yarn":
            original = scaling.pop("original")
            fast, slow = scaling.pop("beta_fast", 32.0), scaling.pop("beta_slow", 1.0)
            mscale = scaling.pop("mscale", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)

            def index_of(turns):  # the pair that turns so many times within the original context
                return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

            low = max(math.floor(index_of(fast)), 0)
            high = min(math.ceil(index_of(slow)), rot - 1)
            for i, f in enumerate(freqs):
                ramp = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
                freqs[i] = f * (1 - ramp) + f / factor * ramp
        elif kind not in (None, "ntk"):
            raise ValueError(f"unknown scaling type {kind!r}")
        if scaling:
            raise ValueError(f"unknown scaling entries {sorted(scaling)}")
        return freqs, float(mscale)


class _RopePlan:
    """What one form of a call (types, shapes, strides, rotation) comes to: its checks passed, its constants packed."""

    __slots__ = ("head", "strides", "q_shape", "k_shape", "like")


def _rope_plan(cache, q, k, v, positions, seqs, rope, wq, wk, eps, weight_offset, q_out, k_out) -> _RopePlan:
    dtype = _Q_DTYPES.get(q.dtype)
    if dtype is None or not q.is_cuda:
        raise ValueError("queries must be bf16 or fp16 CUDA tensors (there is no CPU path)")
    device = q.device
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens, heads, head_dim], got {tuple(q.shape)}")
    if cache is not None:
        if q.shape[2] != cache.head_dim:
            raise ValueError(f"head_dim is {cache.head_dim}")
        if q.device != cache.device:
            raise ValueError("the queries are on another device than the cache")
        if q.dtype != cache._q_dtype and cache._q_dtype is not None:
            raise ValueError("the cache holds another type than the keys")
    tokens, q_heads, dim = q.shape
    if dim % 8:
        check(_lib.XCB_ERR_UNSUPPORTED, "xcb_qk_norm_rope")
    kv_heads = cache.kv_heads if cache is not None else k.shape[1] if k is not None and k.dim() == 3 else 0
    for t, what in ((k, "k"), (v, "v")):
        if t is None:
            continue
        if t.dtype != q.dtype or t.device != device:
            raise ValueError(f"{what} must have the queries' type and device")
        if tuple(t.shape) != (tokens, kv_heads, dim):
            raise ValueError(f"{what} must be [{tokens}, {kv_heads}, {dim}], got {tuple(t.shape)}")
    if rope.turns.device != device:
        raise ValueError("rope is on another device than the queries")
    if rope.rotary_dim > dim:
        raise ValueError(f"rotary_dim {rope.rotary_dim} is larger than head_dim {dim}")
    _check_ints(positions, tokens, device, "positions")
    if cache is not None:
        _check_ints(seqs, tokens, device, "seqs")
    for w, what in ((wq, "q_weight"), (wk, "k_weight")):
        if w is not None and (w.shape != (dim,) or w.device != device or w.dtype not in (q.dtype, torch.float32)):
            raise ValueError(f"{what} must be [head_dim], of the queries' type or float32")
    if wq is not None and wk is not None and wq.dtype != wk.dtype:
        raise ValueError("q_weight and k_weight must have one type")
    for given, like, what in ((q_out, q, "q_out"), (k_out, k, "k_out")):
        if given is not None and (like is None or given.shape != like.shape or given.dtype != q.dtype or
                                  given.device != device or given.stride(2) != 1 or given.stride(0) % 8 or
                                  given.stride(1) % 8):
            raise ValueError(f"{what} must be like its input, with aligned contiguous heads")
    weight = wq if wq is not None else wk
    wtype = dtype if weight is None or weight.dtype == q.dtype else _lib.XCB_DTYPE_F32
    plan = _RopePlan()
    plan.head = (tokens, q_heads, kv_heads, dim, rope.rotary_dim, rope.interleaved, dtype, wtype, eps, weight_offset,
                 rope.mscale)  # and the layer

    def strides(t):
        return (0, 0) if t is None else t.stride()[:2]

    made = (q_heads * dim, dim), (kv_heads * dim, dim)  # of outputs made here
    plan.strides = strides(q) + strides(k) + strides(v) + (made[0] if q_out is None else strides(q_out)) + \
        (made[1] if k_out is None else strides(k_out))
    plan.q_shape = (tokens, q_heads, dim)
    plan.like = q.is_contiguous()  # so is an output like it
    plan.k_shape = (tokens, kv_heads, dim) if cache is None and k is not None else None
    return plan


def _odd_rows(t: torch.Tensor) -> bool:
    """Heads that the kernels cannot read in place: not contiguous, or not on 16-byte boundaries."""
    a, b, c = t.stride() if t.dim() == 3 else (0, 0, 1)
    return c != 1 or a % 8 != 0 or b % 8 != 0 or t.data_ptr() % 16 != 0


# Calls' forms that have passed their checks: types, shapes and strides only; no tensor, no address, no layer.
_PLANS: dict = {}


def _rope_call(cache, layer, q, k, v, positions, seqs, rope, q_weight, k_weight, eps, weight_offset, q_out, k_out):
    plans = _PLANS if cache is None else cache._rope_plans
    layer, eps, weight_offset = index(layer), float(eps), float(weight_offset)
    if cache is not None and not 0 <= layer < cache.layers:
        raise ValueError(f"layer must be in [0, {cache.layers})")
    key = (eps, weight_offset, rope.rotary_dim, rope.interleaved, rope.mscale, rope.turns.get_device(),
           q.dtype, q.shape, q.stride(), q.get_device(),
           k is not None and (k.dtype, k.shape, k.stride(), k.get_device()),
           v is not None and (v.dtype, v.shape, v.stride(), v.get_device()),
           positions.dtype, positions.shape, positions.stride(), positions.get_device(),
           seqs is not None and (seqs.dtype, seqs.shape, seqs.stride(), seqs.get_device()),
           q_weight is not None and (q_weight.dtype, q_weight.shape, q_weight.stride(), q_weight.get_device()),
           k_weight is not None and (k_weight.dtype, k_weight.shape, k_weight.stride(), k_weight.get_device()),
           q_out is not None and (q_out.dtype, q_out.shape, q_out.stride(), q_out.get_device()),
           k_out is not None and (k_out.dtype, k_out.shape, k_out.stride(), k_out.get_device()))
    plan = plans.get(key)
    if plan is None:
        plan = _rope_plan(cache, q, k, v, positions, seqs, rope, q_weight, k_weight, eps, weight_offset, q_out,
                          k_out)
        copies = [t is not None and (_odd_rows(t) if i < 3 else not t.is_contiguous())
                  for i, t in enumerate((q, k, v, positions, seqs, q_weight, k_weight))]
        if any(copies):  # what cannot be read in place is copied, and the call is that of the copies
            q, k, v, positions, seqs, q_weight, k_weight = (
                t.clone(memory_format=torch.contiguous_format) if c else t
                for t, c in zip((q, k, v, positions, seqs, q_weight, k_weight), copies))
            return _rope_call(cache, layer, q, k, v, positions, seqs, rope, q_weight, k_weight, eps, weight_offset,
                              q_out, k_out)
        if len(plans) >= 1024:
            plans.clear()
        plans[key] = plan
    if q_out is None:
        q_out = torch.empty_like(q) if plan.like else torch.empty(plan.q_shape, dtype=q.dtype, device=q.device)
    if k_out is None and plan.k_shape is not None:
        k_out = torch.empty(plan.k_shape, dtype=q.dtype, device=q.device)
    pq, pk, pv = q.data_ptr(), 0 if k is None else k.data_ptr(), 0 if v is None else v.data_ptr()
    pwq, pwk = 0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr()
    if (pq | pk | pv | pwq | pwk) & 15:  # a view of the same form as one seen, but not on a 16-byte boundary
        q, k, v, q_weight, k_weight = (t if t is None or t.data_ptr() % 16 == 0 else
                                       t.clone(memory_format=torch.contiguous_format)
                                       for t in (q, k, v, q_weight, k_weight))
        return _rope_call(cache, layer, q, k, v, positions, seqs, rope, q_weight, k_weight, eps, weight_offset, q_out,
                          k_out)
    if (q_out.data_ptr() | (0 if k_out is None else k_out.data_ptr())) & 15:
        raise ValueError("q_out and k_out must be on 16-byte boundaries")
    args = _ROPE_ARGS.pack(*plan.head, layer, pq, pk, pv, *plan.strides, q_out.data_ptr(),
                           0 if k_out is None else k_out.data_ptr(), pwq, pwk, positions.data_ptr(),
                           0 if seqs is None else seqs.data_ptr(), rope.turns.data_ptr())
    if cache is None:
        _launch(q.device, _lib.load().xcb_qk_norm_rope, "xcb_qk_norm_rope", None, args)
    else:
        _launch(cache.device, cache.lib.xcb_qk_norm_rope, "xcb_qk_norm_rope", cache._address, args)
    return q_out, k_out


def _launch(device, fn, what, *args):
    """Call a C entry on the device's current stream, with that device current."""
    on = device.index
    if on == torch._C._cuda_getDevice():
        rc = fn(*args, _raw_stream(on))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(on))
    if rc:
        check(rc, what)


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: Rope, *,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 weight_offset: float = 0.0, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None):
    """Norms of queries and keys per head and the position rotation, in one pass: ``(q', k')``.

    ``q`` [T, q_heads, D] and ``k`` [T, kv_heads, D] (or None), bf16 or fp16, may be strided views of one projection's
    rows; ``positions`` int32 [T].  ``q_weight`` / ``k_weight`` [D]: y = x * rsqrt(mean(x^2) + eps) * (w +
    weight_offset), no norm where None.  ``q_out`` / ``k_out`` may be the inputs themselves."""
    return _rope_call(None, 0, q, k, None, positions, None, rope, q_weight, k_weight, eps, weight_offset, q_out, k_out)


class PagedKVCache:
    """Keys and values of all layers in pages, and which pages each sequence holds.

    ``kv`` [layers, 2, num_pages, kv_heads, page_size, head_dim] in bf16, fp16 or e4m3; ``page_table`` int32 [max_seqs,
    max_pages] (-1: no page), ``seq_lens`` int32 [max_seqs], ``refcounts`` int32 [num_pages].  An e4m3 cache holds value
    / scale, ``k_scale`` and ``v_scale`` fp32 [kv_heads] (None: 1).  The tensors are the state: a caller may copy them,
    set their contents back (``copy_``; another tensor cannot take their place), or share them with its own code.  Calls
    on one cache, and replays of graphs that hold such calls, must be ordered."""

    kv = property(lambda self: self._kv)
    page_table = property(lambda self: self._page_table)
    seq_lens = property(lambda self: self._seq_lens)
    refcounts = property(lambda self: self._refcounts)
    k_scale = property(lambda self: self._k_scale)
    v_scale = property(lambda self: self._v_scale)
    status = property(lambda self: self._status)

    def __init__(self, layers: int, num_pages: int, kv_heads: int, page_size: int, head_dim: int, *, max_seqs: int,
                 max_pages: int, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
        if dtype not in _CACHE_DTYPES:
            raise ValueError("the cache holds bf16, fp16 or e4m3")
        if min(layers, num_pages, kv_heads, page_size, head_dim, max_seqs, max_pages) <= 0:
            raise ValueError("cache sizes must be positive")
        self._bind(torch.empty((layers, 2, num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device),
                   torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(max_seqs, dtype=torch.int32, device=device),
                   torch.zeros(num_pages, dtype=torch.int32, device=device), k_scale, v_scale)

    @classmethod
    def from_tensors(cls, kv: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                     refcounts: Optional[torch.Tensor] = None, *, k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None) -> "PagedKVCache":
        """A cache over tensors that the caller holds.  Without ``refcounts`` they are counted from the table's entries
        up to each sequence's length."""
        self = cls.__new__(cls)
        if kv.dim() != 6 or kv.shape[1] != 2:
            raise ValueError("kv must be [layers, 2, num_pages, kv_heads, page_size, head_dim]")
        refs = torch.zeros(kv.shape[2], dtype=torch.int32, device=kv.device) if refcounts is None else refcounts
        self._bind(kv, page_table, seq_lens, refs, k_scale, v_scale)
        if refcounts is None:
            page = page_table.clamp(0, self.num_pages - 1)
            first = torch.arange(0, self.max_pages * self.page_size, self.page_size, device=self.device)
            held = (page == page_table) & (first < seq_lens[:, None])
            refs.index_add_(0, page.flatten(), held.flatten().int())
        return self

    def _bind(self, kv, table, lens, refs, k_scale, v_scale):
        if not kv.is_cuda:
            raise ValueError("the cache must be on a CUDA device (there is no CPU path)")
        if kv.dtype not in _CACHE_DTYPES:
            raise ValueError("the cache holds bf16, fp16 or e4m3")
        self.device = kv.device
        self.layers, _, self.num_pages, self.kv_heads, self.page_size, self.head_dim = kv.shape
        for t, shape, what in ((table, (lens.numel(), table.shape[-1]), "page_table"),
                               (lens, (table.shape[0],), "seq_lens"), (refs, (self.num_pages,), "refcounts")):
            if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != self.device or not t.is_contiguous():
                raise ValueError(f"{what} must be contiguous int32 {shape} on {self.device}")
        if not kv.is_contiguous():
            raise ValueError("kv must be contiguous")
        scales = []
        for t, what in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if t is not None:
                if kv.dtype != torch.float8_e4m3fn:
                    raise ValueError(f"{what} belongs to an e4m3 cache")
                if t.dtype != torch.float32 or tuple(t.shape) != (self.kv_heads,) or t.device != self.device:
                    raise ValueError(f"{what} must be float32 [{self.kv_heads}] on {self.device}")
                t = t.contiguous()
            scales.append(t)
        self._kv, self._page_table, self._seq_lens, self._refcounts = kv, table, lens, refs
        self._k_scale, self._v_scale = scales
        self.max_seqs, self.max_pages = table.shape
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.lib = _lib.load()
        self._struct = XcbKvCache(self.layers, self.num_pages, self.kv_heads, self.page_size, self.head_dim,
                                  _CACHE_DTYPES[kv.dtype], self.max_seqs, self.max_pages, kv.data_ptr(),
                                  table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                                  None if scales[0] is None else scales[0].data_ptr(),
                                  None if scales[1] is None else scales[1].data_ptr(), self._status.data_ptr())
        self._address = ctypes.addressof(self._struct)
        self._q_dtype = None if kv.dtype == torch.float8_e4m3fn else kv.dtype
        self._plans: dict = {}       # forms of call that have passed their checks, as _PLANS
        self._rope_plans: dict = {}
        self._attn_ws: dict = {}
        nbytes = self.lib.xcb_kv_workspace_bytes(self._address)
        if nbytes == 0:
            raise ValueError("unsupported cache shape (head_dim * element bytes must be a multiple of 16, at most 256 "
                             "values; kv on a 16-byte boundary; tables and lengths within 31 bits)")
        # The page calls' workspace: zero between calls, which are ordered as they change the same tables.  Made here and
        # not by the first call, which may be captured in a graph.
        self._page_buf = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
        self._page_ws = self._page_buf.data_ptr(), nbytes

    def _attn_workspace(self, nbytes: int) -> int:
        """Address of the current stream's workspace of this size (parts of split sequences).  Sizes are few: one for
        each number of warps that the rows of a kv head can take."""
        key = (_raw_stream(self.device.index), nbytes)
        ws = self._attn_ws.get(key)
        if ws is None:
            ws = self._attn_ws[key] = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return ws.data_ptr()

    # -------------------------------------------------------------------------------------- one layer's step
    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
               seqs: torch.Tensor, rope: Rope, *, q_weight: Optional[torch.Tensor] = None,
               k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, weight_offset: float = 0.0,
               q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Norm and turn ``q`` and ``k`` as ``qk_norm_rope`` does, store k and ``v`` at ``positions`` of sequences
        ``seqs`` (int32 [T]; -1: padding, not stored) in ``layer``'s pages, and return the turned queries.  The pages
        must have been given to the sequences by ``extend``."""
        if k is None or v is None:
            raise ValueError("append needs keys and values")
        return _rope_call(self, layer, q, k, v, positions, seqs, rope, q_weight, k_weight, eps, weight_offset, q_out,
                          None)[0]

    def attend(self, layer: int, q: torch.Tensor, *, seqs: Optional[torch.Tensor] = None, window: int = 0,
               scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None):
        """Attention of new tokens over ``layer``'s pages.

        ``q`` [B, L, q_heads, D] (or [B, q_heads, D]: one token each): the last L tokens of sequences ``seqs`` (int32
        [B], default 0 .. B-1), already stored.  Each sees itself and what comes before it, with ``window`` the last
        ``window`` positions only.  ``scale`` defaults to D^-0.5.  Returns ``out`` like q, and with ``return_lse`` the
        natural log-sum-exp fp32 [B, L, q_heads]; a token that sees nothing gets zeros and -inf.  L is at most 65536, and
        L * q_heads / kv_heads 2^20."""
        layer, window = index(layer), min(index(window), 0x7fffffff)  # no sequence is longer
        if scale is not None:
            scale = float(scale)
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer must be in [0, {self.layers})")
        key = (q.dtype, q.shape, q.stride(), q.get_device(), window, scale,
               seqs is not None and (seqs.dtype, seqs.shape, seqs.get_device()),
               out is not None and (out.dtype, out.shape, out.is_contiguous(), out.get_device()))
        plan = self._plans.get(key)
        if plan is None:
            plan = self._attend_plan(q, seqs, window, scale, out)
            if len(self._plans) >= 1024:
                self._plans.clear()
            self._plans[key] = plan
        (head, rest), strides, shape, ws_bytes, like = plan
        pq = q.data_ptr()
        if strides is None or pq & 15:  # cannot be read in place: the call is that of a copy
            return self.attend(layer, q.clone(memory_format=torch.contiguous_format), seqs=seqs, window=window,
                               scale=scale, return_lse=return_lse, out=out)
        if seqs is not None and not seqs.is_contiguous():
            seqs = seqs.contiguous()
        if out is None:
            out = torch.empty_like(q) if like else torch.empty(shape, dtype=q.dtype, device=self.device)
        elif out.data_ptr() & 15:
            raise ValueError("out must be on a 16-byte boundary")
        lse = torch.empty(shape[:-1], dtype=torch.float32, device=self.device) if return_lse else None
        if shape[0]:
            ws = self._attn_workspace(ws_bytes)
            args = _ATTN_ARGS.pack(*head, layer, *rest, pq, *strides, out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                                   0 if seqs is None else seqs.data_ptr())
            _launch(self.device, self.lib.xcb_paged_attention, "xcb_paged_attention", self._address, args, ws, ws_bytes)
        return (out, lse) if return_lse else out

    def _attend_plan(self, q, seqs, window, scale, out):
        """A form of call checked: the constants of its argument block, the strides (None: q is to be copied), the
        output's shape, the workspace's size."""
        dtype = _Q_DTYPES.get(q.dtype)
        if dtype is None or q.device != self.device:
            raise ValueError(f"queries must be bf16 or fp16 on {self.device}")
        shape = tuple(q.shape)
        if len(shape) not in (3, 4) or shape[-1] != self.head_dim:
            raise ValueError(f"queries must be [batch, new_tokens, heads, {self.head_dim}]")
        s = q.stride()
        if len(shape) == 3:
            (batch, heads, dim), new, s = shape, 1, (s[0], 0, s[1], s[2])
        else:
            batch, new, heads, dim = shape
        if self._q_dtype is not None and q.dtype != self._q_dtype:
            raise ValueError("the cache holds another type than the queries")
        if window < 0:
            raise ValueError("window must be >= 0")
        if heads == 0 or heads % self.kv_heads or new == 0:
            raise ValueError(f"query heads must be a multiple of {self.kv_heads}, new tokens at least 1")
        if seqs is not None:
            _check_ints(seqs, batch, self.device, "seqs")
        elif batch > self.max_seqs:
            raise ValueError(f"the cache has {self.max_seqs} sequences")
        if out is not None and (tuple(out.shape) != shape or out.dtype != q.dtype or out.device != self.device or
                                not out.is_contiguous()):
            raise ValueError(f"out must be contiguous {shape}, of the queries' type")
        head = (batch, new, heads, dtype), (window, dim ** -0.5 if scale is None else float(scale))  # the layer between
        strides = None if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 else tuple(s[:3])
        with torch.cuda.device(self.device):
            ws_bytes = self.lib.xcb_attn_workspace_bytes(self._address, heads, new)
        if ws_bytes == 0:
            raise ValueError(f"unsupported heads: {heads} query heads over {self.kv_heads}, {new} new tokens")
        return head, strides, shape, ws_bytes, q.is_contiguous()

    # -------------------------------------------------------------------------------------- pages
    def _list(self, t: torch.Tensor, n: Optional[int], what: str) -> torch.Tensor:
        t = _check_ints(t, n, self.device, what)
        if n is None and t.shape[0] > self.max_seqs:
            raise ValueError(f"{what} lists more sequences than the cache has")
        return t

    def extend(self, seqs: torch.Tensor, new_tokens: torch.Tensor) -> None:
        """Room for ``new_tokens[i]`` more tokens in sequence ``seqs[i]`` (int32 [n] each); ``seq_lens`` grows.

        The lowest free pages go to the sequences in list order.  A part-full last page that is shared with another
        sequence is replaced by a copy, so that ``append`` never writes to a shared page; where all its holders grow
        in one call the first keeps it.  Too few free pages: nothing changes and XCB_STATUS_NO_PAGES is set."""
        seqs = self._list(seqs, None, "seqs")
        new_tokens = self._list(new_tokens, seqs.shape[0], "new_tokens")
        _launch(self.device, self.lib.xcb_kv_extend, "xcb_kv_extend", self._address, seqs.data_ptr(),
                new_tokens.data_ptr(), seqs.shape[0], *self._page_ws)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Sequence ``dst[i]``, empty before, becomes a copy of ``src[i]`` that shares its pages."""
        src = self._list(src, None, "src")
        dst = self._list(dst, src.shape[0], "dst")
        _launch(self.device, self.lib.xcb_kv_fork, "xcb_kv_fork", self._address, src.data_ptr(), dst.data_ptr(),
                src.shape[0])

    def truncate(self, seqs: torch.Tensor, lens: torch.Tensor) -> None:
        """Sequence ``seqs[i]`` keeps its first ``lens[i]`` tokens; pages that no sequence holds any more are free."""
        seqs = self._list(seqs, None, "seqs")
        lens = self._list(lens, seqs.shape[0], "lens")
        _launch(self.device, self.lib.xcb_kv_truncate, "xcb_kv_truncate", self._address, seqs.data_ptr(),
                lens.data_ptr(), seqs.shape[0])

    def free(self, seqs: torch.Tensor) -> None:
        """The sequences become empty."""
        seqs = self._list(seqs, None, "seqs")
        _launch(self.device, self.lib.xcb_kv_truncate, "xcb_kv_truncate", self._address, seqs.data_ptr(), None,
                seqs.shape[0])

    def compact(self) -> None:
        """Live pages move down into the free ids below them; the upper part of the pool is free afterwards."""
        _launch(self.device, self.lib.xcb_kv_compact, "xcb_kv_compact", self._address, *self._page_ws)

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Contents of page ``src[i]`` to page ``dst[i]`` in all layers (no dst twice, none that is also a src)."""
        src = _check_ints(src, None, self.device, "src")
        dst = _check_ints(dst, src.shape[0], self.device, "dst")
        if src.shape[0] > self.num_pages:
            raise ValueError("more pairs than pages")
        _launch(self.device, self.lib.xcb_kv_copy_pages, "xcb_kv_copy_pages", self._address, src.data_ptr(),
                dst.data_ptr(), src.shape[0])

    def check_device_status(self) -> int:
        """Synchronise the current stream and return (and clear) the cache's device status bits."""
        v = ctypes.c_int32(0)
        with torch.cuda.device(self.device):
            rc = self.lib.xcb_kv_read_status(self._address, ctypes.addressof(v),
                                             torch.cuda.current_stream(self.device).cuda_stream)
        if rc not in (_lib.XCB_OK, _lib.XCB_ERR_DEVICE):
            check(rc, "xcb_kv_read_status")
        return v.value

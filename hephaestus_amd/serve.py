"""A batched serving step of a Qwen3 model around the W8A8 linears: the paged
E4M3 KV cache, the ops of include/hephserve.h and a batch decoder on them.

    per layer, T tokens of S sequences:
        qkv = rmsnorm(x, attn_norm) @ Wqkv^T             heph_rmsnorm_quant_fp8, heph_fp8_linear
              (+ adapters)                               heph_lora_add
        q, k, v: per-head q/k norm, rotation, k/v pages  heph_qk_norm_rope_pages
        att = attention over each sequence's pages,      heph_pages_attention
              shared prefixes once for all
        x  += att @ Wo^T                                 heph_fp8_linear + ADD_RESIDUAL
        act = silu(gate) * up of rmsnorm(x) @ Wgu^T      heph_silu_mul_quant_fp8
        x  += act @ Wdown^T

The step is the batched form of the reference's forward_fp8_batched_decode
(src/hephaestus/forward.mojo:618-871), which keeps one contiguous cache per
sequence and calls attention per sequence.
"""
from __future__ import annotations

import heapq
from array import array
from itertools import accumulate

import numpy as np
import torch

from . import _lib as L
from . import decode as DEC
from . import kernels as HK
from .kernels import HephError
from .loader import Fp8Weight, Qwen3Config, Qwen3Fp8Weights

PAGE = L.PAGE_KEYS
_U8 = (torch.uint8, torch.float8_e4m3fn)
_I32, _BF16, _F32 = (torch.int32,), (torch.bfloat16,), (torch.float32,)


# The checks run before every call of a decode step: one look at each property, and the
# words of a refusal only where there is one.

def _dev(t, name: str, dtypes, numel: int, dev: int) -> int:
    """Pointer of a contiguous tensor on device dev with at least numel elements."""
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.get_device() == dev and \
            t.is_contiguous() and t.numel() >= numel:
        return t.data_ptr()
    HK._dev(t, name, dtypes)
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, not on the current device")
    raise ValueError(f"{name} has {t.numel()} elements, {numel} are needed")


def _rows(t, name: str, n: int, width: int, dev: int) -> tuple[int, int]:
    """Pointer and row stride (elements) of n rows of width bf16 values; the
    rows may lie apart (a slice of a wider buffer)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.get_device() != dev:
        raise ValueError(f"{name} must be in the current device's memory (got {t.device})")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} has dtype {t.dtype}, expected torch.bfloat16")
    shape = t.shape
    if len(shape) >= 2 and shape[0] >= n:
        if t.is_contiguous():
            if t.numel() == shape[0] * width:
                return t.data_ptr(), width
        else:
            strides, run = t.stride(), 1
            for i in range(len(shape) - 1, 0, -1):
                if strides[i] != run and shape[i] != 1:
                    break
                run *= shape[i]
            else:
                if run == width:
                    return t.data_ptr(), strides[0] if shape[0] > 1 else width
    raise ValueError(f"{name} of shape {tuple(shape)} is not {n} rows of {width} "
                     "consecutive values")


def _matrix(t, name: str, dtypes, m: int, n: int, dev: int) -> int:
    """Pointer of a contiguous [m, n] tensor, or of a larger or flat buffer in its place."""
    if isinstance(t, torch.Tensor) and t.shape == (m, n) and t.dtype in dtypes and \
            t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    if isinstance(t, torch.Tensor) and t.dim() > 1 and t.shape[-1] != n:
        raise ValueError(f"{name} of shape {tuple(t.shape)} has no rows of {n}")
    return _dev(t, name, dtypes, m * n, dev)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _at(ctx) -> tuple[int, int]:
    """The current device and the stream of a call: ctx, or its current one."""
    dev = torch.cuda.current_device()
    if ctx is None and _raw_stream is not None:
        return dev, _raw_stream(dev)
    return dev, HK._stream(ctx)


def _call(name: str, *args) -> None:
    status = getattr(L.lib(), name)(*args)
    if status != L.HEPH_OK:
        raise HephError(status, name)


def v_place(j: int) -> int:
    """Where a page's V rows hold key j (0..63)."""
    return j // 4 % 4 * 16 + j // 32 * 8 + j // 16 % 2 * 4 + j % 4


# ------------------------------------------------------------- the ops ----

def rope_table_f32(n_pos: int, theta: float = 1e6, device="cuda", ctx=None) -> torch.Tensor:
    """(cos, sin) in f32 of the 64 pairs of a 128-wide head at positions
    0..n_pos-1, [n_pos, 64, 2], the angles in double."""
    t = torch.empty(n_pos, 64, 2, dtype=torch.float32, device=device)
    dev, stream = _at(ctx)
    _call("heph_rope_table_f32", _dev(t, "table", _F32, 0, dev), n_pos, 128, theta, stream)
    return t


def _pools(k_pages, v_pages, lead: tuple, dev: int) -> tuple[int, int]:
    """Pointers of the K and V pools [*lead, ...], lead ending with n_pages and n_kv."""
    if k_pages.shape != lead + (2, PAGE, 64) or v_pages.shape != lead + (128, PAGE):
        raise ValueError(f"pools of shapes {tuple(k_pages.shape)} and {tuple(v_pages.shape)} are "
                         f"not {list(lead)} pages and heads of [2, 64, 64] and [128, 64]")
    return _dev(k_pages, "k_pages", _U8, 0, dev), _dev(v_pages, "v_pages", _U8, 0, dev)


def qk_norm_rope_pages(q_out, qkv, q_gamma, k_gamma, k_pages, v_pages, kv_inv, rope, positions,
                       slots, eps: float = 1e-6, ctx=None) -> None:
    """For each token: per-head RMSNorm of q and k, rotation by rope's row
    positions[t], q [n_tok, n_heads, 128] to q_out, k and v as E4M3 codes into
    slots[t] (page * 64 + key) of k_pages [n_pages, n_kv, 2, 64, 64] and
    v_pages [n_pages, n_kv, 128, 64]. qkv: [n_tok, n_heads + 2 n_kv, 128], its
    rows may lie apart; q_out may be qkv[:, :n_heads]. A position outside
    rope skips the token, a slot outside the pools the cache write."""
    dev, stream = _at(ctx)
    qs, ks, rs = q_out.shape, k_pages.shape, rope.shape
    if len(qs) != 3 or qs[2] != 128 or len(ks) != 5:
        raise ValueError(f"q_out of shape {tuple(qs)} and k_pages of shape {tuple(ks)} are not "
                         "[n_tok, n_heads, 128] and one layer's pool")
    n_tok, n_heads, n_pages, n_kv = qs[0], qs[1], ks[0], ks[1]
    qp, qs = _rows(q_out, "q_out", n_tok, n_heads * 128, dev)
    xp, xs = _rows(qkv, "qkv", n_tok, (n_heads + 2 * n_kv) * 128, dev)
    if n_tok == 1 and qp == xp:
        qs = xs                   # (one row has no stride of its own)
    kp, vp = _pools(k_pages, v_pages, (n_pages, n_kv), dev)
    if len(rs) != 3 or rs[1] != 64 or rs[2] != 2:
        raise ValueError(f"rope of shape {tuple(rs)} is not [n_pos, 64, 2]")
    _call("heph_qk_norm_rope_pages", qp, qs, xp, xs, _dev(q_gamma, "q_gamma", _BF16, 128, dev),
          _dev(k_gamma, "k_gamma", _BF16, 128, dev), kp, vp, n_pages,
          _dev(kv_inv, "kv_inv", _F32, 2 * n_kv, dev), _dev(rope, "rope", _F32, 0, dev),
          rs[0], _dev(positions, "positions", _I32, n_tok, dev),
          _dev(slots, "slots", _I32, n_tok, dev), n_tok, n_heads, n_kv, 128, eps, stream)


def _bind(p) -> None:
    """Keeps where a plan's own buffers are."""
    p._bound = (p.plan.data_ptr(), p.plan.numel(), p.ws.data_ptr(), p.ws.numel())
    p._dev = p.plan.get_device()


def _bound(p, dev: int) -> tuple:
    if p._dev != dev:
        raise ValueError(f"the plan is on {p.plan.device}, not on the current device")
    return p._bound


class AttentionPlan:
    """The layout of one step's attention and its workspace: update() it from
    the step's lengths in device memory, then call attention_pages for every
    layer. All sizes are fixed, so a captured step can be replayed with other
    lengths. Calls that share a plan are ordered by the caller, its making (a
    fill on the current stream) and its first use on another stream too."""

    def __init__(self, n_seqs: int, n_tok: int, n_heads: int, n_kv: int, table_pages: int,
                 n_groups: int = 0, device="cuda"):
        self.n_seqs, self.n_tok, self.n_groups = n_seqs, n_tok, n_groups
        self.n_heads, self.n_kv, self.table_pages = n_heads, n_kv, table_pages
        sizes = (n_tok, n_seqs, n_groups, n_heads, n_kv)
        nb = L.lib().heph_pages_attention_plan_bytes(*sizes)
        if nb == 0 or not 1 <= table_pages <= L.ATTN_MAX_KEYS // PAGE:
            raise HephError(L.HEPH_ERR_SHAPE, "AttentionPlan")
        # (zeros: no plan until the first update)
        self.plan = torch.zeros(nb, dtype=torch.uint8, device=device)
        self.ws = torch.empty(L.lib().heph_pages_attention_ws_bytes(*sizes), dtype=torch.uint8,
                              device=device)
        _bind(self)

    def update(self, q_start, kv_len, group_start=None, shared_pages=None, ctx=None) -> None:
        """q_start int32 [n_seqs + 1], kv_len int32 [n_seqs]; with groups
        group_start int32 [n_groups + 1], shared_pages int32 [n_groups]."""
        g = self.n_groups > 0
        if g != (group_start is not None) or g != (shared_pages is not None):
            raise ValueError(f"a plan of {self.n_groups} groups "
                             + ("needs" if g else "takes no") + " group_start and shared_pages")
        dev, stream = _at(ctx)
        plan, plan_bytes, _, _ = _bound(self, dev)
        _call("heph_pages_attention_plan", plan, plan_bytes,
              _dev(q_start, "q_start", _I32, self.n_seqs + 1, dev),
              _dev(kv_len, "kv_len", _I32, self.n_seqs, dev),
              _dev(group_start, "group_start", _I32, self.n_groups + 1, dev) if g else None,
              _dev(shared_pages, "shared_pages", _I32, self.n_groups, dev) if g else None,
              self.n_tok, self.n_seqs, self.n_groups, self.table_pages, self.n_heads, self.n_kv,
              stream)


def attention_pages(out, q, k_pages, v_pages, kv_scale, page_table, plan: AttentionPlan,
                    ctx=None) -> None:
    """out[t] = attention of token t over its sequence's keys in the pages,
    laid out by plan (updated with this step's lengths). q [n_tok, n_heads,
    128] (rows may lie apart), out contiguous; page_table int32 [n_seqs,
    table_pages]."""
    p = plan
    dev, stream = _at(ctx)
    n_pages = k_pages.shape[0]
    kp, vp = _pools(k_pages, v_pages, (n_pages, p.n_kv), dev)
    if page_table.shape != (p.n_seqs, p.table_pages):
        raise ValueError(f"page_table of shape {tuple(page_table.shape)} is not "
                         f"[{p.n_seqs}, {p.table_pages}] as planned")
    qp, qs = _rows(q, "q", p.n_tok, p.n_heads * 128, dev)
    _call("heph_pages_attention", _dev(out, "out", _BF16, p.n_tok * p.n_heads * 128, dev), qp, qs,
          kp, vp, n_pages, _dev(kv_scale, "kv_scale", _F32, 2 * p.n_kv, dev),
          _dev(page_table, "page_table", _I32, 0, dev), p.table_pages,
          *_bound(p, dev), p.n_tok, p.n_seqs, p.n_groups, p.n_heads, p.n_kv, 128, stream)


def copy_pages(k_pools, v_pools, src, dst, ctx=None) -> None:
    """Page src[i] of every layer copied to page dst[i] in both pools
    [n_layers, n_pages, ...]; src and dst are host lists of ints. A destination may
    neither repeat nor be a source."""
    ks = k_pools.shape
    if len(ks) != 6:
        raise ValueError(f"k_pools of shape {tuple(ks)} has no layers")
    dev, stream = _at(ctx)
    kp, vp = _pools(k_pools, v_pools, tuple(ks[:3]), dev)
    s, d = array("i", src), array("i", dst)
    if len(s) != len(d):
        raise ValueError(f"{len(s)} sources and {len(d)} destinations")
    _call("heph_copy_pages", kp, vp, *ks[:3], s.buffer_info()[0], d.buffer_info()[0], len(s), stream)


class LoraPlan:
    """The rows of a step grouped by adapter, and the workspace of lora_add for
    projections k -> n of up to this rank and k (of any n): update() it from the rows' adapter ids
    in device memory (an id outside [0, n_adapters): no adapter). Calls that
    share a plan are ordered by the caller, its making (a fill on the current
    stream) and its first use on another stream too."""

    def __init__(self, m: int, n_adapters: int, rank: int, k: int, n: int | None = None,
                 device="cuda"):
        self.m, self.n_adapters = m, n_adapters
        nb = L.lib().heph_lora_plan_bytes(m, n_adapters)
        wb = L.lib().heph_lora_ws_bytes(m, n_adapters, k, rank)
        if nb == 0 or wb == 0:
            raise HephError(L.HEPH_ERR_SHAPE, "LoraPlan")
        self.plan = torch.zeros(nb, dtype=torch.uint8, device=device)
        self.ws = torch.empty(wb, dtype=torch.uint8, device=device)
        _bind(self)

    def update(self, ids, ctx=None) -> None:
        dev, stream = _at(ctx)
        plan, plan_bytes, _, _ = _bound(self, dev)
        _call("heph_lora_plan", plan, plan_bytes, _dev(ids, "ids", _I32, self.m, dev), self.m, self.n_adapters, stream)


def lora_add(c, base, x, a, b, scale, plan: LoraPlan, ctx=None) -> None:
    """c = base + scale[i] * (x @ a[i]^T) @ b[i]^T per row with the adapter i
    that plan holds for it (c may be base, the projection's own output).
    a [n_adapters, rank, k], b [n_adapters, n, rank], x [m, k] bf16; c and base
    [m, n] bf16 or f32."""
    sa, sb, m = a.shape, b.shape, plan.m
    if len(sa) != 3 or len(sb) != 3 or sa[0] != sb[0] or sa[1] != sb[2]:
        raise ValueError(f"a {tuple(sa)} and b {tuple(sb)} are not [adapters, rank, k] "
                         "and [adapters, n, rank]")
    if sa[0] != plan.n_adapters:
        raise ValueError(f"{sa[0]} adapters, planned for {plan.n_adapters}")
    if c.dtype not in HK._OUT or base.dtype != c.dtype:
        raise TypeError(f"lora_add: c {c.dtype} and base {base.dtype} not supported")
    rank, k, n, dt = sa[1], sa[2], sb[1], (c.dtype,)
    dev, stream = _at(ctx)
    _call("heph_lora_add", _matrix(c, "c", dt, m, n, dev), HK._OUT[c.dtype],
          _matrix(base, "base", dt, m, n, dev), _matrix(x, "x", _BF16, m, k, dev),
          _dev(a, "a", _BF16, 0, dev), _dev(b, "b", _BF16, 0, dev),
          _dev(scale, "scale", _F32, plan.n_adapters, dev), *_bound(plan, dev), m, n, k, rank, plan.n_adapters,
          stream)


# --------------------------------------------------------------- the cache ----

class Sequence:
    """A sequence's pages (ids, in key order) and its number of keys."""

    def __init__(self):
        self.pages: list[int] = []
        self.length = 0


class PagedKVCache:
    """K and V pools of all layers with E4M3 codes, k [n_layers, n_pages, n_kv,
    2, 64, 64] and v [n_layers, n_pages, n_kv, 128, 64], f32 scales [n_layers,
    2*n_kv] and their reciprocals, and which sequence holds which page. A page
    may belong to several sequences (a shared prefix): it is freed with the
    last of them. Page copies run on the current stream (or ctx's); steps on other
    streams are ordered by the caller."""

    def __init__(self, cfg: Qwen3Config, n_pages: int, device="cuda"):
        if cfg.head_dim != 128:
            raise ValueError("head_dim must be 128")
        if n_pages < 1:
            raise ValueError(f"a cache of {n_pages} pages")
        self.cfg, self.n_pages = cfg, n_pages
        shape = (cfg.n_layers, n_pages, cfg.n_kv_heads)
        self.k = torch.zeros(*shape, 2, PAGE, 64, dtype=torch.uint8, device=device)
        self.v = torch.zeros(*shape, 128, PAGE, dtype=torch.uint8, device=device)
        self.scale = torch.ones(cfg.n_layers, 2 * cfg.n_kv_heads, dtype=torch.float32,
                                device=device)
        self.inv = torch.ones_like(self.scale)
        self._free = list(range(n_pages))          # a heap: the lowest page first
        self._users = [0] * n_pages
        self._seqs: dict[Sequence, None] = {}      # in the order of their making

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise MemoryError(f"{n} pages wanted, {len(self._free)} free")
        got = [heapq.heappop(self._free) for _ in range(n)]
        for p in got:
            self._users[p] = 1
        return got

    def _drop(self, page: int) -> None:
        self._users[page] -= 1
        if self._users[page] == 0:
            heapq.heappush(self._free, page)

    def _own(self, seq: Sequence) -> Sequence:
        if not isinstance(seq, Sequence) or seq not in self._seqs:
            raise ValueError("the sequence is not in this cache")
        return seq

    def new(self) -> Sequence:
        """An empty sequence."""
        seq = Sequence()
        self._seqs[seq] = None
        return seq

    def extend(self, seq: Sequence, n: int) -> list[int]:
        """Room for n more keys; their slots. Nothing changes if the pages do
        not suffice."""
        if n < 0:
            raise ValueError(f"{n} keys")
        self._own(seq)
        if seq.length + n > L.ATTN_MAX_KEYS:
            raise ValueError(f"{seq.length + n} keys > {L.ATTN_MAX_KEYS}")
        seq.pages += self._take(-(-(seq.length + n) // PAGE) - len(seq.pages))
        keys = range(seq.length, seq.length + n)
        seq.length += n
        return [seq.pages[j // PAGE] * PAGE + j % PAGE for j in keys]

    def fork(self, seq: Sequence, n: int = 1, ctx=None) -> list[Sequence]:
        """n sequences with seq's keys: its full pages are shared, its partly
        filled last page is copied for each (on the current stream)."""
        self._own(seq)
        if n < 0:
            raise ValueError(f"{n} forks")
        full = seq.length // PAGE
        tails = self._take(n if seq.length % PAGE else 0)
        if tails:
            try:
                copy_pages(self.k, self.v, [seq.pages[full]] * n, tails, ctx)
            except BaseException:
                for p in tails:
                    self._drop(p)
                raise
        made = []
        for i in range(n):
            s = self.new()
            s.pages, s.length = seq.pages[:full] + tails[i:i + 1], seq.length
            for p in seq.pages[:full]:
                self._users[p] += 1
            made.append(s)
        return made

    def free(self, seq: Sequence) -> None:
        """The sequence leaves the cache; pages that no other one holds are free."""
        self._own(seq)
        for p in seq.pages:
            self._drop(p)
        del self._seqs[seq]
        seq.pages, seq.length = [], 0

    def compact(self, ctx=None) -> int:
        """Live pages move down into the lowest ids, so that the pages from the
        number of live ones on are free; returns how many moved. Page tables
        made before are stale."""
        live = self.n_pages - len(self._free)
        dst = sorted(p for p in self._free if p < live)
        src = [p for p in range(live, self.n_pages) if self._users[p]]
        copy_pages(self.k, self.v, src, dst, ctx)
        to = dict(zip(src, dst))
        for s in self._seqs:
            s.pages = [to.get(p, p) for p in s.pages]
        for a, b in to.items():
            self._users[b], self._users[a] = self._users[a], 0
        self._free = list(range(live, self.n_pages))
        return len(src)


# ------------------------------------------------------------- the decoder ----

class LoraWeights:
    """Adapters of one model: per layer and projection ("qkv", "o", "gate_up",
    "down"; those absent have none) the pair (a [n_adapters, rank, k], b
    [n_adapters, n, rank]), and scale f32 [n_adapters]."""

    def __init__(self, scale: torch.Tensor, layers: list[dict]):
        self.scale, self.layers = scale, layers
        self.n_adapters = scale.numel()
        for i, d in enumerate(layers):
            for name, (a, b) in d.items():
                if name not in _PROJECTIONS:
                    raise ValueError(f"layer {i}: no projection is named {name!r}")
                if a.dim() != 3 or b.dim() != 3 or a.shape[:2] != (b.shape[0], b.shape[2]) or \
                        a.shape[0] != self.n_adapters or not _rank_ok(a.shape[1]):
                    raise ValueError(f"layer {i}, {name}: a {tuple(a.shape)} and b {tuple(b.shape)} "
                                     f"are not [{self.n_adapters}, rank, k] and "
                                     f"[{self.n_adapters}, n, rank], rank a multiple of 8 up to 128")
        pairs = [p for d in layers for p in d.values()]
        self.max_rank = max((a.shape[1] for a, _ in pairs), default=8)
        self.max_k = max((a.shape[2] for a, _ in pairs), default=128)


_PROJECTIONS = ("qkv", "o", "gate_up", "down")


def _rank_ok(rank: int) -> bool:
    return 8 <= rank <= 128 and rank % 8 == 0


def _common(a: list[int], b: list[int]) -> int:
    """How many first entries two lists share, halving a range that holds the end."""
    m, end = 0, min(len(a), len(b))
    while m < end:
        mid = (m + end + 1) // 2
        if a[m:mid] == b[m:mid]:
            m = mid
        else:
            end = mid - 1
    return m


def _groups(seqs: list[Sequence]) -> tuple[list[int], list[int]]:
    """Runs of neighbouring sequences that share their first pages:
    group_start and shared_pages. A run grows while its common prefix keeps
    at least half of the pages its first two share."""
    start, shared = [0], []
    n = first = None
    for i in range(1, len(seqs) + 1):
        if i < len(seqs):
            m = _common(seqs[start[-1]].pages, seqs[i].pages)
            if n is None:
                if m > 0:
                    n = first = m
                    continue
            elif 2 * min(n, m) >= first:
                n = min(n, m)
                continue
        shared.append(n or 0)
        start.append(i)
        n = None
    return start, shared


class Qwen3BatchDecoder:
    """A step of many sequences: prompts or single tokens, behind whatever
    their caches hold."""

    def __init__(self, weights: Qwen3Fp8Weights, kv: PagedKVCache, n_pos: int = 40960,
                 lora: LoraWeights | None = None):
        if not weights.embed.block:
            raise ValueError("the decoder takes 128x128 block-scaled weights")
        if lora is not None and len(lora.layers) != weights.cfg.n_layers:
            raise ValueError(f"adapters of {len(lora.layers)} layers, "
                             f"{weights.cfg.n_layers} in the model")
        for i, d in enumerate(lora.layers if lora is not None else []):
            for name, (a, b) in d.items():
                fw = getattr(weights.layers[i], name)
                if (b.shape[1], a.shape[2]) != (fw.N, fw.K):
                    raise ValueError(f"layer {i}, {name}: adapters {a.shape[2]} -> {b.shape[1]} "
                                     f"beside a projection {fw.K} -> {fw.N}")
        self.w, self.kv, self.lora = weights, kv, lora
        self.n_pos = min(n_pos, L.ATTN_MAX_KEYS)
        self.rope = rope_table_f32(self.n_pos, weights.cfg.theta, device=weights.embed.w.device)

    def _linear(self, c, x, fw: Fp8Weight, K: int, ws, residual: bool = False,
                quantized: bool = False) -> None:
        fn = HK.linear_add_residual_fp8 if residual else HK.linear_fp8
        fn(c, x, fw.w, fw.scale, ws[0], ws[1], c.shape[0], fw.N, K, do_quantize=not quantized)

    def step(self, tokens: list[list[int]], seqs: list[Sequence],
             adapters: list[int] | None = None) -> torch.Tensor:
        """tokens[i] (one or more) enter sequence seqs[i], with adapter
        adapters[i] (-1: none). Returns the f32 logits [len(seqs), vocab] after
        each sequence's last token. A step that raises leaves the sequences as
        they were."""
        cfg, kv = self.w.cfg, self.kv
        if len(tokens) != len(seqs) or not seqs or any(len(t) < 1 for t in tokens):
            raise ValueError("every sequence brings one token or more")
        if len({id(s) for s in seqs}) != len(seqs):
            raise ValueError("a sequence appears twice")
        if adapters is not None and (self.lora is None or len(adapters) != len(seqs)):
            raise ValueError("adapters without weights, or not one a sequence")
        if len(seqs) > L.PAGES_MAX_SEQS:
            raise ValueError(f"{len(seqs)} sequences > {L.PAGES_MAX_SEQS}")
        if any(not 0 <= i < cfg.vocab for t in tokens for i in t):
            raise ValueError(f"a token outside the vocabulary of {cfg.vocab}")
        if adapters is not None and any(not -1 <= a < self.lora.n_adapters for a in adapters):
            raise ValueError(f"an adapter outside the {self.lora.n_adapters} that there are")
        need = 0
        for t, s in zip(tokens, seqs):
            kv._own(s)
            if s.length + len(t) > self.n_pos:
                raise ValueError(f"position {s.length + len(t) - 1} outside the rotation table "
                                 f"of {self.n_pos}")
            need += -(-(s.length + len(t)) // PAGE) - len(s.pages)
        if need > kv.free_pages:
            raise MemoryError(f"{need} pages wanted, {kv.free_pages} free")
        before = [(s, s.length, len(s.pages)) for s in seqs]
        try:
            return self._run(tokens, seqs, adapters)
        except BaseException:
            for s, length, pages in before:
                for p in s.pages[pages:]:
                    kv._drop(p)
                s.length, s.pages = length, s.pages[:pages]
            raise

    def _layout(self, tokens, seqs, adapters) -> list:
        """The sequences take their tokens; the int32 values that the step's ops read: tokens,
        positions, slots, q_start, kv_len, group_start, shared_pages, adapter ids and the page
        table [len(seqs), most pages]."""
        flat = [i for t in tokens for i in t]
        positions = [s.length + i for t, s in zip(tokens, seqs) for i in range(len(t))]
        slots = [i for t, s in zip(tokens, seqs) for i in self.kv.extend(s, len(t))]
        q_start = [0, *accumulate(len(t) for t in tokens)]
        ids = [-1] * len(flat) if adapters is None else [a for t, a in zip(tokens, adapters) for _ in t]
        table = np.full((len(seqs), max(len(s.pages) for s in seqs)), -1, dtype=np.int32)
        for row, s in zip(table, seqs):
            row[:len(s.pages)] = s.pages
        rows = [flat, positions, slots, q_start, [s.length for s in seqs], *_groups(seqs), ids]
        # (array: what is no whole number is refused, not rounded)
        return [np.frombuffer(array("i", r), dtype=np.int32) for r in rows] + [table]

    def _run(self, tokens, seqs, adapters) -> torch.Tensor:
        cfg, w, kv = self.w.cfg, self.w, self.kv
        parts = self._layout(tokens, seqs, adapters)
        # one upload for everything the step's ops read
        meta = torch.from_numpy(np.concatenate([p.ravel() for p in parts])).to(w.embed.w.device)
        (tok, pos, slot, q_start, kv_len, group_start, shared, ids,
         table) = meta.split([p.size for p in parts])
        T, S, G, width = tok.numel(), len(seqs), shared.numel(), parts[-1].shape[1]

        H, I, Q, KV = cfg.hidden, cfg.inter, cfg.q_out, cfg.kv_out
        dev = w.embed.w.device
        bf = dict(dtype=torch.bfloat16, device=dev)
        x, xn = torch.empty(T, H, **bf), torch.empty(T, H, **bf)
        qkv, att = torch.empty(T, Q + 2 * KV, **bf), torch.empty(T, Q, **bf)
        gu, act = torch.empty(T, 2 * I, **bf), torch.empty(T, I, **bf)
        q_bytes = max(L.lib().heph_fp8_linear_ws_bytes(T, n, k) for n, k in
                      ((Q + 2 * KV, H), (H, Q), (2 * I, H), (H, I)))
        ws = (torch.empty(q_bytes, dtype=torch.uint8, device=dev),
              torch.empty(T * max(H, Q, I) // 128, dtype=torch.float32, device=dev))
        plan = AttentionPlan(S, T, cfg.n_heads, cfg.n_kv_heads, width, n_groups=G, device=dev)
        plan.update(q_start, kv_len, group_start, shared)
        table = table.view(S, width)
        lora = self.lora if adapters is not None else None
        if lora is not None:
            lplan = LoraPlan(T, lora.n_adapters, lora.max_rank, lora.max_k, device=dev)
            lplan.update(ids)

        def adapt(li, op, c, a):
            if lora is not None and op in lora.layers[li]:
                lora_add(c, c, a, *lora.layers[li][op], lora.scale, lplan)

        def norm_linear(li, op, c, gamma, fw):
            if lora is not None and op in lora.layers[li]:
                # the adapter takes the normalized row too
                DEC.rmsnorm(xn, x, gamma, cfg.eps)
                self._linear(c, xn, fw, H, ws)
                adapt(li, op, c, xn)
            else:
                HK.rmsnorm_quant_fp8(ws[0], ws[1], x, gamma, T, H, cfg.eps)
                self._linear(c, None, fw, H, ws, quantized=True)

        DEC.embed_fp8(x, w.embed.w, w.embed.scale, tok)
        q = att.view(T, cfg.n_heads, 128)
        qs = qkv.view(T, -1, 128)[:, :cfg.n_heads]
        for li, lw in enumerate(w.layers):
            norm_linear(li, "qkv", qkv, lw.attn_norm, lw.qkv)
            qk_norm_rope_pages(qs, qkv.view(T, -1, 128), lw.q_norm, lw.k_norm, kv.k[li], kv.v[li],
                               kv.inv[li], self.rope, pos, slot, cfg.eps)
            attention_pages(q, qs, kv.k[li], kv.v[li], kv.scale[li], table, plan)
            self._linear(x, att, lw.o, Q, ws, residual=True)
            adapt(li, "o", x, att)
            norm_linear(li, "gate_up", gu, lw.ffn_norm, lw.gate_up)
            if lora is not None and "down" in lora.layers[li]:
                # (the op takes gate and up each in one piece)
                DEC.silu_mul(act, gu[:, :I].contiguous(), gu[:, I:].contiguous(), T * I)
                self._linear(x, act, lw.down, I, ws, residual=True)
                adapt(li, "down", x, act)
            else:
                HK.silu_mul_quant_fp8(ws[0], ws[1], gu, gu[:, I:], T, I, 2 * I)
                self._linear(x, None, lw.down, I, ws, residual=True, quantized=True)
        last = x[q_start[1:].long() - 1]
        logits = torch.empty(S, cfg.vocab, dtype=torch.float32, device=dev)
        HK.rmsnorm_quant_fp8(ws[0], ws[1], last, w.final_norm, S, H, cfg.eps)
        self._linear(logits, None, w.embed, H, ws, quantized=True)
        return logits

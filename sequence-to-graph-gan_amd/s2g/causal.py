"""Host side of the causal-transformer operators: rotary positions, attention over packed sequences with grouped heads
(and its gradient), and the paged key/value cache that serves single tokens and chunks.  Plans are laid out here from
lengths the host knows; every product and reduction runs in libs2g kernels (include/s2g.h)."""
from __future__ import annotations

import contextlib
import ctypes
import math
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .lib import S2GError, S2GPacked, S2GPaged, S2GRotary, call, get
from .ops import cur_stream, ptr, stream_ptr

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
TILE = 128                       # rows, or keys, of one workgroup


def _launch(device: int, name: str, *args) -> None:
    """A kernel call on the tensors' device, whichever is current, and on its current stream."""
    if device == torch._C._cuda_getDevice():
        call(name, *args, stream_ptr())
    else:
        with torch.cuda.device(device):
            call(name, *args, stream_ptr())


def current_device(x: torch.Tensor):
    """x's device as the current one, for kernels that go to the current device's stream."""
    if not x.is_cuda or x.get_device() == torch._C._cuda_getDevice():
        return contextlib.nullcontext()
    return torch.cuda.device(x.get_device())


def _check(what: str, **tensors: Optional[torch.Tensor]) -> None:
    """One GPU, one element type the kernels have."""
    first = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise S2GError(f"{what}: {name} must be a GPU tensor (MI355X-only implementation, no CPU path)")
        first = t if first is None else first
        if t.dtype not in TYPES:
            raise S2GError(f"{what}: {name} must be float32, bfloat16 or float16, got {t.dtype}")
        if t.dtype != first.dtype or t.device != first.device:
            raise S2GError(f"{what}: {name} ({t.dtype}, {t.device}) differs from {first.dtype}, {first.device}")


def _strides(x: torch.Tensor) -> Tuple[int, int]:
    """Token and head stride of [tokens, heads, dim]; those of a single token or head are what they would be."""
    h = x.stride(1) if x.shape[1] > 1 else x.shape[2]
    return (x.stride(0) if x.shape[0] > 1 else x.shape[1] * h), h


def _fetchable(x: torch.Tensor, group: int = 1) -> bool:
    """Rows that the kernels can fetch in 16-byte units, 64 of them (of `group` heads each, side by side) within 31 bits of
    each other, as far as their strides go."""
    unit = 16 // x.element_size()
    t, h = _strides(x)
    return (x.stride(2) == 1 and t % unit == 0 and h % unit == 0 and max(t, h) < 1 << 22
            and (64 * t + group * h) * x.element_size() < 0x7ffffe00)


def _no_tangent(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """The kernels write new tensors through their addresses: a forward-mode tangent would be lost without a word, also where
    no gradient is asked for."""
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise S2GError(f"{what}: no forward-mode derivative (a tensor carries a tangent)")


def _once(backward):
    """once_differentiable, whose bookkeeping (10 us a call) is needed only where a graph of the gradient is being made."""
    slow = once_differentiable(backward)

    def choose(ctx, *grads):
        _no_tangent("gradient of a causal operator", *grads)
        return slow(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return choose


def _new(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _copy(x: torch.Tensor) -> torch.Tensor:
    return x.clone(memory_format=torch.contiguous_format)


def _layout(*tensors) -> tuple:
    """What the checks of a call and its plan go by: shapes, strides, types, devices; never addresses or values."""
    return tuple([(t.dtype, t.shape, t.stride(), t.get_device()) for t in tensors])


def _dense(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(2) == 1 else _copy(x)      # contiguous() keeps the strides of empty tensors


def _attention_shapes(what: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise S2GError(f"{what}: q, k and v must be [tokens, heads, dim]")
    if k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise S2GError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} must agree, and q {tuple(q.shape)} share their dim")
    _attention_heads(what, q.shape[1], k.shape[1], q.shape[2])


def _attention_heads(what: str, H: int, Hk: int, D: int) -> None:
    if Hk == 0 or H % Hk or not 1 <= H // Hk <= 128:
        raise S2GError(f"{what}: {H} query heads must be 1 to 128 times the {Hk} key/value heads")
    if D % 8 or not 8 <= D <= 128:
        raise S2GError(f"{what}: head dim must be a multiple of 8, at most 128, got {D}")


def _scale(what: str, scale: Optional[float], D: int) -> float:
    s = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 1e-30 <= s <= 1e30:
        raise S2GError(f"{what}: scale must be positive, 1e-30 to 1e30, got {scale}")
    return s


def _no_capture(what: str = "a batch layout") -> None:
    if torch.cuda.is_current_stream_capturing():
        raise S2GError(f"{what} cannot be made inside a graph capture: use it once before")


# What batches, caches and modules keep is made outside inference mode, whichever mode its first call runs in: autograd saves no
# inference tensor, and training steps may come later.
_lasting = torch.inference_mode(False)


@_lasting
def _on_device(values, device) -> torch.Tensor:
    """An int32 device copy of host integers, complete on return (any stream may use it)."""
    _no_capture()
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).to(device)


@_lasting
def lasting_copy(what: str, x: torch.Tensor, device) -> torch.Tensor:
    """x on `device`, for its owner to keep."""
    _no_capture(what)
    return x.to(device)


def _stream(device: int) -> torch.cuda.Stream:
    """A device's current stream."""
    return cur_stream() if device == torch._C._cuda_getDevice() else torch.cuda.current_stream(device)


def _hold(device: int, *tensors: torch.Tensor) -> None:
    """Tensors that a launch on the current stream reads: their memory is not given away before it is done, whichever stream
    they were made on and whenever they go (0.3 us each)."""
    stream = _stream(device)
    for t in tensors:
        t.record_stream(stream)


def _lend(owner, *tensors: torch.Tensor) -> None:
    """The same for a batch's own tensors, which were made on owner.stream."""
    if torch._C._cuda_getCurrentRawStream(owner.device.index) != owner.stream.cuda_stream:
        _hold(owner.device.index, *tensors)


class _Fixed:
    """Attributes are set once: plans have been checked against them."""
    __slots__ = ()

    def __setattr__(self, name, value):
        if hasattr(self, name):
            raise S2GError(f"{type(self).__name__}: {name} is set for good when the batch is made (tensors may be written in place)")
        object.__setattr__(self, name, value)


# ---------------------------------------------------------------------------------------------------------------- rotary
@_lasting
def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 4096, device="cuda") -> Tuple[torch.Tensor, float]:
    """(frequencies [rotary_dim / 2] in radians per position, float64; multiplier) for apply_rotary.
    scaling, for contexts `factor` times as long as the original_length a model was trained at:
      None      base^(-2i / rotary_dim)
      "linear"  every frequency divided by factor
      "base"    base raised to base factor^(rotary_dim / (rotary_dim - 2)): the slowest pair is stretched by factor, the
                quickest not at all
      "ramp"    by how often a pair turns within original_length: at most once, stretched by factor; 32 times or more,
                left alone; between, blended; multiplier 0.1 log(factor) + 1"""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise S2GError(f"rotary_frequencies: rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 0 or not factor > 0:
        raise S2GError("rotary_frequencies: base and factor must be positive")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    f, multiplier = base ** -i, 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "base":
        if rotary_dim > 2:
            f = (base * factor ** (rotary_dim / (rotary_dim - 2))) ** -i
    elif scaling == "ramp":
        turns = original_length * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        f, multiplier = f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    elif scaling is not None:
        raise S2GError(f"rotary_frequencies: scaling must be None, 'linear', 'base' or 'ramp', got {scaling!r}")
    return f.to(device), multiplier


def _frequencies(what: str, frequencies: torch.Tensor, device: int, D: int) -> int:
    """How many features `frequencies` turn."""
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64 or frequencies.get_device() != device or not frequencies.is_contiguous():
        raise S2GError(f"{what}: frequencies must be a contiguous float64 vector on the tensors' device")
    R = 2 * frequencies.numel()
    if R > D or D > 256:
        raise S2GError(f"{what}: {R} rotary features of head dim {D} (at most 256)")
    return R


def _rotary_dims(q, k, v, R, interleaved, multiplier, backward) -> S2GRotary:
    if not math.isfinite(multiplier):
        raise S2GError("rotary positions: multiplier must be finite")
    (ql, qh), (kl, kh), (vl, vh) = (_strides(x) if x is not None else (0, 0) for x in (q, k, v))
    return S2GRotary(TYPES[q.dtype], q.shape[1], 0 if k is None else k.shape[1], q.shape[2], R, int(interleaved), int(backward), multiplier,
                     q.shape[0], ql, qh, kl, kh, vl, vh)


class _TurnPlan:
    """The kernel's arguments for q and k laid out like these, checked once."""
    kept: dict = {}

    def __init__(self, q, k, R, interleaved, multiplier, backward):
        self.copy = q.stride(2) != 1 or (k is not None and k.stride(2) != 1)
        self.rows, self.device = q.shape[0], q.get_device()
        self.args = ctypes.byref(_rotary_dims(q, k, None, R, interleaved, multiplier, backward))


def _turn(q, k, positions, frequencies, interleaved, multiplier, backward):
    how = (frequencies.numel(), interleaved, multiplier, backward)
    key = (_layout(q) if k is None else _layout(q, k), how)
    plan = _TurnPlan.kept.get(key)
    if plan is None:
        if len(_TurnPlan.kept) >= 256:                 # batches of ever new sizes
            _TurnPlan.kept.clear()
        plan = _TurnPlan.kept[key] = _TurnPlan(q, k, 2 * how[0], *how[1:])
    if plan.copy:
        return _turn(_dense(q), None if k is None else _dense(k), positions, frequencies, interleaved, multiplier, backward)
    qo, ko = _new(q), None if k is None else _new(k)
    if plan.rows:
        _hold(plan.device, positions, frequencies)         # a batch's and a module's own, which may go before the launch is done
        _launch(plan.device, "s2g_rotary", q.data_ptr(), ptr(k), positions.data_ptr(), frequencies.data_ptr(), qo.data_ptr(), ptr(ko), plan.args)
    return qo, ko


class RotaryFn(torch.autograd.Function):
    """(q, k) turned by their tokens' positions; the gradient is the turn by the negative angles."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved, multiplier):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (interleaved, multiplier)
        return _turn(q, k, positions, frequencies, interleaved, multiplier, False)

    @staticmethod
    @_once
    def backward(ctx, dq, dk):
        positions, frequencies = ctx.saved_tensors
        return (*_turn(dq, dk, positions, frequencies, *ctx.how, True), None, None, None, None)


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor,
                 interleaved: bool = False, multiplier: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turns pair i of the first 2 len(frequencies) features of every head by positions[token] * frequencies[i] radians
    and scales it by multiplier; further features pass through.  q [tokens, heads, dim], k [tokens, kv heads, dim] or
    None, fp32 / bf16 / fp16 with any strides; positions int32 [tokens]; pairs are features (2i, 2i + 1) if interleaved,
    else (i, i + len(frequencies)).  Returns new tensors; differentiable in q and k."""
    _check("apply_rotary", q=q, k=k)
    _no_tangent("apply_rotary", q, k, frequencies)
    if q.dim() != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
        raise S2GError("apply_rotary: q and k must be [tokens, heads, dim] with the same tokens and dim")
    if q.shape[1] == 0 or q.shape[2] == 0 or (k is not None and k.shape[1] == 0):
        raise S2GError("apply_rotary: no heads, or heads without features")
    if positions.shape != q.shape[:1] or positions.dtype != torch.int32 or positions.device != q.device or not positions.is_contiguous():
        raise S2GError(f"apply_rotary: positions must be contiguous int32 [{q.shape[0]}] on {q.device}")
    _frequencies("apply_rotary", frequencies, q.get_device(), q.shape[2])
    if not torch.is_grad_enabled() or not (q.requires_grad or (k is not None and k.requires_grad)):
        return _turn(q, k, positions, frequencies, bool(interleaved), float(multiplier), False)
    return RotaryFn.apply(q, k, positions, frequencies, bool(interleaved), float(multiplier))


# ----------------------------------------------------------------------------------------------------- packed sequences
class _WorkLists:
    """The kernels' work lists for a batch of sequences, made when they are first used."""

    def __init__(self, q_len: np.ndarray, k_len: np.ndarray, device, stream=None):
        self.q_len, self.k_len, self.device, self.stream = q_len, k_len, device, stream
        self.q_start, self.k_start = np.cumsum(q_len) - q_len, np.cumsum(k_len) - k_len
        self.kept: dict = {}

    def _tiles(self, count: np.ndarray) -> Tuple[np.ndarray, np.ndarray]:
        """(sequence, which) of every tile of `count` rows or keys a sequence."""
        n = -(-count // TILE)
        return np.repeat(np.arange(n.size), n), np.arange(int(n.sum())) - np.repeat(np.cumsum(n) - n, n)

    def _list(self, seq, tile, row_lo, row_hi, slot) -> torch.Tensor:
        entry = np.empty((seq.size, 8), dtype=np.int32)
        for i, column in enumerate((self.q_start[seq], self.q_len[seq], self.k_start[seq], self.k_len[seq], tile, row_lo, row_hi, slot)):
            entry[:, i] = column
        if self.stream is not None:
            _no_capture()                                  # asked of the caller's stream: the batch's own is not being captured
        with torch.cuda.stream(self.stream):
            return _on_device(entry, self.device)

    def query_tiles(self, group: int, causal: bool) -> torch.Tensor:
        """Work list of the query side for `group` query heads to a kv head: the longest first, so that what remains at the
        end of the launch is short."""
        got = self.kept.get((group, causal))
        if got is None:
            count = self.q_len * group
            seq, tile = self._tiles(count)
            work = self.k_len[seq]
            if causal:
                last = (np.minimum((tile + 1) * TILE, count[seq]) - 1) // group
                work = np.minimum(work, last + 1 + (self.k_len - self.q_len)[seq])
            order = np.argsort(-work, kind="stable")
            got = self.kept[group, causal] = self._list(seq[order], tile[order], 0, 0, -1)
        return got

    def key_tiles(self, group: int, causal: bool, kv_heads: int, exact: bool = False) -> Tuple[torch.Tensor, torch.Tensor, int]:
        """Work list of the key side, the tiles that are cut, and how many slots they need.  A tile is as much work as it has
        rows; none is left with more than half of what falls to a compute unit, but 256 rows are not worth a slot.  exact:
        fp32, whose products take eight times as long: 128 rows, but all that falls to a compute unit, where several tiles
        overlap.  (Kernel and sum, us.  16 / 4 bf16 heads of 64, 4 x 500 tokens, at least 128 / 256 / 512 rows: 28 / 28 / 39; 12 /
        1 fp16 heads of 64, 96 up to 203: 38 / 39 / 42; 8 bf16 heads of 128, 1000: 36 / 29 / 32; 2 fp32 heads of 96, 8 up to 722:
        49 / 76 / 124.)"""
        got = self.kept.get((group, causal, kv_heads, exact))
        if got is None:
            seq, tile = self._tiles(self.k_len)
            rows = (self.q_len * group)[seq]
            first = np.maximum(0, tile * TILE - (self.k_len - self.q_len)[seq]) * group // TILE * TILE if causal else np.zeros_like(rows)
            work = np.maximum(0, rows - first)
            most = max(128 if exact else 256, -(-int(work.sum()) * kv_heads // (256 if exact else 512) // TILE) * TILE)
            parts = np.maximum(1, -(-work // most))
            each = -(-work // parts // TILE) * TILE                      # whole tiles of rows
            of = np.repeat(np.arange(parts.size), parts)
            nth = np.arange(of.size) - np.repeat(np.cumsum(parts) - parts, parts)
            lo = np.minimum(first[of] + nth * each[of], rows[of])
            hi = np.minimum(lo + each[of], rows[of])
            is_cut = parts[of] > 1
            slot = np.where(is_cut, np.cumsum(is_cut) - 1, -1)
            order = np.argsort(lo - hi, kind="stable")
            cut = np.flatnonzero(parts > 1)
            start = np.cumsum(parts) - parts
            got = self.kept[group, causal, kv_heads, exact] = (
                self._list(seq[of][order], tile[of][order], np.where(is_cut, lo, 0)[order], np.where(is_cut, hi, rows[of])[order], slot[order]),
                self._list(seq[cut], tile[cut], parts[cut], 0, slot[start[cut]]), int(is_cut.sum()))
        return got


class PackedSequences(_Fixed):
    """The layout of a batch of sequences that lie one after another: `lengths` tokens each (zeros allowed), and
    `key_lengths` keys each where those differ (the newest tokens of longer sequences: query i of n sees the first
    key_length - n + i + 1 keys when causal).  Rows behind the last sequence belong to nobody.
    starts, positions: int32 device tensors, the first row of every sequence (and the end), and every row's position in
    its sequence's keys.  Made once per batch, and kept for forward and backward; the work lists of a grouping of heads
    are laid out when it is first used.  A captured graph reads them on every replay: keep the batch as long as the graph."""

    @_lasting
    def __init__(self, lengths: Sequence[int], device="cuda", key_lengths: Optional[Sequence[int]] = None):
        q = np.asarray(lengths, dtype=np.int64).reshape(-1)
        k = q if key_lengths is None else np.asarray(key_lengths, dtype=np.int64).reshape(-1)
        if q.shape != k.shape or q.size == 0 or q.min() < 0 or k.min() < 0 or q.sum() >= 1 << 30 or k.sum() >= 1 << 30:
            raise S2GError("PackedSequences: lengths and key_lengths must be as many, not negative, below 2^30 in all")
        device = torch.device(device)
        if device.type != "cuda":
            raise S2GError("PackedSequences: needs a GPU device")
        self.device = torch.device("cuda", torch.cuda.current_device()) if device.index is None else device
        self.rows, self.key_rows = int(q.sum()), int(k.sum())
        with torch.cuda.device(self.device):
            both = _on_device(np.concatenate(([0], np.cumsum(q), np.arange(self.rows) - np.repeat(np.cumsum(q) - k, q))), self.device)
        self.starts, self.positions = both[:q.size + 1], both[q.size + 1:]
        self._work, self._plans = _WorkLists(q, k, self.device, torch.cuda.current_stream(self.device)), {}


class _PackedPlan:
    """One layout of q, k and v over one batch: checked once, its work lists and the kernels' arguments kept."""

    def __init__(self, pack, q, k, v, causal, scale):
        _check("packed_attention", q=q, k=k, v=v)
        _attention_shapes("packed_attention", q, k, v)
        if pack.device != q.device:
            raise S2GError(f"packed_attention: pack must be PackedSequences on {q.device}")
        if q.shape[0] < pack.rows or k.shape[0] < pack.key_rows:
            raise S2GError(f"packed_attention: the layout needs {pack.rows} queries and {pack.key_rows} keys, got {q.shape[0]} and {k.shape[0]}")
        if q.shape[0] * q.shape[1] >= 1 << 30 or k.shape[0] >= 1 << 30:
            raise S2GError("packed_attention: 2^30 rows or more")
        (R, H, D), (M, Hk, _) = q.shape, k.shape
        if H * D >= 1 << 22:                           # no layout of the output's gradient could be fetched
            raise S2GError("packed_attention: tokens of q have 2^22 elements or more")
        self.copies = [not _fetchable(q, H // Hk), not _fetchable(k), not _fetchable(v)]
        self.strides = (q.stride(), k.stride(), v.stride())
        self.work, self.causal, self.group, self.kv_heads = pack._work, causal, H // Hk, Hk
        self.device, self.rows, self.key_rows = q.get_device(), pack.rows, pack.key_rows
        self.some = pack.rows > 0 and pack.key_rows > 0
        self.stats = Hk * R * self.group
        self.fields = (TYPES[q.dtype], H, Hk, D, int(causal), _scale("packed_attention", scale, D))
        self.size, self.whole = (R, M), R == pack.rows and M == pack.key_rows
        self.fwd = ctypes.byref(S2GPacked(*self.fields, *_strides(q), *_strides(k), *_strides(v), H * D, D, R, M))
        self.q_tiles = self.work.query_tiles(self.group, causal)
        self.q_list = (ptr(self.q_tiles), self.q_tiles.shape[0])
        self.bwd: dict = {}

    def backward(self, q, k, v, do):
        """(arguments, key-side lists, floats of workspace, the lists' tensors) for inputs and a gradient laid out like these."""
        key = (q.stride(), k.stride(), v.stride(), do.stride())
        got = self.bwd.get(key)
        if got is None:
            dims = S2GPacked(*self.fields, *_strides(q), *_strides(k), *_strides(v), *_strides(do), *self.size)
            k_tiles, cut, slots = self.work.key_tiles(self.group, self.causal, self.kv_heads, self.fields[0] == 0)
            got = self.bwd[key] = (ctypes.byref(dims), (ptr(k_tiles), k_tiles.shape[0], ptr(cut), cut.shape[0]),
                                   get().s2g_packed_attention_bwd_workspace(ctypes.byref(dims), slots), (self.q_tiles, k_tiles, cut))
        return got


class PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, plan):
        out = _new(q)
        if not plan.some:
            out.zero_()
        elif not plan.whole:
            out[plan.rows:].zero_()
        lse = rest = None
        if any(ctx.needs_input_grad):
            lse = q.new_empty(2, plan.stats, dtype=torch.float32)         # and room for D
            rest = torch.empty_like(out) if q.dtype != torch.float32 else None
        if plan.some:
            _lend(plan.work, plan.q_tiles)
            _launch(plan.device, "s2g_packed_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ptr(rest), ptr(lse),
                    *plan.q_list, plan.fwd)
        ctx.save_for_backward(q, k, v, out, rest, lse)
        ctx.plan = plan
        return out

    @staticmethod
    @_once
    def backward(ctx, do):
        q, k, v, out, rest, lse = ctx.saved_tensors
        plan = ctx.plan
        if not plan.some:
            return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), None
        if do.data_ptr() & 15 or not _fetchable(do, plan.group):
            do = _copy(do)
        if (q.stride(), k.stride(), v.stride()) != plan.strides:       # hooks on saved tensors may lay them out anew
            q, k, v = _copy(q), _copy(k), _copy(v)
            out, rest, lse = (None if x is None else x.contiguous() for x in (out, rest, lse))
        dims, lists, floats, kept = plan.backward(q, k, v, do)
        _lend(plan.work, *kept)
        dq, dk, dv = _new(q), _new(k), _new(v)
        if not plan.whole:
            dq[plan.rows:].zero_()
            dk[plan.key_rows:].zero_()
            dv[plan.key_rows:].zero_()
        work = lse.new_empty(floats) if floats else None
        _launch(plan.device, "s2g_packed_attention_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ptr(rest), do.data_ptr(),
                lse.data_ptr(), lse.data_ptr() + 4 * plan.stats, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ptr(work), *plan.q_list, *lists, dims)
        return dq, dk, dv, None


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pack: PackedSequences, causal: bool = True,
                     scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v within every sequence of `pack`, row i of n queries and m keys seeing keys j <= i + m - n
    (causal) or all of them.  q [tokens, heads, dim], k and v [keys, kv heads, dim], fp32 / bf16 / fp16, query head h
    reading kv head h // (heads / kv heads); dim a multiple of 8 up to 128; scale: 1 / sqrt(dim).  A row that sees no key
    gives zeros and has no gradient, and so does one whose scores are all minus infinity (a softmax of those would be NaN); rows
    behind the last sequence give zeros and have no gradient.  Differentiable in q, k and v, with the same bits on every run.
    Sums and softmax are taken in 32 bits; of 16-bit inputs the weights are rounded to their type before they meet v.  A pass
    that is trained keeps two floats a row of a head and, of 16-bit inputs, a tensor of the output's size beside the output.
    Infinities and NaN stay with the rows that see them, but rows or keys near one that others do not see are made anew pair by
    pair, a hundred times as slow (a training step whose gradient has overflowed)."""
    if not isinstance(pack, PackedSequences):
        raise S2GError("packed_attention: pack must be PackedSequences")
    _no_tangent("packed_attention", q, k, v)
    causal, scale = bool(causal), None if scale is None else float(scale)
    try:
        key = (_layout(q, k, v), causal, scale)
    except AttributeError:
        raise S2GError("packed_attention: q, k and v must be GPU tensors") from None
    plan = pack._plans.get(key)
    if plan is None:
        plan = pack._plans[key] = _PackedPlan(pack, q, k, v, causal, scale)
    copies = [c or x.data_ptr() & 15 for c, x in zip(plan.copies, (q, k, v))]
    if any(copies):                                    # rows that cannot be fetched in 16-byte units, or do not start so
        return packed_attention(*(_copy(x) if c else x for c, x in zip(copies, (q, k, v))), pack, causal, scale)
    return PackedAttentionFn.apply(q, k, v, plan)


# ---------------------------------------------------------------------------------------------------------- paged cache
class PagedBatch(_Fixed):
    """What a step of serving reads: for every sequence its row of the page table (int32 [sequences, columns], column c
    the page of tokens c * page size ..), its length in the cache with the new tokens counted in, and how many of them are
    new; the new tokens of all sequences lie one after another, `rows` in all.  table, lengths and starts live on the
    device and may be rewritten there in place between launches (a captured decoding loop does `batch.lengths.add_(1)`; a
    sequence that is done is given length 0), up to max_length tokens and max_new new ones a sequence; what the host knows
    is max_new, max_length and rows.  Rows that rewritten starts leave to no sequence come back undefined.  A captured
    graph reads the tensors on every replay: keep the batch as long as the graph."""

    __slots__ = ("device", "stream", "table", "lengths", "starts", "sequences", "rows", "max_new", "max_length", "_length", "_new", "_cuts", "_plans")

    @_lasting
    def __init__(self, table, lengths: Sequence[int], new_lengths: Sequence[int], max_length: Optional[int] = None, device=None):
        n, c = np.asarray(new_lengths, dtype=np.int64).reshape(-1), np.asarray(lengths, dtype=np.int64).reshape(-1)
        if n.shape != c.shape or n.size == 0 or n.size > 65535 or n.min() < 0 or (c < n).any() or c.max() >= 1 << 30 or n.sum() >= 1 << 30:
            raise S2GError("PagedBatch: lengths must be as many as new_lengths (1 to 65535), and none smaller")
        if not isinstance(table, torch.Tensor):
            table = torch.as_tensor(np.asarray(table, dtype=np.int32))
        if table.dim() != 2 or table.shape[0] != n.size or table.dtype != torch.int32:
            raise S2GError(f"PagedBatch: table must be int32 [{n.size}, columns]")
        dev = table.device if table.is_cuda else torch.device(device or "cuda")
        if dev.type != "cuda":
            raise S2GError("PagedBatch: needs a GPU device")
        # one copy to the device: a step of serving makes a batch
        columns = table.shape[1]
        host = [c, [0], np.cumsum(n)] + ([] if table.is_cuda else [table.numpy().reshape(-1)])
        buffer = _on_device(np.concatenate(host), dev)
        dev = self.device = buffer.device
        self.lengths, self.starts = buffer[:n.size], buffer[n.size:2 * n.size + 1]
        self.table = table.contiguous() if table.is_cuda else buffer[2 * n.size + 1:].view(n.size, columns)
        self.stream = torch.cuda.current_stream(dev)
        self.sequences, self.rows, self.max_new = n.size, int(n.sum()), int(n.max())
        self.max_length = int(c.max()) if max_length is None else int(max_length)
        self._length, self._new, self._cuts, self._plans = c, n, {}, {}
        if self.max_length < c.max():
            raise S2GError("PagedBatch: max_length is below a length")

    def pointers(self) -> Tuple[int, int, int]:
        """The device tensors' addresses, for a launch on the current stream."""
        _lend(self, self.table, self.lengths, self.starts)
        return self.table.data_ptr(), self.lengths.data_ptr(), self.starts.data_ptr()


def _pool(what: str, keys: torch.Tensor, values: torch.Tensor) -> Tuple[int, int, int]:
    if keys.dim() != 4 or keys.shape != values.shape or keys.stride() != values.stride() or keys.stride(3) != 1:
        raise S2GError(f"{what}: keys and values must be [pages, page size, kv heads, dim], alike in shape and strides, dim dense")
    size = keys.shape[1]
    if size < 16 or size > 65536 or size & (size - 1):
        raise S2GError(f"{what}: page size must be a power of two, 16 to 65536, got {size}")
    if keys.shape[0] == 0 or keys.shape[0] >= 1 << 31:
        raise S2GError(f"{what}: {keys.shape[0]} pages")
    return keys.stride(0), keys.stride(1), keys.stride(2)


def _batch(what: str, batch: PagedBatch, q: torch.Tensor, keys: torch.Tensor) -> None:
    if not isinstance(batch, PagedBatch) or batch.table.device != q.device:
        raise S2GError(f"{what}: batch must be a PagedBatch on {q.device}")
    if q.shape[0] < batch.rows:
        raise S2GError(f"{what}: the batch has {batch.rows} new tokens, got {q.shape[0]}")
    if batch.max_length > batch.table.shape[1] * keys.shape[1]:
        raise S2GError(f"{what}: {batch.max_length} tokens do not fit {batch.table.shape[1]} pages of {keys.shape[1]}")
    if batch.table.shape[1] * keys.shape[1] >= 1 << 30:
        raise S2GError(f"{what}: the table covers 2^30 tokens or more")


def _no_grad(what: str, *tensors: torch.Tensor) -> None:
    _no_tangent(what, *tensors)
    if torch.is_grad_enabled() and any([t.requires_grad for t in tensors]):
        raise S2GError(f"{what} serves: it has no gradient (call it under torch.no_grad())")


def _plan_of(batch, what, how, make, *tensors):
    """The batch's plan for tensors laid out like these, made (and they checked) when they first come."""
    if not isinstance(batch, PagedBatch):
        raise S2GError(f"{what}: batch must be a PagedBatch")
    try:
        key = (what, how, _layout(*tensors))
    except AttributeError:
        raise S2GError(f"{what}: needs GPU tensors") from None
    got = batch._plans.get(key)
    if got is None:
        got = batch._plans[key] = make(batch, how, *tensors)
    return got


class _AppendPlan:
    def __init__(self, batch, how, q, k, v, keys, values, frequencies):
        what = "append_rotary"
        _check(what, q=q, k=k, v=v, keys=keys, values=values)
        if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or q.shape[1] == 0:
            raise S2GError(f"{what}: q must be [tokens, heads, dim], k and v [tokens, kv heads, dim]")
        page_ld, token_ld, head_ld = _pool(what, keys, values)
        if tuple(keys.shape[2:]) != tuple(k.shape[1:]) or k.shape[1] == 0:
            raise S2GError(f"{what}: pages hold heads {tuple(keys.shape[2:])}, k has {tuple(k.shape[1:])}")
        _batch(what, batch, q, keys)
        self.copy = any(x.stride(2) != 1 for x in (q, k, v))
        self.device, self.whole = q.get_device(), q.shape[0] == batch.rows
        dims = _rotary_dims(q, k, v, _frequencies(what, frequencies, q.get_device(), q.shape[2]), *how, False)
        paged = S2GPaged(sequences=batch.sequences, page_size=keys.shape[1], pages=keys.shape[0], table_cols=batch.table.shape[1],
                         max_new=batch.max_new, page_ld=page_ld, token_ld=token_ld, head_ld=head_ld)
        self.args, self.paged = ctypes.byref(dims), ctypes.byref(paged)


def append_rotary(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                  batch: PagedBatch, frequencies: torch.Tensor, interleaved: bool = False, multiplier: float = 1.0) -> torch.Tensor:
    """The new tokens of a batch on their way into the cache, in one launch: q and k are turned as apply_rotary turns them,
    by the tokens' positions in their sequences, k and v written to their pages (keys, values: [pages, page size, kv heads,
    dim], in place), the turned q returned.  A token whose position has no page is not written.  Rows of q behind the
    batch's come back as zeros.  No two sequences may own a page that both write to."""
    _no_grad("append_rotary", q, k, v, keys, values)
    _no_tangent("append_rotary", frequencies)
    how = (bool(interleaved), float(multiplier))
    plan = _plan_of(batch, "append_rotary", how, _AppendPlan, q, k, v, keys, values, frequencies)
    if plan.copy:
        q, k, v = _dense(q), _dense(k), _dense(v)
        plan = _plan_of(batch, "append_rotary", how, _AppendPlan, q, k, v, keys, values, frequencies)
    out = _new(q)
    if not plan.whole:
        out[batch.rows:].zero_()
    if batch.rows:
        _hold(plan.device, frequencies)
        _launch(plan.device, "s2g_rotary_append", q.data_ptr(), k.data_ptr(), v.data_ptr(), frequencies.data_ptr(), out.data_ptr(),
                keys.data_ptr(), values.data_ptr(), *batch.pointers(), plan.args, plan.paged)
    return out


def _cut(batch: PagedBatch, Hk: int, G: int, D: int, size: int) -> Tuple[bool, int, int]:
    """(128 rows to a workgroup, keys per part, parts).  One workgroup per (row tile, kv head, part) that exists.  Either all
    of them are resident at once (counting on 85 % of the places, as they are not dealt quite evenly) and take as long as a
    part; or they come in turn, which takes the whole work and, at the end, about 0.6 of a part.  Beginning and ending cost
    a workgroup about 256 keys' time, a part's sums of 128 rows another 4 to write and to join.  (64 sequences of 300 to 8200
    tokens, 8 kv heads of 128 bf16: parts of 512 / 1024 / 2048 / 8192 keys 253 / 232 / 212 / 236 us.)  From the lengths as
    they were when the batch was made, and kept with it.  Of 128 rows it counts one workgroup to a compute unit, as in fp32; of the
    16-bit ones two fit.  (The parts were swept for single tokens only.)"""
    got = batch._cuts.get((Hk, G, D, size))
    if got is None:
        rows = np.maximum(batch._new, 0) * G
        by_rows = batch.max_new * G > 64
        tiles = -(-rows // (TILE if by_rows else 32)) * Hk
        width = 32 if D <= 32 else 64 if D <= 64 else 128
        resident = 256 if by_rows else 256 * max(1, 131072 // (16 * 32 * width * size))
        work = int((tiles * batch._length).sum())
        best, k = None, 128
        while True:
            blocks = int((tiles * -(-batch._length // k)).sum())
            if blocks <= 0.85 * resident:
                cost = min(k, batch.max_length) + 256
            else:
                cost = (work + 256 * blocks) / resident + 0.6 * min(k, batch.max_length)
            if by_rows and k < batch.max_length:
                cost += 4 * blocks * width * 256 / resident / 128
            if best is None or cost < best[0]:
                best = cost, k
            if k >= batch.max_length:
                break
            k += max(128, k // 8 // 128 * 128)
        k = max(best[1], -(-batch.max_length // 4096 // 128) * 128)
        got = batch._cuts[Hk, G, D, size] = by_rows, k, max(1, -(-batch.max_length // k))
    return got


class _PagedPlan:
    """One layout of q and of the pool for one batch: checked once, cut into parts, the kernel's arguments kept."""

    def __init__(self, batch, how, q, keys, values):
        causal, scale = how
        what = "paged_attention"
        _check(what, q=q, keys=keys, values=values)
        page_ld, token_ld, head_ld = _pool(what, keys, values)
        if q.dim() != 3 or q.shape[2] != keys.shape[3]:
            raise S2GError(f"{what}: q must be [tokens, heads, {keys.shape[3]}]")
        (R, H, D), Hk = q.shape, keys.shape[2]
        _attention_heads(what, H, Hk, D)
        unit = 16 // q.element_size()
        if any(s % unit for s in (page_ld, token_ld, head_ld)) or max(token_ld, head_ld) >= 1 << 22:
            raise S2GError(f"{what}: pages must be strided by multiples of 16 bytes, tokens by less than 2^22 elements")
        if page_ld * q.element_size() >= 1 << 36 or keys.shape[1] * token_ld * q.element_size() >= 1 << 32:
            raise S2GError(f"{what}: a page must span less than 4 GiB, and the next begin within 64")
        _batch(what, batch, q, keys)
        if R * H >= 1 << 30:
            raise S2GError(f"{what}: 2^30 rows or more")
        by_rows, part_keys, parts = _cut(batch, Hk, H // Hk, D, q.element_size())
        self.copy, self.device, self.whole = not _fetchable(q), q.get_device(), R == batch.rows
        if H * D >= 1 << 22 and self.copy:             # a copy's tokens would be as far apart
            raise S2GError(f"{what}: tokens of q have 2^22 elements or more")
        dims = S2GPaged(TYPES[q.dtype], batch.sequences, H, Hk, D, int(causal), keys.shape[1], keys.shape[0], batch.table.shape[1],
                        batch.max_new, batch.max_length, part_keys, parts, int(by_rows), _scale(what, scale, D), R, *_strides(q),
                        page_ld, token_ld, head_ld)
        self.args = ctypes.byref(dims)
        self.floats = 0 if self.copy or not batch.rows else get().s2g_paged_attention_workspace(self.args)


def paged_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, batch: PagedBatch, causal: bool = True,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of a batch's new tokens (q [tokens, heads, dim]) over what its sequences hold in the cache: query i of n
    new tokens of a sequence of m sees keys j <= m - n + i (causal) or all m.  One token or thousands per sequence, mixed
    at will; types, heads and scale as in packed_attention.  A page number outside the pool, or a position that the table does
    not cover, is a key that is not there; a query without keys gives zeros, and so do one whose scores are all minus infinity
    and rows of q behind the batch's."""
    _no_grad("paged_attention", q, keys, values)
    causal, scale = bool(causal), None if scale is None else float(scale)
    plan = _plan_of(batch, "paged_attention", (causal, scale), _PagedPlan, q, keys, values)
    if plan.copy or q.data_ptr() & 15:
        return paged_attention(_copy(q), keys, values, batch, causal, scale)
    if (keys.data_ptr() | values.data_ptr()) & 15:
        raise S2GError("paged_attention: pages must start at multiples of 16 bytes")
    out = _new(q)
    if not plan.whole:
        out[batch.rows:].zero_()
    if batch.rows:
        work = q.new_empty(plan.floats, dtype=torch.float32) if plan.floats else None
        _launch(plan.device, "s2g_paged_attention", q.data_ptr(), keys.data_ptr(), values.data_ptr(), *batch.pointers(), out.data_ptr(), ptr(work),
                plan.args)
    return out


class PagedKVCache:
    """Keys and values of many sequences in pages of one pool: `keys`, `values` [pages, page size, kv heads, dim].
    Sequences come and go on the host; `extend` reserves room for new tokens and says where they lie."""

    @_lasting
    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, dtype=torch.float32, device="cuda"):
        if num_pages <= 0 or page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise S2GError("PagedKVCache: needs pages, of a power of two of tokens, 16 to 65536")
        _attention_heads("PagedKVCache", num_kv_heads, num_kv_heads, head_dim)
        if dtype not in TYPES:
            raise S2GError(f"PagedKVCache: float32, bfloat16 or float16, got {dtype}")
        self.keys = torch.empty(num_pages, page_size, num_kv_heads, head_dim, dtype=dtype, device=device)
        self.values = torch.empty_like(self.keys)
        self.page_size = page_size
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: Dict[int, List[int]] = {}
        self._length: Dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def add(self) -> int:
        """A new, empty sequence."""
        self._next += 1
        self._pages[self._next], self._length[self._next] = [], 0
        return self._next

    def length(self, sequence: int) -> int:
        return self._length[self._known(sequence)]

    def remove(self, sequence: int) -> None:
        """Gives a sequence's pages back (to be used again by launches enqueued later on the same stream)."""
        self._free.extend(reversed(self._pages.pop(self._known(sequence))))
        del self._length[sequence]

    def _known(self, sequence: int) -> int:
        if sequence not in self._pages:
            raise S2GError(f"PagedKVCache: no sequence {sequence}")
        return sequence

    def extend(self, sequences: Sequence[int], new_lengths: Sequence[int]) -> PagedBatch:
        """Room for new_lengths[i] more tokens of sequences[i]; the batch of them for append_rotary and paged_attention.
        Refuses, changing nothing, if the pool has too few pages.  The batch's layout is copied to the device before it returns,
        behind what is queued on the stream; a loop that is not to wait reserves all its tokens in one call and makes one
        PagedBatch over that batch's table, whose lengths it advances on the device."""
        if len(sequences) != len(new_lengths) or len(set(sequences)) != len(sequences) or not sequences or min(new_lengths) < 0:
            raise S2GError("PagedKVCache.extend: needs different sequences, each with its number of new tokens")
        lengths = [self._length[self._known(s)] + int(n) for s, n in zip(sequences, new_lengths)]
        need = [-(-m // self.page_size) - len(self._pages[s]) for s, m in zip(sequences, lengths)]
        if sum(need) > len(self._free):
            raise S2GError(f"PagedKVCache.extend: {sum(need)} pages needed, {len(self._free)} free")
        spare = iter(reversed(self._free))
        more = [[next(spare) for _ in range(k)] for k in need]
        table = np.full((len(sequences), max(1, max(len(self._pages[s]) + k for s, k in zip(sequences, need)))), -1, dtype=np.int32)
        for row, s, new in zip(table, sequences, more):
            row[:len(self._pages[s]) + len(new)] = self._pages[s] + new
        batch = PagedBatch(torch.from_numpy(table), lengths, new_lengths, device=self.keys.device)
        del self._free[len(self._free) - sum(need):]
        for s, m, new in zip(sequences, lengths, more):
            self._pages[s] += new
            self._length[s] = m
        return batch

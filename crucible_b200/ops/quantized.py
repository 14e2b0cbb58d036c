"""Rows of activations in 8 bits, and matrix products over 8-bit and 4-bit weights.

A row in 8 bits is e4m3 numbers q [K] with one float32 scale s; it stands for q * s.  `add_rmsnorm8`
and `glu8` make such rows (s: the row's largest magnitude over 448), `linear8` multiplies them by
weights that are kept the same way, a scale per output feature (`Weights8`).

`linear4` multiplies float32 or bfloat16 rows by 4-bit weights (`Weights4`): (code - 8) * group scale *
feature scale, codes 0..15, the group scales e4m3, the feature scales float32.  (code - 8) times an
e4m3 number has at most seven significant bits, so the tensor cores take the weights as they are, in
bfloat16 without a rounding; float32 rows go through them as three bfloat16 parts that add up to the row
exactly (but for what lies below 2^-133).  Sums are float32 in every product, and only the result is rounded.  Which
kernel runs, and with it the order of a sum, goes by the sizes, the number of rows among them.

Everything here launches on torch's current stream of the tensors' device, keeps no buffer between
calls and may be captured into a CUDA graph (a call that has to bring rows into another layout first
allocates from torch's pool, as any captured torch operation does).  Outputs may not overlap inputs, but where
a function says so.  The waits inside the products, and inside `glu8` of many long rows, are bounded;
`tensor_core.check_status` raises if one ran out.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import LAUNCHES, KernelError, _check, _need_cuda, _ptr, _stream, build, tensor_core

build.register_module("rows8", ["common.cuh", "quantized.cuh", "tc_common.cuh"])
build.register_module("linear_quantized_few", ["common.cuh", "quantized.cuh"])
build.register_module("linear_quantized_ring", ["common.cuh", "quantized.cuh", "tc_common.cuh"])
for _name in ("linear_quantized_tcgen05", "linear_quantized_pairs_tcgen05"):
    build.register_module(_name, ["common.cuh", "quantized.cuh", "quantized_tc.cuh", "tc_common.cuh"])

E4M3 = torch.float8_e4m3fn
TOP = 448.0                      # the largest e4m3 number
LEAST = 1e-30                    # a row's largest magnitude counts as this much at least
_FOUR_BF16, _FOUR_F32, _EIGHT = 0, 1, 2
_MOST_PITCH = 1 << 24            # bytes between rows of weights (`csrc/quantized.cuh`)
_FLOATS = (torch.float32, torch.bfloat16)
_MOST_ROWS = (1 << 31) - 1024    # the kernels count rows and features in 32 bits
_SLAB = 1 << 16                  # float32 rows over 4-bit weights at a time, at most
_SCRATCH = 512 << 20             # and at most so many bytes of their three bfloat16 parts, 6 a number
_LEAST_LIMIT = 2.0 ** -126       # (a smaller limit could be zero in float32)
_WAITS_FROM = 296                # rows of `glu8` from which its kernel may wait for copies (`cb_glu8_waits_from`)


# Every function asks first whether all is as it usually is, in one expression over plain attributes; only where it is
# not are the tensors looked over one by one, for what is refused and for what is unusual but taken (a row of any
# stride where there is one row, say).  Looked over one by one they took 6 to 11 us of host time a call, which
# for a few rows is more than the kernel takes; the one expression takes 2 to 3.

_F32 = torch.float32
_device_now = torch._C._cuda_getDevice


def _at(dev: int, call, *args) -> int:
    """call(*args, stream) with device `dev` the current one."""
    now = _device_now()
    if now == dev:
        return call(*args, _stream())
    torch.cuda.set_device(dev)
    try:
        return call(*args, _stream())
    finally:
        torch.cuda.set_device(now)


def _one_device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    for t in others:
        if t is not None and t.device != first.device:
            raise KernelError(f"the tensors lie on {first.device} and {t.device}")


def _rows(t: torch.Tensor, what: str, dtypes, shape=None) -> None:
    """Rows that a kernel walks: 2-D, of a dtype it takes, each row's elements side by side."""
    if t.dim() != 2 or t.dtype not in dtypes or (shape is not None and tuple(t.shape) != shape):
        names = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        want = f" {list(shape)}" if shape is not None else ""
        raise KernelError(f"{what}: {names} rows{want} are taken, got {t.dtype} {list(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise KernelError(f"{what}: rows must be contiguous")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise KernelError(f"{what}: rows must not overlap")
    _count(t.shape[0], what)


def _count(rows: int, what: str) -> None:
    if rows > _MOST_ROWS:
        raise KernelError(f"{what}: up to {_MOST_ROWS} rows are taken, got {rows}")


def _vector(t: torch.Tensor, what: str, size: int) -> None:
    if t.dtype != torch.float32 or tuple(t.shape) != (size,) or (size > 1 and t.stride(0) != 1):
        raise KernelError(f"{what}: a contiguous float32 vector [{size}] is taken, got {t.dtype} {list(t.shape)}")


def new_rows8(rows: int, width: int, device) -> torch.Tensor:
    """Uninitialised e4m3 rows [rows, width] that begin a multiple of 16 bytes apart, as `linear8` takes
    them without a copy."""
    return torch.empty(rows, (width + 15) // 16 * 16, dtype=torch.uint8, device=device).view(E4M3)[:, :width]


# ---------------------------------------------------------------------------
# rows in 8 bits
# ---------------------------------------------------------------------------

def add_rmsnorm8(x: torch.Tensor, delta: Optional[torch.Tensor], gain: torch.Tensor, eps: float, out: torch.Tensor,
                 scales: torch.Tensor, sum_out: Optional[torch.Tensor] = None) -> None:
    """x + delta, its RMS norm, and that in 8 bits: y = sum / sqrt(mean(sum^2) + eps) * gain goes to `out`
    (e4m3 [T, W]) and `scales` (float32 [T]).  `x`: the float32 residual; `delta`: float32 or bfloat16 rows
    to add to it, or None.  The sum goes to `sum_out`, which is `x` itself if a delta is given and
    nothing else is said (without either, `x` is only read)."""
    if sum_out is None and delta is not None:
        sum_out = x
    dev, shape, xs, os = x.get_device(), x.shape, x.stride(), out.stride()
    ss = xs if sum_out is None or sum_out is x else sum_out.stride()
    ds = xs if delta is None else delta.stride()
    if not (dev >= 0 and len(shape) == 2 and x.dtype is _F32 and out.dtype is E4M3 and scales.dtype is _F32
            and gain.dtype is _F32 and out.shape == shape and xs[1] == 1 == os[1] and xs[0] >= shape[1] <= os[0]
            and shape[0] <= _MOST_ROWS and gain.shape == (shape[1],) and gain.is_contiguous()
            and scales.shape == (shape[0],) and scales.is_contiguous()
            and out.get_device() == dev == gain.get_device() and scales.get_device() == dev
            and (delta is None or (delta.shape == shape and delta.dtype in _FLOATS and ds[1] == 1
                                   and ds[0] >= shape[1] and delta.get_device() == dev))
            and (ss is xs or (sum_out.shape == shape and sum_out.dtype is _F32 and ss[1] == 1
                              and ss[0] >= shape[1] and sum_out.get_device() == dev))):
        _look_over_norm8(x, delta, gain, out, scales, sum_out)
    lib = build.load("rows8")
    code = _at(dev, lib.cb_norm8, x.data_ptr(), xs[0], _ptr(delta), 1 if delta is not None and delta.dtype is not _F32 else 0,
               ds[0], gain.data_ptr(), eps, _ptr(sum_out), ss[0], out.data_ptr(), os[0], scales.data_ptr(),
               shape[0], shape[1])
    if code == build.UNSUPPORTED:
        raise KernelError(f"add_rmsnorm8 takes rows of 1 to {lib.cb_rows8_widest()} features, got {shape[1]}")
    _check(code, "add_rmsnorm8")


def _look_over_norm8(x, delta, gain, out, scales, sum_out) -> None:
    _rows(x, "add_rmsnorm8 input", (torch.float32,))
    rows, width = x.shape
    if delta is not None:
        _rows(delta, "add_rmsnorm8 delta", _FLOATS, (rows, width))
    if sum_out is not None:
        _rows(sum_out, "add_rmsnorm8 sum", (torch.float32,), (rows, width))
    _vector(gain, "add_rmsnorm8 gain", width)
    _rows(out, "add_rmsnorm8 output", (E4M3,), (rows, width))
    _vector(scales, "add_rmsnorm8 scales", rows)
    _need_cuda(x, delta, gain, out, scales, sum_out)
    _one_device(x, delta, gain, out, scales, sum_out)


def glu8(both: torch.Tensor, out: torch.Tensor, scales: torch.Tensor, limit: Optional[float] = None,
         alpha: float = 1.0, offset: float = 0.0) -> None:
    """The gated pair of rows [g: F | u: F] in 8 bits: `out` (e4m3 [T, F]) and `scales` (float32 [T]).
    `limit` None: silu(g) * u.  A number: the capped pair of `ops.glu`, g' sigmoid(alpha g') (u' + offset)
    with g' = min(g, limit), u' = clamp(u, -limit, limit)."""
    dev, shape, bs, os = both.get_device(), out.shape, both.stride(), out.stride()
    if not (dev >= 0 and len(shape) == 2 and both.dtype in _FLOATS and out.dtype is E4M3 and scales.dtype is _F32
            and both.shape == (shape[0], 2 * shape[1]) and bs[1] == 1 == os[1] and bs[0] >= 2 * shape[1]
            and os[0] >= shape[1] and scales.shape == (shape[0],) and scales.is_contiguous()
            and out.get_device() == dev == scales.get_device() and shape[0] <= _MOST_ROWS
            and (limit is None or limit >= _LEAST_LIMIT)):
        _look_over_glu8(both, out, scales, limit)
    lib = build.load("rows8")
    code = _at(dev, lib.cb_glu8, both.data_ptr(), 0 if both.dtype is _F32 else 1, bs[0], out.data_ptr(), os[0],
               scales.data_ptr(), shape[0], shape[1], limit if limit is not None else 0.0, alpha, offset,
               _status(dev) if shape[0] >= _WAITS_FROM else 0)
    if code == build.UNSUPPORTED:
        raise KernelError(f"glu8 takes 1 to {lib.cb_rows8_widest()} features, got {shape[1]}")
    _check(code, "glu8")


def _look_over_glu8(both, out, scales, limit) -> None:
    _rows(both, "glu8 input", _FLOATS)
    if both.shape[1] % 2:
        raise KernelError(f"glu8 takes rows [g | u] of an even width, got {both.shape[1]}")
    if limit is not None and not limit >= _LEAST_LIMIT:
        raise KernelError(f"glu8: the limit must be positive, {_LEAST_LIMIT:.3g} or more, got {limit}")
    _rows(out, "glu8 output", (E4M3,), (both.shape[0], both.shape[1] // 2))
    _vector(scales, "glu8 scales", both.shape[0])
    _need_cuda(both, out, scales)
    _one_device(both, out, scales)


# ---------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------

def _aligned16(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or t.stride(0) * t.element_size() % 16 == 0)


def _pitch(t: torch.Tensor) -> int:
    """Elements between rows (one row: as many as would do)."""
    per = 16 // t.element_size()
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + per - 1) // per * per


def _in_aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """The same values in rows that begin on multiples of 16 bytes."""
    per = 16 // t.element_size()
    wide = torch.empty(t.shape[0], (t.shape[1] + per - 1) // per * per, dtype=t.dtype, device=t.device)[:, :t.shape[1]]
    wide.copy_(t)
    return wide


class Weights8:
    """A matrix [N, K] in 8 bits: e4m3 `values` [N, K], float32 `scales` [N]; weight (n, k) is
    values[n, k] * scales[n].  Values whose rows do not begin on multiples of 16 bytes are copied into rows
    that do, once, here."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        shape, dev = values.shape, values.get_device()
        if (len(shape) == 2 and values.dtype is E4M3 and scales.dtype is _F32 and values.is_contiguous()
                and scales.shape == (shape[0],) and scales.is_contiguous() and shape[0] > 0 and shape[1] > 0
                and scales.get_device() == dev and shape[1] % 16 == 0 and values.data_ptr() % 16 == 0):
            self.values, self.pitch = values, shape[1]
        else:
            _rows(values, "8-bit weights", (E4M3,))
            if shape[0] == 0 or shape[1] == 0:
                raise KernelError(f"8-bit weights: an empty matrix {list(shape)}")
            _vector(scales, "8-bit weights' scales", shape[0])
            _one_device(values, scales)
            if not _aligned16(values) or (shape[0] > 1 and values.stride(0) > _MOST_PITCH):
                values = _in_aligned_rows(values.view(torch.uint8)).view(E4M3)
            self.values, self.pitch = values, _pitch(values)
        self.scales, self.shape, self.device = scales, shape, dev
        if dev >= 0 and dev not in tensor_core._status:
            _status(dev)

    @classmethod
    def pack(cls, w: torch.Tensor) -> "Weights8":
        """From a matrix of floating numbers: each row's largest magnitude becomes 448."""
        w = _finite(w)
        scales = w.abs().amax(dim=1).clamp_min(LEAST) * (1 / TOP)
        return cls((w / scales[:, None]).clamp(-TOP, TOP).to(E4M3), scales)

    def dense(self) -> torch.Tensor:
        """The float32 matrix that these weights stand for."""
        return self.values.float() * self.scales[:, None]


def _finite(w: torch.Tensor) -> torch.Tensor:
    if w.dim() != 2 or not w.is_floating_point() or w.numel() == 0:
        raise KernelError(f"weights are packed from a matrix of floating numbers, got {w.dtype} {list(w.shape)}")
    w = w.float().contiguous()
    if not bool(torch.isfinite(w).all()):
        raise KernelError("weights are packed from finite numbers")
    return w


# Code i of eight neighbouring k lies at this bit of their int32: even k in the low half, odd k in the high
# half, so that masking one nibble of both halves gives the codes of two neighbouring k.
CODE_SHIFTS = tuple(4 * (i // 2) + 16 * (i % 2) for i in range(8))


class Weights4:
    """A matrix [N, K] in 4 bits: weight (n, k) is (code - 8) * group_scales[n, k // group] * scales[n].
    `codes`: int32 [N, K / 8], eight codes of neighbouring k a word at the bits `CODE_SHIFTS`;
    `group_scales`: e4m3 [N, K / group] (`group` is read off the shapes: a multiple of 32 that divides K);
    `scales`: float32 [N]."""

    def __init__(self, codes: torch.Tensor, group_scales: torch.Tensor, scales: torch.Tensor):
        shape, groups = codes.shape, group_scales.shape
        if (len(shape) == 2 == len(groups) and codes.dtype is torch.int32 and group_scales.dtype is E4M3
                and scales.dtype is _F32 and groups[0] == shape[0] and scales.shape == (shape[0],) and shape[0] > 0
                and groups[1] > 0 and shape[1] % (4 * groups[1]) == 0 and shape[1] > 0 and scales.is_contiguous()
                and codes.is_contiguous() and group_scales.is_contiguous() and codes.data_ptr() % 16 == 0
                and codes.get_device() == group_scales.get_device() == scales.get_device()):
            self.codes, self.group_scales, self.scales = codes, group_scales, scales
            self.group = shape[1] * 8 // groups[1]
            self.shape = torch.Size((shape[0], shape[1] * 8))
            self.device = codes.get_device()
            if self.device >= 0 and self.device not in tensor_core._status:
                _status(self.device)
            return
        _rows(codes, "4-bit weights' codes", (torch.int32,))
        n, k = codes.shape[0], codes.shape[1] * 8
        if n == 0 or k == 0:
            raise KernelError(f"4-bit weights: an empty matrix [{n}, {k}]")
        _rows(group_scales, "4-bit weights' group scales", (E4M3,))
        groups = group_scales.shape[1]
        if group_scales.shape[0] != n or groups == 0 or k % groups or (k // groups) % 32:
            raise KernelError(f"4-bit weights: group scales [{n}, K / group] are taken, the group a multiple of 32 "
                              f"that divides K = {k}, got {list(group_scales.shape)}")
        _vector(scales, "4-bit weights' scales", n)
        _one_device(codes, group_scales, scales)
        self.codes = codes if codes.is_contiguous() and codes.data_ptr() % 16 == 0 else codes.clone(
            memory_format=torch.contiguous_format)
        self.group_scales = group_scales.contiguous()
        self.scales = scales
        self.group = k // groups
        self.shape = torch.Size((n, k))
        self.device = codes.get_device()
        if self.device >= 0:
            _status(self.device)

    @classmethod
    def pack(cls, w: torch.Tensor, group: int = 64) -> "Weights4":
        """From a matrix of floating numbers [N, K]: a group's largest magnitude becomes code 1 or 15 (before
        its scale is rounded to e4m3; the codes are then the nearest for the scales as they are)."""
        w = _finite(w)
        n, k = w.shape
        if group <= 0 or group % 32 or k % group:
            raise KernelError(f"4-bit weights: a group is a multiple of 32 that divides K = {k}, got {group}")
        parts = w.view(n, k // group, group)
        # (products with reciprocals, and quotients of tensors alone: a quotient by a number is rounded otherwise on
        # another device, and a scale that falls on the other side of a border is 2^-3 off)
        want = parts.abs().amax(dim=2) * (1 / 7)
        scales = want.amax(dim=1).clamp_min(LEAST) * (1 / TOP)
        # (no group's scale may round to zero: the smallest number above it is 2^-9)
        group_scales = (want / scales[:, None]).clamp(2.0 ** -9, TOP).to(E4M3)
        step = group_scales.float() * scales[:, None]
        codes = (torch.round(parts / step[:, :, None]).clamp(-8, 7) + 8).to(torch.int32).view(n, k // 8, 8)
        words = torch.zeros(n, k // 8, dtype=torch.int32, device=w.device)
        for i, shift in enumerate(CODE_SHIFTS):
            words |= codes[:, :, i] << shift
        return cls(words, group_scales, scales)

    def dense(self) -> torch.Tensor:
        """The float32 matrix that these weights stand for."""
        n, k = self.shape
        shifts = torch.tensor(CODE_SHIFTS, dtype=torch.int32, device=self.codes.device)
        codes = ((self.codes[:, :, None] >> shifts) & 15) - 8
        grouped = codes.float().view(n, -1, self.group) * self.group_scales.float()[:, :, None]
        return grouped.view(n, k) * self.scales[:, None]


# ---------------------------------------------------------------------------
# products: out[M, N] = rows[M, K] . W[N, K]^T (+ add)
# ---------------------------------------------------------------------------

def _out_rows(out: torch.Tensor, add: Optional[torch.Tensor], shape, what: str) -> None:
    _rows(out, f"{what} output", _FLOATS, shape)
    if add is not None:
        _rows(add, f"{what} add", (torch.float32,), shape)


# Which kernel, and how.  What follows was measured on B200 for the three kinds of product at 11 sizes of weights, 1,280 by
# 768 to 28,672 by 4,096 (and 50,304 by 768, 4,096 by 14,336), and 1 to 2,048 rows, in every form: the rules below, fitted to
# these, took 0.8% longer than the best form on the average.
#
#   "few"    mma.sync from registers.  Nothing stands between a load and its use, so small matrices end first: us at 64
#            rows of 768 by 1,280, few / tiles: 4.8 / 5.2 (8 bits), 5.2 / 6.8 (4 bits); 8 rows of 2,048 by 2,048 5.2 / 5.9.
#   "ring"   the same arithmetic behind a ring of stages: 4-bit weights, K a multiple of 256, bfloat16 rows.  8 rows of
#            4,096 by 4,096, ring / few / tiles: 4.8 / 7.0 / 8.1; 16 rows by 14,336 14.6 / 20.6 / 16.5; 32 rows by 2,048 (K of
#            8,192) 9.7 / 12.7 / 11.2, by 6,144 (K of 4,096) 13.0 / 19.8 / 11.5.  17 to 32 rows by few features, ring / tiles: by
#            1,920 (tiles of which six share a long K) K of 5,120 7.3 / 8.1, of 6,144 8.2 / 8.2, of 8,192 10.3 / 9.3, of 16,384
#            16.6 / 13.3; by 1,984 (four share it) 7.3 / 9.3, 8.2 / 9.7, 10.3 / 11.3, 16.6 / 17.2.  A block is so many groups of warps by
#            warps that share a group's K: 1 x 8 while the SMs have two blocks or fewer at once, 1 x 4 beyond (8 rows by
#            28,672, 1 x 8 / 1 x 4 / 2 x 4: 22.5 / 19.8 / 22.7; by 4,096 4.8 / 5.4 / 7.1), 2 x 2 where K is short beside
#            the features and the rows are best read less often (by 50,304, K of 768, 1 x 4 / 2 x 2: 9.5 / 8.4), 2 x 4 for
#            16 rows, whose stages are larger (by 14,336, 1 x 4 / 2 x 4: 15.4 / 14.6).  Few features and a long K: blocks of
#            a cluster share K (8 rows by 2,048, K of 14,336, one share / four: 10.9 / 8.0; K of 8,192 7.2 / 5.5; by
#            4,096, K of 4,096, one / two: 4.8 / 5.4).
#            Up to five float32 rows are up to 15 bfloat16 ones here (1 and 5 rows by 28,672, ring / tiles: 20.7 / 40.8 and
#            29.5 / 41.2; by 2,048, K of 8,192, 7.0 / 13.8 and 8.6 / 14.1; of 768 by 1,280, ring / few: 3.7 / 3.4 and 4.0 / 3.6).
#   "tiles"  tcgen05, a block a tile of 128 features by up to 256 rows, up to 8 blocks sharing K (33 float32 rows by 2,048, K of
#            8,192, shared by 4 / 6 / 8: 15.7 / 13.9 / 19.9; a cluster of eight that fill their SMs needs eight free ones
#            side by side).
#   "pairs"  tcgen05, two SMs a tile of 256 features by up to 256 rows, tile after tile.
#
# The tiles add up a block's share of K in one sum, from which the tensor cores cut off a little at every addition.  Over 4-bit
# weights the kernel takes float32 results 2,048 of K at a time; of e4m3 products, which have 8 bits, sums of 4,096 are off by
# 2.3e-7 of the norm, of 8,192 by 4.9e-7, of 12,288 by 8.4e-7 and of 16,384 by 1.2e-6, so there a share is 12,288 at most.
# Where K has no such shares the pairs take it, 2,048 at a time (33 rows of 14,336 by 28,672 75.2 us, in one sum 68.5; by
# 20,000 two blocks share K: 65.6).
#
# Between the last two, and for the rows a tile and the shares of K, a model of what a launch takes decides: a block's
# fixed part, its steps along K (longer where two blocks are on an SM, and never shorter than the memory
# allows), what a cluster costs, and how many blocks follow one another on an SM.  us, in `_COSTS`.
FORM = None                      # tests name one of the forms, "few", "ring", "tiles" or "pairs", to reach it at any size
N_SMS = 148
_LONG_8 = 12288                  # K of one sum of e4m3 products, float32 results
_RING_F32_ROWS = 5               # (three bfloat16 rows each, and the ring takes 16)
_SMALL, _SMALL_8_ROWS = 1_200_000, 4_200_000           # weights of a matrix that "few" ends first: up to 64 rows, up to 8


class _Costs(NamedTuple):
    base: float                  # a launch of tiles
    block: float                 # a block of it, and per row
    block_row: float
    step: float                  # 128 bytes of a row along K (128 k in 8 bits, 64 k else), and per column of sums
    step_col: float
    two: float                   # times that, with two blocks on an SM
    step_bytes: float            # at least, for all blocks on an SM
    share: float                 # a cluster, per row, per block of it
    share_row: float
    share_block: float
    pair_base: float             # a launch of pairs
    pair_step: float             # a step of theirs, and per row
    pair_step_row: float
    pair_out: float              # a tile's way out, per row


_COSTS = {
    _EIGHT: _Costs(1.77, 0.80, 0.0116, 0.1705, 0.0011, 3.26, 0.232, 1.21, 0.0206, 0.13, 6.39, 0.152, 0.0007, 0.008),
    _FOUR_BF16: _Costs(3.58, 1.32, 0.0097, 0.1545, 0.0007, 1.90, 0.192, 1.17, 0.0111, 0.12, 10.1, 0.131, 0.0009, 0.0089),
    _FOUR_F32: _Costs(4.02, 1.16, 0.0190, 0.1736, 0.0005, 1.76, 0.237, 0.40, 0.0209, 0.21, 0.0, 0.0, 0.0, 0.0),
}


def _up(x: int, to: int) -> int:
    return (x + to - 1) // to * to


def _tiles_us(kind: int, m: int, n: int, k: int, tok: int, shares: int) -> float:
    c, parts = _COSTS[kind], 3 if kind == _FOUR_F32 else 1
    unit = 128 if kind == _EIGHT else 256              # K is shared in such units, of one step or four
    units = -(-k // unit)
    steps = -(-units // shares) * (1 if kind == _EIGHT else 4)
    per_sm = _blocks_an_sm(kind, tok)
    fixed = c.block + c.block_row * tok
    if shares > 1:
        fixed += c.share + c.share_row * tok + c.share_block * shares
    alone = c.step + c.step_col * parts * tok

    def round_of(blocks: int) -> float:
        return fixed + steps * max(alone * (c.two if blocks > N_SMS else 1.0), c.step_bytes * blocks / N_SMS)
    full, rest = divmod(-(-n // 128) * -(-m // tok) * shares, N_SMS * per_sm)
    return c.base + full * round_of(N_SMS * per_sm) + (round_of(rest) if rest else 0.0)


def _blocks_an_sm(kind: int, tok: int) -> int:
    return 2 if tok <= (32 if kind == _FOUR_F32 else 64) else 1


def _pairs_us(kind: int, m: int, n: int, k: int, tok: int) -> float:
    c = _COSTS[kind]
    steps = -(-k // (128 if kind == _EIGHT else 64))
    waves = -(-(-(-n // 256) * -(-m // tok)) // (N_SMS // 2))
    out = c.pair_out * tok
    return c.pair_base + waves * max(steps * (c.pair_step + c.pair_step_row * tok), out) + out


def _even(m: int, most: int) -> int:
    """Rows a tile, at most `most`, that cut m into equal tiles."""
    return _up(-(-m // -(-m // most)), 16)


def _ring(m: int, n: int, k: int):
    """Groups of warps a block, warps a group, blocks that share K, for m bfloat16 rows."""
    if n >= (9472 if k <= 1024 else 12000):
        if n >= (16 if m <= 8 else 24) * k:
            return 2, 2, 1
        return (1, 4, 1) if m <= 8 or k <= 1024 else (2, 4, 1)
    blocks, stages, shares = -(-n // 32) * -(-m // (8 if m <= 8 else 16)), -(-k // 1024), 1
    while shares < 8 and 2 * shares <= stages and 2 * shares * blocks <= 2 * N_SMS:
        shares *= 2
    return 1, 8, shares if shares >= 4 or stages >= 12 else 1


@functools.lru_cache(maxsize=4096)
def _rule(forced, kind: int, m: int, n: int, k: int, f32: bool = False):
    """("few",), ("ring", groups of warps, warps a group, shares of K), ("tiles", rows a tile, shares of K) or
    ("pairs", rows a tile, pairs of SMs).  `f32`: float32 results."""
    form = forced
    if form is None:
        small = n * k <= _SMALL and m <= 64
        if kind == _FOUR_BF16:
            narrow = (n <= 2048 and (n > 1920 or k <= 5120)) or (n <= 4096 and k <= 2048)
            form = "ring" if m <= 16 or (m <= 32 and narrow) else "few" if small else None
        elif kind == _FOUR_F32 and m <= _RING_F32_ROWS and k % 256 == 0 and not (small and k <= 1024):
            form = "ring"
        elif small or (n * k <= _SMALL_8_ROWS and m <= 8):
            form = "few"
    if form == "ring" and (kind == _EIGHT or k % 256 or (kind == _FOUR_F32 and m > _RING_F32_ROWS)):
        form = "few"
    if form == "few":
        return ("few",)
    if form == "ring":
        return ("ring",) + _ring(3 * m if kind == _FOUR_F32 else m, n, k)
    units = -(-k // (128 if kind == _EIGHT else 256))
    best = None
    if form != "pairs" or kind == _FOUR_F32:
        for most in (32, 64) if kind == _FOUR_F32 else (32, 64, 128, 256):
            tok = _even(m, most)
            if -(-m // tok) > 65535:
                continue
            tiles, per_sm = -(-n // 128) * -(-m // tok), _blocks_an_sm(kind, tok)
            for shares in (1, 2, 4, 6, 8) if per_sm == 2 else (1, 2, 4, 6):
                if shares > 1 and (shares > units or tiles * shares > 320):
                    continue
                if not (f32 and kind == _EIGHT and form is None and -(-units // shares) * 128 > _LONG_8):
                    us = _tiles_us(kind, m, n, k, tok, shares)
                    if best is None or us < best[0]:
                        best = us, ("tiles", tok, shares)
    if kind != _FOUR_F32 and (form == "pairs" or (form is None and (m >= 48 or best is None))):
        for most in (64, 96, 128, 160, 192, 224, 256):
            tok = _even(m, most)
            us = _pairs_us(kind, m, n, k, tok)
            if best is None or us < best[0]:
                best = us, ("pairs", tok, N_SMS // 2)
    return best[1]


def _status(dev: int) -> int:
    """The address of the word that a kernel writes if one of its bounded waits runs out (`tensor_core.check_status`
    raises then).  None yet, and a graph is being captured: null, since the word's zero would be written by the
    graph's replays and not now.  (`glu8` then takes the kernel that does not wait, a product is refused; whoever made
    his weights before the capture has the word.)"""
    word = tensor_core._status.get(dev)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            return 0
        word = tensor_core.status_word(torch.device("cuda", dev))
    return word.data_ptr()


def form_of(kind: int, m: int, n: int, k: int, f32: bool = False):
    return _rule(FORM, kind, m, n, k, f32)


def _product(kind: int, dev: int, rows, m: int, ldr: int, row_scales, values, ldw: int, group_scales, w, group: int, out,
             ldo: int, add, what: str) -> None:
    if m == 0:
        return
    n, k = w.shape
    _count(max(m, n), what)
    form = form_of(kind, m, n, k, out.dtype is _F32)
    common = (kind, rows.data_ptr(), ldr, row_scales, values.data_ptr(), ldw, group_scales, w.scales.data_ptr(),
              _ptr(add), add.stride(0) if add is not None else 0, out.data_ptr(), 0 if out.dtype is _F32 else 1, ldo, m, n, k,
              group)
    if form[0] == "few":
        code = _at(dev, build.load("linear_quantized_few").cb_linear_quantized_few, *common)
    else:
        status = _status(dev)
        if not status:
            raise KernelError(f"{what}: the first use on a device cannot be inside a graph's capture: its kernels have no place yet "
                              f"to say that a wait ran out")
        parts = None
        if kind == _FOUR_F32:
            parts = torch.empty(3 * m * k, dtype=torch.bfloat16, device=rows.device)
        if form[0] == "ring":
            code = _at(dev, build.load("linear_quantized_ring").cb_linear_quantized_ring, *common, *form[1:], _ptr(parts), status)
        elif form[0] == "pairs":
            code = _at(dev, build.load("linear_quantized_pairs_tcgen05").cb_linear_quantized_pairs, *common, form[1],
                       form[2], status)
        else:
            code = _at(dev, build.load("linear_quantized_tcgen05").cb_linear_quantized_tcgen05, *common, form[1], form[2],
                       _ptr(parts), status)
        if kind == _FOUR_F32 and code == 0:
            LAUNCHES[0] += 1                           # (the rows' parts)
    if code == build.UNSUPPORTED:
        raise KernelError(f"{what}: sizes out of range: rows [{m}, {k}], weights [{n}, {k}]")
    _check(code, what)


def linear8(rows: torch.Tensor, row_scales: torch.Tensor, w: Weights8, out: torch.Tensor,
            add: Optional[torch.Tensor] = None) -> None:
    """out = (rows * row_scales) . W^T (+ add): e4m3 `rows` [M, K], float32 `row_scales` [M]; `out`: float32
    or bfloat16 [M, N]; `add`: float32 [M, N], which may be `out`.  K up to 2^20.  Rows that do not begin on
    multiples of 16 bytes (`new_rows8` makes such that do) are brought into ones that do, at every call."""
    if not isinstance(w, Weights8):
        raise KernelError(f"linear8 takes Weights8, got {type(w).__name__}")
    dev, shape, rs, os = rows.get_device(), rows.shape, rows.stride(), out.stride()
    n, k = w.shape
    if not (dev == w.device >= 0 and len(shape) == 2 and shape[1] == k and rows.dtype is E4M3 and row_scales.dtype is _F32
            and row_scales.shape == (shape[0],) and row_scales.is_contiguous() and out.dtype in _FLOATS
            and out.shape == (shape[0], n) and rs[1] == 1 == os[1] and rs[0] >= k and os[0] >= n
            and out.get_device() == dev == row_scales.get_device() and rs[0] % 16 == 0 and rows.data_ptr() % 16 == 0
            and (add is None or (add.dtype is _F32 and add.shape == out.shape and add.is_contiguous()
                                 and add.get_device() == dev))):
        _rows(rows, "linear8 rows", (E4M3,), (rows.shape[0], k))
        _vector(row_scales, "linear8 row scales", rows.shape[0])
        _out_rows(out, add, (rows.shape[0], n), "linear8")
        _need_cuda(rows, row_scales, w.values, out, add)
        _one_device(rows, row_scales, w.values, out, add)
        if not _aligned16(rows):
            rows = _in_aligned_rows(rows.view(torch.uint8)).view(E4M3)
        rs = (_pitch(rows),)
    _product(_EIGHT, dev, rows, shape[0], rs[0], row_scales.data_ptr(), w.values, w.pitch, None, w, 0, out, os[0],
             add, "linear (8-bit weights)")


def _slab(m: int, k: int) -> int:
    """Rows at a time, of m float32 rows over 4-bit weights: equal slabs, in tiles of 64."""
    most = max(64, min(_SLAB, _SCRATCH // (6 * k)) // 64 * 64)
    return min(most, _up(-(-m // -(-m // most)), 64))


def linear4(a: torch.Tensor, w: Weights4, out: torch.Tensor, add: Optional[torch.Tensor] = None) -> None:
    """out = a . W^T (+ add): float32 or bfloat16 rows `a` [M, K]; `out`: float32 or bfloat16 [M, N]; `add`:
    float32 [M, N], which may be `out`.  K up to 2^20.  Rows that do not begin on multiples of 16 bytes are brought
    into ones that do, at every call.  float32 rows take scratch memory from torch's pool for the call: 6 bytes a number for their
    bfloat16 parts, 512 MB at most (more rows than that holds are taken a part at a time)."""
    if not isinstance(w, Weights4):
        raise KernelError(f"linear4 takes Weights4, got {type(w).__name__}")
    dev, shape, rs, os = a.get_device(), a.shape, a.stride(), out.stride()
    n, k = w.shape
    f32 = a.dtype is _F32
    if not (dev == w.device >= 0 and len(shape) == 2 and shape[1] == k and a.dtype in _FLOATS and out.dtype in _FLOATS
            and out.shape == (shape[0], n) and rs[1] == 1 == os[1] and rs[0] >= k and os[0] >= n
            and out.get_device() == dev and rs[0] % 8 == 0 and a.data_ptr() % 16 == 0
            and (add is None or (add.dtype is _F32 and add.shape == out.shape and add.is_contiguous()
                                 and add.get_device() == dev))):
        _rows(a, "linear4 rows", _FLOATS, (a.shape[0], k))
        _out_rows(out, add, (a.shape[0], n), "linear4")
        _need_cuda(a, w.codes, out, add)
        _one_device(a, w.codes, out, add)
        if not _aligned16(a):
            a = _in_aligned_rows(a)
        rs = (_pitch(a),)
    if f32 and shape[0] > 64 and (shape[0] > _SLAB or 6 * k * shape[0] > _SCRATCH):
        rows = _slab(shape[0], k)
        for at in range(0, shape[0], rows):
            to = at + rows
            linear4(a[at:to], w, out[at:to], add=None if add is None else add[at:to])
        return
    _product(_FOUR_F32 if f32 else _FOUR_BF16, dev, a, shape[0], rs[0], None, w.codes, k // 2, w.group_scales.data_ptr(),
             w, w.group, out, os[0], add, "linear (4-bit weights)")

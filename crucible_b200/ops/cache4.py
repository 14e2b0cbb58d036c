"""A paged key/value cache in 4 bits: writing it, attention over it, and picking the pages to attend to.

A key or value row (one token, one kv head) is held by groups of `group` features as codes 0..15 with a bfloat16
pair (step, low) and stands for code * step + low.  low is the group's least number rounded down to bfloat16, step
is (largest - low) * (1 / 15) rounded to bfloat16 (0 if it is under 1e-30), the code is (x - low) * (1 / step)
rounded to the nearest, ties to even, and held within 0..15; every operation is float32's, rounded once.  A group
that holds a number that is not finite, or numbers further apart than float32 reaches, stands for NaN.  A number is off by at most half a
step, as it is rounded (a group's largest number lies up to 15.06 of these above the low).

`rope_append4` rotates q and k of packed rows by their positions and writes k and v to the rows' places;
`attention4` is causal grouped-query attention over what the pages hold, for single tokens, portions and whole
prompts; `pick_pages4` chooses for every row and kv head the pages whose bounds allow the largest logits, for
`attention4(..., picks=)` to read alone.  Pages that are to be picked keep bounds (`Pages4.new(..., bounds=True)`):
`rope_append4` brings those of every page that it writes up to date.

Long bfloat16 portions of heads of 64 and 128 go to the tensor cores' tiles in float16, whose waits are bounded and tell of
running out by the device's status word (`tensor_core.check_status`; a graph that is captured before there is one walks
instead).  There a value that is no number makes the whole head's result none for the rows that see it; elsewhere only its
group's features.  And there the keys of a request and kv head go into float16 by one power of two, as do the values: what is
more than 2^28 smaller than the largest of them that some row of the step sees loses bits, for the rows before that one, too.

Everything launches on torch's current stream of the tensors' device and may be captured into a CUDA graph; what is
allocated on the way (partial results of very long contexts, pages laid out anew for long portions, 2 GB at a time at most)
comes from torch's pool.  Outputs may not overlap inputs, but where a function says so.  Sums and softmax statistics are
float32.  Page ids, positions and row numbers on the device are looked over by the kernels: a key whose table entry names no
page of the pool is not seen, a row of a request that is none is left as it is.
"""
from __future__ import annotations

import functools
from operator import add as _add
from typing import Optional, Sequence

import torch

from . import KernelError, _check, _code, _need_cuda, build, tensor_core
from .quantized import _at, _one_device, _status

build.register_module("append4", ["common.cuh", "cache4.cuh"])
build.register_module("pick4", ["common.cuh", "cache4.cuh"])
HEAD_DIMS = (64, 128, 192, 256)
for _dim in HEAD_DIMS:
    build.register_module(f"attention4_{_dim}", ["common.cuh", "cache4.cuh", "attention4.cuh"])

GROUPS = (32, 64, 128)
_HALF_DIMS = tuple(d // 2 for d in HEAD_DIMS)
_F32, _BF16, _I32 = torch.float32, torch.bfloat16, torch.int32
_FLOATS = (_F32, _BF16)
_MOST_INT = (1 << 31) - 1
_LEAST_SCALE = 2.0 ** -126        # (one that float32 holds as a normal number, as it does one over it and either times log2 e)


class Pages4:
    """A pool of pages in 4 bits: `codes` uint8 [2, pages, kv heads, page tokens, dim / 2] (keys, values), `scales`
    bfloat16 [2, pages, kv heads, page tokens, dim / group, 2] (step, low); head sizes are multiples of 64 up to 256,
    groups 32, 64 or 128 features that divide them.  Bytes of a row are int32 words; word (dim / 64) g + w, g < 8,
    holds the codes of the features 64 w + 8 k + g, its bits 4n.. 4n + 3 that of k = (0, 1, 4, 5, 2, 3, 6, 7)[n].
    `bounds`: int8 [pages, kv heads, 2, dim] (largest, least key of each feature over the tokens that a page holds)
    with float32 `bound_scales` [pages, kv heads], or neither.  The tensors are kept, not copied."""

    __slots__ = ("codes", "scales", "bounds", "bound_scales", "n_pages", "kv_heads", "page_tokens", "head_dim", "group", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bounds: Optional[torch.Tensor] = None,
                 bound_scales: Optional[torch.Tensor] = None):
        # (one expression over what a pool usually is; only where it is not that are the tensors looked over one by one)
        cs, ss, dev = codes.shape, scales.shape, codes.get_device()
        if not (len(cs) == 5 and len(ss) == 6 and codes.dtype is torch.uint8 and scales.dtype is _BF16 and cs[0] == 2 == ss[5]
                and cs[4] in _HALF_DIMS and ss[:4] == cs[:4] and min(cs) > 0 < ss[4] and (2 * cs[4]) % ss[4] == 0
                and 2 * cs[4] // ss[4] in GROUPS and codes.is_contiguous() and scales.is_contiguous()
                and not (codes.data_ptr() | scales.data_ptr()) & 15 and scales.get_device() == dev
                and (bounds is None) is (bound_scales is None)
                and (bounds is None or (
                    bounds.dtype is torch.int8 and bounds.shape == (cs[1], cs[2], 2, 2 * cs[4]) and bounds.is_contiguous()
                    and not bounds.data_ptr() & 15 and bound_scales.dtype is _F32 and bound_scales.shape == cs[1:3]
                    and bound_scales.is_contiguous() and bounds.get_device() == dev == bound_scales.get_device()))):
            self._refuse(codes, scales, bounds, bound_scales)
        self.codes, self.scales, self.bounds, self.bound_scales = codes, scales, bounds, bound_scales
        _, self.n_pages, self.kv_heads, self.page_tokens, half = cs
        self.head_dim = 2 * half
        self.group, self.device = 2 * half // ss[4], dev

    @staticmethod
    def _refuse(codes, scales, bounds, bound_scales):
        cs, ss = codes.shape, scales.shape
        if len(cs) != 5 or cs[0] != 2 or codes.dtype != torch.uint8 or cs[4] not in _HALF_DIMS or not codes.is_contiguous():
            raise KernelError("a pool's codes are contiguous uint8 [2, pages, kv heads, page tokens, dim / 2] with dim in "
                              f"{HEAD_DIMS}, got {codes.dtype} {list(cs)}")
        dim = 2 * cs[4]
        if (len(ss) != 6 or ss[:4] != cs[:4] or ss[5] != 2 or scales.dtype != _BF16 or not scales.is_contiguous()
                or ss[4] < 1 or dim % ss[4] or dim // ss[4] not in GROUPS):
            raise KernelError("a pool's scales are contiguous bfloat16 [2, pages, kv heads, page tokens, dim / group, 2] with "
                              f"groups of {GROUPS}, got {scales.dtype} {list(ss)} for codes {list(cs)}")
        if min(cs) < 1:
            raise KernelError(f"a pool has pages, kv heads and tokens, got {list(cs)}")
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise KernelError("a pool's codes and scales begin on multiples of 16 bytes")
        if (bounds is None) != (bound_scales is None):
            raise KernelError("bounds come with their scales")
        _one_device(codes, scales, bounds, bound_scales)
        raise KernelError(f"bounds are contiguous int8 [{cs[1]}, {cs[2]}, 2, {dim}] that begin on a multiple of 16 bytes, with "
                          f"float32 scales [{cs[1]}, {cs[2]}], got {bounds.dtype} {list(bounds.shape)} and {bound_scales.dtype} "
                          f"{list(bound_scales.shape)}")

    @classmethod
    def new(cls, n_pages: int, page_tokens: int, kv_heads: int, head_dim: int, group: int = 64, bounds: bool = False,
            device="cuda:0") -> "Pages4":
        """Pages of zeros (every key and value stands for 0)."""
        if head_dim not in HEAD_DIMS or group not in GROUPS or head_dim % group:
            raise KernelError(f"pages in 4 bits take heads of {HEAD_DIMS} features in groups of {GROUPS} that divide them, "
                              f"got {head_dim} and {group}")
        if min(n_pages, page_tokens, kv_heads) < 1:
            raise KernelError("a pool has pages, kv heads and tokens")
        shape = (2, n_pages, kv_heads, page_tokens)
        kept = (torch.zeros(n_pages, kv_heads, 2, head_dim, dtype=torch.int8, device=device),
                torch.zeros(n_pages, kv_heads, device=device)) if bounds else ()
        return cls(torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device),
                   torch.zeros(*shape, head_dim // group, 2, dtype=_BF16, device=device), *kept)

    def values(self, dtype: torch.dtype = _F32):
        """What the pool stands for: (keys, values), each [pages, kv heads, page tokens, dim]."""
        if dtype not in _FLOATS:
            raise KernelError(f"pages are read back as float32 or bfloat16, not {dtype}")
        _need_cuda(self.codes)
        out = torch.empty(2, self.n_pages, self.kv_heads, self.page_tokens, self.head_dim, dtype=dtype, device=self.codes.device)
        lib = build.load("append4")
        _check(_at(self.device, lib.cb_values4, self.codes.data_ptr(), self.scales.data_ptr(), self.group,
                   2 * self.n_pages * self.kv_heads * self.page_tokens, self.head_dim, out.data_ptr(), _code(dtype)),
               "values in 4 bits")
        return out.unbind()

    def bound_values(self) -> torch.Tensor:
        """What the bounds stand for: float32 [pages, kv heads, 2, dim]."""
        if self.bounds is None:
            raise KernelError("these pages keep no bounds")
        _need_cuda(self.bounds)
        out = torch.empty_like(self.bounds, dtype=_F32)
        lib = build.load("append4")
        _check(_at(self.device, lib.cb_bound_values4, self.bounds.data_ptr(), self.bound_scales.data_ptr(),
                   self.n_pages * self.kv_heads, self.head_dim, out.data_ptr()), "bounds in 8 bits")
        return out


class Batch:
    """The packed rows of a step.  On the device, int32: `positions` [rows] and `row_request` [rows] (a row's position in
    its request, its request's number), `row_start` [requests + 1] and `first_pos` [requests] (where a request's
    rows begin, and the position of the first), `table` [requests, pages] (which page of the pool holds a
    request's tokens i * page_tokens onwards).  On the host: how many tokens of every request are
    `new_tokens`, its rows in this step, and `held_tokens`, before them.  A request's rows are consecutive and
    so are their positions; there are at least as many rows as they bring tokens.  Rows behind the last request's are left alone.

    A call that is captured into a graph may be replayed with other numbers on the device, as long as no request brings more rows
    than the most that the host was told of, the same leading requests bring one and, where a request brings more, no request
    then holds more tokens than at the capture; the kernels are shaped by the host's numbers, the results follow the device's.
    `reach`: the longest context that they are shaped for (as long as the host's numbers say, if it is not given); pages
    beyond it are not picked, only attention to all of them reads them."""

    __slots__ = ("positions", "row_request", "row_start", "first_pos", "table", "new_tokens", "held_tokens", "requests",
                 "rows", "stride", "most_new", "alike", "reach", "lead", "device")

    def __init__(self, positions, row_request, row_start, first_pos, table, new_tokens: Sequence[int],
                 held_tokens: Sequence[int], reach: Optional[int] = None):
        self.positions, self.row_request, self.row_start = positions, row_request, row_start
        self.first_pos, self.table = first_pos, table
        self.new_tokens, self.held_tokens = new_tokens, held_tokens
        self.requests = requests = len(new_tokens)
        self.device = dev = positions.get_device()
        # (shapes whole: asked for one size at a time they take twice as long)
        shape, pages = positions.shape, table.shape
        if not (requests > 0 and len(held_tokens) == requests and len(pages) == 2 and pages[0] == requests and pages[1] > 0
                and len(shape) == 1 and row_request.shape == shape and row_start.shape == (requests + 1,)
                and first_pos.shape == (requests,)
                and positions.dtype is _I32 and row_request.dtype is _I32 and row_start.dtype is _I32
                and first_pos.dtype is _I32 and table.dtype is _I32
                and positions.is_contiguous() and row_request.is_contiguous() and row_start.is_contiguous()
                and first_pos.is_contiguous() and table.is_contiguous()
                and dev == row_request.get_device() == row_start.get_device() == first_pos.get_device() == table.get_device()):
            self._refuse()
        self.rows, self.stride = shape[0], pages[1]
        self.most_new = most = max(new_tokens)
        self.alike = alike = requests == 1 or most == min(new_tokens)      # as many rows of every request
        if alike:
            self.lead = requests if most == 1 else 0
            longest = most + max(held_tokens)
        else:
            self.lead = next(i for i, n in enumerate(new_tokens) if n != 1)
            longest = max(map(_add, new_tokens, held_tokens))
        self.reach = longest if reach is None else reach
        if min(new_tokens) < 1 or min(held_tokens) < 0:
            raise KernelError("a batch's requests bring at least one token each, and hold none or more")
        if (most * requests if alike else sum(new_tokens)) > self.rows:
            raise KernelError(f"a batch's requests bring {sum(new_tokens)} tokens, but it has {self.rows} rows")

    def _refuse(self):
        t = {"positions": self.positions, "row_request": self.row_request, "row_start": self.row_start,
             "first_pos": self.first_pos, "table": self.table}
        _one_device(*t.values())
        raise KernelError("a batch takes contiguous int32 tensors positions [rows], row_request [rows], row_start [requests + 1], "
                          "first_pos [requests] and table [requests, pages], and two host lists with a number a request; got "
                          + ", ".join(f"{n} {v.dtype} {list(v.shape)}" for n, v in t.items())
                          + f", {len(self.new_tokens)} and {len(self.held_tokens)} numbers")

    @classmethod
    def of(cls, ctx, group: int) -> "Batch":
        """The step of a `StepContext`, over the pages of one of its cache groups."""
        made = ctx.__dict__.setdefault("_batches4", {})
        batch = made.get(group)
        if batch is None:
            host = ctx.host
            batch = made[group] = cls(ctx.positions, ctx.row_request, ctx.req_row_start, ctx.req_first_pos,
                                      ctx.block_table(group), host.new_tokens, host.first_pos, host.context_bucket)
        return batch


def _rows_ok(t: torch.Tensor, what: str, width: int, dtype, rows: int) -> int:
    """`rows` rows at least, of `width` numbers side by side; of `dtype`, or (None) float32 or bfloat16.  How far apart they are."""
    shape, strides = t.shape, t.stride()
    if not (len(shape) == 2 and shape[1] == width and (t.dtype is dtype if dtype is not None else t.dtype in _FLOATS)
            and strides[1] == 1 and (strides[0] >= width or shape[0] == 1) and shape[0] >= rows):
        names = "float32 or bfloat16" if dtype is None else str(dtype).replace("torch.", "")
        if t.dim() != 2 or t.shape[1] != width or t.dtype not in _FLOATS or (dtype is not None and t.dtype != dtype):
            raise KernelError(f"{what}: {names} rows [T, {width}] are taken, got {t.dtype} {list(t.shape)}")
        if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < width):
            raise KernelError(f"{what}: rows must be contiguous and not overlap")
        raise KernelError(f"{what}: the batch has {rows} rows, the tensor {t.shape[0]}")
    return strides[0]


def _same_device(what: str, batch: "Batch", pages: Pages4, *others) -> None:
    dev = pages.device
    if dev >= 0 and batch.device == dev:
        for t in others:
            if t is not None and t.get_device() != dev:
                break
        else:
            return
    _need_cuda(pages.codes, batch.positions, *others)
    raise KernelError(f"{what}: pages, batch and the other tensors lie on different devices")


def rope_append4(qkv: torch.Tensor, q: torch.Tensor, n_heads: int, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor],
                 batch: Batch, pages: Pages4, neighbours: bool = False, write: bool = True) -> None:
    """Rows [q : n_heads | k : kv heads | v : kv heads] of heads side by side: q rotated by the rows' positions goes to `q`
    (which may be the first columns of `qkv` themselves), k rotated and v as it is go to the rows' places in the
    pages, in 4 bits.  `cos`, `sin`: float32 [positions, r / 2], the angles of every position; the first r
    features of a head turn, (a, b) -> (a cos - b sin, a sin + b cos), feature i with i + r / 2 or (`neighbours`)
    2 i with 2 i + 1.  None: nothing turns.  Rows whose position is beyond the tables are left out.  No two rows are of one place.
    `write` False: q alone (the pages hold the rows already).
    With bounds, every page that the step wrote gets its own anew, from the tokens up to the last that it wrote there."""
    dim, kv = pages.head_dim, pages.kv_heads
    width = (n_heads + 2 * kv) * dim
    if n_heads < 1:
        raise KernelError("rope_append4: a positive number of query heads is needed")
    rows = batch.rows
    qkv_stride = _rows_ok(qkv, "rope_append4 rows", width, None, rows)
    q_stride = _rows_ok(q, "rope_append4 queries", n_heads * dim, qkv.dtype, rows)
    if (cos is None) != (sin is None):
        raise KernelError("rope_append4: cos and sin come together")
    rotary = positions = 0
    if cos is not None:
        shape = cos.shape
        rotary = 2 * shape[-1] if shape else 0
        if (len(shape) != 2 or cos.dtype is not _F32 or sin.dtype is not _F32 or sin.shape != shape or not cos.is_contiguous()
                or not sin.is_contiguous() or rotary > dim):
            raise KernelError(f"rope_append4: the tables are contiguous float32 [positions, r / 2] with r at most {dim}, got "
                              f"{cos.dtype} {list(cos.shape)} and {sin.dtype} {list(sin.shape)}")
        positions = shape[0]
    _same_device("rope_append4", batch, pages, qkv, q, cos, sin)
    lib = build.load("append4")
    code = _at(pages.device, lib.cb_append4, qkv.data_ptr(), _code(qkv.dtype), qkv_stride, q.data_ptr(), q_stride,
               cos.data_ptr() if rotary else 0, sin.data_ptr() if rotary else 0, rotary, positions, 1 if neighbours else 0,
               1 if write else 0, batch.positions.data_ptr(), batch.row_request.data_ptr(), batch.table.data_ptr(),
               batch.stride, batch.requests, pages.codes.data_ptr(), pages.scales.data_ptr(), pages.n_pages,
               pages.page_tokens, n_heads, kv, dim, pages.group, rows,
               pages.bounds.data_ptr() if pages.bounds is not None else 0,
               pages.bound_scales.data_ptr() if pages.bounds is not None else 0)
    _check(code, "rope_append4")


def pick_pages4(q: torch.Tensor, n_heads: int, batch: Batch, pages: Pages4, picks: torch.Tensor, first: int = 1,
                last: int = 2) -> None:
    """For every row and kv head `picks.shape[2]` of the request's pages up to the row's own, by their place in the table
    and in ascending order, -1 behind them where there are fewer: the `first` first and `last` last always, the others
    by the largest bound on a logit that a head of the group has in them, of equal ones the first.  `picks`: int32
    [rows, kv heads, count], or [n, ..] for the first n rows alone.  A query is rounded to 8 bits for it (largest magnitude
    127), as the bounds are."""
    dim, kv = pages.head_dim, pages.kv_heads
    rows = batch.rows
    _rows_ok(q, "pick_pages4 queries", n_heads * dim, None, rows)
    if n_heads < 1 or n_heads % kv:
        raise KernelError(f"pick_pages4: {n_heads} query heads do not share {kv} kv heads evenly")
    if pages.bounds is None:
        raise KernelError("pick_pages4: these pages keep no bounds")
    _picks_ok("pick_pages4", picks, kv)
    rows = min(picks.shape[0], rows)
    if first < 0 or last < 1 or first + last > picks.shape[2]:
        raise KernelError(f"pick_pages4: of {picks.shape[2]} pages the first {first} and the last {last} cannot always be "
                          "among them (the row's own page has to be)")
    _same_device("pick_pages4", batch, pages, q, picks)
    # scores are held for as many pages as the longest context may have
    most = min(batch.stride, -(-batch.reach // pages.page_tokens))
    lib = build.load("pick4")
    code = _at(pages.device, lib.cb_pick4, q.data_ptr(), _code(q.dtype), q.stride(0), batch.positions.data_ptr(),
               batch.row_request.data_ptr(), batch.table.data_ptr(), batch.stride, batch.requests,
               pages.bounds.data_ptr(), pages.bound_scales.data_ptr(), pages.n_pages, pages.page_tokens, n_heads // kv, kv,
               dim, rows, picks.data_ptr(), picks.shape[2], first, last, most, _pick_shares(rows * kv, most))
    if code == build.UNSUPPORTED:
        raise KernelError(f"pick_pages4 takes tables of up to {most_pages(n_heads // kv, dim)} pages a request here, got {most}; "
                          "longer pages make shorter tables")
    _check(code, "pick_pages4")


def most_pages(n_rep: int, head_dim: int) -> int:
    """Pages that a request may have for `pick_pages4`, `n_rep` query heads on a kv head."""
    return (build.load("pick4").cb_pick4_room() - n_rep * (2 * head_dim + 4)) // 16 * 4


def _pick_shares(blocks: int, pages: int) -> int:
    """Blocks of a cluster that score a row's pages: as many as fill the SMs, none with fewer than 128 pages."""
    shares = 1
    while shares < 8 and blocks * shares * 2 <= 2 * tensor_core.N_SMS and pages >= 256 * shares:
        shares *= 2
    return shares


def _picks_ok(what: str, picks: torch.Tensor, kv_heads: int) -> None:
    if (picks.dim() != 3 or picks.dtype != _I32 or not picks.is_contiguous() or picks.shape[1] != kv_heads
            or min(picks.shape) < 1):
        raise KernelError(f"{what}: the picks are contiguous int32 [rows, {kv_heads}, count], got {picks.dtype} {list(picks.shape)}")


def attention4(q: torch.Tensor, out: torch.Tensor, n_heads: int, scale: float, batch: Batch, pages: Pages4,
               window: Optional[int] = None, picks: Optional[torch.Tensor] = None) -> None:
    """out = softmax(scale q . k) v (`scale` from 2^-126 to 2^126): every row over the keys of its request up to its own position (the last `window` of
    them), heads of a group over the same kv head (head h over h // (n_heads / kv heads)).  `q`, `out`: rows [T,
    n_heads * dim] of one type.  A row that sees no key is zero.  `picks` (int32 [rows, kv heads, count], as
    `pick_pages4` leaves them): the pages of the table that a row attends to, each named once, -1 for none; every row is then
    walked by itself, so that this is for a few rows a request; page sizes are multiples of 16, and there is no window.
    Picks of the first n rows alone are for the first n requests, which bring one row each; the others attend to all."""
    dim, kv = pages.head_dim, pages.kv_heads
    rows = batch.rows
    _rows_ok(q, "attention4 queries", n_heads * dim, None, rows)
    _rows_ok(out, "attention4 output", n_heads * dim, q.dtype, rows)
    if n_heads < 1 or n_heads % kv:
        raise KernelError(f"attention4: {n_heads} query heads do not share {kv} kv heads evenly")
    if window is not None and window < 1:
        raise KernelError(f"attention4: a window is positive, got {window}")
    if window is not None and window > _MOST_INT:          # (more than any position; kernels take 32 bits of it)
        window = _MOST_INT
    if not _LEAST_SCALE <= scale <= 1.0 / _LEAST_SCALE:
        raise KernelError(f"attention4: the scale is a positive number from {_LEAST_SCALE:.3g} to {1.0 / _LEAST_SCALE:.3g}, got {scale}")
    behind = 0
    if picks is not None:
        _picks_ok("attention4", picks, kv)
        if window is not None or pages.page_tokens % 16:
            raise KernelError("attention4: picks go with pages of a multiple of 16 tokens and without a window")
        behind = picks.shape[0]
        if behind < rows and behind > batch.lead:
            raise KernelError(f"attention4: picks of {behind} of {rows} rows, but only the first {batch.lead} requests bring one row")
    _same_device("attention4", batch, pages, q, out, picks)
    if picks is not None:
        _walk(q, out, n_heads, scale, batch, pages, None, picks, 0, 0)
    if behind < min(rows, batch.requests):
        lead = max(behind, batch.lead)
        if lead < batch.requests and _laid_out(q, out, n_heads, batch, pages, window, behind, lead):
            if behind < lead:
                _walk(q, out, n_heads, scale, batch, pages, window, None, behind, lead)
            for first, last, counts in _slabs(batch, window, lead, _MOST_BLOCKS // (kv * dim)):
                if counts is None or not _tiles(q, out, n_heads, scale, batch, pages, window, first, last, counts):
                    _walk(q, out, n_heads, scale, batch, pages, window, None, first, last)
            return
        _walk(q, out, n_heads, scale, batch, pages, window, None, behind, batch.requests)


def _most_rows(batch, first, last) -> int:
    """Rows that a launch over the requests first .. last - 1 takes of each: as many as a replay may bring there."""
    return 1 if last <= batch.lead else batch.most_new


def _resident(dim: int, group: int, columns: int, f32: bool) -> int:
    """Blocks of the walking kernel that the SMs hold at once."""
    return tensor_core.N_SMS * (2 if dim > 128 or columns > 1 else 4 if dim // group * (2 if f32 else 1) <= 2 else 3)


@functools.lru_cache(maxsize=4096)
def _shares(blocks: int, tiles: int, total: int, resident: int, weight: float = 1.0) -> tuple:
    """(blocks of a cluster, blocks of a stream or 0, us that it may take): how the keys are dealt, by the launch's row tiles of
    all kv heads (`blocks`), the most tiles of 16 keys that one of them sees, how many they see in all, and the blocks that
    the SMs hold.  A model of what either takes, in us.  A block takes a round of eight tiles in 0.7 alone on its SM and in
    0.53 times the blocks beside it (heads of 128, bfloat16; `weight` for others), and 5 to begin and to end, a cluster half
    more; a launch takes 2.  A stream's blocks take 1.1 and 0.24 times their number on the SM for a round (theirs are not
    alike), and it 10.5 besides, 0.8 more for every 100 blocks, whose results are put together.  Modelled and measured, us:
    1 token of 32 heads of 128 on 8 behind 16,000 keys, clusters of 8 19 and 17, a stream of three blocks an SM 18 and 18;
    behind 131,071 clusters 97 and 105, a stream 44 and 41; 8 behind up to 16,000, clusters of 8 37 and 35, a stream 38
    and 38; 32 clusters of 8 116 and 105, a stream 103 and 100."""
    per_sm = resident / tensor_core.N_SMS
    best = None
    for shares in (1, 2, 4, 8):
        rounds = -(-tiles // (8 * shares))
        each = weight * max(0.7, 0.53 * min(blocks * shares / tensor_core.N_SMS, per_sm))
        mean = total / (8 * shares * blocks)
        waves = blocks * shares / resident
        if waves < 2.0:
            waves = -(-blocks * shares // resident)
        us = 2.0 + waves * (5.0 + mean * each) + max(0.0, rounds - mean) * each + 0.1 * shares + (0.4 if shares > 1 else 0.0)
        if best is None or us < best[0]:
            best = us, shares
        if rounds == 1:
            break
    if best[0] > 10.5 and total < 1 << 30 and blocks < 4 * resident:
        us, stream = min((max(1.0, weight) * (10.5 + 0.008 * each) + weight * (1.1 + 0.24 * n) * max(1.0, total / (8 * each)), each)
                         for n in range(1, int(per_sm) + 1) for each in (max(1, min(n * tensor_core.N_SMS, total // 8)),))
        us += 3.0 * blocks / resident
        if us < best[0]:
            return 1, stream, us
    return best[1], 0, best[0]


def _dealt(dim, kv, n_rep, group, f32, batch, window, first, last) -> tuple:
    """How the requests first .. last - 1 go through the walking kernel: (column tiles a block, blocks of a cluster, blocks of a
    stream, us that it may take)."""
    requests = last - first
    new, held = batch.new_tokens, batch.held_tokens
    if requests < batch.requests:
        new, held = new[first:last], held[first:last]
        most_rows, alike = max(new), max(new) == min(new)
    else:
        most_rows, alike = batch.most_new, batch.alike
    reach = batch.reach if window is None else min(batch.reach, window + most_rows)
    tiles = -(-reach // 16) + (window is not None)
    columns = _columns(n_rep, f32, dim, most_rows)
    if alike:
        per = kv * -(-most_rows * n_rep // (8 * columns))
        blocks = requests * per
        total = per * (requests * tiles if requests == 1 or window is not None else (sum(held) + sum(new)) // 16 + requests)
    else:                                                  # (blocks behind a request's last row end at once)
        per = [kv * -(-n * n_rep // (8 * columns)) for n in new]
        blocks = sum(per)
        total = sum([p * min(tiles, (n + h) // 16 + 1) for p, n, h in zip(per, new, held)])
    return columns, *_dealt_to(dim, group, f32, columns, blocks, tiles, total)


def _columns(n_rep, f32, dim, most_rows) -> int:
    return 1 if f32 or most_rows * n_rep <= 8 or dim > 128 else 2


def _dealt_to(dim, group, f32, columns, blocks, tiles, total) -> tuple:
    return _shares(blocks, tiles, total, _resident(dim, group, columns, f32),
                   (dim / 128) ** 0.6 * (2.0 if f32 else 1.3 if columns == 2 else 1.0))


def _walk(q, out, n_heads, scale, batch, pages, window, picks, first, last) -> None:
    """The kernel that walks the cache as it lies: for the requests first .. last - 1 of the batch, or for the rows that
    have picks."""
    dim, kv = pages.head_dim, pages.kv_heads
    n_rep, f32 = n_heads // kv, q.dtype is _F32
    rows = batch.rows
    if picks is not None:
        most_rows, blocks = 1, min(rows, picks.shape[0])
        tiles = picks.shape[2] * pages.page_tokens // 16
        columns = _columns(n_rep, f32, dim, 1)
        per = blocks * kv * -(-n_rep // (8 * columns))
        shares, stream, _ = _dealt_to(dim, pages.group, f32, columns, per, tiles, tiles * per)
    else:
        most_rows = _most_rows(batch, first, last)
        columns, shares, stream, _ = _dealt(dim, kv, n_rep, pages.group, f32, batch, window, first, last)
    partial = torch.empty(stream * 16 * columns * (dim + 2), dtype=_F32, device=q.device) if stream else None
    lib = build.load(f"attention4_{dim}")
    code = _at(pages.device, lib.cb_attention4, q.data_ptr(), _code(q.dtype), q.stride()[0], out.data_ptr(), out.stride()[0],
               pages.codes.data_ptr(), pages.scales.data_ptr(), pages.n_pages, pages.page_tokens, kv, n_rep, pages.group,
               batch.row_start.data_ptr() + 4 * first, batch.first_pos.data_ptr() + 4 * first,
               batch.table.data_ptr() + 4 * first * batch.stride, batch.stride,
               batch.requests if picks is not None else last - first,
               picks.data_ptr() if picks is not None else 0, picks.shape[2] if picks is not None else 0,
               batch.row_request.data_ptr(), batch.positions.data_ptr(),
               rows if picks is None else min(rows, picks.shape[0]), most_rows, window or 0, scale, columns,
               shares, stream, partial.data_ptr() if partial is not None else 0)
    if code == build.UNSUPPORTED:
        raise KernelError(f"attention4: {rows} rows of {n_heads} heads are more than a launch takes")
    _check(code, "attention4")


LAID_OUT: Optional[bool] = None       # tests fix which way portions go


def _laid_out(q, out, n_heads, batch, pages, window, behind, first) -> bool:
    """Whether the portions of the requests from `first` on go by `_tiles`, those from `behind` on before them walked by
    themselves: bfloat16 rows of heads of 64 and 128, 64 of a kv head and more (others have no kernel there that is quicker).
    us, by what was measured: 8.5 and 1.7 a million features laid out, then a tile of 128 rows walks its keys alone, 7.2
    a thousand, or all of them at 0.75 PFLOP/s."""
    dim, kv = pages.head_dim, pages.kv_heads
    new, held = batch.new_tokens[first:], batch.held_tokens[first:]
    n_rep = n_heads // kv
    if (q.dtype is not _BF16 or dim > 128 or q.stride(0) % 8 or out.stride(0) % 8 or q.data_ptr() % 16 or out.data_ptr() % 16
            or max(new) * n_rep < 64 or not _status(pages.device)):
        return False
    if LAID_OUT is not None:
        return LAID_OUT
    walk = _dealt(dim, kv, n_rep, pages.group, False, batch, window, behind, batch.requests)[3]
    reach = max(map(_add, new, held))
    seen = reach if window is None else min(reach, window + 128)
    pairs = sum([n * min(h + n / 2, seen) for n, h in zip(new, held)])
    laid = sum(new) + sum(held) if window is None else sum([n + min(h, window) for n, h in zip(new, held)])
    tiles = 8.5 + 1.7e-6 * laid * kv * dim + max(0.0072 * min(seen, reach), 4e-6 * dim * n_heads * pairs / 750.0)
    if behind < first:
        tiles += _dealt(dim, kv, n_rep, pages.group, False, batch, window, behind, first)[3]
    return tiles < walk


_MOST_BLOCKS = (2 << 30) // (64 * 4)  # of 64 tokens and a feature that are laid out at a time: 2 GB of keys and values


def _slabs(batch, window, first, most):
    """The requests from `first` on, as many at a time as `most` blocks of 64 tokens hold: (first, last, the blocks of each, or
    None where one request alone has more).  With a window, as many blocks as the step's rows can reach wherever they begin."""
    new, held = batch.new_tokens, batch.held_tokens
    counts, total = [], 0
    for r in range(first, batch.requests):
        n = -(-(new[r] + held[r]) // 64)
        if window is not None:
            n = min(n, (window + batch.most_new + 62) // 64 + 1)     # (a replayed request may bring as many rows as any)
        if total + n > most:
            if counts:
                yield first, r, counts
            first, counts, total = r, [], 0
            if n > most:
                yield r, r + 1, None
                first = r + 1
                continue
        counts.append(n)
        total += n
    if counts:
        yield first, batch.requests, counts


def _tiles(q, out, n_heads, scale, batch, pages, window, first, last, counts) -> bool:
    """bfloat16 portions of many rows: the keys and values of the requests first .. last - 1 are laid out once, in blocks of
    64 tokens (not taken apart again for every tile of rows), and attention runs over these on tcgen05.  Queries, keys, values
    and p are float16 there, with a power of two for each row, key head and value head: eleven bits of them (in bfloat16 the
    results were off by 0.0033 of themselves, half of it the roundings inside, in float16 by 0.0017, which is their own)."""
    dim, kv = pages.head_dim, pages.kv_heads
    new, held = batch.new_tokens[first:last], batch.held_tokens[first:last]
    n_blocks, stride, requests, rows = sum(counts), -(-max(map(_add, new, held)) // 64), len(counts), batch.rows
    both = torch.empty(2, n_blocks + 1, kv, 64, dim, dtype=torch.float16, device=q.device)
    spans = torch.empty(2 * n_blocks * kv + 3 * requests * stride, dtype=_I32, device=q.device)
    seen, blocks = spans[2 * n_blocks * kv:], spans[2 * (n_blocks * kv + requests * stride):]
    factors = torch.empty(2 * requests * kv, dtype=_F32, device=q.device)
    starts, places = batch.row_start.data_ptr() + 4 * first, batch.first_pos.data_ptr() + 4 * first
    _check(_at(pages.device, build.load("append4").cb_expand4, pages.codes.data_ptr(), pages.scales.data_ptr(), pages.n_pages,
               pages.page_tokens, kv, dim, pages.group, starts, places, batch.table.data_ptr() + 4 * first * batch.stride,
               batch.stride, requests, window or 0, both[0].data_ptr(), both[1].data_ptr(), spans.data_ptr(),
               factors.data_ptr(), seen.data_ptr(), blocks.data_ptr(), stride, n_blocks, rows), "pages laid out")
    code = _at(pages.device, build.load("attention_tcgen05").cb_attention_tcgen05_half, q.data_ptr(), q.stride(0), rows,
               out.data_ptr(), out.stride(0), both[0].data_ptr(), both[1].data_ptr(), n_blocks + 1, starts, places,
               blocks.data_ptr(), stride, requests, _most_rows(batch, first, last), n_heads, kv, dim, scale, window or 0, factors.data_ptr(),
               seen.data_ptr(), _status(pages.device))
    if code == build.UNSUPPORTED:
        return False
    _check(code, "attention4 (tiles)")
    return True

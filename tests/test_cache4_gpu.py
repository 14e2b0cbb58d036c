"""The cache in 4 bits on the GPU: what is written, attention over it, and which pages are picked."""
import pytest
import torch

import cache4_cases as cc

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"


def _append(case, qkv, q, rotary, neighbours=False, tables=None):
    from crucible_b200.ops import cache4
    cos, sin = tables or cc.tables(int(case.positions.max()) + 1, rotary // 2, DEV) if rotary else (None, None)
    cache4.rope_append4(qkv, q, case.heads, cos, sin, case.batch, case.pages, neighbours=neighbours)
    return cos, sin


def _expected_rows(case, qkv, cos, sin, neighbours):
    """(q float64, k and v codes, steps, lows)."""
    rows = qkv.double().view(qkv.shape[0], -1, case.dim)
    both = rows[:, :case.heads + case.kv_heads]
    if cos is not None:
        at = case.positions.long()
        both = cc.turned(both, cos[at], sin[at], neighbours)
    return (both[:, :case.heads].flatten(1), cc.coded(both[:, case.heads:], case.group),
            cc.coded(rows[:, case.heads + case.kv_heads:], case.group))


def _check_append(case, before, got_q, expected):
    q, *sides = expected
    assert torch.equal(got_q, q.to(case.dtype))
    where = case.table[case.row_request.long(), torch.div(case.positions, case.page, rounding_mode="floor").long()].long()
    slot = (case.positions % case.page).long()
    codes, scales = before
    for side, (code, step, low) in enumerate(sides):
        codes[side, where, :, slot] = cc.packed(code)
        scales[side, where, :, slot] = torch.stack((step, low), dim=-1)
    assert torch.equal(case.pages.codes, codes)                        # (what was not written is as it was)
    assert torch.equal(case.pages.scales.view(torch.int16), scales.view(torch.int16))


@pytest.mark.parametrize("dim,group,rotary,neighbours,page,dtype", [
    (64, 64, 64, False, 16, BF16), (64, 32, 32, True, 5, F32), (128, 128, 128, False, 16, BF16),
    (128, 64, 64, False, 24, BF16), (128, 32, 128, True, 64, F32), (192, 32, 96, False, 16, BF16),
    (192, 64, 2, False, 7, F32), (256, 128, 256, False, 32, BF16), (256, 32, 0, False, 16, F32), (128, 64, 6, True, 16, BF16)])
def test_append_to_the_bit(dim, group, rotary, neighbours, page, dtype):
    case = cc.Case([(0, 3), (17, 1), (30, 40), (63, 1)], dim=dim, group=group, page=page, dtype=dtype, seed=dim + group + page)
    width = (case.heads + 2 * case.kv_heads) * dim
    wide = case.normal(case.rows, width + 3).to(dtype)                   # rows apart, at odd offsets
    qkv = wide[:, 3:]
    out = torch.zeros(case.rows, case.heads * dim + 5, dtype=dtype, device=DEV)
    before = (case.pages.codes.clone(), case.pages.scales.clone())
    cos, sin = _append(case, qkv, out[:, :case.heads * dim], rotary, neighbours)
    _check_append(case, before, out[:, :case.heads * dim], _expected_rows(case, qkv, cos, sin, neighbours))
    assert not out[:, case.heads * dim:].any()


def test_append_over_its_own_rows_and_rows_that_are_left():
    """q in its own place; rows of no request, rows beyond the tables of angles and rows whose page is none."""
    case = cc.Case([(0, 20), (3, 4), (9, 2)], dim=64, page=8, seed=3)
    width = (case.heads + 2 * case.kv_heads) * 64
    qkv = case.normal(case.rows + 5, width).to(BF16)                       # five rows behind the batch's
    first = qkv.clone()
    before = (case.pages.codes.clone(), case.pages.scales.clone())
    tables = cc.tables(18, 32, DEV)                                     # positions 18 and 19 have no angles
    case.row_request[21] = -1
    case.row_request[22] = 3
    case.table[2, 1] = case.n_pages                                      # row 24, 25 (positions 9, 10): no such page
    _append(case, qkv, qkv[:, :case.heads * 64], 64, tables=tables)
    untouched = [18, 19, 21, 22] + list(range(case.rows, case.rows + 5))
    assert torch.equal(qkv[untouched], first[untouched])
    keep = [r for r in range(case.rows) if r not in untouched]
    case.positions, case.row_request, case.rows = case.positions[keep], case.row_request[keep], len(keep)
    q, *sides = _expected_rows(case, first[keep], *tables, False)
    assert torch.equal(qkv[keep, :case.heads * 64], q.to(BF16))
    assert torch.equal(qkv[:, case.heads * 64:], first[:, case.heads * 64:])
    for name, was in zip(("codes", "scales"), before):
        now = getattr(case.pages, name)
        changed = (now != was).flatten(4).any(dim=-1)
        written = torch.zeros_like(changed)
        for p, r in zip(case.positions.tolist(), case.row_request.tolist()):
            page = int(case.table[r, p // 8])
            if page < case.n_pages:
                written[:, page, :, p % 8] = True
        assert not (changed & ~written).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_groups_that_are_hard_to_code(dtype):
    """All numbers alike, almost alike, far from zero, far apart, huge, tiny, and not finite."""
    case = cc.Case([(0, 12)], dim=64, group=32, kv_heads=1, n_rep=1, dtype=dtype, seed=9)
    base = case.normal(12, 3 * 64)
    base[0] = 1.7
    base[1] = -1e-3 + 1e-9 * base[1]
    base[2] = 1000.0 + 0.01 * base[2]
    base[3, ::7] = 500.0
    base[4] *= 1e36
    base[5] *= 1e-36
    base[6] = 0.0
    base[7, 64::2], base[7, 65::2] = 0.0, -0.0
    base[8, 70] = float("nan")
    base[9, 70] = float("inf")
    base[10, 140] = -float("inf")
    base[11, 130], base[11, 135] = 3.0e38, -3.0e38
    qkv = base.to(dtype)
    q = torch.empty(12, 64, dtype=dtype, device=DEV)
    before = (case.pages.codes.clone(), case.pages.scales.clone())
    _append(case, qkv, q, 0)
    k, v = case.pages.values()
    place = case.table[0, 0].long()
    rows = torch.stack((k[place, 0, :12], v[place, 0, :12]), dim=1).double()        # [12, 2, 64]
    bad = torch.zeros(12, 2, 2, dtype=torch.bool, device=DEV)                       # row, side, group
    bad[8, 0, 0] = bad[9, 0, 0] = bad[10, 1, 0] = bad[11, 1, 0] = True
    spread = bad.repeat_interleave(32, dim=2)
    assert rows[spread].isnan().all() and rows[~spread].isfinite().all()
    fine = [r for r in range(12) if r not in (8, 9, 10, 11)]
    expected = [cc.coded(qkv.double()[fine, 64 * (1 + s):64 * (2 + s)], 32) for s in (0, 1)]
    for side, (code, step, low) in enumerate(expected):
        assert torch.equal(case.pages.codes[side, place, 0, fine], cc.packed(code))
        assert torch.equal(case.pages.scales[side, place, 0, fine].float(), torch.stack((step, low), dim=-1).float())
        # off by half a step at most, and by what the rounding of the step cuts off the largest (15 steps of 2^-8)
        got = rows[fine][:, side]
        x = qkv.double()[fine, 64 * (1 + side):64 * (2 + side)]
        room = step.double().repeat_interleave(32, dim=1) * (0.5 + 15 * 2.0 ** -8 + 1e-5) + LEAST
        assert ((got - x).abs() <= room).all()
    del before


LEAST = 15 * cc.LEAST_STEP


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 32), (192, 64), (256, 128)])
def test_values_read_back(dim, group, dtype):
    case = cc.Case([(0, 30)], dim=dim, group=group, page=7, seed=dim)
    want = case.contents()
    for got, w in zip(case.pages.values(dtype), want):
        assert torch.equal(got, w.float().to(dtype))


def _bounds_by_definition(case, page, held):
    k = case.contents()[0, page, :, :held]
    both = cc.once(torch.stack((k.amax(dim=1), k.amin(dim=1)), dim=1))
    scale = cc.once(both.abs().amax(dim=(1, 2)) * cc.OF_127)
    inverse = torch.where(scale > 0, cc.once(1.0 / scale.clamp_min(1e-300)), 0.0)
    return torch.round(cc.once(both * inverse[:, None, None])), scale


@pytest.mark.parametrize("dim,page,dtype", [(64, 16, BF16), (128, 24, F32), (192, 64, BF16), (256, 5, BF16)])
def test_bounds_follow_what_is_written(dim, page, dtype):
    case = cc.Case([(0, 33), (page - 1, 1), (2 * page, 1), (7, page + 3)], dim=dim, page=page, dtype=dtype, seed=page, bounds=True)
    case.pages.bounds.fill_(55)
    qkv = case.normal(case.rows, (case.heads + 2 * case.kv_heads) * dim).to(dtype)
    _append(case, qkv, torch.empty(case.rows, case.heads * dim, dtype=dtype, device=DEV), dim)
    held = {}
    for p, r in zip(case.positions.tolist(), case.row_request.tolist()):
        held[int(case.table[r, p // page])] = max(held.get(int(case.table[r, p // page]), 0), p % page + 1)
    for i in range(case.n_pages):
        if i not in held:
            assert (case.pages.bounds[i] == 55).all() and (case.pages.bound_scales[i] == 0).all()
            continue
        want, scale = _bounds_by_definition(case, i, held[i])
        assert torch.equal(case.pages.bounds[i].double(), want) and torch.equal(case.pages.bound_scales[i].double(), scale)


def test_bounds_where_the_angles_end():
    """Rows beyond the tables of angles are left out: the page's bounds are those of the rows before them."""
    case = cc.Case([(0, 16)], dim=64, page=16, seed=31, bounds=True)
    qkv = case.normal(16, (case.heads + 2 * case.kv_heads) * 64).to(BF16)
    _append(case, qkv, torch.empty(16, case.heads * 64, dtype=BF16, device=DEV), 64, tables=cc.tables(11, 32, DEV))
    place = int(case.table[0, 0])
    want, scale = _bounds_by_definition(case, place, 11)
    assert torch.equal(case.pages.bounds[place].double(), want) and torch.equal(case.pages.bound_scales[place].double(), scale)


def _attend(case, q, scale, **more):
    from crucible_b200.ops import cache4
    out = torch.full((q.shape[0], case.heads * case.dim), 7.0, dtype=q.dtype, device=q.device)
    cache4.attention4(q, out, case.heads, scale, case.batch, case.pages, **more)
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,group,n_rep,kv_heads,page,requests", [
    (64, 64, 3, 4, 16, [(700, 1)]),
    (64, 32, 1, 2, 16, [(0, 1), (15, 1), (16, 1), (300, 1)]),
    (128, 64, 4, 2, 16, [(1, 1), (2, 2), (200, 3), (500, 1)]),
    (128, 128, 8, 1, 64, [(1023, 1), (63, 1), (64, 1)]),
    (128, 32, 7, 2, 24, [(77, 1), (5, 9), (260, 2)]),
    (192, 32, 2, 1, 7, [(100, 1), (0, 5)]),
    (192, 64, 9, 1, 32, [(250, 1), (31, 2)]),
    (256, 32, 5, 1, 16, [(130, 2), (0, 1)]),
    (256, 128, 16, 1, 5, [(61, 1), (3, 3)]),
    (256, 64, 33, 1, 16, [(90, 1)]),
])
def test_attention_of_few_rows(dim, group, n_rep, kv_heads, page, requests, dtype, monkeypatch):
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", False)               # (the kernel that walks the pages as they lie)
    case = cc.Case(requests, dim=dim, group=group, n_rep=n_rep, kv_heads=kv_heads, page=page, dtype=dtype, seed=dim + n_rep)
    q = case.queries(1.5)
    want, most = case.attention(q, dim ** -0.5)
    cc.assert_attention(_attend(case, q, dim ** -0.5), want, most, dtype)


@pytest.mark.parametrize("dim,group,n_rep,kv_heads,page,requests,window", [
    (64, 64, 3, 2, 16, [(0, 70)], None), (64, 32, 1, 3, 16, [(5, 100), (0, 33)], None), (128, 64, 4, 1, 16, [(200, 40)], None),
    (128, 128, 2, 2, 24, [(30, 65), (129, 64), (0, 130)], None), (128, 32, 7, 1, 7, [(90, 31)], None),
    (64, 64, 4, 2, 64, [(40, 1), (17, 1), (0, 200), (300, 20)], None), (128, 64, 4, 1, 16, [(200, 1), (250, 90), (0, 64)], 100),
    (64, 64, 2, 2, 16, [(500, 40)], 17), (64, 64, 32, 1, 16, [(70, 5), (0, 9)], None), (128, 128, 5, 1, 8, [(3, 140)], None),
    (64, 32, 1, 3, 16, [(0, 64), (1000, 70)], None), (128, 128, 4, 1, 24, [(3000, 70), (5, 1), (64, 66), (0, 60)], 130), (128, 64, 130, 1, 16, [(10, 3)], None)])
def test_attention_of_portions_that_are_laid_out(dim, group, n_rep, kv_heads, page, requests, window, monkeypatch):
    """Long portions, decoded tokens at the step's head walked beside them; what the window has passed is not read."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    tiled, tiles = [], cache4._tiles
    monkeypatch.setattr(cache4, "_tiles", lambda *a: tiled.append(tiles(*a)) or tiled[-1])
    case = cc.Case(requests, dim=dim, group=group, n_rep=n_rep, kv_heads=kv_heads, page=page, seed=dim + n_rep)
    if window is not None:
        for r, (held, new) in enumerate(requests):
            case.table[r, :max(0, held - window + 1) // page] = [-1, case.free][r % 2]
        case.pages.scales[:, case.free] = float("nan")
    scale = dim ** -0.5
    q, spread = case.queries(1.5), []
    want, most = case.attention(q, scale, window=window, spread=spread)
    got = _attend(case, q, scale, window=window)
    assert tiled == [True]
    cc.assert_attention_laid_out(got, want, most, spread[0])
    single = sum(1 for _, n in requests if n == 1)
    cc.assert_attention(got[:single], want[:single], most[:single], BF16) if single else None


@pytest.mark.parametrize("size,stretch,scale", [(1e-7, 1.0, 1.0), (1e8, 1.0, 1e-9), (1.0, 1e-15, 1e14), (1.0, 1e15, 1e-16),
                                                (1e-20, 1e20, 0.1), (1e25, 1e-22, 1e-3), (1e-20, 1e-22, 0.1)])
def test_sizes_in_portions_that_are_laid_out(size, stretch, scale, monkeypatch):
    """Keys and queries whose numbers float16 would not hold as they are."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    case = cc.Case([(30, 50), (0, 40)], dim=64, group=32, n_rep=4, kv_heads=1, seed=23, size=size)
    case.pages.scales[1] *= 1e-3 / size                           # values as ever
    q, spread = case.queries(stretch), []
    q[0, :64] = 0
    want, most = case.attention(q, scale, spread=spread)
    cc.assert_attention_laid_out(_attend(case, q, scale), want, most, spread[0])


@pytest.mark.parametrize("window", [None, 70])
def test_places_without_a_page_in_portions_that_are_laid_out(window, monkeypatch):
    """What the table does not name is not seen, here too; a row that sees nothing is zero."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    case = cc.Case([(300, 40), (0, 150), (0, 33)], dim=64, group=64, n_rep=4, kv_heads=2, page=16, seed=31)
    case.table[0, 3:7] = torch.tensor([-1, case.n_pages, -(1 << 31), 1 << 30], device=DEV)
    case.table[0, 17] = -1
    case.table[1, :2] = -1
    case.table[1, 8] = -1
    q, spread = case.queries(), []
    want, most = case.attention(q, 0.125, window=window, spread=spread)
    got = _attend(case, q, 0.125, window=window)
    assert (got[40:72] == 0).all()
    cc.assert_attention_laid_out(got, want, most, spread[0])
    case.table = case.table[:, :9].contiguous()                    # (positions behind 143 are of no page then)
    case.stride, case.batch = 9, None
    case.batch = case.make_batch()
    spread.clear()
    want, most = case.attention(q, 0.125, window=window, spread=spread)
    cc.assert_attention_laid_out(_attend(case, q, 0.125, window=window), want, most, spread[0])


def test_portions_laid_out_of_a_captured_step(monkeypatch):
    """Replayed with other queries, other places and fewer tokens; and captured where no wait that runs out could be told."""
    from crucible_b200.ops import cache4, tensor_core
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    case = cc.Case([(5, 1), (120, 40), (0, 90)], dim=128, group=64, n_rep=3, kv_heads=1, seed=33)
    q = case.queries()
    outs = [torch.empty_like(q) for _ in range(3)]

    def step(out):
        cache4.attention4(q, out, case.heads, 0.1, case.batch, case.pages)
    step(outs[0])
    graphs = [torch.cuda.CUDAGraph() for _ in range(3)]
    for i, (graph, out) in enumerate(zip(graphs, outs)):
        if i == 2:
            monkeypatch.setattr(tensor_core, "_status", {})
        with torch.cuda.graph(graph):
            step(out)
    for requests in ([(5, 1), (120, 40), (0, 90)], [(4, 1), (60, 30), (3, 80)], [(0, 1), (0, 1), (1, 1)]):
        case.requests = requests
        starts = [0]
        for _, n in requests:
            starts.append(starts[-1] + n)
        positions = [h + i for h, n in requests for i in range(n)]
        case.rows = len(positions)
        case.positions[:case.rows] = torch.tensor(positions, device=DEV, dtype=torch.int32)
        case.row_request.fill_(-1)
        case.row_request[:case.rows] = torch.tensor([r for r, (_, n) in enumerate(requests) for _ in range(n)], device=DEV)
        case.row_start.copy_(torch.tensor(starts))
        case.first_pos.copy_(torch.tensor([h for h, _ in requests]))
        q.copy_(torch.randn_like(q))
        for out in outs:
            out.fill_(7)
        for graph in graphs:                                       # (two that share nothing, one behind the other)
            graph.replay()
        spread = []
        want, most = case.attention(q, 0.1, spread=spread)
        for out in outs:
            cc.assert_attention_laid_out(out[:case.rows], want, most, spread[0]) if out is not outs[2] else \
                cc.assert_attention(out[:case.rows], want, most, BF16)
            assert (out[case.rows:] == 7).all()


def test_portions_laid_out_in_a_window_wherever_they_begin(monkeypatch):
    """A captured step replayed at other places: as many blocks of 64 tokens as the rows may reach, not one more or less."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    case = cc.Case([(700, 50), (640, 33)], dim=64, group=64, n_rep=2, kv_heads=1, page=16, seed=43)
    q, window = case.queries(), 79
    out = torch.empty_like(q)

    def step():
        cache4.attention4(q, out, case.heads, 0.125, case.batch, case.pages, window=window)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for first in ((700, 640), (0, 1), (63, 64), (127, 128), (141, 142), (143, 78), (560, 593)):
        case.requests = [(first[0], 50), (first[1], 33)]
        case.first_pos.copy_(torch.tensor(first))
        case.positions.copy_(torch.cat([f + torch.arange(n) for f, n in case.requests]))
        out.fill_(7)
        graph.replay()
        spread = []
        want, most = case.attention(q, 0.125, window=window, spread=spread)
        cc.assert_attention_laid_out(out, want, most, spread[0])


@pytest.mark.parametrize("blocks,tiled", [(11, 3), (9, 3), (6, 3), (4, 2), (3, 2), (2, 1), (1, 0)])
def test_portions_that_are_laid_out_a_few_requests_at_a_time(blocks, tiled, monkeypatch):
    """No more at a time than scratch memory is for; a request that alone has more is walked."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    monkeypatch.setattr(cache4, "_MOST_BLOCKS", blocks * 2 * 64)
    calls, tiles = [], cache4._tiles
    monkeypatch.setattr(cache4, "_tiles", lambda *a: calls.append(a[-3:]) or tiles(*a))
    case = cc.Case([(7, 1), (100, 70), (0, 90), (300, 40)], dim=64, group=32, n_rep=4, kv_heads=2, seed=45)   # blocks of 3, 2, 6
    q, spread = case.queries(), []
    want, most = case.attention(q, 0.125, spread=spread)
    got = _attend(case, q, 0.125)
    assert sum(last - first for first, last, _ in calls) == tiled and all(sum(counts) <= blocks for _, _, counts in calls)
    cc.assert_attention(got[:1], want[:1], most[:1], BF16)
    cc.assert_attention_laid_out(got, want, most, spread[0])


def test_portions_laid_out_on_two_streams_at_once(monkeypatch):
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    cases = [cc.Case([(100 * i, 200)], dim=64, group=32, n_rep=2, kv_heads=4, seed=35 + i) for i in range(2)]
    qs = [c.queries() for c in cases]
    outs = [[torch.empty_like(q) for _ in range(10)] for q in qs]
    streams = [torch.cuda.Stream(DEV) for _ in cases]
    torch.cuda.synchronize()
    for n in range(10):
        for c, q, out, stream in zip(cases, qs, outs, streams):
            with torch.cuda.stream(stream):
                cache4.attention4(q, out[n], c.heads, 0.125, c.batch, c.pages)
    torch.cuda.synchronize()
    for c, q, out in zip(cases, qs, outs):
        spread = []
        want, most = c.attention(q, 0.125, spread=spread)
        cc.assert_attention_laid_out(out[0], want, most, spread[0])
        assert all(torch.equal(o, out[0]) for o in out[1:])


def test_picks_of_a_padded_step():
    """Rows behind the last request's, whether there are picks of these or not: left as they are."""
    from crucible_b200.ops import cache4
    case = cc.Case([(200, 1), (90, 1), (140, 1)], dim=64, group=64, page=16, bounds=True, seed=37)
    _true_bounds(case)
    rows = case.rows
    q = case.queries()
    by_definition = _picks_by_definition(case, q, 5, 1, 2)
    case.positions = torch.cat((case.positions, torch.zeros(3, dtype=torch.int32, device=DEV)))
    case.row_request = torch.cat((case.row_request, torch.full((3,), -1, dtype=torch.int32, device=DEV)))
    case.batch = case.make_batch()
    q = torch.cat((q, torch.full_like(q, float("nan"))))
    for n in (rows, rows + 3):
        picks = torch.full((n, case.kv_heads, 5), 99, dtype=torch.int32, device=DEV)
        cache4.pick_pages4(q, case.heads, case.batch, case.pages, picks)
        assert torch.equal(picks[:rows], by_definition) and (picks[rows:] == 99).all()
        want, most = case.attention(q, 0.125, picks=picks.cpu())
        out = torch.full_like(q, 7)
        cache4.attention4(q, out, case.heads, 0.125, case.batch, case.pages, picks=picks)
        cc.assert_attention(out[:rows], want[:rows], most[:rows], BF16)
        assert (out[rows:] == 7).all()


@pytest.mark.parametrize("small", [0.0, 1e-12, 1e-7, 1e-3])
def test_spans_in_portions_that_are_laid_out(small, monkeypatch):
    """What a request's keys and values are scaled by goes by all of them that are visible, not by one, and not by what the
    window has passed or what lies behind the last."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    for window in (None, 150):
        case = cc.Case([(90, 70), (200, 40), (0, 40)], dim=64, group=32, n_rep=4, kv_heads=2, seed=29)
        place = case.table[0].long()
        case.pages.scales[:, place[0], :, 0] *= small             # the first visible, in one request
        case.pages.scales[:, place[3]] *= small
        if window is not None:
            for j in range(5):                                    # (positions up to 50 are passed in the second)
                case.pages.scales[:, int(case.table[1, 0]), :, j] *= 1e20
        q, spread = case.queries(), []
        want, most = case.attention(q, 0.125, window=window, spread=spread)
        cc.assert_attention_laid_out(_attend(case, q, 0.125, window=window), want, most, spread[0])


def test_numbers_that_are_none_in_portions_that_are_laid_out(monkeypatch):
    """A value or key that is no number reaches the rows that see it, whole, and no others; nor does what nobody wrote."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    case = cc.Case([(20, 60), (0, 90)], dim=64, group=32, n_rep=4, kv_heads=2, seed=21)
    q, spread = case.queries(), []
    want, most = case.attention(q, 0.125, spread=spread)
    scales = case.pages.scales
    scales[:, case.free] = float("nan")
    for r, last in ((0, 80), (1, 90)):
        for j in range(last, case.stride * 16):
            place = int(case.table[r, j // 16])
            if place != case.free:
                scales[:, place, :, j % 16] = float("nan")
    scales[1, int(case.table[0, 50 // 16]), 1, 50 % 16, 1] = float("nan")       # a value of kv head 1 at position 50: row 30
    scales[0, int(case.table[1, 70 // 16]), 0, 70 % 16, 0] = float("nan")       # a key of kv head 0 at position 70: row 60 + 70
    got = _attend(case, q, 0.125)
    bad = torch.zeros(150, 8, dtype=torch.bool, device=DEV)
    bad[30:60, 4:] = True
    bad[130:, :4] = True
    bad = bad.repeat_interleave(64, dim=1)
    assert got[bad].isnan().all()
    fine = torch.where(bad, want, got.double())
    cc.assert_attention_laid_out(fine, want, most, spread[0])


def test_rows_at_odd_addresses_go_by_the_walking_kernel():
    case = cc.Case([(300, 200)], dim=64, group=64, n_rep=4, kv_heads=1, seed=22)
    wide = torch.zeros(200, 4 * 64 + 3, dtype=BF16, device=DEV)
    q = wide[:, 3:]
    q.copy_(case.queries())
    want, most = case.attention(q, 0.125)
    cc.assert_attention(_attend(case, q, 0.125), want, most, BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [1, 16, 37, 500])
def test_attention_in_a_window(window, dtype):
    case = cc.Case([(300, 1), (0, 1), (40, 7), (15, 2)], dim=64, page=16, dtype=dtype, seed=window)
    q = case.queries()
    # pages that the window has passed were given back
    for r, (held, _) in enumerate(case.requests):
        passed = max(0, held - window + 1) // 16
        case.table[r, :passed] = torch.tensor([-1, case.free][r % 2], device=DEV)
    want, most = case.attention(q, 0.125, window=window)
    cc.assert_attention(_attend(case, q, 0.125, window=window), want, most, dtype)
    if window == 1:                    # a row that sees itself alone is its own value
        own = case.table[0, 300 // 16].long()
        value = case.contents()[1, own, :, 300 % 16].repeat_interleave(3, dim=0).flatten()
        assert ((want[0] - value).abs() <= 1e-12 * value.abs()).all()


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_nobody_wrote_is_not_seen(dtype, page):
    """Places behind the last token hold what is no number, or vast ones; so do pages that no table names."""
    requests = [(5, 1), (33, 1), (50, 3), (0, 1), (127, 1)]
    case = cc.Case(requests, dim=128, group=64, page=page, dtype=dtype, seed=4)
    q = case.queries()
    want, most = case.attention(q, 0.09)
    scales = case.pages.scales
    scales[:, case.free] = float("nan")
    for r, (held, new) in enumerate(requests):
        for j in range(held + new, case.stride * page):
            place = int(case.table[r, j // page])
            if place != case.free:
                scales[:, place, :, j % page] = (float("nan"), float("inf"), 1e38, -1e38)[j % 4]
    cc.assert_attention(_attend(case, q, 0.09), want, most, dtype)


def test_a_number_that_is_none_stays_with_the_rows_that_see_it():
    """NaN and vast values at a later position of a portion: earlier rows of the same tile do not notice."""
    for dtype in (BF16, F32):
        case = cc.Case([(20, 6)], dim=64, group=64, dtype=dtype, seed=8)
        q = case.queries()
        want, most = case.attention(q, 0.125)
        place = int(case.table[0, 24 // 16])
        case.pages.scales[1, place, :, 24 % 16] = float("nan")           # the value of position 24: row 4
        case.pages.scales[0, place, 0, 23 % 16] = 3e37                    # a vast key at 23, a vast value too
        case.pages.scales[1, place, :, 23 % 16] = 3e37
        got = _attend(case, q, 0.125)
        cc.assert_attention(got[:3], want[:3], most[:3], dtype)
        assert got[4:].isnan().all()


def test_rows_of_no_keys_and_rows_behind_the_last():
    case = cc.Case([(10, 1), (40, 2), (3, 1)], dim=64, seed=5)
    q = torch.cat((case.queries(), torch.full((3, case.heads * 64), float("nan"), device=DEV, dtype=BF16)))
    case.table[0, :] = -1
    case.table[1, 1] = case.n_pages + 7                  # keys 16..31 of the second request
    case.table[2, 0] = -(1 << 31)
    want, most = case.attention(q, 0.2)
    got = _attend(case, q, 0.2)
    assert (got[0] == 0).all() and (got[3] == 0).all() and (got[4:] == 7).all()
    cc.assert_attention(got[1:3], want[1:3], most[1:3], BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sizes_of_scores_values_and_queries(dtype):
    """Scores far apart, one key that outweighs all, values and queries that are huge, tiny or zero."""
    for size, stretch, scale in ((1e-6, 1.0, 0.1), (1e6, 1.0, 1e-7), (1.0, 40.0, 0.1), (1e-20, 1.0, 0.1), (1.0, 1e-20, 1.0),
                                 (1.0, 1e20, 1e-20), (3e30, 1.0, 1e-31)):
        case = cc.Case([(200, 1), (90, 2)], dim=64, group=32, dtype=dtype, seed=6, size=size)
        q = case.queries(stretch)
        q[0, :64] = 0
        want, most = case.attention(q, scale)
        if stretch == 40.0:            # scores of up to a few hundred: their rounding counts (2^-24 of a sum of terms 16 times as large)
            most = most * 32
        cc.assert_attention(_attend(case, q, scale), want, most, dtype)


@pytest.mark.parametrize("dtype,dim,held,n_rep,kv_heads", [(BF16, 128, 20000, 4, 1), (F32, 64, 9000, 7, 1), (BF16, 64, 5000, 16, 2),
                                                           (F32, 256, 3000, 3, 1)])
def test_long_contexts_are_dealt_to_many_blocks(dtype, dim, held, n_rep, kv_heads):
    for requests in ([(held, 1)], [(held, 1), (5, 1), (held // 3, 2)]):
        case = cc.Case(requests, dim=dim, group=64, n_rep=n_rep, kv_heads=kv_heads, page=32, dtype=dtype, seed=held)
        q = case.queries(1.2)
        want, most = case.attention(q, dim ** -0.5)
        cc.assert_attention(_attend(case, q, dim ** -0.5), want, most, dtype)


def test_sums_of_a_very_long_context_in_32_bits():
    """Equal weights over 30,000 keys: the mean of the values, to float32's rounding of its sums."""
    case = cc.Case([(30000, 1)], dim=64, group=64, n_rep=1, kv_heads=1, page=64, dtype=F32, seed=2)
    q = torch.zeros(1, 64, device=DEV)
    want, most = case.attention(q, 1.0)
    got = _attend(case, q, 1.0)
    assert ((got.double() - want).abs() <= 2.0 ** -20 * most).all()


def test_strides_streams_and_both_ends_of_a_tensor():
    case = cc.Case([(50, 1), (70, 3)], dim=64, seed=7)
    wide = torch.zeros(case.rows, case.heads * 64 + 11, dtype=BF16, device=DEV)
    q = wide[:, 5:5 + case.heads * 64]
    q.copy_(case.queries())
    want, most = case.attention(q, 0.125)
    from crucible_b200.ops import cache4
    out = torch.zeros(case.rows, case.heads * 64 + 3, dtype=BF16, device=DEV)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        cache4.attention4(q, out[:, 1:-2], case.heads, 0.125, case.batch, case.pages)
    torch.cuda.current_stream().wait_stream(other)
    cc.assert_attention(out[:, 1:-2], want, most, BF16)
    assert not out[:, 0].any() and not out[:, -2:].any()


def _picks_by_definition(case, q, count, first, last):
    rep = case.heads // case.kv_heads
    out = torch.full((case.rows, case.kv_heads, count), -1, dtype=torch.int32)
    for i, (r, p) in enumerate(zip(case.row_request.tolist(), case.positions.tolist())):
        own = p // case.page
        ids = case.table[r, :own + 1].long()
        for h in range(case.kv_heads):
            hi, lo = (case.pages.bounds[ids, h, s].double() for s in (0, 1))
            a = case.pages.bound_scales[ids, h].double()
            best = torch.full((own + 1,), -float("inf"), dtype=torch.float64, device=q.device)
            for j in range(rep):
                row = q[i, (h * rep + j) * case.dim:(h * rep + j + 1) * case.dim].double()
                unit = cc.once(row.abs().max() * cc.OF_127)
                q8 = torch.round(cc.once(row * cc.once(1.0 / unit))) if unit > 0 else torch.zeros_like(row)
                dot = torch.maximum(q8 * hi, q8 * lo).sum(dim=1)
                best = torch.maximum(best, cc.once(dot * cc.once(unit * a)))
            best[:first] = float("inf")
            best[max(0, own - last + 1):] = float("inf")
            rank = torch.argsort(best, descending=True, stable=True)[:count].sort().values
            out[i, h, :rank.numel()] = rank.int().cpu()
    return out.to(q.device)


def _true_bounds(case):
    for i in range(case.n_pages):
        want, scale = _bounds_by_definition(case, i, case.page)
        case.pages.bounds[i], case.pages.bound_scales[i] = want.to(torch.int8), scale.float()


@pytest.mark.parametrize("dim,page,count,first,last,n_rep,dtype", [
    (64, 16, 5, 1, 2, 3, BF16), (128, 32, 8, 0, 1, 4, F32), (192, 16, 3, 1, 2, 1, BF16), (256, 16, 40, 2, 3, 7, F32),
    (64, 16, 600, 1, 2, 2, BF16), (128, 16, 257, 1, 1, 16, BF16)])
def test_picked_pages_and_attention_to_them(dim, page, count, first, last, n_rep, dtype):
    from crucible_b200.ops import cache4
    requests = [(4000, 1), (0, 1), (page * count - 1, 1), (page * count, 1), (777, 2)]
    case = cc.Case(requests, dim=dim, group=64, n_rep=n_rep, kv_heads=2, page=page, dtype=dtype, seed=count, bounds=True)
    _true_bounds(case)
    q = case.queries()
    picks = torch.full((case.rows, 2, count), 99, dtype=torch.int32, device=DEV)
    cache4.pick_pages4(q, case.heads, case.batch, case.pages, picks, first=first, last=last)
    assert torch.equal(picks, _picks_by_definition(case, q, count, first, last))
    want, most = case.attention(q, dim ** -0.5, picks=picks.cpu())
    cc.assert_attention(_attend(case, q, dim ** -0.5, picks=picks), want, most, dtype)


def test_picks_among_equal_pages_and_of_queries_of_nothing():
    """Equal scores: the first pages; a query of zeros scores every page alike."""
    from crucible_b200.ops import cache4
    case = cc.Case([(16 * 700 - 1, 1)], dim=64, n_rep=2, kv_heads=1, seed=1, bounds=True)
    case.pages.bounds[:] = 9
    case.pages.bound_scales.fill_(0.5)
    picks = torch.empty(1, 1, 20, dtype=torch.int32, device=DEV)
    for q in (torch.zeros(1, 128, dtype=BF16, device=DEV), torch.ones(1, 128, dtype=BF16, device=DEV)):
        cache4.pick_pages4(q, 2, case.batch, case.pages, picks)
        assert picks.flatten().tolist() == list(range(18)) + [698, 699]
    case.pages.bound_scales[case.table[0, 300].long()] = 0.75
    cache4.pick_pages4(q, 2, case.batch, case.pages, picks)
    assert picks.flatten().tolist() == list(range(17)) + [300, 698, 699]


def test_picks_that_name_nothing():
    """-1 and pages beyond the table are not there; a row whose picks are all so is zero."""
    case = cc.Case([(200, 1), (90, 1)], dim=64, n_rep=2, kv_heads=2, seed=11)
    q = case.queries()
    picks = torch.tensor([[[0, 3, 12, -1], [-1, -1, -1, -1]], [[5, 1, 1 << 28, -5], [2, 0, 4, 3]]], dtype=torch.int32, device=DEV)
    want, most = case.attention(q, 0.125, picks=picks.cpu())
    got = _attend(case, q, 0.125, picks=picks)
    cc.assert_attention(got, want, most, BF16)
    assert (got[0, 128:] == 0).all()


def test_one_captured_step_replayed_behind_longer_contexts():
    """Append, pick and attend in one graph; positions move on between its replays, past what the host said."""
    from crucible_b200.ops import cache4
    dim, page, steps = 64, 16, 40
    case = cc.Case([(100 + steps, 1), (7 + steps, 1), (300 + steps, 1)], dim=dim, page=page, seed=12, bounds=True)
    _true_bounds(case)
    case.requests = [(100, 1), (7, 1), (300, 1)]
    case.first_pos.copy_(torch.tensor([100, 7, 300]))
    case.positions.copy_(case.first_pos)
    case.batch = case.make_batch()
    cos, sin = cc.tables(400, dim // 2, DEV)
    qkv = torch.empty(3, (case.heads + 2 * case.kv_heads) * dim, dtype=BF16, device=DEV)
    q = torch.empty(3, case.heads * dim, dtype=BF16, device=DEV)
    dense, sparse = torch.empty_like(q), torch.empty_like(q)
    picks = torch.empty(3, case.kv_heads, 6, dtype=torch.int32, device=DEV)

    def step():
        cache4.rope_append4(qkv, q, case.heads, cos, sin, case.batch, case.pages)
        cache4.attention4(q, dense, case.heads, 0.125, case.batch, case.pages)
        cache4.pick_pages4(q, case.heads, case.batch, case.pages, picks)
        cache4.attention4(q, sparse, case.heads, 0.125, case.batch, case.pages, picks=picks)
    qkv.copy_(case.normal(*qkv.shape))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(steps):
        case.positions.copy_(torch.tensor([100 + i, 7 + i, 300 + i]))
        case.first_pos.copy_(case.positions)
        qkv.copy_(case.normal(*qkv.shape))
        graph.replay()
        if i % 13 == 0 or i == steps - 1:
            case.requests = [(100 + i, 1), (7 + i, 1), (300 + i, 1)]
            for got, chosen in ((dense, None), (sparse, picks.cpu())):
                want, most = case.attention(q, 0.125, picks=chosen)
                cc.assert_attention(got, want, most, BF16)


def test_a_pool_whose_offsets_pass_32_bits(monkeypatch):
    """The same pages at the end of a pool of more than 2^32 bytes a side give the same, to the bit."""
    from crucible_b200.ops import cache4
    dim, kv, page = 128, 8, 64
    requests = [(200, 1), (70, 1), (100, 90)]
    far = (1 << 32) // (kv * page * dim // 2) + 50
    cos, sin = cc.tables(300, dim // 2, DEV)
    got = []
    for offset in (0, far):
        case = cc.Case(requests, dim=dim, group=64, n_rep=2, kv_heads=kv, page=page, bounds=True, seed=41)
        if offset:
            small = case.pages
            n = offset + small.n_pages
            case.pages = cache4.Pages4(*(torch.empty(2, n, *t.shape[2:], dtype=t.dtype, device=DEV) for t in (small.codes, small.scales)),
                                       *(torch.empty(n, *t.shape[1:], dtype=t.dtype, device=DEV) for t in (small.bounds, small.bound_scales)))
            case.pages.codes[:, offset:], case.pages.scales[:, offset:] = small.codes, small.scales
            case.pages.bounds[offset:], case.pages.bound_scales[offset:] = small.bounds, small.bound_scales
            case.table += offset
            case.batch = case.make_batch()
        qkv = case.normal(case.rows, (case.heads + 2 * kv) * dim).to(BF16)
        q = torch.empty(case.rows, case.heads * dim, dtype=BF16, device=DEV)
        cache4.rope_append4(qkv, q, case.heads, cos, sin, case.batch, case.pages)
        picks = torch.empty(case.rows, kv, 3, dtype=torch.int32, device=DEV)
        cache4.pick_pages4(q, case.heads, case.batch, case.pages, picks)
        outs = [torch.empty_like(q) for _ in range(3)]
        cache4.attention4(q, outs[0], case.heads, 0.09, case.batch, case.pages, picks=picks)
        for laid_out, out in zip((False, True), outs[1:]):
            monkeypatch.setattr(cache4, "LAID_OUT", laid_out)
            cache4.attention4(q, out, case.heads, 0.09, case.batch, case.pages)
        p = case.pages
        got.append((q, picks, *outs, p.codes[:, offset:].clone(), p.scales[:, offset:].clone(), p.bounds[offset:].clone(),
                    p.bound_scales[offset:].clone()))
        del p
        case.pages = None
    for small, large in zip(*got):
        assert torch.equal(small, large)

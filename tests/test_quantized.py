"""The quantised operators' host side: packed weights and what is refused (no kernel runs)."""
import pytest
import torch

from crucible_b200.ops import KernelError, quantized
from quantized_cases import E4M3, dense4, dense8, random_rows8, random_weights4, random_weights8


def _gen():
    return torch.Generator().manual_seed(7)


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (5, 96, 32), (7, 192, 96), (16, 256, 64), (3, 1024, 128), (4, 160, 160)])
def test_pack4_keeps_weights_within_half_a_step(n, k, group):
    w = torch.randn(n, k, generator=_gen()) * 0.02
    w[0, :group] = 0.0                                 # a group of zeros
    p = quantized.Weights4.pack(w, group)
    assert p.shape == (n, k) and p.group == group
    assert torch.equal(p.dense().double(), dense4(p).float().double()) or \
        torch.allclose(p.dense().double(), dense4(p), rtol=2.0 ** -22, atol=0)
    step = p.group_scales.double().repeat_interleave(group, 1) * p.scales.double()[:, None]
    # 7 steps reach the largest; its scale may round down by half a step of e4m3, 2^-4: 7.47 steps, code 15
    assert ((w.double() - dense4(p)).abs() <= step * (0.5 + 1e-5)).all()
    assert (dense4(p)[0, :group] == 0).all()


@pytest.mark.parametrize("n,k", [(1, 1), (5, 17), (16, 256)])
def test_pack8_rounds_to_nearest(n, k):
    w = torch.randn(n, k, generator=_gen()) * 0.02
    w[n // 2] = 0.0
    p = quantized.Weights8.pack(w)
    assert p.values.stride(0) % 16 == 0 or n == 1
    assert ((w.double() - dense8(p)).abs() <= w.double().abs() * (2.0 ** -4 + 1e-6) + p.scales.double()[:, None] * 2.0 ** -10).all()
    assert torch.allclose(p.dense().double(), dense8(p), rtol=2.0 ** -23, atol=0)


def test_codes_lie_where_they_are_said_to():
    w = torch.arange(-8, 0).float().repeat(4)[None]     # codes 0..7, four times
    p = quantized.Weights4(torch.tensor([[0, 0, 0, 0]], dtype=torch.int32), torch.ones(1, 1).to(E4M3), torch.ones(1))
    assert (p.dense() == -8).all()
    word = sum(i << s for i, s in enumerate(quantized.CODE_SHIFTS))
    p = quantized.Weights4(torch.tensor([[word] * 4], dtype=torch.int32), torch.ones(1, 1).to(E4M3), torch.ones(1))
    assert torch.equal(p.dense(), w)


def test_rows_of_new_rows8_begin_on_16_bytes():
    for width in (1, 15, 16, 17, 100):
        q = quantized.new_rows8(3, width, "cpu")
        assert q.shape == (3, width) and q.dtype == E4M3 and q.stride(0) % 16 == 0


def _refused(match, fn, *args, **kw):
    with pytest.raises(KernelError, match=match):
        fn(*args, **kw)


def test_weights_that_are_refused():
    ok = torch.zeros(4, 8, dtype=torch.int32)
    one = torch.ones(4)
    for groups in (3, 5, 64):
        _refused("group", quantized.Weights4, ok, torch.ones(4, groups).to(E4M3), one)
    _refused("group scales", quantized.Weights4, ok, torch.ones(4, 2), one)
    _refused("codes", quantized.Weights4, ok.long(), torch.ones(4, 2).to(E4M3), one)
    _refused("float32 vector", quantized.Weights4, ok, torch.ones(4, 2).to(E4M3), one.double())
    _refused("float32 vector", quantized.Weights4, ok, torch.ones(4, 2).to(E4M3), torch.ones(5))
    _refused("empty", quantized.Weights4, ok[:0], torch.ones(0, 2).to(E4M3), one[:0])
    _refused("empty", quantized.Weights8, torch.zeros(4, 0).to(E4M3), one)
    _refused("8-bit weights", quantized.Weights8, torch.zeros(4, 8, dtype=torch.uint8), one)
    _refused("finite", quantized.Weights8.pack, torch.tensor([[1.0, float("nan")]]))
    _refused("finite", quantized.Weights4.pack, torch.full((2, 32), float("inf")), 32)
    for group in (0, 16, 48, 33, 64):
        _refused("group", quantized.Weights4.pack, torch.ones(2, 96), group)


def test_calls_that_are_refused():
    g = _gen()
    x, q, s = torch.zeros(3, 20), quantized.new_rows8(3, 20, "cpu"), torch.zeros(3)
    gain = torch.ones(20)
    norm = quantized.add_rmsnorm8
    _refused("CUDA device", norm, x, None, gain, 1e-5, q, s)               # all is well but the device
    _refused("input", norm, x.bfloat16(), None, gain, 1e-5, q, s)
    _refused("delta", norm, x, torch.zeros(3, 19), gain, 1e-5, q, s)
    _refused("delta", norm, x, torch.zeros(3, 20).half(), gain, 1e-5, q, s)
    _refused("overlap", norm, x, torch.zeros(1, 20).expand(3, 20), gain, 1e-5, q, s)
    _refused("gain", norm, x, None, torch.ones(21), 1e-5, q, s)
    _refused("output", norm, x, None, gain, 1e-5, q[:2], s)
    _refused("output", norm, x, None, gain, 1e-5, torch.zeros(3, 20), s)
    _refused("scales", norm, x, None, gain, 1e-5, q, s[:2])
    _refused("sum", norm, x, None, gain, 1e-5, q, s, sum_out=x.bfloat16())
    _refused("contiguous", norm, torch.zeros(20, 3).t(), None, gain, 1e-5, q, s)
    both = torch.zeros(3, 40)
    _refused("CUDA device", quantized.glu8, both, q, s)
    _refused("even", quantized.glu8, torch.zeros(3, 41), q, s)
    _refused("limit", quantized.glu8, both, q, s, 0.0)
    _refused("limit", quantized.glu8, both, q, s, float("nan"))
    _refused("output", quantized.glu8, torch.zeros(3, 42), q, s)

    w8, w4 = random_weights8(6, 64, "cpu", g), random_weights4(6, 64, 32, "cpu", g)
    rows, scales = random_rows8(3, 64, "cpu", g)
    out = torch.zeros(3, 6)
    _refused("CUDA device", quantized.linear8, rows, scales, w8, out)
    _refused("Weights8", quantized.linear8, rows, scales, w4, out)
    _refused("rows", quantized.linear8, rows[:, :63], scales, w8, out)
    _refused("rows", quantized.linear8, torch.zeros(3, 64), scales, w8, out)
    _refused("row scales", quantized.linear8, rows, scales[:2], w8, out)
    _refused("output", quantized.linear8, rows, scales, w8, torch.zeros(3, 7))
    _refused("output", quantized.linear8, rows, scales, w8, out.half())
    _refused("overlap", quantized.linear8, rows, scales, w8, torch.zeros(6).expand(3, 6))
    _refused("add", quantized.linear8, rows, scales, w8, out, add=out.bfloat16())
    a = torch.zeros(3, 64)
    _refused("CUDA device", quantized.linear4, a, w4, out)
    _refused("Weights4", quantized.linear4, a, w8, out)
    _refused("rows", quantized.linear4, a.half(), w4, out)
    _refused("rows", quantized.linear4, torch.zeros(3, 32), w4, out)
    _refused("add", quantized.linear4, a, w4, out, add=torch.zeros(2, 6))


def test_the_rule_names_a_form_that_takes_the_product():
    for kind in (quantized._EIGHT, quantized._FOUR_BF16, quantized._FOUR_F32):
        for forced in (None, "few", "ring", "tiles", "pairs"):
            for m in (1, 5, 6, 8, 9, 16, 17, 33, 64, 65, 100, 129, 256, 257, 1000, 2049, 30000, 1 << 20):
                for n, k in ((1, 32), (127, 256), (129, 96), (768, 2048), (4096, 14336), (28672, 4096), (300000, 64),
                             (512, 8192), (60000, 1024)):
                    form, *how = quantized._rule(forced, kind, m, n, k)
                    if form == "few":
                        assert forced in (None, "few", "ring")
                    elif form == "ring":
                        assert k % 256 == 0 and tuple(how[:2]) in ((1, 8), (1, 4), (2, 4), (2, 2)) and how[2] in (1, 2, 4, 8)
                        assert kind == quantized._FOUR_BF16 or (kind == quantized._FOUR_F32 and m <= 5)
                    else:
                        rows, more = how
                        assert rows % 16 == 0 and 16 <= rows <= (64 if kind == quantized._FOUR_F32 else 256)
                        if form == "tiles":
                            assert more in (1, 2, 4, 6, 8) and more <= -(-k // (128 if kind == quantized._EIGHT else 256))
                            assert -(-m // rows) <= 65535
                        else:
                            assert form == "pairs" and kind != quantized._FOUR_F32 and more == 74


def test_a_config_names_4_bit_feed_forwards():
    from crucible_b200.config import ConfigError, parse_config, shape
    raw = shape("120m")
    assert parse_config(raw).layers[0].feed_forward.kind == "swiglu"
    for group in (32, 128, 256):
        cfg = parse_config({**raw, "feed_forward_weight_group": group})
        assert cfg.layers[0].feed_forward.kind == "swiglu_4bit" and cfg.layers[0].feed_forward.option("group") == group
    for group in (16, 48, 100, 512, 0, -32, "64"):
        with pytest.raises(ConfigError):
            parse_config({**raw, "feed_forward_weight_group": group})


def test_a_described_config_keeps_the_group():
    from crucible_b200.config import get_architecture, parse_config, shape
    for name in ("120m", "llama-1b"):
        for extra in ({}, {"feed_forward_weight_group": 64}):
            cfg = parse_config({**shape(name), **extra})
            again = get_architecture(cfg.architecture).describe(cfg)
            assert again.get("feed_forward_weight_group") == extra.get("feed_forward_weight_group")
            assert parse_config(again).layers == cfg.layers


def test_more_rows_than_32_bits_count_are_refused():
    many = 1 << 31
    x, out, scales = (torch.empty(many, 1, device="meta"), torch.empty(many, 1, dtype=E4M3, device="meta"),
                      torch.empty(many, device="meta"))
    _refused("up to 2147482624 rows", quantized.add_rmsnorm8, x, None, torch.ones(1), 1e-5, out, scales)
    _refused("up to 2147482624 rows", quantized.glu8, torch.empty(many, 2, device="meta"), out, scales)
    w8, w4 = random_weights8(1, 1, "cpu", _gen()), random_weights4(1, 32, 32, "cpu", _gen())
    _refused("up to 2147482624 rows", quantized.linear8, out, scales, w8, x)
    _refused("up to 2147482624 rows", quantized.linear4, torch.empty(many, 32, device="meta"), w4, x)


def test_a_limit_that_float32_may_have_as_zero_is_refused():
    both, q, s = torch.zeros(3, 40), quantized.new_rows8(3, 20, "cpu"), torch.zeros(3)
    for limit in (1e-50, 2.0 ** -127, -1.0):
        _refused("limit", quantized.glu8, both, q, s, limit)
    _refused("CUDA device", quantized.glu8, both, q, s, 2.0 ** -126)


def test_a_wait_of_glu8_that_runs_out_is_told(monkeypatch):
    """Wherever the kernel would wait for copies it is handed a place to say that a wait ran out; where there is none
    (nothing was called yet and a graph is being captured) it does not wait."""
    from crucible_b200.ops import build
    lib = build.load("rows8")
    assert lib.cb_glu8_waits_from() == quantized._WAITS_FROM
    told = {}

    class Recorder:
        cb_rows8_widest = lib.cb_rows8_widest

        @staticmethod
        def cb_glu8(both, dtype, ldb, q, ldq, scales, rows, width, limit, alpha, offset, status):
            told[dtype, rows, width] = status
            return 0
    monkeypatch.setattr(build, "load", lambda name: Recorder)
    monkeypatch.setattr(quantized, "_at", lambda dev, call, *args: call(*args))
    monkeypatch.setattr(quantized, "_look_over_glu8", lambda *args: None)       # (tensors without memory, on no GPU)
    monkeypatch.setattr(quantized, "_status", lambda dev: 1 << 20)
    waiting = 0
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        for rows in (1, 8, 295, 296, 297, 512, 1023, 1024, 1025, 4096):
            for width in (8, 4096, 7168, 7176, 8192, 14336, 14344, 14400, 14408, 20000, 28800, 28808, 32768):
                both, out = torch.empty(rows, 2 * width, dtype=dtype, device="meta"), torch.empty(rows, width, dtype=E4M3, device="meta")
                quantized.glu8(both, out, torch.empty(rows, device="meta"))
                status = told.pop((code, rows, width))
                assert not lib.cb_glu8_waits(code, rows, width, 0)
                waits = lib.cb_glu8_waits(code, rows, width, 1 << 20)
                waiting += waits
                assert status or not waits, f"{dtype} {rows} x {width}"
    assert waiting > 20


def test_shares_of_a_long_k_in_8_bits():
    """float32 results of e4m3 products: no sum of more than 12,288 of K but in the pairs, which take 2,048 at a time, and from
    registers, whose sums keep more."""
    for m in (9, 33, 100, 1000):
        for n in (200, 2048, 28672):
            for k in (8192, 12288, 12289, 14336, 16384, 65536, 262144, 1 << 20):
                form, *how = quantized._rule(None, quantized._EIGHT, m, n, k, True)
                assert form in ("few", "pairs") or -(-(-(-k // 128)) // how[1]) * 128 <= 12288, (m, n, k, form, how)
                assert quantized._rule(None, quantized._EIGHT, m, n, k)[0] != "ring"


def test_4_bit_feed_forwards_take_normalised_rows():
    """The block neither asks the attention's last product to leave rows ahead of the norm, which nobody would read, nor hands
    over rows that are not normalised yet."""
    from crucible_b200.config.model_config import FeedForwardSpec
    from crucible_b200.parts.base import FEED_FORWARDS
    from crucible_b200.parts.block import PreNormBlock
    calls = []

    class Norm:
        supports_ahead = supports_lazy = True

        def forward(self, ctx, x, lazy=False):
            calls.append(("norm", lazy))
            return "rows"

    class Ctx:
        def announce_norm(self, norm, rows):
            calls.append(("announced", norm))
    norm, rows = Norm(), torch.zeros(2, 64)
    for kind, takes in (("swiglu", True), ("swiglu_4bit", False)):
        part = FEED_FORWARDS.build(kind, FeedForwardSpec(kind=kind, width=64, intermediate=128, extra=(("group", 32),) * (kind != "swiglu")))
        calls.clear()
        PreNormBlock._announce(Ctx(), (norm, part), rows)
        assert PreNormBlock._norm(Ctx(), norm, part, rows) == "rows"
        assert calls == [("announced", norm if takes else None), ("norm", takes)]


def test_scratch_of_float32_rows_is_bounded():
    """Slabs of float32 rows: whole tiles, equal but for the last, at most 512 MB of parts, and no more of them than that takes."""
    for k in (32, 256, 4096, 14336, 16384, 100000 // 32 * 32, 1 << 20):
        for m in (65, 2048, 4096, 65536, 65537, 1 << 20, 4_200_000):
            rows = quantized._slab(m, k)
            assert rows % 64 == 0 and 64 <= rows <= quantized._SLAB and 6 * k * rows <= 512 << 20
            least = max(-(-m // quantized._SLAB), -(-6 * k * m // (512 << 20)))
            assert -(-m // rows) <= least + 1 + least // 4 or rows <= 640        # (a slab of few tiles wastes more of the room)


def test_a_transposed_matrix_is_packed():
    w = torch.randn(64, 96, generator=_gen())
    for view in (w.t(), w.t()[:, ::2], w[::2].t(), w.t().double(), w.t().bfloat16(), w.flip(0)):
        rows = view.contiguous()
        for cls, group in ((quantized.Weights8, ()), (quantized.Weights4, (32,))):
            here, there = cls.pack(view, *group), cls.pack(rows, *group)
            assert here.shape == view.shape and torch.equal(here.dense(), there.dense())


def test_few_rows_by_few_features_of_a_long_k():
    """17 to 32 rows: the ring up to 5,120 of K, and beyond it only where no six tiles share K (measured both sides)."""
    for m in (17, 32):
        for n, k, form in ((1536, 5120, "ring"), (1536, 8192, "tiles"), (1920, 16384, "tiles"), (1984, 16384, "ring"),
                           (2048, 8192, "ring"), (1408, 5120, "ring"), (4096, 2048, "ring"), (4096, 4096, "tiles")):
            assert quantized._rule(None, quantized._FOUR_BF16, m, n, k)[0] == form, (m, n, k)


def test_a_product_that_could_not_tell_of_a_wait_is_refused(monkeypatch):
    """Inside a capture on a device that has no status word yet."""
    from crucible_b200.ops import tensor_core
    monkeypatch.setattr(tensor_core, "_status", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    launched = []
    monkeypatch.setattr(quantized, "_at", lambda dev, call, *args: launched.append(call) or 0)
    w = random_weights4(300, 256, 64, "cpu", _gen())
    for rows, dtype in ((1, torch.bfloat16), (100, torch.bfloat16), (100, torch.float32)):
        a, out = torch.zeros(rows, 256, dtype=dtype), torch.zeros(rows, 300)
        kind = quantized._FOUR_F32 if dtype == torch.float32 else quantized._FOUR_BF16
        monkeypatch.setattr(quantized, "FORM", None if rows == 1 else "tiles")
        form = quantized.form_of(kind, rows, 300, 256)[0]
        call = (kind, 0, a, rows, 256, None, w.codes, 128, w.group_scales.data_ptr(), w, 64, out, 300, None, "linear (4-bit weights)")
        assert form in ("ring", "tiles") and not launched
        _refused("inside a graph's capture", quantized._product, *call)

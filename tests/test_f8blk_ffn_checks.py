"""What the feed-forward helper over block-scaled e4m3 planes refuses, on the host alone: a stub pack fails on any launch, so nothing may
have been written when a call is refused."""
import pytest
import torch

from paddock_b200 import planes as P

EMBD, FF, TOKENS = 256, 512, 4


class Refusing:
    """A pack on which nothing may be launched."""
    def call(self, name, *a, **k):
        raise AssertionError(f"{name} launched")


def executor(pack):
    ex = P.GpuExecutor.__new__(P.GpuExecutor)
    ex.pack, ex.device = pack, torch.device("cpu")
    return ex


def plane(in_dim, out_dim):
    return P.F8BlkPlane(torch.zeros(in_dim * out_dim, dtype=torch.uint8), torch.zeros(P._blocks(in_dim) * P._blocks(out_dim)), (in_dim, out_dim))


def forward(pack, monkeypatch, embd=EMBD, ff=FF, batch=TOKENS, **change):
    """One call of the helper whose operands fit, but for what `change` replaces."""
    monkeypatch.setattr(P, "_stream", lambda: 0)
    ex = executor(pack)
    args = {"gate": plane(embd, ff), "up": plane(embd, ff), "down": plane(ff, embd), "ws": P.F8BlkFfnWorkspace(ex, embd, ff, TOKENS),
            "x": torch.zeros(batch * embd), "proj": torch.zeros(batch * embd), "norm": torch.ones(embd), "eps": 1e-6,
            "y": torch.zeros(batch, embd), "batch": batch, **change}
    P.ffn_f8blk_forward(ex, **args)


class Counting:
    def __init__(self):
        self.names = []

    def call(self, name, *a, **k):
        self.names.append(name)


def test_what_fits_is_three_launches(monkeypatch):
    for y in (torch.zeros(TOKENS, EMBD), torch.zeros(TOKENS, EMBD, dtype=torch.bfloat16)):
        pack = Counting()
        forward(pack, monkeypatch, y=y)
        assert pack.names == ["pdk_add_rmsnorm_quant_e4m3_blk", "pdk_f8blk_gate_up", "pdk_f8blk_gemm" + ("" if y.dtype == torch.float32 else "_bf16")]


@pytest.mark.parametrize("embd,ff,tokens", [(EMBD - 128, FF, TOKENS), (EMBD, FF - 128, TOKENS), (EMBD - 16, FF, TOKENS), (EMBD, FF, TOKENS - 1),
                                            (FF, EMBD, TOKENS)])
def test_a_workspace_of_narrower_layers_is_refused(monkeypatch, embd, ff, tokens):
    with pytest.raises(ValueError):
        forward(Refusing(), monkeypatch, ws=P.F8BlkFfnWorkspace(executor(None), embd, ff, tokens))


def test_a_workspace_of_wider_layers_is_taken(monkeypatch):
    pack = Counting()
    forward(pack, monkeypatch, ws=P.F8BlkFfnWorkspace(executor(None), EMBD + 128, FF + 16, TOKENS + 1))
    assert len(pack.names) == 3


# ---- what a later launch of the three would refuse is refused before the first, which adds proj onto x
def test_gate_and_up_of_different_sizes_are_refused_before_x_changes(monkeypatch):
    for up in (plane(EMBD, FF + 128), plane(EMBD + 128, FF)):
        with pytest.raises(ValueError):
            forward(Refusing(), monkeypatch, up=up)


@pytest.mark.parametrize("embd,ff", [(EMBD - 4, FF), (EMBD, FF - 8), (EMBD, FF - 1)])
def test_widths_that_the_products_refuse_are_refused_before_x_changes(monkeypatch, embd, ff):
    with pytest.raises(ValueError):
        forward(Refusing(), monkeypatch, embd=embd, ff=ff)


@pytest.mark.parametrize("y,error", [(torch.zeros(TOKENS, EMBD, dtype=torch.float16), TypeError), (torch.zeros(TOKENS, EMBD, dtype=torch.float64), TypeError),
                                     (None, TypeError)])
def test_a_result_that_the_down_projection_refuses_is_refused_before_x_changes(monkeypatch, y, error):
    with pytest.raises(error):
        forward(Refusing(), monkeypatch, y=y)


@pytest.mark.parametrize("which", ["gate", "up", "down"])
def test_planes_off_a_16_byte_boundary_are_refused_before_x_changes(monkeypatch, which):
    dims = (FF, EMBD) if which == "down" else (EMBD, FF)
    whole = torch.zeros(EMBD * FF + 32, dtype=torch.uint8)
    off = (-whole.data_ptr()) % 16 + 8
    off_boundary = P.F8BlkPlane(whole[off:off + EMBD * FF], torch.zeros(64), dims)
    with pytest.raises(ValueError):
        forward(Refusing(), monkeypatch, **{which: off_boundary})
    with pytest.raises(ValueError):
        forward(Refusing(), monkeypatch, **{which: P.F8BlkPlane(None, torch.zeros(64), dims)})


# ---- types: the launches read f32 whatever floating type they are given, so a narrower tensor is read and written past its end
NARROW = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("which", ["x", "proj", "norm"])
@pytest.mark.parametrize("dtype", [*NARROW, torch.float64])
def test_the_helper_refuses_a_residual_stream_of_other_types(monkeypatch, which, dtype):
    with pytest.raises(TypeError):
        forward(Refusing(), monkeypatch, **{which: torch.zeros(EMBD if which == "norm" else TOKENS * EMBD, dtype=dtype)})


def test_the_residual_may_be_missing(monkeypatch):
    pack = Counting()
    forward(pack, monkeypatch, proj=None)
    assert len(pack.names) == 3


@pytest.mark.parametrize("dtype", [*NARROW, torch.float64])
def test_f32_operands_of_the_single_calls_are_checked(monkeypatch, dtype):
    monkeypatch.setattr(P, "_stream", lambda: 0)
    ex, n, m = executor(Refusing()), 128, 2
    bad, f32, codes, w = torch.zeros(m * n, dtype=dtype), torch.zeros(m * n), torch.zeros(m * n, dtype=torch.uint8), plane(n, m)
    for i in (0, 1, 2, 3, 5):                                  # x, proj, w, xn, scale
        args = [f32, f32, f32, f32, codes, f32]
        args[i] = bad
        with pytest.raises(TypeError):
            ex.add_rmsnorm_quant_e4m3_blk(*args, n, 1e-6, m)
    for call in (lambda: ex.f8blk_dequant(w, bad), lambda: ex.quantize_e4m3_blk(f32, codes, bad, n, m), lambda: ex.f8blk_gemm(w, codes, bad, f32, m),
                 lambda: ex.f8blk_gate_up(w, w, codes, bad, codes, f32, m), lambda: ex.f8blk_gate_up(w, w, codes, f32, codes, bad, m)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
def test_weights_that_are_not_bf16_are_refused(monkeypatch, dtype):
    monkeypatch.setattr(P, "_stream", lambda: 0)
    with pytest.raises(TypeError):
        executor(Refusing()).bf16_to_f8blk(torch.zeros(128 * 128, dtype=dtype), 128, 128)


def test_what_may_be_missing_in_front_of_the_norm_may_still_be(monkeypatch):
    monkeypatch.setattr(P, "_stream", lambda: 0)
    pack = Counting()
    executor(pack).add_rmsnorm_quant_e4m3_blk(torch.zeros(256), None, torch.ones(128), None, torch.zeros(256, dtype=torch.uint8), torch.zeros(2), 128, 1e-6, 2)
    assert len(pack.names) == 1


def test_addresses_and_raw_bytes_pass(monkeypatch):
    """Operands without a floating type: an address, or a slice of a buffer of bytes."""
    monkeypatch.setattr(P, "_stream", lambda: 0)
    pack = Counting()
    ex, raw = executor(pack), torch.zeros(1024, dtype=torch.uint8)
    ex.add_rmsnorm_quant_e4m3_blk(raw.data_ptr(), raw, raw, None, raw, raw.data_ptr(), 128, 1e-6, 1)
    ex.bf16_to_f8blk(raw, 64, 8)
    ex.bf16_to_f8blk(raw.view(torch.int16), 64, 8)
    assert len(pack.names) == 3

"""e4m3 with a scale per block of 128 on a GPU.  The quantizers, the weight loader and the way back are held to the rule's exact bits; the
products to an f64 product of the same codes and scales, within what f32 sums of that length can be off; the gated front to its f64
value within that and half a step of its e4m3 result."""
import ctypes

import numpy as np
import pytest
import torch

import oracle
from gpu_util import dev_f32
from paddock_b200 import executor as X
from paddock_b200 import planes as P

pytestmark = pytest.mark.gpu
B, TOP = 128, 448.0
ULP = 2.0 ** -24          # one f32 rounding, relative


def blocks(n):
    return -(-n // B)


def e4m3_value(code):
    """f64 value of e4m3 codes (numpy uint8)."""
    code = np.asarray(code, np.uint8).astype(np.int64)
    e, m = (code >> 3) & 15, code & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(code & 128, -v, v)


def half_step(v):
    """Half the distance between the e4m3 values around |v|."""
    return 2.0 ** (np.clip(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -60))), -6, 8) - 4.0)


def nearest_code_value(v):
    """Nearest e4m3 value of f64 v, ties to even, saturating."""
    step = 2.0 * half_step(v)
    return np.clip(np.round(v / step) * step, -TOP, TOP)


def by_block(a, rows):
    """[n][k] -> [n / rows][rows][blocks(k)][B], zero-padded."""
    n, k = a.shape
    a = np.pad(a, ((0, -n % rows), (0, -k % B)))
    return a.reshape(a.shape[0] // rows, rows, a.shape[1] // B, B)


def rule(v, rows):
    """(scales, values of the codes) of the quantizer's rule in f32 on f32 v [n][k]."""
    n, k = v.shape
    g = by_block(v.astype(np.float32), rows)
    a = np.fmax.reduce(np.abs(g), axis=(1, 3))
    s = np.maximum(a / np.float32(TOP), np.float32(2.0 ** -126)).astype(np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        p = (g * (np.float32(1.0) / s)[:, None, :, None]).astype(np.float32)
        c = nearest_code_value(np.clip(p.astype(np.float64), -TOP, TOP))
    return s, c.reshape(c.shape[0] * rows, -1)[:n, :k]


def expand(s, rows, n, k):
    """Scales [..][blocks] -> [n][k]."""
    return np.repeat(np.repeat(s, rows, 0)[:n], B, 1)[:, :k]


def wild(rows, k, seed):
    """f32 [rows][k] over many magnitudes: ordinary, tiny, huge and zero blocks."""
    v = oracle.fill_normal(rows * k, seed, 1.0).reshape(rows, k)
    rng = np.random.default_rng(seed)
    mag = rng.choice([1.0, 1.0, 1e-3, 1e-30, 1e-40, 1e30, 0.0], (rows, blocks(k)))
    return (v * np.repeat(mag, B, 1)[:, :k]).astype(np.float32)


def guarded(n, dtype, before=16):
    """A buffer of n elements inside a larger one of a known pattern, and a check that the rest kept it."""
    size = torch.empty(0, dtype=dtype).element_size()
    whole = torch.full(((n + 2 * before) * size,), 0x5A, dtype=torch.uint8, device="cuda").view(dtype)
    view = whole[before:before + n]

    def kept():
        raw = whole.view(torch.uint8)
        return bool((raw[:before * size] == 0x5A).all()) and bool((raw[(before + n) * size:] == 0x5A).all())
    return view, kept


# ---------------------------------------------------------------- quantizers
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 3), (3, 16), (2, 100), (1, 128), (5, 130), (7, 384), (4, 1000), (300, 2880), (64, 5120)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("off", [0, 1])           # elements the input starts behind a 16-byte boundary
def test_quantize_blk_bit_exact(pack, rows, k, t, off):
    x = wild(rows, k, 700 + rows + k)
    d_x = torch.zeros(rows * k + off, dtype=torch.float32, device="cuda")
    d_x[off:] = dev_f32(x.reshape(-1))
    if t == "bf16":
        d_x = d_x.to(torch.bfloat16)
        x = d_x[off:].float().cpu().numpy().reshape(rows, k)
    q, q_kept = guarded(rows * k, torch.uint8)
    s, s_kept = guarded(rows * blocks(k), torch.float32)
    pack.call("pdk_quantize_e4m3_blk" + ("" if t == "f32" else "_bf16"), d_x[off:], q, s, k, rows)
    torch.cuda.synchronize()
    s_ref, v_ref = rule(x, 1)
    assert np.array_equal(s.cpu().numpy().reshape(rows, -1), s_ref)
    assert np.array_equal(e4m3_value(q.cpu().numpy()).reshape(rows, k), v_ref)
    assert q_kept() and s_kept()


def test_quantize_blk_many_blocks_a_warp(pack):
    """Enough blocks for the form with four a group of lanes, and a last thread block that is not full."""
    rows, k = 1237, 5120 + 4
    x = oracle.fill_normal(rows * k, 711, 2.0).reshape(rows, k)
    q = torch.zeros(rows * k, dtype=torch.uint8, device="cuda")
    s = torch.zeros(rows * blocks(k), dtype=torch.float32, device="cuda")
    pack.call("pdk_quantize_e4m3_blk", dev_f32(x.reshape(-1)), q, s, k, rows)
    torch.cuda.synchronize()
    s_ref, v_ref = rule(x, 1)
    assert np.array_equal(s.cpu().numpy().reshape(rows, -1), s_ref)
    assert np.array_equal(e4m3_value(q.cpu().numpy()).reshape(rows, k), v_ref)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("k", [256, 250])
def test_quantize_blk_nan_and_infinity(pack, t, k):
    x = oracle.fill_normal(4 * k, 720, 1.0).reshape(4, k)
    x[1, 5], x[2, 7] = np.nan, np.inf
    d_x = dev_f32(x.reshape(-1)).to(torch.float32 if t == "f32" else torch.bfloat16)
    q = torch.zeros(4 * k, dtype=torch.uint8, device="cuda")
    s = torch.zeros(4 * blocks(k), dtype=torch.float32, device="cuda")
    pack.call("pdk_quantize_e4m3_blk" + ("" if t == "f32" else "_bf16"), d_x, q, s, k, 4)
    torch.cuda.synchronize()
    s = s.cpu().numpy().reshape(4, -1)
    v = e4m3_value(q.cpu().numpy()).reshape(4, k)
    clean = d_x.float().cpu().numpy().reshape(4, k)
    clean[1, 5] = 0.0
    s_ref, v_ref = rule(clean[[0, 1, 3]], 1)
    assert np.array_equal(s[[0, 1, 3]], s_ref)                    # a NaN does not take part in the maximum
    assert np.isnan(v[1, 5]) and np.isnan(v[2, 7]) and np.isinf(s[2, 0]) and np.isfinite(s[2, 1])
    v[1, 5] = 0.0
    assert np.array_equal(v[[0, 1, 3]], v_ref)


def test_quantize_blk_into_codes_off_a_boundary(pack):
    rows, k = 5, 384
    x = wild(rows, k, 725)
    s_ref, v_ref = rule(x, 1)
    for before in (16, 17, 18):
        q, kept = guarded(rows * k, torch.uint8, before)
        s = torch.zeros(rows * blocks(k), dtype=torch.float32, device="cuda")
        pack.call("pdk_quantize_e4m3_blk", dev_f32(x.reshape(-1)), q, s, k, rows)
        torch.cuda.synchronize()
        assert np.array_equal(s.cpu().numpy().reshape(rows, -1), s_ref) and kept()
        assert np.array_equal(e4m3_value(q.cpu().numpy()).reshape(rows, k), v_ref)


@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (129, 144), (37, 640), (300, 1000), (260, 130), (5, 7)])
@pytest.mark.parametrize("before", [16, 17, 20])          # y on a 32-byte, a 4-byte and a 16-byte boundary
def test_bf16_to_f8blk_and_back_bit_exact(pack, n, k, before):
    w = torch.from_numpy(wild(n, k, 730 + n + k)).to(torch.bfloat16)
    ref = w.float().numpy()
    q, q_kept = guarded(n * k, torch.uint8, before)
    s, s_kept = guarded(blocks(n) * blocks(k), torch.float32)
    y, y_kept = guarded(n * k, torch.float32, before)
    pack.call("pdk_bf16_to_f8blk", w.cuda(), q, s, k, n)
    pack.call("pdk_f8blk_dequant", q, s, y, k, n)
    torch.cuda.synchronize()
    s_ref, v_ref = rule(ref, B)
    assert np.array_equal(s.cpu().numpy().reshape(s_ref.shape), s_ref)
    assert np.array_equal(e4m3_value(q.cpu().numpy()).reshape(n, k), v_ref)
    assert np.array_equal(y.cpu().numpy().reshape(n, k), v_ref.astype(np.float32) * expand(s_ref, B, n, k))
    assert q_kept() and s_kept() and y_kept()


# ---------------------------------------------------------------- residual add + norm + quantizer
@pytest.mark.parametrize("rows,n,residual,want_xn", [(1, 4, True, True), (2, 100, True, False), (3, 128, False, True), (7, 5120, True, True),
                                                     (5, 2880, False, False), (70, 5120, True, False), (2, 17408, True, True),
                                                     (1, 40000, True, True), (2, 65536, False, True)])
def test_add_rmsnorm_quant_blk(pack, rows, n, residual, want_xn):
    x = oracle.fill_normal(rows * n, 740 + n, 1.5).reshape(rows, n)
    proj = oracle.fill_normal(rows * n, 741 + n, 0.5).reshape(rows, n) if residual else None
    w = (1.0 + 0.1 * oracle.fill_normal(n, 742, 1.0)).astype(np.float32)
    eps = 1e-6
    v = x + proj if residual else x                                # one f32 addition
    v64 = v.astype(np.float64)
    xn64 = v64 / np.sqrt((v64 * v64).mean(axis=1, keepdims=True) + eps) * w
    d_x, x_kept = guarded(rows * n, torch.float32)
    d_x.copy_(dev_f32(x.reshape(-1)))
    d_xn, xn_kept = guarded(rows * n, torch.float32)
    q, q_kept = guarded(rows * n, torch.uint8)
    s, s_kept = guarded(rows * blocks(n), torch.float32)
    args = (dev_f32(proj.reshape(-1)) if residual else None, dev_f32(w))
    pack.call("pdk_add_rmsnorm_quant_e4m3_blk", d_x, *args, d_xn, q, s, n, eps, rows)
    torch.cuda.synchronize()
    assert np.array_equal(d_x.cpu().numpy().reshape(rows, n), v)
    xn = d_xn.cpu().numpy().reshape(rows, n)
    # the sum of squares: a product's rounding, at most 4 * 16 additions in a thread, 5 over lanes, 32 over warps; half of that behind the
    # root, and five roundings behind it
    assert (np.abs(xn - xn64) <= (0.5 * (1 + 64 + 5 + 32) + 6) * ULP * np.abs(xn64)).all()
    s_ref, v_ref = rule(xn, 1)
    assert np.array_equal(s.cpu().numpy().reshape(rows, -1), s_ref)
    assert np.array_equal(e4m3_value(q.cpu().numpy()).reshape(rows, n), v_ref)
    assert x_kept() and xn_kept() and q_kept() and s_kept()
    if not want_xn:
        d_x.copy_(dev_f32(x.reshape(-1)))
        q2, s2 = torch.zeros_like(q), torch.zeros_like(s)
        pack.call("pdk_add_rmsnorm_quant_e4m3_blk", d_x, *args, None, q2, s2, n, eps, rows)
        torch.cuda.synchronize()
        assert torch.equal(q2, q) and torch.equal(s2, s)


# ---------------------------------------------------------------- products
class Operands:
    """Codes and scales of tokens and of one or two planes, on the device and as f64."""

    def __init__(self, m, n, k, seed, planes=1):
        self.m, self.n, self.k = m, n, k
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(m, k, device="cuda", generator=g)
        x[:, ::17] *= 30.0
        self.xq, self.xs, self.x64 = self._codes(x, 1, g)
        self.w = [self._codes(torch.randn(n, k, device="cuda", generator=g) * 0.02, B, g) for _ in range(planes)]

    @staticmethod
    def _codes(v, rows, g):
        """Scales of a checkpoint: any positive numbers.  The values' largest code of a block is between 240 and 448."""
        n, k = v.shape
        p = torch.nn.functional.pad(v, (0, -k % B, 0, -n % rows))
        p = p.view(p.shape[0] // rows, rows, p.shape[1] // B, B)
        s = p.abs().amax(dim=(1, 3)).clamp_min(1e-20) / (240.0 + 208.0 * torch.rand(p.shape[0], p.shape[2], device=v.device, generator=g))
        q = (p / s[:, None, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
        val = (q.double() * s.double()[:, None, :, None]).reshape(p.shape[0] * rows, -1)[:n, :k]
        return q.reshape(p.shape[0] * rows, -1)[:n, :k].contiguous().view(torch.uint8), s.contiguous(), val

    def product(self, i=0):
        """f64 product and what its f32 sums may be off.  A block: 128 exact products summed in f32 (an addition may truncate: twice ULP
        each).  Over blocks: the two scales' product, one rounding per block and a split's partial sums."""
        w = self.w[i][2]
        y, ab = self.x64 @ w.T, self.x64.abs() @ w.abs().T
        return y, (2 * B + blocks(self.k) + 8 + 2) * ULP * ab


SHAPES = [(1, 1, 16), (1, 128, 128), (3, 5, 48), (2, 1024, 5120), (7, 129, 144), (17, 1000, 400), (31, 300, 17408), (33, 257, 2048),
          (64, 640, 1040), (65, 384, 512), (100, 5000, 640), (130, 260, 272), (200, 1024, 1024), (300, 700, 4000), (513, 1280, 256),
          (257, 19000, 128), (1000, 4900, 400), (1100, 2600, 1536),
          # the plans that these do not take: 64 tokens a tile, whole and split; 256 channels a tile, several rounds, rows off 16 bytes
          # and more than 48 tiles of tokens, whose last group is not full
          (6300, 2200, 144), (33, 48, 16), (3000, 48, 2400), (140, 14192, 288), (2000, 4900, 1040), (1100, 2602, 1536)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_f8blk_gemm(pack, m, n, k, t):
    o = Operands(m, n, k, 800 + m + n + k)
    ref, tol = o.product()
    y, kept = guarded(m * n, torch.float32 if t == "f32" else torch.bfloat16)
    pack.call("pdk_f8blk_gemm" + ("" if t == "f32" else "_bf16"), o.w[0][0], o.w[0][1], o.xq, o.xs, y, k, n, m)
    assert pack.device_error() == 0
    assert kept()
    if t == "bf16":
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs()      # the result's own rounding
    off = (y.view(m, n).double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("m,n,k", [(2, 136, 256), (40, 264, 512), (600, 2056, 256), (600, 2050, 256)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_f8blk_gemm_into_rows_off_a_16_byte_boundary(pack, m, n, k, t):
    """y one element behind a boundary: same values as in aligned rows, nothing around them touched."""
    o = Operands(m, n, k, 830 + n)
    dtype = torch.float32 if t == "f32" else torch.bfloat16
    got = []
    for before in (16, 17):
        y, kept = guarded(m * n, dtype, before)
        pack.call("pdk_f8blk_gemm" + ("" if t == "f32" else "_bf16"), o.w[0][0], o.w[0][1], o.xq, o.xs, y, k, n, m)
        assert pack.device_error() == 0 and kept()
        got.append(y.clone())
    assert torch.equal(got[0], got[1])


def test_f8blk_gemm_of_more_than_32_bits_of_results(pack):
    """Rows of y behind 2^32 elements."""
    m, n, k = 65700, 65600, 128
    o = Operands(m, n, k, 845)
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    pack.call("pdk_f8blk_gemm_bf16", o.w[0][0], o.w[0][1], o.xq, o.xs, y, k, n, m)
    assert pack.device_error() == 0
    for rows in (slice(0, 3), slice(m - 130, m)):
        ref, ab = o.x64[rows] @ o.w[0][2].T, o.x64[rows].abs() @ o.w[0][2].abs().T
        tol = (2 * B + 1 + 10) * ULP * ab * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs()
        assert bool(((y[rows].double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("m,n,k", [(3, 256, 512), (50, 384, 640), (700, 2304, 512)])
def test_f8blk_gemm_keeps_nan_in_its_row_and_column(pack, m, n, k):
    o = Operands(m, n, k, 840)
    wq, ws, _ = o.w[0]
    o.xq[1, 200], wq[130, 7] = 0x7F, 0xFF
    o.xs[m - 1, 1] = float("inf")
    y = torch.zeros(m, n, device="cuda")
    pack.call("pdk_f8blk_gemm", wq, ws, o.xq, o.xs, y, k, n, m)
    assert pack.device_error() == 0
    bad = ~torch.isfinite(y)
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[1], want[m - 1], want[:, 130] = True, True, True
    assert torch.equal(bad, want)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[:, 130]).all())


def check_gate_up(o, hq, hs):
    (g, dg), (u, du) = o.product(0), o.product(1)
    act = g * torch.sigmoid(g)
    h = act * u
    # silu moves by at most 1.1 times its argument; expf, the sum, the quotient and the product are rounded (expf to two units)
    dh = 1.1 * dg * (u.abs() + du) + act.abs() * du + 8 * ULP * h.abs() + 1e-37
    m, ff = o.m, o.n
    h, dh = h.cpu().numpy(), dh.cpu().numpy()
    s = hs.cpu().numpy().reshape(m, -1).astype(np.float64)
    amax = by_block(np.abs(h), 1).max(axis=(1, 3))
    assert (np.abs(s * TOP - amax) <= by_block(dh, 1).max(axis=(1, 3)) + 4 * ULP * amax).all()
    se = expand(s, 1, m, ff)
    v = h / se
    off = np.abs(e4m3_value(hq.cpu().numpy()).reshape(m, ff) - v)
    slack = dh / se + 4 * ULP * np.abs(v)
    assert (off <= np.maximum(half_step(v), half_step(np.abs(v) + slack)) + slack).all()


GATED = [(1, 16, 16), (1, 128, 128), (2, 2880, 2880), (7, 144, 144), (17, 1008, 400), (33, 272, 2048), (64, 640, 1040),
         (65, 384, 512), (130, 272, 272), (200, 1024, 1024), (300, 704, 4000), (257, 9600, 128), (1000, 4912, 400),
         (1100, 2608, 1536), (302, 2064, 7472), (6300, 1104, 144)]


def test_shapes_reach_every_plan(pack):
    """What the product tests run: each kernel, each tile size of it, with and without a split of K."""
    reached = {1: set(), 2: set()}
    for planes, shapes in ((1, SHAPES), (2, GATED)):
        for m, n, k in shapes:
            plan = (ctypes.c_uint32 * 3)()
            assert pack._lib.pdk_f8blk_plan(planes, k, n, m, plan) == 0
            reached[planes].add((plan[0], plan[1], plan[2] > 1))
    assert reached[1] == {(1, 32, False), (1, 32, True), (1, 64, False), (1, 64, True), (2, 128, False), (2, 256, False)}
    assert reached[2] == {(1, 32, False), (1, 32, True), (1, 64, True), (2, 256, False)}


@pytest.mark.parametrize("m,ff,k", GATED)
def test_f8blk_gate_up(pack, m, ff, k):
    o = Operands(m, ff, k, 860 + m + ff + k, planes=2)
    hq, q_kept = guarded(m * ff, torch.uint8)
    hs, s_kept = guarded(m * blocks(ff), torch.float32)
    (g, gs, _), (u, us, _) = o.w
    pack.call("pdk_f8blk_gate_up", g, gs, u, us, o.xq, o.xs, hq, hs, k, ff, m)
    assert pack.device_error() == 0
    assert q_kept() and s_kept()
    check_gate_up(o, hq, hs)


@pytest.mark.parametrize("m", [3, 60, 600])
def test_f8blk_gate_up_of_zero_tokens_and_of_nan(pack, m):
    """A token of zeros leaves codes of zero under the smallest scale; a NaN stays in its token."""
    ff, k = 2320, 512
    o = Operands(m, ff, k, 880, planes=2)
    o.xq[0] = 0
    o.xq[2, 300] = 0x7F
    hq = torch.full((m, ff), 0x11, dtype=torch.uint8, device="cuda")
    hs = torch.zeros(m, blocks(ff), device="cuda")
    (g, gs, _), (u, us, _) = o.w
    pack.call("pdk_f8blk_gate_up", g, gs, u, us, o.xq, o.xs, hq, hs, k, ff, m)
    assert pack.device_error() == 0
    assert bool(((hq[0] & 0x7F) == 0).all()) and bool((hs[0] == 2.0 ** -126).all())
    assert bool(((hq[2] & 0x7F) == 0x7F).all())
    assert not bool(((hq[1] & 0x7F) == 0x7F).any()) and not bool(((hq[3:] & 0x7F) == 0x7F).any())


# ---------------------------------------------------------------- as a program uses them
def test_ffn_forward_eager_captured_and_on_another_stream(pack):
    """Residual add + norm + quantizer, gated front, down projection: eager, replayed from a graph on new inputs, and beside another
    stream's run, give the same bits."""
    ex = P.GpuExecutor(pack)
    embd, ff, m = 1040, 1936, 37
    mk = lambda n, k, seed: ex.bf16_to_f8blk(torch.from_numpy(oracle.fill_normal(n * k, seed, 0.02)).cuda().to(torch.bfloat16), k, n)   # noqa: E731
    gate, up, down = mk(ff, embd, 900), mk(ff, embd, 901), mk(embd, ff, 902)
    norm = 1.0 + 0.1 * dev_f32(oracle.fill_normal(embd, 903, 1.0))
    ins = [(dev_f32(oracle.fill_normal(m * embd, 904 + i, 1.0)), dev_f32(oracle.fill_normal(m * embd, 914 + i, 1.0))) for i in range(3)]
    torch.cuda.synchronize()

    def once(x0, p0, ws, stream):
        with torch.cuda.stream(stream):
            x, y = x0.clone(), torch.zeros(m, embd, device="cuda")
            P.ffn_f8blk_forward(ex, gate, up, down, ws, x, p0, norm, 1e-6, y, m)
        return x, y

    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    ws, ws2 = (P.F8BlkFfnWorkspace(ex, embd, ff, m) for _ in range(2))
    want = [once(x, p, ws, main) for x, p in ins]
    torch.cuda.synchronize()
    for x, p in ins:                                               # the formula, coarsely: e4m3 activations are 2^-4 apart
        v = x + p
        h = (v.view(m, embd).double() * torch.rsqrt(v.view(m, embd).double().square().mean(1, keepdim=True) + 1e-6)) * norm.double()
        w = [torch.zeros(n * k, device="cuda") for n, k in ((ff, embd), (ff, embd), (embd, ff))]
        for pl, out in zip((gate, up, down), w):
            ex.f8blk_dequant(pl, out)
        g, u = (h @ w[i].view(ff, embd).double().T for i in (0, 1))
        ref = (g * torch.sigmoid(g) * u) @ w[2].view(embd, ff).double().T
        y = want[[i for i, (a, _) in enumerate(ins) if a is x][0]][1].double()
        assert float((y - ref).norm() / ref.norm()) < 2.0 ** -4    # each of the two roundings is off by at most 2^-4 of its value
    # two streams at once, a workspace each
    got = [once(*ins[0], ws, main), once(*ins[1], ws2, side)]
    torch.cuda.synchronize()
    for (x, y), (wx, wy) in zip(got, want):
        assert torch.equal(x, wx) and torch.equal(y, wy)
    # captured once, replayed on other inputs
    x_in, p_in, y_out = torch.zeros(m * embd, device="cuda"), torch.zeros(m * embd, device="cuda"), torch.zeros(m, embd, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.ffn_f8blk_forward(ex, gate, up, down, ws, x_in, p_in, norm, 1e-6, y_out, m)
    for (x, p), (wx, wy) in zip(ins, want):
        x_in.copy_(x)
        p_in.copy_(p)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x_in, wx) and torch.equal(y_out, wy)
    assert pack.device_error() == 0


@pytest.mark.parametrize("m,n,k", [(5, 1024, 5120), (300, 700, 2000), (302, 2064, 7472), (700, 2304, 512), (1100, 2608, 1536)])
def test_f8blk_products_repeat_their_bits(pack, m, n, k):
    """Sums are added in a fixed order: calls repeated on two streams at once give the same bits."""
    o = Operands(m, n, k, 890, planes=2)
    (g, gs, _), (u, us, _) = o.w
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for i in range(24):
        with torch.cuda.stream(streams[i % 2]):
            y, hq, hs = torch.zeros(m, n, device="cuda"), torch.zeros(m, n, dtype=torch.uint8, device="cuda"), torch.zeros(m, blocks(n), device="cuda")
            st = streams[i % 2].cuda_stream
            pack.call("pdk_f8blk_gemm", g, gs, o.xq, o.xs, y, k, n, m, stream=st)
            if n % 16 == 0:
                pack.call("pdk_f8blk_gate_up", g, gs, u, us, o.xq, o.xs, hq, hs, k, n, m, stream=st)
            outs.append((y, hq, hs))
    assert pack.device_error() == 0
    for out in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out, outs[0]))


def test_f8blk_through_the_operator_layer():
    """The C++ layer: planes from bf16 and from a checkpoint's two tensors, every launch, its refusals."""
    ex = X.GpuExecutor()
    try:
        m, n, k = 9, 400, 272

        def run(fn, *args):
            torch.cuda.synchronize()
            fn(*args)
            ex.synchronize()

        w = oracle.bf16_round(oracle.fill_normal(n * k, 950, 0.02))
        plane = ex.bf16_to_f8blk((w.view(np.uint32) >> 16).astype(np.uint16), k, n)
        assert plane.kind == "F8Blk" and plane.dims == (k, n) and plane.bytes() == n * k + 4 * blocks(n) * blocks(k)
        s_ref, v_ref = rule(w.reshape(n, k), B)
        y = torch.zeros(n * k, device="cuda")
        run(ex.f8blk_dequant, plane, y)
        assert np.array_equal(y.cpu().numpy().reshape(n, k), v_ref.astype(np.float32) * expand(s_ref, B, n, k))
        o = Operands(m, n, k, 951, planes=2)
        gate, up = (ex.f8blk_upload(q.cpu().numpy(), s.cpu().numpy(), k, n) for q, s, _ in o.w)
        y = torch.zeros(m, n, device="cuda")
        run(ex.f8blk_gemm, gate, o.xq, o.xs, y, m)
        ref, tol = o.product()
        assert bool(((y.double() - ref).abs() <= tol).all())
        hq, hs = torch.zeros(m * n, dtype=torch.uint8, device="cuda"), torch.zeros(m * blocks(n), device="cuda")
        run(ex.f8blk_gate_up, gate, up, o.xq, o.xs, hq, hs, m)
        check_gate_up(o, hq, hs)
        x = oracle.fill_normal(m * k, 952, 1.0).reshape(m, k)
        d_x, q, s = dev_f32(x.reshape(-1)), torch.zeros(m * k, dtype=torch.uint8, device="cuda"), torch.zeros(m * blocks(k), device="cuda")
        run(ex.quantize_e4m3_blk, d_x, q, s, k, m)
        assert np.array_equal(s.cpu().numpy().reshape(m, -1), rule(x, 1)[0])
        q2, s2, xn = torch.zeros_like(q), torch.zeros_like(s), torch.zeros_like(d_x)
        run(ex.add_rmsnorm_quant_e4m3_blk, d_x, None, torch.ones(k, device="cuda"), xn, q2, s2, k, 1e-6, m)
        s_ref, v_ref = rule(xn.cpu().numpy().reshape(m, k), 1)
        assert np.array_equal(s2.cpu().numpy().reshape(m, -1), s_ref)
        assert np.array_equal(e4m3_value(q2.cpu().numpy()).reshape(m, k), v_ref)
        row = ex.f8row_upload(o.w[0][0].cpu().numpy(), np.ones(n, np.float32), k, n)
        for bad in (lambda: ex.f8blk_gemm(row, o.xq, o.xs, y, m), lambda: ex.f8blk_gate_up(gate, row, o.xq, o.xs, hq, hs, m),
                    lambda: ex.f8blk_gate_up(gate, ex.f8blk_upload(np.zeros((128, k), np.uint8), np.zeros((1, blocks(k))), k, 128), o.xq, o.xs, hq, hs, m),
                    lambda: ex.f8blk_upload(np.zeros((4, 24), np.uint8), np.zeros((1, 1)), 24, 4), lambda: ex.f8row_gemm(gate, o.xq, o.xs, y, m)):
            with pytest.raises(X.GpuError) as e:
                bad()
            assert e.value.kind == "Unsupported"
    finally:
        ex.close()

"""Block-scaled e4m3 products at the ends of f32's range: gates where 1 + exp(-g) nears the largest f32, and scales whose product does."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_f8blk import ULP, blocks, by_block, e4m3_value, expand, guarded, half_step

pytestmark = pytest.mark.gpu
ONE, TWO, MINUS_ONE = 0x38, 0x40, 0xB8


def plan(pack, planes, m, n, k):
    p = (ctypes.c_uint32 * 3)()
    assert pack._lib.pdk_f8blk_plan(planes, k, n, m, p) == 0
    return tuple(p)


@pytest.mark.parametrize("m,ff,k,kernel", [(30, 128, 2048, 1), (40, 400, 2048, 1), (4000, 2064, 128, 2)])
def test_gated_unit_of_gates_down_to_where_the_exponential_overflows(pack, m, ff, k, kernel):
    """g / (1 + exp(-g)) * u is an ordinary f32 number for g down to -88.72, where exp(-g) passes f32; below it is 0.  The ups are large enough
    for the result to be far from the smallest scale."""
    assert plan(pack, 2, m, ff, k)[0] == kernel
    xq = torch.zeros(m, k, dtype=torch.uint8, device="cuda")
    xq[:, 0] = ONE
    g = torch.linspace(80.0, 95.0, m, device="cuda")                    # a token's only scale, and minus its gate
    gq = torch.zeros(ff, k, dtype=torch.uint8, device="cuda")
    gq[:, 0] = MINUS_ONE
    uq = torch.zeros(ff, k, dtype=torch.uint8, device="cuda")
    uq[:, 0] = (0x30 + torch.arange(ff, device="cuda") % 16).to(torch.uint8)      # 0.5 to 1.875
    gs, us = torch.ones(blocks(ff), blocks(k), device="cuda"), torch.full((blocks(ff), blocks(k)), 2.0 ** 90, device="cuda")
    hq, q_kept = guarded(m * ff, torch.uint8)
    hs, s_kept = guarded(m * blocks(ff), torch.float32)
    pack.call("pdk_f8blk_gate_up", gq, gs, uq, us, xq, g.view(m, 1).expand(m, blocks(k)).contiguous(), hq, hs, k, ff, m)
    assert pack.device_error() == 0 and q_kept() and s_kept()
    g64 = -g.double().cpu().numpy()[:, None]
    u64 = -g64 * 2.0 ** 90 * e4m3_value(uq[:, 0].cpu().numpy())[None]
    h = g64 / (1.0 + np.exp(-g64)) * u64
    s = hs.cpu().numpy().reshape(m, -1).astype(np.float64)
    v = e4m3_value(hq.cpu().numpy()).reshape(m, ff)
    top = float(np.log(np.finfo(np.float32).max))
    whole, none = (-g64[:, 0] < top - 1e-4), (-g64[:, 0] > top + 1e-4)
    assert whole.sum() > m // 3 and none.sum() > m // 4
    assert (v[none] == 0).all() and (s[none] == 2.0 ** -126).all()
    # expf two units (4 roundings), the sum 1, the quotient two units, the product 1; u: the scales' product and its multiply-add 2
    rel = 12 * ULP
    amax = by_block(np.abs(h), 1).max(axis=(1, 3))
    assert (np.abs(s * 448.0 - amax) <= (rel + 4 * ULP) * amax)[whole].all()
    want = h / expand(s, 1, m, ff)
    slack = (rel + 4 * ULP) * np.abs(want)
    off = np.abs(v - want)
    assert (off <= np.maximum(half_step(want), half_step(np.abs(want) + slack)) + slack)[whole].all()


@pytest.mark.parametrize("m,ff,k,kernel", [(30, 128, 2048, 1), (40, 400, 2048, 1), (4000, 2064, 128, 2)])
def test_gated_unit_of_gates_up_to_the_largest_f32(pack, m, ff, k, kernel):
    """silu(g) is g for large gates, up to where f32 ends; the ups are small, so the result is an ordinary number."""
    assert plan(pack, 2, m, ff, k)[0] == kernel
    xq = torch.zeros(m, k, dtype=torch.uint8, device="cuda")
    xq[:, 0] = ONE
    g = torch.exp2(torch.linspace(120.0, 127.9, m, dtype=torch.float64, device="cuda")).float()           # a token's only scale, and its gate
    gq, uq = torch.zeros(ff, k, dtype=torch.uint8, device="cuda"), torch.zeros(ff, k, dtype=torch.uint8, device="cuda")
    gq[:, 0] = ONE
    uq[:, 0] = (0x30 + torch.arange(ff, device="cuda") % 16).to(torch.uint8)
    gs, us = torch.ones(blocks(ff), blocks(k), device="cuda"), torch.full((blocks(ff), blocks(k)), 2.0 ** -140, device="cuda")
    hq, hs = torch.zeros(m * ff, dtype=torch.uint8, device="cuda"), torch.zeros(m * blocks(ff), device="cuda")
    pack.call("pdk_f8blk_gate_up", gq, gs, uq, us, xq, g.view(m, 1).expand(m, blocks(k)).contiguous(), hq, hs, k, ff, m)
    assert pack.device_error() == 0
    g64 = g.double().cpu().numpy()[:, None]
    h = g64 * (g64 * 2.0 ** -140 * e4m3_value(uq[:, 0].cpu().numpy())[None])
    s = hs.cpu().numpy().reshape(m, -1).astype(np.float64)
    rel = 12 * ULP                                                       # as above
    amax = by_block(np.abs(h), 1).max(axis=(1, 3))
    assert (np.abs(s * 448.0 - amax) <= (rel + 4 * ULP) * amax).all()
    want = h / expand(s, 1, m, ff)
    slack = (rel + 4 * ULP) * np.abs(want)
    off = np.abs(e4m3_value(hq.cpu().numpy()).reshape(m, ff) - want)
    assert (off <= np.maximum(half_step(want), half_step(np.abs(want) + slack)) + slack).all()


@pytest.mark.parametrize("m,n,k", [(5, 272, 2048), (40, 400, 2048), (4000, 2064, 384), (300, 700, 256)])
@pytest.mark.parametrize("xs,ws", [(2.0 ** -60, 2.0 ** -66), (2.0 ** -126, 1.0), (2.0 ** 100, 2.0 ** 9), (2.0 ** -100, 2.0 ** 120)])
def test_products_under_scales_whose_product_f32_holds(pack, m, n, k, xs, ws):
    """The two scales of a block are multiplied first.  Down to 2^-126 and up to where the result itself ends, with codes whose products and
    sums are exact in f32, so is the result."""
    g = torch.Generator(device="cuda").manual_seed(970)
    code = lambda r: torch.tensor([0x00, ONE, TWO, MINUS_ONE], dtype=torch.uint8, device="cuda")[torch.randint(0, 4, (r, k), device="cuda", generator=g)]     # noqa: E731
    xq, wq = code(m), code(n)
    y = torch.zeros(m, n, device="cuda")
    pack.call("pdk_f8blk_gemm", wq, torch.full((blocks(n), blocks(k)), ws, device="cuda"), xq, torch.full((m, blocks(k)), xs, device="cuda"), y, k, n, m)
    assert pack.device_error() == 0
    value = torch.tensor(e4m3_value(np.arange(256)), device="cuda")
    want = (value[xq.long()] @ value[wq.long()].T) * xs * ws
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("m,n,k", [(5, 272, 2048), (4000, 2064, 128)])
def test_products_under_scales_whose_product_passes_f32(pack, m, n, k):
    """Beyond f32 the scales' product is an infinity: a sum of codes becomes one of its sign, a sum of zero NaN.  Below 2^-149 it is 0."""
    xq, wq = torch.zeros(m, k, dtype=torch.uint8, device="cuda"), torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    xq[:, 0], wq[0::3, 0], wq[1::3, 0] = ONE, ONE, MINUS_ONE
    y = torch.zeros(m, n, device="cuda")
    big, small = (lambda r, s: torch.full((r, blocks(k)), s, device="cuda")), 2.0 ** -100
    sx, sw = big(m, 1.0), big(blocks(n), 1.0)
    sx[:, 0], sw[:, 0] = 2.0 ** 100, 2.0 ** 100
    pack.call("pdk_f8blk_gemm", wq, sw, xq, sx, y, k, n, m)
    assert bool((y[:, 0::3] == float("inf")).all()) and bool((y[:, 1::3] == float("-inf")).all()) and bool(y[:, 2::3].isnan().all())
    sx[:, 0], sw[:, 0] = small, small
    pack.call("pdk_f8blk_gemm", wq, sw, xq, sx, y, k, n, m)
    assert pack.device_error() == 0 and bool((y == 0).all())

"""What the block-scaled e4m3 calls refuse or return from by their arguments alone, before anything is launched or read (no GPU; the
addresses are made up and no call here gets as far as using them)."""
import ctypes as C

import pytest
import torch

import paddock_b200 as pb
from paddock_b200 import pack as packmod
from paddock_b200 import planes as P

INVALID, UNSUPPORTED = 1, 801                   # cudaErrorInvalidValue, cudaErrorNotSupported
A = 0x7000_0000_0000                            # an address aligned to anything

# name -> (how many pointers, their strictest offset, numbers of a good call)
PRODUCTS = {"pdk_f8blk_gemm": (5, (128, 128, 4)), "pdk_f8blk_gemm_bf16": (5, (128, 128, 4)), "pdk_f8blk_gate_up": (8, (128, 128, 4))}
QUANTIZERS = {"pdk_quantize_e4m3_blk": (3, (128, 4)), "pdk_quantize_e4m3_blk_bf16": (3, (128, 4)), "pdk_bf16_to_f8blk": (3, (128, 128)),
              "pdk_f8blk_dequant": (3, (128, 128))}
# byte alignment of each pointer
ALIGN = {"pdk_f8blk_gemm": (16, 4, 16, 4, 4), "pdk_f8blk_gemm_bf16": (16, 4, 16, 4, 2), "pdk_f8blk_gate_up": (16, 4, 16, 4, 16, 4, 16, 4),
         "pdk_quantize_e4m3_blk": (4, 1, 4), "pdk_quantize_e4m3_blk_bf16": (2, 1, 4), "pdk_bf16_to_f8blk": (2, 1, 4),
         "pdk_f8blk_dequant": (1, 4, 4)}


def status(name, *args):
    fn = getattr(C.CDLL(pb.lib_path()), name)
    kinds = packmod._EXTRA_SIGS[name]
    assert len(args) == len(kinds)
    fn.argtypes = [packmod._KIND[k] for k in kinds] + [C.c_void_p]
    fn.restype = C.c_int
    return fn(*args, None)


@pytest.mark.parametrize("name", [*PRODUCTS, *QUANTIZERS])
def test_a_missing_operand_is_refused(name):
    n, nums = {**PRODUCTS, **QUANTIZERS}[name]
    for i in range(n):
        assert status(name, *[None if j == i else A for j in range(n)], *nums) == INVALID


@pytest.mark.parametrize("name", ALIGN)
def test_addresses_off_their_boundary_are_refused(name):
    n, nums = {**PRODUCTS, **QUANTIZERS}[name]
    for i, a in enumerate(ALIGN[name]):
        if a > 1:
            assert status(name, *[A + a // 2 if j == i else A for j in range(n)], *nums) == INVALID


@pytest.mark.parametrize("name", [*PRODUCTS, *QUANTIZERS])
def test_nothing_to_do_is_no_error(name):
    n, nums = {**PRODUCTS, **QUANTIZERS}[name]
    for zero in range(1 if name in PRODUCTS else 0, len(nums)):
        assert status(name, *[None] * n, *[0 if j == zero else v for j, v in enumerate(nums)]) == 0


@pytest.mark.parametrize("name", PRODUCTS)
@pytest.mark.parametrize("in_dim", [0, 8, 100, 129, 0xFFFFFFF0])
def test_products_refuse_rows_that_boxes_cannot_start_on(name, in_dim):
    n, nums = PRODUCTS[name]
    assert status(name, *[A] * n, in_dim, *nums[1:]) == INVALID


@pytest.mark.parametrize("out_dim,batch", [(0x80000000, 1), (128, 0x80000000)])
def test_products_refuse_sizes_past_signed_coordinates(out_dim, batch):
    for name, (n, _) in PRODUCTS.items():
        assert status(name, *[A] * n, 128, out_dim, batch) == INVALID


@pytest.mark.parametrize("ff", [1, 8, 100, 1000])
def test_gate_up_refuses_rows_that_the_down_projection_could_not_read(ff):
    assert status("pdk_f8blk_gate_up", *[A] * 8, 128, ff, 4) == INVALID


def test_plan_query_refuses_what_is_no_product():
    lib, plan = C.CDLL(pb.lib_path()), (C.c_uint32 * 3)()
    for args in ((0, 128, 128, 1), (3, 128, 128, 1), (1, 0, 128, 1), (1, 128, 0, 1), (1, 128, 128, 0)):
        assert lib.pdk_f8blk_plan(*args, plan) == INVALID
    assert lib.pdk_f8blk_plan(1, 128, 128, 1, None) == INVALID


def test_quantizers_refuse_more_blocks_than_their_numbers_hold():
    for name in ("pdk_quantize_e4m3_blk", "pdk_quantize_e4m3_blk_bf16", "pdk_bf16_to_f8blk", "pdk_f8blk_dequant"):
        assert status(name, A, A, A, 0xFFFFFFFC, 0xFFFFFFFF) == INVALID
        assert status(name, A, A, A, 0xFFFFFF80, 1) == INVALID           # a row whose last block's end has no number
    assert status("pdk_bf16_to_f8blk", A, A, A, 1, 0xFFFFFF80) == INVALID


def test_add_rmsnorm_quant_refusals():
    call = lambda ptrs, n=256, batch=2: status("pdk_add_rmsnorm_quant_e4m3_blk", *ptrs, n, 1e-6, batch)      # noqa: E731
    good = [A] * 6
    for i in (0, 2, 4, 5):                                       # proj and xn may be missing
        assert call([None if j == i else A for j in range(6)]) == INVALID
    for i, off in ((0, 8), (1, 8), (2, 8), (3, 8), (4, 2), (5, 2)):
        assert call([A + off if j == i else A for j in range(6)]) == INVALID
    for n in (1, 2, 3, 130):
        assert call(good, n) == INVALID
    assert call(good, 65540) == UNSUPPORTED
    assert call(good, 0) == 0 and call(good, 256, 0) == 0


def test_planes_that_do_not_fit_together_are_refused():
    class Fails:
        def call(self, *a, **k):
            raise AssertionError("launched")

    ex = P.GpuExecutor.__new__(P.GpuExecutor)
    ex.pack, ex.device = Fails(), "cpu"
    a, b = P.F8BlkPlane(None, None, (128, 256)), P.F8BlkPlane(None, None, (128, 384))
    with pytest.raises(ValueError):
        ex.f8blk_gate_up(a, b, None, None, None, None, 1)
    ws = P.F8BlkFfnWorkspace(ex, 128, 256, 4)
    with pytest.raises(ValueError):
        P.ffn_f8blk_forward(ex, a, a, b, ws, None, None, None, 1e-6, None, 1)
    with pytest.raises(ValueError):
        P.ffn_f8blk_forward(ex, a, a, P.F8BlkPlane(None, None, (256, 128)), ws, None, None, None, 1e-6, None, 5)
    with pytest.raises(TypeError):
        ex.quantize_e4m3_blk(torch.zeros(128, dtype=torch.float16), None, None, 128, 1)
    with pytest.raises(TypeError):
        ex.f8blk_gemm(a, None, None, torch.zeros(256, dtype=torch.float64), 1)

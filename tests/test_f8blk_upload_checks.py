"""What the operator layer's front end refuses of a checkpoint's block scales, on the host (no device: the upload itself is replaced)."""
import numpy as np
import pytest

from paddock_b200 import executor as X


def upload(monkeypatch, scales):
    ex, taken = X.GpuExecutor.__new__(X.GpuExecutor), []
    ex._h = None
    monkeypatch.setattr(ex, "_plane", lambda fn, codes, s, k, n: taken.append(np.ctypeslib.as_array(s, (4,)).copy()), raising=False)
    ex.f8blk_upload(np.zeros((256, 256), np.uint8), scales, 256, 256)
    return taken[0]


@pytest.mark.parametrize("dtype", [np.float32, np.float64, np.float16])
def test_scales_go_up_as_f32(monkeypatch, dtype):
    s = np.array([[0.5, 2.0], [0.25, 8.0]], dtype)
    assert np.array_equal(upload(monkeypatch, s), s.astype(np.float32).reshape(-1))


@pytest.mark.parametrize("dtype", [np.uint16, np.int16, np.uint8, np.int32])
def test_bits_of_scales_are_not_taken_for_numbers(monkeypatch, dtype):
    """bf16 scales as their bits, the way weights are handed over: 0x3f80 is 1, not 16256."""
    with pytest.raises(TypeError):
        upload(monkeypatch, np.full((2, 2), 0x3F, dtype))


# ---- the operator layer's block calls are f32 in and out: a tensor of another floating type would be read or written at another size
class Launched(Exception):
    pass


class Lib:
    def __getattr__(self, name):
        def call(*a):
            raise Launched(name)
        return call


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float64"])
def test_other_floating_types_are_refused(monkeypatch, dtype):
    import torch
    monkeypatch.setattr(X, "_lib", lambda: Lib())
    ex, w = X.GpuExecutor.__new__(X.GpuExecutor), X.Plane.__new__(X.Plane)
    ex._h = w._h = None
    bad, f32, codes = torch.zeros(256, dtype=getattr(torch, dtype)), torch.zeros(256), torch.zeros(256, dtype=torch.uint8)
    norm = [f32, f32, f32, f32, codes, f32]
    calls = [(ex.quantize_e4m3_blk, (f32, codes, f32, 128, 2), (0, 2)), (ex.add_rmsnorm_quant_e4m3_blk, (*norm, 128, 1e-6, 2), (0, 1, 2, 3, 5)),
             (ex.f8blk_dequant, (w, f32), (1,)), (ex.f8blk_gemm, (w, codes, f32, f32, 2), (2, 3)),
             (ex.f8blk_gate_up, (w, w, codes, f32, codes, f32, 2), (3, 5))]
    for call, good, which in calls:
        with pytest.raises(Launched):
            call(*good)
        for i in which:
            args = list(good)
            args[i] = bad
            with pytest.raises(TypeError):
                call(*args)
            args[i] = bad.data_ptr()                                     # an address passes
            with pytest.raises(Launched):
                call(*args)
    ex.close = w.free = lambda: None

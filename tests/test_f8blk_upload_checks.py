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

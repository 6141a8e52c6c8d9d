"""Host side of the FP8 operators without a GPU: buffer sizes, the row slots of ragged groups, refusals of CPU tensors."""

import ctypes

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def so():
    from lockstep_b200 import _lib, build
    build.build()
    return _lib.lib()


def test_sizes_agree_with_python(so):
    from lockstep_b200 import fp8
    rng = np.random.default_rng(0)
    for _ in range(200):
        rows, K, G = int(rng.integers(1, 5000)), int(rng.integers(1, 5000)), int(rng.integers(1, 65))
        assert so.ls_fp8_sf_bytes(rows, K) == fp8.sf_bytes(rows, K) == -(-rows // 128) * -(-K // 512) * 512
        assert so.ls_fp8_slots(rows, G) == fp8.slots(rows, G)
        assert so.ls_fp8_slots(rows, 0) == -(-rows // 128)


def test_slots_of_groups_do_not_collide(so):
    from lockstep_b200 import fp8
    rng = np.random.default_rng(1)
    for _ in range(300):
        sizes = rng.integers(0, rng.choice([2, 5, 130, 400]), size=rng.integers(1, 40))
        off = np.concatenate([[0], np.cumsum(sizes)])
        taken = [o // 128 + g + i for g, (o, n) in enumerate(zip(off, sizes)) for i in range(-(-n // 128))]
        assert len(set(taken)) == len(taken)
        assert all(0 <= t < fp8.slots(int(off[-1]), len(sizes)) for t in taken)


def test_buffers_grow_with_what_is_kept(so):
    T, N, K = 1000, 600, 520
    bytes_of = lambda what, G, grads: so.ls_fp8_linear_bytes(what, T, N, K, G, grads)
    assert so.ls_fp8_linear_bytes(2, T, N, K, 0, 0) == 0                          # nothing kept without gradients
    assert bytes_of(2, 0, 3) == bytes_of(2, 0, 1) + bytes_of(2, 0, 2)
    assert bytes_of(2, 0, 2) >= T * K and bytes_of(2, 0, 1) >= N * K
    assert bytes_of(2, 4, 2) >= (T // 128 + 4) * 128 * K                          # whole slots
    assert bytes_of(0, 0, 0) >= T * K and so.ls_fp8_linear_bytes(0, 1, 64, 64, 0, 0) == 0
    assert so.ls_fp8_linear_bytes(9, T, N, K, 0, 0) == -1


def test_cpu_tensors_are_refused(so):
    from lockstep_b200 import fp8, fp8_linear
    x, w = torch.zeros(4, 32), torch.zeros(8, 32)
    codes, sf = torch.zeros(8, 32).to(torch.float8_e4m3fn), torch.zeros(512, dtype=torch.uint8)
    off = torch.tensor([0, 4])
    for call in (lambda: fp8.quantize_fp8(x), lambda: fp8.quantize_fp8_packed(x), lambda: fp8.quantize_fp8_both(x),
                 lambda: fp8.quantize_fp8_weight(w), lambda: fp8.fp8_gemm(codes, codes, sf, sf),
                 lambda: fp8.dequantize_fp8(codes, torch.ones(8, 1)),
                 lambda: fp8_linear.linear(x, w), lambda: fp8_linear.linear_quantized(x, codes, sf),
                 lambda: fp8_linear.grouped_linear(x, w[None], off), lambda: fp8_linear.FP8Linear(32, 8)(x)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(AssertionError):
        fp8_linear.FP8Linear(8, 8, bias=True)


def test_shapes_are_checked_before_the_device():
    from lockstep_b200 import fp8_linear
    x, w = torch.zeros(4, 32), torch.zeros(8, 32)
    with pytest.raises(AssertionError):
        fp8_linear.linear(x, w[None])
    with pytest.raises(AssertionError):
        fp8_linear.linear(x, torch.zeros(8, 31))
    with pytest.raises(AssertionError):
        fp8_linear.grouped_linear(x[None], w[None], torch.tensor([0, 4]))
    with pytest.raises(TypeError):
        fp8_linear.linear(x.half(), w)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device error path")
def test_entry_points_refuse_without_a_device(so):
    n = ctypes.c_int64(128)
    assert so.ls_fp8_gemm(0, None, 128, None, 128, None, None, None, 0, 1, 1, 128, None) in (-5, -3)
    assert so.ls_quantize_fp8(None, 0, 1, 128, None, 0, None, 128, None, None, None) in (-5, -3)
    assert so.ls_fp8_linear(None, 0, 1, 128, None, 128, None, 1, None, 0, None, 1, 0, None, None) in (-5, -3)
    assert n.value == 128 and so.ls_last_error()

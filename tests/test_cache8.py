"""Rotary frequencies and the checks of arguments of the 8-bit cache and its operators that need no
device, and the reference that the GPU tests compare with."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from gufo_npu_b200 import _capi, backend, build
from gufo_npu_b200.cache8 import Batch, CudaCache8
from tests import cache8_reference as R


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


def rope_frequencies(lib, **kw):
    args = dict(rope_dim=64, theta=1e7, layout="halves", scaling="none", factor=1.0, original_positions=0.0,
                fast_turns=32.0, slow_turns=1.0, magnitude=0.0)
    args.update(kw)
    params = backend.rope_params(**args)
    out = (C.c_double * 256)()
    magnitude = C.c_double()
    status = lib.gufo_cuda_rope_frequencies(C.byref(params), out, C.byref(magnitude))
    return status, np.array(out[:max(args["rope_dim"], 0) // 2]), magnitude.value


@pytest.mark.parametrize("rope_dim, theta, scaling, more", [
    (64, 1e7, "none", {}), (2, 1e4, "none", {}), (512, 5e5, "none", {}), (128, 1e4, "linear", {"factor": 8.0}),
    (64, 1e7, "by_parts", {"factor": 8.0, "original": 32768.0}), (128, 1e4, "by_parts", {"factor": 4.0, "original": 4096.0}),
    (10, 1e4, "by_parts", {"factor": 40.0, "original": 100.0, "fast": 1e6, "slow": 1e5}),
    (32, 1e6, "by_parts", {"factor": 0.5, "original": 1e30})])
def test_frequencies(lib, rope_dim, theta, scaling, more):
    kw = {{"original": "original_positions", "fast": "fast_turns", "slow": "slow_turns"}.get(k, k): v for k, v in more.items()}
    status, got, magnitude = rope_frequencies(lib, rope_dim=rope_dim, theta=theta, scaling=scaling, **kw)
    assert status == 0
    want = R.frequencies(rope_dim, theta, scaling, **more)
    # (a power, whose argument is off by half a step times its logarithm, and a handful of operations in 64 bits)
    np.testing.assert_allclose(got, want, rtol=64 * 2.0 ** -53, atol=0)
    factor = more.get("factor", 1.0)
    assert magnitude == (0.1 * math.log(factor) + 1.0 if scaling == "by_parts" and factor > 1 else 1.0)
    assert rope_frequencies(lib, scaling="linear", factor=2.0, magnitude=1.25)[2] == 1.25


@pytest.mark.parametrize("kw, status", [
    ({"rope_dim": 0}, 2), ({"rope_dim": 3}, 2), ({"rope_dim": 514}, 2), ({"rope_dim": -2}, 2), ({"theta": 1.0}, 1),
    ({"theta": float("nan")}, 1), ({"theta": float("inf")}, 1), ({"scaling": "linear", "factor": 0.0}, 1),
    ({"scaling": "linear", "factor": -1.0}, 1), ({"scaling": "linear", "factor": 1e-310}, 1), ({"magnitude": 1e300}, 1),
    ({"scaling": "by_parts", "original_positions": 0.0}, 1),
    ({"scaling": "by_parts", "original_positions": 100.0, "fast_turns": 1.0, "slow_turns": 1.0}, 1),
    ({"scaling": "by_parts", "original_positions": 100.0, "slow_turns": 0.0}, 1), ({"magnitude": float("nan")}, 1)])
def test_frequencies_refused(lib, kw, status):
    assert rope_frequencies(lib, **kw)[0] == status
    assert b"rope" in lib.gufo_cuda_last_error(None)


def test_unknown_enumerators_refused(lib):
    params = backend.rope_params(64, 1e4, "halves", "none", 1.0, 0.0, 32.0, 1.0, 0.0)
    out, magnitude = (C.c_double * 32)(), C.c_double()
    assert lib.gufo_cuda_rope_frequencies(C.byref(params), None, C.byref(magnitude)) == 1
    assert lib.gufo_cuda_rope_frequencies(C.byref(params), out, None) == 1
    assert lib.gufo_cuda_rope_frequencies(None, out, C.byref(magnitude)) == 1
    params.layout = 2
    assert lib.gufo_cuda_rope_frequencies(C.byref(params), out, C.byref(magnitude)) == 1
    params.layout, params.scaling = 0, 3
    assert lib.gufo_cuda_rope_frequencies(C.byref(params), out, C.byref(magnitude)) == 1
    for kw in ({"layout": "thirds"}, {"scaling": "ntk"}):
        with pytest.raises(ValueError):
            rope_frequencies(lib, **kw)


def test_null_contexts_refused(lib):
    out, size, ptr = C.c_int64(), C.c_size_t(), C.c_void_p()
    config, batch = _capi.Cache8Config(1, 1, 16, 16, 0, 0), _capi.Cache8Batch()
    assert lib.gufo_cuda_rope_create(None, None, C.byref(out)) == 1
    assert lib.gufo_cuda_rope_free(None, 1) == 1
    assert lib.gufo_cuda_rope_device(None, 1, None, 1, None, 1) == 1
    assert lib.gufo_cuda_cache8_create(None, C.byref(config), C.byref(out)) == 1
    assert lib.gufo_cuda_cache8_free(None, 1) == 1
    assert lib.gufo_cuda_cache8_weights(None, 1, C.byref(ptr)) == 1
    assert lib.gufo_cuda_cache8_append_device(None, 1, C.byref(batch), None, 0, 0, None, 0, 0) == 1
    assert lib.gufo_cuda_cache8_rows_device(None, 1, C.byref(batch), None, None) == 1
    assert lib.gufo_cuda_cache8_attend_scratch(None, 1, 1, 1, 0, C.byref(size)) == 1
    assert lib.gufo_cuda_cache8_attend_device(None, 1, C.byref(batch), None) == 1
    assert lib.gufo_cuda_cache8_evict_device(None, 1, C.byref(batch), 1, 0, 0, None, None, 0, None) == 1


def test_host_tensors_refused():
    with pytest.raises(ValueError):
        Batch(0, torch.zeros(2, dtype=torch.int32), None, None)
    with pytest.raises(ValueError):
        backend.check_rows("rows", 0, torch.zeros(2, 1, 16))
    with pytest.raises(ValueError):
        CudaCache8(None, 1, 1, 16, 16, format="e5m2")


# ---- the reference itself ---------------------------------------------------------------


def test_reference_codes_are_torch_e4m3():
    x = torch.cat([torch.randn(5000) * 2.0 ** torch.randint(-14, 9, (5000,)),
                   torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float(),
                   torch.tensor([0.0, 448.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, 1.0625, 1.1875, 0.9375 * 2.0 ** -6])])
    x = x[torch.isfinite(x)].clamp(-448, 448)
    assert np.array_equal(R.nearest(x.numpy(), "e4m3"), x.to(torch.float8_e4m3fn).float().numpy())
    y = torch.cat([torch.linspace(-127, 127, 1017), torch.tensor([0.5, 1.5, -2.5])])
    assert np.array_equal(R.nearest(y.numpy(), "int8"), torch.round(y).numpy())


@pytest.mark.parametrize("form, top, scale", [("e4m3", 448.0, 1.0), ("e4m3", 449.0, 2.0), ("e4m3", 224.0, 0.5),
                                              ("int8", 127.0, 1.0), ("int8", 127.5, 2.0), ("int8", 63.5, 0.5),
                                              ("int8", 0.0, 2.0 ** -126), ("e4m3", 2.0 ** 127, 2.0 ** 119)])
def test_reference_scales(form, top, scale):
    assert R.scale_for(top, form) == scale

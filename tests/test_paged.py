"""Rotary positions and paged caches without a GPU: frequencies, and what is
refused before anything is launched."""

import ctypes
import math

import numpy as np
import pytest
import torch

from aegaeon_amd import _lib, ops


def test_frequencies():
    f, a = ops.rotary_frequencies(8, base=10000.0)
    assert a == 1.0 and np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-14)
    f, _ = ops.rotary_frequencies(8, scaling="linear", factor=4.0)
    assert np.allclose(f, [0.25, 0.025, 0.0025, 0.00025], rtol=1e-14)
    f, _ = ops.rotary_frequencies(4, base=16.0, scaling="base", factor=4.0)
    assert np.allclose(f, [1.0, 1.0 / math.sqrt(16 * 16)], rtol=1e-14)


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("scaling", ["ramp", "smooth"])
def test_scaled_frequencies_keep_the_fast_pairs_and_divide_the_slow_ones(dim, scaling):
    length, factor = 4096, 8.0
    plain, _ = ops.rotary_frequencies(dim)
    f, a = ops.rotary_frequencies(dim, scaling=scaling, factor=factor, length=length)
    turns = plain * length / (2 * math.pi)
    many, few = (33, 0.9) if scaling == "ramp" else (4, 1)
    assert np.allclose(f[turns >= many], plain[turns >= many], rtol=1e-12)
    # (a ramp ends at whole pairs: the last pair with a turn or more may be past its end)
    slow = np.flatnonzero(turns <= few)[1:]
    assert np.allclose(f[slow], plain[slow] / factor, rtol=1e-12)
    assert ((f <= plain * (1 + 1e-12)) & (f >= plain / factor * (1 - 1e-12))).all()
    assert (np.diff(f) < 0).all()
    assert a == pytest.approx(1 + 0.1 * math.log(factor) if scaling == "ramp" else 1.0)


@pytest.mark.parametrize("kw,match", [
    (dict(dim=7), "even"), (dict(dim=0), "even"), (dict(dim=8, scaling="other"), "unknown"),
    (dict(dim=8, base=0.5), "base"), (dict(dim=8, base=math.inf), "base"),
    (dict(dim=8, factor=0.0), "factor"), (dict(dim=8, factor=math.nan), "factor"),
    (dict(dim=8, scaling="ramp", factor=2.0), "length"),
    (dict(dim=8, scaling="smooth", factor=2.0), "length"),
    (dict(dim=2, scaling="base", factor=2.0), "single pair")])
def test_bad_frequencies(kw, match):
    with pytest.raises(ValueError, match=match):
        ops.rotary_frequencies(**kw)


@pytest.mark.parametrize("args,kw,match", [
    ((0,), {}, "heads of 0"), ((65,), {}, "heads of 65"), ((2048,), {}, "heads of 2048"),
    ((64,), dict(dim=66), "66 rotated"), ((64,), dict(dim=5), "5 rotated"),
    ((64,), dict(frequencies=[1.0]), "1 frequencies for 32"),
    ((4,), dict(frequencies=[1.0, math.inf]), "finite"),
    ((64,), dict(amplitude=math.nan), "finite"), ((64,), dict(device="cpu"), "HIP")])
def test_bad_rotary_positions(args, kw, match):
    with pytest.raises(ValueError, match=match):
        ops.Rotary(*args, **kw)


def test_caches_on_the_host_are_refused():
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device"):
        ops.PagedCache(pages, pages.clone())


def plan():
    """(plan, its bytes) of one sequence of 20 tokens, 2 of them new, in blocks 1 and 2."""
    lib = _lib.load()
    n = ctypes.c_int64()
    ids = lambda *x: (ctypes.c_int64 * len(x))(*x)     # noqa: E731
    args = (1, ids(0, 2), ids(1, 2), ids(20), ids(2), 4, 16, 2, 4, 0, 0, 0, 0, 0, 0)
    assert lib.aegkv_batch_plan(*args, None, ctypes.byref(n)) == 0
    room = ctypes.create_string_buffer(n.value + 16)
    at = (ctypes.addressof(room) + 15) & ~15
    assert lib.aegkv_batch_plan(*args, at, ctypes.byref(n)) == 0
    return room, at


def test_c_calls_check_before_they_launch():
    """Every address here is the host's: a call that got past its checks would say so by
    another error than the one expected."""
    lib = _lib.load()
    keep, host = plan()
    memory = ctypes.create_string_buffer(1 << 16)
    here = (ctypes.addressof(memory) + 15) & ~15
    page = 16 * 2 * 64 * 2

    def cache(**kw):
        c = _lib.PagedCacheArgs(here, here, page, page, 4, 16, 2, 64, _lib.DTYPE_BFLOAT16, 0, 0)
        for key, value in kw.items():
            setattr(c, key, value)
        return ctypes.byref(c)

    def rows(tokens=2, heads=4, dtype=_lib.DTYPE_BFLOAT16):
        return ctypes.byref(_lib.Rows(here, tokens, heads * 64, 64, heads, dtype))

    turn = ctypes.byref(_lib.RotaryArgs(here, 64, 0, 1.0))

    def says(rc, text):
        assert rc < 0
        assert text in lib.aegkv_last_error().decode(), lib.aegkv_last_error()

    def attend(plan_=host, device_plan=here, c=None):
        return lib.aegkv_paged_attend(plan_, device_plan, c or cache(), rows(), rows(), None, 0,
                                      0, 0.1, None, 0, None)

    says(lib.aegkv_paged_attend(host, here, None, rows(), rows(), None, 0, 0, 0.1, None, 0, None),
         "cache must not be null")
    says(attend(plan_=None), "plan must not be null")
    says(attend(plan_=here), "no plan")
    says(attend(device_plan=None), "device copy")
    says(attend(device_plan=here + 8), "device copy")
    says(attend(), "not HIP device memory")
    says(lib.aegkv_rotate(None, here, 2, 8, 64, rows(), rows(), None, None, None), "not be null")
    says(lib.aegkv_rotate(turn, here, 2, 8, 64, rows(), rows(), rows(), None, None),
         "not be null")
    says(lib.aegkv_rotate(turn, here, 2, 8, 63, rows(), rows(), None, None, None), "heads of 63")
    says(lib.aegkv_rotate(turn, here, 2, 8, 32, rows(), rows(), None, None, None),
         "64 rotated values")
    says(lib.aegkv_rotate(turn, here, 2, 8, 64, rows(tokens=-1), rows(), None, None, None),
         "-1 tokens")
    says(lib.aegkv_rotate(ctypes.byref(_lib.RotaryArgs(None, 64, 0, 1.0)), here, 2, 8, 64, rows(),
                          rows(), None, None, None), "turns")
    says(lib.aegkv_rotate(turn, here, 2, 8, 64, rows(), rows(), None, None, None),
         "not HIP device memory")
    del keep

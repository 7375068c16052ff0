"""Quantised caches without a GPU: page sizes, the checks of a batch, and the
64-bit reference the GPU tests go by."""

import ctypes
import shutil
import subprocess
import types
from pathlib import Path

import numpy as np
import pytest
import torch

import quant_reference as ref
from aegaeon_amd import _lib, ops
from aegaeon_amd.layout import make_composite_layout, quant_kv_tensor_specs


REPO = Path(__file__).resolve().parent.parent


def plan(tables, lens, new, *, num_blocks=64, block_size=16, kv_heads=2, heads=4, window=0,
         sinks=0, room=(0, 0, 0), update=None):
    """aegkv_batch_plan's buffer (ValueError where it refuses)."""
    lib = _lib.load()
    offsets = np.zeros(len(tables) + 1, np.int64)
    np.cumsum([len(t) for t in tables], out=offsets[1:])
    ids = np.array([i for t in tables for i in t], np.int64)
    lens, new = np.array(lens, np.int64), np.array(new, np.int64)
    p64 = ctypes.POINTER(ctypes.c_int64)
    args = (len(lens), *(a.ctypes.data_as(p64) for a in (offsets, ids, lens, new)), num_blocks,
            block_size, kv_heads, heads, window, sinks, *room, 0 if update is None else 1)
    if update is not None:
        n = ctypes.c_int64(update.size)
        _lib.check(lib.aegkv_batch_plan(*args, update.ctypes.data, ctypes.byref(n)))
        return update
    n = ctypes.c_int64()
    _lib.check(lib.aegkv_batch_plan(*args, None, ctypes.byref(n)))
    buf = np.zeros(n.value, np.uint8)
    _lib.check(lib.aegkv_batch_plan(*args, buf.ctypes.data, ctypes.byref(n)))
    return buf


def test_page_bytes(aegkv_lib):
    assert ops.quant_page_bytes("mxfp4", 16, 8, 128) == 8 * 16 * (64 + 4)
    assert ops.quant_page_bytes("mxfp8", 64, 3, 64) == 3 * 64 * (64 + 2)
    assert ops.quant_page_bytes("mxfp8", 128, 1, 256) == 128 * (256 + 8)
    for bad in (("int4", 16, 8, 128), ("mxfp4", 24, 8, 128), ("mxfp4", 16, 0, 128),
                ("mxfp4", 16, 8, 96), ("mxfp4", 256, 8, 128)):
        with pytest.raises(ValueError):
            ops.quant_page_bytes(*bad)


def test_quantised_caches_are_segments_of_a_composite_page(aegkv_lib):
    specs = quant_kv_tensor_specs(3, 10, 16, 4, 128, "mxfp8")
    segments, page = make_composite_layout(specs, 10)
    assert [s.layer_name for s in segments][:3] == ["layers.0.k", "layers.0.v", "layers.1.k"]
    assert page == 6 * 4 * 16 * (128 + 4)


@pytest.mark.parametrize("match,args,kw", [
    ("outside", ([[0]], [-1], [0]), {}),
    ("new tokens of", ([[0]], [3], [4]), {}),
    ("new tokens of", ([[0]], [3], [-1]), {}),
    ("blocks of 16", ([[0]], [17], [1]), {}),
    ("block id 64", ([[64]], [3], [1]), {}),
    ("block id -2", ([[-2]], [3], [1]), {}),
    ("released", ([[-1, 0]], [20], [1]), {}),
    ("released", ([[0, -1, 2]], [40], [1]), {"window": 20}),
    ("released", ([[-1, -1, 2]], [40], [1]), {"window": 4, "sinks": 1}),
    ("written twice", ([[0], [0]], [3, 3], [1, 1]), {}),
    ("written twice", ([[1, 0], [2, 0]], [20, 24], [4, 8]), {}),
    ("written twice", ([[0, 0]], [32], [32]), {}),
    ("holds 16, 32", ([[0]], [3], [1]), {"block_size": 48}),
    ("KV heads", ([[0]], [3], [1]), {"heads": 3}),
    ("KV heads", ([[0]], [3], [1]), {"kv_heads": 0}),
    ("outside", ([[0]], [3], [1]), {"num_blocks": 0}),
    ("negative", ([[0]], [3], [1]), {"window": -1}),
    ("negative", ([[0]], [3], [1]), {"sinks": -1}),
    ("room", ([[0]], [3], [1]), {"room": (-1, 0, 0)}),
])
def test_batches_that_are_refused(aegkv_lib, match, args, kw):
    with pytest.raises(ValueError, match=match):
        plan(*args, **kw)


def test_batches_that_are_taken(aegkv_lib):
    plan([], [], [])
    plan([[0], [0]], [3, 3], [0, 0])                     # a shared block that is read
    plan([[1, 0], [2, 0]], [20, 24], [4, 4])             # one block, written apart
    plan([[-1, -1, 2]], [40], [1], window=8)
    plan([[5, -1, 2]], [40], [1], window=4, sinks=16)
    plan([[3, 99, 1]], [10], [1], num_blocks=100)        # columns behind the last


def test_updates_keep_the_plan_they_cannot_change(aegkv_lib):
    room = (4, 20, 4)
    buf = plan([[0]], [3], [1], room=room)
    was = buf.copy()
    for match, args, kw in (("do not fit", ([[0]] * 5, [1] * 5, [0] * 5), {}),
                            ("do not fit", ([list(range(40))], [640], [1]), {}),
                            ("no room", ([[0, 1]], [30], [4]), {"heads": 16}),
                            ("keeps", ([[0]], [3], [1]), {"window": 3}),
                            ("block id", ([[99]], [3], [1]), {})):
        kw = {"heads": 16, **kw} if match == "no room" else kw
        target = plan([[0]], [3], [1], room=room, heads=16) if match == "no room" else buf
        before = target.copy()
        with pytest.raises(ValueError, match=match):
            plan(*args, update=target, **kw)
        assert np.array_equal(target, before)
    plan([[7, 8], [3]], [20, 1], [1, 1], update=buf)
    assert not np.array_equal(buf, was)
    plan([[0]], [3], [1], update=buf)
    with pytest.raises(ValueError, match="no plan"):
        plan([[0]], [3], [1], update=np.zeros(buf.size, np.uint8))


def test_calls_without_a_plan_are_refused(aegkv_lib):
    n = ctypes.c_int64()
    lib = _lib.load()
    buf = plan([[0]], [3], [1])
    assert lib.aegkv_quant_attend_workspace(buf.ctypes.data, 128, ctypes.byref(n)) == 0
    assert n.value == 0                                   # one short sequence is not cut
    assert lib.aegkv_quant_attend_workspace(buf.ctypes.data, 100, ctypes.byref(n)) == _lib.EINVAL
    zero = np.zeros(4096, np.uint8)
    assert lib.aegkv_quant_attend_workspace(zero.ctypes.data, 128,
                                            ctypes.byref(n)) == _lib.EINVAL
    assert lib.aegkv_quant_attend_workspace(None, 128, ctypes.byref(n)) == _lib.EINVAL
    for fmt, d, p, dev in ((1, 128, None, 16), (1, 128, zero.ctypes.data, 16),
                           (3, 128, buf.ctypes.data, 16), (1, 96, buf.ctypes.data, 16),
                           (1, 128, buf.ctypes.data, None), (1, 128, buf.ctypes.data, 8)):
        rc = lib.aegkv_quant_write(p, dev, fmt, d, 16, 16, 16, 1, 1, 16, 1, 1, 1, 1, None)
        assert rc == _lib.EINVAL
        rc = lib.aegkv_quant_read(p, dev, fmt, d, 16, 16, 0, 16, 1, 1, 16, 1, 1, 1, 1, None)
        assert rc == _lib.EINVAL
        rc = lib.aegkv_quant_attend(p, dev, fmt, d, 16, 16, 16, 1, 1, 16, 1, 1, 1, 1, 1.0, None,
                                    0, None)
        assert rc == _lib.EINVAL


def test_python_refuses_what_it_cannot_take(aegkv_lib):
    with pytest.raises(ValueError, match="1 lengths"):
        ops.CacheBatch([[0], [1]], [1], [1, 1], num_blocks=4, block_size=16, kv_heads=1)
    with pytest.raises(ValueError, match="2-D"):
        ops.CacheBatch(np.zeros(3, np.int64), [1], [1], num_blocks=4, block_size=16, kv_heads=1)
    with pytest.raises(ValueError, match="integers"):
        ops.CacheBatch([[0.5]], [1], [1], num_blocks=4, block_size=16, kv_heads=1)
    with pytest.raises(ValueError, match="device"):
        ops.CacheBatch([[0]], [1], [1], num_blocks=4, block_size=16, kv_heads=1, device="cpu")
    page = torch.zeros(2, 16 * 68, dtype=torch.uint8)
    with pytest.raises(ValueError, match="device"):
        ops.QuantCache(page, page, kv_heads=1, head_dim=128, block_size=16)


class Recorded:
    """A stream that notes what it is asked for."""

    def __init__(self, raw, closed=False):
        self.cuda_stream, self.closed = raw, closed
        self.waits, self.synchronized = [], 0

    def record_event(self):
        return self

    def wait_event(self, event):
        self.waits.append(event)

    def synchronize(self):
        self.synchronized += 1


def dropped(monkeypatch, pool, home, used=(), capturing=()):
    """Drop a batch made on `pool`, updated to `home`, with calls on `used`."""
    monkeypatch.setattr(ops, "_capturing", lambda st: st in capturing, raising=False)
    monkeypatch.setattr(ops, "_kept", [], raising=False)
    batch = ops.CacheBatch.__new__(ops.CacheBatch)
    batch._plan, batch._pool, batch._home = object(), pool, home
    batch._used = {st.cuda_stream: st for st in used}
    plan = batch._plan
    del batch
    return plan in ops._kept


def test_a_plan_s_memory_goes_back_behind_all_that_read_it(monkeypatch):
    """The memory is the pool's of the stream a batch was made on, also when an
    update has made another one its home."""
    a, b, c = (Recorded(i) for i in range(3))
    assert not dropped(monkeypatch, a, a) and not a.waits
    assert not dropped(monkeypatch, a, b) and a.waits == [b]
    a.waits.clear()
    assert not dropped(monkeypatch, a, b, [c, a]) and a.waits == [b, c] and not b.waits
    a.waits.clear()
    assert not dropped(monkeypatch, a, a, [c]) and a.waits == [c]
    gone = Recorded(7, closed=True)         # its work was waited for
    assert not dropped(monkeypatch, gone, b, [c])
    assert b.synchronized == 1 and c.synchronized == 1
    a.waits.clear()
    assert not dropped(monkeypatch, a, gone, [c]) and a.waits == [c]
    # what cannot be ordered is not given back
    a.waits.clear()
    assert dropped(monkeypatch, a, b, capturing=[b]) and not a.waits
    assert dropped(monkeypatch, a, b, capturing=[a]) and not a.waits
    b.record_event = lambda: 1 / 0
    assert dropped(monkeypatch, a, b)


def test_calls_on_a_closed_stream_s_handle_are_noted(aegkv_lib, monkeypatch):
    """The runtime may give a new stream the handle of one that was destroyed: calls on
    it are not those of the batch's home, which nothing waits for any more."""
    monkeypatch.setattr(ops, "_capturing", lambda st: False)
    home, new = Recorded(5), Recorded(5)
    batch = ops.CacheBatch.__new__(ops.CacheBatch)
    batch._home = batch._pool = home
    batch._stream, batch._used, batch._uploaded = 5, {}, "uploaded"
    assert batch._enter(5, None) is None
    home.closed = True
    for fails in (False, True):     # also those that fail: something may be enqueued
        batch._used = {}
        cache = types.SimpleNamespace(device=torch.device("cuda", 0))
        monkeypatch.setattr(ops, "_call_on", lambda device, fn: fn())
        if fails:
            with pytest.raises(ValueError):
                ops._on_stream(cache, batch, new, lambda raw: _lib.EINVAL)
        else:
            ops._on_stream(cache, batch, new, lambda raw: 0)
        assert batch._used == {5: new} and not new.waits
    taken = []
    native = types.SimpleNamespace(**{op: lambda *a: taken.append(1) for op in
                                      ("quant_write", "quant_read", "quant_attend")})
    monkeypatch.setattr(_lib, "hostargs", lambda: native)
    batch.device = torch.device("cuda", 1)
    batch.block_size = batch.kv_heads = batch.num_blocks = 1
    other = types.SimpleNamespace(block_size=1, kv_heads=1, num_blocks=1,
                                  device=torch.device("cuda", 0))
    x = torch.zeros(1)
    for call in (lambda: ops.quant_write(other, batch, x, x), lambda: ops.quant_read(other, batch),
                 lambda: ops.quant_attend(other, batch, x)):
        with pytest.raises(ValueError, match="a batch on cuda:1"):
            call()
    assert not taken
    batch._home = None      # nothing to order when it goes


def test_streams_of_another_device_are_refused(aegkv_lib):
    stream = types.SimpleNamespace(device=torch.device("cuda", 1))
    args = ([[0]], [1], [1])
    with pytest.raises(ValueError, match="cuda:1 for work on cuda:0"):
        ops.CacheBatch(*args, num_blocks=4, block_size=16, kv_heads=1, device="cuda:0",
                       stream=stream)
    batch = ops.CacheBatch.__new__(ops.CacheBatch)
    batch.device = torch.device("cuda", 0)
    with pytest.raises(ValueError, match="cuda:1 for work on cuda:0"):
        batch.update(*args, stream=stream)
    like = types.SimpleNamespace(block_size=16, kv_heads=1, num_blocks=4, device=batch.device,
                                 heads=1, head_dim=128, read_tokens=1, num_tokens=1)
    x = torch.zeros(1, 1, 128)
    for call in (lambda: ops.quant_write(like, like, x, x, stream=stream),
                 lambda: ops.quant_read(like, like, stream=stream),
                 lambda: ops.quant_attend(like, like, x, stream=stream)):
        with pytest.raises(ValueError, match="cuda:1 for work on cuda:0"):
            call()


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_the_reference_s_own_rounding(fmt):
    """Every code is read as it was written; the largest value of a group is
    never clipped and no value is off by more than half the gap around it."""
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(1)) * 7
    codes, scales = ref.quantise(fmt, x)
    y = ref.values(fmt, codes, scales)
    again = ref.quantise(fmt, y)
    assert torch.equal(ref.values(fmt, *again), y)
    step = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    gap = {"mxfp4": 2, "mxfp8": 32}[fmt] * step
    assert ((x.double() - y).abs() <= gap / 2).all()
    group = x.abs().unflatten(-1, (-1, 32)).amax(-1).double()
    unit = torch.exp2(scales.double() - 127)
    assert (group <= ref.LARGEST[fmt] * unit).all()
    assert (group > ref.LARGEST[fmt] * unit / 2).all()


def test_the_reference_s_formats():
    """Known answers: E2M1 and E4M3 codes against torch's own 8-bit floats."""
    codes = torch.arange(256, dtype=torch.int16).to(torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().view(8, 32)
    got = ref.values("mxfp8", codes.view(8, 32), torch.full((8, 1), 127, dtype=torch.uint8))
    assert torch.equal(got.nan_to_num(nan=1e3), want.nan_to_num(nan=1e3))
    nibbles = torch.arange(32).remainder(16).to(torch.uint8).view(1, 32)
    got = ref.values("mxfp4", nibbles, torch.full((1, 1), 128, dtype=torch.uint8))[0, :16]
    assert got.tolist() == [0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12]


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not installed")
def test_plans_of_random_batches_under_sanitizers(tmp_path):
    """tests/native/batch_plan_check.cpp: what every row sees lies in exactly one
    of its items, inside the plan's room, whatever was updated."""
    exe = tmp_path / "batch_plan_check"
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-Wall",
           "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
           "-D__HIP_PLATFORM_AMD__", f"-I{REPO / 'include'}", "-I/opt/rocm/include",
           f"-I{REPO / 'aegaeon_amd' / 'csrc'}",
           str(REPO / "tests" / "native" / "batch_plan_check.cpp"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "clean" in run.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not installed")
def test_places_that_overlap_under_sanitizers(tmp_path):
    """tests/native/value_places_check.cpp: rows of values share a byte exactly
    where they are said to."""
    exe = tmp_path / "value_places_check"
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-Wall",
           "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
           f"-I{REPO / 'aegaeon_amd' / 'csrc'}",
           str(REPO / "tests" / "native" / "value_places_check.cpp"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "clean" in run.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not installed")
def test_updates_within_the_room_are_taken_under_sanitizers(tmp_path):
    """tests/native/batch_room_check.cpp: whatever batch a plan was made for, also one
    that fills its room."""
    exe = tmp_path / "batch_room_check"
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-Wall",
           "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-Wno-unused-function",
           "-D__HIP_PLATFORM_AMD__", f"-I{REPO / 'include'}", "-I/opt/rocm/include",
           f"-I{REPO / 'aegaeon_amd' / 'csrc'}", f"-I{REPO / 'tests' / 'native'}",
           str(REPO / "tests" / "native" / "batch_room_check.cpp"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "clean" in run.stdout

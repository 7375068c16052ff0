"""Which batches see a block in two places, on the host."""

import ctypes

import numpy as np
import pytest

from aegaeon_amd import _lib


def shared(tables, lens, new, *, window=0, sinks=0, num_blocks=64, block_size=16):
    lib = _lib.load()
    offsets = np.zeros(len(tables) + 1, np.int64)
    np.cumsum([len(t) for t in tables], out=offsets[1:])
    ids = np.array([i for t in tables for i in t], np.int64)
    lens, new = np.array(lens, np.int64), np.array(new, np.int64)
    args = (len(lens), *(a.ctypes.data_as(ctypes.POINTER(ctypes.c_int64))
                         for a in (offsets, ids, lens, new)),
            num_blocks, block_size, 2, 4, window, sinks, 0, 0, 0, 0)
    n = ctypes.c_int64()
    _lib.check(lib.aegkv_batch_plan(*args, None, ctypes.byref(n)))
    plan = np.zeros(n.value, np.uint8)
    _lib.check(lib.aegkv_batch_plan(*args, plan.ctypes.data, ctypes.byref(n)))
    flag = ctypes.c_int32(7)
    _lib.check(lib.aegkv_batch_shared(plan.ctypes.data, ctypes.byref(flag)))
    return flag.value


# (the second time, few columns of very many blocks, which are sorted)
@pytest.mark.parametrize("num_blocks", [64, 1 << 20])
def test_blocks_count_where_queries_see_them(aegkv_lib, num_blocks):
    def is_shared(*args, **kw):
        return shared(*args, num_blocks=num_blocks, **kw)

    assert is_shared([[1, 2], [1, 3]], [20, 30], [1, 1]) == 1
    assert is_shared([[1, 2], [4, 3]], [20, 30], [1, 1]) == 0
    assert is_shared([[1, 1, 2]], [40], [1]) == 1                     # (one sequence's)
    assert is_shared([[1, 2], [1, 3]], [20, 30], [1, 0]) == 0         # one gathers, alone
    assert is_shared([[1, 2], [1, 3]], [20, 30], [0, 0]) == 0
    assert is_shared([[1, 2, 9], [4, 3, 9]], [20, 30], [1, 1]) == 0   # behind their ends
    assert is_shared([], [], []) == 0
    # a window of 8 has left the common prefix, unless the first tokens stay visible
    tables, lens = [[1, 2, 3], [1, 2, 4]], [48, 48]
    assert is_shared(tables, lens, [1, 1], window=8) == 0
    assert is_shared(tables, lens, [1, 1], window=8, sinks=1) == 1
    assert is_shared(tables, lens, [1, 1], window=16) == 0            # positions 32 to 47
    assert is_shared(tables, lens, [1, 1], window=17) == 1            # 31, too
    assert is_shared(tables, lens, [1, 2], window=16) == 0            # one sees it, alone
    assert is_shared(tables, lens, [2, 2], window=16) == 1
    assert is_shared([[1, 2, 3], [2, 5, 4]], lens, [1, 1], window=8, sinks=16) == 0
    assert is_shared([[1, 2, 3], [5, 1, 4]], lens, [1, 1], window=8, sinks=17) == 1
    assert is_shared([[-1, 2, 3], [-1, 5, 4]], lens, [1, 1], window=20) == 0


def test_refusals(aegkv_lib):
    flag = ctypes.c_int32()
    with pytest.raises(ValueError, match="null"):
        _lib.check(aegkv_lib.aegkv_batch_shared(None, ctypes.byref(flag)))
    other = np.zeros(4096, np.uint8)
    with pytest.raises(ValueError, match="no plan"):
        _lib.check(aegkv_lib.aegkv_batch_shared(other.ctypes.data, ctypes.byref(flag)))

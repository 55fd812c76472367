"""What the page calls refuse before they touch a device, and the size limits of their C entry points."""
from __future__ import annotations

import ctypes

import pytest
import torch

from paged_model import Model
from racetrack_b200 import _lib, build as rt_build, layer, ops, paging


@pytest.fixture(scope="module")
def lib():
    rt_build.build()
    return _lib.load()


def _caches():
    return paging.PagedCaches(layer.DSV32, 6, 16, 4, 4, "cpu")


@pytest.mark.parametrize("call", [
    lambda c: c.append((torch.zeros(1, 512).bfloat16(), torch.zeros(1, 64).bfloat16())),
    lambda c: c.extend(1),
    lambda c: c.fork(torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)),
    lambda c: c.free(torch.zeros(1, dtype=torch.int32)),
    lambda c: c.compact(),
    lambda c: ops.page_copy(c.buffers, torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)),
    lambda c: ops.page_write(c.buffers, c.buffers, torch.zeros(1, dtype=torch.int32)),
])
def test_cpu_tensors_are_refused(call):
    c = _caches()
    with pytest.raises(RuntimeError, match="CUDA"):
        call(c)
    assert (c.block_table == -1).all()


@pytest.mark.parametrize("page", [0, 8, 24, 100, -16])
def test_page_sizes(page):
    with pytest.raises(RuntimeError, match="power of two"):
        paging.PagedCaches(layer.DSV32, 6, page, 4, 4, "cpu")


def test_c_entry_points_check_shapes_before_any_launch(lib):
    buf = ctypes.create_string_buffer(256)
    p = ctypes.addressof(buf) // 16 * 16 + 16
    one = lambda v: (ctypes.c_int64 * 1)(v)
    base = (ctypes.c_void_p * 1)(p)

    def extend(seqs=4, width=4, pages=8, page=16, n=1, tokens=1, stride=4, table=p, offsets=None):
        return lib.rt_page_extend(table, stride, p, p, p, p, offsets, p, p, seqs, width, pages, page, n, tokens, None)
    assert extend(seqs=40000) == -2 and b"at most 32768" in lib.rt_last_error()
    assert extend(pages=1 << 28, page=16) == -2 and b"31 bits" in lib.rt_last_error()
    assert extend(width=5) == -1 and b"overlap" in lib.rt_last_error()
    assert extend(table=None) == -1 and b"null" in lib.rt_last_error()
    assert extend(tokens=2) == -1 and b"one token" in lib.rt_last_error()
    assert extend(page=0) == -1 and extend(n=-1, tokens=-1) == -1
    assert extend(n=0, tokens=0) == 0

    def append(rows=base, row_stride=64, row=64, seqs=4, n=1, tokens=1, n_buffers=1, stride=64 * 16, slots=p):
        return lib.rt_page_append(base, one(stride), one(row), rows, one(row_stride), n_buffers, p, 4, p, p, p, p, None, slots,
                                  p, seqs, 4, 8, 16, n, tokens, None)
    assert append(seqs=40000) == -2 and append(slots=None) == -1 and append(tokens=3) == -1
    assert append(rows=(ctypes.c_void_p * 1)(p + 2)) == -1 and b"4-byte aligned" in lib.rt_last_error()
    assert append(rows=None) == -1 and append(row_stride=-64) == -1 and append(row_stride=6) == -1
    assert append(row=6) == -1 and append(stride=8) == -1 and append(n_buffers=-1) == -2
    assert append(seqs=4, n=1, tokens=1, rows=(ctypes.c_void_p * 1)(None)) == -1
    assert append(n=0, tokens=0) == 0

    def copy(base_ptr=base, stride=64 * 16, row=64, n_buffers=1, page=16):
        return lib.rt_page_copy(base_ptr, one(stride), one(row), n_buffers, p, p, 1, 8, page, None)
    assert copy(row=6) == -1 and b"multiples of 4" in lib.rt_last_error()
    assert copy(stride=64 * 15) == -1                      # pages that overlap
    assert copy(stride=64 * 16 + 8) == -1
    assert copy(base_ptr=(ctypes.c_void_p * 1)(p + 4)) == -1 and b"aligned" in lib.rt_last_error()
    assert copy(n_buffers=129) == -2 and b"at most 128" in lib.rt_last_error()
    assert lib.rt_page_copy(base, one(1024), one(64), 1, None, None, 0, 8, 16, None) == 0
    assert lib.rt_page_fork(base, one(1024), one(64), 1, p, 4, p, p, p, p, p, p + 4, 4, 4, 8, 16, 1, None) == -1
    assert lib.rt_page_free(p, 4, p, p, None, 4, 4, 8, 1, None) == -1
    assert lib.rt_page_compact(base, one(1024), one(64), 1, p, 4, p, None, 4, 4, 8, 16, None) == -1


def test_the_model_keeps_its_own_counts():
    """The restatement that the GPU tests compare with, on a case worked by hand."""
    m = Model([torch.zeros(6, 4, 1)], 6, 4, 3, 3)
    assert m.extend([1, 0], [5, 4]) == [0, 1, 2, 3, 4, 8, 9, 10, 11]
    m.write([torch.arange(1, 10).float().view(9, 1)], [0, 1, 2, 3, 4, 8, 9, 10, 11])
    m.fork([1], [2])
    assert m.table == [[2, -1, -1], [0, 1, -1], [0, 3, -1]] and m.refs == [2, 1, 1, 1, 0, 0]
    assert m.rows_of(2, 0).view(-1).tolist() == [1, 2, 3, 4, 5]
    m.free([0, 1])
    assert m.refs == [1, 0, 0, 1, 0, 0]
    assert m.compact() == (2, 1) and m.table[2] == [0, 1, -1]
    assert m.rows_of(2, 0).view(-1).tolist() == [1, 2, 3, 4, 5]
    m.assert_consistent()

"""Bounds of the operators around the experts' GEMMs that lie where a product or a sum leaves 32 bits, on the CPU."""
import ctypes

import pytest
import torch

from deepgemm_b200 import _lib, build
from deepgemm_b200.permute import _check_rows

P, NULL = ctypes.c_void_p(4096), None


@pytest.fixture(scope='module')
def lib():
    build.build()
    return _lib.lib()


def refused(lib, rc, fragment):
    assert rc == 1 and fragment in lib.dgb200_last_error().decode(), (rc, lib.dgb200_last_error())


def chunks_of(lib, entries):
    """(chunks, entries of a chunk) that the sort takes, from the workspace's one word per chunk and expert."""
    chunks = lib.dgb200_moe_dispatch_plan_workspace_bytes(entries, 1, 1) // 4
    return chunks, -(-entries // (1024 * 128)) * 1024


def test_no_chunk_of_the_sort_ends_past_32_bits(lib):
    """The kernels form a chunk's end in 32 bits. What is not refused must keep the last one below 2^31; the first size past the bound is where
    it would be 2^31 itself."""
    bound = 0x7ffe0000
    for entries in (bound, bound - 1, bound - 131072):
        chunks, entries_of = chunks_of(lib, entries)
        assert chunks == -(-entries // entries_of) <= 128 and chunks * entries_of < 2 ** 31
    for entries in (bound + 1, bound + 4096, 0x7fffefff, 0x7ffff000):
        chunks, entries_of = chunks_of(lib, entries)
        assert chunks * entries_of == 2 ** 31
        refused(lib, lib.dgb200_moe_dispatch_plan(P, entries, 1, 1, 1, P, P, P, P, NULL), 'too many entries')
    refused(lib, lib.dgb200_moe_dispatch_plan(P, 0x7ffe0000 // 8 + 1, 8, 256, 1, P, P, P, P, NULL), 'too many entries')


@pytest.mark.parametrize('shape', [(2 ** 31, 1), (1, 2 ** 31), (1, 2 ** 31 + 5)])
def test_rows_and_columns_beyond_32_bits(monkeypatch, shape):
    """Tensors of unit inner stride, so that nothing but their size can be refused."""
    large, largest = torch.empty(shape, device='meta'), torch.empty(tuple(min(n, 2 ** 31 - 1) for n in shape), device='meta')
    monkeypatch.setattr(torch.Tensor, 'is_cuda', True)
    with pytest.raises(RuntimeError, match='x is too large'):
        _check_rows(large, None, None, (torch.float32,), 'x')
    _check_rows(largest, None, None, (torch.float32,), 'x')

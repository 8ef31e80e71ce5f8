"""Paged cache and sampler: what is refused before a device is needed."""
import ctypes

import pytest
import torch

import tattletale_b200 as ttq
from tattletale_b200 import _lib


def test_null_handles():
    lib = _lib.load()
    h = ctypes.c_void_p()
    assert lib.ttq_paged_create(None, 0, 8, 2, 128, 16, 1, 1, 0, ctypes.byref(h)) == 1
    assert lib.ttq_paged_destroy(None) == 0
    kv, batch, s = _lib.KvPages(), _lib.PagedBatchArgs(), _lib.Sampling()
    assert lib.ttq_paged_append(None, None, ctypes.byref(kv), ctypes.byref(batch), None, 0, None, None, 0.0, None, None, 2, 0, None, 0, None) == 1
    assert lib.ttq_paged_attention(None, None, ctypes.byref(kv), ctypes.byref(batch), None, 0, 1.0, 0, 0, None, 0, None) == 1
    assert lib.ttq_sample(None, None, 2, 1, 1, 1, ctypes.byref(s), None, None, None) == 1


def test_batch_checks_its_tensors():
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ttq.TtqError):
        ttq.PagedBatch(i32, i32[:2], i32.view(1, 3))  # host tensors
    with pytest.raises(ttq.TtqError):
        ttq.PagedBatch(i32.long(), i32[:2], i32.view(1, 3))


def test_structures_match_the_header():
    """Field order and sizes of the structures that cross the C ABI."""
    assert ctypes.sizeof(_lib.KvPages) == 48 and ctypes.sizeof(_lib.PagedBatchArgs) == 80 and ctypes.sizeof(_lib.Sampling) == 48
    assert _lib.PagedBatchArgs.prefix_table_dev.offset == 72 and _lib.Sampling.top_k.offset == 44

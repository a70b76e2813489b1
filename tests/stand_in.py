"""Tensors that are nowhere: what the paged cache's objects ask of a tensor, for tests of their checks without a GPU (or with one of several)."""
import types

import torch


def tensor(shape, dtype, device=0, at=1 << 20):
    """A contiguous tensor on a CUDA device; whatever is made with it may be checked, never run."""
    strides, n = [], 1
    for x in reversed(shape):
        strides.insert(0, n)
        n *= x
    t = types.SimpleNamespace(shape=torch.Size(shape), dtype=dtype, is_cuda=True, nbytes=n * dtype.itemsize)
    t.dim, t.stride = lambda: len(shape), lambda i=None: tuple(strides) if i is None else strides[i]
    t.get_device, t.data_ptr, t.is_contiguous = lambda: device, lambda: at, lambda: True
    return t


def pages(l2, device=0, n_pages=4, page=16, heads=2):
    k = tensor((n_pages, page, heads, 128), torch.float16, device)
    return l2.KvPages(k, k)


def batch(l2, device=0, n_seqs=2, width=3, rows=5, most=4):
    i32 = torch.int32
    return l2.KvBatch(tensor((n_seqs, width), i32, device), tensor((n_seqs,), i32, device), tensor((n_seqs + 1,), i32, device), rows, most)

"""Which layouts of a cache paged_write takes, on the CPU: none whose rows lie on one
another, as different tokens' rows would be written into the same memory."""

import ctypes
import itertools

import pytest
import torch

from kotodama_amd import _capi, paged

FAKE = 0x7F0000000000  # never dereferenced: argument checks run first


def _write(shape, strides):
    """The C entry's answer to a cache of these strides, for more tokens than a launch has threads: a call whose
    strides it takes ends there, before the GPU."""
    pages, hk, page, d = shape
    st = (ctypes.c_int64 * 3)(*strides)
    kst = (ctypes.c_int64 * 2)(hk * d, d)
    return _capi.lib().attnres_paged_write(FAKE, kst, FAKE, kst, 1 << 30, hk, d, _capi.DTYPE_BF16, FAKE, st, FAKE, st,
                                           pages, page, FAKE, 0, None)


def _view(shape, strides):
    n = 1 + sum((s - 1) * st for s, st in zip(shape, (*strides, 1)))
    return torch.zeros(n, dtype=torch.bfloat16).as_strided(shape, (*strides, 1))


OVER = [
    ((3, 2, 16, 64), (0, 1024, 64)),
    ((3, 2, 16, 64), (2048, 0, 64)),
    ((3, 2, 16, 64), (2048, 1024, 0)),
    ((3, 2, 16, 64), (1024, 1024, 64)),  # a page stride shorter than a page
    ((3, 2, 16, 64), (2040, 1024, 64)),
    ((3, 2, 16, 64), (2048, 1024, 56)),  # rows into the next
    ((3, 2, 16, 64), (2048, 512, 64)),  # heads into one another
    ((2, 4, 16, 8), (256, 128, 8)),
    ((3, 2, 16, 64), (2048, 64, 64)),
]
APART = [
    ((3, 2, 16, 64), (2048, 1024, 64)),
    ((3, 2, 16, 64), (2048, 64, 128)),  # tokens outside heads
    ((3, 2, 16, 64), (4096, 64, 256)),  # keys and values side by side
    ((5, 2, 16, 64), (1024, 5120, 64)),  # heads outside pages
    ((3, 2, 16, 64), (2304, 1152, 72)),
    ((1, 2, 16, 64), (0, 1024, 64)),  # one page: no other lies on it
    ((3, 1, 16, 64), (1024, 0, 64)),
    ((1, 1, 16, 64), (8, 8, 64)),
]


@pytest.mark.parametrize("shape,strides", OVER)
def test_rows_on_one_another_are_refused(shape, strides):
    assert _write(shape, strides) == _capi.ERR_ARG
    cache = _view(shape, strides)
    with pytest.raises(ValueError, match="on one another"):
        paged._check_cache_memory("paged_write", cache, cache, written=True)
    good = torch.zeros(shape, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="v_cache lie on one another"):
        paged._check_cache_memory("paged_write", good, cache, written=True)
    paged._check_cache_memory("paged_attention", cache, cache)  # reading them is no harm


@pytest.mark.parametrize("shape,strides", APART)
def test_rows_apart_are_taken(shape, strides):
    assert _write(shape, strides) == _capi.ERR_UNSUPPORTED
    cache = _view(shape, strides)
    paged._check_cache_memory("paged_write", cache, cache, written=True)


def test_one_page_has_no_page_stride():
    # as the C entry has it: how far apart pages lie matters where there are two
    far = torch.zeros(2048, dtype=torch.bfloat16).as_strided((1, 2, 16, 64), (1 << 31, 1024, 64, 1))
    paged._check_cache_memory("paged_attention", far, far)
    paged._check_cache_memory("paged_write", far, far, written=True)
    two = torch.empty((0,), dtype=torch.bfloat16).as_strided((0, 2, 16, 64), (1 << 31, 1024, 64, 1))
    paged._check_cache_memory("paged_write", two, two, written=True)
    far = torch.empty(1, dtype=torch.bfloat16, device="meta").as_strided((2, 2, 16, 64), (1 << 31, 1024, 64, 1))
    with pytest.raises(ValueError, match="so far apart"):
        paged._check_cache_memory("paged_attention", far, far)


def test_against_every_element():
    # what is taken has no two elements in one place
    for shape in ((2, 2, 16, 8), (3, 1, 16, 8), (2, 3, 16, 8)):
        for strides in itertools.product((8, 16, 24, 128, 136, 256, 384), repeat=3):
            cache = _view(shape, strides)
            if not paged._rows_apart(cache):
                continue
            at = sum(torch.arange(n).reshape([-1 if i == j else 1 for j in range(4)]) * st
                     for i, (n, st) in enumerate(zip(shape, cache.stride())))
            assert at.flatten().unique().numel() == cache.numel(), (shape, strides)

"""Page-locked buffers of the output pool (``_hostpool``) without a GPU: a library that hands them out, and one that has none."""

from __future__ import annotations

import ctypes
import gc

import numpy as np
import pytest

from neo_ls_svm_amd import _hostpool as pool

N = 2900  # N^2 doubles: 67 MB


class Library:
    """nls_host_alloc / nls_host_free on ordinary memory; memory that exists already is not to be page-locked."""

    def __init__(self, rc=0):
        self.rc, self.held = rc, {}

    def nls_host_alloc(self, handle, size, out):
        if self.rc == 0:
            memory = (ctypes.c_char * size.value)()
            address = ctypes.addressof(memory)
            self.held[address] = memory
            ctypes.cast(out, ctypes.POINTER(ctypes.c_void_p))[0] = address
        return self.rc

    def nls_host_free(self, handle, p):
        del self.held[p.value]
        return 0

    def nls_host_register(self, handle, p, size):
        return 2


class Context:
    handle = 1

    def __init__(self, rc=0):
        self.lib = Library(rc)


@pytest.fixture(autouse=True)
def clean():
    pool.release()
    yield
    pool.pin_large_outputs(False)
    gc.collect()
    pool.release()
    assert not pool._registered and pool._pooled_bytes() == 0


def output(ctx):
    return pool.factor_output((N, N), np.float64, ctx)


def test_page_locked_buffers_are_allocated_recycled_and_released():
    ctx = Context()
    pool.pin_large_outputs(True)
    a = output(ctx)
    address = a.__array_interface__["data"][0]
    assert type(a.base).__name__ == "_Lease" and len(pool._registered) == len(ctx.lib.held) == 1
    a[:] = 5.0
    view = a[3:5]
    del a
    gc.collect()
    assert pool._pooled_bytes() == 0 and view[0, 0] == 5.0  # (the view keeps the buffer)
    del view
    gc.collect()
    pool.pin_large_outputs(False)
    b = output(ctx)
    assert b.__array_interface__["data"][0] == address and len(ctx.lib.held) == 1
    del b
    gc.collect()
    pool.release()
    assert not ctx.lib.held and not pool._registered


def test_reuse_puts_a_page_locked_buffer_in_the_place_of_a_pageable_one():
    ctx = Context()
    pool.pin_large_outputs("reuse")
    a = output(ctx)
    assert not pool._registered
    del a
    gc.collect()
    b = output(ctx)
    assert len(pool._registered) == len(ctx.lib.held) == 1 and pool._pooled_bytes() == 0
    b[:] = 1.0
    address = b.__array_interface__["data"][0]
    del b
    gc.collect()
    c = output(ctx)
    assert c.__array_interface__["data"][0] == address and len(ctx.lib.held) == 1
    del c


@pytest.mark.parametrize("policy", [True, "reuse"])
def test_where_there_are_none_buffers_are_pageable(policy):
    ctx = Context(rc=2)
    pool.pin_large_outputs(policy)
    for _ in range(3):
        a = output(ctx)
        assert type(a.base).__name__ == "_Lease" and not pool._registered
        a[:] = 2.0
        del a
        gc.collect()
    assert pool.LAST_REGISTER_RC == 2


def test_reserved_buffers():
    ctx = Context()
    assert pool.reserve((N, N), np.float64, ctx, 2) == 2 and pool.reserve((N, N), np.float64, ctx, 1) == 0
    assert len(ctx.lib.held) == len(pool._registered) == 2 and pool._pooled_bytes() == 2 * N * N * 8
    a, b, c = output(ctx), output(ctx), output(ctx)
    assert len(ctx.lib.held) == 2 and len({x.__array_interface__["data"][0] for x in (a, b, c)}) == 3
    del a, b, c
    gc.collect()
    pool.release()
    assert not ctx.lib.held
    assert pool.reserve((N, N), np.float64, Context(rc=2), 1) == 1 and not pool._registered

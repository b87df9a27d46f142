"""CPU checks of the few-bit matrix operators: refusals before anything reaches a GPU, and the arithmetic the kernels rely on."""

from __future__ import annotations

import shutil
import subprocess
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest

import neo_ls_svm_amd as nls

X = np.ones((3, 32), dtype=np.float32)
Q = np.ones((3, 32), dtype=np.int8)
S = np.ones(3, dtype=np.float32)


@pytest.mark.parametrize(
    "call",
    [
        lambda: nls.quantize_rows(X.astype(np.float64)),
        lambda: nls.quantize_rows(X.astype(np.int32)),
        lambda: nls.quantize_rows(np.float32(1.0)),
        lambda: nls.quantize_rows([[1.0, 2.0]]),
        lambda: nls.quantize_rows(np.empty((3, 0), dtype=np.float32)),
        lambda: nls.int8_matmul(X, S, Q, S),
        lambda: nls.int8_matmul(Q, S, Q.astype(np.uint8), S),
        lambda: nls.int8_matmul(Q, S, Q[:, :16], S),
        lambda: nls.int8_matmul(Q, S[:2], Q, S),
        lambda: nls.int8_matmul(Q, S, Q, S[:2]),
        lambda: nls.int8_matmul(Q, S.astype(np.float64), Q, S),
        lambda: nls.int8_matmul(Q, S, Q[None], S[None]),
        lambda: nls.int8_matmul(Q, S, Q, S, bias=S[:2]),
        lambda: nls.int8_matmul(Q, S, Q, S, bias=S.astype(np.float16)),
        lambda: nls.int8_matmul(Q, S, Q, S, dtype="float64"),
        lambda: nls.int8_matmul(Q, S, Q, S, dtype="bfloat16"),
        lambda: nls.int8_matmul(Q, S, Q, S, dtype="nonsense"),
        lambda: nls.int8_matmul(np.ones((1, 131072), np.int8), S[:1], np.ones((1, 131072), np.int8), S[:1]),
        lambda: nls.int8_matmul(np.ones((1, 0), np.int8), S[:1], np.ones((1, 0), np.int8), S[:1]),
        lambda: nls.int8_linear(X, Q[:, :16], S),
        lambda: nls.int8_linear(X.astype(np.float64), Q, S),
        lambda: nls.int8_linear(X, Q, S, bias=X),
        lambda: nls.orthogonalize(X.astype(np.float64)),
        lambda: nls.orthogonalize(X[0]),
        lambda: nls.orthogonalize(X, steps=0),
        lambda: nls.orthogonalize(X, steps=33),
        lambda: nls.orthogonalize(X, steps=2.5),
        lambda: nls.orthogonalize(X, steps=3, coefficients=[(1.5, -0.5, 0.0)] * 2),
        lambda: nls.orthogonalize(X, coefficients=(1.5, -0.5)),
        lambda: nls.orthogonalize(X, coefficients=(float("nan"), 0.0, 0.0)),
        lambda: nls.orthogonalize(X, eps=-1.0),
        lambda: nls.orthogonalize(X, eps=float("nan")),
    ],
)
def test_refused_before_any_gpu_is_asked_for(call):
    with pytest.raises(ValueError):
        call()


def test_host_tensors_and_mixed_arguments_are_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="GPU"):
        nls.quantize_rows(torch.ones(3, 32))
    with pytest.raises(ValueError, match="like the other"):
        nls.int8_matmul(Q, S, torch.ones(3, 32, dtype=torch.int8), S)


def test_sixty_four_bits_decide_a_quotient_next_to_a_half():
    """127 x / top of two float32 numbers: the 64-bit quotient rounds to the integer the exact one rounds to (the kernel's slow path), and the
    32-bit product x * fl(127 / top) is never further from it than the kernel's window of 2e-5 around a half (its fast path)."""
    rng = np.random.default_rng(0)
    top = rng.uniform(1.0, 2.0, 4000).astype(np.float32)
    j = rng.integers(-127, 127, 4000)
    x = ((2 * j + 1).astype(np.float64) * top.astype(np.float64) / 254.0).astype(np.float32)  # as near to a half as float32 gets
    x = np.concatenate([x, np.nextafter(x, np.float32(9)), np.float32([63.5, 0.5, 1.5, -2.5])])
    top = np.concatenate([top, top, np.float32([127.0] * 4)])
    wide = np.rint(x.astype(np.float64) * 127.0 / top.astype(np.float64))
    fast = x * (np.float32(127.0) / top)
    for xi, ti, wi, fi in zip(x, top, wide, fast):
        r = Fraction(float(xi)) * 127 / Fraction(float(ti))
        assert round(r) == int(wi)  # (Fraction rounds ties to even)
        assert abs(Fraction(float(fi)) - r) < Fraction(2, 100000)


def test_arrays_of_the_other_byte_order_are_turned():
    from neo_ls_svm_amd import lowbit

    other = X.dtype.newbyteorder()
    turned = lowbit._Arrays(X, None).take(X.astype(other), "x")
    assert turned.dtype == np.float32 and turned.dtype.isnative and np.array_equal(turned, X)


@pytest.mark.parametrize("m", [5, 16, 17, 48, 49, 4096])
@pytest.mark.parametrize("n,k,ld,flag", [(64, 64, 64, 0), (9000, 48, 64, 0), (300, 301, 304, 2), (8192, 33, 4096, 2)])
def test_the_room_int8_linear_takes_without_asking_is_enough(m, n, k, ld, flag):
    import ctypes as C

    from neo_ls_svm_amd import _lib

    need = C.c_size_t()
    assert _lib.load_library().nls_int8_linear_workspace(4096, ld, m, n, k, flag, need) == 0
    assert need.value <= (m * ((k + 15) & -16) + 255 & -256) + (4 * m + 255 & -256)


def device_array(shape, dtype):
    a = nls.DeviceArray.__new__(nls.DeviceArray)  # (no GPU is needed to be refused)
    a.ctx, a.shape, a.dtype, a.ptr = None, shape, np.dtype(dtype), None
    a.nbytes = int(np.prod(shape)) * a.dtype.itemsize
    return a


class NoContext:
    def held(self, a):
        return a


@pytest.mark.parametrize("dtype", ["float32", "float16", "int8", "complex128"])
def test_the_64_bit_calls_refuse_device_arrays_of_other_types(dtype):
    """The few-bit operators hand out DeviceArrays of 32, 16 and 8 bits: read as float64 they would be read past their end."""
    n, d, D = 6, 3, 4
    ctx, x, y = NoContext(), device_array((n, d), dtype), np.ones(n)
    good, shift, scale, B = device_array((n, d), "float64"), np.zeros(d), np.ones(d), np.ones((d, D))
    for call in (
        lambda: nls.featuremap(x, shift, scale, B, ctx=ctx),
        lambda: nls.gram(x, y, y, shift, scale, B, ctx=ctx),
        lambda: nls.gram(good, device_array((n,), dtype), y, shift, scale, B, ctx=ctx),
        lambda: nls.gram(good, y, device_array((n,), dtype), shift, scale, B, ctx=ctx),
        lambda: nls.rotate(x, shift, scale, B, np.eye(D + 1), np.ones(D + 1), ctx=ctx),
        lambda: nls.primal_fit(x, y, y, shift, scale, B, False, ctx=ctx),
        lambda: nls.primal_predict(x, shift, scale, B, beta=np.ones(D + 1), ctx=ctx),
        lambda: nls.dual_fit(x, y, y, False, ctx=ctx),
        lambda: nls.dual_predict(good, x, alpha=y, ctx=ctx),
        lambda: nls.dual_predict(good, good, L=device_array((n, n), dtype), ctx=ctx),
    ):
        with pytest.raises(ValueError, match="64-bit calls take float64"):
            call()


@pytest.mark.parametrize("out", [((6, 10), "float32"), ((6, 5), "float64"), ((6, 4), "complex128"), ((6, 10), "int8")])
def test_featuremap_refuses_to_write_past_the_end_of_out(out):
    with pytest.raises(ValueError, match="out must hold"):
        nls.featuremap(np.ones((6, 3)), np.zeros(3), np.ones(3), np.ones((3, 4)), ctx=NoContext(), out=device_array(*out))


def test_launches_of_many_workgroups(tmp_path):
    """csrc/nls_tile.h compiled for the host: a kernel of 1024 threads used to get 2^32 threads along x from 2^22 workgroups on."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc not available")
    root, exe = Path(__file__).resolve().parent.parent, tmp_path / "test_grid"
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-I", str(root / "neo_ls_svm_amd" / "csrc"), str(root / "tests" / "csrc" / "test_grid.cpp"), "-o", str(exe)], check=True)  # fmt: skip
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_forward_mode_derivatives_are_refused_not_lost():
    """A dual tensor asks for no gradients, has memory like any other, and its result would have none."""
    torch = pytest.importorskip("torch")
    from neo_ls_svm_amd import lowbit

    sp = lowbit._Tensors(torch, 0, None)
    sp.index = -1  # (tensors of the host pass for the device's)
    x, q, s = torch.ones(3, 32), torch.ones(3, 32, dtype=torch.int8), torch.ones(3)
    assert sp.float_rows(x, "x")[0] is x
    with torch.autograd.forward_ad.dual_level():
        assert sp.float_rows(x, "x")[0] is x and sp.int8_rows(q, "b", s, "b_scale")[0] is q
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        scale = torch.autograd.forward_ad.make_dual(s, torch.ones_like(s))
        for call in (lambda: sp.take(dual, "x"), lambda: sp.float_rows(dual, "x"), lambda: sp.float_rows(dual[:, ::2], "x"), lambda: sp.int8_rows(q, "b", scale, "b_scale"), lambda: lowbit._bias(sp, scale, 3, 0)):  # fmt: skip
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
    assert sp.float_rows(x, "x")[0] is x


@pytest.mark.parametrize("shape", [(2**20 + 1, 1), (1, 2**20 + 1), (65536, 1, 1), (256, 256, 1, 1), (2, 2**20 + 1, 0)])
def test_orthogonalize_refuses_sizes_before_it_makes_room_for_them(shape):
    with pytest.raises(ValueError, match="65535 matrices"):
        nls.orthogonalize(np.zeros(shape, dtype=np.float32))

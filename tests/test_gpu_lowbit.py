"""Few-bit matrix operators on the MI355X against plain 64-bit forms computed on the CPU.

Tolerances: a rounding to a type is off by at most eps / 2 of the value (``HALF``); the float32 part of a product makes three roundings before its last
one, and one in the addition of the bias.  Integers and scales have to be equal.  What Newton-Schulz products do to roundings depends on the matrix: the
oracle itself is run with roundings of the documented sizes put into every product, and the kernel may be off by eight times what that does."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import neo_ls_svm_amd as nls  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
HALF = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}
TINY = {"float32": 2.0**-149, "float16": 2.0**-24, "bfloat16": 2.0**-133}
CUBIC = (1.5, -0.5, 0.0)


def host(t):
    return t.detach().cpu().to(torch.float64).numpy()


def activations(rng, m, k):
    return rng.standard_normal((m, k)) * np.exp(0.5 * rng.standard_normal(k)) * np.exp(0.5 * rng.standard_normal((m, 1)))


# ---- oracles (64 bits) ------------------------------------------------------------------------------------------------------------------------
def quantize_oracle(x):
    top = np.abs(x).max(-1, keepdims=True)
    q = np.where(top > 0, np.rint(x * 127.0 / np.where(top > 0, top, 1.0)), 0.0)
    return q.astype(np.int8), (top[..., 0].astype(np.float32) / np.float32(127))


def product_oracle(a, a_scale, b, b_scale, bias=None):
    s = a.astype(np.float64) @ b.astype(np.float64).T  # (integers below 2^53: exact)
    y = s * a_scale.astype(np.float64)[..., None] * b_scale.astype(np.float64)
    return y, (y if bias is None else y + bias)


def product_check(y, a, a_scale, b, b_scale, bias, name):
    part, want = product_oracle(a, a_scale, b, b_scale, bias)
    off = np.abs(host(y) - want)
    inner = 3 * 2.0**-24 * np.abs(part) + 2.0**-24 * np.abs(want)
    bound = 1.01 * (HALF[name] * (np.abs(want) + inner) + inner) + TINY[name]
    assert np.all(off <= bound), float(np.max(off / bound))


def newton_schulz_oracle(g, coefficients, steps, eps, rng=None, rounding=None):
    """rounding(t): relative size of the random roundings put into the operands of every product of step t."""
    rough = (lambda m, t: m * (1.0 + rounding(t) * rng.uniform(-1, 1, m.shape))) if rng is not None else (lambda m, t: m)
    table = np.broadcast_to(np.asarray(coefficients, dtype=np.float64), (steps, 3))
    tall = g.shape[0] > g.shape[1]
    x = (g.T if tall else g) / (np.linalg.norm(g) + eps)
    for t, (a, b, c) in enumerate(table):
        s = rough(x, t) @ rough(x, t).T
        s = (s + s.T) / 2
        p = b * s + c * (rough(s, t) @ rough(s, t))
        x = a * x + rough(p, t) @ rough(x, t)
        if rounding is not None:
            x = x * (1.0 + 2.0**-22 * rng.uniform(-1, 1, x.shape))
    return x.T if tall else x


def newton_schulz_check(out, g, coefficients, steps, eps, name, seed):
    want = newton_schulz_oracle(g, coefficients, steps, eps)
    exact = {"float32": steps, "float16": 3, "bfloat16": 2}[name]  # the last steps work on 22 bits, the ones before on 11
    rng = np.random.default_rng(seed)
    size = lambda t: 2.0**-21 if t >= steps - exact else 2.0**-12  # noqa: E731
    spread = max(np.linalg.norm(newton_schulz_oracle(g, coefficients, steps, eps, rng, size) - want) for _ in range(3))
    got = host(out)
    assert got.shape == want.shape
    bound = 8 * spread + 2.0**-20 * np.linalg.norm(want) + HALF[name] * np.linalg.norm(want) + TINY[name] * np.sqrt(want.size)
    assert np.linalg.norm(got - want) <= bound, (np.linalg.norm(got - want) / np.linalg.norm(want), bound / np.linalg.norm(want))


# ---- quantise -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 4096), (3, 15), (5, 16), (2, 17), (67, 301), (4, 512), (4, 513), (9, 4099), (2, 40000), (1000, 64)])
def test_quantize_rows(rows, k, name):
    rng = np.random.default_rng(rows * 100003 + k)
    x = torch.tensor(activations(rng, rows, k), dtype=torch.float32).to(DTYPES[name]).cuda()
    q, scale = nls.quantize_rows(x)
    wq, ws = quantize_oracle(host(x))
    assert q.shape == x.shape and q.dtype == torch.int8 and scale.dtype == torch.float32
    assert np.array_equal(q.cpu().numpy(), wq)
    assert np.array_equal(scale.cpu().numpy(), ws)


def test_quantize_ties_zeros_extremes():
    x = np.zeros((9, 20), dtype=np.float32)
    x[0, :6] = [127.0, 0.5, 1.5, -2.5, 63.5, -0.5]  # ties go to even
    x[1] = 0.0
    x[2, 0] = 1e-45  # the smallest number of all
    x[3, :3] = [3e38, -3e38, 1e38]
    x[4, :3] = [1e-38, 5e-39, -2e-39]
    x[5, 3] = np.nan
    x[6, [2, 4]] = [np.inf, 1.0]
    x[7, :2] = [-254.0, 1.0]
    x[8, :2] = [1e-36, 0.5e-36]
    q, scale = (t.cpu().numpy() for t in nls.quantize_rows(torch.tensor(x).cuda()))
    fine = [0, 1, 2, 3, 4, 7, 8]
    wq, ws = quantize_oracle(x[fine].astype(np.float64))
    assert np.array_equal(q[fine], wq) and np.array_equal(scale[fine], ws)
    assert np.isnan(scale[5]) and np.isposinf(scale[6]) and not q[5].any() and not q[6].any()
    b = torch.ones(2, 20, dtype=torch.int8).cuda()
    one = torch.ones(2).cuda()
    y = host(nls.int8_linear(torch.tensor(x).cuda(), b, one))
    assert np.isnan(y[5:7]).all() and np.isfinite(y[fine]).all()


@pytest.mark.parametrize("name", ["float32", "bfloat16"])
def test_quantize_strides(name):
    rng = np.random.default_rng(5)
    base = torch.tensor(rng.standard_normal((130, 200)), dtype=torch.float32).to(DTYPES[name]).cuda()
    views = [base.T, base[::2], base[:, ::3], base[3:, 1:], base[:, :7].T, base[5:6].expand(4, 200), base[:, 5:6].expand(130, 33), base[0], base.view(2, 65, 200)[:, 1:]]
    for x in views:
        q, scale = nls.quantize_rows(x)
        wq, ws = quantize_oracle(host(x))
        assert q.shape == x.shape and scale.shape == x.shape[:-1]
        assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(scale.cpu().numpy(), ws)


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("rows,k,skip", [(2048, 128, 0), (2061, 130, 1), (4096, 257, 0), (2500, 1003, 3), (70000, 129, 0)])
def test_quantize_the_rows_of_a_transposed_matrix(rows, k, skip, name):
    rng = np.random.default_rng(rows + k)
    base = torch.tensor(activations(rng, k, rows + skip), dtype=torch.float32).to(DTYPES[name]).cuda()
    x = base[:, skip:].T
    x[7] = 0
    q, scale = nls.quantize_rows(x)
    want_q, want_scale = quantize_oracle(host(x))
    assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(scale.cpu().numpy(), want_scale)
    held = q.as_strided((rows, q.stride(0)), (q.stride(0), 1))
    assert not held[:, k:].any()
    x[11, k - 1], x[rows - 1, 0] = float("nan"), -float("inf")
    q2, scale2 = nls.quantize_rows(x)
    assert torch.isnan(scale2[11]) and torch.isinf(scale2[rows - 1]) and not q2[11].any() and not q2[rows - 1].any()
    q2[11], q2[rows - 1], scale2[11], scale2[rows - 1] = q[11], q[rows - 1], scale[11], scale[rows - 1]
    assert torch.equal(q2, q) and torch.equal(scale2, scale)


def test_quantize_pads_its_rows_with_zeros():
    q, _ = nls.quantize_rows(torch.ones(3, 21, device="cuda"))
    assert q.stride() == (32, 1)
    held = q.as_strided((3, 32), (32, 1)).cpu().numpy()
    assert (held[:, :21] == 127).all() and (held[:, 21:] == 0).all()


# ---- products -----------------------------------------------------------------------------------------------------------------------------
SIZES = [
    (1, 1, 1), (1, 64, 64), (1, 4096, 4096), (2, 17, 31), (3, 5, 129), (8, 300, 127), (15, 33, 1000), (16, 256, 8192), (17, 64, 128), (31, 100, 255),
    (48, 513, 512), (64, 64, 64), (65, 63, 65), (100, 1000, 300), (128, 128, 128), (130, 129, 131), (300, 4097, 301), (513, 257, 384), (2049, 130, 16),
    (700, 4096, 1024), (1, 3, 20000),
]  # fmt: skip


def eight_bits(rng, rows, k):
    q = rng.integers(-127, 128, (rows, k)).astype(np.int8)
    q[rng.random((rows, k)) < 0.02] = -128
    return q


@pytest.mark.parametrize("tight", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_int8_matmul(m, n, k, tight):
    rng = np.random.default_rng(m * 7 + n * 11 + k)
    a, b = eight_bits(rng, m, k), eight_bits(rng, n, k)
    a_scale, b_scale = rng.uniform(1e-3, 1e-2, m).astype(np.float32), rng.uniform(1e-3, 1e-2, n).astype(np.float32)

    def held(x):
        if tight:
            return torch.tensor(x).cuda()
        room = torch.full((x.shape[0], -(-k // 16) * 16), 77, dtype=torch.int8, device="cuda")  # what lies behind a row does not count
        room[:, :k] = torch.tensor(x).cuda()
        return room[:, :k]

    ta, tb = held(a), held(b)
    for name in DTYPES:
        for bias in (None, rng.standard_normal(n)):
            tbias = None if bias is None else torch.tensor(bias, dtype=torch.float32).to(DTYPES[name]).cuda()
            y = nls.int8_matmul(ta, torch.tensor(a_scale).cuda(), tb, torch.tensor(b_scale).cuda(), bias=tbias, dtype=name)
            assert y.dtype == DTYPES[name] and y.shape == (m, n)
            product_check(y, a, a_scale, b, b_scale, None if bias is None else host(tbias), name)


@pytest.mark.parametrize("m,n,k", [(200, 333, 5001), (1300, 1700, 140), (2300, 2100, 257), (3100, 3100, 700), (3100, 3105, 64), (2500, 4100, 2050)])
def test_int8_matmul_in_every_tile(m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, b = eight_bits(rng, m, k), eight_bits(rng, n, k)
    a_scale, b_scale = rng.uniform(1e-3, 1e-2, m).astype(np.float32), rng.uniform(1e-3, 1e-2, n).astype(np.float32)
    ta, tb, tsa, tsb = (torch.tensor(v).cuda() for v in (a, b, a_scale, b_scale))
    room = torch.full((n, -(-k // 16) * 16 + 16), 99, dtype=torch.int8, device="cuda")
    room[:, :k] = tb
    for name in ("float32", "bfloat16"):
        y = nls.int8_matmul(ta, tsa, tb, tsb, dtype=name)
        product_check(y, a, a_scale, b, b_scale, None, name)
        assert torch.equal(nls.int8_matmul(ta, tsa, room[:, :k], tsb, dtype=name), y)


@pytest.mark.parametrize("m", [2, 4, 16, 33, 48])
@pytest.mark.parametrize("k", [40, 63, 1000, 4097])
def test_few_rows_from_any_address(m, k):
    """Rows of a and b that start anywhere and end where their memory ends."""
    rng = np.random.default_rng(m + k)
    n = 70
    a, b = eight_bits(rng, m, k), eight_bits(rng, n, k)
    a_scale, b_scale = rng.uniform(1e-3, 1e-2, m).astype(np.float32), rng.uniform(1e-3, 1e-2, n).astype(np.float32)
    tsa, tsb = torch.tensor(a_scale).cuda(), torch.tensor(b_scale).cuda()
    x = torch.tensor(activations(rng, m, k), dtype=torch.float32).cuda().half()
    q, scale = quantize_oracle(host(x))
    for off in (0, 1, 7):

        def held(v):
            flat = torch.empty(v.size + off, dtype=torch.int8, device="cuda")
            flat[off:] = torch.tensor(v.ravel()).cuda()
            return flat[off:].view(v.shape)

        product_check(nls.int8_matmul(held(a), tsa, held(b), tsb), a, a_scale, b, b_scale, None, "float32")
        product_check(nls.int8_linear(x, held(b), tsb), q, scale, b, b_scale, None, "float16")


def test_rows_with_a_nan_or_an_infinity_spoil_their_results_only():
    for m, k in ((1, 512), (3, 100), (20, 300), (130, 300)):
        x = torch.randn(m, k, device="cuda", generator=torch.Generator("cuda").manual_seed(m))
        q, s = nls.quantize_rows(torch.randn(90, k, device="cuda", generator=torch.Generator("cuda").manual_seed(k)))
        want = nls.int8_linear(x, q, s)
        for bad in (float("nan"), float("inf"), -float("inf")):
            y = x.clone()
            y[m // 2, k - 1] = bad
            got = nls.int8_linear(y, q, s)
            assert torch.isnan(got[m // 2]).all()
            got[m // 2] = want[m // 2]
            assert torch.equal(got, want)


def test_more_rows_than_one_dimension_of_a_launch_counts():
    rows = 2**26 + 5
    value = torch.arange(rows, device="cuda") % 2001 - 1000
    x = value.half().view(rows, 1)
    q, scale = nls.quantize_rows(x)
    want = torch.tensor(np.arange(1001, dtype=np.float32) / np.float32(127)).cuda()  # (torch divides by a number as a product with its inverse)
    assert torch.equal(q[:, 0].float(), torch.sign(x[:, 0]).float() * 127) and torch.equal(scale, want[value.abs()])
    del q, scale, x, value
    n = 2**27 + 40
    b = (torch.arange(n, device="cuda") % 255 - 127).to(torch.int8).view(n, 1).expand(n, 16).contiguous()
    y = nls.int8_matmul(torch.ones(1, 16, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"), b, torch.ones(n, device="cuda"), dtype="float16")
    assert torch.equal(y[0], (16 * b[:, 0].to(torch.int16)).half())


def test_rows_further_apart_than_the_kernels_count():
    rng = np.random.default_rng(0)
    a, b = eight_bits(rng, 3, 32), eight_bits(rng, 20, 32)
    far = torch.zeros(3, 9_000_000, dtype=torch.int8, device="cuda")
    far[:, :32] = torch.tensor(a).cuda()
    one, many = torch.ones(3, device="cuda"), torch.ones(20, device="cuda")
    product_check(nls.int8_matmul(far[:, :32], one, torch.tensor(b).cuda(), many), a, np.ones(3, np.float32), b, np.ones(20, np.float32), None, "float32")


def test_int8_matmul_sums_to_the_end_of_32_bits():
    k = 131071
    a = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    y = nls.int8_matmul(a, torch.ones(2, device="cuda"), b, torch.ones(3, device="cuda"))
    assert np.array_equal(host(y), np.full((2, 3), float(np.float32(k * 16384))))


def test_int8_matmul_views_and_leading_axes():
    rng = np.random.default_rng(1)
    a, b = eight_bits(rng, 24, 96), eight_bits(rng, 40, 96)
    sa, sb = rng.uniform(0.1, 1, 24).astype(np.float32), rng.uniform(0.1, 1, 40).astype(np.float32)
    ta, tb, tsa, tsb = (torch.tensor(v).cuda() for v in (a, b, sa, sb))
    want = nls.int8_matmul(ta, tsa, tb, tsb)
    product_check(want, a, sa, b, sb, None, "float32")
    wide = torch.zeros(24, 100, dtype=torch.int8, device="cuda")
    wide[:, 3:99] = ta
    double = torch.zeros(80, 96, dtype=torch.int8, device="cuda")
    double[::2] = tb
    for other in (
        nls.int8_matmul(wide[:, 3:99], tsa, tb, tsb),
        nls.int8_matmul(ta, tsa, double[::2], tsb),
        nls.int8_matmul(ta, tsa, tb.T.contiguous().T, tsb),
        nls.int8_matmul(ta.view(2, 3, 4, 96), tsa.view(2, 3, 4), tb, tsb).view(24, 40),
        nls.int8_matmul(ta, torch.stack([tsa, tsa], 1)[:, 0], tb, tsb),
    ):
        assert torch.equal(other, want)
    one = nls.int8_matmul(ta[5], tsa[5], tb, tsb)
    assert one.shape == (40,) and torch.equal(one, want[5])
    same = ta[3:4].expand(24, 96)
    assert torch.equal(nls.int8_matmul(same, tsa[3:4].expand(24), tb, tsb), want[3:4].expand(24, 40))
    assert torch.equal(nls.int8_matmul(same, tsa[3:4].expand(24).contiguous(), tb, tsb), want[3:4].expand(24, 40))
    assert torch.equal(nls.int8_matmul(tb[:0], tsb[:0], tb, tsb), want[:0])


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("m,n,k", SIZES)
def test_int8_linear(m, n, k, name):
    rng = np.random.default_rng(m * 13 + n * 5 + k)
    x = torch.tensor(activations(rng, m, k), dtype=torch.float32).to(DTYPES[name]).cuda()
    b, b_scale = eight_bits(rng, n, k), rng.uniform(1e-3, 1e-2, n).astype(np.float32)
    q, scale = quantize_oracle(host(x))
    for bias in (None, torch.tensor(rng.standard_normal(n), dtype=torch.float32).cuda()):
        y = nls.int8_linear(x, torch.tensor(b).cuda(), torch.tensor(b_scale).cuda(), bias=bias)
        assert y.dtype == x.dtype
        product_check(y, q, scale, b, b_scale, None if bias is None else host(bias), name)


def test_empty_sizes():
    f, i = (lambda *s: torch.empty(s, device="cuda")), (lambda *s: torch.empty(s, dtype=torch.int8, device="cuda"))
    q, s = nls.quantize_rows(f(0, 7))
    assert q.shape == (0, 7) and s.shape == (0,)
    assert nls.quantize_rows(f(2, 0, 7))[0].shape == (2, 0, 7)
    assert nls.int8_matmul(i(0, 9), f(0), i(4, 9), f(4)).shape == (0, 4)
    assert nls.int8_matmul(i(4, 9), f(4), i(0, 9), f(0)).shape == (4, 0)
    assert nls.int8_linear(f(0, 9), i(4, 9), f(4)).shape == (0, 4)
    for shape in ((0, 5), (5, 0), (0, 3, 4), (2, 0, 0)):
        assert nls.orthogonalize(f(*shape)).shape == shape


# ---- orthogonalise ------------------------------------------------------------------------------------------------------------------------
def gradient(rng, m, n):
    r = max(1, min(m, n) // 16)
    return rng.standard_normal((m, r)) @ rng.standard_normal((r, n)) / np.sqrt(r) + 0.3 * rng.standard_normal((m, n))


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize(
    "m,n", [(1, 1), (1, 7), (300, 1), (2, 3), (31, 33), (32, 64), (63, 64), (64, 128), (65, 64), (128, 128), (100, 333), (129, 130), (257, 190), (64, 2000), (700, 512), (1025, 1100), (5, 1100), (1200, 20), (31, 1025), (64, 513), (90, 1500), (128, 257), (128, 3001), (97, 300), (129, 300)]
)
def test_orthogonalize(m, n, name):
    rng = np.random.default_rng(m * 17 + n)
    g = torch.tensor(1e-3 * gradient(rng, m, n), dtype=torch.float32).to(DTYPES[name]).cuda()
    out = nls.orthogonalize(g)
    assert out.dtype == g.dtype and out.is_contiguous()
    newton_schulz_check(out, host(g), nls.NEWTON_SCHULZ, 5, 1e-7, name, m + n)


@pytest.mark.parametrize("batch,m,n", [(1, 64, 64), (5, 48, 80), (33, 80, 48), (3, 200, 260), (2, 1, 9), (3, 120, 700), (4, 1300, 10), (2, 128, 128)])
def test_orthogonalize_batches(batch, m, n):
    rng = np.random.default_rng(batch + m)
    g = np.stack([10.0 ** (2 * i - 4) * gradient(rng, m, n) for i in range(batch)]) if batch < 8 else np.stack([gradient(rng, m, n) for _ in range(batch)])
    t = torch.tensor(g, dtype=torch.float32).cuda()
    out = nls.orthogonalize(t)
    for i in range(batch):
        newton_schulz_check(out[i], host(t[i]), nls.NEWTON_SCHULZ, 5, 1e-7, "float32", i)
    assert torch.equal(nls.orthogonalize(t.view(1, batch, m, n))[0], out)


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("batch,m,n", [(25, 700, 720), (8, 690, 700), (5, 700, 700), (3, 1000, 130)])
def test_orthogonalize_in_every_tile(batch, m, n, name):
    rng = np.random.default_rng(batch)
    g = torch.tensor(np.stack([gradient(rng, m, n)] * 2), dtype=torch.float32)
    g[1] *= 1e-3
    t = torch.stack([g[i % 2] for i in range(batch)]).to(DTYPES[name]).cuda()
    out = nls.orthogonalize(t)
    for i in range(2):
        newton_schulz_check(out[i], host(t[i]), nls.NEWTON_SCHULZ, 5, 1e-7, name, i)
        assert all(torch.equal(out[j], out[i]) for j in range(i, batch, 2))


@pytest.mark.parametrize("m,n,name", [(100, 70001, "float32"), (80001, 128, "bfloat16"), (60, 150000, "float16")])
def test_orthogonalize_with_more_slabs_than_the_card_holds(m, n, name):
    """Workgroups that begin when others are done with the step read what those others read."""
    rng = np.random.default_rng(n)
    g = torch.tensor(rng.standard_normal((m, n)), dtype=torch.float32).to(DTYPES[name]).cuda()
    newton_schulz_check(nls.orthogonalize(g), host(g), nls.NEWTON_SCHULZ, 5, 1e-7, name, 1)


@pytest.mark.parametrize("m,n", [(40, 50), (100, 900), (150, 140)])
def test_orthogonalize_as_many_steps_as_there_may_be(m, n):
    g = torch.tensor(gradient(np.random.default_rng(m), m, n), dtype=torch.float32).cuda()
    newton_schulz_check(nls.orthogonalize(g, steps=32, coefficients=CUBIC), host(g), CUBIC, 32, 1e-7, "float32", m)


@pytest.mark.parametrize("steps,coefficients", [(1, nls.NEWTON_SCHULZ), (2, CUBIC), (9, CUBIC), (8, [nls.NEWTON_SCHULZ] * 5 + [(1.875, -1.25, 0.375)] * 3), (3, (0.5, 0.0, 0.0)), (4, (-1.5, 0.5, 0.0)), (12, nls.NEWTON_SCHULZ)])
@pytest.mark.parametrize("name", sorted(DTYPES))
def test_orthogonalize_polynomials(steps, coefficients, name):
    rng = np.random.default_rng(steps)
    g = torch.tensor(gradient(rng, 90, 140), dtype=torch.float32).to(DTYPES[name]).cuda()
    newton_schulz_check(nls.orthogonalize(g, steps=steps, coefficients=coefficients), host(g), coefficients, steps, 1e-7, name, steps)


def test_orthogonalize_strides_and_sizes_of_numbers():
    rng = np.random.default_rng(2)
    base = torch.tensor(gradient(rng, 150, 260), dtype=torch.float32).cuda()
    for g in (base.T, base[::2, 1:], base[:, ::3], base[:70, :70].T, base[3:4].expand(40, 260), base[:, 5]. view(10, 15)):
        newton_schulz_check(nls.orthogonalize(g), host(g), nls.NEWTON_SCHULZ, 5, 1e-7, "float32", 1)
    for size in (1e-36, 1e-20, 1e-9, 1e9, 1e30):  # from far below eps (the result is tiny then) to near the largest float
        g = size * base[:60, :80].contiguous()
        newton_schulz_check(nls.orthogonalize(g), host(g), nls.NEWTON_SCHULZ, 5, 1e-7, "float32", 1)
    stack = torch.stack([base, base])[:, :50, :60]
    assert torch.equal(nls.orthogonalize(stack)[1], nls.orthogonalize(base[:50, :60].contiguous()))


def test_orthogonalize_zeros_and_what_is_not_finite():
    g = torch.randn(3, 20, 30, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    want = nls.orthogonalize(g)
    h = g.clone()
    h[1] = 0
    out = nls.orthogonalize(h)
    assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2]) and not out[1].any()
    assert not nls.orthogonalize(torch.zeros(5, 4, device="cuda"), eps=0.0).any()
    for bad in (float("nan"), float("inf")):
        h = g.clone()
        h[1, 4, 5] = bad
        out = nls.orthogonalize(h)
        assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2]) and torch.isnan(out[1]).all()
    with pytest.raises(ValueError, match="grow"):
        nls.orthogonalize(g, coefficients=(1e3, 0.0, 0.0))


# ---- in a program -------------------------------------------------------------------------------------------------------------------------
def test_arrays_of_the_framework():
    """NumPy arrays and DeviceArrays give what tensors give."""
    rng = np.random.default_rng(3)
    x, w = activations(rng, 20, 50).astype(np.float32), rng.standard_normal((30, 50)).astype(np.float32)
    q, s = nls.quantize_rows(torch.tensor(w).cuda())
    y = nls.int8_linear(torch.tensor(x).cuda(), q, s)
    o = nls.orthogonalize(torch.tensor(w).cuda())
    hq, hs = nls.quantize_rows(w)
    xq, xs = nls.quantize_rows(x)
    assert np.array_equal(hq, q.cpu().numpy()) and np.array_equal(hs, s.cpu().numpy())
    assert np.array_equal(nls.int8_linear(x, hq, hs), y.cpu().numpy())
    assert np.array_equal(nls.int8_matmul(xq, xs, hq, hs), y.cpu().numpy())
    assert np.array_equal(nls.orthogonalize(w), o.cpu().numpy())
    assert np.array_equal(nls.orthogonalize(w.astype(">f4")), o.cpu().numpy())
    assert np.array_equal(nls.int8_linear(x.astype(">f4"), hq, hs.astype(">f4")), y.cpu().numpy())
    assert np.array_equal(nls.int8_linear(x.astype(np.float16), hq, hs), nls.int8_linear(torch.tensor(x).half().cuda(), q, s).cpu().numpy())
    ctx = nls.default_context()
    dx, dw = ctx.to_device(x, dtype=np.float32), ctx.to_device(w, dtype=np.float32)
    dq, ds = nls.quantize_rows(dw)
    assert isinstance(dq, nls.DeviceArray) and dq.shape == (30, 50) and np.array_equal(dq.to_host(), hq)
    assert np.array_equal(nls.int8_linear(dx, dq, ds).to_host(), y.cpu().numpy())
    assert np.array_equal(nls.int8_matmul(*nls.quantize_rows(dx), dq, ds).to_host(), y.cpu().numpy())
    assert np.array_equal(nls.orthogonalize(dw).to_host(), o.cpu().numpy())
    with pytest.raises(ValueError, match="like the other"):
        nls.int8_linear(dx, hq, hs)


def test_streams_graphs_and_repeats():
    """Other streams than the default one, two graphs replayed side by side, and every result the same bits as the first."""
    rng = np.random.default_rng(4)
    data = []
    for m, n, k in ((4, 256, 300), (200, 512, 1024)):
        x = torch.tensor(activations(rng, m, k), dtype=torch.float32).cuda().bfloat16()
        q, s = nls.quantize_rows(torch.tensor(rng.standard_normal((n, k)), dtype=torch.float32).cuda())
        g = torch.tensor(gradient(rng, n, k), dtype=torch.float32).cuda()
        data.append((x, q, s, g))

    def passes(x, q, s, g):
        xq, xs = nls.quantize_rows(x)
        return [xq, xs, nls.int8_linear(x, q, s), nls.int8_matmul(xq, xs, q, s, dtype="float16"), nls.orthogonalize(g), nls.orthogonalize(g[:40, :70])]

    want = [[t.clone() for t in passes(*d)] for d in data]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for d, st in zip(data, streams):
        with torch.cuda.stream(st):
            for t, w in zip(passes(*d), want[len(graphs)]):
                st.synchronize()
                assert torch.equal(t, w)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(passes(*d))
        graphs.append(graph)
    for turn in range(4):
        for t in outs[0] + outs[1]:
            t.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert all(torch.equal(t, u) for t, u in zip(out, w)), turn
        assert all(torch.equal(t, u) for t, u in zip(passes(*data[0]), want[0]))


def test_threads_with_streams_of_their_own():
    import threading

    rng = np.random.default_rng(5)
    data = []
    for m, n, k in ((3, 128, 200), (70, 256, 320), (300, 64, 96)):
        x = torch.tensor(activations(rng, m, k), dtype=torch.float32).cuda().half()
        q, s = nls.quantize_rows(torch.tensor(rng.standard_normal((n, k)), dtype=torch.float32).cuda())
        data.append((x, q, s, nls.int8_linear(x, q, s), nls.orthogonalize(x)))
    torch.cuda.synchronize()
    wrong = []

    def work(x, q, s, want, ortho):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                y, o = nls.int8_linear(x, q, s), nls.orthogonalize(x)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(y, want) and torch.equal(o, ortho)):
                    wrong.append(x.shape)

    threads = [threading.Thread(target=work, args=d) for d in data]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_context_is_not_made_in_a_capture(monkeypatch):
    from neo_ls_svm_amd import lowbit

    x = torch.ones(4, 32, device="cuda")
    nls.quantize_rows(x)
    with monkeypatch.context() as patch:
        patch.setattr(lowbit, "_default_ctx", {})
        patch.setattr(lowbit, "_on_device", {})
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                x.add_(1.0)
                nls.quantize_rows(x)
    assert nls.quantize_rows(x)[0].shape == (4, 32)


def test_arguments_the_c_calls_refuse():
    """What the Python entry points never pass: workspaces, types, strides and sizes that are checked before anything is launched."""
    import ctypes as C

    ctx = nls.default_context()
    x, q, s, y = torch.ones(64, 48, device="cuda"), torch.ones(64, 48, dtype=torch.int8, device="cuda"), torch.ones(64, device="cuda"), torch.zeros(64, 64, device="cuda")
    ws = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    lib, h, p = ctx.lib, ctx.handle, torch.Tensor.data_ptr
    table = (C.c_double * 3)(1.5, -0.5, 0.0)
    need = C.c_size_t()

    def refused(rc, text):
        with pytest.raises(ValueError, match=text):
            ctx._check(rc)

    refused(lib.nls_quantize_rows(h, p(x), 7, 64, 48, 48, 1, p(q), 48, p(s), None), "type")
    refused(lib.nls_quantize_rows(h, p(x), 0, 64, 40, 48, 1, p(q), 40, p(s), None), "multiples of 16")
    refused(lib.nls_quantize_rows(h, p(x), 0, 64, 48, 48, 1, p(q) + 1, 48, p(s), None), "multiples of 16")
    refused(lib.nls_quantize_rows(h, None, 0, 64, 48, 48, 1, p(q), 48, p(s), None), "null")
    matmul = lambda lda, n_ws, at=0, bias_type=0, m=64: lib.nls_int8_matmul(  # noqa: E731
        h, p(q), lda, p(s), p(q), 48, p(s), p(s), bias_type, m, 64, 47, p(y), 0, 0, p(ws) + at, n_ws, None
    )
    assert lib.nls_int8_matmul_workspace(p(q), 48, p(q), 48, 64, 64, 47, 0, C.byref(need)) == 0 and need.value == 2 * 64 * 48
    refused(matmul(48, need.value - 1), "workspace of")
    refused(matmul(48, need.value, at=16), "aligned")
    refused(matmul(40, need.value), "row strides")
    refused(matmul(48, need.value, bias_type=1), "bias")
    refused(matmul(48, need.value, m=-1), "negative")
    assert matmul(48, need.value) == 0
    lib.nls_orthogonalize_workspace(1, 200, 200, 200, 1, C.byref(need))
    ortho = lambda m, batch, n_ws, steps=1: lib.nls_orthogonalize(h, p(ws), 0, batch, m, 200, m * 200, 200, 1, table, steps, 1e-7, p(ws), p(ws), n_ws, None)  # noqa: E731
    refused(ortho(200, 1, need.value - 1), "workspace of")
    refused(ortho(2**20 + 1, 1, need.value), "2\\^20")
    refused(ortho(200, 65536, need.value), "65535")
    refused(ortho(200, 1, need.value, steps=0), "steps")
    torch.cuda.synchronize()
    assert torch.equal(y, torch.full_like(y, 48.0))  # (47 products and a bias of one)


def test_an_error_left_by_another_call_is_not_taken_for_a_failed_launch():
    ctx = nls.default_context()
    x = torch.ones(4, 32, device="cuda")
    torch.cuda.synchronize()
    page = np.zeros(4096)
    assert ctx.lib.nls_host_unregister(ctx.handle, page.ctypes.data) != 0  # (never registered)
    q, s = nls.quantize_rows(x)
    assert torch.equal(nls.int8_linear(x, q, s), nls.int8_matmul(q, s, q, s)) and nls.orthogonalize(x).shape == (4, 32)


def test_gradients_are_refused_not_lost():
    x = torch.ones(4, 32, device="cuda", requires_grad=True)
    q, s = nls.quantize_rows(x.detach())
    for call in (lambda: nls.quantize_rows(x), lambda: nls.int8_linear(x, q, s), lambda: nls.orthogonalize(x)):
        with pytest.raises(ValueError, match="gradients"):
            call()
        with torch.no_grad():
            call()


def test_frequencies_made_orthogonal_held_and_multiplied_in_eight_bits():
    """The operators together, on the framework's own map: square Gaussian blocks made orthogonal, scaled to frequencies, held in 8 bits, and the angles
    and features of a table computed from 8-bit rows, against ``featuremap`` of the same table and frequencies."""
    d, D, n = 96, 384, 500
    rng = np.random.default_rng(7)
    polar = [nls.NEWTON_SCHULZ] * 6 + [(1.875, -1.25, 0.375)] * 6
    blocks = torch.tensor(rng.standard_normal((D // d, d, d)), dtype=torch.float32).cuda()
    basis = nls.orthogonalize(blocks, steps=len(polar), coefficients=polar)
    eye = basis.cpu().double() @ basis.cpu().double().transpose(1, 2)
    assert float((eye - torch.eye(d, dtype=torch.float64)).abs().max()) < 2e-4
    Z = basis.reshape(D, d) * torch.tensor(np.sqrt(rng.chisquare(d, (D, 1))), dtype=torch.float32).cuda()  # channels x inputs
    X = 0.1 * rng.standard_normal((n, d))
    x = torch.tensor(X, dtype=torch.float32).cuda()
    zq, zs = nls.quantize_rows(Z)
    angles = host(nls.int8_linear(x, zq, zs))
    want = X @ host(Z).T
    # half a step of each operand, against all of the other: |x z - x' z'| <= |x| |dz|_1 + |dx|_1 |z'|
    sx, sz = np.abs(X).max(1, keepdims=True) / 127, np.abs(host(Z)).max(1) / 127
    bound = 0.5 * sz * np.abs(X).sum(1, keepdims=True) + 0.5 * sx * (np.abs(host(Z)).sum(1) + 0.5 * d * sz) + 1e-5
    assert np.all(np.abs(angles - want) <= bound)
    phi = nls.featuremap(X, np.zeros(d), np.ones(d), host(Z).T)
    mine = np.exp(-1j * angles) / np.sqrt(D)
    assert np.all(np.abs(mine - phi[:, :D]) <= bound / np.sqrt(D) + 1e-12)


@pytest.mark.parametrize("m,n", [(4, 304), (3, 25), (16, 17), (17, 500), (28, 4), (5, 2070), (32, 900), (58, 2574), (100, 120), (300, 400)])
def test_orthogonalize_float32_is_as_good_as_plain_float32(m, n):
    """Six steps on Gaussian matrices against 64 bits, beside the same steps in NumPy's float32: at most twice its error, for a pair rounds at 2^-23 where
    float32 does at 2^-24.  The mean over eight matrices: how far single ones are off depends on how their roundings fall."""
    rng = np.random.default_rng(m + n)
    g = rng.standard_normal((8, m, n)).astype(np.float32)
    out = host(nls.orthogonalize(torch.tensor(g).cuda(), steps=6))
    a, b, c = (np.float32(v) for v in nls.NEWTON_SCHULZ)
    mine = plain = 0.0
    for i in range(8):
        want = newton_schulz_oracle(g[i].astype(np.float64), nls.NEWTON_SCHULZ, 6, 1e-7)
        x = g[i].T if m > n else g[i]
        x = x / np.float32(np.linalg.norm(x.astype(np.float64)) + 1e-7)
        for _ in range(6):
            s = x @ x.T
            x = a * x + (b * s + c * (s @ s)) @ x
        mine += np.linalg.norm(out[i] - want) ** 2
        plain += np.linalg.norm((x.T if m > n else x) - want) ** 2
    assert mine <= 4 * plain, (mine / plain) ** 0.5


# ---- 16-bit results: float32's error, rounded once ------------------------------------------------------------------------------------------
FINISH = (1.875, -1.25, 0.375)
TABLES = {
    "5": [nls.NEWTON_SCHULZ] * 5,
    "6": [nls.NEWTON_SCHULZ] * 6,
    "12": [nls.NEWTON_SCHULZ] * 12,
    "5 + 3 finishing": [nls.NEWTON_SCHULZ] * 5 + [FINISH] * 3,
    "5 + 3 of the identity": [nls.NEWTON_SCHULZ] * 5 + [(1.0, 0.0, 0.0)] * 3,
    "16 cubic": [CUBIC] * 16,
}


def sixteen_bit_errors(rng, kind, m, n, table, name):
    """(how far the result is from 64 bits, what its own rounding makes, the error of NumPy float32 products before any rounding, the norm), of one matrix."""
    if kind == "gradient":
        g = gradient(rng, m, n)
    else:  # so many strong directions over a noise floor
        rank, noise = kind
        g = rng.standard_normal((m, rank)) @ rng.standard_normal((rank, n)) + noise * rng.standard_normal((m, n)) if rank else rng.standard_normal((m, n))
    t = torch.tensor(1e-2 * g, dtype=torch.float32).to(DTYPES[name])
    g = host(t)
    want = newton_schulz_oracle(g, table, len(table), 1e-7)
    x = (g.T if m > n else g) / (np.linalg.norm(g) + 1e-7)
    x = x.astype(np.float32)
    for a, b, c in np.asarray(table, dtype=np.float32):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    own = np.linalg.norm(host(torch.tensor(want).to(DTYPES[name])) - want)
    got = host(nls.orthogonalize(t.cuda(), steps=len(table), coefficients=table))
    return np.linalg.norm(got - want), own, np.linalg.norm((x.T if m > n else x) - want), np.linalg.norm(want)


@pytest.mark.parametrize("steps", sorted(TABLES))
@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n", [(130, 200), (300, 420), (400, 400), (700, 150)])
def test_sixteen_bit_results_of_more_than_128_rows_are_float32s_rounded(m, n, name, steps):
    """The error is that of the result's own rounding (norms of tens of thousands of roundings: alike within 5 %) and what the products do before it, which
    is float32's: pairs round at 2^-23 where float32 does at 2^-24, hence twice, and twice that for how single cases fall."""
    rng = np.random.default_rng(m + n)
    for kind in ("gradient", (0, 1.0), (4, 1e-3), (1, 1e-2)):
        off, own, plain, _ = sixteen_bit_errors(rng, kind, m, n, TABLES[steps], name)
        assert off <= 1.05 * own + 4 * plain, (kind, off / own, plain / own)


@pytest.mark.parametrize("steps", [5, 10, 16])
@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n", [(16, 40), (32, 200), (32, 1000), (300, 20), (64, 512), (96, 200), (128, 700), (20, 3000)])
def test_sixteen_bit_results_of_up_to_128_rows(m, n, name, steps):
    """As above, and what the chains of steps on p x p matrices may do to weak directions beside strong ones: roundings of 2^-23 that grow by the square of a
    chain's growth to a sixteenth of half a step of the result, and twice that for the steps behind the chain.  (Hundreds of roundings: alike within 10 %.)"""
    rng = np.random.default_rng(m + n)
    for kind in ((1, 3e-2), (1, 1e-2), (2, 3e-2), (4, 1e-1), (1, 3e-4)):
        for one in (nls.NEWTON_SCHULZ, CUBIC):
            off, own, plain, norm = sixteen_bit_errors(rng, kind, m, n, [one] * steps, name)
            assert off <= 1.1 * own + 4 * plain + HALF[name] / 8 * norm, (kind, one, off / own, plain / own)


def test_an_error_that_the_caller_has_yet_to_ask_for_is_still_there():
    ctx = nls.default_context()
    x = torch.ones(200, 320, device="cuda")
    q, s = nls.quantize_rows(x)
    want = nls.int8_linear(x, q, s), nls.orthogonalize(x), nls.orthogonalize(x[:20])
    torch.cuda.synchronize()
    assert ctx.lib.hipSetDevice(1 << 20) != 0  # (no such device)
    left = ctx.lib.hipPeekAtLastError()
    nls.quantize_rows(x)
    got = nls.int8_linear(x, q, s), nls.orthogonalize(x), nls.orthogonalize(x[:20])
    assert left != 0 and ctx.lib.hipGetLastError() == left and ctx.lib.hipPeekAtLastError() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))

"""Matrix operators of few bits, as a user's program calls them, beside plain forms in elementary torch operations.

* ``quantize_rows``: rows of 16 / 32-bit numbers as 8-bit integers with one scale a row (a row is a token of activations or a
  channel of weights): ``scale = max|x| / 127``, ``q`` = ``127 x / max|x|`` to the nearest integer, ties to even.
* ``int8_matmul``: ``y[m, n] = a_scale[m] b_scale[n] sum_k a[m, k] b[n, k] (+ bias[n])``.
* ``int8_linear``: the two above in one call, ``x`` in 16 / 32 bits against weights held in 8.
* ``orthogonalize``: Newton-Schulz products: ``X = G / (|G|_F + eps)``, then ``X <- a X + (b A + c A A) X`` with ``A = X X^T``
  on the side of the shorter dimension.
"""

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
SIZE = {"bfloat16": 2, "float16": 2, "float32": 4}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def listed():
    return [
        # one token's activations before a projection: latency
        {"name": "quantize_token", "op": "quantize", "rows": 1, "k": 4096, "dtype": "bfloat16"},
        # a prompt's activations: bytes
        {"name": "quantize_prompt", "op": "quantize", "rows": 8192, "k": 8192, "dtype": "bfloat16"},
        # a table of 301 columns (an odd, unaligned row length) in 32 bits
        {"name": "quantize_table", "op": "quantize", "rows": 29300, "k": 301, "dtype": "float32"},
        # rows quantised once and used for several products: a decoding batch, and a prompt
        {"name": "matmul_batch", "op": "matmul", "m": 16, "n": 4096, "k": 4096, "dtype": "bfloat16", "bias": False, "tight": False},
        {"name": "matmul_prompt", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "dtype": "bfloat16", "bias": False, "tight": False},
        # angles of a table on 4096 + 1 frequencies, 32-bit outputs, rows without padding
        {"name": "matmul_angles", "op": "matmul", "m": 2930, "n": 4097, "k": 301, "dtype": "float32", "bias": True, "tight": True},
        # serving: a single token, a decoding batch, a ragged prompt
        {"name": "linear_token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "float16", "bias": True, "tight": False},
        {"name": "linear_batch", "op": "linear", "m": 48, "n": 8192, "k": 8192, "dtype": "bfloat16", "bias": False, "tight": False},
        {"name": "linear_prompt", "op": "linear", "m": 2047, "n": 4096, "k": 4096, "dtype": "bfloat16", "bias": True, "tight": False},
        # a training step's updates: the small matrices of many heads, a wide 32-bit one of odd sizes, a large square one
        {"name": "orthogonalize_heads", "op": "orthogonalize", "batch": 32, "m": 64, "n": 128, "dtype": "float32", "steps": 5},
        {"name": "orthogonalize_odd", "op": "orthogonalize", "batch": 1, "m": 1025, "n": 2930, "dtype": "float32", "steps": 5},
        {"name": "orthogonalize_large", "op": "orthogonalize", "batch": 1, "m": 4096, "n": 4096, "dtype": "bfloat16", "steps": 5},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    largest = {op: max(work(c)["flops"] for c in listed() if c["op"] == op) for op in ("quantize", "matmul", "linear", "orthogonalize")}
    while True:
        op = rng.choice(["quantize", "matmul", "matmul", "linear", "linear", "orthogonalize", "orthogonalize"])
        dtype = rng.choice(sorted(DTYPES))
        if op == "quantize":
            case = {"op": op, "rows": _spread(rng, 1, 32768), "k": _spread(rng, 1, 16384), "dtype": dtype}
        elif op in ("matmul", "linear"):
            sizes = {"m": _spread(rng, 1, 8192), "n": _spread(rng, 16, 16384), "k": _spread(rng, 16, 16384)}
            if rng.random() < 0.6:  # most layers' sizes are multiples of 64
                sizes["n"], sizes["k"] = -(-sizes["n"] // 64) * 64, -(-sizes["k"] // 64) * 64
            case = {"op": op, **sizes, "dtype": dtype, "bias": rng.random() < 0.5, "tight": rng.random() < 0.3}
        else:
            case = {"op": op, "batch": 1, "m": _spread(rng, 1, 4096), "n": _spread(rng, 1, 8192), "dtype": dtype, "steps": rng.choice([4, 5, 5, 6])}
            if max(case["m"], case["n"]) <= 512:
                case["batch"] = _spread(rng, 1, 32)
        if work(case)["flops"] <= largest[op]:
            return case


def work(case):
    op = case["op"]
    if op == "quantize":
        rows, k = case["rows"], case["k"]
        return {"bytes": rows * k * (SIZE[case["dtype"]] + 1) + 4 * rows, "flops": 3 * rows * k}
    if op == "orthogonalize":
        p, q = min(case["m"], case["n"]), max(case["m"], case["n"])
        # X X^T and A A are symmetric: half their entries; (b A + c A A) X whole
        return {
            "bytes": case["batch"] * 2 * p * q * SIZE[case["dtype"]],
            "flops": case["batch"] * case["steps"] * (p * p * q + p * p * p + 2 * p * p * q),
        }
    m, n, k = case["m"], case["n"], case["k"]
    bias = n * SIZE[case["dtype"]] if case["bias"] else 0
    rows = m * k + 4 * m if op == "matmul" else m * k * SIZE[case["dtype"]]
    return {"bytes": rows + n * k + 4 * n + bias + m * n * SIZE[case["dtype"]], "flops": 2 * m * n * k}


def _activations(m, k, generator):
    """Rows of different size with a few channels far above the rest, as activations have them."""
    x = torch.randn(m, k, generator=generator, device="cuda")
    channel = torch.exp(0.5 * torch.randn(k, generator=generator, device="cuda"))
    channel[torch.randint(k, (max(1, k // 256),), generator=generator, device="cuda")] *= 8.0
    return x * channel * torch.exp(0.5 * torch.randn(m, 1, generator=generator, device="cuda"))


def _eight_bits(x, tight):
    """Rows in 8 bits: packed without gaps, or each row starting at a multiple of 16 bytes (as ``quantize_rows`` lays them)."""
    largest = x.abs().amax(1)
    rows, k = x.shape
    held = torch.zeros(rows, k if tight else -(-k // 16) * 16, dtype=torch.int8, device="cuda")
    q = held[:, :k]
    q.copy_((x.double() * 127 / largest.double().clamp_min(1e-30)[:, None]).round())
    return q, largest / 127


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    if op == "quantize":
        return {"case": case, "x": _activations(case["rows"], case["k"], generator).to(dtype)}
    if op == "orthogonalize":
        # a gradient: a few strong directions over a noise floor
        b, m, n = case["batch"], case["m"], case["n"]
        r = max(1, min(m, n) // 16)
        left = torch.randn(b, m, r, generator=generator, device="cuda") / math.sqrt(r)
        right = torch.randn(b, r, n, generator=generator, device="cuda").contiguous()
        g = torch.stack([u @ v for u, v in zip(left, right)]) + 0.3 * torch.randn(b, m, n, generator=generator, device="cuda")
        g = (1e-3 * g).to(dtype)
        return {"case": case, "g": g if b > 1 else g[0]}
    m, n, k = case["m"], case["n"], case["k"]
    state = {"case": case}
    x = _activations(m, k, generator)
    if op == "matmul":
        state["a"], state["a_scale"] = _eight_bits(x, case["tight"])
    else:
        state["x"] = x.to(dtype)
    state["b"], state["b_scale"] = _eight_bits(torch.randn(n, k, generator=generator, device="cuda") / math.sqrt(k), case["tight"])
    state["bias"] = torch.randn(n, generator=generator, device="cuda").to(dtype) if case["bias"] else None
    return state


def _quantize(x):
    wide = x.float()
    largest = wide.abs().amax(-1)
    # a quotient next to a half: in 64 bits, where it cannot fall on the wrong side
    q = (wide.double() * 127 / largest.double().clamp_min(torch.finfo(torch.float64).tiny)[..., None]).round().to(torch.int8)
    return q, largest / 127


def _product(a, a_scale, b, b_scale, bias, dtype):
    y = (a.float() @ b.float().T) * a_scale[:, None] * b_scale[None, :]
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def _newton_schulz(g, steps):
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    x = (x / ((x * x).sum((-2, -1), keepdim=True).sqrt() + EPS)).contiguous()
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.transpose(-2, -1) if tall else x).to(g.dtype).contiguous()


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        import neo_ls_svm_amd as nls

        if op == "quantize":
            q, scale = nls.quantize_rows(state["x"])
            return {"q": q, "scale": scale}
        if op == "matmul":
            return nls.int8_matmul(state["a"], state["a_scale"], state["b"], state["b_scale"], bias=state["bias"], dtype=case["dtype"])
        if op == "linear":
            return nls.int8_linear(state["x"], state["b"], state["b_scale"], bias=state["bias"])
        return nls.orthogonalize(state["g"], steps=case["steps"], coefficients=COEFFICIENTS, eps=EPS)
    if op == "quantize":
        q, scale = _quantize(state["x"])
        return {"q": q, "scale": scale}
    if op == "matmul":
        return _product(state["a"], state["a_scale"], state["b"], state["b_scale"], state["bias"], DTYPES[case["dtype"]])
    if op == "linear":
        q, scale = _quantize(state["x"])
        return _product(q, scale, state["b"], state["b_scale"], state["bias"], state["x"].dtype)
    return _newton_schulz(state["g"], case["steps"])


def exact(case, seed):
    """The definitions, in 64 bits throughout."""
    state = prepare(case, seed)
    op = case["op"]
    if op == "orthogonalize":
        g = state["g"].double()
        side = g if g.shape[-2] <= g.shape[-1] else g.mT
        stack = side if side.dim() == 3 else side[None]
        a, b, c = COEFFICIENTS
        done = []
        for one in stack:
            x = one / (torch.linalg.norm(one) + EPS)
            eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
            for _ in range(case["steps"]):
                s = torch.mm(x, x.T)
                x = torch.mm(a * eye + torch.mm(s, b * eye + c * s), x)
            done.append(x)
        y = torch.stack(done) if side.dim() == 3 else done[0]
        return y.contiguous() if side is g else y.mT.contiguous()
    if op == "matmul":
        a, a_scale = state["a"].double(), state["a_scale"].double()
    else:
        x = state["x"].double()
        top = x.abs().max(dim=1).values
        ratio = torch.where(top[:, None] > 0, x / torch.where(top > 0, top, 1.0)[:, None] * 127, 0.0)
        # the quotient of two numbers of few bits: what is within 1e-12 of a half is that half
        half = torch.floor(ratio) + 0.5
        a = torch.where((ratio - half).abs() < 1e-11, 2 * torch.round(half / 2), torch.round(ratio))
        a_scale = top / 127
        if op == "quantize":
            return {"q": a.to(torch.int8), "scale": a_scale}
    y = torch.mm(a, state["b"].double().T) * torch.outer(a_scale, state["b_scale"].double())
    return y if state["bias"] is None else y + state["bias"].double()

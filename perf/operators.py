"""Cases that measure the framework's operators for 8-bit products and for
orthogonalising a matrix, with a plain form of each.

Operators (the user's call of each is what `run` makes when `own` is true):

- quantize: ``ops.quantize_rows(x)`` gives every row of x a scale
  s = float32(max|x| / 127) and 8-bit integers q = round_half_even(x / s), the
  quotient taken exactly. Works on activations (a scale for each token) and on
  weights (a scale for each output channel) alike.
- matmul: ``ops.int8_matmul(xq, xs, wq, ws, bias)`` gives
  y[i, j] = (sum_k xq[i, k] wq[j, k]) xs[i] ws[j] + bias[j].
- linear: ``ops.int8_linear(x, wq, ws, bias)``, the two joined for weights that
  were quantised once: what a fitted model answers a request with.
- orthogonalize: ``ops.newton_schulz(x)``, X / ||X||_F taken five times through
  X <- a X + b (X X^T) X + c (X X^T)^2 X, the Gram matrix being of the shorter
  side.
"""

import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16,
          "float16": torch.float16}


def listed():
    return [
        # a micro-batch of requests with the 100 features of the benchmark data
        {"name": "quantize_batch", "op": "quantize", "m": 64, "k": 100,
         "dtype": "float32"},
        # a shard of a million such rows
        {"name": "quantize_shard", "op": "quantize", "m": 1_000_000, "k": 100,
         "dtype": "float32"},
        # one request against 50 components: nothing but latency
        {"name": "linear_row", "op": "linear", "m": 1, "k": 100, "n": 50,
         "dtype": "float32"},
        # one token against a large weight matrix: the weights' bytes count
        {"name": "linear_token", "op": "linear", "m": 1, "k": 8192, "n": 8192,
         "dtype": "bfloat16"},
        # a ragged batch of tokens with sizes that no tile divides
        {"name": "linear_ragged", "op": "linear", "m": 333, "k": 5001,
         "n": 4099, "dtype": "bfloat16"},
        # rows of 50,000 features projected on 50 components
        {"name": "matmul_wide", "op": "matmul", "m": 4096, "k": 50_000,
         "n": 50, "dtype": "float32"},
        # similarities of 100,000 rows to 1000 others: the output's bytes count
        {"name": "matmul_scores", "op": "matmul", "m": 100_000, "k": 100,
         "n": 1000, "dtype": "float32"},
        # a long prompt through a large weight matrix: the matrix cores count
        {"name": "matmul_large", "op": "matmul", "m": 8192, "k": 8192,
         "n": 8192, "dtype": "bfloat16"},
        # the update of one small weight matrix
        {"name": "orthogonalize_small", "op": "orthogonalize", "b": 1,
         "m": 48, "k": 100, "dtype": "float32"},
        # a range finder's panel: 50 components and 10 more, a million rows
        {"name": "orthogonalize_panel", "op": "orthogonalize", "b": 1,
         "m": 1_000_000, "k": 60, "dtype": "float32"},
        # the update of a square weight matrix
        {"name": "orthogonalize_square", "op": "orthogonalize", "b": 1,
         "m": 2048, "k": 2048, "dtype": "float32"},
        # the updates of a stack of layers, of odd sizes
        {"name": "orthogonalize_stack", "op": "orthogonalize", "b": 4,
         "m": 1027, "k": 4001, "dtype": "bfloat16"},
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    op = rng.choice(("quantize", "linear", "matmul", "orthogonalize"))
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        dtype = rng.choice(tuple(DTYPES))
        if op == "quantize":
            case = {"op": op, "m": _between(rng, 1, 2_000_000),
                    "k": _between(rng, 1, 60_000), "dtype": dtype}
        elif op == "linear":
            case = {"op": op, "m": _between(rng, 1, 512),
                    "k": _between(rng, 16, 16_384),
                    "n": _between(rng, 1, 16_384), "dtype": dtype}
        elif op == "matmul":
            case = {"op": op, "m": _between(rng, 1, 100_000),
                    "k": _between(rng, 16, 50_000),
                    "n": _between(rng, 16, 16_384), "dtype": dtype}
        else:
            # either a few columns and many rows, or an update's matrix
            if rng.random() < 0.4:
                b, k = 1, _between(rng, 1, 110)
                m = _between(rng, k, 1_000_000)
            else:
                b = rng.choice((1, 1, 2, 3, 5))
                m, k = _between(rng, 16, 4500), _between(rng, 16, 4500)
            case = {"op": op, "b": b, "m": m, "k": k, "dtype": dtype}
        if _cost(case) <= most:
            return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _features(g, m, k, dtype):
    """Rows as scaled features have them, of different norms."""
    x = torch.randn(m, k, generator=g, device="cuda")
    x *= torch.exp(torch.randn(m, 1, generator=g, device="cuda"))
    return x.to(dtype)


def _held(x):
    """8-bit rows and scales that the program has kept. Rows begin at
    multiples of 16 bytes, as the framework lays them out."""
    m, k = x.shape
    q, s = _quantize(x)
    rows = torch.zeros(m, (k + 15) // 16 * 16, dtype=torch.int8,
                       device=x.device)
    rows[:, :k] = q
    return rows[:, :k], s


def _matrix(g, case):
    """A panel of a power iteration (singular values that fall off), or an
    update: a few strong directions over noise."""
    b, m, k = case["b"], case["m"], case["k"]
    x = torch.randn(b, m, k, generator=g, device="cuda")
    if max(m, k) > 4 * min(m, k) and min(m, k) <= 128:
        fall = torch.logspace(0, -1.5, min(m, k), device="cuda")
        x *= fall[None, None, :] if k <= m else fall[None, :, None]
    else:
        r = min(16, m, k)
        strong = torch.randn(b, m, r, generator=g, device="cuda")
        other = torch.randn(b, r, k, generator=g, device="cuda")
        fall = torch.logspace(0, -1, r, device="cuda")
        x += (strong * fall) @ other * 0.5
    x *= 0.01
    return (x if b > 1 else x[0]).to(DTYPES[case["dtype"]])


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"op": case["op"], "dtype": dtype}
    if case["op"] == "quantize":
        state["x"] = _features(g, case["m"], case["k"], dtype)
    elif case["op"] == "orthogonalize":
        state["x"] = _matrix(g, case)
    else:
        x = _features(g, case["m"], case["k"], dtype)
        if case["op"] == "matmul":
            state["xq"], state["xs"] = _held(x)
        else:
            state["x"] = x
        w = _features(g, case["n"], case["k"], torch.float32)
        state["wq"], state["ws"] = _held(w / math.sqrt(case["k"]))
        state["bias"] = torch.randn(case["n"], generator=g, device="cuda")
    return state


def _quantize(x):
    # the quotient in 64 bits: a value next to the middle of two integers
    # would go to the wrong one otherwise
    big = x.abs().amax(dim=1).double()
    s = (big / 127.0).float()
    q = torch.round(x.double() / s.double()[:, None])
    q = torch.where(s[:, None] > 0, q, torch.zeros_like(q))
    return q.to(torch.int8), s


def _product(xq, xs, wq, ws, bias, dtype):
    y = xq.float() @ wq.float().t()
    return (y * xs[:, None] * ws[None, :] + bias).to(dtype)


def _gram(y):
    if y.shape[-1] <= 16384:
        return y @ y.transpose(-2, -1).contiguous()
    # the Gram matrix of a long side is a long sum too: pieces of it in 32
    # bits, their sum in 64
    *batch, n, m = y.shape
    pieces = -(-m // 2048)
    y = torch.nn.functional.pad(y, (0, pieces * 2048 - m))
    y = y.reshape(*batch, n, pieces, 2048).transpose(-3, -2).contiguous()
    parts = y @ y.transpose(-2, -1).contiguous()
    return parts.double().sum(dim=-3).float()


def _orthogonalize(x):
    a, b, c = COEFFICIENTS
    y = x.float()
    tall = y.shape[-2] > y.shape[-1]
    if tall:
        y = y.transpose(-2, -1)
    y = y.contiguous()
    # a long sum: 64 bits
    y = y / y.double().square().sum(dim=(-2, -1), keepdim=True).sqrt().float()
    step = 0
    while step < STEPS:
        gram = _gram(y)
        y = a * y + (b * gram + c * (gram @ gram)) @ y
        step += 1
    return (y.transpose(-2, -1) if tall else y).to(x.dtype)


def run(state):
    op = state["op"]
    if own:
        from mi355ml import ops
        if op == "quantize":
            return ops.quantize_rows(state["x"])
        if op == "linear":
            return ops.int8_linear(state["x"], state["wq"], state["ws"],
                                   bias=state["bias"])
        if op == "matmul":
            return ops.int8_matmul(state["xq"], state["xs"], state["wq"],
                                   state["ws"], bias=state["bias"],
                                   out_dtype=state["dtype"])
        return ops.newton_schulz(state["x"], steps=STEPS,
                                 coefficients=COEFFICIENTS)
    if op == "quantize":
        return _quantize(state["x"])
    if op == "linear":
        xq, xs = _quantize(state["x"])
        return _product(xq, xs, state["wq"], state["ws"], state["bias"],
                        state["dtype"])
    if op == "matmul":
        return _product(state["xq"], state["xs"], state["wq"], state["ws"],
                        state["bias"], state["dtype"])
    return _orthogonalize(state["x"])


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (size + 1) + 4 * m, "flops": 3 * m * k}
    if case["op"] == "orthogonalize":
        b, n, m = case["b"], *sorted((case["m"], case["k"]))
        # a Gram matrix has two equal halves. Either five steps on the whole
        # matrix, or on its Gram matrix with one product at the end.
        whole = STEPS * (n * n * m + n ** 3 + 2 * n * n * m)
        gram = n * n * m + 17 * n ** 3 + 2 * n * n * m
        return {"bytes": 2 * size * b * n * m, "flops": b * min(whole, gram)}
    m, k, n = case["m"], case["k"], case["n"]
    read = m * k * (size if case["op"] == "linear" else 1) + n * k
    return {"bytes": read + size * m * n + 4 * (n + n + m),
            "flops": 2 * m * n * k}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orthogonalize":
        x = state["x"].double()
        x = x if x.dim() == 3 else x[None]
        a, b, c = COEFFICIENTS
        outs = []
        for one in x:
            tall = one.shape[0] > one.shape[1]
            y = (one.t() if tall else one).contiguous()
            y = y / torch.linalg.vector_norm(y)
            for _ in range(STEPS):
                # (b G + c G^2) Y as G (b Y + c G Y), so that it shares no
                # product with the plain form
                gram = torch.mm(y, y.t().contiguous())
                gy = torch.mm(gram, y)
                y = a * y + b * gy + c * torch.mm(gram, gy)
            outs.append(y.t() if tall else y)
        out = torch.stack(outs)
        return out if state["x"].dim() == 3 else out[0]
    if case["op"] != "matmul":
        x = state["x"].double()
        # the scale is a 32-bit number by definition
        s = (x.abs().max(dim=1).values / 127).to(torch.float32)
        s64 = s.double().clamp(min=torch.finfo(torch.float64).tiny)
        q = (x / s64.unsqueeze(1)).round()
        if case["op"] == "quantize":
            return q.to(torch.int8), s.double()
    else:
        q, s = state["xq"].double(), state["xs"]
    y = torch.mm(q, state["wq"].double().t().contiguous())
    y = y * torch.outer(s.double(), state["ws"].double())
    return y + state["bias"].double()

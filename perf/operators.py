"""The linear layers of a language model's feed-forward block, measured over the calls that a user makes.

Three operators and what goes with them: the gated projection pair `act(x Wg^T) * (x Wu^T)` with its
backward pass, dropout whose mask is drawn from a counter and never stored (forward, with the residual
added, and backward), and the 8-bit product that serves the same layers (a scale to each token and each
output channel, tokens quantised on the way in).

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare` makes what a
program has in hand, `run` is one pass. With `own` false `run` computes the operators from elementary torch
operations in 32 bits, with `own` true it calls the framework's operators. `exact` is the same
result from the definitions in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEMSIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------ the cases
def listed():
    return [
        # One token of a decoding sequence through the gated projections: all time goes into reading the weights.
        {"name": "gated_decode_one", "path": "gated", "dtype": "bf16", "activation": "silu", "rows": 1, "inner": 4096, "outer": 11008, "sliced": False},
        # A batch of decoding sequences, one token of each, an odd number of them; x is a slice of a wider buffer.
        {"name": "gated_decode_batch", "path": "gated", "dtype": "f16", "activation": "gelu_tanh", "rows": 53, "inner": 2048, "outer": 5632, "sliced": True},
        # A prompt, or several in one batch: the largest product.
        {"name": "gated_prefill", "path": "gated", "dtype": "bf16", "activation": "silu", "rows": 8192, "inner": 4096, "outer": 11008, "sliced": False},
        # A training step of the pair: output and both gradients.
        {"name": "gated_train", "path": "gated_train", "dtype": "bf16", "activation": "silu", "rows": 4096, "inner": 4096, "outer": 11008, "sliced": False},
        # The same in 32 bits, every size off every grid.
        {"name": "gated_train_f32_ragged", "path": "gated_train", "dtype": "f32", "activation": "gelu", "rows": 1531, "inner": 1027, "outer": 1365, "sliced": False},
        # Dropout on a small activation: the cost of a call.
        {"name": "dropout_small", "path": "dropout", "dtype": "f32", "rows": 16, "cols": 256, "p": 0.1, "residual": True},
        # The output of a block, dropped out and added to the residual stream, and its gradient.
        {"name": "dropout_train", "path": "dropout", "dtype": "bf16", "rows": 8192, "cols": 4096, "p": 0.1, "residual": True},
        # Ragged rows, no residual.
        {"name": "dropout_ragged", "path": "dropout", "dtype": "f16", "rows": 12544, "cols": 2933, "p": 0.5, "residual": False},
        # One token through an 8-bit linear layer: quantised on the way in, the weights read once.
        {"name": "int8_decode_one", "path": "linear_int8", "dtype": "bf16", "rows": 1, "inner": 4096, "outer": 11008, "bias": False},
        # A prompt through an 8-bit linear layer.
        {"name": "int8_prefill", "path": "linear_int8", "dtype": "bf16", "rows": 8192, "inner": 4096, "outer": 11008, "bias": False},
        # The product alone, of tokens that are 8-bit already, ragged, with a bias.
        {"name": "int8_product_ragged", "path": "mm_int8", "dtype": "f16", "rows": 2537, "inner": 1027, "outer": 3709, "bias": True},
        # The product alone at a batch of decoding sequences.
        {"name": "int8_product_batch", "path": "mm_int8", "dtype": "bf16", "rows": 64, "inner": 11008, "outer": 4096, "bias": False},
    ]


PATHS = ("gated", "gated", "gated_train", "dropout", "linear_int8", "mm_int8")
ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def draw(rng):
    """One more case: a path by turns of the die, sizes spread over their logarithm."""
    most = max(_seconds(c) for c in listed())
    while True:
        case = _draw_once(rng)
        if _seconds(case) <= 0.5 * most:
            return case


def _draw_once(rng):
    path = rng.choice(PATHS)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if path == "dropout":
        return {"path": path, "dtype": dtype, "rows": _size(rng, 1, 32768), "cols": _size(rng, 8, 8192), "p": rng.choice((0.0, 0.05, 0.1, 0.5)), "residual": rng.random() < 0.5}
    case = {"path": path, "dtype": dtype, "rows": _size(rng, 1, 8192), "inner": _size(rng, 64, 8192), "outer": _size(rng, 64, 11008)}
    if path in ("gated", "gated_train"):
        return {**case, "activation": rng.choice(ACTIVATIONS), "sliced": rng.random() < 0.25}
    return {**case, "bias": rng.random() < 0.5}


def _size(rng, low, high):
    """An extent between `low` and `high`, even in its logarithm; half of them are rounded to multiples of
    64 or 8, the others stay as odd as they come."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    grid = rng.choice((64, 8, 1, 1))
    return min(max(n // grid * grid, grid if grid <= n else n, low), high)


def _seconds(case):
    """Roughly what a pass of the plain form takes."""
    w = work(case)
    return w["bytes"] / 1e12 + w["flops"] / 5e13


# ------------------------------------------------------------------------------- prepare
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=DEVICE).mul_(std).to(dt)

    def int8(*shape):
        return torch.randn(shape, generator=g, device=DEVICE).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)

    def uniform(low, high, n):
        return torch.rand(n, generator=g, device=DEVICE).mul_(high - low).add_(low)

    path, st = case["path"], {"case": case}
    if path == "dropout":
        rows, cols = case["rows"], case["cols"]
        st["x"], st["dy"] = normal(rows, cols), normal(rows, cols, std=0.1)
        st["residual"] = normal(rows, cols) if case["residual"] else None
        # (seed, offset): the generator's key, and how many draws of four words have gone before
        key = torch.randint(-(2**62), 2**62, (1,), generator=g, device=DEVICE)
        offset = torch.randint(0, 2**40, (1,), generator=g, device=DEVICE)
        st["state"] = torch.cat([key, offset])
        return st
    m, k, n = case["rows"], case["inner"], case["outer"]
    if path in ("gated", "gated_train"):
        st["x"] = normal(m, k + 64)[:, :k] if case["sliced"] else normal(m, k)
        st["w"] = normal(2 * n, k, std=1.0 / math.sqrt(k))  # [gate rows; up rows], each as torch.nn.Linear keeps its weight
        if path == "gated_train":
            st["dh"] = normal(m, n, std=0.1)
        return st
    if path == "linear_int8":
        st["x"] = normal(m, k)
        st["x"][:, torch.randperm(k, generator=g, device=DEVICE)[: max(1, k // 512)]] *= 8  # a few channels stand out, as they do in trained models
    else:
        st["q"], st["scale"] = int8(m, k), uniform(0.01, 0.05, m)
    st["w"], st["w_scale"] = int8(n, k), uniform(0.5, 1.5, n) / (32.0 * math.sqrt(k))
    st["bias"] = normal(n) if case["bias"] else None
    return st


# ----------------------------------------------------------------------------------- run
def run(state):
    return _RUN[state["case"]["path"]](state, state["case"])


def _run_gated(st, case):
    if own:
        return _operators().gated_linear(st["x"], st["w"], case["activation"])
    g, u = _projections(st["x"], st["w"])
    return (_act(g, case["activation"]) * u).to(st["x"].dtype)


def _run_gated_train(st, case):
    x, w, dh, act = st["x"], st["w"], st["dh"], case["activation"]
    if own:
        h, projections = _operators().gated_linear_train(x, w, act)
        dx, dw = _operators().gated_linear_backward(dh, x, w, projections, act, [True, True])
        return h, dx, dw
    g, u = _projections(x, w)
    a, d = _act(g, act), _act_slope(g, act)
    dp = torch.cat([dh.float() * u * d, dh.float() * a], 1)
    return (a * u).to(x.dtype), (dp @ w.float()).to(x.dtype), (dp.t() @ x.float()).to(x.dtype)


def _run_dropout(st, case):
    x, dy, state, residual, p = st["x"], st["dy"], st["state"], st["residual"], case["p"]
    if own:
        return _operators().dropout(x, p, state, residual), _operators().dropout_backward(dy, p, state)
    kept = (_words(x.numel(), state) >= round(p * 2**32)).view(x.shape)
    scale = 1.0 / (1.0 - p)
    y = torch.where(kept, x.float() * scale, 0.0)
    if residual is not None:
        y = residual.float() + y
    return y.to(x.dtype), torch.where(kept, dy.float() * scale, 0.0).to(x.dtype)


def _run_linear_int8(st, case):
    if own:
        q, scale = _operators().quantize_rows(st["x"])
        return _operators().mm_int8(q, st["w"].t(), scale, st["w_scale"], st["bias"], out_dtype=st["x"].dtype)
    x = st["x"].float()
    most = x.abs().amax(1)
    q = torch.round(x * torch.where(most > 0, 127.0 / most, 0.0)[:, None])
    return _scaled(q @ st["w"].float().t(), most / 127.0, st, st["x"].dtype)


def _run_mm_int8(st, case):
    dt = DTYPES[case["dtype"]]
    if own:
        return _operators().mm_int8(st["q"], st["w"].t(), st["scale"], st["w_scale"], st["bias"], out_dtype=dt)
    return _scaled(st["q"].float() @ st["w"].float().t(), st["scale"], st, dt)


_RUN = {"gated": _run_gated, "gated_train": _run_gated_train, "dropout": _run_dropout, "linear_int8": _run_linear_int8, "mm_int8": _run_mm_int8}


def _operators():
    import backendbench_b200.custom_ops  # noqa: F401  (registers torch.ops.b200)

    return torch.ops.b200


def _projections(x, w):
    return (x.float() @ w.float().t()).chunk(2, 1)


def _scaled(sums, scale, st, dt):
    y = sums * scale[:, None] * st["w_scale"]
    return (y if st["bias"] is None else y + st["bias"].float()).to(dt)


def _act(g, name):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    if name == "relu":
        return torch.where(g > 0, g, 0.0)
    return 1 / (1 + torch.exp(-g))


def _act_slope(g, name):
    s = 1 / (1 + torch.exp(-g))
    if name == "silu":
        return s * (1 + g * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    if name == "relu":
        return (g > 0).float()
    return s * (1 - s)


def _words(n, state):
    """The first `n` 32-bit words that Philox-4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random
    numbers: as easy as 1, 2, 3; SC 2011) gives for the counters offset, offset + 1, ...; four words to a counter."""
    low = 0xFFFFFFFF
    at = torch.arange((n + 3) // 4, device=DEVICE) + state[1]
    a, b, c, d = at & low, (at >> 32) & low, torch.zeros_like(at), torch.zeros_like(at)
    k0, k1 = state[0] & low, (state[0] >> 32) & low
    for _ in range(10):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57  # the upper half of a product is taken from its 64 bits, whatever their sign
        a, b, c, d = ((q >> 32) & low) ^ b ^ k0, q & low, ((p >> 32) & low) ^ d ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([a, b, c, d], 1).view(-1)[:n]


# ------------------------------------------------------------------------ 64 bits, work
def exact(case, seed):
    st = prepare(case, seed)
    path = case["path"]
    if path == "dropout":
        x = st["x"]
        keep = torch.from_numpy(_kept(x.numel(), st["state"].tolist(), case["p"])).to(DEVICE).view(x.shape)
        y = x.double().masked_fill(~keep, 0) / (1 - case["p"])
        dx = st["dy"].double().masked_fill(~keep, 0) / (1 - case["p"])
        return (y if st["residual"] is None else y + st["residual"].double()), dx
    w = st["w"].double()
    if path in ("gated", "gated_train"):
        x = st["x"].double()
        n = case["outer"]
        gate = torch.nn.functional.linear(x, w[:n]).requires_grad_()
        up = torch.nn.functional.linear(x, w[n:])
        a = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "relu": torch.relu, "sigmoid": torch.sigmoid}[case["activation"]](gate)
        h = a.detach() * up
        if path == "gated":
            return h
        dh = st["dh"].double()
        (dg,) = torch.autograd.grad(a, gate, dh * up)
        du = dh * a.detach()
        return h, torch.addmm(dg.mm(w[:n]), du, w[n:]), torch.cat([dg.t().mm(x), du.t().mm(x)])
    if path == "linear_int8":
        x = st["x"].double()
        scale = x.abs().max(dim=1).values / 127
        q = torch.round(x / torch.where(scale == 0, 1, scale).unsqueeze(1))
    else:
        q, scale = st["q"].double(), st["scale"].double()
    y = torch.nn.functional.linear(q, w).mul_(torch.outer(scale, st["w_scale"].double()))
    return y if st["bias"] is None else y + st["bias"].double()


def _kept(n, state, p):
    """Which of `n` elements stay, on the host: a word of the generator at or above p * 2^32."""
    seed, offset = (v % 2**64 for v in state)
    draws = (n + 3) // 4
    count = np.arange(draws, dtype=np.uint64) + np.uint64(offset)
    x = [(count & np.uint64(0xFFFFFFFF)).astype(np.uint32), (count >> np.uint64(32)).astype(np.uint32), np.zeros(draws, np.uint32), np.zeros(draws, np.uint32)]
    for r in range(10):
        key = [np.uint32((seed + r * 0x9E3779B9) % 2**32), np.uint32(((seed >> 32) + r * 0xBB67AE85) % 2**32)]
        first, third = x[0].astype(np.uint64) * np.uint64(0xD2511F53), x[2].astype(np.uint64) * np.uint64(0xCD9E8D57)
        x = [(third >> np.uint64(32)).astype(np.uint32) ^ x[1] ^ key[0], third.astype(np.uint32), (first >> np.uint64(32)).astype(np.uint32) ^ x[3] ^ key[1], first.astype(np.uint32)]
    return np.stack(x, 1).reshape(-1)[:n] >= np.uint32(round(p * 2**32))


def work(case):
    """Bytes (each input once, each output once) and operations that a pass cannot do without."""
    e = ITEMSIZE[case["dtype"]]
    m, path = case["rows"], case["path"]
    if path == "dropout":
        return {"bytes": m * case["cols"] * e * (5 if case["residual"] else 4) + 16, "flops": 0}
    k, n = case["inner"], case["outer"]
    if path == "gated":
        return {"bytes": e * (m * k + 2 * n * k + m * n), "flops": 4 * m * k * n}
    if path == "gated_train":
        # x, w, dh read, h, dx, dw written
        return {"bytes": e * (2 * m * k + 4 * n * k + 2 * m * n), "flops": 12 * m * k * n}
    bias = e * n if case["bias"] else 0
    return {"bytes": (m * k * e if path == "linear_int8" else m * k + 4 * m) + n * k + 4 * n + m * n * e + bias, "flops": 2 * m * k * n}

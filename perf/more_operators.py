"""The matrix operators of networks that read signals: plain forms, cases and sizes.

The projections of a localisation network are matrix products.  They are
answered and trained in 8 bits, and their weights are trained by steps whose
directions are orthogonalised:

  quant    rows to e4m3 codes with a power-of-two scale for each block of 128
           (and, for training, the same of the transposed matrix)
  product  codes times a weight's codes, scales for each block or row, a bias
  linear   a projection whose three products (output, gradients of input and
           weight) run on such codes
  polar    orthogonalisation of matrices by Newton-Schulz products
  muon     one step of an optimizer that moves matrices along orthogonalised
           momenta

run() computes a case in elementary torch operations (own = False) or by the
framework's operators (own = True); exact() computes it in float64 from the
definitions.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"
BLOCK = 128               # codes along the summed axis that share a scale
E4M3_MAX = 448.0
LEAST = -126              # the smallest scale's exponent
STEPS, COEFFICIENTS, NS_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, MOMENTUM, DECAY = 1e-3, 0.95, 0.1


# ---- cases -----------------------------------------------------------------

def listed():
    return [
        # a decoding step's rows
        {"name": "quant 16x2048 bf16", "op": "quant", "rows": 16, "D": 2048, "dtype": "bf16", "both": False},
        # a training batch's rows, and their transpose for the weight's gradient
        {"name": "quant 16384x4096 bf16 both", "op": "quant", "rows": 16384, "D": 4096, "dtype": "bf16", "both": True},
        # one sample of one stream; its row comes from an 8-bit norm, with one scale
        {"name": "product 1x2048x4096", "op": "product", "M": 1, "K": 2048, "N": 4096, "dtype": "bf16",
         "scales": "row", "bias": True},
        # a batch of odd sizes, float32 results
        {"name": "product 333x1000x1500 f32", "op": "product", "M": 333, "K": 1000, "N": 1500, "dtype": "f32",
         "scales": "block", "bias": True},
        # the largest batch that is answered at once
        {"name": "product 8192x4096x8192", "op": "product", "M": 8192, "K": 4096, "N": 8192, "dtype": "bf16",
         "scales": "block", "bias": False},
        # a small float32 network's projection in training, odd sizes
        {"name": "linear 515x1000x2000 f32", "op": "linear", "M": 515, "K": 1000, "N": 2000, "dtype": "f32",
         "weight": "f32", "bias": True},
        # inputs and gates of a wide block for a batch of 8 series of 2048 samples
        {"name": "linear 16384x2048x4096 bf16", "op": "linear", "M": 16384, "K": 2048, "N": 4096, "dtype": "bf16",
         "weight": "bf16", "bias": True},
        # a few small matrices
        {"name": "polar 3x130x260 bf16", "op": "polar", "B": 3, "m": 130, "n": 260, "dtype": "bf16"},
        # one tall matrix in float32
        {"name": "polar 4096x2048 f32", "op": "polar", "B": 1, "m": 4096, "n": 2048, "dtype": "f32"},
        # the largest
        {"name": "polar 4096x8192 bf16", "op": "polar", "B": 1, "m": 4096, "n": 8192, "dtype": "bf16"},
        # a small network's matrices, odd sizes
        {"name": "muon 130x4 f32", "op": "muon", "width": 130, "depth": 4, "dtype": "f32"},
        # a wide network's
        {"name": "muon 2048x4 bf16", "op": "muon", "width": 2048, "depth": 4, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["quant", "product", "product", "product", "linear", "linear", "polar", "polar", "muon"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quant":
        D = _log_int(rng, 1, 8192)
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(65536, (1 << 26) // D))), "D": D, "dtype": dtype,
                "both": rng.random() < 0.5}
    if op == "product":
        M, K, N = _log_int(rng, 1, 16384), _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
        M = max(1, min(M, (1 << 38) // (K * N)))
        return {"op": op, "M": M, "K": K, "N": N, "dtype": dtype, "scales": rng.choice(["row", "block", "block"]),
                "bias": rng.random() < 0.5}
    if op == "linear":
        M, K, N = _log_int(rng, 1, 32768), _log_int(rng, 16, 4096), _log_int(rng, 16, 8192)
        M = max(1, min(M, (1 << 37) // (K * N)))
        return {"op": op, "M": M, "K": K, "N": N, "dtype": dtype, "weight": rng.choice([dtype, dtype, "f32"]),
                "bias": rng.random() < 0.5}
    if op == "polar":
        m, n = _log_int(rng, 8, 4096), _log_int(rng, 8, 4096)
        return {"op": op, "B": _log_int(rng, 1, max(1, min(64, (1 << 31) // (min(m, n) ** 2 * max(m, n))))),
                "m": m, "n": n, "dtype": dtype}
    width = _log_int(rng, 8, 1500)
    return {"op": op, "width": width, "depth": _log_int(rng, 1, 8 if width < 512 else 4), "dtype": dtype}


def _shapes(case):
    """A recurrent network's matrices: an input layer, `depth` blocks of a
    projection to inputs and gates and one back, a head."""
    w = case["width"]
    return [(w, 3)] + [s for _ in range(case["depth"]) for s in ((2 * w, w), (w, w))] + [(49, w)]


def _polar_flops(m, n):
    """Of products X X^T and A A, whose results are symmetric (half of each), and B X."""
    m, n = min(m, n), max(m, n)
    return STEPS * (m * m * n + m ** 3 + 2 * m * m * n)


def work(case):
    op, e = case["op"], {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if op == "quant":
        n, R, D = case["rows"] * case["D"], case["rows"], case["D"]
        codes = n + R * -(-D // BLOCK)
        if case["both"]:
            codes += n + D * -(-R // BLOCK)
        return {"bytes": n * e + codes, "flops": 2 * n}
    if op == "product":
        M, K, N = case["M"], case["K"], case["N"]
        b = -(-K // BLOCK)
        scales = 4 * (M + N) if case["scales"] == "row" else b * (M + N)
        return {"bytes": M * K + N * K + M * N * e + scales + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    if op == "linear":
        M, K, N, f = case["M"], case["K"], case["N"], 4 if case["weight"] == "f32" else e
        # x, dy, weight in; y, dx, the weight's gradient out
        return {"bytes": 2 * M * (K + N) * e + 2 * N * K * f, "flops": 6 * M * N * K}
    if op == "polar":
        m, n = case["m"], case["n"]
        return {"bytes": 2 * case["B"] * m * n * e, "flops": case["B"] * _polar_flops(m, n)}
    n = sum(a * b for a, b in _shapes(case))
    return {"bytes": n * (3 * e + 8), "flops": sum(_polar_flops(a, b) for a, b in _shapes(case))}


# ---- inputs ----------------------------------------------------------------

def _encode(x):
    """(codes [R, K], each row from a multiple of 16 bytes, and the scales'
    exponents + 127, uint8 [R, ceil(K / 128)]) of a float32 matrix."""
    R, K = x.shape
    nb = -(-K // BLOCK)
    p = torch.zeros(R, nb * BLOCK, device=x.device)
    p[:, :K] = x
    p = p.view(R, nb, BLOCK)
    bits = p.abs().amax(2).view(torch.int32)                  # 448 = 1.75 * 2^8
    exp = ((bits + 0x1FFFFF) >> 23) - 127 - 8
    exp = exp.clamp_min(LEAST)
    inv = ((127 - exp) << 23).view(torch.float32)
    q = (p * inv[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(R, nb * BLOCK)
    pitch = -(-K // 16) * 16
    return q[:, :pitch].contiguous()[:, :K], (exp + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def normal(*shape, dtype=t, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(dtype)

    def features(rows, width, dtype=t, scale=1.0):
        """Activations: channels differ in size."""
        return (normal(rows, width, dtype=torch.float32) * normal(width, dtype=torch.float32, scale=0.7).exp()
                * scale).to(dtype)

    op = case["op"]
    if op == "quant":
        return {"case": case, "x": features(case["rows"], case["D"])}
    if op == "product":
        M, K, N = case["M"], case["K"], case["N"]
        x = features(M, K, torch.float32)
        w = normal(N, K, dtype=torch.float32, scale=K ** -0.5)
        s = {"case": case, "bias": normal(N, dtype=torch.float32, scale=0.1) if case["bias"] else None}
        if case["scales"] == "row":     # as an 8-bit norm leaves them: one float32 scale for a row
            for k, v in (("x", x), ("w", w)):
                scale = (v.abs().amax(1) / E4M3_MAX).clamp_min(2.0 ** LEAST)
                s[k] = (v / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
                s[k + "_scale"] = scale
        else:
            for k, v in (("x", x), ("w", w)):
                s[k], exp = _encode(v)
                s[k + "_scale"] = exp.view(torch.float8_e8m0fnu)
        return s
    if op == "linear":
        M, K, N, f = case["M"], case["K"], case["N"], TYPES[case["weight"]]
        s = {"case": case, "x": features(M, K).requires_grad_(True),
             "w": normal(N, K, dtype=f, scale=K ** -0.5).requires_grad_(True),
             "b": normal(N, dtype=f, scale=0.1).requires_grad_(True) if case["bias"] else None}
        s["dy"] = features(M, N, scale=1e-2)
        return s

    def direction(m, n, dtype, scale):
        """A gradient's kind of matrix: a few strong directions and many weak ones."""
        r = min(8, m, n)
        low = normal(m, r, dtype=torch.float32) @ normal(r, n, dtype=torch.float32)
        return ((normal(m, n, dtype=torch.float32) + 0.5 * low) * scale).to(dtype)

    if op == "polar":
        return {"case": case, "x": torch.stack([direction(case["m"], case["n"], t, 1e-3) for _ in range(case["B"])])}
    shapes = _shapes(case)
    return {"case": case, "params": [normal(*s, scale=s[1] ** -0.5) for s in shapes],
            "grads": [direction(*s, t, 10.0 ** -(2 + k % 3)) for k, s in enumerate(shapes)],
            "momenta": [direction(*s, torch.float32, 10.0 ** -(2 + k % 3)) for k, s in enumerate(shapes)]}


# ---- plain forms -----------------------------------------------------------

def _scale_of(exp):
    return (exp.int() << 23).view(torch.float32)


def _wide(scale, K):
    return torch.repeat_interleave(scale, BLOCK, 1)[:, :K]


def _through(x):
    """x [R, K] in float32 as its 8-bit codes stand for it."""
    q, exp = _encode(x)
    return q.float() * _wide(_scale_of(exp), x.shape[1])


def _plain_quant(s):
    x = s["x"].float()
    out = _encode(x)
    return (*out, *_encode(x.t())) if s["case"]["both"] else out


def _plain_product(s):
    c = s["case"]
    x, w = s["x"].float(), s["w"].float()
    if c["scales"] == "row":
        y = (x @ w.t()) * s["x_scale"][:, None] * s["w_scale"]
    else:
        x = x * _wide(_scale_of(s["x_scale"].view(torch.uint8)), c["K"])
        w = w * _wide(_scale_of(s["w_scale"].view(torch.uint8)), c["K"])
        y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(TYPES[c["dtype"]])


def _plain_linear(s):
    x, w, dy = s["x"].detach().float(), s["w"].detach().float(), s["dy"].float()
    y = _through(x) @ _through(w).t()
    if s["b"] is not None:
        y = y + s["b"].detach().float()
    dx = _through(dy) @ _through(w.t()).t()
    dw = _through(dy.t()) @ _through(x.t()).t()
    out = (y.to(s["x"].dtype), dx.to(s["x"].dtype), dw.to(s["w"].dtype))
    return out if s["b"] is None else (*out, dy.sum(0).to(s["b"].dtype))


def _plain_polar(x, t):
    """Newton-Schulz steps towards the orthogonal factor of each matrix of x,
    in 64 bits where the result is kept in 32: five steps multiply what the
    first one rounds away by up to 500."""
    x = x.double() if t == torch.float32 else x.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        A = x @ x.mT
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.mT if tall else x


def _plain_muon(s):
    t = TYPES[s["case"]["dtype"]]
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        g = g.float()
        m.mul_(MOMENTUM).add_(g * (1 - MOMENTUM))
        o = _plain_polar(g * (1 - MOMENTUM) + m * MOMENTUM, t)
        rate = LR * 0.2 * math.sqrt(max(p.shape))
        p.copy_(p.float() * (1 - LR * DECAY) - rate * o)
    return s["params"], s["momenta"]


# ---- one pass --------------------------------------------------------------

def _framework():
    at = os.path.join(os.getcwd(), "fg-cpab_b200")
    if at not in sys.path:
        sys.path.insert(0, at)


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if not own:
        if op == "polar":
            return _plain_polar(s["x"], s["x"].dtype).to(s["x"].dtype)
        return {"quant": _plain_quant, "product": _plain_product, "linear": _plain_linear,
                "muon": _plain_muon}[op](s)
    _framework()
    if op == "quant":
        from cpab.pytorch.projection import quantize_blocks
        out = quantize_blocks(s["x"], transposed=c["both"])
        return tuple(v.view(torch.uint8) if i % 2 else v for i, v in enumerate(out))
    if op == "product":
        from cpab.pytorch.projection import matmul_quantized
        return matmul_quantized(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"],
                                dtype=TYPES[c["dtype"]])
    if op == "linear":
        from cpab.pytorch.projection import linear_quantized
        y = linear_quantized(s["x"], s["w"], s["b"])
        leaves = [s[k] for k in ("x", "w", "b") if s[k] is not None]
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    if op == "polar":
        from cpab.optim import orthogonalize
        return orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    from cpab.optim import muon_
    muon_(s["params"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, nesterov=True,
          coefficients=COEFFICIENTS, eps=NS_EPS, steps=STEPS, adjust_lr="match_rms_adamw")
    return s["params"], s["momenta"]


# ---- the definitions in float64 --------------------------------------------

def _two_to(e):
    """2^e exactly (pow may be off in the last place, which decides ties)."""
    return ((e + 1023) << 52).view(torch.float64)


def _codes64(v):
    """Codes and exponents by the definition: the least power of two s with
    max|v| <= 448 s over each 128 values of a row."""
    R, K = v.shape
    codes = torch.empty(R, K, device=v.device, dtype=torch.float64)
    exps = torch.empty(R, -(-K // BLOCK), device=v.device, dtype=torch.int64)
    for j in range(exps.shape[1]):
        part = v[:, j * BLOCK:(j + 1) * BLOCK]
        most = part.abs().max(1).values
        e = torch.ceil(torch.log2(most / E4M3_MAX)).clamp(LEAST, 127).long()
        e = torch.where(most > E4M3_MAX * _two_to(e), e + 1, e)       # (log2 near a whole number)
        e = torch.where((most <= E4M3_MAX * _two_to(e - 1)) & (e > LEAST), e - 1, e)
        codes[:, j * BLOCK:(j + 1) * BLOCK] = (part * _two_to(-e[:, None])).to(torch.float8_e4m3fn).double()
        exps[:, j] = e
    return codes, exps


def _valued(codes, exps):
    at = torch.arange(codes.shape[1], device=codes.device) // BLOCK
    return codes * _two_to(exps[:, at])


def _exact_quant(s):
    x = s["x"].double()
    codes, exps = _codes64(x)
    out = (codes, exps + 127)
    if s["case"]["both"]:
        codes, exps = _codes64(x.t())
        out = (*out, codes, exps + 127)
    return out


def _exact_product(s):
    if s["case"]["scales"] == "row":
        x = s["x"].double() * s["x_scale"].double()[:, None]
        w = s["w"].double() * s["w_scale"].double()[:, None]
    else:
        x = _valued(s["x"].double(), s["x_scale"].view(torch.uint8).long() - 127)
        w = _valued(s["w"].double(), s["w_scale"].view(torch.uint8).long() - 127)
    y = torch.einsum("mk,nk->mn", x, w)
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_linear(s):
    x, w, dy = s["x"].detach().double(), s["w"].detach().double(), s["dy"].double()
    y = torch.einsum("mk,nk->mn", _valued(*_codes64(x)), _valued(*_codes64(w)))
    dx = torch.einsum("mn,kn->mk", _valued(*_codes64(dy)), _valued(*_codes64(w.t())))
    dw = torch.einsum("nm,km->nk", _valued(*_codes64(dy.t())), _valued(*_codes64(x.t())))
    if s["b"] is None:
        return y, dx, dw
    return y + s["b"].detach().double(), dx, dw, torch.einsum("mn->n", dy)


def _polar64(x):
    """p(X) = a X + b (X X^T) X + c (X X^T)^2 X, on the wide side."""
    a, b, c = COEFFICIENTS
    wide = x.transpose(-1, -2) if x.shape[-2] > x.shape[-1] else x
    X = wide.double() / (torch.linalg.vector_norm(wide.double()) + NS_EPS)
    for _ in range(STEPS):
        gram = X @ X.transpose(-1, -2)
        G1 = gram @ X
        X = a * X + b * G1 + c * (gram @ G1)
    return X.transpose(-1, -2) if x.shape[-2] > x.shape[-1] else X


def _exact_muon(s):
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        g, m = g.double(), m.double()
        m = MOMENTUM * m + (1 - MOMENTUM) * g
        o = _polar64((1 - MOMENTUM) * g + MOMENTUM * m)
        params.append((1 - LR * DECAY) * p.double() - LR * 0.2 * max(p.shape) ** 0.5 * o)
        momenta.append(m)
    return params, momenta


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "polar":
        return torch.stack([_polar64(x) for x in s["x"]])
    return {"quant": _exact_quant, "product": _exact_product, "linear": _exact_linear,
            "muon": _exact_muon}[case["op"]](s)

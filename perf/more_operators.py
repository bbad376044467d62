"""The MLP side of a block between its packed linears, and the int8 product: cases, plain forms and values in 64 bits.

A case is a dict of plain values; `op` is one of
  norm         root-mean-square norm with the residual's addition, the output in 8 bits with a scale a token;
  norm_train   the same norm with a 16-bit output, forward and backward;
  act          gated activation, the output in 8 bits with a scale a token;
  act_train    the activation with a 16-bit output, forward and backward;
  linear       matrix product in 8-bit integers with scales for each token and channel.
`rotate` is the size of the Hadamard rotation that rows go through before they are held in 8 bits (0: none), as for weights
that are stored rotated.  What is held in 8 bits is returned as the values it stands for.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one token of one request: the decode step where latency counts
        {"name": "norm_token", "op": "norm", "tokens": 1, "width": 4096, "residual": True, "rotate": 0, "dtype": "bf16"},
        # image tokens of a diffusion transformer
        {"name": "norm_image", "op": "norm", "tokens": 4608, "width": 6144, "residual": True, "rotate": 0, "dtype": "bf16"},
        # one block in LoRA training, 1056 tokens
        {"name": "norm_train_image", "op": "norm_train", "tokens": 1056, "width": 6144, "residual": True, "dtype": "bf16"},
        # the same for video
        {"name": "norm_train_video", "op": "norm_train", "tokens": 9504, "width": 5120, "residual": True, "dtype": "bf16"},
        # the middle of the MLP for one token
        {"name": "act_token", "op": "act", "tokens": 1, "width": 13824, "gated": True, "act": "silu", "rotate": 0, "dtype": "bf16"},
        # the middle of the MLP for video tokens, before weights that are stored rotated
        {"name": "act_video", "op": "act", "tokens": 9504, "width": 13824, "gated": True, "act": "silu", "rotate": 256,
         "dtype": "fp16"},
        # the wide MLP of an image model in LoRA training
        {"name": "act_train_image", "op": "act_train", "tokens": 1056, "width": 16384, "gated": True, "act": "gelu_tanh",
         "dtype": "bf16"},
        # the same for video
        {"name": "act_train_video", "op": "act_train", "tokens": 9504, "width": 13824, "gated": True, "act": "silu", "dtype": "bf16"},
        # a decode step's linear: one token
        {"name": "linear_token", "op": "linear", "rows": 1, "k": 4096, "n": 4096, "bias": False, "residual": False, "dtype": "bf16"},
        # a small decode batch through the MLP's first linear
        {"name": "linear_batch", "op": "linear", "rows": 8, "k": 5120, "n": 13824, "bias": False, "residual": False, "dtype": "bf16"},
        # a prompt of an odd number of tokens, the residual added
        {"name": "linear_prompt", "op": "linear", "rows": 333, "k": 4096, "n": 4096, "bias": True, "residual": True, "dtype": "fp16"},
        # video tokens through the MLP's first linear
        {"name": "linear_video", "op": "linear", "rows": 9504, "k": 5120, "n": 13824, "bias": True, "residual": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _width(rng, lo, hi):
    """Rows as models have them, and odd ones."""
    kind = rng.random()
    if kind < 0.6:
        return 128 * max(1, _log(rng, lo, hi) // 128)
    return 64 * max(1, _log(rng, lo, hi) // 64) if kind < 0.8 else _log(rng, lo, hi)


def draw(rng):
    """One call of the ranges above: from one token to the largest listed ones, odd sizes, with and without the options."""
    op = rng.choice(("norm", "norm", "norm_train", "act", "act", "act_train", "linear", "linear", "linear"))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "linear":
        rows, k, n = _log(rng, 1, 9504), _width(rng, 256, 16384), _width(rng, 256, 16384)
        while rows * k * n > 9504 * 5120 * 13824:
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "k": k, "n": n, "bias": rng.random() < 0.5, "residual": rng.random() < 0.4, "dtype": dtype}
    width, tokens = _width(rng, 256, 16384), _log(rng, 1, 9504)
    most = 9504 * (5120 if op.startswith("norm") else 13824)
    while tokens * width > most:
        tokens //= 2
    case = {"op": op, "tokens": tokens, "width": width, "dtype": dtype}
    if op.startswith("norm"):
        case.update(residual=rng.random() < 0.8)
    else:
        case.update(gated=rng.random() < 0.8, act=rng.choice(("silu", "silu", "gelu_tanh")))
    if not op.endswith("train"):
        group = rng.choice((0, 0, 64, 128, 256))
        case.update(rotate=group if group and width % group == 0 else 0)
    return case


# ------------------------------------------------------------------------------------------ inputs

def _codes(gen, rows, k, spread):
    """Rows of int8 codes as quantization leaves them: normal values whose largest one is at 127."""
    v = torch.randn(rows, k, generator=gen, device=DEV)
    if spread:  # activations: channels of unequal size
        v *= torch.exp(0.3 * torch.randn(k, generator=gen, device=DEV))
    top = v.abs().amax(-1, keepdim=True)
    return torch.round(v * (127.0 / top)).to(torch.int8), (top / 127.0)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype, s = DTYPES[case["dtype"]], {"case": dict(case)}

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=DEV) * scale

    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        s["x"], s["x_scale"] = _codes(gen, m, k, True)
        s["w"], top = _codes(gen, n, k, False)
        s["w_scale"] = top.reshape(-1) * k ** -0.5
        s["bias"] = normal(n, scale=0.2).to(dtype) if case["bias"] else None
        s["residual"] = normal(m, n).to(dtype) if case["residual"] else None
        return s
    t, w = case["tokens"], case["width"]
    gain = torch.exp(0.3 * normal(w))  # channels of unequal size
    if case["op"].startswith("norm"):
        s["x"] = (normal(t, w) * gain).to(dtype)
        s["residual"] = normal(t, w, scale=2.0).to(dtype) if case["residual"] else None
        s["weight"] = (1 + 0.2 * normal(w)).to(dtype)
        if case["op"] == "norm_train":
            s["dy"], s["dh"] = normal(t, w).to(dtype), normal(t, w).to(dtype)
        return s
    # gate and up as the fused projection leaves them: the halves of one row
    both = (normal(t, 2 * w if case["gated"] else w) * torch.cat([gain, gain] if case["gated"] else [gain])).to(dtype)
    s["gate"], s["up"] = both.split(w, 1) if case["gated"] else (both, None)
    if case["op"] == "act_train":
        s["dy"] = normal(t, w).to(dtype)
    return s


# ------------------------------------------------------------------------------------- plain forms

_H4 = ((1, 1, 1, -1), (1, 1, -1, 1), (1, -1, 1, 1), (-1, 1, 1, 1))


def _hadamard(size, dtype):
    """The orthogonal rotation of `size` values: Kronecker powers of a 4 x 4 Hadamard matrix, with a 2 x 2 one in front where
    size is twice a power of 4."""
    h4 = torch.tensor(_H4, dtype=dtype, device=DEV)
    h = torch.ones(1, 1, dtype=dtype, device=DEV)
    while h.shape[0] * 4 <= size:
        h = torch.kron(h, h4)
    if h.shape[0] < size:
        h = torch.kron(torch.tensor(((1, 1), (1, -1)), dtype=dtype, device=DEV), h)
    return h * size ** -0.5


def _plain_rotated(v, size):
    if not size:
        return v
    return torch.matmul(v.reshape(-1, size), _hadamard(size, v.dtype).T.contiguous()).reshape(v.shape)


def _plain_8bit(v, size):
    """v [tokens, width] held in 8 bits with a scale a token: (the values that stands for, the scales)."""
    v = _plain_rotated(v, size)
    top = v.abs().amax(-1, keepdim=True)
    scale = top / 127
    code = torch.round(v / torch.where(top > 0, scale, 1.0)).clamp(-127, 127)
    return code * scale, scale


def _plain_sum(s):
    return s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()


def _plain_norm(s):
    dtype, h = s["x"].dtype, _plain_sum(s)
    y = h * (h.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["weight"].float()
    y, scale = _plain_8bit(y, s["case"]["rotate"])
    return [y.to(dtype), scale, h.to(dtype)]


def _plain_norm_train(s):
    dtype, h, w = s["x"].dtype, _plain_sum(s), s["weight"].float()
    rstd = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    unit, dy = h * rstd, s["dy"].float()
    g = dy * w
    dx = rstd * (g - unit * (g * unit).mean(-1, keepdim=True)) + s["dh"].float()
    return [(unit * w).to(dtype), h.to(dtype), dx.to(dtype), (dy * unit).sum(0).to(dtype)]


def _plain_f(z, act):
    """(f(z), f'(z)) of z sigma(t): t = z, or the argument of GELU's tanh form doubled."""
    if act == "silu":
        t, dt = z, 1.0
    else:
        c = 2 * math.sqrt(2 / math.pi)
        t, dt = c * (z + 0.044715 * z ** 3), c * (1 + 3 * 0.044715 * z ** 2)
    sig = 1 / (1 + torch.exp(-t))
    return z * sig, sig + z * sig * (1 - sig) * dt


def _plain_act(s):
    y, _ = _plain_f(s["gate"].float(), s["case"]["act"])
    if s["up"] is not None:
        y = y * s["up"].float()
    y, scale = _plain_8bit(y, s["case"]["rotate"])
    return [y.to(s["gate"].dtype), scale]


def _plain_act_train(s):
    dtype, dy = s["gate"].dtype, s["dy"].float()
    f, df = _plain_f(s["gate"].float(), s["case"]["act"])
    if s["up"] is None:
        return [f.to(dtype), (dy * df).to(dtype)]
    up = s["up"].float()
    return [(f * up).to(dtype), (dy * up * df).to(dtype), (dy * f).to(dtype)]


def _plain_linear(s):
    y = torch.matmul(s["x"].float(), s["w"].float().T) * s["x_scale"] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


def _qlin():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-kernels-public_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qlin
    return qlin


def _values(code, scale, dtype):
    """What 8-bit codes [tokens, width] with scales [tokens, 1] stand for."""
    return torch.mul(code, scale, out=torch.empty(code.shape, dtype=dtype, device=code.device))


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"norm": _plain_norm, "norm_train": _plain_norm_train, "act": _plain_act, "act_train": _plain_act_train,
                "linear": _plain_linear}[op](s)
    q = _qlin()
    if op == "norm":
        code, scale, h = q.add_rms_norm_int8(s["x"], s["residual"], s["weight"], eps=EPS, convrot_groupsize=case["rotate"])
        return [_values(code, scale, s["x"].dtype), scale, h]
    if op == "norm_train":
        y, h = q.add_rms_norm(s["x"], s["residual"], s["weight"], eps=EPS)
        return [y, h, *q.add_rms_norm_grad(s["dy"], s["dh"], h, s["weight"], eps=EPS)]
    if op == "act":
        code, scale = q.gated_act_int8(s["gate"], s["up"], act=case["act"], convrot_groupsize=case["rotate"])
        return [_values(code, scale, s["gate"].dtype), scale]
    if op == "act_train":
        y = q.gated_act(s["gate"], s["up"], act=case["act"])
        dgate, dup = q.gated_act_grad(s["dy"], s["gate"], s["up"], act=case["act"])
        return [y, dgate] if dup is None else [y, dgate, dup]
    return q.w8a8_int8_linear(s["x"], s["x_scale"], s["w"], s["w_scale"], s["bias"], DTYPES[case["dtype"]], residual=s["residual"])


def work(case):
    op = case["op"]
    if op == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": m * k + n * k + 2 * m * n * (2 if case["residual"] else 1) + 4 * (m + n) + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    t, w = case["tokens"], case["width"]
    turns = 2 * math.log2(case["rotate"]) if case.get("rotate") else 0  # additions of a fast transform, and the scaling
    if op.startswith("norm"):
        add = 1 if case["residual"] else 0
        if op == "norm":  # x and the residual in, their sum and the codes out
            return {"bytes": t * w * (2 + 4 * add + 1) + 4 * t + 2 * w, "flops": t * w * (7 + turns)}
        # forward: x and the residual in, y and the sum out; backward: dy, dh and the sum in, dx out
        return {"bytes": t * w * (4 + 4 * add + 8) + 6 * w, "flops": 18 * t * w}
    gates = 2 if case["gated"] else 1
    if op == "act":
        return {"bytes": t * w * (2 * gates + 1) + 4 * t, "flops": t * w * (9 + turns)}
    return {"bytes": t * w * 2 * (gates + 1 + 2 * gates + 1), "flops": 25 * t * w}


# ----------------------------------------------------------------------------- the results in 64 bits

def _turned(v, size):
    """v's groups of `size` values through the rotation, one base-4 (and base-2) digit of the index after the other."""
    if not size:
        return v
    shape, digits = v.shape, []
    while size > 1:
        digits.insert(0, 4 if size % 4 == 0 else 2)
        size //= digits[0]
    digits.sort()  # the factor 2 is the most significant digit
    v = v.reshape(-1, *digits)
    for i, d in enumerate(digits):
        at = v.movedim(i + 1, 0)
        if d == 4:
            total = at.sum(0, keepdim=True)
            at = (total - 2 * at.flip(0)) / 2
        else:
            at = torch.stack([at[0] + at[1], at[0] - at[1]]) / math.sqrt(2)
        v = at.movedim(0, i + 1)
    return v.reshape(shape)


def _held(y, size):
    y = _turned(y, size)
    scale = torch.linalg.vector_norm(y, ord=math.inf, dim=-1, keepdim=True) / 127
    return torch.round(y / scale).nan_to_num() * scale, scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        y = s["x"].double() @ s["w"].double().T
        y = y * s["x_scale"].double() * s["w_scale"].double()[None]
        for term in ("bias", "residual"):
            y = y if s[term] is None else y + s[term].double()
        return y
    if op in ("norm", "norm_train"):
        names = [n for n in ("x", "residual", "weight") if s[n] is not None]
        leaf = {n: s[n].double().requires_grad_(op == "norm_train") for n in names}
        h = leaf["x"] + leaf["residual"] if "residual" in leaf else leaf["x"] * 1.0
        y = torch.nn.functional.rms_norm(h, (case["width"],), leaf["weight"], EPS)
        if op == "norm":
            return [*_held(y, case["rotate"]), h]
        dx, dw = torch.autograd.grad((y, h), (leaf["x"], leaf["weight"]), (s["dy"].double(), s["dh"].double()))
        return [y.detach(), h.detach(), dx, dw]
    f = {"silu": torch.nn.functional.silu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[case["act"]]
    gate = s["gate"].double().requires_grad_(op == "act_train")
    up = None if s["up"] is None else s["up"].double().requires_grad_(op == "act_train")
    y = f(gate) if up is None else f(gate) * up
    if op == "act":
        return list(_held(y, case["rotate"]))
    leaves = [gate] if up is None else [gate, up]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"].double())]

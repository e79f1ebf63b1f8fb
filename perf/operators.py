"""The dense gated feed-forward block and the 4-bit microscaled products, as cases that can be prepared and run.

`listed()` holds the calls that a program makes of these operators: single tokens and decode batches, ragged
chunks, prefill batches, training steps, quantisation of activations and of weights, and products with weights
that are kept in 4 bits.  `draw(rng)` gives more of the same ranges.  With `own` false, `run` computes the
operators from elementary operations in 32 bits; with `own` true it calls the package.

Operators (w13 holds the I rows of the gate projection, then the I rows of the up projection):
  ffn       y = (silu(x Wg^T) * (x Wu^T)) W2^T
  train     the same and the gradients of x, w13 and w2 for a given gradient of y
  quantize  x to MX4 and back: blocks of 32 along the row share the scale 2^(floor(log2(max|x|)) - 2), the elements
            are rounded to nearest even on {0, 0.5, 1, 1.5, 2, 3, 4, 6} and saturate at 6
  product   x W^T of x, quantised in the call, and W, kept in MX4
  gated     silu(x Wg^T) * (x Wu^T) of x, quantised in the call, and w13, kept in MX4
"""
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
WEIGHT_STD = 0.02


def _case(op, rows, hidden, inter=0, dtype="bf16", **name):
    """rows x hidden is the shape of x; `inter` is I of the block, or the rows of the weights of a product."""
    return dict(op=op, rows=rows, hidden=hidden, inter=inter, dtype=dtype, **name)


def listed():
    return [
        # one sequence being decoded through a dense block: the weights are read once for one token
        _case("ffn", 1, 2048, 6144, name="ffn_decode_1"),
        # a decode batch through a large block
        _case("ffn", 32, 4096, 12288, name="ffn_decode_32"),
        # a ragged chunk of a prefill through a shared expert (the small layer's expert size), fp16 weights
        _case("ffn", 333, 2048, 768, dtype="fp16", name="ffn_chunk_333_fp16"),
        # a prefill batch through a large block
        _case("ffn", 8192, 4096, 12288, name="ffn_prefill_8192"),
        # a training step of a small block with odd sizes
        _case("train", 777, 1000, 2744, dtype="fp16", name="train_777_fp16"),
        # a training step: 4096 tokens, all gradients
        _case("train", 4096, 2048, 6144, name="train_4096"),
        # activations of a decode batch
        _case("quantize", 16, 4096, name="quantize_16"),
        # a weight matrix or the activations of a long prefill
        _case("quantize", 16384, 4096, name="quantize_16384"),
        # one token times a down projection kept in 4 bits
        _case("product", 1, 12288, 4096, name="product_decode_1"),
        # a prefill batch times a square projection kept in 4 bits
        _case("product", 8192, 4096, 4096, name="product_prefill_8192"),
        # a decode batch through the gate and up projections of a large block kept in 4 bits
        _case("gated", 64, 4096, 12288, name="gated_decode_64"),
        # an odd number of tokens and ragged sizes, fp16 in and out
        _case("gated", 1531, 2080, 1544, dtype="fp16", name="gated_1531_fp16"),
    ]


def _spread(rng, low, high, step):
    """A multiple of `step` between low and high, spread over the logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random() / step) * step))


def draw(rng: random.Random):
    op = rng.choice(["ffn", "ffn", "train", "quantize", "product", "gated"])
    if op == "quantize":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return _case(op, _spread(rng, 1, 16384, 1), _spread(rng, 32, 12288, 32), dtype=dtype)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("product", "gated"):
        return _case(op, _spread(rng, 1, 8192, 1), _spread(rng, 256, 12288 if op == "product" else 4096, 32),
                     _spread(rng, 256, 4096 if op == "product" else 12288, 8), dtype=dtype)
    return _case(op, _spread(rng, 1, 8192 if op == "ffn" else 4096, 1), _spread(rng, 256, 4096, 8),
                 _spread(rng, 256, 12288 if op == "ffn" else 6144, 8), dtype=dtype)


def _inputs(case, seed):
    """The tensors of a case: x, then weights, then the gradient of the output, as far as the operator has them."""
    dev, dtype = torch.device("cuda"), _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    rows, hidden, inter = case["rows"], case["hidden"], case["inter"]

    def normal(*shape, std):
        return torch.empty(*shape, dtype=torch.float32, device=dev).normal_(0.0, std, generator=g).to(dtype)

    x = normal(rows, hidden, std=1.0)
    if case["op"] == "quantize":
        return dict(x=x)
    if case["op"] == "product":
        return dict(x=x, w=normal(inter, hidden, std=WEIGHT_STD))
    if case["op"] == "gated":
        return dict(x=x, w=normal(2, inter, hidden, std=WEIGHT_STD))
    t = dict(x=x, w13=normal(2 * inter, hidden, std=WEIGHT_STD), w2=normal(hidden, inter, std=WEIGHT_STD))
    if case["op"] == "train":
        t["dy"] = normal(rows, hidden, std=1.0)
    return t


# ------------------------------------------------------------------ plain forms
def _plain_mx4(x):
    """What x stands for after quantisation to MX4, in 32 bits (64 inside: values next to a border)."""
    v = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    exponent = torch.frexp(v.abs().amax(-1, keepdim=True)).exponent.long() - 3  # floor(log2) is frexp's less 1
    exponent = exponent.clamp(-127, 127)
    scale = ((exponent + 1023) << 52).view(torch.float64)
    m = (v / scale).abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    q = (torch.round(m / step) * step).clamp(max=6.0)
    return (torch.copysign(q, v) * scale).reshape(x.shape).float()


def _plain_ffn(x, w13, w2):
    inter = w2.shape[1]
    x, w13, w2 = x.float(), w13.float(), w2.float()
    gu = x @ w13.t()
    g, u = gu[:, :inter], gu[:, inter:]
    s = 1.0 / (1.0 + torch.exp(-g))
    h = g * s * u
    return x, w13, w2, g, u, s, h, h @ w2.t()


def _plain_train(x, w13, w2, dy):
    dtype = x.dtype
    x, w13, w2, g, u, s, h, y = _plain_ffn(x, w13, w2)
    dy = dy.float()
    dh = dy @ w2
    dgu = torch.cat([dh * u * s * (1.0 + g * (1.0 - s)), dh * g * s], dim=1)
    out = [y, dgu @ w13, dgu.t() @ x, dy.t() @ h]
    return [t.to(dtype) for t in out]


def _plain(state):
    case, t = state.case, state.tensors
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "ffn":
        return _plain_ffn(t["x"], t["w13"], t["w2"])[-1].to(dtype)
    if case["op"] == "train":
        return _plain_train(t["x"], t["w13"], t["w2"], t["dy"])
    x = _plain_mx4(t["x"])
    if case["op"] == "quantize":
        return x.to(dtype)
    if case["op"] == "product":
        return (x @ state.weights.t()).to(dtype)
    g, u = x @ state.weights[0].t(), x @ state.weights[1].t()
    return (g / (1.0 + torch.exp(-g)) * u).to(dtype)


# --------------------------------------------------------------- prepare and run
class State:
    """What a program has in hand: the tensors, and the weights in the form in which it keeps them."""

    def __init__(self, case, tensors, weights):
        self.case, self.tensors, self.weights = case, tensors, weights


def prepare(case, seed):
    t = _inputs(case, seed)
    weights = None
    if "w" in t:  # weights kept in 4 bits; the plain form keeps the values that they stand for
        if own:
            from flash_distributed_moe_b200 import mx4_quantize
            weights = mx4_quantize(t.pop("w"))
        else:
            weights = _plain_mx4(t.pop("w"))
    if case["op"] == "train":
        for name in ("x", "w13", "w2"):
            t[name].requires_grad_(own)
    return State(case, t, weights)


def run(state):
    if not own:
        return _plain(state)
    import flash_distributed_moe_b200 as fm
    t, op = state.tensors, state.case["op"]
    if op == "ffn":
        return fm.gated_ffn(t["x"], t["w13"], t["w2"])
    if op == "train":
        y = fm.gated_ffn(t["x"], t["w13"], t["w2"])
        return [y.detach(), *torch.autograd.grad(y, (t["x"], t["w13"], t["w2"]), t["dy"])]
    q = fm.mx4_quantize(t["x"])
    if op == "quantize":
        return q.dequantize(t["x"].dtype)
    if op == "product":
        return fm.mx4_matmul(q, state.weights, t["x"].dtype)
    return fm.mx4_gated_matmul(q, state.weights, t["x"].dtype)


# ------------------------------------------------------------- the definition in 64 bits
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_mx4(x):
    """Nearest grid point by comparing with the borders between them; a value on a border goes to the even code."""
    v = x.double().unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp_min(2.0 ** -125))) - 2)  # float16 and the normal range of the others
    scale = torch.where(top >= scale * 8, scale * 2, torch.where(top < scale * 4, scale / 2, scale))
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    m = v.abs() / scale
    code = torch.zeros_like(m)
    for i in range(7):
        border = (_GRID[i] + _GRID[i + 1]) / 2
        code += (m > border) if i % 2 == 0 else (m >= border)  # the lower code is even: the border itself stays below
    q = torch.tensor(_GRID, dtype=torch.float64, device=x.device)[code.long()]
    return (torch.sign(v) * q * scale).flatten(-2)


def exact(case, seed):
    t = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_mx4(t["x"])
    silu = torch.nn.functional.silu
    if op == "product":
        return torch.nn.functional.linear(_exact_mx4(t["x"]), _exact_mx4(t["w"]))
    if op == "gated":
        x, w = _exact_mx4(t["x"]), _exact_mx4(t["w"])
        return silu(torch.nn.functional.linear(x, w[0])) * torch.nn.functional.linear(x, w[1])
    x, w13, w2 = (t[n].double().requires_grad_(op == "train") for n in ("x", "w13", "w2"))
    g, u = torch.nn.functional.linear(x, w13).chunk(2, dim=-1)
    y = torch.nn.functional.linear(silu(g) * u, w2)
    if op == "ffn":
        return y
    return [y.detach(), *torch.autograd.grad(y, (x, w13, w2), t["dy"].double())]


def work(case):
    rows, hidden, inter = case["rows"], case["hidden"], case["inter"]
    size = 4 if case["dtype"] == "fp32" else 2
    mx4 = 17 / 32  # bytes of an element with its share of the scale
    x = rows * hidden * size
    if case["op"] == "quantize":  # x is read, its 4-bit form written, and the values it stands for
        return {"bytes": 2 * x + rows * hidden * mx4, "flops": 0}
    if case["op"] == "product":
        return {"bytes": x + inter * hidden * mx4 + rows * inter * size, "flops": 2 * rows * inter * hidden}
    if case["op"] == "gated":
        return {"bytes": x + 2 * inter * hidden * mx4 + rows * inter * size, "flops": 4 * rows * inter * hidden}
    if case["op"] == "ffn":  # x and the weights in, y out
        return {"bytes": 2 * x + 3 * hidden * inter * size, "flops": 6 * rows * hidden * inter}
    # x, dy and the weights in, y and the gradients out
    return {"bytes": 4 * x + 6 * hidden * inter * size, "flops": 18 * rows * hidden * inter}

"""The low-bit operators of the policy's trunk: what is measured of them, in their plain form and as the framework's calls.

Four operators, all on blocks of 32 values that share a power-of-two scale (stored as its biased exponent, one byte;
255 marks a block that holds a NaN or an infinity):

  quantize     4-bit floats (e2m1: 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), scale 2^(floor(log2 max|x|) - 2),
               nearest value, ties to the even code, above 6 to 6
  linear       x in 4 bits times a weight that is kept in 4 bits, plus bias, ReLU if asked
  compress     8-bit integers, the smallest scale with which no |code| passes 127 (255 where no value is negative)
  weight_grad  the parameter gradients of a linear layer whose input was kept in 8 bits: grad^T x, the column sums of
               grad, and grad itself, where a ReLU stood behind the layer with grad cut where its output's code is 0
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = 32


def listed():
    return [
        # a policy's first layer, quantised anew after every update: 202 features, 512 units
        {"name": "quantize_weight_512x202", "op": "quantize", "rows": 512, "cols": 202, "type": "f32", "values": "weight"},
        # the observations of 65,536 two-agent kitchens
        {"name": "quantize_obs_131072x202", "op": "quantize", "rows": 131072, "cols": 202, "type": "f32", "values": "obs"},
        # one rollout step at 16 envs with two agents, where only the call's latency counts
        {"name": "linear_32x202x512", "op": "linear", "rows": 32, "cols": 202, "out": 512, "type": "f32", "values": "obs", "relu": True},
        # the trunk's two layers at 65,536 envs
        {"name": "linear_131072x202x512", "op": "linear", "rows": 131072, "cols": 202, "out": 512, "type": "f32", "values": "obs", "relu": True},
        {"name": "linear_131072x512x256", "op": "linear", "rows": 131072, "cols": 512, "out": 256, "type": "f32", "values": "hidden", "relu": True},
        # four agents' observations (420 features) of a batch that no tile divides, in bfloat16, without ReLU
        {"name": "linear_bf16_21847x420x250", "op": "linear", "rows": 21847, "cols": 420, "out": 250, "type": "bf16", "values": "obs", "relu": False},
        # the centralised critic: one row of all observations of 2,048 two-agent envs
        {"name": "linear_joint_1x827392x512", "op": "linear", "rows": 1, "cols": 827392, "out": 512, "type": "f32", "values": "obs", "relu": True},
        # a minibatch of 16 envs' rollouts: the first layer's input
        {"name": "compress_obs_2048x202", "op": "compress", "rows": 2048, "cols": 202, "type": "f32", "values": "obs", "positive": False},
        # the hidden layer of a large minibatch, behind its ReLU
        {"name": "compress_hidden_131072x512", "op": "compress", "rows": 131072, "cols": 512, "type": "f32", "values": "hidden", "positive": True},
        # the first layer's gradient in the small minibatch, the second's in the large one, and the two heads' (7 logits and a value)
        {"name": "weight_grad_2048x512x202", "op": "weight_grad", "rows": 2048, "out": 512, "cols": 202, "type": "f32", "values": "obs", "positive": False, "relu": True},
        {"name": "weight_grad_131072x256x512", "op": "weight_grad", "rows": 131072, "out": 256, "cols": 512, "type": "f32", "values": "hidden", "positive": True, "relu": True},
        {"name": "weight_grad_bf16_65000x8x256", "op": "weight_grad", "rows": 65000, "out": 8, "cols": 256, "type": "bf16", "values": "hidden", "positive": True, "relu": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "linear", "compress", "weight_grad", "weight_grad"))
    case = {"op": op, "type": rng.choice(("f32", "f32", "bf16", "f16")), "values": rng.choice(("obs", "hidden", "normal"))}
    rows, cols, out = _log(rng, 1, 131072), _log(rng, 5, 512), _log(rng, 1, 512)
    if op == "linear" and rng.random() < 0.25:  # few rows of very many features: a joint observation
        rows, cols = rng.randint(1, 8), _log(rng, 1000, 400000)
    if op in ("linear", "weight_grad"):
        rows = min(rows, max(1, 131072 * 512 * 256 // (cols * out)))
        case.update(out=out, relu=rng.random() < 0.5)
    if op in ("compress", "weight_grad"):
        case["positive"] = case["values"] == "hidden"
    case.update(rows=rows, cols=cols)
    return case


def _values(rows, cols, kind, g):
    """float32 [rows, cols]: small whole numbers, mostly 0 (`obs`: the encoders' distances, counts and flags), what a ReLU
    leaves (`hidden`), weights as they are initialised, or both signs at sizes that differ from row to row (`normal`)"""
    if kind == "obs":
        x = torch.randn((rows, cols), device="cuda", generator=g)
        return (x.abs() > 0.9).float() * (x * 1.3).round()
    x = torch.randn((rows, cols), device="cuda", generator=g)
    if kind == "weight":
        return x * (2.0 / max(cols, 512)) ** 0.5
    size = torch.exp(0.7 * torch.randn((rows, 1), device="cuda", generator=g))
    return torch.relu(x * size) if kind == "hidden" else x * size


def _two(e):
    """2^e exactly, from the bits (e: int32 tensor in [-126, 127])"""
    return ((e + 127) << 23).view(torch.float32)


def _grid4(x):
    """float32 [n, BLOCK]: -> (codes 0..15, exponents [n, 1])"""
    top = x.abs().amax(1, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(-126, 125)
    v = (x * _two(-e)).abs().clamp(max=6.0)
    half = torch.where(v < 2.0, (v * 2.0).round(), torch.where(v < 4.0, v.round() + 2.0, (v * 0.5).round() + 4.0))
    return half.to(torch.uint8) | ((x < 0).to(torch.uint8) << 3), torch.where(top > 0, e, torch.full_like(e, -126))


def _blocks(x):
    rows, cols = x.shape
    n = -(-cols // BLOCK)
    return torch.nn.functional.pad(x, (0, n * BLOCK - cols)).view(rows * n, BLOCK), n


def _pack4(w):
    """a weight as a user's program keeps it: codes uint8 [rows, 16 * blocks] (low half first), scales uint8 [rows, blocks]"""
    x, n = _blocks(w)
    codes, e = _grid4(x)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).view(w.shape[0], n * 16), (e + 127).to(torch.uint8).view(w.shape[0], n)


def _pack8(x, positive):
    """an activation as it was kept: codes uint8 [rows, cols] (plus 128 where there are negative ones), scales uint8 [rows, blocks]"""
    v, e, n = _grid8(x, positive)
    codes = (v + (0.0 if positive else 128.0)).to(torch.uint8).view(x.shape[0], n * BLOCK)[:, :x.shape[1]].contiguous()
    return codes, (e + 127).to(torch.uint8).view(x.shape[0], n)


def _grid8(x, positive):
    x, n = _blocks(x)
    most = 255.0 if positive else 127.0
    top = x.abs().amax(1, keepdim=True)
    e = torch.frexp(top).exponent - (8 if positive else 7)
    e = e.clamp(-126, 126)
    e = torch.where(top * _two(-e) >= most + 0.5, e + 1, e)
    v = (x * _two(-e)).round()
    if positive:
        v = torch.where(x > 0, v.clamp(min=1.0), torch.zeros_like(v))
    return v, torch.where(top > 0, e, torch.full_like(e, -126)), n


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, kind = case["rows"], case["cols"], TYPES[case["type"]]
    x = _values(rows, cols, case["values"], g).to(kind)
    state = {"op": case["op"], "cols": cols, "type": kind}
    if case["op"] == "quantize":
        state["x"] = x
    elif case["op"] == "linear":
        codes, scales = _pack4(_values(case["out"], cols, "weight", g))
        state.update(x=x, codes=codes, scales=scales, relu=case["relu"], bias=0.1 * torch.randn(case["out"], device="cuda", generator=g))
    elif case["op"] == "compress":
        state.update(x=x, positive=case["positive"])
    else:
        codes, scales = _pack8(x.float(), case["positive"])
        # a mean loss over the rows: gradients of a few samples are many times the others'
        size = torch.exp(torch.randn((rows, 1), device="cuda", generator=g)) * (64.0 if kind == torch.float16 else 1.0) / rows
        grad = torch.randn((rows, case["out"]), device="cuda", generator=g) * size
        state.update(codes=codes, scales=scales, positive=case["positive"], grad=grad.to(kind), kept=None)
        if case["relu"]:  # the layer's own output, kept in 8 bits: its codes say where the ReLU let the gradient through
            kept = torch.relu(torch.randn((rows, case["out"]), device="cuda", generator=g))
            state["kept"], state["kept_scales"] = _pack8(kept, True)
    return state


def _two_to(scales, rows):
    return _two(scales.view(rows, -1, 1).int() - 127)


def _dense4(codes, scales, cols):
    """float32 values of a packed 4-bit tensor"""
    value = torch.tensor(VALUES + tuple(-v for v in VALUES), device=codes.device)
    pairs = torch.stack((value.repeat(16), value.repeat_interleave(16)), 1)  # both halves of every byte
    rows = codes.shape[0]
    return (pairs[codes.int()].view(rows, -1, BLOCK) * _two_to(scales, rows)).view(rows, -1)[:, :cols]


def _dense8(codes, scales, positive):
    rows, cols = codes.shape
    n = scales.shape[1]
    v = torch.nn.functional.pad(codes.float() - (0.0 if positive else 128.0), (0, n * BLOCK - cols))
    return (v.view(rows, n, BLOCK) * _two_to(scales, rows)).view(rows, -1)[:, :cols]


def _round4(x):
    """x to the nearest 4-bit values"""
    rows, cols = x.shape
    b, n = _blocks(x.float())
    e = (torch.frexp(b.abs().amax(1, keepdim=True)).exponent - 3).clamp(-126, 125)
    v = b * _two(-e)
    a = v.abs().clamp(max=6.0)
    a = torch.where(a < 2.0, (a * 2.0).round() * 0.5, torch.where(a < 4.0, a.round(), (a * 0.5).round() * 2.0))
    return (torch.copysign(a, v) * _two(e)).view(rows, n * BLOCK)[:, :cols]


def run(state):
    op = state["op"]
    if own:
        from marl_amd import act8, mxfp4

        if op == "quantize":
            return mxfp4.quantize(state["x"]).dequantize()
        if op == "linear":
            weight = mxfp4.MXFP4(state["codes"], state["scales"], state["cols"])
            return mxfp4.linear(state["x"], weight, state["bias"], relu=state["relu"], out_dtype=state["type"])
        if op == "compress":
            return act8.compress(state["x"], nonnegative=state["positive"]).dequantize()
        kept = None if state["kept"] is None else act8.Act8(state["kept"], state["kept_scales"], True)
        return act8.weight_grad(state["grad"], act8.Act8(state["codes"], state["scales"], state["positive"]), mask=kept)
    if op == "quantize":
        return _round4(state["x"])
    if op == "linear":
        y = _round4(state["x"]) @ _dense4(state["codes"], state["scales"], state["cols"]).t() + state["bias"]
        return (torch.relu(y) if state["relu"] else y).to(state["type"])
    if op == "compress":
        x = state["x"].float()
        v, e, n = _grid8(x, state["positive"])
        return (v * _two(e)).view(x.shape[0], n * BLOCK)[:, :x.shape[1]]
    grad, kept = state["grad"], state["kept"]
    if kept is not None:
        grad = torch.where(kept > 0, grad, torch.zeros((), dtype=grad.dtype, device=grad.device))
    wide = grad.float()
    return wide.t() @ _dense8(state["codes"], state["scales"], state["positive"]), wide.sum(0), None if kept is None else grad


def work(case):
    rows, cols, op = case["rows"], case["cols"], case["op"]
    n, size = -(-cols // BLOCK), 4 if case["type"] == "f32" else 2
    if op in ("quantize", "compress"):
        return {"bytes": rows * cols * (size + 4), "flops": rows * cols}
    out = case["out"]
    flops = 2 * rows * cols * out
    if op == "linear":
        return {"bytes": rows * cols * size + out * n * 17 + out * 4 + rows * out * size, "flops": flops}
    masked = rows * out * (1 + size) if case["relu"] else 0
    return {"bytes": rows * out * size + rows * (cols + n) + masked + out * cols * 4 + out * 4, "flops": flops}


def exact(case, seed):
    """From the definitions in 64 bits: 4-bit values by counting the borders between neighbours, 8-bit ones by division."""
    s = prepare(case, seed)
    op = s["op"]

    def power_of_two(e):  # from the bits: pow() may be off by one
        return ((e.long() + 1023) << 52).view(torch.float64)

    def blocks(t):
        t = t.double()
        pad = torch.zeros((t.shape[0], -t.shape[1] % BLOCK), dtype=torch.float64, device="cuda")
        t = torch.cat((t, pad), 1).reshape(t.shape[0], -1, BLOCK)
        top = t.abs().max(2, keepdim=True).values
        return t, top, torch.frexp(top).exponent - 1

    def four(t):
        v, top, power = blocks(t)
        scale = power_of_two(torch.where(top > 0, power - 2, torch.zeros_like(power)).clamp(min=-126))
        grid = torch.tensor(VALUES, dtype=torch.float64, device="cuda")
        border = (grid[1:] + grid[:-1]) / 2
        size = (v / scale).abs()
        below, upto = torch.bucketize(size, border), torch.bucketize(size, border, right=True)
        index = torch.where((upto > below) & (below % 2 == 1), upto, below)
        return (grid[index] * torch.sign(v) * scale).flatten(1)[:, :t.shape[1]]

    if op == "quantize":
        return four(s["x"])
    if op == "linear":
        high, low = (s["codes"] // 16).long(), (s["codes"] % 16).long()
        code = torch.stack((low, high), 2).view(case["out"], -1, BLOCK)
        value = torch.tensor(VALUES, dtype=torch.float64, device="cuda")[code % 8] * (1 - 2 * (code // 8)).double()
        w = (value * power_of_two(s["scales"].int() - 127)[:, :, None]).flatten(1)[:, :case["cols"]]
        y = four(s["x"]) @ w.t() + s["bias"].double()
        return y.clamp(min=0) if case["relu"] else y
    if op == "compress":
        v, top, power = blocks(s["x"])
        most = 255 if s["positive"] else 127
        e = power - (7 if s["positive"] else 6)
        e = torch.where((top / power_of_two(e)).round() > most, e + 1, e)
        scale = power_of_two(torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=-126))
        code = (v / scale).round()
        if s["positive"]:
            code = torch.maximum(code, (v > 0).double())
        return (code * scale).flatten(1)[:, :case["cols"]]
    scale = power_of_two(s["scales"].int() - 127).repeat_interleave(BLOCK, 1)[:, :case["cols"]]
    x = (s["codes"].double() - (0 if s["positive"] else 128)) * scale
    grad = s["grad"].double()
    if s["kept"] is not None:
        grad = grad * (s["kept"] != 0)
    return grad.t() @ x, grad.sum(0), None if s["kept"] is None else grad

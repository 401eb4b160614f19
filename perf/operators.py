"""Measured cases of the operators around a Dense layer with 4-bit operands: layer norm and the MXFP4 format.

A case is one of six kinds of work, each of them a call or a short sequence of calls as a user's program makes them:

  layer_norm           Tensor.layer_norm of a matrix's rows; for training the rows' means and reciprocal deviations too
  layer_norm_backward  the gradients with respect to input, weight and bias, from the statistics that the forward pass saved
  mx_round_trip        Tensor.quantize_mxfp4 along an axis and MxTensor.dequantize: what a tensor is worth in 4 bits
  mx_dot               MxTensor.dot of two operands quantised before
  mx_dense             MxDense.forward: activations quantised along their rows, times a weight quantised once, with bias and relu
  mx_dense_backward    the two products of a Dense layer's backward edge in 4 bits: dx = dy.W^T, dW = x^T.dy, all four operands quantised

MXFP4: blocks of 32 values along the reduction share a scale 2^s, s = floor(log2(largest magnitude)) - 2 held to [-127, 127]; a value is
rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale (half to even, larger ones to 6).  The last block of a row may be short.

Inputs are seeded and made on the GPU.  The plain forms are elementary torch operations in 32 bits.
"""
import math

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
_EPS = 1e-5


def listed():
    return [
        # one token's activations in front of a layer: latency alone
        {"name": "layer_norm_bf16_1x4096", "kind": "layer_norm", "dtype": "bf16", "rows": 1, "cols": 4096, "stats": False},
        # the large layer's input, training
        {"name": "layer_norm_bf16_16384x4096", "kind": "layer_norm", "dtype": "bf16", "rows": 16384, "cols": 4096, "stats": True},
        # ragged rows in front of a classifier head, inference in f32
        {"name": "layer_norm_f32_1999x1001", "kind": "layer_norm", "dtype": "f32", "rows": 1999, "cols": 1001, "stats": False},
        # training of the large layer
        {"name": "layer_norm_backward_bf16_16384x4096", "kind": "layer_norm_backward", "dtype": "bf16", "rows": 16384, "cols": 4096},
        # training of a small network at the batch size that the benchmark uses
        {"name": "layer_norm_backward_f32_100x84", "kind": "layer_norm_backward", "dtype": "f32", "rows": 100, "cols": 84},
        # the large layer's activations along their rows
        {"name": "mx_round_trip_bf16_16384x4096_rows", "kind": "mx_round_trip", "dtype": "bf16", "rows": 16384, "cols": 4096, "axis": 1},
        # a weight of ragged sizes along its columns
        {"name": "mx_round_trip_f32_2047x1001_columns", "kind": "mx_round_trip", "dtype": "f32", "rows": 2047, "cols": 1001, "axis": 0},
        # the square product that fills the chip
        {"name": "mx_dot_bf16_8192", "kind": "mx_dot", "dtype": "bf16", "m": 8192, "k": 8192, "n": 8192},
        # the large layer serving one request
        {"name": "mx_dense_bf16_1x4096x4096", "kind": "mx_dense", "dtype": "bf16", "m": 1, "k": 4096, "n": 4096, "relu": True},
        # the large layer in bulk inference
        {"name": "mx_dense_bf16_16384x4096x4096", "kind": "mx_dense", "dtype": "bf16", "m": 16384, "k": 4096, "n": 4096, "relu": True},
        # a classifier head of ragged sizes
        {"name": "mx_dot_f32_1999x2047x1001", "kind": "mx_dot", "dtype": "f32", "m": 1999, "k": 2047, "n": 1001},
        # training of a mid-sized layer
        {"name": "mx_dense_backward_bf16_4096x2048x1000", "kind": "mx_dense_backward", "dtype": "bf16", "m": 4096, "k": 2048, "n": 1000},
    ]


# ---- the ranges: sizes, types and options that the kinds above are used with ----

_KINDS = ("layer_norm", "layer_norm_backward", "mx_round_trip", "mx_dot", "mx_dense", "mx_dense_backward")


def _log_size(rng, lo, hi):
    """Log-uniform; half of the sizes are whole multiples of 32, the others are left as they fall, odd ones among them."""
    v = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v // 32 * 32 if v >= 32 and rng.random() < 0.5 else v


def _draw_one(rng):
    kind = rng.choice(_KINDS)
    case = {"kind": kind, "dtype": rng.choice(("f32", "bf16"))}
    if kind.startswith("layer_norm"):
        case.update(rows=_log_size(rng, 1, 16384), cols=_log_size(rng, 16, 16384))
        if kind == "layer_norm":
            case.update(stats=rng.random() < 0.5)
    elif kind == "mx_round_trip":
        case.update(rows=_log_size(rng, 1, 16384), cols=_log_size(rng, 16, 16384), axis=rng.choice((0, 1)))
    else:
        case.update(m=_log_size(rng, 1, 16384), k=_log_size(rng, 16, 16384), n=_log_size(rng, 10, 16384))
        if kind == "mx_dense":
            case.update(relu=rng.random() < 0.5)
    return case


def _cost(case):
    """Seconds at everyday rates: the measure by which a drawn case is kept below the largest listed one."""
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 3e15)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw_one(rng)
        if _cost(case) <= most:
            return case


# ---- inputs ----


class _Random:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, shape, std, dtype):
        return (torch.randn(shape, generator=self.gen, device="cuda") * std).to(_TORCH[dtype])

    def activation(self, rows, cols, dtype):
        """Hidden activations: channels of different spread and offset, one in sixty-four or so several times larger."""
        spread = torch.exp(0.5 * torch.randn(cols, generator=self.gen, device="cuda"))
        spread = torch.where(torch.rand(cols, generator=self.gen, device="cuda") < 1 / 64, 8 * spread, spread)
        x = torch.randn((rows, cols), generator=self.gen, device="cuda") * spread
        return (x + 0.3 * torch.randn(cols, generator=self.gen, device="cuda")).to(_TORCH[dtype])


def _inputs(case, seed):
    """The tensors of a case by name, on the GPU."""
    r, dt, kind = _Random(seed), case["dtype"], case["kind"]
    if kind.startswith("layer_norm"):
        rows, cols = case["rows"], case["cols"]
        t = {"x": r.activation(rows, cols, dt), "w": 1 + r.normal((cols,), 0.1, dt)}
        if kind == "layer_norm":
            t["b"] = r.normal((cols,), 0.1, dt)
        else:
            t["dy"] = r.normal((rows, cols), 1, dt)
            x = t["x"].float()
            t["mean"] = x.double().mean(1).float()
            t["rstd"] = (x.double().var(1, correction=0) + _EPS).rsqrt().float()
        return t
    if kind == "mx_round_trip":
        return {"x": r.activation(case["rows"], case["cols"], dt)}
    m, k, n = case["m"], case["k"], case["n"]
    t = {"x": r.activation(m, k, dt), "w": r.normal((k, n), math.sqrt(2 / k), dt)}
    if kind == "mx_dense":
        t["b"] = r.normal((n,), 0.1, dt)
    elif kind == "mx_dense_backward":
        t["dy"] = r.normal((m, n), 1 / m, dt)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _Program(case, t)
    # operands that a program quantises once are held as 4-bit codes and scales
    if case["kind"] == "mx_dot":
        return case, {"x": _mx(t["x"]), "w": _mx(t["w"].t())}
    if case["kind"] == "mx_dense":
        return case, {**t, "w": _mx(t["w"].t())}
    return case, t


# ---- the framework's calls ----


class _Memory:
    """A framework tensor's memory as torch reads it; holds the tensor, so the memory lives as long as torch's view."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.__cuda_array_interface__ = {
            "shape": tensor.shape, "typestr": "<f4" if tensor.dtype == "f32" else "<i2",
            "strides": tuple(s * _SIZE[tensor.dtype] for s in tensor.strides), "data": (tensor._data_ptr(), False), "version": 2}


def _torch(tensor):
    view = torch.as_tensor(_Memory(tensor), device="cuda")
    return view if tensor.dtype == "f32" else view.view(torch.bfloat16)


class _Program:
    """What a program that uses the framework has in hand: the same inputs as framework tensors, weights quantised once."""

    def __init__(self, case, tensors):
        import autograph_amd as ag
        from autograph_amd._ffi import check, lib

        ag.Device(0)
        torch.cuda.synchronize()
        t = {}
        for name, values in tensors.items():
            t[name] = ag.Tensor.uninit(tuple(values.shape), "bf16" if values.dtype == torch.bfloat16 else "f32")
            check(lib.agh_memcpy_d2d(t[name]._ptr(), values.data_ptr(), values.numel() * values.element_size()))
        check(lib.agh_sync())
        if case["kind"] == "mx_dot":
            t = {"x": t["x"].quantize_mxfp4(axis=1), "w": t["w"].quantize_mxfp4(axis=0)}
        elif case["kind"] == "mx_dense":
            t["layer"] = ag.Dense(t["w"], t["b"]).quantize_mxfp4()
        elif case["kind"] == "layer_norm":
            t["layer"] = ag.LayerNorm(t["w"], t["b"], _EPS)
        self.case, self.tensors = case, t

    def run(self):
        case, t = self.case, self.tensors
        kind, dt = case["kind"], case["dtype"]
        if kind == "layer_norm":
            y = t["layer"].forward_train(t["x"]) if case["stats"] else (t["layer"].forward(t["x"]),)
        elif kind == "layer_norm_backward":
            y = t["x"].layer_norm_backward(t["dy"], t["w"], t["mean"], t["rstd"])
        elif kind == "mx_round_trip":
            y = (t["x"].quantize_mxfp4(axis=case["axis"]).dequantize(dt),)
        elif kind == "mx_dot":
            y = (t["x"].dot(t["w"], dtype=dt),)
        elif kind == "mx_dense":
            y = (t["layer"].forward(t["x"], relu=case["relu"]),)
        else:
            dx = t["dy"].quantize_mxfp4(axis=1).dot(t["w"].quantize_mxfp4(axis=1).t(), dtype=dt)
            dw = t["x"].quantize_mxfp4(axis=0).t().dot(t["dy"].quantize_mxfp4(axis=0), dtype=dt)
            y = (dx, dw)
        return [_torch(v) for v in y]


# ---- the plain forms ----

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_tables = {}


def _table():
    """The values of the sixteen codes, of the 256 scale bytes (255: NaN) and their reciprocals."""
    if not _tables:
        _tables["codes"] = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device="cuda")
        scales = torch.tensor([2.0 ** (s - 127) for s in range(255)] + [math.nan], dtype=torch.float64, device="cuda")
        _tables["scales"], _tables["reciprocals"] = scales.float(), (1 / scales).float()
    return _tables


def _mx_parts(x):
    """The rows of x in blocks of 32, short ones filled with zeros: (values over scale rounded to the format, scale bytes)."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(rows, -1, 32)
    scale = (torch.frexp(v.abs().amax(-1)).exponent + 124).clamp(0, 254)
    v = v * _table()["reciprocals"][scale].unsqueeze(-1)
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return torch.copysign((torch.round(size / step) * step).clamp(max=6), v), scale


def _mx(x):
    """Codes, two in a byte, and scale bytes."""
    q, scale = _mx_parts(x)
    size = q.abs()
    code = torch.where(size < 2, size * 2, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    code = code.view(x.shape[0], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), scale.to(torch.uint8), x.shape[1]


def _mx_values(parts):
    codes, scales, k = parts
    t = _table()
    v = t["codes"][torch.stack((codes & 15, codes >> 4), -1).long()].view(codes.shape[0], -1, 32)
    return (v * t["scales"][scales.long()].unsqueeze(-1)).view(codes.shape[0], -1)[:, :k]


def _mx_round_trip(x):
    """The values that x's rows stand for in the format, in f32."""
    q, scale = _mx_parts(x)
    return (q * _table()["scales"][scale].unsqueeze(-1)).view(x.shape[0], -1)[:, : x.shape[1]]


def run(state):
    if own:
        return state.run()
    case, t = state
    kind, dt = case["kind"], _TORCH[case["dtype"]]
    if kind == "layer_norm":
        x = t["x"].float()
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = ((d * d).mean(1, keepdim=True) + _EPS).rsqrt()
        y = (d * rstd * t["w"].float() + t["b"].float()).to(dt)
        return [y, mean.view(-1), rstd.view(-1)] if case["stats"] else [y]
    if kind == "layer_norm_backward":
        dy, rstd = t["dy"].float(), t["rstd"].unsqueeze(1)
        xh = (t["x"].float() - t["mean"].unsqueeze(1)) * rstd
        g = dy * t["w"].float()
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        return [dx.to(dt), (dy * xh).sum(0).to(dt), dy.sum(0).to(dt)]
    if kind == "mx_round_trip":
        return [(_mx_round_trip(t["x"]) if case["axis"] == 1 else _mx_round_trip(t["x"].t()).t()).to(dt)]
    if kind == "mx_dot":
        return [torch.matmul(_mx_values(t["x"]), _mx_values(t["w"]).t()).to(dt)]
    if kind == "mx_dense":
        y = torch.matmul(_mx_round_trip(t["x"]), _mx_values(t["w"]).t()) + t["b"].float()
        return [(y.clamp(min=0) if case["relu"] else y).to(dt)]
    dx = torch.matmul(_mx_round_trip(t["dy"]), _mx_round_trip(t["w"]).t())
    dw = torch.matmul(_mx_round_trip(t["x"].t()), _mx_round_trip(t["dy"].t()).t())
    return [dx.to(dt), dw.to(dt)]


# ---- the same by definition, in 64 bits ----


def _exact_mx(x):
    """Each block against the format's values themselves: the nearest one, of two equally near the one with the even code."""
    x = x.double()
    rows, k = x.shape
    blocks = torch.cat((x, x.new_zeros(rows, -k % 32)), 1).reshape(-1, 32)
    most = blocks.abs().max(1).values
    s = torch.floor(torch.log2(torch.where(most > 0, most, torch.ones_like(most))))
    s = torch.where(torch.exp2(s) > most, s - 1, torch.where(torch.exp2(s + 1) <= most, s + 1, s)) - 2  # (log2 rounds)
    scale = torch.exp2(torch.where(most > 0, s, torch.full_like(s, -127)).clamp(-127, 127)).unsqueeze(1)
    size = blocks.abs() / scale
    values = x.new_tensor(_VALUES)
    between = (values[1:] + values[:-1]) / 2
    code = torch.where(torch.arange(7, device=x.device) % 2 == 0, size.unsqueeze(-1) > between, size.unsqueeze(-1) >= between).sum(-1)
    return (torch.sign(blocks) * values[code] * scale).view(rows, -1)[:, :k]


def _exact_mx_chunked(x):
    """A few million values at a time: the comparisons above take seven of them for each."""
    step = max(1, (1 << 22) // max(1, x.shape[1]))
    return torch.cat([_exact_mx(x[i : i + step]) for i in range(0, x.shape[0], step)])


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "layer_norm":
        x = t["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = 1 / torch.sqrt(var + _EPS)
        y = torch.addcmul(t["b"].double(), (x - mean[:, None]) * rstd[:, None], t["w"].double())
        return [y, mean, rstd] if case["stats"] else [y]
    if kind == "layer_norm_backward":
        x, dy, rstd, cols = t["x"].double(), t["dy"].double(), t["rstd"].double(), case["cols"]
        xh = (x - t["mean"].double()[:, None]) * rstd[:, None]
        g = dy * t["w"].double()
        inner = (cols * g - g.sum(1)[:, None] - xh * (g * xh).sum(1)[:, None]) / cols
        return [inner * rstd[:, None], torch.einsum("rc,rc->c", dy, xh), dy.sum(0)]
    if kind == "mx_round_trip":
        return [_exact_mx_chunked(t["x"]) if case["axis"] == 1 else _exact_mx_chunked(t["x"].t().contiguous()).t()]
    if kind == "mx_dense_backward":
        dx = _exact_mx_chunked(t["dy"]) @ _exact_mx_chunked(t["w"]).t()
        return [dx, _exact_mx_chunked(t["x"].t().contiguous()) @ _exact_mx_chunked(t["dy"].t().contiguous()).t()]
    y = _exact_mx_chunked(t["x"]) @ _exact_mx_chunked(t["w"].t().contiguous()).t()
    if kind == "mx_dense":
        y = y + t["b"].double()
        y = torch.where(y < 0, torch.zeros_like(y), y) if case["relu"] else y
    return [y]


# ---- the work a pass cannot do without ----


def work(case):
    es, kind = _SIZE[case["dtype"]], case["kind"]
    if kind == "layer_norm":  # x, weight, bias in; y and the statistics out
        r, c = case["rows"], case["cols"]
        return {"bytes": es * (2 * r * c + 2 * c) + (8 * r if case["stats"] else 0), "flops": 8.0 * r * c}
    if kind == "layer_norm_backward":  # x, dy, weight, statistics in; three gradients out
        r, c = case["rows"], case["cols"]
        return {"bytes": es * (3 * r * c + 3 * c) + 8 * r, "flops": 14.0 * r * c}
    if kind == "mx_round_trip":
        return {"bytes": 2 * es * case["rows"] * case["cols"], "flops": 4.0 * case["rows"] * case["cols"]}
    m, k, n = case["m"], case["k"], case["n"]
    if kind == "mx_dense_backward":  # x, dy, W in; dx, dW out
        return {"bytes": es * (2 * m * k + 2 * k * n + m * n), "flops": 4.0 * m * k * n}
    four = 17 / 32  # bytes of a value in the format: a code and its share of the scale
    if kind == "mx_dot":
        return {"bytes": int(four * k * (m + n)) + es * m * n, "flops": 2.0 * m * k * n}
    return {"bytes": es * (m * k + m * n + n) + int(four * k * n), "flops": 2.0 * m * k * n}

"""Work in 8-bit rows, as cases to be timed and compared: what a program that
runs a Qwen3 layer on int8 weights and activations asks of the device.

A row of 8 bits stands for the values q s: q the nearest integers (ties to
even) to 127 v / max |v|, s the 32-bit max |v| / 127. Four operators:

- "matmul": products of 8-bit rows, out[t][r] = sx[t] sw[r] sum_k qx[t][k] qw[r][k];
- "norm": the residual's addition and the RMS norm, with its output in 8 bits;
- "silu": silu(gate) * up, in 8 bits (the down projection's input);
- "rows": f32 rows in 8 bits (the output projection's input).

What is held in 8 bits is returned as the values it stands for. Shapes are the
Qwen3-4B layer's, and odd ones.

The framework's calls go to its device's own stream, which neither waits for
torch's streams nor is waited for by them. What `prepare` writes with torch is
there when it returns; a pass of the framework's calls is over, and its outputs
may be read, once the whole device has been waited for
(`torch.cuda.synchronize()`): an event on a torch stream does not see it.
"""

from __future__ import annotations

import ctypes
import math

import torch

own = False

EPS = 1e-6


def listed():
    return [
        # Decode: one token's gate (or up) projection.
        {"name": "token", "kind": "matmul", "n": 1, "rows": 9728, "cols": 2560},
        # A chat's next turn, a few tokens through the q projection.
        {"name": "turn", "kind": "matmul", "n": 11, "rows": 4096, "cols": 2560},
        # One batch of 64 tokens through the down projection: long rows, few tokens.
        {"name": "batch", "kind": "matmul", "n": 64, "rows": 2560, "cols": 9728},
        # Sizes that are whole tiles, or whole words, in no direction.
        {"name": "ragged", "kind": "matmul", "n": 50, "rows": 1003, "cols": 1101},
        # A prompt of 512 tokens through the gate projection.
        {"name": "prompt", "kind": "matmul", "n": 512, "rows": 9728, "cols": 2560},
        # The largest chunk of a document through the down projection.
        {"name": "long prompt", "kind": "matmul", "n": 8192, "rows": 2560, "cols": 9728},
        # The norm before a projection, decoding (the smallest call) and over a
        # long prompt.
        {"name": "norm token", "kind": "norm", "rows": 1, "cols": 2560},
        {"name": "norm prompt", "kind": "norm", "rows": 8192, "cols": 2560},
        # The activation before the down projection, decoding and over a prompt.
        {"name": "silu token", "kind": "silu", "rows": 1, "cols": 9728},
        {"name": "silu prompt", "kind": "silu", "rows": 2048, "cols": 9728},
        # The attention's output before the output projection, decoding and
        # over a long prompt.
        {"name": "rows token", "kind": "rows", "rows": 1, "cols": 4096},
        {"name": "rows prompt", "kind": "rows", "rows": 8192, "cols": 4096},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


# The listed cases' largest: multiplications of a matmul, values of the others.
MOST_PRODUCTS, MOST_VALUES = 8192 * 2560 * 9728, 2048 * 9728


def draw(rng):
    if rng.random() < 0.6:
        # The model's projections, or any matrix.
        rows, cols = rng.choice([(4096, 2560), (1024, 2560), (2560, 4096), (9728, 2560), (2560, 9728)])
        if rng.random() < 0.6:
            rows, cols = _log_int(rng, 1, 16000), _log_int(rng, 1, 16000)
        return {"kind": "matmul", "n": _log_int(rng, 1, min(8192, MOST_PRODUCTS // (rows * cols))), "rows": rows,
                "cols": cols}
    kind = rng.choice(["norm", "silu", "rows"])
    cols = rng.choice([128, 1024, 2560, 4096, 9728, _log_int(rng, 1, 20000), _log_int(rng, 1, 20000)])
    return {"kind": kind, "rows": _log_int(rng, 1, min(8192, MOST_VALUES // cols)), "cols": cols}


# ---- what a program has in hand ----

def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _bytes(g, rows: int, cols: int, scale: float):
    """Rows of normal numbers, each of its own size about `scale`, in 8 bits."""
    v = torch.randn((rows, cols), generator=g, device="cuda")
    most = v.abs().amax(-1, keepdim=True)
    size = scale * (0.5 + torch.rand(rows, generator=g, device="cuda"))
    return torch.round(v * (127 / most)).to(torch.int8), most[:, 0] / 127 * size


def _matmul_inputs(case, seed):
    g = _generator(seed)
    return _bytes(g, case["rows"], case["cols"], 0.02) + _bytes(g, case["n"], case["cols"], 1.0)


def _row_inputs(case, seed):
    """Two arrays of rows (x and y, or gate and up; "rows" has the first alone),
    and the norm's gains."""
    g = _generator(seed)
    shape = (case["rows"], case["cols"])
    a = torch.randn(shape, generator=g, device="cuda")
    b = torch.randn(shape, generator=g, device="cuda") if case["kind"] != "rows" else None
    gain = (1 + 0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(torch.bfloat16)
    return a, b, gain


_device = None


def _hip():
    global _device
    if _device is None:
        from titania_amd.device import Hip

        _device = Hip(0)
    return _device


class _InPlace:
    """A buffer's memory, for torch to look at in place (which keeps the
    buffer): a handle points at the device address first."""

    def __init__(self, buf, shape: tuple):
        self.buf = buf
        address = ctypes.c_void_p.from_address(buf.handle).value
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<f4", "data": (address, False), "version": 2}


def _view(buf, *shape) -> torch.Tensor:
    """A buffer's values where they are: a program that chains operations
    reads none of them back."""
    return torch.as_tensor(_InPlace(buf, shape), device="cuda")


def _buffer(values: torch.Tensor):
    b = _hip().alloc(values.numel())
    _view(b, values.numel()).copy_(values.reshape(-1))
    torch.cuda.current_stream().synchronize()  # the device's own stream does not wait for torch's
    return b


def _q8(values: torch.Tensor, scales: torch.Tensor):
    q = _hip().alloc_q8(*values.shape)
    _hip().write_q8(q, values.cpu().numpy(), scales.cpu().numpy())
    return q


def prepare(case, seed):
    if case["kind"] == "matmul":
        wq, ws, xq, xs = _matmul_inputs(case, seed)
        if not own:
            return case, wq, ws, xq, xs
        out = _hip().alloc(case["n"] * case["rows"])
        return case, _q8(wq, ws), _q8(xq, xs), out, _view(out, case["n"], case["rows"])
    a, b, gain = _row_inputs(case, seed)
    if not own:
        return case, a, b, gain
    from titania_amd.device import Tensor

    rows, cols = case["rows"], case["cols"]
    buf_a, out = _buffer(a), _hip().alloc(a.numel())
    gains = _hip().upload(Tensor((cols,), gain.view(torch.int16).cpu().numpy().view("uint16")))
    return (case, buf_a, _buffer(b) if b is not None else None, gains, _hip().alloc_q8(rows, cols), out,
            _view(buf_a, rows, cols), _view(out, rows, cols))


# ---- a pass ----

def _in_8_bits(v):
    """The values that rows v (64 bits: what is next to a border goes to its own side) stand for in 8 bits."""
    most = v.abs().amax(-1, keepdim=True)
    q = torch.round(v * 127 / torch.where(most > 0, most, 1.0))
    return q.float() * (most / 127).float()


def _plain(state):
    case = state[0]
    if case["kind"] == "matmul":
        _, wq, ws, xq, xs = state
        return (xq.float() @ wq.float().T) * xs[:, None] * ws
    _, a, b, gain = state
    if case["kind"] == "rows":
        return _in_8_bits(a.double())
    if case["kind"] == "silu":
        g = a.double()
        return _in_8_bits(g / (1 + torch.exp(-g)) * b.double())
    a.add_(b)
    x = a.double()
    return {"x": a, "norm": _in_8_bits(x * gain.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))}


def _own(state):
    case, hip = state[0], _hip()
    if case["kind"] == "matmul":
        _, w, x, out, seen = state
        hip.matmul_q8(out, w, x)
        return seen
    _, a, b, gain, q, out, seen_a, seen = state
    if case["kind"] == "norm":
        hip.add_rmsnorm_q8(a, b, q, gain, EPS)
        hip.dequantize_q8(out, q)
        return {"x": seen_a, "norm": seen}
    if case["kind"] == "silu":
        hip.silu_mul_q8(q, a, b)
    else:
        hip.quantize_q8(q, a)
    hip.dequantize_q8(out, q)
    return seen


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----

def work(case):
    if case["kind"] == "matmul":
        n, rows, cols = case["n"], case["rows"], case["cols"]
        return {"bytes": (rows + n) * (cols + 4) + 4 * n * rows, "flops": 2 * n * rows * cols}
    values = case["rows"] * case["cols"]
    # Inputs read (and the residual written), an 8-bit value and its row's scale
    # written and read, the value it stands for written.
    moved = {"norm": 12, "silu": 8, "rows": 4}[case["kind"]] + 2 + 4
    return {"bytes": moved * values + 8 * case["rows"] + (2 * case["cols"] if case["kind"] == "norm" else 0),
            "flops": {"norm": 8, "silu": 10, "rows": 4}[case["kind"]] * values}


# ---- the same in 64 bits ----

def _rows64(v):
    """Rows in 8 bits by their definition: integers nearest to v over a step,
    the step rounded to 32 bits where it is kept."""
    step = torch.amax(torch.abs(v), dim=1) / 127
    q = torch.where(step[:, None] > 0, v / step.clamp_min(1e-300)[:, None], torch.zeros_like(v)).round()
    return q * step.float().double()[:, None]


def exact(case, seed):
    if case["kind"] == "matmul":
        wq, ws, xq, xs = (t.double() for t in _matmul_inputs(case, seed))
        out = torch.empty((case["n"], case["rows"]), dtype=torch.float64, device="cuda")
        w = (wq * ws[:, None]).t().contiguous()
        for at in range(0, case["n"], 1024):
            out[at:at + 1024] = torch.matmul(xq[at:at + 1024] * xs[at:at + 1024, None], w)
        return out
    a, b, gain = _row_inputs(case, seed)
    if case["kind"] == "rows":
        return _rows64(a.double())
    if case["kind"] == "silu":
        return _rows64(a.double() * torch.sigmoid(a.double()) * b.double())
    x = torch.add(a, b).double()  # the sum is kept in 32 bits, and the norm is that sum's
    scale = torch.rsqrt(x.square().sum(1) / case["cols"] + EPS)
    return {"x": x, "norm": _rows64(scale[:, None] * x * gain.double())}

"""Layer norm and microscaled 4-bit products as a user of the framework calls them: what is timed and compared.

Every case is one pass through entry points of the C ABI, by its ctypes binding (`hipabi.Context`), on operands that lie
in device memory.  Activations are [features x batch] with the batch contiguous, as in the framework's layer chain; `pad`
is how many places longer the input's rows are than the batch.  `kind` says which path a case takes:

  norm        so_layer_norm: Y = (X - mean) * rstd * gamma + beta over the features of every column, with the statistics
              that the gradient takes.
  norm_grad   so_layer_norm_grad: dX, dgamma and dbeta from X, dY and the saved statistics.
  round_trip  so_mxfp4_quantize and so_mxfp4_dequantize: a matrix to 4-bit codes with a scale per 32 entries of a row, and back.
  matmul      so_mxfp4_matmul: Y = act(W X + b), W kept in 4 bits, X quantised in blocks of 32 features within the call.
  matvec      so_mxfp4_matvec: y = W x + b, W kept in 4 bits, x as it is.

With `own` false the same passes are made of elementary torch operations in 32 bits.

With `own` true a pass is queued on the context's own stream, with which torch's streams are not ordered.  `prepare` waits for
what torch has to do ahead of it; whoever reads a pass's results, or writes into what a state holds, calls `finish()` before that
(or waits for the whole device).  A state that is dropped waits by itself before its memory goes back to torch."""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MX_BYTES = 0.5 + 1.0 / 32      # a code of 4 bits, a scale per 32 entries
EPS = 1e-5


def listed():
    return [
        # one token between two fully connected layers: all latency
        {"name": "norm_token", "kind": "norm", "F": 4096, "B": 1, "pad": 0, "type": "f32"},
        # the benchmark's MLP batch
        {"name": "norm_batch", "kind": "norm", "F": 4096, "B": 256, "pad": 0, "type": "f32"},
        # a long prompt or a training batch, half precision
        {"name": "norm_prompt", "kind": "norm", "F": 4096, "B": 8192, "pad": 0, "type": "bf16"},
        # no size a multiple of anything, rows longer than the batch
        {"name": "norm_grad_ragged", "kind": "norm_grad", "F": 1531, "B": 203, "pad": 6, "type": "f16"},
        # the backward pass of a training batch
        {"name": "norm_grad_prompt", "kind": "norm_grad", "F": 4096, "B": 8192, "pad": 0, "type": "bf16"},
        # a layer's weights after a step, small
        {"name": "round_trip_1024", "kind": "round_trip", "m": 1024, "n": 1024, "type": "f32"},
        # the largest layer that the encoder's benchmark has
        {"name": "round_trip_8192", "kind": "round_trip", "m": 8192, "n": 8192, "type": "bf16"},
        # ragged everywhere, a small batch of tokens, fused ReLU
        {"name": "matmul_ragged", "kind": "matmul", "m": 3001, "n": 2777, "C": 101, "pad": 3, "type": "f16", "bias": True, "act": "relu"},
        # the benchmark's large fully connected layer at its batch
        {"name": "matmul_4096_c256", "kind": "matmul", "m": 4096, "n": 4096, "C": 256, "pad": 0, "type": "f32", "bias": True, "act": "none"},
        # a prompt through a large layer
        {"name": "matmul_8192_c2048", "kind": "matmul", "m": 8192, "n": 8192, "C": 2048, "pad": 0, "type": "bf16", "bias": False, "act": "none"},
        # one token through a small and a large layer
        {"name": "matvec_1024", "kind": "matvec", "m": 1024, "n": 1024, "bias": True},
        {"name": "matvec_16384", "kind": "matvec", "m": 16384, "n": 16384, "bias": True},
    ]


def _log_size(rng, lo, hi):
    """A whole number of lo..hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm_grad", "round_trip", "matmul", "matmul", "matvec"))
    if kind in ("norm", "norm_grad"):
        F = _log_size(rng, 64, 8192)
        return {"kind": kind, "F": F, "B": _log_size(rng, 1, min(16384, (1 << 25) // F)), "pad": rng.choice((0, 0, 1, 8)),
                "type": rng.choice(("bf16", "f16", "f32")) if F < 4096 else rng.choice(("bf16", "f16"))}
    if kind == "round_trip":
        return {"kind": kind, "m": _log_size(rng, 128, 8192), "n": _log_size(rng, 128, 8192), "type": rng.choice(("f32", "bf16"))}
    if kind == "matvec":
        return {"kind": kind, "m": _log_size(rng, 256, 16384), "n": _log_size(rng, 256, 16384), "bias": rng.random() < 0.5}
    return {"kind": kind, "m": _log_size(rng, 64, 8192), "n": _log_size(rng, 256, 8192), "C": _log_size(rng, 1, 2048), "pad": rng.choice((0, 0, 3, 8)),
            "type": rng.choice(("f32", "f16", "bf16")), "bias": rng.random() < 0.5, "act": rng.choice(("none", "relu", "sigmoid", "tanh"))}


# ---- what a program holds before the call -------------------------------------------------------------------------

_context = None


def context():
    """One context for the process, as a program has it."""
    global _context
    if _context is None:
        path = os.path.join(os.getcwd(), "sparse-ops_amd", "python")
        if path not in sys.path:
            sys.path.insert(0, path)
        import hipabi
        _context = hipabi.Context(0)
    return _context


def finish():
    """Waits until all passes made so far are done: their results can be read, their memory used for something else."""
    if _context is not None:
        _context.sync()


class InUse:
    """Held by a state, ahead of its tensors: passes over them may still be queued when the state is dropped."""

    def __init__(self):
        self.wait = finish

    def __del__(self):
        self.wait()


class OnGpu:
    """A torch tensor's memory as the binding's calls take it (they read only `.ptr`)."""

    def __init__(self, tensor):
        self.tensor, self.ptr = tensor, tensor.data_ptr()


class Weights:
    """A handle that is freed with the state that holds it."""

    def __init__(self, handle):
        self.handle = handle

    def __del__(self):
        self.handle.free()


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(rows, cols, pad, type_, g):
    """[rows x cols] inside rows of cols + pad places: normal values around a mean of each column's own, a few features ten times as large."""
    X = torch.randn(rows, cols + pad, device="cuda", generator=g)
    loud = torch.rand(rows, 1, device="cuda", generator=g) < 0.005
    shift = torch.randn(1, cols + pad, device="cuda", generator=g) * 0.5
    return (X * torch.where(loud, 10.0, 1.0) + shift).to(TYPES[type_])


def _padded(X, n):
    """X with rows of zeros below it up to a multiple of 32."""
    return torch.cat([X, X.new_zeros((n + 31) // 32 * 32 - n, X.shape[1])]) if n % 32 else X


def _power(top):
    """2^(top - 127) in fp32 from the exponent's bits, exactly."""
    top = top.to(torch.int32)
    return (top.clamp_min(1) << 23).view(torch.float32) * torch.where(top > 0, 1.0, 0.5)


def _mx(blocks):
    """The codes 0..15 and the scales' exponents 0..255 of fp32 blocks [..., 32, C], along the dimension before the last."""
    top = (blocks.abs().amax(dim=-2, keepdim=True).view(torch.int32) >> 23).clamp_min(2) - 2
    a = blocks.abs() * _power(254 - top)
    code = (a > 0.25).to(torch.uint8)
    for border, reached in ((1.25, a.gt), (2.5, a.gt), (5.0, a.gt), (0.75, a.ge), (1.75, a.ge), (3.5, a.ge)):
        code = code + reached(border)
    return code + (blocks < 0).to(torch.uint8) * 8, top.to(torch.uint8)


def _stored(W):
    """Row-major [m x n] fp32 to bytes [m][n / 32][16], the even entry of two in the low half, and scales [m][n / 32]."""
    m, n = W.shape
    code, scale = _mx(_padded(W.T, n).reshape(-1, 32, m))
    code = code.permute(2, 0, 1).contiguous()
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), scale.reshape(-1, m).T.contiguous()


def _values(code, top):
    """What codes with scales stand for, in fp32."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=code.device)
    return table[code.to(torch.int32)] * _power(top)


def _weights(s):
    """The stored matrix, dense."""
    code = torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=-1).reshape(s["m"], -1, 32)
    return _values(code, s["scales"].unsqueeze(-1)).reshape(s["m"], -1)[:, :s["n"]]


def _statistics(X):
    mean = X.mean(dim=0)
    return mean, 1.0 / torch.sqrt((X - mean).square().mean(dim=0) + EPS)


def _inputs(case, seed):
    kind, g = case["kind"], _generator(seed)
    s = dict(case)
    if kind in ("norm", "norm_grad"):
        F, B, pad = case["F"], case["B"], case["pad"]
        s["X"] = _activations(F, B, pad, case["type"], g)
        s["gamma"] = 1.0 + 0.1 * torch.randn(F, device="cuda", generator=g)
        s["beta"] = 0.1 * torch.randn(F, device="cuda", generator=g)
        if kind == "norm_grad":
            s["dY"] = (torch.randn(F, B, device="cuda", generator=g) * 0.02).to(TYPES[case["type"]])
            s["mean"], s["rstd"] = _statistics(s["X"][:, :B].float())
        return s
    m, n = case["m"], case["n"]
    W = torch.randn(m, n, device="cuda", generator=g) / math.sqrt(n)
    if kind == "round_trip":
        s["X"] = W.to(TYPES[case["type"]])
        return s
    s["codes"], s["scales"] = _stored(W)
    s["bias"] = torch.randn(m, device="cuda", generator=g) * 0.1 if case["bias"] else None
    s["X"] = _activations(n, case["C"], case["pad"], case["type"], g) if kind == "matmul" else torch.randn(n, device="cuda", generator=g)
    return s


def prepare(case, seed):
    s = {"in_use": InUse()} if own else {}          # the first to go
    s.update(_inputs(case, seed))
    kind, new = case["kind"], lambda *shape, type=torch.float32: torch.zeros(*shape, dtype=type, device="cuda")
    if own:
        if kind == "norm":
            s.update(Y=new(s["F"], s["B"], type=TYPES[s["type"]]), mean=new(s["B"]), rstd=new(s["B"]))
            context().layer_norm_reserve(s["F"], s["B"], type=s["type"])
        elif kind == "norm_grad":
            s.update(dX=new(s["F"], s["B"], type=TYPES[s["type"]]), dgamma=new(s["F"]), dbeta=new(s["F"]))
            context().layer_norm_reserve(s["F"], s["B"], type=s["type"])
        elif kind == "round_trip":
            blocks = (s["n"] + 31) // 32
            s.update(Y=new(s["m"], s["n"], type=TYPES[s["type"]]), codes=new(s["m"], blocks, 16, type=torch.uint8), scales=new(s["m"], blocks, type=torch.uint8))
        else:
            torch.cuda.synchronize()
            s["W"] = Weights(context().mxfp4(OnGpu(s["codes"]), OnGpu(s["scales"]), s["m"], s["n"]))
            s["Y"] = new(s["m"], s["C"], type=TYPES[s["type"]]) if kind == "matmul" else new(s["m"])
            if kind == "matmul":
                context().mxfp4_matmul_reserve(s["W"].handle, s["C"])
        s["on"] = {k: OnGpu(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        torch.cuda.synchronize()   # the framework's calls run on its own stream
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def _run_own(s):
    kind, ctx, on = s["kind"], context(), s["on"]
    if kind == "norm":
        ctx.layer_norm(on["X"], s["F"], s["B"], on["gamma"], on["beta"], EPS, on["Y"], on["mean"], on["rstd"], type=s["type"], x_stride=s["B"] + s["pad"])
        return {"Y": s["Y"], "mean": s["mean"], "rstd": s["rstd"]}
    if kind == "norm_grad":
        ctx.layer_norm_grad(on["X"], on["dY"], s["F"], s["B"], on["gamma"], on["mean"], on["rstd"], on["dX"], on["dgamma"], on["dbeta"], type=s["type"],
                            x_stride=s["B"] + s["pad"])
        return {"dX": s["dX"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
    if kind == "round_trip":
        ctx.mxfp4_quantize(on["X"], s["m"], s["n"], on["codes"], on["scales"], type=s["type"])
        ctx.mxfp4_dequantize(on["codes"], on["scales"], s["m"], s["n"], on["Y"], type=s["type"])
        return s["Y"]
    if kind == "matmul":
        ctx.mxfp4_matmul(s["W"].handle, on["X"], s["C"], on.get("bias"), on["Y"], s["act"], type=s["type"], x_stride=s["C"] + s["pad"])
        return s["Y"]
    ctx.mxfp4_matvec(s["W"].handle, on["X"], on.get("bias"), on["Y"])
    return s["Y"]


def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if kind == "norm":
        X = s["X"][:, :s["B"]].float()
        mean, rstd = _statistics(X)
        Y = (X - mean) * rstd * s["gamma"].unsqueeze(1) + s["beta"].unsqueeze(1)
        return {"Y": Y.to(s["X"].dtype), "mean": mean, "rstd": rstd}
    if kind == "norm_grad":
        h = (s["X"][:, :s["B"]].float() - s["mean"]) * s["rstd"]
        dY = s["dY"].float()
        g = dY * s["gamma"].unsqueeze(1)
        dX = (g - g.mean(dim=0) - h * (g * h).mean(dim=0)) * s["rstd"]
        return {"dX": dX.to(s["X"].dtype), "dgamma": (dY * h).sum(dim=1), "dbeta": dY.sum(dim=1)}
    if kind == "round_trip":
        n = s["n"]
        code, top = _mx(_padded(s["X"].float().T, n).reshape(-1, 32, s["m"]))
        return _values(code, top).reshape(-1, s["m"])[:n].T.contiguous().to(s["X"].dtype)
    W = _weights(s)
    if kind == "matvec":
        y = torch.mv(W, s["X"])
        return y if s["bias"] is None else y + s["bias"]
    n, C = s["n"], s["C"]
    code, top = _mx(_padded(s["X"][:, :C].float(), n).reshape(-1, 32, C))
    Y = torch.mm(W, _values(code, top).reshape(-1, C)[:n])
    if s["bias"] is not None:
        Y = Y + s["bias"].unsqueeze(1)
    if s["act"] == "relu":
        Y = torch.where(Y > 0, Y, torch.zeros_like(Y))
    elif s["act"] == "sigmoid":
        Y = 1.0 / (1.0 + torch.exp(-Y))
    elif s["act"] == "tanh":
        Y = torch.tanh(Y)
    return Y.to(s["X"].dtype)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _two_to(exponent):
    """2^exponent in 64 bits, from its bits."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _nearest(V):
    """Every block of 32 along the first dimension of V, in 64 bits, on its grid of 4-bit values."""
    n, C = V.shape
    blocks = torch.zeros((n + 31) // 32 * 32, C, dtype=torch.float64, device=V.device)
    blocks[:n] = V
    blocks = blocks.view(-1, 32, C)
    largest = blocks.abs().amax(dim=1, keepdim=True)
    exponent = torch.frexp(largest).exponent - 1                                # floor(log2) of what is not zero
    exponent = torch.where(largest > 0, exponent - 2, torch.full_like(exponent, -127)).clamp_min(-127)
    scale = _two_to(exponent)
    a = (blocks / scale).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(blocks) * (torch.round(a / step) * step).clamp_max(6.0) * scale).view(-1, C)[:n]


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        X = s["X"][:, :case["B"]].double()
        gamma = s["gamma"].double()[:, None]
        if kind == "norm":
            centred = X - X.sum(0) / case["F"]
            sigma = ((centred * centred).sum(0) / case["F"] + EPS).sqrt()
            return {"Y": centred / sigma * gamma + s["beta"].double()[:, None], "mean": X.sum(0) / case["F"], "rstd": 1 / sigma}
        rstd, dY = s["rstd"].double(), s["dY"].double()
        h = (X - s["mean"].double()) * rstd
        along, across = (dY * gamma).sum(0), (dY * gamma * h).sum(0)
        return {"dX": (case["F"] * dY * gamma - along - h * across) * rstd / case["F"], "dgamma": (dY * h).sum(1), "dbeta": dY.sum(1)}
    if kind == "round_trip":
        return _nearest(s["X"].double().T).T.contiguous()
    low, high = s["codes"].long() & 15, s["codes"].long() >> 4
    code = torch.stack((low, high), -1).flatten(-2)                              # [m][blocks][32]
    size, half = code % 8, (code % 8) // 2
    value = torch.where(size < 2, size.double() / 2, (1 + (size % 2).double() / 2) * _two_to(half - 1))
    W = (torch.where(code > 7, -value, value) * _two_to(s["scales"].long()[..., None] - 127)).flatten(1)[:, :case["n"]]
    bias = 0.0 if s["bias"] is None else s["bias"].double()
    if kind == "matvec":
        return W @ s["X"].double() + bias
    Y = W @ _nearest(s["X"][:, :case["C"]].double()) + (bias if s["bias"] is None else bias[:, None])
    return {"none": lambda: Y, "relu": lambda: Y.clamp_min(0), "sigmoid": lambda: 1 / (1 + torch.exp(-Y)), "tanh": lambda: torch.tanh(Y)}[case["act"]]()


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        e, F, B = BYTES[case["type"]], case["F"], case["B"]
        if kind == "norm":
            return {"bytes": 2.0 * e * F * B + 8.0 * F + 8.0 * B, "flops": 8.0 * F * B}
        return {"bytes": 3.0 * e * F * B + 12.0 * F + 8.0 * B, "flops": 14.0 * F * B}
    m, n = case["m"], case["n"]
    if kind == "round_trip":
        return {"bytes": 2.0 * (BYTES[case["type"]] + MX_BYTES) * m * n, "flops": 4.0 * m * n}
    bias = 4.0 * m if case["bias"] else 0.0
    if kind == "matvec":
        return {"bytes": MX_BYTES * m * n + 4.0 * (m + n) + bias, "flops": 2.0 * m * n}
    return {"bytes": MX_BYTES * m * n + BYTES[case["type"]] * case["C"] * (m + n) + bias, "flops": 2.0 * m * n * case["C"]}

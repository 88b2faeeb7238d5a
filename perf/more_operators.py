"""Gated feed-forward blocks, low-rank adapters and rotary positions as a user of the framework calls them: what is timed and compared.

Every case is one pass through an entry point of the C ABI, by its ctypes binding (`hipabi.Context`), on operands that lie in
device memory.  Activations are [features x batch] with the batch contiguous, as in the framework's layer chain, a column
being a token; `pad` is how many places longer the input's rows are than the batch.  `kind` says which path a case takes:

  gated       so_gated: H = act(Wg X + G0) * (Wu X + U0), both projections, the activation and the product; `save` asks for
              the two sums as well, which the gradient takes, `add` says that there are G0 and U0 (what adapters make of X).
  gated_grad  so_gated_grad: the gradients of X, Wg and Wu from that of H and the saved sums.
  adapters    so_adapters: Y = base + scale_a B_a (A_a X), a the adapter that each column's request has, if it has one.
  rotary      so_head_rotary: every head of a column's queries and keys over the root of its mean square (if `norm`), times a gain per
              feature, and turned by the column's position; `save` asks for the norms' factors, which the gradient takes.
  rotary_grad so_head_rotary_grad: the gradients of the input and of both gains.

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
EPS = 1e-6
AMPLITUDE = 1.1                # of turned features, as scalings for long contexts have it
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid", "tanh", "none")


def listed():
    return [
        # one token through a large block: a stream of weights
        {"name": "gated_token", "kind": "gated", "m": 16384, "n": 4096, "B": 1, "pad": 0, "type": "bf16", "act": "silu", "save": False, "add": False},
        # the next tokens of a few requests, with adapters on both projections
        {"name": "gated_requests", "kind": "gated", "m": 8192, "n": 4096, "B": 24, "pad": 0, "type": "f16", "act": "gelu", "save": False, "add": True},
        # no size a multiple of anything, rows longer than the batch, fp32
        {"name": "gated_ragged", "kind": "gated", "m": 2777, "n": 1531, "B": 203, "pad": 3, "type": "f32", "act": "gelu_tanh", "save": True, "add": False},
        # a training batch, forward
        {"name": "gated_prompt", "kind": "gated", "m": 8192, "n": 4096, "B": 4096, "pad": 0, "type": "bf16", "act": "silu", "save": True, "add": False},
        # a small ragged training step's backward pass
        {"name": "gated_grad_ragged", "kind": "gated_grad", "m": 1531, "n": 1003, "B": 331, "pad": 6, "type": "f16", "act": "gelu"},
        # a training batch, backward
        {"name": "gated_grad_prompt", "kind": "gated_grad", "m": 8192, "n": 4096, "B": 4096, "pad": 0, "type": "bf16", "act": "silu"},
        # the next tokens of a served batch, nearly every request with an adapter of its own
        {"name": "adapters_requests", "kind": "adapters", "m": 4096, "n": 4096, "C": 48, "requests": 48, "count": 64, "rank": 16, "pad": 0, "type": "f16"},
        # ragged everywhere, fp32
        {"name": "adapters_ragged", "kind": "adapters", "m": 2777, "n": 1531, "C": 203, "requests": 9, "count": 5, "rank": 10, "pad": 3, "type": "f32"},
        # the prompts of a few requests
        {"name": "adapters_prompt", "kind": "adapters", "m": 4096, "n": 4096, "C": 8192, "requests": 6, "count": 8, "rank": 16, "pad": 0, "type": "bf16"},
        # one token of one request: all latency
        {"name": "rotary_token", "kind": "rotary", "q": 32, "k": 8, "D": 128, "rot": 128, "B": 1, "pad": 0, "type": "bf16", "layout": "halves", "norm": True, "save": False},
        # the prompts of a few requests, far into long contexts
        {"name": "rotary_prompt", "kind": "rotary", "q": 32, "k": 8, "D": 128, "rot": 128, "B": 8192, "pad": 0, "type": "bf16", "layout": "halves", "norm": True, "save": True},
        # a training batch's backward pass, neighbouring features in pairs, a part of the head turned, rows longer than the batch
        {"name": "rotary_grad_ragged", "kind": "rotary_grad", "q": 24, "k": 8, "D": 96, "rot": 64, "B": 4099, "pad": 5, "type": "f16", "layout": "pairs", "norm": True},
    ]


def _log_size(rng, lo, hi):
    """A whole number of lo..hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("gated", "gated", "gated_grad", "adapters", "adapters", "rotary", "rotary_grad"))
    if kind in ("rotary", "rotary_grad"):
        k, D = rng.choice((1, 2, 4, 8)), rng.choice((32, 64, 80, 96, 128, 192, 256))
        q = k * rng.choice((1, 2, 4, 7, 8))
        case = {"kind": kind, "q": q, "k": k, "D": D, "rot": rng.choice((D, D, D // 2, D // 4)), "B": _log_size(rng, 1, min(16384, (1 << 25) // (D * (q + k)))), "pad": rng.choice((0, 0, 1, 8)),
                "type": rng.choice(("f32", "f16", "bf16", "bf16")), "layout": rng.choice(("halves", "pairs")), "norm": rng.random() < 0.7}
        if kind == "rotary":
            case["save"] = case["norm"] and rng.random() < 0.5
        return case
    if kind == "adapters":
        rank = rng.choice((4, 8, 10, 16, 24, 32, 64))
        C = _log_size(rng, 1, 8192 * 16 // max(rank, 16))
        return {"kind": kind, "m": _log_size(rng, 256, 8192 if C < 4096 else 4096), "n": _log_size(rng, 256, 4096), "C": C, "requests": C if C <= 64 else _log_size(rng, 1, 40), "count": _log_size(rng, 1, 32),
                "rank": rank, "pad": rng.choice((0, 0, 3, 8)), "type": rng.choice(("f32", "f16", "bf16")) if C < 2048 else rng.choice(("f16", "bf16"))}
    type_ = rng.choice(("f32", "f16", "bf16", "bf16"))
    m, n = _log_size(rng, 128, 8192), _log_size(rng, 128, 4096)
    B = _log_size(rng, 1 if kind == "gated" else 16, 512 if type_ == "f32" else 4096)
    case = {"kind": kind, "m": m, "n": n, "B": B, "pad": rng.choice((0, 0, 3, 8)), "type": type_, "act": rng.choice(ACTS)}
    if kind == "gated":
        case.update(save=rng.random() < 0.5, add=rng.random() < 0.3)
    return case


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


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(rows, cols, pad, type_, g):
    """[rows x cols] inside rows of cols + pad places: what a norm leaves, a few features ten times as large."""
    X = torch.randn(rows, cols + pad, device="cuda", generator=g)
    loud = torch.rand(rows, 1, device="cuda", generator=g) < 0.005
    return (X * torch.where(loud, 10.0, 1.0)).to(TYPES[type_])


def _weights(rows, cols, type_, g):
    return (torch.randn(rows, cols, device="cuda", generator=g) / math.sqrt(cols)).to(TYPES[type_])


def _adapter_of(request, count):
    """The number of a request's adapter before the numbers are shuffled; every eighth request has none."""
    return -1 if request % 8 == 7 else request % count


def _which(case, g):
    """The adapter of every column: a request's columns lie together, and begin anywhere."""
    C, requests, count = case["C"], min(case["requests"], case["C"]), case["count"]
    first = torch.zeros(C, dtype=torch.int64, device="cuda")
    first[torch.randperm(C - 1, device="cuda", generator=g)[:requests - 1] + 1] = 1
    shuffled = torch.randperm(count, device="cuda", generator=g)
    number = torch.tensor([_adapter_of(r, count) for r in range(requests)], device="cuda")
    adapter = torch.where(number < 0, number, shuffled[number.clamp_min(0)])
    return adapter[first.cumsum(0)].to(torch.int32)


def _positions(B, g):
    """Four runs of consecutive positions that begin anywhere in a long context."""
    column = torch.arange(B, device="cuda")
    start = torch.randint(0, 1000000, (4,), device="cuda", generator=g)
    return (start[column * 4 // B] + column).to(torch.int32)


def _inputs(case, seed):
    kind, g, type_ = case["kind"], _generator(seed), case["type"]
    s = dict(case)
    if kind in ("rotary", "rotary_grad"):
        heads, D, B = case["q"] + case["k"], case["D"], case["B"]
        s["X"] = _activations(heads * D, B, case["pad"], type_, g)
        s["position"] = _positions(B, g)
        s["frequency"] = (500000.0 ** (-torch.arange(case["rot"] // 2, device="cuda") * 2.0 / case["rot"])).float() * (0.5 + 0.5 * torch.rand(case["rot"] // 2, device="cuda", generator=g))
        if case["norm"]:
            s["gain_q"], s["gain_k"] = (1.0 + 0.1 * torch.randn(D, device="cuda", generator=g) for _ in range(2))
        if kind == "rotary_grad":
            s["dY"] = (0.02 * torch.randn(heads * D, B, device="cuda", generator=g)).to(TYPES[type_])
            if case["norm"]:
                s["rstd"] = _rstd(s["X"][:, :B].float().view(heads, D, B))
        return s
    m, n = case["m"], case["n"]
    if kind == "adapters":
        C, count, rank = case["C"], case["count"], case["rank"]
        s["X"] = _activations(n, C, case["pad"], type_, g)
        s["A"] = _weights(count * rank, n, type_, g)
        s["B"] = _weights(count * m, rank, type_, g)
        s["scale"] = 0.5 + torch.rand(count, device="cuda", generator=g)
        s["which"] = _which(case, g)
        s["base"] = torch.randn(m, C, device="cuda", generator=g).to(TYPES[type_])
        return s
    B = case["B"]
    s["X"] = _activations(n, B, case["pad"], type_, g)
    s["Wg"], s["Wu"] = _weights(m, n, type_, g), _weights(m, n, type_, g)
    if kind == "gated_grad":
        X = s["X"][:, :B].float()
        s["G"], s["U"] = torch.mm(s["Wg"].float(), X).to(TYPES[type_]), torch.mm(s["Wu"].float(), X).to(TYPES[type_])
        s["dH"] = (0.02 * torch.randn(m, B, device="cuda", generator=g)).to(TYPES[type_])
    elif case["add"]:
        s["G0"], s["U0"] = ((0.3 * torch.randn(m, B, device="cuda", generator=g)).to(TYPES[type_]) for _ in range(2))
    return s


def prepare(case, seed):
    s = {"in_use": InUse()} if own else {}          # the first to go
    s.update(_inputs(case, seed))
    if own:
        kind, new = case["kind"], lambda *shape, type=case["type"]: torch.zeros(*shape, dtype=TYPES[type], device="cuda")
        if kind in ("rotary", "rotary_grad"):
            heads, D, B = s["q"] + s["k"], s["D"], s["B"]
            if kind == "rotary":
                s["Y"] = new(heads * D, B)
                if s["save"]:
                    s["rstd"] = new(heads, B, type="f32")
            else:
                s["dX"] = new(heads * D, B)
                if s["norm"]:
                    s.update(dgain_q=new(D, type="f32"), dgain_k=new(D, type="f32"))
                context().head_rotary_reserve(s["q"], s["k"], D, B, type=s["type"])
        elif kind == "adapters":
            m, n = s["m"], s["n"]
            s["Y"] = new(m, s["C"])
            context().adapters_reserve(m, n, s["C"], s["rank"], type=s["type"])
        else:
            m, n = s["m"], s["n"]
            if kind == "gated":
                s["H"] = new(m, s["B"])
                if s["save"]:
                    s.update(G=new(m, s["B"]), U=new(m, s["B"]))
            else:
                s.update(dX=new(n, s["B"]), dWg=new(m, n), dWu=new(m, n))
            context().gated_reserve(m, n, s["B"], type=s["type"])
        s["on"] = {k: OnGpu(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        torch.cuda.synchronize()   # the framework's calls run on its own stream
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def _run_own(s):
    kind, ctx, on = s["kind"], context(), s["on"]
    if kind == "gated":
        ctx.gated(on["Wg"], on["Wu"], s["m"], s["n"], on["X"], s["B"], s["act"], on["H"], on.get("G"), on.get("U"), on.get("G0"), on.get("U0"), type=s["type"],
                  x_stride=s["B"] + s["pad"])
        return {k: s[k] for k in ("H", "G", "U") if k in s}
    if kind == "gated_grad":
        ctx.gated_grad(on["Wg"], on["Wu"], s["m"], s["n"], on["X"], s["B"], s["act"], on["G"], on["U"], on["dH"], on["dX"], on["dWg"], on["dWu"], type=s["type"],
                       x_stride=s["B"] + s["pad"])
        return {"dX": s["dX"], "dWg": s["dWg"], "dWu": s["dWu"]}
    if kind == "rotary":
        ctx.head_rotary(on["X"], s["q"], s["k"], s["D"], s["B"], on["position"], on["frequency"], s["rot"], on["Y"], layout=s["layout"], amplitude=AMPLITUDE, norm=s["norm"], eps=EPS,
                        dGainQ=on.get("gain_q"), dGainK=on.get("gain_k"), dRstd=on.get("rstd"), type=s["type"], x_stride=s["B"] + s["pad"])
        return {k: s[k] for k in ("Y", "rstd") if k in s}
    if kind == "rotary_grad":
        ctx.head_rotary_grad(on["X"], on["dY"], s["q"], s["k"], s["D"], s["B"], on["position"], on["frequency"], s["rot"], on["dX"], layout=s["layout"], amplitude=AMPLITUDE, norm=s["norm"],
                             dGainQ=on.get("gain_q"), dGainK=on.get("gain_k"), dRstd=on.get("rstd"), dDgainQ=on.get("dgain_q"), dDgainK=on.get("dgain_k"), type=s["type"],
                             x_stride=s["B"] + s["pad"])
        return {k: s[k] for k in ("dX", "dgain_q", "dgain_k") if k in s}
    ctx.adapters(on["A"], on["B"], on["scale"], s["count"], s["rank"], on["which"], s["m"], s["n"], on["X"], s["C"], on["base"], on["Y"], type=s["type"],
                 x_stride=s["C"] + s["pad"])
    return s["Y"]


GELU_TANH = math.sqrt(2.0 / math.pi)


def _act(G, act):
    if act == "silu":
        return G / (1.0 + torch.exp(-G))
    if act == "gelu":
        return 0.5 * G * (1.0 + torch.erf(G * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * G * (1.0 + torch.tanh(GELU_TANH * (G + 0.044715 * G * G * G)))
    if act == "relu":
        return torch.where(G > 0, G, torch.zeros_like(G))
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-G))
    return torch.tanh(G) if act == "tanh" else G


def _slope(G, act):
    """The activation's derivative."""
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-G))
        return p * (1.0 + G * (1.0 - p))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(G * math.sqrt(0.5))) + G * torch.exp(-0.5 * G * G) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(GELU_TANH * (G + 0.044715 * G * G * G))
        return 0.5 * (1.0 + t) + 0.5 * G * (1.0 - t * t) * GELU_TANH * (1.0 + 3.0 * 0.044715 * G * G)
    if act == "relu":
        return torch.where(G > 0, torch.ones_like(G), torch.zeros_like(G))
    if act == "sigmoid":
        p = 1.0 / (1.0 + torch.exp(-G))
        return p * (1.0 - p)
    if act == "tanh":
        return 1.0 - torch.tanh(G) ** 2
    return torch.ones_like(G)


def _rstd(X):
    return 1.0 / torch.sqrt(X.square().mean(dim=1) + EPS)


def _gains(s):
    """[heads, D, 1]: the queries' for the first heads, the keys' for the others."""
    return torch.cat([s["gain_q"].expand(s["q"], -1), s["gain_k"].expand(s["k"], -1)]).unsqueeze(2)


def _turn(X, s, back=False):
    """The first `rot` features of every head of X [heads, D, B] turned by the columns' angles (64 bits: positions are far), times the amplitude."""
    rot = s["rot"]
    angle = s["position"].double().unsqueeze(0) * s["frequency"].double().unsqueeze(1)
    cos, sin = (AMPLITUDE * torch.cos(angle)).float(), (AMPLITUDE * torch.sin(angle)).float()
    if back:
        sin = -sin
    if s["layout"] == "halves":
        a, b = X[:, :rot // 2], X[:, rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=1)
    else:
        a, b = X[:, 0:rot:2], X[:, 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=2).reshape(X.shape[0], rot, X.shape[2])
    return torch.cat([turned, X[:, rot:]], dim=1)


def _run_rotary(s):
    type_, heads, D, B = s["X"].dtype, s["q"] + s["k"], s["D"], s["B"]
    X = s["X"][:, :B].float().view(heads, D, B)
    if s["kind"] == "rotary":
        out = {}
        if s["norm"]:
            rstd = _rstd(X)
            X = X * rstd.unsqueeze(1) * _gains(s)
            if s["save"]:
                out["rstd"] = rstd
        return {"Y": _turn(X, s).reshape(heads * D, B).to(type_), **out}
    g = _turn(s["dY"].float().view(heads, D, B), s, back=True)
    if not s["norm"]:
        return {"dX": g.reshape(heads * D, B).to(type_)}
    rstd = s["rstd"].unsqueeze(1)
    h = X * rstd
    along = g * _gains(s)
    dX = (along - h * (along * h).mean(dim=1, keepdim=True)) * rstd
    dgain = (g * h).sum(dim=2)
    return {"dX": dX.reshape(heads * D, B).to(type_), "dgain_q": dgain[:s["q"]].sum(dim=0), "dgain_k": dgain[s["q"]:].sum(dim=0)}


def run(s):
    if own:
        return _run_own(s)
    kind, type_ = s["kind"], s["X"].dtype
    if kind in ("rotary", "rotary_grad"):
        return _run_rotary(s)
    if kind == "adapters":
        # every adapter on every column, and of these the column's own
        C, m, count, rank = s["C"], s["m"], s["count"], s["rank"]
        T = torch.mm(s["A"].float(), s["X"][:, :C].float()).view(count, rank, C) * s["scale"].view(count, 1, 1)
        mine = s["which"].view(1, 1, C) == torch.arange(count, device="cuda").view(count, 1, 1)
        T = torch.where(mine, T, torch.zeros_like(T)).view(count * rank, C)
        B = s["B"].float().view(count, m, rank).permute(1, 0, 2).reshape(m, count * rank)
        return (s["base"].float() + torch.mm(B, T)).to(type_)
    X, Wg, Wu = s["X"][:, :s["B"]].float(), s["Wg"].float(), s["Wu"].float()
    if kind == "gated":
        G, U = torch.mm(Wg, X), torch.mm(Wu, X)
        if s["add"]:
            G, U = G + s["G0"].float(), U + s["U0"].float()
        out = {"H": (_act(G, s["act"]) * U).to(type_)}
        if s["save"]:
            out.update(G=G.to(type_), U=U.to(type_))
        return out
    G, U, dH = s["G"].float(), s["U"].float(), s["dH"].float()
    dG, dU = dH * U * _slope(G, s["act"]), dH * _act(G, s["act"])
    return {"dX": (torch.mm(Wg.T, dG) + torch.mm(Wu.T, dU)).to(type_), "dWg": torch.mm(dG, X.T).to(type_), "dWu": torch.mm(dU, X.T).to(type_)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _gate(G, act):
    """The activation and its derivative, in 64 bits."""
    if act == "none":
        return G, torch.ones_like(G)
    if act == "relu":
        return G.clamp_min(0.0), (G > 0).double()
    if act == "tanh":
        return torch.tanh(G), 1.0 / torch.cosh(G).square()
    half = torch.tanh(G / 2)
    if act == "sigmoid":
        return (1 + half) / 2, (1 - half * half) / 4
    if act == "silu":
        return G * (1 + half) / 2, (1 + half) / 2 + G * (1 - half * half) / 4
    if act == "gelu":
        below = torch.special.erfc(-G / math.sqrt(2)) / 2
        return G * below, below + G * torch.exp(-G * G / 2) / math.sqrt(2 * math.pi)
    inner, along = G + 0.044715 * G ** 3, 1 + 0.134145 * G ** 2
    half = torch.tanh(math.sqrt(2 / math.pi) * inner)
    return G * (1 + half) / 2, (1 + half) / 2 + G * (1 - half * half) * along / math.sqrt(2 * math.pi)


def _exact_rotary(case, s):
    q, k, D, B, rot = (case[name] for name in ("q", "k", "D", "B", "rot"))
    first = torch.arange(rot // 2, device="cuda") * (1 if case["layout"] == "halves" else 2)
    second = first + (rot // 2 if case["layout"] == "halves" else 1)
    turn = AMPLITUDE * torch.exp(1j * s["frequency"].double()[:, None] * s["position"].double()[None, :])
    X = s["X"][:, :B].double().view(q + k, D, B)
    if case["norm"]:
        gain = torch.stack([s["gain_q"].double()] * q + [s["gain_k"].double()] * k)[:, :, None]
    if case["kind"] == "rotary":
        out = {}
        if case["norm"]:
            size = ((X * X).sum(1, keepdim=True) / D + EPS).sqrt()
            X = X / size * gain
            if case["save"]:
                out["rstd"] = 1 / size[:, 0]
        pair = torch.complex(X[:, first], X[:, second]) * turn
        Y = X.clone()
        Y[:, first], Y[:, second] = pair.real, pair.imag
        return {"Y": Y.view(-1, B), **out}
    g = s["dY"].double().view(q + k, D, B).clone()
    pair = torch.complex(g[:, first], g[:, second]) * turn.conj()
    g[:, first], g[:, second] = pair.real, pair.imag
    if not case["norm"]:
        return {"dX": g.view(-1, B)}
    r = s["rstd"].double()[:, None, :]
    inner = (g * gain * X).sum(1, keepdim=True)
    dX = g * gain * r - X * inner * r ** 3 / D
    each = torch.einsum("hdb,hdb->hd", g, X * r)
    return {"dX": dX.view(-1, B), "dgain_q": each[:q].sum(0), "dgain_k": each[q:].sum(0)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("rotary", "rotary_grad"):
        return _exact_rotary(case, s)
    if case["kind"] == "adapters":
        m, rank, X = case["m"], case["rank"], s["X"][:, :case["C"]].double()
        Y = s["base"].double()
        for a in range(case["count"]):
            columns = (s["which"] == a).nonzero().flatten()
            low = s["A"][a * rank:(a + 1) * rank].double() @ X[:, columns]
            Y[:, columns] += (s["B"][a * m:(a + 1) * m].double() @ low) * s["scale"][a].double()
        return Y
    X, Wg, Wu = s["X"][:, :case["B"]].double(), s["Wg"].double(), s["Wu"].double()
    if case["kind"] == "gated":
        G, U = Wg @ X, Wu @ X
        if case["add"]:
            G, U = G + s["G0"].double(), U + s["U0"].double()
        out = {"H": _gate(G, case["act"])[0] * U}
        if case["save"]:
            out.update(G=G, U=U)
        return out
    value, slope = _gate(s["G"].double(), case["act"])
    dH = s["dH"].double()
    dG, dU = dH * s["U"].double() * slope, dH * value
    return {"dX": (dG.T @ Wg + dU.T @ Wu).T.contiguous(), "dWg": (X @ dG.T).T.contiguous(), "dWu": (X @ dU.T).T.contiguous()}


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    e = BYTES[case["type"]]
    if case["kind"] in ("rotary", "rotary_grad"):
        heads, D, B = case["q"] + case["k"], case["D"], case["B"]
        arrays = 2 if case["kind"] == "rotary" else 3 if case["norm"] else 2
        statistics = 4.0 * heads * B if case["kind"] == "rotary_grad" and case["norm"] or case.get("save") else 0.0
        return {"bytes": float(arrays * e * heads * D * B + 4 * B + 4 * case["rot"] // 2 + (8 * D if case["norm"] else 0)) + statistics, "flops": (8.0 if case["kind"] == "rotary" else 14.0) * heads * D * B}
    m, n = case["m"], case["n"]
    if case["kind"] == "adapters":
        C, rank = case["C"], case["rank"]
        used = {_adapter_of(r, case["count"]) for r in range(min(case["requests"], C))} - {-1}
        return {"bytes": float(e * (len(used) * rank * (m + n) + n * C + 2 * m * C) + 4 * C), "flops": 2.0 * rank * (m + n) * C}
    B = case["B"]
    if case["kind"] == "gated":
        return {"bytes": float(e * (2 * m * n + n * B + m * B * (1 + 2 * case["save"] + 2 * case["add"]))), "flops": 4.0 * m * n * B + 10.0 * m * B}
    return {"bytes": float(e * (4 * m * n + 2 * n * B + 3 * m * B)), "flops": 8.0 * m * n * B + 20.0 * m * B}

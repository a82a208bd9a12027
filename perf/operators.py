"""The linear layers of a transformer as this framework runs them: what is measured, the plain form in elementary torch
operations, and the same in 64 bits.

  linear             y = act(x W^T + b) + r, with the pre-activation z = x W^T + b stored on request (training)
  linear_backward    dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum of dz over the rows
  grouped            y[rows of expert g] = act(x[rows of expert g] W[g]^T + b[g]), rows sorted by expert, offsets on the GPU
  grouped_backward   the four gradients for every expert; an expert without rows has dW = 0 and db = 0

Layouts are the framework's: x [rows, in], W [out, in] ([experts, out, in]), 16-bit, f32 accumulation.
"""
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token through a small layer: what counts is latency
        dict(name="linear 1 token", kind="linear", m=1, n=2048, k=2048, io="bf16", out="bf16", act="silu", bias=True,
             residual=False, save=False),
        # a batch of 16 single tokens through the widest layer of the skinny GEMM benchmark: the weights' bytes count
        dict(name="linear 16 tokens wide", kind="linear", m=16, n=28672, k=8192, io="bf16", out="bf16", act="silu",
             bias=False, residual=False, save=False),
        # a short prompt of no round length, the projection back onto the residual stream
        dict(name="linear prompt 333", kind="linear", m=333, n=4096, k=4096, io="f16", out="f16", act="gelu_tanh",
             bias=True, residual=True, save=False),
        # sizes that are a multiple of nothing, f32 results (logits of a small head)
        dict(name="linear odd sizes", kind="linear", m=77, n=1003, k=1021, io="f16", out="f32", act="relu", bias=True,
             residual=False, save=False),
        # a training step's forward at the GEMM benchmark's size, everything in the epilogue
        dict(name="linear 8192 training", kind="linear", m=8192, n=8192, k=8192, io="bf16", out="bf16", act="gelu",
             bias=True, residual=True, save=True),
        # a training step's backward through an up-projection
        dict(name="linear_backward 8192", kind="linear_backward", m=8192, n=8192, k=2048, io="bf16", out="bf16",
             act="gelu_tanh", bias=True, dw="bf16"),
        # a small ragged batch's backward
        dict(name="linear_backward ragged", kind="linear_backward", m=515, n=1032, k=776, io="f16", out="f16", act="relu",
             bias=True, dw="f16"),
        # serving: 64 tokens over 64 experts, 24 of which get none
        dict(name="grouped 64 tokens", kind="grouped", m=64, n=2048, k=4096, groups=64, active=40, rest=0, io="bf16",
             out="bf16", act="silu", bias=False, save=False),
        # a long prompt over a few large experts
        dict(name="grouped prompt 16384", kind="grouped", m=16384, n=8192, k=4096, groups=8, active=8, rest=0, io="bf16",
             out="bf16", act="silu", bias=False, save=False),
        # many small experts, ragged rows, rows behind the last expert's, z stored
        dict(name="grouped ragged", kind="grouped", m=3001, n=1032, k=1544, groups=32, active=29, rest=13, io="f16",
             out="f16", act="gelu", bias=True, save=True),
        # a training step's backward over 16 experts
        dict(name="grouped_backward 8192", kind="grouped_backward", m=8192, n=4096, k=2048, groups=16, active=15, rest=0,
             io="bf16", out="bf16", act="silu", bias=True, dw="bf16"),
        # small experts without an activation, f32 weight gradients
        dict(name="grouped_backward ragged", kind="grouped_backward", m=700, n=520, k=1288, groups=24, active=20, rest=7,
             io="f16", out="f16", act="none", bias=True, dw="f32"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear_backward", "grouped", "grouped", "grouped_backward"])
    io = rng.choice(["bf16", "f16"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    unit = 1 if rng.random() < 1 / 6 else 8  # features are a multiple of 8 in most models, rows of anything
    m = _log_uniform(rng, 1, 16384)
    n, k = (max(unit, _log_uniform(rng, 128, 16384) // unit * unit) for _ in range(2))
    case = dict(kind=kind, m=m, io=io, act=act, bias=rng.random() < 0.7)
    if kind.startswith("grouped"):
        groups = _log_uniform(rng, 2, 128)
        case.update(groups=groups, active=min(m, rng.randint((groups + 1) // 2, groups)))
        case["rest"] = rng.choice([0, 0, rng.randint(0, m - case["active"])])
        while groups * n * k > 1 << 29:
            n, k = (max(unit, v // 2 // unit * unit) for v in (n, k))
    while m * n * k > 8192 * 8192 * (4096 if kind.startswith("grouped") else 8192):
        n, k = (max(unit, v * 3 // 4 // unit * unit) for v in (n, k))
    case.update(n=n, k=k)
    if kind.endswith("backward"):
        # an activation's gradient is rounded to the operands' type, and the weights' gradient comes in that type then
        case.update(out=io, dw="f32" if act == "none" and rng.random() < 0.5 else io)
    else:
        case.update(out=rng.choice([io, io, "f32"]), save=rng.random() < 0.3)
        if kind == "linear":
            case["residual"] = rng.random() < 0.4
    return case


def _sizes(case, gen):
    """Rows of each expert: `active` of them share m - rest rows unevenly, none gets more than about three times its share."""
    active, rows = case["active"], case["m"] - case["rest"]
    share = torch.rand(active, generator=gen, dtype=torch.float64) + 0.25
    got = 1 + torch.floor((rows - active) * share / share.sum()).to(torch.int64)
    spare = rows - int(got.sum())
    got[:spare] += 1  # fewer than `active` of them
    sizes = torch.zeros(case["groups"], dtype=torch.int64)
    sizes[torch.randperm(case["groups"], generator=gen)[:active].sort().values] = got[torch.randperm(active, generator=gen)]
    return sizes


def prepare(case, seed):
    """Activations and gradients of unit scale, weights that keep it, as they come out of a normalised layer."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    io, m, n, k = DTYPES[case["io"]], case["m"], case["n"], case["k"]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)  # noqa: E731
    state = dict(case=case, x=randn(m, k).to(io))
    lead = ()
    if case["kind"].startswith("grouped"):
        host = torch.Generator()
        host.manual_seed(seed)
        sizes = _sizes(case, host)
        offsets = torch.zeros(case["groups"] + 1, dtype=torch.int64)
        offsets[1:] = sizes.cumsum(0)
        lead = (case["groups"],)
        # `most`: an upper bound of an expert's rows, which the host knows (a capacity); only the plain form wants it
        state.update(offsets=offsets.to(torch.int32).to(dev), most=int(sizes.max()))
    weight = torch.empty(*lead, n, k, dtype=io, device=dev)
    weight.normal_(0, k ** -0.5, generator=gen)
    state["weight"] = weight
    state["bias"] = (0.25 * randn(*lead, n)).to(io) if case["bias"] else None
    if case["kind"].endswith("backward"):
        state["dy"] = (0.05 * randn(m, n)).to(DTYPES[case["out"]])
        state["z"] = randn(m, n).to(io) if case["act"] != "none" else None
    elif case.get("residual"):
        state["residual"] = randn(m, n).to(io)
    return state


# ---------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_gradient(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _by_expert(state):
    """[experts, most]: the row that each expert's j-th row is, and whether it has one."""
    o = state["offsets"].long()
    rows = o[:-1, None] + torch.arange(state["most"], device=o.device)
    live = rows < o[1:, None]
    return torch.where(live, rows, torch.zeros_like(rows)), live


def _by_row(state, padded):
    """[experts, most, width] back to [rows, width], zero for the rows that no expert has."""
    o = state["offsets"].long()
    row = torch.arange(state["x"].shape[0], device=o.device)
    expert = torch.clamp((row[:, None] >= o[1:]).sum(1), max=o.shape[0] - 2)
    at = torch.clamp(row - o[expert], max=state["most"] - 1)
    return torch.where((row < o[-1])[:, None], padded[expert, at], padded.new_zeros(()))


def _plain_forward(s, c):
    io = DTYPES[c["io"]]
    z = s["x"].float() @ s["weight"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, c["act"])
    if s.get("residual") is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(DTYPES[c["out"]]), **(dict(z=z.to(io)) if c["save"] else {}))


def _plain_backward(s, c):
    io = DTYPES[c["io"]]
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _act_gradient(s["z"].float(), c["act"])
    got = dict(dx=(dz @ s["weight"].float()).to(io), dw=(dz.t() @ s["x"].float()).to(DTYPES[c["dw"]]))
    if c["bias"]:
        got["db"] = dz.sum(0)
    return got


def _plain_grouped(s, c):
    io, out = DTYPES[c["io"]], DTYPES[c["out"]]
    rows, _ = _by_expert(s)
    z = torch.bmm(s["x"].float()[rows], s["weight"].float().transpose(1, 2))
    if s["bias"] is not None:
        z = z + s["bias"].float()[:, None, :]
    y = _by_row(s, _act(z, c["act"])).to(out)
    return dict(y=y, **(dict(z=_by_row(s, z).to(io)) if c["save"] else {}))


def _plain_grouped_backward(s, c):
    io = DTYPES[c["io"]]
    rows, live = _by_expert(s)
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _act_gradient(s["z"].float(), c["act"])
    dz = dz[rows] * live[..., None]
    dx = _by_row(s, torch.bmm(dz, s["weight"].float()))
    got = dict(dx=dx.to(io), dw=torch.bmm(dz.transpose(1, 2), s["x"].float()[rows]).to(DTYPES[c["dw"]]))
    if c["bias"]:
        got["db"] = dz.sum(1)
    return got


def run(state):
    s, c = state, state["case"]
    if not own:
        return dict(linear=_plain_forward, linear_backward=_plain_backward, grouped=_plain_grouped,
                    grouped_backward=_plain_grouped_backward)[c["kind"]](s, c)
    ops = importlib.import_module("7_b200.wave_linear")
    if c["kind"].endswith("backward"):
        more = dict(activation=c["act"], pre_activation=s["z"], dweight_dtype=DTYPES[c["dw"]], need_dbias=c["bias"])
        if c["kind"] == "linear_backward":
            dx, dw, db = ops.linear_backward(s["dy"], s["x"], s["weight"], **more)
        else:
            dx, dw, db = ops.grouped_linear_backward(s["dy"], s["x"], s["weight"], s["offsets"], **more)
        return dict(dx=dx, dw=dw, **(dict(db=db) if c["bias"] else {}))
    more = dict(activation=c["act"], out_dtype=DTYPES[c["out"]], save_pre_activation=c["save"])
    if c["kind"] == "linear":
        got = ops.linear(s["x"], s["weight"], s["bias"], residual=s.get("residual"), **more)
    else:
        got = ops.grouped_linear(s["x"], s["weight"], s["offsets"], s["bias"], **more)
    return dict(y=got[0], z=got[1]) if c["save"] else dict(y=got)


# ----------------------------------------------------------------- what it costs
def work(case):
    m, n, k = case["m"], case["n"], case["k"]
    rows = m - case.get("rest", 0)
    experts = case.get("active", 1)
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["kind"].endswith("backward"):
        read = rows * n * size[case["out"]] + (rows * n * 2 if case["act"] != "none" else 0) + rows * k * 2 + experts * n * k * 2
        write = rows * k * 2 + case.get("groups", 1) * n * k * size[case["dw"]] + (case.get("groups", 1) * n * 4 if case["bias"] else 0)
        return dict(bytes=read + write, flops=4 * rows * n * k)
    read = rows * k * 2 + experts * n * k * 2 + (experts * n * 2 if case["bias"] else 0) + (rows * n * 2 if case.get("residual") else 0)
    return dict(bytes=read + rows * n * (size[case["out"]] + (2 if case["save"] else 0)), flops=2 * rows * n * k)


# --------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    act = case["act"]
    d = lambda t: t.to(torch.float64)  # noqa: E731
    normal = lambda v: torch.special.ndtr(v)  # noqa: E731

    def activate(v):
        return {"none": lambda: v, "relu": lambda: torch.clamp(v, min=0), "gelu": lambda: v * normal(v),
                "gelu_tanh": lambda: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)),
                "silu": lambda: v * torch.sigmoid(v)}[act]()

    def slope(v):
        if act == "gelu":
            return normal(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
        if act == "relu":
            return torch.heaviside(v, torch.zeros((), dtype=v.dtype, device=v.device))
        a = 2 * math.sqrt(2 / math.pi) if act == "gelu_tanh" else 1.0
        b = 0.044715 if act == "gelu_tanh" else 0.0
        p = torch.sigmoid(a * (v + b * v ** 3))
        return p + v * p * (1 - p) * a * (1 + 3 * b * v * v)

    ends = s["offsets"].tolist() if "offsets" in s else [0, case["m"]]
    weights = s["weight"] if "offsets" in s else s["weight"][None]
    biases = None if s["bias"] is None else (s["bias"] if "offsets" in s else s["bias"][None])
    m, n, k = case["m"], case["n"], case["k"]
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device=s["x"].device)  # noqa: E731
    if case["kind"].endswith("backward"):
        dx, dw, db = new(m, k), new(len(ends) - 1, n, k), new(len(ends) - 1, n)
        for g, (b, e) in enumerate(zip(ends[:-1], ends[1:])):
            dz = d(s["dy"][b:e])
            if act != "none":
                dz = dz * slope(d(s["z"][b:e]))
            dx[b:e] = torch.einsum("mn,nk->mk", dz, d(weights[g]))
            dw[g] = torch.einsum("mn,mk->nk", dz, d(s["x"][b:e]))
            db[g] = torch.einsum("mn->n", dz)
        if "offsets" not in s:
            dw, db = dw[0], db[0]
        return dict(dx=dx, dw=dw, **(dict(db=db) if case["bias"] else {}))
    y, z = new(m, n), new(m, n)
    for g, (b, e) in enumerate(zip(ends[:-1], ends[1:])):
        z[b:e] = torch.einsum("mk,nk->mn", d(s["x"][b:e]), d(weights[g]))
        if biases is not None:
            z[b:e] += d(biases[g])
        y[b:e] = activate(z[b:e])
    if s.get("residual") is not None:
        y += d(s["residual"])
    return dict(y=y, **(dict(z=z) if case["save"] else {}))

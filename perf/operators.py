"""The operators of a residual stack of routed experts, as measurable cases.

Kinds of case:
  norm     the norm after a block, its gate and residual scale, and the norm
           before the next block, in one pass over the residual stream
           (`train`: with the gradients of everything that goes in)
  act8     an activation kept in 8 bits and brought back
  grouped  rows sorted by expert times that expert's weight (`train`: with
           both gradients; `keep`: the rows kept in 8 bits for the weight
           gradient)

With `own` false `run` computes them from elementary torch operations in 32
bits; with `own` true it calls the framework.  Inputs come from the seed alone;
`exact` evaluates the definitions in float64.
"""

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
QMAX = {"int8": 127.0, "e4m3": 448.0}


def _norm(name, rows, width, dtype, train, gate="none", act="none", seqs=1, stream=None):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype,
            "stream": stream or dtype, "train": train, "gate": gate, "act": act, "seqs": seqs}


def _act8(name, rows, width, dtype, form, group):
    return {"name": name, "kind": "act8", "rows": rows, "width": width, "dtype": dtype,
            "form": form, "group": group}


def _grouped(name, rows, experts, k, n, dtype, train, keep="none", group=128, skew=0.7):
    return {"name": name, "kind": "grouped", "rows": rows, "experts": experts, "k": k, "n": n,
            "dtype": dtype, "train": train, "keep": keep, "group": group, "skew": skew}


def listed():
    return [
        # one token of a served stack between two blocks: latency
        _norm("norm_token_bf16", 1, 1024, "bf16", False),
        # a prompt through the stack, the stream kept in float32
        _norm("norm_prompt_mixed", 4096, 4096, "bf16", False, stream="f32"),
        # a training step at odd sizes, a learned gate for every token
        _norm("norm_train_odd_f32", 5003, 301, "f32", True, gate="token", act="sigmoid"),
        # a training step of a wide stack, conditioned by sequence (the largest norm)
        _norm("norm_train_bf16", 16384, 4096, "bf16", True, gate="sequence", act="tanh", seqs=8),
        # a small minibatch's hidden activations: launches and latency
        _act8("act8_small_f32", 32, 784, "f32", "int8", 128),
        # odd sizes, half precision, the last group of a row short
        _act8("act8_odd_f16", 10007, 1001, "f16", "e4m3", 64),
        # the activations of a wide layer at full batch
        _act8("act8_65536_bf16", 65536, 1024, "bf16", "int8", 128),
        # one decoding step: a few tokens, each at its own experts
        _grouped("grouped_decode_bf16", 8, 16, 1024, 4096, "bf16", False),
        # odd sizes in float32, forward and backward
        _grouped("grouped_train_odd_f32", 5003, 7, 301, 257, "f32", True),
        # a prompt through wide experts
        _grouped("grouped_prompt_bf16", 16384, 8, 4096, 4096, "bf16", False),
        # a training step of many experts in half precision
        _grouped("grouped_train_f16", 8192, 32, 1024, 1024, "f16", True),
        # a training step whose rows are kept in 8 bits
        _grouped("grouped_train_keep_bf16", 32768, 16, 1024, 4096, "bf16", True, keep="int8"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A size over the logarithm of the range: an odd number, an odd multiple
    of 8 or a power of two."""
    v = _log(rng, lo, hi)
    v = rng.choice([v | 1, v // 16 * 16 + 8, 1 << (v.bit_length() - 1)])
    return min(hi, max(lo, v))


def draw(rng):
    kind = rng.choice(["norm", "act8", "grouped", "grouped"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "norm":
        width = _width(rng, 64, 8192)
        seqs = rng.randint(1, 16)
        rows = _log(rng, 1, min(32768, 67108864 // width))
        gate = rng.choice(["none", "element", "token", "sequence"])
        if gate == "sequence":
            rows = max(1, rows // seqs) * seqs
        c = _norm("", rows, width, dtype, rng.random() < 0.6, gate,
                  "none" if gate == "none" else rng.choice(["none", "sigmoid", "tanh", "silu"]),
                  seqs, rng.choice([None, "f32"]))
    elif kind == "act8":
        width = _width(rng, 16, 8192)
        c = _act8("", _log(rng, 1, 67108864 // width), width, dtype,
                  rng.choice(["int8", "e4m3"]), rng.choice([32, 64, 128, 256]))
    else:
        train = rng.random() < 0.6
        k, n = _width(rng, 64, 4096), _width(rng, 64, 4096)
        most = 1 << (36 if dtype == "f32" else 37)  # k n rows: the largest listed one's and below
        rows = _log(rng, 1, min(32768, most // (k * n)))
        c = _grouped("", rows, _log(rng, 1, 64), k, n, dtype, train,
                     rng.choice(["none", "int8", "e4m3"]) if train else "none",
                     rng.choice([32, 64, 128, 256]), rng.uniform(0.0, 1.5))
    del c["name"]
    return c


def _gate_shape(case):
    if case["gate"] == "element":
        return (case["seqs"], case["rows"] // case["seqs"], case["width"])
    if case["gate"] == "token":
        return (case["seqs"], case["rows"] // case["seqs"], 1)
    return (case["seqs"], 1, case["width"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        v = torch.randn(*shape, generator=g, device="cuda") * std + mean
        return v.to(dtype)

    def channels(width):  # some channels of an activation are far larger than the rest
        big = torch.rand(width, generator=g, device="cuda") < 0.01
        return torch.where(big, 12.0, 1.0)

    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["kind"] == "norm":
        seqs = case["seqs"] if case["rows"] % case["seqs"] == 0 else 1
        case = dict(case, seqs=seqs)
        st["case"] = case
        shape = (seqs, case["rows"] // seqs, case["width"])
        c = channels(case["width"])
        sdt = DTYPES[case["stream"]]
        st["x"] = (normal(*shape, std=2.0) * c).to(sdt)
        st["y"] = (normal(*shape) * c).to(dt)
        st["post"] = normal(case["width"], dtype=dt, std=0.1, mean=1.0)
        st["pre"] = normal(case["width"], dtype=dt, std=0.1, mean=1.0)
        st["scale"] = normal(case["width"], dtype=dt, std=0.05, mean=0.2)
        st["gate"] = None if case["gate"] == "none" else normal(*_gate_shape(case), dtype=dt)
        if case["train"]:
            st["dx"] = normal(*shape, dtype=sdt)
            st["dh"] = normal(*shape, dtype=dt)
            for name in ("x", "y", "post", "pre", "scale", "gate"):
                if st[name] is not None:
                    st[name].requires_grad_()
    elif case["kind"] == "act8":
        st["x"] = (normal(case["rows"], case["width"]) * channels(case["width"])).to(dt)
    else:
        e, k, n = case["experts"], case["k"], case["n"]
        load = torch.softmax(torch.randn(e, generator=g, device="cuda") * case["skew"], 0)
        ids = torch.multinomial(load, case["rows"], replacement=True, generator=g)
        offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = torch.bincount(ids, minlength=e).cumsum(0)
        st["offsets"] = offsets
        st["bounds"] = offsets.tolist()  # the plain form's loop needs them on the host
        st["x"] = (normal(case["rows"], k) * channels(k)).to(dt)
        st["w"] = normal(e, n, k, dtype=dt, std=k ** -0.5)
        if case["train"]:
            st["dy"] = normal(case["rows"], n, dtype=dt)
            st["x"].requires_grad_()
            st["w"].requires_grad_()
    return st


# ---------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits, rounded once at the end
# ---------------------------------------------------------------------------

_ACTS = {"none": lambda v: v, "sigmoid": lambda v: 1 / (1 + (-v).exp()),
         "tanh": lambda v: 1 - 2 / (1 + (2 * v).exp()), "silu": lambda v: v / (1 + (-v).exp())}


def _plain_norm(st):
    case = st["case"]
    x, y = st["x"].float(), st["y"].float()
    branch = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * st["post"].float()
    branch = branch * st["scale"].float()
    if st["gate"] is not None:
        branch = branch * _ACTS[case["act"]](st["gate"].float())
    new = x + branch
    h = new * (new.square().mean(-1, keepdim=True) + EPS).rsqrt() * st["pre"].float()
    return new.to(st["x"].dtype), h.to(st["y"].dtype)


def _plain_keep(x, form, group):
    """(restored values in float32, scales) of rows kept in 8 bits."""
    rows, width = x.shape
    parts = -(-width // group)
    v = torch.zeros(rows, parts * group, dtype=torch.float32, device=x.device)
    v[:, :width] = x
    v = v.reshape(rows, parts, group)
    scale = v.abs().amax(-1, keepdim=True) / QMAX[form]
    u = torch.where(scale > 0, v * (1 / scale), torch.zeros_like(v))
    u = u.round() if form == "int8" else u.to(torch.float8_e4m3fn).float()
    back = (u * scale).reshape(rows, parts * group)[:, :width]
    return back, scale[..., 0]


def _plain_grouped(st):
    case, bounds = st["case"], st["bounds"]
    x, w = st["x"].detach(), st["w"].detach()
    y = torch.empty(case["rows"], case["n"], dtype=x.dtype, device=x.device)
    if case["train"]:
        dy = st["dy"]
        kept = x.float() if case["keep"] == "none" else _plain_keep(x, case["keep"], case["group"])[0]
        dx, dw = torch.empty_like(x), torch.empty_like(w)
    for e in range(case["experts"]):
        rows = slice(bounds[e], bounds[e + 1])
        we = w[e].float()
        y[rows] = (x[rows].float() @ we.t()).to(x.dtype)
        if case["train"]:
            de = dy[rows].float()
            dx[rows] = (de @ we).to(x.dtype)
            dw[e] = (de.t() @ kept[rows]).to(x.dtype)
    return {"y": y, "dx": dx, "dw": dw} if case["train"] else {"y": y}


def _norm_grads(st, outs):
    names = [n for n in ("x", "y", "post", "pre", "scale", "gate") if st[n] is not None]
    grads = torch.autograd.grad(outs, [st[n] for n in names], [st["dx"], st["dh"]])
    return {"d" + n: v for n, v in zip(names, grads)}


def run(st):
    case = st["case"]
    if own:
        import torchsplinekan_amd as tk
    if case["kind"] == "norm":
        if own:
            outs = tk.residual_norm(
                st["x"], st["y"], post_weight=st["post"], pre_weight=st["pre"], scale=st["scale"],
                gate=st["gate"], gate_act=None if case["act"] == "none" else case["act"], eps=EPS)
        else:
            outs = _plain_norm(st)
        r = {"x": outs[0].detach(), "h": outs[1].detach()}
        if case["train"]:
            r.update(_norm_grads(st, outs))
        return r
    if case["kind"] == "act8":
        if own:
            kept = tk.quantize_activation(st["x"], group=case["group"], format=case["form"])
            return {"back": kept.dequantize(), "scale": kept.scale}
        back, scale = _plain_keep(st["x"].float(), case["form"], case["group"])
        return {"back": back.to(st["x"].dtype), "scale": scale}
    if own:
        y = tk.grouped_linear(st["x"], st["w"], st["offsets"], group=case["group"],
                              checkpoint=None if case["keep"] == "none" else case["keep"])
        if not case["train"]:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, [st["x"], st["w"]], st["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    return _plain_grouped(st)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    b = size[case["dtype"]]
    if case["kind"] == "norm":
        count, sb = case["rows"] * case["width"], size[case["stream"]]
        gate = 0
        if case["gate"] == "element":
            gate = count
        elif case["gate"] == "token":
            gate = case["rows"]
        elif case["gate"] == "sequence":
            gate = case["seqs"] * case["width"]
        total = count * 2 * (sb + b) + gate * b + 3 * case["width"] * b
        flops = 12 * count
        if case["train"]:
            total += count * 3 * (sb + b) + 2 * gate * b + 6 * case["width"] * b
            flops += 30 * count
        return {"bytes": total, "flops": flops}
    if case["kind"] == "act8":
        count = case["rows"] * case["width"]
        scales = case["rows"] * -(-case["width"] // case["group"]) * 4
        return {"bytes": 2 * (count * (b + 1) + scales), "flops": 4 * count}
    t, k, n = case["rows"], case["k"], case["n"]
    weights = min(case["experts"], t) * k * n * b
    total, flops = t * (k + n) * b + weights, 2 * t * k * n
    if case["train"]:
        kept = t * k * b
        if case["keep"] != "none":
            kept = t * k + t * -(-k // case["group"]) * 4
            total += kept  # written, besides being read below
        total += t * (k + n) * b + kept + weights + case["experts"] * k * n * b
        flops *= 3
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------------------
# the definitions in float64
# ---------------------------------------------------------------------------

def _exact_norm(st):
    case = st["case"]
    x, y = st["x"].detach().double(), st["y"].detach().double()
    post, pre, scale = (st[n].detach().double() for n in ("post", "pre", "scale"))
    r1 = 1 / torch.sqrt((y * y).sum(-1, keepdim=True) / case["width"] + EPS)
    yhat = y * r1
    if st["gate"] is None:
        a, slope = torch.ones((), dtype=torch.float64, device=x.device), None
    else:
        v = st["gate"].detach().double()
        sg = torch.sigmoid(v)
        a, slope = {"none": (v, torch.ones_like(v)), "sigmoid": (sg, sg * (1 - sg)),
                    "tanh": (torch.tanh(v), 1 - torch.tanh(v) ** 2),
                    "silu": (v * sg, sg * (1 + v * (1 - sg)))}[case["act"]]
    u = yhat * post
    new = x + scale * a * u
    r2 = 1 / torch.sqrt((new * new).sum(-1, keepdim=True) / case["width"] + EPS)
    xhat = new * r2
    r = {"x": new, "h": xhat * pre}
    if not case["train"]:
        return r
    dh = st["dh"].double()
    t = dh * pre
    d = st["dx"].double() + r2 * (t - xhat * (t * xhat).sum(-1, keepdim=True) / case["width"])
    v = d * scale * a
    w = v * post
    r["dx"] = d
    r["dy"] = r1 * (w - yhat * (w * yhat).sum(-1, keepdim=True) / case["width"])
    r["dpost"] = (v * yhat).sum((0, 1))
    r["dpre"] = (dh * xhat).sum((0, 1))
    r["dscale"] = (d * a * u).sum((0, 1))
    if slope is not None:
        full = d * scale * u * slope
        r["dgate"] = {"element": lambda: full, "token": lambda: full.sum(-1, keepdim=True),
                      "sequence": lambda: full.sum(1, keepdim=True)}[case["gate"]]()
    return r


def _exact_keep(x, form, group):
    x = x.detach().double()
    back = torch.empty_like(x)
    scales = []
    for lo in range(0, x.shape[1], group):
        part = x[:, lo:lo + group]
        step = part.abs().max(1, keepdim=True).values / QMAX[form]
        scales.append(step)
        q = part / torch.where(step == 0, 1.0, step)
        if form == "int8":
            q = torch.round(q)
        else:  # 3 bits after the leading one, the last of them 2^-9 at least
            _, ex = torch.frexp(q)
            ulp = torch.ldexp(torch.ones_like(q), (ex - 4).clamp(min=-9))
            q = torch.round(q / ulp) * ulp
        back[:, lo:lo + group] = q * step
    return back, torch.cat(scales, 1)


def exact(case, seed):
    st = prepare(case, seed)
    case = st["case"]
    if case["kind"] == "norm":
        return _exact_norm(st)
    if case["kind"] == "act8":
        back, scale = _exact_keep(st["x"], case["form"], case["group"])
        return {"back": back, "scale": scale}
    x, w = st["x"].detach().double(), st["w"].detach()
    y, dx, dw = [], [], []
    kept = x
    if case["keep"] != "none":
        kept = _exact_keep(st["x"], case["keep"], case["group"])[0]
    for e in range(case["experts"]):
        lo, hi = st["bounds"][e], st["bounds"][e + 1]
        we = w[e].double()
        y.append(torch.mm(x[lo:hi], we.t()))
        if case["train"]:
            de = st["dy"][lo:hi].double()
            dx.append(torch.mm(de, we))
            dw.append(torch.mm(de.t(), kept[lo:hi]))
    r = {"y": torch.cat(y)}
    if case["train"]:
        r.update(dx=torch.cat(dx), dw=torch.stack(dw))
    return r

"""The operators that a residual stack needs to be trained on tokens or classes,
as measurable cases.

Kinds of case:
  ln       layer norm (`train`: with the gradients of its input, weight and bias)
  gated    act(x Wg^T) * (x Wu^T), for all rows alike or with weights by expert
           (`experts` > 0: rows sorted by expert; `train`: with both gradients)
  xent     softmax cross entropy of x W^T over a vocabulary (`train`: with the
           gradients of x and W)
  distill  a student's softmax of x W^T against a teacher's top logits (`train`:
           with the gradients of x and W)

With `own` false `run` computes them from elementary torch operations in 32
bits; with `own` true it calls the framework.  Inputs come from the seed alone;
`exact` evaluates the definitions in float64.
"""

import math

import torch

own = False

EPS = 1e-5
IGNORE = -100
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
ACTS = ["silu", "gelu", "sigmoid", "relu"]


def _ln(name, rows, width, dtype, train, stream=None):
    return {"name": name, "kind": "ln", "rows": rows, "width": width, "dtype": dtype,
            "stream": stream or dtype, "train": train}


def _gated(name, rows, k, n, dtype, train, act="silu", experts=0, skew=0.7):
    return {"name": name, "kind": "gated", "rows": rows, "k": k, "n": n, "dtype": dtype,
            "train": train, "act": act, "experts": experts, "skew": skew}


def _xent(name, rows, k, vocab, dtype, train, ignored=0.1, reduction="mean"):
    return {"name": name, "kind": "xent", "rows": rows, "k": k, "vocab": vocab, "dtype": dtype,
            "train": train, "ignored": ignored, "reduction": reduction}


def _distill(name, rows, k, vocab, top, dtype, train, temperature=2.0, absent=0.05):
    return {"name": name, "kind": "distill", "rows": rows, "k": k, "vocab": vocab, "top": top,
            "dtype": dtype, "train": train, "temperature": temperature, "absent": absent}


def listed():
    return [
        # one token of a served stack: latency
        _ln("ln_token_bf16", 1, 1024, "bf16", False),
        # a training step at odd sizes
        _ln("ln_train_odd_f32", 5003, 301, "f32", True),
        # a training step of a wide stack (the largest norm)
        _ln("ln_train_bf16", 16384, 4096, "bf16", True),
        # one decoding step of a small batch
        _gated("gated_decode_bf16", 8, 1024, 4096, "bf16", False),
        # odd sizes in float32, forward and backward
        _gated("gated_train_odd_f32", 5003, 301, 257, "f32", True, act="gelu"),
        # a training step of many experts in half precision
        _gated("gated_experts_f16", 8192, 1024, 1024, "f16", True, experts=16),
        # a training step of a wide block
        _gated("gated_train_bf16", 16384, 1024, 4096, "bf16", True),
        # the scores of a short text under a large vocabulary
        _xent("xent_score_bf16", 33, 1024, 32768, "bf16", False, ignored=0.0, reduction="none"),
        # a classifier of few classes at full batch
        _xent("xent_classes_f32", 4096, 256, 10, "f32", True, ignored=0.0),
        # a training step over a large vocabulary (the largest)
        _xent("xent_train_bf16", 8192, 2048, 65536, "bf16", True),
        # odd sizes, half precision, a few of the teacher's logits
        _distill("distill_odd_f16", 1021, 777, 32003, 8, "f16", True, temperature=1.0),
        # a student of a large vocabulary
        _distill("distill_train_bf16", 4096, 1024, 65536, 64, "bf16", True),
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
    kind = rng.choice(["ln", "gated", "xent", "distill"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.6
    if kind == "ln":
        width = _width(rng, 16, 16384)
        c = _ln("", _log(rng, 1, min(65536, 67108864 // width)), width, dtype, train,
                rng.choice([None, "f32"]))
    elif kind == "gated":
        k, n = _width(rng, 64, 4096), _width(rng, 64, 4096)
        most = 1 << (34 if dtype == "f32" else 36)  # rows k n: the largest listed one's and below
        c = _gated("", _log(rng, 1, min(32768, most // (k * n))), k, n, dtype, train,
                   rng.choice(ACTS), rng.choice([0, 0, _log(rng, 1, 64)]), rng.uniform(0.0, 1.5))
    else:
        k, vocab = _width(rng, 32, 4096), _width(rng, 2, 131072)
        most = 1 << (36 if dtype == "f32" else 39)
        rows = _log(rng, 1, min(16384, (1 << 30) // vocab, most // (k * vocab)))
        if kind == "xent":
            c = _xent("", rows, k, vocab, dtype, train, rng.choice([0.0, 0.3]),
                      rng.choice(["mean", "sum", "none"]))
        else:
            c = _distill("", rows, k, vocab, min(vocab, _log(rng, 1, 256)), dtype, train,
                         rng.choice([1.0, 2.0, 4.0]), rng.choice([0.0, 0.2]))
    del c["name"]
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        v = torch.randn(*shape, generator=g, device="cuda") * std + mean
        return v.to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def channels(width):  # some channels of an activation are far larger than the rest
        return torch.where(uniform(width) < 0.01, 12.0, 1.0)

    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["kind"] == "ln":
        shape = (case["rows"], case["width"])
        sdt = DTYPES[case["stream"]]
        st["x"] = (normal(*shape, std=2.0, mean=0.3) * channels(case["width"])).to(sdt)
        st["w"] = normal(case["width"], dtype=dt, std=0.1, mean=1.0)
        st["b"] = normal(case["width"], dtype=dt, std=0.1)
        if case["train"]:
            st["dy"] = normal(*shape, dtype=dt)
            for name in ("x", "w", "b"):
                st[name].requires_grad_()
        return st
    t, k = case["rows"], case["k"]
    if case["kind"] == "gated":
        e, n = case["experts"], case["n"]
        st["x"] = (normal(t, k) * channels(k)).to(dt)
        st["w"] = normal(*((e, 2, n, k) if e else (2, n, k)), dtype=dt, std=k ** -0.5)
        if e:
            load = torch.softmax(torch.randn(e, generator=g, device="cuda") * case["skew"], 0)
            ids = torch.multinomial(load, t, replacement=True, generator=g).sort().values
            count = torch.bincount(ids, minlength=e)
            st["offsets"] = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
            st["offsets"][1:] = count.cumsum(0)
            # the plain form's places: row t is row `place` of expert `ids`, of `most` at most
            st["ids"], st["most"] = ids, int(count.max())
            st["place"] = torch.arange(t, device="cuda") - st["offsets"].long()[ids]
        if case["train"]:
            st["dh"] = normal(t, n, dtype=dt)
            st["x"].requires_grad_()
            st["w"].requires_grad_()
        return st
    vocab = case["vocab"]
    st["w"] = normal(vocab, k, dtype=dt, std=2 * k ** -0.5)
    # frequent tokens have low numbers, as where a vocabulary is sorted by frequency
    answer = (vocab * uniform(t) ** 3).long().clamp_(max=vocab - 1)
    # a trained model's state: near its answer's weight more than others'
    st["x"] = (normal(t, k) * channels(k) + 2.5 * st["w"][answer]).to(dt)
    if case["kind"] == "xent":
        st["target"] = torch.where(uniform(t) < case["ignored"], IGNORE, answer)
        if case["rows"]:
            st["target"][0] = answer[0]
    else:
        top = case["top"]
        # distinct numbers, low ones more often, in no order; a row may have fewer of them
        u = (torch.arange(top, device="cuda") + uniform(t, top)) / top
        ids = ((vocab - top) * u ** 3).long() + torch.arange(top, device="cuda")
        st["ids"] = ids.gather(1, uniform(t, top).argsort(1))
        st["ids"][:, 0] = torch.where((ids == answer[:, None]).any(1), st["ids"][:, 0], answer)
        st["teacher"] = normal(t, top, std=2.0).sort(1, descending=True).values
        gone = uniform(t, top) < case["absent"]
        gone[0] = False
        st["ids"] = torch.where(gone, -1, st["ids"])
    if case["train"]:
        if case.get("reduction") == "none":  # each row has a weight of its own
            st["g"] = normal(t, std=0.1, mean=1.0)
        else:  # half precision's gradients of a mean need a loss scale
            mean = case.get("reduction", "mean") == "mean"
            scale = 2.0 ** int(math.log2(t)) if mean and case["dtype"] == "f16" else 1.0
            st["g"] = torch.full((), scale, device="cuda")
        st["x"].requires_grad_()
        st["w"].requires_grad_()
    return st


# ---------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits, rounded once at the end
# ---------------------------------------------------------------------------

def _plain_ln(st):
    case = st["case"]
    x, w, b = st["x"].detach().float(), st["w"].detach().float(), st["b"].detach().float()
    xc = x - x.mean(-1, keepdim=True)
    r = (xc.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh = xc * r
    res = {"y": (xh * w + b).to(st["w"].dtype)}
    if case["train"]:
        dy = st["dy"].float()
        u = dy * w
        dx = r * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
        res.update(dx=dx.to(st["x"].dtype), dw=(dy * xh).sum(0).to(st["w"].dtype),
                   db=dy.sum(0).to(st["b"].dtype))
    return res


def _act(name, v):
    """(act(v), act'(v))"""
    if name == "relu":
        on = (v > 0).float()
        return v * on, on
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(v * 0.5 ** 0.5))
        return v * cdf, cdf + v * (v * v * -0.5).exp() * (2 * math.pi) ** -0.5
    s = 1 / (1 + (-v).exp())
    if name == "sigmoid":
        return s, s * (1 - s)
    return v * s, s * (1 + v * (1 - s))


def _plain_gated(st):
    case = st["case"]
    dt, n, k, e = st["x"].dtype, case["n"], case["k"], max(1, case["experts"])
    w = st["w"].detach().float().reshape(e, 2 * n, k)

    def spread(v):  # rows by expert, padded to the largest
        if not case["experts"]:
            return v.float()[None]
        out = v.new_zeros(e, st["most"], v.shape[1], dtype=torch.float32)
        out[st["ids"], st["place"]] = v.float()
        return out

    def rows(v):
        return (v[st["ids"], st["place"]] if case["experts"] else v[0]).to(dt)

    x = spread(st["x"].detach())
    pre = torch.bmm(x, w.transpose(1, 2).contiguous())
    a, slope = _act(case["act"], pre[..., :n])
    up = pre[..., n:]
    res = {"h": rows(a * up)}
    if case["train"]:
        dh = spread(st["dh"])
        dpre = torch.cat([dh * up * slope, dh * a], -1)
        res["dx"] = rows(torch.bmm(dpre, w))
        res["dw"] = torch.bmm(dpre.transpose(1, 2).contiguous(), x).reshape(st["w"].shape).to(dt)
    return res


def _plain_loss(st):
    """Cross entropy and distillation: the loss against probabilities on a few ids."""
    case = st["case"]
    x, w = st["x"].detach().float(), st["w"].detach().float()
    tau = case.get("temperature", 1.0)
    if case["kind"] == "xent":
        ids, p = st["target"][:, None], torch.ones(case["rows"], 1, device=x.device)
        p = torch.where(ids >= 0, p, 0.0)
    else:
        ids = st["ids"]
        v = torch.where(ids >= 0, st["teacher"] / tau, -math.inf)
        p = (v - v.amax(1, keepdim=True).clamp(min=-1e30)).exp()
        p = p / p.sum(1, keepdim=True).clamp(min=1e-30)
    counted = (ids >= 0).any(1)
    z = (x @ w.t()) / tau
    top = z.amax(1, keepdim=True)
    q = (z - top).exp()
    total = q.sum(1, keepdim=True)
    at = ids.clamp(min=0)
    logq = z.gather(1, at) - top - total.log()
    loss = (p * (p.clamp(min=1e-38).log() - logq)).sum(1) * tau * tau
    loss = torch.where(counted, loss, 0.0)
    reduction = case.get("reduction", "mean")
    res = {"loss": loss if reduction == "none" else loss.sum()}
    if reduction == "mean":
        res["loss"] = res["loss"] / counted.sum()
    if case["train"]:
        g = st["g"] / counted.sum() if reduction == "mean" else st["g"]
        q.div_(total)
        q.scatter_add_(1, at, -p)
        q.mul_((g * counted * tau)[:, None])
        res["dx"] = (q @ w).to(st["x"].dtype)
        res["dw"] = (q.t() @ x).to(st["w"].dtype)
    return res


def run(st):
    case = st["case"]
    if not own:
        return {"ln": _plain_ln, "gated": _plain_gated, "xent": _plain_loss,
                "distill": _plain_loss}[case["kind"]](st)
    import torchsplinekan_amd as tk
    if case["kind"] == "ln":
        y = tk.layer_norm(st["x"], st["w"], st["b"], eps=EPS, dtype=st["w"].dtype)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, [st["x"], st["w"], st["b"]], st["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if case["kind"] == "gated":
        h = tk.gated_linear(st["x"], st["w"], st.get("offsets"), act=case["act"])
        if not case["train"]:
            return {"h": h}
        dx, dw = torch.autograd.grad(h, [st["x"], st["w"]], st["dh"])
        return {"h": h.detach(), "dx": dx, "dw": dw}
    if case["kind"] == "xent":
        loss = tk.linear_cross_entropy(st["x"], st["w"], st["target"], ignore_index=IGNORE,
                                       reduction=case["reduction"])
    else:
        loss = tk.linear_distillation(st["x"], st["w"], st["ids"], st["teacher"],
                                      temperature=case["temperature"])
    if not case["train"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, [st["x"], st["w"]], st["g"])
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def work(case):
    b, train = SIZES[case["dtype"]], case["train"]
    if case["kind"] == "ln":
        count, sb = case["rows"] * case["width"], SIZES[case["stream"]]
        total, flops = count * (sb + b) + 2 * case["width"] * b, 8 * count
        if train:
            total += count * (2 * sb + b) + 3 * case["width"] * b
            flops += 14 * count
        return {"bytes": total, "flops": flops}
    t, k = case["rows"], case["k"]
    if case["kind"] == "gated":
        n, e = case["n"], max(1, case["experts"])
        weights = min(e, t) * 2 * n * k * b
        total, flops = t * (k + n) * b + weights, 4 * t * n * k
        if train:
            total += t * (2 * k + n) * b + weights + e * 2 * n * k * b
            flops *= 3
        return {"bytes": total, "flops": flops}
    vocab = case["vocab"]
    label = 8 if case["kind"] == "xent" else 12 * case["top"]
    total, flops = (t + vocab) * k * b + t * label, 2 * t * vocab * k
    if train:
        total += 2 * (t + vocab) * k * b + t * label
        flops *= 3
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------------------
# the definitions in float64
# ---------------------------------------------------------------------------

def _exact_ln(st):
    x, w, b = (st[n].detach().double() for n in ("x", "w", "b"))
    c = x.shape[1]
    m = x.sum(1, keepdim=True) / c
    var = ((x - m) ** 2).sum(1, keepdim=True) / c
    sd = torch.sqrt(var + EPS)
    n = (x - m) / sd
    r = {"y": n * w + b}
    if st["case"]["train"]:
        dy = st["dy"].double()
        r["db"], r["dw"] = dy.sum(0), (dy * n).sum(0)
        u = dy * w
        r["dx"] = (u - (u.sum(1, keepdim=True) + n * (u * n).sum(1, keepdim=True)) / c) / sd
    return r


_DENSITY = 1 / math.sqrt(2 * math.pi)
_EXACT_ACTS = {
    "relu": lambda v: (torch.relu(v), torch.heaviside(v, torch.zeros_like(v))),
    "sigmoid": lambda v: (torch.sigmoid(v), torch.sigmoid(v) * torch.sigmoid(-v)),
    "silu": lambda v: (v * torch.sigmoid(v),
                       torch.sigmoid(v) + v * torch.sigmoid(v) * torch.sigmoid(-v)),
    "gelu": lambda v: (0.5 * v * torch.erfc(-v / math.sqrt(2)),
                       0.5 * torch.erfc(-v / math.sqrt(2)) + _DENSITY * v * torch.exp(-v * v / 2)),
}


def _exact_gated(st):
    case = st["case"]
    x, w = st["x"].detach().double(), st["w"].detach()
    e = case["experts"]
    bounds = st["offsets"].tolist() if e else [0, case["rows"]]
    h, dx, dw = [], [], []
    for i in range(max(1, e)):
        gate, up = (w[i] if e else w).double()
        part = x[bounds[i]:bounds[i + 1]]
        a, slope = _EXACT_ACTS[case["act"]](part @ gate.t())
        u = part @ up.t()
        h.append(a * u)
        if case["train"]:
            d = st["dh"][bounds[i]:bounds[i + 1]].double()
            dgate, dup = d * u * slope, d * a
            dx.append(dgate @ gate + dup @ up)
            dw.append(torch.stack([dgate.t() @ part, dup.t() @ part]))
    r = {"h": torch.cat(h)}
    if case["train"]:
        r.update(dx=torch.cat(dx), dw=torch.stack(dw) if e else dw[0])
    return r


def _exact_loss(st):
    case = st["case"]
    x, w = st["x"].detach().double(), st["w"].detach().double()
    tau = case.get("temperature", 1.0)
    t, vocab = case["rows"], case["vocab"]
    # row blocks: the softmax of all rows at once can take 8 GB a tensor
    step = max(1, (1 << 28) // vocab)
    if case["kind"] == "xent":
        mask = st["target"] != IGNORE
        ids, share = st["target"].clamp(min=0)[:, None], mask.double()[:, None]
    else:
        there = st["ids"] >= 0
        mask, ids = there.any(1), st["ids"].clamp(min=0)
        score = (st["teacher"].double() / tau).masked_fill(~there, -math.inf)
        share = torch.nan_to_num(torch.softmax(score, 1))
    weight = torch.ones(t, dtype=torch.float64, device=x.device)
    if case["train"]:
        weight = weight * st["g"]
    if case.get("reduction", "mean") == "mean":
        weight = weight / mask.sum()
    losses, dx, dw = [], [], torch.zeros_like(w)
    for lo in range(0, t, step):
        s = slice(lo, lo + step)
        logp = torch.log_softmax(x[s] @ w.t() / tau, 1)
        cross = torch.xlogy(share[s], share[s]) - share[s] * logp.gather(1, ids[s])
        losses.append(tau ** 2 * torch.where(mask[s], cross.sum(1), 0.0))
        if case["train"]:
            d = logp.exp_()
            d = d.scatter_add(1, ids[s], -share[s]) * (tau * weight[s] * mask[s])[:, None]
            dx.append(d @ w)
            dw += d.t() @ x[s]
        del logp
    loss = torch.cat(losses)
    reduction = case.get("reduction", "mean")
    if reduction != "none":
        loss = loss.sum() / (mask.sum() if reduction == "mean" else 1)
    r = {"loss": loss}
    if case["train"]:
        r.update(dx=torch.cat(dx), dw=dw)
    return r


def exact(case, seed):
    st = prepare(case, seed)
    return {"ln": _exact_ln, "gated": _exact_gated, "xent": _exact_loss,
            "distill": _exact_loss}[case["kind"]](st)

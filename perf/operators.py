"""What the framework's dense operators cost: the layer of a decoder (matrix product, bias, activation, residual), the
softmax cross entropy of a class head without its logits, and the class of each row, each in its plain form and as the
framework's call."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100


def _linear(name, rows, k, n, dtype, act, *, bias=True, residual=False, train=False, pad=0):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "residual": residual, "train": train, "pad": pad}


def _ce(name, rows, k, n, dtype, *, bias=True, train=True, ignored=0.0, reduction="mean", pad=0):
    return {"name": name, "op": "cross_entropy", "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": bias, "train": train, "ignored": ignored, "reduction": reduction, "pad": pad}


def _label(name, rows, k, n, dtype, *, bias=True, pad=0):
    return {"name": name, "op": "label", "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": bias, "pad": pad}


def listed():
    return [
        # one token through a feed-forward layer: the smallest call, the weight's bytes are all of it
        _linear("linear_one_row_bf16", 1, 4096, 8192, "bf16", "silu"),
        # a hidden layer of the point decoder: 16384 query points with 6 neighbours each (batch_size, query_nn_k), 64 units
        _linear("linear_points_f32", 16384 * 6, 64, 64, "f32", "relu"),
        # its first layer in training: 8 features and 3 coordinates to 64 units, one batch of samples
        _linear("linear_train_first_bf16", 16384, 11, 64, "bf16", "leaky_relu", train=True),
        # a wider decoder trained in single precision
        _linear("linear_train_f32", 4096, 1024, 1024, "f32", "gelu", residual=True, train=True),
        # a large model's layer in training
        _linear("linear_train_wide_bf16", 8192, 4096, 4096, "bf16", "gelu", residual=True, train=True),
        # odd sizes, rows of a wider buffer
        _linear("linear_ragged_f16", 1999, 1000, 777, "f16", "gelu", residual=True, pad=3),
        # the semantic head of the decoder: 20 classes and the unlabelled one, three samples in ten without a label
        _ce("ce_train_semantic_f32", 16384, 64, 21, "f32", ignored=0.3),
        # a vocabulary's head in training, single and half width
        _ce("ce_train_vocab_f32", 2048, 1024, 32000, "f32", bias=False),
        _ce("ce_train_vocab_bf16", 8192, 2048, 65536, "bf16", bias=False, ignored=0.1),
        # evaluation of a text: the loss of each of its tokens
        _ce("ce_eval_f16", 333, 768, 50021, "f16", train=False, reduction="none"),
        # the classes of one chunk of a mesher's grid (infer_bs points)
        _label("label_points_f32", 16384 * 64, 64, 21, "f32"),
        # one token's answer over a vocabulary
        _label("label_one_row_bf16", 1, 4096, 131072, "bf16", bias=False),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    op = rng.choice(["linear", "linear", "cross_entropy", "cross_entropy", "label"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    pad = rng.choice([0, 0, 0, 1, 8])
    bias = rng.random() < 0.7
    while True:
        rows = _log(rng, 1, 16384 if op == "cross_entropy" else 262144)
        k = _log(rng, 8, 8192)
        n = _log(rng, 8, 8192) if op == "linear" else _log(rng, 2, 131072)
        k, n = (v if rng.random() < 0.4 else max(8, v // 8 * 8) for v in (k, n))  # widths are multiples of 8 more often than not
        if rows * k * n <= (1 << 36) and rows * max(n, k) <= (1 << 28) and n * k <= (1 << 29):
            break
    if op == "linear":
        train = rng.random() < 0.5
        acts = ["none", "gelu", "silu"] + ([] if train and dtype == "f32" else ["relu", "leaky_relu"])
        return _linear("", rows, k, n, dtype, rng.choice(acts), bias=bias, residual=rng.random() < 0.4, train=train, pad=pad)
    if op == "cross_entropy":
        return _ce("", rows, k, n, dtype, bias=bias, train=rng.random() < 0.7, ignored=rng.choice([0.0, 0.0, 0.2, 0.8]), reduction=rng.choice(["mean", "sum", "none"]), pad=pad)
    return _label("", rows, k, n, dtype, bias=bias, pad=pad)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    rows, k, n = case["rows"], case["k"], case["n"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    w = normal(n, k).mul_(k ** -0.5)
    x = normal(rows, k)
    s = {"case": case}
    if case["op"] != "linear":  # features as a trained head meets them: most rows lean towards one class
        skew = torch.rand(rows, generator=gen, device="cuda").pow_(3)
        target = skew.mul_(n).long().clamp_(max=n - 1)
        x += 10 * torch.rand(rows, 1, generator=gen, device="cuda") * w[target]
        if case["op"] == "cross_entropy":
            lost = torch.rand(rows, generator=gen, device="cuda") < case["ignored"]
            s["target"] = target.masked_fill(lost, IGNORE)
            if case["train"]:  # 16-bit training scales its loss
                scale = 1024.0 if case["dtype"] == "f16" else 1.0
                g = torch.full((), scale, device="cuda")
                s["g"] = g * normal(rows).abs() / rows if case["reduction"] == "none" else g / rows if case["reduction"] == "sum" else g
    store = torch.zeros(rows, k + case["pad"], dtype=dt, device="cuda")
    store[:, :k] = x
    s["x"], s["w"] = store[:, :k], w.to(dt)
    s["b"] = (0.1 * normal(n)).to(dt) if case["bias"] else None
    if case["op"] == "linear":
        s["r"] = normal(rows, n).to(dt) if case["residual"] else None
        if case["train"]:
            s["dy"] = normal(rows, n).to(dt)
    if case.get("train"):
        for name in ("x", "w", "b"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "leaky_relu":
        return torch.where(z > 0, z, 0.01 * z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "leaky_relu":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, 0.01))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_linear(c, x, w, b, r, dy):
    dt = x.dtype
    x, w = x.float(), w.float()
    z = x @ w.t()
    if b is not None:
        z = z + b.float()
    y = _act(z, c["act"])
    if r is not None:
        y = y + r.float()
    out = {"y": y.to(dt)}
    if c["train"]:
        dz = dy.float() * _act_slope(z, c["act"])
        out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if b is not None:
            out["db"] = dz.sum(0).to(dt)
    return out


def _over_the_largest(z):
    """The lowest column of each row's largest value, the sum of exp(z - largest) over the other columns (log1p of it keeps what
    a confident row has, where log of the whole sum would round it away), and exp(z - largest)."""
    top = z.max(1, keepdim=True).values
    best = torch.where(z == top, torch.arange(z.shape[1], device=z.device), z.shape[1]).min(1, keepdim=True).values
    e = torch.exp(z - top)
    return best, e.scatter(1, best, 0.0).sum(1, keepdim=True), e


def _plain_ce(c, x, w, b, target, g):
    dt = x.dtype
    counts = target != IGNORE
    x, w = x.float(), w.float()
    x = torch.where(counts[:, None], x, torch.zeros_like(x))
    z = x @ w.t()
    if b is not None:
        z = z + b.float()
    best, rest, e = _over_the_largest(z)
    at = torch.where(counts, target, torch.zeros_like(target))[:, None]
    loss = torch.log1p(rest) + (z.gather(1, best) - z.gather(1, at))
    loss = torch.where(counts, loss[:, 0], torch.zeros_like(loss[:, 0]))
    many = counts.sum().clamp(min=1)
    out = {"loss": loss if c["reduction"] == "none" else loss.sum() if c["reduction"] == "sum" else loss.sum() / many}
    if c["train"]:
        row = g / many if c["reduction"] == "mean" else g
        row = torch.where(counts, row.expand(x.shape[0]), torch.zeros_like(loss))
        dz = e / (1 + rest)
        dz.scatter_(1, at, torch.expm1(-loss)[:, None])  # p - 1 where p is close to one
        dz = dz * row[:, None]
        out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if b is not None:
            out["db"] = dz.sum(0).to(dt)
    return out


def _plain_label(x, w, b):
    z = x.float() @ w.float().t()
    if b is not None:
        z = z + b.float()
    best, rest, _ = _over_the_largest(z)
    return {"label": best[:, 0], "log_prob": -torch.log1p(rest)[:, 0]}


def _gradients(out, s, of, g):
    leaves = {"d" + name: s[name] for name in ("x", "w", "b") if s[name] is not None}
    return out | dict(zip(leaves, torch.autograd.grad(of, list(leaves.values()), g)))


def _own_run(s):
    from clid_slam_amd.linear import linear_act, linear_label
    from clid_slam_amd.loss import linear_cross_entropy

    c = s["case"]
    if c["op"] == "label":
        label, log_prob = linear_label(s["x"], s["w"], s["b"])
        return {"label": label, "log_prob": log_prob}
    if c["op"] == "linear":
        y = linear_act(s["x"], s["w"], s["b"], activation=c["act"], residual=s["r"])
        return _gradients({"y": y.detach()}, s, y, s["dy"]) if c["train"] else {"y": y}
    loss = linear_cross_entropy(s["x"], s["w"], s["b"], s["target"], ignore_index=IGNORE, reduction=c["reduction"])
    return _gradients({"loss": loss.detach()}, s, loss, s["g"]) if c["train"] else {"loss": loss}


def run(state):
    if own:
        return _own_run(state)
    c = state["case"]
    with torch.no_grad():
        if c["op"] == "linear":
            return _plain_linear(c, state["x"], state["w"], state["b"], state["r"], state.get("dy"))
        if c["op"] == "cross_entropy":
            return _plain_ce(c, state["x"], state["w"], state["b"], state["target"], state.get("g"))
        return _plain_label(state["x"], state["w"], state["b"])


def work(case):
    m, k, n = case["rows"], case["k"], case["n"]
    size = 4 if case["dtype"] == "f32" else 2
    bias = n if case["bias"] else 0
    values, more, products = m * k + n * k + bias, 0, 1
    if case["op"] == "linear":
        values += m * n * (2 if case["residual"] else 1)
        if case["train"]:
            values += m * n + m * k + n * k + bias
            products = 3
    elif case["op"] == "cross_entropy":
        more = 8 * m + 4 * (m if case["reduction"] == "none" else 1)
        if case["train"]:
            values += m * k + n * k + bias
            products = 3
    else:
        more = 12 * m
    return {"bytes": size * values + more, "flops": 2 * products * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        x, w = s["x"].detach().double(), s["w"].detach().double()
        b = None if s["b"] is None else s["b"].detach().double()
        n = w.shape[0]
        step = max(1, (1 << 27) // n)  # rows at a time
        parts = {}
        dw, db = torch.zeros_like(w), torch.zeros(n, dtype=torch.float64, device=w.device)
        live = None if "target" not in s else (s["target"] != IGNORE)
        for i in range(0, x.shape[0], step):
            xi = x[i:i + step]
            if live is not None:
                xi = xi.masked_fill(~live[i:i + step, None], 0.0)
            z = torch.mm(xi, w.t()) if b is None else torch.addmm(b, xi, w.t())
            dz, got = None, {}
            if case["op"] == "linear":
                y, slope = _exact_act(z, case["act"])
                got["y"] = y if s["r"] is None else y + s["r"][i:i + step].double()
                if case["train"]:
                    dz = s["dy"][i:i + step].double() * slope
            else:
                lp = z - torch.logsumexp(z, 1, keepdim=True)
                if case["op"] == "label":
                    best = torch.argmax(lp, 1)  # a trained head's rows have no ties in 64 bits
                    got["label"], got["log_prob"] = best, lp.amax(1)
                else:
                    t, on = s["target"][i:i + step], live[i:i + step]
                    hot = torch.zeros_like(lp)
                    hot[on, t[on]] = 1.0
                    got["loss"] = -(torch.where(hot > 0, lp, 0.0)).sum(1)
                    if case["train"]:
                        g = s["g"].double()
                        per = g[i:i + step] if g.dim() else g.expand(xi.shape[0])
                        if case["reduction"] == "mean":
                            per = per / max(1, int(live.sum()))
                        dz = (lp.exp_() - hot) * (per * on)[:, None]
            if dz is not None:
                got["dx"] = torch.mm(dz, w)
                dw += torch.mm(dz.t(), xi)
                db += dz.sum(0)
            for name, v in got.items():
                parts.setdefault(name, []).append(v)
        out = {name: torch.cat(v) for name, v in parts.items()}
        if case["op"] == "cross_entropy" and case["reduction"] != "none":
            out["loss"] = out["loss"].sum() / (max(1, int(live.sum())) if case["reduction"] == "mean" else 1)
        if case.get("train"):
            out["dw"] = dw
            if b is not None:
                out["db"] = db
        return out


def _exact_act(z, act):
    """act(z) and its slope in 64 bits."""
    if act in ("relu", "leaky_relu"):
        slope = torch.full_like(z, 0.0 if act == "relu" else 0.01).masked_fill_(z > 0, 1.0)
        return z * slope, slope
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    return z, torch.ones_like(z)

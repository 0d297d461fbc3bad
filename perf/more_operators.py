"""The operators that train and run a gated residual block at the float end of a network, as cases that can be timed and
compared: the gated feed-forward product (two projections, an activation, their product), the norms after and before a
block with its gate, scale and residual stream, and the softmax cross entropy of a linear classifier that keeps no
logits, each with its gradients.  Sizes are those of this library's networks (1024 and 4096 hidden neurons, 512 features, 1000
classes, batches of 256 and 8192) and around them, and vocabularies of general size."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
# A drawn case does no more than the largest listed one of its kind: multiply-adds of the products (one product of each
# kind, forward), values of a norm, values of logits.
MAX_GATED = 8192 * 4096 * 16384
MAX_LOSS = 8192 * 1024 * 131072
MAX_NORM = 16384 * 4096


def listed():
    return [
        # one row through a wide gated block: a request of its own, bound by the weights' bytes
        dict(name="gated_row1", op="gated", rows=1, inp=4096, out=8192, dtype="bf16", act="silu", bias=False, preact=False,
             extra=0),
        # odd sizes throughout, input rows out of a wider array: the tail of a data set
        dict(name="gated_ragged", op="gated", rows=77, inp=1023, out=1537, dtype="f16", act="gelu", bias=True, preact=True,
             extra=3),
        # a wide block over the largest batch, as training runs it (the values before the activation are kept)
        dict(name="gated_large", op="gated", rows=8192, inp=4096, out=8192, dtype="bf16", act="silu", bias=False,
             preact=True, extra=0),
        # gradients of the hidden layer's width over the largest batch
        dict(name="gated_grad", op="gated_grad", rows=8192, inp=1024, out=4096, dtype="bf16", act="silu", bias=True,
             extra=0),
        # one row of a wide stream: latency
        dict(name="norms_row1", op="norms", rows=1, features=4096, dtype="bf16", after="rms", before="rms", gate=False,
             extra=0),
        # a long batch of wide rows: memory
        dict(name="norms_large", op="norms", rows=16384, features=4096, dtype="bf16", after="rms", before="rms", gate=True,
             extra=0),
        # gradients of a long batch of wide rows, all parameters' among them
        dict(name="norms_grad", op="norms_grad", rows=8192, features=4096, dtype="bf16", after="rms", before="rms", gate=True,
             stream=True, extra=0),
        # layer norms of odd rows in fp32, rows out of a wider array
        dict(name="norms_grad_ragged", op="norms_grad", rows=1000, features=1001, dtype="f32", after="layer", before="layer",
             gate=True, stream=True, extra=3),
        # how likely one token of a large vocabulary was: bound by the weights' bytes
        dict(name="loss_row1", op="loss", rows=1, inp=4096, classes=131072, dtype="bf16", bias=False, extra=0),
        # the classifier of the residual networks at their batch, a step of its training
        dict(name="loss_classes", op="loss_step", rows=256, inp=512, classes=1000, dtype="f32", bias=True, extra=0),
        # an odd vocabulary and odd rows
        dict(name="loss_ragged", op="loss_step", rows=333, inp=1000, classes=32003, dtype="f16", bias=True, extra=3),
        # a step over many tokens of a large vocabulary: the logits would take more than the weights
        dict(name="loss_large", op="loss_step", rows=8192, inp=1024, classes=131072, dtype="bf16", bias=False, extra=0),
    ]


def _log_int(rng, lo, hi):
    """An integer of lo..hi, evenly spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _size(rng, lo, hi):
    """A size as layers have them: two times in three a multiple of 8, otherwise whatever comes."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 1 / 3 else max(8, (n + 7) // 8 * 8)


def draw(rng):
    op = rng.choice(["gated", "gated", "gated_grad", "norms", "norms_grad", "loss", "loss_step", "loss_step"])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), extra=rng.choice([0, 0, 0, 8, 3]))
    while True:
        if op in ("gated", "gated_grad"):
            c.update(rows=_log_int(rng, 1, 8192), inp=_size(rng, 16, 8192), out=_size(rng, 10, 8192),
                     act=rng.choice(["silu", "silu", "gelu", "relu", "none"]), bias=rng.random() < 0.5)
            if op == "gated":
                c.update(preact=rng.random() < 0.5)
            # (products in fp32 take eight times as long)
            if c["rows"] * c["inp"] * c["out"] * 2 <= MAX_GATED // (2 if op == "gated_grad" else 1) // (8 if c["dtype"] == "f32" else 1):
                return c
        elif op in ("norms", "norms_grad"):
            c.update(rows=_log_int(rng, 1, 16384), features=_size(rng, 8, 8192), before=rng.choice(["rms", "rms", "layer", "none"]),
                     after=rng.choice(["rms", "layer", "none"]), gate=rng.random() < 0.5)
            if op == "norms_grad":
                c.update(stream=rng.random() < 0.75 or c["before"] == "none")
            if c["before"] == c["after"] == "none":
                c["before"] = "rms"
            if c["rows"] * c["features"] <= MAX_NORM // (2 if op == "norms_grad" else 1):
                return c
        else:
            c.update(rows=_log_int(rng, 1, 8192), inp=_size(rng, 16, 4096), classes=_log_int(rng, 10, 131072),
                     bias=rng.random() < 0.5)
            if c["rows"] * c["inp"] * c["classes"] <= MAX_LOSS // (8 if c["dtype"] == "f32" else 1):
                return c


def _normal(gen, shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(std).add_(mean)


def _rows(x, dtype, extra):
    """The values in the case's type, in rows that lie `extra` elements further apart than they are long."""
    wide = torch.zeros((x.shape[0], x.shape[1] + extra), dtype=DTYPES[dtype], device="cuda")
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


def _statistics(x, kind):
    """mean and 1 / sqrt(variance + eps) of the rows of a matrix in 64 bits (about 0 for "rms"), fp32."""
    if kind == "none":
        return None, None
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    rstd = ((x - mean).square().mean(1) + EPS).rsqrt()
    return (mean[:, 0].float() if kind == "layer" else None), rstd.float()


def _inputs(case, seed):
    """What the operator reads, from the seed alone: activations about N(0, 1), weights N(0, 1/inputs), a residual stream
    wider than a block's output, a trained classifier's rows (most given classes stand out), -1 for rows without a class."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, dt, extra = case["op"], case["dtype"], case["extra"]
    if op in ("gated", "gated_grad"):
        m, k, n = case["rows"], case["inp"], case["out"]
        s = dict(x=_rows(_normal(gen, (m, k)), dt, extra), w=_normal(gen, (2 * n, k), k ** -0.5).to(DTYPES[dt]),
                 bias=_normal(gen, (2 * n,), 0.5) if case["bias"] else None)
        if op == "gated_grad":
            s["z"] = _normal(gen, (m, 2 * n)).to(DTYPES[dt])
            s["dy"] = _rows(_normal(gen, (m, n)), dt, extra)
        return s
    if op in ("norms", "norms_grad"):
        m, n = case["rows"], case["features"]
        s = dict(stream=_rows(_normal(gen, (m, n), 2.0, 0.2), dt, extra), block=_rows(_normal(gen, (m, n), 1.5, 0.3), dt, extra),
                 gate=_normal(gen, (n,), 0.2, 0.7) if case["gate"] else None, scale=0.5)
        for which in ("after", "before"):
            there, layer = case[which] != "none", case[which] == "layer"
            s[which + "_gamma"] = _normal(gen, (n,), 0.2, 1.0) if there else None
            s[which + "_beta"] = _normal(gen, (n,), 0.2) if layer else None
        if op == "norms_grad":  # (`stream` is the one that the forward call wrote)
            s["after_mean"], s["after_rstd"] = _statistics(s["block"].double(), case["after"])
            s["before_mean"], s["before_rstd"] = _statistics(s["stream"].double(), case["before"])
            s["d_output"] = _rows(_normal(gen, (m, n)), dt, extra) if case["before"] != "none" else None
            s["d_stream"] = _rows(_normal(gen, (m, n)), dt, extra) if case["stream"] else None
        return s
    m, k, v = case["rows"], case["inp"], case["classes"]
    w = _normal(gen, (v, k), 2.5 * k ** -0.5)
    target = torch.randint(0, v, (m,), generator=gen, device="cuda")
    boost = torch.where(torch.rand((m,), generator=gen, device="cuda") < 0.7, 9.0 / 6.25, 0.0)
    x = _normal(gen, (m, k)) + boost[:, None] * w[target]
    none = torch.rand((m,), generator=gen, device="cuda") < 0.03
    return dict(x=_rows(x, dt, extra), w=w.to(DTYPES[dt]), bias=_normal(gen, (v,), 0.5) if case["bias"] else None,
                target=torch.where(none, -1, target).int(), g=torch.rand((m,), generator=gen, device="cuda").add_(0.5))


class _Stream:
    """torch's current stream, as the layers take one."""

    @property
    def handle(self):
        return torch.cuda.current_stream().cuda_stream


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if not own:
        return s
    from tcbnn_amd import head
    from tcbnn_amd.device import DeviceView

    def view(t):
        return None if t is None else DeviceView.of(t)

    def out(*shape, dtype=DTYPES[case["dtype"]]):
        return torch.empty(shape, dtype=dtype, device="cuda")

    f32 = torch.float32
    op, dt, m = case["op"], case["dtype"], case["rows"]
    s["stream_handle"] = _Stream()
    if op in ("gated", "gated_grad"):
        k, n = case["inp"], case["out"]
        layer = head.GatedLayerParam("gated", m, k, n, dtype=dt, activation=case["act"])
        if op == "gated":
            y = out(m, n)
            z = out(m, 2 * n) if case["preact"] else None
            layer.initialize(view(s["w"]), view(s["bias"]), view(s["x"]), output_gpu=view(y), preact_gpu=view(z))
            s["outputs"] = [y] if z is None else [y, z]
        else:
            dx, dw = out(m, k), out(2 * n, k)
            db = out(2 * n, dtype=f32) if case["bias"] else None
            layer.initialize(view(s["w"]), view(s["bias"]), view(s["x"]), preact_gpu=view(s["z"]))
            layer.initialize_backward(view(s["dy"]), view(dx), view(dw), view(db))
            s["outputs"] = [dx, dw] if db is None else [dx, dw, db]
    elif op in ("norms", "norms_grad"):
        n = case["features"]
        layer = head.BlockNormLayerParam("norms", m, n, dtype=dt, after=case["after"], before=case["before"], scale=s["scale"],
                                         eps=EPS)
        parameters = {name: view(s[name]) for name in ("gate", "after_gamma", "after_beta", "before_gamma", "before_beta")}
        if op == "norms":
            stream = out(m, n)
            y = out(m, n) if case["before"] != "none" else None
            layer.initialize(view(s["stream"]), view(s["block"]), new_stream_gpu=view(stream), output_gpu=view(y), **parameters)
            s["outputs"] = [stream] if y is None else [stream, y]
        else:
            # (what the forward call read besides is not needed any more: its stream may be the new one)
            layer.initialize(view(s["stream"]), view(s["block"]), new_stream_gpu=view(s["stream"]),
                             **{name + "_gpu": view(s[name]) for name in ("after_mean", "after_rstd", "before_mean", "before_rstd")},
                             **parameters)
            grads = {name: out(n, dtype=f32) for name, p in parameters.items() if p is not None}
            d_stream, d_block = out(m, n), out(m, n)
            layer.initialize_backward(view(s["d_output"]), view(s["d_stream"]), grad_stream_gpu=view(d_stream),
                                      grad_block_gpu=view(d_block), **{"grad_%s_gpu" % name: view(g) for name, g in grads.items()})
            s["outputs"] = [d_stream, d_block] + list(grads.values())
    else:
        k, v = case["inp"], case["classes"]
        layer = head.LinearLossLayerParam("loss", m, k, v, dtype=dt)
        loss, lse = out(m, dtype=f32), out(m, dtype=f32)
        layer.initialize(view(s["w"]), view(s["bias"]), view(s["x"]), view(s["target"]), loss_gpu=view(loss), logsumexp_gpu=view(lse))
        s["outputs"] = [loss, lse]
        if op == "loss_step":
            dx, dw = out(m, k), out(v, k)
            db = out(v, dtype=f32) if case["bias"] else None
            layer.initialize_backward(view(s["g"]), view(dx), view(dw), view(db))
            s["outputs"] += [dx, dw] if db is None else [dx, dw, db]
    s["layer"] = layer
    return s


def run(state):
    if own:
        op = state["case"]["op"]
        if not op.endswith("_grad"):
            state["layer"].forward(state["stream_handle"])
        if op.endswith("_grad") or op == "loss_step":
            state["layer"].backward(state["stream_handle"])
        return state["outputs"]
    return _PLAIN[state["case"]["op"]](state["case"], state)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end
def _act(act, z):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(act, z):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_gated(case, s):
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"]
    n, dt = case["out"], DTYPES[case["dtype"]]
    y = (_act(case["act"], z[:, :n]) * z[:, n:]).to(dt)
    return [y, z.to(dt)] if case["preact"] else [y]


def _plain_gated_grad(case, s):
    n, dt = case["out"], DTYPES[case["dtype"]]
    g, u, dy = s["z"][:, :n].float(), s["z"][:, n:].float(), s["dy"].float()
    dz = torch.cat([dy * u * _slope(case["act"], g), dy * _act(case["act"], g)], 1)
    out = [(dz @ s["w"].float()).to(dt), (dz.t() @ s["x"].float()).to(dt)]
    return out + [dz.sum(0)] if case["bias"] else out


def _plain_norm(x, kind, gamma, beta):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(1)[:, None]
    y = x * (1 / torch.sqrt((x * x).mean(1) + EPS))[:, None] * gamma
    return y if beta is None else y + beta


def _plain_norms(case, s):
    u = _plain_norm(s["block"].float(), case["after"], s["after_gamma"], s["after_beta"]) * s["scale"]
    if s["gate"] is not None:
        u = u * s["gate"]
    stream = s["stream"].float() + u
    dt = DTYPES[case["dtype"]]
    if case["before"] == "none":
        return [stream.to(dt)]
    return [stream.to(dt), _plain_norm(stream, case["before"], s["before_gamma"], s["before_beta"]).to(dt)]


def _plain_hat(x, mean, rstd):
    return (x if mean is None else x - mean[:, None]) * rstd[:, None]


def _plain_norm_grad(dy, xh, gamma, rstd, kind):
    g = dy * gamma
    d = g - xh * (g * xh).mean(1)[:, None]
    if kind == "layer":
        d = d - g.mean(1)[:, None]
    return d * rstd[:, None]


def _plain_norms_grad(case, s):
    d = s["d_stream"].float() if s["d_stream"] is not None else 0.0
    grads = {}
    if case["before"] != "none":
        dy = s["d_output"].float()
        xh = _plain_hat(s["stream"].float(), s["before_mean"], s["before_rstd"])
        d = d + _plain_norm_grad(dy, xh, s["before_gamma"], s["before_rstd"], case["before"])
        grads["before_gamma"], grads["before_beta"] = (dy * xh).sum(0), dy.sum(0)
    du = d * s["scale"]
    u = s["block"].float()
    if case["after"] != "none":
        yh = _plain_hat(u, s["after_mean"], s["after_rstd"])
        u = yh * s["after_gamma"]
        if s["after_beta"] is not None:
            u = u + s["after_beta"]
    if s["gate"] is not None:
        grads["gate"] = (du * u).sum(0)
        du = du * s["gate"]
    if case["after"] != "none":
        grads["after_gamma"], grads["after_beta"] = (du * yh).sum(0), du.sum(0)
        du = _plain_norm_grad(du, yh, s["after_gamma"], s["after_rstd"], case["after"])
    dt = DTYPES[case["dtype"]]
    names = ("gate", "after_gamma", "after_beta", "before_gamma", "before_beta")
    return [d.to(dt), du.to(dt)] + [grads[name] for name in names if s[name] is not None]


def _plain_loss(case, s):
    x, w, t = s["x"].float(), s["w"].float(), s["target"].long()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"]
    m = z.amax(1)
    lse = m + torch.log(torch.exp(z - m[:, None]).sum(1))
    at = t.clamp_min(0)[:, None]
    loss = torch.where(t < 0, 0.0, lse - z.gather(1, at)[:, 0])
    if case["op"] == "loss":
        return [loss, lse]
    g = torch.where(t < 0, 0.0, s["g"])
    d = torch.exp(z - lse[:, None]) * g[:, None]
    del z
    d.scatter_add_(1, at, -g[:, None])
    dt = DTYPES[case["dtype"]]
    out = [loss, lse, (d @ w).to(dt), (d.t() @ x).to(dt)]
    return out + [d.sum(0)] if case["bias"] else out


_PLAIN = {"gated": _plain_gated, "gated_grad": _plain_gated_grad, "norms": _plain_norms, "norms_grad": _plain_norms_grad,
          "loss": _plain_loss, "loss_step": _plain_loss}


# ---- the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    return (_exact_gated if op.startswith("gated") else _exact_norms if op.startswith("norms") else _exact_loss)(case, s)


def _exact_gated(case, s):
    def act_and_slope(z):
        """Both by automatic differentiation of the activation's definition."""
        z = z.detach().requires_grad_(True)
        normal = torch.distributions.Normal(torch.zeros((), dtype=torch.float64, device="cuda"), 1.0, validate_args=False)
        a = {"none": lambda: z * 1.0, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "gelu": lambda: z * normal.cdf(z),
             "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
        return a.detach(), torch.autograd.grad(a.sum(), z)[0]

    n, w, x = case["out"], s["w"].double(), s["x"].double()
    if case["op"] == "gated":
        gate, up = torch.matmul(x, w[:n].transpose(0, 1)), torch.matmul(x, w[n:].transpose(0, 1))
        if s["bias"] is not None:
            gate += s["bias"][:n].double()
            up += s["bias"][n:].double()
        y = act_and_slope(gate)[0] * up
        return [y, torch.cat([gate, up], 1)] if case["preact"] else [y]
    z, dy = s["z"].double(), s["dy"].double()
    a, slope = act_and_slope(z[:, :n])
    d_gate, d_up = dy * z[:, n:] * slope, dy * a
    dx = torch.matmul(d_gate, w[:n]) + torch.matmul(d_up, w[n:])
    dw = torch.cat([torch.matmul(d.transpose(0, 1), x) for d in (d_gate, d_up)])
    return [dx, dw, torch.cat([d_gate.sum(0), d_up.sum(0)])] if case["bias"] else [dx, dw]


def _exact_norms(case, s):
    def norm(x, which):
        kind = case[which]
        if kind == "none":
            return x
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        if kind == "rms":
            var, mean = var + mean * mean, torch.zeros_like(mean)
        y = (x - mean) * (var + EPS).pow(-0.5) * s[which + "_gamma"].double()
        return y if s[which + "_beta"] is None else y + s[which + "_beta"].double()

    gate = s["scale"] * (1.0 if s["gate"] is None else s["gate"].double())
    if case["op"] == "norms":
        stream = s["stream"].double() + norm(s["block"].double(), "after") * gate
        return [stream] if case["before"] == "none" else [stream, norm(stream, "before")]

    def hat(x, which):
        mean = 0.0 if s[which + "_mean"] is None else s[which + "_mean"].double()[:, None]
        return (x.double() - mean) * s[which + "_rstd"].double()[:, None]

    def through(dy, xh, which):
        """The gradient of a norm's input, its row statistics as given."""
        g, n = dy * s[which + "_gamma"].double(), case["features"]
        mean = g.sum(1, keepdim=True) if case[which] == "layer" else 0.0
        return (n * g - mean - xh * (g * xh).sum(1, keepdim=True)) * s[which + "_rstd"].double()[:, None] / n

    grads = {}
    d = torch.zeros_like(s["block"], dtype=torch.float64)
    if s["d_stream"] is not None:
        d += s["d_stream"].double()
    if case["before"] != "none":
        dy, xh = s["d_output"].double(), hat(s["stream"], "before")
        d += through(dy, xh, "before")
        grads.update(before_gamma=torch.einsum("ij,ij->j", dy, xh), before_beta=dy.sum(0))
    if case["after"] == "none":
        u, d_block = s["block"].double(), d * gate
    else:
        yh = hat(s["block"], "after")
        u = yh * s["after_gamma"].double() + (0.0 if s["after_beta"] is None else s["after_beta"].double())
        d_block = through(d * gate, yh, "after")
        grads.update(after_gamma=torch.einsum("ij,ij->j", d * gate, yh), after_beta=(d * gate).sum(0))
    grads["gate"] = s["scale"] * torch.einsum("ij,ij->j", d, u)
    return [d, d_block] + [grads[name] for name in ("gate", "after_gamma", "after_beta", "before_gamma", "before_beta")
                           if s[name] is not None]


def _exact_loss(case, s):
    w = s["w"].double()
    rows = max(1, min(1024, (1 << 27) // case["classes"]))
    loss, lse, dx = [], [], []
    step = case["op"] == "loss_step"
    dw = torch.zeros_like(w) if step else None
    db = torch.zeros_like(w[:, 0]) if step else None
    for i in range(0, case["rows"], rows):
        x, t = s["x"][i:i + rows].double(), s["target"][i:i + rows].long()
        logits = torch.matmul(x, w.transpose(0, 1))
        if s["bias"] is not None:
            logits += s["bias"].double()
        given = t >= 0
        here, at = torch.arange(len(t), device="cuda"), t.clamp(min=0)
        lse.append(torch.logsumexp(logits, 1))
        loss.append(-torch.log_softmax(logits, 1)[here, at] * given)
        if step:
            p = torch.softmax(logits, 1)
            p[here, at] -= 1.0
            p *= (s["g"][i:i + rows].double() * given)[:, None]
            dx.append(torch.matmul(p, w))
            dw += torch.matmul(p.transpose(0, 1), x)
            db += p.sum(0)
    out = [torch.cat(loss), torch.cat(lse)]
    if step:
        out += [torch.cat(dx), dw] + ([db] if case["bias"] else [])
    return out


def work(case):
    """Inputs read once and outputs written once; two operations a multiply-add, a handful a value elsewhere."""
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    if op in ("gated", "gated_grad"):
        m, k, n = case["rows"], case["inp"], case["out"]
        if op == "gated":
            return {"bytes": size * (m * k + 2 * n * k + m * n * (3 if case["preact"] else 1)) + 8 * n * case["bias"],
                    "flops": 4 * m * n * k}
        return {"bytes": size * (2 * m * k + 4 * n * k + 3 * m * n) + 8 * n * case["bias"], "flops": 8 * m * n * k}
    if op in ("norms", "norms_grad"):
        m, n = case["rows"], case["features"]
        layers, norms = [sum(case[which] in kinds for which in ("after", "before")) for kinds in (("layer",), ("rms", "layer"))]
        parameters = 4 * n * (layers + norms + case["gate"])
        there = case["before"] != "none"
        if op == "norms":
            return {"bytes": size * m * n * (3 + there) + parameters, "flops": m * n * (3 + 5 * norms)}
        # (the stream itself is read for the norm before the next block only, the block's output for its norm or its gate)
        block = case["after"] != "none" or case["gate"]
        return {"bytes": size * m * n * (2 + 2 * there + block + case["stream"]) + 4 * m * (layers + norms) + 2 * parameters,
                "flops": m * n * (4 + 10 * norms)}
    # (the gradient takes three products, the logits' own among them; they are not kept, so a step makes those twice, which is
    # not counted here)
    m, k, v = case["rows"], case["inp"], case["classes"]
    steps = 2 if op == "loss_step" else 1
    return {"bytes": size * steps * (m * k + v * k) + 4 * steps * v * case["bias"] + m * (12 + 4 * (steps - 1)),
            "flops": 2 * m * v * k * (3 if op == "loss_step" else 1)}

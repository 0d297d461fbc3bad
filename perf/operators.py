"""The float operators of a head on a binary trunk, as cases that can be timed and compared: linear layers with bias,
activation and residual, layer norms, log probabilities of given classes (or tokens) with entropy and the best
alternatives, and the gradient of each.  Sizes are those of this library's networks (1024 and 4096 hidden neurons, 512
features, 1000 and 10 classes, batches of 256 and 8192) and around them, and vocabularies of general size."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
# A drawn case does no more than the largest listed one of its kind: multiply-adds of a product, values of a norm or of logits.
MAX_MULTIPLIES = 8192 * 4096 * 4096
MAX_NORM = 16384 * 4096
MAX_LOGITS = 2048 * 131072


def listed():
    return [
        # one row through a wide hidden layer: a request of its own, bound by the weights' bytes
        dict(name="linear_row1", op="linear", rows=1, inp=4096, out=4096, dtype="bf16", act="gelu", bias=True, residual=False,
             preact=False, extra=0),
        # the classifier of the residual networks at their batch, in the type its features come in
        dict(name="linear_classes_f32", op="linear", rows=256, inp=512, out=1000, dtype="f32", act="none", bias=True,
             residual=False, preact=False, extra=0),
        # odd sizes throughout, input rows out of a wider array: the tail of a data set through an odd layer
        dict(name="linear_ragged", op="linear", rows=77, inp=1023, out=1537, dtype="f16", act="silu", bias=True, residual=True,
             preact=False, extra=3),
        # a wide residual layer over the largest batch, as training runs it (the values before the activation are kept)
        dict(name="linear_large", op="linear", rows=8192, inp=4096, out=4096, dtype="bf16", act="gelu", bias=True,
             residual=True, preact=True, extra=0),
        # gradients of a hidden layer over the largest batch
        dict(name="linear_grad", op="linear_grad", rows=8192, inp=1024, out=4096, dtype="bf16", act="gelu", extra=0),
        # one row of a wide layer: latency
        dict(name="norm_row1", op="norm", rows=1, features=4096, dtype="bf16", extra=0),
        # a long batch of wide rows: memory
        dict(name="norm_large", op="norm", rows=16384, features=4096, dtype="bf16", extra=0),
        # gradients over the MLP's batch and width, with the reduction over rows
        dict(name="norm_grad", op="norm_grad", rows=8192, features=1024, dtype="bf16", extra=0),
        # the answers of an ImageNet classifier: five best classes of each image
        dict(name="logprobs_classes", op="logprobs", rows=256, classes=1000, top=5, dtype="f32", masked=0.0, extra=0),
        # one token of a large vocabulary with its alternatives, some of the vocabulary forbidden
        dict(name="logprobs_row1", op="logprobs", rows=1, classes=131072, top=20, dtype="bf16", masked=0.25, extra=0),
        # scoring of many tokens
        dict(name="logprobs_large", op="logprobs", rows=2048, classes=131072, top=8, dtype="bf16", masked=0.0, extra=0),
        # the loss' gradient over an odd vocabulary
        dict(name="logprobs_grad", op="logprobs_grad", rows=4095, classes=32003, dtype="bf16", entropy=True, extra=0),
    ]


def _log_int(rng, lo, hi):
    """An integer of lo..hi, evenly spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _size(rng, lo, hi):
    """A size as layers have them: two times in three a multiple of 8, otherwise whatever comes."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 1 / 3 else max(8, (n + 7) // 8 * 8)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "linear_grad", "linear_grad", "norm", "norm_grad", "logprobs", "logprobs",
                     "logprobs_grad"])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), extra=rng.choice([0, 0, 0, 8, 3]))
    while True:
        if op in ("linear", "linear_grad"):
            c.update(rows=_log_int(rng, 1, 8192), inp=_size(rng, 16, 8192), out=_size(rng, 10, 8192),
                     act=rng.choice(["none", "relu", "gelu", "silu"]))
            if op == "linear":
                c.update(bias=rng.random() < 0.75, residual=rng.random() < 0.5, preact=rng.random() < 0.25)
            if c["rows"] * c["inp"] * c["out"] * (2 if op == "linear_grad" else 1) <= MAX_MULTIPLIES:
                return c
        elif op in ("norm", "norm_grad"):
            c.update(rows=_log_int(rng, 1, 16384), features=_size(rng, 8, 8192))
            if c["rows"] * c["features"] <= MAX_NORM // (2 if op == "norm_grad" else 1):
                return c
        else:
            c.update(rows=_log_int(rng, 1, 8192), classes=_log_int(rng, 10, 131072))
            if op == "logprobs":
                c.update(top=rng.choice([0, 1, 5, 8, 20, 32]), masked=rng.choice([0.0, 0.0, 0.25, 0.5]))
                c["top"] = min(c["top"], c["classes"] // 4)
                if c["classes"] < 256:
                    c["masked"] = 0.0
            else:
                c.update(entropy=rng.random() < 0.5)
            if c["rows"] * c["classes"] <= MAX_LOGITS // (2 if op == "logprobs_grad" else 1) // (2 if c["dtype"] == "f32" else 1):
                return c


def _normal(gen, shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(std).add_(mean)


def _rows(x, dtype, extra):
    """The values in the case's type, in rows that lie `extra` elements further apart than they are long."""
    wide = torch.zeros((x.shape[0], x.shape[1] + extra), dtype=DTYPES[dtype], device="cuda")
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


def _inputs(case, seed):
    """What the operator reads, from the seed alone: activations about N(0, 1), weights N(0, 1/inputs), logits of a
    trained classifier (most given classes stand out), -1 for rows without a given class."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, dt, extra = case["op"], case["dtype"], case["extra"]
    if op in ("linear", "linear_grad"):
        m, k, n = case["rows"], case["inp"], case["out"]
        s = dict(x=_rows(_normal(gen, (m, k)), dt, extra), w=_normal(gen, (n, k), k ** -0.5).to(DTYPES[dt]))
        if op == "linear":
            s["bias"] = _normal(gen, (n,), 0.5) if case["bias"] else None
            s["res"] = _normal(gen, (m, n)).to(DTYPES[dt]) if case["residual"] else None
        else:
            s["z"] = _normal(gen, (m, n)).to(DTYPES[dt]) if case["act"] != "none" else None
            s["dy"] = _rows(_normal(gen, (m, n)), dt, extra)
        return s
    if op in ("norm", "norm_grad"):
        m, n = case["rows"], case["features"]
        s = dict(x=_rows(_normal(gen, (m, n), 2.0, 0.5), dt, extra), gamma=_normal(gen, (n,), 0.2, 1.0),
                 beta=_normal(gen, (n,), 0.2))
        if op == "norm_grad":
            s["dy"] = _rows(_normal(gen, (m, n)), dt, extra)
            x = s["x"].double()
            mean = x.mean(1)
            s["mean"] = mean.float()
            s["rstd"] = ((x - mean[:, None]).square_().mean(1) + EPS).rsqrt().float()
        return s
    m, v = case["rows"], case["classes"]
    x = _normal(gen, (m, v), 2.5)
    target = torch.randint(0, v, (m,), generator=gen, device="cuda")
    if case.get("masked"):
        x[:, torch.rand((v,), generator=gen, device="cuda") < case["masked"]] = -math.inf
        x[:, v - 1] = 0.0
        target = torch.where(torch.isinf(x.gather(1, target[:, None])[:, 0]), v - 1, target)
    boost = torch.rand((m,), generator=gen, device="cuda") < 0.7
    x.scatter_add_(1, target[:, None], boost[:, None] * 9.0)
    none = torch.rand((m,), generator=gen, device="cuda") < 0.03
    s = dict(x=_rows(x, dt, extra), target=torch.where(none, -1, target).int())
    del x
    if op == "logprobs_grad":
        s["lse"] = torch.empty((m,), device="cuda")
        s["entropy"] = torch.empty((m,), device="cuda")
        for i in range(0, m, 512):
            y = s["x"][i:i + 512].double()
            lse = torch.logsumexp(y, 1)
            s["lse"][i:i + 512] = lse
            s["entropy"][i:i + 512] = lse - ((y - lse[:, None]).exp() * y).sum(1)
        s["g_logprob"] = _normal(gen, (m,))
        s["g_entropy"] = _normal(gen, (m,), 0.1) if case["entropy"] else None
    return s


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

    op, dt = case["op"], case["dtype"]
    s["stream"] = _Stream()
    if op in ("linear", "linear_grad"):
        layer = head.LinearLayerParam("linear", case["rows"], case["inp"], case["out"], dtype=dt, activation=case["act"])
        if op == "linear":
            y = torch.empty((case["rows"], case["out"]), dtype=DTYPES[dt], device="cuda")
            z = torch.empty_like(y) if case["preact"] else None
            layer.initialize(view(s["w"]), view(s["bias"]), view(s["x"]), residual_gpu=view(s["res"]), output_gpu=view(y),
                             preact_gpu=view(z))
            s["outputs"] = [y] if z is None else [y, z]
        else:
            dx = torch.empty((case["rows"], case["inp"]), dtype=DTYPES[dt], device="cuda")
            dw = torch.empty((case["out"], case["inp"]), dtype=DTYPES[dt], device="cuda")
            db = torch.empty((case["out"],), device="cuda")
            layer.initialize(view(s["w"]), None, view(s["x"]), preact_gpu=view(s["z"]))
            layer.initialize_backward(view(s["dy"]), view(dx), view(dw), view(db))
            s["outputs"] = [dx, dw, db]
    elif op in ("norm", "norm_grad"):
        layer = head.LayerNormLayerParam("norm", case["rows"], case["features"], dtype=dt, eps=EPS)
        if op == "norm":
            y = torch.empty((case["rows"], case["features"]), dtype=DTYPES[dt], device="cuda")
            mean, rstd = (torch.empty((case["rows"],), device="cuda") for _ in range(2))
            layer.initialize(view(s["gamma"]), view(s["beta"]), view(s["x"]), output_gpu=view(y), mean_gpu=view(mean),
                             rstd_gpu=view(rstd))
            s["outputs"] = [y, mean, rstd]
        else:
            dx = torch.empty((case["rows"], case["features"]), dtype=DTYPES[dt], device="cuda")
            dgamma, dbeta = (torch.empty((case["features"],), device="cuda") for _ in range(2))
            layer.initialize(view(s["gamma"]), view(s["beta"]), view(s["x"]), mean_gpu=view(s["mean"]),
                             rstd_gpu=view(s["rstd"]))
            layer.initialize_backward(view(s["dy"]), view(dx), view(dgamma), view(dbeta))
            s["outputs"] = [dx, dgamma, dbeta]
    else:
        rows, v = case["rows"], case["classes"]
        layer = head.LogProbsLayerParam("logprobs", rows, v, top=case.get("top", 0), dtype=dt)
        if op == "logprobs":
            logprob, entropy, lse = (torch.empty((rows,), device="cuda") for _ in range(3))
            rank = torch.empty((rows,), dtype=torch.int32, device="cuda")
            index = torch.empty((rows, case["top"]), dtype=torch.int32, device="cuda")
            value = torch.empty((rows, case["top"]), device="cuda")
            layer.initialize(view(s["x"]), view(s["target"]), logprob_gpu=view(logprob), entropy_gpu=view(entropy),
                             logsumexp_gpu=view(lse), rank_gpu=view(rank), top_index_gpu=view(index) if case["top"] else None,
                             top_logprob_gpu=view(value) if case["top"] else None)
            s["outputs"] = [logprob, entropy, lse, rank, index, value]
        else:
            dx = torch.empty((rows, v), dtype=DTYPES[dt], device="cuda")
            layer.initialize(view(s["x"]), view(s["target"]), logsumexp_gpu=view(s["lse"]), entropy_gpu=view(s["entropy"]))
            layer.initialize_backward(view(s["g_logprob"]), view(s["g_entropy"]), view(dx))
            s["outputs"] = [dx]
    s["layer"] = layer
    return s


def run(state):
    if own:
        if state["case"]["op"].endswith("_grad"):
            state["layer"].backward(state["stream"])
        else:
            state["layer"].forward(state["stream"])
        return state["outputs"]
    return _PLAIN[state["case"]["op"]](state["case"], state)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end
def _plain_linear(case, s):
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"]
    y = _act(case["act"], z)
    if s["res"] is not None:
        y = y + s["res"].float()
    dt = DTYPES[case["dtype"]]
    return [y.to(dt), z.to(dt)] if case["preact"] else [y.to(dt)]


def _act(act, z):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_linear_grad(case, s):
    g = s["dy"].float()
    if s["z"] is not None:
        z = s["z"].float()
        if case["act"] == "relu":
            g = g * (z > 0)
        elif case["act"] == "gelu":
            g = g * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
        else:
            p = 1 / (1 + torch.exp(-z))
            g = g * (p * (1 + z * (1 - p)))
    dt = DTYPES[case["dtype"]]
    return [(g @ s["w"].float()).to(dt), (g.t() @ s["x"].float()).to(dt), g.sum(0)]


def _plain_norm(case, s):
    x = s["x"].float()
    mean = x.mean(1)
    x = x - mean[:, None]
    rstd = 1 / torch.sqrt((x * x).mean(1) + EPS)
    return [(x * rstd[:, None] * s["gamma"] + s["beta"]).to(DTYPES[case["dtype"]]), mean, rstd]


def _plain_norm_grad(case, s):
    xh = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    dy = s["dy"].float()
    g = dy * s["gamma"]
    dx = (g - g.mean(1)[:, None] - xh * (g * xh).mean(1)[:, None]) * s["rstd"][:, None]
    return [dx.to(DTYPES[case["dtype"]]), (dy * xh).sum(0), dy.sum(0)]


def _plain_logprobs(case, s):
    x, t = s["x"].float(), s["target"].long()
    v, top = case["classes"], case["top"]
    m = x.amax(1)
    e = torch.exp(x - m[:, None])
    total = e.sum(1)
    lse = m + torch.log(total)
    # (masked classes have no share: 0 * -inf counts as 0)
    entropy = torch.log(total) - torch.where(e > 0, e * (x - m[:, None]), 0.0).sum(1) / total
    at = t.clamp_min(0)[:, None]
    xt = x.gather(1, at)
    logprob = torch.where(t < 0, 0.0, xt[:, 0] - lse)
    j = torch.arange(v, device=x.device)
    rank = ((x > xt) | ((x == xt) & (j < at))).sum(1)
    rank = torch.where(t < 0, -1, rank).int()
    if not top:
        return [logprob, entropy, lse, rank, t.new_empty((len(t), 0)).int(), x.new_empty((len(t), 0))]
    # largest value first, lowest index among equals: one 64-bit key for both (bits of an ordered float, then ~index)
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits)
    index = (bits * (1 << 32) + ((1 << 32) - 1 - j)).topk(top, 1).values
    index = ((1 << 32) - 1) - (index & ((1 << 32) - 1))
    return [logprob, entropy, lse, rank, index.int(), x.gather(1, index) - lse[:, None]]


def _plain_logprobs_grad(case, s):
    logp = s["x"].float() - s["lse"][:, None]
    p = torch.exp(logp)
    t = s["target"].long()
    g = torch.where(t < 0, 0.0, s["g_logprob"])
    dx = -p * g[:, None]
    dx.scatter_add_(1, t.clamp_min(0)[:, None], g[:, None])
    if s["g_entropy"] is not None:
        dx = dx - s["g_entropy"][:, None] * torch.where(p > 0, p * (logp + s["entropy"][:, None]), 0.0)
    return [dx.to(DTYPES[case["dtype"]])]


_PLAIN = {"linear": _plain_linear, "linear_grad": _plain_linear_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad,
          "logprobs": _plain_logprobs, "logprobs_grad": _plain_logprobs_grad}


# ---- the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op.startswith("linear"):
        x, w = s["x"].double(), s["w"].double()
        normal = torch.distributions.Normal(torch.zeros((), dtype=torch.float64, device="cuda"), 1.0, validate_args=False)
        if op == "linear":
            z = torch.matmul(x, w.transpose(0, 1))
            if s["bias"] is not None:
                z += s["bias"].double()
            y = {"none": lambda: z, "relu": lambda: torch.maximum(z, torch.zeros_like(z)), "gelu": lambda: z * normal.cdf(z),
                 "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
            if s["res"] is not None:
                y = y + s["res"].double()
            return [y, z] if case["preact"] else [y]
        dz = s["dy"].double()
        if s["z"] is not None:
            z = s["z"].double()
            sig = torch.sigmoid(z)
            dz = dz * {"relu": lambda: (z > 0).double(), "gelu": lambda: normal.cdf(z) + z * normal.log_prob(z).exp(),
                       "silu": lambda: sig + z * sig * (1 - sig)}[case["act"]]()
        return [torch.matmul(dz, w), torch.matmul(dz.transpose(0, 1), x), dz.sum(0)]
    if op == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, unbiased=False)
        rstd = (var + EPS).pow(-0.5)
        return [torch.addcmul(s["beta"].double(), (x - mean[:, None]) * rstd[:, None], s["gamma"].double()), mean, rstd]
    if op == "norm_grad":
        rstd = s["rstd"].double()[:, None]
        dy, xh = s["dy"].double(), (s["x"].double() - s["mean"].double()[:, None]) * rstd
        g, n = dy * s["gamma"].double(), case["features"]
        dx = (n * g - g.sum(1, keepdim=True) - xh * (g * xh).sum(1, keepdim=True)) * rstd / n
        return [dx, torch.einsum("ij,ij->j", dy, xh), dy.sum(0)]
    t = s["target"].long()
    none, at = t < 0, t.clamp(min=0)
    parts = []
    for i in range(0, case["rows"], 256):
        x, ni, ti = s["x"][i:i + 256].double(), none[i:i + 256], at[i:i + 256]
        here = torch.arange(len(ti), device="cuda")
        if op == "logprobs":
            logp = torch.log_softmax(x, 1)
            lse = torch.logsumexp(x, 1)
            entropy = -torch.special.xlogy(logp.exp(), logp.exp()).sum(1)
            order = torch.sort(x, dim=1, descending=True, stable=True).indices
            rank = (order == ti[:, None]).int().argmax(1).int()
            best = order[:, :case["top"]]
            parts.append([logp[here, ti].masked_fill(ni, 0.0), entropy, lse, rank.masked_fill(ni, -1), best.int(),
                          logp[here[:, None], best]])
        else:
            logp = x - s["lse"][i:i + 256].double()[:, None]
            p = logp.exp()
            d = -p
            d[here, ti] += 1.0
            d *= s["g_logprob"][i:i + 256].double().masked_fill(ni, 0.0)[:, None]
            if s["g_entropy"] is not None:
                d -= s["g_entropy"][i:i + 256].double()[:, None] * p * (logp + s["entropy"][i:i + 256].double()[:, None])
            parts.append([d])
    return [torch.cat(p) for p in zip(*parts)]


def work(case):
    """Inputs read once and outputs written once; two operations a multiply-add, a handful a value elsewhere."""
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    if op in ("linear", "linear_grad"):
        m, k, n = case["rows"], case["inp"], case["out"]
        if op == "linear":
            return {"bytes": size * (m * k + n * k + m * n * (1 + case["residual"] + case["preact"])) + 4 * n * case["bias"],
                    "flops": 2 * m * n * k}
        return {"bytes": size * (2 * m * k + 2 * n * k + m * n * (1 if case["act"] == "none" else 2)) + 4 * n,
                "flops": 4 * m * n * k}
    if op == "norm":
        m, n = case["rows"], case["features"]
        return {"bytes": size * 2 * m * n + 8 * (m + n), "flops": 8 * m * n}
    if op == "norm_grad":
        m, n = case["rows"], case["features"]
        return {"bytes": size * 3 * m * n + 8 * m + 12 * n, "flops": 14 * m * n}
    m, v = case["rows"], case["classes"]
    if op == "logprobs":
        return {"bytes": size * m * v + m * (20 + 8 * case["top"]), "flops": 6 * m * v}
    return {"bytes": size * 2 * m * v + m * (16 + 4 * case["entropy"]), "flops": 5 * m * v}

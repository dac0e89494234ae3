"""The operators of a training step that decide what is kept between its two passes, as measurable cases.

Four kinds of case, each through the package's public entry points:

* ``ce``: softmax cross entropy of a linear classifier, straight from features, weight and labels (the logits are
  never returned), for evaluation or for training (the gradients of features, weight and bias);
* ``gelu``: exact GELU of ``x + bias`` whose backward pass has only an 8-bit checkpoint of its argument;
* ``ln``: LayerNorm over the last axis whose backward pass has only an 8-bit checkpoint of its input and the
  statistics of its rows;
* ``keep``: an activation put into 8 bits and brought back.

An 8-bit checkpoint: each row is cut into groups of 128 columns (the last one may be shorter).  A group with least
value ``lo`` and greatest value ``hi`` has the step ``s = (hi - lo) * (1/255)``, and a value ``v`` the code
``round((v - lo) * (1/s))`` (ties to even), all in fp32; the code ``q`` stands for ``lo + q*s``.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
GROUP = 128
EPS = 1e-6


def _ce(name=None, N=128, D=768, V=1000, dtype="bf16", bias=True, smoothing=0.0, ignored=0.0, ignore_index=-100, reduction="mean", train=True):
    c = dict(kind="ce", N=N, D=D, V=V, dtype=dtype, bias=bias, smoothing=smoothing, ignored=ignored, ignore_index=ignore_index,
             reduction=reduction, train=train)
    return c if name is None else dict(c, name=name)


def _rows(kind, name=None, rows=196, C=768, dtype="bf16", bias=True):
    c = dict(kind=kind, rows=rows, C=C, dtype=dtype, bias=bias)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one image's loss in an evaluation loop, head of the tiny classifier: nothing but latency
        _ce("ce-eval-1x768x1000-fp32", N=1, dtype="fp32", train=False),
        # the head of the tiny classifier in training, labels smoothed as its recipe has them
        _ce("ce-train-128x768x1000-bf16", N=128, smoothing=0.1),
        # head of the base classifier on a label set of tens of thousands (the largest product)
        _ce("ce-train-4096x1024x21841-bf16", N=4096, D=1024, V=21841),
        # every pixel of a dense-prediction batch's first stage, 150 classes, unlabelled pixels among them
        _ce("ce-train-133200x96x150-bf16", N=2 * 200 * 333, D=96, V=150, ignored=0.1, ignore_index=255),
        # odd sizes in fp32, no bias, a loss for each row that the caller weights itself
        _ce("ce-train-2500x384x10007-fp32-rows", N=2500, D=384, V=10007, dtype="fp32", bias=False, reduction="none"),
        # hidden tensor of one image in the third stage: the smallest call
        _rows("gelu", "gelu-196x1536-fp32", rows=196, C=1536, dtype="fp32", bias=False),
        # hidden tensor of the tiny classifier's second stage at the benchmark's batch
        _rows("gelu", "gelu-100352x768-bf16-bias", rows=128 * 28 * 28, C=768),
        # one image in the last stage: the smallest call
        _rows("ln", "ln-49x768-bf16", rows=49, C=768),
        # first stage of the tiny classifier at the benchmark's batch: short rows, the most of them
        _rows("ln", "ln-401408x96-bf16", rows=128 * 56 * 56, C=96),
        # last stage of the base classifier, fp32, a ragged batch: long rows
        _rows("ln", "ln-3087x1024-fp32", rows=63 * 49, C=1024, dtype="fp32"),
        # hidden tensor of the base 1D++ classifier's third stage
        _rows("keep", "keep-12544x2048-bf16", rows=64 * 14 * 14, C=2048),
        # odd everything: no row but the first starts on a vector, the last group has 105 columns
        _rows("keep", "keep-1001x1001-fp32", rows=1001, C=1001, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "gelu", "ln", "keep"])
    dtype = rng.choice(["bf16", "fp32"])
    if kind == "ce":
        D, V = _log(rng, 8, 1536), _log(rng, 2, 32768)
        most = 4096 * 1024 * 21841 // (4 if dtype == "fp32" else 1)      # products of a pass
        N = _log(rng, 1, max(1, min(133200, most // (D * V))))
        if rng.random() < 0.5:
            D = -(-D // 8) * 8
        return _ce(N=N, D=D, V=V, dtype=dtype, bias=rng.random() < 0.7, smoothing=rng.choice([0.0, 0.0, 0.1, 0.3]),
                   ignored=rng.choice([0.0, 0.0, 0.2]), ignore_index=rng.choice([-100, 255]), reduction=rng.choice(["mean", "sum", "none"]),
                   train=rng.random() < 0.75)
    C = _log(rng, 8 if kind == "ln" else 1, 4096)      # the gradient of shorter normalised rows is all cancellation
    if rng.random() < 0.5:
        C = -(-C // 8) * 8
    most = {"gelu": 100352 * 768, "ln": 401408 * 96, "keep": 12544 * 2048}[kind] // (2 if dtype == "fp32" else 1)
    return _rows(kind, rows=_log(rng, 1, max(1, most // C)), C=C, dtype=dtype, bias=kind != "gelu" or rng.random() < 0.7)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["kind"] == "ce":
        N, D, V = case["N"], case["D"], case["V"]
        w = normal(V, D) * (2.0 / math.sqrt(D))                       # logits of a few units, as a classifier in training has them
        t = torch.randint(0, V, (N,), generator=g, device=dev)
        lean = torch.rand(N, 1, generator=g, device=dev)              # how far a row leans towards its label
        x = normal(N, D) + 3.0 * lean * w[t]
        dropped = torch.rand(N, generator=g, device=dev) < case["ignored"]
        if case["ignored"] and case["ignore_index"] < V:
            t[t == case["ignore_index"]] = 0
        t[dropped] = case["ignore_index"]
        up = normal(N).abs() if case["reduction"] == "none" else normal(()).abs() + 0.5
        s = dict(case, x=x.to(dt), w=w.to(dt), b=(0.5 * normal(V)).to(dt) if case["bias"] else None, t=t, up=up)
        if case["train"]:
            for k in ("x", "w", "b"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
        return s
    rows, C = case["rows"], case["C"]
    spread = 0.3 + torch.rand(C, generator=g, device=dev) * 1.5          # channels differ in scale and in their mean
    x = normal(rows, C).mul_(spread).add_(normal(C).mul_(0.5))
    s = dict(case, x=x.to(dt))
    if case["kind"] == "keep":
        return s
    s["x"].requires_grad_(True)
    s["dy"] = normal(rows, C).to(dt)
    if case["kind"] == "ln":
        s["w"] = (1.0 + 0.2 * normal(C)).to(dt).requires_grad_(True)
    s["b"] = (0.2 * normal(C)).to(dt).requires_grad_(True) if case["bias"] else None
    return s


def run(s):
    return _own(s) if own else _plain(s)


# ---- the framework's calls --------------------------------------------------------------------------

def _own(s):
    from oriented1d_b200 import ops
    if s["kind"] == "ce":
        loss = ops.linear_cross_entropy(s["x"], s["w"], s["t"], s["b"], ignore_index=s["ignore_index"], label_smoothing=s["smoothing"],
                                        reduction=s["reduction"])
        if not s["train"]:
            return {"loss": loss}
        leaves = [s[k] for k in ("x", "w", "b") if s[k] is not None]
        grads = torch.autograd.grad(loss, leaves, s["up"])
        return dict(zip(("dx", "dw", "db"), grads), loss=loss.detach())
    if s["kind"] == "gelu":
        y = ops.gelu_keep8(s["x"], s["b"])
        grads = torch.autograd.grad(y, [s["x"]] + ([s["b"]] if s["b"] is not None else []), s["dy"])
        return dict(zip(("dx", "db"), grads), y=y.detach())
    if s["kind"] == "ln":
        y = ops.layer_norm_keep8(s["x"], s["w"], s["b"], EPS)
        grads = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return dict(zip(("dx", "dw", "db"), grads), y=y.detach())
    codes, ranges = ops.keep8(s["x"])
    return {"x": ops.restore8(codes, ranges, s["x"].dtype)}


# ---- the plain forms --------------------------------------------------------------------------------

def _plain(s):
    with torch.no_grad():
        dt = s["x"].dtype
        x = s["x"].float()
        if s["kind"] == "ce":
            return _plain_ce(s, x, dt)
        b = s["b"].float() if s.get("b") is not None else None
        if s["kind"] == "gelu":
            h = x if b is None else x + b
            out = {"y": (0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))).to(dt)}
            h = _there_and_back(h)
            slope = 0.5 * (1.0 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) * (1.0 / math.sqrt(2.0 * math.pi))
            dx = s["dy"].float() * slope
            out["dx"] = dx.to(dt)
            if b is not None:
                out["db"] = dx.sum(0, dtype=torch.float64).to(dt)
            return out
        if s["kind"] == "ln":
            w, dy = s["w"].float(), s["dy"].float()
            mean = x.mean(1, keepdim=True)
            rstd = torch.rsqrt((x - mean).square().mean(1, keepdim=True) + EPS)
            out = {"y": ((x - mean) * rstd * w + b).to(dt)}
            xhat = (_there_and_back(x) - mean) * rstd
            g = dy * w
            out["dx"] = (rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))).to(dt)
            out["dw"] = (dy * xhat).sum(0, dtype=torch.float64).to(dt)
            out["db"] = dy.sum(0, dtype=torch.float64).to(dt)
            return out
        return {"x": _there_and_back(x).to(dt)}


def _there_and_back(x):
    """The fp32 values that the 8-bit checkpoint of the fp32 matrix x stands for."""
    rows, C = x.shape
    groups = -(-C // GROUP)
    if groups * GROUP != C:                                            # a short last group: its last column once more
        x = x[:, torch.arange(groups * GROUP, device=x.device).clamp(max=C - 1)]
    x = x.view(rows, groups, GROUP)
    lo, hi = x.amin(2, keepdim=True), x.amax(2, keepdim=True)
    step = (hi - lo) * torch.tensor(1.0 / 255.0, dtype=torch.float32, device=x.device)
    code = torch.where(step > 0, ((x - lo) * (1.0 / step)).round(), torch.zeros_like(x))
    return (lo.double() + code.double() * step.double()).float().reshape(rows, groups * GROUP)[:, :C]


def _plain_ce(s, x, dt):
    w, t, eps, V = s["w"].float(), s["t"], s["smoothing"], s["V"]
    logits = x @ w.t()
    if s["b"] is not None:
        logits += s["b"].float()
    kept = t != s["ignore_index"]
    safe = torch.where(kept, t, torch.zeros_like(t))
    top = logits.amax(1, keepdim=True)
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    loss = lse[:, 0] - (1.0 - eps) * logits.gather(1, safe[:, None])[:, 0]
    if eps:
        loss = loss - (eps / V) * logits.sum(1)
    loss = torch.where(kept, loss, torch.zeros_like(loss))
    count = kept.sum()
    if s["reduction"] == "mean":
        total = (loss.sum(dtype=torch.float64) / count).float()
    else:
        total = loss.sum(dtype=torch.float64).float() if s["reduction"] == "sum" else loss
    if not s["train"]:
        return {"loss": total}
    scale = s["up"] / count if s["reduction"] == "mean" else s["up"]
    scale = torch.where(kept, scale.expand(loss.shape), torch.zeros_like(loss))[:, None]
    g = (logits - lse).exp()
    if eps:
        g -= eps / V
    g.scatter_add_(1, safe[:, None], torch.full_like(loss, eps - 1.0)[:, None])
    g *= scale
    out = {"loss": total, "dx": (g @ w).to(dt), "dw": (g.t() @ x).to(dt)}
    if s["b"] is not None:
        out["db"] = g.sum(0, dtype=torch.float64).to(dt)
    return out


# ---- work and exact results -------------------------------------------------------------------------

def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "ce":
        N, D, V = case["N"], case["D"], case["V"]
        params = V * D * e + (V * e if case["bias"] else 0)
        losses = 4 * N if case["reduction"] == "none" else 4
        if not case["train"]:
            return {"bytes": N * D * e + params + 8 * N + losses, "flops": 2 * N * D * V}
        return {"bytes": 2 * (N * D * e + params) + 8 * N + 2 * losses, "flops": 6 * N * D * V}
    rows, C = case["rows"], case["C"]
    n = rows * C
    kept = n + 8 * rows * -(-C // GROUP)                               # codes, and two numbers a group
    if case["kind"] == "keep":
        return {"bytes": 2 * n * e + 2 * kept, "flops": 6 * n}
    if case["kind"] == "gelu":
        return {"bytes": 4 * n * e + 2 * kept + (2 * C * e if case["bias"] else 0), "flops": 40 * n}
    return {"bytes": 4 * n * e + 2 * kept + 16 * rows + 4 * C * e, "flops": 30 * n}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "ce":
            return _exact_ce(s)
        x = s["x"].double()
        b = s["b"].double() if s.get("b") is not None else None
        if case["kind"] == "keep":
            return {"x": _kept(s["x"].float())}
        dy = s["dy"].double()
        if case["kind"] == "gelu":
            h = x + b if b is not None else x
            kept = _kept((s["x"].float() + s["b"].float()) if b is not None else s["x"].float())
            phi = lambda v: torch.special.ndtr(v)  # noqa: E731
            dx = dy * (phi(kept) + kept * torch.exp(-kept.pow(2) / 2) / math.sqrt(2 * math.pi))
            out = {"y": h * phi(h), "dx": dx}
            if b is not None:
                out["db"] = dx.sum(0)
            return out
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        rstd = (var + EPS).pow(-0.5)
        w = s["w"].double()
        xhat = (_kept(s["x"].float()) - mean) * rstd
        g = dy * w
        C = x.shape[1]
        dx = (C * g - g.sum(1, keepdim=True) - xhat * (g * xhat).sum(1, keepdim=True)) * rstd / C
        return {"y": torch.addcmul(b, (x - mean) * rstd, w), "dx": dx, "dw": (dy * xhat).sum(0), "db": dy.sum(0)}


def _kept(x):
    """What the checkpoint of the fp32 matrix x stands for, in fp64: the codes follow from fp32 steps by definition,
    each taken here as the fp64 result rounded to fp32."""
    out = torch.empty_like(x, dtype=torch.float64)
    for c in range(0, x.shape[1], GROUP):
        part = x[:, c:c + GROUP].double()
        lo = part.min(1, keepdim=True).values
        hi = part.max(1, keepdim=True).values
        third = torch.tensor(1.0 / 255.0).double().item()              # the fp32 number nearest to 1/255
        step = ((hi - lo).float().double() * third).float().double()
        inverse = (1.0 / step.clamp_min(1e-300)).float().double()
        code = torch.round(((part - lo).float().double() * inverse).float())
        out[:, c:c + GROUP] = torch.where(step > 0, lo + code.double() * step, lo.expand_as(part))
    return out


def _exact_ce(s):
    x, w = s["x"].double(), s["w"].double()
    N, V, eps, t = s["N"], s["V"], s["smoothing"], s["t"]
    b = s["b"].double() if s["b"] is not None else torch.zeros(V, dtype=torch.float64, device=x.device)
    kept = t.ne(s["ignore_index"])
    count = kept.sum().item()
    want = torch.full((V,), eps / V, dtype=torch.float64, device=x.device)
    losses, dx, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    for lo in range(0, N, 4096):
        k, rows = kept[lo:lo + 4096], x[lo:lo + 4096]
        logp = torch.log_softmax(torch.addmm(b, rows, w.t()), 1)
        target = want.repeat(len(rows), 1)
        target[torch.arange(len(rows), device=x.device)[k], t[lo:lo + 4096][k]] += 1.0 - eps
        target[~k] = 0
        losses.append(-(target * logp).sum(1))
        if s["train"]:
            up = s["up"].double()
            up = up[lo:lo + 4096] if s["reduction"] == "none" else (up / count if s["reduction"] == "mean" else up).expand(len(rows))
            g = (logp.exp() - target) * torch.where(k, up, 0.0)[:, None]
            dx.append(g @ w)
            dw += g.t() @ rows
            db += g.sum(0)
    loss = torch.cat(losses)
    loss = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / count if count else loss.sum() * math.nan}[s["reduction"]]
    if not s["train"]:
        return {"loss": loss}
    out = {"loss": loss, "dx": torch.cat(dx), "dw": dw}
    if s["b"] is not None:
        out["db"] = db
    return out

"""ops.linear_cross_entropy against float64 on the same inputs.

Tolerances, element by element, from the arithmetic (u = 2^-24):
  a logit is a sum over D in fp32: at most 2u for each of the D/16 additions of the tensor core (it truncates) plus 8 more
    for the rest of the formula, at the size of sum |x||w|;
  softmax and loss add the errors of exp2 and log2 (2^-22 each, absolute in the exponent) and two roundings of the logits;
  the gradient of the logits is off by that, relatively, and for bf16 by its rounding to bf16 (2^-8);
  dx, dw and db add the same bound for their own sums, and their rounding to bf16 (2^-8) where they are bf16."""
import gc

import pytest
import torch

import oriented1d_b200 as o1d

ops = o1d.ops
gpu = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def leave_no_garbage():
    """Tensors in reference cycles (an exception's frames) are freed here, not in the middle of a test that counts bytes."""
    yield
    gc.collect()


def make(N, D, V, dtype, bias="same", seed=0, ignored=0.0, ignore_index=-100, logit=2.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g) * (logit / D ** 0.5)
    t = torch.randint(0, V, (N,), generator=g)
    x = torch.randn(N, D, generator=g) + torch.rand(N, 1, generator=g) * w[t]
    t[torch.rand(N, generator=g) < ignored] = ignore_index
    b = None
    if bias:
        b = (0.5 * torch.randn(V, generator=g)).to(DT["fp32" if (bias == "other") == (dtype == "bf16") else "bf16"])
    return x.to(DT[dtype]).cuda(), w.to(DT[dtype]).cuda(), None if b is None else b.cuda(), t.cuda()


def reference(x, w, b, t, up, ignore_index, smoothing, reduction):
    """(loss rows, reduced loss, dx, dw, db) and bounds of their errors, all float64."""
    bf16 = x.dtype == torch.bfloat16
    x, w = x.double(), w.double()
    N, D = x.shape
    V = w.shape[0]
    l = x @ w.t()
    size = (x.abs() @ w.abs().t()).amax(1, keepdim=True)
    if b is not None:
        l = l + b.double()
        size = size + b.double().abs().max()
    e_l = 2 * U * (D / 16 + 8) * size                                     # error of a row's logits
    kept = t != ignore_index
    safe = t.clamp(0, V - 1)
    lse = torch.logsumexp(l, 1, keepdim=True)
    rows = lse[:, 0] - (1 - smoothing) * l.gather(1, safe[:, None])[:, 0] - smoothing * l.mean(1)
    rows = torch.where(kept, rows, torch.zeros_like(rows))
    e_rows = (2 * e_l + 2.0 ** -20 + 8 * U * l.abs().amax(1, keepdim=True))[:, 0]
    count = kept.sum()
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / count}[reduction]
    e_loss = {"none": e_rows, "sum": e_rows.sum(), "mean": e_rows.max()}[reduction] + U * loss.abs()
    scale = up.double() / (count if reduction == "mean" else 1)
    scale = torch.where(kept, scale.expand(N), torch.zeros((), dtype=torch.float64, device=x.device))[:, None]
    p = torch.exp(l - lse)
    onehot = torch.zeros_like(l).scatter_(1, safe[:, None], 1 - smoothing)
    g = (p - onehot - smoothing / V) * scale
    e_g = (p * (2 * e_l + 2.0 ** -20 + 8 * U * l.abs().amax(1, keepdim=True)) + 8 * U * (p + onehot + smoothing / V)) * scale.abs()
    if bf16:
        e_g = e_g + 2.0 ** -8 * 1.01 * g.abs()
    out = []
    for r, m, k in ((g @ w, e_g @ w.abs() + 2 * U * (V / 16 + 40) * (g.abs() @ w.abs()), bf16),
                    (g.t() @ x, e_g.t() @ x.abs() + 2 * U * (N / 16 + 40) * (g.t().abs() @ x.abs()), bf16),
                    (g.sum(0), e_g.sum(0) + 2 * U * (N / 8 + 40) * g.abs().sum(0), b is not None and b.dtype == torch.bfloat16)):
        out.append((r, m + (2.0 ** -8 if k else 4 * U) * r.abs() + 1e-38))
    return loss, e_loss, out


def within(got, ref, bound, what):
    got = got.double()
    assert got.shape == ref.shape, what
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound, worst {float(((got - ref).abs() / bound).max()):.3g} times it"


def check(N, D, V, dtype, bias="same", smoothing=0.0, reduction="mean", ignored=0.0, ignore_index=-100, seed=0, logit=2.0):
    x, w, b, t = make(N, D, V, dtype, bias, seed, ignored, ignore_index, logit)
    up = torch.rand(N if reduction == "none" else (), device="cuda") + 0.5
    loss, e_loss, grads = reference(x, w, b, t, up, ignore_index, smoothing, reduction)
    leaves = [v.requires_grad_(True) for v in (x, w, b) if v is not None]
    kw = dict(ignore_index=ignore_index, label_smoothing=smoothing, reduction=reduction)
    got = ops.linear_cross_entropy(x, w, t, b, **kw)
    assert got.dtype == torch.float32
    within(got.detach(), loss, e_loss, "loss")
    out = torch.autograd.grad(got, leaves, up)
    for leaf, o, (r, bound), what in zip(leaves, out, grads, ("dx", "dw", "db")):
        assert o.dtype == leaf.dtype
        within(o, r, bound, what)
    # the bounds above are worst cases; taken together the errors are random.  No fp32 softmax is nearer than its exponent
    # allows: l, l * log2(e) and l - lse are each rounded at the size of l (u|l| absolute), which exp makes relative: 4u max|l|
    with torch.no_grad():
        most = 4 * U * float((x.double() @ w.double().t()).abs().max())
    for o, (r, _), leaf in zip(out, grads, leaves):
        n = float(r.norm())
        if n > 1e-3 * float(up.mean()):
            assert float((o.double() - r).norm()) <= ((2.0 ** -8 if torch.bfloat16 in (x.dtype, leaf.dtype) else 3e-6) + most) * n
    with torch.no_grad():
        alone = ops.linear_cross_entropy(x, w, t, b, **kw)               # up to eight rows: a kernel of its own, in another order
        assert torch.equal(alone, got) if N > 8 else True
        within(alone, loss, e_loss, "loss without gradients")
    assert o1d.ops.device_status() == 0
    return out


# around every tile edge: rows 128, classes 128 (fp32) and 256 (bf16) and their halves and quarters, features 64 and 8
# (and the kernel for up to eight rows: each of its row counts, vectors and none, the longest row it takes and one it does not)
SHAPES = [(1, 8, 2), (1, 768, 1000), (1, 8192, 40), (1, 8200, 40), (2, 100, 3001), (4, 2048, 77), (5, 48, 700), (8, 1024, 2500), (8, 1025, 50), (9, 64, 300), (2, 64, 10), (3, 1, 1), (7, 72, 31), (31, 16, 33), (64, 65, 64), (127, 63, 63), (128, 64, 256), (129, 100, 257),
          (130, 127, 127), (200, 128, 129), (255, 192, 255), (256, 96, 150), (257, 15, 1000), (300, 384, 511), (513, 1024, 2049), (1000, 33, 5003),
          (2600, 200, 5003), (5003, 1000, 5001)]        # tiles on pairs of CTAs, in some of the products and in all


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N,D,V", SHAPES)
def test_shapes(N, D, V, dtype):
    check(N, D, V, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("bias", [None, "same", "other"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
def test_options(smoothing, bias, reduction, dtype):
    check(150, 40, 300, dtype, bias, smoothing, reduction, ignored=0.3, ignore_index=7)
    check(33, 96, 21, dtype, bias, smoothing, reduction)


@gpu
@pytest.mark.parametrize("N,D,V,dtype,reduction", [
    (2100, 64, 40001, "bf16", "mean"),        # pieces of the classes
    (1500, 72, 20001, "fp32", "none"),
    (80001, 32, 1000, "bf16", "none"),        # pieces of the rows
    (40003, 24, 700, "fp32", "mean"),
    (30000, 64, 10, "bf16", "mean"),          # the gradient of the weight has one tile and a long K axis: parts
    (9000, 100, 3, "fp32", "sum"),
    (5, 64, 30011, "bf16", "sum"),            # dx has one tile and a long K axis
    (3, 40, 9001, "fp32", "mean"),
    (4100, 1000, 17001, "bf16", "mean"),      # pieces whose products have one part: the last one adds the others to what it writes
    (4101, 997, 17001, "bf16", "none"),
    (2500, 1100, 9001, "fp32", "sum"),        # the same in fp32
    (14001, 1002, 5000, "bf16", "sum"),       # and of the rows
    (2100, 64, 50001, "bf16", "mean"), (1500, 72, 24001, "fp32", "none"), (110001, 32, 1000, "bf16", "none"), (50003, 24, 700, "fp32", "mean"),
    (4100, 1000, 28001, "bf16", "mean"), (4101, 997, 28001, "bf16", "none"), (2500, 1100, 14001, "fp32", "sum"), (21001, 1002, 5000, "bf16", "sum"),
])
def test_pieces_and_parts(N, D, V, dtype, reduction):
    check(N, D, V, dtype, reduction=reduction, smoothing=0.1, ignored=0.1)


# more than 2^30 products, up to 192 classes and 128 features: one kernel for the gradients.  Around its blocks of 64 and pieces of 32
DENSE = [(75001, 96, 150), (43700, 128, 192), (60001, 100, 180), (270000, 63, 64), (530011, 64, 33), (2100007, 24, 22), (700001, 8, 192),
         (260000, 65, 65), (560003, 120, 16), (4200001, 128, 2), (2300001, 3, 160), (90112, 127, 97)]


@gpu
@pytest.mark.parametrize("N,D,V", DENSE)
def test_few_classes_and_narrow_features(N, D, V):
    check(N, D, V, "bf16", ignored=0.1)


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("bias", [None, "same", "other"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
def test_options_of_few_classes(smoothing, bias, reduction):
    check(100001, 96, 120, "bf16", bias, smoothing, reduction, ignored=0.3, ignore_index=7)


@gpu
def test_parts_of_the_gradient_of_few_classes():
    """Any of the three gradients alone is the same, bits and all; labels that are no class and rows without a loss."""
    x, w, b, t = make(80003, 96, 150, "bf16", ignored=0.2)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    up = torch.rand(80003, device="cuda")
    f = lambda t, r, *v: ops.linear_cross_entropy(v[0], v[1], t, v[2], reduction=r)  # noqa: E731
    all_of = torch.autograd.grad(f(t, "none", *leaves), leaves, up)
    again = torch.autograd.grad(f(t, "none", *leaves), leaves, up)
    for i in range(3):
        alone, = torch.autograd.grad(f(t, "none", *(v if k == i else v.detach() for k, v in enumerate(leaves))), leaves[i], up)
        assert torch.equal(alone, all_of[i]) and torch.equal(again[i], all_of[i])
    assert not all_of[0][t == -100].any() and all_of[0][t != -100].any(1).all()
    none = torch.autograd.grad(f(torch.full_like(t, -100), "mean", *leaves), leaves)
    assert not any(g.any() for g in none)
    wrong = t.clone()
    wrong[[5, 79999]] = torch.tensor([150, -1], device="cuda")
    rows = f(wrong, "none", *leaves)
    dx, = torch.autograd.grad(rows, x, up)
    bad = torch.zeros(80003, dtype=torch.bool, device="cuda")
    bad[[5, 79999]] = True
    assert rows[bad].isnan().all() and dx[bad].isnan().all()
    assert torch.equal(dx[~bad], all_of[0][~bad])


@gpu
def test_sums_over_very_many_rows_do_not_drift():
    """Few classes, 29 million rows: the upstream gradient of the first half is 1, of the second, the same rows, -1, so that the weight's
    gradient is zero.  All weights are zero: G = 1/64 (and 1/64 - 1 of class 0) is exact in bf16, and what dw is off by is what the tensor
    core's additions lose: half a unit (2^-24) of the sum so far, on average, for each of at most 2048 that one sum takes (its mean is half
    of what its terms add up to)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    half, D, V = 6 * 128 * sms * 128, 24, 64                                   # six launches' worth of rounds; every SM gets both halves
    x = torch.rand(half, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.bfloat16) + 0.25
    x = torch.cat([x, x])
    w = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    b = torch.zeros(V, device="cuda", requires_grad=True)
    t = torch.zeros(2 * half, dtype=torch.int64, device="cuda")
    up = torch.ones(2 * half, device="cuda")
    up[half:] = -1
    dw, db = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, b, reduction="none"), (w, b), up)
    terms = 2 * x[:half].double().sum(0) / V * torch.where(torch.arange(V, device="cuda") == 0, V - 1, 1)[:, None]
    assert float((dw.double().abs() / terms).max()) <= 2048 * 2.0 ** -24 / 2
    assert not db.any()                                                        # whole numbers of 1/64


@gpu
@pytest.mark.parametrize("extra", [0, 1, 128, 40001])
def test_few_classes_in_several_launches(extra):
    """Rows around the number that one launch takes (256 tiles of 128 an SM): each row's gradient is the one it has among few rows, and
    the sums are those of float64."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    N, D, V = 256 * 128 * sms + extra, 9, 31
    g = torch.Generator(device="cuda").manual_seed(extra)
    x = torch.randn(N, D, device="cuda", generator=g).bfloat16().requires_grad_(True)
    w = torch.randn(V, D, device="cuda", generator=g).bfloat16().requires_grad_(True)
    b = torch.randn(V, device="cuda", generator=g).requires_grad_(True)
    t = torch.randint(-1, V, (N,), device="cuda", generator=g)
    up = torch.rand(N, device="cuda", generator=g)
    f = lambda x, t, up: torch.autograd.grad(ops.linear_cross_entropy(x, w, t, b, ignore_index=-1, reduction="none"), (x, w, b), up)  # noqa: E731
    dx, dw, db = f(x, t, up)
    rdw, rdb, s_db = 0, 0, 0
    with torch.no_grad():
        for lo in range(0, N, 1 << 20):
            xs, ts, us = x[lo:lo + (1 << 20)].double(), t[lo:lo + (1 << 20)], up[lo:lo + (1 << 20)].double()
            G = torch.softmax(xs @ w.double().t() + b.double(), 1)
            G[torch.arange(len(ts), device="cuda"), ts.clamp_min(0)] -= 1
            G *= torch.where(ts == -1, 0, us)[:, None]
            ref = G @ w.double()
            # each element of G to half a unit of bf16, a few units of fp32 in its exponent, and the result's own rounding
            assert ((dx[lo:lo + (1 << 20)].double() - ref).abs() <= 2.0 ** -8 * (G.abs() @ w.double().abs()) + 2.0 ** -8 * ref.abs() + 1e-6).all()
            rdw, rdb, s_db = rdw + G.t() @ xs, rdb + G.sum(0), s_db + G.abs().sum(0)
    # (labels are random: a class's sums are of its rows' own size, and the roundings of millions of rows' G cancel in them)
    assert float((dw.double() - rdw).norm()) <= 2.0 ** -8 * float(rdw.norm())
    assert ((db.double() - rdb).abs() <= 1e-5 * s_db).all()
    tail = slice(N - 100_000, N)
    assert torch.equal(f(x[tail].detach().repeat(40, 1).requires_grad_(True), t[tail].repeat(40), up[tail].repeat(40))[0][:100_000], dx[tail])


@gpu
def test_extreme_rows_of_few_classes():
    """Masked classes, targets among them, rows that are not finite with and without a loss: each row alone is affected."""
    N, D, V = 80003, 96, 150
    x, w, b, t = make(N, D, V, "bf16", bias=None, ignored=0.1)
    b = torch.zeros(V, device="cuda")
    b[140:145], b[145:] = -float("inf"), torch.finfo(torch.float32).min
    t[t >= 140] = 3
    t[7], t[8], t[9], t[10] = 141, 2, -100, -100
    x[8] = float("nan")
    x[9] = float("inf")
    x[10, 5] = float("nan")
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    rows = ops.linear_cross_entropy(x, w, t, b, reduction="none")
    dx, _, db = torch.autograd.grad(rows, leaves, torch.ones_like(rows))
    odd = torch.zeros(N, dtype=torch.bool, device="cuda")
    odd[7:11] = True
    assert rows[7] == float("inf") and rows[8].isnan() and rows[9] == 0 and rows[10] == 0
    assert dx[8].isnan().all() and not dx[9:11].any() and dx[7].isfinite().all() and rows[~odd].isfinite().all()
    l = x.detach()[~odd].double() @ w.detach()[:140].double().t()
    tt = t[~odd]
    kept = tt != -100
    p = torch.softmax(l, 1)
    p[torch.arange(len(tt), device="cuda"), tt.clamp_min(0)] -= 1
    p[~kept] = 0
    ref = p @ w.detach()[:140].double()
    assert float((dx[~odd].double() - ref).norm()) <= 2.0 ** -8 * float(ref.norm())
    with torch.no_grad():
        x[8], x[9], x[10] = 0, 0, 0
    rows = ops.linear_cross_entropy(x, w, t, b, reduction="none")
    again, db = torch.autograd.grad(rows, (leaves[0], leaves[2]), torch.ones_like(rows))
    assert torch.equal(again[~odd], dx[~odd]) and not db[145:].any() and not db[142:145].any() and db[141] == -1


@gpu
@pytest.mark.parametrize("rows", ["sure", "alike"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 0.3, 0.9])
@pytest.mark.parametrize("N,D,V", [(80003, 96, 150), (8190, 512, 1000)])
def test_gradients_that_all_rows_round_alike(N, D, V, smoothing, rows):
    """More than 2^30 products, where the logits' gradient G is rounded to bf16 (2^-8 of an element at most), and rows whose G are the
    same numbers, so that roundings do not average out: every row sure of its class (smoothing leaves e/V for each other class), or equal
    logits everywhere.  They add up to 2^-8 of the gradient at most, and its own rounding is another 2^-8."""
    x, w, b, t = make(N, D, V, "bf16", bias=None)
    with torch.no_grad():
        if rows == "sure":
            w.copy_(torch.randn(V, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)))
            x.copy_(1.5 * w[t].float() + torch.rand(x.shape, device="cuda"))
        else:
            w.zero_()
    up = torch.ones((), device="cuda")
    loss, e_loss, grads = reference(x, w, None, t, up, -100, smoothing, "mean")
    leaves = [v.requires_grad_(True) for v in (x, w)]
    got = ops.linear_cross_entropy(x, w, t, label_smoothing=smoothing)
    within(got.detach(), loss, e_loss, "loss")
    for o, (ref, bound), what in zip(torch.autograd.grad(got, leaves), grads, ("dx", "dw")):
        within(o, ref, bound, what)
        assert float((o.double() - ref).norm()) <= 2 * 2.0 ** -8 * float(ref.norm()), what


@gpu
@pytest.mark.parametrize("N,D,V,dtype", [(20001, 16, 24001, "bf16"), (60001, 16, 4001, "bf16"), (50001, 24, 1000, "bf16"), (17001, 8, 18001, "fp32"),
                                         (40001, 8, 3001, "fp32")])
def test_bias_gradient_of_many_rows(N, D, V, dtype):
    """More than 16384 rows a piece, whose column sums are added in two steps: pieces of the classes, of the rows (a short last one), and one."""
    check(N, D, V, dtype, "other" if dtype == "bf16" else "same", ignored=0.1, reduction="sum")


@gpu
@pytest.mark.parametrize("N,V", [(131072, 131072), (500_000, 500_000), (2_000_000, 300_000), (300_000, 2_000_000), (4096, 21841), (9, 10_000_000)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_workspace_of_the_backward_pass(N, V, dtype):
    """What include/o1d.h says of it: the logits' gradient in pieces of 192 MB, or of 256 rows or columns where those are more, and
    beside it planes of the operands (none for bf16 rows of whole vectors), fp32 sums of the pieces' products and column sums of 32 rows."""
    D, planes = 8, 1 if dtype else 3
    piece = max(192 << 20, 256 * 2 * planes * (min(N, V) + 64))
    operands = 0 if dtype else planes * 2 * D * (N + V)
    sums = 4 * D * (N + V) + 4 * D * 148 * 4096                              # of one part each, or parts that are short
    assert o1d._lib.lib.o1d_linear_xent_workspace_bytes(N, D, V, dtype, 1) <= piece * (1 + 1 / 16) + operands + sums + (64 << 20)


@gpu
def test_gradients_against_differences():
    """The fp32 gradient against central differences of the float64 loss along random directions."""
    x, w, b, t = make(70, 48, 90, "fp32", ignored=0.2)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    grads = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, b, label_smoothing=0.1), leaves)
    f = lambda x, w, b: torch.nn.functional.cross_entropy(x @ w.t() + b, t, label_smoothing=0.1)  # noqa: E731
    torch.manual_seed(0)
    base = [v.detach().double() for v in leaves]
    for i in range(3):
        step = torch.randn_like(base[i])
        hi = [v + 1e-5 * step if k == i else v for k, v in enumerate(base)]
        lo = [v - 1e-5 * step if k == i else v for k, v in enumerate(base)]
        num = (f(*hi) - f(*lo)) / 2e-5
        assert abs(float((grads[i].double() * step).sum() - num)) <= 1e-5 * float((grads[i].double() * step).abs().sum())


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_without_a_loss_and_labels_that_are_none(dtype):
    x, w, b, t = make(200, 64, 100, dtype, ignored=0.4)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    none = torch.full_like(t, -100)
    for reduction in ("mean", "sum", "none"):
        loss = ops.linear_cross_entropy(x, w, none, b, reduction=reduction)
        grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
        assert loss.isnan().all() if reduction == "mean" else not loss.any()
        assert not any(g.any() for g in grads)
    rows = ops.linear_cross_entropy(x, w, t, b, reduction="none")
    assert not rows[t == -100].any() and (rows[t != -100] != 0).all()
    dx, = torch.autograd.grad(rows.sum(), x)
    assert not dx[t == -100].any() and dx[t != -100].any(1).all()
    for bad in (100, -1, 2 ** 40, -2 ** 62):
        s = t.clone()
        s[3] = bad
        rows = ops.linear_cross_entropy(x, w, s, b, reduction="none")
        dx, dw = torch.autograd.grad(rows, (x, w), torch.ones_like(rows))
        others = torch.arange(200, device="cuda") != 3
        assert rows[3].isnan() and rows[others].isfinite().all()
        assert dx[3].isnan().all() and dx[others].isfinite().all() and dw.isnan().all()
        assert ops.linear_cross_entropy(x, w, s, b).isnan()
    assert o1d.ops.device_status() == 0


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_extreme_logits(dtype):
    """Large logits (exp would overflow), classes switched off by a bias of -inf, rows of NaN and infinities."""
    check(64, 32, 70, dtype, logit=60.0)
    x, w, b, t = make(64, 32, 70, dtype)
    b = b.float()
    off = torch.zeros(70, dtype=torch.bool, device="cuda")
    off[10:40] = True
    b[off] = -float("inf")
    t = torch.where(off[t], torch.zeros_like(t), t)
    up = torch.ones((), device="cuda")
    keep = (~off).nonzero()[:, 0]
    new = torch.full((70,), -1, device="cuda")
    new[keep] = torch.arange(len(keep), device="cuda")
    loss, e_loss, grads = reference(x, w[keep], b[keep], new[t], up, -100, 0.0, "mean")
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    got = ops.linear_cross_entropy(x, w, t, b)
    dx, dw, db = torch.autograd.grad(got, leaves)
    within(got.detach(), loss, e_loss, "loss")
    within(dx, *grads[0], "dx")
    within(dw[keep], *grads[1], "dw")
    within(db[keep], *grads[2], "db")
    assert not dw[off].any() and not db[off].any()
    y = x.detach().clone()
    y[5, 3], y[6, 3] = float("nan"), float("inf")
    rows = ops.linear_cross_entropy(y, w.detach(), t, b.detach(), reduction="none")
    others = torch.ones(64, dtype=torch.bool, device="cuda")
    others[5:7] = False
    assert rows[~others].isnan().all() and rows[others].isfinite().all()
    assert o1d.ops.device_status() == 0


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_layouts(dtype):
    """More axes, strided and misaligned inputs, a channels-last map with a label a pixel, one row without a batch axis."""
    x, w, b, t = make(96, 40, 50, dtype)
    want = ops.linear_cross_entropy(x, w, t, b, reduction="none").detach()
    assert torch.equal(ops.linear_cross_entropy(x.view(4, 24, 40), w, t.view(4, 24), b, reduction="none"), want.view(4, 24))
    assert torch.equal(ops.linear_cross_entropy(x.t().contiguous().t(), w.t().contiguous().t(), t, b, reduction="none"), want)
    pad = torch.empty(96 * 40 + 1, device="cuda", dtype=x.dtype)
    pad[1:] = x.reshape(-1)
    assert torch.equal(ops.linear_cross_entropy(pad[1:].view(96, 40), w, t, b, reduction="none"), want)      # off a 16-byte boundary
    # (a single row has a kernel of its own, which adds in another order: 40 products of a few units each, to 2^-24 of them)
    assert float((ops.linear_cross_entropy(x[5], w, t[5], b, reduction="none") - want[5]).abs()) <= 1e-5
    a = x.view(2, 6, 8, 40).permute(0, 3, 1, 2).detach().requires_grad_(True)                                   # an NCHW view of NHWC data
    loss = ops.linear_cross_entropy(a.permute(0, 2, 3, 1), w, t.view(2, 6, 8), b)
    assert torch.autograd.grad(loss, a)[0].shape == a.shape
    other = torch.float32 if dtype == "bf16" else torch.bfloat16
    v = w.to(other).requires_grad_(True)
    loss = ops.linear_cross_entropy(x, v, t, b)
    assert torch.autograd.grad(loss, v)[0].dtype == other


@gpu
def test_only_the_gradients_asked_for_and_empty_batches():
    x, w, b, t = make(100, 64, 300, "bf16")
    full = torch.autograd.grad(ops.linear_cross_entropy(*(v.requires_grad_(True) for v in (x, w)), t, b.requires_grad_(True)), (x, w, b))
    for i in range(3):
        part = [v.detach().requires_grad_(k == i) for k, v in enumerate((x, w, b))]
        g, = torch.autograd.grad(ops.linear_cross_entropy(part[0], part[1], t, part[2]), part[i])
        assert torch.equal(g, full[i])
    e = x[:0].detach().requires_grad_(True)
    for reduction, value in (("sum", 0.0), ("mean", float("nan")), ("none", None)):
        loss = ops.linear_cross_entropy(e, w, t[:0], b, reduction=reduction)
        assert loss.shape == ((0,) if value is None else ()) and (value is None or torch.equal(loss, torch.tensor(value, device="cuda")) or (value != value and loss.isnan()))
        ge, gw, gb = torch.autograd.grad(loss, (e, w, b), torch.ones_like(loss))
        assert ge.shape == (0, 64) and not gw.any() and not gb.any()


@gpu
def test_more_than_32_bits_of_logits():
    """70000 x 32768 logits, 2.3e9: the last rows' losses and gradients are those of the same rows alone."""
    x, w, b, t = make(70000, 8, 32768, "bf16")
    rows = ops.linear_cross_entropy(x.requires_grad_(True), w.requires_grad_(True), t, b, reduction="none")
    up = torch.ones_like(rows)
    dx, dw = torch.autograd.grad(rows, (x, w), up)
    tail = x.detach()[-200:].clone().requires_grad_(True)
    want = ops.linear_cross_entropy(tail, w.detach(), t[-200:], b, reduction="none")
    assert float((rows[-200:] - want).detach().abs().max()) <= 1e-4
    ref, = torch.autograd.grad(want, tail, up[-200:])
    assert float((dx[-200:] - ref).float().norm()) <= 2.0 ** -8 * float(ref.float().norm())
    assert dw.isfinite().all() and dx.isfinite().all()


@gpu
def test_repeats_bit_for_bit_streams_and_graphs():
    x, w, b, t = make(700, 96, 2000, "bf16", ignored=0.1)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]

    def step():
        loss = ops.linear_cross_entropy(*leaves[:2], t, leaves[2], label_smoothing=0.1)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    first = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:                                                    # two calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(step())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(first, o))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        x.mul_(0.5)
    graph.replay()
    again = step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(captured, again)) and not torch.equal(first[0], again[0])


@gpu
def test_the_logits_are_not_kept():
    """16384 x 30000 bf16 logits alone would be 983 MB."""
    x, w, b, t = make(16384, 64, 30000, "bf16")
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    loss = ops.linear_cross_entropy(*leaves[:2], t, leaves[2])
    assert torch.cuda.memory_allocated() - base <= 16384 * 12 + 8192       # three floats a row
    torch.autograd.grad(loss, leaves)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - base <= 256 << 20


def test_refusals():
    x, w, t = torch.zeros(4, 16), torch.zeros(10, 16), torch.zeros(4, dtype=torch.int64)
    f = ops.linear_cross_entropy
    with pytest.raises(ValueError, match="reduction"):
        f(x, w, t, reduction="average")
    with pytest.raises(ValueError, match="weight must be"):
        f(x, torch.zeros(10, 15), t)
    with pytest.raises(ValueError, match="weight must be"):
        f(x, torch.zeros(0, 16), t)
    with pytest.raises(ValueError, match="bias has"):
        f(x, w, t, torch.zeros(9))
    with pytest.raises(ValueError, match="target has shape"):
        f(x, w, t[:3])
    with pytest.raises(TypeError, match="int64"):
        f(x, w, t.int())
    with pytest.raises(TypeError, match="int64"):
        f(x, w, torch.zeros(4, 10))
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        f(x.half(), w.half(), t)
    for s in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="label_smoothing"):
            f(x, w, t, label_smoothing=s)
    with pytest.raises(ValueError, match="feature"):
        f(torch.zeros(4, 0), torch.zeros(10, 0), t)
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x, w, t)


def test_sizes_that_indices_do_not_hold():
    """One-row steps past the last class stay within 32 bits up to 2^31 - 65536; sizes above are refused before any device is asked."""
    lib, p = o1d._lib.lib, torch.zeros(256).data_ptr()
    for k in range(3):
        n = [4, 8, 10]
        n[k] = 2 ** 31 - 65535
        assert lib.o1d_linear_xent(p, p, None, p, p, None, p, p, 0, *n, -100, 0.0, 2, 0, None) == 2
        assert lib.o1d_linear_xent_bwd(p, p, None, p, p, p, p, p, p, None, p, 0, *n, -100, 0.0, 2, 0, None) == 2
        assert lib.o1d_linear_xent_workspace_bytes(*n, 0, 0) == 0
    one = torch.zeros(1, 1)
    wide = torch.zeros(1).expand(1, 2 ** 31 - 1)
    for x, w, t in ((one, one.expand(2 ** 31 - 65535, 1), torch.zeros(1, dtype=torch.int64)), (wide, wide, torch.zeros(1, dtype=torch.int64)),
                    (one.expand(2 ** 31 - 65535, 1), one, torch.zeros((), dtype=torch.int64).expand(2 ** 31 - 65535))):
        with pytest.raises(ValueError, match="65536"):
            ops.linear_cross_entropy(x, w, t)


def test_entry_points_reject_bad_arguments():
    lib, buf = o1d._lib.lib, torch.zeros(256)
    p = buf.data_ptr()
    ok = dict(x=p, w=p, b=None, t=p, loss=p, lse=p, count=p, ws=p, n=0, N=4, D=8, V=10, ig=-100, s=0.0, red=2, dt=0, st=None)
    call = lambda **k: lib.o1d_linear_xent(*{**ok, **k}.values())  # noqa: E731
    for k in ("x", "w", "t", "loss", "count"):
        assert call(**{k: None}) == 1, k
    for k in (dict(N=0), dict(D=0), dict(V=-1), dict(s=-1.0), dict(s=float("nan")), dict(red=3), dict(dt=2)):
        assert call(**k) == 1, k
    okb = dict(x=p, w=p, b=None, t=p, lse=p, count=p, dl=p, dx=p, dw=p, db=None, ws=p, n=0, N=4, D=8, V=10, ig=-100, s=0.0, red=2, dt=0, st=None)
    callb = lambda **k: lib.o1d_linear_xent_bwd(*{**okb, **k}.values())  # noqa: E731
    for k in ("x", "w", "t", "lse", "count", "dl"):
        assert callb(**{k: None}) == 1, k
    assert lib.o1d_linear_xent_workspace_bytes(0, 8, 10, 0, 0) == 0


@gpu
def test_refusals_on_the_device():
    x, w, b, t = make(4, 16, 10, "fp32")
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.linear_cross_entropy(x, w, t.cpu(), b)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.linear_cross_entropy(x, w, t, b), x, create_graph=True)
    lib = o1d._lib.lib
    n = lib.o1d_linear_xent_workspace_bytes(4, 16, 10, 0, 0)
    assert n > 0
    out, ws = torch.empty(8, device="cuda"), torch.empty(n, dtype=torch.uint8, device="cuda")
    args = lambda p, n: (x.data_ptr(), w.data_ptr(), None, t.data_ptr(), out.data_ptr(), out[4:].data_ptr(), out[1:].data_ptr(), p, n, 4, 16, 10, -100, 0.0, 2, 0, None)  # noqa: E731
    assert lib.o1d_linear_xent(*args(ws.data_ptr(), n - 1)) == 4
    assert lib.o1d_linear_xent(*args(None, n)) == 4
    assert lib.o1d_linear_xent(*args(ws.data_ptr() + 16, n)) == 4

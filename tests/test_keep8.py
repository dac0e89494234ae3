"""8-bit activation checkpoints (ops.keep8 / restore8) and the GELU and LayerNorm that keep one for their backward pass.

References are float64.  The codes of a checkpoint follow from fp32 operations by definition, so the reference does those
steps in numpy float32 and the codes have to be equal, one by one.  Tolerances: an fp32 result may be off by the fp32
operations of its formula (about ten roundings of 2^-24 at the size of its terms: 2e-6 of the largest), a bf16 one by half
a unit of its last place (2^-8 relative) on top."""
import gc
import math
import os
import re

import numpy as np
import pytest
import torch

import oriented1d_b200 as o1d

ops = o1d.ops
gpu = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def leave_no_garbage():
    """Tensors in reference cycles (an exception's frames) are freed here, not in the middle of a test that counts bytes."""
    yield
    gc.collect()


def ref_codes(x):
    """(codes, ranges) of a float32 matrix by the definition, each operation rounded to fp32."""
    rows, C = x.shape
    G = -(-C // 128)
    codes, ranges = np.zeros((rows, C), np.uint8), np.zeros((rows, G, 2), np.float32)
    with np.errstate(all="ignore"):
        for g in range(G):
            v = x[:, 128 * g:128 * g + 128]
            lo, hi = v.min(1), v.max(1)                              # numpy's propagate NaN
            s = ((hi - lo) * np.float32(1 / 255)).astype(np.float32)
            lost = ~np.isfinite(s)
            s = np.where(s < np.finfo(np.float32).tiny, np.float32(0), s)
            inv = np.where(s > 0, np.float32(1) / np.where(s > 0, s, 1), 0).astype(np.float32)
            q = np.rint((v - lo[:, None]) * inv[:, None])
            codes[:, 128 * g:128 * g + 128] = np.where(lost[:, None], 0, q)
            ranges[:, g, 0], ranges[:, g, 1] = lo, np.where(lost, np.nan, s)
    return codes, ranges


def ref_values(codes, ranges):
    C = codes.shape[1]
    r = np.repeat(ranges.astype(np.float64), 128, axis=1)[:, :C]
    return r[..., 0] + codes.astype(np.float64) * r[..., 1]


def make(rows, C, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=g) * (0.3 + torch.rand(C, generator=g)) + 0.5 * torch.randn(C, generator=g)
    return x.to(DT[dtype])


def close(got, ref, dtype, terms=None, what=""):
    """|got - ref| within the roundings of the formula at the size of its terms, and of the output type."""
    got, ref = got.double().cpu(), ref.cpu()
    size = (ref if terms is None else terms.cpu()).abs().max().clamp_min(1e-30)
    tol = 2e-6 * size + (2.0 ** -8 * ref.abs() if dtype == "bf16" else 0)
    bad = (got - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((got - ref).abs().max()):.3g} at size {float(size):.3g}"


# rows of one element, below / at / above every width at which another kernel takes over, odd and even, and the longest
WIDTHS = [1, 3, 4, 7, 8, 31, 32, 33, 64, 65, 100, 127, 128, 129, 132, 256, 260, 385, 512, 516, 1001, 1024, 1028, 2048, 2052, 4096, 4100, 8192]


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("C", WIDTHS + [20000])
def test_codes_and_values(C, dtype):
    for rows in (1, 2, 13, 333):
        x = make(rows, C, dtype, seed=rows)
        codes, ranges = ops.keep8(x.cuda())
        rc, rr = ref_codes(x.float().numpy())
        assert codes.dtype == torch.uint8 and codes.shape == x.shape and ranges.shape == (rows, -(-C // 128), 2)
        assert np.array_equal(ranges.cpu().numpy(), rr)
        assert np.array_equal(codes.cpu().numpy(), rc)
        val = ref_values(rc, rr)
        back = ops.restore8(codes, ranges, DT[dtype])
        assert back.dtype == DT[dtype]
        close(back, torch.from_numpy(val), dtype, what=f"restore {rows}x{C}")
        # at most half a step off, plus the roundings of lo + q*s
        step = np.repeat(rr[..., 1], 128, axis=1)[:, :C]
        assert (np.abs(val - x.double().numpy()) <= 0.5 * step * (1 + 1e-5) + 1e-6 * np.abs(val).max()).all()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_special_groups(dtype):
    """Equal values, zeros of both signs, NaN, infinities, an overflowing range, numbers below the normal ones: each in a
    group of its own, which alone is affected."""
    big = torch.finfo(DT[dtype]).max
    x = make(10, 300, dtype)
    x[0, 128:256] = 3.5
    x[1, :128] = 0.0
    x[1, 5] = -0.0
    x[2, 130] = float("nan")
    x[3, 299] = float("inf")
    x[4, 0] = -float("inf")
    x[5, 10], x[5, 20] = big, -big
    x[6, :128] = torch.linspace(0, 1, 128) * 2.0 ** -130
    x[7, 128:] = float("inf")
    x[8, :] = float("nan")
    lost = torch.zeros(10, 300, dtype=torch.bool)
    lost[2, 128:256] = lost[3, 256:] = lost[4, :128] = lost[5, :128] = lost[7, 128:] = lost[8] = True
    codes, ranges = ops.keep8(x.cuda())
    back = ops.restore8(codes, ranges, torch.float32).cpu()
    rc, rr = ref_codes(x.float().numpy())
    assert np.array_equal(codes.cpu().numpy(), rc)
    assert torch.equal(back.isnan(), lost)
    assert torch.equal(back[0, 128:256], torch.full((128,), 3.5)) and (back[1, :128] == 0).all()
    assert (back[6, :128] >= 0).all() and (back[6, :128] <= 2.0 ** -130).all()
    fine = ~lost
    assert (back[fine].double() - torch.from_numpy(ref_values(rc, rr))[fine]).abs().max() <= 1e-6


def _gelu(h):
    return 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))


def _gelu_grad(h):
    return 0.5 * (1 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)


def _kept(h32):
    rc, rr = ref_codes(h32.numpy())
    return torch.from_numpy(ref_values(rc, rr))


def test_the_fit_of_gelu_is_as_good_as_it_says():
    """The stored fp32 coefficients of t q(t), t = 1/(1 + slope m), against exp(z^2) erfc(z), z = m/sqrt 2, in float64: the relative errors
    that the comment beside them states, at the centre, in the tail and on average."""
    src = open(os.path.join(os.path.dirname(o1d.__file__), "csrc", "o1d_keep8.cuh")).read()
    slope = float(re.search(r"constexpr float slope = ([\d.]+)f;", src).group(1))
    table = re.findall(r"FP32 \? (-?[\d.]+)f : (-?[\d.]+)f", src[src.index("fit[10]"):src.index("fit[10]") + 1500])[:10]
    assert len(table) == 10 and np.float32(slope) == slope
    m = torch.linspace(0, 10 * math.sqrt(2), 40001, dtype=torch.float64)
    t = 1 / (1 + slope * m)
    for column, worst, mean in ((0, 5e-9, 1e-9), (1, 1e-7, 1e-8)):
        coef = [float(np.float32(row[column])) for row in table]
        e = t * sum(c * t ** k for k, c in enumerate(coef)) / torch.special.erfcx(m / math.sqrt(2)) - 1
        assert float(e.abs().max()) <= worst and abs(float(e.mean())) <= mean, (column, float(e.abs().max()), float(e.mean()))


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bias", [None, "same", "other"])
@pytest.mark.parametrize("C", [1, 7, 32, 64, 96, 128, 129, 384, 1001, 2304])
def test_gelu_keep8(C, bias, dtype):
    for rows in (1, 5, 700):
        x, dy = make(rows, C, dtype, 1), make(rows, C, dtype, 2)
        bt = DT["fp32" if (bias == "other") == (dtype == "bf16") else "bf16"] if bias else None
        b = make(1, C, "fp32", 3)[0].to(bt) if bias else None
        h32 = x.float() + b.float() if bias else x.float()
        kept = _kept(h32)
        xd = x.cuda().requires_grad_(True)
        bd = b.cuda().requires_grad_(True) if bias else None
        y = ops.gelu_keep8(xd, bd)
        y.backward(dy.cuda())
        assert y.dtype == x.dtype and xd.grad.dtype == x.dtype
        h = x.double() + b.double() if bias else x.double()
        close(y.detach(), _gelu(h), dtype, terms=h, what="y")
        ref = dy.double() * _gelu_grad(kept)
        close(xd.grad, ref, dtype, terms=dy.double() * 1.2, what="dx")
        if bias:
            assert bd.grad.dtype == bt
            # a sum of `rows` terms in fp32, at most rows/8 of them in a row; the terms' own error on top
            close(bd.grad, ref.sum(0), "bf16" if bt == torch.bfloat16 else "fp32", terms=ref.abs().sum(0), what="db")
        with torch.no_grad():
            assert torch.equal(ops.gelu_keep8(xd, bd), y)


def _ln_ref(x, dy, w, b, eps, kept):
    x, dy, w, b = x.double(), dy.double(), w.double(), b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    y = (x - mean) * rstd * w + b
    xhat = (kept - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return y, dx, (dy * xhat).sum(0), dy.sum(0), xhat, rstd, g


@gpu
@pytest.mark.parametrize("dtype,params", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("C", WIDTHS)
def test_layer_norm_keep8(C, dtype, params):
    eps = 1e-6 if C > 2 else 1e-2                    # two equal columns: their variance alone would be a division by nothing
    for rows in (1, 6, 401):
        x, dy = make(rows, C, dtype, 4), make(rows, C, dtype, 5)
        w, b = (1 + 0.2 * make(1, C, "fp32", 6)[0]).to(DT[params]), make(1, C, "fp32", 7)[0].to(DT[params])
        kept = _kept(x.float())
        y, dx, dw, db, xhat, rstd, g = _ln_ref(x, dy, w, b, eps, kept)
        xd, wd, bd = (t.cuda().requires_grad_(True) for t in (x, w, b))
        out = ops.layer_norm_keep8(xd, wd, bd, eps)
        out.backward(dy.cuda())
        assert out.dtype == xd.grad.dtype == x.dtype and wd.grad.dtype == bd.grad.dtype == w.dtype
        # x - mean cancels: an error of the mean (2^-24 of the row's size) is scaled by rstd * w
        size = (x.double().abs().amax(1, keepdim=True) * rstd * (w.double().abs().max())).max() + b.double().abs().max()
        close(out.detach(), y, dtype, terms=size, what="y")
        hat = (x.double().abs().amax(1, keepdim=True) * rstd).max() + xhat.abs().max()
        close(xd.grad, dx, dtype, terms=(rstd * g.abs().amax(1, keepdim=True)).max() * (1 + hat * xhat.abs().max()), what="dx")
        close(wd.grad, dw, params, terms=(dy.double().abs().sum(0) * hat).max(), what="dw")
        close(bd.grad, db, params, terms=dy.double().abs().sum(0), what="db")
        with torch.no_grad():
            assert torch.equal(ops.layer_norm_keep8(xd, wd, bd, eps), out)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("C", [8, 24, 40, 64, 72, 80, 88, 96, 97, 104, 128, 136, 200])
def test_many_rows(C, dtype):
    """Enough rows for the kernels that hold several vectors of a lane at once: a row's checkpoint and GELU are those it has
    among few rows, bit for bit; LayerNorm, whose sums are in another order, is within the roundings of the formula."""
    rows, some = 120001, 500
    x, dy = (make(2 * some, C, dtype, k).cuda().repeat(-(-rows // (2 * some)), 1)[:rows] for k in (8, 9))
    x = (x.float() * torch.linspace(0.5, 2, rows, device="cuda")[:, None]).to(DT[dtype])
    b = make(1, C, "fp32", 3)[0].cuda().to(DT[dtype])
    codes, ranges = ops.keep8(x)
    back = ops.restore8(codes, ranges, DT[dtype])
    leaves = [t.requires_grad_(True) for t in (x, b)]
    y = ops.gelu_keep8(*leaves)
    dx, db = torch.autograd.grad(y, leaves, dy)
    for at in (0, 60000, rows - some):
        part = x.detach()[at:at + some].clone().requires_grad_(True)
        pc, pr = ops.keep8(part)
        assert torch.equal(pc, codes[at:at + some]) and torch.equal(pr, ranges[at:at + some])
        assert torch.equal(ops.restore8(pc, pr, DT[dtype]), back[at:at + some])
        py = ops.gelu_keep8(part, b.detach())
        assert torch.equal(py, y[at:at + some])
        assert torch.equal(torch.autograd.grad(py, part, dy[at:at + some])[0], dx[at:at + some])
    ref = dx.double() if dtype == "fp32" else None                           # (bf16: the sum is of what dx was rounded from)
    if ref is not None:
        assert ((db.double() - ref.sum(0)).abs() <= 2e-6 * ref.abs().sum(0)).all()

    w = (1 + 0.2 * make(1, C, "fp32", 6)[0]).cuda()
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b.float())]
    y = ops.layer_norm_keep8(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    kept = ops.restore8(codes, ranges).double()                              # fp32: a rounding away from what the kernel holds
    ry, rdx, rdw, rdb, xhat, rstd, g = _ln_ref(x.detach(), dy, w, b.detach(), 1e-6, kept)
    hat = (x.detach().double().abs().amax(1, keepdim=True) * rstd) + xhat.abs().amax(1, keepdim=True)
    half = 2.0 ** -8 if dtype == "bf16" else 0.0
    assert ((y.double() - ry).abs() <= 2e-6 * (hat * w.abs().max() + b.detach().double().abs().max()) + half * ry.abs()).all()
    most = rstd * g.abs().amax(1, keepdim=True) * (1 + hat * xhat.abs().amax(1, keepdim=True))
    assert ((grads[0].double() - rdx).abs() <= 2e-6 * most + half * rdx.abs()).all()
    assert ((grads[1].double() - rdw).abs() <= 2e-6 * (dy.double().abs() * hat).sum(0)).all()
    assert ((grads[2].double() - rdb).abs() <= 2e-6 * dy.double().abs().sum(0)).all()


@gpu
def test_gradients_against_differences():
    """The gradient belongs to the function at the kept values: with an input that the checkpoint holds exactly (256
    evenly spaced values a group) it is the derivative of the forward pass itself."""
    torch.manual_seed(0)
    x = (torch.stack([torch.randperm(256)[:128] for _ in range(6)]).float() - 100) / 32
    x[:, 0], x[:, 1] = -100 / 32, 155 / 32                            # the group's ends: the step is 1/32 exactly
    dy, w, b = torch.randn(6, 128), torch.rand(128) + 0.5, torch.randn(128)
    codes, ranges = ops.keep8(x.cuda())
    assert torch.equal(ops.restore8(codes, ranges).cpu(), x)
    for f, double in ((lambda t: ops.gelu_keep8(t), _gelu),
                      (lambda t: ops.layer_norm_keep8(t, w.cuda(), b.cuda()), lambda t: torch.nn.functional.layer_norm(t, (128,), w.double(), b.double(), 1e-6))):
        xd = x.cuda().requires_grad_(True)
        (f(xd) * dy.cuda()).sum().backward()
        step = torch.randn(6, 128, dtype=torch.float64)
        eps = 1e-5
        num = ((double(x.double() + eps * step) - double(x.double() - eps * step)) * dy.double()).sum() / (2 * eps)
        assert abs(float((xd.grad.cpu().double() * step).sum() - num)) <= 1e-5 * float((xd.grad.cpu().double() * step).abs().sum())


@gpu
def test_layouts_views_and_empty_tensors():
    """Strided inputs and gradients, storage that starts off a vector, more axes, and no rows at all."""
    x = make(64, 96, "bf16").cuda()
    for v in (x.t(), x[:, 1:], x[:, ::2], x[1:, :95].reshape(63, 5, 19), x.view(4, 16, 96)[:, 1:15], x.view(-1)[3:3 + 93 * 8].view(93, 8),
              x[0], x[:1].expand(5, 96)):
        c1, r1 = ops.keep8(v)
        c2, r2 = ops.keep8(v.contiguous().clone())
        assert torch.equal(c1, c2) and torch.equal(r1, r2)
        w, b = torch.rand(v.shape[-1], device="cuda"), torch.rand(v.shape[-1], device="cuda")
        outs = []
        for t in (v.detach(), v.contiguous().clone()):
            t = t.requires_grad_(True)
            for f in (lambda t: ops.gelu_keep8(t, b), lambda t: ops.layer_norm_keep8(t, w, b)):
                y = f(t)
                assert y.shape == v.shape
                dy = torch.ones((), device="cuda", dtype=y.dtype).expand(y.shape)      # stride 0
                outs.append((y.detach(), *torch.autograd.grad(y, t, dy)))
        for a, c in zip(outs[:2], outs[2:]):
            assert all(torch.equal(p, q) for p, q in zip(a, c))
    for shape in ((0, 96), (2, 0, 5)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        b = torch.ones(shape[-1], device="cuda", requires_grad=True)
        (ops.layer_norm_keep8(e, w, b).sum() + ops.gelu_keep8(e, b).sum()).backward()
        assert e.grad.shape == shape and not w.grad.any() and not b.grad.any()
        c, r = ops.keep8(e)
        assert ops.restore8(c, r).shape == shape


@gpu
def test_a_checkpoint_stored_anywhere():
    """Codes and ranges that are views of a larger buffer, off every alignment, or strided."""
    x = make(64, 200, "fp32").cuda()
    codes, ranges = ops.keep8(x)
    want = ops.restore8(codes, ranges)
    c, r = torch.empty(64 * 200 + 3, dtype=torch.uint8, device="cuda"), torch.empty(64 * 4 + 1, device="cuda")
    c[3:], r[1:] = codes.reshape(-1), ranges.reshape(-1)
    assert torch.equal(ops.restore8(c[3:].view(64, 200), r[1:].view(64, 2, 2)), want)
    assert torch.equal(ops.restore8(codes.t().contiguous().t(), ranges.permute(2, 0, 1).contiguous().permute(1, 2, 0)), want)


@gpu
def test_parameters_of_any_shape():
    """Only the number of elements counts; a gradient has its parameter's shape."""
    x = make(6, 40, "fp32").cuda()
    for shape in ((40,), (1, 40), (1, 1, 40), (5, 8)):
        w, b = (torch.rand(shape, device="cuda").requires_grad_(True) for _ in range(2))
        gb, = torch.autograd.grad(ops.gelu_keep8(x, b).sum(), b)
        gw, gc = torch.autograd.grad(ops.layer_norm_keep8(x, w, b).sum(), (w, b))
        assert gb.shape == gw.shape == gc.shape == shape
        flat = b.detach().reshape(40).requires_grad_(True)
        assert torch.equal(torch.autograd.grad(ops.gelu_keep8(x, flat).sum(), flat)[0], gb.reshape(40))


@gpu
def test_more_than_32_bits_of_elements():
    """2.2e9 elements: the last rows are those of the same rows alone."""
    rows, C = 67000, 33000
    x = torch.empty(rows, C, device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    tail = x[-3:].clone()
    codes, ranges = ops.keep8(x)
    c, r = ops.keep8(tail)
    assert torch.equal(codes[-3:], c) and torch.equal(ranges[-3:], r)
    back = ops.restore8(codes, ranges, torch.bfloat16)
    assert torch.equal(back[-3:], ops.restore8(c, r, torch.bfloat16))
    del codes, ranges, back
    b = torch.linspace(-1, 1, C, device="cuda")
    y = ops.gelu_keep8(x.requires_grad_(True), b)
    dx, = torch.autograd.grad(y, x, x.detach())
    t = tail.clone().requires_grad_(True)
    z = ops.gelu_keep8(t, b)
    assert torch.equal(y[-3:], z) and torch.equal(dx[-3:], torch.autograd.grad(z, t, tail)[0])
    del y, dx
    x = x.detach().reshape(-1)[:33000 * 67000 // 4096 * 4096].reshape(-1, 4096).requires_grad_(True)
    w = torch.linspace(0.5, 1, 4096, device="cuda")
    y = ops.layer_norm_keep8(x, w, w)
    dx, = torch.autograd.grad(y, x, x.detach())
    t = x.detach()[-3:].clone().requires_grad_(True)
    z = ops.layer_norm_keep8(t, w, w)
    assert torch.equal(y[-3:], z) and torch.equal(dx[-3:], torch.autograd.grad(z, t, t.detach())[0])


@gpu
def test_sums_repeat_bit_for_bit_and_streams():
    x, dy = make(5000, 385, "bf16").cuda(), make(5000, 385, "bf16", 1).cuda()
    w, b = torch.rand(385, device="cuda"), torch.rand(385, device="cuda")

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.gelu_keep8(ops.layer_norm_keep8(*leaves), leaves[2])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    x.copy_(make(5000, 385, "bf16", 2))
    graph.replay()
    fourth = step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(third, fourth)) and not torch.equal(first[0], third[0])


@gpu
def test_what_stays_in_memory():
    """Between the passes GELU and LayerNorm hold 1.0625 bytes an element (and 8 a row), not the 2 of a bf16 tensor."""
    x = make(4096, 1024, "bf16").cuda()
    w, b = torch.ones(1024, device="cuda", requires_grad=True), torch.zeros(1024, device="cuda", requires_grad=True)
    for f, kept in ((lambda: ops.gelu_keep8(x, b), 4096 * 1024 * 1.0625), (lambda: ops.layer_norm_keep8(x, w, b), 4096 * (1024 * 1.0625 + 8))):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = f()
        got = torch.cuda.memory_allocated() - before - y.numel() * 2
        assert kept <= got <= kept + 4096
        del y


def test_refusals():
    """Checked before the device is, so that they show on any machine."""
    x, w = torch.zeros(4, 16), torch.ones(16)
    for f in (lambda: ops.gelu_keep8(x, torch.ones(15)), lambda: ops.layer_norm_keep8(x, w, torch.ones(17)),
              lambda: ops.layer_norm_keep8(x, torch.ones(0), w)):
        with pytest.raises(ValueError, match="elements, expected 16"):
            f()
    for f in (ops.keep8, ops.gelu_keep8, lambda t: ops.layer_norm_keep8(t, w, w)):
        with pytest.raises(TypeError, match="float32 and bfloat16"):
            f(x.half())
        with pytest.raises(ValueError, match="one column"):
            f(torch.zeros(3, 0))
        with pytest.raises(ValueError, match="one column"):
            f(torch.zeros(()))
        with pytest.raises(RuntimeError, match="CUDA"):
            f(x)
    codes, ranges = torch.zeros(4, 200, dtype=torch.uint8), torch.zeros(4, 2, 2)
    for bad in (torch.zeros(4, 1, 2), torch.zeros(3, 2, 2), torch.zeros(4, 2)):
        with pytest.raises(ValueError, match="ranges have shape"):
            ops.restore8(codes, bad)
    with pytest.raises(TypeError, match="uint8"):
        ops.restore8(codes.float(), ranges)
    with pytest.raises(TypeError, match="uint8"):
        ops.restore8(codes, ranges.double())
    with pytest.raises(TypeError, match="float16"):
        ops.restore8(codes, ranges, torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.restore8(codes, ranges)


def test_entry_points_reject_bad_arguments():
    lib, p = o1d._lib.lib, torch.zeros(64).data_ptr()
    assert lib.o1d_keep8(None, p, p, 1, 8, 0, None) == 1
    assert lib.o1d_keep8(p, p, p, 0, 8, 0, None) == 1
    assert lib.o1d_keep8(p, p, p, 1, 8, 2, None) == 1
    assert lib.o1d_keep8(p, p, p + 4, 1, 8, 0, None) == 2
    assert lib.o1d_keep8(p, p, p, 1, 2 ** 24 + 1, 0, None) == 2
    assert lib.o1d_restore8(p, None, p, 1, 8, 0, None) == 1
    assert lib.o1d_gelu_keep8(p, None, p, p, None, 1, 8, 0, None) == 1          # codes without ranges
    assert lib.o1d_gelu_keep8_bwd(p, p, p, None, None, None, None, 0, 1, 8, 0, None) == 1
    assert lib.o1d_layernorm_keep8(p, p, p, p, p, p, None, 1, 8, 1e-6, 0, None) == 1          # codes without statistics
    assert lib.o1d_layernorm_keep8(p, p, p, p, None, p, p, 1, 8, 1e-6, 0, None) == 1
    assert lib.o1d_layernorm_keep8(p, p, p, p, p, p, p, 1, 8193, 1e-6, 0, None) == 2
    assert lib.o1d_layernorm_keep8_bwd(p, p, p, p, p, None, p, p, p, p, p, 64, 1, 8, 0, None) == 1      # y wanted, beta missing
    assert lib.o1d_layernorm_keep8_bwd(p, p, p, p, p, p, p, None, p, p, None, 0, 1, 8, 0, None) == 4
    assert lib.o1d_layernorm_keep8_bwd_workspace_bytes(1, 9000) == 0


@gpu
def test_refusals_on_the_device():
    x = make(4, 16, "fp32").cuda().requires_grad_(True)
    with pytest.raises(o1d._lib.O1dError):
        ops.layer_norm_keep8(torch.zeros(2, 8193, device="cuda"), torch.ones(8193, device="cuda"), torch.ones(8193, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gelu_keep8(x, torch.zeros(16))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.gelu_keep8(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.layer_norm_keep8(x, x[0].detach(), x[1].detach()).sum(), x, create_graph=True)

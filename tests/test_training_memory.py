"""The training step that keeps little: blocks with 8-bit checkpoints, the head's loss without logits, all together."""
import gc

import pytest
import torch
import torch.nn.functional as F
import torch.nn.utils.prune

import oriented1d_b200 as o1d
from oriented1d_b200 import backbone, convnext1d

ops = o1d.ops
gpu = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def leave_no_garbage():
    """Tensors in reference cycles (an exception's frames) are freed here, not in the middle of a test that counts bytes."""
    yield
    gc.collect()


def mlp_args(rows, C, hidden, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = r(rows, C) * (0.5 + torch.rand(C, generator=g)) + 0.3 * r(C)
    out = [x, 1 + 0.1 * r(C), 0.1 * r(C), r(hidden, C) * (1.5 / C ** 0.5), 0.2 * r(hidden), r(C, hidden) / hidden ** 0.5, 0.1 * r(C)]
    return [t.to(DT[dtype]).cuda().requires_grad_(True) for t in out]


def kept_of(x):
    """What the checkpoint of a float32 matrix stands for, float64."""
    return ops.restore8(*ops.keep8(x.float().reshape(-1, x.shape[-1]))).double().reshape(x.shape)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,C,hidden", [(1, 8, 16), (50, 96, 384), (333, 100, 130), (2000, 128, 512)])
def test_mlp_keep8(rows, C, hidden, dtype):
    """Output and gradients against float64: the gradient of each layer at the values its checkpoint stands for.  The GEMM
    library rounds every product's result to the type (2^-8 relative for bf16) and the hidden tensor's rounding shows in its
    codes; fp32 products carry 2^-24 sqrt(K) or so.  Norm-wise tolerance: four such roundings in a row."""
    torch.backends.cuda.matmul.allow_tf32 = False
    leaves = mlp_args(rows, C, hidden, dtype)
    dz = torch.randn(rows, C, generator=torch.Generator().manual_seed(9)).to(DT[dtype]).cuda()
    out = ops.mlp_keep8(*leaves)
    grads = torch.autograd.grad(out, leaves, dz)
    with torch.no_grad():
        assert torch.equal(ops.mlp_keep8(*leaves), out)
        x, g, b, w1, b1, w2, b2 = (t.detach() for t in leaves)
        # the stored hidden tensor is the library's rounded one; its checkpoint is taken of that plus the bias
        hidden32 = F.linear(ops.layer_norm_keep8(x, g, b), w1).float() + b1.float()
        kx, kh = kept_of(x), kept_of(hidden32)
        x, g, b, w1, b1, w2, b2, d = (t.double() for t in (x, g, b, w1, b1, w2, b2, dz))
        mean = x.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + 1e-6)
        ref_out = F.gelu(((x - mean) * rstd * g + b) @ w1.t() + b1) @ w2.t() + b2
        xhat = (kx - mean) * rstd
        da = d @ w2
        slope = 0.5 * (1 + torch.erf(kh / 2 ** 0.5)) + kh * torch.exp(-kh * kh / 2) / (2 * torch.pi) ** 0.5
        dh = da * slope
        dy = dh @ w1
        gg = dy * g
        dx = rstd * (gg - gg.mean(1, keepdim=True) - xhat * (gg * xhat).mean(1, keepdim=True))
        refs = [dx, (dy * xhat).sum(0), dy.sum(0), dh.t() @ (xhat * g + b), dh.sum(0), d.t() @ F.gelu(kh), d.sum(0)]
    tol = 4 * 2.0 ** -8 if dtype == "bf16" else 2e-5
    assert float((out.detach().double() - ref_out).norm()) <= tol * float(ref_out.norm())
    for name, a, r, leaf in zip(("dx", "dgamma", "dbeta", "dw1", "db1", "dw2", "db2"), grads, refs, leaves):
        assert a.dtype == leaf.dtype and a.shape == leaf.shape
        assert float((a.double() - r).norm()) <= tol * float(r.norm()) + 1e-6, name


@gpu
def test_mlp_keep8_is_near_the_whole_gradient():
    """Against the gradient with everything kept: a code is off by at most half a 255th of its group's range, about six
    standard deviations of normal data, so by 0.007 of one, r.m.s.; that reaches the gradients scaled by slopes of about one."""
    leaves = mlp_args(1500, 96, 384, "fp32")
    dz = torch.randn(1500, 96, device="cuda")
    grads = torch.autograd.grad(ops.mlp_keep8(*leaves), leaves, dz)
    x, g, b, w1, b1, w2, b2 = leaves
    full = torch.autograd.grad(F.linear(F.gelu(F.linear(F.layer_norm(x, (96,), g, b, 1e-6), w1, b1)), w2, b2), leaves, dz)
    for a, r in zip(grads, full):
        assert float((a - r).norm()) <= 0.02 * float(r.norm())


@gpu
def test_only_the_gradients_asked_for():
    leaves = mlp_args(40, 32, 64, "fp32")
    dz = torch.randn(40, 32, device="cuda")
    full = torch.autograd.grad(ops.mlp_keep8(*leaves), leaves, dz)
    for i in range(7):
        part = [t.detach().requires_grad_(k == i) for k, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(ops.mlp_keep8(*part), part[i], dz)[0], full[i])


def small(keep8, variant="1d"):
    torch.manual_seed(3)
    m = convnext1d.ConvNeXt1D(depths=(1, 1, 2, 1), dims=(32, 64, 96, 128), variant=variant, stem_dim1=16, layer_scale_init_value=0.5,
                              num_classes=37, keep8=keep8)
    for p in m.parameters():
        if p.dim() > 1:
            torch.nn.init.normal_(p, std=0.1)
    return m.cuda().train()


@gpu
@pytest.mark.parametrize("variant", ["1d", "2d"])
def test_a_training_step_together(variant):
    """loss() against F.cross_entropy of forward(), with and without checkpoints, on the same weights and batch."""
    torch.backends.cudnn.allow_tf32 = torch.backends.cuda.matmul.allow_tf32 = False
    img = torch.randn(4, 3, 64, 64, generator=torch.Generator().manual_seed(0)).cuda()
    t = torch.tensor([3, 36, -100, 0], device="cuda")
    models = [small(False, variant), small(True, variant)]
    losses, grads = [], []
    for m in models:
        loss = m.loss(img, t, label_smoothing=0.1)
        loss.backward()
        want = F.cross_entropy(m(img).float(), t, label_smoothing=0.1)
        assert abs(float(loss - want)) <= 1e-5 * float(want)
        losses.append(loss.detach())
        grads.append({k: p.grad for k, p in m.named_parameters() if p.grad is not None})
    assert abs(float(losses[0] - losses[1])) <= 1e-5 * float(losses[0])          # the forward pass is the same arithmetic
    assert grads[0].keys() == grads[1].keys()
    for k, a in grads[0].items():
        assert float((a - grads[1][k]).norm()) <= 0.05 * float(a.norm()) + 1e-6, k
    m = models[0]
    m.zero_grad(set_to_none=True)
    F.cross_entropy(m(img), t, label_smoothing=0.1).backward()
    for k, p in m.named_parameters():
        if p.grad is not None:
            assert float((p.grad - grads[0][k]).norm()) <= 1e-4 * float(p.grad.norm()) + 1e-7, k


@gpu
def test_under_autocast():
    m = small(True)
    img = torch.randn(4, 3, 64, 64, device="cuda")
    t = torch.tensor([3, 36, 1, 0], device="cuda")
    with torch.autocast("cuda", torch.bfloat16):
        loss = m.loss(img, t)
    loss.backward()
    want = m.loss(img, t)
    assert abs(float(loss.detach() - want.detach())) <= 0.02 * float(want.detach())
    assert all(p.grad is None or p.grad.isfinite().all() and p.grad.dtype == p.dtype for p in m.parameters())


@gpu
@pytest.mark.parametrize("region", [torch.bfloat16, torch.float16])
def test_blocks_under_autocast_run_their_products_in_its_type(region):
    """The MLP of a block with checkpoints against the separate layers in the same region, fp32 parameters and input.  Four roundings
    to the type in a row on either side (the input's, the normalised one's, the hidden tensor's, the result's), 2^-8 of each at most; a
    region of a type without checkpoints (float16) is served by the separate layers."""
    torch.manual_seed(0)
    block = convnext1d.Block1D(64).cuda().train()
    x = torch.randn(2, 20, 20, 64, device="cuda", requires_grad=True)
    outs = []
    for block.keep8 in (False, True):
        with torch.autocast("cuda", region):
            y = block._mlp(x)
        params = [*block.norm.parameters(), *block.pwconv1.parameters(), *block.pwconv2.parameters()]
        outs.append((y.detach(), *torch.autograd.grad(y, [x, *params], torch.ones_like(y) / 8)))
    assert all(a.dtype == b.dtype and a.shape == b.shape for a, b in zip(*outs)) and outs[1][0].dtype == region
    if region == torch.float16:
        assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert float((outs[0][0] - outs[1][0]).float().norm()) <= 8 * 2.0 ** -8 * float(outs[0][0].float().norm())
    for a, b in zip(outs[0][1:], outs[1][1:]):                                 # 8-bit codes of normal data on top: 0.007 r.m.s.
        assert float((a - b).float().norm()) <= 0.05 * float(a.float().norm())


@gpu
@pytest.mark.parametrize("region", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_backward_pass_inside_autocast(dtype, region):
    """A region around the backward pass (or around both) changes nothing: the products' type is that of x."""
    leaves = mlp_args(64, 32, 128, dtype)
    x, g, b, w1, b1 = leaves[:5]
    dz = torch.randn(64, 32, device="cuda").to(DT[dtype])
    t = torch.arange(64, device="cuda")
    calls = [(lambda: ops.mlp_keep8(*leaves), leaves, dz), (lambda: ops.gelu_keep8(x, b), [x, b], dz), (lambda: ops.layer_norm_keep8(x, g, b), [x, g, b], dz),
             (lambda: ops.linear_cross_entropy(x, w1, t, b1), [x, w1, b1], torch.ones((), device="cuda"))]
    for f, ins, up in calls:
        want = torch.autograd.grad(f(), ins, up)
        y = f()
        with torch.autocast("cuda", region):
            got = torch.autograd.grad(y, ins, up)
            both = torch.autograd.grad(f(), ins, up)
        assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, got, both))


def test_the_loss_calls_a_head_that_is_more_than_a_linear():
    """Hooks on the head run, a pruned head is pruned anew, and a head that is another module is that module (on the CPU: those take torch's
    own operators)."""
    m = convnext1d.ConvNeXt1D(depths=(1, 1, 1, 1), dims=(8, 8, 8, 8), num_classes=5, stem_dim1=8)
    m.forward_features = lambda x: x
    x, t = torch.randn(6, 8, 3, 3), torch.tensor([0, 1, -100, 4, 4, 2])
    want = lambda: F.cross_entropy(m(x), t, label_smoothing=0.1)  # noqa: E731
    seen = []
    handle = m.head.register_forward_hook(lambda mod, i, o: seen.append(o.shape) or 2 * o)
    assert torch.equal(m.loss(x, t, label_smoothing=0.1), want()) and seen == [(6, 5), (6, 5)]
    handle.remove()
    torch.nn.utils.prune.l1_unstructured(m.head, "weight", 0.5)
    for _ in range(2):                                                         # its weight is a new tensor at every call
        m.loss(x, t).backward()
    assert torch.equal(m.loss(x, t, label_smoothing=0.1), want())
    assert (m.head.weight_orig.grad[m.head.weight_mask == 0] == 0).all()
    m.head = torch.nn.Sequential(torch.nn.Linear(8, 8), torch.nn.ReLU(), torch.nn.Linear(8, 5))
    assert torch.equal(m.loss(x, t, label_smoothing=0.1), want())
    m.head = torch.nn.Linear(8, 5)
    with pytest.raises(RuntimeError, match="CUDA"):                            # the plain head: ops.linear_cross_entropy
        m.loss(x, t)


@gpu
@pytest.mark.parametrize("keep8", [False, True])
def test_hooks_on_the_layers_of_a_block(keep8):
    block = convnext1d.Block1D(64).cuda().train()
    block.keep8 = keep8
    x = torch.randn(50, 64, device="cuda", requires_grad=True)
    for name in ("norm", "pwconv1", "pwconv2"):
        layer = getattr(block, name)
        seen = []
        handles = [layer.register_forward_pre_hook(lambda mod, i: seen.append("before")), layer.register_forward_hook(lambda mod, i, o: seen.append("after") or o * 0),
                   layer.register_full_backward_hook(lambda mod, i, o: seen.append("back"))]
        block._mlp(x).sum().backward()
        assert seen == ["before", "after", "back"], name
        for h in handles:
            h.remove()
    block.pwconv1 = torch.nn.Linear(64, 256, bias=False).cuda()                # a layer in its place that has no bias
    block._mlp(x).sum().backward()
    assert block.pwconv1.weight.grad is not None


@gpu
def test_nodes_of_the_graph():
    """What autograd does with any node: outputs changed in place, graphs kept and used up, inputs changed behind its back, saved
    tensors through hooks, hooks on inputs, no forward-mode derivative."""
    leaves = mlp_args(6, 32, 64, "fp32")
    x, g, b, w1, b1 = leaves[:5]
    t = torch.tensor([0, 5, 63, 1, 2, 3], device="cuda")
    calls = {"mlp": (lambda: ops.mlp_keep8(x.unsqueeze(0), *leaves[1:])[0], leaves),
             "gelu": (lambda: ops.gelu_keep8(x), [x]),
             "ln": (lambda: ops.layer_norm_keep8(x, g, b), [x, g, b]),
             "ce": (lambda: ops.linear_cross_entropy(x, w1, t, b1, reduction="none"), [x, w1, b1])}
    for name, (f, ins) in calls.items():
        y = f()
        up = torch.rand_like(y)
        want = torch.autograd.grad(y, ins, up, retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(y, ins, up)))
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, ins, up)
        y = f()
        y.add_(1).mul_(2)                                                      # before the backward pass
        assert all(torch.equal(2 * p, q) or torch.allclose(2 * p, q, rtol=1e-5, atol=1e-6) for p, q in zip(want, torch.autograd.grad(y, ins, up)))
        packed = []
        with torch.autograd.graph.saved_tensors_hooks(lambda v: packed.append(v.shape) or v.cpu(), lambda v: v.cuda()):
            y = f()
        assert packed and all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(y, ins, up)))
        seen = []
        handle = ins[0].register_hook(lambda v: seen.append(v.shape))
        f().backward(up)
        handle.remove()
        assert seen == [ins[0].shape] and torch.equal(ins[0].grad, want[0])
        for v in ins:
            v.grad = None
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
            ops.gelu_keep8(dual)
    y = ops.linear_cross_entropy(x, w1, t, b1)
    with torch.no_grad():
        w1.mul_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


@gpu
def test_no_rows_and_inference_mode():
    leaves = mlp_args(3, 32, 64, "fp32")
    empty = leaves[0].detach()[:0].requires_grad_(True)
    out = ops.mlp_keep8(empty, *leaves[1:])
    grads = torch.autograd.grad(out, [empty, *leaves[1:]], torch.zeros_like(out))
    assert out.shape == (0, 32) and grads[0].shape == (0, 32)
    assert all(g.shape == t.shape and not g.any() for g, t in zip(grads[1:], leaves[1:]))
    with torch.inference_mode():
        x, g, b, w1, b1 = (t.detach() for t in leaves[:5])
        t = torch.tensor([0, 5, 63], device="cuda")
        outs = [ops.mlp_keep8(*(v.detach() for v in leaves)), ops.gelu_keep8(x), ops.layer_norm_keep8(x, g, b), ops.linear_cross_entropy(x, w1, t, b1),
                *ops.keep8(x)]
    assert all(not o.requires_grad for o in outs) and torch.equal(outs[0], ops.mlp_keep8(*leaves).detach())


@gpu
def test_gradients_that_start_off_a_vector():
    leaves = mlp_args(30, 32, 64, "bf16")
    dz = torch.randn(30 * 32 + 1, device="cuda").bfloat16()
    out = ops.mlp_keep8(*leaves)
    a = torch.autograd.grad(out, leaves, dz[1:].view(30, 32), retain_graph=True)
    b = torch.autograd.grad(out, leaves, dz[1:].view(30, 32).clone())
    for p, q in zip(a, b):
        assert float((p - q).float().norm()) <= 2.0 ** -7 * float(q.float().norm())      # the library may pick another product


@gpu
def test_a_captured_training_step_repeats():
    m = small(True)
    img = torch.randn(2, 3, 64, 64, device="cuda")
    t = torch.tensor([1, 5], device="cuda")
    params = [p for p in m.parameters() if p.requires_grad]

    def step():
        loss = m.loss(img, t)
        return [loss.detach(), *[g for g in torch.autograd.grad(loss, params, allow_unused=True) if g is not None]]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, captured))


@gpu
def test_memory_between_the_passes():
    """A block's MLP keeps 1.06 bytes an element of x and of the hidden tensor: of 2 x (1 + 1 + 4 + 4) bytes, 5.3."""
    for keep8, least, most in ((False, 19.0, 21.0), (True, 5.0, 5.6)):
        block = convnext1d.Block1D(128).cuda().bfloat16().train()
        block.keep8 = keep8
        x = torch.randn(8, 56, 56, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        block._mlp(x * 1).sum().backward()                                     # the library's workspaces are there now
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = block._mlp(x * 1)                                                  # an input that only the block holds on to
        torch.cuda.synchronize()
        got = (torch.cuda.memory_allocated() - before - y.numel() * 2) / (x.numel())
        assert least <= got <= most, (keep8, got)
        del y


@gpu
def test_backbone_with_checkpoints():
    torch.manual_seed(0)
    m = backbone.ConvNeXt1DBackbone(depths=(1, 1, 1, 1), dims=(32, 64, 96, 128), stem_dim1=16, keep8=True).cuda().train()
    x = torch.randn(1, 3, 75, 90, device="cuda")
    with torch.no_grad():
        want = m(x)
    outs = m(x)
    assert all(float((a - b).norm()) <= 1e-5 * float(b.norm()) for a, b in zip(outs, want))
    sum(o.square().mean() for o in outs).backward()
    for k, p in m.stages.named_parameters():
        if not k.endswith("theta"):                                            # angles never receive a gradient
            assert p.grad is not None and p.grad.isfinite().all(), k


def test_refusals():
    with pytest.raises(ValueError, match="keep8"):
        convnext1d.ConvNeXt1D(variant="1dpp", depths=(1, 1, 1, 1), dims=(8, 8, 8, 8), keep8=True)
    t = torch.zeros
    ok = [t(4, 8), t(8), t(8), t(16, 8), t(16), t(8, 16), t(8)]
    for i, bad, what in ((1, t(7), "weight has"), (2, t(7), "bias has"), (3, t(16, 7), "weight1"), (4, t(15), "bias1"), (5, t(8, 15), "weight2"),
                         (6, t(9), "bias2")):
        with pytest.raises(ValueError, match=what):
            ops.mlp_keep8(*[bad if k == i else a for k, a in enumerate(ok)])
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        ops.mlp_keep8(ok[0].half(), *ok[1:])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.mlp_keep8(*ok)

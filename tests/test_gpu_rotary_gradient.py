"""Gradients of ops.rotary through autograd, and the version counters of what the paged calls write."""
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import dev, freqs, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("inverse", [False, True])
def test_gradient(ops, layout, inverse, dtype):  # noqa: F811
    """x.grad is the rotation back, of a gradient of any strides, for a leaf that is broadcast over heads too."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    pos, f = dev([0, 5, 1000, 70000, 3]), freqs(24)
    leaf = torch.randn(5, 1, 64, generator=gen, device="cuda").to(dtype).requires_grad_()
    y = ops.rotary(leaf.expand(5, 4, 64), pos, f.cuda(), layout=layout, factor=1.25, inverse=inverse)
    want = plain.rotate(leaf.detach().cpu().expand(5, 4, 64), pos.cpu(), f, layout, 1.25, inverse)
    assert bool(((y.detach().cpu().double() - want).abs() <= plain.rotate_bound(leaf.detach().cpu().expand(5, 4, 64), want, f, layout, 1.25)).all())
    g = torch.randn(5, 64, 4, generator=gen, device="cuda").to(dtype).transpose(1, 2)
    (seen,) = torch.autograd.grad(y, leaf, g, retain_graph=True)
    back = plain.rotate(g.cpu(), pos.cpu(), f, layout, 1.25, not inverse)
    each = plain.rotate_bound(g.cpu(), back, f, layout, 1.25)
    eps = torch.finfo(dtype).eps / 2
    total, size = back.sum(1, keepdim=True), (back.abs() + each).sum(1, keepdim=True)
    assert bool(((seen.cpu().double() - total).abs() <= each.sum(1, keepdim=True) + 4 * eps * size).all())     # (torch's sum of four: rounded four times at most)
    (again,) = torch.autograd.grad(y, leaf, g)
    assert torch.equal(seen, again)


def test_gradient_of_the_gradient(ops):  # noqa: F811
    """The rotation is linear: its gradient's gradient is the rotation."""
    pos, f = dev([9, 40]), freqs(16).cuda()
    x, g, h = (torch.randn(2, 3, 32, device="cuda").half() for _ in range(3))
    x.requires_grad_(), g.requires_grad_()
    (gx,) = torch.autograd.grad(ops.rotary(x, pos, f), x, g, create_graph=True)
    (gg,) = torch.autograd.grad(gx, g, h)
    assert torch.equal(gg, ops.rotary(h, pos, f))
    with torch.no_grad():
        assert not ops.rotary(x, pos, f).requires_grad


def test_results_to_be_written_carry_no_gradient(ops):  # noqa: F811
    from kvcomp_b200._lib import KvcError
    pos, f = dev([9, 40]), freqs(16).cuda()
    x = torch.randn(2, 3, 32, device="cuda").half().requires_grad_()
    with pytest.raises(KvcError):
        ops.rotary(x, pos, f, out=torch.empty_like(x))
    with torch.no_grad():
        out = torch.empty_like(x)
        assert ops.rotary(x, pos, f, out=out) is out


def test_versions(ops):  # noqa: F811
    """Tensors that a call writes in place are known to autograd as changed."""
    x, pos, f = torch.randn(2, 2, 64, device="cuda").half(), dev([1, 2]), freqs(32).cuda()
    kp, vp = (torch.zeros(3, 4, 2, 64, device="cuda").half() for _ in range(2))
    table, lengths, free, head, new = dev([[0, -1], [1, -1]]), dev([3, 4]), dev([0, 1, 2]), dev([2]), dev([1, 0])
    out, slots = torch.zeros_like(x), dev([3, 5])
    plan = ops.PagePlan(lengths, head, *torch.zeros(9, dtype=torch.int32, device="cuda").split((3, 2, 2, 2)))
    for call, written in ((lambda: ops.rotary(x, pos, f, out=out), (out,)), (lambda: ops.rotary_paged_store(x, x, x, pos, slots, f, kp, vp, out=out), (out, kp, vp)),
                          (lambda: ops.paged_attn(x, kp, vp, table, lengths, 0.1, out=out), (out,)),
                          (lambda: ops.page_plan(lengths, new, table, free, head, 4, 2, out=plan), (lengths, head, table, plan.slots, plan.positions, plan.taken, plan.starts)),
                          (lambda: ops.page_release(lengths, new > 0, table, free, head, 4, out=(lengths, head)), (lengths, head, free))):
        before = [t._version for t in written]
        call()
        assert all(t._version > n for t, n in zip(written, before))
    y = torch.randn(2, 2, 64, device="cuda").half().requires_grad_()
    z = (y * out).sum()
    ops.rotary(x, pos, f, out=out)
    with pytest.raises(RuntimeError):
        z.backward()
    with torch.inference_mode():
        kept = torch.zeros_like(x)
        ops.rotary(x, pos, f, out=kept)
        ops.rotary(x, pos, f, out=out)
    ops.rotary(x, pos, f, out=kept)


def test_captured(ops):  # noqa: F811
    """Forward and backward in a graph.  (No eager graph of the same leaf may live then: torch gives up such a capture of any operator, since it keeps the leaf's node on
    the stream that it was made on.)"""
    pos, f = dev([9, 40, 2]), freqs(32).cuda()
    x, g = (torch.randn(3, 2, 64, device="cuda").half() for _ in range(2))
    x.requires_grad_()
    torch.autograd.grad(ops.rotary(x, pos, f), x, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.rotary(x, pos, f)
        (gx,) = torch.autograd.grad(y, x, g)
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x)), g.copy_(torch.randn_like(g))
        pos += 5
        graph.replay()
        with torch.no_grad():
            assert torch.equal(y, ops.rotary(x, pos, f)) and torch.equal(gx, ops.rotary(g, pos, f, inverse=True))

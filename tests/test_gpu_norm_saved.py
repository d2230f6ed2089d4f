"""RMSNorm's backward pass on saved values that hooks keep elsewhere, that are recomputed or used twice, and on what it refuses of them."""
import pytest
import torch

from test_gpu_norm import make

pytestmark = pytest.mark.gpu


def given(cuda, T, H, dt, **k):
    leaves = [t.requires_grad_() for t in make(cuda, T, H, dt, **k)]
    g = torch.Generator(device=cuda)
    g.manual_seed(T)
    return leaves, [torch.randn((T, H), device=cuda, generator=g).to(t) for t in (dt, leaves[1].dtype)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_saved_values_elsewhere(cuda, wide, residual):
    """Kept in host memory, as copies that start at any address, recomputed (checkpoint), used twice (retain_graph), accumulated into
    .grad: the plain gradients' bits."""
    import torch.utils.checkpoint as C
    import bmx
    (x, res, w), (dy, dr) = given(cuda, 90, 136, torch.float16, x32=wide, w32=wide)
    norm = bmx.RMSNorm(w, dtype=torch.float16)
    leaves = [x, res, w] if residual else [x, w]
    run = (lambda: norm(x, res)) if residual else (lambda: (norm(x),))
    back = lambda outs, **k: torch.autograd.grad(outs, leaves, (dy, dr)[:len(outs)], **k)
    want = back(run())
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))

    def copy(t):
        c = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return c.copy_(t.detach())

    keep = lambda t: t
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), keep), torch.autograd.graph.saved_tensors_hooks(copy, keep),
                  torch.autograd.graph.saved_tensors_hooks(keep, keep), torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t.t().contiguous().t())):
        with hooks:
            outs = run()
        assert same(back(outs))
    for reentrant in (False, True):
        outs = C.checkpoint(norm, x, res, use_reentrant=reentrant) if residual else (C.checkpoint(norm, x, use_reentrant=reentrant),)
        torch.autograd.backward(outs, (dy, dr)[:len(outs)])
        assert same([t.grad for t in leaves])
        for t in leaves:
            t.grad = None
    outs = run()
    assert same(back(outs, retain_graph=True)) and same(back(outs))


def test_hooks_keep_the_forward_passes_values(cuda):
    """A weight whose data is replaced behind the forward pass is refused, unless a hook has kept what the forward pass had."""
    import bmx
    (x, res, w), (dy, _) = given(cuda, 5, 64, torch.bfloat16)
    norm = bmx.RMSNorm(w)
    want = torch.autograd.grad(norm(x, res)[0], [x, w], dy)
    y = norm(x, res)[0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t):
        z = norm(x, res)[0]
    held = w.data                                       # (so that the new one lies elsewhere)
    w.data = torch.ones_like(held) * 2
    with pytest.raises(RuntimeError, match="replaced"):
        torch.autograd.grad(y, [x, w], dy)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(z, [x, w], dy), want))
    assert bool((held != w.data).any())


def test_saved_values_in_another_form_are_refused(cuda):
    """What a hook gives back in another type, size or place never reaches the kernels."""
    import bmx
    (x, res, w), (dy, _) = given(cuda, 6, 64, torch.float16)
    norm = bmx.RMSNorm(w)
    for change in (lambda t: t.float(), lambda t: t[..., :32], lambda t: t[:3], lambda t: t.cpu(), lambda t: t[None]):
        for which in (1, 2):                            # the weight, then the rows
            unpack = lambda t, n=which: change(t) if t.dim() == n else t
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
                y = norm(x, res)[0]
            with pytest.raises(RuntimeError, match="saved"):
                torch.autograd.grad(y, [x, w], dy)

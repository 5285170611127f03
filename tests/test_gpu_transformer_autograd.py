"""GPU: the encoder-layer operators as autograd nodes: leaves that need no gradient, outputs nobody uses, graphs of gradients,
leaves changed before the backward, checkpoints, backward passes from several threads."""
import pytest
import torch

from tests._transformer_ref import poison

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _calls():
    from asr_amd.Models.transformer_ops import bucket_attention, gated_feed_forward, qk_norm_rope
    g = torch.Generator().manual_seed(3)

    def n(*shape):
        return torch.randn(*shape, generator=g).to(DEV)
    return {"rope": (lambda q, k, a, b: qk_norm_rope(q, k, a, b, rot_dim=16), [n(2, 50, 4, 32), n(2, 50, 2, 32), n(32), n(32)]),
            "attention": (lambda q, k, v, t: (bucket_attention(q, k, v, t, lengths=torch.tensor([50, 31], device=DEV)),),
                          [n(2, 50, 4, 32), n(2, 50, 2, 32), n(2, 50, 2, 32), n(32, 4)]),
            "ff": (lambda x, a, b, c: (gated_feed_forward(x, a, b, c),), [n(2, 35, 24), n(40, 24), n(40, 24), n(24, 40)])}


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
def test_any_subset_of_the_leaves(name):
    fn, args = _calls()[name]
    full = [t.clone().requires_grad_() for t in args]
    out = fn(*full)
    up = [torch.randn(o.shape, generator=torch.Generator().manual_seed(i)).to(DEV) for i, o in enumerate(out)]
    want = torch.autograd.grad(out, full, up, retain_graph=True)
    again = torch.autograd.grad(out, full, up)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    with pytest.raises(RuntimeError):                         # the graph is gone
        torch.autograd.grad(out, full, up)
    for mask in range(1, 16):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(args)]
        poison()
        got = fn(*leaves)
        assert all(o.requires_grad for o in got)
        grads = torch.autograd.grad(got, [t for t in leaves if t.requires_grad], up)
        for a, b in zip(grads, [w for i, w in enumerate(want) if mask >> i & 1]):
            assert torch.equal(a, b), mask
    for i in range(4):                                        # all leaves, the gradient of one
        leaves = [t.clone().requires_grad_() for t in args]
        assert torch.equal(torch.autograd.grad(fn(*leaves), leaves[i], up)[0], want[i])
    assert not any(o.requires_grad for o in fn(*args))
    with torch.no_grad():
        assert not any(o.requires_grad for o in fn(*full))


def test_an_output_nobody_uses():
    fn, args = _calls()["rope"]
    leaves = [t.clone().requires_grad_() for t in args]
    q, k = fn(*leaves)
    up = torch.ones_like(k)
    got = torch.autograd.grad(k, leaves, up)
    both = fn(*leaves)
    want = torch.autograd.grad(both, leaves, [torch.zeros_like(q), up])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[0].any() and got[1].any()


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
def test_gradients_of_gradients_raise(name):
    fn, args = _calls()[name]
    leaves = [t.clone().requires_grad_() for t in args]
    out = fn(*leaves)
    up = [torch.ones_like(o).requires_grad_() for o in out]
    grads = torch.autograd.grad(out, leaves, up, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        grads[0].sum().backward()


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
def test_leaves_changed_before_the_backward_raise(name):
    fn, args = _calls()[name]
    leaves = [t.clone().requires_grad_() for t in args]
    out = fn(*leaves)
    with torch.no_grad():
        leaves[1].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
def test_recomputed_by_a_checkpoint(name):
    from torch.utils.checkpoint import checkpoint
    fn, args = _calls()[name]
    a, b = ([t.clone().requires_grad_() for t in args] for _ in range(2))
    ya, yb = fn(*a), checkpoint(fn, *b, use_reentrant=False)
    up = [torch.ones_like(o) for o in ya]
    for x, y in zip(torch.autograd.grad(ya, a, up), torch.autograd.grad(yb, b, up)):
        assert torch.equal(x, y)


def test_backward_from_two_threads():
    import threading
    calls = _calls()
    want, got = {}, {}

    def work(name, out):
        fn, args = calls[name]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                leaves = [t.clone().requires_grad_() for t in args]
                y = fn(*leaves)
                out[name] = torch.autograd.grad(y, leaves, [torch.ones_like(o) for o in y])
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    for name in calls:
        work(name, want)
    threads = [threading.Thread(target=work, args=(name, got)) for name in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for name in calls:
        assert all(torch.equal(a, b) for a, b in zip(want[name], got[name])), name

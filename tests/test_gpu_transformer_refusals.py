"""GPU: calls of the encoder-layer operators that have no right answer and must say so."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("H,Hk", [(0, 2), (2, 0)])
@pytest.mark.parametrize("train", [False, True])
def test_norm_and_rotation_of_one_side_without_heads(H, Hk, train):
    from asr_amd.Models.transformer_ops import qk_norm_rope
    q, k, w = (torch.ones(s, device=DEV).requires_grad_(train) for s in ((1, 3, H, 8), (1, 3, Hk, 8), (8,)))
    with pytest.raises(RuntimeError, match="do not match"):
        qk_norm_rope(q, k, w, w)


def test_norm_and_rotation_of_nothing():
    from asr_amd.Models.transformer_ops import qk_norm_rope
    for shape in ((1, 3, 0, 8), (0, 3, 2, 8), (1, 0, 2, 8)):
        q, k = (torch.ones(shape, device=DEV).requires_grad_() for _ in range(2))
        w = torch.ones(8, device=DEV).requires_grad_()
        y = qk_norm_rope(q, k, w, w)
        assert all(o.shape == q.shape for o in y)
        assert not torch.autograd.grad(y, w, [torch.ones_like(o) for o in y])[0].any()


def _calls():
    from asr_amd.Models.transformer_ops import bucket_attention, gated_feed_forward, qk_norm_rope
    g = torch.Generator().manual_seed(3)

    def n(*shape):
        return torch.randn(*shape, generator=g).to(DEV)
    return {"rope": (lambda q, k, a, b: qk_norm_rope(q, k, a, b, rot_dim=16), [n(2, 50, 4, 32), n(2, 50, 2, 32), n(32), n(32)]),
            "attention": (lambda q, k, v, t: (bucket_attention(q, k, v, t),), [n(2, 50, 4, 32), n(2, 50, 2, 32), n(2, 50, 2, 32), n(32, 4)]),
            "ff": (lambda x, a, b, c: (gated_feed_forward(x, a, b, c),), [n(2, 35, 24), n(40, 24), n(40, 24), n(24, 40)])}


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
@pytest.mark.parametrize("leaf", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_raise(name, leaf, grad):
    import torch.autograd.forward_ad as fwd
    fn, args = _calls()[name]
    args = [t.requires_grad_(grad) for t in args]
    with fwd.dual_level():
        duals = list(args)
        duals[leaf] = fwd.make_dual(args[leaf], torch.ones_like(args[leaf]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            fn(*duals)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            fn(*duals)
        fn(*args)                                             # no tangent among them


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
@pytest.mark.parametrize("grad", [False, True])
def test_traces_raise(name, grad):
    fn, args = _calls()[name]
    args = tuple(t.requires_grad_(grad) for t in args)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(fn, args, check_trace=False)
    fn(*args)


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
def test_a_second_derivative_raises_and_is_never_left_out(name):
    """Also where the upstream gradient is a constant: the gradients depend on the inputs all the same."""
    fn, args = _calls()[name]
    leaves = [t.requires_grad_() for t in args]
    out = fn(*leaves)
    grads = torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out], create_graph=True)
    assert all(g.requires_grad for g in grads)
    for i in range(4):
        with pytest.raises(RuntimeError, match="twice"):
            torch.autograd.grad((grads[i] ** 2).sum() + (leaves[0] ** 2).sum(), leaves, retain_graph=True, allow_unused=True)
        for leaf in leaves:                                   # with respect to one input, through any
            with pytest.raises(RuntimeError, match="twice"):
                torch.autograd.grad((grads[i] ** 2).sum() + (leaf ** 2).sum(), leaf, retain_graph=True)
    # as numbers they are the gradients, and what does not go through them has its second derivatives
    plain = torch.autograd.grad(fn(*leaves), leaves, [torch.ones_like(o) for o in out])
    assert all(torch.equal(a, b) and not b.requires_grad for a, b in zip(grads, plain))
    total = sum((o * o).sum() for o in fn(*leaves)) + (leaves[0] ** 3).sum()
    total.backward(create_graph=True)
    assert all(t.grad is not None for t in leaves)
    for t in leaves:
        t.grad = None

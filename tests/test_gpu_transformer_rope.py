"""GPU: qk_norm_rope against its definition in float64: element types, head layouts, widths that fill no vector, partial
rotation, strides, far positions, single frames, gradients (the formula's and by differences)."""
import pytest
import torch

from tests._transformer_ref import poison, rope64, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# forward: the sum of squares (<= 16 terms in a lane, 6 steps across lanes), its root and quotient, two products, the angle's
# float32 tail and the rotation's product pair stay below 64 roundings of the row's largest normed element; backward: two
# such sums and their products, below 160 roundings of the terms of dx
FWD_TERMS, BWD_TERMS = 64, 160


def _case(B, T, H, Hk, D, dtype, seed=0, packed=False):
    g = torch.Generator().manual_seed(seed)
    if packed:
        p = torch.randn(B, T, (H + 2 * Hk) * D, generator=g).to(dtype).to(DEV)
        q, k = p[..., :H * D].unflatten(-1, (H, D)), p[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))
    else:
        q, k = (torch.randn(B, T, h, D, generator=g).to(dtype).to(DEV) for h in (H, Hk))
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(DEV) for _ in range(2)]
    gr = [torch.randn(B, T, h, D, generator=g).to(dtype).to(DEV) for h in (H, Hk)]
    return q, k, w, gr


def _check(q, k, w, gr, pos, rot, base=10000.0, eps=1e-6):
    from asr_amd.Models.transformer_ops import qk_norm_rope
    poison()
    T = q.shape[1]
    p64 = pos if pos is not None else torch.arange(T, device=q.device)
    leaves = [t.detach().requires_grad_() for t in (q, k, *w)]
    out = qk_norm_rope(*leaves, positions=pos, rot_dim=rot, base=base, eps=eps)
    grads = torch.autograd.grad(out, leaves, gr)
    with torch.no_grad():
        again = qk_norm_rope(q, k, *w, positions=pos, rot_dim=rot, base=base, eps=eps)
    for x, xw, o, o2, g, dx, dw in zip((q, k), w, out, again, gr, grads[:2], grads[2:]):
        assert torch.equal(o, o2) and o.is_contiguous() and o.dtype == x.dtype
        x64, w64 = x.detach().double().requires_grad_(), xw.detach().double().requires_grad_()
        y64 = rope64(x64, w64, p64, rot, base, eps)
        dx64, dw64 = torch.autograd.grad(y64, (x64, w64), g.double())
        r = torch.rsqrt((x64 * x64).mean(-1, keepdim=True) + eps).detach()
        xh = x64.detach() * r
        within(o.detach(), y64.detach(), 2 * (xh * w64.detach()).abs().amax(-1, keepdim=True), FWD_TERMS)
        gw = 2 * g.double().abs().amax(-1, keepdim=True) * w64.detach().abs().max()
        within(dx, dx64, r * gw * (1 + xh.abs().amax(-1, keepdim=True)), BWD_TERMS)
        terms = 2 * g.double().abs().amax(-1, keepdim=True) * xh.abs()
        within(dw, dw64, terms.sum((0, 1, 2)), FWD_TERMS)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("B,T,H,Hk,D,rot", [
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 4, 64, 64), (3, 33, 6, 3, 80, 40), (2, 17, 2, 1, 38, 18), (1, 5, 3, 3, 128, 128),
    (2, 9, 1, 1, 126, 2), (1, 40, 16, 2, 128, 64), (2, 11, 5, 5, 24, 0), (8, 1, 8, 2, 64, 64), (1, 700, 12, 4, 96, 96)])
def test_shapes_and_types(B, T, H, Hk, D, rot, dtype):
    q, k, w, gr = _case(B, T, H, Hk, D, dtype)
    _check(q, k, w, gr, None, rot)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_views_of_a_packed_projection_and_other_strides(dtype):
    q, k, w, gr = _case(3, 19, 4, 2, 64, dtype, packed=True)
    assert not q.is_contiguous()
    _check(q, k, w, gr, None, 64)
    q, k, w, gr = _case(3, 19, 4, 2, 64, dtype)
    _check(q.transpose(1, 2).contiguous().transpose(1, 2), k, w, [g.transpose(1, 2).contiguous().transpose(1, 2) for g in gr],
           None, 64)
    _check(q.transpose(2, 3).contiguous().transpose(2, 3), k, w, gr, None, 64)               # heads not contiguous
    _check(q[:, :1].expand(-1, 19, -1, -1), k, w, [gr[0], gr[1][:, :, :1].expand(-1, -1, 2, -1)], None, 64)
    # a view that starts off the 16-byte grid
    big = torch.randn(3 * 19 * 4 * 64 + 1, device=DEV).to(dtype)
    _check(big[1:].view(3, 19, 4, 64), k, w, gr, None, 64)


@pytest.mark.parametrize("start", [0, 1000003, -7, 2 ** 33])
def test_far_positions(start):
    q, k, w, gr = _case(2, 5, 2, 2, 64, torch.float32)
    pos = start + torch.arange(5, device=DEV) + torch.tensor([[0], [12345]], device=DEV)
    _check(q, k, w, gr, pos, 64)
    _check(q, k, w, gr, pos[0], 64, base=500.0)
    if start < 2 ** 31:
        _check(q, k, w, gr, pos.int(), 64)


def test_rows_of_zeros_and_large_values():
    q, k, w, gr = _case(2, 6, 2, 2, 64, torch.float32)
    q[0, 1] = 0
    q[1, 2] *= 1e15
    k[0, 3] *= 1e-12
    _check(q, k, w, gr, None, 64)


def test_gradient_by_differences():
    from asr_amd.Models.transformer_ops import qk_norm_rope
    q, k, w, gr = _case(1, 7, 2, 1, 32, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (q, k, *w)]
    out = qk_norm_rope(*leaves, rot_dim=16)
    grads = torch.autograd.grad(out, leaves, gr)
    f = lambda ts: sum((o.double() * g.double()).sum() for o, g in zip(qk_norm_rope(*ts, rot_dim=16), gr))  # noqa: E731
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        d = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(5)).to(DEV)
        h = 2.0 ** -6
        with torch.no_grad():
            ts = [t.detach() for t in leaves]
            up = f([t + h * d if j == i else t for j, t in enumerate(ts)])
            dn = f([t - h * d if j == i else t for j, t in enumerate(ts)])
        want = (grad.double() * d.double()).sum()
        # a central difference is off by h^2 f''' / 6; the norm's third derivative along d is of order |d|^3
        assert abs(float((up - dn) / (2 * h) - want)) < 2e-2 * float(grad.double().norm() * d.double().norm())


def test_empty_batches():
    from asr_amd.Models.transformer_ops import qk_norm_rope
    for B, T in ((0, 3), (2, 0)):
        q, k, w, gr = _case(B, T, 2, 1, 16, torch.float32)
        leaves = [t.detach().requires_grad_() for t in (q, k, *w)]
        out = qk_norm_rope(*leaves)
        assert out[0].shape == q.shape and out[1].shape == k.shape
        grads = torch.autograd.grad(out, leaves, gr)
        assert not grads[2].any() and not grads[3].any()


def test_another_stream_and_a_captured_graph():
    from asr_amd.Models.transformer_ops import qk_norm_rope
    q, k, w, _ = _case(4, 50, 4, 2, 64, torch.bfloat16)
    want = qk_norm_rope(q, k, *w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = qk_norm_rope(q, k, *w)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rep = qk_norm_rope(q, k, *w)
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(n)).to(q.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(rep, qk_norm_rope(q, k, *w)))


def test_refusals():
    from asr_amd.Models.transformer_ops import qk_norm_rope
    q, k, w, _ = _case(2, 3, 2, 1, 16, torch.float32)
    for bad in ((q.cpu(), k, *w), (q.double(), k.double(), *w), (q, k.half(), *w), (q[0], k, *w), (q, k[:, :2], *w),
                (q, k, w[0][:8], w[1]), (q, k, w[0].half(), w[1]), (q[..., :15], k[..., :15], w[0][:15], w[1][:15]),
                (q, k[..., :8], *w)):
        with pytest.raises(RuntimeError):
            qk_norm_rope(*bad)
    for kw in (dict(rot_dim=3), dict(rot_dim=18), dict(rot_dim=-2), dict(base=0.0), dict(eps=-1.0), dict(eps=float("nan")),
               dict(positions=torch.arange(3)), dict(positions=torch.arange(2, device=DEV)),
               dict(positions=torch.zeros(3, device=DEV))):
        with pytest.raises(RuntimeError):
            qk_norm_rope(q, k, *w, **kw)
    big = torch.zeros(1, 1, 1, 130, device=DEV)
    with pytest.raises(RuntimeError):
        qk_norm_rope(big, big, torch.ones(130, device=DEV), torch.ones(130, device=DEV))

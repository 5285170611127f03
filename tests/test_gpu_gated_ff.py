"""GPU: gated_feed_forward against its definition in float64: element types, sizes around the tiles, padded and unpadded
widths, few rows, gradients (the formula's and by differences), streams, captured graphs, refusals."""
import pytest
import torch

from tests._transformer_ref import gated_ff64, held, poison

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(M, d, f, n, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x, dy = (scale * torch.randn(M, w, generator=g) for w in (d, n))
    wg, wu, wd = (torch.randn(*s, generator=g) * s[1] ** -0.5 for s in ((f, d), (f, d), (n, f)))
    return [t.to(dtype).to(DEV) for t in (x, wg, wu, wd, dy)]


def _check(x, wg, wu, wd, dy, act="swish"):
    from asr_amd.Models.transformer_ops import gated_feed_forward
    poison()
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves, act=act)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        plain = gated_feed_forward(x, wg, wu, wd, act=act)
    d64 = [t.detach().double().reshape(-1, t.shape[-1]) for t in (x, wg, wu, wd, dy)]
    want = gated_ff64(*d64, act, x.dtype)
    flat = lambda t: t.detach().reshape(-1, t.shape[-1])  # noqa: E731
    held(flat(plain), want[0])
    for got, w in zip((y, *grads), want):
        held(flat(got), w)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,d,f,n", [
    (1, 1, 1, 1), (5, 3, 7, 2), (16, 64, 64, 64), (17, 40, 96, 24), (64, 128, 192, 64), (65, 64, 64, 64), (129, 200, 683, 200),
    (128, 256, 128, 256), (200, 33, 65, 130), (300, 256, 320, 128), (1003, 64, 128, 64)])
def test_shapes_and_types(M, d, f, n, dtype):
    _check(*_inputs(M, d, f, n, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gelu(dtype):
    _check(*_inputs(70, 64, 100, 64, dtype, scale=3.0), act="gelu")
    _check(*_inputs(7, 64, 100, 64, dtype, scale=3.0), act="gelu")


@pytest.mark.parametrize("M,d,f,n", [(2060, 40, 2041, 33), (4000, 64, 2048, 64), (4100, 40, 2041, 33), (2100, 200, 1500, 72), (8200, 64, 1030, 64)])
def test_tiles_of_every_width(M, d, f, n):
    """16-bit products of enough tiles for the widest, with ragged last ones."""
    _check(*_inputs(M, d, f, n, torch.bfloat16))
    _check(*_inputs(M, d, f, n, torch.float16))


@pytest.mark.parametrize("M,d,f", [(70, 64, 96), (300, 64, 96), (2100, 256, 1024)])         # the last one as it lies in the backward too
@pytest.mark.parametrize("xs,ws,ds,gs", [(60.0, 1.0, 1e-3, 1.0), (200.0, 4.0, 1e-4, 1e-4), (1e-6, 1.0, 1.0, 1e-6), (1.0, 1e-3, 1.0, 3e-7), (0.0, 1.0, 1.0, 1.0),
                                         (1.0, 1.0, 0.0, 1.0), (1.0, 1.0, 1.0, 0.0), (1.0, 100.0, 1e-3, 50.0)])
def test_float16_hidden_values_out_of_its_range(M, d, f, xs, ws, ds, gs):
    """h, da and db far above the largest float16 and below its normal numbers, where y and gradients may be neither."""
    x, wg, wu, wd, dy = _inputs(M, d, f, 40, torch.float32)
    _check(*[(t.float() * s).to(torch.float16) for t, s in ((x, xs), (wg, ws), (wu, ws), (wd, ds), (dy, gs))])


def test_float16_rows_with_infinities_leave_the_others():
    from asr_amd.Models.transformer_ops import gated_feed_forward
    x, wg, wu, wd, _ = _inputs(130, 64, 96, 40, torch.float16)
    want = gated_feed_forward(x, wg, wu, wd)
    bad = x.clone()
    bad[3, 5], bad[77, 0], bad[129, 63] = float("inf"), float("nan"), -float("inf")
    got = gated_feed_forward(bad, wg, wu, wd)
    rest = torch.ones(130, dtype=torch.bool, device=x.device)
    rest[[3, 77, 129]] = False
    close = (got[rest].float() - want[rest].float()).abs() <= 2.0 ** -10 * want[rest].float().abs() + 2.0 ** -9 * float(want.abs().max())
    assert bool(close.all()) and not got[~rest].isfinite().any()


def test_many_tiles_and_split_sums():
    _check(*_inputs(3000, 128, 256, 128, torch.bfloat16))
    _check(*_inputs(2100, 64, 192, 96, torch.float32))


def test_large_and_small_values():
    """Saturated activations, and float16 gradients far below what float16 products would hold."""
    x, wg, wu, wd, dy = _inputs(90, 64, 96, 64, torch.float32)
    _check(x * 40, wg, wu, wd, dy)
    x, wg, wu, wd, dy = _inputs(90, 64, 96, 64, torch.float16)
    _check(x, wg, wu, wd, dy * 2.0 ** -12)
    _check(x * 8, wg * 8, wu * 8, wd, dy)


def test_layouts():
    from asr_amd.Models.transformer_ops import gated_feed_forward
    x, wg, wu, wd, dy = _inputs(90, 64, 96, 64, torch.bfloat16)
    _check(x.view(3, 30, 64), wg, wu, wd, dy.view(3, 30, 64))
    _check(x.t().contiguous().t(), wg.t().contiguous().t(), wu, wd, dy.t().contiguous().t())
    both = torch.cat([wg, wu])
    _check(x, both[:96], both[96:], wd, dy)
    buf = torch.empty(90 * 64 + 1, device=DEV, dtype=torch.bfloat16)       # off the 16-byte grid
    off = buf[1:].view(90, 64).copy_(x)
    _check(off, wg, wu, wd, dy)
    with torch.no_grad():
        assert torch.equal(gated_feed_forward(off[:8], wg, wu, wd), gated_feed_forward(x[:8], wg, wu, wd))
    # one weight used twice: both gradients arrive
    w = wg.detach().requires_grad_()
    y = gated_feed_forward(x, w, w, wd)
    g, = torch.autograd.grad(y, w, dy)
    want = gated_ff64(*[t.double() for t in (x, wg, wg, wd, dy)], "swish", torch.bfloat16)
    held(g, (want[2][0] + want[3][0], want[2][1] + want[3][1] + 2.0 ** -8 * (want[2][0] + want[3][0]).abs()))


def test_gradient_by_differences():
    from asr_amd.Models.transformer_ops import gated_feed_forward
    ts = _inputs(70, 24, 40, 16, torch.float32)
    leaves = [t.detach().requires_grad_() for t in ts[:4]]
    grads = torch.autograd.grad(gated_feed_forward(*leaves), leaves, ts[4])
    for i, grad in enumerate(grads):
        d = torch.randn(ts[i].shape, generator=torch.Generator().manual_seed(3)).to(DEV)
        d = d / d.norm()
        h = 2.0 ** -5
        with torch.no_grad():
            up, dn = (sum((gated_feed_forward(*[t + s * h * d if j == i else t for j, t in enumerate(ts[:4])]).double()
                           * ts[4].double()).flatten()) for s in (1, -1))
        # h^2 / 6 of a third derivative of the order of the gradient itself along a unit direction
        assert abs(float((up - dn) / (2 * h) - (grad.double() * d.double()).sum())) < 4e-3 * float(grad.double().norm())


def test_only_what_is_asked_for():
    from asr_amd.Models.transformer_ops import gated_feed_forward
    x, wg, wu, wd, dy = _inputs(70, 64, 64, 64, torch.float32)
    full = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
    want = torch.autograd.grad(gated_feed_forward(*full), full, dy)
    for keep in ([0], [1], [3], [2, 0]):
        leaves = [t.detach().requires_grad_(i in keep) for i, t in enumerate((x, wg, wu, wd))]
        got = torch.autograd.grad(gated_feed_forward(*leaves), [leaves[i] for i in keep], dy)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, keep))


def test_no_rows():
    from asr_amd.Models.transformer_ops import gated_feed_forward
    x, wg, wu, wd, _ = _inputs(4, 64, 64, 32, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x[:0], wg, wu, wd)]
    y = gated_feed_forward(*leaves)
    assert y.shape == (0, 32)
    assert not any(g.any() for g in torch.autograd.grad(y.sum(), leaves))


@pytest.mark.parametrize("M", [8, 200])
def test_another_stream_and_captured_graphs(M):
    from asr_amd.Models.transformer_ops import gated_feed_forward
    x, wg, wu, wd, _ = _inputs(M, 64, 128, 64, torch.float32)
    want = gated_feed_forward(x, wg, wu, wd)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gated_feed_forward(x, wg, wu, wd)
    s.synchronize()
    assert torch.equal(got, want)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(gated_feed_forward(x, wg, wu, wd))
    for n in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(n)))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = gated_feed_forward(x, wg, wu, wd)
        assert all(torch.equal(o, want) for o in outs)


def test_refusals():
    from asr_amd.Models.transformer_ops import gated_feed_forward
    x, wg, wu, wd, _ = _inputs(4, 16, 24, 16, torch.float32)
    for bad in ((x.cpu(), wg, wu, wd), (x.half(), wg, wu, wd), (x.double(), wg.double(), wu.double(), wd.double()),
                (x[:, :8], wg, wu, wd), (x, wg[:8], wu, wd), (x, wg, wu, wd[:, :8]), (x, wg, wu, wd.half()),
                (x, wg[0], wu[0], wd), (x, wg[:0], wu[:0], wd[:, :0])):
        with pytest.raises(RuntimeError):
            gated_feed_forward(*bad)
    with pytest.raises(RuntimeError):
        gated_feed_forward(x, wg, wu, wd, act="tanh")

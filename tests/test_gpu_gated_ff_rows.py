"""GPU: gated_feed_forward with rows and weights of very different sizes: no row's result may depend on another row's size."""
import pytest
import torch

from tests._transformer_ref import gated_ff64, held, poison

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inputs(M, d, f, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, dy = (torch.randn(M, w, generator=g) for w in (d, n))
    wg, wu, wd = (torch.randn(*s, generator=g) * s[1] ** -0.5 for s in ((f, d), (f, d), (n, f)))
    return x, wg, wu, wd, dy


def _by_groups(x, wg, wu, wd, dy, groups, act):
    """gated_ff64 of each group of rows by itself, so that no tolerance knows another group's size: y and dx by rows, the
    weights' gradients and their tolerances added up.  (A group's sum over its own rows leaves out (M - M_g) 2^-24 of the terms'
    sizes for a sum over all M of them; at M <= 2100 that is 2^-13, and what h, da and db are kept in, 2^-16, leaves as much of the
    2^-11 that the tolerance has for it.)"""
    M = x.shape[0]
    rows = [[torch.zeros(M, w, device=x.device, dtype=torch.float64) for _ in range(2)] for w in (wd.shape[0], x.shape[1])]
    sums = [[torch.zeros_like(w) for _ in range(2)] for w in (wg, wu, wd)]
    for at in groups:
        y, dx, *dw = gated_ff64(x[at], wg, wu, wd, dy[at], act, torch.float16)
        for to, got in ((rows[0], y), (rows[1], dx)):
            to[0][at], to[1][at] = got
        for to, got in zip(sums, dw):
            to[0] += got[0]
            to[1] += got[1]
    return [tuple(t) for t in (*rows, *sums)]


def _check(x, wg, wu, wd, dy, groups, act="swish"):
    from asr_amd.Models.transformer_ops import gated_feed_forward
    ts = [t.to(torch.float16).to(DEV) for t in (x, wg, wu, wd, dy)]
    assert all(bool(t.isfinite().all()) for t in ts)
    want = _by_groups(*[t.double() for t in ts], groups, act)
    poison()
    leaves = [t.detach().requires_grad_() for t in ts[:4]]
    y = gated_feed_forward(*leaves, act=act)
    for got, w in zip((y.detach(), *torch.autograd.grad(y, leaves, ts[4])), want):
        held(got, w)
    with torch.no_grad():
        held(gated_feed_forward(*ts[:4], act=act), want[0])
        few = torch.cat([gated_feed_forward(t, *ts[1:4], act=act) for t in ts[0].split(64)])      # the form for up to 64 rows
    held(few, want[0])


SIZES = [(66, 64, 96, 40), (600, 200, 683, 72), (2100, 256, 1024, 256)]


def _one_and_the_rest(M, at):
    rest = torch.ones(M, dtype=torch.bool, device=DEV)
    rest[at] = False
    return [~rest, rest]


@pytest.mark.parametrize("M,d,f,n", SIZES)
@pytest.mark.parametrize("times", [100.0, 1000.0, 8000.0])
@pytest.mark.parametrize("act", ["swish", "gelu"])
def test_one_large_row_of_x(M, d, f, n, times, act):
    x, wg, wu, wd, dy = _inputs(M, d, f, n)
    x[17] *= times
    _check(x, wg, wu, wd * 2.0 ** -6, dy * 2.0 ** -4, _one_and_the_rest(M, 17), act)


@pytest.mark.parametrize("M,d,f,n", SIZES)
@pytest.mark.parametrize("xs,gs", [(100.0, 1e5), (100.0, 1e6), (1.0, 1e7)])
def test_one_large_row_of_the_gradient(M, d, f, n, xs, gs):
    x, wg, wu, wd, dy = _inputs(M, d, f, n, seed=1)
    x[M - 1] *= xs
    dy = dy * 2.0 ** -12
    dy[M - 1] *= gs
    _check(x * 2.0 ** -4, wg, wu, wd, dy, _one_and_the_rest(M, M - 1))


@pytest.mark.parametrize("M,d,f,n", SIZES)
def test_rows_of_many_sizes(M, d, f, n):
    x, wg, wu, wd, dy = _inputs(M, d, f, n, seed=2)
    k = torch.arange(M)
    x *= (2.0 ** (k % 14 - 8))[:, None]
    dy *= (2.0 ** (k * 5 % 11 - 6))[:, None]
    kinds = (k % 14 * 11 + k * 5 % 11).to(DEV)
    _check(x, wg, wu, wd, dy, [kinds == c for c in kinds.unique()])


@pytest.mark.parametrize("M,d,f,n", SIZES)
def test_one_large_hidden_unit_that_the_output_leaves_out(M, d, f, n):
    """Weight rows far larger than the others' whose hidden unit counts for nothing."""
    x, wg, wu, wd, dy = _inputs(M, d, f, n, seed=3)
    wg[5] *= 1000
    wu[5] *= 1000
    wd[:, 5] = 0
    x, dy = x * 2.0 ** -3, dy
    ts = [t.to(torch.float16).to(DEV) for t in (x, wg, wu, wd, dy)]
    from asr_amd.Models.transformer_ops import gated_feed_forward
    got = gated_feed_forward(*ts[:4])
    # the same sum without the unit: its own products are zeros
    rest = torch.arange(f, device=DEV) != 5
    held(got, gated_ff64(*[t.double() for t in (ts[0], ts[1][rest], ts[2][rest], ts[3][:, rest])], None, "swish", torch.float16)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M", [20, 130, 600])
def test_rows_with_infinities_leave_the_others_as_they_were(M, dtype):
    from asr_amd.Models.transformer_ops import gated_feed_forward
    x, wg, wu, wd, dy = (t.to(dtype).to(DEV) for t in _inputs(M, 64, 96, 40))
    bad_x, bad_dy = x.clone(), dy.clone()
    bad_x[3, 5], bad_x[7, 0], bad_x[M - 1, 63], bad_dy[11, 2] = float("inf"), float("nan"), -float("inf"), float("nan")
    rest = torch.ones(M, dtype=torch.bool, device=DEV)
    rest[[3, 7, 11, M - 1]] = False

    def run(a, g):
        a = a.detach().requires_grad_()
        y = gated_feed_forward(a, wg, wu, wd)
        return y.detach(), torch.autograd.grad(y, a, g)[0]
    for want, got in zip(run(x, dy), run(bad_x, bad_dy)):
        assert torch.equal(got[rest], want[rest])

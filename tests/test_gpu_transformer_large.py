"""GPU: the encoder-layer operators on tensors whose element offsets pass 32 bits: views with large strides give the bits of their
compact copies, and results at the far end of large outputs are those of the same rows alone."""
import pytest
import torch

from tests._transformer_ref import attention64, gated_ff64, held

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 * 2 ** 30:
        pytest.skip("needs 100 GB of free device memory")
    yield
    torch.cuda.empty_cache()


def _spread(t, axis, step):
    """A view equal to t whose stride along `axis` is `step` elements."""
    n = t.shape[axis]
    inner = t.select(axis, 0).contiguous()
    flat = torch.empty((n - 1) * step + inner.numel(), device=DEV, dtype=t.dtype)
    strides = list(inner.stride())
    strides.insert(axis, step)
    view = flat.as_strided(t.shape, strides)
    view.copy_(t)
    return view


def _rand(*shape, seed=0, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize("axis,step", [(0, 2 ** 30 + 64), (1, 2 ** 25 + 128)])
@pytest.mark.parametrize("Tq", [1, 70])
def test_attention_of_views_with_large_strides(axis, step, Tq):
    from asr_amd.Models.transformer_ops import bucket_attention
    q, k, v, up = _rand(3, Tq, 4, 64), _rand(3, 70, 2, 64, seed=1), _rand(3, 70, 2, 64, seed=2), _rand(3, Tq, 4, 64, seed=3)
    t = _rand(32, 4, seed=4, dtype=torch.float32)
    off = torch.full((3,), 70 - Tq, device=DEV)
    kv = [_spread(x, axis, step) for x in (k, v)]
    far = [_spread(q, axis, step) if Tq > 1 or axis == 0 else q, *kv]
    assert torch.equal(bucket_attention(*far, t, offset=off, causal=True), bucket_attention(q, k, v, t, offset=off, causal=True))
    leaves = [[x.detach().requires_grad_() for x in xs] for xs in ((*far, t), (q, k, v, t))]
    (ya, a), (yb, b) = ((y, torch.autograd.grad(y, x, up)) for x in leaves for y in [bucket_attention(*x, offset=off, causal=True)])
    assert torch.equal(ya, yb) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_norm_and_rotation_of_views_with_large_strides():
    from asr_amd.Models.transformer_ops import qk_norm_rope
    q, k = _rand(3, 50, 4, 64), _rand(3, 50, 2, 64, seed=1)
    w = [_rand(64, seed=s, dtype=torch.float32) for s in (2, 3)]
    up = [_rand(3, 50, 4, 64, seed=4), _rand(3, 50, 2, 64, seed=5)]

    def run(x, y, g):
        leaves = [t.detach().requires_grad_() for t in (x, y, *w)]
        out = qk_norm_rope(*leaves)
        return (*out, *torch.autograd.grad(out, leaves, g))
    want = run(q, k, up)
    for got in (run(_spread(q, 0, 2 ** 30 + 64), _spread(k, 1, 2 ** 26), up), run(q, k, [_spread(up[0], 1, 2 ** 26), _spread(up[1], 0, 2 ** 30 + 64)])):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_with_more_than_2_31_outputs():
    from asr_amd.Models.transformer_ops import bucket_attention
    T, H, D, n = 2 ** 20 + 90, 16, 128, 77
    q = torch.zeros(1, T, H, D, device=DEV, dtype=BF16)
    up = torch.zeros_like(q)
    q[:, -n:], up[:, -n:] = _rand(1, n, H, D), _rand(1, n, H, D, seed=1)
    k, v, t = _rand(1, 40, 2, D, seed=2), _rand(1, 40, 2, D, seed=3), _rand(32, H, seed=4, dtype=torch.float32)
    off = torch.tensor([30 - T], device=DEV)                          # the last rows are the ones next to the keys
    leaves = [x.detach().requires_grad_() for x in (q, k, v, t)]
    y = bucket_attention(*leaves, offset=off)
    grads = torch.autograd.grad(y, leaves, up)
    want = attention64(q[:, -n:].double(), k.double(), v.double(), t.double(), up[:, -n:].double(), BF16, train=True, lengths=None, keep=None,
                       offset=torch.tensor([30 - n], device=DEV), causal=False, reach=128, scale=D ** -0.5)
    held(y.detach()[:, -n:], want[0])
    held(grads[0][:, -n:], want[1])
    for g, w in zip(grads[1:], want[2:]):
        held(g, w)
    with torch.no_grad():
        assert torch.isfinite(bucket_attention(q, k, v, t, offset=off)[:, ::4099]).all()


@pytest.mark.parametrize("dtype", [BF16, torch.float16], ids=str)
def test_feed_forward_with_more_than_2_31_hidden_values(dtype):
    from asr_amd.Models.transformer_ops import gated_feed_forward
    M, d, f, n = 2 ** 19 + 300, 64, 4160, 201
    x = torch.zeros(M, d, device=DEV, dtype=dtype)
    dy = torch.zeros_like(x)
    x[-n:], dy[-n:] = _rand(n, d, dtype=dtype), _rand(n, d, seed=1, dtype=dtype)
    w = [(_rand(*s, seed=i, dtype=torch.float32) * s[1] ** -0.5).to(dtype) for i, s in ((2, (f, d)), (3, (f, d)), (4, (d, f)))]
    leaves = [t.detach().requires_grad_() for t in (x, *w)]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    want = gated_ff64(*(t.double() for t in (x[-n:], *w, dy[-n:])), "swish", dtype)
    held(y.detach()[-n:], want[0])
    held(grads[0][-n:], want[1])
    for g, v in zip(grads[1:], want[2:]):
        held(g, v)

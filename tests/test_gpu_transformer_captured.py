"""GPU: forward and backward of the encoder-layer operators captured into one HIP graph and replayed on new inputs, with eager
work of the program's own between the replays."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _n(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _calls():
    from asr_amd.Models.transformer_ops import bucket_attention, gated_feed_forward, qk_norm_rope
    n = torch.tensor([150, 31], device=DEV, dtype=torch.int32)
    attn = lambda reach: lambda q, k, v, t: (bucket_attention(q, k, v, t, lengths=n, causal=True, max_distance=reach),)  # noqa: E731
    qkv = lambda D, dt: [_n(2, 150, h, D, dtype=dt, seed=h) for h in (4, 2, 2)]  # noqa: E731
    ff = lambda x, a, b, c: (gated_feed_forward(x, a, b, c),)  # noqa: E731
    sizes = ((300, 96), (136, 96), (136, 96), (96, 136))
    return {"rope": (lambda q, k, a, b: qk_norm_rope(q, k, a, b), [_n(2, 150, 4, 64), _n(2, 150, 2, 64), _n(64), _n(64)]),
            "attention": (attn(128), [*qkv(64, torch.bfloat16), _n(32, 4)]),
            "attention, much LDS": (attn(1024), [*qkv(128, torch.float32), _n(32, 4)]),        # beyond 64 KB a workgroup
            "ff float16": (ff, [_n(*s, dtype=torch.float16, seed=i) * 0.1 for i, s in enumerate(sizes)]),
            "ff float32": (ff, [_n(*s, seed=i) * 0.1 for i, s in enumerate(sizes)])}


@pytest.mark.parametrize("name", ["rope", "attention", "attention, much LDS", "ff float16", "ff float32"])
def test_a_captured_training_call(name):
    fn, args = _calls()[name]

    def step(leaves, up):
        out = fn(*leaves)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, up))
    leaves = [t.clone().requires_grad_() for t in args]
    up = [torch.ones_like(o) for o in fn(*args)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step(leaves, up)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            got.append(step(leaves, up))
    for seed in range(4):
        with torch.no_grad():
            for i, t in enumerate(leaves + up):
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * seed + i)) * (0.1 if name.startswith("ff") else 1.0))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step([t.detach().clone().requires_grad_() for t in leaves], up)
        for outs in got:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), seed
        torch.cuda.synchronize()

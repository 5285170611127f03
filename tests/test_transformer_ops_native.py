"""CPU: what the native module of the encoder-layer operators refuses before it looks for a GPU."""
import pytest
import torch


def _native():
    from asr_amd import _lib
    return _lib.native()


@pytest.mark.parametrize("H,Hk", [(0, 2), (2, 0)])
def test_norm_and_rotation_of_one_side_without_heads(H, Hk):
    """The other side must not come back as memory that nobody wrote."""
    q, k, w = torch.ones(1, 3, H, 8), torch.ones(1, 3, Hk, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="both or none"):
        _native().rope_fwd(q, k, w, w, None, 8, 1e4, 1e-6)
    with pytest.raises(RuntimeError, match="both or none"):
        _native().rope_bwd(q, k, w, w, None, 8, 1e4, 1e-6, q, k)


@pytest.mark.parametrize("shape", [(1, 3, 0, 8), (0, 3, 2, 8), (1, 0, 2, 8)])
def test_norm_and_rotation_of_nothing(shape):
    q, w = torch.ones(shape), torch.ones(8)
    for out in _native().rope_fwd(q, q, w, w, None, 8, 1e4, 1e-6):
        assert out.shape == q.shape
    dq, dk, dwq, dwk = _native().rope_bwd(q, q, w, w, None, 8, 1e4, 1e-6, q, q)
    assert dq.shape == dk.shape == q.shape and not dwq.any() and not dwk.any()


def _calls():
    """The three operators as their Python functions call them, on tensors that no GPU holds."""
    m, n = _native(), torch.randn
    return {"rope": (lambda q, k, a, b: m.rope(q, k, a, b, None, 8, 1e4, 1e-6), [n(1, 3, 2, 8), n(1, 3, 1, 8), n(8), n(8)]),
            "attention": (lambda q, k, v, t: m.attention(q, k, v, t, None, None, None, 0, True, 1.0), [n(1, 3, 2, 8), n(1, 3, 1, 8), n(1, 3, 1, 8), n(2, 2)]),
            "ff": (lambda x, a, b, c: m.ff(x, a, b, c, 0), [n(3, 8), n(4, 8), n(4, 8), n(8, 4)])}


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
@pytest.mark.parametrize("leaf", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_raise(name, leaf, grad):
    """A tangent that no kernel carries on must not vanish, whether or not the call is a node of a graph."""
    import torch.autograd.forward_ad as fwd
    fn, args = _calls()[name]
    args = [t.requires_grad_(grad) for t in args]
    with fwd.dual_level():
        args[leaf] = fwd.make_dual(args[leaf], torch.ones_like(args[leaf]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            fn(*args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            fn(*args)


@pytest.mark.parametrize("name", ["rope", "attention", "ff"])
@pytest.mark.parametrize("grad", [False, True])
def test_traces_raise(name, grad):
    """A trace would hold the outputs' allocation and no kernel."""
    fn, args = _calls()[name]
    args = tuple(t.requires_grad_(grad) for t in args)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(fn, args, check_trace=False)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_long_utterances_do_not_take_the_form_for_few_queries(dtype):
    """Told by the workspace: float32 partial rows of the split form, or the planes of the other one."""
    import ctypes as C
    from asr_amd import _lib
    edges = (C.c_int32 * 7)(12, 16, 23, 32, 46, 64, 91)

    def few(T, H):
        a = _lib.BucketAttentionArgs()
        a.edges_host = C.addressof(edges)
        a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, a.nb, a.dtype, a.scale = 1, T, T, H, H, 64, 32, dtype, 1.0
        # (the pointers' addresses are on the 16-byte grid, strides zero: bfloat16 is an operand as it lies)
        n = _lib.load().asr_bucket_attention_ws_bytes(C.byref(a), 0)
        planes = {0: 3, 1: 0, 2: 2}[dtype] * 2 * 64 * 3 * H * T
        return n != planes
    assert few(374, 4) and few(1500, 4) and few(4096, 4) and few(8192, 1)
    for T, H in ((8192, 4), (16384, 4), (32768, 4), (32768, 1), (16384, 2), (1 << 20, 1)):
        assert not few(T, H), (T, H)

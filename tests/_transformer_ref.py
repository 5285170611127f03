"""Float64 definitions of the encoder-layer operators (asr_amd/Models/transformer_ops.py), used by their tests."""
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of each type
U32 = U[torch.float32]


def rope64(x, w, pos, rot, base, eps):
    """x (B,T,H,D) float64; pos (T,) or (B,T)."""
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=x.device) / max(rot, 1))
    t = pos.double()[..., None] * f
    t = (t if t.dim() == 3 else t[None])[:, :, None]
    a, b = n[..., :rot // 2], n[..., rot // 2:rot]
    return torch.cat([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin(), n[..., rot:]], -1)


def within(got, want, scale, terms):
    """|got - want| <= u(type) |want| + terms u(float32) scale, element by element (scale broadcasts): the rounding of the
    stored type plus `terms` float32 roundings of quantities no larger than `scale`."""
    assert got.shape == want.shape, (got.shape, want.shape)
    err = (got.double() - want).abs()
    tol = U[got.dtype] * want.abs() + terms * U32 * scale
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25                       # half a step of the subnormals
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol.clamp(min=1e-300)).max()), float(err.max()))

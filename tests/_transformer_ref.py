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


def act64(a, kind):
    if kind == "swish":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    c = 0.5 * (1 + torch.erf(a * 0.5 ** 0.5))
    return a * c, c + a * torch.exp(-0.5 * a * a) * (2 * torch.pi) ** -0.5


def gated_ff64(x, wg, wu, wd, dy, kind, dtype):
    """Float64 block and gradients with their tolerances: a list of (value, tolerance).

    u_h: half step of what h, da and db are kept in between the products; drop: what the products leave out of a term
    (pieces.h: 2^-24 for each of two dropped products and for the rest behind three pieces, one dropped product of two
    halves of at most 2^-8 for two pieces); every sum of n terms in float32 is off by at most n u of the sum of its terms'
    sizes."""
    u = U[dtype]
    u_h, drop = {torch.float32: (2.0 ** -24, 3 * 2.0 ** -24), torch.bfloat16: (2.0 ** -8, 0.0),
                 torch.float16: (2.0 ** -16, 2.0 ** -16)}[dtype]
    d, f, n, M = x.shape[1], wg.shape[0], wd.shape[0], x.shape[0]
    a, b = x @ wg.t(), x @ wu.t()
    ea, eb = ((d * U32 + drop) * (x.abs() @ w.abs().t()) for w in (wg, wu))
    act, slope = act64(a, kind)
    h = act * b
    own = 16 * U32                                        # exp, reciprocal or erf and the products around them
    slope_max = 1.13                                      # the largest slope of either activation; of the slope, 1.0
    eact, eslope = slope_max * ea + own * (act.abs() + a.abs() * slope.abs()), ea + own * (1 + a.abs())
    eh = eact * b.abs() + act.abs() * eb + eact * eb + (u_h + U32) * h.abs()
    y = h @ wd.t()
    out = [(y, eh @ wd.abs().t() + (f * U32 + drop) * (h.abs() @ wd.abs().t()))]
    if dy is not None:
        dh = dy @ wd
        edh = (n * U32 + drop) * (dy.abs() @ wd.abs())
        da, db = dh * b * slope, dh * act
        eda = (edh * (b * slope).abs() + eb * (dh * slope).abs() + eslope * (dh * b).abs()) * 1.01 + (u_h + 4 * U32) * da.abs()
        edb = (edh * act.abs() + eact * dh.abs()) * 1.01 + (u_h + 2 * U32) * db.abs()
        s = M * U32 + drop
        out.append((da @ wg + db @ wu, eda @ wg.abs() + edb @ wu.abs()
                    + (2 * f * U32 + drop) * (da.abs() @ wg.abs() + db.abs() @ wu.abs())))
        out.append((da.t() @ x, eda.t() @ x.abs() + s * (da.abs().t() @ x.abs())))
        out.append((db.t() @ x, edb.t() @ x.abs() + s * (db.abs().t() @ x.abs())))
        out.append((dy.t() @ h, dy.abs().t() @ eh + s * (dy.abs().t() @ h.abs())))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return [(v, t + u * (v.abs() + t) + tiny) for v, t in out]


def held(got, want):
    v, tol = want
    assert got.shape == v.shape, (got.shape, v.shape)
    err = (got.double() - v).abs()
    # a value beyond the type's largest one rounds to infinity (float16: from 65520 on, the largest plus half a step)
    top = torch.finfo(got.dtype).max * (1 + U[got.dtype] / 2)
    over = torch.isinf(got) & (got.sign().double() == v.sign()) & (v.abs() + tol >= top)
    err = torch.where(over, 0.0, err)
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol.clamp(min=1e-300)).max()), float(err.max()))
    return float((err / tol.clamp(min=1e-300)).max())

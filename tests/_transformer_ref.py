"""Float64 definitions of the encoder-layer operators (asr_amd/Models/transformer_ops.py), used by their tests."""
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of each type
U32 = U[torch.float32]


def poison():
    """Fill what the caching allocator hands out next with NaN: a kernel that reads workspace nobody wrote shows it."""
    sizes = [1 << 26] + 4 * [1 << 20] + 6 * [1 << 18] + 8 * [1 << 16] + 8 * [1 << 13]
    keep = [torch.full((n // 4,), float("nan"), device="cuda:0") for n in sizes]
    del keep


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
    (pieces.h: 2^-24 for each of two dropped products and for the rest behind three pieces; up to 64 rows without gradients
    float16 has two pieces, one dropped product of two halves of at most 2^-8); every sum of n terms in float32 is off by at
    most n u of the sum of its terms' sizes.  float16 h, da and db are kept times a power of two that brings a bound on them
    above 2^14: a value below the normal numbers is off by half of 2^-24, 2^-39 of the bound."""
    u = U[dtype]
    u_h, drop = {torch.float32: (2.0 ** -24, 3 * 2.0 ** -24), torch.bfloat16: (2.0 ** -8, 0.0),
                 torch.float16: (2.0 ** -11, 2.0 ** -16)}[dtype]
    d, f, n, M = x.shape[1], wg.shape[0], wd.shape[0], x.shape[0]
    a, b = x @ wg.t(), x @ wu.t()
    ea, eb = ((d * U32 + drop) * (x.abs() @ w.abs().t()) for w in (wg, wu))
    act, slope = act64(a, kind)
    h = act * b
    low = 2.0 ** -39 if dtype == torch.float16 else 0.0
    norm_x, norm_g, norm_u = (t.norm(dim=1).max() for t in (x, wg, wu))
    own = 16 * U32                                        # exp, reciprocal or erf and the products around them
    slope_max = 1.13                                      # the largest slope of either activation; of the slope, 1.0
    eact, eslope = slope_max * ea + own * (act.abs() + a.abs() * slope.abs()), ea + own * (1 + a.abs())
    eh = eact * b.abs() + act.abs() * eb + eact * eb + (u_h + U32) * h.abs() + low * norm_x ** 2 * norm_g * norm_u
    y = h @ wd.t()
    out = [(y, eh @ wd.abs().t() + (f * U32 + drop) * (h.abs() @ wd.abs().t()))]
    if dy is not None:
        dh = dy @ wd
        edh = (n * U32 + drop) * (dy.abs() @ wd.abs())
        da, db = dh * b * slope, dh * act
        low = low * 1.13 * dy.norm(dim=1).max() * wd.norm(dim=0).max() * norm_x * torch.maximum(norm_g, norm_u)
        eda = (edh * (b * slope).abs() + eb * (dh * slope).abs() + eslope * (dh * b).abs()) * 1.01 + (u_h + 4 * U32) * da.abs() + low
        edb = (edh * act.abs() + eact * dh.abs()) * 1.01 + (u_h + 2 * U32) * db.abs() + low
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


def bucket64(r, nb, reach, causal):
    """Bucket of each distance r (int64), by the definition, in whole numbers."""
    n = nb if causal else nb // 2
    first, steps = n // 2, n - n // 2

    def one(x):
        away = max(-x, 0) if causal else abs(x)
        k = away
        if away >= first:
            k = first
            while k < n - 1 and away ** steps * first ** (k - first + 1) >= reach ** (k - first + 1) * first ** steps:
                k += 1
        return k + (0 if causal or x <= 0 else n)
    lo, hi = int(r.min()), int(r.max())
    line = torch.tensor([one(x) for x in range(lo, hi + 1)], device=r.device)
    return line[r - lo]


def attention64(q, k, v, table, g, dtype, *, lengths, keep, offset, causal, reach, scale, train):
    """Float64 attention and gradients with tolerances: [(value, tolerance)] for out, dq, dk, dv, dtable.

    drop / u_p: what the products leave out of a term and the half step of the probabilities and score gradients between two
    products, by type (pieces.h; bfloat16 probabilities carry at least 16 bits in training's forward).  A score's absolute error es (its product,
    the bias and scale in base 2) makes a relative error es of its probability; one exponential, the sum's roundings and
    the quotient add `own`."""
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    drop, u_p, u_ds = {torch.float32: (3 * 2.0 ** -24, 2.0 ** -24, 2.0 ** -24), torch.float16: (2.0 ** -16, 2.0 ** -16, 2.0 ** -16),
                       torch.bfloat16: (0.0, 2.0 ** -16 if train else 2.0 ** -8, 2.0 ** -8)}[dtype]
    qq, gg = q.transpose(1, 2), None if g is None else g.transpose(1, 2)
    j = torch.arange(Tk, device=q.device)
    pos = torch.arange(Tq, device=q.device)[None] + (0 if offset is None else offset.long()[:, None])
    r = j - pos[..., None]                                               # (B or 1, Tq, Tk)
    slot = bucket64(r, table.shape[0], reach, causal)
    ok = torch.ones(B, 1, Tq, Tk, dtype=torch.bool, device=q.device)
    if lengths is not None:
        ok = ok & (j < lengths[:, None])[:, None, None]
    if keep is not None:
        ok = ok & keep.bool()[:, None, None]
    if causal:
        ok = ok & (r <= 0)[:, None]
    seen = ok.any(2).squeeze(1)                                          # keys that no query may read hold anything
    kk, vv = (torch.where(seen[:, :, None, None], t, 0.0).transpose(1, 2).repeat_interleave(G, 1) for t in (k, v))
    bias = table[slot].movedim(-1, 1)
    s = torch.where(ok, qq @ kk.transpose(-1, -2) * scale + bias, -torch.inf)
    size = (qq.abs() @ kk.abs().transpose(-1, -2)) * abs(scale)
    es = (D * U32 + drop) * size + 6 * U32 * (size + bias.abs() + 1) + 4 * U32 * torch.where(ok, s.abs(), 0.0)
    es = torch.where(ok, es, 0.0)
    top = torch.where(ok.any(-1, keepdim=True), s.amax(-1, keepdim=True), 0.0)
    es = es + 4 * U32 * (top.abs() + torch.where(ok, (s - top).abs(), 0.0))   # differences from the running maximum
    e = torch.exp(s - top) * ok
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    own = (Tk / 16 + 16) * U32
    # float32 holds nothing below 2^-126 and the running maximum may lag by 2^8: a smaller probability becomes zero
    ep = p * (es + (p * es).sum(-1, keepdim=True) + own) + 2.0 ** -118 * ok
    out = p @ vv
    eo = (ep + u_p * p) @ vv.abs() + (Tk * U32 + drop) * (p @ vv.abs())
    res = [(out.transpose(1, 2), eo.transpose(1, 2))]
    if gg is not None:
        dp = gg @ vv.transpose(-1, -2)
        edp = (D * U32 + drop) * (gg.abs() @ vv.abs().transpose(-1, -2))
        delta = (gg * out).sum(-1, keepdim=True)
        edelta = (gg.abs() * (eo + U32 * out.abs())).sum(-1, keepdim=True) + D * U32 * (gg * out).abs().sum(-1, keepdim=True)
        ds = p * (dp - delta)
        eds = ep * (dp - delta).abs() + p * (edp + edelta) + 4 * U32 * p * (dp.abs() + delta.abs())
        back = lambda t: t.unflatten(1, (Hk, G)).sum(2).transpose(1, 2)  # noqa: E731
        pt, dst, eph, edsh = (t.transpose(-1, -2) for t in (p, ds, ep + u_p * p if dtype != torch.bfloat16 else ep + 2.0 ** -8 * p,
                                                            eds + u_ds * ds.abs()))
        res.append(((ds @ kk * scale).transpose(1, 2),
                    ((edsh.transpose(-1, -2) + (Tk * U32 + drop) * ds.abs()) @ kk.abs() * abs(scale)).transpose(1, 2)))
        res.append((back(dst @ qq * scale), back((edsh + (G * Tq * U32 + drop) * dst.abs()) @ qq.abs() * abs(scale))))
        res.append((back(pt @ gg), back((eph + (G * Tq * U32 + drop) * pt) @ gg.abs())))
        dt, et = torch.zeros_like(table), torch.zeros_like(table)
        slot = slot.expand(B, Tq, Tk).reshape(-1)
        n = B * Tq * min(Tk, 4 * reach)
        dt.index_add_(0, slot, ds.movedim(1, -1).reshape(-1, H))
        et.index_add_(0, slot, (eds + min(n, 4096) * U32 * ds.abs()).movedim(1, -1).reshape(-1, H))
        res.append((dt, et))
    u = U[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return [(a, t + (u if i < 4 else U32) * (a.abs() + t) + (tiny if i < 4 else 0.0)) for i, (a, t) in enumerate(res)]

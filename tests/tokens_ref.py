"""The layers of token models in 64 bits, from their formulas, on whatever device the tensors are. Every function returns
pairs (value, M): M is the sum of the magnitudes of the terms that make up the value, the scale of its rounding errors.

Tolerances. U is half the distance of neighbouring 32-bit floats, relative: one rounding of a value x is off by at most
U |x|. A sum of L terms that are rounded one after the other is off by at most L U M; the roundings of a long sum are not
aligned, so the tests ask for (16 + 4 sqrt(L)) U M, where 16 covers the roundings of a term itself (at most ten products,
differences and conversions) and of the epilogue.
"""
import torch

U = 2.0 ** -24


def sum_tol(L):
    return (16 + 4 * L ** 0.5) * U


def d(t):
    return None if t is None else t.double()


def check(name, got, pair, tol, floor=1e-37):
    """|got - value| <= tol * M everywhere; tol may be a tensor."""
    ref, M = pair
    assert tuple(got.shape) == tuple(ref.shape), (name, got.shape, ref.shape)
    if ref.numel() == 0:
        return
    err, lim = (got.double() - ref).abs(), tol * M + floor
    assert bool(torch.isfinite(got).all()), f"{name}: non-finite values"
    worst = (err / lim).max().item()
    assert worst <= 1.0, f"{name}: error is {worst:.2f} times the tolerance (largest error {err.max().item():.3e})"


def ln_fwd(mw, vw, mb, vb, ma, va, eps):
    mw, vw, mb, vb, ma, va = map(d, (mw, vw, mb, vb, ma, va))
    n = ma.shape[1]
    m = ma.mean(1, keepdim=True)
    v = ((ma - m).square().sum(1, keepdim=True) + va.sum(1, keepdim=True)) / (n - 1)
    i = (v + eps).rsqrt()
    t = ma - m
    z, vz = i * t * mw, i * i * (va * (mw * mw + vw) + vw * t * t)
    # rounding: the mean is a sum of n terms in at most 64 + n/1024 dependent additions; it enters t, v only in second order
    L = 64 + n / 1024
    em = L * ma.abs().mean(1, keepdim=True)
    Mz = em * (i * mw).abs() + (L / 2 + 10) * z.abs()
    Mv = (L + 16) * vz + 2 * i * i * vw * t.abs() * em
    Mr = (L + 6) * v.squeeze(1) + U * em.squeeze(1).square()
    if mb is not None:
        z, vz = z + mb, vz + vb
        Mz, Mv = Mz + 2 * mb.abs() + z.abs(), Mv + 2 * vb + vz
    return (z, Mz), (vz, Mv), (m.squeeze(1), em.squeeze(1)), (v.squeeze(1), Mr)   # the M here carry their factors: tol = U


def ln_bwd(mw, vw, vb, ma, jcb, m, v, dm, dv, eps):
    mw, vw, vb, ma, jcb, m, v, dm, dv = map(d, (mw, vw, vb, ma, jcb, m, v, dm, dv))
    i = (v[:, None] + eps).rsqrt()
    t = i * mw * (1.0 if jcb is None else jcb)
    u = i * (ma - m[:, None]) * vw
    out = [t * dm, t * t * dv, (u * dm).sum(0), (u * u * dv).sum(0)]
    M = [x.abs() for x in out[:2]] + [(u * dm).abs().sum(0), (u * u * dv).abs().sum(0)]
    if vb is not None:
        out += [vb * dm.sum(0), vb * vb * dv.sum(0)]
        M += [vb * dm.abs().sum(0), vb * vb * dv.abs().sum(0)]
    return list(zip(out, M))


def softmax_jacobian(g):
    """J[t, i, j] = g_i ((i == j) - g_j), with 1 - g_i as the sum of the others."""
    eye = torch.eye(g.shape[1], dtype=torch.bool, device=g.device)
    rest = torch.where(eye, 0.0, g[:, None, :].expand(*g.shape, g.shape[1])).sum(2)
    return torch.where(eye, (g * rest)[:, :, None], -g[:, :, None] * g[:, None, :])


def route_fwd(ms, vs, k):
    """(expert, (mu_g, M), (var_g, M), offsets, token, pos)."""
    T, E = ms.shape
    s = torch.where(torch.isnan(ms), -torch.inf, ms.double())
    score, idx = torch.sort(s, dim=1, descending=True, stable=True)
    score, idx = score[:, :k], idx[:, :k]
    ok = score > -torch.inf
    top = score[:, :1]
    gap = torch.where(ok & (score != top), score - top, 0.0)
    p = torch.where(ok, gap.exp(), 0.0)
    g = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    v = torch.where(ok, torch.gather(vs.double(), 1, idx), 0.0) if vs is not None else torch.zeros_like(g)
    var_g = (softmax_jacobian(g).square() * v[:, None, :]).sum(2)
    # a gate: exp of a difference that was rounded once (U |gap|, relative, once it is in the exponent), exp itself (two
    # units in the last place), at most k + 5 additions, a division
    gap = torch.where(torch.isfinite(gap), gap.abs(), 0.0).amax(1, keepdim=True)
    rel = 16 + 2 * gap + 2 * k
    expert = torch.where(ok, idx, -1)
    flat = torch.where(ok, idx, E).reshape(-1)
    order = torch.argsort(flat, stable=True)
    live = int((flat < E).sum())
    offsets = torch.cat([flat.new_zeros(1), torch.bincount(flat, minlength=E + 1)[:E].cumsum(0)])
    token = torch.full((T * k,), -1, dtype=torch.int64, device=ms.device)
    token[:live] = order[:live] // k
    pos = torch.full((T * k,), -1, dtype=torch.int64, device=ms.device)
    pos[order[:live]] = torch.arange(live, device=ms.device)
    return expert, (g, rel * g), (var_g, 4 * rel * var_g), offsets, token, pos.reshape(T, k)


def route_bwd(expert, g, dg, vg, E):
    has = expert >= 0
    g, dg, vg = (torch.where(has, x.double(), 0.0) for x in (g, dg, vg))
    J = softmax_jacobian(g)
    dm, dv = (J * dg[:, :, None]).sum(1), (J.square() * vg[:, :, None]).sum(1)
    Mm, Mv = (J.abs() * dg.abs()[:, :, None]).sum(1), (J.square() * vg.abs()[:, :, None]).sum(1)
    # the kernel forms g_j sum g_i (d_j - d_i): its terms are those of J
    T, k = expert.shape
    full = [torch.zeros(T, E, dtype=torch.float64, device=g.device) for _ in range(4)]
    t = torch.arange(T, device=g.device)[:, None].expand(T, k)
    for f, x in zip(full, (dm, Mm, dv, Mv)):
        f[t[has], expert.long()[has]] = x[has]
    return (full[0], full[1]), (full[2], full[3])


def _spans(offsets, S):
    o = [min(max(int(x), 0), S) for x in offsets.tolist()]
    return [(o[e], max(o[e], o[e + 1])) for e in range(len(o) - 1)]


def _gather(x, token):
    if token is None:
        return x
    t = token.long()
    ok = (t >= 0) & (t < x.shape[0])
    return torch.where(ok[:, None], x[t.clamp(0, max(0, x.shape[0] - 1))], 0.0)


def grouped_fwd(mw, vw, mb, vb, ma, va, offsets, token):
    mw, vw, mb, vb = map(d, (mw, vw, mb, vb))
    S, N = (ma.shape[0] if token is None else token.numel()), mw.shape[1]
    a, v = _gather(ma.double(), token), _gather(va.double(), token)
    z, Mz, vz = (torch.zeros(S, N, dtype=torch.float64, device=ma.device) for _ in range(3))
    for e, (r0, r1) in enumerate(_spans(offsets, S)):
        r = slice(r0, r1)
        z[r], Mz[r] = a[r] @ mw[e].t(), a[r].abs() @ mw[e].abs().t()
        vz[r] = v[r] @ (mw[e].square() + vw[e]).t() + a[r].square() @ vw[e].t()
        if mb is not None:
            z[r], vz[r], Mz[r] = z[r] + mb[e], vz[r] + vb[e], Mz[r] + mb[e].abs()
    return (z, Mz), (vz, vz)


def grouped_state(mw, jcb, dm, dv, offsets):
    mw, jcb, dm, dv = map(d, (mw, jcb, dm, dv))
    S = dm.shape[0]
    o = [torch.zeros(S, mw.shape[2], dtype=torch.float64, device=dm.device) for _ in range(4)]
    for e, (r0, r1) in enumerate(_spans(offsets, S)):
        r = slice(r0, r1)
        w = mw[e]
        o[0][r], o[1][r] = dm[r] @ w, dm[r].abs() @ w.abs()
        o[2][r], o[3][r] = dv[r] @ w.square(), dv[r].abs() @ w.square()
    if jcb is not None:
        o = [o[0] * jcb, o[1] * jcb.abs(), o[2] * jcb * jcb, o[3] * jcb * jcb]
    return (o[0], o[1]), (o[2], o[3])


def grouped_param(vw, vb, ma, dm, dv, offsets, token):
    vw, vb, dm, dv = map(d, (vw, vb, dm, dv))
    a = _gather(ma.double(), token)
    w = [torch.zeros_like(vw) for _ in range(4)]
    b = [torch.zeros(vw.shape[:2], dtype=torch.float64, device=dm.device) for _ in range(4)]
    for e, (r0, r1) in enumerate(_spans(offsets, dm.shape[0])):
        r = slice(r0, r1)
        w[0][e], w[1][e] = dm[r].t() @ a[r], dm[r].abs().t() @ a[r].abs()
        w[2][e], w[3][e] = dv[r].t() @ a[r].square(), dv[r].abs().t() @ a[r].square()
        b[0][e], b[1][e], b[2][e], b[3][e] = dm[r].sum(0), dm[r].abs().sum(0), dv[r].sum(0), dv[r].abs().sum(0)
    out = [(vw * w[0], vw * w[1]), (vw * vw * w[2], vw * vw * w[3])]
    if vb is not None:
        out += [(vb * b[0], vb * b[1]), (vb * vb * b[2], vb * vb * b[3])]
    return out


def _slots(pos, S):
    ok = (pos >= 0) & (pos < S)
    return ok, torch.where(ok, pos, 0).long()


def _taken(x, pos):
    ok, p = _slots(pos, x.shape[0])
    if x.shape[0] == 0:
        return torch.zeros(*pos.shape, x.shape[1], dtype=torch.float64, device=x.device)
    return torch.where(ok[:, :, None], x.double()[p], 0.0)


def combine_fwd(pos, g, vg, mx, vx):
    x, v = _taken(mx, pos), _taken(vx, pos)
    g, vg = g.double()[:, :, None], vg.double()[:, :, None]
    y, vy = (g * x).sum(1), (vg * (x * x + v) + g * g * v).sum(1)
    return (y, (g * x).abs().sum(1)), (vy, vy.abs())


def combine_bwd(pos, g, mx, jcb, dm, dv):
    """dmu_x, dvar_x (rows that no slot names: NaN), dmu_g, dvar_g."""
    S, N = mx.shape
    ok, p = _slots(pos, S)
    t = torch.arange(pos.shape[0], device=pos.device)[:, None].expand_as(pos)
    dx = torch.full((S, N), torch.nan, dtype=torch.float64, device=mx.device)
    vx = dx.clone()
    j = torch.ones_like(dx) if jcb is None else jcb.double()
    f = g.double()[ok][:, None] * j[p[ok]]
    dx[p[ok]], vx[p[ok]] = f * dm.double()[t[ok]], f * f * dv.double()[t[ok]]
    x = _taken(mx, pos)
    a, b = x * dm.double()[:, None, :], x * x * dv.double()[:, None, :]
    return (dx, dx.abs()), (vx, vx.abs()), (a.sum(2), a.abs().sum(2)), (b.sum(2), b.abs().sum(2))


def dispatch_bwd(pos, jcb, dm, dv):
    a, b = _taken(dm, pos), _taken(dv, pos)
    j = 1.0 if jcb is None else jcb.double()
    return (j * a.sum(1), abs(j) * a.abs().sum(1)), (j * j * b.sum(1), j * j * b.abs().sum(1))

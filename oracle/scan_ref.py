"""The gated linear recurrences (include/pt_scan.h) in 64 bits, one step after
the other, with bounds on what an f32 evaluation of the same formulas may be
off by.

Every function returns values and bounds.  The bounds follow the recurrence:
an error made at one step is carried on by the product of the a's, so with u =
2^-24 (half an f32 step, relative)

  e_t = a_t e_{t-1} + (error of a_t) |h_{t-1}| + (error of b_t) + K u m_t

Time is cut into pieces that are joined as P h + q, with q the piece's result
from zero.  q and P h may be large and cancel where the walk's own terms are
small (a large input right after a large state of the other sign), and each is
rounded relative to itself: so the roundings are taken relative to m_t = a_t
m_{t-1} + |b_t|, which is at least |q| + |P h| for every way to cut.
Below 2^-126 an f32 rounding is off by up to 2^-150 whatever the value, which a
relative bound does not hold: K of them a step come to less than F = 2^-145, and
the few products that make a gradient from the state (factors below 2^8) to less
than 2^-139.

The error of a logistic value is (2 |x| + 8) u relative: |x| log2(e) is rounded
once and its constant once (2 |x| u in the exponent), exp2 and the reciprocal
are good to an ulp (2 u each), the sum to u.  tanh is good to 8 u absolute and
to 40 u relative: (1 - e) / (1 + e) with e = exp(-2|x|) is taken from 1/64 on at
the least, where 1 - e >= 0.0307 makes at most 32.6 u of the ulp of e (u), the
exponent adds 1.5 u (3 |x| u in e), the sum, the reciprocal and the products 5 u;
below, 2x - 2x^2 + 4/3 x^3 leaves out 1/3 x^3 < 21.4 u of 1 - e and rounds four
times.  tanh's derivative is good to 16 u.  K = 24 covers the roundings of a step's own products and
of joining the pieces (at most 16 a chunk, of 4 steps or more each).
"""
import torch

U = 2.0 ** -24
K = 24.0
F = 2.0 ** -145
FG = 2.0 ** -139


def _s(x):
    return torch.sigmoid(x)


def _es(x):
    """Relative error of s(x) and s(-x); saturated values are exact."""
    return (2.0 * x.abs().clamp(max=104.0) + 8.0) * U


def _et(th):
    """Error of tanh where its value is at most th in size."""
    return (40.0 * th.abs()).clamp(max=8.0) * U


def walk(form, gates, h0=None, lengths=None, dy=None, dh=None, dc=None, backward=True):
    """The recurrence over [B, T, F] gates (f64), its gradients, and bounds.

    Returns (values, bounds), dicts with y, h (last output), c (last state) and,
    with ``backward``, dgates (a list) and dh0.
    """
    gates = [g.double() for g in gates]
    b, t_len, f = gates[0].shape
    h = torch.zeros(b, f, dtype=torch.float64) if h0 is None else h0.double().clone()
    n = torch.full((b,), t_len) if lengths is None else lengths.clamp(0, t_len)
    on = (torch.arange(t_len)[None, :] < n[:, None])[:, :, None]            # [B, T, 1]
    last = (torch.arange(t_len)[None, :] == n[:, None] - 1)[:, :, None]
    gates = [torch.where(on, g, torch.zeros_like(g)) for g in gates]        # nothing behind the end is read
    one, zero = torch.ones((), dtype=torch.float64), torch.zeros((), dtype=torch.float64)
    if form == "leaky":
        z, cand = gates
        a, take = _s(-z), _s(z)
        ea, eb = a * _es(z), (take * cand).abs() * (_es(z) + 2 * U)
    else:
        i, fg, pre, o = gates
        a, take, cand, show = _s(fg), _s(i), torch.tanh(pre), _s(o)
        ea = a * _es(fg)
        eb = (take * cand).abs() * (_es(i) + 2 * U) + take * _et(cand)
    put = take * cand
    a, put = torch.where(on, a, one), torch.where(on, put, zero)
    ea, eb = torch.where(on, ea, zero), torch.where(on, eb, zero)
    states, befores, err, ebefore = [], [], [], []
    e = torch.zeros_like(h)
    m = h.abs()
    for t in range(t_len):
        befores.append(h)
        ebefore.append(e)
        live = on[:, t].double()
        new = a[:, t] * h + put[:, t]
        m = a[:, t] * m + put[:, t].abs()
        e = a[:, t] * e + ea[:, t] * h.abs() + eb[:, t] + live * (K * U * m + F)
        h = torch.where(on[:, t], new, h)
        states.append(h)
        err.append(e)
    st, est = torch.stack(states, 1), torch.stack(err, 1)
    bf, ebf = torch.stack(befores, 1), torch.stack(ebefore, 1)
    if form == "leaky":
        y, ey = st, est
        h_last, eh_last = h, e
    else:
        th = torch.tanh(st)
        y = show * th
        ey = y.abs() * (_es(o) + 2 * U) + show * (est + _et(th.abs() + est))
        h_last = torch.where(last, y, zero).sum(1)
        eh_last = torch.where(last, ey, zero).sum(1)
    val = dict(y=torch.where(on, y, zero), h=h_last, c=h)
    bnd = dict(y=torch.where(on, ey, zero), h=eh_last, c=e)
    if not backward:
        return val, bnd

    d = torch.zeros_like(y) if dy is None else torch.where(on, dy.double(), zero)
    g = torch.zeros_like(h)
    if form == "leaky":
        if dh is not None:
            g = g + dh.double()
        if dc is not None:
            g = g + dc.double()
        local, el = d, torch.zeros_like(d)
    else:
        if dh is not None:
            d = d + torch.where(last, dh.double()[:, None], zero)
        if dc is not None:
            g = g + dc.double()
        sech = 1.0 - th * th
        local = d * show * sech
        el = d.abs() * show * (est + 16 * U) + local.abs() * (_es(o) + 6 * U)
    eg = torch.zeros_like(g)
    mg = g.abs()
    grads, egr = [None] * t_len, [None] * t_len
    for t in reversed(range(t_len)):
        tot = local[:, t] + g
        mt = local[:, t].abs() + mg
        et = el[:, t] + eg + 2 * U * mt
        grads[t], egr[t] = tot, et
        g = a[:, t] * tot
        mg = a[:, t] * mt
        eg = a[:, t] * et + ea[:, t] * tot.abs() + on[:, t].double() * (K * U * mg + F)
    G, eG = torch.stack(grads, 1), torch.stack(egr, 1)
    if form == "leaky":
        k = take * a
        dz, dn = G * (cand - bf) * k, G * take
        ez = (eG * (cand - bf).abs() + G.abs() * (ebf + 2 * U * (cand.abs() + bf.abs()))) * k \
            + dz.abs() * (2 * _es(z) + 4 * U)
        en = eG * take + dn.abs() * (_es(z) + 4 * U)
        dg, ed = [dz, dn], [ez, en]
    else:
        ki, kf, dt, ko = take * _s(-i), a * _s(-fg), 1.0 - cand * cand, show * _s(-o)
        dg = [G * cand * ki, G * bf * kf, G * take * dt, d * th * ko]
        ed = [eG * cand.abs() * ki + G.abs() * ki * _et(cand) + dg[0].abs() * (2 * _es(i) + 6 * U),
              (eG * bf.abs() + G.abs() * ebf) * kf + dg[1].abs() * (2 * _es(fg) + 6 * U),
              eG * take * dt + G.abs() * take * 16 * U + dg[2].abs() * (_es(i) + 6 * U),
              d.abs() * ko * (est + _et(th.abs() + est)) + dg[3].abs() * (2 * _es(o) + 6 * U)]
    val["dgates"] = [torch.where(on, v, zero) for v in dg]
    bnd["dgates"] = [torch.where(on, v + FG, zero) for v in ed]
    val["dh0"], bnd["dh0"] = g, eg
    return val, bnd


def rounding(value, dtype):
    """Half a step of ``dtype`` at ``value``: relative, or the subnormals' own step."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.tiny * info.eps / 2

"""64-bit oracle of the gated-block operators, with the error that 32-bit arithmetic may make.

Each function returns its results and, for every value, a bound on the absolute error of an evaluation in fp32 whose
roundings are counted in units of 2^-24: the formula evaluated on magnitudes times that count. The counts:

  sigmoid   e = 2^(-g log2 e): the product's rounding and the constant's make at most 2 |g| units, the approximate power
            of two 4, the sum 1, the approximate reciprocal 2 and the product with e 1: for |g| <= 8 under 32 units of
            2^-24, for a gate and for one minus it alike (each is formed without a difference)
  scan      a step adds a product, a sum and (where parts of a sequence are joined) one factor of a product of gates:
            40 units of the magnitude, which is the recurrence of |u| (parts may cancel), carried on by the recurrence
  norm      a sum of D squares in 256 or more lanes: D / 256 + 10 <= 74 units, halved by the root, the root 4, the
            gate 32, six products: under 128 units of the magnitude of each sum or product; behind the second norm the
            same again
"""
import torch

U = 2.0 ** -24


def half_step(dtype):
    """Largest relative rounding error of a conversion to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def assert_within(got, ref, err, what=""):
    """|got - ref| within the fp32 error bound plus the rounding to got's type (and its subnormal step)."""
    fi = torch.finfo(got.dtype)
    tol = err + (ref.abs() + err) * half_step(got.dtype) + fi.tiny * fi.eps
    g = got.detach().double().cpu()
    ref, tol = ref.cpu(), tol.cpu()
    assert g.shape == ref.shape, (what, g.shape, ref.shape)
    bad = ~((g - ref).abs() <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by "
                                 f"{float(((g - ref).abs() / tol).nan_to_num(float('inf')).max()):.3g} times its bound")


# ------------------------------------------------------------------------------------------------- scan ----
def gated_scan(x, gate, h0, kind, leaky, lengths=None):
    """x, gate [T,B,D]; returns (h, err_h, h_last, err_last), fp64."""
    x, g = x.double(), gate.double()
    T, B, D = x.shape
    a = torch.sigmoid(g) if kind == "sigmoid" else g
    b = torch.sigmoid(-g) if kind == "sigmoid" else 1 - g
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.double()
    err, mag = torch.zeros_like(h), h.abs()
    out, outerr = torch.zeros_like(x), torch.zeros_like(x)
    n = torch.full((B,), T) if lengths is None else lengths.long().clamp(0, T)
    for t in range(T):
        live = (t < n)[:, None]
        u = b[t] * x[t] if leaky else x[t]
        mag = torch.where(live, a[t].abs() * mag + u.abs(), mag)
        e = a[t].abs() * err + 40 * U * mag
        err = torch.where(live, e, err)
        h = torch.where(live, a[t] * h + u, h)
        out[t], outerr[t] = torch.where(live, h, 0.0), torch.where(live, err, 0.0)
    return out, outerr, h, err


def gated_scan_backward(dh, dh_last, x, gate, h0, kind, leaky, lengths=None):
    """Returns ((dx, dgate, dh_init), the errors of each), fp64."""
    hs, herr, _, _ = gated_scan(x, gate, h0, kind, leaky, lengths)
    x, g, dh = x.double(), gate.double(), dh.double()
    T, B, D = x.shape
    a = torch.sigmoid(g) if kind == "sigmoid" else g
    b = torch.sigmoid(-g) if kind == "sigmoid" else 1 - g
    lam = torch.zeros(B, D, dtype=torch.float64) if dh_last is None else dh_last.double()
    err, mag = torch.zeros_like(lam), lam.abs()
    n = torch.full((B,), T) if lengths is None else lengths.long().clamp(0, T)
    dx, dg = torch.zeros_like(x), torch.zeros_like(x)
    ex, eg = torch.zeros_like(x), torch.zeros_like(x)
    first = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.double()
    for t in range(T - 1, -1, -1):
        live = (t < n)[:, None]
        L = dh[t] + lam
        M = dh[t].abs() + mag
        e = err + 40 * U * M
        before, be = (hs[t - 1], herr[t - 1]) if t else (first, torch.zeros_like(first))
        diff = before - x[t] if leaky else before
        de = be + U * (before.abs() + x[t].abs())
        f = a[t] * b[t] if kind == "sigmoid" else torch.ones_like(L)
        gx = b[t] * L if leaky else L
        dx[t] = torch.where(live, gx, 0.0)
        ex[t] = torch.where(live, (b[t].abs() * e if leaky else e) + 40 * U * gx.abs(), 0.0)
        dg[t] = torch.where(live, L * diff * f, 0.0)
        eg[t] = torch.where(live, f.abs() * (e * diff.abs() + (L.abs() + e) * de) + 80 * U * (L * diff * f).abs(), 0.0)
        lam = torch.where(live, a[t] * L, lam)
        err = torch.where(live, a[t].abs() * (e + 40 * U * M), err)
        mag = torch.where(live, a[t].abs() * M, mag)
    return (dx, dg, lam), (ex, eg, err)


# ------------------------------------------------------------------------------------------------- norm ----
def _act(kind, g):
    if kind == "none":
        return 1.0, 0.0, 1.0
    g = g.double()
    p, m = torch.sigmoid(g), torch.sigmoid(-g)
    if kind == "sigmoid":
        return p, p * m, p * m
    return g * p, p * (1 + g * m), p * (1 + g.abs() * m)       # value, derivative, the derivative's magnitude


def block_norm(y, gate, res, w_post, scale, w_pre, act, post, pre, alpha, eps):
    """Returns dict(res_out, z) and the errors of each, and the parts the backward pass uses; tensors [M, D] or None."""
    lead = y if y is not None else res
    d = lambda t, other: other if t is None else t.double()  # noqa: E731
    r = d(res, torch.zeros(lead.shape, dtype=torch.float64))
    s = dict(ry=1.0, n=None, c=0.0, av=1.0, dav=0.0, dmag=0.0)
    out, mag = r, r.abs()
    if y is not None:
        yd = y.double()
        s["ry"] = 1 / torch.sqrt((yd * yd).mean(-1, keepdim=True) + eps) if post else 1.0
        s["n"] = yd * s["ry"]
        s["c"] = alpha * d(scale, 1.0) * d(w_post, 1.0)
        s["av"], s["dav"], s["dmag"] = _act(act, gate)
        out = r + s["c"] * s["av"] * s["n"]
        mag = r.abs() + (s["c"] * s["av"] * s["n"]).abs()
    s["out"], s["mag"] = out, mag
    ret, err = dict(res_out=out, z=None), dict(res_out=128 * U * mag, z=None)
    if pre:
        s["ro"] = 1 / torch.sqrt((out * out).mean(-1, keepdim=True) + eps)
        # the relative error of rstd(out): that of the sum of squares, sum |out| err / sum out^2, and its roundings
        rel = 128 * U * ((out.abs() * mag).mean(-1, keepdim=True) * s["ro"] ** 2 + 1)
        s["rel_ro"] = rel
        w = d(w_pre, 1.0)
        ret["z"] = out * s["ro"] * w
        err["z"] = abs(w) * s["ro"] * (128 * U * mag + rel * out.abs())
    return ret, err, s


def block_norm_backward(dro, dz, y, gate, res, w_post, scale, w_pre, act, post, pre, alpha, eps):
    """Returns dict(dy, dgate, dresidual, dw_post, dres_scale, dw_pre) and the errors of each."""
    lead = y if y is not None else res
    M, D = lead.shape
    d = lambda t, other: other if t is None else t.double()  # noqa: E731
    _, _, s = block_norm(y, gate, res, w_post, scale, w_pre, act, post, dz is not None, alpha, eps)
    zero = torch.zeros(lead.shape, dtype=torch.float64)
    G, E = d(dro, zero), zero.clone()
    out, err = {}, {}
    rows = M + 40           # additions of a column's sum, each rounding once, in whatever order
    if dz is not None:
        u, v, ro, rel = dz.double() * d(w_pre, 1.0), s["out"], s["ro"], s["rel_ro"]
        verr = 128 * U * s["mag"]
        m, mm = (v * u).mean(-1, keepdim=True), (v * u).abs().mean(-1, keepdim=True)
        em = (verr * u.abs()).mean(-1, keepdim=True) + 128 * U * mm
        G = G + ro * u - v * ro ** 3 * m
        E = (rel + 128 * U) * ro * u.abs() + ro ** 3 * (verr * m.abs() + v.abs() * em + (3 * rel + 128 * U) * v.abs() * m.abs())
        E = E + 128 * U * (d(dro, zero).abs() + ro * u.abs() + v.abs() * ro ** 3 * m.abs())
        t, te = dz.double() * v * ro, dz.double().abs() * ro * (verr + (rel + 128 * U) * v.abs())
        out["dw_pre"], err["dw_pre"] = t.sum(0), te.sum(0) + rows * U * t.abs().sum(0)
    out["dresidual"], err["dresidual"] = G, E
    if y is not None:
        k = 256 * U
        e, ee = G * s["c"] * s["av"], abs(s["c"] * s["av"]) * (E + k * G.abs())
        yd, ry = y.double(), s["ry"]
        if post:
            m, mm = (yd * e).mean(-1, keepdim=True), (yd * e).abs().mean(-1, keepdim=True)
            em = (yd.abs() * ee).mean(-1, keepdim=True) + k * mm
            out["dy"] = ry * e - yd * ry ** 3 * m
            err["dy"] = ry * ee + yd.abs() * ry ** 3 * em + 2 * k * (ry * e.abs() + yd.abs() * ry ** 3 * mm)
        else:
            out["dy"], err["dy"] = e, ee
        if gate is not None:
            out["dgate"] = G * s["c"] * s["n"] * s["dav"]
            err["dgate"] = abs(s["c"] * s["n"]) * s["dmag"] * (E + 2 * k * G.abs())
        q, qe = alpha * G * s["av"] * s["n"], abs(alpha * s["av"] * s["n"]) * (E + 2 * k * G.abs())
        Q, QE = q.sum(0), qe.sum(0) + rows * U * q.abs().sum(0)
        out["dw_post"], err["dw_post"] = Q * d(scale, 1.0), QE * abs(d(scale, 1.0))
        out["dres_scale"], err["dres_scale"] = Q * d(w_post, 1.0), QE * abs(d(w_post, 1.0))
    return out, err


# ----------------------------------------------------------------------------------------------- linear ----
def unpack_w4(q, scales, zeros, group):
    """[N, K] fp64 weights."""
    N, half = q.shape
    w = torch.stack([q & 15, q >> 4], -1).reshape(N, 2 * half).double()
    i = torch.arange(2 * half) // group
    return (w - (8.0 if zeros is None else zeros.double()[:, i])) * scales.double()[:, i]


def linear_w4(x, q, scales, zeros, bias, group):
    """x [M, K]; returns (y, err), fp64. A value is a sum of K products, K / 32 of them in sequence at the most, and each
    sum on the tensor cores may drop the bits below 2^-23 of its largest part: K / 16 + 64 units of the magnitude."""
    w = unpack_w4(q, scales, zeros, group)
    y, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, (x.shape[1] / 16 + 64) * U * mag

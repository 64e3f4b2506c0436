"""Plain 64-bit forms of the training operators, each with a bound on how far a kernel may be from it.

u = finfo(dtype).eps / 2 is one rounding to the storage type, w = 2^-24 one fp32 rounding.  A sum of n products in fp32 is off
by at most about (n + 1) w times the sum of their magnitudes, in any order."""
import torch

W = 2.0 ** -24


def rounding(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the smallest numbers: what rounding may add where the result is (nearly) zero."""
    return torch.finfo(dtype).smallest_normal * rounding(dtype) * 2


def assert_within(got, want, bound, what):
    got, want, bound = got.detach().double().cpu(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, "%s: shape %s, want %s" % (what, tuple(got.shape), tuple(want.shape))
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN in other places"
    off = (got - want).abs()
    bad = off > bound
    if bool(bad.any()):
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError("%s: %d of %d outside, first %s: %g, want %g, bound %g; worst %.3g of its bound" % (
            what, int(bad.sum()), bad.numel(), i, got[i], want[i], bound[i], float((off / bound).nan_to_num(0).max())))


def layer_norm(x, w, b, g, eps):
    """(values, bounds) of out, dx, dweight, dbias."""
    dt, E, T = x.dtype, x.size(1), x.size(0)
    u = rounding(dt)
    x, g = x.double(), g.double()
    w64 = torch.ones(E, dtype=torch.float64, device=x.device) if w is None else w.double()
    b64 = torch.zeros(E, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rs = 1 / torch.sqrt(var + eps)
    n = (x - mean) * rs
    gw = g * w64
    c1, c2 = gw.mean(1, keepdim=True), (gw * n).mean(1, keepdim=True)
    out, dx = n * w64 + b64, rs * (gw - c1 - n * c2)
    dw, db = (g * n).sum(0), g.sum(0)
    # fp32: the mean is off by (E + 2) w mean|x|, so is x - mean (plus w of each term); rstd by (E + 8) w relative plus what the
    # mean's error does to the variance; n by both
    e_mean = (E + 2) * W * x.abs().mean(1, keepdim=True)
    e_n = (e_mean + 2 * W * (x.abs() + mean.abs())) * rs + n.abs() * ((E + 8) * W + 2 * e_mean * rs)
    e_c1 = (E + 2) * W * gw.abs().mean(1, keepdim=True)
    e_c2 = (E + 2) * W * (gw * n).abs().mean(1, keepdim=True) + (gw.abs() * e_n).mean(1, keepdim=True)
    e_out = e_n * w64.abs() + 4 * W * (n * w64).abs() + W * b64.abs()
    e_rs = (E + 8) * W + 2 * e_mean * rs
    e_dx = rs * (4 * W * gw.abs() + e_c1 + n.abs() * e_c2 + e_n * c2.abs() + 4 * W * (n * c2).abs()) + dx.abs() * e_rs
    e_dw = (T + 2) * W * (g * n).abs().sum(0) + (g.abs() * e_n).sum(0)
    e_db = (T + 2) * W * g.abs().sum(0)
    values = dict(out=out, dx=dx, dweight=dw, dbias=db)
    errors = dict(out=e_out, dx=e_dx, dweight=e_dw, dbias=e_db)
    return values, {k: u * (values[k].abs() + errors[k]) + errors[k] + tiny(dt) for k in values}


def embedding(weight, index, g, scale, padding_idx):
    dt, V = weight.dtype, weight.size(0)
    u = rounding(dt)
    ok = (index >= 0) & (index < V)
    i = torch.where(ok, index, torch.zeros_like(index)).long()
    out = weight.double()[i] * scale * ok[:, None]
    keep = ok if padding_idx is None else ok & (index != padding_idx)
    rows = i[keep]
    dw = torch.zeros(V, weight.size(1), dtype=torch.float64, device=weight.device).index_add_(0, rows, g.double()[keep]) * scale
    mag = torch.zeros_like(dw).index_add_(0, rows, g.double().abs()[keep]) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64, device=weight.device).index_add_(0, rows, torch.ones_like(rows, dtype=torch.float64))
    e = (n[:, None] + 3) * W * mag  # the sum's additions, the factor (itself rounded to fp32) and the product
    e_out = 2 * W * out.abs()
    return dict(out=out, dweight=dw), dict(out=u * (out.abs() + e_out) + e_out + tiny(dt) * (scale != 1),
                                           dweight=u * (dw.abs() + e) + e + tiny(dt) * (mag > 0))


def attention(q, k, v, g, lq, lk, heads, scaling):
    """(values, bounds) of out, dq, dk, dv for packed rows q, k, v and lengths lq, lk."""
    dt = q.dtype
    d = q.size(1) // heads
    # 16-bit kernels round P and dS to the storage type before the products that use them (the forward pass P too) and D is
    # taken from the rounded output where a row has more than 16 keys, from the probabilities where it has fewer; fp32 kernels
    # round nothing.  The forward kernel for 16-bit types may take a quarter of its
    # exponentials from a polynomial of relative error 1.9e-4, which also enters the row's denominator.
    half = dt != torch.float32
    u = rounding(dt)
    up = u if half else 0.0
    ex = 2e-4 if half else 0.0
    vals = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    errs = {n: torch.zeros_like(t) for n, t in vals.items()}
    a = c = 0
    for n, m in zip(lq, lk):
        rows, cols = slice(a, a + n), slice(c, c + m)
        a, c = a + n, c + m
        if n == 0 or m == 0:
            continue
        Q, G = (t[rows].double().view(n, heads, d).transpose(0, 1) for t in (q, g))
        K, V = (t[cols].double().view(m, heads, d).transpose(0, 1) for t in (k, v))
        S = Q @ K.transpose(1, 2) * scaling
        P = torch.softmax(S, 2)
        O = P @ V
        dP = G @ V.transpose(1, 2)
        D = (G * O).sum(2, keepdim=True)
        dS = P * (dP - D)
        # S: d products in fp32, and a few roundings of the exponent's argument (the largest |S| of the row: lse holds it)
        smax = (Q.abs() @ K.abs().transpose(1, 2) * abs(scaling)).amax(2, keepdim=True)
        e_s = (d + 8) * W * smax
        e_p = P * (2 * e_s + (m + 16) * W + 2 * ex)        # absolute error of a probability, unrounded
        e_o = (e_p + up * P) @ V.abs() + (m + 4) * W * (P @ V.abs())
        e_d = (G.abs() * (e_o + (u if half else W) * (O.abs() + e_o))).sum(2, keepdim=True) + (d + 2) * W * (G * O).abs().sum(2, keepdim=True)
        e_dp = (d + 2) * W * (G.abs() @ V.abs().transpose(1, 2))
        if half and m <= 16:  # D = sum_j P_ij dP_ij
            e_d = (e_p * dP.abs() + P * e_dp).sum(2, keepdim=True) + (m + 4) * W * (P * dP).abs().sum(2, keepdim=True)
        e_ds = e_p * (dP - D).abs() + P * (e_dp + e_d + 2 * W * (dP.abs() + D.abs()))
        # rounded for the products; below the type's normal range by half its smallest step, where dS is held relative to the
        # power of two at or below the head's largest |dO| (at most that number times 2)
        e_ds = e_ds + up * (dS.abs() + e_ds) + half * tiny(dt) * G.abs().amax((1, 2), keepdim=True) * 2
        e_pr = e_p + up * (P + e_p) + half * tiny(dt)
        sc = abs(scaling)
        out = {"out": (O, e_o, rows), "dq": (scaling * (dS @ K), sc * (e_ds @ K.abs() + (m + 4) * W * (dS.abs() @ K.abs())), rows),
               "dk": (scaling * (dS.transpose(1, 2) @ Q), sc * (e_ds.transpose(1, 2) @ Q.abs() + (n + 4) * W * (dS.abs().transpose(1, 2) @ Q.abs())), cols),
               "dv": (P.transpose(1, 2) @ G, e_pr.transpose(1, 2) @ G.abs() + (n + 4) * W * (P.transpose(1, 2) @ G.abs()), cols)}
        for name, (y, e, r) in out.items():
            vals[name][r] = y.transpose(0, 1).reshape(-1, heads * d)
            errs[name][r] = e.transpose(0, 1).reshape(-1, heads * d)
    return vals, {n: u * (vals[n].abs() + errs[n]) + errs[n] + tiny(dt) for n in vals}

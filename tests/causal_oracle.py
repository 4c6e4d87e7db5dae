"""64-bit definitions of the causal attention operators with error bounds, shared by their tests.

Bounds: u = 2^-24 (half an fp32 step), e = half a step of the operand type (0 for fp32 where nothing is rounded below fp32).  Sums of n rounded
terms are taken to err by 4 sqrt(n) u of the sum of magnitudes (rounding errors of independent signs, four deviations)."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def norm_rope(x, gamma, positions, theta=10000.0, eps=1e-6, dy=None):
    """-> (y, tolerance of y), or with dy (.., dx, tolerance, dgamma, tolerance)."""
    e = half_step(x.dtype)
    D = x.shape[-1]
    xd, gd = x.detach().double(), gamma.detach().double()
    ang = positions.double()[:, None, None] * theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device=x.device) / D)
    c, s = ang.cos(), ang.sin()
    rstd = 1 / (xd.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    n = xd * rstd
    z = n * gd
    a, b = z[..., :D // 2], z[..., D // 2:]
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    mag = (a * a + b * b).sqrt()
    mag = torch.cat([mag, mag], -1)
    # a row's rounding errors: the mean of D squares (a thread's 16 in order, then a tree), rsqrt, three products, the rotation's two and sum;
    # an angle's: rounding of the reduced fraction (pi u) and of sine and cosine (2 u)
    rel = (20 + 8 + 6) * U
    out = [y, e * y.abs() + rel * mag]
    if dy is not None:
        dd = dy.detach().double()
        da, db = dd[..., :D // 2], dd[..., D // 2:]
        dz = torch.cat([da * c + db * s, db * c - da * s], -1)
        dmag = (da * da + db * db).sqrt()
        dmag = torch.cat([dmag, dmag], -1)
        dn = dz * gd
        dot = (dn * n).mean(-1, keepdim=True)
        dx = rstd * (dn - n * dot)
        terms = rstd * (dmag * gd.abs() + n.abs() * (dmag * gd.abs() * n.abs()).mean(-1, keepdim=True))
        out += [dx, e * dx.abs() + 2 * rel * terms]
        each = (dmag * n.abs()).sum((0, 1))
        rows = x.shape[0] * x.shape[1]
        out += [(dz * n).sum((0, 1)), (rel + 4 * math.sqrt(rows) * U) * each + 1e-30]
    return out


def attention(q, k, v, q_lens, k_lens, causal=True, scale=None, dout=None):
    """q [M, H, D], k, v [N, G, D] -> (out, tol) or with dout (out, tol, dq, tol, dk, tol, dv, tol), all 64-bit."""
    dt = q.dtype
    e = half_step(dt)
    ep = 0.0 if dt == torch.float32 else e                       # probabilities and dS are rounded to the operand type
    H, G, D = q.shape[1], k.shape[1], q.shape[2]
    R, scale = H // G, D ** -0.5 if scale is None else scale
    qd, kd, vd = q.detach().double(), k.detach().double(), v.detach().double()
    zeros = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=x.device)                 # noqa: E731
    out, tol = zeros(q), zeros(q)
    gr = None if dout is None else [zeros(q), zeros(q), zeros(k), zeros(k), zeros(v), zeros(v)]
    q0 = k0 = 0
    for n, t in zip(q_lens, k_lens):
        first = max(0, n - t) if causal else (0 if t else n)     # rows before it see nothing
        for h in range(H):
            g = h // R
            qs, ks, vs = qd[q0 + first:q0 + n, h], kd[k0:k0 + t, g], vd[k0:k0 + t, g]
            if qs.shape[0] == 0:
                continue
            s = scale * (qs @ ks.t())
            size = (scale * (qs.abs() @ ks.abs().t())).amax() if t else 0.0
            if causal:
                i, j = torch.arange(first, n, device=q.device), torch.arange(t, device=q.device)
                s = s.masked_fill(j[None, :] > i[:, None] + (t - n), -math.inf)
            p = torch.softmax(s, -1)
            o = p @ vs
            # a logit errs by 4 sqrt(D) u of its magnitude sum, the base-2 exponent and exp by a few u each of their own argument
            rel = 4 * U * (math.sqrt(D) * size + math.sqrt(t) + 8) + 8 * U * size
            out[q0 + first:q0 + n, h] = o
            tol[q0 + first:q0 + n, h] = e * o.abs() + (ep + 2 * rel) * (p @ vs.abs())
            if gr is not None:
                do = dout[q0 + first:q0 + n, h].double()
                # a row whose dO is not finite has no finite gradient, nor have the keys it sees; the others do not hear of it
                lost = ~torch.isfinite(do).all(-1)
                do = do.masked_fill(lost[:, None], 0)
                dp = do @ vs.t()
                dsum = (do * o).sum(-1, keepdim=True)
                ds = p * (dp - dsum)
                # dS: the probabilities' rounding in the output that D is made of (the output's own is kept), fp32 sums of dP and D, the
                # recomputed probability, its own rounding
                errd = (ep + e * e + 2 * rel + 4 * math.sqrt(D) * U) * (do.abs() * (p @ vs.abs())).sum(-1, keepdim=True)
                errp = 4 * math.sqrt(D) * U * (do.abs() @ vs.abs().t())
                eds = p * (errd + errp) + (ep + 2 * rel) * ds.abs()
                acc = 4 * math.sqrt(max(t, n * R)) * U
                gr[0][q0 + first:q0 + n, h] = scale * (ds @ ks)
                gr[1][q0 + first:q0 + n, h] = scale * (eds @ ks.abs() + acc * (ds.abs() @ ks.abs()))
                gr[2][k0:k0 + t, g] += scale * (ds.t() @ qs)
                gr[3][k0:k0 + t, g] += scale * (eds.t() @ qs.abs() + acc * (ds.abs().t() @ qs.abs()))
                gr[4][k0:k0 + t, g] += p.t() @ do
                gr[5][k0:k0 + t, g] += (ep + 2 * rel + acc) * (p.t() @ do.abs())
                gr[0][q0 + first:q0 + n, h][lost] = math.nan
                for x in (gr[2], gr[4]):
                    x[k0:k0 + t, g][torch.isfinite(s[lost]).any(0)] = math.nan
        q0, k0 = q0 + n, k0 + t
    if gr is None:
        return out, tol
    for i in (0, 2, 4):
        gr[i + 1] += e * gr[i].abs()
    return (out, tol, *gr)


def check(got, want, tol, what=''):
    """Every value within its own tolerance (where the definition has a value); the smallest subnormal of the type is always allowed."""
    floor = 2.0 ** -149 if got.dtype == torch.float32 else torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bad = ~((got.double() - want).abs() <= tol + floor) & ~torch.isnan(want)
    if bad.any():
        i = tuple(int(x[0]) for x in bad.nonzero(as_tuple=True))
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: {got[i].item()} for {want[i].item()} (tolerance {tol[i].item()})')

"""Plain float64 forms of the sequence operators, each with a bound of what the kernels may be off by.

The bounds are sums of rounding errors, no element of them fitted: u = 2^-24 is half a unit in the
last place of float32, e the same for the tensors' own type (2^-8 bfloat16, 2^-11 float16, u
float32).  A sum of n products kept in float32 by the matrix cores is taken off by at most
(n / 16 + 16) u of the sum of the products' magnitudes (sixteen are joined at a time); a weight of
the softmax carries the error of its score and of the row's log-sum, and one rounding to the tensors'
type before it is multiplied; a result carries one rounding to that type."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest step of the type: what a rounding is off by where eps / 2 of the value is less."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def sum_error(n):
    return (n / 16 + 16) * U


def attention(q, k, v, q_off, k_off, causal, scale, grad=None):
    """q [tq,hq,d] ... on the CPU, q_off / k_off lists.  -> dict name -> (value, bound)."""
    e, t0 = half_step(q.dtype), tiny(q.dtype)
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    q, k, v = q.double(), k.double(), v.double()
    zero = lambda t: torch.zeros(t.shape, dtype=torch.float64)      # noqa: E731
    out, lse = (zero(q), zero(q)), torch.full((hq, q.shape[0]), float("-inf"), dtype=torch.float64)
    lse_bound = torch.zeros_like(lse)
    dq, dk, dv = ((zero(t), zero(t)) for t in (q, k, v))
    for s in range(len(q_off) - 1):
        a, b, c, f = q_off[s], q_off[s + 1], k_off[s], k_off[s + 1]
        lq, lk = b - a, f - c
        if lq == 0 or lk == 0:
            continue
        allowed = torch.ones(lq, lk, dtype=torch.bool)
        if causal:
            allowed = torch.arange(lk)[None, :] <= torch.arange(lq)[:, None] + lk - lq
        for h in range(hq):
            g = h // (hq // hk)
            qs, ks, vs = q[a:b, h], k[c:f, g], v[c:f, g]
            z = scale * qs @ ks.t()
            # score: its sum, the product with scale and log2 e, the subtraction of the maximum, the exponential
            mass_z = abs(scale) * qs.abs() @ ks.abs().t()
            dz = (sum_error(d) + 4 * U) * mass_z + 4 * U * z.abs()
            z = z.masked_fill(~allowed, float("-inf"))
            some = allowed.any(1, keepdim=True)
            top = torch.where(some, z.amax(1, keepdim=True), torch.zeros(1, 1, dtype=torch.float64))
            p = torch.exp(z - top)
            total = p.sum(1, keepdim=True)
            ls = top + torch.log(torch.where(some, total, torch.ones_like(total)))
            p = torch.where(some, p / torch.where(some, total, torch.ones_like(total)), torch.zeros_like(p))
            worst = torch.where(allowed, dz, torch.zeros_like(dz)).amax(1, keepdim=True) + 4 * U * top.abs()
            rel = 2 * worst + (lk / 2 + 16) * U          # score and log-sum; the row's sum runs in sequence
            o = p @ vs
            mass = p @ vs.abs()
            bo = mass * (rel + e + sum_error(lk)) + e * o.abs() + t0 * (1 + vs.abs().sum(0))
            out[0][a:b, h], out[1][a:b, h] = o, bo
            lse[h, a:b] = torch.where(some, ls, torch.full_like(ls, float("-inf")))[:, 0]
            lse_bound[h, a:b] = (rel + 4 * U * ls.abs() + 4 * U)[:, 0]
            if grad is None:
                continue
            do = grad[a:b, h].double()
            relb = 2 * rel + 8 * U * ls.abs()            # rebuilt from the saved log-sum
            dp, delta = do @ vs.t(), (do * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            err = p * (relb * (dp - delta).abs() + (sum_error(d) + 2 * U) * (do.abs() @ vs.abs().t())
                       + (do.abs() * bo).sum(1, keepdim=True) + sum_error(d) * (do * o).abs().sum(1, keepdim=True))
            err = err + e * (ds.abs() + err) + t0 * allowed
            dv[0][c:f, g] += p.t() @ do
            dv[1][c:f, g] += (p * (relb + e + sum_error(lq * hq // hk)) + t0 * allowed).t() @ do.abs()
            dq[0][a:b, h] = scale * ds @ ks
            dq[1][a:b, h] = abs(scale) * (err + sum_error(lk) * ds.abs()) @ ks.abs()
            dk[0][c:f, g] += scale * ds.t() @ qs
            dk[1][c:f, g] += abs(scale) * (err + sum_error(lq * hq // hk) * ds.abs()).t() @ qs.abs()
    res = dict(out=out, lse=(lse, lse_bound))
    if grad is not None:
        for name, (x, bound) in (("dq", dq), ("dk", dk), ("dv", dv)):
            res[name] = (x, bound + (e + 2 * U) * (x.abs() + bound) + t0)
    return res


def linear_ce(feat, weight, label, ignore, reduction, grad=None):
    """-> dict name -> (value, bound); grad: of the loss (None: no gradients)."""
    e, t0 = half_step(feat.dtype), tiny(feat.dtype)
    n, d = feat.shape
    v = weight.shape[0]
    kept = (label != ignore) & (label >= 0) & (label < v)
    x, w = feat.double(), weight.double()
    idx = kept.nonzero()[:, 0]
    z = x[idx] @ w.t()
    dz = (sum_error(d) + 4 * U) * (x[idx].abs() @ w.abs().t()) + 4 * U * z.abs()
    ls = torch.logsumexp(z, 1)
    y = label[idx].long()
    pick = torch.arange(len(idx))
    worst = dz.amax(1) if len(idx) else torch.zeros(0, dtype=torch.float64)
    rel = 2 * worst + (64 + v / 128) * U                 # tiles of 128 classes, joined in sequence
    loss, bound = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    lse, lse_bound = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    lse[idx], lse_bound[idx] = ls, rel + 4 * U * ls.abs() + 4 * U
    loss[idx], bound[idx] = ls - z[pick, y], rel + 8 * U * (ls.abs() + z[pick, y].abs()) + 4 * U
    count = max(1, len(idx))
    res = dict(lse=(lse, lse_bound))
    if reduction == "none":
        res["loss"] = (loss, bound)
    else:
        by = 1.0 / count if reduction == "mean" else 1.0
        res["loss"] = (loss.sum() * by, bound.sum() * by + 2 * U * loss.sum().abs() * by)
    if grad is None:
        return res
    g = (grad.double().expand(n)[idx] / (count if reduction == "mean" else 1)).unsqueeze(1)
    p = torch.exp(z - ls.unsqueeze(1))
    relb = (2 * rel + 8 * U * ls.abs()).unsqueeze(1)
    hit = torch.zeros_like(p)
    hit[pick, y] = 1
    dzv = (p - hit) * g
    err = (p * relb + 2 * U * (p - hit).abs()) * g.abs() + 2 * U * dzv.abs()
    err = err + e * (dzv.abs() + err)
    if len(idx):                                         # float16 keeps dz as multiples of the largest |g| / 2^14
        err = err + t0 * g.abs().max() * (2.0 ** -14 if feat.dtype == torch.float16 else 1.0)
    dx, bx = torch.zeros_like(x), torch.zeros_like(x)
    dx[idx] = dzv @ w
    bx[idx] = (err + sum_error(v) * dzv.abs()) @ w.abs()
    dw, bw = dzv.t() @ x[idx], (err + sum_error(n) * dzv.abs()).t() @ x[idx].abs()
    res["dx"] = (dx, bx + (e + 2 * U) * (dx.abs() + bx) + t0)
    res["dw"] = (dw, bw + (e + 2 * U) * (dw.abs() + bw) + t0)
    return res


def check(got, want, what):
    """|got - value| <= bound everywhere; infinities equal."""
    value, bound = (t.detach().cpu() for t in want)
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    inf = torch.isinf(value)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], value[inf]), what
    ok = torch.where(inf, torch.zeros_like(value), (got - value).abs()) <= torch.where(inf, torch.zeros_like(value), bound)
    if not bool(ok.all()):
        i = int((~ok).flatten().nonzero()[0, 0])
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} off; first at {i}: got {got.flatten()[i].item():.9g}, "
                             f"want {value.flatten()[i].item():.9g} +- {bound.flatten()[i].item():.3g}")

"""Plain 64-bit forms of attention over rows with a mask and of token log
probabilities, and how far a kernel in fp32 sums with operands of a type may be
from them.

Bounds, for one head, with u the type's half step (finfo.eps / 2), e = 2^-24
fp32's, z_j = scale q . k_j, S = max_j scale |q| . |k_j| over what the row sees
and n its keys:
  a score           (d + 3) e S: d products and sums, the factor, the exponent's
                    own rounding; the exponential doubles a distance as long as
                    it is small, and its own error is 2 e: each unnormalised p,
                    and likewise their sum, is off by r = 2 (d + 3) e S + 8 e,
                    the sum by n e more
  a probability     r + (r + n e) relative, R in all; rounded to the type for
                    the next product: u more, and below fp16's least normal
                    2^-25 absolute
  o = sum p v       (u + R + n e) sum p |v| + u |o|, and 2^-25 where fp16 holds
                    it below its least normal (any result of the type alike)
  lse               r + n e + 4 e |lse|
The gradients carry these through their own sums, term by term below.
"""
import torch

E = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def attention_row_sets(q, k, v, seen, scale, dt, grad=None):
    """q [n, d], k and v [m, d], seen [n, m] booleans, all float64 but seen:
    (o, lse, their bounds) and, with grad [n, d], dq, dk, dv and theirs.  What
    is not seen is taken out of k and v before any product."""
    u = half_step(dt)
    out_u = u
    if dt == torch.float32:
        u = 0.0                       # probabilities and ds are not rounded
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    n, d = q.shape
    m = k.size(0)
    s = (q @ k.T) * scale
    sa = (q.abs() @ k.abs().T) * scale
    s = torch.where(seen, s, torch.full_like(s, -torch.inf))
    S = torch.where(seen, sa, torch.zeros_like(sa)).amax(1, keepdim=True)
    mx = s.amax(1, keepdim=True)
    empty = mx == -torch.inf
    mx = torch.where(empty, torch.zeros_like(mx), mx)
    ex = torch.where(seen, torch.exp(s - mx), torch.zeros_like(s))
    l = ex.sum(1, keepdim=True)
    p = torch.where(empty, torch.zeros_like(ex), ex / l)
    lse = (mx + torch.log(l))[:, 0]
    r = 2 * (d + 3) * E * S + 8 * E
    R = 2 * r + m * E
    va = v.abs()
    o = p @ v
    pva = p @ va
    seen_va = seen.double() @ va
    o_tol = (u + R + m * E) * pva + out_u * o.abs() + tiny * seen_va + tiny + 1e-30
    lse_tol = (r + m * E)[:, 0] + 4 * E * lse.abs()
    if grad is None:
        return (o, lse), (o_tol, lse_tol)
    ga = grad.abs()
    D = (grad * o).sum(1, keepdim=True)
    D_tol = (ga * o_tol).sum(1, keepdim=True) + (d + 2) * E * (ga * o.abs()).sum(1, keepdim=True)
    dp = torch.where(seen, grad @ v.T, torch.zeros_like(s))
    dp_tol = (d + 2) * E * (ga @ va.T)
    # p from the kept lse: its bound and the exponent's own
    P = R + lse_tol.nan_to_num(0.0, 0.0, 0.0)[:, None] + 4 * E * lse.nan_to_num(0.0, 0.0, 0.0).abs()[:, None]
    ds = p * (dp - D)
    ds_tol = p * (dp_tol + D_tol) + P * p * (dp - D).abs() + 4 * E * p * (dp.abs() + D.abs()) + u * ds.abs()
    ds_tol = torch.where(seen, ds_tol + tiny, torch.zeros_like(ds_tol))
    p_tol = torch.where(seen, (u + P) * p + tiny, torch.zeros_like(p))
    # half a step of the sums' rounded result, and their own rounding in fp32
    dq, dk, dv = scale * (ds @ k), scale * (ds.T @ q), p.T @ grad
    dq_tol = scale * (ds_tol @ k.abs()) + m * E * scale * (ds.abs() @ k.abs()) + out_u * dq.abs() + tiny + 1e-30
    dk_tol = scale * (ds_tol.T @ q.abs()) + n * E * scale * (ds.abs().T @ q.abs())
    dv_tol = p_tol.T @ ga + n * E * (p.T @ ga)
    return (o, lse, dq, dk, dv), (o_tol, lse_tol, dq_tol, dk_tol, dv_tol)


def packed_reference(q, k, v, lens, scale, grad=None, start=0):
    """All rows and heads of packed sequences: outputs and bounds as dicts of
    float64 CPU tensors (zeros outside the sequences)."""
    dt = q.dtype
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    grad = grad.double().cpu() if grad is not None else None
    total, H, d = q.shape
    G = k.size(1)
    names = ["out"] + (["dq", "dk", "dv"] if grad is not None else [])
    shapes = dict(out=q.shape, dq=q.shape, dk=k.shape, dv=v.shape)
    want = {n: torch.zeros(shapes[n], dtype=torch.float64) for n in names}
    tol = {n: torch.zeros(shapes[n], dtype=torch.float64) for n in names}
    want["lse"] = torch.zeros((H, total), dtype=torch.float64)
    tol["lse"] = torch.zeros((H, total), dtype=torch.float64)
    a = start
    for n in lens:
        b = a + n
        seen = torch.ones((n, n), dtype=torch.bool).tril()
        for h in range(H if n else 0):
            g = h // (H // G)
            w, t = attention_row_sets(q[a:b, h], k[a:b, g], v[a:b, g], seen, scale, dt,
                                      grad[a:b, h] if grad is not None else None)
            for x, y in ((want, w), (tol, t)):
                x["out"][a:b, h], x["lse"][h, a:b] = y[0], y[1]
                if grad is not None:
                    x["dq"][a:b, h] = y[2]
                    x["dk"][a:b, g] += y[3]
                    x["dv"][a:b, g] += y[4]
        a = b
    for n in ("dk", "dv"):
        if n in tol:
            # the group's heads in one fp32 sum, rounded once
            tol[n] += (half_step(dt) + H // G * E) * want[n].abs() + (2.0 ** -25 if dt == torch.float16 else 1e-30)
    return want, tol


def tree_seen(length, parents):
    T = len(parents)
    seen = torch.zeros((T, length + T), dtype=torch.bool)
    seen[:, :length] = True
    for t in range(T):
        u = t
        while u >= 0:
            seen[t, length + u] = True
            u = parents[u]
    return seen


def logprob_reference(x, tokens):
    """(logprob, entropy, lse) in 64 bits; see token_logprobs for the rules."""
    x = x.double().cpu()
    tokens = tokens.cpu()
    lse = torch.logsumexp(x, -1)
    logp = x - lse[:, None]
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    lp = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    empty = lse == -torch.inf
    lp = torch.where(empty, torch.full_like(lp, -torch.inf), lp)
    ent = torch.where(empty, torch.zeros_like(ent), ent)
    return torch.where(tokens < 0, torch.zeros_like(lp), lp), ent, lse, logp, p


def check(got, want, tol, what):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    same = got[~fin & ~torch.isnan(want)] == want[~fin & ~torch.isnan(want)]
    assert bool(same.all()), f"{what}: infinities differ"
    diff = (got - want).abs()
    over = torch.where(diff == 0, diff, diff / tol)[fin]
    assert over.numel() == 0 or float(over.max()) <= 1.0, f"{what}: {float(over.max()):.3g} times its bound"

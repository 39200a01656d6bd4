"""Plain 64-bit forms of the recurrent layers' operators and of the verification
of drafted tokens, and the bounds their kernels' outputs are held to."""
import math

import torch


def offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _half(y):
    """Half a step of fp16 at y (2^-25: half its smallest step)."""
    return 2.0 ** -11 * y.abs() + 2.0 ** -25


def check(got, want, bound, what=""):
    got = got.double()
    same = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), same), f"{what}: other values are not finite"
    if not got.numel():
        return
    worst = torch.where(same, (got - want).abs() / bound, 0.0).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"


def short_conv(x, state, weight, bias, silu):
    """(out, bound, new state) of one sequence's rows x [n][channels] behind state
    [width - 1][channels] (fp16)."""
    width = weight.shape[1]
    if not len(x):
        return x.double(), x.double(), state
    rows = torch.cat([state, x]).double().unfold(0, width, 1)       # [n][channels][width]
    y = (rows * weight.double()).sum(-1)
    mass = (rows * weight.double()).abs().sum(-1)
    if bias is not None:
        y, mass = y + bias.double(), mass + bias.double().abs()
    near = (width + 1) * 2.0 ** -24 * mass                          # fma by fma in 32 bits
    if silu:
        # silu's slope is below 1.1; its exponential, sum and quotient are off by some 2^-22 of it
        y, near = y * torch.sigmoid(y), 1.1 * near
        near = near + 2.0 ** -20 * y.abs()
    return y, near + _half(y) * (1 + 2.0 ** -10), torch.cat([state, x])[x.shape[0]:]


def gated_norm(x, z, gamma, eps):
    x, z = x.double(), z.double()
    y = x * (x.square().mean(-1, keepdim=True) + eps).clamp(min=1e-20).rsqrt()
    y = y * z * torch.sigmoid(z)
    if gamma is not None:
        y = y * gamma.double()
    # a sum of up to 512 squares, a root, an exponential and five products in 32 bits
    return y, _half(y) * (1 + 2.0 ** -10) + 2.0 ** -18 * y.abs()


def delta(q, k, v, a, b, a_log, dt_bias, state, scale, eps):
    """(out, bound, new state, its bound) of one sequence's rows from state
    [heads_v][dim_k][dim_v], row after row in 64 bits.

    The bounds follow the recurrence.  A row multiplies what the state is off by
    with e^g (1 - beta k^ k^T), which lengthens no column, and adds the rounding of
    its own sums: of some 2^-24 (the row by row form: at most dim_k + 16 of them, whose
    errors are of both signs) or of products whose factors are split into two fp16
    numbers (2^-22 of each factor, in sums over 64 rows and dim_k values, both signs),
    of the column's length and of v.  8 times 2^-22 of both covers either.  The decay
    is off by some 2^-22 of itself for each unit of its logarithm, at most 2^-22 of the
    column."""
    n, hk, dk = q.shape
    hv, dv = v.shape[1:]
    group = hv // hk
    S, E = state.double().clone(), torch.zeros((hv, 1, dv), dtype=torch.float64, device="cuda")
    out = torch.empty((n, hv, dv), dtype=torch.float64, device="cuda")
    near = torch.empty_like(out)
    kn, qn = (x.double() / (x.double().square().sum(-1, keepdim=True) + eps).sqrt()
              for x in (k, q))
    kn, qn = kn.repeat_interleave(group, 1), qn.repeat_interleave(group, 1)
    t = a.double() + dt_bias.double()
    soft = torch.where(t > 30, t, torch.log1p(torch.exp(t.clamp(max=30))))
    g = -torch.exp(a_log.double()) * soft
    beta = torch.sigmoid(b.double())
    one = 8 * 2.0 ** -22
    for i in range(n):
        e = torch.exp(g[i])[:, None, None]
        S = S * e
        u = beta[i][:, None] * (v[i].double() - (S * kn[i][..., None]).sum(1))
        S = S + kn[i][..., None] * u[:, None]
        size = S.square().sum(1, keepdim=True).sqrt() + v[i].double().abs()[:, None]
        E = E * e + one * size
        out[i] = scale * (S * qn[i][..., None]).sum(1)
        near[i] = abs(scale) * (E + one * size)[:, 0]
    bound = near + _half(out) * (1 + 2.0 ** -10)
    return out, bound, S, E.expand_as(S) + 2.0 ** -24 * S.abs() + 2.0 ** -140


def verify(x, counts, drafts, probs, heat, accept_u, sample_u):
    """(counts, tokens) lists, row by row in 64 bits."""
    at, kept, tokens = 0, [], []
    for s, n in enumerate(counts):
        out = [-1] * n
        keep = 0
        t = float(heat[s]) if heat is not None else 1.0
        for i in range(n):
            row = at + i
            y = x[row].double()
            keep = i + 1
            if bool(torch.isnan(y).any()) or bool((y == math.inf).any()) or float(y.max()) == -math.inf:
                break
            d, last = int(drafts[row]), i == n - 1
            best = int(torch.nonzero(y == y.max())[0])
            if t <= 0:
                if not last and d == best:
                    out[i] = d
                    continue
                out[i] = best
                break
            p = torch.exp((y - y.max()) / t)
            p[y == -math.inf] = 0.0
            p = p / p.sum()
            w = p
            if not last:
                if 0 <= d < y.numel():
                    qd = float(probs[row, d]) if probs is not None else 1.0
                    if float(accept_u[row]) * qd < float(p[d]):
                        out[i] = d
                        continue
                if probs is not None:
                    w = (p - probs[row].double()).clamp(min=0)
                elif 0 <= d < y.numel():
                    w = p.clone()
                    w[d] = 0.0
                if float(w.sum()) <= 0:
                    w = p
            total = torch.cumsum(w, 0)
            over = torch.nonzero((total > float(sample_u[s]) * float(total[-1])) & (w > 0))
            out[i] = int(over[0]) if len(over) else int(torch.nonzero(w > 0)[-1])
            break
        kept.append(keep)
        tokens += out
        at += n
    return kept, tokens

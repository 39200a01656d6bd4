"""Plain 64-bit forms of the operators for many sequences, and the bounds their
kernels' outputs are held to."""
import math

import torch


def offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def make_cache(lengths, hkv, page, d, seed, spare=3, width=None, fill=None):
    """(k, v, table, lengths) with the pages handed out in no order and table
    entries past a sequence's last page outside the pool.  Rows that no sequence
    keeps hold `fill` (N(0, 1) where None)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + spare
    width = max([1] + need) if width is None else width
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    table[:, 1::2] = pool + 1000
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    k, v = (torch.randn((pool, hkv, page, d), generator=g, device="cuda", dtype=torch.float16)
            for _ in range(2))
    if fill is not None:
        keep = torch.zeros((pool, page), dtype=torch.bool)
        for s, n in enumerate(lengths):
            for b in range(need[s]):
                keep[table[s, b], :min(page, n - b * page)] = True
        dead = ~keep.cuda()[:, None, :, None]
        k.masked_fill_(dead, fill)
        v.masked_fill_(dead, fill)
    return k, v, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")


def gather(pages, table, s, n):
    """The first n positions of sequence s, [n][hkv][d]."""
    page = pages.shape[2]
    ids = table[s, :-(-n // page)].long()
    return pages[ids].transpose(1, 2).reshape(-1, pages.shape[1], pages.shape[3])[:n]


def attend(q, k, v, scale, causal):
    """(out, absolute) in 64 bits of q [n][hq][d] over k, v [m][hkv][d]: the
    attention and, for the bound, the same weights over |v|.  Causal: the queries
    are the last n of the m positions.  A row that sees nothing is 0."""
    n, hq, d = q.shape
    m, group = k.shape[0], hq // k.shape[1]
    out, mass = (torch.zeros((n, hq, d), dtype=torch.float64, device="cuda") for _ in range(2))
    for h in range(hq):
        for i0 in range(0, n, 2048):
            i1 = min(n, i0 + 2048)
            sees = m - n + i1 if causal else m
            if sees <= 0:
                continue
            kh, vh = k[:sees, h // group].double(), v[:sees, h // group].double()
            x = q[i0:i1, h].double() @ kh.T.contiguous() * scale
            if causal:
                last = torch.arange(m - n + i0, m - n + i1, device="cuda")[:, None]
                x = x.masked_fill(torch.arange(sees, device="cuda")[None] > last, -math.inf)
                blind = (last < 0).expand(-1, d)
            p = torch.softmax(x, -1)
            # what a row does not see does not reach it, infinities and NaN included
            odd = ~torch.isfinite(vh).all(1)
            a, b = p @ vh.masked_fill(odd[:, None], 0.0), p @ vh.abs().masked_fill(odd[:, None], 0.0)
            for j in odd.nonzero()[:, 0].tolist():
                sees_j = ~torch.isneginf(x[:, j])[:, None]
                a = torch.where(sees_j, a + p[:, j:j + 1] * vh[j], a)
                b = torch.where(sees_j, b + p[:, j:j + 1] * vh[j].abs(), b)
            if causal:
                a, b = a.masked_fill(blind, 0.0), b.masked_fill(blind, 0.0)
            out[i0:i1, h], mass[i0:i1, h] = a, b
    return out, mass


def check_attention(got, want, mass):
    """The output's rounding to fp16 (2^-11 of it), the weights' (2^-11 of what
    they carry of |v|), and half as much again for scores, exponentials and sums in
    32 bits; NaN and infinities where the reference has them."""
    got = got.double()
    same = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), same), "other rows are not finite"
    bound = 2.0 ** -11 * want.abs() + 1.5 * 2.0 ** -11 * mass + 2.0 ** -24
    worst = torch.where(same, (got - want).abs() / bound, 0.0).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{worst:.2f} times the bound"


def axis_of_pair(half, sections, interleaved):
    axes = len(sections)
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [j % axes if j < axes * sections[j % axes] else 0 for j in range(half)]


def rotate(x, cos, sin, rows, axis):
    """x [n][heads][d] turned by the table rows `rows` [axes][n], in 64 bits, with
    the bound of the fp16 result."""
    half = cos.shape[1]
    c, z = (torch.stack([t[rows[a].long(), j] for j, a in enumerate(axis)], -1).double()[:, None]
            for t in (cos, sin))
    y = x.double().clone()
    a, b = y[..., :half].clone(), y[..., half:2 * half].clone()
    y[..., :half], y[..., half:2 * half] = a * c - b * z, a * z + b * c
    # two products and a sum in 32 bits, then fp16 (2^-25: half its smallest step)
    near = torch.zeros_like(y)
    near[..., :half] = 2.0 ** -22 * ((a * c).abs() + (b * z).abs())
    near[..., half:2 * half] = 2.0 ** -22 * ((a * z).abs() + (b * c).abs())
    near[..., :2 * half] += 2.0 ** -11 * y[..., :2 * half].abs() + 2.0 ** -25
    return y, near


def logprobs(x, tokens, top):
    """(logprob, entropy, ids, values) of rows x in 64 bits."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    ln = torch.log(z)
    lp = (x - m) - ln
    entropy = ln[:, 0] - torch.where(e > 0, e * (x - m), 0.0).sum(-1) / z[:, 0]
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
    t = tokens.long().clamp(0, x.shape[1] - 1)[:, None]
    return lp.gather(1, t)[:, 0], entropy, order.int(), lp.gather(1, order)

"""Short convolution, gated delta rule, gated norm and the verification of drafted
tokens against plain forms in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

import recurrent_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def aexq():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from aiimage_amd import aexq as mod
    return mod


@pytest.fixture(scope="module")
def ctx(aexq):
    c = aexq.Context(0)
    yield c
    torch.cuda.synchronize()
    c.close()


class Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def f32(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def f16(self, *shape):
        return self.f32(*shape).half()

    def u(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")


# ---------------------------------------------------------------- short convolution

@pytest.mark.parametrize("lens,channels,width,bias,silu", [
    ([1], 8, 2, False, True), ([1, 1, 1], 2056, 4, False, True), ([3, 0, 17, 16, 1], 40, 4, True, True),
    ([33, 2, 200], 1000, 3, False, False), ([15, 16, 17, 31, 32, 33], 72, 5, True, True),
    ([700], 6144, 4, False, True), ([2] * 130, 16, 4, True, False)])
def test_short_conv(aexq, ctx, lens, channels, width, bias, silu):
    """States in no order, sequences that begin, that have no slot, rows behind the last."""
    print(f"[gpu-case] conv {lens[:8]} channels={channels} width={width}", flush=True)
    r, n, total = Draw(1), len(lens), sum(lens)
    wide = r.f16(total + 3, channels + 16)
    x = wide[:, 8:8 + channels]
    weight = r.f32(channels, width)
    b = r.f32(channels) if bias else None
    slot = [(5 * i + 2) % (n + 2) if i % 4 != 3 else (-1 if i % 8 == 3 else n + 9) for i in range(n)]
    slot = [s if s in (-1, n + 9) or slot.index(s) == i else -7 for i, s in enumerate(slot)]
    past = [0 if i % 3 == 1 else 100 + i for i in range(n)]
    state = r.f16(n + 2, width - 1, channels)
    before, out = state.clone(), torch.full((total + 3, channels), 7.0, device="cuda").half()
    slots = aexq.slots(n + 2, n, slot=ref.i32(slot),
                       lengths=ref.i32([p + m for p, m in zip(past, lens)]))
    ctx.short_conv(slots, state, ref.offsets(lens), x, weight, out, bias=b, silu=silu)
    torch.cuda.synchronize()
    at, want = 0, before.clone()
    for i, m in enumerate(lens):
        inside = 0 <= slot[i] < n + 2
        begin = torch.zeros_like(before[0]) if past[i] == 0 or not inside else before[slot[i]]
        y, near, left = ref.short_conv(x[at:at + m], begin, weight, b, silu)
        ref.check(out[at:at + m], y, near, f"sequence {i}")
        if inside and m:
            want[slot[i]] = left
        at += m
    assert torch.equal(state, want)
    assert (out[total:] == 7).all()


@pytest.mark.parametrize("lens", [[5, 3, 1, 4], [40, 2, 17, 19]])
def test_short_conv_of_some_rows(aexq, ctx, lens):
    """counts: the first rows alone, none of one sequence; states read only; no output."""
    print(f"[gpu-case] conv of some rows of {lens}", flush=True)
    r, n, c = Draw(2), len(lens), 64
    kept = [lens[0], 0, 1, lens[3] - 1]
    x, weight, state = r.f16(sum(lens), c), r.f32(c, 4), r.f16(n, 3, c)
    before, off = state.clone(), ref.offsets(lens)
    counts = ref.i32(kept)
    out = torch.full_like(x, 7.0)
    ctx.short_conv(aexq.slots(n, n, counts=counts, read_only=True), state, off, x, weight, out)
    torch.cuda.synchronize()
    assert torch.equal(state, before)
    ctx.short_conv(aexq.slots(n, n, counts=counts), state, off, x, weight, None)
    torch.cuda.synchronize()
    at = 0
    for i, m in enumerate(lens):
        y, near, left = ref.short_conv(x[at:at + kept[i]], before[i], weight, None, True)
        ref.check(out[at:at + kept[i]], y, near)
        assert (out[at + kept[i]:at + m] == 7).all()
        assert torch.equal(state[i], left)
        at += m
    # counts past a sequence's rows are all of them, below 0 none
    state.copy_(before)
    ctx.short_conv(aexq.slots(n, n, counts=ref.i32([1 << 30, -5, 0, 2])), state, off, x, weight, out)
    torch.cuda.synchronize()
    assert torch.equal(state[0], torch.cat([before[0], x[:lens[0]]])[-3:])
    assert torch.equal(state[1:3], before[1:3])


@pytest.mark.parametrize("bad", [INF, NAN])
def test_short_conv_odd_values_stay_in_reach(aexq, ctx, bad):
    print(f"[gpu-case] conv odd values {bad}", flush=True)
    r, c = Draw(3), 24
    x, weight, state = r.f16(60, c), r.f32(c, 4), r.f16(2, 3, c)
    x[20, 5] = bad
    out = torch.zeros_like(x)
    ctx.short_conv(aexq.slots(2, 2), state, ref.offsets([30, 30]), x, weight, out, silu=False)
    torch.cuda.synchronize()
    odd = torch.zeros_like(x, dtype=torch.bool)
    odd[20:24, 5] = True
    assert torch.equal(~torch.isfinite(out), odd)


# ---------------------------------------------------------------- gated delta rule

def _inputs(r, n, hk, hv, dk, dv, view=True):
    wide = r.f16(n, 2 * hk * dk + hv * dv + 24)
    q = wide[:, 8:8 + hk * dk].unflatten(1, (hk, dk))
    k = wide[:, 8 + hk * dk:8 + 2 * hk * dk].unflatten(1, (hk, dk))
    v = wide[:, 8 + 2 * hk * dk:8 + 2 * hk * dk + hv * dv].unflatten(1, (hv, dv))
    ab = r.f16(n, 2 * hv + 3)
    if not view:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    return dict(q=q, k=k, v=v, a=ab[:, 1:1 + hv], b=ab[:, 1 + hv:1 + 2 * hv],
                a_log=r.f32(hv), dt_bias=r.f32(hv) - 1.5)


def _rows(d, at):
    return {x: y if x in ("a_log", "dt_bias") else y[at] for x, y in d.items()}


def _check_delta(d, lens, kept, begin, out, state, slot, scale, eps, hv, what=""):
    at = 0
    for i, m in enumerate(lens):
        if kept[i]:
            y, near, S, err = ref.delta(**_rows(d, slice(at, at + kept[i])), state=begin[i],
                                        scale=scale, eps=eps)
            if out is not None:
                ref.check(out[at:at + kept[i]], y, near, f"{what} sequence {i}")
            if slot[i] is not None:
                ref.check(state[slot[i]], S, err, f"{what} state {i}")
        if out is not None:
            assert (out[at + kept[i]:at + m] == 7).all()
        at += m


SHAPES = [([1], 1, 1, 128, 128), ([33], 2, 4, 128, 128), ([64, 65, 0, 63], 2, 2, 64, 64),
          ([1, 2, 3, 5], 1, 3, 128, 64), ([200, 7, 129], 2, 2, 128, 256), ([130, 300], 1, 2, 64, 256),
          ([500], 1, 1, 128, 128), ([16, 17, 15, 31, 48], 3, 6, 64, 128), ([2] * 70, 1, 1, 64, 64)]


@pytest.mark.parametrize("lens,hk,hv,dk,dv", SHAPES)
def test_delta_prompt(aexq, ctx, lens, hk, hv, dk, dv):
    """States in no order, sequences that begin or have no slot, rows behind the last."""
    print(f"[gpu-case] delta prompt {lens[:8]} {hk}/{hv} {dk}x{dv}", flush=True)
    r, n, total = Draw(4), len(lens), sum(lens)
    d = _inputs(r, total + 2, hk, hv, dk, dv)
    state = r.f32(n + 2, hv, dk, dv)
    before = state.clone()
    slot = [n + 1 - i if i % 4 != 3 else (-1 if i % 8 == 3 else n + 9) for i in range(n)]
    past = [0 if i % 3 == 1 else 50 for i in range(n)]
    out = torch.full((total + 2, hv, dv), 7.0, device="cuda").half()
    slots = aexq.slots(n + 2, n, slot=ref.i32(slot),
                       lengths=ref.i32([p + m for p, m in zip(past, lens)]))
    ctx.delta_prompt(slots, state, ref.offsets(lens), **d, out=out, scale=dk ** -0.5, eps=1e-6)
    torch.cuda.synchronize()
    inside = [0 <= s < n + 2 for s in slot]
    begin = [before[s] if ok and p else torch.zeros_like(before[0])
             for s, p, ok in zip(slot, past, inside)]
    _check_delta(d, lens, lens, begin, out[:total], state,
                 [s if ok else None for s, ok in zip(slot, inside)], dk ** -0.5, 1e-6, hv)
    assert (out[total:] == 7).all()
    used = [s for s, ok, m in zip(slot, inside, lens) if ok and m]
    for s in range(n + 2):
        if s not in used:
            assert torch.equal(state[s], before[s]), f"state {s} is no sequence's"


@pytest.mark.parametrize("lens,hk,hv,dk,dv", [([5, 3, 1, 4], 2, 2, 128, 128),
                                              ([70, 2, 130, 66], 1, 2, 64, 128)])
def test_delta_of_some_rows(aexq, ctx, lens, hk, hv, dk, dv):
    """counts, as the verification of drafts leaves them: the first rows alone, none of
    one sequence; states read only; no output."""
    print(f"[gpu-case] delta of some rows of {lens}", flush=True)
    r, n = Draw(5), len(lens)
    kept = [lens[0], 0, 1, lens[3] - 1]
    d = _inputs(r, sum(lens), hk, hv, dk, dv)
    state = r.f32(n, hv, dk, dv)
    before, off, counts = state.clone(), ref.offsets(lens), ref.i32(kept)
    out = torch.full((sum(lens), hv, dv), 7.0, device="cuda").half()
    args = dict(scale=0.1, eps=1e-6)
    ctx.delta_prompt(aexq.slots(n, n, counts=counts, read_only=True), state, off, **d, out=out, **args)
    torch.cuda.synchronize()
    assert torch.equal(state, before)
    ctx.delta_prompt(aexq.slots(n, n, counts=counts), state, off, **d, out=None, **args)
    torch.cuda.synchronize()
    _check_delta(d, lens, kept, before, out, state, range(n), 0.1, 1e-6, hv)
    assert torch.equal(state[1], before[1])


@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 256)])
@pytest.mark.parametrize("cut", [1, 64, 77, 150])
def test_delta_in_two_calls(aexq, ctx, dk, dv, cut):
    """A prompt in two pieces, the second from the state the first one left."""
    print(f"[gpu-case] delta in two calls at {cut} {dk}x{dv}", flush=True)
    r, n = Draw(6), 200
    d = _inputs(r, n, 1, 2, dk, dv)
    state = r.f32(1, 2, dk, dv)
    before, slots = state.clone(), aexq.slots(1, 1)
    out = torch.full((n, 2, dv), 7.0, device="cuda").half()
    for a, b in ((0, cut), (cut, n)):
        ctx.delta_prompt(slots, state, ref.offsets([b - a]), **_rows(d, slice(a, b)), out=out[a:b],
                         scale=0.2)
    torch.cuda.synchronize()
    _check_delta(d, [n], [n], before, out, state, [0], 0.2, 1e-6, 2)


@pytest.mark.parametrize("kind", ["reset", "keep", "mixed", "closed", "open"])
def test_delta_gates_at_their_ends(aexq, ctx, kind):
    """Decays that are 0 or 1, strengths that are 0 or 1, gates of infinity."""
    print(f"[gpu-case] delta gates {kind}", flush=True)
    r, n, hv, dk, dv = Draw(7), 150, 2, 128, 64
    d = _inputs(r, n, 2, hv, dk, dv)
    d["a"], d["b"] = d["a"].contiguous(), d["b"].contiguous()
    if kind == "reset":
        d["a"].fill_(60000.0)
    elif kind == "keep":
        d["a"].fill_(-60000.0)
    elif kind == "mixed":
        d["a"][::7] = INF
        d["a"][3::11] = -INF
        d["a"][5::13] = 1000.0
    elif kind == "closed":
        d["b"].fill_(-60000.0)
    else:
        d["b"].fill_(INF)
        d["a"].fill_(-9.0)
    state = r.f32(1, hv, dk, dv)
    before = state.clone()
    out = torch.full((n, hv, dv), 7.0, device="cuda").half()
    ctx.delta_prompt(aexq.slots(1, 1), state, ref.offsets([n]), **d, out=out, scale=0.09)
    torch.cuda.synchronize()
    _check_delta(d, [n], [n], before, out, state, [0], 0.09, 1e-6, hv, kind)


@pytest.mark.parametrize("what", ["same", "opposite", "tiny", "huge", "zero", "values"])
def test_delta_keys_that_repeat_and_sizes(aexq, ctx, what):
    """One key over and over (a chunk's rows then correct one another most), keys far
    below eps and near fp16's end, values of 60000 beside ones of 1e-6."""
    print(f"[gpu-case] delta keys {what}", flush=True)
    r, n, hv, dk, dv = Draw(8), 140, 2, 64, 128
    d = _inputs(r, n, 2, hv, dk, dv, view=False)
    d["a"], d["b"] = torch.full_like(d["a"], -8.0), torch.full_like(d["b"], 6.0)
    if what == "same":
        d["k"][:] = d["k"][:1].clone()
    elif what == "opposite":
        d["k"][:] = d["k"][:1].clone()
        d["k"][::2] *= -1
    elif what == "tiny":
        d["k"].mul_(1e-6)
        d["q"].mul_(1e-5)
    elif what == "huge":
        d["k"].mul_(12000.0).clamp_(-60000, 60000)
        d["q"].mul_(12000.0).clamp_(-60000, 60000)
    elif what == "zero":
        d["k"][::3] = 0
        d["q"][::5] = 0
    else:
        d["v"][:, :, ::2] *= 1e-6
        d["v"][:, :, 1::2] = d["v"][:, :, 1::2].clamp(-3, 3) * 20000
    state = 1e-3 * r.f32(1, hv, dk, dv)
    before = state.clone()
    out = torch.full((n, hv, dv), 7.0, device="cuda").half()
    ctx.delta_prompt(aexq.slots(1, 1), state, ref.offsets([n]), **d, out=out, scale=0.1)
    torch.cuda.synchronize()
    _check_delta(d, [n], [n], before, out, state, [0], 0.1, 1e-6, hv, what)


# (an infinite gate is a gate)
@pytest.mark.parametrize("where,bad", [(w, b) for w in ("v", "k", "q", "state") for b in (INF, -INF, NAN)]
                         + [("a", NAN), ("b", NAN)])
def test_delta_odd_values_reach_only_what_follows(aexq, ctx, where, bad):
    """A value that is not finite in row 70 of the first sequence: rows before it, other
    heads and sequences and, of v, other columns are as without it."""
    print(f"[gpu-case] delta odd {where} {bad}", flush=True)
    r, lens, hv, dk, dv, at = Draw(9), [100, 30], 2, 128, 64, 70
    d = _inputs(r, 130, 2, hv, dk, dv, view=False)
    d["a"], d["b"] = d["a"].contiguous(), d["b"].contiguous()
    state = r.f32(2, hv, dk, dv)
    clean, begin = {x: y.clone() for x, y in d.items()}, state.clone()
    if where == "state":
        state[0, 1, 3, 5], at = bad, 0
    else:
        t = d[where]
        if t.dim() == 3:
            t[at, 1, 5] = bad
        else:
            t[at, 1] = bad
    out = torch.zeros((130, hv, dv), device="cuda").half()
    ctx.delta_prompt(aexq.slots(2, 2), state, ref.offsets(lens), **d, out=out, scale=0.1)
    torch.cuda.synchronize()
    odd = torch.zeros_like(out, dtype=torch.bool)
    odd_state = torch.zeros_like(state, dtype=torch.bool)
    if where == "q":
        odd[at, 1] = True
    elif where in ("v", "state"):
        odd[at:100, 1, 5] = True
        odd_state[0, 1, :, 5] = True
    else:
        odd[at:100, 1] = True
        odd_state[0, 1] = True
    got = ~torch.isfinite(out)
    assert torch.equal(got, odd), "other outputs are not finite"
    assert torch.equal(~torch.isfinite(state), odd_state), "other states are not finite"
    first = 0
    for i, m in enumerate(lens):
        y, near, S, err = ref.delta(**_rows(clean, slice(first, first + m)), state=begin[i], scale=0.1,
                                    eps=1e-6)
        o = odd[first:first + m]
        ref.check(out[first:first + m].masked_fill(o, 0), y.masked_fill(o, 0), near)
        ref.check(state[i].masked_fill(odd_state[i], 0), S.masked_fill(odd_state[i], 0), err)
        first += m


@pytest.mark.parametrize("n,hk,hv,dk,dv", [(1, 1, 1, 128, 128), (3, 2, 6, 128, 64), (40, 4, 8, 64, 256),
                                           (9, 16, 16, 128, 128), (65, 3, 3, 64, 64),
                                           (20, 16, 32, 128, 256)])
def test_delta_decode(aexq, ctx, n, hk, hv, dk, dv):
    print(f"[gpu-case] delta decode {n} {hk}/{hv} {dk}x{dv}", flush=True)
    r = Draw(10)
    d = _inputs(r, n, hk, hv, dk, dv)
    state = r.f32(n + 2, hv, dk, dv)
    before = state.clone()
    slot = [n + 1 - i if i % 5 != 4 else -1 for i in range(n)]
    past = [0 if i % 3 == 1 else 50 for i in range(n)]
    kept = [0 if i % 7 == 6 else 1 for i in range(n)]
    out = torch.full((n, hv, dv), 7.0, device="cuda").half()
    slots = aexq.slots(n + 2, n, slot=ref.i32(slot), lengths=ref.i32([p + 1 for p in past]),
                       counts=ref.i32(kept))
    ctx.delta_decode(slots, state, **d, out=out, scale=dk ** -0.5)
    torch.cuda.synchronize()
    begin = [before[s] if s >= 0 and p else torch.zeros_like(before[0]) for s, p in zip(slot, past)]
    _check_delta(d, [1] * n, kept, begin, out, state, [s if s >= 0 else None for s in slot],
                 dk ** -0.5, 1e-6, hv)
    used = [s for s, m in zip(slot, kept) if s >= 0 and m]
    for s in range(n + 2):
        if s not in used:
            assert torch.equal(state[s], before[s])


def test_delta_decode_read_only_and_states_alone(aexq, ctx):
    print("[gpu-case] delta decode read only, states alone", flush=True)
    r, n, hv, dk, dv = Draw(11), 5, 2, 128, 128
    d = _inputs(r, n, 2, hv, dk, dv)
    state = r.f32(n, hv, dk, dv)
    before = state.clone()
    out = torch.full((n, hv, dv), 7.0, device="cuda").half()
    ctx.delta_decode(aexq.slots(n, n, read_only=True), state, **d, out=out, scale=0.1)
    torch.cuda.synchronize()
    assert torch.equal(state, before)
    ctx.delta_decode(aexq.slots(n, n), state, **d, out=None, scale=0.1)
    torch.cuda.synchronize()
    _check_delta(d, [1] * n, [1] * n, before, out, state, range(n), 0.1, 1e-6, hv)


def test_delta_offsets_out_of_range(aexq, ctx):
    """Offsets that reach past the tokens or go back are kept within them."""
    print("[gpu-case] delta offsets out of range", flush=True)
    r, hv, dk, dv = Draw(12), 1, 64, 64
    d = _inputs(r, 80, 1, hv, dk, dv)
    state = r.f32(3, hv, dk, dv)
    before = state.clone()
    out = torch.full((80, hv, dv), 7.0, device="cuda").half()
    off = ref.i32([-5, 30, 20, 1 << 30])
    ctx.delta_prompt(aexq.slots(3, 3), state, off, **d, out=out, scale=0.1)
    x, conv = r.f16(80, 16), r.f16(3, 3, 16)
    ctx.short_conv(aexq.slots(3, 3), conv, off, x, r.f32(16, 4), torch.zeros_like(x))
    torch.cuda.synchronize()
    assert torch.equal(state[1], before[1])
    assert torch.isfinite(out).all()


# ---------------------------------------------------------------- gated norm

@pytest.mark.parametrize("tokens,heads,dim,gamma", [
    (1, 1, 8, True), (3, 5, 64, False), (17, 16, 128, True), (7, 3, 200, True), (2, 2, 512, True),
    (129, 4, 256, False), (5, 1, 264, True), (1000, 7, 96, True)])
def test_gated_rmsnorm(ctx, tokens, heads, dim, gamma):
    print(f"[gpu-case] gated norm {tokens} x {heads} x {dim}", flush=True)
    r = Draw(13)
    wide = r.f16(tokens, heads * dim + 8)
    x, z = wide[:, 8:].unflatten(1, (heads, dim)), 3 * r.f16(tokens, heads, dim)
    x[0, 0] *= 1e-3
    if tokens > 2:
        x[1], z[2] = 0, 0
    g = 1 + 0.3 * r.f32(dim) if gamma else None
    y, near = ref.gated_norm(x, z, g, 1e-6)
    out = torch.full((tokens, heads, dim), 7.0, device="cuda").half()
    ctx.gated_rmsnorm(x, z, g, out)
    torch.cuda.synchronize()
    ref.check(out, y, near)
    for which in ("x", "z"):     # in place
        a, b = x.clone(), z.clone()
        ctx.gated_rmsnorm(a, b, g, a if which == "x" else b)
        torch.cuda.synchronize()
        assert torch.equal(a if which == "x" else b, out)


def test_gated_rmsnorm_odd_values_stay_in_their_row(ctx):
    print("[gpu-case] gated norm odd values", flush=True)
    r = Draw(14)
    x, z = r.f16(6, 3, 128), r.f16(6, 3, 128)
    x[2, 1, 7], z[4, 0, 9], z[5, 2, 3] = NAN, INF, -60000.0
    out = torch.zeros_like(x)
    ctx.gated_rmsnorm(x, z, None, out)
    torch.cuda.synchronize()
    odd = torch.zeros_like(x, dtype=torch.bool)
    odd[2, 1], odd[4, 0, 9] = True, True
    assert torch.equal(~torch.isfinite(out), odd)
    assert out[5, 2, 3].item() == 0.0


# ---------------------------------------------------------------- drafted tokens

def _verify(aexq, ctx, x, lens, drafts, probs, heat, au, su, tail=0):
    counts = torch.full((len(lens),), 77, dtype=torch.int32, device="cuda")
    tokens = torch.full((x.shape[0],), 77, dtype=torch.int32, device="cuda")
    ctx.verify_drafts(aexq.describe(x, *x.shape), ref.offsets(lens), drafts, au, su, counts, tokens,
                      temperature=heat, draft_probs=probs)
    torch.cuda.synchronize()
    want = ref.verify(x, lens, drafts, probs, heat, au, su)
    assert counts.tolist() == want[0]
    n = sum(lens)
    assert tokens[:n].tolist() == want[1]
    assert (tokens[n:] == 77).all()
    return want


@pytest.mark.parametrize("lens,vocab,dtype,with_probs,heat", [
    ([1], 5, "f32", False, None), ([5], 151936, "f32", False, "mixed"), ([3, 1, 0, 9], 1001, "f16", True, "mixed"),
    ([2] * 67, 333, "f32", True, None), ([40, 7], 4099, "f16", False, "cold"),
    ([4, 4, 4], 70000, "f32", True, "mixed"), ([6] * 20, 50, "f32", True, "hot")])
def test_verify(aexq, ctx, lens, vocab, dtype, with_probs, heat):
    print(f"[gpu-case] verify {lens[:6]} vocab={vocab} {dtype} {heat}", flush=True)
    r, n = Draw(15), sum(lens) + 2
    x = 2 * r.f32(n, vocab)
    x = x.half() if dtype == "f16" else x
    x[:, ::7] = -INF
    probs = None
    if with_probs:
        probs = torch.softmax(x.float() + 0.5 * r.f32(n, vocab), -1)
        drafts = torch.multinomial(probs, 1, generator=r.g)[:, 0].int()
    else:
        drafts = torch.where(r.u(n) < 0.8, x.argmax(-1), (vocab * r.u(n)).long()).int()
    temperature = {"mixed": 0.6 * r.u(len(lens)).mul(3).round(), "cold": torch.zeros(len(lens), device="cuda"),
                   "hot": torch.full((len(lens),), INF, device="cuda"), None: None}[heat]
    _verify(aexq, ctx, x, lens, drafts, probs, temperature, r.u(n), r.u(len(lens)))


def test_verify_at_the_borders(aexq, ctx):
    """Numbers of 0 and just below 1, drafts of probability 0 and outside the vocabulary,
    drafts as likely as the target's, draft probabilities that leave nothing."""
    print("[gpu-case] verify at the borders", flush=True)
    r, vocab = Draw(16), 700
    lens = [2] * 8
    x = r.f32(16, vocab)
    x[:, -5:] = -INF
    probs = torch.softmax(x, -1)
    drafts = ref.i32([3, 0, vocab - 1, 0, -4, 0, vocab, 0, 5, 0, 6, 0, 7, 0, 8, 0])
    below = 1 - 2.0 ** -24
    au = torch.tensor([0.0, 0, 0, 0, 0, 0, 0, 0, below, 0, below, 0, 0.5, 0, 0.5, 0], device="cuda")
    su = torch.tensor([0.0, below, 0.5, 0.0, below, 0.0, below, 0.3], device="cuda")
    _verify(aexq, ctx, x, lens, drafts, None, None, au, su)
    probs[8:12] = 0.0               # a draft of probability 0 that the target takes
    probs[12:14] = 3.0              # more than the target's everywhere: nothing is left
    _verify(aexq, ctx, x, lens, drafts, probs, None, au, su)


def test_verify_rows_without_probabilities(aexq, ctx):
    print("[gpu-case] verify rows without probabilities", flush=True)
    r, vocab = Draw(17), 5000
    lens = [2, 3, 1, 2, 1, 2]
    x = r.f32(11, vocab)
    x[0, 9], x[3, 70], x[5], x[7] = NAN, INF, -INF, -INF
    x[8, 4321] = NAN
    drafts = x.nan_to_num(-1.0, 0.0, -1.0).argmax(-1).int()
    for heat in (None, torch.zeros(6, device="cuda")):
        want = _verify(aexq, ctx, x, lens, drafts, None, heat, torch.zeros(11, device="cuda"), r.u(6))
        assert want[1][0] == -1 and want[1][5] == -1


@pytest.mark.parametrize("scale", [1e-30, 1e30, 3e38])
def test_verify_logits_of_any_size(aexq, ctx, scale):
    """Logits whose differences are past exp's range, and temperatures to match."""
    print(f"[gpu-case] verify logits of size {scale}", flush=True)
    r, vocab = Draw(18), 3000
    x = (r.u(12, vocab) * 2 - 1) * scale
    drafts = x.argmax(-1).int()
    heat = torch.tensor([scale, scale / 10, 1.0], device="cuda")
    _verify(aexq, ctx, x, [4, 4, 4], drafts, None, heat, r.u(12), r.u(3))


def test_verify_numbers_beside_borders(aexq, ctx):
    """A flat row of 151936 logits: the numbers lie 2^-26 of the sum beside the borders
    between two tokens, nearer than 32-bit sums place them."""
    print("[gpu-case] verify beside borders", flush=True)
    r, vocab, n = Draw(19), 151936, 24
    x = 0.5 * r.f32(n, vocab)
    p = torch.softmax(x.double(), -1).cumsum(-1)
    at = (vocab * r.u(n)).long()[:, None]
    edge = p.gather(1, at)[:, 0]
    su = (edge + torch.where(torch.arange(n, device="cuda") % 2 == 0, 1, -1) * 2.0 ** -26).float()
    _verify(aexq, ctx, x, [1] * n, torch.zeros(n, dtype=torch.int32, device="cuda"), None, None,
            r.u(n), su.clamp(0, 1 - 2.0 ** -24))

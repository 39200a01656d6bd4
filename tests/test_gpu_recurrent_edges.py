"""Edges of the recurrent layers' operators and of the verification of drafted tokens:
values that are not finite, gates and keys at the ends of their types, rows behind a
sequence's last, sequences of thousands of rows, numbers beside a border."""
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


def _randn(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def _rand(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(shape, generator=g, device="cuda")


def _inputs(n, hk, hv, dk, dv, seed=0):
    s = 100 * seed
    return dict(q=_randn(n, hk, dk, seed=s + 1).half(), k=_randn(n, hk, dk, seed=s + 2).half(),
                v=_randn(n, hv, dv, seed=s + 3).half(), a=_randn(n, hv, seed=s + 4).half(),
                b=_randn(n, hv, seed=s + 5).half(), a_log=_randn(hv, seed=s + 6),
                dt_bias=_randn(hv, seed=s + 7) - 1.5)


def _rows(d, at):
    return {x: y if x in ("a_log", "dt_bias") else y[at] for x, y in d.items()}


# ---------------------------------------------------------------- gated norm

@pytest.mark.parametrize("tokens,heads,dim", [(3, 2, 8), (5, 3, 64), (4, 2, 128), (6, 1, 200),
                                              (3, 2, 512), (9000, 4, 128)])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_gated_norm_of_rows_that_are_not_finite(ctx, tokens, heads, dim, bad):
    """The mean of a row with a NaN is NaN and so is all of it, its zeros and its small
    values as well; an infinity leaves zeros and a NaN in its own place.  No other row meets
    either."""
    print(f"[gpu-case] gated norm with {bad}: {tokens} x {heads} x {dim}", flush=True)
    x, z = _randn(tokens, heads, dim, seed=1).half(), 2 * _randn(tokens, heads, dim, seed=2).half()
    x[1, 0] *= 1e-6
    x[1, 0, ::2] = 0
    z[1, 0, 1::3] = 0
    clean, at = x.clone(), dim // 2 + 1
    x[1, 0, at] = bad
    gamma = 1 + 0.1 * _randn(dim, seed=3)
    outs = []
    for t in (clean, x):
        outs.append(torch.zeros_like(t))
        ctx.gated_rmsnorm(t, z, gamma, outs[-1])
    torch.cuda.synchronize()
    row = outs[1][1, 0].clone()
    if math.isnan(bad):
        assert torch.isnan(row).all()
    else:
        assert torch.isnan(row[at])
        row[at] = 0
        assert (row == 0).all()
    outs[1][1, 0] = outs[0][1, 0]
    assert torch.equal(*outs)


# ---------------------------------------------------------------- gated delta rule

@pytest.mark.parametrize("decode", [False, True])
def test_delta_decays_of_large_rates(aexq, ctx, decode):
    """a_log past the largest logarithm of fp32 with gates that undo it: e^a_log is an
    infinity and the softplus 0 in fp32, their product is neither.  (a, a_log and their
    sums are whole quarters: nothing is rounded before the exponential.)"""
    print(f"[gpu-case] delta rates past fp32 decode={decode}", flush=True)
    rates = [89.0, 100.0, 128.0, 95.5]
    n, hv, dk, dv = (40, 4, 64, 64) if decode else (90, 4, 64, 64)
    d = _inputs(n, 2, hv, dk, dv, seed=1)
    d["a_log"], d["dt_bias"] = torch.tensor(rates, device="cuda"), torch.zeros(hv, device="cuda")
    past = torch.tensor([2.0, 1.0, 0.5, -1.5, 8.0, 30.0, -4.0, 0.0], device="cuda").repeat(n // 8 + 1)
    d["a"] = (-d["a_log"][None] - past[:n, None]).half()
    if decode:
        state = _randn(n, hv, dk, dv, seed=2)
        before, out = state.clone(), torch.zeros((n, hv, dv), device="cuda").half()
        ctx.delta_decode(aexq.slots(n, n), state, **d, out=out, scale=0.2)
        spans = [slice(i, i + 1) for i in range(n)]
    else:
        state = _randn(2, hv, dk, dv, seed=2)
        before, out = state.clone(), torch.zeros((n, hv, dv), device="cuda").half()
        ctx.delta_prompt(aexq.slots(2, 2), state, ref.offsets([n - 9, 9]), **d, out=out, scale=0.2)
        spans = [slice(0, n - 9), slice(n - 9, n)]
    torch.cuda.synchronize()
    for i, r in enumerate(spans):
        y, near, S, err = ref.delta(**_rows(d, r), state=before[i], scale=0.2, eps=1e-6)
        ref.check(out[r], y, near, f"sequence {i}")
        ref.check(state[i], S, err, f"state {i}")


@pytest.mark.parametrize("eps", [1e-40, 1e-38, 1e-6])
@pytest.mark.parametrize("n", [9, 100])
def test_delta_keys_of_zero_beside_the_smallest_eps(aexq, ctx, n, eps):
    """Keys and queries of nothing but zeros have length 0 whatever eps is above 0, also
    where 1 / eps is past fp32."""
    print(f"[gpu-case] delta zero keys eps={eps}", flush=True)
    d = _inputs(n, 1, 2, 128, 64, seed=3)
    d["k"][::3], d["q"][::2] = 0, 0
    d["k"][4:7] = 0
    state = _randn(1, 2, 128, 64, seed=4)
    before, out = state.clone(), torch.zeros((n, 2, 64), device="cuda").half()
    ctx.delta_prompt(aexq.slots(1, 1), state, ref.offsets([n]), **d, out=out, scale=0.1, eps=eps)
    torch.cuda.synchronize()
    y, near, S, err = ref.delta(**d, state=before[0], scale=0.1, eps=eps)
    ref.check(out, y, near)
    ref.check(state[0], S, err)


@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
@pytest.mark.parametrize("n", [1000, 970])
def test_delta_odd_values_leave_other_columns_alone(aexq, ctx, n, dk, dv):
    """Values that are not finite in some rows of a long sequence, several in one block
    among them, and in its last: the outputs before them and every other column's, all of
    them, and the other columns' states have the bits that they have without."""
    print(f"[gpu-case] delta odd values in {n} rows {dk}x{dv}", flush=True)
    hv = 2
    d = _inputs(n, 1, hv, dk, dv, seed=5)
    d["a"] -= 2.0
    state = _randn(1, hv, dk, dv, seed=6)
    begin = state.clone()
    odd = {(1, 5): 130, (1, 7): 131, (1, 40): 131, (1, 3): 500, (1, 10): 514, (1, 11): 577,
           (1, 20): n - 1, (0, 9): n - 3, (0, 33): 0}
    runs = []
    for bad in (False, True):
        s, x = begin.clone(), dict(d, v=d["v"].clone())
        if bad:
            for i, ((h, c), t) in enumerate(odd.items()):
                x["v"][t, h, c] = (NAN, INF, -INF)[i % 3]
            s[0, 0, 3, 50] = NAN
        out = torch.zeros((n, hv, dv), device="cuda").half()
        ctx.delta_prompt(aexq.slots(1, 1), s, ref.offsets([n]), **x, out=out, scale=0.1)
        torch.cuda.synchronize()
        runs.append((out, s))
    (clean, clean_state), (out, left) = runs
    odd[0, 50] = 0
    good = torch.ones((hv, dv), dtype=torch.bool, device="cuda")
    y, near, _, _ = ref.delta(**d, state=begin[0], scale=0.1, eps=1e-6)
    for (h, c), t in odd.items():
        good[h, c] = False
        assert not torch.isfinite(out[t:, h, c]).any() and not torch.isfinite(left[0, h, :, c]).any()
        ref.check(out[:t, h, c], y[:t, h, c], near[:t, h, c], f"column {c} of head {h}")
        assert torch.equal(out[:t // 64 * 64, h, c], clean[:t // 64 * 64, h, c])
    assert torch.equal(out[:, good], clean[:, good])
    assert torch.equal(left[0].transpose(1, 2)[good], clean_state[0].transpose(1, 2)[good])


def test_delta_odd_values_in_every_column_and_without_outputs(aexq, ctx):
    """Each of 16 columns stops being finite in another block, two in the last: the states
    of a call that has no outputs are those of one that has, and a call that reads states
    alone leaves them."""
    print("[gpu-case] delta odd values in every column", flush=True)
    n, hv, dk, dv = 14 * 64 + 30, 1, 128, 64
    d = _inputs(n, 1, hv, dk, dv, seed=24)
    state = _randn(1, hv, dk, dv, seed=25)
    clean = torch.zeros((n, hv, dv), device="cuda").half()
    ctx.delta_prompt(aexq.slots(1, 1, read_only=True), state, ref.offsets([n]), **d, out=clean, scale=0.1)
    place = [min(64 * c + 5 * c, n - 1) for c in range(16)]
    for c, t in enumerate(place):
        d["v"][t, 0, 16 + c] = NAN
    y, near, _, _ = ref.delta(**dict(d, v=d["v"].nan_to_num(0.0)), state=state[0], scale=0.1, eps=1e-6)
    states, out = [], torch.zeros((n, hv, dv), device="cuda").half()
    for o, only in ((out, False), (None, False), (out.clone(), True)):
        s = state.clone()
        ctx.delta_prompt(aexq.slots(1, 1, read_only=only), s, ref.offsets([n]), **d, out=o, scale=0.1)
        torch.cuda.synchronize()
        states.append(s)
    assert torch.equal(states[2], state)
    for c, t in enumerate(place):
        assert not torch.isfinite(out[t:, 0, 16 + c]).any()
        ref.check(out[:t, 0, 16 + c], y[:t, 0, 16 + c], near[:t, 0, 16 + c], f"column {16 + c}")
        assert torch.equal(out[:t // 64 * 64, 0, 16 + c], clean[:t // 64 * 64, 0, 16 + c])
    odd = torch.zeros(dv, dtype=torch.bool, device="cuda")
    odd[16:32] = True
    assert torch.equal(out[..., ~odd], clean[..., ~odd])
    for s in states[:2]:
        assert torch.equal(~torch.isfinite(s), odd.expand_as(s))
    assert torch.equal(states[0][..., ~odd], states[1][..., ~odd])


def test_delta_odd_values_of_short_sequences(aexq, ctx):
    """The same where there are many sequences of a few rows each."""
    print("[gpu-case] delta odd values, short sequences", flush=True)
    n, m, hv, dk, dv = 60, 9, 4, 128, 128
    d = _inputs(n * m, 2, hv, dk, dv, seed=5)
    state = _randn(n, hv, dk, dv, seed=6)
    runs = []
    for bad in (False, True):
        s, x = state.clone(), dict(d, v=d["v"].clone())
        if bad:
            x["v"][3 * m + 4, 1, 7], x["v"][3 * m + 8, 1, 9], x["v"][59 * m, 0, 127] = NAN, INF, -INF
        out = torch.zeros((n * m, hv, dv), device="cuda").half()
        ctx.delta_prompt(aexq.slots(n, n), s, ref.offsets([m] * n), **x, out=out, scale=0.1)
        torch.cuda.synchronize()
        runs.append((out.view(n, m, hv, dv), s))
    (clean, clean_state), (out, left) = runs
    y, near, _, _ = ref.delta(**_rows(d, slice(3 * m, 4 * m)), state=state[3], scale=0.1, eps=1e-6)
    odd, odd_state = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(left, dtype=torch.bool)
    for s, t, h, c in ((3, 4, 1, 7), (3, 8, 1, 9), (59, 0, 0, 127)):
        odd[s, t:, h, c], odd_state[s, h, :, c] = True, True
        if t:
            ref.check(out[s, :t, h, c], y[:t, h, c], near[:t, h, c])
            out[s, :t, h, c] = clean[s, :t, h, c]
    assert torch.equal(~torch.isfinite(out), odd) and torch.equal(~torch.isfinite(left), odd_state)
    assert torch.equal(out.masked_fill(odd, 0), clean.masked_fill(odd, 0))
    assert torch.equal(left.masked_fill(odd_state, 0), clean_state.masked_fill(odd_state, 0))


@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 256)])
@pytest.mark.parametrize("n", [1, 16, 17, 18, 31, 32, 33, 40, 48, 49, 63, 65, 81, 90, 96, 100])
def test_delta_rows_behind_the_last_one(aexq, ctx, n, dk, dv):
    """Rows around a sequence's, more than a block of them, hold NaN: nothing of them is
    read, and their outputs stay."""
    print(f"[gpu-case] delta rows behind {n} {dk}x{dv}", flush=True)
    hk, hv, room = 1, 2, 130
    total = n + 2 * room
    d = _inputs(total, hk, hv, dk, dv, seed=7)
    here = slice(room, room + n)
    for x in ("q", "k", "v", "a", "b"):
        d[x][:room], d[x][room + n:] = NAN, NAN
    state = _randn(1, hv, dk, dv, seed=8)
    begin, out = state.clone(), torch.full((total, hv, dv), 7.0, device="cuda").half()
    ctx.delta_prompt(aexq.slots(1, 1), state, ref.offsets([n]) + room, **d, out=out, scale=0.1)
    torch.cuda.synchronize()
    y, near, S, err = ref.delta(**_rows(d, here), state=begin[0], scale=0.1, eps=1e-6)
    ref.check(out[here], y, near)
    ref.check(state[0], S, err)
    assert (out[:room] == 7).all() and (out[room + n:] == 7).all()


@pytest.mark.parametrize("lens,hk,hv,dk,dv", [([5000, 3001], 1, 2, 128, 128), ([4100], 2, 2, 64, 64)])
def test_delta_of_thousands_of_rows(aexq, ctx, lens, hk, hv, dk, dv):
    """Tens of blocks in turn, with decays that forget and decays that keep."""
    print(f"[gpu-case] delta of {lens} rows", flush=True)
    n = sum(lens)
    d = _inputs(n, hk, hv, dk, dv, seed=9)
    d["dt_bias"][0] = -7.0          # keeps some thousand rows
    state = _randn(len(lens), hv, dk, dv, seed=10)
    begin, out = state.clone(), torch.zeros((n, hv, dv), device="cuda").half()
    ctx.delta_prompt(aexq.slots(len(lens), len(lens)), state, ref.offsets(lens), **d, out=out,
                     scale=dk ** -0.5)
    torch.cuda.synchronize()
    at = 0
    for i, m in enumerate(lens):
        y, near, S, err = ref.delta(**_rows(d, slice(at, at + m)), state=begin[i], scale=dk ** -0.5,
                                    eps=1e-6)
        ref.check(out[at:at + m], y, near, f"sequence {i}")
        ref.check(state[i], S, err, f"state {i}")
        at += m


@pytest.mark.parametrize("n,drafted,hk,hv,dk,dv", [
    (3, 8, 2, 4, 128, 128), (1, 5, 4, 16, 128, 128), (48, 8, 2, 16, 128, 128),
    (20, 40, 4, 16, 128, 128),     # too long to go apart with their drafts, not without them
    (20, 100, 4, 16, 64, 256)])
def test_states_behind_accepted_rows_are_those_of_these_rows_alone(aexq, ctx, n, drafted, hk, hv, dk,
                                                                  dv):
    """Bit for bit, whichever kernels either call takes."""
    print(f"[gpu-case] accepted rows of {n} x {drafted} {hk}/{hv} {dk}x{dv}", flush=True)
    c = 2 * hk * dk + hv * dv
    g = torch.Generator().manual_seed(n + drafted)
    kept = [int(torch.randint(1, min(drafted, 20) + 1, (1,), generator=g)) for _ in range(n)]
    kept[0] = drafted
    x, w = _randn(n * drafted, c, seed=11).half(), _randn(c, 4, seed=12)
    d = _inputs(n * drafted, hk, hv, dk, dv, seed=13)
    gates = [d.pop(t) for t in ("a_log", "dt_bias")]
    conv, state = _randn(n, 3, c, seed=14).half(), _randn(n, hv, dk, dv, seed=15)
    rows = torch.cat([torch.arange(k, device="cuda") + drafted * s for s, k in enumerate(kept)])
    got = []
    for whole in (True, False):
        s, t = conv.clone(), state.clone()
        off = ref.offsets([drafted] * n if whole else kept)
        slots = aexq.slots(n, n, counts=ref.i32(kept) if whole else None)
        y, e = (x, d) if whole else (x[rows], {k: v[rows] for k, v in d.items()})
        ctx.short_conv(slots, s, off, y, w, None)
        ctx.delta_prompt(slots, t, off, **e, a_log=gates[0], dt_bias=gates[1], out=None, scale=0.1)
        torch.cuda.synchronize()
        got.append((s, t))
    assert torch.equal(got[0][0], got[1][0])
    assert torch.equal(got[0][1], got[1][1])


# ---------------------------------------------------------------- drafted tokens

def test_verify_numbers_next_to_a_border(aexq, ctx):
    """A flat row of 151936 logits, and for each row the two numbers of 32 bits on either
    side of a border between two tokens.  Weights within 2^-39 of theirs place the border,
    at most 1, within 2^-38 of its place; of 64 borders that one is taken whose nearer
    neighbour is nearest, but no nearer than 2^-36."""
    print("[gpu-case] verify numbers next to a border", flush=True)
    vocab, n, some = 151936, 12, 64
    x = 0.5 * _randn(n, vocab, seed=16)
    p = torch.softmax(x.double(), -1).cumsum(-1)
    p /= p[:, -1:].clone()
    at = (vocab * _rand(n, some, seed=17)).long().clamp(max=vocab - 2)
    border = p.gather(1, at)
    near = border.float()
    up = torch.where(near.double() > border, near, torch.nextafter(near, torch.full_like(near, 2.0)))
    down = torch.nextafter(up, torch.zeros_like(up))
    gap = torch.minimum(up.double() - border, border - down.double())
    pick = torch.where(gap >= 2.0 ** -36, gap, 1.0).argmin(-1, keepdim=True)
    at, up, down = (t.gather(1, pick)[:, 0] for t in (at, up, down))
    assert (gap.gather(1, pick) < 2.0 ** -27).all()
    for su, step in ((up, 1), (down, 0)):
        counts = torch.zeros(n, dtype=torch.int32, device="cuda")
        tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
        ctx.verify_drafts(aexq.describe(x, n, vocab), ref.offsets([1] * n),
                          torch.zeros(n, dtype=torch.int32, device="cuda"), _rand(n, seed=18), su,
                          counts, tokens)
        torch.cuda.synchronize()
        assert counts.tolist() == [1] * n
        assert tokens.tolist() == (at + step).tolist()


# ---------------------------------------------------------------- refusals

def test_outputs_over_inputs_are_refused(aexq, ctx):
    """out inside the rows of an input, by rows or by columns; beside them it may lie."""
    from aiimage_amd import _abi
    print("[gpu-case] outputs over inputs", flush=True)
    n, hk, hv, d = 20, 1, 2, 64
    wide = _randn(n + 1, 8 * d, seed=20).half()
    part = lambda at, h, row=0: wide[row:row + n, at * d:(at + h) * d].unflatten(1, (h, d))  # noqa: E731
    g = _inputs(n, hk, hv, d, d, seed=21)
    args = dict(q=part(0, hk), k=part(1, hk), v=part(2, hv), **{x: g[x] for x in ("a", "b", "a_log",
                                                                                   "dt_bias")}, scale=0.1)
    state, conv, w = _randn(n, hv, d, d, seed=22), _randn(1, 3, 2 * d, seed=23).half(), _randn(2 * d, 4)
    one, off, before = aexq.slots(n, 1), ref.offsets([n]), wide.clone()
    for at, row in ((0, 0), (1, 0), (2, 0), (3, 0), (2, 1), (0, 1)):
        with pytest.raises(_abi.ArgumentError, match="overlaps"):
            ctx.delta_prompt(one, state, off, **args, out=part(at, hv, row))
        with pytest.raises(_abi.ArgumentError, match="overlaps"):
            ctx.delta_decode(aexq.slots(n, n), state, **args, out=part(at, hv, row))
    x = wide[:n, 2 * d:4 * d]
    for out in (x, wide[1:, 2 * d:4 * d], wide[:n, 2 * d + 8:4 * d + 8], wide[1:, d:3 * d]):
        with pytest.raises(_abi.ArgumentError, match="overlaps"):
            ctx.short_conv(aexq.slots(1, 1), conv, off, x, w, out)
    with pytest.raises(_abi.ArgumentError, match="overlaps"):
        ctx.gated_rmsnorm(part(2, hv), part(4, hv), None, part(2, hv, 1))
    assert torch.equal(wide, before)
    begin = state.clone()
    ctx.delta_prompt(one, state, off, **args, out=part(4, hv))
    ctx.short_conv(aexq.slots(1, 1), conv, off, x, w, wide[:n, 6 * d:])
    torch.cuda.synchronize()
    y, near, _, _ = ref.delta(**args, state=begin[0], eps=1e-6)
    ref.check(part(4, hv), y, near)
    y, near, _ = ref.short_conv(x, _randn(1, 3, 2 * d, seed=23).half()[0], w, None, True)
    ref.check(wide[:n, 6 * d:], y, near)
    assert torch.equal(wide[:, :4 * d], before[:, :4 * d])
    assert torch.equal(wide[n], before[n])

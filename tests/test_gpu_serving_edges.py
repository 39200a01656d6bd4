"""The operators for many sequences at the calls that the other tests leave out:
arrays at the ends of their types, forms that only large calls take, infinities."""
import math

import pytest

torch = pytest.importorskip("torch")

import serving_ref as ref  # noqa: E402

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
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)


# ---------------------------------------------------------------- rotary append

def test_append_to_the_lowest_length(aexq, ctx):
    """A length of -2^31 is before every position: nothing is stored, also where the
    table holds so many positions that the difference to a token would wrap into it."""
    print("[gpu-case] append, length -2^31, table of 2^31 - 8192 positions", flush=True)
    hq, hkv, d, page, n = 2, 1, 64, 4096, 8300
    k, v = _randn(1, hkv, page, d, seed=1), _randn(1, hkv, page, d, seed=2)
    table = torch.zeros((1, ((1 << 31) - 8192) // page), dtype=torch.int32, device="cuda")
    lengths = torch.tensor([-1 << 31], dtype=torch.int32, device="cuda")
    before = k.clone(), v.clone()
    cos, sin = torch.zeros((9, d // 2), device="cuda"), torch.ones((9, d // 2), device="cuda")
    cos[0], sin[0] = 1.0, 0.0  # the row that places before the cache are clamped to
    q, kn, vn = _randn(n, hq, d, seed=3), _randn(n, hkv, d, seed=4), _randn(n, hkv, d, seed=5)
    out = torch.zeros_like(q)
    ctx.rope_append_paged(aexq.paged_kv(k, v, table, lengths), aexq.rope(cos, sin),
                          ref.offsets([n]), q, kn, vn, out)
    torch.cuda.synchronize()
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    assert torch.equal(out, q)


# ---------------------------------------------------------------- paged decode

@pytest.mark.parametrize("n,hq,hkv,d", [(257, 8, 2, 128), (700, 4, 1, 64), (300, 20, 1, 128),
                                        (513, 2, 2, 256), (1500, 6, 2, 64)])
def test_cut_decode_of_more_sequences_than_threads(aexq, ctx, n, hq, hkv, d):
    """More sequences than a workgroup has threads, most of them short, some cut into
    several pieces: at the ends, next to the threads' borders, beside empty ones."""
    print(f"[gpu-case] cut decode of {n} sequences {hq}/{hkv} d={d}", flush=True)
    each = -(-n // 256)  # sequences of a thread
    long = sorted({0, 1, each - 1, each, 128 * each, n // 2, n - 2, n - 1})
    lens = [(37 * i) % 90 for i in range(n)]
    for i, s in enumerate(long):
        lens[s] = 1500 + 61 * i
    lens[2], lens[n // 2 + 1] = 0, 0
    k, v, table, lengths = ref.make_cache(lens, hkv, 16, d, 6, width=140, fill=NAN)
    q = _randn(n, hq, d, seed=1)
    out, again = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    kv, scale = aexq.paged_kv(k, v, table, lengths), 1.0 / math.sqrt(d)
    ctx.attention_decode_paged(kv, q, scale, out)
    ctx.attention_decode_paged(kv, q, scale, again)
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    for s in sorted(set(long + [2, n // 2 + 1] + list(range(3, n, 13)))):
        ref.check_attention(out[s:s + 1], *ref.attend(q[s:s + 1], ref.gather(k, table, s, lens[s]),
                                                      ref.gather(v, table, s, lens[s]), scale,
                                                      False))
    dead = torch.tensor([m == 0 for m in lens], device="cuda")
    assert (out[dead] == 0).all() and torch.isfinite(out).all()


def test_decode_scratch_of_a_large_batch(aexq):
    """Sequences that are not cut take no scratch: a batch of 2048 in 8 key heads of
    128 takes the 13 MB of partial rows that one of 4 takes."""
    print("[gpu-case] decode scratch of 2048 sequences", flush=True)
    n, hq, hkv, d = 2048, 32, 8, 128
    lens = [(5 * i) % 40 for i in range(n)]
    k, v, table, lengths = ref.make_cache(lens, hkv, 16, d, 6, width=80)
    q = _randn(n, hq, d, seed=1)
    out, kv = torch.zeros_like(q), aexq.paged_kv(k, v, table, lengths)
    own = aexq.Context(0)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    own.attention_decode_paged(kv, q, 0.09, out)
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] <= 64 << 20
    for s in range(0, n, 97):
        ref.check_attention(out[s:s + 1], *ref.attend(q[s:s + 1], ref.gather(k, table, s, lens[s]),
                                                      ref.gather(v, table, s, lens[s]), 0.09, False))
    own.close()


# ---------------------------------------------------------------- infinities and NaN

def _check_exactly(got, want, mass):
    """ref.check_attention, and NaN where NaN is due, infinities of the due sign."""
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN elsewhere"
    for sign in (INF, -INF):
        assert torch.equal(got == sign, want == sign), f"{sign} elsewhere"
    ref.check_attention(got, want, mass)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_prompt_odd_values_exactly(ctx, d, bad):
    """An infinity or a NaN in v: in rows of tiles that are seen in part and whole,
    both signs in one dim, in the last position."""
    print(f"[gpu-case] prompt odd values exactly {bad} d={d}", flush=True)
    n, hq, hkv = 330, 4, 2
    q, k, v = _randn(n, hq, d, seed=1), _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
    v[20, 0, 5] = bad
    v[90, 0, 5] = -bad
    v[130, 1, d - 1] = bad
    v[n - 1, 0, 0] = bad
    for causal in (True, False):
        out = torch.zeros_like(q)
        ctx.attention_prompt(q, k, v, ref.offsets([n]), 0.06, out, causal=causal)
        torch.cuda.synchronize()
        _check_exactly(out, *ref.attend(q, k, v, 0.06, causal))


@pytest.mark.parametrize("n", [70, 500, 3000])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_decode_odd_values_exactly(aexq, ctx, n, d, bad):
    """The same in paged decode, whole and cut; rows past the end hold NaN."""
    print(f"[gpu-case] decode odd values exactly {bad} n={n} d={d}", flush=True)
    hq, hkv, page = 8, 2, 64
    k, v, table, lengths = ref.make_cache([n, 40], hkv, page, d, 6, fill=NAN)
    for x, h, e, y in ((20, 0, 5, bad), (60, 0, 5, -bad), (n - 1, 1, d - 1, bad), (3, 1, 0, bad)):
        v[table[0, x // page], h, x % page, e] = y
    q = _randn(2, hq, d, seed=1)
    out = torch.zeros_like(q)
    ctx.attention_decode_paged(aexq.paged_kv(k, v, table, lengths), q, 0.06, out)
    torch.cuda.synchronize()
    for s, m in enumerate((n, 40)):
        _check_exactly(out[s:s + 1], *ref.attend(q[s:s + 1], ref.gather(k, table, s, m),
                                                 ref.gather(v, table, s, m), 0.06, False))


@pytest.mark.parametrize("bits", [20.0, 28.0, 30.5, 40.0, 200.0])
@pytest.mark.parametrize("form", ["prompt", "paged prompt", "decode", "cut decode"])
def test_infinities_of_little_weight(aexq, ctx, form, bits):
    """An infinite v whose weight is 2^-bits of the row's largest: that infinity down to
    2^-31, there or NaN below (weights are fp16); all else of the row as ever.  The
    largest weight before the infinity and behind it."""
    print(f"[gpu-case] {form}, infinity of weight 2^-{bits}", flush=True)
    n, hq, hkv, d, page = 3000 if form == "cut decode" else 400, 4, 2, 128, 64
    for at, peak in ((70, 0), (200, 0), (70, 300)):
        k, v, table, lengths = ref.make_cache([n], hkv, page, d, 6)
        k[..., 0] = -3.0   # the other positions weigh 2^-3 of the largest
        k[..., 1:] = 0.0
        for x, y in ((at, -bits), (peak, 0.0)):
            k[table[0, x // page], :, x % page, 0] = y
        v[table[0, at // page], 0, at % page, 7] = INF
        v[table[0, at // page], 1, at % page, 9] = -INF
        kk, vv = ref.gather(k, table, 0, n), ref.gather(v, table, 0, n)
        rows = 1 if "decode" in form else n
        q = torch.zeros((rows, hq, d), dtype=torch.float16, device="cuda")
        q[:, :, 0] = 1.0
        out, scale = torch.zeros_like(q), math.log(2.0)
        kv, off = aexq.paged_kv(k, v, table, lengths), ref.offsets([rows])
        if "decode" in form:
            ctx.attention_decode_paged(kv, q, scale, out)
        elif form == "prompt":
            ctx.attention_prompt(q, kk.contiguous(), vv.contiguous(), off, scale, out)
        else:
            ctx.attention_prompt_paged(kv, q, off, scale, out)
        torch.cuda.synchronize()
        want, mass = ref.attend(q, kk, vv, scale, True)
        if bits > 31:
            # the rows that see both the infinity and a larger weight: others are sure
            last = torch.arange(n - rows, n, device="cuda")
            loose = torch.isinf(want) & (last >= min(at, peak))[:, None, None]
            assert not torch.isfinite(out[loose]).any()
            assert (torch.isnan(out) | (out.double() == want))[loose].all()
            out = torch.where(loose, want.half(), out)
        _check_exactly(out, want, mass)


# ---------------------------------------------------------------- forms of large calls

def _few_tokens(n):
    """0 to 2 new tokens of each of n sequences, none around every 64th."""
    new = [(i * 7 + 1) % 3 for i in range(n)]
    for b in range(64, n + 1, 64):
        new[b - 1] = 0
        if b < n:
            new[b] = 0
    if n % 64:
        new[-1] = 2
    return new


APPENDS = [([1024], [0]), ([1025], [7]), ([700, 0, 801], [40, 3, 0]), ([2, 1101, 200], [5, 0, 300])] + [
    (_few_tokens(n), [(5 * i) % 23 for i in range(n)]) for n in (64, 65, 130, 600)]


@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("d,rot,sections,interleaved,hq,hkv", [
    (128, 128, [64], False, 6, 2), (256, 64, [12, 10, 10], True, 4, 1), (64, 48, [8, 16], False, 9, 3)])
def test_append_of_many_tokens_and_sequences(aexq, ctx, case, d, rot, sections, interleaved, hq,
                                             hkv):
    """More tokens than a workgroup for each takes, not in fours, and more sequences
    than a wave looks through at a time; apart and in place."""
    new, past = APPENDS[case]
    print(f"[gpu-case] append of {sum(new)} tokens of {len(new)} sequences d={d}", flush=True)
    page, lens = 32, [a + b for a, b in zip(new, past)]
    k, v, table, lengths = ref.make_cache(lens, hkv, page, d, 4)
    live, rows = sum(new), 500
    n = live + 3
    q, kn, vn = _randn(n, hq, d, seed=1), _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
    g = torch.Generator(device="cuda").manual_seed(9)
    angle = torch.rand((rows, rot // 2), generator=g, device="cuda") * 6.28
    cos, sin = torch.cos(angle), torch.sin(angle)
    pos = torch.randint(-3, rows + 5, (len(sections), n), generator=g, device="cuda",
                        dtype=torch.int32)
    rope = aexq.rope(cos, sin, pos, sections=sections, interleaved=interleaved)
    kv, off, out = aexq.paged_kv(k, v, table, lengths), ref.offsets(new), torch.full_like(q, 7.0)
    kb, vb = k.clone(), v.clone()
    ctx.rope_append_paged(kv, rope, off, q, kn, vn, out)
    torch.cuda.synchronize()
    axis, at = ref.axis_of_pair(rot // 2, sections, interleaved), pos.clamp(0, rows - 1)
    want, near = ref.rotate(q, cos, sin, at, axis)
    assert ((out.double() - want).abs() <= near)[:live].all()
    assert torch.equal(out[:live, :, rot:], q[:live, :, rot:]) and (out[live:] == 7).all()
    # where each token's rows are
    x = torch.cat([torch.arange(b, b + a) for a, b in zip(new, past)])
    s = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    ids, row = table.cpu()[s, x // page].long().cuda(), (x % page).cuda()
    want, near = ref.rotate(kn, cos, sin, at, axis)
    assert ((k[ids, :, row].double() - want[:live]).abs() <= near[:live]).all()
    kb[ids, :, row], vb[ids, :, row] = k[ids, :, row], vn[:live]
    assert torch.equal(k, kb) and torch.equal(v, vb)  # the appended rows, and no others
    buf = torch.cat([q, kn, vn], 1).contiguous()
    views = buf.split([hq, hkv, hkv], 1)
    ctx.rope_append_paged(kv, rope, off, *views, views[0])
    torch.cuda.synchronize()
    assert torch.equal(views[0][:live], out[:live]) and torch.equal(views[0][live:], q[live:])
    assert torch.equal(views[1], kn) and torch.equal(views[2], vn)
    assert torch.equal(k, kb) and torch.equal(v, vb)


@pytest.mark.parametrize("paged", [False, True])
def test_prompt_layout_of_many_sequences(aexq, ctx, paged):
    """A layout of more sequences, and of more tiles, than it has threads, with long
    sequences that are cut among them."""
    print(f"[gpu-case] layout of 1500 sequences, paged={paged}", flush=True)
    lens = [(7 * i) % 9 for i in range(1500)]
    long = {3: 700, 1023: 300, 1024: 5000, 1490: 1300}
    for s, m in long.items():
        lens[s] = m
    n, hq, hkv, d, page = sum(lens), 4, 2, 64, 64
    q, off = _randn(n, hq, d, seed=1), ref.offsets(lens)
    out = torch.full_like(q, 7.0)
    if paged:
        kp, vp, table, lengths = ref.make_cache(lens, hkv, page, d, 6, fill=NAN)
        ctx.attention_prompt_paged(aexq.paged_kv(kp, vp, table, lengths), q, off, 0.125, out)
    else:
        k, v = _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
        ctx.attention_prompt(q, k, v, off, 0.125, out)
    torch.cuda.synchronize()
    at = off.tolist()
    assert torch.isfinite(out).all() and not (out == 7).all(-1).any()
    for s in sorted(set(list(long) + list(range(1000, 1050)) + list(range(5, 1500, 31)) + [1499])):
        a, m = slice(at[s], at[s + 1]), lens[s]
        kk, vv = ((ref.gather(kp, table, s, m), ref.gather(vp, table, s, m)) if paged
                  else (k[a], v[a]))
        ref.check_attention(out[a], *ref.attend(q[a], kk, vv, 0.125, True))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("short,long,hq,hkv,d", [(2200, 3000, 4, 2, 64), (2, 5000, 64, 1, 128),
                                                 (2100, 2500, 4, 2, 256)])
def test_prompts_of_more_tiles_than_a_layout_takes(ctx, short, long, hq, hkv, d, causal):
    """Without a layout: sequences of several tiles of keys among many of a few tokens."""
    print(f"[gpu-case] {short} short prompts and one of {long}, {hq}/{hkv} d={d}", flush=True)
    lens = [(5 * i) % 4 for i in range(short)]
    lens.insert(short // 2, long)
    n = sum(lens)
    q, k, v = _randn(n, hq, d, seed=1), _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
    off, out, scale = ref.offsets(lens), torch.full_like(q, 7.0), 1.0 / math.sqrt(d)
    ctx.attention_prompt(q, k, v, off, scale, out, causal=causal)
    torch.cuda.synchronize()
    at = off.tolist()
    assert torch.isfinite(out).all()
    for s in list(range(0, short, max(1, short // 40))) + [short]:
        if s != short // 2:
            a = slice(at[s], at[s + 1])
            ref.check_attention(out[a], *ref.attend(q[a], k[a], v[a], scale, causal))
    first, end = at[short // 2], at[short // 2 + 1]
    for b in (1, 130, long // 2, long):  # rows of the long one, heads at the ends of groups
        a = slice(first + max(0, b - 70), first + b)
        heads = sorted({0, hq - 1})
        kk, vv = (t[first:first + b if causal else end][:, [h // (hq // hkv) for h in heads]]
                  for t in (k, v))
        ref.check_attention(out[a][:, heads], *ref.attend(q[a][:, heads], kk, vv, scale, causal))


@pytest.mark.parametrize("dtype,rows,n", [
    (torch.float32, 450, 150001), (torch.float32, 600, 120003), (torch.float16, 900, 150001),
    (torch.float16, 500, 270001)])
def test_logprobs_of_more_than_the_caches_hold(aexq, ctx, dtype, rows, n):
    """Logits read past the caches, in one part a row and in two, rows that start
    anywhere in a 16-byte chunk."""
    print(f"[gpu-case] logprobs {rows} x {n} {dtype}, past the caches", flush=True)
    top = 20
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    x = 3 * torch.randn((rows, n), generator=g, device="cuda", dtype=dtype)
    assert x.numel() * x.element_size() > 256 << 20
    x[:, 100:140] = -INF
    x[rows - 1] = torch.floor(x[rows - 1])  # many equal ones
    tokens = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    tokens[0] = 120
    lp, ent, val = (torch.full(s, 7.0, device="cuda") for s in ((rows,), (rows,), (rows, top)))
    ids = torch.full((rows, top), 7, dtype=torch.int32, device="cuda")
    ctx.logprobs(aexq.describe(x, rows, n), tokens, lp, ent, ids, val)
    torch.cuda.synchronize()
    # the bound of test_gpu_logprobs.py: n / 256 sums of a lane, one after the other
    eps = (n / 256 + 64) * 2.0 ** -24
    for a in list(range(0, rows - 1, 61)) + [rows - 1]:
        want = ref.logprobs(x[a:a + 1], tokens[a:a + 1], top)
        assert torch.equal(ids[a:a + 1], want[2])
        for got, w in ((lp[a:a + 1], want[0]), (val[a:a + 1], want[3])):
            assert torch.equal(torch.isneginf(got.double()), torch.isneginf(w))
            near = (got.double() - w).abs() <= eps + 2.0 ** -22 * w.abs()
            assert (near | torch.isneginf(w)).all()
        assert ((ent[a:a + 1].double() - want[1]).abs() <= 2 * eps * (1 + want[1].abs())).all()


def test_logits_past_32_bit_offsets(aexq, ctx):
    """Rows whose logits lie past 2^31 elements and 2^32 bytes."""
    print("[gpu-case] logprobs of more than 2^31 logits", flush=True)
    n, top = 151937, 5
    rows = (1 << 31) // n + 9
    x = torch.zeros((rows, n), dtype=torch.float16, device="cuda")
    picked = [0, rows // 2, rows - 9, rows - 1]
    for i, r in enumerate(picked):
        x[r] = _randn(n, seed=i)
    tokens = torch.arange(rows, dtype=torch.int32, device="cuda") % n
    lp, ent, val = (torch.full(s, 7.0, device="cuda") for s in ((rows,), (rows,), (rows, top)))
    ids = torch.full((rows, top), 7, dtype=torch.int32, device="cuda")
    ctx.logprobs(aexq.describe(x, rows, n), tokens, lp, ent, ids, val)
    torch.cuda.synchronize()
    eps = (n / 256 + 64) * 2.0 ** -24
    for r in picked + [rows - 2]:
        want = ref.logprobs(x[r:r + 1], tokens[r:r + 1], top)
        assert torch.equal(ids[r:r + 1], want[2])
        for got, w in ((lp[r:r + 1], want[0]), (val[r:r + 1], want[3])):
            assert ((got.double() - w).abs() <= eps + 2.0 ** -22 * w.abs()).all()
        assert ((ent[r:r + 1].double() - want[1]).abs() <= 2 * eps * (1 + want[1].abs())).all()


@pytest.mark.parametrize("form", ["decode", "cut decode", "paged prompt"])
def test_rows_that_are_views(aexq, ctx, form):
    """q and out as views into wider buffers: what lies beside them stays."""
    print(f"[gpu-case] {form} of views", flush=True)
    lens = [2500, 0, 700] if form == "cut decode" else [300, 0, 41]
    hq, hkv, d = 12, 2, 128
    k, v, table, lengths = ref.make_cache(lens, hkv, 64, d, 6, fill=NAN)
    kv, new = aexq.paged_kv(k, v, table, lengths), [1, 1, 1] if "decode" in form else [20, 2, 41]
    n = sum(new)
    wide_q = _randn(n, hq + 4, d, seed=1)
    wide = torch.full((n, hq + 6, d), 7.0, dtype=torch.float16, device="cuda")
    q, out = wide_q[:, 3:hq + 3], wide[:, 2:hq + 2]
    if "decode" in form:
        ctx.attention_decode_paged(kv, q, 0.09, out)
    else:
        ctx.attention_prompt_paged(kv, q, ref.offsets(new), 0.09, out)
    torch.cuda.synchronize()
    at = ref.offsets(new).tolist()
    for s, m in enumerate(lens):
        a = slice(at[s], at[s + 1])
        _check_exactly(out[a], *ref.attend(q[a], ref.gather(k, table, s, m),
                                           ref.gather(v, table, s, m), 0.09, True))
    assert (wide[:, :2] == 7).all() and (wide[:, hq + 2:] == 7).all()


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("form", ["prompt", "paged prompt", "decode", "cut decode"])
def test_finite_values_stay_finite(aexq, ctx, form, d):
    """v of the type's largest magnitude: an average of 65504s is 65504, also where the
    weights' rounding to fp16 adds up.  Scores of -(1 - 2^-10) in log2 units, every 32nd
    of 0: weights of 64.043 in the kernels' scale, rounded to 64.0625, 3.0e-4 more than
    they are, and 31 to every one of 128: 2.8e-4 more in all, which takes 65504 past
    65520, where fp16 rounds to infinity."""
    print(f"[gpu-case] {form} of the largest values d={d}", flush=True)
    n, hq, hkv, page = 3000 if form == "cut decode" else 460, 4, 2, 64
    k, v, table, lengths = ref.make_cache([n], hkv, page, d, 6)
    k[..., 0] = -(1 - 2.0 ** -10)
    k[..., 1:] = 0.0
    k[:, :, ::32, 0] = 0.0
    v[:] = 65504.0
    v[..., 1::2] = -65504.0
    kk, vv = ref.gather(k, table, 0, n), ref.gather(v, table, 0, n)
    rows = 1 if "decode" in form else n
    q = torch.zeros((rows, hq, d), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    out, scale = torch.zeros_like(q), math.log(2.0)
    kv, off = aexq.paged_kv(k, v, table, lengths), ref.offsets([rows])
    if "decode" in form:
        ctx.attention_decode_paged(kv, q, scale, out)
    elif form == "prompt":
        ctx.attention_prompt(q, kk.contiguous(), vv.contiguous(), off, scale, out)
    else:
        ctx.attention_prompt_paged(kv, q, off, scale, out)
    torch.cuda.synchronize()
    _check_exactly(out, *ref.attend(q, kk, vv, scale, True))

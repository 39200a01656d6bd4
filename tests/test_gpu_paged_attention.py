"""Attention over prompts and paged caches, and the rotary append, against
64-bit references (serving_ref.py holds them and their bounds)."""
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


# ---------------------------------------------------------------- prompts

PROMPTS = [([1], 16, 4, 128), ([33], 16, 4, 128), ([0, 5, 0, 130, 1], 4, 1, 128),
           ([64, 65, 127, 129, 300], 8, 8, 64), ([200, 31, 32], 6, 2, 256),
           ([700], 7, 1, 128), ([90, 257], 20, 1, 64), ([1000, 3], 12, 4, 128),
           ([2, 511], 3, 1, 256), ([1] * 300, 2, 1, 64)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,hq,hkv,d", PROMPTS)
def test_prompt(ctx, lens, hq, hkv, d, causal):
    print(f"[gpu-case] prompt {lens[:6]} {hq}/{hkv} d={d} causal={causal}", flush=True)
    n = sum(lens)
    q, k, v = _randn(n, hq, d, seed=1), _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
    off, out = ref.offsets(lens), torch.full_like(q, 7.0)
    scale = 1.0 / math.sqrt(d)
    ctx.attention_prompt(q, k, v, off, scale, out, causal=causal)
    torch.cuda.synchronize()
    at = off.tolist()
    for a, b in zip(at, at[1:]):
        ref.check_attention(out[a:b], *ref.attend(q[a:b], k[a:b], v[a:b], scale, causal))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,kv_lens", [([5, 70], [100, 300]), ([100, 20, 3], [10, 0, 64]),
                                            ([33], [32])])
def test_prompt_with_other_key_lengths(ctx, q_lens, kv_lens, causal):
    """More keys than queries, and fewer: then the first rows see nothing."""
    print(f"[gpu-case] prompt {q_lens} over {kv_lens} causal={causal}", flush=True)
    hq, hkv, d = 8, 2, 128
    q = _randn(sum(q_lens), hq, d, seed=1)
    k, v = (_randn(sum(kv_lens), hkv, d, seed=s) for s in (2, 3))
    qo, ko, out = ref.offsets(q_lens), ref.offsets(kv_lens), torch.full_like(q, 7.0)
    ctx.attention_prompt(q, k, v, qo, 0.1, out, causal=causal, kv_offsets=ko)
    torch.cuda.synchronize()
    qa, ka = qo.tolist(), ko.tolist()
    for i in range(len(q_lens)):
        a, b = slice(qa[i], qa[i + 1]), slice(ka[i], ka[i + 1])
        ref.check_attention(out[a], *ref.attend(q[a], k[b], v[b], 0.1, causal))


def test_prompt_views_and_rows_behind_the_last_sequence(ctx):
    """q, k and v as views into one buffer; rows past the offsets stay."""
    print("[gpu-case] prompt views", flush=True)
    lens, hq, hkv, d = [70, 60], 4, 2, 128
    n = sum(lens) + 9
    buf = _randn(n, (hq + 2 * hkv) * d, seed=5)
    q, k, v = (t.view(n, -1, d) for t in buf.split([hq * d, hkv * d, hkv * d], 1))
    wide = torch.full((n, hq + 3, d), 7.0, dtype=torch.float16, device="cuda")
    off = ref.offsets(lens)
    ctx.attention_prompt(q, k, v, off, 0.09, wide[:, 1:hq + 1])
    torch.cuda.synchronize()
    for a, b in ((0, 70), (70, 130)):
        ref.check_attention(wide[a:b, 1:hq + 1],
                            *ref.attend(q[a:b], k[a:b], v[a:b], 0.09, True))
    assert (wide[130:] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, hq + 1:] == 7).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_prompt_odd_values_reach_only_rows_that_see_them(ctx, d, bad):
    print(f"[gpu-case] prompt odd values {bad} d={d}", flush=True)
    n, hq, hkv = 150, 4, 2
    q, k, v = _randn(n, hq, d, seed=1), _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
    v[20, 0, 5] = bad
    v[130, 1, d - 1] = bad
    v[149, 0, 0] = bad
    off, out = ref.offsets([n]), torch.zeros_like(q)
    ctx.attention_prompt(q, k, v, off, 0.09, out)
    torch.cuda.synchronize()
    ref.check_attention(out, *ref.attend(q, k, v, 0.09, True))
    v = _randn(n, hkv, d, seed=3)
    k[100, 0, 3] = bad
    ctx.attention_prompt(q, k, v, off, 0.09, out)
    torch.cuda.synchronize()
    want, mass = ref.attend(q, k, v, 0.09, True)
    ref.check_attention(out[:100], want[:100], mass[:100])
    ref.check_attention(out[:, 2:], want[:, 2:], mass[:, 2:])
    if math.isnan(bad):
        assert torch.isnan(out[100:, :2]).all()


@pytest.mark.parametrize("gain", [1.0, 30.0])
def test_prompt_maxima_that_grow_along_the_keys(ctx, gain):
    """Scores that rise, and fall, from tile to tile by much more than a weight's
    range, and the last key alone holding the weight."""
    print(f"[gpu-case] prompt growing maxima {gain}", flush=True)
    n, d = 400, 128
    q, k, v = _randn(n, 2, d, seed=1), _randn(n, 2, d, seed=2), _randn(n, 2, d, seed=3)
    ramp = torch.linspace(0, 1, n, device="cuda", dtype=torch.float16)
    q[:, :, 0] = 4.0
    k[:, 0, 0], k[:, 1, 0] = gain * ramp, -gain * ramp
    off, out = ref.offsets([n]), torch.zeros_like(q)
    for causal in (True, False):
        ctx.attention_prompt(q, k, v, off, 1.0, out, causal=causal)
        torch.cuda.synchronize()
        # scores up to 120: their fp32 rounding is 2^-24 of the sums of |q k| (below
        # 400 at scale 1), 128 terms: 3e-4 at most, a sixth of the bound's slack of
        # 2^-12 or more at gain 1, and weights of one key alone at gain 30
        ref.check_attention(out, *ref.attend(q, k, v, 1.0, causal))


@pytest.mark.parametrize("n,hq,hkv,d", [(5000, 2, 1, 128), (4097, 8, 2, 64), (2600, 2, 2, 256)])
def test_prompt_long(ctx, n, hq, hkv, d):
    print(f"[gpu-case] prompt long {n} {hq}/{hkv} d={d}", flush=True)
    q, k, v = _randn(n, hq, d, seed=1), _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
    off, out, scale = ref.offsets([n]), torch.zeros_like(q), 1.0 / math.sqrt(d)
    ctx.attention_prompt(q, k, v, off, scale, out)
    torch.cuda.synchronize()
    ref.check_attention(out, *ref.attend(q, k, v, scale, True))


# ---------------------------------------------------------------- paged prompts

@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("new,past,hq,hkv,d", [
    ([40], [0], 16, 4, 128), ([1, 17, 64], [100, 0, 300], 8, 2, 128),
    ([130, 0, 5], [70, 30, 1000], 4, 4, 64), ([33, 2], [500, 15], 6, 1, 256)])
def test_prompt_paged(aexq, ctx, page, new, past, hq, hkv, d):
    print(f"[gpu-case] paged prompt {new} after {past} page={page} {hq}/{hkv} d={d}", flush=True)
    lens = [a + b for a, b in zip(new, past)]
    # rows that no sequence keeps hold NaN: nothing of them may show
    k, v, table, lengths = ref.make_cache(lens, hkv, page, d, 4, fill=NAN)
    q, off = _randn(sum(new) + 3, hq, d, seed=1), ref.offsets(new)
    out = torch.full_like(q, 7.0)
    ctx.attention_prompt_paged(aexq.paged_kv(k, v, table, lengths), q, off, 0.1, out)
    torch.cuda.synchronize()
    at = off.tolist()
    for s, length in enumerate(lens):
        a = slice(at[s], at[s + 1])
        ref.check_attention(out[a], *ref.attend(q[a], ref.gather(k, table, s, length),
                                                ref.gather(v, table, s, length), 0.1, True))
    assert (out[at[-1]:] == 7).all()


# ---------------------------------------------------------------- decode

LENGTHS = [[1], [0, 1, 2, 15, 16, 17, 31, 32, 33], [127, 128, 129, 0, 255, 256, 257],
           [300, 511, 512], [700, 1, 0, 1025, 513]]


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("hq,hkv,d", [(16, 4, 128), (8, 8, 64), (8, 1, 256), (7, 1, 128),
                                      (20, 1, 128), (32, 2, 64), (3, 3, 256)])
@pytest.mark.parametrize("lens", LENGTHS)
def test_decode(aexq, ctx, lens, hq, hkv, d, page):
    print(f"[gpu-case] paged decode {lens} page={page} {hq}/{hkv} d={d}", flush=True)
    k, v, table, lengths = ref.make_cache(lens, hkv, page, d, 6, fill=NAN)
    q = _randn(len(lens), hq, d, seed=1)
    out, scale = torch.full_like(q, 7.0), 1.0 / math.sqrt(d)
    ctx.attention_decode_paged(aexq.paged_kv(k, v, table, lengths), q, scale, out)
    torch.cuda.synchronize()
    for s, n in enumerate(lens):
        ref.check_attention(out[s:s + 1], *ref.attend(q[s:s + 1], ref.gather(k, table, s, n),
                                                      ref.gather(v, table, s, n), scale, False))


@pytest.mark.parametrize("width", [2, 60])
def test_decode_of_many_short_sequences(aexq, ctx, width):
    """More sequences than a workgroup has threads; a table far wider than the
    lengths need."""
    print(f"[gpu-case] paged decode, many sequences, table of {width}", flush=True)
    lens = [(7 * i) % 33 for i in range(600)]
    hq, hkv, d = 4, 2, 64
    k, v, table, lengths = ref.make_cache(lens, hkv, 16, d, 7, width=max(3, width))
    q = _randn(len(lens), hq, d, seed=1)
    out = torch.full_like(q, 7.0)
    ctx.attention_decode_paged(aexq.paged_kv(k, v, table, lengths), q, 0.125, out)
    torch.cuda.synchronize()
    for s in list(range(40)) + [299, 300, 511, 512, 599]:
        n = lens[s]
        ref.check_attention(out[s:s + 1], *ref.attend(q[s:s + 1], ref.gather(k, table, s, n),
                                                      ref.gather(v, table, s, n), 0.125, False))
    dead = torch.tensor([n == 0 for n in lens], device="cuda")
    assert (out[dead] == 0).all()


@pytest.mark.parametrize("lens,hq,hkv,d", [([70001], 8, 2, 128), ([30000, 9, 20011], 16, 1, 64),
                                           ([25000, 3000], 4, 2, 256)])
def test_decode_long(aexq, ctx, lens, hq, hkv, d):
    print(f"[gpu-case] paged decode long {lens} {hq}/{hkv} d={d}", flush=True)
    k, v, table, lengths = ref.make_cache(lens, hkv, 256, d, 8)
    q = _randn(len(lens), hq, d, seed=1)
    out, scale = torch.zeros_like(q), 1.0 / math.sqrt(d)
    ctx.attention_decode_paged(aexq.paged_kv(k, v, table, lengths), q, scale, out)
    torch.cuda.synchronize()
    for s, n in enumerate(lens):
        ref.check_attention(out[s:s + 1], *ref.attend(q[s:s + 1], ref.gather(k, table, s, n),
                                                      ref.gather(v, table, s, n), scale, False))


def test_decode_scores_of_minus_infinity(aexq, ctx):
    """Keys that score -inf weigh nothing next to finite ones; a sequence of
    nothing else has no weights: NaN, as in aexq_attention_decode."""
    print("[gpu-case] paged decode -inf", flush=True)
    lens, hq, hkv, d = [700, 40, 600], 4, 2, 128
    k, v, table, lengths = ref.make_cache(lens, hkv, 64, d, 9)
    q = _randn(3, hq, d, seed=1).abs() + 0.5
    for s, low in ((0, range(0, 400)), (1, range(40)), (2, range(100, 600))):
        for x in low:
            k[table[s, x // 64], :, x % 64] = -INF
    out = torch.zeros_like(q)
    ctx.attention_decode_paged(aexq.paged_kv(k, v, table, lengths), q, 0.05, out)
    torch.cuda.synchronize()
    for s, keep in ((0, slice(400, 700)), (2, slice(0, 100))):
        kk, vv = (ref.gather(t, table, s, lens[s])[keep] for t in (k, v))
        ref.check_attention(out[s:s + 1], *ref.attend(q[s:s + 1], kk, vv, 0.05, False))
    assert torch.isnan(out[1]).all()


@pytest.mark.parametrize("form", ["decode", "prompt", "append"])
def test_pool_past_32_bit_offsets(aexq, ctx, form):
    """Pages whose elements lie past 2^31, and whose bytes past 2^32."""
    print(f"[gpu-case] {form} in a pool of more than 2^31 elements", flush=True)
    hq, hkv, d, page, n = 8, 2, 128, 256, 600
    pool = (1 << 31) // (hkv * page * d) + 5
    k, v = (torch.zeros((pool, hkv, page, d), dtype=torch.float16, device="cuda")
            for _ in range(2))
    ids = [pool - 1, 3, pool - 2]
    for t, seed in ((k, 2), (v, 3)):
        for i, p in enumerate(ids):
            t[p] = _randn(hkv, page, d, seed=seed + 10 * i)
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    kv = aexq.paged_kv(k, v, table, lengths)
    new = 1 if form == "decode" else 40
    q, off = _randn(new, hq, d, seed=1), ref.offsets([new])
    out = torch.zeros_like(q)
    if form == "append":
        kn, vn = _randn(new, hkv, d, seed=20), _randn(new, hkv, d, seed=21)
        ones, zeros = torch.ones((8, d // 2), device="cuda"), torch.zeros((8, d // 2), device="cuda")
        ctx.rope_append_paged(kv, aexq.rope(ones, zeros), off, q, kn, vn, out)
        torch.cuda.synchronize()
        assert torch.equal(ref.gather(k, table, 0, n)[n - new:], kn)
        assert torch.equal(ref.gather(v, table, 0, n)[n - new:], vn)
        return
    if form == "decode":
        ctx.attention_decode_paged(kv, q, 0.09, out)
    else:
        ctx.attention_prompt_paged(kv, q, off, 0.09, out)
    torch.cuda.synchronize()
    ref.check_attention(out, *ref.attend(q, ref.gather(k, table, 0, n),
                                         ref.gather(v, table, 0, n), 0.09, True))


def test_table_entries_and_lengths_out_of_range(aexq, ctx):
    """A page outside the pool is read as its nearest page, a length past the
    table as the table's end, a negative one as none; nothing is stored there."""
    print("[gpu-case] table entries out of range", flush=True)
    hq, hkv, d, page = 4, 2, 128, 16
    k, v = _randn(5, hkv, page, d, seed=1), _randn(5, hkv, page, d, seed=2)
    table = torch.tensor([[-7, 1], [2, 1 << 30], [3, 0]], dtype=torch.int32, device="cuda")
    fixed = torch.tensor([[0, 1], [2, 4], [3, 0]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([20, 1000, -4], dtype=torch.int32, device="cuda")
    kv = aexq.paged_kv(k, v, table, lengths)
    q = _randn(3, hq, d, seed=3)
    out = torch.full_like(q, 7.0)
    off = ref.offsets([1, 1, 1])
    for form in range(2):
        if form:
            ctx.attention_prompt_paged(kv, q, off, 0.1, out)
        else:
            ctx.attention_decode_paged(kv, q, 0.1, out)
        torch.cuda.synchronize()
        for s, n in enumerate([20, 32, 0]):
            ref.check_attention(out[s:s + 1], *ref.attend(q[s:s + 1], ref.gather(k, fixed, s, n),
                                                          ref.gather(v, fixed, s, n), 0.1, True))
    before = k.clone(), v.clone()
    cos, sin = torch.ones((4, 64), device="cuda"), torch.zeros((4, 64), device="cuda")
    # positions 19 (page 1), 999 (past the table), -5 (none)
    kn, vn = _randn(3, hkv, d, seed=4), _randn(3, hkv, d, seed=5)
    ctx.rope_append_paged(kv, aexq.rope(cos, sin), off, q, kn, vn, out)
    torch.cuda.synchronize()
    before[0][1, :, 3], before[1][1, :, 3] = kn[0], vn[0]
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    assert torch.equal(out, q)


# ---------------------------------------------------------------- rotary append

@pytest.mark.parametrize("d,rot,sections,interleaved", [
    (128, 128, [64], False), (64, 32, [16], False), (256, 64, [12, 10, 10], False),
    (256, 64, [12, 10, 10], True), (128, 128, [24, 20, 20], True), (128, 96, [16, 0, 32], False),
    (64, 64, [9, 8, 8, 7], False), (128, 16, [3, 5], False), (64, 16, [4, 4], True)])
@pytest.mark.parametrize("new,past,hq,hkv,page", [([1], [0], 16, 4, 64),
                                                  ([5, 0, 37, 1], [100, 3, 0, 16], 6, 2, 16)])
def test_rope_append(aexq, ctx, d, rot, sections, interleaved, new, past, hq, hkv, page):
    print(f"[gpu-case] append d={d} rot={rot} {sections} {interleaved} {new}", flush=True)
    lens = [a + b for a, b in zip(new, past)]
    k, v, table, lengths = ref.make_cache(lens, hkv, page, d, 4)
    n, rows = sum(new) + 2, 300
    q, kn, vn = _randn(n, hq, d, seed=1), _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
    g = torch.Generator(device="cuda").manual_seed(9)
    angle = torch.rand((rows, rot // 2), generator=g, device="cuda") * 6.28
    cos, sin = torch.cos(angle), torch.sin(angle)
    pos = torch.randint(-3, rows + 5, (len(sections), n), generator=g, device="cuda",
                        dtype=torch.int32)
    out, off = torch.full_like(q, 7.0), ref.offsets(new)
    kb, vb = k.clone(), v.clone()
    kv = aexq.paged_kv(k, v, table, lengths)
    ctx.rope_append_paged(kv, aexq.rope(cos, sin, pos, sections=sections,
                                        interleaved=interleaved), off, q, kn, vn, out)
    torch.cuda.synchronize()
    live = n - 2
    axis = ref.axis_of_pair(rot // 2, sections, interleaved)
    at = pos.clamp(0, rows - 1)
    want, near = ref.rotate(q, cos, sin, at, axis)
    assert ((out.double() - want).abs() <= near)[:live].all()
    assert torch.equal(out[:live, :, rot:], q[:live, :, rot:]) and (out[live:] == 7).all()
    want, near = ref.rotate(kn, cos, sin, at, axis)
    t = 0
    for s, (a, b) in enumerate(zip(new, past)):
        for x in range(b, b + a):
            page_id, row = int(table[s, x // page]), x % page
            assert ((k[page_id, :, row].double() - want[t]).abs() <= near[t]).all()
            kb[page_id, :, row], vb[page_id, :, row] = k[page_id, :, row], vn[t]
            t += 1
    assert torch.equal(k, kb) and torch.equal(v, vb)  # the appended rows, and no others
    # in place, with q, k and v as views into one buffer
    buf = torch.cat([q, kn, vn], 1).contiguous()
    views = buf.split([hq, hkv, hkv], 1)
    k2 = k.clone()
    ctx.rope_append_paged(kv, aexq.rope(cos, sin, pos, sections=sections,
                                        interleaved=interleaved), off, *views, views[0])
    torch.cuda.synchronize()
    assert torch.equal(views[0][:live], out[:live]) and torch.equal(k, k2)
    assert torch.equal(views[0][live:], q[live:])


def test_rope_append_at_the_place_in_the_cache(aexq, ctx):
    """Without positions a token's is its place in the cache, as
    aexq_rope_kv_append has it."""
    print("[gpu-case] append at cache positions", flush=True)
    from aiimage_amd import decoder
    hq, hkv, d, page = 16, 4, 128, 32
    new, past = [3, 40], [60, 0]
    lens = [a + b for a, b in zip(new, past)]
    k, v, table, lengths = ref.make_cache(lens, hkv, page, d, 4)
    q, kn, vn = _randn(43, hq, d, seed=1), _randn(43, hkv, d, seed=2), _randn(43, hkv, d, seed=3)
    cos, sin = (torch.as_tensor(t).cuda() for t in decoder.rope_tables(64, d, 1e6))
    out = torch.zeros_like(q)
    ctx.rope_append_paged(aexq.paged_kv(k, v, table, lengths), aexq.rope(cos, sin),
                          ref.offsets(new), q, kn, vn, out)
    t = 0
    for s in range(2):
        cap = lens[s]
        kc, vc = (torch.zeros((hkv, cap, d), dtype=torch.float16, device="cuda") for _ in range(2))
        for x in range(past[s], lens[s]):
            one = q[t].clone()
            ctx.rope_kv_append(one, kn[t], vn[t], kc, vc, hq, hkv, d, cap, x, cos[x], sin[x])
            torch.cuda.synchronize()
            # the same products, which may be contracted in another order
            assert (out[t].float() - one.float()).abs().max() <= 2.0 ** -10 * 8
            t += 1
        got = ref.gather(k, table, s, cap).transpose(0, 1)[:, past[s]:]
        assert (got.float() - kc[:, past[s]:].float()).abs().max() <= 2.0 ** -10 * 8
        assert torch.equal(ref.gather(v, table, s, cap).transpose(0, 1)[:, past[s]:],
                           vc[:, past[s]:])

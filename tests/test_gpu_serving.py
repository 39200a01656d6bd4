"""The operators for many sequences together, as a serving program uses them:
prompts into a paged cache, chunks, single tokens, probabilities; captured and
replayed; on streams and contexts of their own; and work cut along the positions."""
import math

import pytest

torch = pytest.importorskip("torch")

import serving_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 16, 4, 128, 32
SCALE = 1.0 / math.sqrt(D)


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


def _tables(rows):
    from aiimage_amd import decoder
    return [torch.as_tensor(t).cuda() for t in decoder.rope_tables(rows, D, 1e6)]


def _empty_cache(lens, steps):
    """Pages enough for lens + steps positions of each sequence; lengths lens."""
    k, v, table, lengths = ref.make_cache([n + steps for n in lens], HKV, PAGE, D, 11)
    lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    return k.zero_(), v.zero_(), table, lengths


def test_prompts_then_tokens(aexq, ctx):
    """Prompts in one call, or in chunks, then tokens one by one: the cache and
    every attention row are those of the single-sequence operators and of 64 bits."""
    print("[gpu-case] prompts, chunks, tokens", flush=True)
    lens, steps = [70, 1, 200], 4
    total = sum(lens)
    cos, sin = _tables(256)
    q, k, v = _randn(total, HQ, D, seed=1), _randn(total, HKV, D, seed=2), _randn(total, HKV, D, seed=3)
    kp, vp, table, lengths = _empty_cache(lens, steps)
    kv, rope = aexq.paged_kv(kp, vp, table, lengths), aexq.rope(cos, sin)
    off = ref.offsets(lens)
    qr, out = torch.zeros_like(q), torch.zeros_like(q)
    ctx.rope_append_paged(kv, rope, off, q, k, v, qr)
    ctx.attention_prompt_paged(kv, qr, off, SCALE, out)
    torch.cuda.synchronize()
    at = off.tolist()
    kr = torch.cat([ref.gather(kp, table, s, n) for s, n in enumerate(lens)])
    for s, n in enumerate(lens):
        a = slice(at[s], at[s + 1])
        assert torch.equal(ref.gather(vp, table, s, n), v[a])
        ref.check_attention(out[a], *ref.attend(qr[a], kr[a], v[a], SCALE, True))
    # the packed form over the rotated rows: the same products in the same order
    packed = torch.zeros_like(q)
    ctx.attention_prompt(qr, kr, v, off, SCALE, packed)
    torch.cuda.synchronize()
    assert torch.equal(packed, out)

    # in two chunks into another cache
    kp2, vp2, table2, lengths2 = _empty_cache(lens, steps)
    kv2 = aexq.paged_kv(kp2, vp2, table2, lengths2)
    part = [40, 0, 137]
    out2 = torch.zeros_like(q)
    for first in (True, False):
        a, b = ([0] * 3, part) if first else (part, lens)
        rows = torch.cat([torch.arange(at[s] + a[s], at[s] + b[s]) for s in range(3)]).cuda()
        lengths2.copy_(torch.tensor(b, dtype=torch.int32))
        o2 = ref.offsets([y - x for x, y in zip(a, b)])
        qc, oc = torch.zeros_like(q[rows]), torch.zeros_like(q[rows])
        ctx.rope_append_paged(kv2, rope, o2, q[rows], k[rows], v[rows], qc)
        ctx.attention_prompt_paged(kv2, qc, o2, SCALE, oc)
        torch.cuda.synchronize()
        out2[rows] = oc
    for s, n in enumerate(lens):
        assert torch.equal(ref.gather(kp2, table2, s, n), ref.gather(kp, table, s, n))
        a = slice(at[s], at[s + 1])
        ref.check_attention(out2[a], *ref.attend(qr[a], kr[a], v[a], SCALE, True))

    # tokens, against the operators of one sequence over a cache of its own
    cap = 256
    kc, vc = (torch.zeros((3, HKV, cap, D), dtype=torch.float16, device="cuda") for _ in range(2))
    for s, n in enumerate(lens):
        kc[s, :, :n] = ref.gather(kp, table, s, n).transpose(0, 1)
        vc[s, :, :n] = ref.gather(vp, table, s, n).transpose(0, 1)
    one = ref.offsets([1, 1, 1])
    for step in range(steps):
        lengths.add_(1)
        q1, k1, v1 = (_randn(3, h, D, seed=50 + 3 * step + i) for i, h in enumerate((HQ, HKV, HKV)))
        qr1, o1, want = torch.zeros_like(q1), torch.zeros_like(q1), torch.zeros_like(q1)
        ctx.rope_append_paged(kv, rope, one, q1, k1, v1, qr1)
        ctx.attention_decode_paged(kv, qr1, SCALE, o1)
        for s, n in enumerate(lens):
            p = n + step
            ctx.attention_decode_rope(q1[s], k1[s], v1[s], kc[s], vc[s], HQ, HKV, D, cap, p + 1,
                                      cos[p], sin[p], SCALE, want[s])
        torch.cuda.synchronize()
        for s, n in enumerate(lens):
            m = n + step + 1
            ref.check_attention(o1[s:s + 1], *ref.attend(qr1[s:s + 1], ref.gather(kp, table, s, m),
                                                         ref.gather(vp, table, s, m), SCALE, False))
            # two roundings of the output, and of q and k, apart
            assert (o1[s].float() - want[s].float()).abs().max() <= 4e-3 * want[s].abs().max()


def test_probabilities_of_the_lm_heads_logits(aexq, ctx):
    """logprobs over the logits that the LM head writes: its greedy token is the
    first alternative."""
    print("[gpu-case] LM head and log probabilities", flush=True)
    from aiimage_amd import synth
    n, k, m = 5000, 256, 3
    words, scales, _ = synth.q8_weights(n, k, 5)
    w = ctx.weight(aexq.QuantizedTensor(n * k, k, words, scales, bits=8), n, k)
    x = torch.as_tensor(synth.activations(m, k, 6)).cuda()
    lay = aexq.LAYOUT_PACK4_LINEAR
    buf = aexq.new_activation(m, n, torch.float32, lay)
    logits = aexq.describe(buf, m, n, lay)
    best = torch.zeros(m, dtype=torch.int32, device="cuda")
    ctx.lmhead_argmax(w, aexq.describe(x, m, k), logits, best)
    lp, ids = torch.zeros(m, device="cuda"), torch.zeros((m, 3), dtype=torch.int32, device="cuda")
    val = torch.zeros((m, 3), device="cuda")
    ctx.logprobs(logits, best, lp, None, ids, val)
    torch.cuda.synchronize()
    assert torch.equal(ids[:, 0], best) and torch.equal(val[:, 0], lp)
    want = ref.logprobs(buf.view(m, -1)[:, :n], best, 3)
    assert torch.equal(ids, want[2]) and (val.double() - want[3]).abs().max() <= 1e-5


@pytest.mark.parametrize("width", [8, 40])
def test_a_captured_step_follows_lengths_on_the_device(aexq, width):
    """One step of three sequences, captured: lengths advance in the graph, the
    cache grows, and every replay equals the eager calls; whole and cut launches."""
    print(f"[gpu-case] captured step, table of {width}", flush=True)
    own = aexq.Context(0)
    lens, replays, vocab = [60, 3, 130], 4, 3000
    cos, sin = _tables(512)
    states = []
    for _ in range(2):  # the graph's cache and the eager one
        k, v, table, lengths = ref.make_cache([n + 10 for n in lens], HKV, PAGE, D, 11,
                                              width=width)
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        states.append((aexq.paged_kv(k, v, table, lengths), k, v, lengths))
    rope, one = aexq.rope(cos, sin), ref.offsets([1, 1, 1])
    q, k1, v1 = _randn(3, HQ, D, seed=1), _randn(3, HKV, D, seed=2), _randn(3, HKV, D, seed=3)
    x = torch.randn((3, vocab), device="cuda")
    logits = aexq.describe(x, 3, vocab)
    tokens = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")

    def buffers():
        z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        return (torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q), z(3), z(3),
                torch.zeros((3, 4), dtype=torch.int32, device="cuda"), z(3, 4))

    def step(state, out):
        kv, _, _, lengths = state
        lengths.add_(1)
        own.rope_append_paged(kv, rope, one, q, k1, v1, out[0])
        own.attention_decode_paged(kv, out[0], SCALE, out[1])
        own.attention_prompt_paged(kv, out[0], one, SCALE, out[2])
        own.logprobs(logits, tokens, *out[3:])

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    own.set_stream(stream)
    got, want = buffers(), buffers()
    with torch.cuda.stream(stream):
        step(states[0], got)  # sizes the scratch; its position is written again
        states[0][3].sub_(1)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        step(states[0], got)
    for i in range(replays):
        x.copy_(torch.randn((3, vocab), generator=torch.Generator(device="cuda").manual_seed(i),
                            device="cuda"))
        q.copy_(_randn(3, HQ, D, seed=100 + i))
        k1.copy_(_randn(3, HKV, D, seed=200 + i))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step(states[1], want)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for a, b in zip(states[0][1:], states[1][1:]):
            assert torch.equal(a, b)
    del graph
    own.close()


def test_scratch_does_not_grow_under_capture(aexq):
    print("[gpu-case] capture before a first run", flush=True)
    from aiimage_amd import _abi
    own = aexq.Context(0)
    k, v, table, lengths = ref.make_cache([700], 1, 16, D, 3)
    kv = aexq.paged_kv(k, v, table, lengths)
    q = _randn(1, 2, D, seed=1)
    out, off = torch.zeros_like(q), ref.offsets([1])
    x = torch.randn((1, 20000), device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    own.set_stream(stream)
    lp = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        out.zero_()
        for call in (lambda: own.attention_decode_paged(kv, q, 0.1, out),
                     lambda: own.attention_prompt_paged(kv, q, off, 0.1, out),
                     lambda: own.logprobs(aexq.describe(x, 1, 20000), off[:1], lp)):
            with pytest.raises(_abi.NotSupportedError, match="capturing"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    own.close()


def test_a_batch_that_grows_step_by_step(aexq):
    """Scratch that is outgrown stays (graphs may hold it), but not once per size:
    64 sizes of up to 768 + 64 * 8 pieces of 16 rows, 10.8 MB, would keep 556 MB."""
    print("[gpu-case] growing batch", flush=True)
    most = 64
    k, v, table, lengths = ref.make_cache([1100] * most, 8, 16, D, 3)
    q = _randn(most, 8, D, seed=1)
    out, probs = torch.zeros_like(q), torch.zeros(most, device="cuda")
    x, tok = torch.randn((most, 20000), device="cuda"), lengths.clone()
    own = aexq.Context(0)
    own.attention_decode_paged(aexq.paged_kv(k, v, table[:1], lengths[:1]), q[:1], SCALE, out[:1])
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for n in range(1, most + 1):
        kv = aexq.paged_kv(k, v, table[:n], lengths[:n])
        own.attention_decode_paged(kv, q[:n], SCALE, out[:n])
        own.logprobs(aexq.describe(x[:n], n, 20000), tok[:n], probs[:n])
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] <= 128 << 20
    for s in (0, most - 1):
        kk, vv = ref.gather(k, table, s, 1100), ref.gather(v, table, s, 1100)
        ref.check_attention(out[s:s + 1], *ref.attend(q[s:s + 1], kk, vv, SCALE, False))
    own.close()


def test_two_contexts_at_once(aexq):
    """Each context has a stream and scratch of its own."""
    print("[gpu-case] two contexts", flush=True)
    k, v, table, lengths = ref.make_cache([5000, 900], 2, 64, D, 3)
    kv = aexq.paged_kv(k, v, table, lengths)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [aexq.Context(0, s) for s in streams]
    qs = [_randn(2, 8, D, seed=i) for i in range(2)]
    news = [_randn(60, 8, D, seed=10 + i) for i in range(2)]
    off = ref.offsets([20, 40])
    x = [torch.randn((2, 30000), device="cuda") for _ in range(2)]
    tok = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    outs = []
    for i in range(2):
        outs.append([[torch.zeros_like(qs[i]), torch.zeros_like(news[i]),
                      torch.zeros(2, device="cuda")] for _ in range(6)])
    torch.cuda.synchronize()
    for r in range(6):
        for i in range(2):
            a = outs[i][r]
            ctxs[i].attention_decode_paged(kv, qs[i], SCALE, a[0])
            ctxs[i].attention_prompt_paged(kv, news[i], off, SCALE, a[1])
            ctxs[i].logprobs(aexq.describe(x[i], 2, 30000), tok, a[2])
    torch.cuda.synchronize()
    for i in range(2):
        for r in range(1, 6):  # the same bits every time
            for a, b in zip(outs[i][0], outs[i][r]):
                assert torch.equal(a, b)
        for s, n in enumerate((5000, 900)):
            kk, vv = ref.gather(k, table, s, n), ref.gather(v, table, s, n)
            ref.check_attention(outs[i][0][0][s:s + 1],
                                *ref.attend(qs[i][s:s + 1], kk, vv, SCALE, False))
            a = slice(*off.tolist()[s:s + 2])
            ref.check_attention(outs[i][0][1][a], *ref.attend(news[i][a], kk, vv, SCALE, True))
    for c in ctxs:
        c.close()


@pytest.mark.parametrize("new,past,hq,hkv,d", [
    ([1], [9000], 4, 1, 128), ([16], [9000], 16, 4, 128), ([40, 3], [6000, 4000], 4, 2, 64),
    ([9, 700], [5000, 0], 8, 1, 256), ([100], [3500], 16, 16, 64)])
def test_few_rows_over_many_positions(aexq, ctx, new, past, hq, hkv, d):
    """Tiles cut along the positions, and a NaN among positions only the last
    token sees."""
    print(f"[gpu-case] few rows {new} after {past} {hq}/{hkv} d={d}", flush=True)
    lens = [a + b for a, b in zip(new, past)]
    k, v, table, lengths = ref.make_cache(lens, hkv, 64, d, 4, fill=math.nan)
    last = lens[0] - 1
    v[table[0, last // 64], 0, last % 64, 1] = math.nan
    kv, off = aexq.paged_kv(k, v, table, lengths), ref.offsets(new)
    q = _randn(sum(new), hq, d, seed=1)
    out, again = torch.zeros_like(q), torch.zeros_like(q)
    scale = 1.0 / math.sqrt(d)
    ctx.attention_prompt_paged(kv, q, off, scale, out)
    ctx.attention_prompt_paged(kv, q, off, scale, again)
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    at = off.tolist()
    for s, n in enumerate(lens):
        a = slice(at[s], at[s + 1])
        ref.check_attention(out[a], *ref.attend(q[a], ref.gather(k, table, s, n),
                                                ref.gather(v, table, s, n), scale, True))


def test_more_sequences_than_a_layout_takes(ctx):
    print("[gpu-case] 2500 sequences", flush=True)
    lens = [(5 * i) % 4 for i in range(2500)]
    n = sum(lens)
    q, k, v = _randn(n, 4, 64, seed=1), _randn(n, 2, 64, seed=2), _randn(n, 2, 64, seed=3)
    off, out = ref.offsets(lens), torch.full_like(q, 7.0)
    ctx.attention_prompt(q, k, v, off, 0.125, out)
    torch.cuda.synchronize()
    at = off.tolist()
    for s in list(range(20)) + list(range(2480, 2500)):
        a = slice(at[s], at[s + 1])
        ref.check_attention(out[a], *ref.attend(q[a], k[a], v[a], 0.125, True))


def test_refusals_leave_the_outputs(aexq, ctx):
    print("[gpu-case] refusals", flush=True)
    from aiimage_amd import _abi
    k, v, table, lengths = ref.make_cache([40, 50], 2, 16, D, 3)
    kv = aexq.paged_kv(k, v, table, lengths)
    q, off = _randn(2, 4, D, seed=1), ref.offsets([1, 1])
    out = torch.full_like(q, 7.0)
    arg = _abi.ArgumentError
    with pytest.raises(arg, match="q is"):
        ctx.attention_decode_paged(kv, q[:1], 0.1, out)
    with pytest.raises(arg, match="out is"):
        ctx.attention_decode_paged(kv, q, 0.1, out.float())
    with pytest.raises(arg, match="out is q"):
        ctx.attention_decode_paged(kv, q, 0.1, q)
    with pytest.raises(arg, match="scale"):
        ctx.attention_decode_paged(kv, q, 0.0, out)
    with pytest.raises(arg, match="offsets"):
        ctx.attention_prompt_paged(kv, q, off[:2], 0.1, out)
    with pytest.raises(arg, match="offsets"):
        ctx.attention_prompt(q, q, q, off.long(), 0.1, out)
    with pytest.raises(arg, match="heads_q"):
        ctx.attention_prompt(q, q[:, :3], q[:, :3], off, 0.1, out)
    with pytest.raises(arg, match="kv is|PagedKv"):
        ctx.attention_decode_paged(None, q, 0.1, out)
    cos = torch.ones((8, D // 2), device="cuda")
    with pytest.raises(arg, match="positions of 3"):
        ctx.rope_append_paged(kv, aexq.rope(cos, cos, torch.zeros((1, 3), dtype=torch.int32,
                                                                  device="cuda")),
                              off, q, q[:, :2], q[:, :2], out)
    x = torch.zeros((2, 30), device="cuda")
    d = aexq.describe(x, 2, 30)
    lp = torch.full((2,), 7.0, device="cuda")
    with pytest.raises(arg, match="tokens"):
        ctx.logprobs(d, off[:2].long(), lp)
    with pytest.raises(arg, match="top=31"):
        ctx.logprobs(d, off[:2], lp, None, torch.zeros((2, 31), dtype=torch.int32, device="cuda"))
    with pytest.raises(arg, match="no output"):
        ctx.logprobs(d, off[:2], None)
    torch.cuda.synchronize()
    assert (out == 7).all() and (lp == 7).all()


@pytest.mark.parametrize("lens,hq,hkv,d,causal", [
    ([1613, 300], 16, 16, 64, False), ([900, 1700], 16, 4, 128, True), ([800, 65], 8, 2, 256, True)])
def test_repeated_calls_give_the_same_bits(ctx, lens, hq, hkv, d, causal):
    """Tiles follow one another through two buffers; a read that is late, or a row
    that is early, shows in some of many passes only."""
    print(f"[gpu-case] repeated prompts {lens} {hq}/{hkv} d={d}", flush=True)
    n = sum(lens)
    q, k, v = _randn(n, hq, d, seed=1), _randn(n, hkv, d, seed=2), _randn(n, hkv, d, seed=3)
    off, first, out = ref.offsets(lens), torch.zeros_like(q), torch.zeros_like(q)
    other = torch.zeros((), dtype=torch.int64, device="cuda")
    ctx.attention_prompt(q, k, v, off, 0.1, first, causal=causal)
    for _ in range(150):
        ctx.attention_prompt(q, k, v, off, 0.1, out, causal=causal)
        other += (out != first).sum()
    torch.cuda.synchronize()
    assert other.item() == 0
    at = off.tolist()
    for a, b in zip(at, at[1:]):
        ref.check_attention(first[a:b], *ref.attend(q[a:b], k[a:b], v[a:b], 0.1, causal))

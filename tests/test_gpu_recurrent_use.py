"""The recurrent layers' operators and the verification of drafted tokens as a serving
program uses them: a layer over prompts, single tokens and drafts, captured graphs, two
contexts, pools and rows past 32-bit offsets, thousands of sequences."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import recurrent_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

HK, HV, D, HIDDEN, VOCAB = 2, 4, 64, 256, 600
CHANNELS = 2 * HK * D + HV * D
SCALE, EPS = D ** -0.5, 1e-6


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


class Layer:
    """A recurrent layer: projections, convolution, delta rule, gated norm, projection."""

    def __init__(self, aexq, ctx, pool, seed=1):
        self.aexq, self.ctx = aexq, ctx
        rng = np.random.default_rng(seed)
        w = lambda n, k: ctx.weight_from_float(  # noqa: E731
            (rng.standard_normal((n, k)) * k ** -0.5).astype(np.float32), n, k)
        self.qkv, self.z, self.ab = w(CHANNELS, HIDDEN), w(HV * D, HIDDEN), w(2 * HV, HIDDEN)
        self.o, self.head = w(HIDDEN, HV * D), w(VOCAB, HIDDEN)
        self.conv_w, self.gamma = _randn(CHANNELS, 4, seed=2), 1 + 0.2 * _randn(D, seed=3)
        self.a_log, self.dt_bias = _randn(HV, seed=4), _randn(HV, seed=5) - 1.5
        self.conv = torch.zeros((pool, 3, CHANNELS), device="cuda").half()
        self.state = torch.zeros((pool, HV, D, D), device="cuda")

    def clone_states(self):
        return self.conv.clone(), self.state.clone()

    def put_states(self, states):
        self.conv.copy_(states[0])
        self.state.copy_(states[1])

    def linear(self, w, x, n):
        y = torch.zeros((x.shape[0], n), device="cuda").half()
        self.ctx.linear(w, self.aexq.describe(x, *x.shape), self.aexq.describe(y, *y.shape))
        return y

    def split(self, y):
        q, k, v = y.split([HK * D, HK * D, HV * D], 1)
        return q.unflatten(1, (HK, D)), k.unflatten(1, (HK, D)), v.unflatten(1, (HV, D))

    def run(self, x, slots, off, single=False, alone=False):
        """Hidden states of rows x; every buffer on the way in self.seen.  single: the
        single-token form; alone: the states, no outputs."""
        n = x.shape[0]
        qkv, z, ab = (self.linear(w, x, m) for w, m in ((self.qkv, CHANNELS), (self.z, HV * D),
                                                        (self.ab, 2 * HV)))
        mixed = torch.full_like(qkv, 7.0)
        self.ctx.short_conv(slots, self.conv, off, qkv, self.conv_w, mixed)
        q, k, v = self.split(mixed)
        out = None if alone else torch.full((n, HV, D), 7.0, device="cuda").half()
        args = (q, k, v, ab[:, :HV], ab[:, HV:], self.a_log, self.dt_bias, out)
        if single:
            self.ctx.delta_decode(slots, self.state, *args, scale=SCALE)
        else:
            self.ctx.delta_prompt(slots, self.state, off, *args, scale=SCALE)
        self.seen = (qkv, z, ab, mixed, out)
        if alone:
            return None
        normed = torch.zeros_like(out)
        self.ctx.gated_rmsnorm(out, z.unflatten(1, (HV, D)), self.gamma, normed)
        self.seen += (normed,)
        return self.linear(self.o, normed.flatten(1), HIDDEN)

    def check(self, lens, before, slot, stored=True):
        """Every stage of the last run against its plain form on the stage's own input."""
        torch.cuda.synchronize()
        qkv, z, ab, mixed, out, normed = self.seen
        at = 0
        for s, m in enumerate(lens):
            rows = slice(at, at + m)
            y, near, left = ref.short_conv(qkv[rows], before[0][slot[s]], self.conv_w, None, True)
            ref.check(mixed[rows], y, near, f"conv of {s}")
            q, k, v = (t[rows] for t in self.split(mixed))
            y, near, S, err = ref.delta(q, k, v, ab[rows, :HV], ab[rows, HV:], self.a_log,
                                        self.dt_bias, before[1][slot[s]], SCALE, EPS)
            ref.check(out[rows], y, near, f"delta of {s}")
            y, near = ref.gated_norm(out[rows], z[rows].unflatten(1, (HV, D)), self.gamma, 1e-6)
            ref.check(normed[rows], y, near, f"norm of {s}")
            if stored:
                assert torch.equal(self.conv[slot[s]], left)
                ref.check(self.state[slot[s]], S, err, f"state of {s}")
            at += m


def test_a_layer_over_prompts_tokens_and_drafts(aexq, ctx):
    """Prompts, then single tokens, then drafts that run without storing, are verified,
    and whose accepted rows advance the states: the states are then, bit for bit, those
    of a run of the accepted rows alone."""
    print("[gpu-case] a recurrent layer, prompts to drafts", flush=True)
    lens, slot = [70, 3, 130], [4, 0, 2]
    n, pool = len(lens), 5
    layer, slots_of = Layer(aexq, ctx, pool), ref.i32(slot)
    before = layer.clone_states()
    layer.run(_randn(sum(lens), HIDDEN, seed=10).half(),
              aexq.slots(pool, n, slot=slots_of, lengths=ref.i32(lens)), ref.offsets(lens))
    layer.check(lens, before, slot)
    one = ref.offsets([1] * n)
    for step in range(3):
        before = layer.clone_states()
        layer.run(_randn(n, HIDDEN, seed=20 + step).half(),
                  aexq.slots(pool, n, slot=slots_of, lengths=ref.i32([m + 1 + step for m in lens])),
                  one, single=True)
        layer.check([1] * n, before, slot)
    for turn in range(3):
        drafted = [5, 2, 4]
        rows, off = sum(drafted), ref.offsets(drafted)
        x = _randn(rows, HIDDEN, seed=30 + turn).half()
        before = layer.clone_states()
        hidden = layer.run(x, aexq.slots(pool, n, slot=slots_of, read_only=True), off)
        layer.check(drafted, before, slot, stored=False)
        for a, b in zip(layer.clone_states(), before):
            assert torch.equal(a, b)
        logits = layer.linear(layer.head, hidden, VOCAB).float() * 3
        probs = torch.softmax(logits + _randn(rows, VOCAB, seed=40 + turn), -1)
        drafts = probs.argmax(-1).int()
        au, su = _rand(rows, seed=50 + turn), _rand(n, seed=60 + turn)
        counts = torch.zeros(n, dtype=torch.int32, device="cuda")
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        ctx.verify_drafts(aexq.describe(logits, rows, VOCAB), off, drafts, au, su, counts, tokens,
                          draft_probs=probs)
        layer.run(x, aexq.slots(pool, n, slot=slots_of, counts=counts), off, alone=True)
        torch.cuda.synchronize()
        want = ref.verify(logits, drafted, drafts, probs, None, au, su)
        assert (counts.tolist(), tokens.tolist()) == want
        got = layer.clone_states()
        # the same rows, and no others
        layer.put_states(before)
        kept = want[0]
        first = off.tolist()
        layer.run(torch.cat([x[first[s]:first[s] + kept[s]] for s in range(n)]),
                  aexq.slots(pool, n, slot=slots_of), ref.offsets(kept))
        layer.check(kept, before, slot)
        assert torch.equal(layer.state, got[1])
        assert torch.equal(layer.conv, got[0])


def _step_inputs(seed, rows):
    """What one step of everything takes: rows of three sequences."""
    r = lambda *s, k=0: _randn(*s, seed=100 * seed + k)  # noqa: E731
    return dict(x=r(rows, CHANNELS).half(), ab=r(rows, 2 * HV, k=1).half(),
                z=r(rows, HV, D, k=2).half(), logits=2 * r(rows, VOCAB, k=3),
                au=_rand(rows, seed=seed), su=_rand(3, seed=seed + 1))


class Step:
    """Every operator once, on buffers of its own."""

    def __init__(self, aexq, ctx, lens, seed=7):
        self.ctx, self.n, rows = ctx, len(lens), sum(lens)
        self.d = _step_inputs(seed, rows)
        self.off, self.weight = ref.offsets(lens), _randn(CHANNELS, 4, seed=8)
        self.one = ref.offsets([1] * self.n)
        self.gates = _randn(HV, seed=9), _randn(HV, seed=10) - 1
        self.conv = _randn(4, 3, CHANNELS, seed=11).half()
        self.states = [_randn(4, HV, D, D, seed=12 + i) for i in range(2)]
        self.lengths = ref.i32([0, 40, 9]) + ref.i32(lens)
        self.counts = torch.full((self.n,), 1, dtype=torch.int32, device="cuda")
        self.tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.drafts = self.d["logits"].argmax(-1).int()
        slot = ref.i32([3, 0, 1])
        self.all = aexq.slots(4, self.n, slot=slot, lengths=self.lengths)
        self.some = aexq.slots(4, self.n, slot=slot, counts=self.counts)
        self.logits = aexq.describe(self.d["logits"], rows, VOCAB)
        z = lambda *s: torch.zeros(s, device="cuda").half()  # noqa: E731
        self.mixed, self.out, self.normed = z(rows, CHANNELS), z(rows, HV, D), z(rows, HV, D)
        self.single = z(self.n, HV, D)

    def run(self):
        c, d = self.ctx, self.d
        c.verify_drafts(self.logits, self.off, self.drafts, d["au"], d["su"], self.counts,
                        self.tokens)
        c.short_conv(self.all, self.conv, self.off, d["x"], self.weight, self.mixed)
        q, k, v = self.mixed.split([HK * D, HK * D, HV * D], 1)
        rows = (q.unflatten(1, (HK, D)), k.unflatten(1, (HK, D)), v.unflatten(1, (HV, D)),
                d["ab"][:, :HV], d["ab"][:, HV:])
        c.delta_prompt(self.some, self.states[0], self.off, *rows, *self.gates, self.out, scale=SCALE)
        c.delta_decode(self.all, self.states[1], *(t[:self.n] for t in rows), *self.gates, self.single,
                       scale=SCALE)
        c.gated_rmsnorm(self.out, d["z"], None, self.normed)

    def results(self):
        return [t.clone() for t in (self.counts, self.tokens, self.mixed, self.conv, self.out,
                                    *self.states, self.single, self.normed)]

    def take(self, seed):
        """Other values in the same buffers; lengths grow."""
        for k, t in _step_inputs(seed, self.d["x"].shape[0]).items():
            self.d[k].copy_(t)
        self.lengths.add_(1)


@pytest.mark.parametrize("lens", [[5, 1, 3], [100, 17, 64]])
def test_captured_steps(aexq, lens):
    """Everything in one graph; states, lengths and counts change from replay to replay.
    Eager work runs between the replays, a second graph shares the context's scratch."""
    print(f"[gpu-case] captured steps of {lens}", flush=True)
    own, plain = aexq.Context(0), aexq.Context(0)
    stream = torch.cuda.Stream()
    steps = [Step(aexq, own, lens, 7), Step(aexq, own, [m + 1 for m in lens], 70)]
    eager = [Step(aexq, plain, lens, 7), Step(aexq, plain, [m + 1 for m in lens], 70)]
    torch.cuda.synchronize()
    own.set_stream(stream)
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    for s, e in zip(steps, eager):
        with torch.cuda.stream(stream):
            s.run()                       # sizes the scratch
        stream.synchronize()
        e.run()
        torch.cuda.synchronize()
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
            s.run()
        graphs.append(g)
    for i in range(4):
        for s, e, g in zip(steps, eager, graphs):
            s.take(200 + i)
            e.take(200 + i)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
            e.run()
            torch.cuda.synchronize()
            for a, b in zip(s.results(), e.results()):
                assert torch.equal(a, b)
        with torch.cuda.stream(stream):   # both, with no wait between them
            for s in steps:
                s.take(300 + i)
            for g in graphs:
                g.replay()
        for e in eager:
            e.take(300 + i)
            e.run()
        torch.cuda.synchronize()
        for s, e in zip(steps, eager):
            for a, b in zip(s.results(), e.results()):
                assert torch.equal(a, b)
    del graphs
    own.close()
    plain.close()


def test_scratch_does_not_grow_under_capture(aexq):
    print("[gpu-case] recurrent scratch under capture", flush=True)
    from aiimage_amd import _abi
    own = aexq.Context(0)
    step = Step(aexq, own, [5, 1, 3])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    own.set_stream(stream)
    d = step.d
    q, k, v = d["x"].split([HK * D, HK * D, HV * D], 1)
    rows = (q.unflatten(1, (HK, D)), k.unflatten(1, (HK, D)), v.unflatten(1, (HV, D)),
            d["ab"][:, :HV], d["ab"][:, HV:])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        step.out.zero_()
        with pytest.raises(_abi.NotSupportedError, match="capturing"):
            own.delta_prompt(step.all, step.states[0], step.off, *rows, *step.gates, step.out,
                             scale=SCALE)
        with pytest.raises(_abi.NotSupportedError, match="capturing"):
            own.verify_drafts(step.logits, step.off, step.drafts, d["au"], d["su"], step.counts,
                              step.tokens)
        # (these take none)
        own.short_conv(step.all, step.conv, step.off, d["x"], step.weight, step.mixed)
        own.delta_decode(step.all, step.states[1], *(t[:3] for t in rows), *step.gates, step.single,
                         scale=SCALE)
    graph.replay()
    torch.cuda.synchronize()
    del graph
    own.close()


def test_two_contexts_at_once(aexq):
    """Each context has a stream and scratch of its own; the same bits every time."""
    print("[gpu-case] two contexts, recurrent", flush=True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [aexq.Context(0, s) for s in streams]
    lens = [[300, 20, 64], [5, 1, 3]]
    steps = [[Step(aexq, c, m) for _ in range(5)] for c, m in zip(ctxs, lens)]
    alone = [Step(aexq, c, m) for c, m in zip(ctxs, lens)]
    torch.cuda.synchronize()
    for i in range(5):
        for j in range(2):
            steps[j][i].run()
    torch.cuda.synchronize()
    for j in range(2):
        alone[j].run()
        torch.cuda.synchronize()
        want = alone[j].results()
        for s in steps[j]:
            for a, b in zip(s.results(), want):
                assert torch.equal(a, b)
    for c in ctxs:
        c.close()


def test_pools_past_32_bit_offsets(aexq, ctx):
    """States whose offsets in bytes and in elements pass 2^32: the first, one in the
    middle and the last."""
    print("[gpu-case] pools past 32 bits", flush=True)
    hv, dk, dv, c = 32, 128, 128, 6144
    pool = 2 ** 32 // (hv * dk * dv) + 5
    state = torch.empty((pool, hv, dk, dv), device="cuda")
    slot = [pool - 1, 0, pool // 2 + 3]
    begin = _randn(3, hv, dk, dv, seed=1)
    for i, s in enumerate(slot):
        state[s] = begin[i]
    lens = [3, 70, 1]
    n = sum(lens)
    d = dict(q=_randn(n, 2, dk, seed=2).half(), k=_randn(n, 2, dk, seed=3).half(),
             v=_randn(n, hv, dv, seed=4).half(), a=_randn(n, hv, seed=5).half(),
             b=_randn(n, hv, seed=6).half(), a_log=_randn(hv, seed=7), dt_bias=_randn(hv, seed=8))
    out = torch.zeros((n, hv, dv), device="cuda").half()
    slots = aexq.slots(pool, 3, slot=ref.i32(slot))
    ctx.delta_prompt(slots, state, ref.offsets(lens), **d, out=out, scale=0.1)
    torch.cuda.synchronize()
    at = 0
    for i, m in enumerate(lens):
        rows = {k: t if k in ("a_log", "dt_bias") else t[at:at + m] for k, t in d.items()}
        y, near, S, err = ref.delta(**rows, state=begin[i], scale=0.1, eps=1e-6)
        ref.check(out[at:at + m], y, near, f"sequence {i}")
        ref.check(state[slot[i]], S, err, f"state {i}")
        begin[i] = state[slot[i]]
        at += m
    one = {k: t if k in ("a_log", "dt_bias") else t[:3] for k, t in d.items()}
    ctx.delta_decode(slots, state, **one, out=out[:3], scale=0.1)
    torch.cuda.synchronize()
    for i in range(3):
        rows = {k: t if k in ("a_log", "dt_bias") else t[i:i + 1] for k, t in d.items()}
        y, near, S, err = ref.delta(**rows, state=begin[i], scale=0.1, eps=1e-6)
        ref.check(out[i:i + 1], y, near, f"token {i}")
        ref.check(state[slot[i]], S, err, f"state {i}")
    del state
    pool = 2 ** 32 // (3 * c) + 5
    conv = torch.empty((pool, 3, c), device="cuda", dtype=torch.float16)
    slot = [pool - 1, 0, pool // 2 + 3]
    begin = _randn(3, 3, c, seed=9).half()
    for i, s in enumerate(slot):
        conv[s] = begin[i]
    x, w = _randn(n, c, seed=10).half(), _randn(c, 4, seed=11)
    got = torch.zeros_like(x)
    ctx.short_conv(aexq.slots(pool, 3, slot=ref.i32(slot)), conv, ref.offsets(lens), x, w, got)
    torch.cuda.synchronize()
    at = 0
    for i, m in enumerate(lens):
        y, near, left = ref.short_conv(x[at:at + m], begin[i], w, None, True)
        ref.check(got[at:at + m], y, near, f"rows of {i}")
        assert torch.equal(conv[slot[i]], left)
        at += m


def test_rows_as_far_apart_as_they_may_be(aexq, ctx):
    """Strides of 2^24 elements, offsets past 2^32 bytes, sequences that begin there."""
    print("[gpu-case] rows 2^24 elements apart", flush=True)
    far, n, hv, dk, dv = 1 << 24, 150, 2, 64, 64
    wide = torch.empty((n, far), device="cuda", dtype=torch.float16)
    result = torch.empty((n, far), device="cuda", dtype=torch.float16)
    part = lambda t, i, h, d: t[:, 4096 * i:4096 * i + h * d].unflatten(1, (h, d))  # noqa: E731
    q, k, v, z = (part(wide, i, h, d) for i, (h, d) in enumerate(((1, dk), (1, dk), (hv, dv),
                                                                  (hv, dv))))
    for i, t in enumerate((q, k, v, z)):
        t.copy_(_randn(*t.shape, seed=i))
    a, b = _randn(n, hv, seed=5).half(), _randn(n, hv, seed=6).half()
    gates = _randn(hv, seed=7), _randn(hv, seed=8) - 1
    lens = [20, n - 20]
    state = _randn(2, hv, dk, dv, seed=9)
    before, slots, off = state.clone(), aexq.slots(2, 2), ref.offsets(lens)
    out, normed, x = part(result, 0, hv, dv), part(result, 1, hv, dv), wide[:, 8192:8192 + hv * dv]
    mixed = result[:, 65536:65536 + hv * dv]
    ctx.delta_prompt(slots, state, off, q, k, v, a, b, *gates, out, scale=0.1)
    ctx.gated_rmsnorm(out, z, None, normed)
    conv, w = torch.zeros((2, 3, hv * dv), device="cuda").half(), _randn(hv * dv, 4, seed=10)
    ctx.short_conv(slots, conv, off, x, w, mixed)
    torch.cuda.synchronize()
    at = 0
    for i, m in enumerate(lens):
        r = slice(at, at + m)
        y, near, S, err = ref.delta(q[r], k[r], v[r], a[r], b[r], *gates, before[i], 0.1, 1e-6)
        ref.check(out[r], y, near, f"sequence {i}")
        ref.check(state[i], S, err, f"state {i}")
        y, near, left = ref.short_conv(x[r], torch.zeros_like(conv[0]), w, None, True)
        ref.check(mixed[r], y, near, f"rows of {i}")
        assert torch.equal(conv[i], left)
        at += m
    ref.check(normed, *ref.gated_norm(out, z, None, 1e-6), "norm")
    # single tokens: row s is sequence s
    ctx.delta_decode(aexq.slots(2, n, slot=ref.i32([-1] * n)), state, q, k, v, a, b, *gates, out,
                     scale=0.1)
    torch.cuda.synchronize()
    zero = torch.zeros_like(state[0])
    for i in (0, 77, n - 1):
        r = slice(i, i + 1)
        y, near, _, _ = ref.delta(q[r], k[r], v[r], a[r], b[r], *gates, zero, 0.1, 1e-6)
        ref.check(out[r], y, near, f"token {i}")
    del wide, result, q, k, v, z, x, out, normed, mixed
    # logits and draft probabilities past 2^32 bytes
    vocab, rows = 1 << 23, 140
    logits = torch.empty((rows, vocab), device="cuda", dtype=torch.float16)
    logits.normal_(generator=torch.Generator(device="cuda").manual_seed(3))
    probs = torch.softmax(logits[-3:].float() + 1, -1)
    whole = torch.empty((rows, vocab), device="cuda")
    whole[-3:] = probs
    drafts = torch.zeros(rows, dtype=torch.int32, device="cuda")
    drafts[-3:] = torch.multinomial(probs, 1)[:, 0].int()
    au, su = _rand(rows, seed=4), _rand(2, seed=5)
    counts = torch.zeros(2, dtype=torch.int32, device="cuda")
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    off = ref.i32([rows - 4, rows - 3, rows])
    ctx.verify_drafts(aexq.describe(logits, rows, vocab), off, drafts, au, su, counts, tokens,
                      draft_probs=whole)
    torch.cuda.synchronize()
    want = ref.verify(logits[-4:], [1, 3], drafts[-4:], torch.cat([probs[:1], probs]), None, au[-4:],
                      su)
    assert (counts.tolist(), tokens[-4:].tolist()) == want
    assert (tokens[:-4] == 0).all()


@pytest.mark.parametrize("n,hk,hv,dk,dv", [(100, 2, 4, 128, 128), (300, 1, 2, 64, 256)])
def test_short_sequences_and_a_few_long_ones(aexq, ctx, n, hk, hv, dk, dv):
    """Many sequences of 0 to 17 rows with longer ones, a state that is not finite, counts
    that leave a long one short, slots of no state: each as by itself."""
    print(f"[gpu-case] {n} sequences, mostly short, {hk}/{hv} {dk}x{dv}", flush=True)
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 18, (n,), generator=g).tolist()
    for s, m in ((3, 200), (64, 65), (65, 16), (66, 17), (n - 1, 130), (n - 2, 80)):
        lens[s] = m
    kept = list(lens)
    kept[n - 2], kept[7] = 9, 0
    total, off = sum(lens), ref.offsets(lens)
    d = dict(q=_randn(total, hk, dk, seed=1).half(), k=_randn(total, hk, dk, seed=2).half(),
             v=_randn(total, hv, dv, seed=3).half(), a=_randn(total, hv, seed=4).half(),
             b=_randn(total, hv, seed=5).half(), a_log=_randn(hv, seed=6),
             dt_bias=_randn(hv, seed=7) - 1)
    state = _randn(n, hv, dk, dv, seed=8)
    state[65, 0, 3, 5], state[3, 1, 7, 9] = math.inf, math.nan
    before = state.clone()
    slot = [s if s % 10 != 9 or s in (n - 1,) else -1 for s in range(n)]
    out = torch.full((total, hv, dv), 7.0, device="cuda").half()
    ctx.delta_prompt(aexq.slots(n, n, slot=ref.i32(slot), counts=ref.i32(kept)), state, off, **d,
                     out=out, scale=0.1)
    torch.cuda.synchronize()
    at = off.tolist()
    for s in list(range(0, n, 23)) + [3, 7, 64, 65, 66, n - 2, n - 1]:
        r = slice(at[s], at[s] + kept[s])
        assert (out[at[s] + kept[s]:at[s + 1]] == 7).all()
        if not kept[s]:
            assert torch.equal(state[s], before[s])
            continue
        rows = {k: t if k in ("a_log", "dt_bias") else t[r] for k, t in d.items()}
        begin = before[s] if slot[s] >= 0 else torch.zeros_like(before[s])
        y, near, S, err = ref.delta(**rows, state=begin, scale=0.1, eps=1e-6)
        if s in (3, 65):   # the other columns; this one is not finite from the start
            h, j = (1, 9) if s == 3 else (0, 5)
            assert not torch.isfinite(out[r][:, h, j]).any()
            assert not torch.isfinite(state[s, h, :, j]).any()
            keep = torch.ones((hv, dv), dtype=torch.bool, device="cuda")
            keep[h, j] = False
            ref.check(out[r][:, keep], y[:, keep], near[:, keep], f"sequence {s}")
            ref.check(state[s].transpose(1, 2)[keep], S.transpose(1, 2)[keep],
                      err.transpose(1, 2)[keep], f"state {s}")
            continue
        ref.check(out[r], y, near, f"sequence {s}")
        if slot[s] >= 0:
            ref.check(state[s], S, err, f"state {s}")
        else:
            assert torch.equal(state[s], before[s])


@pytest.mark.parametrize("n", [65, 4097, 20000])
def test_thousands_of_sequences(aexq, ctx, n):
    """Sequences of 0 to 3 rows, found by their rows in several steps: the same bits as
    calls of a few sequences each."""
    print(f"[gpu-case] {n} sequences", flush=True)
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 4, (n,), generator=g).tolist()
    lens[0] = 1
    total, c, vocab = sum(lens), 16, 40
    off = ref.offsets(lens)
    x, w = _randn(total, c, seed=1).half(), _randn(c, 4, seed=2)
    conv = _randn(n, 3, c, seed=3).half()
    d = [_randn(total, 1, 64, seed=4 + i).half() for i in range(3)]
    ab = _randn(total, 2, seed=7).half()
    gates = _randn(1, seed=8), _randn(1, seed=9)
    states = _randn(n, 1, 64, 64, seed=10)
    logits, au, su = _randn(total, vocab, seed=11), _rand(total, seed=12), _rand(n, seed=13)
    drafts = logits.argmax(-1).int()
    at = off.tolist()

    def run(a, b, conv, states):
        r = slice(at[a], at[b])
        rows, o = at[b] - at[a], off[a:b + 1] - at[a]
        mixed, out = torch.zeros_like(x[r]), torch.zeros_like(d[0][r])
        counts = torch.zeros(b - a, dtype=torch.int32, device="cuda")
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        if rows:
            ctx.short_conv(aexq.slots(b - a, b - a), conv[a:b], o, x[r], w, mixed)
            ctx.delta_prompt(aexq.slots(b - a, b - a), states[a:b], o, *(t[r] for t in d), ab[r, :1],
                             ab[r, 1:], *gates, out, scale=0.1)
            ctx.verify_drafts(aexq.describe(logits[r], rows, vocab), o, drafts[r], au[r], su[a:b],
                              counts, tokens)
        torch.cuda.synchronize()
        return mixed, out, counts, tokens

    before = conv.clone(), states.clone()
    whole = run(0, n, conv, states)
    step = 50
    places = sorted({0, 50, (n // 100) * 50, n - step} if n > 200 else {0, n - step})
    for a in places:
        conv2, states2 = (t.clone() for t in before)
        some = run(a, a + step, conv2, states2)
        r, s = slice(at[a], at[a + step]), slice(a, a + step)
        for got, want in zip((whole[0][r], whole[1][r], whole[2][s], whole[3][r], conv[s], states[s]),
                             (*some, conv2[s], states2[s])):
            assert torch.equal(got, want)


@pytest.mark.parametrize("layout", ["LAYOUT_PACK4_LINEAR", "LAYOUT_PACK4_TILED"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_logits_as_the_head_leaves_them(aexq, ctx, layout, dtype):
    """Rows padded to whole packs, rows of an odd width: what lies between them is no
    token's."""
    print(f"[gpu-case] verify {layout} {dtype}", flush=True)
    rows, vocab, lens = 7, 33001, [4, 3]
    layout = getattr(aexq, layout)
    buf = aexq.new_activation(rows, vocab, dtype=dtype, layout=layout)
    wide = buf.view(rows, -1)
    wide.fill_(50.0)        # above every logit
    wide[:, :vocab] = 2 * _randn(rows, vocab, seed=1)
    x = wide[:, :vocab]
    probs = torch.softmax(x.float() + _randn(rows, vocab, seed=2), -1)
    drafts = probs.argmax(-1).int()
    for heat in (None, torch.zeros(2, device="cuda")):
        au, su = _rand(rows, seed=3), _rand(2, seed=4)
        counts = torch.zeros(2, dtype=torch.int32, device="cuda")
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        ctx.verify_drafts(aexq.describe(buf, rows, vocab, layout), ref.offsets(lens), drafts, au, su,
                          counts, tokens, temperature=heat, draft_probs=probs)
        torch.cuda.synchronize()
        assert (counts.tolist(), tokens.tolist()) == ref.verify(x, lens, drafts, probs, heat, au, su)


def test_rows_before_the_first_sequence(aexq, ctx):
    """Offsets that begin far behind the first row: rows of no sequence are not touched,
    the others have the bits of a call of their own."""
    print("[gpu-case] rows before the first sequence", flush=True)
    skip, lens, hv, d, vocab = 1000, [5, 90], 2, 64, 300
    n = skip + sum(lens) + 2
    x, w = _randn(n, 16, seed=1).half(), _randn(16, 4, seed=2)
    rows = [_randn(n, h, d, seed=3 + i).half() for i, h in enumerate((1, 1, hv))]
    a, b = _randn(n, hv, seed=6).half(), _randn(n, hv, seed=7).half()
    gates = _randn(hv, seed=8), _randn(hv, seed=9)
    logits, au, su = _randn(n, vocab, seed=10), _rand(n, seed=11), _rand(2, seed=12)
    drafts = logits.argmax(-1).int()
    got = []
    for first, cut in ((skip, slice(0, n)), (0, slice(skip, skip + sum(lens)))):
        conv, state = _randn(2, 3, 16, seed=13).half(), _randn(2, hv, d, d, seed=14)
        m = n if cut.start == 0 else sum(lens)
        off = ref.offsets(lens) + first
        mixed, out = torch.full((m, 16), 7.0, device="cuda").half(), torch.full(
            (m, hv, d), 7.0, device="cuda").half()
        counts = torch.zeros(2, dtype=torch.int32, device="cuda")
        tokens = torch.full((m,), 77, dtype=torch.int32, device="cuda")
        slots = aexq.slots(2, 2)
        ctx.short_conv(slots, conv, off, x[cut], w, mixed)
        ctx.delta_prompt(slots, state, off, *(t[cut] for t in rows), a[cut], b[cut], *gates, out,
                         scale=0.1)
        ctx.verify_drafts(aexq.describe(logits[cut], m, vocab), off, drafts[cut], au[cut], su, counts,
                          tokens)
        torch.cuda.synchronize()
        used = slice(first, first + sum(lens))
        for t in (mixed, out):
            assert (t[:first] == 7).all() and (t[used.stop:] == 7).all()
        assert (tokens[:first] == 77).all() and (tokens[used.stop:] == 77).all()
        got.append([t[used].clone() for t in (mixed, out, tokens)] + [conv, state, counts])
    for p, q in zip(*got):
        assert torch.equal(p, q)


def test_a_layer_without_a_gpu_stream_of_its_own(aexq, ctx):
    """A context's stream may be any: results do not depend on it."""
    print("[gpu-case] recurrent operators on another stream", flush=True)
    a, b = Step(aexq, ctx, [64, 2, 130]), None
    a.run()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    own = aexq.Context(0, stream)
    with torch.cuda.stream(stream):
        b = Step(aexq, own, [64, 2, 130])
        b.run()
    stream.synchronize()
    for x, y in zip(a.results(), b.results()):
        assert torch.equal(x, y)
    own.close()
    assert math.isfinite(a.normed.float().abs().max().item())

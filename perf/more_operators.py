"""Performance cases of the recurrent layers and of drafted tokens: the short
causal convolution with its state, the gated delta rule over packed prompts and
for one token per sequence, the norm gated by silu behind it, and the
verification of drafted tokens.

A case is one call that a serving program makes over and over:

  conv    causal convolution of packed tokens along each sequence, channel by
          channel, with silu; the last inputs of a sequence are its state
  delta   the gated delta rule over packed prompts, chunks of prompts or drafted
          tokens, from and to each sequence's state
  step    the gated delta rule for one new token of each sequence
  norm    root-mean-square norm of each head, gated by silu
  verify  drafted tokens against the target's probabilities

Sequence s has rows offsets[s] .. offsets[s + 1] - 1 of the packed tokens; its
state is entry slot[s] of a pool.  A sequence whose length is its number of new
rows starts from zeros.  Activations are fp16, as everywhere in the library,
states fp32 (the convolution's are its fp16 inputs), logits fp32 or fp16.
"""
import math
import random

import torch

own = False

VOCAB = 151936
CHUNK = 64
EPS = 1e-6


def listed():
    return [
        # the next token of each sequence of a serving batch: q, k and v of 16
        # heads of 128 together
        {"name": "conv_tokens", "op": "conv", "seqs": 64, "lo": 1, "hi": 1, "channels": 6144,
         "width": 4, "bias": False, "drafts": False, "pick": 1},
        # ordinary prompts of different lengths, packed
        {"name": "conv_packed", "op": "conv", "seqs": 12, "lo": 50, "hi": 2048, "channels": 6144,
         "width": 4, "bias": False, "drafts": False, "pick": 2},
        # the smallest prompt: one short question
        {"name": "delta_short", "op": "delta", "seqs": 1, "lo": 33, "hi": 33, "hk": 16, "hv": 16,
         "dk": 128, "dv": 128, "drafts": False, "pick": 3},
        # ordinary prompts of different lengths, some of them continued
        {"name": "delta_packed", "op": "delta", "seqs": 12, "lo": 50, "hi": 2048, "hk": 16,
         "hv": 16, "dk": 128, "dv": 128, "drafts": False, "pick": 4},
        # one long document, two value heads to a key head
        {"name": "delta_long", "op": "delta", "seqs": 1, "lo": 16384, "hi": 16384, "hk": 16,
         "hv": 32, "dk": 128, "dv": 128, "drafts": False, "pick": 5},
        # drafted tokens of a batch, whose accepted rows advance the states
        {"name": "delta_drafts", "op": "delta", "seqs": 48, "lo": 2, "hi": 8, "hk": 16, "hv": 16,
         "dk": 128, "dv": 128, "drafts": True, "pick": 6},
        # the next token of one conversation
        {"name": "step_one", "op": "step", "seqs": 1, "hk": 16, "hv": 16, "dk": 128, "dv": 128,
         "pick": 7},
        # the next token of each sequence of a serving batch
        {"name": "step_batch", "op": "step", "seqs": 128, "hk": 16, "hv": 32, "dk": 128,
         "dv": 128, "pick": 8},
        # the heads of a batch's tokens
        {"name": "norm_tokens", "op": "norm", "rows": 64, "heads": 16, "d": 128, "gamma": True,
         "pick": 9},
        # the heads of packed prompts
        {"name": "norm_prompts", "op": "norm", "rows": 9973, "heads": 16, "d": 128, "gamma": True,
         "pick": 10},
        # one conversation whose drafts come from its own text: no probabilities
        {"name": "verify_one", "op": "verify", "seqs": 1, "lo": 5, "hi": 5, "vocab": VOCAB,
         "f16": False, "probs": False, "greedy": False, "pick": 11},
        # a serving batch with the draft model's probabilities
        {"name": "verify_batch", "op": "verify", "seqs": 64, "lo": 2, "hi": 8, "vocab": VOCAB,
         "f16": False, "probs": True, "greedy": False, "pick": 12},
    ]


# what a drawn case stays below: tokens times heads_v * dim_k * dim_v of the
# delta rule, and bytes of all operators
MOST_DELTA = 16384 * 32 * 128 * 128
MOST_BYTES = 2 * 128 * 32 * 128 * 128 * 4


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "delta", "delta", "delta", "step", "norm", "verify", "verify"])
    while True:
        c = {"op": op, "pick": rng.randrange(1 << 30)}
        if op == "norm":
            c["rows"], c["heads"] = _log_int(rng, 1, 16384), _log_int(rng, 1, 64)
            c["d"], c["gamma"] = rng.choice([64, 96, 128, 128, 200, 256]), rng.random() < 0.8
        else:
            c["seqs"] = _log_int(rng, 1, 128)
        if op in ("conv", "delta"):
            c["hi"] = _log_int(rng, 1, 16384)
            c["lo"] = _log_int(rng, 1, c["hi"])
            c["drafts"] = c["hi"] <= 16 and rng.random() < 0.5
        if op == "conv":
            c["channels"], c["width"] = 8 * _log_int(rng, 8, 1200), rng.choice([2, 3, 4, 4, 4, 5])
            c["bias"] = rng.random() < 0.3
        if op in ("delta", "step"):
            c["hk"] = rng.choice([1, 2, 4, 6, 8, 16])
            c["hv"] = c["hk"] * rng.choice([1, 1, 2, 3, 4])
            c["dk"], c["dv"] = rng.choice([64, 128, 128]), rng.choice([64, 128, 128, 256])
        if op == "verify":
            c["hi"] = rng.randint(1, 9)
            c["lo"] = rng.randint(1, c["hi"])
            c["vocab"] = _log_int(rng, 1000, VOCAB)
            c["f16"], c["probs"] = rng.random() < 0.5, rng.random() < 0.6
            c["greedy"] = rng.random() < 0.3
        if op == "delta" and sum(_new(c)) * c["hv"] * c["dk"] * c["dv"] > MOST_DELTA:
            continue
        if work(c)["bytes"] > MOST_BYTES:
            continue
        return c


# ---------------------------------------------------------------- inputs

def _new(case):
    """Rows of each sequence: spread over their logarithm, the first is the longest."""
    rng, lo, hi = random.Random(case["pick"]), case.get("lo", 1), case.get("hi", 1)
    return [hi] + [max(lo, min(hi, _log_int(rng, lo, hi))) for _ in range(case["seqs"] - 1)]


def _past(case):
    """Positions before the call: a third of the prompts start with it."""
    rng = random.Random(case["pick"] + 1)
    return [0 if case["op"] == "delta" and not case["drafts"] and rng.random() < 0.34 else
            _log_int(rng, 1, 30000) for _ in range(case["seqs"])]


def _kept(case):
    """Rows of each sequence that are taken: all, or the accepted ones of drafts."""
    rng = random.Random(case["pick"] + 2)
    return [rng.randint(1, n) if case.get("drafts") else n for n in _new(case)]


def _offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


class _Inputs:
    """Seeded inputs on the GPU, drawn in a fixed order."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def slots(self, case):
        """(offsets, slot, lengths, counts) of the sequences; the pool is a little
        larger than its use, its entries handed out in no order."""
        new, n = _new(case), case["seqs"]
        order = torch.randperm(n + 3, generator=self.g, device="cuda")[:n].to(torch.int32)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        lengths = i32([p + m for p, m in zip(_past(case), new)])
        counts = i32(_kept(case)) if case.get("drafts") else None
        return {"offsets": i32(_offsets(new)), "slot": order, "lengths": lengths, "counts": counts}


def _prepare_conv(case, seed):
    r = _Inputs(seed)
    s = r.slots(case)
    n, channels, width = sum(_new(case)), case["channels"], case["width"]
    s["x"] = r.normal(n, channels).half()
    s["weight"] = r.normal(channels, width) / math.sqrt(width)
    s["bias"] = 0.1 * r.normal(channels) if case["bias"] else None
    s["state"] = r.normal(case["seqs"] + 3, width - 1, channels).half()
    s["out"] = torch.zeros_like(s["x"])
    return s


def _prepare_delta(case, seed):
    r = _Inputs(seed)
    s = r.slots(case)
    n, hk, hv, dk, dv = sum(_new(case)), case["hk"], case["hv"], case["dk"], case["dv"]
    # q, k and v lie in one buffer, as the convolution leaves them
    x = torch.nn.functional.silu(r.normal(n, 2 * hk * dk + hv * dv)).half()
    s["q"] = x[:, :hk * dk].unflatten(1, (hk, dk))
    s["k"] = x[:, hk * dk:2 * hk * dk].unflatten(1, (hk, dk))
    s["v"] = x[:, 2 * hk * dk:].unflatten(1, (hv, dv))
    s["a"], s["b"] = r.normal(n, hv).half(), r.normal(n, hv).half()
    # decays as layers of this kind begin with: rates 1 to 16, steps 0.001 to 0.1
    s["a_log"] = torch.log(1 + 15 * r.uniform(hv))
    step = torch.exp(math.log(1e-3) + math.log(100.0) * r.uniform(hv))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["state"] = 0.2 * r.normal(case["seqs"] + 3, hv, dk, dv)
    s["out"] = torch.zeros((n, hv, dv), device="cuda", dtype=torch.float16)
    return s


_prepare_step = _prepare_delta


def _prepare_norm(case, seed):
    r = _Inputs(seed)
    shape = (case["rows"], case["heads"], case["d"])
    return {"x": r.normal(*shape).half(), "z": r.normal(*shape).half(),
            "gamma": 1 + 0.1 * r.normal(case["d"]) if case["gamma"] else None,
            "out": torch.zeros(shape, device="cuda", dtype=torch.float16)}


def _prepare_verify(case, seed):
    r = _Inputs(seed)
    new, vocab = _new(case), case["vocab"]
    n = sum(new)
    x = 3.0 * r.normal(n, vocab)
    x = x.half() if case["f16"] else x
    s = {"x": x, "probs": None, "offsets": torch.tensor(_offsets(new), dtype=torch.int32).cuda()}
    if case["probs"]:
        # a draft model that is near the target; its tokens come from its probabilities
        s["probs"] = torch.softmax(0.9 * x.float() + 0.6 * r.normal(n, vocab), -1)
        at = torch.cumsum(s["probs"], -1, dtype=torch.float64)
        at /= at[:, -1:].clone()
        drafts = torch.searchsorted(at, r.uniform(n, 1).double(), right=True)[:, 0]
        drafts = drafts.clamp(max=vocab - 1)
    else:
        # mostly the likeliest token
        drafts = torch.where(r.uniform(n) < 0.7, x.argmax(-1), (vocab * r.uniform(n)).long())
    s["drafts"] = drafts.to(torch.int32)
    s["accept_u"], s["sample_u"] = r.uniform(n), r.uniform(case["seqs"])
    s["temperature"] = 0.5 + r.uniform(case["seqs"])
    if case["greedy"]:
        s["temperature"][::2] = 0.0
    s["counts"] = torch.zeros(case["seqs"], device="cuda", dtype=torch.int32)
    s["tokens"] = torch.zeros(n, device="cuda", dtype=torch.int32)
    return s


_ctx = None


def _context():
    """The program's one context."""
    global _ctx
    if _ctx is None:
        from aiimage_amd import aexq
        _ctx = aexq.Context(0)
    return _ctx


def prepare(case, seed):
    state = globals()["_prepare_" + case["op"]](case, seed)
    state["case"] = case
    if own:
        from aiimage_amd import aexq
        state["ctx"] = _context()
        if "state" in state:
            state["slots"] = aexq.slots(case["seqs"] + 3, case["seqs"], slot=state["slot"],
                                        lengths=state["lengths"], counts=state["counts"])
        if case["op"] == "verify":
            state["logits"] = aexq.describe(state["x"], *state["x"].shape)
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state, state["case"])


def _own_conv(s, c):
    s["ctx"].short_conv(s["slots"], s["state"], s["offsets"], s["x"], s["weight"], s["out"],
                        bias=s["bias"])
    return {"out": s["out"], "state": s["state"]}


def _own_delta(s, c):
    s["ctx"].delta_prompt(s["slots"], s["state"], s["offsets"], s["q"], s["k"], s["v"], s["a"],
                          s["b"], s["a_log"], s["dt_bias"], s["out"], scale=c["dk"] ** -0.5,
                          eps=EPS)
    return {"out": s["out"], "state": s["state"]}


def _own_step(s, c):
    s["ctx"].delta_decode(s["slots"], s["state"], s["q"], s["k"], s["v"], s["a"], s["b"],
                          s["a_log"], s["dt_bias"], s["out"], scale=c["dk"] ** -0.5, eps=EPS)
    return {"out": s["out"], "state": s["state"]}


def _own_norm(s, c):
    s["ctx"].gated_rmsnorm(s["x"], s["z"], s["gamma"], s["out"], eps=EPS)
    return s["out"]


def _own_verify(s, c):
    s["ctx"].verify_drafts(s["logits"], s["offsets"], s["drafts"], s["accept_u"], s["sample_u"],
                           s["counts"], s["tokens"], temperature=s["temperature"],
                           draft_probs=s["probs"])
    return {"counts": s["counts"], "tokens": s["tokens"]}


def _rows(s, c):
    """Of each packed row: its sequence, its place among that one's rows, and
    whether it is taken."""
    first = s["offsets"].long()
    new = first[1:] - first[:-1]
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), new,
                                  output_size=s["out"].shape[0])
    place = torch.arange(s["out"].shape[0], device="cuda") - first[seq]
    kept = new if s["counts"] is None else torch.minimum(new, s["counts"].long())
    return seq, place, kept


def _plain_conv(s, c):
    seq, place, kept = _rows(s, c)
    back = c["width"] - 1
    fresh = s["lengths"].long() <= s["offsets"].long().diff()
    old = torch.where(fresh[:, None, None], 0, s["state"][s["slot"].long()])  # [seqs][back][channels]

    def inputs(seq, place):
        """The inputs at `place`, the state's where that is below 0."""
        row = (s["offsets"].long()[seq] + place).clamp(0, s["x"].shape[0] - 1)
        before = old[seq, (place + back).clamp(0, max(back - 1, 0))]
        return torch.where((place >= 0)[..., None], s["x"][row], before)

    y = torch.zeros(s["x"].shape, device="cuda") if s["bias"] is None else s["bias"].expand(
        s["x"].shape)
    for j in range(c["width"]):
        y = y + s["weight"][:, j] * inputs(seq, place - back + j).float()
    y = y / (1 + torch.exp(-y))
    s["out"].copy_(torch.where((place < kept[seq])[:, None], y.half(), s["out"]))
    at = kept[:, None] + torch.arange(back, device="cuda") - back
    left = inputs(torch.arange(c["seqs"], device="cuda")[:, None].expand(at.shape), at)
    s["state"][s["slot"].long()] = left
    return {"out": s["out"], "state": s["state"]}


def _unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)


def _gates(s):
    """Log decays and strengths [tokens][heads_v] in 64 bits."""
    t = s["a"].double() + s["dt_bias"].double()
    soft = torch.clamp(t, min=0) + torch.log1p(torch.exp(-t.abs()))
    return -torch.exp(s["a_log"].double()) * soft, 1 / (1 + torch.exp(-s["b"].double()))


def _plain_delta(s, c):
    """Chunks of 64 rows: inside a chunk the rows' corrections of one another are
    the inverse of a triangular matrix; from chunk to chunk goes the state."""
    hv, dk = c["hv"], c["dk"]
    g, beta = _gates(s)
    _, place, kept = _rows(s, c)
    first, fresh = s["offsets"].long(), s["lengths"].long() <= s["offsets"].long().diff()
    q, k, v = _unit(s["q"].float()), _unit(s["k"].float()), s["v"].float()
    eye = torch.eye(CHUNK, device="cuda")
    below = torch.ones((CHUNK, CHUNK), device="cuda").tril(-1) > 0
    upto = below | (eye > 0)
    same = {}                                 # sequences of as many chunks go together
    for i, n in enumerate(_new(c)):
        same.setdefault(-(-n // CHUNK), []).append(i)
    for chunks, members in same.items():
        seq = torch.tensor(members, device="cuda")
        at = torch.arange(chunks * CHUNK, device="cuda")
        real = at < kept[seq][:, None]                                     # [B][rows]
        row = torch.where(real, first[seq][:, None] + at, 0)

        def cut(x, heads):
            """[B][heads_v][chunks][64][...] of packed rows, zero where there is none."""
            y = torch.where(real[(...,) + (None,) * (x.dim() - 1)], x[row], 0)
            y = y.repeat_interleave(hv // heads, 2).unflatten(1, (chunks, CHUNK))
            return y.movedim(3, 1)

        Q, K, V = cut(q, c["hk"]), cut(k, c["hk"]), cut(v, hv)
        G, B = torch.cumsum(cut(g, hv), -1), cut(beta, hv).float()
        pairs = torch.exp(torch.where(upto, G[..., :, None] - G[..., None, :], -math.inf)).float()
        A = torch.where(below, B[..., None] * pairs * (K @ K.mT), 0)
        T = eye.expand(A.shape).clone()
        for i in range(1, CHUNK):
            T[..., i, :i] = -(A[..., i, None, :i] @ T[..., :i, :i])[..., 0, :]
        P = torch.where(upto, pairs * (Q @ K.mT), 0)
        S = torch.where(fresh[seq][:, None, None, None], 0, s["state"][s["slot"][seq].long()])
        out = torch.empty_like(V)
        for n in range(chunks):
            e = torch.exp(G[:, :, n]).float()[..., None]
            U = T[:, :, n] @ (B[:, :, n, :, None] * (V[:, :, n] - e * (K[:, :, n] @ S)))
            out[:, :, n] = e * (Q[:, :, n] @ S) + P[:, :, n] @ U
            left = torch.exp(G[:, :, n, -1:] - G[:, :, n]).float()[..., None]
            S = e[:, :, -1:] * S + (left * K[:, :, n]).mT @ U
        s["state"][s["slot"][seq].long()] = S
        out = (out * dk ** -0.5).half().movedim(1, 3).flatten(1, 2)
        s["out"][row[real]] = out[real]
    return {"out": s["out"], "state": s["state"]}


def _plain_step(s, c):
    group, slot = c["hv"] // c["hk"], s["slot"].long()
    g, beta = _gates(s)
    q, k = (_unit(s[x].float()).repeat_interleave(group, 1) for x in ("q", "k"))
    S = torch.where((s["lengths"] <= 1)[:, None, None, None], 0, s["state"][slot])
    S = S * torch.exp(g).float()[..., None, None]
    u = beta.float()[..., None] * (s["v"].float() - (S * k[..., None]).sum(2))
    S = S + k[..., None] * u[:, :, None]
    s["state"][slot] = S
    s["out"].copy_((S * q[..., None]).sum(2) * c["dk"] ** -0.5)
    return {"out": s["out"], "state": s["state"]}


def _plain_norm(s, c):
    x, z = s["x"].float(), s["z"].float()
    y = x / torch.sqrt(torch.clamp((x * x).mean(-1, keepdim=True) + EPS, min=1e-20))
    if s["gamma"] is not None:
        y = y * s["gamma"]
    s["out"].copy_(y * z / (1 + torch.exp(-z)))
    return s["out"]


def _plain_verify(s, c):
    n, seqs = s["x"].shape[0], c["seqs"]
    first = s["offsets"].long()
    new = first[1:] - first[:-1]
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), new, output_size=n)
    place = torch.arange(n, device="cuda") - first[seq]
    drafts, heat = s["drafts"].long(), s["temperature"]
    x = s["x"].float()
    best = x.argmax(-1)
    cold = heat[seq] <= 0
    over = torch.where(cold, 1.0, heat[seq])[:, None]
    e = torch.exp((x - x.amax(-1, keepdim=True)) / over)
    p = e.gather(1, drafts[:, None])[:, 0] / e.sum(-1)
    q = s["probs"].gather(1, drafts[:, None])[:, 0] if s["probs"] is not None else 1.0
    good = torch.where(cold, drafts == best, s["accept_u"] * q < p)
    # the rows that are accepted from a sequence's first on
    bad = (~good | (place == new[seq] - 1)).long()
    passed = torch.cumsum(bad, 0) - bad
    passed = passed - passed[first[:-1]][seq]
    counts = torch.zeros(seqs, dtype=torch.long, device="cuda").index_add_(
        0, seq, (passed == 0).long())
    row = first[:-1] + counts - 1                       # the row that the new token comes from
    last = counts == new
    # 64 bits: a cumulative sum over the vocabulary meets a number next to a border
    y = s["x"][row].double()
    e = torch.exp((y - y.amax(-1, keepdim=True)) / over[row].double())
    w = e / e.sum(-1, keepdim=True)
    if s["probs"] is not None:
        taken = s["probs"][row].double()
    else:
        taken = torch.zeros_like(w).scatter_(1, drafts[row][:, None], 2.0)
    rest = torch.clamp(w - taken, min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    w = torch.where(last[:, None], w, rest)
    upto = torch.cumsum(w, -1)
    token = (upto <= s["sample_u"].double()[:, None] * upto[:, -1:]).sum(-1)
    token = torch.where(cold[row], best[row], token.clamp(max=c["vocab"] - 1))
    tokens = torch.where(place < counts[seq] - 1, drafts, -1)
    tokens[row] = token
    s["counts"].copy_(counts)
    s["tokens"].copy_(tokens)
    return {"counts": s["counts"], "tokens": s["tokens"]}


# ---------------------------------------------------------------- what it takes

def work(case):
    """Every input read once, every output written once; states read where a
    sequence has a past, and written."""
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["heads"] * case["d"]
        return {"bytes": 6 * n + (4 * case["d"] if case["gamma"] else 0), "flops": 10 * n}
    new, kept, past = _new(case), _kept(case), _past(case)
    if op == "verify":
        n, each = sum(new), 2 if case["f16"] else 4
        # (of the draft's probabilities one row of a sequence, and one value of the others)
        probs = 4 * (case["seqs"] * case["vocab"] + n) if case["probs"] else 0
        return {"bytes": n * (case["vocab"] * each + 12) + 12 * case["seqs"] + probs,
                "flops": 5 * n * case["vocab"]}
    rows, states = sum(kept), sum(2 if p else 1 for p in past)
    if op == "conv":
        c, w = case["channels"], case["width"]
        return {"bytes": 4 * rows * c + 2 * states * (w - 1) * c + 4 * c * (w + case["bias"]),
                "flops": (2 * w + 4) * rows * c}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    return {"bytes": 2 * rows * (2 * hk * dk + 2 * hv * dv + 2 * hv) + 4 * states * hv * dk * dv,
            "flops": 7 * rows * hv * dk * dv}


# ---------------------------------------------------------------- 64-bit results

def exact(case, seed):
    return globals()["_exact_" + case["op"]](case, seed)


def _exact_conv(case, seed):
    s = _prepare_conv(case, seed)
    back, at = case["width"] - 1, _offsets(_new(case))
    out, state = s["out"].double(), s["state"].double()
    w = s["weight"].double()
    for i, (slot, kept) in enumerate(zip(s["slot"].tolist(), _kept(case))):
        x = torch.cat([state[slot], s["x"][at[i]:at[i] + kept].double()])
        if _past(case)[i] == 0:
            x[:back] = 0
        y = (x.unfold(0, back + 1, 1) * w).sum(-1)
        if s["bias"] is not None:
            y = y + s["bias"].double()
        out[at[i]:at[i] + kept] = y * torch.sigmoid(y)
        state[slot] = x[kept:]
    return {"out": out, "state": state}


def _exact_delta(case, seed):
    """Row by row, all sequences at once."""
    s = _prepare_delta(case, seed)
    new, kept = _new(case), _kept(case)
    first, slot = torch.tensor(_offsets(new)[:-1], device="cuda"), s["slot"].long()
    kept_dev = torch.tensor(kept, device="cuda")
    group = case["hv"] // case["hk"]
    out, pool = s["out"].double(), s["state"].double()
    S = pool[slot].clone()
    S[torch.tensor([p == 0 for p in _past(case)], device="cuda")] = 0
    rate, bias = s["a_log"].double().exp(), s["dt_bias"].double()
    for t in range(max(kept)):
        on = torch.nonzero(kept_dev > t)[:, 0]
        row = first[on] + t
        q, k = (torch.nn.functional.normalize(x, dim=-1, eps=0.0) * (
            x.norm(dim=-1, keepdim=True) / (x.square().sum(-1, keepdim=True) + EPS).sqrt())
            for x in (s["q"][row].double(), s["k"][row].double()))
        q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
        decay = torch.exp(-rate * torch.nn.functional.softplus(s["a"][row].double() + bias))
        part = S[on] * decay[..., None, None]
        seen = torch.matmul(k[:, :, None], part)[:, :, 0]
        u = torch.sigmoid(s["b"][row].double())[..., None] * (s["v"][row].double() - seen)
        part = part + k[..., None] * u[:, :, None]
        S[on] = part
        out[row] = torch.matmul(q[:, :, None], part)[:, :, 0] / math.sqrt(case["dk"])
    pool[slot] = S
    return {"out": out, "state": pool}


def _exact_step(case, seed):
    return _exact_delta({**case, "lo": 1, "hi": 1}, seed)


def _exact_norm(case, seed):
    s = _prepare_norm(case, seed)
    x, z = s["x"].double(), s["z"].double()
    y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * torch.nn.functional.silu(z)
    return y if s["gamma"] is None else y * s["gamma"].double()


def _exact_verify(case, seed):
    s = _prepare_verify(case, seed)
    at, drafts = _offsets(_new(case)), s["drafts"].tolist()
    counts, tokens = [], [-1] * at[-1]
    for i in range(case["seqs"]):
        heat = float(s["temperature"][i])
        for r in range(at[i], at[i + 1]):
            x = s["x"][r].double()
            p = torch.softmax(x / heat, -1) if heat > 0 else (
                torch.arange(x.numel(), device="cuda") == x.argmax()).double()
            w = p
            if r < at[i + 1] - 1:
                d = drafts[r]
                q = s["probs"][r].double() if s["probs"] is not None else torch.zeros_like(p)
                if s["probs"] is None:
                    q[d] = 1.0
                if float(p[d]) > 0 and (heat <= 0 or
                                        float(s["accept_u"][r]) * float(q[d]) < float(p[d])):
                    tokens[r] = d
                    continue
                w = torch.relu(p - q) if heat > 0 else p
                w = w if float(w.sum()) > 0 else p
            total = torch.cumsum(w, 0)
            goal = float(s["sample_u"][i]) * float(total[-1]) if heat > 0 else 0.0
            tokens[r] = int(torch.nonzero(total > goal)[0])
            counts.append(r - at[i] + 1)
            break
    return {"counts": torch.tensor(counts, dtype=torch.int32).cuda(),
            "tokens": torch.tensor(tokens, dtype=torch.int32).cuda()}

"""Log probabilities, entropy and top alternatives against 64 bits.

Bound: a lane adds up n / 256 exponentials one after the other, each sum off by
2^-24 of it, and an exponent of y in log2 units is off by 2^-23 |y| (y below 40
where the weight matters): the logarithm of the sum by (n / 256 + 64) 2^-24 at
most, the mean of x - m by that times its size, each result by its own rounding."""
import math

import pytest

torch = pytest.importorskip("torch")

import serving_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu


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


def _outputs(rows, top):
    f = lambda *s: torch.full(s, 7.0, device="cuda")  # noqa: E731
    return (f(rows), f(rows), torch.full((rows, top), 7, dtype=torch.int32, device="cuda"),
            f(rows, top))


def _check(x, tokens, got):
    top = got[2].shape[1]
    want = ref.logprobs(x, tokens, top)
    n = x.shape[1]
    eps = (n / 256 + 64) * 2.0 ** -24
    assert torch.equal(got[2], want[2])
    for g, w in ((got[0], want[0]), (got[3], want[3])):
        g, w = g.double(), w.double()
        low = torch.isneginf(w)
        assert torch.equal(torch.isneginf(g), low)
        assert ((g - w).abs() <= eps + 2.0 ** -22 * w.abs())[~low].all()
    assert ((got[1].double() - want[1]).abs() <= 2 * eps * (1 + want[1].abs())).all()


def _run(aexq, ctx, x, tokens, top, stride=None):
    rows, n = x.shape
    out = _outputs(rows, top)
    ctx.logprobs(aexq.describe(x, rows, n), tokens, *out)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,n,top", [
    (1, 1, 1), (1, 7, 0), (3, 7, 7), (2, 64, 64), (5, 1001, 20), (1, 4099, 5), (1, 20011, 20),
    (1, 151936, 20), (4, 151936, 64), (2, 50257, 1), (600, 3001, 8), (9, 12345, 33)])
def test_rows(aexq, ctx, rows, n, top, dtype):
    print(f"[gpu-case] logprobs {rows} x {n} top={top} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    x = (3 * torch.randn((rows, n), generator=g, device="cuda")).to(dtype)
    tokens = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    _check(x, tokens, _run(aexq, ctx, x, tokens, top))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,n", [(1, 9000), (700, 2500)])
@pytest.mark.parametrize("kind", ["equal", "steps", "rising", "falling", "one lane", "banned",
                                  "far", "lowest", "zeros"])
def test_orders_and_ties(aexq, ctx, rows, n, kind, dtype):
    """Ties go to the lower index, wherever the largest logits lie."""
    print(f"[gpu-case] logprobs {kind} {rows} x {n} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    i = torch.arange(n, device="cuda").float()
    x = torch.randn((rows, n), generator=g, device="cuda")
    if kind == "equal":
        x = torch.full((rows, n), 2.5, device="cuda")
    elif kind == "steps":
        x = torch.floor(x * 2)
    elif kind == "rising":
        x = (i / n * 20).expand(rows, n).contiguous()
    elif kind == "falling":
        x = (-i / n * 20).expand(rows, n).contiguous()
    elif kind == "one lane":  # every large logit in the chunks of one lane
        x = torch.where((i.long() // 8) % 256 == 77, x + 15, x)
        x = torch.where((i.long() // 4) % 256 == 30, x + 15, x)
    elif kind == "banned":
        x[:, torch.rand(n, generator=g, device="cuda") < 0.9] = -math.inf
        x[:, 11] = 0.5
    elif kind == "far":  # one logit holds all the weight
        x[:, 300] = 1000.0
    elif kind == "lowest":  # masks of the type's lowest value
        x[:, 100:] = torch.finfo(dtype).min
    else:
        x = torch.where(x > 0, 0.0, -0.0)
    x = x.to(dtype)
    tokens = torch.full((rows,), 11, dtype=torch.int32, device="cuda")
    _check(x, tokens, _run(aexq, ctx, x, tokens, 20))


def test_more_alternatives_than_finite_logits(aexq, ctx):
    print("[gpu-case] logprobs few finite logits", flush=True)
    for n in (50, 9000):
        x = torch.full((2, n), -math.inf, device="cuda")
        x[:, 30], x[:, 33], x[1, 40] = 1.0, 2.0, 2.0
        tokens = torch.tensor([30, 5], dtype=torch.int32, device="cuda")
        got = _run(aexq, ctx, x, tokens, 6)
        _check(x, tokens, got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,n", [(1, 9000), (700, 2500)])
def test_masks_of_the_lowest_value(aexq, ctx, rows, n, dtype):
    """A masked logit's own probability, and rows of nothing but masks: finite."""
    print(f"[gpu-case] logprobs lowest values {rows} x {n} {dtype}", flush=True)
    low = torch.finfo(dtype).min
    x = torch.full((rows, n), low, device="cuda", dtype=dtype)
    tokens = torch.full((rows,), n - 3, dtype=torch.int32, device="cuda")
    _check(x, tokens, _run(aexq, ctx, x, tokens, 20))
    x[:, n // 2:n // 2 + 5] = 3.0  # fewer than the alternatives
    _check(x, tokens, _run(aexq, ctx, x, tokens, 20))
    x[:, n // 2] = -low / 2 ** 40
    _check(x, tokens, _run(aexq, ctx, x, tokens, 20))
    x[:] = -math.inf
    x[:, 7:9] = low
    _check(x, tokens, _run(aexq, ctx, x, tokens, 20))


@pytest.mark.parametrize("n", [500, 9000])
def test_rows_without_probabilities(aexq, ctx, n):
    """A NaN, a +inf or nothing but -inf: NaN and ids of -1, the rows beside them
    untouched; token -1 is 0, one outside the row NaN."""
    print(f"[gpu-case] logprobs odd rows n={n}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((7, n), generator=g, device="cuda")
    x[0, 3], x[2, n - 1], x[4] = math.nan, math.inf, -math.inf
    tokens = torch.tensor([1, 2, 3, -1, 4, n, -2], dtype=torch.int32, device="cuda")
    lp, ent, ids, val = _run(aexq, ctx, x, tokens, 4)
    for r in (0, 2, 4):
        assert math.isnan(lp[r]) and math.isnan(ent[r])
        assert (ids[r] == -1).all() and torch.isnan(val[r]).all()
    assert lp[3] == 0 and math.isnan(lp[5]) and math.isnan(lp[6])
    good = torch.tensor([1, 3, 5, 6], device="cuda")
    ref_ = ref.logprobs(x[good], tokens[good], 4)
    assert torch.equal(ids[good], ref_[2])
    assert (ent[good].double() - ref_[1]).abs().max() <= 1e-4
    assert abs(lp[1].item() - ref_[0][0].item()) <= 1e-5


@pytest.mark.parametrize("layout", ["PACK4_LINEAR", "PACK4_TILED"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_layouts_and_single_outputs(aexq, ctx, layout, dtype):
    """The layouts the LM head writes, whose rows are padded, and each output alone."""
    print(f"[gpu-case] logprobs {layout} {dtype}", flush=True)
    lay = getattr(aexq, "LAYOUT_" + layout)
    rows, n, top = 3, 40003, 5
    buf = aexq.new_activation(rows, n, dtype, lay)
    buf.fill_(50.0)  # padding must not count
    x = buf.view(rows, -1)[:, :n]
    g = torch.Generator(device="cuda").manual_seed(5)
    x.copy_(torch.randn((rows, n), generator=g, device="cuda"))
    d = aexq.describe(buf, rows, n, lay)
    tokens = torch.tensor([0, n - 1, 17], dtype=torch.int32, device="cuda")
    out = _outputs(rows, top)
    ctx.logprobs(d, tokens, *out)
    torch.cuda.synchronize()
    _check(x, tokens, out)
    alone = _outputs(rows, top)
    ctx.logprobs(d, tokens, alone[0])
    ctx.logprobs(d, None, None, alone[1])
    ctx.logprobs(d, None, None, None, alone[2])
    ctx.logprobs(d, None, None, None, None, alone[3])
    torch.cuda.synchronize()
    for a, b in zip(alone, out):
        assert torch.equal(a, b)

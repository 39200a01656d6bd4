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

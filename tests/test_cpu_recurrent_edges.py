"""Outputs of the recurrent layers' operators and of the verification of drafted tokens
that overlap their inputs, without a GPU."""
import ctypes
import random

import pytest

import fake_hip
from aiimage_amd import _abi
from test_cpu_recurrent import INVALID, PRELUDE, PTR, _norm, _verify, handle, lib  # noqa: F401


def _meet(a, a_stride, a_width, b, b_stride, b_width, rows):
    """By their elements."""
    of = lambda p, s, w: {p // 2 + i * s + j for i in range(rows) for j in range(w)}  # noqa: E731
    return bool(of(a, a_stride, a_width) & of(b, b_stride, b_width))


def _layouts(n, seed=1):
    r = random.Random(seed)
    for _ in range(n):
        rows, (wa, wb) = r.randint(1, 6), (r.randint(1, 9) for _ in range(2))
        sa = wa + r.randint(0, 20)
        sb = r.choice([max(sa, wb), wb + r.randint(0, 20)])
        sa = sb if r.random() < 0.5 and sb >= wa else sa
        yield 2000, sa, wa, 2000 + 2 * r.randint(-100, 100), sb, wb, rows


def test_rows_that_share_memory():
    aexq = pytest.importorskip("aiimage_amd.aexq")
    met = 0
    for layout in _layouts(4000):
        want = _meet(*layout)
        met += want
        assert aexq._rows_meet(*layout) == want, layout
    assert 500 < met < 3500


def test_norm_over_rows_that_are_still_read(lib, handle):  # noqa: F811
    """The rows' elements decide, in units of 8, as the entry point takes them; in place is
    no overlap.  (What does not overlap is answered by a later check: no context is there.)"""
    from aiimage_amd import aexq
    r, met = random.Random(2), 0
    for _ in range(400):
        rows, width = r.randint(1, 5), 8 * r.randint(1, 4)
        a_stride = width + 8 * r.randint(0, 6)
        b_stride = r.choice([a_stride, width + 8 * r.randint(0, 6)])
        by = 16 * r.randint(-40, 40)
        if not aexq._rows_meet(PTR, a_stride, width, PTR + by, b_stride, width, rows) or by == 0:
            continue
        met += 1
        far = PTR + (1 << 18)
        for x, z in (((PTR, a_stride), (far, width)), ((far, width), (PTR, a_stride))):
            assert _norm(lib, handle, x=x[0], x_stride=x[1], z=z[0], z_stride=z[1], out=PTR + by,
                         out_stride=b_stride, tokens=rows, heads=1, dim=width) == INVALID
            assert b"overlaps" in lib.aexq_last_error()
    assert met > 50    # (of 400 draws: enough of either stride)


@pytest.mark.parametrize("over", [
    dict(tokens=PTR + 4), dict(tokens=PTR - 32), dict(tokens=PTR + 64), dict(counts=PTR + 128 + 32),
    dict(counts=PTR), dict(accept_u=PTR + 128 - 4), dict(sample_u=PTR + 64 + 8),
    dict(temperature=PTR + 128), dict(offsets=PTR + 64 - 12)])
def test_verify_over_arrays_that_are_still_read(lib, handle, over):  # noqa: F811
    assert _verify(lib, handle, **over) == INVALID
    assert lib.aexq_last_error()


def test_rows_side_by_side_are_no_overlap(tmp_path):
    """Views of one buffer, rows between rows, in place, and arrays one behind the other."""
    fake_hip.run(tmp_path, PRELUDE + """
norm = lambda x, xs, z, zs, o, os: lib.aexq_gated_rmsnorm(ctx, x, xs, z, zs, PTR, 1e-6, 9, 1, 128, o, os)
for args in ((PTR, 384, PTR + 256, 384, PTR + 512, 384), (PTR, 128, PTR, 128, PTR, 128),
             (PTR, 128, PTR + 2304, 128, PTR + 4608, 128), (PTR, 128, PTR + 2304, 256, PTR, 128),
             (PTR + 4608, 128, PTR + 2304, 128, PTR, 128), (PTR, 512, PTR + 256, 512, PTR + 512, 256 + 768),
             (PTR, 512, PTR + 256, 1024, PTR + 256, 1024)):
    assert norm(*args) == 0, (args, lib.aexq_last_error())
assert lib.aexq_verify_drafts(ctx, logits, PTR, 3, PTR, None, 0, None, PTR, PTR, PTR + 36,
                              PTR + 48) == 0, lib.aexq_last_error()
""")


# ---- scratch: sizes whose need is so little above a power of two that what is allocated
# for it without any one of its parts does not hold it

@pytest.mark.parametrize("sequences,rows,vocab,f16", [(7, 35, 5000, True), (10, 10, 5000, False),
                                                      (28, 35, 33000, True)])
def test_scratch_of_a_verification_holds_all_of_its_parts(tmp_path, sequences, rows, vocab, f16):
    """Of each sequence what was decided and what its row sums to, of each of its runs two
    sums; of each row its draft, of each of its parts a sum, a logit and an index."""
    chunks = (vocab * (2 if f16 else 4) + 15) // 16
    parts = max(1, min(64, (8 * 256 + rows - 1) // rows, (chunks + 511) // 512))
    runs = min(256, ((vocab + 255) // 256 + 3) // 4 * 4)
    held = [16 * sequences, 16 * sequences, 16 * rows, 16 * sequences * runs, 8 * rows * parts,
            4 * rows * parts, 4 * rows * parts]
    need, power = sum(held), 4096
    while 2 * power < need:
        power *= 2
    assert need - min(held) <= power < need
    fake_hip.run(tmp_path, PRELUDE + f"""
logits.logical = logits.storage = _abi.Shape(2, {vocab}, {rows}, 1, 1)
logits.dtype = _abi.{"DTYPE_F16" if f16 else "DTYPE_F32"}
before = fake.fake_bytes()
assert lib.aexq_verify_drafts(ctx, logits, PTR, {sequences}, PTR, PTR, {vocab}, PTR, PTR, PTR,
                              PTR + 4096, PTR + 8192) == 0, lib.aexq_last_error()
got = fake.fake_bytes() - before
assert {need} <= got <= {2 * need}, got
""")


def test_scratch_of_the_delta_rule_holds_its_list_of_long_sequences(tmp_path):
    """Blocks that fill a power of two but for 64 bytes, and behind them the number of the
    sequences of more than 16 rows and their names."""
    n, tokens, hk, hv, dk, dv = 89, 44 * 64, 1, 3, 128, 128
    blocks = (tokens // 64 + n) * (hv * (24 * 1024 + 4 * 64 * 4 + 64) + hk * 3 * 64 * dk * 2)
    assert blocks == 2 ** 24 - 64 and blocks + 4 * (n + 1) > 2 ** 24
    fake_hip.run(tmp_path, PRELUDE + f"""
before = fake.fake_bytes(), fake.fake_launches()
assert lib.aexq_delta_prompt(ctx, slots(sequences={n}, count={n}), PTR, PTR, {tokens}, PTR, {hk * dk}, PTR,
    {hk * dk}, PTR, {hv * dv}, PTR, {hv}, PTR, {hv}, PTR, PTR, {hk}, {hv}, {dk}, {dv}, 0.1, 1e-6,
    PTR + 64, {hv * dv}) == 0, lib.aexq_last_error()
assert fake.fake_launches() - before[1] == 3    # (the sequences of up to 16 rows go apart)
got = fake.fake_bytes() - before[0]
assert {blocks + 4 * (n + 1)} <= got, got
""")

"""The recurrent layers' operators and the verification of drafted tokens without a
GPU: refusals that come before the device or the context is touched, the layout of
their struct, what the host side launches and allocates."""
import ctypes
import os
import re
import subprocess

import pytest

import fake_hip
from aiimage_amd import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20    # 16-byte aligned, never read
INVALID, SHAPE, UNSUPPORTED = _abi.ERR_INVALID_ARGUMENT, _abi.ERR_SHAPE, _abi.ERR_UNSUPPORTED
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib():
    return _abi.load()


_keep = ctypes.create_string_buffer(1 << 12)


@pytest.fixture
def handle():
    """Stands where a context would; the refusals come before it is read."""
    return ctypes.addressof(_keep)


def _slots(**over):
    d = dict(slot=PTR, lengths=PTR, counts=PTR, count=8, sequences=3, read_only=0)
    d.update(over)
    return _abi.Slots(**d)


def _conv(lib, handle, **over):
    a = dict(slots=_slots(), state=PTR, offsets=PTR, tokens=9, x=PTR, x_stride=256, weight=PTR,
             bias=None, channels=256, width=4, silu=1, out=PTR + 64, out_stride=256)
    assert set(over) <= set(a)
    a.update(over)
    return lib.aexq_short_conv(handle, *a.values())


def _delta(lib, handle, decode=False, **over):
    a = dict(slots=_slots(), state=PTR, offsets=PTR, tokens=9, q=PTR, q_stride=256, k=PTR,
             k_stride=256, v=PTR, v_stride=512, a=PTR, a_stride=4, b=PTR, b_stride=4, a_log=PTR,
             dt_bias=PTR, heads_k=2, heads_v=4, dim_k=128, dim_v=128, scale=0.1, eps=1e-6,
             out=PTR + 64, out_stride=512)
    assert set(over) <= set(a)
    a.update(over)
    if decode:
        a.pop("offsets")
        a.pop("tokens")
        return lib.aexq_delta_decode(handle, *a.values())
    return lib.aexq_delta_prompt(handle, *a.values())


def _norm(lib, handle, **over):
    a = dict(x=PTR, x_stride=512, z=PTR, z_stride=512, gamma=PTR, eps=1e-6, tokens=9, heads=4,
             dim=128, out=PTR + 64, out_stride=512)
    assert set(over) <= set(a)
    a.update(over)
    return lib.aexq_gated_rmsnorm(handle, *a.values())


def _logits(data=PTR, dtype=_abi.DTYPE_F32, w=500, h=9, batch=1):
    t = _abi.Tensor()
    t.logical = t.storage = _abi.Shape(2, w, h, 1, 1)
    t.layout, t.dtype, t.data, t.batch = _abi.LAYOUT_LINEAR, dtype, data, batch
    return t


def _verify(lib, handle, **over):
    a = dict(logits=_logits(), offsets=PTR, sequences=3, drafts=PTR, probs=PTR, stride=500,
             temperature=PTR, accept_u=PTR, sample_u=PTR, counts=PTR + 64, tokens=PTR + 128)
    assert set(over) <= set(a)
    a.update(over)
    return lib.aexq_verify_drafts(handle, *a.values())


@pytest.mark.parametrize("over,status", [
    (dict(count=0), INVALID), (dict(count=-1), INVALID), (dict(sequences=0), INVALID),
    (dict(sequences=65536), UNSUPPORTED)])
def test_slots(lib, handle, over, status):
    for call in (_conv, _delta, lambda l, h, **o: _delta(l, h, decode=True, **o)):
        assert call(lib, handle, slots=_slots(**over)) == status
        assert call(lib, handle, slots=None) == INVALID
        assert call(lib, handle, state=None) == INVALID
        assert call(lib, handle, state=PTR + 4) == UNSUPPORTED
        assert call(lib, None) == INVALID
        assert lib.aexq_last_error()


@pytest.mark.parametrize("over,status", [
    (dict(offsets=None), INVALID), (dict(tokens=0), INVALID), (dict(tokens=(1 << 23) + 1), INVALID),
    (dict(x=None), INVALID), (dict(weight=None), INVALID), (dict(out=PTR), INVALID),
    (dict(channels=0), UNSUPPORTED), (dict(channels=252), UNSUPPORTED),
    (dict(channels=(1 << 20) + 8, x_stride=1 << 21, out_stride=1 << 21), UNSUPPORTED),
    (dict(width=1), UNSUPPORTED), (dict(width=6), UNSUPPORTED), (dict(x_stride=248), SHAPE),
    (dict(x_stride=260), UNSUPPORTED), (dict(x_stride=(1 << 24) + 8), UNSUPPORTED),
    (dict(out_stride=248), SHAPE), (dict(x=PTR + 8), UNSUPPORTED), (dict(out=PTR + 8), UNSUPPORTED),
    (dict(tokens=1 << 23, channels=1 << 16, x_stride=1 << 16, out_stride=1 << 16), UNSUPPORTED)])
def test_conv_arguments(lib, handle, over, status):
    assert _conv(lib, handle, **over) == status
    assert lib.aexq_last_error()


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("over,status", [
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(a=None), INVALID), (dict(b=None), INVALID), (dict(a_log=None), INVALID),
    (dict(dt_bias=None), INVALID), (dict(heads_k=0), INVALID), (dict(heads_k=3), INVALID),
    (dict(heads_v=0), INVALID), (dict(dim_k=256), UNSUPPORTED), (dict(dim_k=96), UNSUPPORTED),
    (dict(dim_v=96), UNSUPPORTED), (dict(dim_v=32), UNSUPPORTED),
    (dict(eps=0.0), INVALID), (dict(eps=NAN), INVALID), (dict(eps=INF), INVALID),
    (dict(scale=NAN), INVALID), (dict(scale=-INF), INVALID),
    (dict(q_stride=248), SHAPE), (dict(k_stride=252), SHAPE), (dict(v_stride=504), SHAPE),
    (dict(out_stride=504), SHAPE), (dict(q_stride=260), UNSUPPORTED), (dict(v=PTR + 8), UNSUPPORTED),
    (dict(k_stride=(1 << 24) + 8), UNSUPPORTED), (dict(a_stride=3), SHAPE), (dict(b_stride=3), SHAPE),
    (dict(a_stride=(1 << 24) + 1), SHAPE), (dict(a=PTR + 1), UNSUPPORTED),
    (dict(b=PTR + 1), UNSUPPORTED), (dict(out=PTR), INVALID),
    (dict(slots=_slots(sequences=65535), heads_k=64, heads_v=64, q_stride=8192, k_stride=8192,
          v_stride=8192, out_stride=8192, a_stride=64, b_stride=64), UNSUPPORTED)])
def test_delta_arguments(lib, handle, decode, over, status):
    assert _delta(lib, handle, decode, **over) == status
    assert lib.aexq_last_error()


@pytest.mark.parametrize("over,status", [
    (dict(offsets=None), INVALID), (dict(tokens=0), INVALID), (dict(tokens=(1 << 23) + 1), INVALID)])
def test_delta_rows(lib, handle, over, status):
    assert _delta(lib, handle, **over) == status


@pytest.mark.parametrize("over,status", [
    (dict(x=None), INVALID), (dict(z=None), INVALID), (dict(out=None), INVALID),
    (dict(tokens=0), INVALID), (dict(tokens=(1 << 23) + 1), INVALID), (dict(heads=0), INVALID),
    (dict(heads=65536), INVALID), (dict(dim=0), UNSUPPORTED), (dict(dim=100), UNSUPPORTED),
    (dict(dim=520), UNSUPPORTED), (dict(eps=-1.0), INVALID), (dict(eps=NAN), INVALID),
    (dict(x_stride=504), SHAPE), (dict(z_stride=516), UNSUPPORTED), (dict(x=PTR + 2), UNSUPPORTED),
    (dict(out=PTR, out_stride=520), INVALID), (dict(out=PTR + 128, z=PTR + 128, out_stride=520), INVALID),
    (dict(tokens=1 << 23, heads=1024, dim=8, x_stride=8192, z_stride=8192, out_stride=8192),
     UNSUPPORTED)])
def test_norm_arguments(lib, handle, over, status):
    assert _norm(lib, handle, **over) == status
    assert lib.aexq_last_error()


@pytest.mark.parametrize("over,status", [
    (dict(logits=None), INVALID), (dict(offsets=None), INVALID), (dict(drafts=None), INVALID),
    (dict(accept_u=None), INVALID), (dict(sample_u=None), INVALID), (dict(counts=None), INVALID),
    (dict(tokens=None), INVALID), (dict(tokens=PTR), INVALID), (dict(sequences=0), INVALID),
    (dict(sequences=65536), INVALID), (dict(stride=499), SHAPE), (dict(stride=(1 << 28) + 1), SHAPE),
    (dict(logits=_logits(data=PTR + 2)), UNSUPPORTED), (dict(logits=_logits(dtype=3)), UNSUPPORTED),
    (dict(logits=_logits(batch=2)), UNSUPPORTED), (dict(logits=_logits(w=0)), SHAPE),
    (dict(logits=_logits(w=1 << 25), stride=1 << 25), UNSUPPORTED),
    (dict(logits=_logits(h=(1 << 20) + 1)), UNSUPPORTED)])
def test_verify_arguments(lib, handle, over, status):
    assert _verify(lib, handle, **over) == status
    assert lib.aexq_last_error()


def test_python_entry_points_refuse_before_the_library():
    torch = pytest.importorskip("torch")
    from aiimage_amd import aexq
    i32, f16 = torch.int32, torch.float16
    for name in ("slot", "lengths", "counts"):
        with pytest.raises(_abi.ArgumentError, match="on a GPU"):
            aexq.slots(4, 3, **{name: torch.zeros(3, dtype=i32)})
    d = aexq.slots(4, 3, read_only=True)
    assert (d.count, d.sequences, d.read_only, d.slot, d.lengths, d.counts) == (4, 3, 1, None, None,
                                                                                None)
    rows = torch.zeros((3, 5), dtype=f16)
    assert aexq._gate_rows(rows[:, 1:3], "a", 3, 2, -1) == 5
    assert aexq._gate_rows(rows[:, 1:2], "a", 3, 1, -1) == 5
    for bad in (rows[:, ::2], rows.float()[:, :3], rows[:2, :3]):
        with pytest.raises(_abi.ArgumentError, match="fp16 rows"):
            aexq._gate_rows(bad, "a", 3, 3, -1)


def test_struct_matches_the_c_compiler_and_the_binding(tmp_path):
    fields = _abi.Slots._fields_
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "aexq.h"', "int main(void){",
             'printf("size %zu\\n", sizeof(aexq_slots));']
    lines += [f'printf("{f} %zu\\n", offsetof(aexq_slots, {f}));' for f, _ in fields]
    probe, exe = tmp_path / "probe.c", tmp_path / "probe"
    probe.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(probe), "-o", str(exe)],
                   check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(_abi.Slots)
    for f, _ in fields:
        assert int(got[f]) == getattr(_abi.Slots, f).offset, f
    text = open(os.path.join(ROOT, "bindings", "csharp", "Native.cs")).read()
    body = re.search(r"Sequential\)\]\s*public struct AexqSlots\s*\{(.*?)\n    \}", text,
                     re.S).group(1)
    members = []
    for kind, names in re.findall(r"public (IntPtr|int) ([\w, ]+);", body):
        members += [(kind, n.strip()) for n in names.split(",")]
    snake = lambda n: re.sub(r"(?<=[a-z])([A-Z])", r"_\1", n).lower()  # noqa: E731
    assert [(k == "IntPtr", snake(n)) for k, n in members] == [
        (t is ctypes.c_void_p, f) for f, t in fields]


# ---- launches and scratch, the runtime's calls answered by a stand-in
PRELUDE = """
def slots(**over):
    d = dict(slot=PTR, lengths=PTR, counts=PTR, count=8, sequences=3, read_only=0)
    d.update(over)
    return _abi.Slots(**d)
logits = _abi.Tensor()
logits.logical = logits.storage = _abi.Shape(2, 5000, 9, 1, 1)
logits.layout, logits.dtype, logits.data, logits.batch = (_abi.LAYOUT_LINEAR, _abi.DTYPE_F32,
                                                          PTR, 1)
"""
CALLS = {
    "conv": ("lib.aexq_short_conv(ctx, slots(), PTR, PTR, 900, PTR, 256, PTR, None, 256, 4, 1,"
             " PTR + 64, 256)", 1),
    "prompt": ("lib.aexq_delta_prompt(ctx, slots(), PTR, PTR, 900, PTR, 256, PTR, 256, PTR, 512, PTR,"
               " 4, PTR, 4, PTR, PTR, 2, 4, 128, 128, 0.1, 1e-6, PTR + 64, 512)", 2),
    "prompt, mostly short": (
        "lib.aexq_delta_prompt(ctx, slots(sequences=100, count=100), PTR, PTR, 900, PTR, 256, PTR, 256,"
        " PTR, 512, PTR, 4, PTR, 4, PTR, PTR, 2, 4, 128, 128, 0.1, 1e-6, PTR + 64, 512)", 3),
    "prompt, all short": (  # 16 rows: no sequence can have more
        "lib.aexq_delta_prompt(ctx, slots(sequences=100, count=100), PTR, PTR, 16, PTR, 256, PTR, 256,"
        " PTR, 512, PTR, 4, PTR, 4, PTR, PTR, 2, 4, 128, 128, 0.1, 1e-6, PTR + 64, 512)", 2),
    "decode": ("lib.aexq_delta_decode(ctx, slots(), PTR, PTR, 256, PTR, 256, PTR, 512, PTR, 4, PTR,"
               " 4, PTR, PTR, 2, 4, 128, 128, 0.1, 1e-6, PTR + 64, 512)", 1),
    "norm": ("lib.aexq_gated_rmsnorm(ctx, PTR, 512, PTR, 512, PTR, 1e-6, 9, 4, 128, PTR, 512)", 1),
    "verify": ("lib.aexq_verify_drafts(ctx, logits, PTR, 3, PTR, PTR, 5000, PTR, PTR, PTR, PTR + 64,"
               " PTR + 128)", 3),
}


@pytest.mark.parametrize("name", CALLS)
def test_a_failed_launch_is_reported(tmp_path, name):
    """Whichever of a call's launches fails, the call does, and no later one of its
    launches runs on what the failed one should have left."""
    call, launches = CALLS[name]
    fake_hip.run(tmp_path, PRELUDE + f"""
before = fake.fake_launches()
assert {call} == 0, lib.aexq_last_error()
assert fake.fake_launches() - before == {launches}
for n in range({launches}):
    before = fake.fake_launches()
    fake.fake_fail(n)
    assert {call} != 0, f"launch {{n}} failed unseen"
    assert fake.fake_launches() - before == n + 1, f"launches after the failed {{n}}"
    assert {call} == 0
""")


def test_scratch(tmp_path):
    """Blocks of 64 rows of the delta rule: 25.06 KB a value head and 3 * 64 rows of
    dim_k fp16 a key head, tokens / 64 + sequences blocks; the other operators but the
    verification take none; none grows on a second call.  Sizes round up to a power of two."""
    fake_hip.run(tmp_path, PRELUDE + f"""
def grown(call):
    before = fake.fake_bytes()
    assert call() == 0, lib.aexq_last_error()
    return fake.fake_bytes() - before
for call in (lambda: {CALLS["conv"][0]}, lambda: {CALLS["decode"][0]}, lambda: {CALLS["norm"][0]}):
    assert grown(call) == 0
blocks = 900 // 64 + 3
need = blocks * (4 * (24 * 1024 + 4 * 64 * 4 + 64) + 2 * 3 * 64 * 128 * 2)
got = grown(lambda: {CALLS["prompt"][0]})
assert need <= got <= 2 * need, (need, got)
assert grown(lambda: {CALLS["prompt"][0]}) == 0
got = grown(lambda: {CALLS["verify"][0]})
assert 3 * 32 + 9 * 16 <= got <= 1 << 16, got
assert grown(lambda: {CALLS["verify"][0]}) == 0
""")


def test_refusals_launch_nothing(tmp_path):
    """Calls of more workgroups than a launch may have."""
    fake_hip.run(tmp_path, PRELUDE + f"""
before = fake.fake_launches(), fake.fake_bytes()
assert {CALLS["norm"][0].replace("512", "8192").replace("9, 4, 128", "1 << 23, 1024, 8")} == \
    _abi.ERR_UNSUPPORTED
assert b"one call" in lib.aexq_last_error()
assert {CALLS["conv"][0].replace("900,", "1 << 23,").replace("256", "65536")} == _abi.ERR_UNSUPPORTED
assert b"one call" in lib.aexq_last_error()
assert (fake.fake_launches(), fake.fake_bytes()) == before
""")

"""Refusals of the operators for many sequences, which the library answers
before it touches the device or the context, and the layout of their structs.
No GPU call is made here."""
import ctypes
import os
import re
import subprocess

import pytest

from aiimage_amd import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20    # 16-byte aligned, never read


@pytest.fixture(scope="module")
def lib():
    return _abi.load()


_keep = ctypes.create_string_buffer(1 << 12)


@pytest.fixture
def handle():
    """Stands where a context would; the refusals come before it is read."""
    return ctypes.addressof(_keep)


def _kv(**over):
    d = dict(k=PTR, v=PTR, pages=8, page_size=64, heads_kv=2, head_dim=128, table=PTR,
             lengths=PTR, sequences=3, table_width=4)
    d.update(over)
    return _abi.PagedKv(**d)


def _rope(**over):
    d = dict(cos_table=PTR, sin_table=PTR, positions=PTR, rows=100, rotary_dim=128, axes=1,
             interleaved=0, section0=64)
    d.update(over)
    return _abi.Rope(**d)


BAD_CACHES = [
    (dict(k=None), _abi.ERR_INVALID_ARGUMENT), (dict(v=None), _abi.ERR_INVALID_ARGUMENT),
    (dict(table=None), _abi.ERR_INVALID_ARGUMENT), (dict(lengths=None), _abi.ERR_INVALID_ARGUMENT),
    (dict(pages=0), _abi.ERR_INVALID_ARGUMENT), (dict(heads_kv=0), _abi.ERR_INVALID_ARGUMENT),
    (dict(sequences=0), _abi.ERR_INVALID_ARGUMENT), (dict(table_width=0), _abi.ERR_INVALID_ARGUMENT),
    (dict(page_size=8), _abi.ERR_UNSUPPORTED), (dict(page_size=48), _abi.ERR_UNSUPPORTED),
    (dict(page_size=8192), _abi.ERR_UNSUPPORTED), (dict(head_dim=96), _abi.ERR_UNSUPPORTED),
    (dict(sequences=65536), _abi.ERR_UNSUPPORTED),
    (dict(table_width=1 << 25, page_size=64), _abi.ERR_UNSUPPORTED),
    (dict(k=PTR + 2), _abi.ERR_UNSUPPORTED)]


@pytest.mark.parametrize("over,status", BAD_CACHES)
def test_cache_descriptors(lib, handle, over, status):
    kv = _kv(**over)
    assert lib.aexq_attention_decode_paged(handle, kv, PTR, 512, 4, 0.1, PTR + 64, 512) == status
    assert lib.aexq_attention_prompt_paged(handle, kv, PTR, 512, PTR, 9, 4, 0.1, PTR, 512) == status
    assert lib.aexq_rope_append_paged(handle, kv, _rope(), PTR, 9, 4, PTR, 512, PTR, 256, PTR, 256,
                                      PTR, 512) == status
    assert lib.aexq_last_error()


@pytest.mark.parametrize("args,status", [
    (dict(q=None), _abi.ERR_INVALID_ARGUMENT), (dict(out=None), _abi.ERR_INVALID_ARGUMENT),
    (dict(out=PTR), _abi.ERR_INVALID_ARGUMENT), (dict(heads=3), _abi.ERR_INVALID_ARGUMENT),
    (dict(heads=0), _abi.ERR_INVALID_ARGUMENT), (dict(scale=0.0), _abi.ERR_INVALID_ARGUMENT),
    (dict(scale=-1.0), _abi.ERR_INVALID_ARGUMENT),
    (dict(scale=float("nan")), _abi.ERR_INVALID_ARGUMENT),
    (dict(scale=float("inf")), _abi.ERR_INVALID_ARGUMENT),
    (dict(q_stride=500), _abi.ERR_SHAPE), (dict(q_stride=516), _abi.ERR_UNSUPPORTED),
    (dict(q_stride=(1 << 24) + 8), _abi.ERR_UNSUPPORTED),
    (dict(out_stride=8), _abi.ERR_SHAPE), (dict(q=PTR + 8), _abi.ERR_UNSUPPORTED),
    (dict(kv=_kv(sequences=65000, table_width=1 << 14, page_size=4096, heads_kv=4)),
     _abi.ERR_UNSUPPORTED)])
def test_decode_arguments(lib, handle, args, status):
    a = dict(kv=_kv(), q=PTR, q_stride=512, heads=4, scale=0.1, out=PTR + 64, out_stride=512)
    a.update(args)
    assert lib.aexq_attention_decode_paged(handle, a["kv"], a["q"], a["q_stride"], a["heads"],
                                           a["scale"], a["out"], a["out_stride"]) == status


def test_no_context(lib):
    kv, bad = _kv(), _abi.ERR_INVALID_ARGUMENT
    assert lib.aexq_attention_decode_paged(None, kv, PTR, 512, 4, 0.1, PTR, 512) == bad
    assert lib.aexq_attention_prompt_paged(None, kv, PTR, 512, PTR, 9, 4, 0.1, PTR, 512) == bad
    assert lib.aexq_rope_append_paged(None, kv, _rope(), PTR, 9, 4, PTR, 512, PTR, 256, PTR, 256,
                                      PTR, 512) == bad
    assert lib.aexq_logprobs(None, _abi.Tensor(), PTR, PTR, PTR, 0, None, None) == bad


@pytest.mark.parametrize("args,status", [
    (dict(n=0), _abi.ERR_INVALID_ARGUMENT), (dict(tokens=0), _abi.ERR_INVALID_ARGUMENT),
    (dict(kv_tokens=0), _abi.ERR_INVALID_ARGUMENT),
    (dict(kv_tokens=8), _abi.ERR_INVALID_ARGUMENT),   # another count without offsets of its own
    (dict(off=None), _abi.ERR_INVALID_ARGUMENT), (dict(k=None), _abi.ERR_INVALID_ARGUMENT),
    (dict(v=None), _abi.ERR_INVALID_ARGUMENT), (dict(d=80), _abi.ERR_UNSUPPORTED),
    (dict(heads_kv=3), _abi.ERR_INVALID_ARGUMENT), (dict(scale=0.0), _abi.ERR_INVALID_ARGUMENT),
    (dict(ks=128), _abi.ERR_SHAPE), (dict(vs=257), _abi.ERR_UNSUPPORTED),
    (dict(n=70000), _abi.ERR_UNSUPPORTED),
    (dict(tokens=1 << 30, kv_tokens=1 << 30), _abi.ERR_UNSUPPORTED)])
def test_prompt_arguments(lib, handle, args, status):
    a = dict(q=PTR, qs=512, k=PTR, ks=256, v=PTR, vs=256, off=PTR, kvo=None, n=2, tokens=9,
             kv_tokens=9, heads=4, heads_kv=2, d=128, scale=0.1, out=PTR, os=512)
    a.update(args)
    assert lib.aexq_attention_prompt(handle, a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"],
                                     a["off"], a["kvo"], a["n"], a["tokens"], a["kv_tokens"],
                                     a["heads"], a["heads_kv"], a["d"], 1, a["scale"], a["out"],
                                     a["os"]) == status


def test_outputs_over_inputs(lib, handle):
    """Attention into its own queries, and rotation in place with other row strides."""
    kv, bad = _kv(), _abi.ERR_INVALID_ARGUMENT
    assert lib.aexq_attention_prompt_paged(handle, kv, PTR, 512, PTR, 9, 4, 0.1, PTR, 512) == bad
    assert lib.aexq_attention_prompt(handle, PTR, 512, PTR + 64, 256, PTR + 64, 256, PTR, None, 2,
                                     9, 9, 4, 2, 128, 1, 0.1, PTR, 512) == bad
    assert b"out is q" in lib.aexq_last_error()
    assert lib.aexq_rope_append_paged(handle, kv, _rope(), PTR, 9, 4, PTR, 520, PTR, 256, PTR, 256,
                                      PTR, 512) == bad
    assert b"q_out is q" in lib.aexq_last_error()


@pytest.mark.parametrize("over,status", [
    (dict(rotary_dim=24, section0=12), _abi.ERR_UNSUPPORTED),
    (dict(rotary_dim=144, section0=72), _abi.ERR_UNSUPPORTED),
    (dict(rotary_dim=0, section0=0), _abi.ERR_UNSUPPORTED),
    (dict(rows=0), _abi.ERR_INVALID_ARGUMENT), (dict(axes=0), _abi.ERR_INVALID_ARGUMENT),
    (dict(axes=5), _abi.ERR_INVALID_ARGUMENT),
    (dict(axes=3, positions=None, section0=24, section1=20, section2=20),
     _abi.ERR_INVALID_ARGUMENT),
    (dict(section0=63), _abi.ERR_INVALID_ARGUMENT),
    (dict(axes=2, section0=65, section1=-1), _abi.ERR_INVALID_ARGUMENT),
    (dict(axes=3, interleaved=1, section0=18, section1=23, section2=23), _abi.ERR_INVALID_ARGUMENT),
    (dict(cos_table=None), _abi.ERR_INVALID_ARGUMENT)])
def test_rope_arguments(lib, handle, over, status):
    assert lib.aexq_rope_append_paged(handle, _kv(), _rope(**over), PTR, 9, 4, PTR, 512, PTR, 256,
                                      PTR, 256, PTR, 512) == status


@pytest.mark.parametrize("args,status", [
    (dict(tokens=None), _abi.ERR_INVALID_ARGUMENT), (dict(top=65), _abi.ERR_INVALID_ARGUMENT),
    (dict(top=-1), _abi.ERR_INVALID_ARGUMENT), (dict(top=51), _abi.ERR_INVALID_ARGUMENT),
    (dict(lp=None, top=0), _abi.ERR_INVALID_ARGUMENT),
    (dict(lp=None, ids=None), _abi.ERR_INVALID_ARGUMENT),
    (dict(data=PTR + 2), _abi.ERR_UNSUPPORTED), (dict(dtype=3), _abi.ERR_UNSUPPORTED),
    (dict(w=0), _abi.ERR_SHAPE), (dict(h=1 << 24), _abi.ERR_UNSUPPORTED)])
def test_logprob_arguments(lib, handle, args, status):
    a = dict(tokens=PTR, lp=PTR, top=5, ids=PTR, data=PTR, dtype=_abi.DTYPE_F32, w=50, h=2)
    a.update(args)
    t = _abi.Tensor()
    t.logical = _abi.Shape(2, a["w"], a["h"], 1, 1)
    t.storage = _abi.Shape(2, a["w"], a["h"], 1, 1)
    t.layout, t.dtype, t.data, t.batch = _abi.LAYOUT_LINEAR, a["dtype"], a["data"], 1
    assert lib.aexq_logprobs(handle, t, a["tokens"], a["lp"], None, a["top"], a["ids"],
                             None) == status


def test_python_entry_points_refuse_before_the_library():
    """Tensors that are no device tensors of the right type and shape."""
    torch = pytest.importorskip("torch")
    from aiimage_amd import aexq
    f16, i32 = torch.float16, torch.int32
    pool, table = torch.zeros((2, 1, 16, 64), dtype=f16), torch.zeros((1, 2), dtype=i32)
    with pytest.raises(_abi.ArgumentError, match="on a GPU"):
        aexq.paged_kv(pool, pool, table, torch.zeros(1, dtype=i32))
    with pytest.raises(_abi.ArgumentError, match="pool"):
        aexq.paged_kv(pool[0], pool[0], table, torch.zeros(1, dtype=i32))
    with pytest.raises(_abi.ArgumentError, match="on a GPU"):
        aexq.rope(torch.zeros((4, 8)), torch.zeros((4, 8)))
    with pytest.raises(_abi.ArgumentError, match="rows"):
        aexq._head_rows(torch.zeros((3, 2, 64)), "q", (3, 2, 64), -1)
    with pytest.raises(_abi.ArgumentError, match="dense heads"):
        aexq._head_rows(torch.zeros((3, 64, 2), dtype=f16).transpose(1, 2), "q", (3, 2, 64), -1)
    assert aexq._head_rows(torch.zeros((3, 5, 64), dtype=f16)[:, 1:3], "q", (3, 2, 64), -1) == 320
    with pytest.raises(_abi.ArgumentError, match="int32"):
        aexq._device_array(torch.zeros(3, dtype=torch.int64), "offsets", i32, (3,), -1)
    with pytest.raises(_abi.ArgumentError, match="rows"):
        aexq._head_shape(torch.zeros((3, 64)), "q")


def test_structs_match_the_c_compiler_and_the_binding(tmp_path):
    """aexq_paged_kv and aexq_rope: the ctypes mirrors have the C compiler's sizes
    and offsets, the C# structs (sequential) its members in order."""
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "aexq.h"', "int main(void){"]
    structs = {"aexq_paged_kv": (_abi.PagedKv, "AexqPagedKv"), "aexq_rope": (_abi.Rope, "AexqRope")}
    for name, (cls, _) in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for field, _type in cls._fields_:
            lines.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
    lines.append("return 0;}")
    probe, exe = tmp_path / "probe.c", tmp_path / "probe"
    probe.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(probe), "-o", str(exe)],
                   check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    text = open(os.path.join(ROOT, "bindings", "csharp", "Native.cs")).read()
    for name, (cls, cs) in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for field, _type in cls._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(cls, field).offset, field
        body = re.search(r"Sequential\)\]\s*public struct " + cs + r"\s*\{(.*?)\n    \}", text,
                         re.S).group(1)
        members = []
        for kind, names in re.findall(r"public (IntPtr|int) ([\w, ]+);", body):
            members += [(kind, n.strip()) for n in names.split(",")]
        snake = lambda n: re.sub(r"(?<=[a-z])([A-Z])", r"_\1", n).lower()  # noqa: E731
        assert [(k == "IntPtr", snake(n)) for k, n in members] == [
            (t is ctypes.c_void_p, f) for f, t in cls._fields_]


def test_a_wait_state_between_m0_and_the_load_that_reads_it():
    """Loads to LDS take their LDS address from M0.  A scalar write of M0 needs one
    wait state before such a load on gfx9; the compiler adds it to its own code and
    not inside assembly."""
    import glob
    found = 0
    for path in glob.glob(os.path.join(ROOT, "aiimage_amd", "csrc", "*.h*")):
        for text in re.findall(r'asm volatile\(\s*((?:"[^"]*"\s*)+)', open(path).read()):
            lines = [l.strip() for l in re.sub(r'"\s*"', "", text).strip().strip('"')
                     .replace("\\t", " ").split("\\n")]
            for i, line in enumerate(lines):
                if re.match(r"s_mov_b32 m0\b", line):
                    found += 1
                    assert lines[i + 1].startswith("s_nop"), (os.path.basename(path), lines)
    assert found >= 2  # the two widths of dma(), which every kernel calls

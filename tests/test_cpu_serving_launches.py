"""What the host side of the operators for many sequences launches and allocates,
and that a launch that fails is reported (fake_hip.py stands for the runtime)."""
import pytest

import fake_hip

CALLS = {
    "prompt": ("lib.aexq_attention_prompt(ctx, PTR, 512, PTR, 256, PTR, 256, PTR, None, 2, 900, 900,"
               " 4, 2, 128, 1, 0.1, PTR + 64, 512)", 2),
    "prompt_paged": ("lib.aexq_attention_prompt_paged(ctx, paged(), PTR, 512, PTR, 900, 4, 0.1,"
                     " PTR + 64, 512)", 2),
    "decode": ("lib.aexq_attention_decode_paged(ctx, paged(), PTR, 512, 4, 0.1, PTR + 64, 512)", 2),
    "append": ("lib.aexq_rope_append_paged(ctx, paged(), _abi.Rope(PTR, PTR, PTR, 100, 128, 1, 0,"
               " 64), PTR, 9, 4, PTR, 512, PTR, 256, PTR, 256, PTR, 512)", 1),
    "logprobs": ("lib.aexq_logprobs(ctx, logits, PTR, PTR, None, 5, PTR, PTR)", 2),
}
LOGITS = """
logits = _abi.Tensor()
logits.logical = logits.storage = _abi.Shape(2, 150000, 2, 1, 1)
logits.layout, logits.dtype, logits.data, logits.batch = (_abi.LAYOUT_LINEAR, _abi.DTYPE_F32,
                                                          PTR, 1)
"""


@pytest.mark.parametrize("name", CALLS)
def test_a_failed_launch_is_reported(tmp_path, name):
    """Whichever of a call's launches fails, the call does, and no later one of its
    launches runs on what the failed one should have left."""
    call, launches = CALLS[name]
    fake_hip.run(tmp_path, LOGITS + f"""
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


@pytest.mark.parametrize("name", ["prompt", "prompt_paged", "decode"])
def test_scales_whose_log2_form_is_past_fp32_are_refused(tmp_path, name):
    """Scores are formed in log2 units, by scale * log2 e: past fp32's range from
    2.36e38 on, where every row would be NaN."""
    call, launches = CALLS[name]
    fake_hip.run(tmp_path, f"""
before = fake.fake_launches()
assert {call.replace("0.1,", "2.4e38,")} == _abi.ERR_INVALID_ARGUMENT, "2.4e38 taken"
assert b"scale" in lib.aexq_last_error()
assert fake.fake_launches() == before
assert {call.replace("0.1,", "2.3e38,")} == 0, lib.aexq_last_error()
assert fake.fake_launches() - before == {launches}
""")


@pytest.mark.parametrize("sequences,hq,d", [(1, 4, 128), (1024, 32, 128), (8192, 32, 128),
                                            (20000, 8, 256), (8192, 128, 64)])
def test_decode_scratch_does_not_grow_with_the_batch(tmp_path, sequences, hq, d):
    """Only a (sequence, head block) longer than a share of the work leaves partial
    rows, and those are few however many sequences there are: 2 * 768 pieces (at most)
    of 16 rows of 260 floats are 26 MB, rounded up to 32; an int a sequence."""
    fake_hip.run(tmp_path, f"""
before = fake.fake_bytes()
kv = paged(sequences={sequences}, heads_kv=8 if {hq} % 8 == 0 else 2, head_dim={d}, table_width=64)
assert lib.aexq_attention_decode_paged(ctx, kv, PTR, {hq * d}, {hq}, 0.1, PTR + 64,
                                       {hq * d}) == 0, lib.aexq_last_error()
assert fake.fake_bytes() - before <= (32 << 20) + 8 * {sequences} + 4096, fake.fake_bytes() - before
""")

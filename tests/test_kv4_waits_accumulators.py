"""The search of `test_kv4_waits.py` for results of matrix instructions that are touched too early, for those that stand in accumulation
registers (a0 .. a255), which it takes for none: they become vector registers from v512 on, a file of their own, before it looks."""
import os
import re
import subprocess

import pytest

from braidinfer_amd.csrc import build
from test_kv4_waits import registers, too_early


def as_vectors(text):
    text = re.sub(r"\ba\[(\d+):(\d+)\]", lambda m: f"v[{512 + int(m[1])}:{512 + int(m[2])}]", text)
    return re.sub(r"\ba(\d+)\b", lambda m: f"v{512 + int(m[1])}", text)


def results(text):
    """The registers that every matrix instruction writes."""
    return [registers(line.split(None, 1)[1].split(",")[0].strip()) for line in (raw.split(";")[0].strip() for raw in text.splitlines())
            if line.startswith("v_mfma")]


def test_the_search_sees_accumulation_registers():
    early = """
f:
\tv_mfma_f32_16x16x32_bf16 a[0:3], v[2:5], v[6:9], a[0:3]
\tv_accvgpr_read_b32 v1, a0
\ts_endpgm
"""
    assert results(early) == [set()] and too_early(early)[1] == []                       # as they are they are not seen
    got = as_vectors(early)
    assert results(got) == [{512, 513, 514, 515}]
    assert too_early(got)[1] == [("v_mfma_f32_16x16x32_bf16 v[512:515], v[2:5], v[6:9], v[512:515]", "v_accvgpr_read_b32 v1, v512")]
    assert too_early(got.replace("\tv_accvgpr_read", "\ts_nop 7\n\tv_accvgpr_read")) == (1, [])
    # written again, in the next block; the vector register of the same number is another
    again = early.replace("v_accvgpr_read_b32 v1, a0", "s_branch .L\n.L:\n\tv_accvgpr_write_b32 a3, v1")
    assert len(too_early(as_vectors(again))[1]) == 1
    assert too_early(as_vectors(again.replace("a3, v1", "a4, v3"))) == (1, [])
    moved = early.replace("v_accvgpr_read_b32 v1, a0", "v_accvgpr_mov_b32 a9, a2")
    assert len(too_early(as_vectors(moved))[1]) == 1


@pytest.mark.timeout(300)
def test_no_result_in_any_register_is_touched_before_it_is_there(tmp_path):
    hipcc = build._hipcc()
    if hipcc is None:
        pytest.skip("no hipcc here")
    out = str(tmp_path / "attention_kv4.s")
    flags = [f for f in build.FLAGS if f not in ("-shared", "-fPIC")]
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", os.path.join(build.HERE, "attention_kv4.hip"), "-o", out], check=True,
                   env={**os.environ, "HOME": str(tmp_path)}, capture_output=True)
    text = as_vectors(open(out).read())
    assert all(results(text))
    products, found = too_early(text)
    assert products == len(results(text)) > 1000 and not found, found[:5]

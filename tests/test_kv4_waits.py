"""What the compiler made of the attention over 4-bit pages: no result of a matrix instruction may be read, or its register written again,
before it is there.  The compiler puts wait states between such a pair within a block, but has been seen to leave them out where the second
instruction is a copy at the head of the next block."""
import os
import re
import subprocess

import pytest

from braidinfer_amd.csrc import build


def registers(operand):
    m = re.match(r"^[-|]*v\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.match(r"^[-|]*v(\d+)\b", operand)
    return {int(m[1])} if m else set()


def too_early(text):
    """(matrix instructions, [(one of them, what touches its result too early)]): states are counted along every path, one an
    instruction and what `s_nop` says, until the result is there (8 for 16 x 16 blocks, 12 for 32 x 32)."""
    lines, labels = [], {}
    for raw in text.splitlines():
        line = raw.split(";")[0].strip()
        label = re.match(r"^([\w.$]+):$", line)
        if label:
            labels[label[1]] = len(lines)
        elif line and not line.startswith("."):
            lines.append(line)
    found = []
    for i, line in enumerate(lines):
        if not line.startswith("v_mfma"):
            continue
        need = 8 if "16x16" in line else 12
        todo, seen = [(i + 1, 0, frozenset(registers(line.split(None, 1)[1].split(",")[0].strip())))], set()
        while todo:
            j, states, live = todo.pop()
            if j >= len(lines) or states >= need or not live or (j, states, live) in seen:
                continue
            seen.add((j, states, live))
            op, _, rest = lines[j].partition(" ")
            if op == "s_endpgm":
                continue
            if op == "s_nop":
                todo.append((j + 1, states + int(rest, 0) + 1, live))
                continue
            if op == "s_branch" or op.startswith("s_cbranch"):
                if rest.strip() in labels:
                    todo.append((labels[rest.strip()], states + 1, live))
                if op == "s_branch":
                    continue
            elif not op.startswith("s_"):
                args = [registers(x.strip()) for x in re.split(r",(?![^\[]*\])", rest)]
                stores = op.startswith(("global_store", "ds_write", "buffer_store"))
                if op.startswith("v_mfma"):                      # handed on as the sum to add to, a result needs no wait
                    read, written = args[1] | args[2], set()
                    live_after = live - args[0]
                else:
                    read = set().union(*(args if stores else args[1:]))
                    written = set() if stores else args[0]
                    live_after = live - written
                if (read | written) & live:
                    found.append((line, lines[j]))
                live = frozenset(live_after)
            todo.append((j + 1, states + 1, live))
    return sum(x.startswith("v_mfma") for x in lines), found


def test_the_search_sees_what_it_is_for():
    early = """
f:
\tv_mfma_f32_16x16x32_bf16 v[50:53], v[2:5], v[6:9], v[50:53]
\ts_and_b64 vcc, exec, vcc
\ts_cbranch_vccnz .LBB0_2
\ts_nop 7
\ts_endpgm
.LBB0_2:
\tv_mov_b64_e32 v[14:15], v[50:51]
\ts_endpgm
"""
    assert too_early(early)[1] == [("v_mfma_f32_16x16x32_bf16 v[50:53], v[2:5], v[6:9], v[50:53]", "v_mov_b64_e32 v[14:15], v[50:51]")]
    assert too_early(early.replace(".LBB0_2:", ".LBB0_2:\n\ts_nop 6")) == (1, [])
    chain = """
f:
\tv_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], v[24:27], 0
\tv_mfma_f32_32x32x16_bf16 v[0:15], v[28:31], v[32:35], v[0:15]
\tds_write_b128 v40, v[12:15]
\ts_endpgm
"""
    assert [b for _, b in too_early(chain)[1]] == ["ds_write_b128 v40, v[12:15]"]


@pytest.mark.timeout(300)
def test_no_result_is_touched_before_it_is_there(tmp_path):
    hipcc = build._hipcc()
    if hipcc is None:
        pytest.skip("no hipcc here")
    out = str(tmp_path / "attention_kv4.s")
    flags = [f for f in build.FLAGS if f not in ("-shared", "-fPIC")]
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", os.path.join(build.HERE, "attention_kv4.hip"), "-o", out], check=True,
                   env={**os.environ, "HOME": str(tmp_path)}, capture_output=True)
    products, found = too_early(open(out).read())
    assert products > 1000 and not found, found[:5]

"""Vector instructions and the matrix instructions that read what they wrote, in
the built gfx950 code: there is no forwarding between them, two wait states have
to pass (an instruction each, s_nop n more). The compiler sees to that for its
own instructions, and cannot for those in inline asm. Read from the disassembly:
too early a read need not show in a run. Needs no GPU."""
import os
import re

import pytest

from test_lds_waits import OBJDUMP, code  # noqa: F401  (code: fixture)

pytestmark = pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")

WAIT = 2


def registers(text):
    """Vector registers that an operand list names."""
    out = set()
    for kind, one, lo, hi in re.findall(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])", text):
        out.update((kind, i) for i in (range(int(lo), int(hi) + 1) if lo else [int(one)]))
    return out


def written(t):
    """Vector registers that a vector instruction writes."""
    if not t.startswith("v_") or t.startswith(("v_mfma", "v_smfmac", "v_cmp", "v_readlane", "v_readfirstlane", "v_nop")):
        return set()
    ops = t.split(None, 1)[1].split(",") if " " in t else []
    both = "swap" in t
    return registers(",".join(ops[:2] if both else ops[:1]))


def early_reads(ins):
    """(writer, reader, wait states between) of every read that comes too early,
    along every way the code can go."""
    text = [t for _, t in ins]
    at = {a: i for i, (a, _) in enumerate(ins)}
    before = [[] for _ in ins]
    for i, (a, t) in enumerate(ins):
        m = re.match(r"s_c?branch\S* (\d+)", t)
        to = at.get(a + 4 + 4 * ((int(m.group(1)) ^ 0x8000) - 0x8000)) if m else None
        if to is not None:
            before[to].append(i)
        if i + 1 < len(ins) and not t.startswith(("s_branch", "s_endpgm", "s_setpc")):
            before[i + 1].append(i)
    found = []
    for i, t in enumerate(text):
        if not t.startswith(("v_mfma", "v_smfmac")):
            continue
        reads = registers(t.split(None, 1)[1].split(",", 1)[1])
        todo = [(j, 0, reads) for j in before[i]]
        while todo:
            j, states, regs = todo.pop()
            hit = written(text[j]) & regs
            if hit:
                found.append((text[j], t, states))
            m = re.match(r"s_nop (\d+)", text[j])
            states += int(m.group(1)) + 1 if m else 1
            if states < WAIT:
                todo += [(k, states, regs - hit) for k in before[j]]
    return found


def test_parsing():
    """What the check itself can tell, on a few lines."""
    ins = ["v_perm_b32 v4, v1, v2, v3", "s_nop 0", "v_mfma_f32_16x16x32_f16 v[8:11], v[4:7], v[12:15], v[8:11]", "s_endpgm"]
    asm = [(4 * i, t) for i, t in enumerate(ins)]
    assert len(early_reads(asm)) == 1 and early_reads(asm)[0][2] == 1
    ins[1] = "s_nop 1"
    assert not early_reads([(4 * i, t) for i, t in enumerate(ins)])
    loop = ["s_nop 7", "v_mfma_f32_16x16x32_f16 v[8:11], v[4:7], v[12:15], v[8:11]", "s_nop 7", "v_mov_b32_e32 v15, 0", "s_cbranch_scc1 65532"]
    assert len(early_reads([(4 * i, t) for i, t in enumerate(loop)])) == 1
    assert written("v_permlane16_swap_b32_e32 v1, v2") == {("v", 1), ("v", 2)}


def test_no_matrix_instruction_reads_too_early(code):  # noqa: F811
    seen = 0
    for name, ins in code.items():
        if not any(t.startswith("v_mfma") for _, t in ins):
            continue
        early = early_reads(ins)
        assert not early, f"{name}: {len(early)} reads too early, as {early[0]}"
        seen += 1
    assert seen >= 100

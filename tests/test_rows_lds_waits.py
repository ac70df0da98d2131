"""The attention's loads with an LDS destination, in the built gfx950 code (as
test_lds_waits.py does for the matrix products): before such a load goes out,
the wave's reads of the slot it fills have returned. Needs no GPU."""
import os
import re

import pytest

from test_lds_waits import OBJDUMP, code, outstanding  # noqa: F401  (code: fixture)

pytestmark = pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")


def is_load(t):
    return re.match(r"buffer_load_dwordx4\b.* lds", t)


def main_loop(ins):
    """The shortest backward branch's body that both loads and multiplies (the
    masked steps' code jumps back and forth inside it)."""
    at = {a: i for i, (a, _) in enumerate(ins)}
    found = []
    for i, (a, t) in enumerate(ins):
        m = re.match(r"s_c?branch\S* (\d+)", t)
        to = at.get(a + 4 + 4 * ((int(m.group(1)) ^ 0x8000) - 0x8000)) if m else None
        if to is not None and to <= i:
            body = [x for _, x in ins[to:i + 1]]
            if any("v_mfma" in x for x in body) and any(is_load(x) for x in body):
                found.append(body)
    return min(found, key=len)


def test_attention_reloads_read_slots_only(code):  # noqa: F811
    """tree_attention_kernel: a turn's loads wait for the turn before's reads
    (few rows: of the slot itself; shared tiles: ahead of the barrier)."""
    seen = 0
    for name, ins in code.items():
        if "tree_attention_kernel" not in name:
            continue
        worst = outstanding(main_loop(ins), is_load)
        assert worst and max(worst) == 0, f"{name}: {worst} reads not waited for"
        seen += 1
    assert seen == 24  # head sizes, types, four tiles, the shared ones through and past the caches

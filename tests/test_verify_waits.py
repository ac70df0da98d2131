"""The judging of drafts, in the built gfx950 code: a row that waits for another
round overwrites what the round before left for it, which every wave of the
workgroup reads. Between those reads and that store stands a barrier, right in
front of the store's own condition. Read from the disassembly, as no run can show
a barrier that is missing but seldom needed. Needs no GPU."""
import os

import pytest

from test_lds_waits import OBJDUMP, code  # noqa: F401  (code: fixture)

pytestmark = pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")


def test_a_waiting_rows_state_is_stored_behind_a_barrier(code):  # noqa: F811
    seen = 0
    for name, ins in code.items():
        if "verify_step_kernel" not in name:
            continue
        text = [t for _, t in ins]
        stores = [i for i, t in enumerate(text) if t.startswith("global_store_dwordx4")]  # (the only 16 bytes it stores)
        assert len(stores) == 1, name
        before = text[max(0, stores[0] - 10):stores[0]]
        assert "s_barrier" in before, f"{name}: no barrier right before the state's store"
        behind = before[len(before) - before[::-1].index("s_barrier"):]
        assert not any("load" in t for t in behind), f"{name}: {behind}"
        seen += 1
    assert seen == 4  # types, small and large chunks

"""long_attention's loads with an LDS destination, in the built gfx950 code (as
test_rows_lds_waits.py does for tree_attention's): before such a load goes out,
the wave's reads of the slot it fills have returned. Needs no GPU."""
import os

import pytest

from test_lds_waits import OBJDUMP, code, outstanding  # noqa: F401  (code: fixture)
from test_rows_lds_waits import is_load, main_loop

pytestmark = pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")


def test_long_attention_reloads_read_slots_only(code):  # noqa: F811
    """The turns of fp16 rows: a turn's loads wait for the turn before's reads
    (few rows: of the slot itself; shared tiles: ahead of the barrier)."""
    seen = 0
    for name, ins in code.items():
        if "long_attention_kernel" not in name:
            continue
        worst = outstanding(main_loop(ins), is_load)
        assert worst and max(worst) == 0, f"{name}: {worst} reads not waited for"
        seen += 1
    # head sizes and types; few rows: 16 and 32 rows over fp16 rows, one tile of 16 and more
    # over blocks; shared: 64 and 128 rows, with blocks and without, through and past the caches
    assert seen == 4 * (2 + 2 + 8)

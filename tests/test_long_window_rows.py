"""A window over masks is refused where it is shorter than a sequence's rows can
be: than max_rows, or than all rows of the call where they are fewer. Needs no
GPU: the calls that pass it are turned away by a later argument."""
import math

import pytest

import q3vl_int8 as q
from test_long_capi import attn
from test_rows_capi import refused


@pytest.mark.parametrize("window,rows,max_rows", [(50, 10, 100), (10, 10, 100), (3, 3, 3), (3, 3, 1 << 30), (1, 1, 8), (8, 20, 8)])
def test_windows_of_all_rows_there_are(window, rows, max_rows):
    refused(attn(window=window, rows=rows, max_rows=max_rows, scale=math.nan), q.ERR_INVALID_ARGUMENT, "scale")


@pytest.mark.parametrize("window,rows,max_rows", [(9, 10, 100), (2, 3, 3), (7, 20, 8), (19, 20, 1 << 30)])
def test_shorter_windows_are_refused(window, rows, max_rows):
    refused(attn(window=window, rows=rows, max_rows=max_rows, scale=math.nan), q.ERR_UNSUPPORTED, f"masks of up to {min(rows, max_rows)} rows")


def test_without_a_mask_any_window():
    refused(attn(window=1, rows=10, max_rows=10, mask=None, words=0, scale=math.nan), q.ERR_INVALID_ARGUMENT, "scale")

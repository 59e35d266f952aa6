"""riallm_paged_row with a page size that no cache has: no row, at once."""
import ctypes
import subprocess
import sys

import pytest

from conftest import ROOT


def test_page_sizes(rb):
    L = rb.lib()
    table = (ctypes.c_int32 * 2)(1, 0)
    for ps, want in ((16, 1 * 16 + 5), (32, 1 * 32 + 5), (64, 1 * 64 + 5), (128, 1 * 128 + 5), (0, -1), (-16, -1), (8, -1),
                     (17, -1), (48, -1), (256, -1)):
        assert L.riallm_paged_row(table, 2, 2, 4, 1, ps, 0, 0, 5) == want, ps


@pytest.mark.parametrize("ps", [2**30 + 1, 2**31 - 1])
def test_a_page_size_past_every_power_ends(ps):
    code = ("import ctypes, riallm_b200 as r; t = (ctypes.c_int32 * 2)(1, 0); "
            f"print(r.lib().riallm_paged_row(t, 2, 2, 4, 1, {ps}, 0, 0, 5))")
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=60)
    assert out.stdout.strip() == "-1", out.stderr

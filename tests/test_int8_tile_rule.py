"""The int8 GEMM's token tile: the library's rule, and the expert layer's
restatement of it for the global expert count."""

from __future__ import annotations

import pytest

from moe_serving_profile_b200 import _lib, experts


@pytest.mark.parametrize("rows,n,tile", [(0, 128, 16), (8, 128, 16), (682, 128, 16), (683, 128, 32), (1365, 128, 32),
                                         (1366, 128, 64), (2731, 128, 128), (14335, 128, 128), (14336, 128, 256),
                                         (1, 1, 16), (5, 1, 16), (6, 1, 32), (111, 1, 128), (112, 1, 256),
                                         (2 ** 31 - 1, 1024, 256), (2 ** 31 - 1, 1, 256)])
def test_rule(rows, n, tile):
    """Three times the mean rows per expert, rounded up to a tile of 16 to 128;
    256 from a mean of 112 (restated)."""
    assert _lib.lib.b200moe_int8_token_tile(rows, n) == tile
    want = 256 if rows >= 112 * n else next((t for t in (16, 32, 64, 128) if t * n >= 3 * rows), 128)
    assert experts._int8_tile(rows, n) == want == tile


def test_both_rules_agree():
    for n in (1, 3, 8, 128, 384, 1024):
        for mean in (0.01, 0.3, 1, 5, 5.4, 10, 10.7, 21, 21.4, 42, 42.7, 100, 111.9, 112, 113, 5000):
            for rows in {int(mean * n), int(mean * n) + 1, max(0, int(mean * n) - 1)}:
                assert experts._int8_tile(rows, n) == _lib.lib.b200moe_int8_token_tile(rows, n), (rows, n)

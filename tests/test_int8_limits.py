"""The int8 GEMM's 32-bit counts: launches whose row chunks could pass them."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moe_serving_profile_b200 import _lib, layout, ops
from tests.test_int8 import _args

FAKE = 0x10000


@pytest.mark.parametrize("rows,experts,tile,unit", [
    (2 ** 30, 1024, 16, 128), (2 ** 31 - 1, 1024, 128, 128), (2 ** 31 - 1, 1024, 0, 128),
    (2 ** 29, 2, 16, 128 * 64)])           # the last: too many tiles of ascending offsets
def test_too_many_chunks_or_tiles(rows, experts, tile, unit):
    a = _args(max_rows=rows, b_rows=rows, n_experts=experts, token_tile=tile, feat_pad=unit, n_feat=unit, ldo=unit)
    chunks = experts * -(-rows // (tile or 256))
    assert chunks > 2 ** 31 - 1 or (min(experts, rows) + rows // tile) * (unit // 128) > 0x7fff0000
    assert _lib.lib.b200moe_int8_gemm(0, None, ctypes.byref(a), FAKE, FAKE, FAKE, None) == _lib.ERR_UNSUPPORTED
    assert b"too many" in _lib.lib.b200moe_last_error()


@pytest.mark.gpu
def test_offsets_that_go_up_and_down(cuda):
    """Every second expert has all rows: each is computed, the last one's result
    stays or an earlier one's (both have the same weights here)."""
    g = torch.Generator().manual_seed(1)
    E, rows, N, K = 512, 300, 136, 128
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    lin = layout.int8_linear(w.to(cuda), torch.ones(N, device=cuda))
    m = ops.Int8Matrix(E, 1, N, K, 256, K, lin.weight.repeat(E, 1, 1, 1, 1), lin.scale.repeat(E, 1, 1), None,
                       _lib.EPI_DOWN_ONCE)
    q = torch.randint(-127, 128, (rows, K), generator=g, dtype=torch.int8)
    off = torch.tensor([0, rows] * (E // 2) + [0], dtype=torch.int32, device=cuda)
    want = (q.double() @ w.double().t()).to(torch.float32).to(torch.bfloat16)
    for tile in (16, 128, 256):
        y = ops.int8_gemm(m, ops.QuantRows(q.to(cuda), torch.ones(rows, device=cuda)), offsets=off, token_tile=tile)
        assert torch.equal(y.cpu(), want) and _lib.device_status(0) == 0

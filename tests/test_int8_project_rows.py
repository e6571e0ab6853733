"""b200moe_int8_project multiplies only rows that its x gives: through the C
interface, where the rows of x and of the launch are separate arguments."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moe_serving_profile_b200 import _lib, layout, ops

FAKE = 0x10000
L = _lib.lib


def args(**over):
    a = _lib.GemmArgs(n_experts=1, max_rows=64, wfmt=_lib.W_INT8, planes=1, feat_pad=256, n_feat=256, k_pad=128,
                      weight=FAKE, b_rows=64, b_div=1, epilogue=_lib.EPI_DOWN_ONCE, out=FAKE, ldo=256)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def project(a, rows, inverse=None, copies=1, x=FAKE, scale=FAKE, ws=FAKE, kv=128, stream=None):
    return L.b200moe_int8_project(0, stream, ctypes.byref(a), x, kv, rows, kv, inverse, copies, scale, None, ws,
                                  L.b200moe_int8_project_workspace(a.b_rows, a.k_pad))


@pytest.mark.parametrize("rows,inverse,copies", [(63, None, 1), (0, None, 1), (15, FAKE, 4), (0, FAKE, 8)])
def test_dense_rows_that_x_does_not_give(rows, inverse, copies):
    assert project(args(), rows, inverse, copies) == _lib.ERR_INVALID
    assert b"dense rows" in L.b200moe_last_error()


def test_no_rows_of_segments():
    """Segments over no rows at all: nothing to do (and no device needed)."""
    assert project(args(offsets=FAKE), 0) == _lib.OK


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [16, 256])
def test_segments_past_the_rows(cuda, tile):
    """Segments that end behind x's rows: the rows behind them stay as they were."""
    g = torch.Generator().manual_seed(tile)
    E, rows, most, K, N = 3, 40, 64, 128, 136
    w = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8)
    lin = [layout.int8_linear(w[e].to(cuda), torch.ones(N, device=cuda)) for e in range(E)]
    weight, scale = torch.cat([m.weight for m in lin]), torch.cat([m.scale for m in lin])
    x = torch.randint(-127, 128, (rows, K), generator=g).to(torch.bfloat16)
    x[:, 0] = 127                                      # a scale of one
    xd = x.to(cuda)
    off = torch.tensor([0, 10, 30, most], dtype=torch.int32, device=cuda)
    out = torch.full((most, N), 7.0, dtype=torch.bfloat16, device=cuda)
    size = L.b200moe_int8_project_workspace(most, K)
    ws = torch.zeros(size, dtype=torch.uint8, device=cuda)
    a = args(offsets=off.data_ptr(), n_experts=E, max_rows=most, b_rows=most, token_tile=tile, feat_pad=256, n_feat=N,
             weight=weight.data_ptr(), out=out.data_ptr(), ldo=N)
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(project(a, rows, x=xd.data_ptr(), scale=scale.data_ptr(), ws=ws.data_ptr(), kv=K, stream=st), "project")
    want = torch.full((most, N), 7.0, dtype=torch.float64)
    for e, (lo, hi) in enumerate(((0, 10), (10, 30), (30, rows))):
        want[lo:hi] = x[lo:hi].double() @ w[e].double().t()
    # sums below 2^24 are exact in fp32; one rounding to bf16
    assert torch.equal(out.cpu(), want.to(torch.float32).to(torch.bfloat16))
    assert _lib.device_status(0) == 0


@pytest.mark.gpu
def test_dense_rows_and_copies(cuda):
    """As many rows as the launch has, by themselves or as copies."""
    g = torch.Generator().manual_seed(2)
    lin = layout.int8_linear(*layout.quantize_int8(torch.randn(136, 256, generator=g).to(cuda)))
    x = torch.randn(16, 256, generator=g).to(torch.bfloat16).to(cuda)
    y = ops.int8_project(lin, x)
    inv = torch.randperm(48, generator=g).to(torch.int32).to(cuda)
    z = ops.int8_project(lin, x, inverse=inv, copies=3)
    assert torch.equal(z[inv.long()].view(16, 3, 136), y[:, None].expand(16, 3, 136))

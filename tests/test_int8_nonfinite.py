"""Rows with infinities and NaN through the 8-bit quantisers and products:
no finite number comes out of them, and their neighbours are untouched."""

from __future__ import annotations

import pytest
import torch

from moe_serving_profile_b200 import _lib, experts, layout, norm, ops
from tests.test_int8 import on, packed

BAD = {2: float("inf"), 5: float("-inf"), 7: float("nan"), 19: float("inf")}


def rows_with(g, T, H, dev):
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    clean = x.clone()
    for r, v in BAD.items():
        x[r, (37 * r) % H] = v
    x[19, 3] = float("-inf")
    return x.to(dev), clean.to(dev), torch.tensor([r in BAD for r in range(T)], device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("clamp", [False, True])
@pytest.mark.parametrize("tile", [16, 256])
def test_products(cuda, clamp, tile):
    """bf16 rows through every epilogue: NaN in all features of a bad row."""
    g = torch.Generator().manual_seed(tile + clamp)
    H, I, T = 256, 136, 40
    _, parts, more = packed(g, 1, H, I, clamp, bias=True)
    parts, more = on(cuda, *parts, **more)
    w = layout.int8_experts(*parts, **more)
    x, clean, bad = rows_with(g, T, H, cuda)
    act = ops.int8_project(w.m1, x, token_tile=tile)[:, :I]
    want = ops.int8_project(w.m1, clean, token_tile=tile)[:, :I]
    assert act[bad].isnan().all() and torch.equal(act[~bad], want[~bad])
    y, y0 = ops.int8_project(w.m2, act.contiguous(), token_tile=tile), ops.int8_project(w.m2, want.contiguous(), token_tile=tile)
    assert y[bad].isnan().all() and torch.equal(y[~bad], y0[~bad])
    q = ops.act_quant_int8(x)
    assert q.scale[bad].isnan().all() and q.scale[~bad].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("quant", ["int8", "fp8"])
def test_layer_from_a_norm(cuda, quant):
    """A norm's 8-bit rows into the experts: an infinite weight makes a value of
    every row infinite or NaN, an infinite input a row of NaN."""
    g = torch.Generator().manual_seed(3)
    E, K, H, I, T = 4, 2, 256, 128, 24
    if quant == "int8":
        w = layout.int8_experts(*on(cuda, *packed(g, E, H, I)[1])[0])
    else:
        def block(*s):
            return (torch.randn(*s, generator=g).to(torch.float8_e4m3fn).to(cuda),
                    (torch.rand(E, s[1] // 128, s[2] // 128, generator=g) * 0.1).to(cuda))
        w = layout.fp8_experts(*block(E, I, H), *block(E, I, H), *block(E, H, I), (128, 128))
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(cuda)
    wt = torch.rand(T, K, generator=g).to(cuda)
    m = norm.AddRMSNorm(H, 1e-6, quant=quant).to(cuda)

    def layer(x):
        n = m(x)
        return n, experts.layer_forward(w, n.out, idx, wt, num_experts=E, expert_begin=0, numerics="efficient",
                                        rows=n.rows)

    x, clean, bad = rows_with(g, T, H, cuda)
    (n, y), (n0, y0) = layer(x), layer(clean)
    assert n.rows.scale.view(T, -1)[bad].isnan().any(1).all()
    assert y[bad].isnan().all() and torch.equal(y[~bad], y0[~bad]) and y0.isfinite().all()
    m.weight.data[200] = float("inf")
    n, y = layer(clean)
    s = n.rows.scale.view(T, -1)
    assert s[:, -1].isnan().all() and y.isnan().all()
    if quant == "fp8":                       # the other group of 128 columns is what it was
        assert torch.equal(s[:, 0], n0.rows.scale[:, 0])
        assert torch.equal(n.rows.q.view(torch.uint8)[:, :128], n0.rows.q.view(torch.uint8)[:, :128])
    assert _lib.device_status(0) == 0


def test_weights_that_are_not_finite():
    """A channel with NaN or an infinity has the scale NaN: its products are NaN,
    where a scale of 1 made them zero."""
    w = torch.randn(6, 64, generator=torch.Generator().manual_seed(0)) * 0.02
    w[1, 3], w[2, 5], w[3, 7], w[4] = float("nan"), float("inf"), float("-inf"), 0.0
    q, s = layout.quantize_int8(w)
    bad = torch.tensor([False, True, True, True, False, False])
    assert s[bad].isnan().all() and s[~bad].isfinite().all() and s[4] == 1
    assert (q[bad] == 0).all() and (q[4] == 0).all()
    good = layout.quantize_int8(w[~bad])
    assert torch.equal(q[~bad], good[0]) and torch.equal(s[~bad], good[1])
    # in a layer the channel of either gate plane stays NaN
    lin = layout.int8_linear(*layout.quantize_int8(w.repeat(4, 1)))
    assert int(lin.scale.isnan().sum()) == 12


@pytest.mark.gpu
def test_products_of_weights_that_are_not_finite(cuda):
    g = torch.Generator().manual_seed(6)
    E, H, I, T = 2, 128, 64, 9
    gate, up, down = ((torch.randn(E, *s, generator=g) * 0.1).to(cuda) for s in ((I, H), (I, H), (H, I)))
    gate[0, 5, 3], up[0, 9, 1] = float("nan"), float("inf")
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
    off = torch.tensor([0, T, T], dtype=torch.int32, device=cuda)
    for epi in (_lib.EPI_SWIGLU_F32, _lib.EPI_CLAMP_SWIGLU_F32):
        w = layout.int8_experts_from(gate, up, down, gated_epilogue=epi)
        act = ops.int8_project(w.m1, x, offsets=off)[:, :I]
        bad = torch.zeros(I, dtype=torch.bool, device=cuda)
        bad[5] = bad[9] = True
        assert act[:, bad].isnan().all() and act[:, ~bad].isfinite().all()

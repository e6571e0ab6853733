"""A NaN in a token's hidden row comes out of the expert layer as NaN, in every
weight format and numerics, and touches no other token."""

from __future__ import annotations

import pytest
import torch

from moe_serving_profile_b200 import _lib, experts, layout

E, K, H, I = 8, 2, 256, 128


def weights(fmt, g, dev):
    if fmt == "bf16":
        return layout.bf16_experts(*((torch.randn(E, *s, generator=g) * 0.05).to(torch.bfloat16).to(dev)
                                     for s in ((I, H), (I, H), (H, I))))
    if fmt == "fp8":
        def block(*s):
            return (torch.randn(E, *s, generator=g).to(torch.float8_e4m3fn).to(dev),
                    (torch.rand(E, s[0] // 128, s[1] // 128, generator=g) * 0.1).to(dev))
        return layout.fp8_experts(*block(I, H), *block(I, H), *block(H, I), (128, 128))
    if fmt == "int8":
        return layout.int8_experts_from(*((torch.randn(E, *s, generator=g) * 0.05).to(dev)
                                          for s in ((I, H), (I, H), (H, I))))
    blocks = lambda f, k: torch.randint(0, 256, (E, f, k // 32, 16), generator=g, dtype=torch.uint8).to(dev)  # noqa: E731
    scales = lambda f, k: torch.randint(118, 124, (E, f, k // 32), generator=g, dtype=torch.uint8).to(dev)   # noqa: E731
    bias = lambda f: (torch.randn(E, f, generator=g) * 0.1).to(torch.bfloat16).to(dev)                       # noqa: E731
    return layout.gpt_oss_mxfp4_experts(blocks(2 * I, H), scales(2 * I, H), bias(2 * I), blocks(H, I), scales(H, I),
                                        bias(H), 1.702, 7.0)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 40, 600])
@pytest.mark.parametrize("fmt,numerics", [("bf16", "reference"), ("bf16", "fast"), ("fp8", "reference"),
                                          ("fp8", "fast"), ("fp8", "efficient"), ("mxfp4", "reference"),
                                          ("mxfp4", "fast"), ("mxfp4", "efficient"), ("int8", "efficient")])
def test_nan_rows(cuda, fmt, numerics, T):
    g = torch.Generator().manual_seed(T)
    w = weights(fmt, g, cuda)
    clean = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(cuda)
    wt = torch.rand(T, K, generator=g).to(cuda)
    x = clean.clone()
    bad = torch.zeros(T, dtype=torch.bool, device=cuda)
    bad[::3] = True
    x[::3, 77] = float("nan")

    def layer(h):
        return experts.layer_forward(w, h, idx, wt, num_experts=E, expert_begin=0, numerics=numerics)

    y, y0 = layer(x), layer(clean)
    assert y0.isfinite().all() and torch.equal(y[~bad], y0[~bad])
    assert y[bad].isnan().all()
    assert _lib.device_status(0) == 0

"""Grouped routing where 64-bit scores meet: logits whose scores are one number
in 64 bits go by id, others by score, whatever the logits' type."""

from __future__ import annotations

import pytest
import torch

from tests.test_route_grouped import check


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_tiny_logits(cuda, scoring):
    """Around zero: 1e-20 and 0 have one score (0.5, or that of the row's
    largest), 2^-29 and the numbers beside it have their own."""
    step = 2.0 ** -29 * (1 + 2.0 ** -7)
    rows = [
        [0.0, 1e-20, -1.0, 2e-20, -1e-30, -2.0, 1e-38, -0.0],
        [1e-20, 2e-20, 1.0, -1e-20, 0.0, -1.0, 0.5, 3e-20],
        [-1e-20, 0.0, 300.0, 2e-20, 1e-25, -1.0, 5.0, 0.0],
        [2.0 ** -29, step, -step, 0.0, -2.0 ** -29, 2.0 ** -28, -0.0, -2.0 ** -28],
        [-3.0, -2.0, -1.0, 2e-20, 1e-20, 0.0, -1e-20, -4.0],
        [0.0] * 8,
        [1e-39, 9e-41, 0.0, -9e-41, -1e-39, 2e-39, 1e-45, -2e-39],
    ]
    x = torch.tensor(rows)
    x = torch.cat([x, x.roll(3, 1), x.flip(1)]).to(cuda)
    for dtype in (torch.bfloat16, torch.float32):
        for kw in (dict(), dict(n_group=4, topk_group=2, group_top=1), dict(n_group=8, topk_group=5, group_top=2)):
            for K in (1, 3, 4):
                check(x.to(dtype), None, K, scoring=scoring, **kw)
                check(x.to(dtype), torch.zeros(8, device=cuda), K, scoring=scoring, **kw)
    # among many experts: the tiny one is in no lane's or group's best place
    g = torch.Generator().manual_seed(4)
    wide = -torch.rand(40, 160, generator=g) - 0.5
    wide[:, 7::20], wide[:, 11::20] = 1e-20, 0.0
    wide[::2, 31] = 3e-20
    for kw in (dict(), dict(n_group=8, topk_group=3, group_top=1)):
        check(wide.to(torch.bfloat16).to(cuda), None, 6, scoring=scoring, **kw)


@pytest.mark.gpu
def test_subnormal_scores(cuda):
    """Sigmoids between the smallest subnormal and the smallest normal 64-bit
    number (logits of -708.4 to -709.7) still order their experts; below them
    the formula's exp overflows and the scores are zero."""
    x = torch.tensor([[-709.5, -709.0, -708.75, -709.25, -710.0, -711.0, -708.0, -707.0],
                      [-720.0, -709.75, -709.5, -708.5, -800.0, -708.5, -900.0, -709.0]]).to(cuda)
    for kw in (dict(), dict(n_group=4, topk_group=2, group_top=1), dict(n_group=4, topk_group=3, group_top=2)):
        for K in (1, 3, 4):
            check(x, None, K, **kw)
            check(x, torch.zeros(8, device=cuda), K, **kw)
    check(x, None, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("E,G", [(510, 17), (512, 1), (256, 8)])
def test_softmax_keys_that_nearly_tie(cuda, E, G):
    """One expert with most of the score against one whose bias brings its key
    within a few 2^-23 of it. The row's sum of many equal terms carries an
    error of its own in fp32 (up to 13 such units where a lane adds 30 of them
    one after the other), which is not the two keys' but the first one's alone."""
    unit = 2.0 ** -23
    far = torch.cat([torch.linspace(-7.95, -7.88, 24), torch.linspace(-6.5, -4.0, 8)]).tolist()
    for v in far:
        x = torch.full((1, E), v)
        x[0, 3] = 0.0
        s = torch.softmax(x.double(), 1)[0]
        for gap in (-6, -3, -1.5, 1.5, 3, 6):
            bias = torch.full((E,), -10.0)
            bias[3] = -s[3].float()
            for other in (1, E - 2):           # in the same group and in another
                b = bias.clone()
                b[other] = (s[3] + bias[3].double() - s[other] + gap * unit).float()
                key = s + b.double()
                assert (key[other] > key[3]) == (gap > 0)
                for K in (1, 2):
                    check(x.to(cuda), b.to(cuda), K, G, G, 1, "softmax", False)
                if G > 1:
                    check(x.to(cuda), b.to(cuda), 1, G, 1, 1, "softmax", False)


@pytest.mark.gpu
def test_sigmoids_one_step_above_a_half(cuda):
    """1 / (1 + exp(-2.4e-16)) rounds up to the number above 0.5, correctly
    rounded; an estimate that is one step short would tie it with 0.5."""
    x = torch.tensor([[0.0, 2.4e-16, -1.0, 0.0, 2.4e-16, -1e-30], [-2.0, 0.0, 0.0, 2.4e-16, 1e-20, -3.0]]).to(cuda)
    for dtype in (torch.float32, torch.bfloat16):
        for kw in (dict(), dict(n_group=3, topk_group=2, group_top=1)):
            check(x.to(dtype), None, 3, **kw)

"""Grouped expert routing (``ops.route_grouped``): scores, balance bias,
groups, top-k, renormalised weights.

The plain form below restates the formula in 64 bits. Selections have to be
equal to it; weights are fp32 results of fp32 arithmetic: exp is good to 2
units in the last place (4 half-steps of 2^-24), its argument l - max l is
rounded once (|l - max l| <= 32 in these inputs: 32 half-steps), a sum over a
row adds at most 16 + 5 roundings, a quotient and the scale one each, and the
renormalising sum carries the scores' errors once more: below 128 half-steps.
"""

from __future__ import annotations

import pytest
import torch

from moe_serving_profile_b200 import _lib, ops

TOL = 128 * 2.0 ** -24
FAKE = 0x10000


def plain(logits, bias, K, n_group, topk_group, group_top, scoring, normalize, scale):
    x = logits.double()
    T, E = x.shape
    s = 1.0 / (1.0 + torch.exp(-x)) if scoring == "sigmoid" else torch.exp(x - x.amax(1, keepdim=True))
    if scoring == "softmax":
        s = s / s.sum(1, keepdim=True)
    key = s if bias is None else s + bias.double()
    if topk_group < n_group:
        parts = key.view(T, n_group, -1)
        best = torch.topk(parts, min(group_top, parts.shape[2]), dim=2).values.sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :topk_group]
        open_ = torch.zeros(T, n_group, dtype=torch.bool).scatter_(1, kept, True)
        open_ = open_.repeat_interleave(E // n_group, 1)
    else:
        open_ = torch.ones(T, E, dtype=torch.bool)
    idx = torch.empty(T, K, dtype=torch.int64)
    for t in range(T):   # NaN first, then descending, equal keys by id; only open experts
        ids = open_[t].nonzero().flatten().tolist()
        v = key[t].tolist()
        ids.sort(key=lambda e: (0 if v[e] != v[e] else 1, -v[e] if v[e] == v[e] else 0.0, e))
        idx[t] = torch.tensor(ids[:K])
    w = s.gather(1, idx)
    if normalize:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return idx, w * scale, torch.bincount(idx.flatten(), minlength=E)


def check(logits, bias, K, n_group=1, topk_group=1, group_top=2, scoring="sigmoid", normalize=True, scale=1.0):
    want = plain(logits.cpu(), None if bias is None else bias.cpu(), K, n_group, topk_group, group_top, scoring,
                 normalize, scale)
    got = ops.route_grouped(logits, bias, K, n_group=n_group, topk_group=topk_group, group_top=group_top,
                            scoring=scoring, normalize=normalize, scale=scale)
    assert torch.equal(got.indices.cpu(), want[0])
    assert torch.equal(got.counts.cpu().long(), want[2])
    g, w = got.scores.cpu().double(), want[1]
    assert torch.equal(g.isnan(), w.isnan())
    ok = ~w.isnan()
    assert (g[ok] - w[ok]).abs().le(TOL * w[ok].abs() + 2.0 ** -126).all()
    return got


CASES = [  # T, E, K, n_group, topk_group, group_top
    (1, 1, 1, 1, 1, 2), (1, 8, 2, 1, 1, 2), (1, 256, 8, 8, 4, 2), (33, 256, 8, 8, 4, 2), (65, 128, 8, 1, 1, 2),
    (17, 160, 6, 8, 3, 1), (40, 512, 32, 1, 1, 2), (40, 512, 32, 32, 2, 2), (9, 21, 5, 3, 2, 2),
    (9, 510, 7, 17, 5, 2), (300, 32, 4, 32, 9, 1), (77, 100, 10, 5, 5, 2), (1025, 64, 6, 4, 1, 2),
    (8, 96, 16, 2, 1, 1), (5, 6, 2, 6, 2, 2), (50, 384, 8, 1, 1, 2), (31, 12, 12, 4, 4, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K,G,keep,top", CASES)
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_matches_the_formula(cuda, T, E, K, G, keep, top, scoring):
    for i, (dtype, use_bias, norm) in enumerate([(torch.float32, True, True), (torch.bfloat16, False, True),
                                                 (torch.bfloat16, True, False), (torch.float32, False, False)]):
        g = torch.Generator().manual_seed(T * 31 + E + i)
        logits = (torch.randn(T, E, generator=g) * 2).to(dtype).to(cuda)
        bias = (torch.randn(E, generator=g) * 0.1).to(cuda) if use_bias else None
        check(logits, bias, K, G, keep, top, scoring, norm, 2.5 if i else 1.0)


@pytest.mark.gpu
def test_no_tokens(cuda):
    r = ops.route_grouped(torch.empty(0, 16, device=cuda), None, 4, n_group=4, topk_group=2)
    assert r.indices.shape == (0, 4) and r.scores.shape == (0, 4) and (r.counts == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_ties_go_to_the_lower_id(cuda, scoring):
    """Few distinct logits: ties inside the selection, at its border, among
    groups, and rows of one value only."""
    g = torch.Generator().manual_seed(5)
    logits = (torch.randint(0, 4, (200, 64), generator=g).float() - 1.5)
    logits[3] = 0.25
    logits[4] = -50.0
    for bias in (None, torch.randint(0, 2, (64,), generator=g).float().to(cuda) * 0.125):
        for G, keep, top in ((1, 1, 2), (8, 3, 2), (16, 5, 1)):
            check(logits.to(cuda), bias, 8 if G < 16 else 5, G, keep, top, scoring)


@pytest.mark.gpu
@pytest.mark.parametrize("G,keep", [(1, 1), (8, 4)])
def test_keys_that_fp32_cannot_tell_apart(cuda, G, keep):
    """The bias cancels the scores to within its own rounding, so that keys
    differ by less than one fp32 step and their order is that of 64 bits."""
    g = torch.Generator().manual_seed(11)
    row = torch.randn(256, generator=g)
    bias = (1.0 - torch.sigmoid(row.double())).float()
    logits = row.repeat(50, 1)
    logits[1:] += torch.randn(49, 256, generator=g) * torch.logspace(-7, -3, 49)[:, None]
    check(logits.to(cuda), bias.to(cuda), 8, G, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_masked_experts(cuda, scoring):
    """-inf, the types' lowest values, +inf, huge and NaN logits, also in all
    of a row or of a group."""
    g = torch.Generator().manual_seed(7)
    for dtype in (torch.float32, torch.bfloat16):
        low = torch.finfo(dtype).min
        x = torch.randn(24, 64, generator=g)
        x[:, ::3] = float("-inf")
        x[1] = float("-inf")
        x[2] = low
        x[3, 5:] = low
        x[4, 8:16] = float("-inf")
        x[5, 7] = float("inf")
        x[6, 9] = float("nan")
        x[7] = float("nan")
        x[8, 3], x[8, 4] = float("nan"), float("inf")
        x[9] *= 1e4
        x[10, 10:20] = 100.0
        x[11, 2:5], x[11, 6:] = 2.0, low
        x = x.to(dtype).to(cuda)
        bias = (torch.randn(64, generator=g) * 0.1).to(cuda)
        for b in (None, bias):
            for G, keep, top in ((1, 1, 2), (8, 3, 2), (8, 2, 1)):
                check(x, b, 9, G, keep, top, scoring)
    # a bias of -inf keeps an expert out, of NaN puts it first
    bias = bias.clone()
    bias[::2] = float("-inf")
    bias[17] = float("nan")
    check(x.float(), bias, 9, 8, 3, 2, scoring)
    check(x.float(), bias, 9, 1, 1, 2, scoring)


@pytest.mark.gpu
def test_strided_and_offset_rows(cuda):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(70, 200, generator=g)
    for dtype in (torch.float32, torch.bfloat16):
        x = wide.to(dtype).to(cuda)
        for lo in (0, 1, 3, 8):
            check(x[:, lo:lo + 160], None, 6, 8, 3)
            check(x[5:6, lo:lo + 160], None, 6, 8, 3)


def test_refusals():
    L = _lib.lib

    def call(T=4, E=64, K=4, n_group=8, topk_group=4, group_top=2, scoring=0, ld=None, logits=FAKE, scores=FAKE,
             indices=FAKE, bf16=0):
        return L.b200moe_route_grouped(0, None, logits, bf16, E if ld is None else ld, None, T, E, K, n_group,
                                       topk_group, group_top, scoring, 1, 1.0, scores, indices, None)

    for bad in (dict(T=-1), dict(K=0), dict(n_group=0), dict(n_group=7), dict(topk_group=0), dict(topk_group=9),
                dict(group_top=3), dict(group_top=0), dict(scoring=2), dict(ld=63), dict(logits=None),
                dict(scores=None), dict(indices=None), dict(K=33, n_group=8, topk_group=8, E=32), dict(bf16=2),
                dict(K=9, topk_group=1), dict(E=0, n_group=1, topk_group=1)):
        code = call(**bad)
        assert code in (_lib.ERR_INVALID, _lib.ERR_UNSUPPORTED), bad
        assert _lib.lib.b200moe_last_error()
    for bad in (dict(E=1024, n_group=1, topk_group=1), dict(E=128, n_group=64, topk_group=8),
                dict(E=128, K=33, n_group=1, topk_group=1)):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad
    with pytest.raises(ValueError, match="CUDA"):
        ops.route_grouped(torch.zeros(4, 8), None, 2)
    from types import SimpleNamespace

    from moe_serving_profile_b200.router import GroupedRouter
    cfg = dict(num_experts=12, num_experts_per_tok=2, hidden_size=64)
    with pytest.raises(ValueError, match="groups"):
        GroupedRouter(SimpleNamespace(**cfg, n_group=5))
    with pytest.raises(ValueError, match="scoring"):
        GroupedRouter(SimpleNamespace(**cfg, scoring_func="tanh"))
    with pytest.raises(ValueError, match="logits"):
        GroupedRouter(SimpleNamespace(**cfg), logits="fused")


@pytest.mark.gpu
def test_wrapper_refusals(cuda):
    x = torch.zeros(4, 64, device=cuda)
    for kw in (dict(bias=torch.zeros(63, device=cuda)), dict(bias=torch.zeros(64, device=cuda, dtype=torch.bfloat16)),
               dict(bias=torch.zeros(64)), dict(top_k=0), dict(top_k=65), dict(scoring="tanh"),
               dict(n_group=7), dict(n_group=8, topk_group=1, top_k=9)):
        args = {"bias": None, "top_k": 4, **kw}
        with pytest.raises(ValueError):
            ops.route_grouped(x, args.pop("bias"), args.pop("top_k"), **args)
    for bad in (x.half(), x.t(), x[0]):
        with pytest.raises(ValueError):
            ops.route_grouped(bad, None, 4)


@pytest.mark.gpu
def test_router_module(cuda):
    from types import SimpleNamespace

    from moe_serving_profile_b200.router import GroupedRouter
    g = torch.Generator().manual_seed(1)
    cfg = SimpleNamespace(num_experts=64, num_experts_per_tok=6, hidden_size=256, n_group=8, topk_group=3,
                          routed_scaling_factor=2.5)
    for mode in ("fp32", "exact"):
        r = GroupedRouter(cfg, logits=mode).to(cuda)
        r.weight.data = (torch.randn(64, 256, generator=g) * 0.06).to(cuda)
        r.balance_bias.data = (torch.randn(64, generator=g) * 0.05).to(cuda)
        h = torch.randn(3, 20, 256, generator=g).to(torch.bfloat16).to(cuda)
        logits, scores, idx = r(h)
        assert logits.shape == (60, 64) and logits.dtype == (torch.float32 if mode == "fp32" else torch.bfloat16)
        want = plain(logits.cpu(), r.balance_bias.cpu(), 6, 8, 3, 2, "sigmoid", True, 2.5)
        assert torch.equal(idx.cpu(), want[0]) and torch.equal(r.last_counts.cpu().long(), want[2])
        assert (scores.cpu().double() - want[1]).abs().le(TOL * want[1]).all()

"""Int8 products with a scale per token and channel: the grouped and the dense
GEMM, the expert layer on them, and the modules that offer them.

The integer sums are exact, so a GEMM output is off by its fp32 epilogue (one
conversion, two products, a bias: 8 half-steps of 2^-24 of the largest term;
the gates' exp and quotient 16 more, times at most 1 + |g|) and one bf16
rounding (2^-8). Layers are compared with a float64 restatement that rounds
where the layer does (bf16 activations, their int8 codes, bf16 rows): what is
left are codes and roundings that land on the other side of a border, and the
output's own rounding.
"""

from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch

from moe_serving_profile_b200 import _lib, experts, layout, native, norm, ops, qwen3
from moe_serving_profile_b200.parallel import ParallelGroup
from moe_serving_profile_b200.router import GroupedRouter, GroupedRouting
from tests.conftest import rel_l2

FAKE = 0x10000
F32 = 24 * 2.0 ** -24


def weights(g, E, rows, K, full=False):
    if full:
        q = torch.randint(-128, 128, (E, rows, K), generator=g)
    else:
        q = (torch.randn(E, rows, K, generator=g) * 36).round().clamp(-127, 127)
    return q.to(torch.int8), (0.5 + torch.rand(E, rows, generator=g)) * 1e-3


def sums(q, s, w, ws, bounds):
    """float64 D of rows in expert segments [bounds[e], bounds[e + 1])."""
    out = torch.zeros(q.shape[0], w.shape[1], dtype=torch.float64)
    for e in range(w.shape[0]):
        a, b = bounds[e], bounds[e + 1]
        if b > a:
            out[a:b] = (q[a:b].double() @ w[e].double().t()) * ws[e].double()
    return out * s.double()[:, None]


def gate(d, bias, bounds, I, clamp):
    g, u = d[:, :I].clone(), d[:, I:].clone()
    if bias is not None:
        for e in range(bias.shape[0]):
            g[bounds[e]:bounds[e + 1]] += bias[e, 0].double()
            u[bounds[e]:bounds[e + 1]] += bias[e, 1].double()
    if clamp:
        g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        return g, g * torch.sigmoid(1.702 * g) * (u + 1)
    return g, g * torch.sigmoid(g) * u


def packed(g, E, H, I, clamp=False, bias=False, full=False):
    gw, gs = weights(g, E, I, H, full)
    uw, us = weights(g, E, I, H, full)
    dw, ds = weights(g, E, H, I, full)
    more, raw = {}, dict(w1=torch.cat([gw, uw], 1), s1=torch.cat([gs, us], 1), w2=dw, s2=ds, b1=None, b2=None)
    if bias:
        raw["b1"], raw["b2"] = torch.randn(E, 2, I, generator=g) * 0.1, torch.randn(E, H, generator=g) * 0.1
        more = dict(gate_bias=raw["b1"][:, 0], up_bias=raw["b1"][:, 1], down_bias=raw["b2"])
    if clamp:
        more["gated_epilogue"] = _lib.EPI_CLAMP_SWIGLU_F32
    return raw, (gw, gs, uw, us, dw, ds), more


def on(dev, *ts, **kw):
    return [t.to(dev) for t in ts], {k: v.to(dev) if torch.is_tensor(v) else v for k, v in kw.items()}


# --------------------------------------------------------------------------- layout (CPU)
def test_tile_layout_round_trip():
    """The images' rows and chunks, restated element by element."""
    g = torch.Generator().manual_seed(0)
    raw, parts, _ = packed(g, 2, 200, 72)
    w = layout.int8_experts(*parts)
    assert w.fmt == _lib.W_INT8 and w.h_k == 256 and w.i_pad == 128 and w.h_f == 256
    assert w.w1.shape == (2, 2, 2, 128, 128) and w.w2.shape == (2, 2, 1, 128, 128)
    assert w.s1.shape == (2, 2, 128) and w.s2.shape == (2, 2, 128)
    for e, f, k in ((0, 0, 0), (1, 71, 199), (0, 17, 130), (1, 35, 64), (0, 63, 15), (1, 64, 16)):
        for plane in (0, 1):
            r = (f % 64) // 16 * 32 + plane * 16 + f % 16
            c = (k % 128) // 16
            img = w.w1[e, f // 64, k // 128, r]
            assert img[16 * (c ^ (r & 7)) + k % 16] == raw["w1"][e, plane * 72 + f, k]
            assert w.s1[e, f // 64, r] == raw["s1"][e, plane * 72 + f]
    for e, f, k in ((0, 0, 0), (1, 199, 71), (0, 130, 33)):
        r, c = f % 128, (k % 128) // 16
        assert w.w2[e, f // 128, k // 128, r, 16 * (c ^ (r & 7)) + k % 16] == raw["w2"][e, f, k]
        assert w.s2[e, f // 128, r] == raw["s2"][e, f]
    lin = layout.int8_linear(parts[4][0], parts[5][0])
    assert torch.equal(lin.weight[0], w.w2[0]) and torch.equal(lin.scale[0], w.s2[0])
    q, s = layout.quantize_int8(torch.tensor([[0.0, 0.0], [1.0, -127.0], [2.54, 1.0]]))
    assert q.tolist() == [[0, 0], [1, -127], [127, 50]] and s[0] == 1 and s[1] == 1


# --------------------------------------------------------------------------- GEMM
def run_gemm(cuda, g, counts, planes, F, K, tile, *, clamp=False, bias=False, full=False, row_w=None, begin=0, spare=3):
    """One launch over len(counts) experts; checks every row, and that rows of
    no expert stay as they were."""
    E, R = len(counts), sum(counts)
    pre = 5 if begin else 0
    bounds = [pre]
    for c in counts:
        bounds.append(bounds[-1] + c)
    rows = bounds[-1] + spare
    kp, fp = -(-K // 128) * 128, -(-F // 128) * 128
    q = torch.zeros(rows, kp, dtype=torch.int8)
    q[:, :K] = torch.randint(-128 if full else -127, 128, (rows, K), generator=g).to(torch.int8)
    s = (0.5 + torch.rand(rows, generator=g)) * 0.02
    w, ws = weights(g, E, planes * F, K, full)
    b = torch.randn(E, planes, F, generator=g) * 0.1 if bias else None
    w4, ws3 = w.view(E, planes, F, K), ws.view(E, planes, F)
    tiles = layout._int8_tiles(w4.to(cuda), fp, kp)
    off = torch.tensor([0] * begin + bounds, dtype=torch.int32, device=cuda)
    out = torch.full((rows, F), 7.0, dtype=torch.bfloat16, device=cuda)
    epi = _lib.EPI_DOWN_ONCE if planes == 1 else (_lib.EPI_CLAMP_SWIGLU_F32 if clamp else _lib.EPI_SWIGLU_F32)
    src = torch.randperm(rows, generator=g).int()
    rw = None if row_w is None else torch.rand(rows, generator=g).to(row_w)
    m = ops.Int8Matrix(E, planes, F, K, fp, kp, tiles, layout._int8_channels(ws3, fp).to(cuda),
                       None if b is None else layout._int8_channels(b, fp).to(cuda), epi)
    ops.int8_gemm(m, ops.QuantRows(q.to(cuda), s.to(cuda)), offsets=off, expert_begin=begin,
                  row_weight=None if rw is None else rw.to(cuda), row_src=None if rw is None else src.to(cuda),
                  out=out, token_tile=tile)
    assert _lib.device_status(0) == 0
    got = out.cpu().double()
    d = sums(q[:, :K], s, w, ws, bounds)
    if planes == 2:
        gt, want = gate(d, b, bounds, F, clamp)
        slack = F32 * (1 + gt.abs()) * want.abs()
        if bias:   # the sums may cancel the bias: their errors stay, times |u| or |g|
            big = d.abs().amax() + 1
            slack = slack + F32 * big * (1 + gt.abs() + big)
    else:
        want, slack = d, F32 * d.abs()
        if b is not None:
            for e in range(E):
                want[bounds[e]:bounds[e + 1]] += b[e, 0].double()
            slack = slack + F32 * 0.5
        if rw is not None:
            want = want * rw.double()[src.long()][:, None]
    a, z = bounds[0], bounds[-1]
    assert (got[a:z] - want[a:z]).abs().le(want[a:z].abs() * 2.0 ** -8 + slack[a:z] + 1e-30).all()
    assert (got[:a] == 7).all() and (got[z:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("planes", [1, 2])
def test_gemm_ragged_experts(cuda, tile, planes):
    g = torch.Generator().manual_seed(tile + planes)
    run_gemm(cuda, g, [0, 1, 17, tile, tile + 1, 3 * tile - 5, 0, 16], planes, 136, 264, tile)
    run_gemm(cuda, g, [5, 40], planes, 8, 8, tile, begin=3)


@pytest.mark.gpu
@pytest.mark.parametrize("planes,F,K", [(1, 2048, 768), (2, 768, 2048), (1, 2880, 2880), (2, 2880, 2880), (2, 64, 128),
                                        (1, 128, 4096), (1, 1000, 1112)])
def test_gemm_sizes(cuda, planes, F, K):
    g = torch.Generator().manual_seed(F + K)
    for counts in ([1], [3, 0, 130], [300, 2]):
        run_gemm(cuda, g, counts, planes, F, K, 0, bias=True, clamp=planes == 2,
                 row_w=torch.float32 if planes == 1 else None)
    run_gemm(cuda, g, [9, 20], planes, F, K, 16, row_w=torch.bfloat16 if planes == 1 else None)


@pytest.mark.gpu
def test_gemm_full_range(cuda):
    """-128 on both sides: the largest sums, at every tile and with many rows
    beside each other in one CTA's share."""
    g = torch.Generator().manual_seed(1)
    for tile in (16, 64, 256):
        run_gemm(cuda, g, [70, 5], 1, 264, 4096, tile, full=True)
    q = torch.full((40, 16384), -128, dtype=torch.int8, device=cuda)
    lin = layout.int8_linear(torch.full((128, 16384), -128, dtype=torch.int8, device=cuda), torch.ones(128, device=cuda))
    out = experts.int8_linear(lin, ops.QuantRows(q, torch.ones(40, device=cuda)))
    assert (out.float() == float(2 ** 28)).all()          # 16384 * 2^14, exact in int32
    # many tiles per CTA: the accumulator slots and the ring wrap
    run_gemm(cuda, g, [33] * 40, 1, 1280, 256, 16)
    run_gemm(cuda, g, [290] * 12, 2, 640, 384, 256)


@pytest.mark.gpu
def test_gemm_non_finite_scales(cuda):
    """A row whose scale is NaN or infinite comes out without finite values,
    its neighbours are untouched."""
    lin = layout.int8_linear(torch.ones(128, 128, dtype=torch.int8, device=cuda), torch.ones(128, device=cuda))
    x = torch.ones(20, 128, dtype=torch.bfloat16, device=cuda)
    x[3, 5], x[7, 6] = float("nan"), float("inf")
    y = experts.int8_linear(lin, x)
    bad = torch.zeros(20, dtype=torch.bool, device=cuda)
    bad[3] = bad[7] = True
    assert not y[bad].isfinite().any() and y[~bad].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(1, 8, 8), (1, 4096, 2048), (33, 136, 2880), (257, 1000, 200), (1000, 256, 4096)])
def test_linear(cuda, T, N, K):
    g = torch.Generator().manual_seed(T + N)
    w, ws = weights(g, 1, N, K)
    bias = torch.randn(N, generator=g)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16)
    lin = layout.int8_linear(w[0].to(cuda), ws[0].to(cuda), bias.to(cuda))
    y = experts.int8_linear(lin, x.to(cuda))
    s = x.float().abs().amax(1) / 127
    q = torch.round(x.float() / s[:, None])
    want = sums(q, s, w, ws, [0, T])
    slack = F32 * (want.abs() + bias.abs())
    want = want + bias.double()
    assert (y.cpu().double() - want).abs().le(want.abs() * 2.0 ** -8 + slack).all()
    # into a caller's buffer with wider rows
    buf = torch.full((T + 2, N + 16), 3.0, dtype=torch.bfloat16, device=cuda)
    experts.int8_linear(lin, ops.act_quant_int8(x.to(cuda)), out=buf[:T, :N])
    assert torch.equal(buf[:T, :N], y) and (buf[T:] == 3).all() and (buf[:, N:] == 3).all()


# --------------------------------------------------------------------------- layer
def layer64(raw, q, s, idx, wt, E, clamp=False):
    """float64 layer from quantised token rows, rounded where the layer rounds."""
    T, K = idx.shape
    H, I = raw["w2"].shape[1:]
    src = torch.argsort(((idx * K + torch.arange(K)) * T + torch.arange(T)[:, None]).flatten())
    e_of = idx.flatten()[src]
    bounds = torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(e_of, minlength=E).cumsum(0)]).tolist()
    tok = src // K
    d = sums(q[tok], s[tok], raw["w1"], raw["s1"], bounds)
    act = gate(d, raw["b1"], bounds, I, clamp)[1].to(torch.bfloat16).float()
    s2 = act.abs().amax(1) / 127
    s2 = torch.where(s2 > 0, s2, torch.ones_like(s2))
    y = sums(torch.round(act / s2[:, None]), s2, raw["w2"], raw["s2"], bounds)
    if raw["b2"] is not None:
        for e in range(E):
            y[bounds[e]:bounds[e + 1]] += raw["b2"][e].double()
    y = (y * wt.double().flatten()[src][:, None]).to(torch.bfloat16).double()
    out = torch.zeros(T, H, dtype=torch.float64)
    return out.index_add_(0, tok, y)


def quant(x):
    s = x.float().abs().amax(1) / 127
    s = torch.where(s > 0, s, torch.ones_like(s))
    return torch.round(x.float() / s[:, None]), s


def distinct(g, T, K, E):
    return torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)])


LAYERS = [(1, 8, 2, 256, 128), (7, 16, 4, 200, 72), (64, 32, 8, 512, 256), (300, 8, 2, 128, 264), (33, 128, 8, 256, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K,H,I", LAYERS)
@pytest.mark.parametrize("clamp", [False, True])
def test_layer(cuda, T, E, K, H, I, clamp):
    g = torch.Generator().manual_seed(T + E)
    raw, parts, more = packed(g, E, H, I, clamp, bias=clamp)
    parts, more = on(cuda, *parts, **more)
    w = layout.int8_experts(*parts, **more)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    idx, wt = distinct(g, T, K, E), torch.softmax(torch.randn(T, K, generator=g), 1)
    xd, idxd, wtd = x.to(cuda), idx.to(cuda), wt.to(cuda)
    y = experts.layer_forward(w, xd, idxd, wtd, num_experts=E, expert_begin=0, numerics="efficient")
    want = layer64(raw, *quant(x), idx, wt, E, clamp)
    assert rel_l2(y, want) <= 2.0 ** -8
    # a rank's share of the experts: partial sums over the ranks add up to the whole
    part = torch.zeros(T, H, dtype=torch.float64)
    for r in range(2):
        n = E // 2
        share = layout.int8_experts(*[p[r * n:(r + 1) * n] for p in parts],
                                    **{k: v[r * n:(r + 1) * n] if torch.is_tensor(v) else v for k, v in more.items()})
        part += experts.layer_forward(share, xd, idxd, wtd, num_experts=E, expert_begin=r * n,
                                      numerics="efficient").cpu().double()
    assert rel_l2(part, want) <= 2.0 ** -8
    # rows that a norm quantised: the same codes here, so the same bits
    rows = ops.act_quant_int8(xd, k_pad=w.h_k)
    y2 = experts.layer_forward(w, xd, idxd, wtd, num_experts=E, expert_begin=0, numerics="efficient", rows=rows)
    assert torch.equal(y, y2)
    # dropped slots add nothing
    drop = idxd.clone()
    drop[0, 0] = -1
    y3 = experts.layer_forward(w, xd, drop, wtd, num_experts=E, expert_begin=0, numerics="efficient")
    assert torch.equal(y3[1:], y[1:]) and _lib.device_status(0) == _lib.STATUS_BAD_INDEX
    e = experts.layer_forward(w, xd[:0], idxd[:0], wtd[:0], num_experts=E, expert_begin=0, numerics="efficient")
    assert e.shape == (0, H)


def qwen_experts(parts, numerics="efficient"):
    gw, gs, uw, us, dw, ds = parts
    m = qwen3.ParallelExperts(SimpleNamespace(num_experts=gw.shape[0], hidden_act="silu"), ParallelGroup(1), numerics)
    for e, mods in enumerate(m.local):
        mods["gate_proj"] = qwen3.ExpertProjection(gw[e], gs[e])
        mods["up_proj"] = qwen3.ExpertProjection(uw[e], us[e])
        mods["down_proj"] = qwen3.ExpertProjection(dw[e], ds[e])
    return m


@pytest.mark.gpu
def test_norm_router_experts_together(cuda):
    """A decode block as it is used: norm with the residual, grouped router on
    its bf16 output, int8 experts on its int8 rows; then on another stream and
    in two captured graphs whose replays interleave."""
    g = torch.Generator().manual_seed(9)
    T, E, K, H, I = 24, 32, 4, 512, 128
    raw, parts, _ = packed(g, E, H, I)
    m = qwen_experts(on(cuda, *parts)[0])
    nrm = norm.AddRMSNorm(H, 1e-6, quant="int8").to(cuda)
    nrm.weight.data = (1 + 0.1 * torch.randn(H, generator=g)).to(cuda)
    router = GroupedRouter(SimpleNamespace(num_experts=E, num_experts_per_tok=K, hidden_size=H, n_group=4,
                                           topk_group=2, routed_scaling_factor=2.5)).to(cuda)
    router.weight.data = (torch.randn(E, H, generator=g) * 0.05).to(cuda)
    router.balance_bias.data = (torch.randn(E, generator=g) * 0.05).to(cuda)

    def block(x, res):
        n = nrm(x, res)
        _, wt, idx = router(n.out)
        return n, wt, idx, m(n.out, idx, wt, rows=n.rows)

    xs = [torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda) for _ in range(4)]
    rs = [(torch.randn(T, H, generator=g) * 3).to(torch.bfloat16).to(cuda) for _ in range(4)]
    outs = []
    for x, r in zip(xs, rs):
        n, wt, idx, y = block(x, r)
        want = layer64(raw, n.rows.q.cpu()[:, :H].float(), n.rows.scale.cpu(), idx.cpu(), wt.cpu(), E)
        assert rel_l2(y, want) <= 2.0 ** -8
        assert torch.equal(router.last_counts.cpu().long(), torch.bincount(idx.cpu().flatten(), minlength=E))
        outs.append(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = block(xs[0], rs[0])[3]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, outs[0])
    # two calls at once on two streams
    s2 = torch.cuda.Stream()
    s2.wait_stream(torch.cuda.current_stream())
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            a = block(xs[1], rs[1])[3]
        with torch.cuda.stream(s2):
            b = block(xs[2], rs[2])[3]
        torch.cuda.synchronize()
        assert torch.equal(a, outs[1]) and torch.equal(b, outs[2])
    graphs = []
    for i in range(2):
        gx, gr = xs[i].clone(), rs[i].clone()
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            gy = block(gx, gr)[3]
        graphs.append((cg, gx, gr, gy))
    for i, j in ((0, 1), (2, 3), (3, 0)):
        for (cg, gx, gr, gy), k in zip(graphs, (i, j)):
            gx.copy_(xs[k])
            gr.copy_(rs[k])
        for cg, *_ in graphs:
            cg.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][3], outs[i]) and torch.equal(graphs[1][3], outs[j])
    assert _lib.device_status(0) == 0


@pytest.mark.gpu
def test_fp8_experts_take_the_norms_rows(cuda):
    """W8A8 FP8 experts on rows the norm quantised: the same bits as the same
    rows through the quantising gather, when the rows are exact in bf16."""
    from moe_serving_profile_b200 import synthetic as S
    cfg = S.CONFIGS["qwen3-tiny"]
    w = S.make_qwen(cfg, seed=0)
    dev = cuda
    packed8 = layout.fp8_experts(w.gate.to(dev), w.gate_scale.to(dev), w.up.to(dev), w.up_scale.to(dev),
                                 w.down.to(dev), w.down_scale.to(dev), cfg.block)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(50, cfg.hidden, generator=g).to(torch.bfloat16).to(dev)
    q, s = ops.act_quant_fp8(x, k_pad=packed8.h_k)
    idx = distinct(g, 50, cfg.top_k, cfg.experts).to(dev)
    wt = torch.rand(50, cfg.top_k, generator=g).to(dev)
    kw = dict(num_experts=cfg.experts, expert_begin=0, numerics="efficient")
    a = experts.layer_forward(packed8, x, idx, wt, **kw)
    b = experts.layer_forward(packed8, x, idx, wt, rows=ops.QuantRows(q, s), **kw)
    assert torch.equal(a, b)
    n = ops.add_rmsnorm(x, torch.ones(cfg.hidden, device=dev), 1e-6, quant="fp8")
    c = experts.layer_forward(packed8, n.out, idx, wt, **kw)
    d = experts.layer_forward(packed8, n.out, idx, wt, rows=n.rows, **kw)
    # the codes come from the norm before or after its bf16 rounding: two
    # quantisations of values 2^-8 apart at most, e4m3 steps of 2^-4
    assert rel_l2(d, c) <= 2.0 ** -4


@pytest.mark.gpu
def test_native_layer_in_int8(cuda):
    """MoELayer with int8 experts, an int8 shared expert and grouped routing,
    against the bf16 layer of the weights that the int8 codes stand for."""
    g = torch.Generator().manual_seed(21)
    E, K, H, I, T = 16, 4, 256, 128, 40

    def deq(shape):
        q, s = layout.quantize_int8(torch.randn(shape, generator=g) * 0.05)
        return (q.float() * s[..., None])

    gu, dn = deq((E, 2 * I, H)).to(torch.bfloat16).to(cuda), deq((E, H, I)).to(torch.bfloat16).to(cuda)
    sg, su, sd = (deq(s).to(torch.bfloat16).to(cuda) for s in ((I, H), (I, H), (H, I)))
    score = (torch.randn(1, H, generator=g) * 0.05).to(torch.bfloat16).to(cuda)
    gw = (torch.randn(E, H, generator=g) * 0.1).to(torch.bfloat16).to(cuda)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
    routing = GroupedRouting(n_group=4, topk_group=2, scale=1.5, bias=(torch.randn(E, generator=g) * 0.05).to(cuda))
    outs = {}
    for storage in ("bf16", "int8"):
        layer = native.MoELayer(gw, native.LocalSwiGLUExperts(gu, dn, storage=storage), native.ExpertPlan(E, 1, 0), K,
                                shared=native.SharedSwiGLU(sg, su, sd, score, storage=storage), routing=routing)
        y, stats = layer(x)
        outs[storage] = y
        lg = torch.nn.functional.linear(x.float(), gw.float())
        assert torch.equal(stats.counts, torch.bincount(routing.select(lg, K, True).indices.cpu().flatten(),
                                                        minlength=E))
    # int8 activations: the bar that the 8-bit paths have against 16-bit ones
    assert rel_l2(outs["int8"], outs["bf16"]) < 0.08
    # every rank in one process equals one rank (exact integer sums), and so does the call per row
    ids, wts = (routing.select(torch.nn.functional.linear(x.float(), gw.float()), K, True).indices,
                torch.rand(T, K, device=cuda))
    whole = native.LocalSwiGLUExperts(gu, dn, storage="int8")
    one = native.simulate_routed([x], [ids], [wts], [whole], E)[0]
    halves = [native.LocalSwiGLUExperts(gu[r * 8:(r + 1) * 8], dn[r * 8:(r + 1) * 8], storage="int8") for r in range(2)]
    two = native.simulate_routed([x[:17], x[17:]], [ids[:17], ids[17:]], [wts[:17], wts[17:]], halves, E)
    for t, (a, b) in enumerate(zip(one, torch.cat(two))):
        assert rel_l2(a, b) <= 2.0 ** -6      # the bf16 sums run in another order
    direct = whole(x, ids[:, 0])
    perm = ops.permute(ids[:, :1].contiguous(), E)
    placed = native.run_experts_received(whole.weights, x[perm.perm_src.long()].contiguous(), perm.offsets,
                                         tile_tokens=T, K=1, num_experts=E)
    assert torch.equal(placed[perm.inverse.long()], direct)


# --------------------------------------------------------------------------- refusals
def _args(**over):
    a = _lib.GemmArgs(offsets=FAKE, expert_begin=0, n_experts=8, max_rows=64, token_tile=0, wfmt=_lib.W_INT8, planes=1,
                      feat_pad=256, n_feat=256, k_pad=128, weight=FAKE, b_rows=64, b_div=1,
                      epilogue=_lib.EPI_DOWN_ONCE, out=FAKE, ldo=256)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code", [
    ({"wfmt": _lib.W_BF16}, _lib.ERR_INVALID), ({"wfmt": _lib.W_FP8}, _lib.ERR_INVALID),
    ({"planes": 3}, _lib.ERR_INVALID), ({"planes": 2}, _lib.ERR_INVALID),
    ({"planes": 2, "epilogue": _lib.EPI_SWIGLU}, _lib.ERR_INVALID), ({"epilogue": _lib.EPI_DOWN}, _lib.ERR_INVALID),
    ({"planes": 2, "epilogue": _lib.EPI_SWIGLU_F32, "row_weight": FAKE, "row_src": FAKE}, _lib.ERR_INVALID),
    ({"feat_pad": 200}, _lib.ERR_INVALID), ({"n_feat": 300}, _lib.ERR_INVALID), ({"k_pad": 64}, _lib.ERR_INVALID),
    ({"k_pad": 192}, _lib.ERR_INVALID), ({"k_pad": 131072}, _lib.ERR_UNSUPPORTED),
    ({"n_experts": 2000}, _lib.ERR_UNSUPPORTED), ({"n_experts": 0}, _lib.ERR_INVALID),
    ({"offsets": None}, _lib.ERR_INVALID), ({"offsets": None, "n_experts": 1, "expert_begin": 2}, _lib.ERR_INVALID),
    ({"b_rows": 63}, _lib.ERR_INVALID), ({"weight": FAKE + 8}, _lib.ERR_INVALID), ({"out": FAKE + 8}, _lib.ERR_INVALID),
    ({"ldo": 248}, _lib.ERR_INVALID), ({"ldo": 260}, _lib.ERR_INVALID), ({"n_feat": 250}, _lib.ERR_INVALID),
    ({"token_tile": 160}, _lib.ERR_INVALID), ({"bias": FAKE}, _lib.ERR_INVALID), ({"b_map": FAKE}, _lib.ERR_INVALID),
    ({"row_weight": FAKE}, _lib.ERR_INVALID),
])
def test_gemm_refusals(over, code):
    a = _args(**over)
    assert _lib.lib.b200moe_int8_gemm(0, None, ctypes.byref(a), FAKE, FAKE, FAKE, None) == code
    assert _lib.lib.b200moe_last_error()


def test_other_refusals():
    L = _lib.lib
    assert L.b200moe_int8_gemm(0, None, None, FAKE, FAKE, FAKE, None) == _lib.ERR_INVALID
    for ptrs in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None), (FAKE + 4, FAKE, FAKE)):
        assert L.b200moe_int8_gemm(0, None, ctypes.byref(_args()), *ptrs, None) == _lib.ERR_INVALID
    a = _args(max_rows=0)
    assert L.b200moe_int8_gemm(0, None, ctypes.byref(a), None, None, None, None) == _lib.OK
    # the bf16 GEMM does not take int8 weights or the int8 epilogues
    b = _lib.GemmArgs(offsets=FAKE, n_experts=8, max_rows=64, wfmt=_lib.W_INT8, planes=1, feat_pad=256, n_feat=256,
                      k_pad=128, weight=FAKE, b_src=FAKE, ldb=128, b_rows=64, k_valid=128, b_div=1,
                      epilogue=_lib.EPI_DOWN, out=FAKE, ldo=256)
    assert L.b200moe_expert_gemm(0, None, ctypes.byref(b)) == _lib.ERR_INVALID
    b.wfmt, b.epilogue = _lib.W_BF16, _lib.EPI_DOWN_ONCE
    assert L.b200moe_expert_gemm(0, None, ctypes.byref(b)) == _lib.ERR_INVALID

    g = torch.Generator().manual_seed(0)
    raw, parts, _ = packed(g, 2, 64, 16)
    w = layout.int8_experts(*parts)
    x, idx, wt = torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(3, 1, dtype=torch.int64), torch.ones(3, 1)
    kw = dict(num_experts=2, expert_begin=0)
    for numerics in ("reference", "fast"):
        with pytest.raises(ValueError, match="efficient"):
            experts.layer_forward(w, x, idx, wt, numerics=numerics, **kw)
    rows = ops.QuantRows(torch.zeros(3, 128, dtype=torch.int8), torch.ones(3))
    bf = layout.bf16_experts(*(torch.zeros(2, *s, dtype=torch.bfloat16) for s in ((16, 64), (16, 64), (64, 16))))
    with pytest.raises(ValueError, match="quantised rows"):
        experts.layer_forward(bf, x, idx, wt, numerics="efficient", rows=rows, **kw)
    for bad in (ops.QuantRows(rows.q[:, :64], rows.scale), ops.QuantRows(rows.q.view(torch.float8_e4m3fn), rows.scale),
                ops.QuantRows(rows.q, rows.scale.double()), ops.QuantRows(rows.q, rows.scale[:2]),
                ops.QuantRows(rows.q[:2], rows.scale[:2])):
        with pytest.raises(ValueError):
            experts.layer_forward(w, x, idx, wt, numerics="efficient", rows=bad, **kw)
    with pytest.raises(ValueError, match="efficient"):
        qwen_experts(parts, "reference").prepare()
    with pytest.raises(ValueError, match="int8"):
        layout.int8_experts(parts[0].float(), *parts[1:])
    with pytest.raises(ValueError, match="scale"):
        layout.int8_experts(parts[0], parts[1][:, :3], *parts[2:])
    with pytest.raises(ValueError, match="gate with"):
        layout.int8_experts(*parts, gated_epilogue=_lib.EPI_SWIGLU)
    with pytest.raises(NotImplementedError):
        layout.int8_linear(torch.zeros(12, 64, dtype=torch.int8), torch.ones(12))
    with pytest.raises(ValueError, match="storage"):
        native.LocalSwiGLUExperts(torch.zeros(2, 32, 64, dtype=torch.bfloat16),
                                  torch.zeros(2, 64, 16, dtype=torch.bfloat16), storage="fp4")
    with pytest.raises(ValueError, match="logits"):
        native.MoELayer(torch.zeros(2, 64), None, native.ExpertPlan(2, 1, 0), 1, logits="fused",
                        routing=GroupedRouting())
    with pytest.raises(ValueError, match="CUDA"):
        experts.int8_linear(layout.int8_linear(parts[0][0], parts[1][0]), x)

"""The grouped routing, norm and int8 calls where calls go wrong: offsets past
32 bits, the same expert twice, signed zeros, two host threads, captured
replays of long batches, copies of the packed weights."""

from __future__ import annotations

import copy
import pickle
import threading

import pytest
import torch

from moe_serving_profile_b200 import _lib, experts, layout, native, ops
from tests.test_int8 import distinct, layer64, on, packed, quant, run_gemm
from tests.test_route_grouped import check, plain


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """Rows behind the 4 GB mark of bf16 inputs and the 2 GB mark of codes equal
    the same rows alone."""
    T, H = 600_000, 4096
    part = torch.randn(64, H, device=cuda).to(torch.bfloat16)
    x = part.repeat(T // 64, 1)
    w = torch.rand(H, device=cuda)
    want = ops.add_rmsnorm(part, w, 1e-6, residual=part, quant="int8")
    n = ops.add_rmsnorm(x, w, 1e-6, residual=x, quant="int8")
    for a, b in ((n.out, want.out), (n.residual, want.residual), (n.rows.q, want.rows.q),
                 (n.rows.scale, want.rows.scale)):
        assert torch.equal(a[-64:], b) and torch.equal(a[:64], b)
    lin = layout.int8_linear(*layout.quantize_int8(torch.randn(136, H, device=cuda)))
    y, y0 = experts.int8_linear(lin, n.rows), experts.int8_linear(lin, want.rows)
    assert torch.equal(y[-64:], y0) and torch.equal(y[T // 2 // 64 * 64:][:64], y0)
    del n
    y = experts.int8_linear(lin, x)
    assert torch.equal(y[-64:], experts.int8_linear(lin, part))
    del x, y
    torch.cuda.empty_cache()
    logits = torch.randn(64, 512, device=cuda)
    many = logits.repeat(70_000, 1)                       # 9 GB of fp32 logits
    r = ops.route_grouped(many, None, 8, n_group=8, topk_group=4)
    r0 = ops.route_grouped(logits, None, 8, n_group=8, topk_group=4)
    assert torch.equal(r.indices[-64:], r0.indices) and torch.equal(r.scores[-64:], r0.scores)
    assert torch.equal(r.counts, r0.counts * 70_000)


@pytest.mark.gpu
def test_one_expert_many_times(cuda):
    """A token may name an expert twice, and all tokens the same expert."""
    g = torch.Generator().manual_seed(5)
    E, H, I, T, K = 8, 128, 64, 90, 3
    raw, parts, _ = packed(g, E, H, I)
    w = layout.int8_experts(*on(cuda, *parts)[0])
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    wt = torch.rand(T, K, generator=g)
    for idx in (torch.full((T, K), 5), torch.randint(0, E, (T, K), generator=g)):
        y = experts.layer_forward(w, x.to(cuda), idx.to(cuda), wt.to(cuda), num_experts=E, expert_begin=0,
                                  numerics="efficient")
        want = layer64(raw, *quant(x), idx, wt, E)
        assert float((y.cpu().double() - want).norm() / want.norm()) <= 2.0 ** -8


@pytest.mark.gpu
def test_signed_zero_logits_tie(cuda):
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.full((6, 32), -2.0)
        x[:, 5::7] = 0.0
        x[:, 3] = -0.0
        x[1, 20] = -0.0
        for kw in (dict(), dict(n_group=4, topk_group=2, group_top=1), dict(scoring="softmax")):
            check(x.to(dtype).to(cuda), None, 4, **kw)
            check(x.to(dtype).to(cuda), torch.zeros(32, device=cuda), 4, **kw)


@pytest.mark.gpu
def test_saturated_scores_tie(cuda):
    """Logits whose scores 64 bits round together go by id, others by score."""
    x = torch.tensor([[40.0, 50.0, 45.0, 38.0, 16.0, 15.5, 17.0, 37.5],
                      [-800.0, -750.0, -900.0, -600.0, -500.0, -1000.0, -20.0, -700.0]])
    for dtype in (torch.float32, torch.bfloat16):
        for scoring in ("sigmoid", "softmax"):
            for kw in (dict(), dict(n_group=4, topk_group=3, group_top=1)):
                check(x.to(dtype).to(cuda), None, 6, scoring=scoring, **kw)


@pytest.mark.gpu
def test_calls_of_two_threads(cuda):
    """Two host threads, each on its own stream, get what one gets."""
    g = torch.Generator().manual_seed(8)
    E, H, I, T, K = 16, 256, 128, 500, 4
    raw, parts, _ = packed(g, E, H, I)
    w = layout.int8_experts(*on(cuda, *parts)[0])
    xs = [torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2)]
    gate = torch.randn(E, H, generator=g).to(cuda)
    bias = (torch.randn(E, generator=g) * 0.05).to(cuda)

    def block(x):
        n = ops.add_rmsnorm(x, torch.ones(H, device=cuda), 1e-6, residual=x, quant="int8")
        r = ops.route_grouped(n.out.float() @ gate.t(), bias, K, n_group=4, topk_group=2)
        return experts.layer_forward(w, n.out, r.indices, r.scores, num_experts=E, expert_begin=0,
                                     numerics="efficient", rows=n.rows), r.counts

    want = [block(x) for x in xs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[i].append(block(xs[i]))
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    for i in range(2):
        assert len(got[i]) == 20
        for y, c in got[i]:
            assert torch.equal(y, want[i][0]) and torch.equal(c, want[i][1])


@pytest.mark.gpu
def test_captured_long_batches(cuda):
    """Routing (whose counts a second kernel zeroes), the quantiser and the
    products of a long batch, replayed on new inputs."""
    g = torch.Generator().manual_seed(2)
    T, E, K = 3000, 64, 6
    logits = [torch.randn(T, E, generator=g).to(cuda) for _ in range(3)]
    lin = layout.int8_linear(*layout.quantize_int8(torch.randn(520, 328, generator=g).to(cuda)))
    xs = [torch.randn(T, 328, generator=g).to(torch.bfloat16).to(cuda) for _ in range(3)]

    def step(a, x):
        r = ops.route_grouped(a, None, K, n_group=8, topk_group=3, scoring="softmax")
        return r.indices, r.scores, r.counts, experts.int8_linear(lin, x)

    want = [step(a, x) for a, x in zip(logits, xs)]
    a, x = logits[0].clone(), xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, x)
    for i in (1, 2, 0, 0):
        a.copy_(logits[i])
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(out, want[i]):
            assert torch.equal(o, w)
    idx, _, counts = plain(logits[1].cpu(), None, K, 8, 3, 2, "softmax", True, 1.0)
    assert torch.equal(want[1][0].cpu(), idx) and torch.equal(want[1][2].cpu().long(), counts)


@pytest.mark.gpu
def test_many_tiles_of_pairs(cuda):
    """256-row tiles: odd numbers of feature tiles, chunks of all sizes and more
    tiles than CTA pairs."""
    from tests.test_int8 import run_gemm
    g = torch.Generator().manual_seed(12)
    for planes, F, K in ((1, 1160, 136), (2, 456, 136), (1, 264, 1112)):
        run_gemm(cuda, g, [1, 31, 32, 33, 255, 256, 257, 0, 511, 700], planes, F, K, 256)
    run_gemm(cuda, g, [260] * 60, 1, 640, 256, 256, row_w=torch.float32)
    assert _lib.device_status(0) == 0


def test_packed_weights_copy_and_pickle():
    g = torch.Generator().manual_seed(3)
    _, parts, _ = packed(g, 2, 64, 16)
    w = layout.int8_experts(*parts)
    for other in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        for m, o in ((w.m1, other.m1), (w.m2, other.m2)):
            assert torch.equal(m.weight, o.weight) and torch.equal(m.scale, o.scale) and o.bias is None
            assert m.weight.data_ptr() != o.weight.data_ptr()
            assert (m.n_experts, m.planes, m.n_feat, m.k_valid, m.feat_pad, m.k_pad, m.epilogue) == (
                o.n_experts, o.planes, o.n_feat, o.k_valid, o.feat_pad, o.k_pad, o.epilogue)
    r = pickle.loads(pickle.dumps(ops.QuantRows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2))))
    assert r.q.shape == (2, 128) and r.scale.shape == (2,)
    with pytest.raises(ValueError, match="tiles"):
        ops.Int8Matrix(2, 2, 16, 64, 128, 128, w.w1[:1], w.s1, None, _lib.EPI_SWIGLU_F32)
    with pytest.raises(ValueError, match="sizes"):
        ops.Int8Matrix(2, 2, 200, 64, 128, 128, w.w1, w.s1, None, _lib.EPI_SWIGLU_F32)
    with pytest.raises(ValueError, match="scale"):
        ops.Int8Matrix(2, 2, 16, 64, 128, 128, w.w1, w.s1.double(), None, _lib.EPI_SWIGLU_F32)


@pytest.mark.gpu
def test_int8_wrapper_refusals(cuda):
    g = torch.Generator().manual_seed(0)
    _, parts, _ = packed(g, 2, 64, 16)
    w = layout.int8_experts(*on(cuda, *parts)[0])
    x = torch.zeros(6, 64, dtype=torch.bfloat16, device=cuda)
    idx = torch.zeros(3, 2, dtype=torch.int64, device=cuda)
    perm = ops.permute(idx, 2)
    rows = ops.act_quant_int8(x)
    kw = dict(offsets=perm.offsets)
    out = torch.empty(6, 64, dtype=torch.bfloat16, device=cuda)
    bad = [
        lambda: ops.int8_gemm(w.m1, rows, offsets=None),                                   # two experts
        lambda: ops.int8_gemm(w.m1, rows, offsets=perm.offsets[:2]),
        lambda: ops.int8_gemm(w.m1, rows, offsets=perm.offsets.long()),
        lambda: ops.int8_gemm(w.m1, rows, offsets=perm.offsets.cpu()),
        lambda: ops.int8_gemm(w.m1, rows, expert_begin=-1, **kw),
        lambda: ops.int8_gemm(w.m1, ops.QuantRows(rows.q.cpu(), rows.scale), **kw),
        lambda: ops.int8_gemm(w.m1, rows, max_rows=7, **kw),
        lambda: ops.int8_gemm(w.m1, rows, out=out[:5], **kw),
        lambda: ops.int8_gemm(w.m1, rows, out=out[:, :8], **kw),
        lambda: ops.int8_gemm(w.m1, rows, out=out.float(), **kw),
        lambda: ops.int8_gemm(w.m1, rows, out=out.t(), **kw),
        lambda: ops.int8_gemm(w.m1, rows, out=out[:, 1:], **kw),                           # not 16-byte aligned
        lambda: ops.int8_gemm(w.m1, rows, token_tile=48, **kw),
        lambda: ops.int8_gemm(w.m1, rows, row_weight=torch.ones(6, device=cuda), row_src=perm.perm_src, **kw),  # gated
        lambda: ops.int8_gemm(w.m2, ops.act_quant_int8(x[:, :16], k_pad=128), row_weight=torch.ones(5, device=cuda),
                              row_src=perm.perm_src, **kw),
        lambda: ops.int8_gemm(w.m2, ops.act_quant_int8(x[:, :16], k_pad=128), row_weight=torch.ones(6, device=cuda), **kw),
        lambda: ops.int8_project(w.m1, x.float(), **kw),
        lambda: ops.int8_project(w.m1, x[:, :32], **kw),
        lambda: ops.int8_project(w.m1, x[:, 1:], **kw),
        lambda: ops.int8_project(w.m1, x[:3], inverse=perm.inverse, copies=3, **kw),
        lambda: ops.int8_project(w.m1, x[:3], copies=2, **kw),
        lambda: experts.int8_gate_up(w, x[:3, :56], perm, K=2, num_experts=2, expert_begin=0),
        lambda: experts.int8_down(w, x[:5], perm, None, K=2, num_experts=2, expert_begin=0),
        lambda: experts.int8_linear(w.m1, x),
        lambda: experts.int8_swiglu(w, x),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was accepted")
    e = native.LocalSwiGLUExperts(torch.zeros(2, 32, 64, dtype=torch.bfloat16, device=cuda),
                                  torch.zeros(2, 64, 16, dtype=torch.bfloat16, device=cuda), storage="int8")
    assert e(x[:0], idx[:0, 0]).shape == (0, 64) and (e(x, idx.reshape(-1)) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [16, 256])
@pytest.mark.parametrize("offsets", [[0, 40, 100, 260], [-7, 40, 30, 30], [70, 80, 90, 100], [0, 64, 64, 0]])
def test_offsets_outside_the_rows(cuda, tile, offsets):
    """Offsets are kept within the launch's rows, a segment that would end
    before it begins is empty, and rows of no segment are left as they were."""
    rows, K, N = 64, 256, 136
    g = torch.Generator().manual_seed(11)
    w = torch.randint(-127, 128, (3, N, K), generator=g, dtype=torch.int8)
    lin = [layout.int8_linear(w[e].to(cuda), torch.ones(N, device=cuda)) for e in range(3)]
    m = ops.Int8Matrix(3, 1, N, K, 256, K, torch.cat([l.weight for l in lin]), torch.cat([l.scale for l in lin]), None,
                       _lib.EPI_DOWN_ONCE)
    q = torch.randint(-127, 128, (rows, K), generator=g, dtype=torch.int8)
    guard = torch.full((rows + 64, N), 7.0, device=cuda, dtype=torch.bfloat16)
    ops.int8_gemm(m, ops.QuantRows(q.to(cuda), torch.ones(rows, device=cuda)), token_tile=tile, out=guard,
                  offsets=torch.tensor(offsets, dtype=torch.int32, device=cuda))
    want = torch.full((rows + 64, N), 7.0, dtype=torch.float64)
    at = [min(max(o, 0), rows) for o in offsets]
    for e in range(3):
        for r in range(at[e], max(at[e], at[e + 1])):
            want[r] = w[e].double() @ q[r].double()
    # sums below 2^24 are exact in fp32; one rounding to bf16
    assert torch.equal(guard.cpu(), want.to(torch.float32).to(torch.bfloat16))


@pytest.mark.gpu
def test_negative_sizes_are_refused(cuda):
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=cuda)
    lin = layout.int8_linear(*layout.quantize_int8(torch.randn(8, 64, device=cuda)))
    for call in (lambda: ops.act_quant_int8(x, k_pad=-128), lambda: ops.act_quant_int8(x, k_pad=48),
                 lambda: ops.int8_gemm(lin, ops.act_quant_int8(x), max_rows=-1)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("planes", [1, 2])
def test_last_chunks_of_every_size(cuda, planes):
    """Token tile 256: experts whose last chunk of rows comes in each box size,
    with ragged ends; an odd number of feature tiles; many tiles a CTA."""
    g = torch.Generator().manual_seed(21 + planes)
    run_gemm(cuda, g, [0, 1, 31, 64, 65, 128, 129, 255, 256, 257, 320, 321, 385, 513, 1100, 3], planes, 136, 264, 256)
    run_gemm(cuda, g, [300, 5, 270], planes, 264, 1000, 256, begin=2)
    run_gemm(cuda, g, [290, 600, 40, 700, 258], planes, 4096, 128, 256)


@pytest.mark.gpu
def test_calls_back_to_back(cuda):
    """Kernels that begin before their predecessor ends read nothing too early:
    buffers rewritten between calls, with and without a wait after every call,
    and captured."""
    g = torch.Generator().manual_seed(31)
    E, K, H, I, T, n = 16, 4, 512, 256, 200, 24
    _, parts, _ = packed(g, E, H, I)
    w = layout.int8_experts(*on(cuda, *parts)[0])
    weight = torch.rand(H, generator=g).to(torch.bfloat16).to(cuda)
    xs = torch.randn(n, T, H, generator=g).to(torch.bfloat16).to(cuda)
    ls = torch.randn(n, T, E, generator=g).to(cuda)
    few = torch.arange(T, device=cuda)[None] < (torch.arange(n, device=cuda) % 3 * 90 + 9)[:, None]
    xs *= few[:, :, None]
    x, logits, res = torch.empty_like(xs[0]), torch.empty_like(ls[0]), torch.zeros_like(xs[0])
    out = torch.empty_like(xs)

    def run(wait):
        res.zero_()
        for i in range(n):
            x.copy_(xs[i])
            logits.copy_(ls[i])
            for rows in (T, 10):   # two launches of the router, and one
                r = ops.route_grouped(logits[:rows], None, K, n_group=4, topk_group=2)
                wait()
                norm = ops.add_rmsnorm(x[:rows], weight, 1e-6, residual=res[:rows], residual_out=res[:rows], quant="int8")
                wait()
                y = experts.layer_forward(w, norm.out, r.indices, r.scores, num_experts=E, expert_begin=0,
                                          numerics="efficient", rows=norm.rows)
                wait()
                y = y + experts.layer_forward(w, norm.out, r.indices, r.scores, num_experts=E, expert_begin=0,
                                              numerics="efficient")
                out[i, :rows] = y
            wait()
        return out.clone()

    want = run(torch.cuda.synchronize)
    got = run(lambda: None)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(lambda: None)
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)

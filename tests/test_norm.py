"""RMS norm with the residual's addition and an 8-bit output
(``ops.add_rmsnorm``), the int8 row quantiser and the movers of 8-bit rows.

Tolerances: the new residual is exact (one fp32 sum, one rounding). fp32
rounding errors of y are below 64 half-steps (2^-24 each): the squares' sum
(at most 32 serial additions and 10 of a tree, halved by the root), the
quotient, the root, two products. out adds a bf16 half-step of 2^-8. An e4m3
value is off by half a step, 2^-4 of it or 2^-10 below the smallest normal; an
int8 value by half a step of its scale; a quotient that lands next to a border
moves by the fp32 error times at most 448 (or 127) steps.
"""

from __future__ import annotations

import pytest
import torch

from moe_serving_profile_b200 import _lib, norm, ops

FAKE = 0x10000
F32 = 64 * 2.0 ** -24


def rows(g, T, H, pad, scale=1.0):
    return (torch.randn(T, H + pad, generator=g) * scale).to(torch.bfloat16)[:, :H]


def plain(x, residual, weight, eps):
    h = x if residual is None else (x.float() + residual.float()).to(torch.bfloat16)
    f = h.double()
    return h, f / torch.sqrt(f.square().mean(1, keepdim=True) + eps) * weight.double()


def check_fp8(r: ops.QuantRows, y, H, k_pad):
    q, s = r.q.cpu().float().double(), r.scale.cpu().double()
    G = -(-k_pad // 128)
    assert q.shape == (y.shape[0], k_pad) and s.shape == (y.shape[0], G)
    assert (q[:, H:] == 0).all()
    p = torch.zeros(y.shape[0], G * 128, dtype=torch.float64)
    p[:, :H] = y
    amax = p.view(-1, G, 128).abs().amax(2)
    want = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    assert (s - want).abs().le((F32 + 2 ** -24) * want).all()
    step = s.repeat_interleave(128, 1)[:, :H]
    err = (q[:, :H] * step - y).abs()
    assert err.le(y.abs() * (2.0 ** -4 + 2 * F32) + step * (2.0 ** -10 + 448 * F32)).all()


def check_int8(r: ops.QuantRows, y, H, k_pad):
    q, s = r.q.cpu().double(), r.scale.cpu().double()
    assert q.shape == (y.shape[0], k_pad) and s.shape == (y.shape[0],)
    assert (q[:, H:] == 0).all()
    amax = y.abs().amax(1)
    want = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    assert (s - want).abs().le((F32 + 2 ** -24) * want).all()
    assert (q[:, :H] * s[:, None] - y).abs().le(s[:, None] * (0.5 + 127 * 2 * F32)).all()


CASES = [(1, 8, 0), (1, 2048, 0), (3, 16, 8), (5, 136, 0), (7, 2880, 0), (33, 2048, 64), (64, 4096, 0), (2, 8192, 8),
         (2, 4104, 0), (9, 768, 8), (1, 32768, 0), (130, 1024, 0), (4, 1032, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,pad", CASES)
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_matches_the_formula(cuda, T, H, pad, wdtype):
    g = torch.Generator().manual_seed(T + H)
    x, res = rows(g, T, H, pad), rows(g, T, H, pad, 5.0)
    res[:, ::37] *= 40
    w = (1 + 0.2 * torch.randn(H, generator=g)).to(wdtype)
    xd, rd, wd = (torch.empty(T, H + pad, dtype=torch.bfloat16, device=cuda)[:, :H].copy_(x),
                  torch.empty(T, H + pad, dtype=torch.bfloat16, device=cuda)[:, :H].copy_(res), w.to(cuda))
    for residual, rdev in ((None, None), (res, rd)):
        h, y = plain(x, residual, w, 1e-6)
        for quant in (None, "fp8", "int8"):
            k_pads = (None,) if quant is None else (None, -(-H // 16) * 16, -(-H // 128) * 128)
            for k_pad in k_pads:
                n = ops.add_rmsnorm(xd, wd, 1e-6, residual=rdev, quant=quant, k_pad=k_pad)
                assert (n.out.cpu().double() - y).abs().le(y.abs() * (2.0 ** -8 + F32)).all()
                if residual is None:
                    assert n.residual is None
                else:
                    assert torch.equal(n.residual.cpu(), h)
                if quant == "fp8":
                    check_fp8(n.rows, y, H, k_pad or -(-H // 64) * 64)
                elif quant == "int8":
                    check_int8(n.rows, y, H, k_pad or -(-H // 128) * 128)


@pytest.mark.gpu
def test_in_place_and_partial_outputs(cuda):
    g = torch.Generator().manual_seed(2)
    x, res = rows(g, 21, 512, 0).to(cuda), rows(g, 21, 512, 0, 3.0).to(cuda)
    m = norm.AddRMSNorm(512, 1e-5, quant="int8").to(cuda)
    m.weight.data = torch.rand(512, generator=g).to(cuda)
    want = m(x, res)
    keep = res.clone()
    n = m(x, res, inplace=True, normed=False)
    assert n.out is None and n.residual.data_ptr() == res.data_ptr()
    assert torch.equal(res, want.residual) and not torch.equal(res, keep)
    assert torch.equal(n.rows.q, want.rows.q) and torch.equal(n.rows.scale, want.rows.scale)
    # a view of a wider buffer: columns outside it and rows behind it stay
    wide = torch.full((30, 640), 7.0, dtype=torch.bfloat16, device=cuda)
    out = wide[:21, 64:576]
    ops.add_rmsnorm(x, m.weight, 1e-5, residual=keep, residual_out=out)
    assert torch.equal(out, want.residual)
    assert (wide[21:] == 7).all() and (wide[:, :64] == 7).all() and (wide[:, 576:] == 7).all()
    e = m(x[:0], res[:0])
    assert e.out.shape == (0, 512) and e.rows.q.shape == (0, 512)


@pytest.mark.gpu
def test_zero_tiny_and_non_finite_rows(cuda):
    x = torch.zeros(9, 256, dtype=torch.bfloat16)
    x[1, 3] = 1.0
    x[2] = 1e-40                     # subnormal in bf16
    x[3, 130] = float("inf")
    x[4, 7] = float("nan")
    x[5] = 3e38
    x[6, :128] = 2.0                 # a group of zeros beside one of values
    x[7] = -1.0
    w = torch.ones(256)
    d = x.to(cuda)
    fp8 = ops.add_rmsnorm(d, w.to(cuda), 1e-6, quant="fp8").rows
    n = ops.add_rmsnorm(d, w.to(cuda), 1e-6, quant="int8")
    i8 = n.rows
    ok = [0, 1, 2, 6, 7]
    _, y = plain(x[ok], None, w, 1e-6)
    check_int8(ops.QuantRows(i8.q[ok], i8.scale[ok]), y, 256, 256)
    check_fp8(ops.QuantRows(fp8.q.view(torch.uint8)[ok].view(torch.float8_e4m3fn), fp8.scale[ok]), y, 256, 256)
    assert (i8.scale[0] == 1) and (fp8.scale[0] == 1).all() and fp8.scale[6, 1] == 1
    # nothing finite comes out of a row that holds inf or NaN
    for r in (3, 4):
        assert not (i8.q[r].float() * i8.scale[r]).isfinite().any()
    # the squares of a huge row overflow fp32: the norm is zero, not NaN
    assert (n.out[5] == 0).all() and (i8.q[5] == 0).all() and i8.scale[5] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,k_valid,k_pad,E", [(1, 1, 8, 16, 4), (1, 8, 2048, 2048, 128), (37, 4, 2880, 2944, 32),
                                                (200, 8, 768, 768, 16), (5, 3, 32768, 32768, 8), (64, 2, 72, 128, 8)])
def test_act_quant_int8(cuda, T, K, k_valid, k_pad, E):
    """Codes and scales equal plain fp32 arithmetic (one quotient each), at
    every place of the permuted order, of all experts or of a rank's."""
    g = torch.Generator().manual_seed(T * K + k_valid)
    x = (torch.randn(T, k_valid + 8, generator=g) * torch.rand(T, 1, generator=g) * 9).to(torch.bfloat16)[:, :k_valid]
    if T > 3:
        x[2] = 0
        x[3, 1] = 3e38
    amax = x.float().abs().amax(1)
    s = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    q = torch.zeros(T, k_pad, dtype=torch.int8)
    q[:, :k_valid] = torch.round(x.float() / s[:, None]).to(torch.int8)
    xd = torch.empty(T, k_valid + 8, dtype=torch.bfloat16, device=cuda)[:, :k_valid].copy_(x)
    r = ops.act_quant_int8(xd, k_pad=k_pad)
    assert torch.equal(r.q.cpu(), q) and torch.equal(r.scale.cpu(), s)
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(cuda)
    if T > 5:
        idx[5, 0] = E                # a dropped slot
    perm = ops.permute(idx, E)
    _lib.device_status(0)            # the dropped id raised its flag
    inv = perm.inverse.cpu().view(T, K).long()
    at = perm.offsets.cpu()
    for lo, hi in ((0, E), (E // 4, E // 2)):
        kw = {} if (lo, hi) == (0, E) else dict(offsets=perm.offsets, expert_lo=lo, expert_hi=hi)
        moved = (ops.act_quant_int8(xd, k_pad=k_pad, inverse=perm.inverse, copies=K, **kw),
                 ops.scatter_rows_8bit(r, perm.inverse, K, **kw))
        for m in moved:
            for t in range(T):
                for c in range(K):
                    d = inv[t, c].item()
                    if d >= 0 and at[lo] <= d < at[hi]:
                        assert torch.equal(m.q[d].cpu(), q[t]) and m.scale[d].item() == s[t].item()


@pytest.mark.gpu
def test_scatter_leaves_other_rows(cuda):
    """Rows of no token and of other ranks' experts are not written, fp8 rows
    keep all their scales."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(11, 320, generator=g).to(torch.bfloat16).to(cuda)
    q, s = ops.act_quant_fp8(x, k_pad=320)
    idx = torch.stack([torch.randperm(8, generator=g)[:3] for _ in range(11)]).to(cuda)
    perm = ops.permute(idx, 8)
    out = torch.full((33, 320), 3, dtype=torch.uint8, device=cuda)
    sc = torch.full((33, 3), -1.0, device=cuda)
    at = perm.offsets.tolist()
    _lib.check(_lib.lib.b200moe_scatter_rows_8bit(
        0, torch.cuda.current_stream().cuda_stream, q.data_ptr(), 320, s.data_ptr(), 3, 11, perm.inverse.data_ptr(), 3,
        33, perm.offsets.data_ptr(), 2, 5, out.data_ptr(), sc.data_ptr()), "scatter")
    assert (out[:at[2]] == 3).all() and (out[at[5]:] == 3).all()
    assert (sc[:at[2]] == -1).all() and (sc[at[5]:] == -1).all()
    src = perm.perm_src[at[2]:at[5]].long() // 3
    assert torch.equal(out[at[2]:at[5]], q.view(torch.uint8)[src]) and torch.equal(sc[at[2]:at[5]], s[src])


def test_refusals():
    L = _lib.lib

    def nrm(T=4, H=64, ldx=None, res=None, ldr=64, ro=None, ldro=64, w=FAKE, wf=0, eps=1e-6, out=FAKE, ldo=64,
            quant=0, q=FAKE, k_pad=64, s=FAKE, x=FAKE):
        return L.b200moe_add_rmsnorm(0, None, x, H if ldx is None else ldx, res, ldr, ro, ldro, w, wf, eps, T, H, out,
                                     ldo, quant, q, k_pad, s)

    for bad in (dict(T=-1), dict(H=0), dict(H=12), dict(ldx=60), dict(ldx=68), dict(res=FAKE, ldr=60), dict(ro=FAKE),
                dict(res=FAKE, ro=FAKE, ldro=32), dict(w=None), dict(wf=2), dict(eps=-1.0), dict(ldo=32),
                dict(quant=3), dict(quant=1, k_pad=48), dict(quant=1, k_pad=72), dict(quant=2, q=None),
                dict(quant=2, s=None), dict(x=None), dict(x=FAKE + 8), dict(out=FAKE + 2), dict(w=FAKE + 4),
                dict(quant=1, q=FAKE + 8), dict(res=FAKE + 4), dict(eps=float("nan"))):
        assert nrm(**bad) == _lib.ERR_INVALID, bad
    assert nrm(H=32776, ldo=40000) == _lib.ERR_UNSUPPORTED
    assert nrm(quant=1, k_pad=32784) == _lib.ERR_UNSUPPORTED
    assert nrm(T=0, x=None) == _lib.OK

    def act(x=FAKE, ldx=128, rows=4, kv=128, kp=128, inv=None, copies=1, out=4, off=None, lo=0, hi=0, q=FAKE, s=FAKE):
        return L.b200moe_act_quant_int8(0, None, x, ldx, rows, kv, kp, inv, copies, out, off, lo, hi, q, s)

    for bad in (dict(rows=-1), dict(kv=0), dict(kv=124), dict(kp=120), dict(kp=136), dict(ldx=120), dict(ldx=132),
                dict(copies=0), dict(copies=2), dict(out=3), dict(off=FAKE, lo=3, hi=2), dict(x=None), dict(q=None),
                dict(s=None), dict(x=FAKE + 4), dict(q=FAKE + 4)):
        assert act(**bad) == _lib.ERR_INVALID, bad
    assert act(kp=32784) == _lib.ERR_UNSUPPORTED
    assert act(rows=0, x=None) == _lib.OK

    def sct(q=FAKE, nb=128, sc=FAKE, groups=1, rows=4, inv=FAKE, copies=2, out=8, off=None, lo=0, hi=0, o=FAKE, os=FAKE):
        return L.b200moe_scatter_rows_8bit(0, None, q, nb, sc, groups, rows, inv, copies, out, off, lo, hi, o, os)

    for bad in (dict(nb=0), dict(nb=24), dict(groups=0), dict(rows=-1), dict(inv=None), dict(copies=0), dict(q=None),
                dict(o=None), dict(sc=None), dict(os=None), dict(q=FAKE + 8), dict(off=FAKE, lo=-1, hi=2)):
        assert sct(**bad) == _lib.ERR_INVALID, bad
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.add_rmsnorm(x, torch.ones(64), 1e-6)
    with pytest.raises(ValueError, match="CUDA"):
        ops.act_quant_int8(x)
    with pytest.raises(ValueError, match="quant"):
        norm.AddRMSNorm(64, quant="int4")
    with pytest.raises(NotImplementedError):
        norm.AddRMSNorm(60)


@pytest.mark.gpu
def test_wrapper_refusals(cuda):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda)
    w = torch.ones(64, device=cuda)
    for kw in (dict(quant="int4"), dict(residual=x[:3]), dict(residual=x.float()), dict(residual_out=x),
               dict(residual=x.cpu()), dict(normed=False), dict(quant="fp8", k_pad=40),
               dict(residual=torch.zeros(4, 65, dtype=torch.bfloat16, device=cuda)[:, 1:])):
        with pytest.raises(ValueError):
            ops.add_rmsnorm(x, w, 1e-6, **kw)
    for bad in (w[:32], w.half(), w.cpu()):
        with pytest.raises(ValueError):
            ops.add_rmsnorm(x, bad, 1e-6)
    r = ops.act_quant_int8(x)
    inv = torch.zeros(8, dtype=torch.int32, device=cuda)
    for fn in (lambda: ops.scatter_rows_8bit(r, inv, 3), lambda: ops.scatter_rows_8bit(r, inv.long(), 2),
               lambda: ops.act_quant_int8(x, copies=2), lambda: ops.act_quant_int8(x, inverse=inv.cpu(), copies=2),
               lambda: ops.scatter_rows_8bit(ops.QuantRows(r.q, r.scale[:3]), inv, 2),
               lambda: ops.act_quant_int8(x.float())):
        with pytest.raises(ValueError):
            fn()

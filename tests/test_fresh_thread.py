"""Calls that are a host thread's first CUDA work: the thread has no current
context then, which the GEMMs' tensor maps need."""

from __future__ import annotations

import threading

import pytest
import torch

from moe_serving_profile_b200 import _lib, layout, ops


def in_thread(f):
    got = []

    def work():
        try:
            f()
            got.append(None)
        except Exception as e:   # noqa: BLE001
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join(120)
    assert got == [None], got


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "bf16", "w8a8"])
def test_gemm_is_a_threads_first_call(cuda, fmt):
    """Inputs and outputs exist already, and the library has served the main thread."""
    g = torch.Generator().manual_seed(1)
    H, I, T = 256, 128, 64
    off = torch.tensor([0, T], dtype=torch.int32, device=cuda)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
    out = torch.zeros(T, I, dtype=torch.bfloat16, device=cuda)
    if fmt == "int8":
        lin = layout.int8_linear(*layout.quantize_int8(torch.randn(I, H, generator=g).to(cuda)))
        rows = ops.act_quant_int8(x)
        call = lambda: ops.int8_gemm(lin, rows, out=out)                           # noqa: E731
    else:
        kw = dict(offsets=off, expert_begin=0, n_experts=1, max_rows=T, planes=2, epilogue=_lib.EPI_SWIGLU, out=out)
        if fmt == "bf16":
            w = layout.bf16_experts(*((torch.randn(1, *s, generator=g) * 0.1).to(torch.bfloat16).to(cuda)
                                      for s in ((I, H), (I, H), (H, I))))
            kw.update(wfmt=w.fmt, b_src=x, k_valid=H, bias=None)
        else:
            def block(*s):
                return (torch.randn(1, *s, generator=g).to(torch.float8_e4m3fn).to(cuda),
                        torch.ones(1, s[0] // 128, s[1] // 128, device=cuda))
            w = layout.fp8_experts(*block(I, H), *block(I, H), *block(H, I), (128, 128))
            q, s = ops.act_quant_fp8(x)
            kw.update(q=q, q_scale=s, fp8_block=w.block)
        kw.update(feat_pad=w.i_pad, n_feat=w.inter, k_pad=w.h_k, weight=w.w1)
        call = (lambda: ops.expert_gemm(**kw)) if fmt == "bf16" else (lambda: ops.w8a8_gemm(**kw))
    call()
    torch.cuda.synchronize()
    want = out.clone()
    assert want.isfinite().all() and (want != 0).any()
    out.zero_()
    torch.cuda.synchronize()
    in_thread(call)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and _lib.device_status(0) == 0

"""The torch binding where it does not load (CPU): what goes through ctypes stays
usable, and calls that need the binding say how to build it."""

from __future__ import annotations

import subprocess
import sys
import textwrap

from tests.conftest import ROOT


def run(code: str) -> str:
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


def test_package_without_the_binding():
    out = run("""
        import sys
        sys.modules["moe_serving_profile_b200._ext"] = None     # its import fails
        import torch
        from moe_serving_profile_b200 import experts, gpt_oss, layout, native, norm, ops, qwen3, router
        w = layout.bf16_experts(*(torch.zeros(2, *s, dtype=torch.bfloat16) for s in ((16, 64), (16, 64), (64, 16))))
        assert w.n_experts == 2
        x = torch.zeros(4, 64, dtype=torch.bfloat16)
        calls = [
            lambda: ops.route_grouped(torch.zeros(4, 8), None, 2),
            lambda: ops.act_quant_int8(x),
            lambda: ops.add_rmsnorm(x, torch.ones(64), 1e-6),
            lambda: norm.AddRMSNorm(64)(x),
            lambda: ops.scatter_rows_8bit(None, None, 1),
            lambda: ops.int8_gemm(None, None),
            lambda: ops.int8_project(None, x),
            lambda: ops.QuantRows(x, x),
            lambda: layout.int8_linear(torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)),
        ]
        for call in calls:
            try:
                call()
            except ImportError as e:
                assert "moe_serving_profile_b200.build" in str(e)
            else:
                raise SystemExit("accepted")
        try:
            ops.act_quant_fp8(x)                                # through ctypes: its own check
        except ValueError as e:
            print("ok", e)
        """)
    assert out.startswith("ok")


def test_binding_of_another_torch_is_not_used():
    out = run("""
        import sys, types
        other = types.ModuleType("moe_serving_profile_b200._ext")
        other.built_for = "torch 1.0 cpython-30"
        sys.modules["moe_serving_profile_b200._ext"] = other
        import torch
        from moe_serving_profile_b200 import ops
        try:
            ops.add_rmsnorm(torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64), 1e-6)
        except ImportError as e:
            print(e)
        """)
    assert "built for torch 1.0 cpython-30" in out


def test_binding_of_another_torch_is_rebuilt(tmp_path, monkeypatch):
    """A torch of another version, with no file newer than the binding."""
    from moe_serving_profile_b200 import build

    runs = []

    def compile_(cmd, check):
        runs.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "wb") as f:
            f.write(b"\0" + build.ext_key().encode() + b"\0")

    ext = tmp_path / "_ext.so"
    ext.write_bytes(build.EXT.read_bytes())      # newer than every source
    monkeypatch.setattr(build, "EXT", ext)
    monkeypatch.setattr(build.subprocess, "run", compile_)
    build.build_ext()
    assert not runs                                     # the torch that it was built for
    import torch
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".post1")
    build.build_ext()
    assert len(runs) == 1 and any("post1" in a for a in runs[0])
    build.build_ext()
    assert len(runs) == 1

"""Backend labels name the storage that the experts have."""

from __future__ import annotations

import pytest

from moe_serving_profile_b200 import backend


def test_labels_of_every_storage():
    label = lambda *a: backend.backend_metadata(*a)["experts"]   # noqa: E731
    assert label("qwen3", "efficient", "int8") == "b200_tcgen05_grouped_int8_channel_w8a8_dynamic_act_row"
    assert label("qwen3", "efficient", "fp8") == label("qwen3", "efficient") == (
        "b200_tcgen05_grouped_fp8_e4m3_block128_w8a8_dynamic_act_128")
    assert label("qwen3", "reference") == "b200_tcgen05_grouped_fp8_e4m3_block128_weight_only"
    assert label("qwen3", "reference", "bf16") == "b200_tcgen05_grouped_bf16_weight_only"
    assert label("gpt_oss", "efficient") == label("gpt_oss", "efficient", "mxfp4") == (
        "b200_tcgen05_grouped_mxfp4_e2m1_ue8m0_weight_only")
    with pytest.raises(ValueError, match="efficient"):
        backend.backend_metadata("qwen3", "reference", "int8")
    with pytest.raises(ValueError, match="storage"):
        backend.backend_metadata("gpt_oss", "efficient", "int8")

"""What bench.py sets a prompt's time against, by the type that its products run in."""
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import bench


def test_layers_in_16_bits():
    cfg, T = bench.QWEN3_8B, 2048
    nums = bench.model_numbers(cfg, 36)
    flops = 2.0 * (nums["linear_params"] - cfg["vocab_size"] * cfg["hidden_size"]) * T + 2.0 * cfg["vocab_size"] * cfg["hidden_size"] \
        + 36 * 4.0 * nums["Q"] * T * (T + 1) / 2
    assert bench.prefill_floor_s(cfg, nums, 36, T, 1600.0) == pytest.approx(flops / 1600e12, rel=1e-12)


@pytest.mark.parametrize("cfg", [bench.QWEN3_8B, bench.LLAMA3_8B])
@pytest.mark.parametrize("T", [1, 512, 2048, 8192])
def test_layers_in_8_bits(cfg, T):
    """Only the layers' products run at twice the rate: the floor lies between half of the 16-bit one and the whole of it, by the products' share."""
    n = cfg["num_hidden_layers"]
    nums, eight = bench.model_numbers(cfg, n), bench.model_numbers(cfg, n, "float8")
    stored, floor = bench.prefill_floor_s(cfg, nums, n, T, 1600.0), bench.prefill_floor_s(cfg, eight, n, T, 1600.0, "float8")
    assert floor == pytest.approx(stored - nums["per_layer"] * n * T / 1600e12, rel=1e-12)
    assert stored / 2 < floor < stored


def test_no_more_than_the_peak_for_what_was_measured():
    """A prompt of 2,048 tokens through 8-bit layers of the Qwen3-8B shape took 16.6 ms at a bfloat16 peak of 1,598 TFLOP/s: above that peak if everything were set against it."""
    cfg = bench.QWEN3_8B
    nums = bench.model_numbers(cfg, 36, "float8")
    assert bench.prefill_floor_s(cfg, nums, 36, 2048, 1598.1) > 16.6e-3
    assert 0.5 < bench.prefill_floor_s(cfg, nums, 36, 2048, 1598.1, "float8") / 16.6e-3 < 0.7

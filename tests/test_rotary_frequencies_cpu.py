"""CPU: rotary frequencies of further scaling entries, and requests refused."""
import math

import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


def _g(factor, m):
    return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0


MSCALE = [({"mscale": 0.707, "mscale_all_dim": 0.707}, 1.0),
          ({"mscale": 1.0, "mscale_all_dim": 0.5}, _g(40.0, 1.0) / _g(40.0, 0.5)),
          ({"mscale": 1, "mscale_all_dim": 1}, 1.0),
          ({"mscale": 1.0}, _g(40.0, 1.0)), ({"mscale_all_dim": 0.5}, _g(40.0, 1.0)),
          ({"mscale": None, "mscale_all_dim": 0.5}, _g(40.0, 1.0)),
          ({"mscale": 0.0, "mscale_all_dim": 1.0}, _g(40.0, 1.0)),
          ({"mscale": 1.0, "mscale_all_dim": 0.5, "attention_factor": 1.25}, 1.25),
          ({"mscale": 1.0, "mscale_all_dim": 0.5, "factor": 0.5}, 1.0)]


@pytest.mark.parametrize("keys, want", MSCALE, ids=[str(i) for i in range(len(MSCALE))])
def test_yarn_mscale(keys, want):
    """The factor of cos and sin; the frequencies do not depend on it.  Both
    sides are the same few operations in 64 bits, eps/2 = 2^-53 each."""
    freq, a = kd.kv_rotary_inv_freq(128, 500000.0, {**YARN, **keys})
    assert abs(a - want) <= 8 * 2.0 ** -53 * want
    assert torch.equal(freq, kd.kv_rotary_inv_freq(128, 500000.0, {**YARN, "factor": keys.get("factor", 40.0)})[0])


@pytest.mark.parametrize("keys", [k for k, _ in MSCALE], ids=[str(i) for i in range(len(MSCALE))])
def test_yarn_mscale_equals_transformers(keys):
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import LlamaConfig
    spec = {**YARN, **keys}
    cfg = LlamaConfig(hidden_size=1024, num_attention_heads=8, head_dim=128, max_position_embeddings=163840,
                      rope_parameters={**spec, "rope_theta": 500000.0})
    _, want = rope.ROPE_INIT_FUNCTIONS["yarn"](cfg, torch.device("cpu"))
    assert abs(kd.kv_rotary_inv_freq(128, 500000.0, spec)[1] - want) <= 1e-12


LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
DYNAMIC = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048, "seq_len": 8192}
LINEAR = {"rope_type": "linear", "factor": 4.0}
BAD = [0.0, -2.0, math.inf, math.nan]


@pytest.mark.parametrize("spec", [LINEAR, DYNAMIC, YARN, LLAMA3], ids=lambda s: s["rope_type"])
@pytest.mark.parametrize("bad", BAD, ids=str)
def test_senseless_numbers_are_refused(spec, bad):
    """No division by zero, no infinite, negative or complex frequencies."""
    for key in ("factor", "original_max_position_embeddings", "seq_len", "high_freq_factor"):
        if key in spec:
            with pytest.raises(RuntimeError):
                kd.kv_rotary_inv_freq(64, 10000.0, {**spec, key: bad})
    with pytest.raises(RuntimeError):
        kd.kv_rotary_inv_freq(64, bad, spec)
    with pytest.raises(RuntimeError):
        kd.kv_rotary_inv_freq(64, bad)


@pytest.mark.parametrize("keys", [
    {"attention_factor": 0.0}, {"attention_factor": -1.0}, {"attention_factor": math.nan}, {"beta_fast": -1.0},
    {"beta_slow": math.inf}, {"beta_fast": math.nan}, {"mscale": math.nan, "mscale_all_dim": 1.0},
    {"mscale": -10.0, "mscale_all_dim": 1.0}, {"mscale": 1.0, "mscale_all_dim": -10.0 / math.log(40.0)}], ids=str)
def test_senseless_yarn_keys_are_refused(keys):
    with pytest.raises(RuntimeError):
        kd.kv_rotary_inv_freq(64, 10000.0, {**YARN, **keys})


def test_frequencies_beyond_fp32_are_refused():
    # the slowest pair: 10000^(-62/64) = 1.3e-4, divided by 1e-45 beyond 3.4e38
    for spec in ({**LINEAR, "factor": 1e-45}, {**YARN, "factor": 1e-45}, {**LLAMA3, "factor": 1e-45}):
        with pytest.raises(RuntimeError):
            kd.kv_rotary_inv_freq(64, 10000.0, spec)


def test_low_freq_factor_may_be_zero_but_a_number():
    freq, _ = kd.kv_rotary_inv_freq(64, 10000.0, {**LLAMA3, "low_freq_factor": 0.0})
    plain = 10000.0 ** -(torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    keep = (8192 * plain / (2 * math.pi) / 4.0).clamp(0.0, 1.0)
    want = keep * plain + (1 - keep) * plain / 8.0
    assert torch.allclose(freq.double(), want, rtol=2.0 ** -23)
    for low in (math.nan, -math.inf, None):
        with pytest.raises(RuntimeError):
            kd.kv_rotary_inv_freq(64, 10000.0, {**LLAMA3, "low_freq_factor": low})


def test_entry_with_another_base_is_refused():
    """An entry that carries its own base is not answered with another one."""
    spec = {**LLAMA3, "rope_theta": 500000.0}
    with pytest.raises(RuntimeError, match="rope_theta"):
        kd.kv_rotary_inv_freq(64, scaling=spec)
    assert torch.equal(kd.kv_rotary_inv_freq(64, 500000, spec)[0], kd.kv_rotary_inv_freq(64, 500000.0, LLAMA3)[0])

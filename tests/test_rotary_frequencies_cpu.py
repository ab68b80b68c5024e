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

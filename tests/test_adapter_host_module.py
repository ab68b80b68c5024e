"""The vLLM impl in a process where the prompt kernel's host module does not
load (another torch or Python than it was built for)."""
import pytest
import torch

from slm_turbo_b200 import _lib


def _broken(monkeypatch):
    def host():
        raise ImportError("_host.so is built for another torch")
    monkeypatch.setattr(_lib, "host", host)


def test_the_impl_looks_at_the_start(monkeypatch, caplog):
    """Found when the impl is made, not in the first prompt step; the store and
    the decode are as they were."""
    ad = pytest.importorskip("slm_turbo_b200.adapters.vllm_adapter")
    if ad.QuantizedKVAttentionImpl is None:
        pytest.skip("vLLM backend API not available")
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    said = []
    monkeypatch.setattr(ad.logger, "warning", lambda text, *args: said.append(text % args))
    make = lambda: ad.QuantizedKVAttentionImpl(  # noqa: E731
        num_heads=8, head_size=64, scale=0.125, num_kv_heads=2, alibi_slopes=None, sliding_window=None,
        kv_cache_dtype="auto")
    impl = make()
    assert impl._slm_kernel and impl._slm_prompt_kernel and not said
    _broken(monkeypatch)
    impl = make()
    assert impl._slm_kernel and not impl._slm_prompt_kernel
    assert len(said) == 1 and "another torch" in said[0]


@pytest.mark.gpu
@pytest.mark.parametrize("capture_path", [False, True])
def test_fresh_prompts_go_to_sdpa(monkeypatch, capture_path):
    from tests.helpers import assert_close
    from tests.test_gpu_adapter import _expected, _impl, _run, _step
    ad, impl = _impl()
    if capture_path:
        monkeypatch.setattr(ad, "_capturing", lambda: True)
    _broken(monkeypatch)
    impl._slm_prompt_kernel = False
    st = _step([(0, 33), (300, 20), (0, 5)], seed=9)
    assert_close(_run(impl, st, torch.device("cuda", torch.cuda.current_device())), _expected(st), what="step")

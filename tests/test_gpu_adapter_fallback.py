"""GPU: steps of the vLLM impl whose tensors the prompt kernel does not take
are served as before, by scaled_dot_product_attention."""
import numpy as np
import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd
from tests.helpers import assert_close
from tests.test_gpu_adapter import BS, D, HQ, KV, _causal_ref, _expected, _impl, _run, _step

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev():
    d = torch.device("cuda", torch.cuda.current_device())
    assert kd.read_device_errors(d) == 0
    yield d
    assert kd.read_device_errors(d) == 0


def _on(st, dev):
    md = st["md"]
    for name, t in list(vars(md).items()):
        if torch.is_tensor(t):
            setattr(md, name, t.to(dev))
    return (st[n].to(dev) for n in ("q", "k", "v", "cache"))


@pytest.mark.parametrize("capture_path", [False, True])
@pytest.mark.parametrize("off", [1, 4])
def test_output_rows_at_any_element(dev, monkeypatch, capture_path, off):
    """An output that starts at an odd element, or on 8 bytes."""
    ad, impl = _impl()
    if capture_path:
        monkeypatch.setattr(ad, "_capturing", lambda: True)
    st = _step([(0, 33), (0, 70), (0, 5)], seed=4)
    want = _expected(st)
    q, k, v, cache = _on(st, dev)
    n = q.shape[0]
    store = torch.full((n * HQ * D + off + 8,), 7.5, dtype=torch.float16, device=dev)
    out = store[off:off + n * HQ * D].view(n, HQ * D)
    impl.forward(None, q, k, v, cache, st["md"], out)
    assert_close(out.float().view(n, HQ, D).cpu().numpy(), want, what="step")
    assert (store[:off] == 7.5).all() and (store[off + n * HQ * D:] == 7.5).all()


@pytest.mark.parametrize("which", ["key", "value"])
def test_key_or_value_that_requires_a_gradient(dev, which):
    """Autograd records; the step is differentiable where it was."""
    _, impl = _impl()
    st = _step([(0, 33), (0, 20)], seed=5)
    want = _expected(st)
    q, k, v, cache = _on(st, dev)
    (k if which == "key" else v).requires_grad_()
    out = torch.zeros(q.shape[0], HQ * D, dtype=torch.float16, device=dev)
    impl.forward(None, q, k, v, cache, st["md"], out)
    assert_close(out.detach().float().view(-1, HQ, D).cpu().numpy(), want, what="step")
    out.float().sum().backward()
    assert (k if which == "key" else v).grad is not None


def test_other_types_and_head_sizes(dev):
    """An output in 64 bits, a head size and a scale that the kernel has not."""
    _, impl = _impl()
    st = _step([(0, 33), (0, 20)], seed=6)
    want = _expected(st)
    q, k, v, cache = _on(st, dev)
    out = torch.zeros(q.shape[0], HQ * D, dtype=torch.float64, device=dev)
    impl.forward(None, q, k, v, cache, st["md"], out)
    assert_close(out.view(-1, HQ, D).cpu().numpy(), want, what="64 bits")
    q2, k2, v2 = (torch.cat([t, t[..., :32]], -1) for t in (q, k, v))  # 96 dims
    impl.head_size = 96
    out = torch.zeros(q.shape[0], HQ * 96, dtype=torch.float16, device=dev)
    impl.forward(None, q2, k2, v2, cache, st["md"], out)
    want = np.concatenate([_causal_ref(q2[a:b].cpu(), k2[a:b].cpu(), v2[a:b].cpu(), impl.scale)
                           for a, b in zip(st["qsl"], st["qsl"][1:])])
    assert_close(out.float().view(-1, HQ, 96).cpu().numpy(), want, what="96 dims")
    impl.head_size, impl.scale = D, 3e38  # times log2 e beyond fp32
    out = torch.zeros(q.shape[0], HQ * D, dtype=torch.float16, device=dev)
    impl.forward(None, q, k, v, cache, st["md"], out)

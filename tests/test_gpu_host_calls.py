"""GPU: what the serving-step entry points refuse, and the errors they raise."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from slm_turbo_b200.kernels import kv_dequant as kd

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev():
    d = torch.device("cuda:0")
    assert kd.read_device_errors(d) == 0
    yield d
    assert kd.read_device_errors(d) == 0


def _args(dev):
    q, k, v = (torch.randn(4, h, 64, device=dev).half() for h in (4, 2, 2))
    pos, freq = torch.arange(4, device=dev), kd.kv_rotary_inv_freq(64, device=dev)[0]
    cache = torch.zeros(2, 16, 2, 72, dtype=torch.uint8, device=dev)
    start = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    return q, k, v, pos, freq, cache, torch.arange(4, device=dev), start


@pytest.mark.parametrize("which", ["query", "key", "value"])
def test_forward_mode_tangents_are_not_dropped(dev, which):
    """A dual tensor is refused like one that requires a gradient: there is no
    forward-mode rule, and its tangent would be lost.  no_grad does not end
    forward mode."""
    q, k, v, pos, freq, cache, slots, start = _args(dev)
    with fwd.dual_level():
        t = {"query": q, "key": k, "value": v}
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        q2, k2, v2 = t.values()
        calls = [lambda: kd.kv_rotary_store(q2, k2, v2, pos, freq, cache, slots),
                 lambda: kd.kv_prompt_attention(q2, k2, v2, start, 4)]
        if which != "value":
            calls.append(lambda: kd.kv_rotary(q2, k2, pos, freq))
        for call in calls:
            with pytest.raises(RuntimeError, match="backward"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="backward"):
                call()
    assert (cache == 0).all()
    kd.kv_rotary_store(q2, k2, v2, pos, freq, cache, slots)  # the level is over


def test_memory_that_runs_out_is_an_out_of_memory_error(dev):
    """Outputs of 2 x 550 GB: torch's own error, as from the other functions."""
    cache = torch.zeros(1, 16, 64, 136, dtype=torch.uint8, device=dev)
    slots = torch.zeros(1 << 24, dtype=torch.int64, device=dev)
    with pytest.raises(torch.OutOfMemoryError):
        kd.kv_dequantize_load(cache, slots, torch.float32)
    k, _ = kd.kv_dequantize_load(cache, slots[:3])
    assert k.shape == (3, 64, 128)


def test_outputs_that_share_memory_are_refused(dev):
    """And buffers next to one another are not."""
    *_, cache, slots, start = _args(dev)
    both = torch.zeros(8, 2, 64, device=dev)
    for a, b in ((both[:4], both[:4]), (both[:4], both[3:7])):
        with pytest.raises(RuntimeError):
            kd.kv_dequantize_load(cache, slots, torch.float32, key_out=a, value_out=b)
    kd.kv_dequantize_load(cache, slots, torch.float32, key_out=both[:4], value_out=both[4:])
    bt = torch.tensor([[1]], dtype=torch.int32, device=dev)
    lens = torch.tensor([4], dtype=torch.int32, device=dev)
    ids = torch.zeros(8, dtype=torch.int64, device=dev)
    for a, b in ((ids[:4], ids[:4]), (ids[3:7], ids[:4])):
        with pytest.raises(RuntimeError):
            kd.kv_page_plan(start, lens, bt, 16, 4, slot_mapping=a, positions=b)
    kd.kv_page_plan(start, lens, bt, 16, 4, slot_mapping=ids[:4], positions=ids[4:])
    assert ids.tolist() == [16, 17, 18, 19, 0, 1, 2, 3]
    assert kd.kv_page_plan(start[:1], lens[:0], bt[:0], 16, 0, slot_mapping=ids[:0], positions=ids[:0])[2].item() == 0

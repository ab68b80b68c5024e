"""GPU: the kernel variants of large steps -- four tokens per CTA in the
rotary kernels, tokens split over blocks and several steps per block in the
load -- at sizes around their edges, bit for bit."""
import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd
from tests.test_gpu_step_ops import _load_ref, _rot_case, _rotate_ref

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev():
    d = torch.device("cuda:0")
    assert kd.read_device_errors(d) == 0
    yield d
    assert kd.read_device_errors(d) == 0


# (tokens, Hq, KV, D, rot): kv heads of one, and of more than a CTA has rows of
BIG_ROT = [(1184, 4, 1, 64, 64), (1185, 3, 33, 64, 32), (1186, 5, 17, 128, 128), (1187, 2, 1, 80, 80),
           (2500, 8, 2, 128, 64), (2501, 1, 19, 80, 16), (1183, 4, 2, 128, 128), (1187, 33, 3, 64, 8),
           (1185, 4, 2, 80, 20), (1186, 2, 1, 128, 118)]


@pytest.mark.parametrize("case", BIG_ROT, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_rotary_of_many_tokens(dev, case, interleaved, dtype):
    q, k, v, pos, freq = _rot_case(*case, dtype, dev)
    wq, wk = (_rotate_ref(t, pos, freq, interleaved, 1.1875) for t in (q, k))
    gq, gk = kd.kv_rotary(q, k, pos, freq, interleaved, 1.1875)
    assert torch.equal(gq, wq) and torch.equal(gk, wk)
    n, _, kv, d, _ = case
    nb = n // 16 + 3
    g = torch.Generator(device=dev).manual_seed(n)
    slots = torch.randperm(nb * 16, device=dev, generator=g)[:n]
    slots[::7], slots[-1] = -1, -1
    fill = torch.randint(0, 256, (nb, 16, kv, d + 8), device=dev, generator=g, dtype=torch.uint8)
    want, got = fill.clone(), fill.clone()
    kd.kv_quantize_store(wk, v, want, slots, 16)
    gq, gk = kd.kv_rotary_store(q, k, v, pos, freq, got, slots, interleaved, 1.1875)
    assert torch.equal(gq, wq) and torch.equal(gk, wk) and torch.equal(got, want)
    # in place, 32-bit positions; then the rows without the store
    got, q2, k2 = fill.clone(), q.clone(), k.clone()
    kd.kv_rotary_store(q2, k2, v, pos.int(), freq, got, slots, interleaved, 1.1875, query_out=q2, key_out=k2)
    assert torch.equal(q2, wq) and torch.equal(k2, wk) and torch.equal(got, want)
    kd.kv_rotary(q, k, pos, freq, interleaved, 1.1875, query_out=q, key_out=k)
    assert torch.equal(q, wq) and torch.equal(k, wk)


# pieces of a token beyond a block's threads (the last block not full), and
# tokens enough for 2 to 8 steps per block, not a multiple of a step
BIG_LOAD = [(77, 32, 80), (1003, 33, 128), (9, 65, 64), (40001, 8, 128), (120001, 1, 64), (50003, 3, 80), (5003, 40, 128),
            (20011, 16, 64)]


@pytest.mark.parametrize("case", BIG_LOAD, ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
def test_load_of_many_tokens_and_heads(dev, case, dtype):
    n, kv, d = case
    nb = n // 16 + 2
    g = torch.Generator(device=dev).manual_seed(n)
    cache = torch.randint(0, 256, (nb, 16, kv, d + 8), device=dev, generator=g, dtype=torch.uint8)
    rulers = torch.randn(nb, 16, kv, 4, device=dev, generator=g).half()
    cache[..., d:] = rulers.view(torch.uint8)
    slots = torch.randint(0, nb * 16, (n,), device=dev, generator=g)
    slots[::11], slots[-1] = -1, -3
    wk, wv = _load_ref(cache, slots.clamp(min=0), dtype)
    wk[slots < 0], wv[slots < 0] = 0, 0
    gk, gv = kd.kv_dequantize_load(cache, slots, dtype)
    assert torch.equal(gk, wk) and torch.equal(gv, wv)
    # rows around the given outputs stay
    ko, vo = (torch.full((n + 2, kv, d), 9.0, dtype=dtype, device=dev) for _ in range(2))
    kd.kv_dequantize_load(cache, slots, dtype, key_out=ko[1:-1], value_out=vo[1:-1])
    for o, w in ((ko, wk), (vo, wv)):
        assert torch.equal(o[1:-1], w) and (o[0] == 9).all() and (o[-1] == 9).all()

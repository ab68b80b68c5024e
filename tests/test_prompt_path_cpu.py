"""CPU: argument checks of the serving-step entries (nothing is launched) and
the rotary frequencies against their formulas."""
import math

import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd

P = 1 << 20  # a made-up device pointer: every call here is refused or empty
HEAD_DIM, SHAPE, DTYPE, ALIGN, NULL, UNSUPPORTED = -2, -3, -4, -5, -1, -7


@pytest.fixture(scope="module")
def lib():
    from slm_turbo_b200 import _lib
    from slm_turbo_b200.build import build_library
    build_library()
    return _lib.load()


def _call(fn, order, base, **kw):
    assert set(kw) <= set(order)
    return fn(*[{**base, **kw}[n] for n in order])


PLAN = "qsl sl r bt bts mb bs fb nf cur n slots pos out err st".split()
PLAN_BASE = dict(qsl=P, sl=P, r=2, bt=P, bts=4, mb=4, bs=16, fb=P, nf=8, cur=P, n=5, slots=P, pos=P, out=2 * P,
                 err=None, st=None)


@pytest.mark.parametrize("kw, rc", [
    (dict(bs=0), SHAPE), (dict(n=-1), SHAPE), (dict(r=-1), SHAPE), (dict(nf=-1), SHAPE), (dict(mb=-1), SHAPE),
    (dict(bts=3), SHAPE), (dict(out=P), SHAPE), (dict(n=1 << 31), SHAPE), (dict(qsl=None), NULL), (dict(sl=None), NULL),
    (dict(bt=None), NULL), (dict(slots=None), NULL), (dict(pos=None), NULL), (dict(n=0, out=None), 0),
])
def test_page_plan_argument_checks(lib, kw, rc):
    assert _call(lib.slmt_page_plan, PLAN, PLAN_BASE, **kw) == rc


ROT = "q qt qh k kt kh dt pos pdt freq rot il sc n hq kv d qo qot qoh ko kot koh st".split()
ROT_BASE = dict(q=P, qt=1024, qh=128, k=P, kt=256, kh=128, dt=0, pos=P, pdt=4, freq=P, rot=128, il=0, sc=1.0, n=3,
                hq=8, kv=2, d=128, qo=P, qot=1024, qoh=128, ko=P, kot=256, koh=128, st=None)
ROT_BAD = [
    (dict(d=96), HEAD_DIM), (dict(rot=130), SHAPE), (dict(rot=63), SHAPE), (dict(rot=-2), SHAPE), (dict(n=-1), SHAPE),
    (dict(dt=2), DTYPE), (dict(pdt=0), DTYPE), (dict(sc=math.inf), SHAPE), (dict(sc=math.nan), SHAPE),
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(pos=None), NULL), (dict(freq=None), NULL), (dict(qo=None), NULL),
    (dict(qot=0), SHAPE), (dict(qoh=0), SHAPE), (dict(kot=0), SHAPE), (dict(n=0), 0),
]


@pytest.mark.parametrize("kw, rc", ROT_BAD + [(dict(ko=None), NULL)])
def test_rotary_argument_checks(lib, kw, rc):
    assert _call(lib.slmt_rotary, ROT, ROT_BASE, **kw) == rc


STORE = ("q qt qh k kt kh v vt vh dt pos pdt freq rot il sc n hq kv d qo qot qoh ko kot koh cache nb bs slots err st"
         .split())
STORE_BASE = dict(ROT_BASE, v=P, vt=256, vh=128, cache=P, nb=4, bs=16, slots=P, err=None)


@pytest.mark.parametrize("kw, rc", ROT_BAD + [
    (dict(v=None), NULL), (dict(cache=None), NULL), (dict(slots=None), NULL), (dict(cache=P + 4), ALIGN),
    (dict(bs=0), SHAPE), (dict(nb=-1), SHAPE), (dict(kv=0), SHAPE)])
def test_rotary_store_argument_checks(lib, kw, rc):
    assert _call(lib.slmt_rotary_store, STORE, STORE_BASE, **kw) == rc


LOAD = "cache nb bs kv d slots n k v dt err st".split()
LOAD_BASE = dict(cache=P, nb=4, bs=16, kv=8, d=128, slots=P, n=3, k=P, v=P, dt=0, err=None, st=None)


@pytest.mark.parametrize("kw, rc", [
    (dict(d=72), HEAD_DIM), (dict(n=-1), SHAPE), (dict(kv=0), SHAPE), (dict(bs=0), SHAPE), (dict(nb=-1), SHAPE),
    (dict(dt=3), DTYPE), (dict(cache=None), NULL), (dict(slots=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL),
    (dict(cache=P + 4), ALIGN), (dict(k=P + 8), ALIGN), (dict(v=P + 2), ALIGN), (dict(n=0), 0)])
def test_load_argument_checks(lib, kw, rc):
    assert _call(lib.slmt_kv_dequantize_load, LOAD, LOAD_BASE, **kw) == rc


PROMPT = "q qt qh k kt kh v vt vh dt qsl sl r mq n hq kv d sc out odt ot oh err st".split()
PROMPT_BASE = dict(q=P, qt=1024, qh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, dt=0, qsl=P, sl=None, r=2, mq=8,
                   n=9, hq=8, kv=2, d=128, sc=0.1, out=P, odt=2, ot=1024, oh=128, err=None, st=None)


@pytest.mark.parametrize("kw, rc", [
    (dict(d=96), HEAD_DIM), (dict(hq=9), SHAPE), (dict(kv=0), SHAPE), (dict(r=-1), SHAPE), (dict(mq=-1), SHAPE),
    (dict(n=-1), SHAPE), (dict(hq=258, kv=2), UNSUPPORTED), (dict(dt=2), DTYPE), (dict(odt=3), DTYPE),
    (dict(sc=0.0), SHAPE), (dict(sc=-1.0), SHAPE), (dict(sc=math.inf), SHAPE), (dict(sc=math.nan), SHAPE),
    (dict(sc=3e38), SHAPE),  # its log2 e is not finite
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(out=None), NULL), (dict(qsl=None), NULL),
    (dict(q=P + 2), ALIGN), (dict(k=P + 8), ALIGN), (dict(v=P + 8), ALIGN), (dict(out=P + 4), ALIGN),
    (dict(qt=1028), ALIGN), (dict(kh=130), ALIGN), (dict(vt=257), ALIGN), (dict(ot=1022), ALIGN), (dict(ot=0), SHAPE),
    (dict(oh=0), SHAPE), (dict(r=0), 0), (dict(mq=0), 0), (dict(n=0), 0)])
def test_prompt_attention_argument_checks(lib, kw, rc):
    assert _call(lib.slmt_prompt_attention, PROMPT, PROMPT_BASE, **kw) == rc


def test_host_tensors_are_refused():
    q, k = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(2, 2, 64, dtype=torch.float16)
    i32, i64 = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    cache = torch.zeros(1, 16, 2, 72, dtype=torch.uint8)
    for call in (lambda: kd.kv_rotary(q, k, i64, torch.ones(32)),
                 lambda: kd.kv_rotary_store(q, k, k, i64, torch.ones(32), cache, i64),
                 lambda: kd.kv_dequantize_load(cache, i64),
                 lambda: kd.kv_page_plan(i32, i32[:1], i32.view(1, 2), 16, 2),
                 lambda: kd.kv_prompt_attention(q, k, k, i32, 2)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


# -------------------------------------------------------- rotary frequencies
def test_plain_frequencies():
    freq, a = kd.kv_rotary_inv_freq(80, 500000.0)
    want = torch.tensor([500000.0 ** (-2.0 * i / 80) for i in range(40)], dtype=torch.float64).to(torch.float32)
    assert a == 1.0 and freq.dtype == torch.float32 and torch.equal(freq, want)


def test_linear_and_dynamic_frequencies():
    base, _ = kd.kv_rotary_inv_freq(64)
    freq, a = kd.kv_rotary_inv_freq(64, scaling={"rope_type": "linear", "factor": 4.0})
    assert a == 1.0 and torch.equal(freq, base / 4)  # a power of two: exact
    spec = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048, "seq_len": 2048}
    assert torch.equal(kd.kv_rotary_inv_freq(64, scaling=spec)[0], base)  # within the original length: unchanged
    freq, _ = kd.kv_rotary_inv_freq(64, scaling={**spec, "seq_len": 8192})
    stretched = 10000.0 * (2.0 * 8192 / 2048 - 1.0) ** (64 / 62)
    assert torch.allclose(freq.double(), torch.tensor([stretched ** (-2.0 * i / 64) for i in range(32)],
                                                      dtype=torch.float64), rtol=2.0 ** -23)


@pytest.mark.parametrize("spec", [
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096, "attention_factor": 1.0},
])
def test_banded_frequencies(spec):
    """Fast pairs stay, slow pairs are divided by the factor, monotone between."""
    dim, base = 128, 500000.0
    plain = kd.kv_rotary_inv_freq(dim, base)[0].double()
    freq, a = kd.kv_rotary_inv_freq(dim, base, spec)
    ratio = plain / freq.double()
    turns = spec["original_max_position_embeddings"] * plain / (2 * math.pi)
    fast, slow = (4.0, 1.0) if spec["rope_type"] == "llama3" else (32.0, 1.0)
    tol = 2.0 ** -22
    assert torch.all((ratio[turns > 1.3 * fast] - 1).abs() < tol)
    assert torch.all((ratio[turns < slow / 1.3] / spec["factor"] - 1).abs() < tol)
    assert torch.all(ratio[1:] >= ratio[:-1] * (1 - tol)) and float(ratio.min()) > 1 - tol
    if spec["rope_type"] == "llama3":
        mid = (turns > 1.0) & (turns < 4.0)
        share = (turns[mid] - 1.0) / 3.0
        assert torch.allclose(1 / ratio[mid], share + (1 - share) / 8.0, rtol=2.0 ** -21)
        assert a == 1.0
    else:
        assert a == (spec["attention_factor"] if "attention_factor" in spec else 0.1 * math.log(4.0) + 1.0)


def test_frequencies_equal_transformers():
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import LlamaConfig
    for spec in ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                  "original_max_position_embeddings": 8192},
                 {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096},
                 {"rope_type": "linear", "factor": 3.0}):
        cfg = LlamaConfig(hidden_size=1024, num_attention_heads=8, head_dim=128, max_position_embeddings=32768,
                          rope_parameters={**spec, "rope_theta": 500000.0})
        want, a = rope.ROPE_INIT_FUNCTIONS[spec["rope_type"]](cfg, torch.device("cpu"))
        freq, mine = kd.kv_rotary_inv_freq(128, 500000.0, spec)
        # theirs is a chain of fp32 operations: the power, and up to five more
        assert torch.allclose(freq, want, rtol=16 * 2.0 ** -24) and abs(mine - a) < 1e-12


def test_bad_frequency_requests():
    for args in ((7,), (0,), (64, 0.0), (64, 10000.0, {"rope_type": "linear"}), (64, 10000.0, {"rope_type": "spiral"}),
                 (64, 10000.0, {"rope_type": "llama3", "factor": 8.0}),
                 (64, 10000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
                                "original_max_position_embeddings": 8192}),
                 (64, 1.0, {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 8192})):
        with pytest.raises(RuntimeError):
            kd.kv_rotary_inv_freq(*args)

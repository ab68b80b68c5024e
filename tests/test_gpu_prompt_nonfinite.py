"""GPU: NaN and infinities in V at every head size, and in some of many
requests, whose items follow one another on an SM."""
import math

import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd
from tests.test_gpu_prompt_attention import _inputs, _ref

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev():
    d = torch.device("cuda:0")
    assert kd.read_device_errors(d) == 0
    yield d
    assert kd.read_device_errors(d) == 0


def _expected(v, lens, group):
    """0 where a row's output is finite, else the NaN or the infinity that the
    formula gives: weights are positive, so an infinity attended to stays, and
    a NaN or two infinities of opposite signs are a NaN."""
    n, kv, d = v.shape
    want = torch.zeros(n, kv * group, d, dtype=torch.float64, device=v.device)
    at = 0
    for m in lens:
        x = v[at:at + m].double()
        nan = x.isnan().cumsum(0) > 0
        up, down = (x == math.inf).cumsum(0) > 0, (x == -math.inf).cumsum(0) > 0
        y = torch.zeros_like(x)
        y[up], y[down] = math.inf, -math.inf
        y[nan | (up & down)] = math.nan
        want[at:at + m] = y.repeat_interleave(group, 1)
        at += m
    return want


def _check(got, clean, want):
    fin = want == 0
    assert torch.equal(got[fin], clean[fin])
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf].double(), want[inf])


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_one_bad_value_at_each_place(dev, d, dtype):
    """A bad value on the diagonal, before it and in the last row, in the first
    and last dims, one of each kind.  (Values stay finite elsewhere, so the
    rows that do not attend to them keep their bits.)"""
    lens, hq, kv = [100, 300, 45, 1], 4, 2
    q, k, v, start = _inputs(lens + [30], hq, kv, d, dtype, dev)
    start = start[:5]
    clean = kd.kv_prompt_attention(q, k, v, start, 300, out=torch.zeros(q.shape, device=dev))
    for rows in ([(40, 0, 9, math.nan)], [(100, 1, 0, math.inf)], [(100 + 299, 0, d - 1, -math.inf)],
                 [(313, 1, 3, math.inf), (350, 1, 3, -math.inf)], [(227, 0, 33, math.nan), (228, 1, 63, math.inf)],
                 [(400, 0, d - 1, math.inf), (445, 1, 17, math.nan), (99, 1, d - 16, -math.inf)],
                 [(t, t % 2, (5 * t) % d, math.inf) for t in range(0, 446, 3)]):
        v2 = v.clone()
        for t, h, c, x in rows:
            v2[t, h, c] = x
        v2[446:] = math.nan  # rows of no request
        got = kd.kv_prompt_attention(q, k, v2, start, 300, out=torch.zeros(q.shape, device=dev))
        want = _expected(v2, lens + [30], 2)
        want[446:] = 0
        _check(got, clean, want)


@pytest.mark.parametrize("d, kv", [(64, 4), (80, 4), (128, 4), (64, 1)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_some_of_many_requests_hold_bad_values(dev, d, kv, dtype):
    """Several items per SM: requests with bad values and clean ones follow one
    another in every accumulator; the clean ones keep their bits."""
    lens = [5 + (37 * i * i) % 389 for i in range(160)] + [1, 0, 700, 2]
    hq = 4 * kv
    q, k, v, start = _inputs(lens, hq, kv, d, dtype, dev)
    clean = kd.kv_prompt_attention(q, k, v, start, 700)
    exact, tol = _ref(q, k, v, lens, 1 / math.sqrt(d), torch.float32)
    assert ((clean.double() - exact).abs() <= tol).all()
    v2 = v.clone()
    g = torch.Generator().manual_seed(d)
    first = start.tolist()
    for r, n in enumerate(lens):
        if n and r % 3 == 1:
            for _ in range(3):
                t, h, c = (int(torch.randint(0, x, (1,), generator=g)) for x in (n, kv, d))
                v2[first[r] + t, h, c] = (math.nan, math.inf, -math.inf)[(r // 3) % 3]
    got = kd.kv_prompt_attention(q, k, v2, start, 700)
    _check(got, clean, _expected(v2, lens, 4))


def test_output_in_the_place_of_the_queries(dev):
    """out may be the queries themselves: each row is read by its own item."""
    for d, heads in ((64, (8, 2)), (80, (4, 4)), (128, (16, 1))):
        lens = [300, 5, 0, 129, 700]
        q, k, v, start = _inputs(lens, *heads, d, torch.bfloat16, dev)
        want = kd.kv_prompt_attention(q, k, v, start, 700, out=torch.empty_like(q))
        kd.kv_prompt_attention(q, k, v, start, 700, out=q)
        assert torch.equal(q, want)

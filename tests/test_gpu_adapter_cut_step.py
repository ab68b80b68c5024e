"""GPU: the vLLM impl's device path on a step whose offsets run past its tokens."""
import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd
from tests.helpers import assert_close
from tests.test_gpu_adapter import D, HQ, _expected, _impl, _step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [30, 31, 55, 70])
def test_captured_step_cut_behind_the_actual_tokens(n):
    """A fresh request that is cut keeps its rows' attention."""
    _, impl = _impl()
    dev = torch.device("cuda", torch.cuda.current_device())
    st = _step([(0, 30), (0, 40)], seed=7)
    want = _expected(st)
    md = st["md"]
    for name in ("query_start_loc", "seq_lens", "block_table"):
        setattr(md, name, getattr(md, name).to(dev))
    q, k, v, cache = (st[x].to(dev) for x in ("q", "k", "v", "cache"))
    out = torch.full((n, HQ, D), float("nan"), dtype=torch.float16, device=dev)
    impl._prefill_attention_device(q[:n], k[:n], v[:n], cache, md, out)
    assert kd.read_device_errors(dev) == 0
    assert_close(out.float().cpu().numpy(), want[:n], what="cut step")

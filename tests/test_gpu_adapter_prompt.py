"""GPU: fresh prompts of the vLLM impl go through the packed prompt kernel,
eagerly and in a captured step that is replayed with other lengths."""
from types import SimpleNamespace

import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd
from tests.helpers import assert_close
from tests.test_gpu_adapter import BS, D, HQ, _expected, _impl, _run, _step

pytestmark = pytest.mark.gpu


def _counted(monkeypatch):
    calls = []
    real = kd.kv_prompt_attention

    def counted(*args, **kw):
        calls.append(args[4])
        return real(*args, **kw)

    monkeypatch.setattr(kd, "kv_prompt_attention", counted)
    return calls


@pytest.mark.parametrize("requests, longest", [
    ([(0, 33), (0, 70), (0, 5)], 70), ([(300, 40), (0, 25), (0, 1), (1000, 1), (0, 200)], 200), ([(5, 9), (40, 1)], None)])
def test_one_launch_for_all_fresh_prompts(monkeypatch, requests, longest):
    calls = _counted(monkeypatch)
    _, impl = _impl()
    dev = torch.device("cuda", torch.cuda.current_device())
    st = _step(requests, seed=len(requests))
    got = _run(impl, st, dev)
    assert kd.read_device_errors(dev) == 0
    assert calls == ([] if longest is None else [longest])
    assert_close(got, _expected(st), what="step")


def test_captured_mixed_step_replays_with_other_lengths():
    _, impl = _impl()
    dev = torch.device("cuda", torch.cuda.current_device())
    steps = [_step(r, seed=20) for r in ([(40, 30), (0, 50), (0, 4)], [(0, 60), (90, 8), (0, 16)])]
    width = max(s["bt"].shape[1] for s in steps)
    pool = max(s["cache"].shape[0] for s in steps)
    buf = None
    for s in steps:
        cache = torch.zeros(pool, *s["cache"].shape[1:], dtype=torch.uint8)
        cache[:s["cache"].shape[0]] = s["cache"]
        s["cache"] = cache
        bt = torch.zeros(len(s["requests"]), width, dtype=torch.int32)
        bt[:, :s["bt"].shape[1]] = s["bt"]
        s["bt"] = s["md"].block_table = bt

    def load(s):
        hk, hv, hs = s["hist"]
        buf["cache"].copy_(s["cache"])
        if hs.numel():
            kd.kv_quantize_store(hk.to(dev), hv.to(dev), buf["cache"], hs.to(dev), BS)
        for name in ("q", "k", "v"):
            buf[name].copy_(s[name])
        for name in ("query_start_loc", "seq_lens", "block_table", "slot_mapping"):
            getattr(buf["md"], name).copy_(getattr(s["md"], name))

    s0 = steps[0]
    buf = {n: s0[n].to(dev) for n in ("cache", "q", "k", "v")}
    buf["md"] = SimpleNamespace(**{n: (x.to(dev) if torch.is_tensor(x) else x) for n, x in vars(s0["md"]).items()})
    out = torch.zeros(s0["q"].shape[0], HQ * D, dtype=torch.float16, device=dev)

    def step():
        impl.do_kv_cache_update(None, buf["k"], buf["v"], buf["cache"], buf["md"].slot_mapping)
        impl._prefill_attention(buf["q"], buf["k"], buf["v"], buf["cache"], buf["md"], out.view(-1, HQ, D))

    load(s0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for s in (steps[1], steps[0]):
        load(s)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize(dev)
        assert kd.read_device_errors(dev) == 0
        assert_close(out.float().view(-1, HQ, D).cpu().numpy(), _expected(s), what="replayed step")

"""GPU: causal attention of packed prompts against the formula in 64 bits."""
import math

import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd

pytestmark = pytest.mark.gpu

SEQ_LEN = 8
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture
def dev():
    d = torch.device("cuda:0")
    assert kd.read_device_errors(d) == 0
    yield d
    assert kd.read_device_errors(d) == 0


def _inputs(lens, hq, kv, d, dtype, dev, seed=0, spread=1.0):
    g = torch.Generator(device=dev).manual_seed(seed + sum(lens) + hq + d)
    n = sum(lens)
    q, k, v = (torch.randn(n, h, d, device=dev, generator=g).mul_(s).to(dtype)
               for h, s in ((hq, spread), (kv, 1.0), (kv, 1.0)))
    start = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    return q, k, v, start


def _ref(q, k, v, lens, scale, out_dtype):
    """Output in 64 bits, and how far a kernel may be from it, per element.

    With weights p_j (held in the inputs' 16-bit type for the second product:
    u = its half step), A = sum p_j |v_j|:  the weights' rounding moves the
    output by u A; a score is a sum of D fp32 products, off by at most (D + 4)
    2^-24 B, B = scale * sum |q||k| at its largest over the row, and scales its
    weight and the sum of weights by as much (2 B (D + 4) 2^-24 A); the
    exponential may be 2^-14 off, relative, in both (2 * 2^-14 A); sums of n
    terms in fp32 add 2 n 2^-24 A; weights too small for fp16 (below 2^-24 of
    the largest, which the kernel holds at 1 or more) may vanish: n 2^-24 max|v|;
    the output is rounded once.
    """
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    u = HALF[q.dtype]
    at = 0
    for m in lens:
        if m:
            qs, ks, vs = (t[at:at + m].double().transpose(0, 1) for t in (q, k, v))
            ks, vs = ks.repeat_interleave(group, 0), vs.repeat_interleave(group, 0)
            s = qs @ ks.transpose(1, 2) * scale
            hidden = torch.ones(m, m, dtype=torch.bool, device=q.device).triu(1)
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            o = p @ vs
            a = p @ vs.abs()
            b = (qs.abs() @ ks.abs().transpose(1, 2) * scale).masked_fill(hidden, 0).amax(-1, keepdim=True)
            t = (u + 2 * b * (d + 4) * 2.0 ** -24 + 2 * 2.0 ** -14 + 2 * m * 2.0 ** -24) * a
            t = t + m * 2.0 ** -24 * vs.abs().amax() + HALF[out_dtype] * (o.abs() + t)
            out[at:at + m], tol[at:at + m] = o.transpose(0, 1), t.transpose(0, 1)
        at += m
    return out, tol


def _check(got, want, tol, rows=None):
    if rows is not None:
        got, want, tol = got[rows], want[rows], tol[rows]
    off = (got.double() - want).abs() - tol
    assert (off <= 0).all(), f"{int((off > 0).sum())} of {off.numel()} outside, worst by {float(off.max()):.3e}"


LENS = {"one": [1], "small": [1, 17, 40, 130], "edges": [127, 128, 129, 0, 256, 257, 1, 63, 64, 65],
        "empty": [0, 0, 5, 0], "long": [2049, 3, 700], "many": [(7 * i * i) % 61 for i in range(300)]}
HEADS = [(32, 8, 128), (32, 4, 64), (8, 8, 80), (14, 2, 64), (16, 1, 128), (6, 6, 128), (64, 1, 80), (3, 1, 64),
         (10, 2, 80)]


@pytest.mark.parametrize("name", LENS)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_prompt_attention(dev, name, heads, dtype):
    lens, (hq, kv, d) = LENS[name], heads
    q, k, v, start = _inputs(lens, hq, kv, d, dtype, dev)
    scale = 1.0 / math.sqrt(d)
    out_dtype = torch.float32 if hq % 3 else dtype
    out = kd.kv_prompt_attention(q, k, v, start, max(lens), out=torch.empty(q.shape, dtype=out_dtype, device=dev))
    _check(out, *_ref(q, k, v, lens, scale, out_dtype))


@pytest.mark.parametrize("lens, heads", [([1999, 777, 63], (32, 32, 80)), ([700] * 6 + [5, 90] * 150, (16, 4, 64)),
                                         ([2100, 50, 1500, 1], (16, 16, 128))], ids=["d80", "d64", "d128"])
def test_several_items_of_unequal_length_per_sm(dev, lens, heads):
    """Hundreds of tile pairs of falling length: every one is done, once."""
    hq, kv, d = heads
    q, k, v, start = _inputs(lens, hq, kv, d, torch.bfloat16, dev)
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device=dev)
    kd.kv_prompt_attention(q, k, v, start, max(lens), out=out)
    _check(out, *_ref(q, k, v, lens, 1 / math.sqrt(d), torch.bfloat16))


@pytest.mark.parametrize("hq", [127, 128])
def test_widest_groups(dev, hq):
    lens = [3, 130, 1]
    q, k, v, start = _inputs(lens, hq, 1, 64, torch.bfloat16, dev)
    _check(kd.kv_prompt_attention(q, k, v, start, 130), *_ref(q, k, v, lens, 0.125, torch.float32))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_peaked_scores_and_scales(dev, dtype):
    """Scores of some hundreds (weights from 1 down to 0, maxima that keep
    growing along the row) and a scale of one's own."""
    lens = [600, 77]
    q, k, v, start = _inputs(lens, 4, 2, 128, dtype, dev, spread=8.0)
    k *= torch.linspace(0.2, 3.0, sum(lens), device=dev).to(dtype)[:, None, None]
    for scale in (0.3, 2.0 ** -9):
        got = kd.kv_prompt_attention(q, k, v, start, 600, sm_scale=scale)
        _check(got, *_ref(q, k, v, lens, scale, torch.float32))


@pytest.mark.parametrize("value", [1e30, 3e38])
def test_enormous_scores(dev, value):
    """Scores of up to 1e31: the largest key takes all of the weight."""
    q = torch.zeros(200, 1, 64, device=dev, dtype=torch.bfloat16)
    k, v = torch.zeros_like(q), torch.randn(200, 1, 64, device=dev).bfloat16()
    q[:, 0, 0] = 8.0
    k[:, 0, 0] = torch.linspace(-1, 1, 200, device=dev).mul(value / 64).bfloat16()
    start = torch.tensor([0, 200], dtype=torch.int32, device=dev)
    got = kd.kv_prompt_attention(q, k, v, start, 200)
    s = 8.0 * k[:, 0, 0].double() * 0.125
    p = torch.softmax(s[None].expand(200, 200).masked_fill(torch.ones(200, 200, device=dev).triu(1) > 0, -math.inf), -1)
    want = p @ v[:, 0].double()
    assert ((got[:, 0].double() - want).abs() <= 2.0 ** -8 * (p @ v[:, 0].double().abs()) + 1e-6).all()


def test_equal_scores_and_tiny_weights(dev):
    """Zero queries: plain means of the values seen, over 1500 keys."""
    q, k, v, start = _inputs([1500], 2, 1, 64, torch.float16, dev)
    q.zero_()
    _check(kd.kv_prompt_attention(q, k, v, start, 1500), *_ref(q, k, v, [1500], 0.125, torch.float32))


def test_strided_inputs_and_outputs(dev):
    """Views of one fused projection, [H, N, D] storage, rows at odd offsets."""
    lens, hq, kv, d = [70, 1, 200], 8, 2, 128
    n = sum(lens)
    _, _, _, start = _inputs(lens, 1, 1, 64, torch.float16, dev)
    fused = torch.randn(n, hq + 2 * kv, d, device=dev).half()
    q, k, v = fused[:, :hq], fused[:, hq:hq + kv], fused[:, hq + kv:]
    want, tol = _ref(q, k, v, lens, 1 / math.sqrt(d), torch.float16)
    wide = torch.zeros(n, 2 * hq, d, device=dev, dtype=torch.float16)
    _check(kd.kv_prompt_attention(q, k, v, start, 200, out=wide[:, hq:]), want, tol)
    assert (wide[:, :hq] == 0).all()
    qt, kt, vt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    ot = torch.empty(hq, n, d, dtype=torch.float16, device=dev).transpose(0, 1)
    _check(kd.kv_prompt_attention(qt, kt, vt, start, 200, out=ot), want, tol)
    odd = torch.empty(n * (hq + 2 * kv) * d + 1, dtype=torch.float16, device=dev)[1:].view(n, hq + 2 * kv, d)
    odd.copy_(fused)
    got = kd.kv_prompt_attention(odd[:, :hq], odd[:, hq:hq + kv], odd[:, hq + kv:], start, 200)
    _check(got, *_ref(q, k, v, lens, 1 / math.sqrt(d), torch.float32))
    k1, v1 = k[:, :1].expand(n, kv, d), v[:, :1].expand(n, kv, d)  # one kv head for all
    _check(kd.kv_prompt_attention(q, k1, v1, start, 200), *_ref(q, k1, v1, lens, 1 / math.sqrt(d), torch.float32))


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_output_rows_on_16_bytes(dev, d, out_dtype):
    """Rows that start on 16 bytes but not on 32: the same bits as elsewhere."""
    lens, hq, kv = [70, 1, 200], 4, 2
    q, k, v, start = _inputs(lens, hq, kv, d, torch.bfloat16, dev)
    want = kd.kv_prompt_attention(q, k, v, start, 200, out=torch.empty(q.shape, dtype=out_dtype, device=dev))
    pad = 16 // want.element_size()
    rows = torch.full((sum(lens), hq * d + 2 * pad), 7.5, dtype=out_dtype, device=dev)
    got = rows[:, pad:pad + hq * d].view(-1, hq, d)
    assert got.data_ptr() % 32 == 16
    kd.kv_prompt_attention(q, k, v, start, 200, out=got)
    assert torch.equal(got, want)
    assert (rows[:, :pad] == 7.5).all() and (rows[:, pad + hq * d:] == 7.5).all()


def test_skipped_requests_and_rows_outside(dev):
    """Requests with a cached context, and the padding, are left as they were."""
    lens, hq, kv, d = [30, 5, 129, 1], 4, 2, 64
    q, k, v, start = _inputs(lens + [40], hq, kv, d, torch.bfloat16, dev)
    want, tol = _ref(q, k, v, lens + [40], 0.125, torch.float32)
    out = torch.full(q.shape, 7.5, device=dev)
    seq = torch.tensor([30, 50, 129, 9], dtype=torch.int32, device=dev)
    kd.kv_prompt_attention(q, k, v, start[:5], 129, seq_lens=seq, out=out)
    rows = torch.tensor([True] * 30 + [False] * 5 + [True] * 129 + [False] * 41, device=dev)
    _check(out, want, tol, rows)
    assert (out[~rows] == 7.5).all()


def test_nothing_leaks_from_what_is_not_attended(dev):
    """NaN and infinities in later rows, in other requests and behind the last
    one change nothing, bit for bit, in the rows that do not attend to them;
    the rows that do become what the formula gives."""
    lens, hq, kv, d = [100, 300, 45], 4, 2, 128
    n = sum(lens)
    for dtype in (torch.float16, torch.bfloat16):
        q, k, v, start = _inputs(lens + [35], hq, kv, d, dtype, dev)
        start = start[:4]
        clean = kd.kv_prompt_attention(q, k, v, start, 300, out=torch.zeros(q.shape, device=dev))
        k2, v2 = k.clone(), v.clone()
        k2[n:], v2[n:] = math.nan, math.inf
        v2[100 + 213, 1, 3], v2[100 + 250, 1, 3] = math.inf, -math.inf  # in the middle of the second request
        v2[40, 0, 9] = math.nan
        k2[400, :, 0] = math.nan  # the third request's first row
        got = kd.kv_prompt_attention(q, k2, v2, start, 300, out=torch.zeros(q.shape, device=dev))
        same = torch.ones(q.shape, dtype=torch.bool, device=dev)
        same[313:400, 2:, 3] = False
        same[40:100, :2, 9] = False
        same[400:445] = False
        assert torch.equal(got[same], clean[same])
        assert (got[313:350, 2:, 3] == math.inf).all() and got[350:400, 2:, 3].isnan().all()
        assert got[40:100, :2, 9].isnan().all() and got[400:445].isnan().all()


def test_rows_beyond_the_bound_are_reported(dev):
    q, k, v, start = _inputs([50, 20], 4, 2, 64, torch.float16, dev)
    want, tol = _ref(q, k, v, [50, 20], 0.125, torch.float32)
    out = torch.full(q.shape, 7.5, device=dev)
    kd.kv_prompt_attention(q, k, v, start, 33, out=out)
    assert kd.read_device_errors(dev) == SEQ_LEN
    rows = torch.arange(70, device=dev)
    _check(out, want, tol, (rows < 33) | (rows >= 50))
    assert (out[33:50] == 7.5).all()
    # rows outside the tensors
    out.fill_(7.5)
    kd.kv_prompt_attention(q[:60], k[:60], v[:60], start, 50, out=out[:60])
    assert kd.read_device_errors(dev) == SEQ_LEN and (out[60:] == 7.5).all()
    _check(out, want, tol, rows < 60)


def test_many_requests_and_offsets_beyond_32_bits(dev):
    """5000 requests; q and out of more than 2^31 elements."""
    hq, kv, d = 64, 2, 128
    lens = [(11 * i) % 113 for i in range(5000)]
    n = sum(lens)
    assert n * hq * d > 1 << 31
    q = torch.empty(n, hq, d, dtype=torch.bfloat16, device=dev).normal_()
    k, v = (torch.empty(n, kv, d, dtype=torch.bfloat16, device=dev).normal_() for _ in range(2))
    start = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    out = torch.empty_like(q)
    kd.kv_prompt_attention(q, k, v, start, max(lens), out=out)
    for r in (0, 1, 9, 2047, 2048, 4095, 4096, 4999):
        a, b = int(start[r]), int(start[r + 1])
        if a < b:
            _check(out[a:b], *_ref(q[a:b], k[a:b], v[a:b], [b - a], 1 / math.sqrt(d), torch.bfloat16))


def test_same_call_twice_and_on_two_streams(dev):
    q, k, v, start = _inputs([700, 31, 260], 8, 2, 128, torch.bfloat16, dev)
    first = kd.kv_prompt_attention(q, k, v, start, 700)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs += [kd.kv_prompt_attention(q, k, v, start, 700) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_captured_and_replayed_with_other_lengths(dev):
    q, k, v, start = _inputs([100, 20, 300], 8, 2, 64, torch.float16, dev)
    out = torch.zeros(q.shape, device=dev)
    kd.kv_prompt_attention(q, k, v, start, 420, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kd.kv_prompt_attention(q, k, v, start, 420, out=out)
    for lens in ([100, 20, 300], [1, 0, 419], [420, 0, 0], [7, 7, 7]):
        start.copy_(torch.tensor([0] + lens).cumsum(0))
        out.fill_(7.5)
        graph.replay()
        want, tol = _ref(q, k, v, lens, 0.125, torch.float32)
        _check(out, want, tol, torch.arange(420, device=dev) < sum(lens))
        assert (out[sum(lens):] == 7.5).all()


def test_refusals(dev):
    q, k, v, start = _inputs([5, 6], 4, 2, 64, torch.float16, dev)
    bad = [dict(query=q.float()), dict(key=k.bfloat16()), dict(value=v[:10]), dict(key=k[:, :, :32]),
           dict(key=k[:, :0], value=v[:, :0]), dict(query=q[:, :3]), dict(query_start_loc=start[:0]),
           dict(seq_lens=start[:1]), dict(out=torch.empty(11, 4, 32, device=dev)),
           dict(out=torch.empty(11, 4, 64, device=dev, dtype=torch.float64)), dict(sm_scale=0.0), dict(sm_scale=-1.0),
           dict(sm_scale=math.nan), dict(max_query_len=-1), dict(query_start_loc=start.cpu()),
           dict(out=torch.empty(1, 4, 64, device=dev).expand(11, 4, 64)),
           dict(query=q.clone().requires_grad_()), dict(value=v.clone().requires_grad_())]
    for kw in bad:
        args = dict(query=q, key=k, value=v, query_start_loc=start, max_query_len=6)
        with pytest.raises(RuntimeError):
            kd.kv_prompt_attention(**{**args, **kw})
    assert kd.kv_prompt_attention(q[:0], k[:0], v[:0], start[:1], 0).shape == (0, 4, 64)


# -------------------------------------------------------- the whole step
def test_prompt_step_then_decode_step(dev):
    """A prompt step and a decode step through every operator, as a serving
    loop runs them: page plan, rotary store, prompt attention; then page plan,
    rotary store and paged decode over what the first step stored."""
    from tests.helpers import assert_close
    import oracle
    hq, kv, d, bs = 8, 2, 64, 16
    lens = [37, 16, 120]
    R = len(lens)
    dtype = torch.float16
    g = torch.Generator(device=dev).manual_seed(3)
    freq = kd.kv_rotary_inv_freq(d, device=dev)[0]
    free = torch.randperm(20, device=dev, generator=g).int()
    bt = torch.zeros(R, 10, dtype=torch.int32, device=dev)
    cache = torch.zeros(20, bs, kv, d + 8, dtype=torch.uint8, device=dev)
    n = sum(lens)
    q, k, v, start = _inputs(lens, hq, kv, d, dtype, dev)
    slots, pos, cur = kd.kv_page_plan(start, torch.tensor(lens, device=dev), bt, bs, n, free_blocks=free)
    qr, kr = kd.kv_rotary_store(q, k, v, pos, freq, cache, slots)
    out = kd.kv_prompt_attention(qr, kr, v, start, max(lens))
    _check(out, *_ref(qr, kr, v, lens, 0.125, torch.float32))
    # the cache holds the rotated prompt: what is read back is what the chunked prefill attends to
    q1, k1, v1, start1 = _inputs([1] * R, hq, kv, d, dtype, dev, seed=9)
    seq = torch.tensor([x + 1 for x in lens], dtype=torch.int32, device=dev)
    slots1, pos1, cur1 = kd.kv_page_plan(start1, seq, bt, bs, R, free_blocks=free, free_cursor=cur)
    assert pos1.tolist() == lens and int(cur1 - cur) == sum(x % bs == 0 for x in lens)
    qr1, _ = kd.kv_rotary_store(q1, k1, v1, pos1, freq, cache, slots1, return_key=False)
    out1 = kd.kv_decode_paged_batched(qr1, cache, bt, seq)
    want = oracle.paged_decode(qr1.cpu(), cache.cpu().numpy(), bt.cpu(), seq.cpu(), bs, kv)
    assert_close(out1.cpu().numpy(), want, what="decode after prompt")
    # the same rows through the cache, read back and attended in 64 bits
    for r, x in enumerate(lens):
        p = torch.arange(x + 1, device=dev)
        rows = bt[r].long()[p // bs] * bs + p % bs
        kk, vv = kd.kv_dequantize_load(cache, rows, torch.float32)
        s = torch.einsum("hd,nhd->hn", qr1[r].double(), kk.double().repeat_interleave(hq // kv, 1)) * 0.125
        o = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), vv.double().repeat_interleave(hq // kv, 1))
        assert_close(out1[r].cpu().numpy(), o.cpu().numpy(), what=f"request {r}")


def test_a_wait_that_runs_out_is_reported(dev):
    """The test hook makes one softmax wait run out after 2 ms: every role
    gives up in its own time, nothing hangs, and the next call is right."""
    import time
    from slm_turbo_b200 import _lib
    lib = _lib.load()
    for d, heads in ((128, (8, 2)), (64, (8, 2)), (80, (4, 4))):
        lens = [900, 40, 1, 300]
        q, k, v, start = _inputs(lens, *heads, d, torch.bfloat16, dev)
        torch.cuda.synchronize()
        prev = lib.slmt_set_wait_limit_ns(2_000_000)
        lib.slmt_set_debug_stall(1)
        try:
            t0 = time.perf_counter()
            kd.kv_prompt_attention(q, k, v, start, 900)
            torch.cuda.synchronize()
            took = time.perf_counter() - t0
        finally:
            lib.slmt_set_debug_stall(0)
            lib.slmt_set_wait_limit_ns(prev)
        assert kd.read_device_errors(dev) == 4 and took < 1.0
        _check(kd.kv_prompt_attention(q, k, v, start, 900), *_ref(q, k, v, lens, d ** -0.5, torch.float32))


@pytest.mark.parametrize("d, dtype", [(64, torch.bfloat16), (80, torch.float16), (128, torch.bfloat16)])
def test_a_request_does_not_depend_on_the_batch(dev, d, dtype):
    """The same bits alone, among others, and next to rows of NaN or enormous
    queries (which share its last tile of rows)."""
    lens, (hq, kv) = [77, 300, 5, 513], (8, 2)
    q, k, v, start = _inputs(lens, hq, kv, d, dtype, dev)
    whole = kd.kv_prompt_attention(q, k, v, start, 513)
    for r, n in enumerate(lens):
        a, b = int(start[r]), int(start[r + 1])
        alone = kd.kv_prompt_attention(q[a:b], k[a:b], v[a:b], torch.tensor([0, n], dtype=torch.int32, device=dev), n)
        assert torch.equal(alone, whole[a:b])
        dirty = q.clone()
        dirty[:a], dirty[b:] = math.nan, math.nan
        if r == 1:
            dirty[b:] = 3e4
        got = kd.kv_prompt_attention(dirty, k, v, start, 513)
        assert torch.equal(got[a:b], whole[a:b])

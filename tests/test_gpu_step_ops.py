"""GPU: page plan, rotary, rotary store and dequantize-load against plain
restatements (loops and torch fp64), bit for bit."""
import math

import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd

pytestmark = pytest.mark.gpu

BLOCK_ID, SLOT, SEQ_LEN, FREE_BLOCKS = 1, 2, 8, 32


@pytest.fixture
def dev():
    d = torch.device("cuda:0")
    assert kd.read_device_errors(d) == 0
    yield d
    assert kd.read_device_errors(d) == 0


# ------------------------------------------------------------------- plan
def _plan_ref(start, seq, tables, bs, n, free, cursor):
    tables = [list(r) for r in tables]
    slots, pos = [-1] * n, [0] * n
    for r, length in enumerate(seq):
        new = start[r + 1] - start[r]
        ctx = length - new
        for b in range(-(-ctx // bs), -(-length // bs)):
            if free is not None:
                tables[r][b] = free[cursor]
                cursor += 1
        for i in range(new):
            p = ctx + i
            slots[start[r] + i] = tables[r][p // bs] * bs + p % bs
            pos[start[r] + i] = p
    return slots, pos, tables, cursor


def _plan_case(requests, bs, seed, pad=0, width_extra=1):
    """requests: (cached, new) pairs."""
    g = torch.Generator().manual_seed(seed)
    seq = [c + n for c, n in requests]
    start = [0]
    for _, n in requests:
        start.append(start[-1] + n)
    need, have = [-(-x // bs) for x in seq], [-(-c // bs) for c, _ in requests]
    perm = torch.randperm(sum(need) + 5, generator=g).tolist()
    width = max(need + [0]) + width_extra
    tables, at = [], 0
    for h in have:
        tables.append(perm[at:at + h] + [-7] * (width - h))
        at += h
    return start, seq, tables, perm[at:], start[-1] + pad


PLAN_CASES = [
    ([(0, 1)], 16, 0), ([(15, 1)], 16, 3), ([(16, 1)], 16, 0), ([(0, 16), (16, 16), (31, 2)], 16, 1),
    ([(5, 0), (0, 0), (7, 9), (0, 33)], 16, 2), ([(100, 1)] * 300, 16, 0), ([(0, 1)] * 2500, 16, 7),
    ([(0, 5000), (3, 1), (0, 4097)], 16, 0), ([(i % 37, i % 5) for i in range(1500)], 32, 11),
    ([(9, 7), (0, 100)], 1, 0), ([(9, 7), (0, 100), (50, 1)], 7, 5), ([], 16, 4),
]


@pytest.mark.parametrize("case", PLAN_CASES, ids=[str(i) for i in range(len(PLAN_CASES))])
@pytest.mark.parametrize("alloc", [True, False])
def test_page_plan(dev, case, alloc):
    requests, bs, pad = case
    start, seq, tables, free, n = _plan_case(requests, bs, seed=len(requests) + bs, pad=pad)
    cursor = 0
    if not alloc:  # complete tables
        _, _, tables, _ = _plan_ref(start, seq, tables, bs, n, free, 0)
    else:
        free, cursor = [9999, 9998] + free, 2
    want_slots, want_pos, want_tables, want_cursor = _plan_ref(start, seq, tables, bs, n, free if alloc else None, cursor)
    width = len(tables[0]) if tables else 3
    bt = torch.tensor(tables, dtype=torch.int32).reshape(len(seq), width).to(dev)
    slots, pos, cur = kd.kv_page_plan(
        torch.tensor(start, dtype=torch.int32, device=dev), torch.tensor(seq, dtype=torch.int32, device=dev), bt, bs, n,
        free_blocks=torch.tensor(free, dtype=torch.int32, device=dev) if alloc else None,
        free_cursor=torch.tensor([cursor], dtype=torch.int32, device=dev) if alloc else None)
    assert slots.tolist() == want_slots and pos.tolist() == want_pos
    assert bt.tolist() == want_tables and cur.item() == want_cursor


def test_page_plan_strided_tables_and_given_outputs(dev):
    start, seq, tables, free, n = _plan_case([(3, 20), (16, 1), (0, 40)], 16, seed=5, pad=6)
    want_slots, want_pos, want_tables, _ = _plan_ref(start, seq, tables, 16, n, free, 0)
    wide = torch.full((3, 40), -3, dtype=torch.int32, device=dev)
    bt = wide[:, 2:2 + len(tables[0])]
    bt.copy_(torch.tensor(tables))
    slots, pos = (torch.full((n,), 77, dtype=torch.int64, device=dev) for _ in range(2))
    a, b, _ = kd.kv_page_plan(torch.tensor(start, device=dev), torch.tensor(seq, device=dev), bt, 16, n,
                              free_blocks=torch.tensor(free, dtype=torch.int32, device=dev), slot_mapping=slots,
                              positions=pos)  # int64 lengths are accepted
    assert a is slots and b is pos and slots.tolist() == want_slots and pos.tolist() == want_pos
    assert bt.tolist() == want_tables
    assert (wide[:, :2] == -3).all() and (wide[:, 2 + len(tables[0]):] == -3).all()


def test_page_plan_reports_what_does_not_fit(dev):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    # a free list of one block for two new pages
    bt = torch.full((2, 4), -1, dtype=torch.int32, device=dev)
    slots, _, cur = kd.kv_page_plan(i32(0, 1, 2), i32(1, 1), bt, 16, 2, free_blocks=i32(5))
    assert slots.tolist() == [80, -1] and bt[:, 0].tolist() == [5, -1] and cur.item() == 1
    assert kd.read_device_errors(dev) == FREE_BLOCKS
    # an empty list
    slots, _, cur = kd.kv_page_plan(i32(0, 1), i32(1), bt[:1], 16, 1, free_blocks=i32())
    assert slots.tolist() == [-1] and cur.item() == 0 and kd.read_device_errors(dev) == FREE_BLOCKS
    # a cursor behind the list
    slots, _, cur = kd.kv_page_plan(i32(0, 1), i32(1), bt[:1], 16, 1, free_blocks=i32(5), free_cursor=i32(3))
    assert slots.tolist() == [-1] and kd.read_device_errors(dev) == FREE_BLOCKS
    # a length beyond the table: the pages that it has are used
    bt = torch.full((1, 2), -1, dtype=torch.int32, device=dev)
    slots, pos, cur = kd.kv_page_plan(i32(0, 40), i32(40), bt, 16, 40, free_blocks=i32(3, 4, 5))
    assert slots.tolist() == [48 + i for i in range(16)] + [64 + i for i in range(16)] + [-1] * 8
    assert cur.item() == 2 and kd.read_device_errors(dev) == SEQ_LEN
    # more rows than tokens: that request gets nothing, its neighbour is served
    bt = torch.tensor([[1], [2]], dtype=torch.int32, device=dev)
    slots, pos, _ = kd.kv_page_plan(i32(0, 3, 5), i32(2, 2), bt, 16, 5)
    assert slots.tolist() == [-1, -1, -1, 32, 33] and kd.read_device_errors(dev) == SEQ_LEN
    # rows beyond num_tokens
    slots, _, _ = kd.kv_page_plan(i32(0, 3), i32(3), bt[:1], 16, 2)
    assert slots.tolist() == [16, 17] and kd.read_device_errors(dev) == SEQ_LEN
    # an entry that names no block
    bt = torch.tensor([[-1]], dtype=torch.int32, device=dev)
    slots, _, _ = kd.kv_page_plan(i32(0, 3), i32(3), bt, 16, 3)
    assert slots.tolist() == [-1] * 3 and kd.read_device_errors(dev) == BLOCK_ID


def test_page_plan_refusals(dev):
    i32 = torch.zeros(3, dtype=torch.int32, device=dev)
    bt = torch.zeros(2, 4, dtype=torch.int32, device=dev)
    for kw in (dict(block_tables=bt.long()), dict(block_tables=bt[:1]), dict(block_tables=bt.t()),
               dict(query_start_loc=i32[:2]), dict(num_tokens=-1), dict(free_blocks=i32.long()),
               dict(free_cursor=i32), dict(slot_mapping=i32), dict(positions=torch.zeros(4, dtype=torch.int64, device=dev)),
               dict(block_size=0), dict(seq_lens=i32[:2].cpu())):
        args = dict(query_start_loc=i32, seq_lens=i32[:2], block_tables=bt, block_size=16, num_tokens=2)
        with pytest.raises(RuntimeError):
            kd.kv_page_plan(**{**args, **kw})


# ----------------------------------------------------------------- rotary
def _rotate_ref(x, pos, freq, interleaved, factor):
    """The formula with every fp32 rounding of the definition (separate torch
    operations do not contract), angles in 64 bits."""
    ang = pos.double()[:, None] * freq.double()[None, :]
    c, s = (torch.cos(ang).float() * factor)[:, None], (torch.sin(ang).float() * factor)[:, None]
    h = freq.numel()
    y = x.float().clone()
    first, second = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    a, b = x.float()[..., first], x.float()[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y.to(x.dtype)


def _rot_case(n, hq, kv, d, rot, dtype, dev, seed=0, far=131072):
    g = torch.Generator(device=dev).manual_seed(seed + n + d + rot)
    q, k, v = (torch.randn(n, h, d, device=dev, generator=g).to(dtype) for h in (hq, kv, kv))
    pos = torch.randint(0, far, (n,), device=dev, generator=g)
    return q, k, v, pos, kd.kv_rotary_inv_freq(rot, 500000.0, device=dev)[0] if rot else torch.empty(0, device=dev)


ROT_CASES = [(1, 32, 8, 128, 128), (5, 4, 4, 64, 64), (33, 14, 2, 80, 80), (130, 3, 1, 128, 32), (7, 8, 2, 80, 70),
             (64, 32, 4, 64, 54), (2, 1, 1, 128, 118), (3, 2, 1, 64, 2), (9, 4, 2, 128, 0), (1001, 5, 5, 128, 64)]


@pytest.mark.parametrize("case", ROT_CASES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_rotary(dev, case, interleaved, dtype):
    q, k, _, pos, freq = _rot_case(*case, dtype, dev)
    factor = 1.0 if case[0] % 2 else 1.1875
    wq, wk = (_rotate_ref(t, pos, freq, interleaved, factor) for t in (q, k))
    gq, gk = kd.kv_rotary(q, k, pos, freq, interleaved, factor)
    assert torch.equal(gq, wq) and torch.equal(gk, wk)
    # in place, 32-bit positions
    kd.kv_rotary(q, k, pos.int(), freq, interleaved, factor, query_out=q, key_out=k)
    assert torch.equal(q, wq) and torch.equal(k, wk)


def test_rotary_views_of_a_fused_projection(dev):
    """q, k, v as slices of one [N, (Hq + 2 KV) * D] tensor, at an odd element
    offset too, rotated in place; v and everything around stay."""
    for off in (0, 1, 8):
        n, hq, kv, d = 37, 8, 2, 128
        store = torch.randn(off + n * (hq + 2 * kv) * d, device=dev).half()
        fused = store[off:].view(n, hq + 2 * kv, d)
        before = fused.clone()
        pos = torch.arange(n, device=dev) * 1000
        freq = kd.kv_rotary_inv_freq(d, device=dev)[0]
        q, k = fused[:, :hq], fused[:, hq:hq + kv]
        kd.kv_rotary(q, k, pos, freq, query_out=q, key_out=k)
        assert torch.equal(q, _rotate_ref(before[:, :hq], pos, freq, False, 1.0))
        assert torch.equal(k, _rotate_ref(before[:, hq:hq + kv], pos, freq, False, 1.0))
        assert torch.equal(fused[:, hq + kv:], before[:, hq + kv:])


def test_rotary_head_strides(dev):
    """[H, N, D] storage (token stride smaller than the head stride)."""
    q, k, _, pos, freq = _rot_case(19, 6, 3, 64, 64, torch.bfloat16, dev)
    qt, kt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k))
    qo = torch.empty(6, 19, 64, dtype=q.dtype, device=dev).transpose(0, 1)
    gq, gk = kd.kv_rotary(qt, kt, pos, freq, query_out=qo)
    assert gq is qo and torch.equal(qo, _rotate_ref(q, pos, freq, False, 1.0))
    assert torch.equal(gk, _rotate_ref(k, pos, freq, False, 1.0))


def test_rotary_turns_back_and_keeps_far_angles(dev):
    """Negative positions undo the turn: y and back is x within the two
    roundings to the type (each eps/2 relative to the pair's length), at
    positions up to 2^28 -- where angles in fp32 would be off by radians."""
    q, k, _, pos, freq = _rot_case(64, 4, 2, 128, 128, torch.float16, dev, far=1 << 28)
    gq, gk = kd.kv_rotary(q, k, pos, freq)
    assert torch.equal(gq, _rotate_ref(q, pos, freq, False, 1.0))
    back, _ = kd.kv_rotary(gq, gk, -pos, freq)
    pair = (q.float()[..., :64] ** 2 + q.float()[..., 64:] ** 2).sqrt().repeat(1, 1, 2)
    # first rounding: both of a pair, turned, at most sqrt(2) half steps; second: one; fp32: 8 steps
    tol = (math.sqrt(2.0) + 1.0) * 2.0 ** -11 * pair + 8 * 2.0 ** -24 * pair + 2.0 ** -24
    assert ((back.float() - q.float()).abs() <= tol).all()


def test_rotary_gradient_is_the_turn_back(dev):
    """d<g, R q>/dq = R^T g = kv_rotary(g, -positions), against autograd of the
    formula in 64 bits: one rounding to the type, eps/2 relative to the pair."""
    q, _, _, pos, freq = _rot_case(9, 2, 1, 64, 64, torch.bfloat16, dev)
    g = torch.randn(q.shape, device=dev).to(q.dtype)
    x = q.double().requires_grad_()
    ang = pos.double()[:, None] * freq.double()[None]
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :32], x[..., 32:]
    torch.cat([a * c - b * s, b * c + a * s], -1).backward(g.double())
    got, _ = kd.kv_rotary(g, g[:, :1], -pos, freq)
    pair = (g.double()[..., :32] ** 2 + g.double()[..., 32:] ** 2).sqrt().repeat(1, 1, 2)
    assert ((got.double() - x.grad).abs() <= (2.0 ** -8 + 8 * 2.0 ** -24) * pair).all()


def test_rotary_passes_special_values(dev):
    """Infinities and NaN stay in their own pair."""
    q, k, _, pos, freq = _rot_case(3, 2, 1, 64, 64, torch.float16, dev)
    q[0, 0, 5], q[1, 1, 40] = math.inf, math.nan
    gq, _ = kd.kv_rotary(q, k, pos, freq)
    want = _rotate_ref(q, pos, freq, False, 1.0)
    assert torch.equal(gq.isnan(), want.isnan()) and torch.equal(gq[~want.isnan()], want[~want.isnan()])


def test_rotary_refusals(dev):
    q, k, v, pos, freq = _rot_case(4, 4, 2, 64, 64, torch.float16, dev)
    for args in ((q, k.bfloat16(), pos, freq), (q[:3], k, pos, freq), (q, k, pos[:3], freq), (q, k, pos.float(), freq),
                 (q, k, pos, freq.half()), (q, k, pos, freq.repeat(2)), (q.float(), k.float(), pos, freq),
                 (q, k, pos, freq.cpu()), (q[..., :62], k[..., :62], pos, freq[:31])):
        with pytest.raises(RuntimeError):
            kd.kv_rotary(*args)
    with pytest.raises(RuntimeError):
        kd.kv_rotary(q, k, pos, freq, query_out=q[:, :2])
    with pytest.raises(RuntimeError):
        kd.kv_rotary(q, k, pos, freq, query_out=torch.empty(1, 4, 64, device=dev).half().expand(4, 4, 64))
    with pytest.raises(RuntimeError, match="backward"):
        kd.kv_rotary(q.detach().clone().requires_grad_(), k, pos, freq)
    with torch.no_grad():
        kd.kv_rotary(q.detach().clone().requires_grad_(), k, pos, freq)
    cache = torch.zeros(2, 16, 2, 72, dtype=torch.uint8, device=dev)
    slots = torch.arange(4, device=dev)
    for kw in (dict(value=v[:, :1]), dict(value=v.bfloat16()), dict(kv_cache=cache[:, :, :1]), dict(slot_mapping=slots[:3]),
               dict(slot_mapping=slots.int()), dict(kv_cache=cache.int()), dict(return_key=False, key_out=k),
               dict(kv_cache=torch.zeros(2, 16, 2, 136, dtype=torch.uint8, device=dev)), dict(slot_mapping=slots.cpu())):
        args = dict(query=q, key=k, value=v, positions=pos, inv_freq=freq, kv_cache=cache, slot_mapping=slots)
        with pytest.raises(RuntimeError):
            kd.kv_rotary_store(**{**args, **kw})
    assert (cache == 0).all()


# ----------------------------------------------------------- rotary + store
@pytest.mark.parametrize("case", ROT_CASES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_rotary_store_is_rotary_then_store(dev, case, interleaved, dtype):
    n, hq, kv, d, rot = case
    q, k, v, pos, freq = _rot_case(*case, dtype, dev)
    k[n // 2] = 0.25  # a constant row (before rotation) and a constant value row
    v[n // 3] = -1.5
    nb = n // 16 + 3
    g = torch.Generator(device=dev).manual_seed(n)
    slots = torch.randperm(nb * 16, device=dev, generator=g)[:n]
    slots[::5] = -1
    fill = torch.randint(0, 256, (nb, 16, kv, d + 8), device=dev, generator=g, dtype=torch.uint8)
    wq, wk = kd.kv_rotary(q, k, pos, freq, interleaved, 1.0)
    want, got = fill.clone(), fill.clone()
    kd.kv_quantize_store(wk, v, want, slots, 16)
    gq, gk = kd.kv_rotary_store(q, k, v, pos, freq, got, slots, interleaved)
    assert torch.equal(gq, wq) and torch.equal(gk, wk) and torch.equal(got, want)
    # in place, the rotated key kept in the cache only
    got = fill.clone()
    q2, none = kd.kv_rotary_store(q, k, v, pos, freq, got, slots, interleaved, query_out=q, return_key=False)
    assert none is None and q2 is q and torch.equal(q, wq) and torch.equal(got, want)


def test_rotary_store_slot_beyond_the_cache(dev):
    q, k, v, pos, freq = _rot_case(3, 4, 2, 64, 64, torch.float16, dev)
    cache = torch.zeros(1, 16, 2, 72, dtype=torch.uint8, device=dev)
    kd.kv_rotary_store(q, k, v, pos, freq, cache, torch.tensor([3, 16, 1 << 40], device=dev))
    assert kd.read_device_errors(dev) == SLOT
    assert (cache[0, :3] == 0).all() and (cache[0, 4:] == 0).all() and (cache[0, 3] != 0).any()


# -------------------------------------------------------------------- load
def _load_ref(cache, slots, dtype):
    d = cache.shape[-1] - 8
    rows = cache.view(-1, *cache.shape[2:])[slots]
    rul = rows[..., d:].contiguous().view(torch.float16).float()
    out = []
    for i in (0, 1):
        half = rows[..., i * d // 2:(i + 1) * d // 2]
        code = torch.stack([half & 15, half >> 4], -1).flatten(-2).float()
        out.append((code * rul[..., 2 * i + 1:2 * i + 2] + rul[..., 2 * i:2 * i + 1]).to(dtype))
    return out


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("n, kv, bs", [(1, 1, 16), (17, 3, 16), (130, 8, 32), (1003, 5, 7)])
def test_load(dev, d, dtype, n, kv, bs):
    nb = n // bs + 2
    k, v = (torch.randn(nb * bs, kv, d, device=dev).half() for _ in range(2))
    cache = torch.zeros(nb, bs, kv, d + 8, dtype=torch.uint8, device=dev)
    kd.kv_quantize_store(k, v, cache, torch.randperm(nb * bs, device=dev), bs)
    slots = torch.randint(0, nb * bs, (n,), device=dev)  # repeats are fine
    slots[n // 2] = -1 if n > 1 else slots[n // 2]
    wk, wv = _load_ref(cache, slots.clamp(min=0), dtype)
    wk[slots < 0], wv[slots < 0] = 0, 0
    gk, gv = kd.kv_dequantize_load(cache, slots, dtype)
    assert torch.equal(gk, wk) and torch.equal(gv, wv)
    ko = torch.full_like(gk, 9)
    assert kd.kv_dequantize_load(cache, slots, dtype, key_out=ko)[0] is ko and torch.equal(ko, wk)


def test_load_bad_slots_and_refusals(dev):
    cache = torch.ones(2, 16, 2, 72, dtype=torch.uint8, device=dev)
    k, v = kd.kv_dequantize_load(cache, torch.tensor([32, 1 << 50, -5], device=dev))
    assert kd.read_device_errors(dev) == SLOT and (k == 0).all() and (v == 0).all()
    k, v = kd.kv_dequantize_load(cache, torch.empty(0, dtype=torch.int64, device=dev))
    assert k.shape == (0, 2, 64)
    s = torch.zeros(3, dtype=torch.int64, device=dev)
    for args in ((cache[:, :, :1], s), (cache, s.int()), (cache.int(), s), (cache, s, torch.int32),
                 (cache, s, torch.float64), (torch.zeros(2, 16, 2, 70, dtype=torch.uint8, device=dev), s),
                 (cache, s, torch.float16, torch.zeros(3, 2, 64, device=dev)), (cache, s.cpu())):
        with pytest.raises(RuntimeError):
            kd.kv_dequantize_load(*args)


def test_load_offsets_beyond_32_bits(dev):
    """Rows behind the 2^32nd byte of the pool (35 M slots of 136 bytes)."""
    nb, kv, d = 2_200_000, 1, 128
    cache = torch.zeros(nb, 16, kv, d + 8, dtype=torch.uint8, device=dev)
    slots = torch.tensor([nb * 16 - 1, (1 << 32) // 136 + 1, 0], device=dev)
    q, k, v, pos, freq = _rot_case(3, 1, 1, 128, 128, torch.float16, dev)
    _, wk = kd.kv_rotary_store(q, k, v, pos, freq, cache, slots)
    gk, gv = kd.kv_dequantize_load(cache, slots)
    for got, x in ((gk, wk), (gv, v)):
        x = x.float()
        lo = x.amin(-1, keepdim=True)
        step = (x.amax(-1, keepdim=True) - lo) / 15
        # half a step of the code, the fp16 rulers (15 steps and a minimum off by eps/2 each), one rounding
        tol = step * (0.5 + 15 * 2.0 ** -11) + lo.abs() * 2.0 ** -11 + x.abs() * 2.0 ** -11 + step * 2.0 ** -10
        assert ((got.float() - x).abs() <= tol).all()


# ------------------------------------------------------- streams and graphs
def test_step_ops_on_a_side_stream_and_in_a_graph(dev):
    """plan -> rotary store -> load captured once, replayed with other lengths."""
    n, hq, kv, d, bs = 48, 8, 2, 128, 16
    q, k, v, _, freq = _rot_case(n, hq, kv, d, d, torch.bfloat16, dev)
    start = torch.tensor([0, 20, 21, 40], dtype=torch.int32, device=dev)
    seq = torch.tensor([20, 33, 19], dtype=torch.int32, device=dev)
    free = torch.randperm(12, device=dev).int()
    bt = torch.tensor([[0] * 4, [12, 13, 14, 0], [0] * 4], dtype=torch.int32, device=dev)
    cache = torch.zeros(16, bs, kv, d + 8, dtype=torch.uint8, device=dev)
    qo = torch.empty_like(q)

    def step():
        slots, pos, cur = kd.kv_page_plan(start, seq, bt, bs, n, free_blocks=free)
        kd.kv_rotary_store(q, k, v, pos, freq, cache, slots, query_out=qo, return_key=False)
        return slots, pos, cur, *kd.kv_dequantize_load(cache, slots, torch.bfloat16)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for s0, l0 in (([0, 20, 21, 40], [20, 33, 19]), ([0, 3, 10, 48], [3, 40, 38]), ([0, 0, 1, 1], [0, 47, 0])):
        start.copy_(torch.tensor(s0))
        seq.copy_(torch.tensor(l0))
        bt.copy_(torch.tensor([[0] * 4, [12, 13, 14, 0], [0] * 4]))
        graph.replay()
        got = [t.clone() for t in outs] + [qo.clone(), bt.clone()]
        bt.copy_(torch.tensor([[0] * 4, [12, 13, 14, 0], [0] * 4]))
        want = [*step(), qo, bt]
        for a, b in zip(got, want):
            assert torch.equal(a, b)

"""GPU: rows of NaN, infinities, signed zeros, and steps at the edges of the
quantizer's range.  The rotary store writes the bytes that the store kernel
writes for the same rows, at every head size and pair layout."""
import math

import pytest
import torch

from slm_turbo_b200.kernels import kv_dequant as kd

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev():
    d = torch.device("cuda:0")
    assert kd.read_device_errors(d) == 0
    yield d
    assert kd.read_device_errors(d) == 0


def _special_rows(d, dtype):
    """[rows, d]: each row one thing that a quantizer meets rarely."""
    g = torch.Generator().manual_seed(d)
    rows = []

    def add(fill, **at):
        row = fill.clone() if torch.is_tensor(fill) else torch.full((d,), float(fill))
        for i, x in at.items():
            row[int(i[1:])] = x
        rows.append(row)

    plain = torch.randn(d, generator=g)
    inf, nan = math.inf, math.nan
    add(nan), add(inf), add(-inf), add(0.0), add(-0.0)
    add(plain, i3=nan), add(plain, i0=nan, i7=inf), add(plain, i9=inf), add(plain, i11=-inf)
    add(plain, i1=inf, i2=-inf), add(nan, i5=1.5), add(nan, i5=inf), add(inf, i4=-inf)
    add(plain.abs() + 1, i6=0.0, i20=-0.0), add(plain.abs() + 1, i6=-0.0, i20=0.0)
    add(-plain.abs() - 1, i6=0.0, i20=-0.0), add(-0.0, i30=0.0)
    # the step is (15 - 2^-20) / 15, which rounds to 1 - 2^-24: its mantissa is all ones
    ones = torch.rand(d, generator=g) * 14 + 0.5
    ones[2], ones[d - 1] = 2.0 ** -20, 15.0
    add(ones)
    assert (torch.tensor([15.0]) - 2.0 ** -20).div(15.0).view(torch.int32).item() & 0x7FFFFF == 0x7FFFFF
    # steps of the type's largest and smallest values; the difference may overflow
    big = float(torch.finfo(dtype).max)
    tiny = float(torch.finfo(dtype).smallest_normal) * float(torch.finfo(dtype).eps)
    add(torch.rand(d, generator=g) * 2 - 1, i0=1.0, i1=-1.0)
    rows[-1] = rows[-1] * big
    add(torch.randint(0, 16, (d,), generator=g).float() * tiny)
    if dtype == torch.bfloat16:
        for e in (-126, -100, -61, -60, -59, 58, 59, 60, 61, 64, 100):
            rows.append(torch.rand(d, generator=g) * 15 * 2.0 ** e)
    # values half way between two codes
    rows.append((torch.randint(0, 31, (d,), generator=g).float() * 0.5).index_fill(0, torch.tensor([0]), 0.0)
                .index_fill(0, torch.tensor([1]), 15.0))
    return torch.stack(rows).to(dtype)


def _both(k, v, layout, dev):
    """Caches of the store kernel and of the rotary store (no dim turns)."""
    n, kv, d = k.shape
    nb = n // 16 + 1
    fill = torch.randint(0, 256, (nb, 16, kv, d + 8), dtype=torch.uint8, device=dev)
    slots = torch.arange(n, device=dev)
    want, got = fill.clone(), fill.clone()
    kd.kv_quantize_store(k, v, want, slots, 16)
    kk = k
    if layout == "any":  # rows at an odd element
        store = torch.empty(k.numel() + 1, dtype=k.dtype, device=dev)
        kk = store[1:].view(k.shape)
        kk.copy_(k)
    q = torch.zeros(n, 1, d, dtype=k.dtype, device=dev)
    none = torch.empty(0, device=dev)
    _, ko = kd.kv_rotary_store(q, kk, v, torch.zeros(n, dtype=torch.int64, device=dev), none, got, slots,
                               interleaved=layout == "interleaved")
    return want, got, ko


@pytest.mark.parametrize("layout", ["half", "interleaved", "any"])
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_special_rows_get_the_store_kernels_bytes(dev, dtype, d, layout):
    rows = _special_rows(d, dtype).to(dev)
    r = rows.shape[0]
    # a token's two heads, and its k and v, hold different rows
    k = torch.stack([rows, rows.roll(1, 0)], 1).contiguous()
    v = torch.stack([rows.roll(5, 0), rows.flip(0)], 1).contiguous()
    want, got, _ = _both(k, v, layout, dev)
    bad = (want != got).flatten(0, 1).any(-1).nonzero().tolist()
    assert not bad, f"(token, head) of {r} rows whose bytes differ: {bad}"


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_rows_of_all_sizes_get_the_store_kernels_bytes(dev, dtype, d):
    """Rows of random spread and offset over the type's range: the corrected
    quotient is the divided one, on the bit."""
    g = torch.Generator(device=dev).manual_seed(7 * d)
    n, kv = 4096, 4
    lo, hi = (-20, 12) if dtype == torch.float16 else (-70, 70)
    e = torch.randint(lo, hi, (2, n, kv, 1), device=dev, generator=g)
    shift = torch.randint(-3, 8, (2, n, kv, 1), device=dev, generator=g)
    x = torch.randn(2, n, kv, d, device=dev, generator=g) + shift.float()
    x = (x * torch.exp2(e.float())).to(dtype)
    x = torch.where(x.isfinite(), x, torch.zeros_like(x))
    want, got, _ = _both(x[0].contiguous(), x[1].contiguous(), "half", dev)
    assert torch.equal(want, got)

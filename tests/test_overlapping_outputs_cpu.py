"""CPU: outputs of one call that share memory are refused (their writes would
race); made-up pointers, nothing is launched."""
import pytest

from tests.test_prompt_path_cpu import LOAD, LOAD_BASE, PLAN, PLAN_BASE, P, SHAPE, _call, lib  # noqa: F401

FAR = 1 << 30


@pytest.mark.parametrize("off", [0, 8, 32, -8, -32])
def test_page_plan_slots_and_positions(lib, off):  # noqa: F811
    """5 tokens: 40 bytes each."""
    assert _call(lib.slmt_page_plan, PLAN, PLAN_BASE, slots=FAR, pos=FAR + off) == SHAPE


@pytest.mark.parametrize("dt, size", [(0, 2), (1, 2), (2, 4)])
def test_load_key_and_value(lib, dt, size):  # noqa: F811
    bytes_ = 3 * 8 * 128 * size
    cache = dict(cache=4 * FAR)
    for off in (0, 16, bytes_ - 16, 16 - bytes_):
        assert _call(lib.slmt_kv_dequantize_load, LOAD, LOAD_BASE, k=FAR, v=FAR + off, dt=dt, **cache) == SHAPE


def test_load_outputs_and_the_cache(lib):  # noqa: F811
    """4 blocks of 16 tokens, 8 heads, 136 bytes a row."""
    pool, out = 4 * 16 * 8 * 136, 3 * 8 * 128 * 2
    for off in (0, pool - 16, 16 - out):
        for one, other in (("k", "v"), ("v", "k")):
            kw = {one: FAR + off, other: 4 * FAR}
            assert _call(lib.slmt_kv_dequantize_load, LOAD, LOAD_BASE, cache=FAR, **kw) == SHAPE

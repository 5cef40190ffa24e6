"""Allocations of the calls as torch's own: with its deterministic setting new memory that a call leaves as it is holds NaN, and its profiler lists them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def deterministic():
    kept = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    yield
    torch.use_deterministic_algorithms(kept[0])
    torch.utils.deterministic.fill_uninitialized_memory = kept[1]


def test_deterministic_fill(gpu, deterministic):
    from dscuda_b200 import mla
    codes = torch.zeros(3, 64, mla.FP8_CACHE_ROW_BYTES, dtype=torch.uint8, device=gpu)
    cache = mla.cache_dequantize_fp8(codes, None, 70, 20).view(-1, 576)
    assert bool((cache[70:90] == 0).all())
    assert bool(torch.isnan(cache[:70]).all()) and bool(torch.isnan(cache[90:]).all())


def test_profiler_lists_allocations(gpu):
    from dscuda_b200 import flash
    query, positions = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device=gpu), torch.zeros(1, 4, dtype=torch.int32, device=gpu)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as profiler:
        flash.rope(query, None, positions, [64])
    assert any(event.key == "aten::empty" for event in profiler.key_averages())

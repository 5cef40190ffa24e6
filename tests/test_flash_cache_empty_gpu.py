"""Entries of an append without new tokens have no position, so none outside the cache either: whatever their start is, nothing is written or reported."""
import pytest
import torch

from test_flash_cache_gpu import append_and_compare, filled, normal, tables

pytestmark = pytest.mark.gpu


def test_entries_without_tokens(gpu):
    from dscuda_b200 import flash
    assert flash.device_status(reset=True) == 0
    starts, counts = torch.tensor([-1, 30, -2 ** 31, 2 ** 31 - 1, 64], dtype=torch.int32), torch.tensor([0, 3, 0, -1, 0], dtype=torch.int32)
    table = tables(5, 2, 12, 1)
    table[0], table[4] = -1, 99
    append_and_compare(gpu, filled(torch.int8, 12, 2, 32, 2), normal(3, 5, 4, 2, 128), normal(4, 5, 4, 2, 128), table, starts, counts)
    assert flash.device_status(reset=True) == 0


def test_a_start_in_front_of_the_cache_is_still_reported(gpu):
    from dscuda_b200 import flash
    append_and_compare(gpu, filled(torch.int8, 12, 2, 32, 5), normal(6, 2, 4, 2, 128), normal(7, 2, 4, 2, 128), tables(2, 2, 12, 8), torch.tensor([-2, 5], dtype=torch.int32), None)
    assert flash.device_status(reset=True) == 3

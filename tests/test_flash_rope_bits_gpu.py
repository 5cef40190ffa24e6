"""Rotary positions have the bits of their steps: sines and cosines in 64 bits rounded to fp32, two fp32 products and their sum, rounded to bf16.  An 8-bit cache
filled from them then holds the same codes as one filled from the same steps in torch."""
import pytest
import torch

from oracle import flash_oracle as oracle
from test_flash_cache_gpu import filled, same, tables

pytestmark = pytest.mark.gpu


def stepwise(x, positions, sections, restart=False, inverse=False, theta=10000.0):
    half = x.shape[-1] // 2
    frequency = [(axis, theta ** -(j / count if restart else (sum(sections[:axis]) + j) / half)) for axis, count in enumerate(sections) for j in range(count)]
    angle = torch.stack([positions[axis].double() * f for axis, f in frequency], -1)[:, None]
    c, s = torch.cos(angle).float(), torch.sin(angle).float() * (-1.0 if inverse else 1.0)
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * c - b * s, a * s + b * c], -1).bfloat16()


@pytest.mark.parametrize("rows,heads,width,sections,restart,inverse", [
    (2000, 6, 128, [16, 24, 24], False, False), (1500, 3, 128, [64], False, True), (3000, 4, 64, [10, 22], True, False), (16, 40, 128, [31, 33], True, True),
])
def test_bits(gpu, rows, heads, width, sections, restart, inverse):
    from dscuda_b200 import flash
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, heads, width, generator=g).bfloat16()
    positions = torch.randint(0, 40000, (len(sections), rows), generator=g, dtype=torch.int32)
    out, _ = flash.rope(x.to(gpu), None, positions.to(gpu), sections, restart=restart, inverse=inverse)
    assert torch.equal(out.cpu().view(torch.int16), stepwise(x, positions, sections, restart, inverse).view(torch.int16))


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_codes_of_turned_keys(gpu, kind):
    from dscuda_b200 import flash
    batch, tokens, heads, page, sections = 4, 500, 4, 64, [16, 24, 24]
    g = torch.Generator().manual_seed(5)
    key, value = (torch.randn(batch, tokens, heads, 128, generator=g).bfloat16() for _ in range(2))
    positions = torch.randint(0, 30000, (3, batch, tokens), generator=g, dtype=torch.int32)
    cache, table, starts = filled(kind, 40, heads, page, 6), tables(batch, 9, 40, 7), torch.tensor([0, 5, 64, 70], dtype=torch.int32)
    device = [x.to(gpu) for x in cache]
    _, turned = flash.rope(None, key.to(gpu), positions.to(gpu), sections)
    flash.cache_append(*device, turned, value.to(gpu), table.to(gpu), starts.to(gpu))
    plain = stepwise(key.view(-1, heads, 128), positions.view(3, -1), sections).view(key.shape)
    oracle.append(cache[0], cache[2], plain, table, starts, torch.full((batch,), tokens))
    oracle.append(cache[1], cache[3], value, table, starts, torch.full((batch,), tokens))
    for x, y in zip(device, cache):
        assert same(x, y)

"""The 8-bit paged cache: appends against the fp32 steps that define them (equal codes and scales), the decode against attention in
64 bits over the values that the cache holds."""
import math

import pytest
import torch

from oracle import flash_oracle as oracle

pytestmark = pytest.mark.gpu

KINDS = [torch.int8, torch.float8_e4m3fn]
SCALE = 128 ** -0.5


def normal(seed, *shape, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).bfloat16()


def filled(kind, blocks, heads, page, seed):
    """A cache with codes everywhere: what lies behind a sequence must not matter, and must stay."""
    g = torch.Generator().manual_seed(seed)
    top = oracle.LARGEST[kind]
    codes = [(torch.randn(blocks, heads, page, 128, generator=g) * top / 4).clamp(-top, top) for _ in range(2)]
    codes = [x.round().to(torch.int8) if kind == torch.int8 else x.to(kind) for x in codes]
    scales = [torch.rand(blocks, heads, generator=g) * 0.05 + 0.005 for _ in range(2)]
    return [*codes, *scales]


def tables(batch, pages, blocks, seed):
    return torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))[: batch * pages].view(batch, pages).int()


def same(a, b):
    return torch.equal(a.cpu().view(torch.int8) if a.dtype != torch.float32 else a.cpu(), b.view(torch.int8) if b.dtype != torch.float32 else b)


def append_and_compare(gpu, cache, key, value, table, starts, counts):
    from dscuda_b200 import flash
    device = [x.to(gpu) for x in cache]
    flash.cache_append(*device, key.to(gpu), value.to(gpu), table.to(gpu), starts.to(gpu) if starts is not None else None, counts.to(gpu) if counts is not None else None)
    b, t = key.shape[:2]
    s, n = starts if starts is not None else torch.zeros(b), counts if counts is not None else torch.full((b,), t)
    oracle.append(cache[0], cache[2], key, table, s, n)
    oracle.append(cache[1], cache[3], value, table, s, n)
    for x, y in zip(device, cache):
        assert same(x, y)
    return device


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,tokens,heads,page,high", [(1, 1, 1, 16, 0), (5, 1, 3, 64, 200), (3, 7, 2, 32, 90), (2, 130, 4, 64, 70), (2, 300, 1, 128, 130), (1, 65, 2, 16, 15), (2, 200, 2, 144, 10)])
def test_append(gpu, kind, batch, tokens, heads, page, high):
    g = torch.Generator().manual_seed(tokens)
    starts = torch.randint(0, high + 1, (batch,), generator=g).int()
    counts = torch.randint(0, tokens + 1, (batch,), generator=g).int()
    pages = -(-(high + tokens) // page)
    blocks = batch * pages + 2
    for n in (None, counts):
        append_and_compare(gpu, filled(kind, blocks, heads, page, 1), normal(2, batch, tokens, heads, 128, std=3.0), normal(3, batch, tokens, heads, 128),
                           tables(batch, pages, blocks, 4), starts, n)


@pytest.mark.parametrize("kind", KINDS)
def test_appends_in_a_row(gpu, kind):
    """Token by token: a page's scale grows with its values, and its codes are those of the same appends on the host."""
    from dscuda_b200 import flash
    page, heads, steps = 32, 2, 70
    key, value = normal(5, 1, steps, heads, 128), normal(6, 1, steps, heads, 128)
    key[0, 40] *= 20
    table = tables(1, 3, 5, 7)
    host = filled(kind, 5, heads, page, 8)
    device = [x.to(gpu) for x in host]
    for t in range(steps):
        start = torch.tensor([t], dtype=torch.int32)
        flash.cache_append(*device, key[:, t:t + 1].contiguous().to(gpu), value[:, t:t + 1].contiguous().to(gpu), table.to(gpu), start.to(gpu))
        oracle.append(host[0], host[2], key[:, t:t + 1], table, start, torch.ones(1))
        oracle.append(host[1], host[3], value[:, t:t + 1], table, start, torch.ones(1))
    for x, y in zip(device, host):
        assert same(x, y)
    # what the cache holds is near what went in: every growth of the scale costs at most half a code more
    held = oracle.cached(device[1].cpu(), device[3].cpu(), table[0], steps)
    step = device[3].cpu()[table[0].long()].repeat_interleave(page, 0)[:steps, :, None].double()
    error = (held - value[0].double()).abs()
    limit = 4 * step if kind == torch.int8 else 4 * step * 2.0 ** -10 + 2.0 ** -2 * value[0].double().abs()
    assert bool((error <= limit).all())


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_are_not_finite_and_pages_of_zeros(gpu, kind):
    key, value = normal(9, 1, 40, 2, 128), normal(10, 1, 40, 2, 128)
    key[0, 3, 0, 5], key[0, 4, 0, 6], key[0, 5, 0, 7] = math.inf, -math.inf, math.nan
    value[0, :32] = 0.0
    value[0, 33, 1] = 2.0 ** -110
    value[0, 34:, 1] = 0.0
    key[0, 32:, 1] = math.inf
    append_and_compare(gpu, filled(kind, 4, 2, 32, 11), key, value, tables(1, 2, 4, 12), None, None)


def test_parts_of_a_projection(gpu):
    from dscuda_b200 import flash
    b, t, heads = 2, 9, 3
    fused = normal(13, b, t, 4 * heads * 128).to(gpu)
    key, value = fused[..., heads * 128:2 * heads * 128].view(b, t, heads, 128), fused[..., 3 * heads * 128:].view(b, t, heads, 128)
    table = tables(b, 1, 4, 14).to(gpu)
    caches = [[x.to(gpu) for x in filled(torch.int8, 4, heads, 16, 15)] for _ in range(2)]
    flash.cache_append(*caches[0], key, value, table)
    flash.cache_append(*caches[1], key.contiguous(), value.contiguous(), table)
    for x, y in zip(*caches):
        assert torch.equal(x, y)


def test_append_outside_the_cache(gpu):
    """Positions in front of and behind the cache and page numbers outside it are left out and raise status 3."""
    from dscuda_b200 import flash
    table = tables(4, 2, 10, 16)
    table[1, 0], table[2, 1] = 10, -1
    starts = torch.tensor([20, 0, 0, -5], dtype=torch.int32)
    append_and_compare(gpu, filled(torch.int8, 10, 2, 16, 17), normal(18, 4, 30, 2, 128), normal(19, 4, 30, 2, 128), table, starts, None)
    assert flash.device_status(reset=True) == 3
    assert flash.device_status() == 0


def decode_and_compare(gpu, kind, lengths, tokens, hq, hkv, page, seed, pages=None, std=1.0):
    from dscuda_b200 import flash
    batch = len(lengths)
    pages = pages or max(1, -(-max(lengths) // page))
    blocks = batch * pages + 1
    cache = filled(kind, blocks, hkv, page, seed)
    if kind == torch.float8_e4m3fn:
        # stale codes behind a sequence's end: NaN
        table = tables(batch, pages, blocks, seed + 1)
        for b, n in enumerate(lengths):
            if 0 < n < pages * page and n % page:
                cache[1].view(torch.uint8)[table[b, n // page], :, n % page:] = 0x7f
                cache[0].view(torch.uint8)[table[b, n // page], :, n % page:] = 0x7f
    table = tables(batch, pages, blocks, seed + 1)
    query = normal(seed + 2, batch, tokens, hq, 128, std=std)
    device = [x.to(gpu) for x in cache]
    out, lse = flash.decode(query.to(gpu), *device, table.to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu), SCALE)
    torch.cuda.synchronize()
    for b, n in enumerate(lengths):
        n = min(max(n, 0), pages * page)
        limits = (n - tokens + 1 + torch.arange(tokens)).clamp(min=0)
        keys, values = oracle.cached(cache[0], cache[2], table[b], n).to(gpu), oracle.cached(cache[1], cache[3], table[b], n).to(gpu)
        r_out, r_lse, out_slack, lse_slack = oracle.attention(query[b].to(gpu), keys, values, SCALE, limits, oracle.F16)
        assert bool(((out[b].double() - r_out).abs() <= out_slack).all()), (b, n)
        empty = ~torch.isfinite(r_lse)
        assert torch.equal(lse[b] == -math.inf, empty)
        assert bool(((lse[b].double() - r_lse).abs()[~empty] <= lse_slack[~empty]).all()), (b, n)
    return out, lse


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,tokens,hq,hkv,page", [
    ([1], 1, 1, 1, 16), ([700], 1, 32, 8, 64), ([0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129], 1, 8, 2, 16), ([64, 65, 63, 500], 1, 16, 1, 32),
    ([300, 5, 1, 0], 4, 12, 4, 64), ([1000, 129], 2, 32, 2, 128), ([700, 128, 0, 129, 1, 3000], 8, 32, 2, 64), ([640, 20], 17, 1, 1, 16), ([2000, 33, 256], 5, 24, 2, 32),
    ([513, 64], 64, 4, 1, 128), ([400], 9, 130, 2, 48), ([90, 4000], 8, 28, 4, 64), ([40, 64, 65], 64, 3, 1, 48), ([2500, 17], 3, 5, 5, 144),
])
def test_decode(gpu, kind, lengths, tokens, hq, hkv, page):
    decode_and_compare(gpu, kind, lengths, tokens, hq, hkv, page, 20 + tokens)


def test_decode_long_and_many(gpu):
    decode_and_compare(gpu, torch.int8, [70001], 1, 8, 2, 64, 31)
    decode_and_compare(gpu, torch.float8_e4m3fn, [3 + 37 * i % 900 for i in range(200)], 1, 8, 4, 64, 32)
    decode_and_compare(gpu, torch.int8, [9000] + [0] * 140 + [1] * 20, 1, 4, 4, 32, 33)
    decode_and_compare(gpu, torch.float8_e4m3fn, [5 + 53 * i % 700 for i in range(90)], 5, 16, 4, 32, 34)
    decode_and_compare(gpu, torch.int8, [30000, 0, 70, 15000], 8, 8, 2, 64, 35)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,tokens,hq,hkv,page", [
    # on both sides of the change from whole items to parts (it depends on the keys that a table holds and the number of items)
    ([384, 0], 1, 8, 2, 64), ([400, 0], 1, 8, 2, 16), ([1024 - 7 * i for i in range(48)], 1, 8, 2, 64), ([1040, 0, 3] * 16, 1, 8, 2, 16),
    ([0] * 3 + [512, 500] * 90, 2, 15, 3, 32), ([528, 1, 0] * 60, 1, 12, 3, 16), ([0, 0, 1] * 40, 8, 32, 4, 32), ([0, 100], 64, 6, 1, 32), ([0, 0], 3, 4, 4, 16),
])
def test_whole_items_and_parts(gpu, kind, lengths, tokens, hq, hkv, page):
    decode_and_compare(gpu, kind, lengths, tokens, hq, hkv, page, 60)


def test_lengths_behind_the_table_and_large_queries(gpu):
    decode_and_compare(gpu, torch.int8, [1000, -3], 1, 8, 2, 64, 34, pages=3)
    # sharp softmax, values of Q far from 1 on both sides: the power of two in front of f16
    decode_and_compare(gpu, torch.int8, [333], 2, 8, 2, 64, 35, std=2.0 ** 6)
    decode_and_compare(gpu, torch.int8, [333], 2, 8, 2, 64, 36, std=2.0 ** -40)


def test_scales_of_very_different_sizes(gpu):
    """Pages whose value scales lie 2^12 apart, zero among them."""
    from dscuda_b200 import flash
    cache = filled(torch.int8, 9, 1, 32, 37)
    cache[3][:, 0] = torch.tensor([1e-3, 4.0, 0.0, 1e-3, 2.0, 1e-3, 0.5, 3.0, 1.0])
    table, query = torch.arange(9).view(1, 9).int(), normal(38, 1, 1, 8, 128)
    out, lse = flash.decode(query.to(gpu), *[x.to(gpu) for x in cache], table.to(gpu), torch.tensor([280], dtype=torch.int32, device=gpu), SCALE)
    keys, values = oracle.cached(cache[0], cache[2], table[0], 280), oracle.cached(cache[1], cache[3], table[0], 280)
    r_out, r_lse, out_slack, lse_slack = oracle.attention(query[0], keys, values, SCALE, torch.tensor([280]), oracle.F16)
    assert bool(((out[0].cpu().double() - r_out).abs() <= out_slack).all()) and bool(((lse[0].cpu().double() - r_lse).abs() <= lse_slack).all())


def test_pages_outside_the_cache(gpu):
    """A page number outside the cache is read as page 0 and reported."""
    from dscuda_b200 import flash
    cache = [x.to(gpu) for x in filled(torch.int8, 4, 2, 32, 39)]
    query, lengths = normal(40, 1, 1, 4, 128).to(gpu), torch.tensor([90], dtype=torch.int32, device=gpu)
    bad, good = (torch.tensor([[1, page, 2]], dtype=torch.int32, device=gpu) for page in (99, 0))
    expected = flash.decode(query, *cache, good, lengths, SCALE)
    assert flash.device_status(reset=True) == 0
    actual = flash.decode(query, *cache, bad, lengths, SCALE)
    assert torch.equal(actual[0], expected[0]) and torch.equal(actual[1], expected[1])
    assert flash.device_status(reset=True) == 3


def test_the_same_bits_again_and_given_memory(gpu):
    from dscuda_b200 import flash
    cache = [x.to(gpu) for x in filled(torch.float8_e4m3fn, 70, 4, 64, 41)]
    table = tables(3, 23, 70, 42).to(gpu)
    query, lengths = normal(43, 3, 2, 16, 128).to(gpu), torch.tensor([1400, 3, 700], dtype=torch.int32, device=gpu)
    first = flash.decode(query, *cache, table, lengths, SCALE)
    workspace = flash.decode_workspace(3, 2, 16, 4, gpu).fill_(0xff)
    out, lse = torch.empty_like(query), torch.empty(3, 16, 2, device=gpu)
    flash.decode(query, *cache, table, lengths, SCALE, workspace, out, lse)
    assert torch.equal(first[0], out) and torch.equal(first[1], lse)


def test_refusals(gpu):
    from dscuda_b200 import flash
    cache = [x.to(gpu) for x in filled(torch.int8, 4, 2, 32, 44)]
    table, lengths, query = torch.zeros(1, 2, dtype=torch.int32, device=gpu), torch.tensor([9], dtype=torch.int32, device=gpu), normal(45, 1, 1, 4, 128).to(gpu)
    with pytest.raises(RuntimeError, match="divisible"):
        flash.decode(normal(1, 1, 1, 3, 128).to(gpu), *cache, table, lengths, SCALE)
    with pytest.raises(RuntimeError, match="at most 64"):
        flash.decode(normal(1, 1, 65, 4, 128).to(gpu), *cache, table, lengths, SCALE)
    with pytest.raises(RuntimeError, match="scale"):
        flash.decode(query, *cache, table, lengths, 0.0)
    with pytest.raises(ValueError, match="dtype"):
        flash.decode(query, *cache, table.long(), lengths, SCALE)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        flash.decode(query, *[x.to(gpu) for x in filled(torch.int8, 4, 2, 24, 44)], table, lengths, SCALE)

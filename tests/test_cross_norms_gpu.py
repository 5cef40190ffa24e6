"""Errors of whole heads: cross attention and decode against 64 bits, with the roundings added as independent ones.  A tile left out of a long loop, which the
bounds for single elements cannot tell from roundings, is many times over these (test_norms_cpu.py leaves one out of every shape here)."""
import pytest
import torch

from oracle import flash_oracle as oracle
from test_cross_attention_gpu import SCALE, SHAPES, inputs, run
from test_flash_cache_gpu import KINDS, filled, normal, tables

pytestmark = pytest.mark.gpu

# A head's error is a sum over 128 columns and more, but the error of delta is one for a row: of a single row it is a normal number, 4 deviations of which
# happen once in 16000.  The variances count the largest value of a step, twice the mean square over a binade.
LIMIT = 4.0
NAMES = ("output", "dquery", "dkey", "dvalue")


def counts(b, tk, lengths):
    return [tk] * b if lengths is None else lengths


@pytest.mark.parametrize("b,tq,tk,hq,hkv,lengths", SHAPES)
def test_heads(gpu, b, tq, tk, hq, hkv, lengths):
    x = inputs(gpu, b, tq, tk, hq, hkv)
    results = run(x, lengths)
    expected, variances = oracle.cross_variances(x[3], *x[:3], SCALE, counts(b, tk, lengths))
    found = {name: oracle.deviations(a, e, v) for name, a, e, v in zip(NAMES, (results[0], *results[2:]), expected, variances)}
    assert max(found.values()) <= LIMIT, found


@pytest.mark.parametrize("b,tq,tk,hq,hkv,lengths", [(2, 600, 3, 8, 8, [2, 3]), (30, 700, 4, 8, 8, [2 + i % 3 for i in range(30)]), (2, 512, 1000, 4, 4, [2, 3]), (1, 512, 130, 2, 2, [2])])
def test_few_keys_have_the_error_of_their_roundings(gpu, b, tq, tk, hq, hkv, lengths):
    """With all keys in one tile delta comes from the tile: what is left are the roundings of dS and of the result.  Hundreds of rows to a head: the
    sums are within their variances, where a delta from the rounded output is not (test_norms_cpu.py)."""
    x = inputs(gpu, b, tq, tk, hq, hkv)
    results = run(x, lengths)
    expected, variances = oracle.cross_variances(x[3], *x[:3], SCALE, lengths)
    for i in (1, 2):
        assert oracle.deviations(results[1 + i], expected[i], variances[i]) <= 1.0, NAMES[i]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,tokens,hq,hkv,page", [([700, 1, 0, 130], 1, 32, 8, 64), ([70001], 1, 8, 2, 64), ([9000, 33, 3000], 4, 32, 4, 32), ([30000, 0, 15000], 8, 8, 2, 64),
                                                        ([3 + 37 * i % 900 for i in range(100)], 1, 8, 4, 64), ([5000, 20], 64, 6, 1, 48)])
def test_decode_heads(gpu, kind, lengths, tokens, hq, hkv, page):
    from dscuda_b200 import flash
    pages = -(-max(lengths) // page)
    blocks = len(lengths) * pages + 1
    cache, table, query = filled(kind, blocks, hkv, page, 70), tables(len(lengths), pages, blocks, 71), normal(72, len(lengths), tokens, hq, 128)
    out, _ = flash.decode(query.to(gpu), *[x.to(gpu) for x in cache], table.to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu), SCALE)
    for b, n in enumerate(lengths):
        keys, values = (oracle.cached(cache[i], cache[2 + i], table[b], n).to(gpu) for i in range(2))
        limits = (n - tokens + 1 + torch.arange(tokens)).clamp(min=0)
        expected, variance = oracle.attention_variances(query[b].to(gpu), keys, values, SCALE, limits, oracle.F16)
        assert oracle.deviations(out[b:b + 1], expected[None], variance[None]) <= LIMIT, (b, n)

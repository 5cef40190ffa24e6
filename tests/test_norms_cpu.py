"""What the checks of test_cross_norms_gpu.py tell apart, on the CPU: results with the kernels' roundings pass, results without one tile of a loop do not, and for
few keys a delta from the rounded output does not."""
import pytest
import torch

from oracle import flash_oracle as oracle
from test_cross_attention_gpu import SCALE, SHAPES, inputs
from test_cross_norms_gpu import LIMIT, NAMES, counts

KEY_TILE, ROW_TILE = 128, 64


def one_head(shape):
    """The entry with the most keys and its first key head."""
    b, tq, tk, hq, hkv, lengths = shape
    n = counts(b, tk, lengths)
    entry = max(range(b), key=lambda i: n[i])
    group = hq // hkv
    query, key, value, dout = inputs("cpu", b, tq, tk, hq, hkv)
    return [x[entry:entry + 1, :, :h].contiguous() for x, h in ((query, group), (key, 1), (value, 1), (dout, group))], n[entry]


def emulated(x, n, exact_delta=True):
    """Results with P, dS, O and the results rounded to bf16, from 64 bits; terms(keys, tokens) are the same over parts of the loops."""
    query, key, value, dout = (t[0].double() for t in x)
    group = query.shape[1]
    k, v = key[:n, 0], value[:n, 0]
    rounded = lambda t: t.bfloat16().double()  # noqa: E731
    p, ds = [], []
    for h in range(group):
        weights = torch.softmax(query[:, h] @ k.t() * SCALE, -1)
        dp = dout[:, h] @ v.t()
        delta = (weights * dp).sum(-1, keepdim=True) if exact_delta else (dout[:, h] * rounded(rounded(weights) @ v)).sum(-1, keepdim=True)
        p.append(rounded(weights))
        ds.append(rounded(weights * (dp - delta) * SCALE))

    def terms(keys, tokens):
        out = torch.stack([a[:, keys] @ v[keys] for a in p], 1)
        dq = torch.stack([a[:, keys] @ k[keys] for a in ds], 1)
        dk, dv = torch.zeros(2, *key.shape, dtype=torch.float64)
        dk[:n, 0] = sum(a[tokens].t() @ query[tokens, h] for h, a in enumerate(ds))
        dv[:n, 0] = sum(a[tokens].t() @ dout[tokens, h] for h, a in enumerate(p))
        return [t[None] for t in (out, dq, dk, dv)]
    return terms


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_tile_left_out_is_seen(shape):
    x, n = one_head(shape)
    tokens, group = x[0].shape[1], x[0].shape[2]
    row_tile = ROW_TILE // group
    expected, variances = oracle.cross_variances(x[3], *x[:3], SCALE, [n])
    terms = emulated(x, n, n <= oracle.EXACT_DELTA)
    everything = terms(slice(None), slice(None))
    far = lambda results: [oracle.deviations(a.bfloat16(), e, v) for a, e, v in zip(results, expected, variances)]  # noqa: E731
    assert max(far(everything)) <= LIMIT / 2
    missing = terms(slice(0, KEY_TILE), slice(0, row_tile))
    without = far([a - b for a, b in zip(everything, missing)])
    looked_at = ([0, 1] if n > KEY_TILE else []) + ([2, 3] if tokens > row_tile and n > 1 else [])
    for i in looked_at:
        assert without[i] > LIMIT, (NAMES[i], without[i])


@pytest.mark.parametrize("n,tokens", [(2, 600), (3, 600), (4, 700)])
def test_delta_from_the_rounded_output_is_seen(n, tokens):
    x = inputs("cpu", 1, tokens, n, 1, 1)
    expected, variances = oracle.cross_variances(x[3], *x[:3], SCALE, [n])
    for exact in (True, False):
        results = emulated(x, n, exact)(slice(None), slice(None))
        far = [oracle.deviations(results[i].bfloat16(), expected[i], variances[i]) for i in (1, 2)]
        assert (max(far) <= 1.0) if exact else (min(far) > 1.0), far

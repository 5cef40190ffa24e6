"""Entries that see a single key: its weight is 1 whatever the score, so queries and keys have gradients of exactly zero.  One shape for each
form of the two gradient kernels (whole loops, loops in parts, several tiles to a CTA), entries of one key beside longer ones."""
import pytest
import torch

from oracle import flash_oracle as oracle

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


@pytest.mark.parametrize("b,tq,tk,hq,hkv,lengths", [
    (1, 9, 1, 4, 4, None), (2, 1700, 1, 8, 8, None), (3, 300, 1, 6, 2, [1, 0, 1]), (60, 700, 1, 8, 8, None),
    (3, 77, 333, 6, 2, [333, 1, 128]), (2, 64, 1000, 8, 1, [1000, 1]), (1, 2000, 100, 4, 2, [1]), (2, 1500, 1030, 3, 1, [1, 600]),
    (40, 130, 500, 8, 8, [1 if i % 3 == 0 else (53 * i) % 501 for i in range(40)]), (6, 900, 300, 16, 8, [300, 0, 1, 129, 1, 257]),
    (5, 90, 1100, 12, 12, [1, 0, 1100, 1, 1]),
])
def test_one_key_has_no_gradient(gpu, b, tq, tk, hq, hkv, lengths):
    from dscuda_b200 import flash
    g = torch.Generator().manual_seed(tq + 7 * tk)
    query, key, value, dout = [(torch.randn(b, n, h, 128, generator=g) * s).bfloat16().to(gpu) for n, h, s in ((tq, hq, 1.0), (tk, hkv, 1.0), (tk, hkv, 1.0), (tq, hq, 0.1))]
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=gpu)
    out, lse = flash.cross_forward(query, key, value, SCALE, n)
    grads = flash.cross_backward(dout, out, lse, query, key, value, SCALE, n)
    assert flash.device_status() == 0
    counts = [tk] * b if lengths is None else lengths
    for i, count in enumerate(counts):
        if count == 1:
            assert torch.equal(out[i], value[i, :1].repeat_interleave(hq // hkv, 1).expand(tq, -1, -1)), i
            assert bool((grads[0][i] == 0).all()) and bool((grads[1][i] == 0).all()), i
    # and the others have theirs
    expected, slacks = oracle.cross_gradients(dout, query, key, value, SCALE, counts)
    for actual, wanted, slack in zip(grads, expected, slacks):
        assert bool(((actual.double() - wanted).abs() <= slack).all())

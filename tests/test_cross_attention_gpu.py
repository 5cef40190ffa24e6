"""Cross attention forward and backward against attention in 64 bits, each element within the error its roundings allow."""
import math

import pytest
import torch

from oracle import flash_oracle as oracle

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def inputs(gpu, b, tq, tk, hq, hkv, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed + tq + 7 * tk)
    return [(torch.randn(*shape, generator=g) * s).bfloat16().to(gpu) for shape, s in (((b, tq, hq, 128), std), ((b, tk, hkv, 128), std), ((b, tk, hkv, 128), 1.0), ((b, tq, hq, 128), 0.1))]


def poison(x, lengths, value=math.nan):
    x = x.clone()
    for b, n in enumerate(lengths):
        x[b, n:] = value
    return x


def run(x, lengths):
    from dscuda_b200 import flash
    query, key, value, dout = x
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=query.device)
    out, lse = flash.cross_forward(query, key, value, SCALE, n)
    grads = flash.cross_backward(dout, out, lse, query, key, value, SCALE, n)
    torch.cuda.synchronize()
    assert flash.device_status() == 0
    return out, lse, *grads


def check(x, lengths, results):
    query, key, value, dout = x
    n = [key.shape[1]] * query.shape[0] if lengths is None else [min(max(v, 0), key.shape[1]) for v in lengths]
    out, lse, out_slack, lse_slack = oracle.cross(query, key, value, SCALE, n)
    grads, slacks = oracle.cross_gradients(dout, query, key, value, SCALE, n)
    empty = ~torch.isfinite(lse)
    assert torch.equal(results[1] == -math.inf, empty)
    assert bool(((results[1].double() - lse).abs()[~empty] <= lse_slack[~empty]).all()), "lse"
    for name, actual, expected, slack in zip(("output", "dquery", "dkey", "dvalue"), (results[0], *results[2:]), (out, *grads), (out_slack, *slacks)):
        error = (actual.double() - expected).abs()
        assert bool((error <= slack).all()), (name, float((error / slack.clamp_min(1e-30)).max()))
    for b, count in enumerate(n):
        assert bool((results[3][b, count:] == 0).all()) and bool((results[4][b, count:] == 0).all())


SHAPES = [
    (1, 1, 1, 1, 1, None), (1, 33, 1, 1, 1, None), (2, 1, 300, 8, 2, [300, 7]), (1, 17, 129, 3, 3, None), (3, 77, 333, 6, 2, [333, 0, 128]),
    (2, 130, 257, 5, 1, [257, 200]), (1, 300, 64, 4, 4, [64]), (2, 64, 1000, 8, 1, [1000, 1]), (1, 257, 513, 14, 2, [500]), (2, 100, 140, 64, 1, [139, 3]),
    (1, 50, 90, 33, 1, None), (1, 700, 300, 2, 2, [129]), (4, 9, 65, 16, 4, [0, 64, 65, 63]),
    # few CTAs and long loops: cut into parts, some of them without a tile of the shorter entries
    (1, 40, 3000, 4, 1, [2900]), (3, 20, 2600, 8, 2, [2600, 100, 0]), (1, 2000, 100, 4, 2, None), (2, 1500, 1030, 3, 1, [1030, 600]), (1, 33, 2049, 1, 1, None),
]

# few rows under many keys: CTAs of the key kernel that go over several items
SHAPES += [
    (40, 5, 700, 8, 4, [(97 * i) % 701 for i in range(40)]), (2, 12, 5000, 28, 4, [5000, 2500]), (1, 700, 4850, 8, 8, None), (70, 3, 130, 6, 3, [0, 130, 128, 1, 129] * 14),
    (5, 90, 1100, 12, 12, [0, 0, 0, 0, 1]),
]
# few keys under many rows: CTAs of the query kernel that go over several items
SHAPES += [
    (6, 900, 300, 16, 8, [300, 0, 128, 129, 1, 257]), (3, 4000, 20, 8, 4, [20, 3, 17]), (2, 3000, 1000, 14, 2, [1000, 129]), (40, 130, 500, 8, 8, [(53 * i) % 501 for i in range(40)]),
    (1, 5000, 700, 24, 8, None), (2, 2400, 64, 8, 8, None), (3, 1700, 256, 33, 11, [0, 256, 100]),
]


@pytest.mark.parametrize("b,tq,tk,hq,hkv,lengths", SHAPES)
def test_forward_and_gradients(gpu, b, tq, tk, hq, hkv, lengths):
    x = inputs(gpu, b, tq, tk, hq, hkv)
    check(x, lengths, run(x, lengths))


@pytest.mark.parametrize("b,tq,tk,hq,hkv,lengths", [(2, 1, 300, 8, 2, [290, 7]), (3, 77, 333, 6, 2, [300, 0, 128]), (2, 200, 1000, 8, 1, [999, 1]),
                                                      (2, 20, 2600, 8, 2, [2500, 130]), (40, 5, 700, 8, 4, [(97 * i) % 701 for i in range(40)]), (6, 900, 300, 16, 8, [290, 0, 128, 129, 1, 257])])
def test_padding_is_never_used(gpu, b, tq, tk, hq, hkv, lengths):
    """NaN or infinities behind the lengths: the same bits as zeros there."""
    query, key, value, dout = inputs(gpu, b, tq, tk, hq, hkv)
    clean = run((query, poison(key, lengths, 0.0), poison(value, lengths, 0.0), dout), lengths)
    for bad in (math.nan, math.inf, torch.finfo(torch.bfloat16).min):
        for a, c in zip(run((query, poison(key, lengths, bad), poison(value, lengths, bad), dout), lengths), clean):
            assert torch.equal(a, c)


def test_entries_do_not_see_one_another(gpu):
    """A query, key or gradient that is not finite stays in its entry and head."""
    x = inputs(gpu, 2, 70, 200, 4, 2)
    clean = run(x, None)
    bad = [t.clone() for t in x]
    bad[0][1, 5, 3] = math.nan
    bad[1][1, 150, 1] = math.inf
    bad[3][1, 60, 2] = math.nan
    for a, c in zip(run(bad, None), clean):
        assert torch.equal(a[0], c[0])
    assert bool(torch.isfinite(run(bad, None)[0][1, :, :2].float()).all())


def test_lengths_outside_the_states(gpu):
    x = inputs(gpu, 2, 40, 100, 4, 4)
    for a, c in zip(run(x, [500, -2]), run(x, [100, 0])):
        assert torch.equal(a, c)


def test_sharp_softmax(gpu):
    x = inputs(gpu, 1, 150, 500, 4, 2, std=4.0)
    check(x, [480], run(x, [480]))


def test_the_same_bits_again_and_given_memory(gpu):
    from dscuda_b200 import flash
    query, key, value, dout = inputs(gpu, 2, 90, 700, 8, 2)
    n = torch.tensor([700, 650], dtype=torch.int32, device=gpu)
    first = run((query, key, value, dout), [700, 650])
    out, lse = torch.empty_like(query), torch.empty(2, 8, 90, device=gpu)
    grads = [torch.full_like(t, math.nan) for t in (query, key, value)]
    flash.cross_forward(query, key, value, SCALE, n, flash.cross_forward_workspace(2, 90, 700, 8, 2, gpu).fill_(0xff), out, lse)
    flash.cross_backward(dout, out, lse, query, key, value, SCALE, n, flash.cross_backward_workspace(2, 90, 700, 8, 2, gpu).fill_(0xff), grads)
    for a, c in zip((out, lse, *grads), first):
        assert torch.equal(a, c)


def test_gradients_against_differences(gpu):
    """The slope of <dout, output> along a direction, from the forward in 64 bits."""
    x = inputs(gpu, 2, 35, 150, 6, 2)
    lengths = [150, 99]
    results = run(x, lengths)
    _, slacks = oracle.cross_gradients(x[3], *x[:3], SCALE, lengths)
    step = 2.0 ** -12
    for i in range(3):
        u = torch.randn(x[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(gpu)
        sides = []
        for sign in (1, -1):
            moved = [t.double() for t in x[:3]]
            moved[i] = moved[i] + sign * step * u
            sides.append(float((x[3].double() * oracle.cross(*moved, SCALE, lengths)[0]).sum()))
        slope = (sides[0] - sides[1]) / (2 * step)
        allowed = float((slacks[i] * u.abs()).sum()) + 1e-5 * abs(slope) + 1e-6
        assert abs(float((results[2 + i].double() * u).sum()) - slope) <= allowed


def test_refusals(gpu):
    from dscuda_b200 import flash
    query, key, value, dout = inputs(gpu, 1, 40, 50, 4, 2)
    with pytest.raises(RuntimeError, match="divisible"):
        flash.cross_forward(query[:, :, :3].contiguous(), key, value, SCALE)
    with pytest.raises(RuntimeError, match="scale"):
        flash.cross_forward(query, key, value, -1.0)
    with pytest.raises(RuntimeError, match="64 query heads"):
        flash.cross_forward(torch.zeros(1, 4, 65, 128, device=gpu, dtype=torch.bfloat16), key[:, :, :1].contiguous(), value[:, :, :1].contiguous(), SCALE)
    with pytest.raises(ValueError, match="shape"):
        flash.cross_forward(query, key, value[:, :40].contiguous(), SCALE)
    with pytest.raises(ValueError, match="contiguous"):
        flash.cross_forward(query, key.transpose(1, 2), value, SCALE)
    with pytest.raises(ValueError, match="dtype"):
        flash.cross_forward(query.half(), key, value, SCALE)

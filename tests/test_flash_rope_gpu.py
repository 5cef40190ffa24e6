"""Rotary positions with several axes against the definition in 64 bits."""
import pytest
import torch

from oracle import flash_oracle as oracle

pytestmark = pytest.mark.gpu


def draw(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


def positions(seed, axes, rows, high=100000):
    return torch.randint(-5, high, (axes, rows), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def check(actual, x, pos, *rest, **more):
    expected, slack = oracle.rope_axes(x.cpu(), pos, *rest, **more)
    error = (actual.cpu().double() - expected).abs()
    assert bool((error <= oracle.BF16 * expected.abs() + slack).all()), float((error / (expected.abs() + 1e-9)).max())


@pytest.mark.parametrize("rows,hq,hk,width,sections,restart,inverse", [
    (1, 1, 1, 128, [64], False, False), (1, 40, 1, 64, [32], False, False), (16, 32, 8, 128, [16, 24, 24], False, False), (333, 5, 5, 128, [1, 62, 1], True, False),
    (700, 6, 2, 64, [16, 16], True, True), (77, 28, 4, 128, [10, 20, 30, 4], False, True), (5000, 16, 2, 128, [16, 24, 24], False, False), (3, 130, 7, 128, [31, 33], False, False),
])
def test_matches_definition(gpu, rows, hq, hk, width, sections, restart, inverse):
    from dscuda_b200 import flash
    q, k, pos = draw(1, rows, hq, width), draw(2, rows, hk, width), positions(3, len(sections), rows)
    out_q, out_k = flash.rope(q.to(gpu), k.to(gpu), pos.to(gpu), sections, restart=restart, inverse=inverse)
    check(out_q, q, pos, sections, restart=restart, inverse=inverse)
    check(out_k, k, pos, sections, restart=restart, inverse=inverse)


def test_far_positions_and_another_base(gpu):
    from dscuda_b200 import flash
    q, pos = draw(4, 64, 3, 128), torch.randint(1 << 23, 1 << 24, (2, 64), generator=torch.Generator().manual_seed(5), dtype=torch.int32)
    out, none = flash.rope(q.to(gpu), None, pos.to(gpu), [32, 32], theta=500000.0)
    assert none is None
    check(out, q, pos, [32, 32], theta=500000.0)


def test_parts_of_a_projection_and_in_place(gpu):
    """Queries and keys as views of one tensor, outputs into views of another, and in place: the same bits; what lies between stays."""
    from dscuda_b200 import flash
    b, t, hq, hk = 3, 37, 12, 4
    fused = draw(6, b, t, (hq + 2 * hk) * 128).to(gpu)
    q, k, v = (x.view(b, t, -1, 128) for x in fused.split([hq * 128, hk * 128, hk * 128], -1))
    pos = positions(7, 3, b * t).to(gpu)
    plain = flash.rope(q.contiguous(), k.contiguous(), pos, [20, 22, 22])
    views = flash.rope(q, k, pos.view(3, b, t), [20, 22, 22])
    other = torch.full_like(fused, 7.0)
    into = [x.view(b, t, -1, 128) for x in other.split([hq * 128, hk * 128, hk * 128], -1)]
    given = flash.rope(q, k, pos, [20, 22, 22], query_out=into[0], key_out=into[1])
    assert given[0] is into[0] and bool((into[2] == 7.0).all())
    kept = v.clone()
    flash.rope(q, k, pos, [20, 22, 22], query_out=q, key_out=k)
    for i, inplace in enumerate((q, k)):
        assert torch.equal(plain[i], views[i]) and torch.equal(plain[i], into[i]) and torch.equal(plain[i], inplace)
    assert torch.equal(v, kept)


def test_gradient_is_the_inverse_turn(gpu):
    """<g, rope(x)> = <rope_inverse(g), x> in the definition; the kernel's inverse against differences of the definition's forward."""
    from dscuda_b200 import flash
    rows, h, sections = 9, 2, [24, 40]
    x, g, u, pos = draw(8, rows, h, 128), draw(9, rows, h, 128), draw(10, rows, h, 128), positions(11, 2, rows)
    back, _ = flash.rope(g.to(gpu), None, pos.to(gpu), sections, inverse=True)
    step = 2.0 ** -10
    up, down = (oracle.rope_axes(x.double() + s * step * u.double(), pos, sections)[0] for s in (1, -1))
    slope = float((g.double() * (up - down) / (2 * step)).sum())
    expected, slack = oracle.rope_axes(g, pos, sections, inverse=True)
    allowed = float(((oracle.BF16 * expected.abs() + slack) * u.double().abs()).sum())
    assert abs(float((back.cpu().double() * u.double()).sum()) - slope) <= allowed


def test_refusals(gpu):
    from dscuda_b200 import flash
    q, pos = draw(12, 4, 2, 128).to(gpu), positions(13, 2, 4).to(gpu)
    for sections in ([32, 31], [64, 0], [65, -1], [10, 10, 10, 10, 24]):
        with pytest.raises((ValueError, RuntimeError)):
            flash.rope(q, None, positions(13, len(sections), 4).to(gpu), sections)
    with pytest.raises(RuntimeError, match="head_size"):
        flash.rope(draw(1, 4, 2, 96).to(gpu), None, pos, [24, 24])
    with pytest.raises(ValueError, match="positions"):
        flash.rope(q, None, positions(13, 2, 5).to(gpu), [32, 32])
    with pytest.raises(ValueError):
        flash.rope(q, draw(1, 5, 2, 128).to(gpu), pos, [32, 32])
    with pytest.raises(ValueError, match="contiguous"):
        flash.rope(draw(1, 4, 128, 2).to(gpu).transpose(1, 2), None, pos, [32, 32])

"""The grouped-query operators as a decoder layer runs them: rotary positions, append, decode over the cache, attention to an encoder's
states and its gradients; on other streams, captured and replayed, with a shared workspace."""
import math

import pytest
import torch

from oracle import flash_oracle as oracle

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5
HQ, HKV, PAGE, PAGES, STATES = 12, 3, 48, 6, 140
SECTIONS = (16, 24, 24)


def normal(seed, *shape, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).bfloat16()


class Layer:
    """Buffers of one layer for `batch` conversations, `tokens` new tokens each, and its step."""

    def __init__(self, gpu, kind, batch, tokens, workspace=None, seed=0):
        from dscuda_b200 import flash
        self.kind, self.batch, self.tokens = kind, batch, tokens
        blocks = batch * PAGES + 1
        self.cache = [torch.zeros(blocks, HKV, PAGE, 128, dtype=kind, device=gpu) for _ in range(2)] + [torch.zeros(blocks, HKV, device=gpu) for _ in range(2)]
        self.table = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))[: batch * PAGES].view(batch, PAGES).int().to(gpu)
        self.fused = torch.empty(batch, tokens, HQ + 2 * HKV, 128, dtype=torch.bfloat16, device=gpu)
        self.positions = torch.zeros(3, batch, tokens, dtype=torch.int32, device=gpu)
        self.starts, self.lengths, self.counts = (torch.zeros(batch, dtype=torch.int32, device=gpu) for _ in range(3))
        self.states = [normal(seed + 7 + i, batch, STATES, HKV, 128).to(gpu) for i in range(2)]
        self.state_lengths = torch.tensor([STATES - 37 * b if b < 3 else 0 for b in range(batch)], dtype=torch.int32, device=gpu)
        self.rotated = torch.empty(batch, tokens, HQ, 128, dtype=torch.bfloat16, device=gpu)
        self.out, self.crossed = torch.empty_like(self.rotated), torch.empty_like(self.rotated)
        self.lse, self.crossed_lse = (torch.empty(batch, HQ, tokens, device=gpu) for _ in range(2))
        self.workspace = flash.decode_workspace(batch, tokens, HQ, HKV, gpu) if workspace is None else workspace
        self.cross_workspace = flash.cross_forward_workspace(batch, tokens, STATES, HQ, HKV, gpu)

    def set(self, fused, starts, counts=None):
        self.fused.copy_(fused)
        counts = counts if counts is not None else torch.full((self.batch,), self.tokens)
        self.starts.copy_(starts)
        self.counts.copy_(counts)
        # row t of the query is position length - tokens + t: padded entries count their missing tokens in front
        self.lengths.copy_(starts + self.tokens)
        at = starts[:, None] + torch.arange(self.tokens)
        self.positions.copy_(torch.stack([at, at // 7, at % 7]))

    def step(self):
        from dscuda_b200 import flash
        query, key, value = self.fused.split([HQ, HKV, HKV], 2)
        flash.rope(query, key, self.positions, SECTIONS, query_out=self.rotated, key_out=key)
        flash.cache_append(*self.cache, key, value, self.table, self.starts, self.counts)
        flash.decode(self.rotated, *self.cache, self.table, self.lengths, SCALE, self.workspace, self.out, self.lse)
        flash.cross_forward(self.out, *self.states, SCALE, self.state_lengths, self.cross_workspace, self.crossed, self.crossed_lse)

    def results(self):
        return [t.clone() for t in (self.rotated, *self.cache, self.out, self.lse, self.crossed, self.crossed_lse)]


class Host:
    """The same steps on the CPU, from the kernels' rotated rows where a rounding could go either way."""

    def __init__(self, layer):
        self.cache = [t.cpu() for t in layer.cache]

    def check(self, layer, fused, starts):
        query, key, value = fused.split([HQ, HKV, HKV], 2)
        positions = layer.positions.cpu().view(3, -1)
        turned, slack = oracle.rope_axes(torch.cat([query, key], 2).reshape(-1, HQ + HKV, 128), positions, SECTIONS)
        actual = torch.cat([layer.rotated, layer.fused[:, :, HQ:HQ + HKV]], 2).cpu().view(-1, HQ + HKV, 128)
        assert bool(((actual.double() - turned).abs() <= oracle.BF16 * turned.abs() + (1 + oracle.BF16) * slack).all())
        oracle.append(self.cache[0], self.cache[2], layer.fused[:, :, HQ:HQ + HKV].cpu(), layer.table.cpu(), starts, layer.counts.cpu())
        oracle.append(self.cache[1], self.cache[3], value, layer.table.cpu(), starts, layer.counts.cpu())
        for a, b in zip(layer.cache, self.cache):
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
        for b in range(layer.batch):
            n = int(layer.lengths[b])
            keys, values = (oracle.cached(self.cache[i], self.cache[2 + i], layer.table[b].cpu(), n) for i in range(2))
            limits = (n - layer.tokens + 1 + torch.arange(layer.tokens)).clamp(min=0)
            out, lse, out_slack, lse_slack = oracle.attention(layer.rotated[b].cpu(), keys, values, SCALE, limits, oracle.F16)
            assert bool(((layer.out[b].cpu().double() - out).abs() <= out_slack).all())
            assert bool(((layer.lse[b].cpu().double() - lse).abs() <= lse_slack).all())
        out, lse, out_slack, lse_slack = oracle.cross(layer.out.cpu(), *[t.cpu() for t in layer.states], SCALE, layer.state_lengths.tolist())
        assert bool(((layer.crossed.cpu().double() - out).abs() <= out_slack).all())
        empty = ~torch.isfinite(lse)
        assert torch.equal(layer.crossed_lse.cpu() == -math.inf, empty)
        assert bool(((layer.crossed_lse.cpu().double() - lse).abs()[~empty] <= lse_slack[~empty]).all())


def inputs(step, batch, tokens):
    return normal(100 + step, batch, tokens, HQ + 2 * HKV, 128, std=1.0 + step % 3)


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_prompt_drafts_and_single_tokens(gpu, kind):
    """A prompt of 60 tokens, a draft of 4 of which some are refused, single tokens over the refused ones."""
    from dscuda_b200 import flash
    batch = 4
    prompt = Layer(gpu, kind, batch, 60)
    host = Host(prompt)
    starts = torch.zeros(batch, dtype=torch.int32)
    x = inputs(0, batch, 60)
    prompt.set(x, starts)
    prompt.step()
    host.check(prompt, x, starts)
    held = torch.full((batch,), 60, dtype=torch.int32)
    for step, tokens in enumerate((4, 1, 1, 4, 1), 1):
        layer = Layer(gpu, kind, batch, tokens)
        layer.cache, layer.table, layer.states, layer.state_lengths = prompt.cache, prompt.table, prompt.states, prompt.state_lengths
        x = inputs(step, batch, tokens)
        layer.set(x, held)
        layer.step()
        host.check(layer, x, held)
        held = held + torch.tensor([tokens, max(1, tokens - 1), max(1, tokens - 2), 1], dtype=torch.int32)
    assert flash.device_status() == 0


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_replayed_steps(gpu, kind):
    """One graph, replayed with new tokens and positions in the same buffers, against direct launches on another cache."""
    batch, tokens = 3, 1
    replayed, direct = (Layer(gpu, kind, batch, tokens) for _ in range(2))
    starts = torch.zeros(batch, dtype=torch.int32)
    for layer in (replayed, direct):
        layer.set(inputs(0, batch, tokens), starts)
        layer.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed.step()
    for step in range(1, 56):               # over the end of a page
        starts = starts + torch.tensor([1, 1, step % 2], dtype=torch.int32)
        replayed.set(inputs(step, batch, tokens), starts)
        direct.set(inputs(step, batch, tokens), starts)
        graph.replay()
        direct.step()
        if step % 18 == 1:
            for a, b in zip(replayed.results(), direct.results()):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_graphs_share_a_workspace(gpu):
    """Steps of different sizes, captured with one workspace and replayed in turn."""
    from dscuda_b200 import flash
    workspace = flash.decode_workspace(5, 4, HQ, HKV, gpu)
    layers = [Layer(gpu, torch.int8, 5, 4, workspace), Layer(gpu, torch.int8, 2, 1, workspace, seed=3)]
    alone = [Layer(gpu, torch.int8, 5, 4), Layer(gpu, torch.int8, 2, 1, seed=3)]
    graphs = []
    for i, layer in enumerate(layers):
        for x in (layer, alone[i]):
            x.set(inputs(i, x.batch, x.tokens), torch.full((x.batch,), 130 - 100 * i, dtype=torch.int32))
            x.cache[2].fill_(0.02)
            x.cache[3].fill_(0.02)
            x.step()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            layer.step()
    for step in range(6):
        for i in (0, 1):
            for x in (layers[i], alone[i]):
                x.set(inputs(10 + step, x.batch, x.tokens), torch.full((x.batch,), 131 + step - 100 * i, dtype=torch.int32))
            graphs[i].replay()
            alone[i].step()
    for layer, other in zip(layers, alone):
        for a, b in zip(layer.results(), other.results()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_streams_at_once(gpu):
    """Calls of two streams at the same time, each with its own (or no given) workspace, have the bits of calls in a row."""
    from dscuda_b200 import flash
    b, tk = 2, 900
    cache = [torch.randint(-127, 128, (40, 4, 64, 128), device=gpu, dtype=torch.int8, generator=torch.Generator(gpu).manual_seed(i)) for i in range(2)]
    cache += [torch.full((40, 4), 0.02, device=gpu) for _ in range(2)]
    table = torch.arange(40, device=gpu).view(2, 20).int()
    lengths, n = torch.tensor([1280, 700], device=gpu).int(), torch.tensor([900, 350], device=gpu).int()
    calls = []
    for i in range(2):
        query, key, value = normal(50 + i, b, 3, 16, 128).to(gpu), normal(52 + i, b, tk, 4, 128).to(gpu), normal(54 + i, b, tk, 4, 128).to(gpu)
        wide, dout = normal(56 + i, b, 60, 16, 128).to(gpu), normal(58 + i, b, 60, 16, 128, std=0.1).to(gpu)

        def call(query=query, key=key, value=value, wide=wide, dout=dout):
            results = [*flash.decode(query, *cache, table, lengths, SCALE), *flash.cross_forward(query, key, value, SCALE, n), *flash.cross_forward(wide, key, value, SCALE, n)]
            return results + list(flash.cross_backward(dout, results[4], results[5], wide, key, value, SCALE, n))
        calls.append(call)
    expected = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu) for _ in calls]
    for _ in range(5):
        actual = []
        for stream, call in zip(streams, calls):
            with torch.cuda.stream(stream):
                actual.append(call())
        torch.cuda.synchronize()
        for mine, wanted in zip(actual, expected):
            for a, c in zip(mine, wanted):
                assert torch.equal(a, c)


def test_captured_training_step(gpu):
    """Rotary positions, cross attention and all gradients in one graph, replayed on new values."""
    from dscuda_b200 import flash
    b, t, tk = 2, 70, 300
    make = lambda seed: [normal(seed + i, *shape).to(gpu) for i, shape in enumerate([(b, t, HQ, 128), (b, tk, HKV, 128), (b, tk, HKV, 128), (b, t, HQ, 128)])]
    x, other = make(70), make(80)
    positions = torch.arange(t, device=gpu).int().repeat(3, b, 1)
    n = torch.tensor([300, 0], device=gpu).int()
    kept = []

    def step():
        query = flash.rope(x[0], None, positions, SECTIONS)[0]
        out, lse = flash.cross_forward(query, x[1], x[2], SCALE, n)
        dquery, dkey, dvalue = flash.cross_backward(x[3], out, lse, query, x[1], x[2], SCALE, n)
        flash.rope(dquery, None, positions, SECTIONS, inverse=True, query_out=dquery)
        kept[:] = [out, lse, dquery, dkey, dvalue]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    captured = list(kept)
    for a, c in zip(x, other):
        a.copy_(c)
    n.copy_(torch.tensor([130, 299]))
    graph.replay()
    torch.cuda.synchronize()
    replayed = [t.clone() for t in captured]
    step()
    torch.cuda.synchronize()
    for a, c in zip(replayed, kept):
        assert torch.equal(a, c)
    # against the formula, from the kernel's rotated queries
    query = flash.rope(x[0], None, positions, SECTIONS)[0]
    grads, slacks = oracle.cross_gradients(x[3], query, x[1], x[2], SCALE, [130, 299])
    for a, g, s in zip(kept[3:], grads[1:], slacks[1:]):
        assert bool(((a.double() - g).abs() <= s).all())
    # the query's gradient is turned back: a pair's error is turned with it, and rounded once more
    back, slack = oracle.rope_axes(grads[0].cpu().view(b * t, HQ, 128), positions.cpu().view(3, -1), SECTIONS, inverse=True)
    error = slacks[0].cpu().view(b * t, HQ, 128)
    pair = error[..., :64] + error[..., 64:]
    allowed = torch.cat([pair, pair], -1) * (1 + oracle.BF16) + oracle.BF16 * back.abs() + (1 + oracle.BF16) * slack
    assert bool(((kept[2].cpu().double().view(b * t, HQ, 128) - back).abs() <= allowed).all())


def test_a_page_shared_by_readers(gpu):
    """Two conversations with the same first pages, decoded together, have the bits of each alone."""
    from dscuda_b200 import flash
    cache = [torch.randint(-127, 128, (9, HKV, PAGE, 128), device=gpu, dtype=torch.int8, generator=torch.Generator(gpu).manual_seed(i)) for i in range(2)]
    cache += [torch.rand(9, HKV, device=gpu, generator=torch.Generator(gpu).manual_seed(3)) * 0.05 for _ in range(2)]
    table = torch.tensor([[1, 2, 5], [1, 2, 7], [1, 1, 1]], device=gpu).int()
    query, lengths = normal(90, 3, 1, HQ, 128).to(gpu), torch.tensor([130, 110, 144], device=gpu).int()
    out, lse = flash.decode(query, *cache, table, lengths, SCALE)
    for b in range(3):
        held = [oracle.cached(cache[i].cpu(), cache[2 + i].cpu(), table[b].cpu(), int(lengths[b])) for i in range(2)]
        r_out, r_lse, out_slack, lse_slack = oracle.attention(query[b].cpu(), *held, SCALE, lengths[b:b + 1].cpu(), oracle.F16)
        assert bool(((out[b].cpu().double() - r_out).abs() <= out_slack).all()) and bool(((lse[b].cpu().double() - r_lse).abs() <= lse_slack).all())


@pytest.mark.parametrize("rows", [(17, 1), (9, 2), (3, 10), (8, 4), (1, 33)])
def test_cross_attention_around_the_change_of_kernels(gpu, rows):
    """17 to 33 rows to a key head: blocks of 32 rows of the one kernel, a tile of the other."""
    from dscuda_b200 import flash
    tokens, group = rows
    query, key, value = normal(1, 2, tokens, 2 * group, 128).to(gpu), normal(2, 2, 1111, 2, 128).to(gpu), normal(3, 2, 1111, 2, 128).to(gpu)
    n = [1100, 15]
    out, lse = flash.cross_forward(query, key, value, SCALE, torch.tensor(n, device=gpu).int())
    r_out, r_lse, out_slack, lse_slack = oracle.cross(query, key, value, SCALE, n)
    assert bool(((out.double() - r_out).abs() <= out_slack).all()) and bool(((lse.double() - r_lse).abs() <= lse_slack).all())


def test_cache_of_more_than_four_gigabytes(gpu):
    """Byte offsets behind 2^32: the last blocks of a large cache."""
    from dscuda_b200 import flash
    blocks, page, heads = 36000, 128, 8                     # 4.7 GB for keys and for values
    cache = [torch.zeros(blocks, heads, page, 128, dtype=torch.int8, device=gpu) for _ in range(2)] + [torch.zeros(blocks, heads, device=gpu) for _ in range(2)]
    pages = torch.tensor([[blocks - 1, 3, blocks - 2]], dtype=torch.int32)
    key, value, query = normal(5, 1, 300, heads, 128), normal(6, 1, 300, heads, 128), normal(7, 1, 1, 16, 128)
    flash.cache_append(*cache, key.to(gpu), value.to(gpu), pages.to(gpu))
    out, lse = flash.decode(query.to(gpu), *cache, pages.to(gpu), torch.tensor([300], dtype=torch.int32, device=gpu), SCALE)
    used = pages[0].long().to(gpu)
    small = [t[used].cpu() for t in cache]
    mine = [torch.zeros(3, heads, page, 128, dtype=torch.int8), torch.zeros(3, heads)]
    order = torch.tensor([[0, 1, 2]])
    for i, rows in enumerate((key, value)):
        codes, scales = mine[0].clone(), mine[1].clone()
        oracle.append(codes, scales, rows, order, torch.zeros(1), torch.full((1,), 300))
        assert torch.equal(small[i][:2], codes[:2]) and torch.equal(small[i][2, :, :44], codes[2, :, :44]) and torch.equal(small[2 + i], scales)
    held = [oracle.cached(small[i], small[2 + i], order[0], 300) for i in range(2)]
    r_out, r_lse, out_slack, lse_slack = oracle.attention(query[0], *held, SCALE, torch.tensor([300]), oracle.F16)
    assert bool(((out[0].cpu().double() - r_out).abs() <= out_slack).all()) and bool(((lse[0].cpu().double() - r_lse).abs() <= lse_slack).all())
    for x in cache[:2]:
        assert int(x[4:blocks - 2].count_nonzero()) == 0

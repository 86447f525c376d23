"""Split calls, whose second kernel is let in while the first still runs, right behind kernels that write what they read: lengths, queries,
tables and pages; eagerly, on another stream and in replayed graphs, each answer against attention in 64 bits over what it should have seen."""

import pytest
import torch

import libcertex_b200 as certex

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def expect(q, keys, values, table, n, page, dtype):
    """Out, its bound, lse and its bound for rows of q over the first n tokens each (keys, values: places, kv, d; 64 bits). A score is
    off by (d + 2) 2^-23 of its absolute terms, a weight by that, 2^-21 (exp), t 2^-24 (sums), 2^-16 (two 16-bit parts); twice for a quotient."""
    rows, heads, d = q.shape
    kv = torch.arange(heads, device="cuda") // (heads // keys.shape[1])
    t = torch.arange(n, device="cuda")
    at = table[:, t // page].long() * page + t % page
    k, v = (x.double()[at][:, :, kv].transpose(1, 2) for x in (keys, values))
    x = q.double()
    s = torch.einsum("rhtd,rhd->rht", k, x) * d**-0.5
    terms = torch.einsum("rhtd,rhd->rht", k.abs(), x.abs()) * d**-0.5
    l = torch.logsumexp(s, -1)
    p = torch.exp(s - l[..., None])
    out, size = torch.einsum("rht,rhtd->rhd", p, v), torch.einsum("rht,rhtd->rhd", p, v.abs())
    weight = (d + 2) * 2.0**-23 * terms.amax(-1) + 2.0**-21 + (n + 100) * 2.0**-24 + (0 if dtype == torch.float32 else 2.0**-16)
    off = 2 * weight[..., None] * size + 1.01 * HALF_STEP[dtype] * out.abs() + (2.0**-25 if dtype == torch.float16 else 0)
    return out, off, l, weight + 2.0**-22 * l.abs()


def check(got, want):
    out, off, l, l_off = want
    far = (got[0].double() - out).abs() - off
    assert float(far.max()) <= 0, float(far.max())
    assert bool(((got[1].double() - l).abs() <= l_off).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 40])
@pytest.mark.parametrize("named", [False, True])
def test_split_calls_see_what_was_enqueued_right_before_them(rows, named, dtype):
    """A step writes everything that the attention reads, attends, and spoils it all; rows of one length (a row by itself finds its shares before the
    first kernel has ended) and of several."""
    page, kv, heads, d, pages = 16, 2, 4, 64, 400
    g = torch.Generator(device="cuda").manual_seed(rows)
    sources = [[torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((rows, heads, d), (pages, page, kv, d), (pages, page, kv, d))] for _ in range(3)]
    tables = [torch.stack([torch.randperm(pages, generator=g, device="cuda") for _ in range(rows)]).to(torch.int32) for _ in range(3)]
    keys, values, q = (torch.zeros_like(x) for x in (sources[0][1], sources[0][2], sources[0][0]))
    table = torch.zeros_like(tables[0])
    lengths, to = (torch.zeros(rows, device="cuda", dtype=torch.int32) for _ in range(2))
    cache = certex.PagedCache(keys=keys, values=values)
    big, n = torch.empty(1 << 26, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int32)
    chosen = [torch.zeros_like(x) for x in (q, keys, values, table)]

    def step():
        big.add_(1)  # a long kernel in front
        for x, y in zip((q, keys, values, table), chosen):
            x.copy_(y)
        to.copy_(torch.arange(rows, device="cuda"))
        lengths.copy_(n.expand(rows))
        got = cache.attend(q, table, lengths, row_to_batch=to if named else None, return_lse=True)
        lengths.fill_(1)
        to.fill_(0)
        for x in (q, keys, values, table):
            x.zero_()
        return got

    def choose(i, length):
        for x, y in zip(chosen, (*sources[i], tables[i])):
            x.copy_(y)
        n.fill_(length)
        return expect(sources[i][0], sources[i][1].view(-1, kv, d), sources[i][2].view(-1, kv, d), tables[i], length, page, dtype)

    turns = [(0, 6400), (1, 1), (2, 3000), (1, 6399), (0, 33), (2, 5000)]
    for i, length in turns:
        want = choose(i, length)
        check(step(), want)
    side = torch.cuda.Stream()
    for i, length in turns:
        want = choose(i, length)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        check(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i, length in turns:
        want = choose(i, length)
        for x in got:
            x.fill_(9)
        graph.replay()
        check(got, want)
    assert not cache.faulted()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_sequence_that_grows_in_a_replayed_graph(dtype):
    """One sequence, one new token a replay: the graph moves the length and the position on by itself, turns, appends and attends in shares."""
    page, kv, heads, d, start = 16, 2, 8, 64, 4090
    rotary = certex.Rotary(d)
    g = torch.Generator(device="cuda").manual_seed(0)
    pages = [torch.randn((300, page, kv, d), generator=g, device="cuda").to(dtype) for _ in range(2)]
    cache = certex.PagedCache(keys=pages[0], values=pages[1], rotary=rotary)
    table = torch.randperm(300, generator=g, device="cuda").to(torch.int32)[None]
    new = [torch.randn((12, 1, h, d), generator=g, device="cuda").to(dtype) for h in (heads, kv, kv)]
    q0, k0, v0 = (torch.zeros_like(x[0]) for x in new)
    length = torch.full((1,), start, device="cuda", dtype=torch.int32)
    position = length - 1

    def step():
        position.add_(1)
        length.add_(1)
        q = cache.append(k0, v0, table, position, q=q0)
        return (q, *cache.attend(q, table, length, return_lse=True))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out, lse = step()
    for i in range(12):
        for x, y in zip((q0, k0, v0), new):
            x.copy_(y[i])
        graph.replay()
        turned = rotary(new[0][i], torch.tensor([start + i], device="cuda"))
        assert torch.equal(q, turned)
        place = table[0, (start + i) // page].long(), (start + i) % page
        assert torch.equal(cache.values[place], new[2][i, 0]) and torch.equal(cache.keys[place], rotary(new[1][i], torch.tensor([start + i], device="cuda"))[0])
        check((out, lse), expect(turned, cache.keys.view(-1, kv, d), cache.values.view(-1, kv, d), table, start + i + 1, page, dtype))
    assert int(length) == start + 12 and not cache.faulted()

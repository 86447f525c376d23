"""How the attention over a paged cache is cut into shares: more units than blocks and fewer, rows beyond one pass over the lengths,
units side by side and behind one another, shares that end with their units, one row of everything; every answer against
attention in 64 bits, and no answer dependent on what ran before."""

import pytest
import torch

import libcertex_b200 as certex

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(out, lse, q, keys, values, places):
    """places (rows, heads, most): places of the cache that every query head sees, -1 none; keys, values (places, kv, d). In 64 bits on
    the GPU, as many rows at a time as fit. The bound is that of a score, (d + 2) 2^-23 of its absolute terms, of the weights' sums (t + 100) 2^-24,
    their two 16-bit parts 2^-16 and exp 2^-21, twice for a quotient, and the rounding of the result."""
    heads, d = q.shape[1:]
    kv = torch.arange(heads, device="cuda") // (heads // keys.shape[1])
    step = max(1, int(2e8 / (heads * d * places.shape[2])))
    for r0 in range(0, q.shape[0], step):
        at, x = places[r0 : r0 + step], q[r0 : r0 + step].double()
        k, v = (t[at.clamp(min=0), kv[:, None]].double().masked_fill_((at < 0)[..., None], 0) for t in (keys, values))
        s = torch.einsum("rhtd,rhd->rht", k, x) * d**-0.5
        terms = torch.einsum("rhtd,rhd->rht", k.abs(), x.abs()) * d**-0.5
        s = s.masked_fill(at < 0, -torch.inf)
        l = torch.logsumexp(s, -1)
        p = torch.exp(s - l.clamp(min=-1e300)[..., None])
        want, size = torch.einsum("rht,rhtd->rhd", p, v), torch.einsum("rht,rhtd->rhd", p, v.abs())
        t = out.dtype
        weight = (d + 2) * 2.0**-23 * terms.amax(-1) + 2.0**-21 + (places.shape[2] + 100) * 2.0**-24 + (0 if t == torch.float32 else 2.0**-16)
        off = 2 * weight[..., None] * size + 1.01 * HALF_STEP[t] * want.abs() + (2.0**-25 if t == torch.float16 else 0)
        far = (out[r0 : r0 + step].double() - want).abs() - off
        assert float(far.max()) <= 0, (r0, float(far.max()))
        if lse is not None:
            got = lse[r0 : r0 + step].double()
            assert torch.equal(got == -torch.inf, l == -torch.inf)
            some = l > -torch.inf
            assert bool(((got - l).abs()[some] <= (weight + 2.0**-22 * l.abs())[some]).all())


def make(dtype, pages, page, kv, d, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    keys, values = (torch.randn((pages, page, kv, d), generator=g, device="cuda").to(dtype) for _ in range(2))
    return certex.PagedCache(keys=keys, values=values), keys.view(-1, kv, d), values.view(-1, kv, d), g


def table_places(table, lengths, page, heads, window=None):
    t = torch.arange(max(1, int(lengths.max())), device="cuda")
    at = table.long()[:, (t // page).clamp(max=table.shape[1] - 1)] * page + t % page
    keep = t < lengths[:, None]
    if window:
        keep &= t >= lengths[:, None] - window
    return torch.where(keep, at, -1)[:, None].expand(-1, heads, -1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,kv,heads,d,most", [(130, 8, 16, 32, 900), (300, 4, 4, 64, 1200), (1000, 2, 2, 16, 700), (65, 16, 32, 128, 400), (33, 1, 5, 24, 3000),
                                                  (3, 100, 100, 16, 2000), (2, 500, 500, 8, 900), (1, 1, 1, 64, 9000), (1, 8, 128, 64, 5000), (64, 8, 8, 200, 600)])
def test_ragged_batches(rows, kv, heads, d, most, dtype):
    page = 16
    cache, keys, values, g = make(dtype, 400, page, kv, d, rows)
    table = torch.randint(0, 400, (rows, -(-most // page)), generator=g, device="cuda", dtype=torch.int32)  # pages may be shared
    lengths = (torch.rand(rows, generator=g, device="cuda") ** 3 * most).to(torch.int32)
    lengths[0] = most
    lengths[rows // 3 :: 7] = 0
    lengths[-1] = most if rows < 3 else 1
    q = torch.randn((rows, heads, d), generator=g, device="cuda").to(dtype)
    out, lse = cache.attend(q, table, lengths, return_lse=True)
    check(out, lse, q, keys, values, table_places(table, lengths, page, heads))
    window = most // 3
    out, lse = cache.attend(q, table, lengths, window=window, return_lse=True)
    check(out, lse, q, keys, values, table_places(table, lengths, page, heads, window))
    assert torch.equal(out, cache.attend(q, table, lengths, window=window)) and not cache.faulted()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,kv,heads,d,k", [(40, 8, 64, 64, 600), (111, 8, 8, 32, 512), (111, 8, 8, 32, 513), (148, 2, 8, 16, 1024), (3, 2, 6, 128, 5000), (1, 1, 1, 80, 20_000),
                                               (500, 4, 8, 8, 300), (5, 3, 9, 256, 1500)])
def test_selected_lists(rows, kv, heads, d, k, dtype):
    cache, keys, values, g = make(dtype, 300, 8, kv, d, k)
    q = torch.randn((rows, heads, d), generator=g, device="cuda").to(dtype)
    for lists in {1, kv, heads}:
        at = torch.randint(-300, 2400, (rows, lists, k), generator=g, device="cuda", dtype=torch.int32)
        out, lse = cache.attend_selected(q, at, return_lse=True)
        doubled = out * 2  # a kernel right behind the call sees what it left
        check(out, lse, q, keys, values, at.long().repeat_interleave(heads // lists, 1))
        assert torch.equal(doubled, out * 2)


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_of_all_kinds_in_a_row(dtype):
    """Calls that need workspaces of other sizes, clusters and splits, one behind another without a wait: each answers as it does alone."""
    cache, keys, values, g = make(dtype, 500, 16, 4, 64)
    calls = []
    for rows, most in ((1, 100), (1, 6000), (3, 2500), (40, 300), (200, 900), (1, 8000)):
        table = torch.randint(0, 500, (rows, -(-most // 16)), generator=g, device="cuda", dtype=torch.int32)
        lengths = torch.randint(0, most + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        q = torch.randn((rows, 16, 64), generator=g, device="cuda").to(dtype)
        at = torch.randint(0, 8000, (rows, 16, 700), generator=g, device="cuda")
        calls += [lambda q=q, t=table, n=lengths: cache.attend(q, t, n), lambda q=q, at=at: cache.attend_selected(q, at)]
    alone = []
    for call in calls:
        torch.cuda.synchronize()
        alone.append(call())
    torch.cuda.synchronize()
    for _ in range(3):
        for a, b in zip([call() for call in calls], alone):
            assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [call() for call in calls]
    graph.replay()
    for a, b in zip(captured, alone):
        assert torch.equal(a, b)


def test_the_tables_width_changes_nothing_that_is_seen():
    """The same rows with a table that is far wider than they need: another plan, the same answer to rounding."""
    cache, keys, values, g = make(torch.float32, 300, 16, 2, 64)
    lengths = torch.tensor([100, 0, 257, 16], dtype=torch.int32, device="cuda")
    table = torch.randint(0, 300, (4, 2000), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn((4, 8, 64), generator=g, device="cuda")
    for width in (17, 40, 200, 2000):
        out, lse = cache.attend(q, table[:, :width], lengths, return_lse=True)
        check(out, lse, q, keys, values, table_places(table, lengths, 16, 8))
    assert not cache.faulted()


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_see_what_was_enqueued_right_before_them(dtype):
    """Kernels that are let in before the one in front has ended: fills, copies from and to the host, other streams' work and the library's
    own kernels right before and behind them, eagerly and in a graph; whatever reads early would read the old."""
    rotary = certex.Rotary(64)
    pages = torch.zeros((700, 16, 4, 64), device="cuda").to(dtype)
    cache = certex.PagedCache(keys=pages, values=torch.zeros_like(pages), rotary=rotary)
    g = torch.Generator(device="cuda").manual_seed(4)
    table = torch.arange(700, device="cuda", dtype=torch.int32).view(2, 350)
    source = [torch.randn((2, 4, 64), generator=g, device="cuda").to(dtype) for _ in range(4)]
    big = torch.empty((1 << 26,), device="cuda")
    k, q, lengths, p = (torch.zeros_like(source[0]), torch.zeros((2, 8, 64), device="cuda").to(dtype), torch.zeros(2, dtype=torch.int32, device="cuda"),
                        torch.zeros(2, dtype=torch.int32, device="cuda"))
    side = torch.cuda.Stream()

    def step(i, n):
        big.fill_(float(i))                       # a long kernel in front
        k.copy_(source[i])
        q.copy_(torch.cat([source[i], source[(i + 1) % 4]], 1))
        p.fill_(n - 1)
        r = cache.append(k, k, table, p, q=q)
        k.zero_()
        q.zero_()
        lengths.fill_(n)
        a, lse = cache.attend(r, table, lengths, return_lse=True)   # split: the table is wide
        lengths.fill_(1)
        b = cache.attend(r, table[:, :4], lengths)                   # a cluster
        lengths.fill_(0)
        at = (table[:, :1, None] * 16 + n - 1).expand(2, 8, 3)
        at = torch.where(p[:, None, None] >= 0, table[:, (n - 1) // 16, None, None] * 16 + (n - 1) % 16, at)
        c = cache.attend_selected(r, at.contiguous())
        p.fill_(0)
        t = rotary(r, p, inverse=True)
        r.zero_()
        return a, lse, b, c, t

    def expected(i, n):
        kk, qq = source[i], torch.cat([source[i], source[(i + 1) % 4]], 1)
        pos = torch.full((2,), n - 1, dtype=torch.int32, device="cuda")
        return rotary(qq, pos), kk.repeat_interleave(2, 1)

    def verify(i, n, got):
        turned, values = expected(i, n)
        a, lse, b, c, t = got
        assert torch.equal(t, turned)  # position 0 turns nothing
        # one key, named three times, with equal weights: the sum of three values, 1 / 3 and their product are rounded, 3 * 2^-24, and the result
        off = (c.double() - values.double()).abs() - values.double().abs() * (4 * 2.0**-24 + 1.01 * HALF_STEP[dtype])
        assert float(off.max()) <= 0, float(off.max())
        assert bool(torch.isfinite(a.float()).all()) and bool(torch.isfinite(lse).all())

    for n in (1, 2, 17, 900):
        for i in range(4):
            got = step(i, n)
            torch.cuda.synchronize()
            verify(i, n, got)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        got = step(1, 33)
    side.synchronize()
    verify(1, 33, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(2, 40)
    for _ in range(3):
        for x in got:
            x.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        verify(2, 40, got)
    # the whole attention over what the steps appended, against 64 bits
    n = torch.tensor([900, 900], dtype=torch.int32, device="cuda")
    x = torch.randn((2, 8, 64), generator=g, device="cuda").to(dtype)
    out, lse = cache.attend(x, table, n, return_lse=True)
    check(out, lse, x, cache.keys.view(-1, 4, 64), cache.values.view(-1, 4, 64), table_places(table, n, 16, 8))

"""The paged cache: append against plain indexing, both attentions against the definition in 64 bits on the CPU, at the lengths,
pages, heads, types and masks where they can go wrong; refusals; a decoding loop as it is used, with the exact selection."""

import copy
import ctypes
import io
import math
import pickle
import struct

import pytest
import torch

import libcertex_b200 as certex
from libcertex_b200 import _lib, flashinfer, paged

gpu = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


# ------------------------------------------------------------------------------------------------------------ oracle
def softmax_sum(q, k, v, scale, dtype):
    """One head: q (d), k and v (t, d) in 64 bits. Returns out, lse, and how far the kernel's may be off.

    A score is off by at most (d + 2) steps of 2^-23 (tensor cores may cut instead of rounding) of scale * sum |q_i k_i|, so a
    weight by e = that + 2^-21 (exp of a difference up to 100 that is itself rounded adds 100 * 2^-24) and by 2^-16 where
    16-bit weights are kept as two numbers (8 + 8 bits at least); sums of t terms by t * 2^-24 at most. A quotient of two such
    sums is off by twice that of the mean of |v|, and is rounded once; lse by the scores' and the sum's."""
    if len(k) == 0:
        return torch.zeros_like(q), -math.inf, torch.zeros_like(q), 0.0
    s = (k @ q) * scale
    lse = torch.logsumexp(s, 0)
    p = torch.exp(s - lse)
    out = p @ v
    score = (len(q) + 2) * 2.0**-23 * float(((k.abs() @ q.abs()) * abs(scale)).max())
    weight = score + 2.0**-21 + 100 * 2.0**-24 + len(k) * 2.0**-24 + (2.0**-16 if dtype != torch.float32 else 0)
    off = 2 * weight * (p @ v.abs()) + 1.01 * HALF_STEP[dtype] * out.abs() + (2.0**-25 if dtype == torch.float16 else 0)
    return out, float(lse), off, weight + 2.0**-22 * abs(float(lse))


def check(out, lse, q, cache, places, scale=None):
    """places[i][h]: the (page, place) pairs that row i's query head h sees, or None for a row that is not looked at."""
    heads, d = q.shape[1:]
    keys, values = (t.cpu() if cache.layout == "NHD" else t.cpu().transpose(1, 2) for t in (cache.keys, cache.values))
    q, got, lse = q.cpu().double(), out.cpu(), None if lse is None else lse.cpu()
    for i in range(q.shape[0]):
        for h in range(heads):
            at = places[i][h]
            kv = h // (heads // cache.n_kv_heads)
            k, v = (t[at[:, 0], at[:, 1], kv].double() for t in (keys, values))
            want, l, off, l_off = softmax_sum(q[i, h], k, v, d**-0.5 if scale is None else scale, got.dtype)
            far = (got[i, h].double() - want).abs() - off
            assert float(far.max()) <= 0, (i, h, len(at), float(far.max()), float(off.max()))
            if lse is not None:
                assert (lse[i, h] == -math.inf) if l == -math.inf else abs(float(lse[i, h]) - l) <= l_off, (i, h, float(lse[i, h]), l)


def table_places(cache, table, lengths, to_batch, heads, window=None):
    table, ps = table.cpu().long(), cache.page_size
    rows = []
    for i, n in enumerate(lengths.tolist()):
        b = i if to_batch is None else int(to_batch[i])
        t = torch.arange(max(0, n - window) if window else 0, max(n, 0))
        at = torch.stack([table[b][t // ps], t % ps], 1) if len(t) else torch.zeros((0, 2), dtype=torch.long)
        rows.append([at] * heads)
    return rows


def selected_places(cache, selected, heads):
    at = selected.cpu().long()
    at = at.repeat_interleave(heads // at.shape[1], 1)
    return [[torch.stack([a[a >= 0] // cache.page_size, a[a >= 0] % cache.page_size], 1) for a in row] for row in at]


def make(dtype, sequences, most, page, kv, dim, layout="NHD", seed=0, poison=True):
    """A cache whose pages are dealt in a random order; what no sequence has holds NaN, and so do the places behind a
    sequence's last token that `lengths` will not reach."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = -(-most // page) + 1
    n = sequences * per + 3
    shape = (n, page, kv, dim) if layout == "NHD" else (n, kv, page, dim)
    keys, values = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    keys[..., 3] *= 6
    table = torch.randperm(n, generator=g, device="cuda")[: sequences * per].to(torch.int32).view(sequences, per)
    cache = certex.PagedCache(keys=keys, values=values, layout=layout)
    return cache, table, g


def poison(cache, table, lengths, value=float("nan")):
    """Everything but the first `lengths` tokens of the sequences becomes `value` (NaN, inf)."""
    keep = torch.zeros(cache.n_pages * cache.page_size, dtype=torch.bool, device="cuda")
    for row, n in zip(table, lengths):
        t = torch.arange(n, device="cuda")
        keep[row.long()[t // cache.page_size] * cache.page_size + t % cache.page_size] = True
    keep = keep.view(cache.n_pages, cache.page_size)
    for t in (cache.keys, cache.values):
        t = t if cache.layout == "NHD" else t.transpose(1, 2)
        t[~keep] = value


# ------------------------------------------------------------------------------------------------------------ refusals
def _cache_args(**change):
    f = dict(keys=64, values=64, k0=64, k1=64, k2=64, v0=64, v1=64, v2=64, n_pages=1, page_size=1, kv=1, dim=8, dtype=0, fault=64)
    return paged._CACHE.pack(*{**f, **change}.values())


def test_the_library_refuses_what_it_cannot_read(built_library):
    """Nothing is launched: every one of these is an error before the device is looked at."""
    L, table, rows = built_library, paged._TABLE.pack(64, 1, 1, 1, 0), paged._ROWS.pack(64, 8, 8)
    plan = lambda r=8: paged._ROTARY.pack(64, r, 0, 1.0)  # noqa: E731

    def attend(cache=_cache_args(), table=table, lengths=64, window=0, heads=1, n=1, scale=1.0):
        return L.certexB200PagedAttend(None, cache, table, lengths, window, rows, rows, n, heads, scale, None, None, 0)

    def selected(cache=_cache_args(), at=64, lists=1, k=1, heads=1):
        return L.certexB200PagedAttendSelected(None, cache, at, 0, lists, k, rows, rows, 1, heads, 1.0, None, None, 0)

    def append(cache=_cache_args(), rotary=None, table=table, k=rows, q=None, n=1, heads=0, positions=64):
        return L.certexB200PagedAppend(None, cache, rotary, table, k, rows, q, q, n, heads, positions, 0)

    def rotate(rotary=plan(), x=rows, n=1, heads=1, dim=8, dtype=0, positions=64):
        return L.certexB200Rotate(None, rotary, x, rows, n, heads, dim, dtype, positions, 0, 0)

    for call, text in (
        (lambda: attend(cache=None), b"null cache"), (lambda: attend(cache=_cache_args(dim=12)), b"multiple of 8"),
        (lambda: attend(cache=_cache_args(dim=264)), b"at most 256"), (lambda: attend(cache=_cache_args(dtype=3)), b"dtype"),
        (lambda: attend(cache=_cache_args(keys=72)), b"16 bytes"), (lambda: attend(cache=_cache_args(v1=2)), b"16 bytes"),
        (lambda: attend(cache=_cache_args(fault=0)), b"null cache"), (lambda: attend(cache=_cache_args(page_size=0)), b"pages"),
        (lambda: attend(table=None), b"table"), (lambda: attend(lengths=None), b"lengths"), (lambda: attend(window=-1), b"window"),
        (lambda: attend(cache=_cache_args(kv=2), heads=3), b"multiple"), (lambda: attend(n=-1), b"rows"), (lambda: attend(n=2**31), b"rows"), (lambda: attend(n=2**27), b"rows"),
        (lambda: attend(cache=_cache_args(n_pages=2**16, page_size=2**15)), b"places"), (lambda: attend(cache=_cache_args(n_pages=2**20, page_size=16, k0=-64)), b"strides"),
        (lambda: attend(scale=math.inf), b"finite"), (lambda: attend(scale=math.nan), b"finite"), (lambda: attend(), b"null resources"),
        (lambda: selected(lists=2, heads=4), b"list"), (lambda: selected(at=None), b"positions"), (lambda: selected(k=-1), b"positions"),
        (lambda: selected(), b"null resources"), (lambda: append(k=None), b"null keys"), (lambda: append(heads=2, q=rows), b"rotation"),
        (lambda: append(rotary=plan(), heads=1), b"null queries"), (lambda: append(rotary=plan(10)), b"even number"),
        (lambda: append(positions=None), b"positions"), (lambda: append(n=2**31), b"rows"), (lambda: append(), b"null resources"),
        (lambda: rotate(rotary=None), b"null rotation"), (lambda: rotate(plan(3)), b"even"), (lambda: rotate(dim=7), b"even"),
        (lambda: rotate(dtype=-1), b"dtype"), (lambda: rotate(x=None), b"null rows"), (lambda: rotate(positions=None), b"positions"),
        (lambda: rotate(n=2**31), b"rows"), (lambda: rotate(), b"null resources"),
    ):
        assert call() == 0 and text in L.cuvsGetLastErrorText(), (text, L.cuvsGetLastErrorText())
    assert attend(n=0) == 1 and append(n=0) == 1 and rotate(n=0) == 1  # nothing to do needs nothing
    need = ctypes.c_size_t()
    assert L.certexB200PagedWorkspace(None, _cache_args(dim=9), 1, 1, 0, 1, 0, ctypes.byref(need)) == 0


def test_sizes_beyond_all_bounds_are_refused(built_library):
    """Products of sizes that would wrap, and those that the other calls refuse, are errors before the device is looked at."""
    L, table, rows, need = built_library, paged._TABLE.pack(64, 1, 1, 1, 0), paged._ROWS.pack(64, 8, 8), ctypes.c_size_t()

    def workspace(n=1, heads=1, lists=0, k=1):
        return L.certexB200PagedWorkspace(None, _cache_args(), n, heads, lists, k, 0, ctypes.byref(need))

    def attend(n, heads):
        return L.certexB200PagedAttend(None, _cache_args(), table, 64, 0, rows, rows, n, heads, 1.0, None, None, 0)

    for call, text in (
        (lambda: workspace(n=2**27), b"too many rows"), (lambda: workspace(n=2**40), b"too many rows"), (lambda: workspace(n=2**62, heads=4), b"too many rows"),
        (lambda: workspace(heads=65536), b"multiple"), (lambda: workspace(n=-1), b"null argument"), (lambda: attend(2**62, 4), b"too many rows"),
        (lambda: attend(2**26, 2), b"too many rows"), (lambda: workspace(n=2**27 - 1, k=2**62), b"null resources"),
    ):
        assert call() == 0 and text in L.cuvsGetLastErrorText(), (text, L.cuvsGetLastErrorText())


def test_packed_structures_have_the_headers_sizes(built_library, tmp_path):
    import os
    import shutil
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, exe = tmp_path / "sizes.c", str(tmp_path / "sizes")
    src.write_text('#include <stdio.h>\n#include "certex_b200.h"\nint main(void) { printf("%zu %zu %zu %zu", sizeof(certexB200Rows_t), '
                   "sizeof(certexB200PageTable_t), sizeof(certexB200Rotary_t), sizeof(certexB200PagedCache_t)); return 0; }\n")
    subprocess.run([shutil.which("gcc"), "-I" + os.path.join(root, "include"), str(src), "-o", exe], check=True)
    sizes = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert [int(s) for s in sizes] == [s.size for s in (paged._ROWS, paged._TABLE, paged._ROTARY, paged._CACHE)]
    assert all(isinstance(s, struct.Struct) for s in (paged._ROWS, paged._TABLE))


def test_caches_that_make_no_sense_are_refused():
    t = torch.zeros((2, 4, 1, 8))
    for kwargs in (dict(n_pages=0, page_size=1, n_kv_heads=1, head_dim=8), dict(n_pages=1, page_size=1, n_kv_heads=1), dict(keys=t),
                   dict(keys=t, values=t), dict(n_pages=1, page_size=1, n_kv_heads=1, head_dim=8, layout="DNH")):
        with pytest.raises(ValueError):
            certex.PagedCache(**kwargs, device="cpu")


@gpu
def test_refusals():
    kv = torch.zeros((4, 2, 2, 16), device="cuda")
    for kwargs in (dict(keys=kv, values=kv[:3]), dict(keys=kv, values=kv.half()), dict(keys=kv.double(), values=kv.double()),
                   dict(keys=kv[..., :12], values=kv[..., :12]), dict(keys=kv[..., ::2], values=kv[..., ::2]), dict(keys=kv[..., 1:9], values=kv[..., 1:9]),
                   dict(keys=kv, values=kv, page_size=3), dict(keys=kv, values=kv, rotary=certex.Rotary(8)),
                   dict(keys=kv[:1].expand(4, 2, 2, 16), values=kv), dict(n_pages=1, page_size=1, n_kv_heads=1, head_dim=264)):
        with pytest.raises(ValueError):
            certex.PagedCache(**kwargs)
    cache = certex.PagedCache(keys=kv, values=kv.clone())
    q, n, t = torch.zeros((2, 4, 16), device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda"), torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    at = torch.zeros((2, 4, 3), dtype=torch.int32, device="cuda")
    k = q[:, :2]
    for bad in (lambda: cache.attend(q[:, :3], t, n), lambda: cache.attend(q.half(), t, n), lambda: cache.attend(q, t.long(), n),
                lambda: cache.attend(q, t, n.long()), lambda: cache.attend(q, t, n[:1]), lambda: cache.attend(q, t[:1], n), lambda: cache.attend(q, t.cpu(), n),
                lambda: cache.attend(q, t, n, window=0), lambda: cache.attend(q, t, n, scale=math.inf), lambda: cache.attend(q[0], t, n),
                lambda: cache.attend(q, t, n, row_to_batch=[0, 1]), lambda: cache.attend(q, t, n, out=q), lambda: cache.attend(q.cpu(), t, n),
                lambda: cache.attend(q.requires_grad_(), t, n), lambda: cache.attend_selected(q, at[:, :3]), lambda: cache.attend_selected(q, at[:1]),
                lambda: cache.attend_selected(q, at.float()), lambda: cache.append(k, k[:1], t, n), lambda: cache.append(k, k, t, n.float()),
                lambda: cache.append(k[:, :1], k, t, n), lambda: cache.append(k, k, t, n, q=q)):
        q.requires_grad_(False)
        with pytest.raises(ValueError):
            bad()
    q.requires_grad_(False)
    lib, need = _lib.lib(), ctypes.c_size_t()
    big = torch.zeros((1, 4096), dtype=torch.int32, device="cuda")
    _lib.check(lib.certexB200PagedWorkspace(_lib.resources(), cache._args, 1, 4, 0, 8192, 0, ctypes.byref(need)))
    if need.value:  # a workspace that is too small
        table = paged._TABLE.pack(big.data_ptr(), 4096, 1, 4096, 0)
        rows = paged._packed(q)
        assert lib.certexB200PagedAttend(_lib.resources(), cache._args, table, n.data_ptr(), 0, rows, rows, 1, 4, 1.0, None, big.data_ptr(), need.value - 1) == 0
        assert b"workspace" in lib.cuvsGetLastErrorText()


# ------------------------------------------------------------------------------------------------------------ append
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("sequences,tokens,kv,heads,dim,page,r", [(1, 1, 1, 0, 8, 1, 0), (3, 1, 2, 6, 80, 16, 80), (2, 37, 3, 3, 96, 7, 32), (1, 5, 8, 64, 128, 64, 128),
                                                                   (3, 700, 8, 32, 128, 16, 64), (2, 9, 1, 2, 24, 5, 6)])
def test_append(sequences, tokens, kv, heads, dim, page, r, layout, dtype):
    cache, table, g = make(dtype, sequences, 1000, page, kv, dim, layout)
    cache = certex.PagedCache(keys=cache.keys, values=cache.values, layout=layout, rotary=certex.Rotary(dim, r, interleaved=r == 32) if r else None)
    n = sequences * tokens + 2
    qkv = torch.randn((n, heads + 2 * kv, dim), generator=g, device="cuda").to(dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv], qkv[:, heads + kv :]
    start = torch.randint(0, 1000 - tokens, (sequences,), generator=g, device="cuda")
    positions = torch.cat([(start[:, None] + torch.arange(tokens, device="cuda")).flatten(), torch.tensor([-1, -7], device="cuda")])
    to = torch.cat([torch.arange(sequences, device="cuda").repeat_interleave(tokens), torch.tensor([0, 99], device="cuda")]).to(torch.int32)
    order = torch.randperm(n, generator=g, device="cuda")
    q, k, v, positions, to = (qkv[order][:, :heads], qkv[order][:, heads : heads + kv], qkv[order][:, heads + kv :], positions[order], to[order])
    keys, values = cache.keys.clone(), cache.values.clone()
    got = cache.append(k, v, table, positions, row_to_batch=to, q=q if heads and r else None)
    real = positions >= 0
    page_of = table[to[real].long(), positions[real] // page].long()
    for new, old, x in ((cache.keys, keys, cache.rotary(k, positions) if r else k), (cache.values, values, v)):
        view = old if layout == "NHD" else old.transpose(1, 2)
        view[page_of, positions[real] % page] = x[real]
        assert torch.equal(new, old)  # the rest of the cache as well
    assert (got is None) == (not (heads and r)) and (got is None or torch.equal(got, cache.rotary(q, positions)))
    assert not cache.faulted()
    again = cache.keys.clone()
    cache.append(k, v, table, positions.int(), row_to_batch=to)
    assert torch.equal(cache.keys, again)


@gpu
def test_append_with_indices_out_of_range_writes_nothing():
    cache, table, g = make(torch.float16, 2, 32, 8, 2, 64)
    keys, values = cache.keys.clone(), cache.values.clone()
    k = torch.randn((1, 2, 64), device="cuda").half()
    one = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
    for positions, to, tab in ((one(40), one(0), table), (one(2**31 - 1), one(1), table), (torch.tensor([2**60], device="cuda"), one(0), table), (one(0), one(2), table),
                               (one(0), one(-1), table), (one(0), one(0), torch.full_like(table, cache.n_pages)), (one(0), one(0), torch.full_like(table, -1))):
        cache.append(k, k, tab, positions, row_to_batch=to)
        assert cache.faulted() and not cache.faulted()
        assert torch.equal(cache.keys, keys) and torch.equal(cache.values, values)
    cache.append(k[:0], k[:0], table[:0], one(0)[:0])
    assert not cache.faulted()


# ------------------------------------------------------------------------------------------------------------ attention
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv,heads,dim,page,layout", [(1, 1, 8, 1, "NHD"), (2, 8, 128, 16, "NHD"), (3, 3, 80, 7, "HND"), (1, 16, 64, 32, "HND"), (2, 10, 96, 5, "NHD"),
                                                      (1, 17, 256, 16, "NHD"), (2, 128, 128, 64, "HND"), (1, 6, 200, 3, "HND")])
def test_attend_every_length(kv, heads, dim, page, layout, dtype):
    """Lengths around every border of the kernels: none, one, tiles of 16, 32, 64 and 128, a few thousand."""
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500, 1025, 2049, -3]
    cache, table, g = make(dtype, len(lens), 2049, page, kv, dim, layout, seed=dim)
    poison(cache, table, [max(n, 0) for n in lens])
    q = torch.randn((len(lens), heads, dim), generator=g, device="cuda").to(dtype)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, table, lengths, return_lse=True)
    rows = torch.tensor([0, 1, 4, 5, 10, 13, 17, 18, 19])  # the oracle is slow: these, and every length for two heads
    check(out[rows], lse[rows], q[rows], cache, [table_places(cache, table, lengths, None, heads)[i] for i in rows])
    few = sorted({0, heads - 1})
    full = table_places(cache, table, lengths, None, heads)
    keys, values = (t.cpu() if layout == "NHD" else t.cpu().transpose(1, 2) for t in (cache.keys, cache.values))
    for i in range(len(lens)):
        for h in few:
            kvh = h // (heads // kv)
            at = full[i][h]
            want, l, off, _ = softmax_sum(q[i, h].cpu().double(), keys[at[:, 0], at[:, 1], kvh].double(), values[at[:, 0], at[:, 1], kvh].double(), dim**-0.5, dtype)
            assert float(((out[i, h].cpu().double() - want).abs() - off).max()) <= 0, (i, h)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all()) and not cache.faulted()
    assert torch.equal(out, cache.attend(q, table, lengths))  # the same again, bit for bit


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most,window,scale", [(40_000, None, None), (40_000, 333, 0.3), (9000, 1, None), (9000, 5000, -0.05), (9000, 10_000, 0.0)])
def test_attend_long_and_windows(most, window, scale, dtype):
    cache, table, g = make(dtype, 3, most, 16, 2, 64)
    lens = [most, most // 3, 1]
    poison(cache, table, lens, float("inf"))
    q = torch.randn((3, 8, 64), generator=g, device="cuda").to(dtype)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, table, lengths, window=window, scale=scale, return_lse=True)
    check(out, lse, q, cache, table_places(cache, table, lengths, None, 8, window), scale)


@gpu
def test_attend_drafts_and_padded_batches():
    """Several rows of one sequence with lengths of their own, rows in any order, rows that are padding, one sequence in many rows."""
    cache, table, g = make(torch.bfloat16, 4, 700, 16, 2, 128)
    to = torch.tensor([2, 2, 2, 0, 3, 3, 1, 0, 2], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([500, 501, 502, 1, 0, 700, 64, 699, 3], dtype=torch.int32, device="cuda")
    q = torch.randn((9, 8, 128), generator=g, device="cuda").bfloat16()
    out, lse = cache.attend(q, table, lengths, row_to_batch=to, return_lse=True)
    check(out, lse, q, cache, table_places(cache, table, lengths, to, 8))
    wide = torch.full((9, 20, 128), 5.0, device="cuda").bfloat16()
    assert cache.attend(q, table, lengths, row_to_batch=to, out=wide[:, 4:12]).data_ptr() == wide[:, 4:12].data_ptr()
    assert torch.equal(wide[:, 4:12], out) and bool((wide[:, :4] == 5).all()) and bool((wide[:, 12:] == 5).all())
    big = torch.randn((9, 64, 128), generator=g, device="cuda").bfloat16()
    view = big[:, ::8]  # queries that are a view, and a table that is a part of a wider one
    a = cache.attend(view, torch.cat([table, table], 1)[:, : table.shape[1]], lengths, row_to_batch=to)
    assert torch.equal(a, cache.attend(view.contiguous(), table, lengths, row_to_batch=to))
    assert cache.attend(q[:0], table[:0], lengths[:0]).shape == (0, 8, 128)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_with_indices_out_of_range(dtype):
    """What is named wrongly is left out, and said."""
    cache, table, g = make(dtype, 2, 300, 16, 1, 64)
    q = torch.randn((2, 4, 64), generator=g, device="cuda").to(dtype)
    n = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    assert bool((cache.attend(q, table, n(10, 300)) != 0).any()) and not cache.faulted()
    most = table.shape[1] * 16
    assert torch.equal(cache.attend(q, table, n(2**31 - 1, 5)), cache.attend(q, table, n(most, 5))) and cache.faulted()
    assert bool((cache.attend(q, table, n(7, 7), row_to_batch=n(2, -1)) == 0).all()) and cache.faulted()
    bad = table.clone()
    bad[0, 1], bad[0, 3] = cache.n_pages, -5
    out = cache.attend(q, bad, n(80, 0))
    assert cache.faulted()
    t = torch.cat([torch.arange(0, 16), torch.arange(32, 48), torch.arange(64, 80)])
    at = torch.stack([table[0].cpu().long()[t // 16], t % 16], 1)
    check(out[:1], None, q[:1], cache, [[at] * 4])
    assert bool((cache.attend(q, torch.full_like(table, -1), n(300, 300)) == 0).all()) and cache.faulted()
    at = torch.full((2, 4, 9), cache.n_pages * 16, dtype=torch.int64, device="cuda")
    at[:, :, 4] = 17
    assert torch.equal(cache.attend_selected(q, at), cache.attend_selected(q, at[:, :, 4:5])) and cache.faulted()
    at[:, :, 4] = 2**40
    assert bool((cache.attend_selected(q, at) == 0).all()) and cache.faulted()
    empty = table[:, :0]
    assert bool((cache.attend(q, empty, n(0, 0)) == 0).all()) and not cache.faulted()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv,heads,dim,page,layout", [(2, 8, 128, 16, "NHD"), (1, 1, 64, 1, "NHD"), (3, 6, 80, 7, "HND"), (1, 40, 96, 32, "NHD"), (8, 8, 256, 5, "HND")])
@pytest.mark.parametrize("k", [1, 17, 128, 1000])
def test_attend_selected(k, kv, heads, dim, page, layout, dtype):
    cache, table, g = make(dtype, 3, 1500, page, kv, dim, layout, seed=k)
    q = torch.randn((3, heads, dim), generator=g, device="cuda").to(dtype)
    total = cache.n_pages * cache.page_size
    for lists in sorted({1, kv, heads}):
        at = torch.randint(0, total, (3, lists, k), generator=g, device="cuda")
        if k > 1:
            at[:, 0, k // 2 :] = -1          # a list that is not full
            at[1, -1] = at[1, -1, :1]        # one position over and over
            at[2, -1, ::2] = -1 - at[2, -1, ::2]
        out, lse = cache.attend_selected(q, at, return_lse=True)
        check(out, lse, q, cache, selected_places(cache, at, heads))
        assert torch.equal(out, cache.attend_selected(q, at.to(torch.int32)))
    none, lse = cache.attend_selected(q, torch.full((3, 1, k), -1, device="cuda"), return_lse=True)
    assert bool((none == 0).all()) and bool((lse == -math.inf).all())
    assert bool((cache.attend_selected(q, torch.zeros((3, 1, 0), dtype=torch.int32, device="cuda")) == 0).all())
    assert not cache.faulted()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_values_at_the_edge(dtype):
    """A key that outweighs everything, scores of minus infinity, an infinite value that weighs nothing's neighbour, NaN where it is seen."""
    cache, table, g = make(dtype, 1, 400, 16, 1, 64)
    keys, values = cache.keys, cache.values
    q = torch.zeros((1, 2, 64), device="cuda").to(dtype)
    q[..., 0] = 8
    at = lambda t: (int(table[0, t // 16]), t % 16, 0)  # noqa: E731
    keys[at(200)][0] = 29_952.0
    n = torch.tensor([400], dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, table, n, return_lse=True)
    assert torch.equal(out[0], values[at(200)].expand(2, 64)) and bool(((lse - 29_952).abs() <= 29_952 * 2.0**-22).all())
    for t in range(400):
        keys[at(t)][0] = -float("inf") if t % 3 else 1.0
    out, lse = cache.attend(q, table, n, return_lse=True)
    kept = [(torch.stack([table[0].cpu().long()[torch.arange(0, 400, 3) // 16], torch.arange(0, 400, 3) % 16], 1))] * 2
    q0 = q.clone()
    check(out, lse, q0, cache, [kept])
    values[at(3)][5] = float("inf")
    out = cache.attend(q, table, n)
    assert bool((out[0, :, 5] == float("inf")).all()) and bool(torch.isfinite(out[0, :, 6]).all())
    keys[at(6)][1] = float("nan")
    assert bool(torch.isnan(cache.attend(q, table, n)).all())
    assert bool(torch.isfinite(cache.attend(q, table, torch.tensor([3], dtype=torch.int32, device="cuda"))).all())


@gpu
def test_offsets_beyond_32_bits():
    """Pages whose places in memory lie beyond 2^31 and 2^32 elements: a cache of 9 GiB whose last pages are used."""
    page, kv, dim = 64, 8, 128
    n = 2**32 // (page * kv * dim) + 100
    keys = torch.empty((n, page, kv, dim), dtype=torch.float16, device="cuda")
    values = keys  # the same memory serves both: nothing says that it may not
    cache = certex.PagedCache(keys=keys, values=values, rotary=None)
    table = torch.tensor([[n - 1, n // 2 + 3, 5]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((192, kv, dim), generator=g, device="cuda").half()
    cache.append(x, x, table, torch.arange(192, device="cuda"), row_to_batch=torch.zeros(192, dtype=torch.int32, device="cuda"))
    assert torch.equal(torch.cat([keys[n - 1], keys[n // 2 + 3], keys[5]]), x)
    small = certex.PagedCache(keys=x.view(3, 64, kv, dim).clone(), values=x.view(3, 64, kv, dim).clone())
    q, length = torch.randn((1, 32, dim), generator=g, device="cuda").half(), torch.tensor([190], dtype=torch.int32, device="cuda")
    want = small.attend(q, torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), length)
    assert torch.equal(cache.attend(q, table, length), want)
    at = torch.arange(190, device="cuda")
    at = (table[0, at // 64].long() * 64 + at % 64)[None, None]
    got = cache.attend_selected(q, at)
    assert torch.equal(got, small.attend_selected(q, torch.arange(190, device="cuda")[None, None]))
    assert not cache.faulted()


# ------------------------------------------------------------------------------------------------------------ as it is used
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_a_decoding_loop(dtype):
    """Prompts are appended, then steps: queries and keys turned, stored, attended over everything, over a window and over the exact top k that the selector
    finds among the same keys; the selected attention over all positions is the whole attention."""
    kv, heads, dim, page, k = 2, 8, 64, 16, 48
    rotary = certex.Rotary(dim, scaling="yarn", factor=4.0)
    cache = certex.PagedCache(200, page, kv, dim, dtype=dtype, rotary=rotary)
    g = torch.Generator(device="cuda").manual_seed(3)
    table = torch.randperm(200, generator=g, device="cuda").to(torch.int32)[:120].view(3, 40)
    selector = flashinfer.ExactTopK(kv, dim, k_max=k)
    lens = [333, 20, 128]
    for b, n in enumerate(lens):
        x, v = (torch.randn((n, kv, dim), generator=g, device="cuda").to(dtype) for _ in range(2))
        pos = torch.arange(n, device="cuda")
        cache.append(x, v, table, pos, row_to_batch=torch.full((n,), b, dtype=torch.int32, device="cuda"))
        selector.append(b, rotary(x, pos))
    for step in range(3):
        q0, x, v = (torch.randn((3, h, dim), generator=g, device="cuda").to(dtype) for h in (heads, kv, kv))
        pos = torch.tensor([n + step for n in lens], device="cuda")
        q = cache.append(x, v, table, pos, q=q0)
        turned = rotary(x, pos)
        for b in range(3):
            selector.append(b, turned[b : b + 1])
        lengths = (pos + 1).to(torch.int32)
        out, lse = cache.attend(q, table, lengths, return_lse=True)
        check(out, lse, q, cache, table_places(cache, table, lengths, None, heads))
        at = selector.page_table_transform(q, table, k, page_size=page)
        assert at.shape == (3, heads, k) and int((at[1, 0] >= 0).sum()) == min(k, lens[1] + step + 1)
        sparse, part = cache.attend_selected(q, at, return_lse=True)
        check(sparse, part, q, cache, selected_places(cache, at, heads))
        assert bool((part <= lse + 1e-3).all())  # a part of the sum
        every = torch.arange(400, device="cuda")[None, :]
        places = table[:, (every[0] // page).clamp(max=39)] * page + (every % page).to(torch.int32)
        whole = cache.attend_selected(q, torch.where(every < lengths[:, None], places, -1)[:, None].to(torch.int32), return_lse=True)
        check(whole[0], whole[1], q, cache, table_places(cache, table, lengths, None, heads))
    assert not cache.faulted()


@gpu
def test_two_graphs_two_streams_and_eager_calls_at_once():
    """Graphs of the same cache replay beside one another and beside eager calls: every call has its own workspace."""
    cache, table, g = make(torch.bfloat16, 4, 20_000, 16, 2, 128)
    q = [torch.randn((4, 8, 128), generator=g, device="cuda").bfloat16() for _ in range(3)]
    lengths = torch.tensor([20_000, 777, 0, 12_345], dtype=torch.int32, device="cuda")
    at = torch.randint(0, cache.n_pages * 16, (4, 8, 4000), generator=g, device="cuda")
    want = [(cache.attend(x, table, lengths), cache.attend_selected(x, at)) for x in q]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in q[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((cache.attend(x, table, lengths), cache.attend_selected(x, at)))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = cache.attend(q[2], table, lengths), cache.attend_selected(q[2], at)
    torch.cuda.synchronize()
    for got, ref in zip(outs + [eager], want):
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    lengths.copy_(torch.tensor([5, 20_000, 13, 1], dtype=torch.int32))  # a captured call sees the new lengths
    graphs[0].replay()
    assert torch.equal(outs[0][0], cache.attend(q[0], table, lengths))


@gpu
def test_what_the_library_overwrites_is_known_to_autograd():
    """A tensor that a graph saved and a call overwrote makes the backward pass fail instead of using what lies there now."""
    rotary = certex.Rotary(64)
    cache = certex.PagedCache(4, 16, 1, 64, dtype=torch.float32)
    p, table = torch.arange(5, device="cuda"), torch.arange(4, device="cuda", dtype=torch.int32)[None]
    n, to = torch.full((5,), 5, device="cuda", dtype=torch.int32), torch.zeros(5, device="cuda", dtype=torch.int32)
    x = torch.randn((5, 1, 64), device="cuda")
    a = torch.ones((5, 1, 64), device="cuda", requires_grad=True)
    overwrite = ((x, lambda: rotary(x, p, out=x)), (cache.keys, lambda: cache.append(x, x, table, p, row_to_batch=to)),
                 (cache.values, lambda: cache.append(x, x, table, p, row_to_batch=to)), (x, lambda: cache.attend(x.clone(), table, n, row_to_batch=to, out=x)),
                 (x, lambda: cache.attend_selected(x.clone(), p.int().view(5, 1, 1), out=x)))
    for t, call in overwrite:
        loss = (a * t.view(-1)[: a.numel()].view_as(a)).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        y = torch.randn((5, 1, 64), device="cuda")
        rotary(y, p, out=y)
        cache.append(y, y, table, p, row_to_batch=to)


@gpu
def test_outputs_whose_rows_overlap_are_refused():
    rotary, p = certex.Rotary(8), torch.arange(4, device="cuda")
    x, memory = torch.randn((4, 3, 8), device="cuda"), torch.zeros(400, device="cuda")
    for strides in ((8, 8, 1), (16, 8, 1), (24, 4, 1), (0, 8, 1), (8, 16, 1), (24, 8, 2)):
        with pytest.raises(ValueError, match="memory of its own"):
            rotary(x, p, out=memory.as_strided((4, 3, 8), strides))
    for strides in ((24, 8, 1), (30, 9, 1), (8, 32, 1), (9, 40, 1)):
        out = memory.as_strided((4, 3, 8), strides)
        assert torch.equal(rotary(x, p, out=out), rotary(x, p))


@gpu
def test_a_cache_stays_what_it_was_made_of():
    cache = certex.PagedCache(4, 16, 1, 64, dtype=torch.float16)
    for name, value in (("keys", cache.values), ("values", cache.keys), ("layout", "HND")):
        with pytest.raises(AttributeError):
            setattr(cache, name, value)
    for rotary in (certex.Rotary(32), certex.Rotary(64, device="cpu")):
        with pytest.raises(ValueError, match="rotation"):
            cache.rotary = rotary
    cache.rotary = certex.Rotary(64)
    k, p, t = torch.ones((1, 1, 64), device="cuda").half(), torch.zeros(1, device="cuda", dtype=torch.int32), torch.zeros((1, 1), device="cuda", dtype=torch.int32)
    cache.append(k, k, t, p)
    selected = p.view(1, 1)
    assert torch.equal(cache.attend_selected(k, selected), cache.attend(k, t, p + 1))
    keys = cache.keys
    keys.data = torch.zeros_like(keys)
    for call in (lambda: cache.append(k, k, t, p), lambda: cache.attend(k, t, p + 1), lambda: cache.attend_selected(k, selected)):
        with pytest.raises(ValueError, match="other memory"):
            call()


@gpu
def test_the_first_calls_of_a_process_may_be_captured():
    """Kernels that were never launched before, recorded in a graph."""
    import subprocess
    import sys

    code = """
import torch, libcertex_b200 as certex
rotary = certex.Rotary(64)
cache = certex.PagedCache(600, 16, 2, 64, dtype=torch.float16, rotary=rotary)
k = torch.randn((1, 2, 64), device="cuda").half(); q = torch.randn((1, 8, 64), device="cuda").half()
table = torch.arange(600, device="cuda", dtype=torch.int32)[None]
p, n = torch.tensor([9000], device="cuda", dtype=torch.int32), torch.tensor([9001], device="cuda", dtype=torch.int32)
cache.keys.normal_(); cache.values.normal_()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    r = cache.append(k, k, table, p, q=q)
    a = cache.attend(r, table, n)
    b = cache.attend(r, table[:, :5], torch.clamp(n, max=70))
    c = cache.attend_selected(r, p.view(1, 1, 1))
g.replay(); torch.cuda.synchronize()
assert torch.equal(a, cache.attend(r, table, n)) and torch.equal(c, k.repeat_interleave(4, 1)) and not cache.faulted()
print("captured")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert "captured" in done.stdout, done.stderr[-2000:]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_pages_that_are_views(dtype):
    """Keys and values as the two halves of one tensor, every second head of wider pages, and one memory for both."""
    g = torch.Generator(device="cuda").manual_seed(9)
    both = torch.randn((50, 2, 16, 6, 40), generator=g, device="cuda").to(dtype)
    q = torch.randn((2, 9, 40), generator=g, device="cuda").to(dtype)
    table = torch.randperm(50, generator=g, device="cuda").to(torch.int32).view(2, 25)
    n = torch.tensor([390, 77], dtype=torch.int32, device="cuda")
    at = torch.randint(-99, 800, (2, 9, 99), generator=g, device="cuda")
    for keys, values in ((both[:, 0, :, :3], both[:, 1, :, 3:]), (both[:, 0, :, ::2], both[:, 1, :, 1::2]), (both[:, 1, :, 1:4], both[:, 1, :, 1:4])):
        cache = certex.PagedCache(keys=keys, values=values)
        dense = certex.PagedCache(keys=keys.contiguous(), values=values.contiguous())
        assert torch.equal(cache.attend(q, table, n), dense.attend(q, table, n))
        assert torch.equal(cache.attend_selected(q, at), dense.attend_selected(q, at))
        out, lse = cache.attend(q, table, n, return_lse=True)
        check(out, lse, q, cache, table_places(cache, table, n, None, 9))
    rest = both.clone()
    cache = certex.PagedCache(keys=both[:, 0, :, ::2], values=both[:, 1, :, 1::2], rotary=certex.Rotary(40, 16))
    k, v = (torch.randn((2, 3, 40), generator=g, device="cuda").to(dtype) for _ in range(2))
    cache.append(k, v, table, n)
    for i in range(2):
        page, place = int(table[i, int(n[i]) // 16]), int(n[i]) % 16
        rest[page, 0, place, ::2] = cache.rotary(k, n)[i]
        rest[page, 1, place, 1::2] = v[i]
    assert torch.equal(both, rest)


@gpu
def test_copies_of_a_cache_have_their_own_memory():
    cache, table, _ = make(torch.bfloat16, 2, 40, 8, 2, 16)
    cache.rotary = certex.Rotary(16)
    q = torch.randn((2, 4, 16), device="cuda").bfloat16()
    lengths = torch.tensor([40, 3], device="cuda", dtype=torch.int32)
    kv = torch.randn((2, 2, 2, 16), device="cuda").bfloat16()
    want = cache.attend(q, table, lengths)
    for twin in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert twin.keys.data_ptr() != cache.keys.data_ptr() and twin.rotary is not cache.rotary
        assert torch.equal(twin.attend(q, table, lengths), want)
        twin.append(kv[0], kv[1], table, torch.tensor([1, 99], device="cuda"))  # the second lies behind its table
        assert twin.faulted() and not cache.faulted()
        assert torch.equal(cache.attend(q, table, lengths), want) and not torch.equal(twin.attend(q, table, lengths), want)
    stored = io.BytesIO()
    torch.save(cache, stored)
    stored.seek(0)
    with pytest.raises(ValueError, match="CUDA"):
        torch.load(stored, map_location="cpu", weights_only=False)


@gpu
def test_keys_and_values_of_one_memory():
    both = torch.randn((3, 4, 1, 8), device="cuda")
    cache = certex.PagedCache(keys=both, values=both)
    table, n = torch.tensor([[2, 0]], device="cuda", dtype=torch.int32), torch.tensor([1], device="cuda", dtype=torch.int32)
    row = torch.ones((1, 1, 8), device="cuda")
    assert torch.equal(cache.attend(row, table, n), both[2, :1])  # one key: its value, weight 1
    cache.append(row, row, table, n)
    assert torch.equal(both[2, 1], row[0]) and torch.equal(cache.attend(row, table, n), both[2, :1])


@gpu
def test_captured_calls_wait_for_all_that_is_in_front_of_them():
    """A call whose place in a graph is behind a kernel of the library, a copy and another stream's work at once sees them all."""
    cache, table, _ = make(torch.float32, 2, 2000, 16, 1, 8)
    q, lengths, host = torch.randn((2, 1, 8), device="cuda"), torch.zeros(2, device="cuda", dtype=torch.int32), torch.zeros(2, dtype=torch.int32).pin_memory()
    side, new = torch.cuda.Stream(), torch.zeros((2, 1, 8), device="cuda")
    source = torch.zeros((2, 1, 8), device="cuda")
    rotary = certex.Rotary(8)

    def step():
        now = torch.cuda.current_stream()
        side.wait_stream(now)
        lengths.copy_(host, non_blocking=True)
        turned = rotary(q, lengths)
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000)
            new.copy_(source)
        now.wait_stream(side)
        cache.append(new, new, table, lengths - 1)
        return turned, cache.attend(new, table, lengths)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, out = step()
    for turn, n in enumerate((1, 2000, 3, 700, 1999)):
        source.normal_()
        host.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        got = turned.clone(), out.clone()
        want = rotary(q, torch.full((2,), n, device="cuda")), cache.attend(source, table, torch.full((2,), n, device="cuda", dtype=torch.int32))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), turn
        for i in range(2):
            place = table[i, (n - 1) // 16].item(), (n - 1) % 16
            assert torch.equal(cache.values[place], source[i])

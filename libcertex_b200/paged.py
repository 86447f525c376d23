"""What a decoding step does beside the selection of positions (`KeyCache`, `flashinfer.ExactTopK`): a cache of keys and
values in pages, the rotation of queries and keys by their positions, and attention of new tokens over the cache, whole or at
the positions that were selected. The reference stops at the selection (certex/attention.py:44-114, certex/flashinfer.py:50-138).

    rotary = certex.Rotary(128)
    cache = certex.PagedCache(n_pages, 16, n_kv_heads=8, head_dim=128, rotary=rotary)
    q = cache.append(k, v, page_table, positions, q=q)            # one launch: keys turned, stored, queries turned
    out = cache.attend(q, page_table, lengths)                    # over the whole sequences, or
    at = selector.page_table_transform(q, page_table, k=2048, page_size=16)
    out = cache.attend_selected(q, at)                            # over the exact top 2048 keys of every query head

Layouts follow `flashinfer.ExactTopK`: rows (n, heads, head_dim); row i belongs to sequence row_to_batch[i] (default i) of a
page table (sequences, pages_per_sequence); token p of a sequence lies at place p % page_size of its page p // page_size.

Every call enqueues on torch's current stream of the tensors' device and returns; nothing is copied to the host, so that calls
can be captured in a graph. Indices are therefore checked on the device: what a wrong one names is neither read nor written,
and `PagedCache.faulted` tells.
"""

import math
import struct

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib as L
from .index import _need

_KIND = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ROWS = struct.Struct("3q")
_TABLE = struct.Struct("5q")
_ROTARY = struct.Struct("3qd")
_CACHE = struct.Struct("14q")
_MOST_DIM = 256
# 2 pi in units of 10**-39: a frequency's share of a turn is rounded once, to 2**-64
_TURN = 6283185307179586476925286766559005768394


def _fail(message):
    raise ValueError(message)


# The checks below stand in front of kernels of a few microseconds: one expression decides, and messages are made when it fails.
_I32, _I64 = torch.int32, torch.int64


def _check_rows(x, what, index, dtype, heads, dim):
    """A tensor (n, heads, dim) on CUDA device `index` whose last axis is dense, as the kernels read it; `heads` and `dtype` may be
    None: any number, any of the types."""
    try:
        shape = x.shape
        fine = (x.get_device() == index and (x.dtype is dtype or (dtype is None and x.dtype in _KIND)) and shape[2] == dim
                and (heads is None or shape[1] == heads) and len(shape) == 3)
    except (AttributeError, IndexError):
        fine = False
    if not fine:
        _explain_rows(x, what, index, dtype, heads, dim)
    if x.is_neg():
        x = x.resolve_neg()
    return x if x.stride(2) == 1 else x.contiguous()


def _explain_rows(x, what, index, dtype, heads, dim):
    _need(isinstance(x, torch.Tensor) and x.is_cuda, f"{what} must be a CUDA tensor")
    _need(x.get_device() == index, f"{what} must be on cuda:{index}, not {x.device}")
    _need(x.ndim == 3 and x.shape[2] == dim and heads in (None, x.shape[1]),
          f"{what} must have shape (n, {'heads' if heads is None else heads}, {dim}), not {tuple(x.shape)}")
    _fail(f"{what} must be {dtype or 'float32, float16 or bfloat16'}, not {x.dtype}")


def _check_index(t, what, shape, index, wide=False):
    """An index tensor of this shape on CUDA device `index`: int32 (or int64 if `wide`), dense."""
    try:
        fine = t.get_device() == index and (t.dtype is _I32 or (wide and t.dtype is _I64)) and t.shape == shape
    except AttributeError:
        fine = False
    if not fine:
        _need(isinstance(t, torch.Tensor) and t.get_device() == index, f"{what} must be a tensor on cuda:{index}")
        _need(t.shape == shape, f"{what} must have shape {tuple(shape)}, not {tuple(t.shape)}")
        _fail(f"{what} must be {'int32 or int64' if wide else 'int32'}, not {t.dtype}")
    if t.is_neg():
        t = t.resolve_neg()
    return t if t.is_contiguous() else t.contiguous()


def _new_like(x):
    """A dense tensor of x's shape."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


def _packed(x):
    s = x.stride()
    return _ROWS.pack(x.data_ptr(), s[0], s[1])


def _span(x):
    """First byte and the byte behind the last that a tensor's elements take."""
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def _check_out(out, x, in_place):
    """A caller's output for rows like x: written by kernels that read x, in any order of rows."""
    _need(isinstance(out, torch.Tensor) and out.shape == x.shape and out.dtype == x.dtype and out.device == x.device,
          f"out must be a {x.dtype} tensor of shape {tuple(x.shape)} on {x.device}")
    _need(not out.is_neg() and not (torch.is_grad_enabled() and out.requires_grad), "out must be a plain tensor without a gradient")
    if out.numel():
        (n, heads, dim), (row, head, one) = out.shape, out.stride()
        _need(one == 1 and (row >= (heads - 1) * head + dim or n == 1 or head >= (n - 1) * row + dim) and (head >= dim or heads == 1)
              and (row >= dim or n == 1), "out must have memory of its own for every head, with a dense last axis")
        if not (in_place and out.data_ptr() == x.data_ptr() and out.stride() == x.stride()):
            (a, b), (c, d) = _span(out), _span(x)
            _need(b <= c or d <= a, "out must not share memory with the rows" + (" unless it is them" if in_place else ""))
    return out


def _has_tangent(x):
    """Whether forward-mode differentiation goes through x (asked only inside of it)."""
    return _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(x).tangent is not None


# Tells autograd that the library wrote into tensors of the caller's: a graph that saved one of them before finds out.
_written = torch.autograd.graph.increment_version


def _no_gradient(*tensors):
    for t in tensors:
        if isinstance(t, torch.Tensor) and (t.requires_grad and torch.is_grad_enabled() or _has_tangent(t)):
            _fail("no gradient flows through a paged cache: call it under torch.no_grad()")


try:
    _current_device = torch._C._cuda_getDevice  # torch.cuda.current_device() without asking whether CUDA is initialised
except AttributeError:
    _current_device = torch.cuda.current_device


# ------------------------------------------------------------------------------------------------------------ rotation
class _Turn(torch.autograd.Function):
    """The rotation is linear and its transpose turns back, with the same magnitude."""

    @staticmethod
    def forward(ctx, x, positions, rotary, inverse):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        return rotary._turn(x, positions, inverse, None)

    @staticmethod
    def backward(ctx, dy):
        (positions,) = ctx.saved_tensors
        return ctx.rotary(dy, positions, inverse=not ctx.inverse), None, None, None

    @staticmethod
    def jvp(ctx, dx, *_):
        (positions,) = ctx.saved_tensors
        return ctx.rotary(dx, positions, inverse=ctx.inverse)


class Rotary:
    """Turns queries and keys by their positions: pair i of the first `rotary_dim` coordinates of a head (default: all) by
    the angle position * w_i, w_i = base ** (-2 i / rotary_dim). Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) with
    interleaved=True. Angles are reduced exactly at every position, so no table of sines limits the length. Sines and cosines
    are off by 2**-21.4 of themselves at most for float32, by 2**-20 for 16-bit types, and by 2**-65 of a turn a position for the
    frequency's rounding.

    scaling stretches the frequencies for sequences longer than the `original_length` a model was trained on, by `factor`:
      "linear"      w_i / factor
      "ntk"         the base grows by factor ** (rotary_dim / (rotary_dim - 2)): slow pairs are stretched, fast ones kept
      "wavelength"  pairs that turn more than `high` times within original_length are kept, those that turn less than `low`
                    times (1 and 4) are divided by factor, those between are mixed
      "yarn"        the ramp over pairs of "YaRN: Efficient Context Window Extension" (Peng et al. 2023) between the pairs that
                    turn `high` and `low` times (32 and 1), with its magnitude 0.1 ln(factor) + 1
    frequencies, if given, are the w_i themselves (rotary_dim / 2 numbers). magnitude multiplies the result (default 1, or
    what "yarn" says)."""

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, interleaved=False, scaling=None, factor=1.0,
                 original_length=4096, low=None, high=None, magnitude=None, frequencies=None, device="cuda"):
        r = head_dim if rotary_dim is None else rotary_dim
        _need(head_dim >= 2 and head_dim % 2 == 0, "head_dim must be even")
        _need(2 <= r <= head_dim and r % 2 == 0, f"rotary_dim must be even and at most head_dim={head_dim}, not {r}")
        _need(scaling in (None, "linear", "ntk", "wavelength", "yarn"), f"unknown scaling {scaling!r}")
        _need(base > 0 and factor > 0 and original_length > 0, "base, factor and original_length must be positive")
        self.head_dim, self.rotary_dim, self.interleaved = int(head_dim), int(r), bool(interleaved)
        if frequencies is not None:
            _need(scaling is None, "frequencies are given: there is nothing to scale")
            w = [float(f) for f in frequencies]
        else:
            w = _frequencies(int(r), float(base), scaling, float(factor), float(original_length), low, high)
        _need(len(w) == r // 2 and all(math.isfinite(f) for f in w), f"{r // 2} finite frequencies are needed")
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" and factor > 1 else 1.0
        self.frequencies, self.magnitude = w, float(magnitude)
        # what one position adds to an angle, as a fraction of a turn in units of 2**-64
        turns = [_turns(f) for f in w]
        self._turns = torch.tensor([t - 2**64 if t >= 2**63 else t for t in turns], dtype=torch.int64, device=device)
        self._bind()

    def _bind(self):
        """What the library is told, with addresses in it."""
        self.device = self._turns.device
        self._index = self._turns.get_device() if self._turns.is_cuda else -2  # (no row is there)
        self._plan = _ROTARY.pack(self._turns.data_ptr(), self.rotary_dim, int(self.interleaved), self.magnitude)

    def __setstate__(self, state):  # a copy, or another process: its tensors lie elsewhere
        self.__dict__.update(state)
        self._bind()

    def __call__(self, x, positions, inverse=False, out=None):
        """x (n, heads, head_dim) float32, float16 or bfloat16, its rows turned by positions (n,) int32 or int64, which may be
        negative. inverse=True is the transpose: it turns back, and multiplies by magnitude too, so that both in a row leave
        magnitude ** 2 times x. Differentiable in x, backward and by torch.autograd.forward_ad; the transforms of torch.func are
        refused (as for every function of torch, a backward pass that is captured in a CUDA graph wants leaves of which no eager
        graph is alive). out: where to write, x itself allowed; without a gradient."""
        x = _check_rows(x, "x", self._index, None, None, self.head_dim)
        positions = _check_index(positions, "positions", x.shape[:1], self._index, True)
        if x.requires_grad and torch.is_grad_enabled() or _has_tangent(x):
            _need(out is None, "out takes no gradient: call without it, or under torch.no_grad()")
            return _Turn.apply(x, positions, self, bool(inverse))
        return self._turn(x, positions, inverse, out)

    def _turn(self, x, positions, inverse, out):
        if _current_device() != self._index:  # kernels, streams and handles are the current device's
            with torch.cuda.device(self._index):
                return self._turn(x, positions, inverse, out)
        y = _new_like(x) if out is None else _check_out(out, x, True)
        n, heads, dim = x.shape
        if n and heads:
            L.check(L.lib().certexB200Rotate(L.resources(self._index), self._plan, _packed(x), _packed(y), n, heads, dim, _KIND[x.dtype],
                                             positions.data_ptr(), positions.dtype is torch.int64, bool(inverse)))
        if out is not None:
            _written(y)
        return y


def _turns(w):
    """w radians as a fraction of a turn in units of 2**-64, whole turns left out."""
    n, d = w.as_integer_ratio()
    return ((n * 10**39 << 65) // (d * _TURN) + 1) // 2 % 2**64


def _frequencies(r, base, scaling, factor, length, low, high):
    """Radians per position of the r / 2 pairs."""
    if scaling == "ntk":
        _need(r > 2, "this scaling needs a rotary_dim of at least 4")
        base = base * factor ** (r / (r - 2))
    w = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if scaling == "linear":
        return [f / factor for f in w]
    if scaling == "wavelength":
        low, high = 1.0 if low is None else float(low), 4.0 if high is None else float(high)
        _need(0 < low < high, "low must be below high")
        kept = [min(1.0, max(0.0, (length * f / (2 * math.pi) - low) / (high - low))) for f in w]
        return [a * f + (1 - a) * f / factor for a, f in zip(kept, w)]
    if scaling == "yarn":
        low, high = 1.0 if low is None else float(low), 32.0 if high is None else float(high)
        _need(0 < low < high and base > 1, "low must be below high, and base above 1")
        # the (fractional) pair that turns so many times within the length
        first, last = (r * math.log(length / (2 * math.pi * t)) / (2 * math.log(base)) for t in (high, low))
        first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
        ramp = [min(1.0, max(0.0, (i - first) / max(last - first, 0.001))) for i in range(r // 2)]
        return [(1 - a) * f + a * f / factor for a, f in zip(ramp, w)]
    return w


# ------------------------------------------------------------------------------------------------------------ cache
class PagedCache:
    """Keys and values of many sequences in pages of page_size tokens. `keys` and `values` are tensors (n_pages, page_size,
    n_kv_heads, head_dim), or (n_pages, n_kv_heads, page_size, head_dim) with layout="HND"; they are made here, or given (views
    with a dense last axis and 16-byte strides will do, such as the two halves of one tensor). Which page belongs to whom is the
    caller's: page tables (sequences, pages_per_sequence), int32. head_dim is a multiple of 8, at most 256; float32, float16
    or bfloat16. rotary: a `Rotary` that append() turns keys (and queries) with."""

    def __init__(self, n_pages=None, page_size=None, n_kv_heads=None, head_dim=None, dtype=torch.bfloat16, layout="NHD",
                 rotary=None, keys=None, values=None, device="cuda"):
        _need(layout in ("NHD", "HND"), f"layout must be 'NHD' or 'HND', not {layout!r}")
        _need((keys is None) == (values is None), "give both keys and values, or neither")
        if keys is None:
            for v, what in ((n_pages, "n_pages"), (page_size, "page_size"), (n_kv_heads, "n_kv_heads"), (head_dim, "head_dim")):
                _need(v is not None and v >= 1, f"{what} must be positive")
            inner = (page_size, n_kv_heads) if layout == "NHD" else (n_kv_heads, page_size)
            keys, values = (torch.zeros((n_pages, *inner, head_dim), dtype=dtype, device=device) for _ in range(2))
        _need(all(isinstance(t, torch.Tensor) and t.is_cuda and t.ndim == 4 and not t.is_neg() and not t.requires_grad
                  for t in (keys, values)), "keys and values must be CUDA tensors of four axes, without a gradient")
        _need(keys.shape == values.shape and keys.dtype == values.dtype and keys.device == values.device,
              "keys and values must have the same shape, type and device")
        _need(keys.dtype in _KIND, f"a paged cache holds float32, float16 or bfloat16, not {keys.dtype}")
        token, head = (1, 2) if layout == "NHD" else (2, 1)
        self._keys, self._values, self._layout = keys, values, layout
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = (
            keys.shape[0], keys.shape[token], keys.shape[head], keys.shape[3])
        for given, have, what in ((n_pages, self.n_pages, "n_pages"), (page_size, self.page_size, "page_size"),
                                  (n_kv_heads, self.n_kv_heads, "n_kv_heads"), (head_dim, self.head_dim, "head_dim")):
            _need(have >= 1 and (given is None or given == have), f"{what} is {given}, but the pages say {have}")
        self.dtype, self.device = keys.dtype, keys.device
        _need(self.head_dim % 8 == 0 and self.head_dim <= _MOST_DIM,
              f"head_dim must be a multiple of 8 and at most {_MOST_DIM}, not {self.head_dim}")
        self.rotary = rotary
        self._fault = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._bind()

    def _bind(self):
        """What the library is told, with addresses in it."""
        keys, values = self._keys, self._values
        token, head = (1, 2) if self._layout == "NHD" else (2, 1)
        size = keys.element_size()
        for t in (keys, values):
            _need(t.is_cuda and t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s > 0 and s * size % 16 == 0 for s in t.stride()[:3]),
                  "keys and values need a dense last axis and strides of whole 16 bytes, on a CUDA device")
        self._index, self._at = keys.get_device(), (keys.data_ptr(), values.data_ptr())
        self._pages = (keys, values)
        self._needs = {}  # sizes of a call -> bytes of its workspace
        self._args = _CACHE.pack(*self._at,
                                 *(t.stride(i) for t in (keys, values) for i in (0, token, head)), self.n_pages,
                                 self.page_size, self.n_kv_heads, self.head_dim, _KIND[self.dtype], self._fault.data_ptr())

    def __setstate__(self, state):  # a copy, or another process: its tensors lie elsewhere
        self.__dict__.update(state)
        self.device = self._keys.device
        self._bind()

    keys = property(lambda self: self._keys, doc="The pages of keys.")
    values = property(lambda self: self._values, doc="The pages of values.")
    layout = property(lambda self: self._layout, doc='"NHD" or "HND".')

    @property
    def rotary(self):
        """What append() turns keys and queries with, or None."""
        return self._rotary

    @rotary.setter
    def rotary(self, rotary):
        _need(rotary is None or (rotary.head_dim == self.head_dim and rotary.device == self.device),
              "the rotation must be for heads of this size, on this device")
        self._rotary = rotary

    def faulted(self):
        """Whether an index of a call since the last time was out of range (and was left out). Waits for the current stream, and
        speaks for calls that were enqueued there, or that it waited for; what a call on another stream finds meanwhile is in this
        answer or in the next."""
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.faulted()
        was = torch.empty_like(self._fault)
        L.check(L.lib().certexB200PagedTakeFault(L.resources(self._index), self._args, was.data_ptr()))
        return bool(was.item())

    def _unmoved(self):
        """The cache as the library takes it, whose memory must still be where it was."""
        if self._keys.data_ptr() != self._at[0] or self._values.data_ptr() != self._at[1]:
            _fail("the pages were given other memory since this cache was made of them: make a new one")
        return self._args

    def _table(self, page_table, row_to_batch, n):
        try:
            sequences, pages = page_table.shape
            fine = page_table.get_device() == self._index and page_table.dtype is _I32
        except (AttributeError, ValueError):
            fine = False
        if not fine:
            _fail(f"the page table must be an int32 tensor (sequences, pages) on {self.device}")
        if page_table.stride(1) != 1:
            page_table = page_table.contiguous()
        rows = 0
        if row_to_batch is not None:
            row_to_batch = _check_index(row_to_batch, "row_to_batch", (n,), self._index)
            rows = row_to_batch.data_ptr()
        elif sequences != n:
            _fail(f"{n} rows and a table of {sequences} sequences: give row_to_batch")
        args = _TABLE.pack(page_table.data_ptr(), page_table.stride(0), sequences, pages, rows)
        return args, (page_table, row_to_batch)  # what must live until the launch

    def append(self, k, v, page_table, positions, row_to_batch=None, q=None):
        """Stores k, v (n, n_kv_heads, head_dim) at positions (n,) int32 or int64 of their sequences; a negative position is
        padding. With a rotation the keys are turned by their positions first, and q (n, heads, head_dim), if given, is
        returned turned (rows of padding too, by the position as it stands). No two rows have the same place, k and v do not
        lie in places that the call writes, and where the cache's keys and values are the same memory k and v are equal and
        unturned. The keys as they are stored are what a selector wants: `rotary(k, positions)` gives them."""
        _no_gradient(k, v, q)
        if _current_device() != self._index:  # kernels, streams and handles are the current device's
            with torch.cuda.device(self._index):
                return self.append(k, v, page_table, positions, row_to_batch, q)
        k = _check_rows(k, "k", self._index, self.dtype, self.n_kv_heads, self.head_dim)
        v = _check_rows(v, "v", self._index, self.dtype, self.n_kv_heads, self.head_dim)
        n = k.shape[0]
        if v.shape[0] != n:
            _fail(f"{n} keys and {v.shape[0]} values")
        positions = _check_index(positions, "positions", (n,), self._index, True)
        table, alive = self._table(page_table, row_to_batch, n)
        heads, q_in, q_to, turned, rotary = 0, None, None, None, self._rotary
        if q is not None:
            _need(rotary is not None, "queries come along to be turned, but this cache has no rotation")
            q = _check_rows(q, "q", self._index, self.dtype, None, self.head_dim)
            if q.shape[0] != n:
                _fail(f"{n} keys and {q.shape[0]} queries")
            turned = _new_like(q)
            heads = q.shape[1]
            if heads:
                q_in, q_to = _packed(q), _packed(turned)
        if n:
            L.check(L.lib().certexB200PagedAppend(L.resources(self._index), self._unmoved(), rotary._plan if rotary else None, table,
                                                  _packed(k), _packed(v), q_in, q_to, n, heads, positions.data_ptr(),
                                                  positions.dtype is torch.int64))
            _written(self._pages)
        return turned

    def _prepared(self, q, scale, return_lse, out):
        """What both attentions do with their queries: checks, outputs."""
        _no_gradient(q)
        q = _check_rows(q, "q", self._index, self.dtype, None, self.head_dim)
        n, heads, dim = q.shape
        if heads < 1 or heads % self.n_kv_heads:
            _fail(f"{heads} query heads are no multiple of {self.n_kv_heads} KV heads")
        out = _new_like(q) if out is None else _check_out(out, q, False)
        lse = torch.empty((n, heads), dtype=torch.float32, device=self.device) if return_lse else None
        scale = dim ** -0.5 if scale is None else float(scale)
        if not math.isfinite(scale):
            _fail("the scale must be finite")
        return q, out, lse, scale

    @staticmethod
    def _answer(out, lse, given):
        if given is not None:
            _written(out)
        return out if lse is None else (out, lse)

    def _workspace(self, n, heads, lists, k, window):
        """(tensor or None, its address, its bytes): memory for the partial results of one call, of the stream's allocator, so
        that calls on other streams and in captured graphs have their own."""
        sizes = (n, heads, lists, k, window)
        need = self._needs.get(sizes)
        if need is None:
            size = L.ctypes.c_size_t()
            L.check(L.lib().certexB200PagedWorkspace(L.resources(), self._args, *sizes, L.ctypes.byref(size)))
            if len(self._needs) > 1000:
                self._needs.clear()
            need = self._needs[sizes] = size.value
        if not need:
            return None, None, 0
        w = torch.empty(need, dtype=torch.uint8, device=self.device)
        return w, w.data_ptr(), need

    def attend(self, q, page_table, lengths, row_to_batch=None, scale=None, window=None, return_lse=False, out=None):
        """Softmax attention of every row of q (n, heads, head_dim) over the first lengths[i] tokens of its sequence (n,)
        int32, or over the last `window` of those; heads is a multiple of n_kv_heads, query head h reads KV head
        h // (heads / n_kv_heads). scale defaults to head_dim ** -0.5. Returns (n, heads, head_dim), and with return_lse the
        float32 logarithm of the sum of exponentials (n, heads). A row that sees nothing gets zeros and -inf, one whose keys
        all have scores of minus infinity NaN and -inf, as a softmax of them has. Several rows of one sequence (drafted tokens)
        name it in row_to_batch and have their own lengths. out, if given, is written: memory that no other argument and no page
        has."""
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.attend(q, page_table, lengths, row_to_batch, scale, window, return_lse, out)
        given = out
        q, out, lse, scale = self._prepared(q, scale, return_lse, out)
        n, heads, _ = q.shape
        if window is None:
            window = 0
        elif window < 1:
            _fail("window must be positive")
        lengths = _check_index(lengths, "lengths", (n,), self._index)
        table, alive = self._table(page_table, row_to_batch, n)
        if n:
            w, at, size = self._workspace(n, heads, 0, page_table.shape[1] * self.page_size, window)
            L.check(L.lib().certexB200PagedAttend(L.resources(self._index), self._unmoved(), table, lengths.data_ptr(), window, _packed(q),
                                                  _packed(out), n, heads, scale, None if lse is None else lse.data_ptr(), at, size))
        return self._answer(out, lse, given)

    def attend_selected(self, q, selected, scale=None, return_lse=False, out=None):
        """attend() over positions that were selected before: selected (n, heads, k), (n, n_kv_heads, k), (n, 1, k) or (n, k), int32
        or int64, are places of the cache, page * page_size + place, as `flashinfer.ExactTopK.page_table_transform` returns them;
        negative ones are left out, one that is named twice counts twice."""
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.attend_selected(q, selected, scale, return_lse, out)
        given = out
        q, out, lse, scale = self._prepared(q, scale, return_lse, out)
        n, heads, _ = q.shape
        if isinstance(selected, torch.Tensor) and selected.ndim == 2:
            selected = selected[:, None]
        if (not isinstance(selected, torch.Tensor) or selected.ndim != 3 or selected.shape[0] != n
                or selected.shape[1] not in (heads, self.n_kv_heads, 1)):
            _fail(f"selected must have shape ({n}, {heads}, k), ({n}, {self.n_kv_heads}, k), ({n}, 1, k) or ({n}, k)")
        selected = _check_index(selected, "selected", selected.shape, self._index, True)
        lists, k = selected.shape[1:]
        if n:
            w, at, size = self._workspace(n, heads, lists, k, 0)
            L.check(L.lib().certexB200PagedAttendSelected(L.resources(self._index), self._unmoved(), selected.data_ptr(),
                                                          selected.dtype is torch.int64, lists, k, _packed(q), _packed(out), n,
                                                          heads, scale, None if lse is None else lse.data_ptr(), at, size))
        return self._answer(out, lse, given)

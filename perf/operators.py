"""The operators of a decoding step over a paged cache of keys and values, as cases that can be timed and compared: the plain
form of each in elementary torch operations, and the call that a user makes of this package.

  rotary     `Rotary`: queries or keys turned by their positions, forward and (with "grad") backward
  append     `PagedCache.append`: new keys and values go to their pages, keys (and queries) are turned on the way
  attend     `PagedCache.attend`: every row's query heads attend to the first keys of its sequence
  selected   `PagedCache.attend_selected`: every row's heads attend to positions that were chosen before (the exact top k)

`own` says which of the two `run` computes. What a case works on is made from the case and a seed by `prepare`; the lengths of
its sequences belong to the case, so that the work does not depend on the seed. `exact` gives the answers in 64 bits.
"""

import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}


def _rotary(name, n, heads, dim, dtype="bfloat16", rotary_dim=None, interleaved=False, scaling="none", factor=1.0, most=131_072,
            grad=False):
    return {"name": name, "path": "rotary", "n": n, "heads": heads, "dim": dim, "dtype": dtype, "rotary_dim": rotary_dim or dim,
            "interleaved": interleaved, "scaling": scaling, "factor": factor, "most": most, "grad": grad}


def _append(name, sequences, tokens, kv_heads, heads, dim, page, dtype="bfloat16", layout="NHD", rotary_dim=None,
            interleaved=False, most=8192, padding=0):
    """`tokens` new tokens for each sequence, behind up to `most` old ones; `padding` rows of the batch hold no token."""
    return {"name": name, "path": "append", "sequences": sequences, "tokens": tokens, "kv_heads": kv_heads, "heads": heads,
            "dim": dim, "page": page, "dtype": dtype, "layout": layout, "rotary_dim": rotary_dim or dim,
            "interleaved": interleaved, "most": most, "padding": padding}


def _attend(name, sequences, least, most, kv_heads, heads, dim, page, dtype="bfloat16", layout="NHD", rows=1, window=0,
            empty=0, lse=False):
    """`rows` query rows for each sequence (drafted tokens see one key more each); every `empty`-th sequence has no keys."""
    return {"name": name, "path": "attend", "sequences": sequences, "least": least, "most": most, "kv_heads": kv_heads,
            "heads": heads, "dim": dim, "page": page, "dtype": dtype, "layout": layout, "rows": rows, "window": window,
            "empty": empty, "lse": lse}


def _selected(name, sequences, keys, k, kv_heads, heads, dim, page, dtype="bfloat16", layout="NHD", shared="query", lse=False):
    """`shared`: one list of positions for every "query" head, every "kv" head, or "all" heads together."""
    return {"name": name, "path": "selected", "sequences": sequences, "keys": keys, "k": k, "kv_heads": kv_heads, "heads": heads,
            "dim": dim, "page": page, "dtype": dtype, "layout": layout, "shared": shared, "lse": lse}


def listed():
    return [
        # the queries of one decoding step for a batch of 16: latency only
        _rotary("rotary_step", 16, 32, 128),
        # the queries of a long prompt, frequencies stretched for long contexts
        _rotary("rotary_prompt", 32_768, 32, 128, scaling="yarn", factor=8.0),
        # a training step of a model that turns part of every head, in pairs of neighbours: output and gradient
        _rotary("rotary_grad_f32", 4099, 12, 96, "float32", rotary_dim=64, interleaved=True, most=8192, grad=True),
        # one new token for each of 16 sequences, its queries turned by the same call
        _append("append_step", 16, 1, 8, 32, 128, 16),
        # the tokens of four prompts, out of one projection that holds queries, keys and values side by side
        _append("append_prompt", 4, 4096, 8, 32, 128, 16),
        # pages of an odd size with heads outermost, part of the head turned, a batch that is padded
        _append("append_ragged_f16", 37, 75, 3, 0, 96, 7, "float16", "HND", rotary_dim=32, interleaved=True, padding=13),
        # the first tokens of an answer: one sequence, a short prompt
        _attend("attend_short", 1, 200, 200, 8, 32, 128, 16),
        # one sequence with a long context
        _attend("attend_long", 1, 131_072, 131_072, 8, 32, 128, 16, lse=True),
        # a batch of sequences of every length, some of which have no keys yet
        _attend("attend_ragged_f16", 64, 1, 8192, 8, 64, 128, 32, "float16", "HND", empty=9),
        # float32 keys in pages of ten, heads of 80, the last 4096 tokens only
        _attend("attend_window_f32", 6, 500, 20_000, 2, 12, 80, 10, "float32", window=4096, lse=True),
        # the step behind the exact selection of one sequence: 2048 of 131 072 keys for every query head
        _selected("selected_step", 1, 131_072, 2048, 8, 32, 128, 16),
        # the same for a batch of 16 sequences
        _selected("selected_batch", 16, 40_000, 2048, 8, 32, 128, 16, lse=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    path = rng.choice(["rotary", "append", "attend", "attend", "selected"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 8, 16])
    page, layout = rng.choice([1, 5, 16, 32, 64]), rng.choice(["NHD", "HND"])
    token = 2 * kv * dim * _BYTES[dtype]  # bytes of one token's keys and values
    if path == "rotary":
        grad = rng.random() < 0.3
        n = _log(rng, 1, max(1, min(32_768, int(2.4e8 / (heads * dim * _BYTES[dtype] * (2 if grad else 1))))))
        scaling = rng.choice(["none", "linear", "ntk", "wavelength", "yarn"])
        c = _rotary("", n, heads, dim, dtype, rng.choice([dim, dim // 2]), rng.random() < 0.5, scaling,
                    1.0 if scaling == "none" else float(rng.choice([2, 4, 8, 32])), _log(rng, 2048, 1_000_000), grad)
    elif path == "append":
        sequences = _log(rng, 1, 64)
        tokens = rng.choice([1, 1, _log(rng, 2, 4096)])
        heads = rng.choice([0, heads])
        tokens = max(1, min(tokens, int(4e8 / (2 * sequences * (kv * 2 + heads) * dim * _BYTES[dtype]))))
        c = _append("", sequences, tokens, kv, heads, dim, page, dtype, layout, rng.choice([dim, dim // 2]), rng.random() < 0.5,
                    max(1, min(_log(rng, 64, 8192), int(5e8 / (sequences * token)))), rng.choice([0, 0, 5]))
    elif path == "attend":
        sequences = _log(rng, 1, 128)
        most = _log(rng, 64, 131_072)
        # keys of the longest sequence times sequences: what a plain form holds in 32 bits
        most = max(16, min(most, int(5.2e8 / (sequences * token))))
        rows = rng.choice([1, 1, 1, 4])
        most = max(16, most // rows)
        c = _attend("", sequences, rng.choice([1, most // 2 + 1, most]), most, kv, heads, dim, page, dtype, layout, rows,
                    rng.choice([0, 0, 0, most // 3 + 1]), rng.choice([0, 0, 5]), rng.random() < 0.5)
    else:
        shared = rng.choice(["query", "query", "kv", "all"])
        sequences = _log(rng, 1, 16)
        lists = heads if shared == "query" else kv
        k = _log(rng, 16, 2048)
        k = max(1, min(k, int(5.3e8 / (sequences * lists * 2 * dim * _BYTES[dtype]))))
        keys = max(k + 1, min(_log(rng, 2000, 131_072), int(2e9 / (sequences * token))))
        c = _selected("", sequences, keys, k, kv, heads, dim, page, dtype, layout, shared, rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """The number of keys of every sequence: spread over the case's range, the longest among them."""
    r = random.Random(case["sequences"] * 1_000_003 + case["most"])
    lens = [_log(r, case.get("least", 1), case["most"]) for _ in range(case["sequences"])]
    lens[0] = case["most"]
    if case.get("empty"):
        for i in range(1, len(lens), case["empty"]):
            lens[i] = 0
    return lens


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _keys(g, shape, dtype):
    """Keys as they come: normal, with a few channels that are far larger."""
    k = _normal(g, shape, dtype)
    k[..., torch.randperm(shape[-1], generator=g, device="cuda")[:4]] *= 8
    return k


def _cache(g, case, lens):
    """Pages in a random order, the table of every sequence's pages, and twenty pages that nobody has."""
    page, dtype = case["page"], _TYPES[case["dtype"]]
    per = [-(-n // page) for n in lens]
    total, width = sum(per) + 20, max(1, max(per))
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), width), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at : at + n]
        at += n
    inner = (page, case["kv_heads"]) if case["layout"] == "NHD" else (case["kv_heads"], page)
    shape = (total, *inner, case["dim"])
    return {"keys": _keys(g, shape, dtype), "values": _normal(g, shape, dtype), "table": table}


def _plan(case):
    """What a `Rotary` is made from."""
    return {"head_dim": case["dim"], "rotary_dim": case["rotary_dim"], "base": 10000.0, "interleaved": case["interleaved"],
            "scaling": None if case.get("scaling", "none") == "none" else case["scaling"], "factor": case.get("factor", 1.0),
            "original_length": 4096}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    s = {"case": case}
    if case["path"] == "rotary":
        s["x"] = _normal(g, (case["n"], case["heads"], case["dim"]), dtype)
        s["positions"] = torch.randint(0, case["most"], (case["n"],), generator=g, device="cuda", dtype=torch.int32)
        s["dy"] = _normal(g, s["x"].shape, dtype) if case["grad"] else None
        s["x"].requires_grad_(case["grad"])
    elif case["path"] == "append":
        b, t = case["sequences"], case["tokens"]
        old = _lengths(case)
        random.Random(seed).shuffle(old)
        s.update(_cache(g, case, [n + t for n in old]))
        rows, pad = b * t, case["padding"]
        positions = (torch.tensor(old, device="cuda")[:, None] + torch.arange(t, device="cuda")).reshape(-1)
        s["positions"] = torch.cat([positions, positions.new_full((pad,), -1)]).to(torch.int32)
        s["to_batch"] = torch.arange(rows + pad, device="cuda", dtype=torch.int32).div_(t, rounding_mode="floor").clamp_(max=b - 1)
        # one projection's output: the heads of queries, keys and values side by side
        h, kv = case["heads"], case["kv_heads"]
        s["qkv"] = _normal(g, (rows + pad, h + 2 * kv, case["dim"]), dtype)
        s["q"] = s["qkv"][:, :h] if h else None
        s["k"], s["v"] = s["qkv"][:, h : h + kv], s["qkv"][:, h + kv :]
    elif case["path"] == "attend":
        lens = _lengths(case)
        random.Random(seed).shuffle(lens)
        s.update(_cache(g, case, lens))
        m = case["rows"]
        s["q"] = _normal(g, (len(lens) * m, case["heads"], case["dim"]), dtype)
        rows = torch.tensor(lens, device="cuda")[:, None] - torch.arange(m - 1, -1, -1, device="cuda")
        s["lengths"] = rows.reshape(-1).clamp_(min=0).to(torch.int32)
        s["to_batch"] = torch.arange(len(lens), device="cuda", dtype=torch.int32).repeat_interleave(m) if m > 1 else None
    else:
        b, n, k = case["sequences"], case["keys"], case["k"]
        s.update(_cache(g, case, [n] * b))
        s["q"] = _normal(g, (b, case["heads"], case["dim"]), dtype)
        lists = {"query": case["heads"], "kv": case["kv_heads"], "all": 1}[case["shared"]]
        at = torch.stack([torch.rand((lists, n), generator=g, device="cuda").topk(k).indices for _ in range(b)])
        page = s["table"][torch.arange(b, device="cuda")[:, None, None], at // case["page"]]
        s["selected"] = page * case["page"] + (at % case["page"]).to(torch.int32)
        s["selected"][:, ::5, k - k // 7 :] = -1  # lists that are not full
    if own:
        import libcertex_b200 as certex

        if case["path"] in ("rotary", "append"):
            s["rotary"] = certex.Rotary(**_plan(case))
        if "keys" in s:
            s["cache"] = certex.PagedCache(keys=s["keys"], values=s["values"], layout=case["layout"], rotary=s.get("rotary"))
    elif case["path"] in ("rotary", "append"):
        s["frequencies"], s["magnitude"] = _frequencies(_plan(case))
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _frequencies(plan):
    """Radians per position of every pair, in 64 bits, and the factor on the result."""
    r, base, f, length = plan["rotary_dim"], plan["base"], plan["factor"], plan["original_length"]
    i = torch.arange(0, r, 2, device="cuda", dtype=torch.float64)
    magnitude = 1.0
    if plan["scaling"] == "ntk":
        base = base * f ** (r / (r - 2))
    w = base ** (-i / r)
    if plan["scaling"] == "linear":
        w = w / f
    elif plan["scaling"] == "wavelength":
        turns = length * w / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        w = keep * w + (1 - keep) * w / f
    elif plan["scaling"] == "yarn":
        edge = [r * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), r - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        w = (1 - ramp) * w + ramp * w / f
        magnitude = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
    return w, magnitude


def _turn(x, positions, frequencies, magnitude, interleaved, backward=False):
    """x (n, heads, dim), any type, turned in 32 bits by angles in 64, rounded once."""
    a = positions.double()[:, None, None] * frequencies
    c, s = (a.cos() * magnitude).float(), (a.sin() * magnitude).float()
    s = -s if backward else s
    r = 2 * len(frequencies)
    x = x.detach()
    y = x.float()
    p, q = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., : r // 2], y[..., r // 2 : r])
    u, v = p * c - q * s, q * c + p * s
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, y[..., r:]], -1).to(x.dtype)


def _softmax_sum(q, k, v, keep, scale):
    """q (r, h, g, d); k, v (r, h, t, d); keep (r, h, t) or (r, 1, t): the weighted sum of the kept values, and log-sum-exp."""
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    s = s.masked_fill(~keep[:, :, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).min)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    return out, (top + total.log()).squeeze(-1)


def _by_token(pages, layout):
    """Pages as (page, token, head, dim)."""
    return pages if layout == "NHD" else pages.transpose(1, 2)


def _gathered(s, kind):
    """Keys and values of every row's sequence, (rows, heads, tokens, dim) in `kind`, with what the row may see."""
    case, table = s["case"], s["table"] if s["to_batch"] is None else s["table"][s["to_batch"].long()]
    t = torch.arange(table.shape[1] * case["page"], device="cuda")[: case["most"]]
    page = table[:, t // case["page"]].long()
    n = s["lengths"].long()[:, None]
    keep = t < n
    if case["window"]:
        keep = keep & (t >= n - case["window"])
    both = [_by_token(s[x], case["layout"])[page, t % case["page"]].to(kind).masked_fill_(~keep[..., None, None], 0).transpose(1, 2)
            for x in ("keys", "values")]
    return both[0], both[1], keep[:, None]


def _chosen(s, kind):
    """Keys and values that were chosen, (rows, lists, k, dim) in `kind`; a list for all heads counts for every KV head."""
    case, at = s["case"], s["selected"]
    if at.shape[1] == 1:
        at = at.expand(-1, case["kv_heads"], -1)
    head = torch.arange(at.shape[1], device="cuda") // (at.shape[1] // case["kv_heads"])
    place = at.clamp(min=0).long()
    both = [_by_token(s[x], case["layout"])[place // case["page"], place % case["page"], head[:, None]].to(kind) for x in ("keys", "values")]
    return both[0], both[1], at >= 0


def _answer(out, lse, q, case):
    out = out.reshape(q.shape).to(q.dtype)
    return (out, lse.reshape(q.shape[:2])) if case["lse"] else out


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["path"] == "rotary":
        turn = (s["positions"], s["frequencies"], s["magnitude"], case["interleaved"])
        y = _turn(s["x"], *turn)
        return (y, _turn(s["dy"], *turn, backward=True)) if case["grad"] else y
    if case["path"] == "append":
        turn = (s["positions"], s["frequencies"], s["magnitude"], case["interleaved"])
        k = _turn(s["k"], *turn)
        real = s["positions"] >= 0
        p = s["positions"][real].long()
        page = s["table"][s["to_batch"][real].long(), p // case["page"]].long()
        _by_token(s["keys"], case["layout"])[page, p % case["page"]] = k[real]
        _by_token(s["values"], case["layout"])[page, p % case["page"]] = s["v"][real]
        return (s["keys"], s["values"], _turn(s["q"], *turn)) if case["heads"] else (s["keys"], s["values"])
    q = s["q"]
    k, v, keep = _gathered(s, torch.float32) if case["path"] == "attend" else _chosen(s, torch.float32)
    out, lse = _softmax_sum(q.float().reshape(q.shape[0], k.shape[1], -1, q.shape[2]), k, v, keep, q.shape[2] ** -0.5)
    return _answer(out, lse, q, case)


def _run_own(s, case):
    if case["path"] == "rotary":
        y = s["rotary"](s["x"], s["positions"])
        return (y, *torch.autograd.grad(y, s["x"], s["dy"])) if case["grad"] else y
    if case["path"] == "append":
        q = s["cache"].append(s["k"], s["v"], s["table"], s["positions"], row_to_batch=s["to_batch"], q=s["q"])
        return (s["keys"], s["values"], q) if case["heads"] else (s["keys"], s["values"])
    if case["path"] == "attend":
        return s["cache"].attend(s["q"], s["table"], s["lengths"], row_to_batch=s["to_batch"], window=case["window"] or None,
                                 return_lse=case["lse"])
    return s["cache"].attend_selected(s["q"], s["selected"], return_lse=case["lse"])


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _exact_turn(x, positions, plan, sign=1.0):
    """The rotation as a product of complex numbers, in numpy's 64 bits; angles from frequencies made one by one."""
    r = plan["rotary_dim"]
    f, length = plan["factor"], plan["original_length"]
    base = plan["base"] * (f ** (r / (r - 2)) if plan["scaling"] == "ntk" else 1.0)
    magnitude, w = 1.0, []
    if plan["scaling"] == "yarn" and f > 1:
        magnitude = 1.0 + math.log(f) / 10
    for i in range(r // 2):
        one = math.exp(-2 * i / r * math.log(base))
        if plan["scaling"] == "linear":
            one /= f
        if plan["scaling"] == "wavelength":
            wave = 2 * math.pi / one
            share = 1.0 if wave < length / 4 else 0.0 if wave > length else (length / wave - 1) / 3
            one = share * one + (1 - share) * one / f
        if plan["scaling"] == "yarn":
            lo = max(0, math.floor(r * math.log(length / (32 * 2 * math.pi)) / (2 * math.log(base))))
            hi = min(r - 1, math.ceil(r * math.log(length / (2 * math.pi)) / (2 * math.log(base))))
            share = 1 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            one = share * one + (1 - share) * one / f
        w.append(one)
    angle = positions.double()[:, None] * torch.from_numpy(np.array(w)).cuda()
    turn = torch.polar(torch.full_like(angle, magnitude), sign * angle)[:, None]
    y = x.detach().double().clone()
    if plan["interleaved"]:
        z = torch.view_as_complex(y[..., :r].reshape(*y.shape[:-1], r // 2, 2).contiguous()) * turn
        y[..., :r] = torch.view_as_real(z).reshape(*y.shape[:-1], r)
    else:
        z = torch.complex(y[..., : r // 2].contiguous(), y[..., r // 2 : r].contiguous()) * turn
        y[..., : r // 2], y[..., r // 2 : r] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] == "rotary":
        y = _exact_turn(s["x"], s["positions"], _plan(case))
        return (y, _exact_turn(s["dy"], s["positions"], _plan(case), -1.0)) if case["grad"] else y
    if case["path"] == "append":
        k = _exact_turn(s["k"], s["positions"], _plan(case))
        keys, values = s["keys"].double(), s["values"].double()
        table = s["table"].cpu().numpy()
        where, what = [], []
        for i, (b, p) in enumerate(zip(s["to_batch"].tolist(), s["positions"].tolist())):
            if p >= 0:
                where.append(int(table[b, p // case["page"]]) * case["page"] + p % case["page"])
                what.append(i)
        where, what = torch.tensor(where, device="cuda"), torch.tensor(what, device="cuda")
        for pages, new in ((keys, k), (values, s["v"].double())):
            flat = _by_token(pages, case["layout"]).reshape(-1, case["kv_heads"], case["dim"])
            flat = flat.index_copy(0, where, new[what])
            flat = flat.reshape(-1, case["page"], case["kv_heads"], case["dim"])
            pages.copy_(flat if case["layout"] == "NHD" else flat.transpose(1, 2))
        return (keys, values, _exact_turn(s["q"], s["positions"], _plan(case))) if case["heads"] else (keys, values)
    # row by row and head by head over the tokens that count, nothing padded
    q, group = s["q"].double(), case["heads"] // case["kv_heads"]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    pages = {x: _by_token(s[x], case["layout"]) for x in ("keys", "values")}
    for i in range(q.shape[0]):
        if case["path"] == "attend":
            b = i if s["to_batch"] is None else int(s["to_batch"][i])
            n = int(s["lengths"][i])
            t = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
            lists = [(s["table"][b].long()[t // case["page"]], t % case["page"])]
        else:
            lists = [(at[at >= 0].long() // case["page"], at[at >= 0].long() % case["page"]) for at in s["selected"][i]]
        for h in range(case["heads"]):
            page, place = lists[h * len(lists) // case["heads"]]
            if len(page) == 0:
                continue
            k, v = (pages[x][page, place, h // group].double() for x in ("keys", "values"))
            x = (k * q[i, h]).sum(-1) / math.sqrt(case["dim"])
            lse[i, h] = torch.logsumexp(x, 0)
            out[i, h] = (torch.exp(x - lse[i, h])[:, None] * v).sum(0)
    return (out, lse) if case["lse"] else out


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    """Inputs read once, outputs written once; two operations for a product and its sum."""
    size, d, h = _BYTES[case["dtype"]], case["dim"], case["heads"]
    if case["path"] == "rotary":
        n = case["n"] * h * d * (2 if case["grad"] else 1)
        return {"bytes": 2 * n * size + 4 * case["n"], "flops": 3 * n}
    kv = case["kv_heads"]
    if case["path"] == "append":
        rows = case["sequences"] * case["tokens"]
        moved = rows * (2 * kv + h) * d
        return {"bytes": 2 * moved * size + 8 * rows, "flops": 3 * rows * (kv + h) * d}
    if case["path"] == "attend":
        seen = [[max(0, n - j) for j in range(case["rows"])] for n in _lengths(case)]
        cut = (lambda n: min(n, case["window"])) if case["window"] else (lambda n: n)
        read, used = sum(max(map(cut, n)) for n in seen), sum(sum(map(cut, n)) for n in seen)
        rows = case["sequences"] * case["rows"]
        return {"bytes": (2 * read * kv * d + 2 * rows * h * d) * size + 4 * -(-read // case["page"]), "flops": 4 * used * h * d}
    rows, n, k = case["sequences"], case["keys"], case["k"]
    lists = {"query": h, "kv": kv, "all": 1}[case["shared"]]
    short = -(-lists // 5)
    entries = rows * (lists * k - short * (k // 7))
    # keys that several lists of one KV head name are read once: what that leaves of random lists
    each = max(1, lists // kv)
    distinct = rows * kv * n * (1 - (1 - entries / (rows * lists) / n) ** each)
    return {"bytes": (2 * distinct * d + 2 * rows * h * d) * size + 4 * rows * lists * k,
            "flops": 4 * entries * (h // lists) * d}

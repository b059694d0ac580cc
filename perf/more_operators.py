"""Operators for serving from a paged cache, each as a user of the package
calls it (``own``) and in its plain form (elementary torch operations in 32
bits, rounded once at the end).

A case is a dict of plain values.  ``op`` names the operator:

* ``append``  the way of new tokens' keys and values into the pages: norms of
  the query and key heads, the rotary embedding (of the whole head or of its
  first ``rot`` elements, in either layout), the queries out.  With ``bits`` 8
  the pages hold 8-bit floats with a power of two for each page and head, and
  the pass ends with the dense values that the sequences' pages stand for, as
  a program takes them to look at or to move;
* ``attend``  attention of the newest tokens of every sequence over its pages,
  with a window and first tokens that stay visible where the case has them.

Sizes are those of the 8B-shaped model of :mod:`nibblegemm_amd.decode_step`
(32 query heads on 8, head size 128) and generic ragged ones.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
THETA = 500000.0
#: Largest 8-bit float (four exponent bits, three mantissa bits).
E4M3_MAX = 448.0


def listed():
    llama = {"kv": 8, "qpk": 4, "D": 128}
    return [
        # The token of one decode step: the smallest call.
        {"name": "append_token", "op": "append", "B": 1, "T": 1, **llama, "ctx": 1000, "page": 16,
         "bits": 16, "layout": "head", "dtype": "float16", "norm": False, "rot": 128,
         "interleaved": False},
        # Four prompts' next parts at once, pages with a row's heads side by side.
        {"name": "append_prompts", "op": "append", "B": 4, "T": 2000, **llama, "ctx": 500,
         "page": 64, "bits": 16, "layout": "row", "dtype": "bfloat16", "norm": True, "rot": 64,
         "interleaved": True},
        # The tokens of 64 young conversations into an 8-bit cache.
        {"name": "append_batch_8bit", "op": "append", "B": 64, "T": 1, **llama, "ctx": 200,
         "page": 32, "bits": 8, "layout": "head", "dtype": "float16", "norm": False, "rot": 128,
         "interleaved": False},
        # Prompts into an 8-bit cache.
        {"name": "append_prompts_8bit", "op": "append", "B": 4, "T": 2000, **llama, "ctx": 100,
         "page": 64, "bits": 8, "layout": "head", "dtype": "bfloat16", "norm": True, "rot": 128,
         "interleaved": False},
        # One conversation's decode step.
        {"name": "decode_1", "op": "attend", "B": 1, "T": 1, **llama, "ctx": 4000, "page": 16,
         "bits": 16, "layout": "head", "dtype": "float16", "window": 0, "sinks": 0},
        # The same far into a very long one.
        {"name": "decode_1_long", "op": "attend", "B": 1, "T": 1, **llama, "ctx": 65000,
         "page": 256, "bits": 16, "layout": "head", "dtype": "bfloat16", "window": 0, "sinks": 0},
        # The decode step of 32 conversations on an 8-bit cache.
        {"name": "decode_32_8bit", "op": "attend", "B": 32, "T": 1, **llama, "ctx": 8100,
         "page": 64, "bits": 8, "layout": "head", "dtype": "bfloat16", "window": 0, "sinks": 0},
        # Conversations that outgrew a window, its pages alone kept.
        {"name": "decode_window_8bit", "op": "attend", "B": 16, "T": 1, **llama, "ctx": 16000,
         "page": 16, "bits": 8, "layout": "row", "dtype": "float16", "window": 4000, "sinks": 4},
        # Short runs of tokens of some sequences together, heads of 64.
        {"name": "ragged_60", "op": "attend", "B": 7, "T": 60, "kv": 2, "qpk": 5, "D": 64,
         "ctx": 2003, "page": 32, "bits": 16, "layout": "row", "dtype": "float16", "window": 0,
         "sinks": 0},
        # The second half of a prompt.
        {"name": "prompt_2048", "op": "attend", "B": 1, "T": 2048, **llama, "ctx": 2048,
         "page": 64, "bits": 16, "layout": "head", "dtype": "bfloat16", "window": 0, "sinks": 0},
        # Parts of two prompts over an 8-bit cache.
        {"name": "prompts_8bit", "op": "attend", "B": 2, "T": 1000, **llama, "ctx": 3001,
         "page": 32, "bits": 8, "layout": "head", "dtype": "float16", "window": 0, "sinks": 0},
        # A whole prompt under a window.
        {"name": "prompt_window", "op": "attend", "B": 1, "T": 4096, **llama, "ctx": 0,
         "page": 64, "bits": 16, "layout": "head", "dtype": "bfloat16", "window": 1000,
         "sinks": 4},
    ]


# ---------------------------------------------------------------- drawn cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    case = {"op": rng.choice(["append", "attend", "attend"]), "B": _log_int(rng, 1, 64),
            "T": rng.choice([1, _log_int(rng, 1, 4096)]), "kv": rng.choice([1, 2, 4, 8]),
            "qpk": rng.choice([1, 2, 4, 5, 8]), "D": rng.choice([64, 128, 128]),
            "ctx": _log_int(rng, 1, 65000) - 1, "page": rng.choice([16, 32, 64, 128, 256]),
            "bits": rng.choice([16, 8]), "layout": rng.choice(["head", "row"]),
            "dtype": rng.choice(["float16", "bfloat16"])}
    if case["op"] == "append":
        return {**case, "norm": rng.random() < 0.5, "interleaved": rng.random() < 0.3,
                "rot": rng.choice([0, 32, case["D"] // 2, case["D"], case["D"]])}
    window = rng.random() < 0.4
    return {**case, "window": _log_int(rng, 16, 8192) if window else 0,
            "sinks": rng.choice([0, 1, 4, _log_int(rng, 1, 200)]) if window else 0}


def _rows(case):
    """Rows that a sequence's pages have room for."""
    return -(-(case["ctx"] + case["T"]) // case["page"]) * case["page"]


def _plain_size(case):
    """Values of the plain form's caches and of its scores."""
    dense = case["B"] * case["kv"] * _rows(case) * case["D"]
    scores = case["B"] * case["kv"] * case["qpk"] * case["T"] * _rows(case)
    return dense, scores if case["op"] == "attend" else 0


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = [max(a, b) for a, b in zip(most.get(c["op"], (0, 0, 0, 0)),
                                                   (w["bytes"], w["flops"], *_plain_size(c)))]
    while True:
        case = _draw(rng)
        w = work(case)
        size = (w["bytes"], w["flops"], *_plain_size(case))
        if all(a <= b for a, b in zip(size, most[case["op"]])):
            return case


# --------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _lengths(case):
    """Cached tokens of each sequence before this call: the longest is ``ctx``."""
    return [int(case["ctx"] * (1 - 0.75 * ((b * 0.618034) % 1.0))) for b in range(case["B"])]


def _sizes(case):
    """New tokens of each sequence: the largest has ``T``."""
    return [max(1, case["T"] - (b * 5) % max(1, case["T"] // 2)) for b in range(case["B"])]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(case, gen):
    """Pages, in any order, of the rows that a sequence has or gets; under a
    window those alone that some token still sees."""
    B, P = case["B"], case["page"]
    M = _rows(case) // P
    order = torch.randperm(B * M + 3, generator=gen, device="cuda")[:B * M].view(B, M)
    first = torch.arange(M, device="cuda") * P
    lengths = _ints(_lengths(case))[:, None]
    there = first < lengths + _ints(_sizes(case))[:, None]
    if case.get("window"):
        there &= (first + P > lengths - case["window"] + 1) | (first < case["sinks"])
    return torch.where(there, order, -1).to(torch.int32)


def _pages(case, gen):
    """Keys or values that earlier calls left, and, of 8-bit ones, their scales
    (biased exponents): of channels that differ, in pages that differ."""
    B, kv, P, D = (case[k] for k in ("B", "kv", "page", "D"))
    n = B * (_rows(case) // P) + 3
    dtype = getattr(torch, case["dtype"])
    shape = (n, kv, P, D) if case["layout"] == "head" else (n, P, kv, D)
    x = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    x *= torch.where(torch.rand(D, generator=gen, device="cuda") < 0.03, 3.0, 1.0).to(dtype)
    x = x if case["layout"] == "head" else x.transpose(1, 2)
    if case["bits"] == 16:
        return x, None
    x *= torch.exp2(torch.randint(-1, 2, (n, 1, 1, 1), generator=gen, device="cuda")).to(dtype)
    e = _exponents(x.abs().amax((2, 3)), dtype)
    codes = (x * _power(254 - e)[..., None, None].to(dtype)).to(torch.float8_e4m3fn)
    return codes, e.to(torch.uint8)


def prepare(case, seed):
    gen = _gen(seed)
    B, T, D = case["B"], case["T"], case["D"]
    dtype = getattr(torch, case["dtype"])
    heads = case["kv"] * case["qpk"]
    (k, ks), (v, vs) = _pages(case, gen), _pages(case, gen)
    state = {"case": case, "k": k, "v": v, "scales": (ks, vs) if ks is not None else None,
             "table": _table(case, gen), "lengths": _ints(_lengths(case)),
             "sizes": _ints(_sizes(case))}
    if case["op"] == "attend":
        return {**state, "q": (2 * _randn(gen, B, T, heads * D)).to(dtype)}
    rot = case["rot"]
    rope = None
    if rot:
        inv = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        angle = torch.outer(torch.arange(_rows(case), dtype=torch.float64, device="cuda"), inv)
        rope = (angle.cos().float(), angle.sin().float())
    norms = [(1 + 0.1 * _randn(gen, D)).to(dtype) for _ in range(2)]
    return {**state, "qkv": _randn(gen, B, T, (heads + 2 * case["kv"]) * D).to(dtype),
            "norms": norms if case["norm"] else [None, None], "rope": rope,
            # what the sequences hold afterwards
            "ends": state["lengths"] + state["sizes"]}


# ------------------------------------------------------------- the plain forms

def _exponents(top, dtype):
    """Biased exponents of the least power of two that ``top`` fits under as an
    8-bit float, as far as the 8-bit floats times it are values of ``dtype``
    too."""
    m, x = torch.frexp(top.double() / E4M3_MAX)
    e = torch.where(m > 0.5, x, x - 1)
    low, high = (-15, 8) if dtype == torch.float16 else (-117, 120)
    return 127 + torch.where(top > 0, e, low).clamp(low, high)


def _power(e):
    """2^(e - 127), exact (an exponential's is not on every device)."""
    return ((e.long() + (1023 - 127)) << 52).view(torch.float64).float()


def _dense(pages, scales, table):
    """The rows of every sequence, ``[B, kv, rows, D]`` in 32 bits; zeros where
    there is no page."""
    at = table.clamp(min=0).long()
    x = pages[at].float()  # [B, M, kv, P, D]
    if scales is not None:
        x = x * _power(scales[at])[..., None, None]
    x = torch.where((table >= 0)[:, :, None, None, None], x, 0.0)
    return x.transpose(1, 2).flatten(2, 3)


def _turned(x, w, rope, at, interleaved):
    """Heads ``x`` ``[B, T, heads, D]`` normalised and rotated."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    if rope is None:
        return x
    cos, sin = (t[at.clamp(max=t.shape[0] - 1)][:, :, None] for t in rope)
    R = 2 * cos.shape[-1]
    if interleaved:
        lo, hi = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([lo * cos - hi * sin, hi * cos + lo * sin], -1).flatten(-2)
    else:
        lo, hi = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _append_8(pages, scales, table, lengths, live, at, y, dtype):
    """Rows ``y`` ``[B, T, kv, D]`` quantised into the pages: a page that begins
    with one takes their scale, another the larger of its own and theirs, its
    earlier rows rescaled to it."""
    B, M = table.shape
    P = pages.shape[2]
    page = table.clamp(min=0).long()
    rows = torch.zeros((B, M * P, *y.shape[2:]), device=y.device)
    new = torch.zeros((B, M * P), dtype=torch.bool, device=y.device)
    b, t = live.nonzero(as_tuple=True)
    rows[b, at[b, t]], new[b, at[b, t]] = y[b, t], True
    rows = rows.unflatten(1, (M, P)).transpose(2, 3)  # [B, M, kv, P, D]
    new = new.unflatten(1, (M, P))
    first = torch.arange(M, device=y.device) * P
    need = _exponents(rows.abs().amax((3, 4)), dtype)
    was = scales[page].long()
    fresh = (first >= lengths[:, None])[..., None]
    e = torch.where(fresh, need, torch.maximum(need, was))
    old = pages[page].float()
    earlier = (first[:, None] + torch.arange(P, device=y.device) < lengths[:, None, None])
    new, earlier = new[:, :, None, :, None], earlier[:, :, None, :, None]
    scaled = torch.where(new, rows / _power(e)[..., None, None],
                         old * _power(was - e + 127)[..., None, None])
    codes = torch.where(new | earlier, scaled.clamp(-E4M3_MAX, E4M3_MAX), old)
    b, m = new.flatten(2).any(-1).nonzero(as_tuple=True)
    pages[page[b, m]] = codes[b, m].to(pages.dtype)
    scales[page[b, m]] = e[b, m].to(torch.uint8)


def _plain_append(s):
    c, table = s["case"], s["table"]
    B, T, kv, D, P = (c[k] for k in ("B", "T", "kv", "D", "page"))
    x = s["qkv"].view(B, T, -1, D)
    n_q = x.shape[2] - 2 * kv
    lengths = s["lengths"].long()
    t = torch.arange(T, device=x.device)
    at = lengths[:, None] + t
    live = t < s["sizes"][:, None]
    q = _turned(x[:, :, :n_q].float(), s["norms"][0], s["rope"], at, c["interleaved"])
    k = _turned(x[:, :, n_q:n_q + kv].float(), s["norms"][1], s["rope"], at, c["interleaved"])
    v = x[:, :, n_q + kv:]
    q = torch.where(live[:, :, None, None], q, 0.0).to(x.dtype).view(B, T, n_q * D)
    if s["scales"] is None:
        b, t = live.nonzero(as_tuple=True)
        row = at[b, t]
        page = table[b, row // P].long()
        s["k"][page, :, row % P] = k[b, t].to(x.dtype)
        s["v"][page, :, row % P] = v[b, t]
        return [q, s["k"], s["v"]]
    out = [q]
    held = torch.arange(_rows(c), device=x.device) < s["ends"][:, None]
    for pages, scales, y in ((s["k"], s["scales"][0], k), (s["v"], s["scales"][1], v.float())):
        _append_8(pages, scales, table, lengths, live, at, y, x.dtype)
        dense = _dense(pages, scales, table)
        out.append(torch.where(held[:, None, :, None], dense, 0.0).to(x.dtype))
    return out


def _plain_attend(s):
    c = s["case"]
    B, T, kv, D = (c[k] for k in ("B", "T", "kv", "D"))
    ks, vs = s["scales"] or (None, None)
    k, v = _dense(s["k"], ks, s["table"]), _dense(s["v"], vs, s["table"])
    S = k.shape[2]
    q = s["q"].float().view(B, T, kv, -1, D).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, D)
    score = q @ k.transpose(2, 3).contiguous() / math.sqrt(D)  # rows (head, token)
    score = score.view(B, kv, -1, T, S)
    j = torch.arange(S, device=q.device)
    i = torch.arange(T, device=q.device)[:, None]
    at = s["lengths"].long()[:, None, None] + i
    there = (s["table"] >= 0).repeat_interleave(c["page"], 1)[:, None]
    seen = (j <= at) & (i < s["sizes"][:, None, None]) & there  # [B, T, S]
    if c["window"]:
        seen &= (j > at - c["window"]) | (j < c["sinks"])
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    out = p.view(B, kv, -1, S) @ v
    return out.view(B, kv, -1, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, -1).to(s["q"].dtype)


# ------------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain_append(s) if c["op"] == "append" else _plain_attend(s)
    from nibblegemm_amd import paged
    if c["op"] == "attend":
        return paged.attention_paged(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["sizes"],
                                     window=c["window"] or None, sinks=c["sinks"],
                                     scales=s["scales"])
    q = paged.paged_append(s["qkv"], s["k"], s["v"], s["table"], s["lengths"], s["sizes"],
                           q_weight=s["norms"][0], k_weight=s["norms"][1], eps=EPS,
                           rope=s["rope"], interleaved=c["interleaved"], scales=s["scales"])
    if s["scales"] is None:
        return [q, s["k"], s["v"]]
    return [q, *paged.paged_values(s["k"], s["v"], s["table"], s["ends"], s["scales"], q.dtype)]


# ------------------------------------------- what a pass cannot do without

def work(case):
    kv, D, heads = case["kv"], case["D"], case["kv"] * case["qpk"]
    lengths, sizes = np.array(_lengths(case)), np.array(_sizes(case))
    element = case["bits"] // 8
    if case["op"] == "append":
        tokens, padded = int(sizes.sum()), case["B"] * case["T"]
        rope = min(_rows(case), tokens) * case["rot"] * 4
        moved = tokens * ((heads + 2 * kv) * D * 2 + 2 * kv * D * element) + padded * heads * D * 2
        if case["bits"] == 8:  # the rows' codes read, their dense values written
            moved += int((lengths + sizes).sum()) * 2 * kv * D
            moved += case["B"] * _rows(case) * 2 * kv * D * 2
        return {"bytes": moved + rope, "flops": tokens * (heads + kv) * D * 7}
    rows = pairs = 0
    for n, t in zip(lengths.tolist(), sizes.tolist()):
        end = n + 1 + np.arange(t)
        begin = np.maximum(0, end - case["window"]) if case["window"] else 0 * end
        pairs += int((end - begin + np.minimum(case["sinks"], begin)).sum())
        rows += n + t - int(begin[0]) + min(case["sinks"], int(begin[0]))
    return {"bytes": rows * 2 * kv * D * element + int(sizes.sum()) * heads * D * 2
            + case["B"] * case["T"] * heads * D * 2, "flops": pairs * heads * D * 4}


# ----------------------------------------------- the same in 64-bit arithmetic

def _ldexp64(x, n):
    """``x 2^n``, exact (torch's takes a power that is not on every device)."""
    powers = torch.from_numpy(np.ldexp(1.0, np.arange(-300, 301))).to(x.device)
    return x * powers[n.long() + 300]


def _sequence64(s, which, b):
    """A sequence's rows ``[rows, kv, D]``, NaN where there is no page."""
    pages, P = s[which], s["case"]["page"]
    out = torch.full((s["table"].shape[1] * P, pages.shape[1], pages.shape[3]), math.nan,
                     dtype=torch.float64, device=pages.device)
    for m, page in enumerate(s["table"][b].tolist()):
        if page >= 0:
            x = pages[page].double()
            if s["scales"] is not None:
                e = s["scales"][0 if which == "k" else 1][page].long() - 127
                x = _ldexp64(x, e[:, None, None])
            out[m * P:(m + 1) * P] = x.transpose(0, 1)
    return out


def _exact_attend(s):
    c = s["case"]
    B, T, kv, D = (c[k] for k in ("B", "T", "kv", "D"))
    q = s["q"].double().view(B, T, kv, -1, D)
    out = torch.zeros_like(q)
    for b, (n, t) in enumerate(zip(_lengths(c), _sizes(c))):
        k, v = (_sequence64(s, which, b)[:n + t] for which in "kv")
        held = ~k[:, 0, 0].isnan()
        j = torch.arange(n + t, device=q.device)[held]
        back = torch.arange(n, n + t, device=q.device)[:, None] - j
        hidden = back < 0
        if c["window"]:
            hidden |= (back >= c["window"]) & (j >= c["sinks"])
        for h in range(kv):
            kh, vh = k[held, h], v[held, h]
            score = torch.matmul(q[b, :t, h].reshape(-1, D), kh.t()).view(t, -1, len(j))
            score = (score * D ** -0.5).masked_fill_(hidden[:, None], -math.inf)
            p = torch.softmax(score, -1)
            out[b, :t, h] = torch.matmul(p.flatten(0, 1), vh).view(t, -1, D)
    return out.view(B, T, -1)


def _grid64(u):
    """The nearest 8-bit floats, ties to the even one."""
    _, ex = torch.frexp(u.abs())
    step = _ldexp64(torch.ones_like(u), ex.clamp(min=-5) - 4)
    return torch.round(u / step) * step


def _write64(s, which, y, dtype):
    """New rows ``y`` ``[B, T, kv, D]`` in an 8-bit cache: the sequences' dense
    values afterwards."""
    c = s["case"]
    P, low = c["page"], -15 if dtype == torch.float16 else -117
    codes = s[which].double()
    scales = s["scales"][0 if which == "k" else 1].long() - 127
    out = torch.zeros((c["B"], c["kv"], _rows(c), c["D"]), dtype=torch.float64, device=y.device)
    for b, (n, t) in enumerate(zip(_lengths(c), _sizes(c))):
        for m, page in enumerate(s["table"][b].tolist()):
            if m * P >= n + t:
                break
            stop = min(P, n + t - m * P)  # rows of the page that are held
            begin = max(0, min(n - m * P, stop))  # its first new one
            held, e = codes[page, :, :stop], scales[page]
            if begin < stop:
                fresh = y[b, m * P + begin - n:m * P + stop - n].transpose(0, 1)
                top = fresh.abs().amax((1, 2))
                powers = _ldexp64(E4M3_MAX + 0 * top[:, None], torch.arange(low, 121,
                                                                            device=y.device))
                need = low + (powers < top[:, None]).sum(1)
                to = need if begin == 0 else torch.maximum(need, e)
                moved = _ldexp64(held[:, :begin], (e - to)[:, None, None])
                written = _ldexp64(fresh, -to[:, None, None])
                held, e = _grid64(torch.cat([moved, written], 1)), to
            out[b, :, m * P:m * P + stop] = _ldexp64(held, e[:, None, None])
    return out


def _exact_append(s):
    c = s["case"]
    kv, D, P, R = c["kv"], c["D"], c["page"], c["rot"]
    x = s["qkv"].double().unflatten(2, (-1, D))
    n_q = x.shape[2] - 2 * kv
    turned = x[:, :, :n_q + kv].clone()
    for part, w in ((slice(0, n_q), s["norms"][0]), (slice(n_q, n_q + kv), s["norms"][1])):
        if w is not None:
            h = turned[:, :, part]
            turned[:, :, part] = h / (h.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
    if R:
        row = s["lengths"].long()[:, None] + torch.arange(c["T"], device=x.device)
        cos, sin = (t.double()[row.clamp(max=len(t) - 1)].unsqueeze(2) for t in s["rope"])
        a, b = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else \
            (slice(0, R // 2), slice(R // 2, R))
        z = torch.complex(turned[..., a], turned[..., b]) * torch.complex(cos, sin)
        turned[..., a], turned[..., b] = z.real, z.imag
    q = turned[:, :, :n_q].clone()
    for b, t in enumerate(_sizes(c)):
        q[b, t:] = 0
    new = {"k": turned[:, :, n_q:], "v": x[:, :, n_q + kv:]}
    if s["scales"] is not None:
        return [q.flatten(2)] + [_write64(s, which, new[which], s["qkv"].dtype) for which in "kv"]
    out = {which: s[which].double() for which in "kv"}
    for b, (n, t) in enumerate(zip(_lengths(c), _sizes(c))):
        row = torch.arange(n, n + t, device=x.device)
        page = s["table"][b, row // P].long()
        for which in "kv":
            out[which][page, :, row % P] = new[which][b, :t]
    return [q.flatten(2), out["k"], out["v"]]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)

"""Operators for serving on 4-bit floating-point weights and with drafted
tokens, each as a user of the package calls it (``own``) and in its plain form
(elementary torch operations in 32 bits, rounded once at the end).

A case is a dict of plain values.  ``op`` names the operator:

* ``quantize``  a matrix to microscaled 4-bit floats (blocks of 32 along a row
  share a power of two) and back to the values they stand for;
* ``matmul``    a product of two such matrices, ``x w^T``; ``x`` either dense
  (quantised within the call) or quantised already;
* ``qk_norm``   RMSNorm of every query and key head, the rotary embedding, and
  the keys' and values' way into the cache;
* ``tree``      attention of a tree of drafted tokens (or, without a mask, of
  a run of tokens) over the cache that holds what came before and themselves.

Sizes are those of the 8B-shaped model of :mod:`nibblegemm_amd.decode_step`
(32 query heads on 8, head size 128, projections of 4096 and 14336) and
generic ragged ones.
"""
import math

import torch

own = False

EPS = 1e-5
BLOCK = 32
#: Values of the 16 codes of a 4-bit float: sign, two exponent bits, one mantissa bit.
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def listed():
    return [
        # A weight of an fp16 checkpoint quantised while a model is loaded (and
        # expanded again, as a check of the quantised model does).
        {"name": "quantize_up", "op": "quantize", "rows": 14336, "K": 4096, "dtype": "float16",
         "transposed": False},
        # A weight held [K, N], as this package holds dense weights, quantised
        # along K: the rows are a transposed view.
        {"name": "quantize_kn", "op": "quantize", "rows": 4102, "K": 5536, "dtype": "float32",
         "transposed": True},
        # One k or v projection for one token: the smallest call.
        {"name": "kv_proj_1", "op": "matmul", "M": 1, "N": 1024, "K": 4096, "x": "dense",
         "dtype": "float16"},
        # The gate and up projections of 27 drafted tokens being verified.
        {"name": "gate_up_27", "op": "matmul", "M": 27, "N": 28672, "K": 4096, "x": "dense",
         "dtype": "bfloat16"},
        # Prefill of a long prompt: the gate or up projection.
        {"name": "gate_2048", "op": "matmul", "M": 2048, "N": 14336, "K": 4096, "x": "dense",
         "dtype": "float16"},
        # Sizes that fill no tile, activations quantised beforehand (one input
        # of several projections), 32-bit outputs.
        {"name": "ragged_1000", "op": "matmul", "M": 1000, "N": 4102, "K": 5536, "x": "codes",
         "dtype": "float32"},
        # The token of one decode step.
        {"name": "qk_token", "op": "qk_norm", "B": 1, "T": 1, "kv": 8, "qpk": 4, "D": 128,
         "S": 4096, "dtype": "float16", "norm": True, "rope": True},
        # A prompt's tokens, four sequences at once.
        {"name": "qk_prompts", "op": "qk_norm", "B": 4, "T": 2000, "kv": 8, "qpk": 4, "D": 128,
         "S": 4096, "dtype": "bfloat16", "norm": True, "rope": True},
        # A tree of 16 drafted tokens early in a conversation.
        {"name": "tree_16", "op": "tree", "B": 1, "T": 16, "kv": 8, "qpk": 4, "D": 128,
         "ctx": 1000, "S": 4096, "dtype": "float16", "mask": True},
        # Sixteen conversations of different lengths verified together, trees
        # of up to 27 tokens.
        {"name": "trees_16x27", "op": "tree", "B": 16, "T": 27, "kv": 8, "qpk": 4, "D": 128,
         "ctx": 8100, "S": 8192, "dtype": "bfloat16", "mask": True},
        # A tree late in a very long conversation.
        {"name": "tree_64_long", "op": "tree", "B": 1, "T": 64, "kv": 8, "qpk": 4, "D": 128,
         "ctx": 65000, "S": 65536, "dtype": "float16", "mask": True},
        # The second half of a prompt over the cache of the first.
        {"name": "prompt_2048", "op": "tree", "B": 1, "T": 2048, "kv": 8, "qpk": 4, "D": 128,
         "ctx": 2048, "S": 4096, "dtype": "bfloat16", "mask": False},
    ]


# ---------------------------------------------------------------- drawn cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "matmul", "qk_norm", "tree", "tree", "tree"])
    if op == "quantize":
        return {"op": op, "rows": _log_int(rng, 1, 14336), "K": 32 * _log_int(rng, 2, 448),
                "dtype": rng.choice(["float16", "bfloat16", "float32"]),
                "transposed": rng.random() < 0.3}
    if op == "matmul":
        return {"op": op, "M": _log_int(rng, 1, 4096), "N": _log_int(rng, 64, 28672),
                "K": 32 * _log_int(rng, 2, 448), "x": rng.choice(["dense", "dense", "codes"]),
                "dtype": rng.choice(["float16", "bfloat16", "float32"])}
    heads = {"kv": rng.choice([1, 2, 4, 8]), "qpk": rng.choice([1, 2, 4, 5, 8]),
             "D": rng.choice([64, 128, 128])}
    if op == "qk_norm":
        T = _log_int(rng, 1, 4096)
        return {"op": op, "B": _log_int(rng, 1, 16), "T": T, **heads,
                "S": T + _log_int(rng, 1, 4096), "dtype": rng.choice(["float16", "bfloat16"]),
                "norm": rng.random() < 0.75, "rope": rng.random() < 0.75}
    T = _log_int(rng, 1, 512)
    ctx = _log_int(rng, 1, 65000)
    return {"op": op, "B": _log_int(rng, 1, 32), "T": T, **heads, "ctx": ctx,
            "S": ctx + T + rng.randint(0, 64), "dtype": rng.choice(["float16", "bfloat16"]),
            "mask": rng.random() < 0.75}


#: The largest listed work of each operator, in bytes and in flops.
_LARGEST = {"quantize": (320e6, 1), "matmul": (80e6, 2.41e11), "qk_norm": (250e6, 1e9),
            "tree": (540e6, 1.1e11)}


def _scores(case):
    """Values of the plain form's score matrix (and its state's caches)."""
    return case["B"] * case["kv"] * case["qpk"] * case["T"] * case["S"] if case["op"] == "tree" else 0


def draw(rng):
    while True:
        case = _draw(rng)
        w, most = work(case), _LARGEST[case["op"]]
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and _scores(case) <= 2.7e8:
            return case


# --------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _activations(gen, rows, K):
    """Unit activations with a few channels that are an order larger."""
    x = _randn(gen, rows, K)
    return x * torch.where(torch.rand(K, generator=gen, device="cuda") < 0.01, 10.0, 1.0)


def _lengths(case):
    """Cached tokens of each sequence before this call: the longest is ``ctx``."""
    return [max(1, int(case["ctx"] * (1 - 0.75 * ((b * 0.618034) % 1.0))))
            for b in range(case["B"])]


def _sizes(case):
    """Tokens of each sequence's tree: the largest has ``T``."""
    return [max(1, case["T"] - (b * 5) % max(1, case["T"] // 2)) for b in range(case["B"])]


def _tree_mask(gen, B, T):
    """Who is whose ancestor (or itself) in random trees: a token's parent is
    one of the eight before it, or the root."""
    i = torch.arange(T, device="cuda")
    back = torch.randint(1, 9, (B, T), generator=gen, device="cuda")
    parent = i - back
    seen = torch.eye(T, device="cuda").expand(B, T, T).clone()
    step = torch.zeros((B, T, T), device="cuda")
    b, t = (parent >= 0).nonzero(as_tuple=True)
    step[b, t, parent[b, t]] = 1.0
    reach = seen + step
    for _ in range(max(1, T.bit_length())):
        reach = (reach @ reach).clamp(max=1.0)
    return reach > 0


def _prepare_tree(case, gen):
    B, T, kv, D = case["B"], case["T"], case["kv"], case["D"]
    dtype = getattr(torch, case["dtype"])
    caches = [torch.randn((B, kv, case["S"], D), generator=gen, device="cuda", dtype=dtype)
              for _ in range(2)]
    return {"q": (2 * _randn(gen, B, T, kv * case["qpk"] * D)).to(dtype), "k": caches[0],
            "v": caches[1], "mask": _tree_mask(gen, B, T) if case["mask"] else None,
            "lengths": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda"),
            "sizes": torch.tensor(_sizes(case), dtype=torch.int32, device="cuda")}


def _prepare_qk(case, gen):
    B, T, kv, D, S = (case[k] for k in ("B", "T", "kv", "D", "S"))
    dtype = getattr(torch, case["dtype"])
    heads = kv * case["qpk"]
    caches = [torch.randn((B, kv, S, D), generator=gen, device="cuda").to(dtype) for _ in range(2)]
    start = torch.randint(0, S - T + 1, (B, 1), generator=gen, device="cuda")
    slots = start + torch.arange(T, device="cuda")
    filled = torch.tensor(_sizes(case), device="cuda")[:, None] > torch.arange(T, device="cuda")
    angle = torch.outer(torch.arange(S, dtype=torch.float64, device="cuda"), 500000.0 ** (
        -torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
    norms = [1 + 0.1 * _randn(gen, D) for _ in range(2)]
    return {"qkv": _randn(gen, B, T, (heads + 2 * kv) * D).to(dtype), "k": caches[0],
            "v": caches[1], "positions": slots.to(torch.int32),
            # tokens behind a sequence's last are padding: they go nowhere
            "slots": torch.where(filled, slots, -1).to(torch.int32),
            "norms": [n.to(dtype) for n in norms] if case["norm"] else [None, None],
            "rope": (angle.cos().float(), angle.sin().float()) if case["rope"] else None}


def _prepare_matmul(case, gen):
    M, N, K = case["M"], case["N"], case["K"]
    w = _encode(_randn(gen, N, K) * 0.02)
    x = _activations(gen, M, K)
    state = {"w": w, "N": N, "K": K, "M": M, "dtype": getattr(torch, case["dtype"])}
    if case["x"] == "dense":
        state["x"] = x.to(state["dtype"])
    else:
        state["codes"] = _encode(x)
    return state


def _prepare_quantize(case, gen):
    rows, K = case["rows"], case["K"]
    shape = (K, rows) if case["transposed"] else (rows, K)
    x = (_randn(gen, *shape) * 0.02).to(getattr(torch, case["dtype"]))
    return {"x": x.t() if case["transposed"] else x}


_PREPARE = {"tree": _prepare_tree, "qk_norm": _prepare_qk, "matmul": _prepare_matmul,
            "quantize": _prepare_quantize}


def prepare(case, seed):
    return {"op": case["op"], **_PREPARE[case["op"]](case, _gen(seed))}


# ------------------------------------------------------------- the plain forms

def _blocks(x):
    """``x`` in blocks of 32 along its rows: each block's exponent (that of its
    largest value, less 2, the exponent of the largest 4-bit value) and its
    values over that power of two, rounded half to even onto the 4-bit floats.
    In 64 bits, where every step but the rounding is exact."""
    v = x.float().reshape(x.shape[0], -1, BLOCK)
    top = v.abs().amax(-1)
    e = ((top.view(torch.int32) >> 23) - 129).clamp(min=-127)
    u = v.double() * torch.exp2(-e.double())[..., None]
    a = u.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return e, torch.where(u < 0, -q, q)


def _values(x):
    """What the quantised ``x`` stands for, in 32 bits (exact)."""
    e, q = _blocks(x)
    return (q * torch.exp2(e.double())[..., None]).float().reshape(x.shape)


def _encode(x):
    """Codes, two to a byte along a row (the even one low), and block exponents
    (biased by 127), those of four blocks to a word: ``[ceil(K / 128), rows,
    4]``, zero behind the last."""
    rows, K = x.shape
    e, q = _blocks(x)
    a = q.abs().reshape(rows, K)
    code = (a * 2).round().to(torch.int64)  # 0, 1, 2, 3, 4, 6, 8, 12
    code = torch.where(code < 4, code, torch.where(code < 8, code // 2 + 2, code // 4 + 4))
    code = code + 8 * (q < 0).reshape(rows, K)
    codes = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    groups = -(-K // 128)
    scales = torch.zeros((rows, groups * 4), dtype=torch.uint8, device=x.device)
    scales[:, :K // BLOCK] = (e + 127).to(torch.uint8)
    return codes, scales.view(rows, groups, 4).transpose(0, 1).contiguous()


def _decode(codes, scales):
    """The values of codes and exponents, in 32 bits (exact)."""
    rows, half = codes.shape
    table = torch.tensor(E2M1, device=codes.device)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1)
    e = scales.transpose(0, 1).reshape(rows, -1)[:, :2 * half // BLOCK]
    power = torch.exp2(e.double() - 127).float()
    return (v.view(rows, -1, BLOCK) * power[..., None]).view(rows, 2 * half)


def _plain_qk(s):
    k_cache, v_cache = s["k"], s["v"]
    B, kv, S, D = k_cache.shape
    T = s["qkv"].shape[1]
    x = s["qkv"].float().view(B, T, -1, D)
    n_q = x.shape[2] - 2 * kv
    q, k, v = x.split([n_q, kv, kv], 2)

    def turned(h, w):
        if w is not None:
            h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.float()
        if s["rope"] is not None:
            cos, sin = (t[s["positions"].long()][:, :, None] for t in s["rope"])
            lo, hi = h.split(D // 2, -1)
            h = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
        return h

    q, k = turned(q, s["norms"][0]), turned(k, s["norms"][1])
    b, t = (s["slots"] >= 0).nonzero(as_tuple=True)
    to = s["slots"][b, t].long()
    k_cache[b, :, to] = k[b, t].to(k_cache.dtype)
    v_cache[b, :, to] = s["qkv"].view(B, T, -1, D)[b, t, n_q + kv:]
    q = torch.where((s["slots"] >= 0)[:, :, None, None], q, 0.0)
    return [q.to(s["qkv"].dtype).view(B, T, n_q * D), k_cache, v_cache]


def _plain_tree(s):
    k_cache, v_cache = s["k"], s["v"]
    B, kv, S, D = k_cache.shape
    T = s["q"].shape[1]
    q = s["q"].float().view(B, T, kv, -1, D).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, D)
    # rows (head, token) by cached tokens
    score = q @ k_cache.float().transpose(2, 3).contiguous() / math.sqrt(D)
    score = score.view(B, kv, -1, T, S)
    at = torch.arange(S, device=q.device)
    first = s["lengths"].long()[:, None, None]
    node = at - first  # [B, 1, S]: which of the drafted tokens a row holds
    i = torch.arange(T, device=q.device)[:, None]
    if s["mask"] is None:
        seen = node <= i
    else:
        seen = torch.gather(s["mask"], 2, node.clamp(0, T - 1).expand(B, T, S))
        seen = (seen & (node < T)) | (node < 0)
    live = s["sizes"].long()[:, None, None]
    seen = seen & (node < live) & (i < live)
    seen = seen[:, None, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    v = torch.where((node < live).transpose(1, 2)[:, None], v_cache.float(), 0.0)
    out = p.view(B, kv, -1, S) @ v
    return out.view(B, kv, -1, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, -1).to(s["q"].dtype)


# ------------------------------------------------------------------- one pass

def run(state):
    op = state["op"]
    if not own:
        if op == "quantize":
            return _values(state["x"]).to(torch.bfloat16)
        if op == "matmul":
            x = _values(state["x"]) if "x" in state else _decode(*state["codes"])
            return (x @ _decode(*state["w"]).t()).to(state["dtype"])
        return _plain_qk(state) if op == "qk_norm" else _plain_tree(state)
    from nibblegemm_amd import glue, mx
    if op == "quantize":
        return mx.dequantize_mx(mx.quantize_mx(state["x"]), torch.bfloat16)
    if op == "matmul":
        x = state["x"] if "x" in state else mx.MXMatrix(*state["codes"], state["M"], state["K"])
        return mx.matmul_mx(x, mx.MXMatrix(*state["w"], state["N"], state["K"]), state["dtype"])
    if op == "qk_norm":
        q = glue.qk_norm_rope(state["qkv"], state["k"], state["v"], state["positions"],
                              state["slots"], state["norms"][0], state["norms"][1], EPS,
                              state["rope"])
        return [q, state["k"], state["v"]]
    return glue.attention_tree(state["q"], state["k"], state["v"], state["lengths"],
                               state["mask"], state["sizes"])


# ------------------------------------------- what a pass cannot do without

def _size(case):
    return 4 if case["dtype"] == "float32" else 2


def _mx_bytes(rows, K):
    return rows * (K // 2 + K // BLOCK)


def work(case):
    op = case["op"]
    if op == "quantize":  # read once; codes and values written
        n = case["rows"] * case["K"]
        return {"bytes": n * (_size(case) + 2) + _mx_bytes(case["rows"], case["K"]), "flops": 0}
    if op == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        x = M * K * _size(case) if case["x"] == "dense" else _mx_bytes(M, K)
        return {"bytes": x + _mx_bytes(N, K) + M * N * _size(case), "flops": 2 * M * N * K}
    kv, D, q = case["kv"], case["D"], case["kv"] * case["qpk"]
    if op == "qk_norm":
        tokens = case["B"] * case["T"]
        rope = min(case["S"], tokens) * D * 4 if case["rope"] else 0
        return {"bytes": tokens * (q + 2 * kv) * D * 2 * 2 + rope + tokens * 8,
                "flops": tokens * (q + kv) * D * 7}
    lengths, sizes = _lengths(case), _sizes(case)
    rows = sum(n + t for n, t in zip(lengths, sizes))
    pairs = sum(t * n + (t * (t + 1)) // 2 for n, t in zip(lengths, sizes))
    masks = case["B"] * case["T"] ** 2 if case["mask"] else 0
    return {"bytes": rows * kv * D * 4 + case["B"] * case["T"] * q * D * 4 + masks,
            "flops": pairs * q * D * 4}


# ----------------------------------------------- the same in 64-bit arithmetic

def _grid64(x):
    """The nearest 4-bit floats of a block's values, found among all of them:
    ties go to the one whose code is even."""
    v = x.double().view(-1, BLOCK)
    top = v.abs().amax(1, keepdim=True)
    _, ex = torch.frexp(top)  # top = f 2^ex, 1/2 <= f < 1
    power = torch.ldexp(torch.ones_like(top), torch.where(top > 0, ex - 3, -127).clamp(min=-127))
    u = (v / power).abs()
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64,
                         device=x.device)  # halfway between neighbours
    code = torch.bucketize(u, edges)  # u at an edge: the lower one
    up = (code < 7) & (u == edges[code.clamp(max=6)]) & (code % 2 == 1)
    grid = torch.tensor(E2M1[:8], dtype=torch.float64, device=x.device)
    return (torch.copysign(grid[code + up.long()], v) * power).view(x.shape)


def _decode64(codes, scales):
    rows = codes.shape[0]
    nibbles = torch.stack([codes.long() % 16, codes.long() // 16], 2).flatten(1)
    mag, sign = nibbles % 8, 1.0 - 2.0 * (nibbles // 8).double()
    ex, man = mag // 2, (mag % 2).double()
    v = torch.where(ex == 0, man / 2, torch.ldexp(1 + man / 2, ex - 1)) * sign
    per = scales.permute(1, 0, 2).flatten(1)[:, :v.shape[1] // BLOCK]
    return torch.ldexp(v, (per.long() - 127).repeat_interleave(BLOCK, 1)).view(rows, -1)


def _exact_qk(s):
    B, kv, S, D = s["k"].shape
    x = s["qkv"].double().unflatten(2, (-1, D))
    n_q = x.shape[2] - 2 * kv
    out = x.clone()
    for part, w in ((slice(0, n_q), s["norms"][0]), (slice(n_q, n_q + kv), s["norms"][1])):
        if w is not None:
            h = out[:, :, part]
            out[:, :, part] = h / (h.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
    if s["rope"] is not None:
        cos, sin = (t.double()[s["positions"].long()].unsqueeze(2) for t in s["rope"])
        z = torch.complex(out[:, :, :n_q + kv, :D // 2], out[:, :, :n_q + kv, D // 2:])
        z = z * torch.complex(cos, sin)
        out[:, :, :n_q + kv] = torch.cat([z.real, z.imag], -1)
    k64, v64 = s["k"].double(), s["v"].double()
    live = s["slots"] >= 0
    for b in range(B):
        to = s["slots"][b][live[b]].long()
        k64[b, :, to] = out[b, live[b], n_q:n_q + kv].transpose(0, 1)
        v64[b, :, to] = out[b, live[b], n_q + kv:].transpose(0, 1)
    return [(out[:, :, :n_q] * live[:, :, None, None]).flatten(2), k64, v64]


def _exact_tree(s):
    """One sequence and one kv head at a time, over that sequence's rows only."""
    B, kv, S, D = s["k"].shape
    T = s["q"].shape[1]
    q = s["q"].double().view(B, T, kv, -1, D)
    out = torch.zeros_like(q)
    for b, (n, t) in enumerate(zip(s["lengths"].tolist(), s["sizes"].tolist())):
        seen = torch.ones((t, n + t), dtype=torch.bool, device=q.device)
        seen[:, n:] = torch.tril(seen[:, n:]) if s["mask"] is None else s["mask"][b, :t, :t]
        hide = torch.zeros((t, n + t), dtype=torch.float64, device=q.device)
        hide.masked_fill_(~seen, -math.inf)
        for h in range(kv):
            k, v = s["k"][b, h, :n + t].double(), s["v"][b, h, :n + t].double()
            score = torch.matmul(q[b, :t, h].reshape(-1, D), k.t()).view(t, -1, n + t)
            p = torch.softmax(score * D ** -0.5 + hide[:, None], -1)
            out[b, :t, h] = torch.matmul(p.flatten(0, 1), v).view(t, -1, D)
    return out.view(B, T, -1)


def exact(case, seed):
    op, gen = case["op"], _gen(seed)
    s = _PREPARE[op](case, gen)
    if op == "quantize":
        return _grid64(s["x"].contiguous())
    if op == "matmul":
        x = _grid64(s["x"]) if "x" in s else _decode64(*s["codes"])
        return torch.matmul(x, _decode64(*s["w"]).t())
    return _exact_qk(s) if op == "qk_norm" else _exact_tree(s)

"""Head norms with the rotary embedding and the cache append, and attention of
trees of drafted tokens over the cache.

The oracle is plain float64 on the CPU, token by token for attention.
Tolerances count roundings: half a step of the output's type, half a step for
the probabilities, and the fp32 sums' own errors.
"""
from __future__ import annotations

import math

import pytest
import torch

import nibblegemm_amd as ng
from nibblegemm_amd import glue

INVALID, WORKSPACE = 1, 3
P = 1 << 20  # aligned, never dereferenced
dev = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DTYPES = [F16, BF16]


# ---------------------------------------------------------------------------
# oracles (float64, CPU)
# ---------------------------------------------------------------------------
def oracle_qk(qkv, k_cache, v_cache, positions, slots, qw, kw, eps, rope):
    """q [B, T, heads, D], the caches, and magnitudes that bound q's and k's
    rounding errors."""
    B, n_kv, S, D = k_cache.shape
    x = qkv.double().view(*qkv.shape[:2], -1, D)
    n_q = x.shape[2] - 2 * n_kv
    rows = rope[0].shape[0] if rope is not None else 1 << 40
    live = (slots >= 0) & (slots < S) & (positions >= 0) & (positions < rows) if rope is not None \
        else (slots >= 0) & (slots < S)
    parts = []
    for h, w in ((x[:, :, :n_q], qw), (x[:, :, n_q:n_q + n_kv], kw)):
        if w is not None:
            h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()
        mag = h.abs()
        if rope is not None:
            at = positions.long().clamp(0, rows - 1)
            c, s = (t.double()[at][:, :, None] for t in rope)
            lo, hi = h[..., :D // 2], h[..., D // 2:]
            h = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
            mag = torch.cat([mag[..., :D // 2] + mag[..., D // 2:]] * 2, -1)
        parts.append((h, mag))
    (q, q_mag), (k, k_mag) = parts
    q = torch.where(live[:, :, None, None], q, 0.0)
    k64, v64, kept = k_cache.double(), v_cache.double(), torch.ones(k_cache.shape, dtype=torch.bool)
    k_bound = torch.zeros_like(k64)
    for b in range(B):
        for t in range(qkv.shape[1]):
            if live[b, t]:
                at = int(slots[b, t])
                k64[b, :, at], v64[b, :, at] = k[b, t], x[b, t, n_q + n_kv:]
                k_bound[b, :, at] = k_mag[b, t]
                kept[b, :, at] = False
    return q, q_mag, k64, k_bound, v64, kept


def check_qk(B, T, n_heads, n_kv, D, S, dtype, norm=True, rope=True, layout="bhsd", slots=None,
             positions=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((B, T, (n_heads + 2 * n_kv) * D), generator=g).to(dtype)
    k = torch.randn((B, n_kv, S, D), generator=g).to(dtype)
    v = torch.randn((B, n_kv, S, D), generator=g).to(dtype)
    if slots is None:
        slots = torch.stack([torch.randperm(S, generator=g)[:T] for _ in range(B)])
    if positions is None:
        positions = torch.randint(0, S + 3, (B, T), generator=g)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    if norm is not True:
        qw, kw = (qw, None) if norm == "q" else (None, kw) if norm == "k" else (None, None)
    tables = glue.rope_tables(S + 3, D, device="cpu") if rope else None

    def cache(t):
        if layout == "bshd":
            return t.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
        if layout == "part":  # rows of a wider cache
            wide = torch.zeros((B, n_kv, S, D + 24), dtype=dtype, device=dev)
            wide[..., 8:8 + D] = t.to(dev)
            return wide[..., 8:8 + D]
        return t.to(dev)

    kd, vd = cache(k), cache(v)
    to = lambda t: t.to(dev) if t is not None else None  # noqa: E731
    got = glue.qk_norm_rope(qkv.to(dev), kd, vd, positions.int().to(dev), slots.int().to(dev),
                            to(qw), to(kw), 1e-5, tuple(map(to, tables)) if rope else None).cpu()
    q, q_mag, k64, k_bound, v64, kept = oracle_qk(qkv, k, v, positions, slots, qw, kw, 1e-5, tables)
    assert got.shape == (B, T, n_heads * D) and got.dtype == dtype
    info = torch.finfo(dtype)
    # fp32: D additions of squares (halved by the root), and ten operations
    slack = (D / 2 + 10) * 2.0 ** -24

    def near(x, want, mag):
        off = (x.double() - want).abs()
        assert (off <= want.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2
                + mag * slack).all(), off.max()

    near(got.view(B, T, n_heads, D), q, q_mag)
    near(kd.cpu(), k64, k_bound)
    assert torch.equal(kd.cpu()[kept], k[kept]), "other rows stay as they were"
    assert torch.equal(vd.cpu().double(), v64)
    return got


def oracle_attention(q, k, v, lengths, mask, sizes, scale):
    """[B, T, heads, D], and a bound of the error per element."""
    B, T, n_heads, D = q.shape
    n_kv, S = k.shape[1], k.shape[2]
    out = torch.zeros((B, T, n_heads, D), dtype=torch.float64)
    bound = torch.zeros_like(out)
    info = torch.finfo(q.dtype)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), S)
        live = T if sizes is None else min(max(int(sizes[b]), 0), T)
        for i in range(live):
            rows = torch.arange(S)
            seen = rows < n
            for j in range(min(live, S - n)):
                if j <= i if mask is None else bool(mask[b if mask.dim() == 3 else 0][i, j]) \
                        if mask.dim() == 3 else bool(mask[i, j]):
                    seen[n + j] = True
            if not seen.any():
                continue
            for h in range(n_heads):
                kk = k[b, h // (n_heads // n_kv)][seen].double()
                vv = v[b, h // (n_heads // n_kv)][seen].double()
                qq = q[b, i, h].double()
                s = kk @ qq * scale
                p = torch.softmax(s, 0)
                out[b, i, h] = p @ vv
                fine = torch.nan_to_num(vv, 0.0, 0.0, 0.0).abs()
                away = (kk.abs() @ qq.abs()).max() * abs(scale) * (D + 4) * 2.0 ** -24 \
                    + s.abs().max() * 2.0 ** -22
                a = p @ fine
                bound[b, i, h] = out[b, i, h].abs().nan_to_num(0.0, 0.0) * info.eps / 2 \
                    + a * (info.eps / 2 + 2 * away + 2.0 ** -20) + info.smallest_normal * info.eps
                if q.dtype == F16:  # probabilities below 2^-14 of the largest: steps of 2^-24
                    bound[b, i, h] += len(vv) * 2.0 ** -25 * fine.max()
    return out, bound


def random_tree(T, g, back=4):
    return torch.tensor([i - int(torch.randint(1, back + 1, (1,), generator=g)) for i in range(T)]
                        ).clamp(min=-1)


def tree_case(B, T, n_heads, n_kv, D, S, dtype, lengths, masked, sizes=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (1.5 * torch.randn((B, T, n_heads, D), generator=g)).to(dtype)
    k, v = (torch.randn((B, n_kv, S, D), generator=g).to(dtype) for _ in range(2))
    mask = None
    if masked:
        mask = glue.tree_mask(torch.stack([random_tree(T, g) for _ in range(B)]))
    lengths = torch.tensor(lengths, dtype=torch.int32)
    sizes = None if sizes is None else torch.tensor(sizes, dtype=torch.int32)
    return q, k, v, lengths, mask, sizes


def run_tree(q, k, v, lengths, mask=None, sizes=None, scale=None):
    to = lambda t: t.to(dev) if t is not None else None  # noqa: E731
    B, T, n_heads, D = q.shape
    return glue.attention_tree(to(q.reshape(B, T, -1)), to(k), to(v), to(lengths), to(mask),
                               to(sizes), scale).view(B, T, n_heads, D)


def check_tree(*case, scale=None):
    q, k, v, lengths, mask, sizes = case
    got = run_tree(*case, scale=scale)
    want, bound = oracle_attention(q, k, v, lengths, mask, sizes,
                                   q.shape[3] ** -0.5 if scale is None else scale)
    assert got.dtype == q.dtype
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or (off <= 0).all(), f"{off.max():.3g} beyond its bound"
    return got


# ---------------------------------------------------------------------------
# masks and refusals (CPU)
# ---------------------------------------------------------------------------
def test_tree_mask():
    #       0
    #      / \      5 (a second root)
    #     1   2
    #    / \   \
    #   3   4   6
    m = glue.tree_mask(torch.tensor([-1, 0, 0, 1, 1, -1, 2]))
    want = {0: [0], 1: [0, 1], 2: [0, 2], 3: [0, 1, 3], 4: [0, 1, 4], 5: [5], 6: [0, 2, 6]}
    assert m.dtype == torch.bool
    assert {i: m[i].nonzero().flatten().tolist() for i in range(7)} == want
    chain = glue.tree_mask(torch.arange(-1, 40).view(1, -1).expand(3, -1))
    assert chain.shape == (3, 41, 41) and torch.equal(chain[2], torch.ones(41, 41).tril().bool())
    assert glue.tree_mask(torch.zeros((2, 0), dtype=torch.long)).shape == (2, 0, 0)
    for bad in ([0], [-1, 1], [-2], [-1, 3, 0]):
        with pytest.raises(ValueError, match="parent"):
            glue.tree_mask(torch.tensor(bad))
    with pytest.raises(ValueError, match="integer"):
        glue.tree_mask(torch.zeros(3))


def qk(ext, qkv=P, dt=0, B=1, T=2, nh=4, nkv=2, D=128, kc=P, st=(4096, 2048, 128), vc=P, S=16,
       pos=P, slots=P, qw=None, kw=None, eps=1e-5, cos=None, sin=None, rows=0, out=P):
    return ext.qk_norm_rope(qkv, dt, B, T, nh, nkv, D, kc, *st, vc, *st, S, pos, slots, qw, kw, eps,
                            cos, sin, rows, out, None)


def tree(ext, q=P, dt=0, B=1, T=2, nh=4, nkv=2, D=128, kc=P, st=(4096, 2048, 128), vc=P, S=16,
         lengths=P, mask=None, mb=1, sizes=None, scale=0.1, out=P, ws=None, wsb=0):
    return ext.attention_tree(q, dt, B, T, nh, nkv, D, kc, *st, vc, *st, S, lengths, mask, mb, sizes,
                              scale, out, ws, wsb, None)


@pytest.mark.parametrize("kwargs,needle", [
    (dict(dt=2), "dtype"), (dict(D=96), "head_dim"), (dict(nkv=0), "n_kv_heads"),
    (dict(nh=0), "n_heads"), (dict(B=-1), "batch"), (dict(T=1 << 31), "tokens"),
    (dict(S=-1), "max_seq"), (dict(cos=P), "both"), (dict(cos=P, sin=P, rows=0), "rows"),
    (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"), (dict(st=(4096, 2044, 128)), "strides"),
    (dict(qkv=0), "null"), (dict(kc=0), "null"), (dict(pos=0), "null"), (dict(slots=0), "null"),
    (dict(out=0), "null"), (dict(qkv=P + 8), "aligned"), (dict(qw=P + 8), "aligned"),
    (dict(vc=P + 2), "aligned"), (dict(pos=P + 2), "aligned"), (dict(B=1 << 30, T=1 << 30), "too many"),
    (dict(B=1 << 20, T=1 << 10), "too many"),
])
def test_qk_rejections(kwargs, needle):
    ext = ng.extension()
    assert qk(ext, **kwargs) == INVALID
    assert needle in ext.last_error()


@pytest.mark.parametrize("kwargs,needle", [
    (dict(dt=2), "dtype"), (dict(D=256), "head_dim"), (dict(nkv=0), "n_kv_heads"),
    (dict(nh=5), "multiple of n_kv_heads"), (dict(B=-1), "batch"), (dict(T=(1 << 20) + 1), "tokens"),
    (dict(S=1 << 30), "max_seq"), (dict(scale=float("inf")), "scale"),
    (dict(st=(4096, 2048, 132)), "strides"), (dict(st=(0, 0, (1 << 22) + 8)), "2^22"),
    (dict(B=3, mask=P, mb=2), "mask"), (dict(q=0), "null"), (dict(lengths=0), "null"),
    (dict(kc=0), "null"), (dict(out=0), "null"), (dict(q=P + 8), "aligned"),
    (dict(lengths=P + 1), "aligned"), (dict(sizes=P + 2), "aligned"),
    (dict(B=65535, T=1 << 20), "2^30"),
])
def test_tree_rejections(kwargs, needle):
    ext = ng.extension()
    assert tree(ext, **kwargs) == INVALID
    assert needle in ext.last_error()


def test_tree_workspace():
    ext = ng.extension()
    assert ext.attention_tree_workspace_bytes(1, 16, 32, 8, 128, 128) == 0  # one tile of rows
    need = ext.attention_tree_workspace_bytes(1, 16, 32, 8, 128, 65536)
    # whole shares of (sums, top, sum), and where each sequence's begin
    assert need > 0 and (need - 8) % (8 * 64 * 130 * 4) == 0
    assert ext.attention_tree_workspace_bytes(1, 16, 32, 8, 96, 65536) == 0  # a refused plan
    st = (8 * 65536 * 128, 65536 * 128, 128)
    big = dict(T=16, nh=32, nkv=8, S=65536, st=st)
    assert tree(ext, **big) == WORKSPACE and "workspace" in ext.last_error()
    assert tree(ext, **big, ws=P, wsb=need - 1) == WORKSPACE
    assert tree(ext, **big, ws=P + 64, wsb=need) == WORKSPACE and "256-byte" in ext.last_error()


def test_library_takes_empty_sizes():
    ext = ng.extension()
    assert qk(ext, B=0, qkv=0, out=0) == 0 and qk(ext, T=0, qkv=0) == 0
    assert tree(ext, B=0, q=0) == 0 and tree(ext, T=0, q=0) == 0


def test_refusals_without_a_gpu():
    x, c = torch.zeros((1, 2, 512), dtype=F16), torch.zeros((1, 1, 8, 128), dtype=F16)
    i = torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        glue.qk_norm_rope(x, c, c, i, i)
    with pytest.raises(RuntimeError, match="GPU"):
        glue.attention_tree(x, c, c, i[:, 0])
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        glue.attention_tree(x.float(), c, c, i[:, 0])


# ---------------------------------------------------------------------------
# norms, rotation and the cache (GPU)
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,n_heads,n_kv,D,S", [
    (1, 1, 1, 1, 64, 1), (1, 1, 32, 8, 128, 64), (2, 3, 5, 1, 128, 7), (3, 17, 8, 2, 64, 40),
    (1, 130, 4, 4, 128, 131), (5, 2, 7, 7, 64, 9)])
def test_qk(B, T, n_heads, n_kv, D, S, dtype):
    check_qk(B, T, n_heads, n_kv, D, S, dtype, seed=T)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm,rope", [(True, False), (False, True), (False, False), ("q", True),
                                       ("k", False)])
def test_qk_without_norms_or_rotation(norm, rope, dtype):
    check_qk(2, 5, 6, 2, 128, 11, dtype, norm=norm, rope=rope)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["bshd", "part"])
@pytest.mark.parametrize("D", [64, 128])
def test_qk_cache_layouts(layout, D):
    check_qk(2, 5, 6, 2, D, 11, BF16, layout=layout)


@pytest.mark.gpu
def test_qk_padding_goes_nowhere():
    S = 12
    slots = torch.tensor([[0, -1, 11, 12, 5], [-7, 2 ** 31 - 1, 3, -2 ** 31, 4]])
    positions = torch.tensor([[0, 3, 15, 2, 14], [1, 1, -1, 2, 2 ** 31 - 1]])
    got = check_qk(2, 5, 6, 2, 128, S, F16, slots=slots, positions=positions)
    dead = torch.tensor([[0, 1, 1, 1, 0], [1, 1, 1, 1, 1]]).bool()
    assert not got[dead].any() and got[~dead].any(-1).all()


@pytest.mark.gpu
def test_qk_one_sequence_and_refusals():
    g = torch.Generator().manual_seed(1)
    x = torch.randn((4, 8 * 128), generator=g).to(F16).to(dev)
    k1, v1 = (torch.zeros((2, 16, 128), dtype=F16, device=dev) for _ in range(2))
    k2, v2 = k1.clone()[None], v1.clone()[None]
    at = torch.arange(4, dtype=torch.int32, device=dev)
    a = glue.qk_norm_rope(x, k1, v1, at, at)
    b = glue.qk_norm_rope(x[None], k2, v2, at[None], at[None])
    assert a.shape == (4, 4 * 128) and torch.equal(a, b[0])
    assert torch.equal(k1, k2[0]) and torch.equal(v1, v2[0]) and k1[:, :4].any()
    for bad, error in [(lambda: glue.qk_norm_rope(x, k2, v2, at, at), ValueError),
                       (lambda: glue.qk_norm_rope(x, k1, v1[:, :8], at, at), ValueError),
                       (lambda: glue.qk_norm_rope(x, k1, v1, at.long(), at), RuntimeError),
                       (lambda: glue.qk_norm_rope(x, k1, v1, at[:3], at), ValueError),
                       (lambda: glue.qk_norm_rope(x, k1, v1.bfloat16(), at, at), RuntimeError),
                       (lambda: glue.qk_norm_rope(x[:, ::2], k1, v1, at, at), RuntimeError),
                       (lambda: glue.qk_norm_rope(x[:, :512].contiguous(), k1, v1, at, at), ValueError),
                       (lambda: glue.qk_norm_rope(x, k1.expand(2, 16, 128)[:1].expand(2, 16, 128), v1,
                                                  at, at), RuntimeError),
                       (lambda: glue.qk_norm_rope(x, k1[..., :1].expand(2, 16, 128), v1, at, at),
                        RuntimeError),
                       (lambda: glue.qk_norm_rope(x.clone().requires_grad_(), k1, v1, at, at),
                        RuntimeError),
                       (lambda: glue.qk_norm_rope(x, k1, v1, at, at, x[0, :64]), ValueError),
                       (lambda: glue.qk_norm_rope(x, k1, v1, at, at, rope=(x, x)), RuntimeError)]:
        with pytest.raises(error):
            bad()


# ---------------------------------------------------------------------------
# attention (GPU)
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("B,T,n_heads,n_kv,D,lengths,extra", [
    (1, 1, 1, 1, 64, [0], 0),
    (1, 1, 4, 1, 128, [1], 0),
    (1, 3, 8, 2, 128, [126], 5),      # the tree ends behind the first tile
    (2, 4, 4, 4, 64, [127, 128], 2),  # one key and two in the second
    (3, 7, 10, 2, 128, [0, 300, 31], 9),
    (1, 16, 8, 2, 128, [500], 0),
    (2, 13, 16, 2, 64, [129, 1000], 3),   # 104 rows: two waves along the keys
    (1, 33, 12, 2, 128, [70], 1),         # 198 rows: a wave per 64 rows
    (1, 70, 8, 1, 64, [40], 64),          # 560 rows: three workgroups
    (1, 65, 8, 2, 128, [600], 0),         # 260 rows: four of them in a second one
    (1, 2, 7, 1, 128, [3000], 30),        # an odd group of heads, several splits
    (1, 2, 4, 2, 64, [20000], 0),         # 63 splits
    (2, 3, 2, 1, 64, [20000, 0], 0),
])
def test_tree_attention(B, T, n_heads, n_kv, D, lengths, extra, masked, dtype):
    check_tree(*tree_case(B, T, n_heads, n_kv, D, max(lengths) + T + extra, dtype, lengths, masked,
                          seed=T))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_sizes_and_shared_masks(dtype):
    q, k, v, lengths, mask, sizes = tree_case(4, 9, 8, 2, 128, 300, dtype, [200, 0, 37, 290], True,
                                              sizes=[9, 4, 0, 1])
    got = check_tree(q, k, v, lengths, mask, sizes)
    assert not got[1, 4:].any() and not got[2].any() and not got[3, 1:].any()
    check_tree(q, k, v, lengths, mask[0].contiguous(), sizes)
    check_tree(q, k, v, lengths, None, sizes)
    check_tree(q, k, v, lengths, mask, None)  # 290 + 9 rows fit
    assert torch.equal(run_tree(q, k, v, lengths, mask, sizes, scale=128 ** -0.5).cpu().double(), got)
    check_tree(q, k, v, lengths, mask, sizes, scale=0.3)
    check_tree(q, k, v, lengths, mask, sizes, scale=0.0)
    check_tree(q, k, v, lengths, mask, sizes, scale=-0.1)


@pytest.mark.gpu
def test_counts_beyond_the_cache_end_with_it():
    q, k, v, _, mask, _ = tree_case(3, 5, 4, 2, 64, 130, F16, [0, 0, 0], True)
    lengths = torch.tensor([128, 1000, -3], dtype=torch.int32)
    sizes = torch.tensor([5, 7, -1], dtype=torch.int32)
    got = check_tree(q, k, v, lengths, mask, sizes)
    assert not got[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_that_see_nothing(dtype):
    """A tree at the start of a sequence whose masks leave rows empty."""
    q, k, v, lengths, mask, _ = tree_case(2, 40, 4, 1, 128, 64, dtype, [0, 0], True)
    mask[0, 3], mask[0, 17], mask[1] = False, False, False
    got = check_tree(q, k, v, lengths, mask, None)
    assert not got[0, 3].any() and not got[0, 17].any() and not got[1].any() and got[0, 4].any()


@pytest.mark.gpu
@pytest.mark.parametrize("qpk", [1, 8])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 6, 9, 66, 131])
def test_masks_of_any_pattern(T, qpk):
    """Trees that begin at every place of a group of four keys and of a tile,
    masks without the token itself and with later ones, and bytes other than 1."""
    lengths = [0, 1, 2, 3, 61, 64, 126]
    q, k, v, lengths, _, _ = tree_case(len(lengths), T, qpk, 1, 64, 126 + T + 1, F16, lengths, False,
                                       seed=T)
    g = torch.Generator().manual_seed(T)
    mask = torch.rand((len(lengths), T, T), generator=g) < 0.3
    mask[:, T // 2] = False
    got = check_tree(q, k, v, lengths, mask, None)
    odd = torch.randint(1, 256, mask.shape, generator=g, dtype=torch.uint8) * mask
    assert torch.equal(run_tree(q, k, v, lengths, odd.view(torch.bool)).cpu().double(), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,n_heads", [(6, 2), (6, 8), (24, 8), (40, 8), (90, 8)])
def test_strange_values_in_rows_not_seen(T, n_heads, dtype):
    """Infinities and NaN in tree rows reach those that see them only, and what
    lies behind the tree nobody."""
    q, k, v, lengths, mask, _ = tree_case(2, T, n_heads, 1, 64, T + 170, dtype, [125, 3], True, seed=T)
    inf, nan = float("inf"), float("nan")
    for b in range(2):
        n = int(lengths[b])
        mask[b, :, 2] = False
        k[b, 0, n + 2, 5], v[b, 0, n + 2, 7] = nan, inf
        mask[b, :, 4] = torch.arange(T) % 3 == 0
        v[b, 0, n + 4, 9], v[b, 0, n + 4, 10], v[b, 0, n + 4, 11] = inf, -inf, nan
        mask[b, :, 1] = torch.arange(T) % 4 == 1
        k[b, 0, n + 1, 3] = nan
        k[b, 0, n + T:], v[b, 0, n + T:] = nan, inf
    got = check_tree(q, k, v, lengths, mask, None)
    assert got.isnan().any() and got.isinf().any() and got.isfinite().all(-1).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [[3, 900], [700, 20]])
def test_strange_values_seen_by_all(lengths, dtype):
    """A NaN in a query is its own output's alone; infinities in cached rows
    that every query sees come out where they belong."""
    q, k, v, lengths, mask, _ = tree_case(2, 9, 4, 2, 128, 920, dtype, lengths, True)
    q[0, 3, 1, 17] = float("nan")
    q[1, 0, 2, 5] = float("nan")
    v[1, 1, 2, 40], v[1, 1, 1, 41] = float("inf"), -float("inf")
    k[0, 0, 1, 3] = float("nan")
    got = check_tree(q, k, v, lengths, mask, None)
    assert got[0, :, :2].isnan().all() and got[0, 2, 2:].isfinite().all()
    assert got[1, 0, 2].isnan().all() and got[1, 1, 0].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("n_kv,n_heads,B", [(1, 2, 70), (1, 1, 300), (2, 4, 33), (1, 3, 511)])
def test_many_sequences_of_uneven_lengths(n_kv, n_heads, B):
    """Shares of the cached rows by the lengths: one long sequence among many
    short and empty ones, all alike, and all empty."""
    S, T, D = 1500, 2, 64
    g = torch.Generator().manual_seed(B)
    q = torch.randn((B, T, n_heads, D), generator=g).to(F16)
    k, v = (torch.randn((1, n_kv, S, D), generator=g).to(F16).expand(B, n_kv, S, D) for _ in range(2))
    for kind in range(3):
        lengths = torch.randint(0, 40, (B,), generator=g)
        lengths[B // 2] = 1490
        lengths[::7] = 0
        if kind:
            lengths[:] = 700 if kind == 1 else 0
        sizes = torch.randint(0, T + 1, (B,), generator=g)
        got = run_tree(q, k, v, lengths.int(), None, sizes.int()).cpu().double()
        for b in sorted({0, 1, 6, 7, B // 2, B // 2 + 1, B - 1}):
            want, bound = oracle_attention(q[b:b + 1], k[:1], v[:1], lengths[b:b + 1], None,
                                           sizes[b:b + 1], D ** -0.5)
            assert ((got[b:b + 1] - want).abs() <= bound).all(), (kind, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_far_apart_and_moving_up(dtype):
    """The running maximum climbs tile by tile, by more and by less than its
    slack, and falls again."""
    q, k, v, lengths, mask, _ = tree_case(1, 4, 4, 2, 128, 1200, dtype, [1190], True)
    ramp = torch.cat([torch.linspace(-3, 3, 900), torch.linspace(3, -2, 300)])
    k = (q[0, 0, 0].float() * ramp[None, None, :, None] + 0.05 * k.float()).to(dtype)
    check_tree(q, k, v, lengths, mask, None)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_cache_layouts_and_one_sequence(D):
    q, k, v, lengths, mask, _ = tree_case(2, 5, 8, 2, D, 400, BF16, [333, 77], True)
    want = run_tree(q, k, v, lengths, mask)
    kd, vd = k.to(dev), v.to(dev)
    bshd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kd, vd)]
    assert torch.equal(run_tree(q, *bshd, lengths, mask), want)
    wide = []
    for t in (kd, vd):
        w = torch.full((2, 2, 400, D + 40), float("nan"), dtype=BF16, device=dev)
        w[..., 16:16 + D] = t
        wide.append(w[..., 16:16 + D])
    assert torch.equal(run_tree(q, *wide, lengths, mask), want)
    for b in range(2):
        one = glue.attention_tree(q[b].reshape(5, -1).to(dev), kd[b], vd[b], lengths[b:b + 1].to(dev),
                                  mask[b].contiguous().to(dev))
        assert one.shape == (5, 8 * D)
        torch.testing.assert_close(one.view(5, 8, D).float(), want[b].float(), atol=0.03, rtol=0.02)
    qd = q.reshape(2, 5, -1).to(dev)
    ln, md = lengths.to(dev), mask.to(dev)
    for bad, error in [(lambda: glue.attention_tree(qd, kd, vd, ln.long()), RuntimeError),
                       (lambda: glue.attention_tree(qd, kd, vd, ln[:1]), ValueError),
                       (lambda: glue.attention_tree(qd, kd, vd, ln, md.to(torch.uint8)), RuntimeError),
                       (lambda: glue.attention_tree(qd, kd, vd, ln, md[:, :4, :4].contiguous()), ValueError),
                       (lambda: glue.attention_tree(qd, kd, vd, ln, md.transpose(1, 2)), RuntimeError),
                       (lambda: glue.attention_tree(qd, kd, vd, ln, md, ln[:1]), ValueError),
                       (lambda: glue.attention_tree(qd, kd, vd.half(), ln), RuntimeError),
                       (lambda: glue.attention_tree(qd, kd[:1], vd[:1], ln), ValueError),
                       (lambda: glue.attention_tree(qd, kd[:, :, :0], vd[:, :, :0], ln), ValueError),
                       (lambda: glue.attention_tree(qd[..., 8:], kd, vd, ln), RuntimeError),
                       (lambda: glue.attention_tree(qd, kd, vd, lengths), RuntimeError),
                       (lambda: glue.attention_tree(qd, kd.clone().requires_grad_(), vd, ln), RuntimeError)]:
        with pytest.raises(error):
            bad()


@pytest.mark.gpu
def test_a_row_stride_that_passes_32_bits():
    """A cache whose last rows lie beyond 2^32 bytes."""
    S, width = 1100, 1 << 21  # 1100 rows of 4 MiB
    if torch.cuda.mem_get_info()[0] < 3 * S * width * 2:
        pytest.skip("not enough memory")
    q, k, v, lengths, mask, _ = tree_case(1, 3, 4, 1, 64, S, F16, [S - 3], True)
    big = torch.empty((1, 1, S, width), dtype=F16, device=dev)
    kd, vd = big[..., 64:128], big[..., width - 64:]
    kd.copy_(k), vd.copy_(v)
    assert torch.equal(run_tree(q, kd, vd, lengths, mask), run_tree(q, k, v, lengths, mask))
    slots = torch.tensor([[S - 1, S - 2, 0]], dtype=torch.int32, device=dev)
    x = torch.randn((1, 3, 6 * 64), device=dev).to(F16)
    small_k, small_v = k.to(dev), v.to(dev)
    a = glue.qk_norm_rope(x, small_k, small_v, slots, slots)
    assert torch.equal(glue.qk_norm_rope(x, kd, vd, slots, slots), a)
    assert torch.equal(kd, small_k) and torch.equal(vd, small_v)


@pytest.mark.gpu
def test_empty_batches():
    for B, T in ((0, 3), (2, 0)):
        q = torch.zeros((B, T, 256), dtype=F16, device=dev)
        c = torch.zeros((B, 1, 8, 64), dtype=F16, device=dev)
        n = torch.zeros(B, dtype=torch.int32, device=dev)
        i = torch.zeros((B, T), dtype=torch.int32, device=dev)
        if B:
            assert glue.attention_tree(q, c, c.clone(), n).shape == (B, T, 256)
            assert glue.qk_norm_rope(q, c, c.clone(), i, i).shape == (B, T, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("T,length", [(3, 50), (16, 3000)])
def test_graphs_and_streams(T, length):
    """Two captured calls of the same sizes, replayed between eager ones, with
    lengths and masks that change between the replays."""
    cases = [tree_case(2, T, 8, 2, 128, 4096, F16, [length + 7 * i, length // 2 + i], True, seed=i)
             for i in range(3)]
    want = [run_tree(*c) for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_tree(*cases[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[1])
    graphs = []
    for _ in range(2):
        state = [t.clone().to(dev) if t is not None else None for t in cases[0]]
        state[0] = state[0].reshape(2, T, -1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = glue.attention_tree(*state)
        graphs.append((graph, state, out))
    for i in (0, 1, 2, 0):
        for n, (graph, state, out) in enumerate(graphs):
            case = cases[(i + n) % 3]
            for dst, src in zip(state, case):
                if dst is not None:
                    dst.copy_(src.view(dst.shape))
            graph.replay()
        assert torch.equal(run_tree(*cases[2]), want[2])
        torch.cuda.synchronize()
        for n, (graph, state, out) in enumerate(graphs):
            assert torch.equal(out.view_as(want[0]), want[(i + n) % 3])


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_layer_verifies_a_tree(dtype):
    """One attention layer on microscaled weights verifies two drafted trees:
    the product, the norms into the cache, the tree's attention and the output
    product, against the same steps in float64 from each step's own inputs; and
    each path of a tree gives what its tokens give one by one."""
    B, T, n_heads, n_kv, D, S, hidden = 2, 6, 8, 2, 128, 200, 512
    g = torch.Generator().manual_seed(5)
    x = torch.randn((B * T, hidden), generator=g).to(dtype).to(dev)
    w_qkv = ng.quantize_mx((0.05 * torch.randn(((n_heads + 2 * n_kv) * D, hidden), generator=g)).to(dev))
    w_o = ng.quantize_mx((0.05 * torch.randn((hidden, n_heads * D), generator=g)).to(dev))
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)).to(dtype).to(dev) for _ in range(2))
    caches = [torch.randn((B, n_kv, S, D), generator=g).to(dtype).to(dev) for _ in range(2)]
    rope = glue.rope_tables(S, D)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 4], [-1, -1, 1, 2, 3, 0]])
    mask = glue.tree_mask(parents).to(dev)
    lengths = torch.tensor([130, 7], dtype=torch.int32, device=dev)
    depth = (mask.sum(-1) - 1).int()
    slots = lengths[:, None] + torch.arange(T, dtype=torch.int32, device=dev)

    def layer(x, k, v, positions, slots, mask, lengths):
        qkv = ng.matmul_mx(x, w_qkv).view(*positions.shape, -1)
        q = glue.qk_norm_rope(qkv, k, v, positions, slots, qw, kw, 1e-5, rope)
        att = glue.attention_tree(q, k, v, lengths, mask)
        return qkv, q, att, ng.matmul_mx(att.flatten(0, 1), w_o)

    k, v = (c.clone() for c in caches)
    qkv, q, att, y = layer(x, k, v, lengths[:, None] + depth, slots, mask, lengths)

    def same(got, want, rel):
        assert (got.double() - want).norm() <= rel * want.norm()

    step = torch.finfo(dtype).eps
    deq = lambda m: ng.dequantize_mx(m, F32).double()  # noqa: E731
    same(qkv.flatten(0, 1), deq(ng.quantize_mx(x)) @ deq(w_qkv).t().contiguous(), step)
    cpu = lambda t: t.cpu()  # noqa: E731
    q64, _, k64, _, _, _ = oracle_qk(cpu(qkv), cpu(caches[0]), cpu(caches[1]),
                                     cpu(lengths[:, None] + depth), cpu(slots), cpu(qw), cpu(kw),
                                     1e-5, tuple(map(cpu, rope)))
    same(q.cpu().view(B, T, n_heads, D), q64, step)
    same(k.cpu(), k64, step)
    a64, _ = oracle_attention(cpu(q).view(B, T, n_heads, D), cpu(k), cpu(v), cpu(lengths), cpu(mask),
                              None, D ** -0.5)
    same(att.cpu().view(B, T, n_heads, D), a64, 2 * step)
    same(y, deq(ng.quantize_mx(att.flatten(0, 1))) @ deq(w_o).t().contiguous(), step)

    # The deepest path of the first tree, token by token on its own cache.
    path = [0, 2, 4, 5]
    k1, v1 = (c[:1].clone() for c in caches)
    for n, t in enumerate(path):
        at = torch.tensor([[130 + n]], dtype=torch.int32, device=dev)
        one = layer(x[t:t + 1], k1, v1, at, at, None, at[0])
        same(one[2][0, 0], att[0, t].double(), 4 * step)

    # The whole layer in a graph.
    kg, vg = (c.clone() for c in caches)
    xs, pos = x.clone(), lengths[:, None] + depth
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = layer(xs, kg, vg, pos, slots, mask, lengths)
    for scale in (1.0, 0.5, 1.0):
        xs.copy_(x * scale)
        graph.replay()
        k2, v2 = (c.clone() for c in caches)
        want = layer(xs, k2, v2, pos, slots, mask, lengths)
        torch.cuda.synchronize()
        assert torch.equal(out[3], want[3]) and torch.equal(kg, k2) and torch.equal(vg, v2)


# ---------------------------------------------------------------------------
# rows of very different weight
# ---------------------------------------------------------------------------
def far_case(T, n_heads, D, S, n, dtype, nats, at, seed=0):
    """Scores of 0 but for row ``at``, the sink, whose score is ``nats``; its
    values are zero and the others' near one."""
    g = torch.Generator().manual_seed(seed)
    q = torch.zeros((1, T, n_heads, D), dtype=dtype)
    q[..., 3] = 4.0
    k = torch.randn((1, 1, S, D), generator=g).to(dtype)
    k[..., 3] = 0.0
    k[0, 0, at, 3] = nats / 4
    assert k[0, 0, at, 3].item() == nats / 4
    v = (1 + 0.25 * torch.randn((1, 1, S, D), generator=g)).to(dtype)
    v[0, 0, at] = 0.0
    return q, k, v, torch.tensor([n], dtype=torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [10, 14, 17, 17.5, 19])
@pytest.mark.parametrize("T,n_heads,n,at", [
    (1, 1, 200, 0), (1, 4, 8192, 0), (1, 4, 8192, 8000), (6, 4, 8192, 70), (12, 4, 8000, 7990),
    (40, 4, 8192, 100), (40, 4, 250, 5), (3, 4, 60000, 1), (40, 2, 60000, 59990)])
def test_small_weights_of_many_rows_add_up(T, n_heads, n, at, nats, dtype):
    """One row outweighs each of thousands by far, and they are what is left of
    the output.  A probability is rounded in its type, fp16's in steps of 2^-24
    at least, where the largest is 2^7 or more: each row's weight is off by half
    a step of its own, or by 2^-25 of 2^7.  An error d of a row's weight moves
    the output by d (v - out).  (bf16's least step is below all of this.)"""
    D = 128
    q, k, v, lengths = far_case(T, n_heads, D, n + T, n, dtype, nats, at)
    got = run_tree(q, k, v, lengths, scale=1.0).cpu().double()
    info = torch.finfo(dtype)
    for i in range(T):
        s = torch.zeros(n + i + 1, dtype=torch.float64)
        s[at] = nats
        w, vv = torch.softmax(s, 0), v[0, 0, :n + i + 1].double()
        want = w @ vv
        apart = (vv - want).abs()
        # rounded weights; fp32 scores (exact but for the factor log2 e), exponentials, sums
        off = w @ apart * (info.eps / 2 + (nats + 2) * 2.0 ** -22 + 2.0 ** -20)
        if dtype == F16:
            off = off + 2.0 ** -32 * apart.sum(0)
        off = off + (want.abs() + off) * info.eps / 2 + info.smallest_normal * info.eps
        for h in range(n_heads):
            assert ((got[0, i, h] - want).abs() <= off).all(), (i, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [40, 120])
@pytest.mark.parametrize("T,n_heads", [(3, 1), (3, 4), (8, 4), (16, 4), (40, 4)])
def test_strange_values_of_no_weight(T, n_heads, nats, dtype):
    """An infinity or a NaN in a row that a token sees is not lost where the
    row's weight rounds to zero, wherever the row lies: among other cached rows,
    in the last tile of them, or in the tree; and it reaches nobody else."""
    D, inf, nan = 64, float("inf"), float("nan")
    mask = torch.ones((1, T, T)).tril().bool()
    mask[0, :, 1] = torch.arange(T) % 2 == 1
    for n, at in ((60, 3), (199, 3), (199, 197), (3000, 2), (3000, 2990)):
        q, k, v, lengths = far_case(T, n_heads, D, n + T, n, dtype, nats, at)
        v[0, 0, 10, 5], v[0, 0, 11, 6], v[0, 0, n - 1, 7], v[0, 0, n - 1, 8] = inf, nan, -inf, nan
        v[0, 0, n + 1, 9], v[0, 0, n + 1, 10] = inf, nan
        got = run_tree(q, k, v, lengths, mask, scale=1.0).cpu()
        bad = ~got.isfinite()
        want = torch.zeros((1, T, n_heads, D), dtype=torch.bool)
        want[..., 5:9] = True
        want[:, 1::2, :, 9:11] = True
        assert torch.equal(bad, want), (n, at)
        assert got[..., [6, 8]].isnan().all() and got[:, 1::2, :, 10].isnan().all()


@pytest.mark.parametrize("kwargs,needle", [
    (dict(B=65535, T=1, nh=512, nkv=512, D=64), "2^32 threads"),
    (dict(B=65535, T=3, nh=65535, nkv=257, D=64), "2^30 query rows"),
])
def test_tree_rejects_what_no_launch_holds(kwargs, needle):
    ext = ng.extension()
    assert tree(ext, **kwargs) == INVALID
    assert needle in ext.last_error()
    assert ext.attention_tree_workspace_bytes(65535, 1, 512, 512, 64, 16) == 0


@pytest.mark.parametrize("scale", [3e38, -3e38, float("nan"), 1e39])
def test_tree_rejects_a_scale_beyond_fp32(scale):
    ext = ng.extension()
    assert tree(ext, scale=scale) == INVALID
    assert "scale" in ext.last_error()


@pytest.mark.gpu
def test_written_caches_are_marked_as_changed():
    """Autograd notices that a cache it has saved was written since."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn((1, 2, 4 * 128), generator=g).to(F16).to(dev)
    at = torch.arange(2, dtype=torch.int32, device=dev)[None]
    for which in range(2):
        caches = [torch.ones((1, 1, 8, 128), dtype=F16, device=dev) for _ in range(2)]
        before = [c._version for c in caches]
        w = torch.ones(1, dtype=F16, device=dev, requires_grad=True)
        y = (w * caches[which]).sum()
        glue.qk_norm_rope(x, *caches, at, at)
        assert [c._version > b for c, b in zip(caches, before)] == [True, True]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    caches = [torch.ones((1, 1, 8, 128), dtype=F16, device=dev) for _ in range(2)]
    before = [c._version for c in caches]
    glue.attention_tree(x, *caches, at[0, :1])  # only reads
    assert [c._version for c in caches] == before
    caches = [torch.ones((1, 8, 128), dtype=F16, device=dev) for _ in range(2)]
    before = [c._version for c in caches]
    glue.attention_decode(x[0, :1], *caches, 3)
    assert [c._version > b for c, b in zip(caches, before)] == [True, True]
    with torch.inference_mode():
        caches = [torch.ones((1, 1, 8, 128), dtype=F16, device=dev) for _ in range(2)]
        glue.qk_norm_rope(x, *caches, at, at)
    glue.qk_norm_rope(x, *caches, at, at)  # (such tensors count no versions)
    glue.attention_decode(x[0, :1], caches[0][0], caches[1][0], 3)


@pytest.mark.gpu
def test_a_batch_of_none():
    for T in (0, 3):
        q = torch.zeros((0, T, 256), dtype=F16, device=dev)
        c = torch.zeros((0, 1, 8, 64), dtype=F16, device=dev)
        n = torch.zeros(0, dtype=torch.int32, device=dev)
        i = torch.zeros((0, T), dtype=torch.int32, device=dev)
        mask = torch.zeros((0, T, T), dtype=torch.bool, device=dev)
        assert glue.attention_tree(q, c, c.clone(), n).shape == (0, T, 256)
        assert glue.attention_tree(q, c, c.clone(), n, mask, n).shape == (0, T, 256)
        assert glue.qk_norm_rope(q, c, c.clone(), i, i).shape == (0, T, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("up", [2, 4, 16, 36])
@pytest.mark.parametrize("power", [10, 11, 12, 12.5, 13])
@pytest.mark.parametrize("T,n_heads", [(1, 4), (7, 4), (15, 4), (40, 4)])
def test_scores_whose_steps_are_whole_powers_of_two(T, n_heads, power, up, dtype):
    """Scores of up to 2^26 in powers of two, where fp32 has steps of 8, and a
    maximum that rises by 4 up in a later tile: no probability overflows."""
    D, n = 128, 128
    base = 2.0 ** power if power != 12.5 else 6144.0
    q = torch.zeros((1, T, n_heads, D), dtype=dtype)
    k = torch.zeros((1, 1, n + T, D), dtype=dtype)
    q[..., 0], q[..., 1] = base, 4.0
    k[0, 0, 0, 0], k[0, 0, 0, 1] = base, 2.0
    k[0, 0, 64, 0], k[0, 0, 64, 1] = base, 2.0 + up
    v = torch.randn((1, 1, n + T, D), generator=torch.Generator().manual_seed(3)).to(dtype)
    got = run_tree(q, k, v, torch.tensor([n], dtype=torch.int32), scale=math.log(2.0)).cpu().double()
    # The scores differ by 4 up, each off by a few steps of 2^-24 of itself at most.
    far = 4.0 * up - 4 * base * base * 2.0 ** -23
    lo, hi = (v[0, 0, i].double() for i in (0, 64))
    info = torch.finfo(dtype)
    off = (lo - hi).abs() * min(1.0, 2.0 ** -far) + hi.abs() * info.eps + 2.0 ** -20
    assert ((got - hi).abs() <= off).all()

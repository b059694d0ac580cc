"""Paged caches: the append with norms and rotation to 16-bit and 8-bit pages,
attention over them with a window and first tokens that stay visible, and the
dense values they hold.

The oracle is plain float64 on the CPU.  Tolerances count roundings: half a
step of the output's type, half a step for the probabilities, the fp32 sums' own
errors, and, of 8-bit codes, the nearest one of a value known that well.
"""
from __future__ import annotations

import math
import os
import re
import shutil
import subprocess

import pytest
import torch

import nibblegemm_amd as ng
from nibblegemm_amd import build, glue, paged

OBJDUMP = os.path.join(os.path.dirname(os.path.dirname(build._hipcc())), "llvm", "bin", "llvm-objdump")
INVALID, WORKSPACE = 1, 3
P = 1 << 20  # aligned, never dereferenced
dev = "cuda"
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
DTYPES = [F16, BF16]
#: Exponents (not biased) that the append gives: codes times them are values of the type.
RANGE = {F16: (-15, 8), BF16: (-117, 120)}


def to_dev(t):
    return t.to(dev) if t is not None else None


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


# ---------------------------------------------------------------------------
# caches
# ---------------------------------------------------------------------------
class Cache:
    """A cache on the CPU and its copy on the GPU: pages in random places, those
    that no sequence has, and the rows behind the sequences' last, full of NaN."""

    def __init__(self, held, n_kv, D, page, dtype, bits=16, width=None, layout="head", seed=0,
                 spare=3, exponents=(-4, 2)):
        g = torch.Generator().manual_seed(seed)
        self.B, self.page, self.dtype, self.bits, self.layout = len(held), page, dtype, bits, layout
        width = max(1, -(-max(held) // page)) if width is None else width
        n = self.B * width + spare
        self.table = torch.randperm(n, generator=g)[:self.B * width].view(self.B, width).int()
        owned = torch.zeros((n, page), dtype=torch.bool)
        for b, h in enumerate(held):
            for m in range(width):
                owned[self.table[b, m], :max(0, min(page, h - m * page))] = True
        self.owned = owned
        shape = (n, n_kv, page, D)
        self.scales = None
        pools = []
        for _ in range(2):
            x = torch.randn(shape, generator=g)
            x = x.to(dtype) if bits == 16 else (64 * x).clamp(-448, 448).to(F8)
            nan = torch.full((), math.nan).to(x.dtype)
            pools.append(torch.where(owned[:, None, :, None], x.float(), nan.float()).to(x.dtype))
        self.k, self.v = pools
        if bits == 8:
            self.scales = tuple(torch.randint(127 - 6 + exponents[0], 127 - 6 + exponents[1],
                                              (n, n_kv), generator=g).to(torch.uint8)
                                for _ in range(2))

    def gpu(self, t):
        if self.layout == "row":  # a row's heads side by side
            return t.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
        if self.layout == "part":  # rows of a wider pool
            wide = torch.zeros((*t.shape[:3], t.shape[3] + 32), dtype=t.dtype, device=dev)
            wide[..., 16:16 + t.shape[3]] = t.to(dev)
            return wide[..., 16:16 + t.shape[3]]
        return t.to(dev)

    def on_gpu(self):
        scales = None if self.scales is None else tuple(s.to(dev) for s in self.scales)
        return self.gpu(self.k), self.gpu(self.v), self.table.to(dev), scales

    def rows(self, which, b, k=None, scales=None):
        """Sequence b's rows [width page, n_kv, D] in float64, and which have a page."""
        pool = (self.k, self.v)[which] if k is None else k
        out, there = [], []
        for page in self.table[b].tolist():
            ok = 0 <= page < pool.shape[0]
            x = pool[page if ok else 0].double()
            if self.bits == 8:
                e = (self.scales if scales is None else scales)[which][page if ok else 0]
                x = x * torch.exp2(e.double() - 127)[:, None, None]
            out.append(x.transpose(0, 1))
            there += [ok] * self.page
        if not out:
            return torch.zeros((0, pool.shape[1], pool.shape[3]), dtype=torch.float64), \
                torch.zeros(0, dtype=torch.bool)
        return torch.cat(out), torch.tensor(there)


# ---------------------------------------------------------------------------
# attention: the oracle
# ---------------------------------------------------------------------------
def oracle_attention(q, cache, lengths, sizes, window, sinks, scale):
    """[B, T, heads, D], and a bound of the error per element."""
    B, T, n_heads, D = q.shape
    n_kv = cache.k.shape[1]
    info = torch.finfo(q.dtype)
    out = torch.zeros((B, T, n_heads, D), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b in range(B):
        k, there = cache.rows(0, b)
        v, _ = cache.rows(1, b)
        room = len(there)
        n = min(max(int(lengths[b]), 0), room)
        live = T if sizes is None else min(max(int(sizes[b]), 0), T)
        total = min(n + live, room)
        if live == 0 or total == 0:
            continue
        j = torch.arange(total)
        r = n + torch.arange(live)[:, None]
        seen = (j <= r) & there[:total]
        if window is not None:
            seen &= (r - j < window) | (j < sinks)
        some = seen.any(0)
        j, seen = j[some], seen[:, some]
        if len(j) == 0:
            continue
        for h in range(n_heads):
            kk, vv = k[j, h // (n_heads // n_kv)], v[j, h // (n_heads // n_kv)]
            qq = q[b, :live, h].double()
            s = torch.where(seen, qq @ kk.t() * scale, -math.inf)
            none = ~seen.any(1)
            p = torch.where(none[:, None], 0.0, torch.softmax(s, 1))
            odd = ~vv.isfinite().all(1)
            fine = torch.where(vv.isfinite(), vv, 0.0)
            o = p @ fine
            for i in odd.nonzero().flatten().tolist():
                o += torch.where(seen[:, i, None], torch.where(vv[i].isfinite(), 0.0, vv[i]), 0.0)
            a = p @ fine.abs()
            away = (torch.where(seen, qq.abs() @ kk.abs().t(), 0.0).amax(1) * abs(scale) * (D + 4)
                    * 2.0 ** -24 + torch.where(seen, s.abs(), 0.0).amax(1) * 2.0 ** -22)[:, None]
            off = o.abs().nan_to_num(0.0, 0.0, 0.0) * info.eps / 2 \
                + a * (info.eps / 2 + 2 * away + 2.0 ** -20) + info.smallest_normal * info.eps
            if q.dtype == F16:  # probabilities below 2^-14 of the largest: steps of 2^-24
                off = off + seen.sum(1, keepdim=True) * 2.0 ** -25 * fine.abs().max()
            out[b, :live, h], bound[b, :live, h] = o, off
    return out, bound


def run_attention(q, cache, lengths, sizes=None, window=None, sinks=0, scale=None, table=None):
    B, T, n_heads, D = q.shape
    k, v, t, scales = cache.on_gpu()
    t = t if table is None else table.to(dev)
    return paged.attention_paged(to_dev(q.reshape(B, T, -1)), k, v, t, to_dev(lengths),
                                 to_dev(sizes), window, sinks, scale, scales).view(B, T, n_heads, D)


def check_attention(q, cache, lengths, sizes=None, window=None, sinks=0, scale=None):
    got = run_attention(q, cache, lengths, sizes, window, sinks, scale)
    want, bound = oracle_attention(q, cache, lengths, sizes, window, sinks,
                                   q.shape[3] ** -0.5 if scale is None else scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or (off <= 0).all(), f"{off.max():.3g} beyond its bound"
    return got


def queries(B, T, n_heads, D, dtype, seed=0):
    g = torch.Generator().manual_seed(1000 + seed)
    return (1.5 * torch.randn((B, T, n_heads, D), generator=g)).to(dtype)


def attention_case(T, n_heads, n_kv, D, page, lengths, dtype, bits=16, sizes=None, layout="head",
                   seed=0, **more):
    live = [T] * len(lengths) if sizes is None else sizes
    cache = Cache([n + t for n, t in zip(lengths, live)], n_kv, D, page, dtype, bits, layout=layout,
                  seed=seed, **more)
    return (queries(len(lengths), T, n_heads, D, dtype, seed), cache, ints(lengths),
            None if sizes is None else ints(sizes))


# ---------------------------------------------------------------------------
# the append: the oracle
# ---------------------------------------------------------------------------
def turned(x, w, eps, rope, at, interleaved):
    """Heads x [T, heads, D] normalised and rotated, and magnitudes that bound
    their rounding errors."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if rope is None:
        return x, x.abs()
    cos, sin = (t.double()[at.clamp(0, t.shape[0] - 1)][:, None] for t in rope)
    R = 2 * cos.shape[-1]
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y, mag = x.clone(), x.abs().clone()
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    mag[..., a] = mag[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, mag


def check_append(cache, qkv, lengths, sizes=None, qw=None, kw=None, eps=1e-5, rope=None,
                 interleaved=False, positions=None):
    """Runs the append on a copy of ``cache`` on the GPU and checks everything
    it holds afterwards; returns the copy's tensors and q."""
    B, T, width = qkv.shape
    n, n_kv, page, D = cache.k.shape
    n_heads = width // D - 2 * n_kv
    k, v, table, scales = cache.on_gpu()
    got = paged.paged_append(to_dev(qkv), k, v, table, to_dev(lengths), to_dev(sizes), to_dev(qw),
                             to_dev(kw), eps, None if rope is None else tuple(map(to_dev, rope)),
                             interleaved, to_dev(positions), scales)
    assert got.shape == (B, T, n_heads * D) and got.dtype == qkv.dtype
    info = torch.finfo(qkv.dtype)
    slack = (D / 2 + 10) * 2.0 ** -24  # fp32: D additions of squares, halved; ten operations
    after = (k.cpu(), v.cpu())
    after_scales = None if scales is None else tuple(s.cpu() for s in scales)
    touched = torch.zeros((n, page), dtype=torch.bool)
    moved = torch.zeros(n, dtype=torch.bool)
    for b in range(B):
        x = qkv[b].double().view(T, -1, D)
        room = cache.table.shape[1] * page
        first = min(max(int(lengths[b]), 0), room)
        live = T if sizes is None else min(max(int(sizes[b]), 0), T)
        row = first + torch.arange(T)
        at = row if positions is None else positions[b].long()
        q, q_mag = turned(x[:, :n_heads], qw, eps, rope, at, interleaved)
        kk, k_mag = turned(x[:, n_heads:n_heads + n_kv], kw, eps, rope, at, interleaved)
        vv = x[:, n_heads + n_kv:]
        good = (torch.arange(T) < live) & (row < room)
        if rope is not None:
            good &= (at >= 0) & (at < rope[0].shape[0])
        pages = cache.table[b, (row // page).clamp(max=max(cache.table.shape[1] - 1, 0))] \
            if room else torch.full((T,), -1)
        good &= (pages >= 0) & (pages < n)
        q = torch.where(good[:, None, None], q, 0.0)
        off = (got[b].cpu().double().view(T, n_heads, D) - q).abs()
        assert (off <= q.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2
                + q_mag * slack).all()
        for which, (y, slop) in enumerate(((kk, k_mag * slack), (vv, 0 * vv))):
            pool, old = after[which], (cache.k, cache.v)[which]
            for m in row[good].div(page, rounding_mode="floor").unique().tolist():
                to = int(cache.table[b, m])
                new = good & (row // page == m)
                r = row[new] % page
                touched[to, r] = True
                held = pool[to][:, r].transpose(0, 1)  # [tokens, n_kv, D]
                want, err = y[new], slop[new].nan_to_num(0.0, 0.0)
                if cache.bits == 16:
                    off = (held.double() - want).abs()
                    assert (off <= want.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2
                            + err).all()
                    continue
                before = min(max(first - m * page, 0), page)
                low, high = RANGE[qkv.dtype]
                most = torch.finfo(qkv.dtype).max
                capped = want.clamp(-most, most)
                sized = torch.where(want.isfinite(), capped, 0.0).abs()
                for h in range(n_kv):
                    e = int(after_scales[which][to, h]) - 127
                    need = [max(low, min(high, math.ceil(math.log2(max(t, 1e-300) / 448))))
                            for t in ((sized - err).clamp(min=0)[:, h].max().item(),
                                      (sized + err)[:, h].max().item())]
                    was = int(cache.scales[which][to, h]) - 127
                    if before:
                        need = [max(x, was) for x in need]
                    assert need[0] <= e <= need[1], (which, to, h, e, need)
                    last = 240.0 if e == high else 448.0
                    u = (capped[:, h] / 2.0 ** e).clamp(-last, last)
                    code = held[:, h]
                    assert torch.equal(code.isnan(), ~want[:, h].isfinite())
                    fine = want[:, h].isfinite()
                    near = u.float().to(F8).double()
                    exact = err[:, h] == 0
                    assert torch.equal(code.double()[fine & exact], near[fine & exact])
                    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
                    reach = step / 2 + 2 * err[:, h] / 2.0 ** e
                    assert ((code.double() - u).abs() <= reach)[fine].all()
                    if before:
                        moved[to] = True
                        earlier = old[to, h, :before].float()
                        want_codes = (earlier * 2.0 ** (was - e)).to(F8)
                        have = pool[to, h, :before]
                        nan = want_codes.isnan()
                        assert torch.equal(have.isnan(), nan)
                        assert torch.equal(have.float()[~nan], want_codes.float()[~nan])
    bits = torch.int16 if cache.bits == 16 else torch.uint8
    for pool, old, sc, osc in zip(after, (cache.k, cache.v), after_scales or (None,) * 2,
                                  cache.scales or (None,) * 2):
        still = ~touched
        still[moved] = False
        a, o = pool.transpose(1, 2)[still], old.transpose(1, 2)[still]
        assert torch.equal(a.view(bits), o.view(bits)), "other rows stay as they were"
        for page_, in zip(moved.nonzero().flatten().tolist()):  # rows behind the new ones
            last = touched[page_].nonzero().max() + 1
            assert torch.equal(pool[page_, :, last:].view(bits), old[page_, :, last:].view(bits))
        if sc is not None:
            assert torch.equal(sc[~touched.any(1)], osc[~touched.any(1)])
    return got, k, v, table, scales


def append_case(T, n_heads, n_kv, D, page, lengths, dtype, bits=16, sizes=None, layout="head",
                seed=0, size=1.0, **more):
    cache = Cache([n + T for n in lengths], n_kv, D, page, dtype, bits, layout=layout, seed=seed,
                  **more)
    g = torch.Generator().manual_seed(2000 + seed)
    qkv = size * torch.randn((len(lengths), T, (n_heads + 2 * n_kv) * D), generator=g)
    return cache, qkv.to(dtype), ints(lengths), None if sizes is None else ints(sizes)


def weights(D, dtype, seed=0):
    g = torch.Generator().manual_seed(3000 + seed)
    return [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)]


# ---------------------------------------------------------------------------
# refusals (CPU)
# ---------------------------------------------------------------------------
CACHE = dict(k=P, v=P, ks=None, vs=None, table=P, pages=9, nkv=2, page=16, D=128, width=4,
             st=(4096, 2048, 128))


def cache_args(c):
    return (c["k"], c["v"], c["ks"], c["vs"], c["table"], c["pages"], c["nkv"], c["page"], c["D"],
            c["width"], *c["st"], *c["st"])


def split(kwargs):
    return {**CACHE, **{k: v for k, v in kwargs.items() if k in CACHE}}, \
        {k: v for k, v in kwargs.items() if k not in CACHE}


def append(ext, **kwargs):
    c, kw = split(kwargs)
    a = dict(qkv=P, dt=0, B=1, T=2, nh=4, lengths=P, sizes=None, pos=None, qw=None, kw=None, eps=1e-5,
             cos=None, sin=None, rows=0, dim=0, inter=0, out=P)
    a.update(kw)
    return ext.paged_append(a["qkv"], a["dt"], a["B"], a["T"], a["nh"], *cache_args(c), a["lengths"],
                            a["sizes"], a["pos"], a["qw"], a["kw"], a["eps"], a["cos"], a["sin"],
                            a["rows"], a["dim"], a["inter"], a["out"], None)


def attend(ext, **kwargs):
    c, kw = split(kwargs)
    a = dict(q=P, dt=0, B=1, T=2, nh=4, lengths=P, sizes=None, window=0, sinks=0, scale=0.1, out=P,
             ws=None, wsb=0)
    a.update(kw)
    return ext.attention_paged(a["q"], a["dt"], a["B"], a["T"], a["nh"], *cache_args(c),
                               a["lengths"], a["sizes"], a["window"], a["sinks"], a["scale"],
                               a["out"], a["ws"], a["wsb"], None)


def values(ext, **kwargs):
    c, kw = split(kwargs)
    a = dict(dt=0, B=1, lengths=P, rows=64, ko=P, vo=P)
    a.update(kw)
    return ext.paged_values(*cache_args(c), a["dt"], a["B"], a["lengths"], a["rows"], a["ko"],
                            a["vo"], None)


@pytest.mark.parametrize("call", [append, attend, values])
@pytest.mark.parametrize("kwargs,needle", [
    (dict(dt=2), "dtype"), (dict(D=96), "head_dim"), (dict(nkv=0), "n_kv_heads"),
    (dict(page=48), "a page"), (dict(page=8), "a page"), (dict(page=512), "a page"),
    (dict(pages=-1), "n_pages"), (dict(pages=1 << 31), "n_pages"), (dict(width=-1), "rows"),
    (dict(width=1 << 26), "2^30 rows"), (dict(B=-1), "batch"), (dict(B=65536), "batch"),
    (dict(ks=P), "both"), (dict(st=(4096, 2044, 128)), "strides"),
    (dict(st=(4096, 2056, 128), ks=P, vs=P), "strides"), (dict(st=(-8, 2048, 128)), "strides"),
    (dict(st=(0, 0, (1 << 22) + 8)), "2^22"), (dict(k=0), "null"), (dict(v=0), "null"),
    (dict(table=0), "null"), (dict(k=P + 8), "aligned"), (dict(table=P + 2), "aligned"),
    (dict(lengths=0), "null"), (dict(lengths=P + 1), "aligned"),
])
def test_cache_rejections(call, kwargs, needle):
    ext = ng.extension()
    assert call(ext, **kwargs) == INVALID
    assert needle in ext.last_error()


@pytest.mark.parametrize("kwargs,needle", [
    (dict(nh=0), "n_heads"), (dict(T=(1 << 20) + 1), "tokens"), (dict(cos=P), "both"),
    (dict(cos=P, sin=P, rows=0, dim=128), "rows"), (dict(cos=P, sin=P, rows=4, dim=24), "multiple of 16"),
    (dict(cos=P, sin=P, rows=4, dim=0), "multiple of 16"), (dict(cos=P, sin=P, rows=4, dim=144), "of 16"),
    (dict(inter=2), "interleaved"), (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"),
    (dict(qkv=0), "null"), (dict(out=0), "null"), (dict(qkv=P + 8), "aligned"),
    (dict(kw=P + 8), "aligned"), (dict(cos=P + 4, sin=P, rows=4, dim=32), "aligned"),
    (dict(sizes=P + 2), "aligned"), (dict(pos=P + 2), "aligned"),
    (dict(B=65535, T=1 << 20), "too many"), (dict(B=65535, T=1 << 20, ks=P, vs=P), "too many"),
])
def test_append_rejections(kwargs, needle):
    ext = ng.extension()
    assert append(ext, **kwargs) == INVALID
    assert needle in ext.last_error()


@pytest.mark.parametrize("kwargs,needle", [
    (dict(nh=5), "multiple of n_kv_heads"), (dict(T=(1 << 20) + 1), "tokens"),
    (dict(scale=float("inf")), "scale"), (dict(scale=3e38), "scale"), (dict(window=-1), "window"),
    (dict(window=(1 << 30) + 1), "window"), (dict(sinks=-1), "sinks"),
    (dict(sinks=(1 << 30) + 1), "sinks"), (dict(q=0), "null"), (dict(out=0), "null"),
    (dict(q=P + 8), "aligned"), (dict(sizes=P + 2), "aligned"), (dict(B=65535, T=1 << 20), "2^30"),
    (dict(B=65535, T=1, nh=512, nkv=512, D=64), "2^32 threads"),
])
def test_attention_rejections(kwargs, needle):
    ext = ng.extension()
    assert attend(ext, **kwargs) == INVALID
    assert needle in ext.last_error()


@pytest.mark.parametrize("kwargs,needle", [
    (dict(rows=-1), "rows"), (dict(rows=1 << 30), "rows"), (dict(ko=0), "null"),
    (dict(vo=P + 8), "aligned"), (dict(B=65535, rows=1 << 20), "too many"),
])
def test_values_rejections(kwargs, needle):
    ext = ng.extension()
    assert values(ext, **kwargs) == INVALID
    assert needle in ext.last_error()


def test_attention_workspace():
    ext = ng.extension()
    assert ext.attention_paged_workspace_bytes(1, 1, 32, 8, 128, 128) == (0, 0)
    need, counters = ext.attention_paged_workspace_bytes(1, 1, 32, 8, 128, 65536)
    assert need > counters > 0 and counters % 256 == 0
    assert ext.attention_paged_workspace_bytes(1, 1, 32, 8, 96, 65536) == (0, 0)  # a refused plan
    # the tiles of all sequences are counted in 32 bits: not where they may pass them
    assert ext.attention_paged_workspace_bytes(63, 1, 8, 2, 64, (1 << 30) - 16)[0] > 0
    assert ext.attention_paged_workspace_bytes(400, 1, 8, 2, 64, (1 << 30) - 16) == (0, 0)
    big = dict(T=1, nh=32, nkv=8, width=4096)
    assert attend(ext, **big) == WORKSPACE and "workspace" in ext.last_error()
    assert attend(ext, **big, ws=P, wsb=need - 1) == WORKSPACE
    assert attend(ext, **big, ws=P + 64, wsb=need) == WORKSPACE and "256-byte" in ext.last_error()


def test_library_takes_empty_sizes():
    ext = ng.extension()
    for kwargs in (dict(B=0), dict(T=0)):
        assert append(ext, qkv=0, out=0, **kwargs) == 0
        assert attend(ext, q=0, out=0, **kwargs) == 0
    assert values(ext, B=0, ko=0) == 0 and values(ext, rows=0, ko=0) == 0


def test_refusals_without_a_gpu():
    x, c = torch.zeros((1, 2, 512), dtype=F16), torch.zeros((3, 1, 16, 128), dtype=F16)
    t, n = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: paged.paged_append(x, c, c, t, n), lambda: paged.paged_values(c, c, t, n),
                 lambda: paged.attention_paged(x, c, c, t, n)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    c8, s = c.to(F8), torch.zeros((3, 1), dtype=torch.uint8)
    for call in (lambda: paged.paged_append(x, c8, c8, t, n, scales=(s, s)),
                 lambda: paged.paged_values(c8, c8, t, n, (s, s)),
                 lambda: paged.attention_paged(x, c8, c8, t, n, scales=(s, s))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        paged.attention_paged(x.float(), c, c, t, n)
    with pytest.raises(ValueError, match="rows"):
        paged.paged_cache(4, 2, 24)
    with pytest.raises(RuntimeError, match="dtype"):
        paged.paged_cache(4, 2, 16, dtype=torch.float32)


# ---------------------------------------------------------------------------
# the append (GPU)
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,n_heads,n_kv,D,page,lengths", [
    (1, 1, 1, 64, 16, [0]), (1, 32, 8, 128, 16, [40]), (3, 5, 1, 128, 32, [0, 31, 62]),
    (17, 8, 2, 64, 16, [15, 16, 17, 0]), (130, 4, 4, 128, 64, [5]), (70, 2, 2, 64, 128, [127, 3]),
    (300, 3, 1, 128, 256, [0, 255]), (40, 4, 2, 128, 128, [100, 7, 0]), (65, 2, 1, 64, 256, [200]),
    (64, 2, 2, 64, 64, [64, 1])])
def test_append(T, n_heads, n_kv, D, page, lengths, dtype, bits):
    qw, kw = weights(D, dtype)
    rope = glue.rope_tables(max(lengths) + T, D, device="cpu")
    check_append(*append_case(T, n_heads, n_kv, D, page, lengths, dtype, bits, seed=T), qw, kw,
                 rope=rope)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,R,interleaved", [
    (128, 128, True), (128, 64, False), (128, 32, True), (128, 16, False), (64, 64, True),
    (64, 48, False), (128, 112, True), (64, 16, True), (64, 0, False)])
def test_append_rotations(D, R, interleaved, bits):
    case = append_case(9, 3, 2, D, 16, [3, 30], BF16, bits, seed=R)
    rope = glue.rope_tables(50, R, device="cpu") if R else None
    check_append(*case, rope=rope, interleaved=interleaved)
    check_append(*case, *weights(D, BF16), rope=rope, interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("layout", ["row", "part"])
@pytest.mark.parametrize("D", [64, 128])
def test_append_layouts_and_one_norm(D, layout, bits):
    case = append_case(20, 6, 2, D, 32, [7, 33, 0], F16, bits, sizes=[20, 5, 13], layout=layout)
    qw, kw = weights(D, F16)
    check_append(*case, qw=qw, rope=glue.rope_tables(60, D, device="cpu"))
    check_append(*case, kw=kw)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_append_padding_goes_nowhere(bits):
    """Tokens behind the sizes, without a page, beyond the table, or at positions
    that the tables do not have; counts of any value."""
    cache, qkv, lengths, _ = append_case(40, 4, 2, 128, 16, [10, 20, 40, 30, 5], BF16, bits, width=5)
    cache.table[0, 1], cache.table[1, 2], cache.table[1, 3] = -1, cache.k.shape[0], 2 ** 31 - 1
    positions = torch.arange(40).expand(5, 40).clone()
    positions[3, 3], positions[3, 4], positions[4, 0], positions[4, 39] = -1, 50, -2 ** 31, 2 ** 31 - 1
    rope = glue.rope_tables(50, 128, device="cpu")
    for sizes in (None, ints([40, 7, 0, -3, 2 ** 31 - 1])):
        for n in (lengths, ints([2 ** 31 - 1, -5, 70, 64, 79]), ints([0, 80, 81, 16, -2 ** 31])):
            check_append(cache, qkv, n, sizes, rope=rope, positions=positions.int())
            check_append(cache, qkv, n, sizes)


@pytest.mark.gpu
def test_append_to_no_pages_at_all():
    for bits in (16, 8):
        cache, qkv, lengths, _ = append_case(3, 4, 2, 64, 16, [0], F16, bits)
        for table in (torch.full((1, 3), -1, dtype=torch.int32), torch.zeros((1, 0), dtype=torch.int32)):
            k, v, _, scales = cache.on_gpu()
            before = [t.clone().view(torch.uint8) for t in (k, v)]
            q = paged.paged_append(to_dev(qkv), k, v, table.to(dev), to_dev(lengths), scales=scales)
            assert not q.any()
            assert all(torch.equal(a.view(torch.uint8), b) for a, b in zip((k, v), before))
            out = paged.attention_paged(q + 1, k, v, table.to(dev), to_dev(lengths), scales=scales)
            assert not out.any()
            dense = paged.paged_values(k, v, table.to(dev), to_dev(lengths) + 40, scales)
            assert not dense[0].any() and dense[0].shape[2] == 16 * table.shape[1]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T", [1, 40, 200])
def test_attention_over_no_pages_at_all(T, bits):
    k, v, scales = paged.paged_cache(0, 1, 16, 64, F16 if bits == 16 else F8)
    table = torch.zeros((2, 40), dtype=torch.int32, device=dev)
    n = to_dev(ints([0, 400]))
    q = torch.full((2, T, 64), 3.0, dtype=F16, device=dev)
    out = paged.attention_paged(q, k, v, table, n, scales=scales)
    assert torch.equal(out, torch.zeros_like(q))
    dense = paged.paged_values(k, v, table, n, scales, rows=500)
    assert not dense[0].any() and not dense[1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 32), (128, 64), (64, 128), (128, 256)])
def test_append_raises_the_scale(D, page, dtype):
    """Earlier rows of small and large powers, and new ones far above and below
    them: the codes are halved as often as the power rises."""
    for seed, (size, exponents) in enumerate([(1.0, (-14, -10)), (60.0, (-6, 0)), (2.0 ** -12, (0, 3)),
                                              (2.0 ** -30, (-8, -5)), (900.0, (-9, -8))]):
        check_append(*append_case(5, 2, 2, D, page, [page - 3, page // 2, 1, page], dtype, 8, seed=seed,
                                  size=size, exponents=exponents))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_extremes_in_8_bits(dtype):
    """Zeros, subnormals, the largest values, infinities and NaN; values at and
    next to the borders of a power and of a rounding."""
    D, T = 128, 16
    most, least = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    inf, nan = math.inf, math.nan
    top = 2.0 ** -3 * 448
    up = top * (1 + torch.finfo(dtype).eps)
    rows = [[0.0], [least], [least / 4], [most], [-most, 1.0], [inf, 3.0], [nan, 5.0], [nan], [-inf],
            [inf, -inf, most], [top], [up], [top, 17.0, 18.0, 19.0, -17.0, 2 ** -9.0, 1.5 * 2 ** -9],
            [448.0 * 2 ** 6, 1.0], [240.0 * 2 ** 7], [1.0, 2.0 ** -10, 3 * 2.0 ** -10]]
    qkv = torch.zeros((len(rows), T, 3 * D))
    for b, r in enumerate(rows):
        for i, x in enumerate(r):
            qkv[b, 3 + i % 5, D + 7 * i] = x  # key
            qkv[b, 2 + i % 5, 2 * D + 11 * i] = x  # value
    for lengths in ([0] * len(rows), [5] * len(rows)):
        cache = Cache([21] * len(rows), 1, D, 16, dtype, 8, exponents=(-9, -7))
        got, k, v, table, scales = check_append(cache, qkv.to(dtype), ints(lengths))
        if lengths[0] == 0:
            # What the pages stand for is finite in the 16-bit type, and near.
            dk, dv = paged.paged_values(k, v, table, to_dev(ints([16] * len(rows))), scales, dtype)
            for b in (0, 1, 2, 3, 4, 10, 11, 12, 13, 14, 15):
                for dense, at in ((dk, D), (dv, 2 * D)):
                    want = qkv[b, :16, at:at + D].to(dtype).double()
                    have = dense[b, 0, :16].cpu().double()
                    assert have.isfinite().all()
                    # a normal code is off by 2^-4 of it at most (the largest of all by a
                    # step of 240's, 2^-4), a subnormal one by half its step, 2^-9 of the power
                    power = 2.0 ** (scales[0 if at == D else 1][table[b, 0], 0].double().cpu() - 127)
                    assert ((have - want).abs() <= want.abs() * 2.0 ** -4 + power * 2.0 ** -10).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [16, 8])
def test_values(bits, dtype):
    for D, page, layout in ((64, 16, "head"), (128, 32, "row"), (128, 256, "part"), (64, 64, "row")):
        held = [0, 1, page, 2 * page + 5, 3 * page]
        cache = Cache(held, 3, D, page, dtype, bits, width=4, layout=layout)
        cache.table[3, 1], cache.table[4, 0] = -1, cache.k.shape[0]
        k, v, table, scales = cache.on_gpu()
        for rows in (None, 1, page + 3, 5 * page):
            for n in (held, [-1, 2 ** 31 - 1, 7, 3, 0]):
                got = paged.paged_values(k, v, table, to_dev(ints(n)), scales, dtype, rows)
                for which in range(2):
                    assert got[which].dtype == dtype
                    assert got[which].shape == (5, 3, 4 * page if rows is None else rows, D)
                    for b in range(5):
                        x, there = cache.rows(which, b)
                        r = torch.arange(len(x))
                        x = torch.where(((r < n[b]) & there)[:, None, None], x, 0.0).transpose(0, 1)
                        x = torch.nn.functional.pad(x, (0, 0, 0, page))[:, :got[which].shape[2]]
                        have = got[which][b].cpu()
                        assert torch.equal(have.isnan(), x.isnan())
                        assert torch.equal(have.double().nan_to_num(), x.nan_to_num())


# ---------------------------------------------------------------------------
# attention (GPU)
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,n_heads,n_kv,D,page,lengths", [
    (1, 1, 1, 64, 16, [0]), (1, 32, 8, 128, 16, [1000]), (1, 4, 1, 128, 32, [0, 1, 63, 64, 65, 300]),
    (1, 5, 1, 64, 64, [700, 30]), (3, 8, 2, 128, 128, [125, 500]), (4, 8, 2, 64, 16, [77, 1500, 0]),
    (9, 6, 2, 128, 256, [3, 400]), (17, 4, 4, 128, 64, [47, 900]), (33, 8, 4, 64, 32, [0, 31, 260]),
    (70, 4, 2, 128, 16, [5, 64, 130]), (200, 2, 1, 128, 32, [0, 111]), (1, 64, 1, 128, 64, [500]),
    (129, 5, 1, 64, 128, [200]), (2, 16, 2, 128, 32, [2500, 60])])
def test_attention(T, n_heads, n_kv, D, page, lengths, dtype, bits):
    check_attention(*attention_case(T, n_heads, n_kv, D, page, lengths, dtype, bits, seed=T))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window,sinks", [
    (1, 0), (1, 1), (2, 5), (16, 4), (63, 0), (64, 64), (65, 70), (100, 130), (300, 1), (5000, 3),
    (1 << 40, 0), (40, 1 << 40)])
@pytest.mark.parametrize("T,n_heads,n_kv,D,page", [
    (1, 4, 1, 128, 16), (5, 8, 2, 64, 32), (24, 4, 2, 128, 64), (150, 2, 1, 64, 128)])
def test_windows(T, n_heads, n_kv, D, page, window, sinks, bits):
    lengths = [0, 3, 64, 200, 777]
    dtype = F16 if window % 2 else BF16
    q, cache, lengths, sizes = attention_case(T, n_heads, n_kv, D, page, lengths, dtype, bits,
                                              sizes=[T, T, max(T - 3, 1), T, (T + 1) // 2], seed=sinks % 99)
    whole = check_attention(q, cache, lengths, sizes, window, sinks)
    # the pages that no token sees any more may go
    for b, n in enumerate(lengths.tolist()):
        for m in range(cache.table.shape[1]):
            if m * page >= sinks and (m + 1) * page <= n - window + 1:
                cache.table[b, m] = -1
    assert torch.equal(check_attention(q, cache, lengths, sizes, window, sinks), whole)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T,n_heads", [(1, 4), (6, 4), (12, 4), (40, 4)])
def test_missing_pages(T, n_heads, bits):
    q, cache, lengths, _ = attention_case(T, n_heads, 1, 128, 16, [300, 500, 40, 0], BF16, bits, spare=5)
    g = torch.Generator().manual_seed(T)
    gone = torch.rand(cache.table.shape, generator=g) < 0.3
    gone[2] = True  # a sequence without pages
    cache.table[gone] = torch.where(torch.rand(int(gone.sum()), generator=g) < 0.5, -1,
                                    cache.k.shape[0] + 7).int()
    got = check_attention(q, cache, lengths)
    assert not got[2].any()
    check_attention(q, cache, lengths, None, 100, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["row", "part"])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_layouts(D, bits, layout):
    check_attention(*attention_case(7, 6, 2, D, 32, [50, 333], F16, bits, layout=layout))
    check_attention(*attention_case(60, 6, 2, D, 16, [50, 333], BF16, bits, layout=layout))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_counts_of_any_value(bits):
    q, cache, _, _ = attention_case(5, 4, 2, 64, 16, [59] * 6, F16, bits)
    n, t = [59, -1, 62, 64, 2 ** 31 - 1, -2 ** 31], [5, 5, 5, -2, 2 ** 31 - 1, 0]
    # (rows that the clamped counts reach hold values)
    cache.k, cache.v = (torch.nan_to_num(x.float(), 0.5).to(x.dtype) for x in (cache.k, cache.v))
    for sizes in (None, ints(t), ints(t[::-1])):
        check_attention(q, cache, ints(n), sizes)
        check_attention(q, cache, ints(n), sizes, 20, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 2.0 ** -40])
@pytest.mark.parametrize("bits", [16, 8])
def test_scales_of_either_sign(scale, bits):
    check_attention(*attention_case(3, 4, 2, 64, 32, [90, 10], F16, bits), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,n_heads", [(1, 4), (6, 2), (6, 8), (24, 8), (40, 8), (90, 8)])
def test_strange_values_in_rows_that_some_see(T, n_heads, dtype, bits):
    """An infinity or a NaN in the values of a row that later tokens alone see,
    and, under a window, earlier ones alone, comes out of those."""
    for n, window, sinks in ((3, None, 0), (130, None, 0), (200, 30, 4), (100, 7, 70)):
        q, cache, lengths, _ = attention_case(T, n_heads, 2, 128, 16, [n, n], dtype, bits)
        for at, (d, x) in {n + T // 2: (5, math.inf), n + T - 1: (9, -math.inf), n + T // 3: (70, math.nan),
                           n - 3: (100, math.nan), max(n - 40, 0): (101, math.nan), 1: (127, -math.inf)}.items():
            x = x if bits == 16 else math.nan
            cache.v[cache.table[0, at // 16], :, at % 16, d] = x
        q[..., :] *= 0.25  # (every weight far from zero)
        check_attention(q, cache, lengths, None, window, sinks)
        cache.k[cache.table[0, (n + T - 1) // 16], :, (n + T - 1) % 16] = math.nan  # the last token's own
        got = check_attention(q, cache, lengths, None, window, sinks)
        assert got[0, -1].isnan().all() and not got[1].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_8_bit_values_beyond_the_type(dtype):
    """Powers of two that a caller wrote: a value that the 16-bit type does not
    hold is infinite, of the rows that a token sees alone."""
    high = 127 + RANGE[dtype][1]
    q, cache, lengths, _ = attention_case(6, 4, 1, 64, 16, [14], dtype, 8)
    q *= 0.01
    cache.scales[0][:] = 110
    page = int(cache.table[0, 1])  # rows 16 ..: tokens 2 and later
    cache.scales[1][page] = high
    cache.v[page, 0] = cache.v[page, 0].float().clamp(-8, 8).to(F8)
    cache.v[page, 0, 1, 3] = 448.0  # row 17, token 3's own
    got = run_attention(q, cache, lengths).cpu()
    want = torch.zeros((1, 6, 4, 64), dtype=torch.bool)
    want[:, 3:, :, 3] = True
    assert torch.equal(~got.isfinite(), want) and (got[want] == math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n_kv,n_heads,B", [(1, 2, 70), (1, 1, 300), (2, 4, 33), (1, 3, 511), (1, 1, 600)])
def test_many_sequences_of_uneven_lengths(n_kv, n_heads, B, bits):
    g = torch.Generator().manual_seed(B)
    lengths = (torch.rand(B, generator=g) ** 6 * 2000).int().tolist()
    sizes = torch.randint(0, 3, (B,), generator=g).int().tolist()
    case = attention_case(2, n_heads, n_kv, 64, 32, lengths, F16, bits, sizes=sizes)
    check_attention(*case)
    check_attention(*case, 150, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T,n_heads,n_kv,B", [(40, 1, 1, 100), (34, 2, 2, 255), (130, 1, 1, 9), (1, 8, 8, 300),
                                              (2, 64, 64, 9), (9, 16, 2, 70)])
def test_many_sequences_of_many_rows_or_heads(T, n_heads, n_kv, B, bits):
    """More sequences than a wave has lanes, of calls that are split or not, with and
    without tokens, by either kernel; more kv heads than room for shares."""
    g = torch.Generator().manual_seed(B)
    lengths = (torch.rand(B, generator=g) ** 8 * 1500).int().tolist()
    sizes = torch.randint(0, T + 1, (B,), generator=g).int().tolist()
    case = attention_case(T, n_heads, n_kv, 64, 16, lengths, BF16, bits, sizes=sizes)
    check_attention(*case)
    check_attention(*case, 70, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 60])
def test_expanded_pages_are_read(T):
    """One page for all places of the pool, one row for all of a page: strides of zero."""
    g = torch.Generator().manual_seed(T)
    page = torch.randn((1, 2, 16, 64), generator=g).half()
    row = torch.randn((5, 1, 1, 64), generator=g).half()
    k, v = to_dev(page).expand(5, 2, 16, 64), to_dev(row).expand(5, 2, 16, 64)
    table, n = to_dev(ints([[4, 0, 2, 1, 3] * 5])), to_dev(ints([300]))
    q = to_dev(torch.randn((1, T, 4 * 64), generator=g).half())
    want = paged.attention_paged(q, k.contiguous(), v.contiguous(), table, n)
    assert torch.equal(paged.attention_paged(q, k, v, table, n), want)
    with pytest.raises(RuntimeError, match="expanded"):
        paged.paged_append(to_dev(torch.zeros((1, T, 8 * 64)).half()), k, v, table, n)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_a_page_that_passes_32_bits(bits):
    """Pages 4 GiB and more into a pool, read and written."""
    n_kv, page, D, dtype = 8, 256, 128, BF16
    element = bits // 8
    n = (9 << 29) // (n_kv * page * D * element) + 2
    pools = [torch.empty((n, n_kv, page, D), dtype=torch.uint8 if bits == 8 else dtype, device=dev)
             for _ in range(2)]
    pools = [p.view(F8) if bits == 8 else p for p in pools]
    small = Cache([300, 100], n_kv, D, page, dtype, bits)
    far = torch.arange(small.k.shape[0]) + n - small.k.shape[0]
    for pool, s in zip(pools, (small.k, small.v)):
        pool[far[0]:] = s.to(dev)
    scales = None
    if bits == 8:
        scales = tuple(torch.full((n, n_kv), 255, dtype=torch.uint8, device=dev) for _ in range(2))
        for s, t in zip(scales, small.scales):
            s[far[0]:] = t.to(dev)
    table = far[small.table.long()].int().to(dev)
    assert int(far[0]) * n_kv * page * D * element >= 1 << 32
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn((2, 3, (16 + 2 * n_kv) * D), generator=g).to(dtype)
    lengths = ints([290, 20])
    got, k, v, _, s = check_append(small, qkv, lengths)
    q = paged.paged_append(to_dev(qkv), *pools, table, to_dev(lengths), scales=scales)
    assert torch.equal(q, got)
    for pool, small_pool in zip(pools, (k, v)):
        assert torch.equal(pool[far[0]:].view(torch.uint8), small_pool.view(torch.uint8))
    a = paged.attention_paged(q, *pools, table, to_dev(lengths), scales=scales)
    b = paged.attention_paged(q, k, v, small.table.to(dev), to_dev(lengths), scales=s)
    assert torch.equal(a, b) and a.isfinite().all()
    ends = to_dev(lengths + 3)
    for x, y in zip(paged.paged_values(*pools, table, ends, scales, dtype),
                    paged.paged_values(k, v, small.table.to(dev), ends, s, dtype)):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_far_apart_and_moving_up(dtype):
    q, cache, lengths, _ = attention_case(20, 4, 2, 128, 16, [600, 64], dtype)
    ramp = torch.linspace(0, 6, cache.page * cache.table.shape[1])
    for b in range(2):
        for m, page in enumerate(cache.table[b].tolist()):
            cache.k[page, :, :, 0] = ramp[m * 16:(m + 1) * 16].to(dtype)
    q[..., 0] = 30.0
    check_attention(q, cache, lengths)
    q[..., 0] = -30.0
    check_attention(q, cache, lengths, None, 100, 10)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [10, 14, 17, 19])
@pytest.mark.parametrize("T,n_heads,n,at", [
    (1, 1, 200, 0), (1, 4, 8192, 0), (1, 4, 8192, 8000), (6, 4, 8192, 70), (12, 4, 8000, 7990),
    (40, 4, 8192, 100)])
def test_small_weights_of_many_rows_add_up(T, n_heads, n, at, nats, dtype, bits):
    """One row outweighs each of thousands by far, and they are what is left of
    the output.  A probability is rounded in its type, fp16's in steps of 2^-24
    at least, where the largest is 2^7 or more: each row's weight is off by half
    a step of its own, or by 2^-25 of 2^7.  An error d of a row's weight moves
    the output by d (v - out)."""
    D = 128
    q, cache, lengths, _ = attention_case(T, n_heads, 1, D, 64, [n], dtype, bits)
    q.zero_()
    q[..., 3] = 4.0
    if bits == 8:
        cache.scales[0][:], cache.scales[1][:] = 127 - 4, 127 - 8
    k, v = cache.k.float(), cache.v.float()
    k[..., 3] = 0.0
    one, unit = (16.0, 256.0) if bits == 8 else (1.0, 1.0)  # codes that stand for 1
    k[cache.table[0, at // 64], 0, at % 64, 3] = nats / 4 * one
    v = unit * (1 + v / v.nan_to_num().abs().max() / 2)
    v[cache.table[0, at // 64], 0, at % 64] = 0.0
    # (3.5 and 4.25, 4.75, 2.5: values of every type here but for 4.75 and 4.25 in 8 bits)
    cache.k, cache.v = k.to(cache.k.dtype), v.to(cache.v.dtype)
    kk, vv = cache.rows(0, 0)[0][:, 0], cache.rows(1, 0)[0][:, 0]
    top = 4 * kk[at, 3].item()
    got = run_attention(q, cache, lengths, scale=1.0).cpu().double()
    info = torch.finfo(dtype)
    for i in range(T):
        s = torch.zeros(n + i + 1, dtype=torch.float64)
        s[at] = top
        w, x = torch.softmax(s, 0), vv[:n + i + 1]
        want = w @ x
        apart = (x - want).abs()
        off = w @ apart * (info.eps / 2 + (top + 2) * 2.0 ** -22 + 2.0 ** -20)
        if dtype == F16:
            off = off + 2.0 ** -32 * apart.sum(0)
        off = off + (want.abs() + off) * info.eps / 2 + info.smallest_normal * info.eps
        for h in range(n_heads):
            assert ((got[0, i, h] - want).abs() <= off).all(), (i, h)


# ---------------------------------------------------------------------------
# together, and around the calls (GPU)
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_as_over_a_contiguous_cache(dtype):
    """A run of tokens over dense caches (:func:`glue.attention_tree`) and over
    the pages of which they are the values."""
    q, cache, lengths, sizes = attention_case(30, 8, 2, 128, 32, [400, 20, 0], dtype, sizes=[30, 11, 2])
    k, v, table, _ = cache.on_gpu()
    dense = paged.paged_values(k, v, table, to_dev(lengths + sizes))
    flat = to_dev(q.reshape(3, 30, -1))
    a = paged.attention_paged(flat, k, v, table, to_dev(lengths), to_dev(sizes))
    b = glue.attention_tree(flat, *dense, to_dev(lengths), None, to_dev(sizes))
    # two ways of summing, each within a rounding of its probabilities and outputs
    assert (a.double() - b.double()).norm() <= 2 * torch.finfo(dtype).eps * b.double().norm()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_layer_step_by_step(dtype, bits):
    """One attention layer on INT4 weights: a prompt in two parts, then tokens
    one by one in a graph, under a window, the pages that it leaves behind taken
    back; each step against the oracle from its own inputs."""
    hidden, n_heads, n_kv, D, page, B = 512, 4, 2, 128, 16, 2
    window, sinks, width = 40, 3, 10
    g = torch.Generator().manual_seed(7)
    w_qkv = ng.quantize(0.05 * torch.randn((hidden, (n_heads + 2 * n_kv) * D), generator=g)).to(dev)
    qw, kw = (t.to(dev) for t in weights(D, dtype))
    rope = glue.rope_tables(width * page, 64)
    kind = dtype if bits == 16 else F8
    k, v, scales = paged.paged_cache(B * width + 1, n_kv, page, D, kind)
    order = torch.randperm(B * width + 1, generator=g)[:B * width].view(B, width).int()
    table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)

    def layer(x, sizes):
        T = x.shape[1]
        qkv = ng.matmul(x.view(-1, hidden), w_qkv).view(B, T, -1).to(dtype)
        q = paged.paged_append(qkv, k, v, table, lengths, sizes, qw, kw, 1e-5, rope, True, scales=scales)
        return qkv, q, paged.attention_paged(q, k, v, table, lengths, sizes, window, sinks, scales=scales)

    def grow(upto):
        for b in range(B):
            for m in range(width):
                at = m * page
                if at < upto[b] and (at < sinks or at + page > int(lengths[b]) - window + 1):
                    table[b, m] = order[b, m]
                else:
                    table[b, m] = -1

    held = [torch.zeros((B, width * page, n_kv, D), dtype=torch.float64) for _ in range(2)]

    def check(qkv, q, out, before, sizes):
        """The rows written this step, and attention over what the cache stands for."""
        T = qkv.shape[1]
        cache = Cache([1] * B, n_kv, D, page, dtype, bits, width=width)
        cache.k, cache.v, cache.table = k.cpu(), v.cpu(), table.cpu()
        cache.scales = None if scales is None else tuple(s.cpu() for s in scales)
        want, bound = oracle_attention(q.cpu().view(B, T, n_heads, D), cache, before, sizes, window, sinks,
                                       D ** -0.5)
        assert ((out.cpu().double().view(B, T, n_heads, D) - want).abs() <= bound).all()
        for b in range(B):
            x = qkv[b].cpu().double().view(T, -1, D)
            at = int(before[b]) + torch.arange(T)
            kk, _ = turned(x[:, n_heads:n_heads + n_kv], kw.cpu(), 1e-5, tuple(t.cpu() for t in rope), at, True)
            for i in range(int(sizes[b])):
                held[0][b, at[i]], held[1][b, at[i]] = kk[i], x[i, n_heads + n_kv:]
            for which in range(2):
                rows, there = cache.rows(which, b)
                n = int(before[b]) + int(sizes[b])
                there = there[:n]
                off = (rows[:n] - held[which][b, :n])[there].norm() / held[which][b, :n][there].norm()
                # 16 bits: a rounding; 8 bits: codes off by 2^-4 of a value at most, 1/4 of it on average squares
                assert off <= (torch.finfo(dtype).eps if bits == 16 else 2.0 ** -4), off

    for T, sizes in ((30, [30, 17]), (33, [20, 33])):
        sizes = ints(sizes)
        x = torch.randn((B, T, hidden), generator=g).half().to(dev)
        grow([int(n) + int(s) for n, s in zip(lengths, sizes)])
        before = lengths.cpu().clone()
        out = layer(x, to_dev(sizes))
        check(*out, before, sizes)
        lengths += to_dev(sizes)

    xs = torch.randn((B, 1, hidden), generator=g).half().to(dev)
    one = torch.ones(B, dtype=torch.int32, device=dev)
    saved = [t.clone() for t in (k, v, *(scales or ()))]
    grow([int(n) + 1 for n in lengths])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = layer(xs, one)
    for t, s in zip((k, v, *(scales or ())), saved):
        t.copy_(s)
    for step in range(25):
        xs.copy_(torch.randn((B, 1, hidden), generator=g).half())
        grow([int(n) + 1 for n in lengths])
        before = lengths.cpu().clone()
        graph.replay()
        torch.cuda.synchronize()
        check(*outs, before, ints([1, 1]))
        eager = paged.attention_paged(outs[1], k, v, table, lengths, one, window, sinks, scales=scales)
        assert torch.equal(outs[2], eager)
        lengths += 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T,length", [(1, 3000), (3, 50), (16, 3000), (70, 500)])
def test_graphs_and_streams(T, length, bits):
    """A captured call follows its inputs; two graphs that share the stream's
    workspace, and calls on another stream, give the eager bits."""
    q, cache, lengths, _ = attention_case(T, 4, 2, 64, 32, [length, length // 3], BF16, bits)
    k, v, table, scales = cache.on_gpu()
    n = to_dev(lengths)
    qd = to_dev(q.reshape(2, T, -1))
    call = lambda w: paged.attention_paged(qd, k, v, table, n, None, w, 2, scales=scales)  # noqa: E731
    eager = {w: call(w) for w in (None, 33)}
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = {}
    for w in (None, 33):
        graphs[w] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[w], stream=side):
            graphs[w].out = call(w)
    for half in (False, True, False):
        n.copy_(to_dev(lengths // 2 if half else lengths))
        want = {w: call(w) for w in (None, 33)}
        for w in (None, 33):
            graphs[w].replay()
            graphs[w].replay()
        torch.cuda.synchronize()
        for w in (None, 33):
            assert torch.equal(graphs[w].out, want[w])
            assert half or torch.equal(want[w], eager[w])
    with torch.cuda.stream(side):
        other = call(None)
    here = call(None)
    torch.cuda.synchronize()
    assert torch.equal(other, eager[None]) and torch.equal(here, eager[None])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_written_pages_are_marked_as_changed(bits):
    cache, qkv, lengths, _ = append_case(2, 2, 1, 128, 16, [3], F16, bits)
    k, v, table, scales = cache.on_gpu()
    written = (k, v) if scales is None else (k, v, *scales)
    before = [t._version for t in written]
    q = paged.paged_append(to_dev(qkv), k, v, table, to_dev(lengths), scales=scales)
    assert [t._version > b for t, b in zip(written, before)] == [True] * len(written)
    before = [t._version for t in written]
    paged.attention_paged(q, k, v, table, to_dev(lengths), scales=scales)
    paged.paged_values(k, v, table, to_dev(lengths), scales)
    assert [t._version for t in written] == before


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_a_batch_of_none(bits):
    k, v, scales = paged.paged_cache(3, 1, 16, 64, F16 if bits == 16 else F8)
    n = torch.zeros(0, dtype=torch.int32, device=dev)
    table = torch.zeros((0, 2), dtype=torch.int32, device=dev)
    for T in (0, 3):
        q = torch.zeros((0, T, 256), dtype=F16, device=dev)
        assert paged.paged_append(q, k, v, table, n, scales=scales).shape == (0, T, 128)
        assert paged.attention_paged(q, k, v, table, n, scales=scales).shape == (0, T, 256)
    assert paged.paged_values(k, v, table, n, scales)[0].shape == (0, 1, 32, 64)
    x = torch.zeros((1, 0, 256), dtype=F16, device=dev)
    n, table = torch.zeros(1, dtype=torch.int32, device=dev), torch.zeros((1, 2), dtype=torch.int32, device=dev)
    assert paged.attention_paged(x, k, v, table, n, scales=scales).shape == (1, 0, 256)


@pytest.mark.gpu
def test_refusals():
    k, v, _ = paged.paged_cache(4, 2, 16, 128)
    k8, v8, s = paged.paged_cache(4, 2, 16, 128, F8)
    x = torch.zeros((1, 2, 8 * 128), dtype=F16, device=dev)
    t, n = torch.zeros((1, 2), dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    cs = glue.rope_tables(8, 128)
    both = [paged.paged_append, paged.attention_paged]
    for call in both:
        with pytest.raises(RuntimeError, match="bfloat16"):
            call(x.to(BF16), k, v, t, n)
        with pytest.raises(RuntimeError, match="need scales|fp16 or bf16"):
            call(x, k8, v8, t, n)
        with pytest.raises(RuntimeError, match="float8_e4m3fn"):
            call(x, k, v, t, n, scales=s)
        with pytest.raises(RuntimeError, match="float8_e4m3fn"):
            call(x, k8.view(torch.uint8), v8, t, n, scales=s)
        with pytest.raises(RuntimeError, match="uint8"):
            call(x, k8, v8, t, n, scales=(s[0].int(), s[1]))
        with pytest.raises(ValueError, match="k_scales must be"):
            call(x, k8, v8, t, n, scales=(s[0][:3], s[1]))
        with pytest.raises(RuntimeError, match="contiguous uint8"):
            call(x, k8, v8, t, n, scales=(s[0].t().contiguous().t(), s[1]))
        with pytest.raises(RuntimeError, match="GPU"):
            call(x, k8.cpu(), v8, t, n, scales=s)
        with pytest.raises(RuntimeError, match="GPU"):
            call(x, k, v, t.cpu(), n)
        with pytest.raises(RuntimeError, match="int32"):
            call(x, k, v, t.long(), n)
        with pytest.raises(ValueError, match="width"):
            call(x, k, v, t[0], n)
        with pytest.raises(ValueError, match="lengths"):
            call(x, k, v, t, torch.zeros(2, dtype=torch.int32, device=dev))
        with pytest.raises(ValueError, match="sizes"):
            call(x, k, v, t, n, torch.zeros(2, dtype=torch.int32, device=dev))
        with pytest.raises(ValueError, match="sequences"):
            call(x, k, v, t.expand(2, 2).contiguous(), n)
        with pytest.raises(ValueError, match="pages must both"):
            call(x, k, v[:, :1], t, n)
        with pytest.raises(ValueError, match="page must have"):
            call(x, k[:, :, :8], v[:, :, :8], t, n)
        with pytest.raises(RuntimeError, match="adjacent"):
            call(x, k.transpose(2, 3).contiguous().transpose(2, 3), v, t, n)
        with pytest.raises(RuntimeError, match="contiguous"):
            call(x.repeat(1, 1, 2)[:, :, :1024], k, v, t, n)
        with pytest.raises(RuntimeError, match="contiguous"):
            call(x[0], k, v, t, n)
        with pytest.raises(RuntimeError, match="no backward"):
            call(x.clone().requires_grad_(), k, v, t, n)
        with pytest.raises(RuntimeError, match="strides"):
            wide = torch.zeros((4, 2, 16, 132), dtype=F16, device=dev)[..., :128]
            call(x, wide, wide.clone(), t, n)
        with pytest.raises(ValueError, match="must be"):
            call(x[:, :, :-8].contiguous(), k, v, t, n)
    with pytest.raises(RuntimeError, match="expanded"):
        paged.paged_append(x, k[:1].expand(4, 2, 16, 128), v, t, n)
    with pytest.raises(ValueError, match="qkv must be"):
        paged.paged_append(x[:, :, :512].contiguous(), k, v, t, n)  # no query heads
    with pytest.raises(ValueError, match="R a multiple of 16"):
        paged.paged_append(x, k, v, t, n, rope=tuple(c[:, :12].contiguous() for c in cs))
    with pytest.raises(ValueError, match="R a multiple of 16"):
        paged.paged_append(x, k, v, t, n, rope=glue.rope_tables(8, 256))
    with pytest.raises(ValueError, match="positions"):
        paged.paged_append(x, k, v, t, n, positions=n)
    with pytest.raises(ValueError, match="q_weight"):
        paged.paged_append(x, k, v, t, n, q_weight=x[0, 0, :64])
    for window in (0, -3):
        with pytest.raises(ValueError, match="window"):
            paged.attention_paged(x, k, v, t, n, window=window)
    with pytest.raises(ValueError, match="sinks"):
        paged.attention_paged(x, k, v, t, n, window=3, sinks=-1)
    with pytest.raises(RuntimeError, match="scale"):
        paged.attention_paged(x, k, v, t, n, scale=math.nan)
    with pytest.raises(RuntimeError, match="pages are"):
        paged.paged_values(k, v, t, n, dtype=BF16)
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        paged.paged_values(k8, v8, t, n, s, torch.float32)
    with pytest.raises(ValueError, match="rows"):
        paged.paged_values(k, v, t, n, rows=-1)
    # pages that are read may be expanded views
    assert paged.attention_paged(x, k[:1].expand(4, 2, 16, 128), v, t, n).shape == x.shape


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,n_heads", [(1, 4), (3, 8), (6, 8), (40, 8), (90, 8)])
def test_scales_of_pages_that_are_not_seen(T, n_heads, dtype, D):
    """What the scale is of a page that nothing sees does not matter: of pages that no
    sequence has (the first among them), of those that a table names for rows to come."""
    for n, window, sinks in ((37, None, 0), (130, None, 0), (300, 60, 20)):
        q, cache, lengths, _ = attention_case(T, n_heads, 2, D, 16, [n, n // 2], dtype, 8,
                                              width=-(-(n + T) // 16) + 3)
        cache.table[cache.table == 0] = -1
        seen = torch.zeros(len(cache.k), dtype=torch.bool)
        for b, first in enumerate(lengths.tolist()):
            for m, page in enumerate(cache.table[b].tolist()):
                in_window = window is None or (m + 1) * 16 > first - window + 1 or m * 16 < sinks
                seen[page] |= page >= 0 and m * 16 < first + T and in_window
        assert not seen[0]
        for s in cache.scales:
            s[~seen] = 255
        check_attention(q, cache, lengths, None, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,n_heads", [(6, 2), (6, 8), (24, 8), (40, 8), (90, 8)])
def test_a_scale_that_is_none(T, n_heads, dtype):
    """The values of a page whose scale is 255 are NaN, for the tokens that see it alone."""
    for n in (14, 125):  # its rows: the last token's own, and some before
        q, cache, lengths, _ = attention_case(T, n_heads, 2, 128, 16, [n, n], dtype, 8)
        first = (n + T - 1) // 16
        want, bound = oracle_attention(q, cache, lengths, None, None, 0, 128 ** -0.5)
        for which in range(2):
            was = cache.scales[which].clone()
            cache.scales[which][cache.table[0, first]] = 255
            got = run_attention(q, cache, lengths).cpu().double()
            cache.scales[which][:] = was
            nan = torch.zeros((2, T), dtype=torch.bool)
            nan[0] = n + torch.arange(T) >= 16 * first
            assert got[nan].isnan().all() and ((got - want).abs() <= bound)[~nan].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("was,size", [(254, 1.0), (254, 2.0 ** 13), (253, 2.0 ** 13), (0, 1.0), (1, 2.0 ** -14)])
def test_append_beside_any_scale(was, size, dtype):
    """Pages of earlier rows whose scale a caller wrote: one of all that a byte holds."""
    size = size if dtype == F16 else size ** 9.5
    cache, qkv, lengths, _ = append_case(5, 2, 2, 64, 16, [13, 8, 1, 0], dtype, 8, size=size,
                                         exponents=(was - 121, was - 120))
    assert cache.scales[0].eq(was).all() and qkv.isfinite().all()
    check_append(cache, qkv, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_beside_rows_without_a_scale(dtype):
    """Earlier rows under a scale of 255 are NaN, and stay so under the new rows' scale,
    which is that of a page of their own."""
    cache, qkv, lengths, _ = append_case(5, 2, 2, 64, 16, [11, 8, 1], dtype, 8)
    for s in cache.scales:
        s[:] = 255
    k, v, table, scales = cache.on_gpu()
    paged.paged_append(to_dev(qkv), k, v, table, to_dev(lengths), scales=scales)
    alone = Cache([5] * 3, 2, 64, 16, dtype, 8)
    k1, v1, t1, s1 = alone.on_gpu()
    paged.paged_append(to_dev(qkv), k1, v1, t1, to_dev(ints([0] * 3)), scales=s1)
    for got, want in zip(paged.paged_values(k, v, table, to_dev(lengths + 5), scales, dtype),
                         paged.paged_values(k1, v1, t1, to_dev(ints([5] * 3)), s1, dtype)):
        for b, n in enumerate(lengths.tolist()):
            assert got[b, :, :n].isnan().all()
            assert torch.equal(got[b, :, n:n + 5], want[b, :, :5])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_of_every_code_and_scale(dtype):
    """All codes under all scales: the value that the two stand for, rounded once (it
    has four bits); a scale of 255 is no power, its values are NaN."""
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 4, 64).expand(256, 1, 4, 64)
    k = torch.zeros((256, 1, 16, 64), dtype=torch.uint8)
    k[:, :, :4] = codes
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1)
    k, s = k.view(F8), scales
    got, same = paged.paged_values(k.to(dev), k.to(dev), torch.arange(256, device=dev, dtype=torch.int32)[None],
                                   to_dev(ints([4096])), (s.to(dev), s.to(dev)), dtype)
    want = torch.ldexp(k.double(), scales[:, :, None, None].double() - 127).to(dtype)
    want[255] = math.nan
    have = got.view(256, 1, 16, 64).cpu()
    assert torch.equal(have.isnan(), want.isnan())
    assert (have == want)[~want.isnan()].all()
    assert torch.equal(same.view(torch.int16), got.view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1])
def test_8_bit_pages_that_autograd_follows_are_refused(which):
    """A followed cache, in reverse and in forward mode: no gradient is cut off, and
    no followed page is written."""
    k, v, scales = paged.paged_cache(3, 1, 16, 64, F8)
    n, t = torch.zeros(1, dtype=torch.int32, device=dev), torch.zeros((1, 2), dtype=torch.int32, device=dev)
    x = torch.zeros((1, 1, 3 * 64), dtype=F16, device=dev)
    calls = [lambda p: paged.paged_append(x, *p, t, n, scales=scales),
             lambda p: paged.attention_paged(x, *p, t, n, scales=scales),
             lambda p: paged.paged_values(*p, t, n, scales)]
    leaf = (k, v)[which].clone().requires_grad_()
    made = torch.ones((3, 1, 16, 64), device=dev, requires_grad=True).to(F8)
    assert made.grad_fn is not None
    for call in calls:
        for followed in (leaf, made):
            pages = [k, v]
            pages[which] = followed
            with pytest.raises(RuntimeError, match="no backward"):
                call(pages)
            with torch.no_grad():  # followed by nothing here
                call(pages)
        with torch.autograd.forward_ad.dual_level():
            pages = [k, v]
            call(pages)
            pages[which] = torch.autograd.forward_ad.make_dual(pages[which], torch.ones_like(pages[which]))
            with pytest.raises(RuntimeError, match="no backward"):
                call(pages)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T,qpk,n_kv,B,D", [
    (1, 1, 1024, 2, 128), (1, 2, 1024, 2, 64), (6, 4, 1024, 2, 128),  # a decode step's, not split
    (1, 1, 128, 9, 64), (6, 4, 128, 9, 64), (9, 2, 128, 2, 128),  # cut in a line, and each by itself
    (40, 1, 256, 2, 64), (70, 1, 256, 2, 128), (40, 1, 128, 2, 128)])  # prompts', and split
def test_pieces_of_many_tiles(T, qpk, n_kv, B, D, bits):
    """More tiles than the 64 whose places are looked up at once in one workgroup: pages
    in any order, their scales, pages that are missing and masks that end in later ones.
    All kv heads read the same pages (a stride of zero) under scales of their own."""
    dtype = F16 if T % 2 else BF16
    lengths = [9000 - 70 * b for b in range(B)]
    q, cache, n, _ = attention_case(T, qpk * n_kv, 1, D, 16, lengths, dtype, bits, seed=T)
    for m in (0, 270, 300, 301, 520):  # tiles 0, 67, 75, 130
        cache.table[:, m] = -1 if m % 2 else cache.k.shape[0]
    g = torch.Generator().manual_seed(T)
    heads = [0, 1, n_kv - 1]  # those that are compared
    few = Cache([1], 1, D, 16, dtype, bits)
    few.B, few.table = B, cache.table
    few.k, few.v = (x.expand(-1, 3, -1, -1) for x in (cache.k, cache.v))
    scales = None
    if bits == 8:
        scales = [torch.randint(119, 124, (len(cache.k), n_kv), generator=g).to(torch.uint8) for _ in range(2)]
        few.scales = [s[:, heads] for s in scales]
        scales = tuple(s.to(dev) for s in scales)
    k, v = (to_dev(x).expand(-1, n_kv, -1, -1) for x in (cache.k, cache.v))
    some = q.view(B, T, n_kv, qpk, D)[:, :, heads].reshape(B, T, 3 * qpk, D)
    flat, table = to_dev(q.reshape(B, T, -1)), to_dev(cache.table)
    for window, sinks in ((None, 0), (3000, 4200)):
        got = paged.attention_paged(flat, k, v, table, to_dev(n), None, window, sinks, scales=scales)
        got = got.cpu().double().view(B, T, n_kv, qpk, D)[:, :, heads].reshape(B, T, 3 * qpk, D)
        want, bound = oracle_attention(some, few, n, None, window, sinks, D ** -0.5)
        assert ((got - want).abs() <= bound).all()


# ---------------------------------------------------------------------------
# the built code
# ---------------------------------------------------------------------------

@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="llvm-objdump not installed")
def test_rows_kernel_waits_match_its_copies(tmp_path):
    """The kernel of a decode step reads a ring in LDS that is its wave's alone, and lets
    all copies but the next ones stay in flight, by count: each of its four waits (k and
    v, with and without a mask) has as many copies behind it as the ring has room for, less
    those that it waits for.  Right only if k and v are as many copies each as counted, and
    if whatever else the loop loads (pages, scales) is waited for in full.  Seen in the built
    code, for every form and type."""
    lib = shutil.copy(build.LIB, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, capture_output=True, check=True)
    objects = [p for p in sorted(tmp_path.iterdir())
               if "gfx950" in p.name and b"rows_kernel" in p.read_bytes()]
    forms = set()
    for at in objects:
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(at)], capture_output=True,
                              text=True, check=True).stdout
        parts = re.split(r"\n[0-9a-f]+ <([^>]+)>:\n", text)
        for name, body in zip(parts[1::2], parts[2::2]):
            form = re.search(r"rows_kernelINS_(4Half|6Bfloat)ELi(\d+)ELi(\d+)ELb(\d)EEE", name)
            if form is None:
                continue
            forms.add(form.groups())
            unit = 16 * int(form[2]) * (1 if form[4] == "1" else 2)  # bytes of 16 rows of k
            copies, ring = unit // 1024, 8192 // (2 * unit)
            seen = []  # copies, other memory operations, waits and barriers, in order
            for line in body.splitlines():
                op = line.split("//")[0].strip()
                if re.match(r"(buffer|global|flat|scratch)_", op):
                    seen.append("copy" if op.endswith("lds") else op.split()[0])
                elif op.startswith("s_waitcnt") and "vmcnt" in op:
                    seen.append(int(re.search(r"vmcnt\((\d+)\)", op)[1]))
                elif op.startswith("s_barrier"):
                    seen.append("barrier")
            last = len(seen) - seen[::-1].index("copy")
            seen = seen[seen.index("copy"):seen.index("barrier", last) + 1]
            # pages' and scales' loads, each with its wait
            rest, i = [], 0
            while i < len(seen):
                loads = 0
                while seen[i + loads] in ("global_load_dword", "global_load_ubyte"):
                    loads += 1
                if loads == 0:
                    rest.append(seen[i])
                else:
                    assert seen[i + loads] == 0, name
                i += loads + 1
            turn = [(2 * ring - 1) * copies] + ["copy"] * copies
            assert rest == ["copy"] * (2 * copies) + turn * 4 + [0, "barrier"], name
    assert len(forms) == 2 * 2 * 2 * 2  # types, heads, tiles of 16 query rows, bits

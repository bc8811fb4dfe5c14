"""The operators of a step of drafted tokens: head norms with rotation, the Q8_0
cache, attention of a tree of drafted tokens over a cache, penalties / biases /
masks on logits. On the GPU each is compared with its formula in 64 bits, the
integers and the cache bytes exactly; refusals are checked without a GPU.

Tolerances (u = 2^-24, half a step of a float relative to the value):
  heads   a head's sum of squares is at most 13 roundings deep (8 per lane, 5 over
          the lanes), its root and quotient add 4: y is off by 13/2 + 4 + 2 < 13 u; the
          angle's rounding to a float (2 u of up to pi) and sincosf (2 ulp) turn by
          4 u, products and sum add 2: 19 u of |y_p| + |y_q|, 24 u are allowed.
  attn    a score is a sum of D products of magnitude at most max|q| |k_e|, each
          rounded (or split into two 11-bit halves: 2^-22 of max|q|) and summed in
          some order: off by at most d = (D + 8) u scale max|q| sum|k|; p then by
          e^(2d) - 1 of itself after the division, the value sum by its chain (under
          256 roundings or tensor-core steps): (4 d + 256 u) max|v|. The 2-norm of
          the difference is also held to 2e-5 of the result's.
  logits  the same float operations as numpy's, bit for bit.
"""
import ctypes as C
import math
import shutil
import subprocess
import sys

import numpy as np
import pytest

import mi_cuda
from conftest import PKG

U = 2.0 ** -24
F = 256  # a fake, 16-byte aligned pointer: the arguments are refused before it is used


# ---------------------------------------------------------------------------
# Without a GPU: refusals, sizes, the tree's mask
# ---------------------------------------------------------------------------

def _refused(rc):
    assert rc == mi_cuda.ERR_ARG and mi_cuda.lib().mi_cuda_last_error() != b""


def _heads_args(**kw):
    a = dict(q=F, qs=896, k=1 << 20, ks=128, wq=None, wk=None, eps=1e-6, d=64, h=14, kv=2, t=3, pos=None, past=0, nd=64,
             base=1e6, qo=1 << 21, ko=1 << 22)
    a.update(kw)
    return [a[x] for x in ("q", "qs", "k", "ks", "wq", "wk", "eps", "d", "h", "kv", "t", "pos", "past", "nd", "base", "qo", "ko")] + [None]


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(d=0), dict(d=257), dict(h=0), dict(kv=0),
                                 dict(t=-1), dict(past=-1), dict(qs=895), dict(ks=127), dict(nd=0), dict(nd=63), dict(nd=66), dict(base=0.0),
                                 dict(base=-1.0), dict(base=math.inf), dict(base=math.nan), dict(eps=-1.0), dict(eps=math.nan),
                                 dict(t=2, past=2**31 - 1), dict(qo=F + 4), dict(qo=F, qs=900), dict(ko=F), dict(qo=1 << 22),
                                 dict(ko=(1 << 20) + 128)])
def test_qk_norm_rope_refusals(bad):
    _refused(mi_cuda.lib().mi_cuda_qk_norm_rope(*_heads_args(**bad)))


def test_kv_q8_0_bytes():
    L = mi_cuda.lib()
    assert L.mi_cuda_kv_q8_0_bytes(2048, 2, 64) == 2048 * 2 * 64 * 34 // 32
    assert L.mi_cuda_kv_q8_0_bytes(1, 1, 32) == 34
    for bad in ((0, 2, 64), (-1, 2, 64), (10, 0, 64), (10, 2, 48), (10, 2, 288), (10, 2, 0), (1 << 31, 1, 32), (10, 1 << 40, 32)):
        assert L.mi_cuda_kv_q8_0_bytes(*bad) == 0


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(ck=None), dict(cv=None), dict(ck=F + 8), dict(cv=F + 2), dict(d=48),
                                 dict(d=288), dict(kv=0), dict(t=-1), dict(ctx=0), dict(past=-1), dict(past=8), dict(past=2**62),
                                 dict(ks=127), dict(vs=1)])
def test_kv_append_refusals(bad):
    a = dict(k=F, ks=128, v=F, vs=128, d=64, kv=2, t=3, ctx=10, past=7, slots=None, ck=F, cv=F)
    a.update(bad)
    _refused(mi_cuda.lib().mi_cuda_kv_append_q8_0(*[a[x] for x in ("k", "ks", "v", "vs", "d", "kv", "t", "ctx", "past", "slots", "ck", "cv")], None))


@pytest.mark.parametrize("bad", [dict(ck=None), dict(cv=F + 1), dict(k=F + 4), dict(v=None), dict(d=40), dict(first=-1), dict(n=-1),
                                 dict(first=11), dict(first=8, n=3), dict(n=2**62)])
def test_kv_read_refusals(bad):
    a = dict(ck=F, cv=F, d=64, kv=2, ctx=10, first=0, n=10, k=F, v=F)
    a.update(bad)
    _refused(mi_cuda.lib().mi_cuda_kv_read_q8_0(*[a[x] for x in ("ck", "cv", "d", "kv", "ctx", "first", "n", "k", "v")], None))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("bad", [dict(q=None), dict(ck=None), dict(cv=None), dict(scratch=None), dict(out=None), dict(ck=F + 8),
                                 dict(cv=F + 4), dict(scratch=F + 8), dict(d=48), dict(d=160), dict(d=256), dict(h=15), dict(h=0), dict(kv=0),
                                 dict(t=-1), dict(t=1025, ctx=4096), dict(past=-1), dict(past=98), dict(past=2**62), dict(ctx=0),
                                 dict(ctx=1 << 31), dict(qs=895)])
def test_attention_tree_refusals(bad, q8):
    a = dict(q=F, qs=896, ck=F, cv=F, d=64, h=14, kv=2, ctx=100, past=97, t=3, mask=None, scale=0.125, scratch=F, out=F)
    a.update(bad)
    fn = mi_cuda.lib().mi_cuda_attention_tree_q8_0 if q8 else mi_cuda.lib().mi_cuda_attention_tree
    _refused(fn(*[a[x] for x in ("q", "qs", "ck", "cv", "d", "h", "kv", "ctx", "past", "t", "mask", "scale", "scratch", "out")], None))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_attention_tree_refuses_a_scale_that_is_not_finite(scale, q8):
    fn = mi_cuda.lib().mi_cuda_attention_tree_q8_0 if q8 else mi_cuda.lib().mi_cuda_attention_tree
    _refused(fn(F, 896, F, F, 64, 14, 2, 100, 97, 3, None, scale, F, F, None))


def test_attention_tree_scratch_bytes():
    fn = mi_cuda.lib().mi_cuda_attention_tree_scratch_bytes
    assert fn(14, 2, 2048, 1, 64) > 0
    for bad in ((14, 3, 100, 1, 64), (14, 2, 100, 1, 48), (14, 2, 3, 4, 64), (14, 2, 1 << 31, 1, 64), (14, 2, 4000, 1025, 64), (0, 2, 10, 1, 64)):
        assert fn(*bad) == 0
    # enough for every shorter context too
    for h, kv, d in ((14, 2, 64), (28, 4, 128), (16, 16, 32), (6, 2, 96)):
        for t in (1, 2, 7, 33, 64, 200):
            n = [fn(h, kv, m, t, d) for m in sorted({t, 300, 1000, 1024, 2047, 4096, 5000, 8191, 20000, 32768, 131072, 1 << 20})]
            assert n == sorted(n)
    # and for fewer tokens
    for h, kv, d in ((14, 2, 64), (28, 4, 128), (16, 16, 32), (6, 2, 96), (96, 1, 64)):
        for m in (1024, 32768):
            n = [fn(h, kv, m, t, d) for t in range(1, 1025)]
            assert n == sorted(n)


@pytest.mark.parametrize("bad", [dict(x=None), dict(out=None), dict(v=0), dict(n=-1), dict(n=65536), dict(stride=99), dict(hist=None),
                                 dict(nh=-1), dict(hs=4), dict(ids=None), dict(bias=None), dict(nb=-1), dict(als=3), dict(repeat=0.0),
                                 dict(repeat=-1.0), dict(repeat=math.nan), dict(repeat=math.inf), dict(freq=math.nan), dict(freq=math.inf),
                                 dict(pres=-math.inf), dict(out=F + 4), dict(out=F, stride=104)])
def test_logits_process_refusals(bad):
    a = dict(x=F, stride=100, v=100, n=2, hist=F, nh=5, hs=5, repeat=1.1, freq=0.0, pres=0.0, ids=F, bias=F, nb=3, allowed=F, als=4,
             out=1 << 20, tok=F)
    a.update(bad)
    _refused(mi_cuda.lib().mi_cuda_logits_process(*[a[x] for x in ("x", "stride", "v", "n", "hist", "nh", "hs", "repeat", "freq", "pres",
                                                                   "ids", "bias", "nb", "allowed", "als", "out", "tok")], None))


def test_python_calls_refuse_other_tensors():
    import torch
    f, i = torch.zeros((3, 2, 64)), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: mi_cuda.qk_norm_rope(f, f, None, None, 1e-6, 0, 64, 1e6),
                 lambda: mi_cuda.kv_append_q8_0(f, f, i, i, 10),
                 lambda: mi_cuda.kv_read_q8_0(i, i, 2, 64, 10, 0, 3),
                 lambda: mi_cuda.kv_q8_0_cache(10, 2, 40),
                 lambda: mi_cuda.attention_tree(f, f, f, 2, 0, 0.1),
                 lambda: mi_cuda.attention_tree_q8_0(f, i, i, 2, 10, 0, 0.1),
                 lambda: mi_cuda.attention_tree_scratch(14, 3, 10, 1, 64),
                 lambda: mi_cuda.logits_process(f[0])):
        with pytest.raises(ValueError):
            call()


def test_tree_mask():
    m = mi_cuda.tree_mask([-1, 0, 0, 2, -1])
    assert m.shape == (5, 1) and m.dtype == np.int32
    assert m[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1101, 0b10000]
    chain = mi_cuda.tree_mask(list(range(-1, 39)))
    assert chain.shape == (40, 2) and chain.view(np.uint32)[39].tolist() == [0xffffffff, 0xff]
    assert mi_cuda.tree_mask([]).shape == (0, 0)
    with pytest.raises(ValueError):
        mi_cuda.tree_mask([0])


# ---------------------------------------------------------------------------
# Formulas in 64 bits
# ---------------------------------------------------------------------------

def heads_f64(torch, x, w, eps, pos, n_dims, base):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    half = n_dims // 2
    a = pos.double()[:, None, None] * torch.pow(torch.tensor(float(base), dtype=torch.float64, device=x.device),
                                                -2.0 * torch.arange(half, device=x.device).double() / n_dims)
    lo, hi = y[..., :half], y[..., half:n_dims]
    size = torch.cat([lo.abs() + hi.abs()] * 2 + [y[..., n_dims:].abs()], -1)
    return torch.cat([lo * a.cos() - hi * a.sin(), lo * a.sin() + hi * a.cos(), y[..., n_dims:]], -1), size


def quantise_f64(torch, x):
    """[T, HKV, D] -> (q int8 [HKV, T, D], d fp16 [HKV, T, D / 32])."""
    b = x.double().transpose(0, 1).unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    d = (top.float() * torch.tensor(1 / 127, dtype=torch.float32, device=x.device)).clamp(max=65504.0).half()  # the header's product
    f = d.double()
    q = torch.where(f > 0, torch.round(b / torch.where(f > 0, f, 1.0)).clamp(-127, 127), 0.0)
    bad = ~torch.isfinite(b).all(-1, keepdim=True)
    q = torch.where(bad, 0.0, q)
    return q.to(torch.int8).flatten(-2), torch.where(bad, torch.tensor(math.nan, dtype=torch.float16, device=x.device), d).squeeze(-1)


def planes(buf, kv, n_ctx, d):
    import torch
    n = kv * n_ctx * d
    return buf[:n].view(torch.int8).view(kv, n_ctx, d), buf[n:].view(torch.float16).view(kv, n_ctx, d // 32)


def attn_f64(torch, q, k, v, seen, scale):
    """q [T, H, D], k / v [n, HKV, D], seen bool [T, n]: (out, the bound of the docstring)."""
    T, H, D = q.shape
    rep = H // k.shape[1]
    kk, vv = (x.double().repeat_interleave(rep, 1).transpose(0, 1) for x in (k, v))  # [H, n, D]
    # what nothing attends to does not count, whatever it holds
    used = seen.any(0)
    kk, vv = (torch.where(used[None, :, None], x, 0.0) for x in (kk, vv))
    s = torch.where(seen, q.double().transpose(0, 1) @ kk.transpose(1, 2) * scale, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    l = p.sum(-1, keepdim=True)
    o = (p @ vv) / torch.where(l > 0, l, 1.0)
    delta = (D + 8) * U * abs(scale) * float(q.abs().max()) * float(kk.abs().sum(-1).max())
    return o.transpose(0, 1), (4 * delta + 256 * U) * float(vv.abs().max())


def check_attn(torch, got, q, k, v, seen, scale):
    want, tol = attn_f64(torch, q, k, v, seen, scale)
    diff = got.double() - want
    assert torch.isfinite(got).all()
    assert float(diff.abs().max()) <= tol
    assert float(diff.norm()) <= 2e-5 * float(want.norm())
    empty = ~seen.any(1)
    assert not got[empty].any()


def seen_of(torch, mask, T, past, dev="cuda"):
    seen = torch.ones((T, past + T), dtype=torch.bool, device=dev)
    if mask is None:
        seen[:, past:] = torch.ones((T, T), device=dev).tril() > 0
    else:
        j = np.arange(T)
        seen[:, past:] = torch.from_numpy((mask.view(np.uint32)[:, j // 32] >> (j % 32).astype(np.uint32)) & 1 > 0).to(dev)
    return seen


def random_tree(rng, T):
    return [-1 if i == 0 or rng.random() < 0.1 else int(rng.integers(max(0, i - 6), i)) for i in range(T)]


def logits_f32(x, hist, repeat, freq, pres, ids, bias, allowed):
    """The formula in numpy's float32, one row; returns (processed, token)."""
    f = np.float32
    x = x.copy()
    V = x.size
    h = hist[(hist >= 0) & (hist < V)]
    t, c = np.unique(h, return_counts=True)
    l = x[t]
    with np.errstate(over="ignore", invalid="ignore"):
        x[t] = np.where(l > 0, l / f(repeat), l * f(repeat)) - (c.astype(f) * f(freq) + f(pres))
        if ids is not None:
            b = np.zeros(V, dtype=f)
            for i, w in zip(ids, bias):
                if 0 <= i < V:
                    b[i] = b[i] + w
            x = x + b
    if allowed is not None:
        bits = np.unpackbits(allowed.view(np.uint8), bitorder="little")[:V]
        x[bits == 0] = -np.inf
    y = np.where(np.isnan(x), -np.inf, x)
    return x, int(np.argmax(y)) if y.max() > -np.inf else -1


# ---------------------------------------------------------------------------
# On the GPU
# ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def torch(torch_cuda):
    return torch_cuda


def check_heads(torch, got, x, w, eps, pos, n_dims, base):
    want, size = heads_f64(torch, x, w, eps, pos, n_dims, base)
    assert ((got.double() - want).abs() <= 24 * U * size + 1e-37).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,HKV,D,n_dims,norm,stacked", [
    (1, 14, 2, 64, 64, True, True), (1, 14, 2, 64, 64, False, False), (7, 28, 4, 128, 128, True, True), (5, 3, 1, 256, 256, True, False),
    (3, 4, 2, 64, 32, True, True), (9, 5, 3, 40, 40, True, True), (4, 2, 1, 7, 6, True, True), (2, 1, 1, 2, 2, True, False),
    (6, 3, 3, 100, 50, False, True), (300, 4, 2, 64, 64, True, True), (33, 6, 2, 96, 96, True, False), (3, 2, 2, 1 + 128, 128, True, False),
    (2, 9, 5, 256, 2, True, True), (17, 40, 8, 128, 64, False, True)])
def test_qk_norm_rope(torch, T, H, HKV, D, n_dims, norm, stacked):
    g = torch.Generator(device="cuda").manual_seed(T * H + D)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    if stacked:  # parts of stacked q|k|v rows
        qkv = rnd(T, (H + 2 * HKV) * D) * 3
        q, k = qkv[:, : H * D].unflatten(1, (H, D)), qkv[:, H * D : (H + HKV) * D].unflatten(1, (HKV, D))
    else:
        q, k = rnd(T, H, D) * 3, rnd(T, HKV, D)
    wq, wk = (rnd(D), rnd(D)) if norm else (None, None)
    pos = torch.randint(0, 200000, (T,), generator=g, device="cuda", dtype=torch.int32)
    for p, past in ((pos, 0), (None, 32100)):
        qo, ko = mi_cuda.qk_norm_rope(q, k, wq, wk, 1e-6, past, n_dims, 1e6, pos=p)
        at = p if p is not None else past + torch.arange(T, device="cuda")
        check_heads(torch, qo, q, wq, 1e-6, at, n_dims, 1e6)
        check_heads(torch, ko, k, wk, 1e-6, at, n_dims, 1e6)
    # one of the two norms alone, and in place
    if norm and not stacked:
        want, _ = mi_cuda.qk_norm_rope(q, k, wq, None, 1e-5, 3, n_dims, 1e4)
        a, b = q.clone(), k.clone()
        qo, ko = mi_cuda.qk_norm_rope(a, b, wq, None, 1e-5, 3, n_dims, 1e4, q_out=a, k_out=b)
        assert qo is a and torch.equal(a, want)
        check_heads(torch, b, k, None, 1e-5, 3 + torch.arange(T, device="cuda"), n_dims, 1e4)


@pytest.mark.gpu
def test_qk_norm_rope_far_positions_and_unaligned_rows(torch):
    g = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn(6 * 200 + 3, generator=g, device="cuda")
    q = base[1:1 + 6 * 200].view(6, 200)[:, :192].unflatten(1, (3, 64))  # 4-byte aligned rows
    k = base[3:3 + 6 * 200].view(6, 200)[:, 7:135].unflatten(1, (2, 64))
    pos = torch.tensor([0, 1, 2**20 + 1, 2**30 + 7, 2**31 - 1, -5], dtype=torch.int32, device="cuda")
    qo, ko = mi_cuda.qk_norm_rope(q, k, None, None, 0.0, 0, 64, 1e4, pos=pos)
    check_heads(torch, qo, q, None, 0.0, pos, 64, 1e4)
    check_heads(torch, ko, k, None, 0.0, pos, 64, 1e4)
    z = torch.zeros((2, 1, 64), device="cuda")  # a zero head stays zero
    assert not mi_cuda.qk_norm_rope(z, z, torch.ones(64, device="cuda"), None, 1e-6, 0, 64, 1e4)[0].any()


def put(torch, cache, kv, n_ctx, d, rows, at):
    """The expected cache bytes after rows [n, HKV, D] went to slots `at` (a list)."""
    q, s = planes(cache.clone(), kv, n_ctx, d)
    q, s = q.clone(), s.clone()
    nq, ns = quantise_f64(torch, rows)
    for t, a in enumerate(at):
        if a >= 0:
            q[:, a], s[:, a] = nq[:, t], ns[:, t]
    return q, s


@pytest.mark.gpu
@pytest.mark.parametrize("T,HKV,D,n_ctx,past", [(1, 2, 64, 9, 8), (13, 2, 64, 40, 20), (5, 3, 96, 5, 0), (70, 1, 32, 129, 59),
                                                (9, 4, 128, 77, 0), (3, 1, 256, 4, 1), (257, 4, 128, 300, 11), (1000, 2, 64, 1000, 0)])
@pytest.mark.parametrize("aligned", [True, False])
def test_kv_append_and_read(torch, T, HKV, D, n_ctx, past, aligned):
    g = torch.Generator(device="cuda").manual_seed(T + D)
    off, row = (0, HKV * D) if aligned else (1, HKV * D + 5)
    k, v = (torch.randn(T * row + 8, generator=g, device="cuda")[off:off + T * row].view(T, row)[:, : HKV * D].unflatten(1, (HKV, D))
            for _ in range(2))
    caches = [torch.randint(0, 60, (mi_cuda.lib().mi_cuda_kv_q8_0_bytes(n_ctx, HKV, D),), generator=g, device="cuda", dtype=torch.uint8)
              for _ in range(2)]
    want = [put(torch, c, HKV, n_ctx, D, x, range(past, past + T)) for c, x in zip(caches, (k, v))]
    mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx, past)
    for c, (q, s) in zip(caches, want):  # other rows as they were
        gq, gs = planes(c, HKV, n_ctx, D)
        assert torch.equal(gq, q) and torch.equal(gs.view(torch.int16), s.view(torch.int16))
    for first, n in ((0, n_ctx), (past, T), (n_ctx - 1, 1), (2, 0)):
        back = mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, first, n)
        for x, (q, s) in zip(back, want):
            f = (q.float().unflatten(-1, (-1, 32)) * s.float()[..., None]).flatten(-2).transpose(0, 1)[first:first + n]
            assert x.shape == (n, HKV, D) and torch.equal(x, f)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 8, 9, 40, 600])
def test_kv_append_slots(torch, T):
    """Skipped tokens, slots out of order, named twice (the later token is kept) and outside the cache."""
    rng = np.random.default_rng(T)
    HKV, D, n_ctx = 2, 64, 700
    slots = rng.integers(-1, min(n_ctx, max(2, T // 2)), T).astype(np.int32)
    k, v = (torch.from_numpy(rng.standard_normal((T, HKV, D), dtype=np.float32)).cuda() for _ in range(2))
    code = C.c_int32(-1)
    for outside in (False, True):
        if outside:
            slots[T // 2] = n_ctx + 3
        caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
        want = [put(torch, c, HKV, n_ctx, D, x, [s if s < n_ctx else -1 for s in slots]) for c, x in zip(caches, (k, v))]
        mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx, slots=torch.from_numpy(slots).cuda())
        for c, (q, s) in zip(caches, want):
            gq, gs = planes(c, HKV, n_ctx, D)
            assert torch.equal(gq, q) and torch.equal(gs.view(torch.int16), s.view(torch.int16))
        assert mi_cuda.lib().mi_cuda_device_error(0, C.byref(code)) == 0
        assert code.value == (mi_cuda.ERR_ARG if outside else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("HKV,D", [(2, 64), (16, 128), (3, 96)])
@pytest.mark.parametrize("T,span", [(2049, 5000), (3001, 40), (9000, 4000), (5000, 5000)])
def test_kv_append_many_slots(torch, HKV, D, T, span):
    """A prompt's rows into slots: some skipped, some outside the cache, many named again and again."""
    rng = np.random.default_rng(T)
    n_ctx = 5000
    slots = rng.integers(-1, span, T).astype(np.int32) if T != span else rng.permutation(T).astype(np.int32)
    outside = T == 9000
    if outside:
        slots[[5, 8000]] = n_ctx, 2**31 - 1
    k, v = (torch.randn((T, HKV, D), device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(T)
    caches = [torch.randint(0, 256, (mi_cuda.lib().mi_cuda_kv_q8_0_bytes(n_ctx, HKV, D),), generator=g, device="cuda", dtype=torch.uint8)
              for _ in range(2)]
    last = {int(s): t for t, s in enumerate(slots) if 0 <= s < n_ctx}
    at, src = (torch.tensor(x, device="cuda") for x in (list(last), list(last.values())))
    want = []
    for c, x in zip(caches, (k, v)):
        q, s = (p.clone() for p in planes(c, HKV, n_ctx, D))
        q[:, at], s[:, at] = (p[:, src] for p in quantise_f64(torch, x))
        want.append((q, s))
    mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx, slots=torch.from_numpy(slots).cuda())
    for c, (q, s) in zip(caches, want):
        gq, gs = planes(c, HKV, n_ctx, D)
        assert torch.equal(gq, q) and torch.equal(gs.view(torch.int16), s.view(torch.int16))
    code = C.c_int32(-1)
    assert mi_cuda.lib().mi_cuda_device_error(0, C.byref(code)) == 0
    assert code.value == (mi_cuda.ERR_ARG if outside else 0)


@pytest.mark.gpu
def test_kv_append_many_slots_captured(torch):
    """Recorded once and replayed with other rows and other slots, over rows that the replay before wrote."""
    T, HKV, D, n_ctx = 1500, 2, 64, 900
    k, v = (torch.empty((T, HKV, D), device="cuda") for _ in range(2))
    slots = torch.zeros(T, device="cuda", dtype=torch.int32)
    caches, alone = ([mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)] for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx, slots=slots)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        k.normal_(generator=g)
        v.normal_(generator=g)
        slots.random_(-1, n_ctx, generator=g)
        graph.replay()
        for t, s in enumerate(slots.tolist()):  # one after another
            if s >= 0:
                mi_cuda.kv_append_q8_0(k[t:t + 1], v[t:t + 1], *alone, n_ctx, s)
        assert all(torch.equal(a, b) for a, b in zip(caches, alone))


@pytest.mark.gpu
def test_kv_append_time_grows_with_the_slots(torch):
    """Four times the tokens take some four times as long at most (not sixteen)."""
    took = []
    for T in (30000, 120000):
        k, v = (torch.randn((T, 2, 64), device="cuda") for _ in range(2))
        caches = [mi_cuda.kv_q8_0_cache(T, 2, 64) for _ in range(2)]
        slots = torch.randperm(T, device="cuda").to(torch.int32)
        best = math.inf
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            mi_cuda.kv_append_q8_0(k, v, *caches, T, slots=slots)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        took.append(best)
    assert took[1] <= 8 * took[0], took


@pytest.mark.gpu
def test_kv_append_values(torch):
    """Zeros, subnormal scales, borders between two integers, saturated scales, infinities and NaN."""
    rows = torch.zeros((12, 1, 32), device="cuda")
    rows[1] = torch.linspace(-1, 1, 32, device="cuda")
    rows[2, 0, 0], rows[2, 0, 1:] = 127.0, torch.arange(31, device="cuda") - 15.5  # d = 1: ties to even
    rows[3] = 1e-9 * torch.arange(32, device="cuda")            # d below the smallest fp16: 0
    rows[4] = 3e-6 * torch.linspace(-1, 1, 32, device="cuda")   # a subnormal d
    rows[5] = 3e7 * torch.linspace(-1, 1, 32, device="cuda")    # past 127 * 65504: clamped
    rows[6, 0, 3] = math.inf
    rows[7, 0, 31] = math.nan
    rows[8, 0, 5] = -math.inf
    rows[9] = 3.4e38
    rows[10] = -1e-45
    rows[11, 0, 0], rows[11, 0, 1:] = 127 * 0.1, (torch.arange(31, device="cuda") + 0.5) * float(torch.tensor(0.1).half())
    cache = [mi_cuda.kv_q8_0_cache(12, 1, 32) for _ in range(2)]
    mi_cuda.kv_append_q8_0(rows, rows, *cache, 12)
    q, d = quantise_f64(torch, rows)
    for c in cache:
        gq, gd = planes(c, 1, 12, 32)
        assert torch.equal(gq, q)
        assert torch.equal(torch.isnan(gd), torch.isnan(d)) and torch.equal(gd.nan_to_num(7.0), d.nan_to_num(7.0))
    k, _ = mi_cuda.kv_read_q8_0(*cache, 1, 32, 12, 0, 12)
    assert torch.isnan(k[6:9]).all() and torch.isfinite(k[:6]).all() and torch.isfinite(k[9:]).all()


def attn_inputs(torch, T, H, HKV, D, past, seed, q8, spare=3):
    """(q, the caches, the rows that they stand for [n_past + T, HKV, D], n_ctx)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_ctx = past + T + spare
    q = torch.randn((T, H, D), generator=g, device="cuda") * 1.5
    k, v = (torch.randn((n_ctx, HKV, D), generator=g, device="cuda") + 2 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    if not q8:
        return q, (k, v), (k[: past + T], v[: past + T]), n_ctx
    caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
    mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx)
    return q, caches, mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, 0, past + T), n_ctx


def tree(torch, q8, q, caches, HKV, n_ctx, past, scale, mask=None, scratch=None):
    m = torch.from_numpy(mask).cuda() if mask is not None else None
    if q8:
        return mi_cuda.attention_tree_q8_0(q, *caches, HKV, n_ctx, past, scale, mask=m, scratch=scratch)
    return mi_cuda.attention_tree(q, *caches, HKV, past, scale, mask=m, scratch=scratch)


SHAPES = [(14, 2, 64), (28, 4, 128), (16, 16, 32), (6, 2, 96), (4, 2, 64), (17, 1, 64), (1, 1, 128), (40, 1, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,HKV,D", SHAPES)
@pytest.mark.parametrize("T,past", [(1, 0), (1, 1), (1, 30), (1, 31), (1, 500), (1, 3001), (2, 0), (3, 127), (5, 1000), (8, 129), (13, 254),
                                    (33, 60), (64, 0), (64, 449), (65, 2000), (200, 77)])
def test_attention_tree(torch, q8, H, HKV, D, T, past):
    q, caches, rows, n_ctx = attn_inputs(torch, T, H, HKV, D, past, T + past + D, q8)
    scale = 1 / math.sqrt(D)
    mask = mi_cuda.tree_mask(random_tree(np.random.default_rng(T + past), T))
    for m in (None, mask):
        check_attn(torch, tree(torch, q8, q, caches, HKV, n_ctx, past, scale, m), q, *rows, seen_of(torch, m, T, past), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,HKV,D,T,past", [(14, 2, 64, 1, 32767), (14, 2, 64, 64, 20001), (28, 4, 128, 11, 16389), (16, 16, 32, 1, 9000),
                                            (6, 2, 96, 300, 5000), (14, 2, 64, 1024, 1500), (14, 2, 64, 7, 131071),
                                            (28, 4, 128, 1, 40000), (14, 2, 64, 2, 16000), (14, 2, 64, 2, 16383), (28, 4, 128, 4, 4092),
                                            (28, 4, 128, 4, 4093), (16, 16, 32, 8, 131071), (4, 2, 96, 4, 60001)])
def test_attention_tree_long(torch, q8, H, HKV, D, T, past):
    q, caches, rows, n_ctx = attn_inputs(torch, T, H, HKV, D, past, 3, q8)
    mask = mi_cuda.tree_mask(random_tree(np.random.default_rng(T), T))
    check_attn(torch, tree(torch, q8, q, caches, HKV, n_ctx, past, 0.11, mask), q, *rows, seen_of(torch, mask, T, past), 0.11)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("T,past", [(4, 0), (40, 0), (70, 5)])
def test_attention_tree_empty_rows_and_poisoned_masked_rows(torch, q8, T, past):
    """Any mask: tokens that attend to nothing, and NaN / infinities in rows that none (or only
    others) attend to and behind the last row."""
    rng = np.random.default_rng(T)
    H, HKV, D = 14, 2, 64
    q, caches, rows, n_ctx = attn_inputs(torch, T, H, HKV, D, past, T, False, spare=40)
    words = (T + 31) // 32
    bits = rng.random((T, words * 32)) < 0.3
    bits[:, T // 2] = False           # no one's row
    bits[T - 1] = False               # attends to nothing drafted
    mask = (bits.astype(np.uint32).reshape(T, words, 32) << np.arange(32, dtype=np.uint32)).sum(-1, dtype=np.uint32).view(np.int32)
    k, v = (x.clone() for x in caches)
    k[past + T // 2], v[past + T // 2] = math.nan, math.inf
    k[past + T:], v[past + T:] = math.inf, math.nan
    rows = (k[: past + T], v[: past + T])
    if q8:
        caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
        mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx)
        rows = mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, 0, past + T)
    else:
        caches = (k, v)
    seen = seen_of(torch, mask, T, past)
    check_attn(torch, tree(torch, q8, q, caches, HKV, n_ctx, past, 0.125, mask), q, *rows, seen, 0.125)
    # a row that some attend to, with a NaN: those tokens get NaN, the others their result
    k2 = rows[0].clone()
    k2[past] = math.nan
    if q8:
        mi_cuda.kv_append_q8_0(k2[past:past + 1], rows[1][past:past + 1], *caches, n_ctx, past)
    else:
        caches[0][past] = math.nan
    got = tree(torch, q8, q, caches, HKV, n_ctx, past, 0.125, mask)
    hit = seen[:, past]
    assert torch.isnan(got[hit]).all()
    want, tol = attn_f64(torch, q[~hit], *rows, seen[~hit], 0.125)
    assert float((got[~hit].double() - want).abs().max()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
def test_attention_tree_sizes_of_values(torch, q8):
    """Large, tiny, zero and far apart queries and keys; a scale of either sign and zero."""
    H, HKV, D, T, past = 14, 2, 64, 9, 333
    for qs, ks, scale in ((1e4, 1e-5, 0.125), (1e-6, 3e5, 0.1), (0.0, 1.0, 0.125), (8.0, 1.0, 0.125), (1.0, 1.0, -0.125), (1.0, 1.0, 0.0),
                          (1e-20, 1e3, 1e15)):
        q, caches, rows, n_ctx = attn_inputs(torch, T, H, HKV, D, past, 8, False)
        q = q * qs
        k, v = caches[0] * ks, caches[1]
        rows = (k[: past + T], v[: past + T])
        if q8:
            caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
            mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx)
            rows = mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, 0, past + T)
        else:
            caches = (k, v)
        got = tree(torch, q8, q, caches, HKV, n_ctx, past, scale)
        want, tol = attn_f64(torch, q, *rows, seen_of(torch, None, T, past), scale)
        assert float((got.double() - want).abs().max()) <= tol, (qs, ks, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,HKV,D", [(14, 2, 64), (4, 2, 128)])
def test_attention_tree_rows_of_different_size(torch, q8, H, HKV, D):
    """Rows whose magnitudes are far apart, and huge rows that only some tokens attend to: the
    others' results keep the precision of the rows that they do attend to."""
    T, past = 24, 150
    q, caches, _, n_ctx = attn_inputs(torch, T, H, HKV, D, past, 6, False)
    g = torch.Generator(device="cuda").manual_seed(9)
    size = lambda lo, hi: torch.exp(torch.empty((n_ctx, 1, 1), device="cuda").uniform_(math.log(lo), math.log(hi), generator=g))  # noqa: E731
    mask = mi_cuda.tree_mask(random_tree(np.random.default_rng(3), T))
    seen = seen_of(torch, mask, T, past)
    for ks, vs, huge in ((size(1e-5, 1), size(1e-4, 1e2), 1.0), (size(1, 1), size(1e-3, 1), 5e6), (size(1e-6, 1), size(1, 1), 8e6)):
        k, v = caches[0] * ks, caches[1] * vs
        for c in (k, v):  # drafted tokens 0, 7 and 19: huge
            c[[past, past + 7, past + 19]] *= huge
        if q8:
            both = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
            mi_cuda.kv_append_q8_0(k, v, *both, n_ctx)
            rows = mi_cuda.kv_read_q8_0(*both, HKV, D, n_ctx, 0, past + T)
        else:
            both, rows = (k, v), (k[: past + T], v[: past + T])
        got = tree(torch, q8, q, both, HKV, n_ctx, past, 0.1, mask)
        hit = seen[:, [past, past + 7, past + 19]].any(1)
        assert 0 < int(hit.sum()) < T
        for part in (hit, ~hit):
            want, tol = attn_f64(torch, q[part], *rows, seen[part], 0.1)
            assert float((got[part].double() - want).abs().max()) <= tol
            if part is not hit or huge == 1.0:
                assert float((got[part].double() - want).norm()) <= 2e-5 * float(want.norm())


@pytest.mark.gpu
def test_attention_tree_strided_queries_and_offsets_past_32_bits(torch):
    """Queries that are parts of stacked rows; a cache whose last head lies past 2^31 bytes."""
    HKV, D, n_ctx, T, past = 16, 128, 1200000, 3, 700
    assert (HKV - 1) * n_ctx * D > 2**31
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn((T, (32 + 2 * HKV) * D), generator=g, device="cuda")
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([32 * D, HKV * D, HKV * D], 1))
    caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
    old = torch.randn((2, past, HKV, D), generator=g, device="cuda")
    mi_cuda.kv_append_q8_0(old[0], old[1], *caches, n_ctx)
    mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx, past)
    rows = mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, 0, past + T)
    want = [torch.cat([o, x]) for o, x in zip(old, (k, v))]
    assert all(float((a - b).abs().max()) < 0.05 for a, b in zip(rows, want))
    check_attn(torch, mi_cuda.attention_tree_q8_0(q, *caches, HKV, n_ctx, past, 0.09), q, *rows, seen_of(torch, None, T, past), 0.09)


@pytest.mark.gpu
def test_attention_tree_same_from_call_to_call_and_over_batches(torch):
    """The same bits on every call, with a scratch that holds another call's values."""
    H, HKV, D, T, past = 14, 2, 64, 12, 3000
    q, caches, _, n_ctx = attn_inputs(torch, T, H, HKV, D, past, 4, True)
    scratch = mi_cuda.attention_tree_scratch(H, HKV, 2 * n_ctx, T, D)
    first = tree(torch, True, q, caches, HKV, n_ctx, past, 0.125, scratch=scratch)
    scratch.fill_(255)
    assert torch.equal(first, tree(torch, True, q, caches, HKV, n_ctx, past, 0.125, scratch=scratch))
    assert torch.equal(first, tree(torch, True, q, caches, HKV, n_ctx, past, 0.125))


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,HKV,D,T,past,bad", [(14, 2, 64, 2, 70, math.inf), (28, 4, 128, 1, 200, -math.inf), (6, 2, 96, 9, 30, math.nan),
                                                (14, 2, 64, 40, 300, math.inf), (17, 1, 32, 20, 129, math.nan)])
def test_attention_tree_values_that_are_not_finite(torch, q8, H, HKV, D, T, past, bad):
    """An infinity or a NaN in a value row: NaN for the tokens that attend to it, nothing for the others."""
    q, caches, _, n_ctx = attn_inputs(torch, T, H, HKV, D, past, T, False)
    k, v = (x.clone() for x in caches)
    v[past + T - 1, HKV - 1, 1] = bad  # (the last token's own row)
    if q8:
        caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
        mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx)
        rows = mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, 0, past + T)
    else:
        caches, rows = (k, v), (k[: past + T], v[: past + T])
    got = tree(torch, q8, q, caches, HKV, n_ctx, past, 0.125).unflatten(1, (HKV, -1))
    assert torch.isnan(got[-1, -1]).any(-1).all()
    clean = torch.where(torch.isfinite(rows[1]), rows[1], 0.0)
    want, tol = attn_f64(torch, q, rows[0], clean, seen_of(torch, None, T, past), 0.125)
    want = want.unflatten(1, (HKV, -1))
    assert T == 1 or float((got[:-1].double() - want[:-1]).abs().max()) <= tol
    assert HKV == 1 or float((got[:, :-1].double() - want[:, :-1]).abs().max()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("H,HKV,D,T,past", [(14, 2, 64, 40, 3000), (28, 4, 128, 20, 900), (40, 1, 32, 9, 2000)])
def test_attention_tree_two_at_once(torch, H, HKV, D, T, past):
    """Calls on two streams, each with its own scratch, and a replayed graph beside an eager call."""
    sets = [attn_inputs(torch, T, H, HKV, D, past, seed, True) for seed in (1, 2)]
    scratch = [mi_cuda.attention_tree_scratch(H, HKV, past + T, T, D) for _ in sets]
    call = lambda i: tree(torch, True, sets[i][0], sets[i][1], HKV, sets[i][3], past, 0.125, scratch=scratch[i])  # noqa: E731
    want = [call(0).clone(), call(1).clone()]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        out = call(0)
    torch.cuda.synchronize()
    for _ in range(5):
        graph.replay()
        with torch.cuda.stream(streams[1]):
            other = call(1)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(other, want[1])


def attn_componentwise(torch, got, q, k, v, seen, scale, rows=None):
    """Holds got [T, H, D] (or its tokens `rows`) to a bound of its own per value, from the rows that the
    token attends to alone, so that nothing a masked row holds may cost precision. Weight j is off by
    d_j + eps of itself and the sum of the weights by what that comes to: d_j is the score's error,
    (D + 8) u scale max|q| sum|k_j| as in check_attn plus 4 u |s_j| for its scaling and the difference to
    the maximum; eps 2 * 2^-22 for exp2 in numerator and sum, 2^-20 for operands held as halves (11 + 11
    bits) and 256 u for the sums. A weight's lower half stops 2^-37 below the largest weight times value:
    n of those are added. Rows with a NaN may be passed where no checked token attends to them."""
    T, H, D = q.shape
    rep, n = H // k.shape[1], k.shape[0]
    for i in range(T) if rows is None else rows:
        at = torch.nonzero(seen[i])[:, 0]
        kk, vv = (x[at].double().repeat_interleave(rep, 1).transpose(0, 1) for x in (k, v))  # [H, m, D]
        s = (kk @ q[i].double()[:, :, None]).squeeze(-1) * scale  # [H, m]
        p = torch.softmax(s, -1)
        d = (D + 8) * U * abs(scale) * q[i].double().abs().amax(-1)[:, None] * kk.abs().sum(-1) + 4 * U * s.abs()
        eps = 2.0**-21 + 2.0**-20 + 256 * U + (p * d).sum(-1, keepdim=True)
        want = (p[:, None] @ vv).squeeze(1)
        tol = ((p * (d + eps))[:, None] @ vv.abs()).squeeze(1) + n * 2.0**-37 * (p * vv.abs().amax(-1)).amax(-1)[:, None]
        diff = (got[i].double() - want).abs()
        assert (diff <= tol).all(), (i, float((diff / tol).max()), float(diff.norm() / want.norm()))


def set_row(torch, caches, kv, n_ctx, d, at, what):
    """Row `at` of both Q8_0 caches: quants 127 with a scale of NaN, of 65504, or of 1000 times the row's own."""
    for c in caches:
        q, s = planes(c, kv, n_ctx, d)
        q[:, at] = 127
        s[:, at] = {"nan": math.nan, "max": 65504.0}[what] if what != "1000" else s[:, at] * 1000


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["nan", "max", "1000"])
@pytest.mark.parametrize("H,HKV,D,T,past", [(14, 2, 64, 1, 20), (14, 2, 64, 2, 18), (14, 2, 64, 4, 30), (28, 4, 128, 2, 40), (28, 4, 128, 1, 7),
                                            (6, 2, 96, 2, 300), (6, 2, 96, 5, 20), (16, 16, 32, 4, 20), (16, 16, 32, 20, 11), (14, 2, 64, 2, 3000),
                                            (28, 4, 128, 24, 150)])
def test_attention_tree_q8_0_beside_masked_rows(torch, H, HKV, D, T, past, what):
    """A masked row of a large scale (or a NaN, as in a row that was never written) takes nothing from the
    precision of the others, however small their values; nor does an attended row whose weight is negligible."""
    g = torch.Generator(device="cuda").manual_seed(T + past + D)
    uniform = lambda *s: torch.rand(s, generator=g, device="cuda") * 2 - 1  # noqa: E731
    n_ctx, n = past + T + 3, past + T
    for size in (1.0, 0.01, 0.001):
        q, k, v = uniform(T, H, D) * 0.3, uniform(n_ctx, HKV, D), uniform(n_ctx, HKV, D) * size
        caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
        mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx)
        # the last token's row: no one's, or (causal) its own alone
        set_row(torch, caches, HKV, n_ctx, D, n - 1, what)
        mask = mi_cuda.tree_mask(list(range(-1, T - 1)))
        mask[T - 1, (T - 1) // 32] &= ~np.int32(1 << (T - 1) % 32) if (T - 1) % 32 < 31 else np.int32(2**31 - 1)
        rows = mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, 0, n)
        attn_componentwise(torch, tree(torch, True, q, caches, HKV, n_ctx, past, 0.125, mask), q, *rows, seen_of(torch, mask, T, past), 0.125)
        if T > 1:
            attn_componentwise(torch, tree(torch, True, q, caches, HKV, n_ctx, past, 0.125), q, *rows, seen_of(torch, None, T, past), 0.125,
                               range(T - 1))
    # attended, but at a score of -60 below the others': a value of 8e6 counts 1e-19
    q, k, v = uniform(T, H, D) * 0.1 + 0.5, uniform(n_ctx, HKV, D), uniform(n_ctx, HKV, D) * 0.01
    k[past - 1], v[past - 1] = -2.0 * 60 / (0.125 * D), 8e6
    caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
    mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx)
    rows = mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, 0, n)
    attn_componentwise(torch, tree(torch, True, q, caches, HKV, n_ctx, past, 0.125), q, *rows, seen_of(torch, None, T, past), 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("word", [0x7f800000, 0xff800000, 0x7f800001, 0x7fc00000])
@pytest.mark.parametrize("H,HKV,D,T,past", [(14, 2, 64, 1, 40), (28, 4, 128, 1, 200), (6, 2, 96, 2, 30), (14, 2, 64, 2, 70), (16, 16, 32, 9, 500),
                                            (14, 2, 64, 24, 300)])
def test_attention_tree_f32_keys_that_are_not_finite(torch, H, HKV, D, T, past, word):
    """An infinity of either sign or a NaN (of any payload) in an F32 key: NaN for the tokens that attend to
    it, whatever their queries' signs, nothing for the others."""
    q, caches, rows, n_ctx = attn_inputs(torch, T, H, HKV, D, past, T + past, False)
    bad = past + T - 1  # the last token's own row
    at = (bad, HKV - 1, D // 2 + 3)
    k = caches[0].clone()
    k.view(torch.int32)[at] = word - (word >> 31 << 32)
    clean = rows[0].clone()
    clean[at] = 0.0
    for sign in (1.0, -1.0, 0.0):
        x = q.clone()
        x[..., at[2]] = x[..., at[2]].abs() * sign
        got = tree(torch, False, x, (k, caches[1]), HKV, n_ctx, past, 0.125).unflatten(1, (HKV, -1))
        assert torch.isnan(got[-1, -1]).any(-1).all(), sign
        want, tol = attn_f64(torch, x, clean, rows[1], seen_of(torch, None, T, past), 0.125)
        want = want.unflatten(1, (HKV, -1))
        assert T == 1 or float((got[:-1].double() - want[:-1]).norm()) <= 2e-5 * float(want[:-1].norm())
        assert HKV == 1 or float((got[-1, :-1].double() - want[-1, :-1]).norm()) <= 2e-5 * float(want[-1, :-1].norm())


def check_scores_past_a_floats_range(torch, H, HKV, D, T, past):
    """Finite F32 keys with a score below a float's range: weight 0, and 1 each for the others' scores of 0."""
    q, caches, rows, n_ctx = attn_inputs(torch, T, H, HKV, D, past, 5, False)
    k = torch.zeros_like(caches[0])
    k[1] = -3e38
    got = tree(torch, False, torch.full_like(q, 3e38), (k, caches[1]), HKV, n_ctx, past, 0.125)
    for i in range(T):
        v = rows[1][: past + i + 1].double()
        want = ((v.sum(0) - v[1]) / (past + i)).repeat_interleave(H // HKV, 0)
        assert float((got[i].double() - want).norm()) <= 2e-5 * float(want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("H,HKV,D,T,past", [(14, 2, 64, 1, 40), (6, 2, 96, 3, 30)])
def test_attention_tree_scores_past_a_floats_range(torch, H, HKV, D, T, past):
    check_scores_past_a_floats_range(torch, H, HKV, D, T, past)


@pytest.mark.gpu
@pytest.mark.parametrize("H,HKV,D,T,past", [(14, 2, 64, 24, 300), (14, 2, 64, 10, 30), (16, 16, 32, 140, 5)])
def test_attention_tree_many_rows_with_scores_past_a_floats_range(torch, H, HKV, D, T, past):
    check_scores_past_a_floats_range(torch, H, HKV, D, T, past)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,HKV,D,T,past", [(14, 2, 64, 1, 100), (14, 2, 64, 30, 100), (28, 4, 128, 64, 3000), (14, 14, 32, 200, 70), (6, 2, 96, 80, 500)])
def test_attention_tree_values_of_any_size(torch, q8, H, HKV, D, T, past):
    """All values of one size, tiny to huge (Q8_0: its scales' range)."""
    for size in (6e-5, 1.0, 60000.0) if q8 else (2.0**-105, 2.0**-101, 2.0**-99, 2.0**-60, 2.0**100, 2.0**110):
        q, caches, _, n_ctx = attn_inputs(torch, T, H, HKV, D, past, 7, False)
        k, v = caches[0], caches[1].clamp(-7, 7) * size
        rows = (k[: past + T], v[: past + T])
        caches = (k, v)
        if q8:
            caches = [mi_cuda.kv_q8_0_cache(n_ctx, HKV, D) for _ in range(2)]
            mi_cuda.kv_append_q8_0(k, v, *caches, n_ctx)
            rows = mi_cuda.kv_read_q8_0(*caches, HKV, D, n_ctx, 0, past + T)
        got = tree(torch, q8, q, caches, HKV, n_ctx, past, 0.125)
        want, _ = attn_f64(torch, q, *rows, seen_of(torch, None, T, past), 0.125)
        assert float((got.double() - want).norm()) <= 2e-5 * float(want.norm()), size


def check_logits(torch, x, out, tokens, hist, repeat, freq, pres, ids, bias, allowed):
    for i in range(x.shape[0]):
        h = hist[i] if hist.ndim == 2 else hist
        a = None if allowed is None else allowed[i] if allowed.ndim == 2 else allowed
        want, tok = logits_f32(x[i], h, repeat, freq, pres, ids, bias, a)
        got = out[i].cpu().numpy()
        same = (got.view(np.uint32) == want.view(np.uint32)) | (np.isnan(got) & np.isnan(want)) | (got == want)
        assert same.all(), np.flatnonzero(~same)[:5]
        assert int(tokens[i]) == tok


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,nh,nb,mask", [(1, 151936, 300, 0, False), (3, 151936, 2000, 50, True), (2, 152064, 0, 7, False),
                                            (5, 257, 40, 9, True), (4, 1, 3, 2, True), (2, 31, 0, 0, True), (2, 33, 100, 0, False),
                                            (7, 50001, 999, 300, True), (64, 2048, 64, 1, True), (1, 600001, 70, 3, True),
                                            (2, 8192, 5000, 2000, False), (1, 5003, 40000, 20, True), (2, 4096, 70001, 3, False),
                                            (9, 40000, 32767, 5, True), (10, 40000, 32768, 700, False)])
@pytest.mark.parametrize("form", ["rows", "shared", "strided"])
def test_logits_process(torch, n, V, nh, nb, mask, form):
    rng = np.random.default_rng(V + nh)
    x = (rng.standard_normal((n, V)) * 4).astype(np.float32)
    shape = lambda m: (m,) if form == "shared" else (n, m)  # noqa: E731
    hist = np.minimum(rng.zipf(1.2, shape(nh)) - 2, 2**31 - 1).astype(np.int32)  # -1 and ids past V are padding
    if nh > 3:
        hist[..., 0], hist[..., 1] = V - 1, -2**31
    ids = rng.integers(-1, V + 1, nb).astype(np.int32) if nb else None  # some twice, some outside
    bias = (rng.standard_normal(nb) * 3).astype(np.float32) if nb else None
    words = (V + 31) // 32
    allowed = rng.integers(0, 2**32, shape(words), dtype=np.uint64).astype(np.uint32) if mask else None
    if mask and form == "rows":
        allowed[-1] = 0  # nothing is left
    up = lambda a: None if a is None else torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()  # noqa: E731
    X, H, A = up(x), up(hist), up(allowed)
    if form == "strided":
        pad = lambda t, m: torch.nn.functional.pad(t, (m, 4))[:, m:-4]  # noqa: E731
        X, H, A = pad(X, 3), pad(H, 1), None if A is None else pad(A, 2)
    kw = dict(repeat=1.15, frequency=0.3, presence=-0.2, bias_ids=up(ids), bias=up(bias), allowed=A)
    out, tok = mi_cuda.logits_process(X, hist=H, **kw)
    check_logits(torch, x, out, tok, hist, 1.15, 0.3, -0.2, ids, bias, allowed)
    if form != "strided":  # in place
        Y = X.clone()
        o2, t2 = mi_cuda.logits_process(Y, hist=H, out=Y, **kw)
        assert o2 is Y and torch.equal(o2.view(torch.int32), out.view(torch.int32)) and torch.equal(t2, tok)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [6, 7, 20, 21, 40])
@pytest.mark.parametrize("V", [3001, 40004, 200000])
def test_logits_process_numbers_of_rows(torch, n, V):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((n, V)) * 4).astype(np.float32)
    hist = rng.integers(0, V, (n, 700)).astype(np.int32)
    hist[:, ::3] = hist[:, :1]
    allowed = rng.integers(0, 2**32, (n, (V + 31) // 32), dtype=np.uint64).astype(np.uint32)
    out, tok = mi_cuda.logits_process(torch.from_numpy(x).cuda(), hist=torch.from_numpy(hist).cuda(), repeat=1.15, frequency=0.3,
                                      presence=-0.2, allowed=torch.from_numpy(allowed.view(np.int32)).cuda())
    check_logits(torch, x, out, tok, hist, 1.15, 0.3, -0.2, None, None, allowed)


@pytest.mark.gpu
def test_logits_process_values(torch):
    """Ties, infinities, NaN, a row without a value above -infinity, the largest floats."""
    V = 1000
    x = np.zeros((7, V), dtype=np.float32)
    x[0, [17, 500, 999]] = 2.0
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 3], x[3, 900] = np.inf, np.nan
    x[4] = -1.0
    x[4, 10:20] = -np.inf
    x[5] = 3.4e38
    x[6, 998], x[6, 999] = -0.0, 0.0
    hist = np.array([[17, 17, 3], [1, 2, 3], [5, 5, 5], [3, 900, 901], [10, 11, 30], [7, 8, 9], [0, 998, 1]], dtype=np.int32)
    H, X = torch.from_numpy(hist).cuda(), torch.from_numpy(x).cuda()
    for repeat, freq, pres in ((1.3, 0.1, 0.2), (0.5, -0.1, 0.0), (1.0, 0.0, 0.0)):
        out, tok = mi_cuda.logits_process(X, hist=H, repeat=repeat, frequency=freq, presence=pres)
        check_logits(torch, x, out, tok, hist, repeat, freq, pres, None, None, None)
    out, tok = mi_cuda.logits_process(X)
    assert torch.equal(out.view(torch.int32), X.view(torch.int32)) and tok.tolist()[:2] == [17, -1]
    # more tokens with a count in one part than its list holds
    V2 = 151936
    x2 = (np.random.default_rng(5).standard_normal((11, V2)) * 3).astype(np.float32)
    hist2 = np.arange(1000, 31000, dtype=np.int32)
    for rows in (1, 11):
        out, tok = mi_cuda.logits_process(torch.from_numpy(x2[:rows]).cuda(), hist=torch.from_numpy(hist2).cuda(), repeat=1.3, presence=0.5)
        check_logits(torch, x2[:rows], out, tok, hist2, 1.3, 0.0, 0.5, None, None, None)
    # one token named by every bias: the list's order
    ids = torch.full((1500,), 321, dtype=torch.int32, device="cuda")
    bias = np.random.default_rng(0).standard_normal(1500).astype(np.float32) * 1000
    out, tok = mi_cuda.logits_process(X[:1], bias_ids=ids, bias=torch.from_numpy(bias).cuda())
    check_logits(torch, x[:1], out, tok, np.zeros(0, np.int32), 1.0, 0.0, 0.0, ids.cpu().numpy(), bias, None)


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,nb", [(1, 152064, 30000), (2, 5000, 9000), (13, 40004, 513), (24, 151936, 6000), (1, 700001, 100000),
                                    (2, 655360, 2048)])
@pytest.mark.parametrize("wide", [False, True])
def test_logits_process_many_biases(torch, n, V, nb, wide):
    """More biases than a part keeps at hand, most of their tokens distinct, some named many times."""
    rng = np.random.default_rng(nb)
    x = (rng.standard_normal((n, V)) * 4).astype(np.float32)
    ids = rng.integers(-1, V + 1, nb).astype(np.int32)
    ids[::7] = ids[0]
    ids[1::5] = V - 1 - rng.integers(0, 20, ids[1::5].size)
    bias = (rng.standard_normal(nb) * 3).astype(np.float32)
    hist = rng.integers(0, V, 33000 if wide else 700).astype(np.int32)
    allowed = rng.integers(0, 2**32, (n, (V + 31) // 32), dtype=np.uint64).astype(np.uint32)
    X = torch.from_numpy(x).cuda()
    kw = dict(hist=torch.from_numpy(hist).cuda(), repeat=1.15, frequency=0.3, presence=-0.2, bias_ids=torch.from_numpy(ids).cuda(),
              bias=torch.from_numpy(bias).cuda(), allowed=torch.from_numpy(allowed.view(np.int32)).cuda())
    out, tok = mi_cuda.logits_process(X, **kw)
    check_logits(torch, x, out, tok, hist, 1.15, 0.3, -0.2, ids, bias, allowed)
    o2, t2 = mi_cuda.logits_process(X, out=X, **kw)
    assert torch.equal(o2.view(torch.int32), out.view(torch.int32)) and torch.equal(t2, tok)


@pytest.mark.gpu
def test_logits_process_time_grows_with_the_biases(torch):
    """Four times the biases take some four times as long at most (not sixteen)."""
    V, rng = 151936, np.random.default_rng(0)
    X = torch.zeros((4, V), device="cuda")
    took = []
    for nb in (20000, 80000):
        ids = torch.from_numpy(rng.permutation(V)[:nb].astype(np.int32)).cuda()
        bias = torch.ones(nb, device="cuda")
        best = math.inf
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            mi_cuda.logits_process(X, bias_ids=ids, bias=bias)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        took.append(best)
    assert took[1] <= 8 * took[0], took


@pytest.mark.gpu
def test_calls_with_no_tokens(torch):
    e = torch.empty((0, 2, 64), device="cuda")
    q, k = mi_cuda.qk_norm_rope(e, e, None, None, 1e-6, 0, 64, 1e6)
    assert q.shape == (0, 2, 64) and k.shape == (0, 2, 64)
    caches = [mi_cuda.kv_q8_0_cache(4, 2, 64) for _ in range(2)]
    mi_cuda.kv_append_q8_0(e, e, *caches, 4)
    assert not caches[0].any()
    assert mi_cuda.attention_tree_q8_0(e, *caches, 2, 4, 4, 0.1).shape == (0, 2, 64)
    out, tok = mi_cuda.logits_process(torch.empty((0, 100), device="cuda"))
    assert out.shape == (0, 100) and tok.shape == (0,)


NOT_PREPARED = """
import ctypes, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # (found before the library's own)
sys.path.insert(0, sys.argv[2])
import torch, mi_cuda
mi_cuda.init(0)
x = torch.arange(64, device="cuda", dtype=torch.float32)
assert int(mi_cuda.argmax(x)) == 63
q, c = torch.ones((1, 2, 64), device="cuda"), torch.zeros((4, 2, 64), device="cuda")
for sign, call in zip(sys.argv[3], (lambda: mi_cuda.attention_tree(q, c, c, 2, 2, 0.1), lambda: mi_cuda.logits_process(x[None]))):
    try:
        call()
        assert sign == "1"
    except mi_cuda.MiCudaError as e:
        assert sign == "0" and e.code == mi_cuda.ERR_CUDA and "could not be prepared" in str(e), e
torch.cuda.synchronize()
"""


@pytest.mark.gpu
@pytest.mark.parametrize("symbol,works", [("_ZN2mi25prepare_attn_tree_kernelsEv", "01"), ("_ZN2mi24prepare_attn_few_kernelsEv", "01"),
                                          ("_ZN2mi22prepare_logits_kernelsEv", "10")])
def test_kernels_that_cannot_be_prepared_refuse_their_own_calls_alone(torch, tmp_path, symbol, works):
    """As in a build that gives a kernel too few registers: a stand-in for the host function that finds out."""
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    (tmp_path / "f.c").write_text(f"int {symbol}(void) {{ return 9; }}  /* cudaErrorInvalidConfiguration */\n")
    fake = str(tmp_path / "f.so")
    subprocess.run(["gcc", "-shared", "-fPIC", str(tmp_path / "f.c"), "-o", fake], check=True)
    r = subprocess.run([sys.executable, "-c", NOT_PREPARED, fake, PKG, works], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


class Step:
    """A drafted step of one attention layer through the operators, and its formula in 64 bits
    over a cache that the operators quantised."""

    H, HKV, D, V, n_ctx = 14, 2, 64, 2048, 600

    def __init__(self, torch):
        g = torch.Generator(device="cuda").manual_seed(0)
        rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.wq, self.wk = 1 + 0.1 * rnd(self.D), 1 + 0.1 * rnd(self.D)
        self.head = rnd(self.H * self.D, self.V) * 0.2
        self.torch, self.rnd = torch, rnd
        self.caches = [mi_cuda.kv_q8_0_cache(self.n_ctx, self.HKV, self.D) for _ in range(2)]
        self.scratch = mi_cuda.attention_tree_scratch(self.H, self.HKV, self.n_ctx, self.n_ctx, self.D)

    def qkv(self, T):
        return self.rnd(T, (self.H + 2 * self.HKV) * self.D)

    def split(self, qkv):
        return (x.unflatten(1, (-1, self.D)) for x in qkv.split([self.H * self.D, self.HKV * self.D, self.HKV * self.D], 1))

    def run(self, qkv, past, pos, mask, hist, allowed):
        q, k, v = self.split(qkv)
        q, k = mi_cuda.qk_norm_rope(q, k, self.wq, self.wk, 1e-6, past, self.D, 1e6, pos=pos)
        mi_cuda.kv_append_q8_0(k, v, *self.caches, self.n_ctx, past)
        o = mi_cuda.attention_tree_q8_0(q, *self.caches, self.HKV, self.n_ctx, past, 0.125, mask=mask, scratch=self.scratch)
        logits = o.flatten(1) @ self.head
        return (k, o) + mi_cuda.logits_process(logits, hist=hist, repeat=1.2, frequency=0.1, allowed=allowed) + (logits,)


@pytest.mark.gpu
def test_drafted_step(torch):
    """A prompt, a drafted tree checked in one step, the accepted path moved into place, the next
    single token: every output against 64 bits, where each drafted token sees its own path only."""
    s = Step(torch)
    rng = np.random.default_rng(1)
    past = 201
    s.run(s.qkv(past), 0, None, None, None, None)
    parents = random_tree(rng, 23)
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    mask = mi_cuda.tree_mask(parents)
    pos = torch.tensor([past + d for d in depth], dtype=torch.int32, device="cuda")
    hist = rng.integers(0, s.V, (23, 50)).astype(np.int32)
    allowed = rng.integers(0, 2**32, (23, s.V // 32), dtype=np.uint64).astype(np.uint32)
    qkv = s.qkv(23)
    k, o, out, tok, logits = s.run(qkv, past, pos, torch.from_numpy(mask).cuda(), torch.from_numpy(hist).cuda(),
                                   torch.from_numpy(allowed.view(np.int32)).cuda())
    q_raw, k_raw, v_raw = s.split(qkv)
    check_heads(torch, k, k_raw, s.wk, 1e-6, pos, s.D, 1e6)
    rows = mi_cuda.kv_read_q8_0(*s.caches, s.HKV, s.D, s.n_ctx, 0, past + 23)
    q64, _ = heads_f64(torch, q_raw, s.wq, 1e-6, pos, s.D, 1e6)
    for i in range(23):  # token i alone, behind the cached text and its ancestors
        path = [i]
        while parents[path[-1]] >= 0:
            path.append(parents[path[-1]])
        at = torch.tensor(list(range(past)) + [past + j for j in reversed(path)], device="cuda")
        want, tol = attn_f64(torch, q64[i:i + 1], rows[0][at], rows[1][at], torch.ones((1, at.numel()), dtype=torch.bool, device="cuda"), 0.125)
        # (the queries' own rounding, 24 u of two elements, counts like the scores')
        assert float((o[i].double() - want[0]).abs().max()) <= 4 * tol
    check_logits(torch, logits.cpu().numpy(), out, tok, hist, 1.2, 0.1, 0.0, None, None, allowed)
    # accept the path to the deepest token: its rows move up behind the text, the others are dropped
    path = [int(np.argmax(depth))]
    while parents[path[-1]] >= 0:
        path.append(parents[path[-1]])
    path.reverse()
    slots = np.full(23, -1, dtype=np.int32)
    slots[path] = past + np.arange(len(path))
    mi_cuda.kv_append_q8_0(k, v_raw, *s.caches, s.n_ctx, slots=torch.from_numpy(slots).cuda())
    moved = mi_cuda.kv_read_q8_0(*s.caches, s.HKV, s.D, s.n_ctx, past, len(path))
    assert all(torch.equal(a, b[[past + j for j in path]]) for a, b in zip(moved, rows))
    past += len(path)
    qkv = s.qkv(1)
    _, o, _, _, _ = s.run(qkv, past, None, None, None, None)
    rows = mi_cuda.kv_read_q8_0(*s.caches, s.HKV, s.D, s.n_ctx, 0, past + 1)
    q64, _ = heads_f64(torch, next(s.split(qkv)), s.wq, 1e-6, torch.tensor([past], device="cuda"), s.D, 1e6)
    want, tol = attn_f64(torch, q64, *rows, torch.ones((1, past + 1), dtype=torch.bool, device="cuda"), 0.125)
    assert float((o.double() - want).abs().max()) <= 4 * tol


@pytest.mark.gpu
def test_drafted_step_captured_and_on_other_streams(torch):
    """The step recorded into a CUDA graph and replayed on new inputs; two steps on two streams at once."""
    s = Step(torch)
    past, T = 300, 9
    s.run(s.qkv(past), 0, None, None, None, None)
    parents = random_tree(np.random.default_rng(2), T)
    mask = torch.from_numpy(mi_cuda.tree_mask(parents)).cuda()
    hist = torch.randint(0, s.V, (T, 30), device="cuda", dtype=torch.int32)
    held, pos = s.qkv(T), torch.arange(past, past + T, device="cuda", dtype=torch.int32)
    steps = [s.qkv(T) for _ in range(3)]
    want = [[x.clone() for x in s.run(x, past, pos, mask, hist, None)] for x in steps]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.run(held, past, pos, mask, hist, None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.run(held, past, pos, mask, hist, None)
    for x, w in zip(steps, want):
        held.copy_(x)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got[:4], w[:4]))
    # two caches, two scratches, two streams
    other = Step(torch)
    other.run(other.qkv(past), 0, None, None, None, None)
    w2 = [x.clone() for x in other.run(steps[1], past, pos, mask, hist, None)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        b = other.run(steps[1], past, pos, mask, hist, None)
    a = s.run(steps[0], past, pos, mask, hist, None)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a[:4], want[0][:4])) and all(torch.equal(x, y) for x, y in zip(b[:4], w2[:4]))

"""Timed cases of the drafted-token operators: norms and rotation of queries and
keys per head, the Q8_0 key/value cache (append and read back), attention of a
tree of drafted tokens over a cache, and penalties, biases and grammar masks on
logits.

Every case has the operators' plain form (elementary torch operations in 32
bits) and, with `own` set, the calls of mini-infer-llama.cpp_b200/mi_cuda.py.
Sizes are those of the repository's own model shapes (14 / 2 heads of 64, 28 / 4
heads of 128, vocabularies of 151936 and 152064) and generic ones.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32  # values per scale of the Q8_0 cache
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-infer-llama.cpp_b200")
_mc = None


def _binding():
    """The framework's Python binding (loaded on the first use by a kernel's case)."""
    global _mc
    if _mc is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import mi_cuda
        _mc = mi_cuda
    return _mc


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decoded token's queries and keys (0.5B heads): launch latency
        dict(name="heads_token", kind="heads", tokens=1, n_past=2047, heads=14, kv_heads=2, dim=64, n_dims=64, norm=True, tree=False),
        # a prompt chunk's stacked q|k|v rows (7B heads), no head norms
        dict(name="heads_prompt", kind="heads", tokens=4096, n_past=1021, heads=28, kv_heads=4, dim=128, n_dims=128, norm=False, tree=False),
        # 13 drafted tokens written (some rejected ones skipped), the cache handed back as F32
        dict(name="cache_draft", kind="cache", tokens=13, n_past=2035, kv_heads=2, dim=64, slots=True),
        # a prompt chunk written behind another and read back (7B heads)
        dict(name="cache_prompt", kind="cache", tokens=4096, n_past=4001, kv_heads=4, dim=128, slots=False),
        # single-token decode over the quantised cache: a short and the longest context
        dict(name="attn_token_2k", kind="attn", tokens=1, n_past=2046, heads=14, kv_heads=2, dim=64, cache="q8_0", tree=False),
        dict(name="attn_token_32k", kind="attn", tokens=1, n_past=32767, heads=14, kv_heads=2, dim=64, cache="q8_0", tree=False),
        # a small tree over the F32 cache (7B heads, an odd context)
        dict(name="attn_tree13_f32", kind="attn", tokens=13, n_past=1021, heads=28, kv_heads=4, dim=128, cache="f32", tree=True),
        # wide trees over the quantised cache: 7B heads, and the longest context
        dict(name="attn_tree64_8k", kind="attn", tokens=64, n_past=8111, heads=28, kv_heads=4, dim=128, cache="q8_0", tree=True),
        dict(name="attn_tree64_32k", kind="attn", tokens=64, n_past=32700, heads=14, kv_heads=2, dim=64, cache="q8_0", tree=True),
        # one decoded row with penalties; a drafted tree's rows under a grammar; a large batch of rows
        dict(name="logits_token", kind="logits", rows=1, vocab=151936, hist=511, bias=0, allowed="", repeat=1.1, frequency=0.0, presence=0.0),
        dict(name="logits_grammar13", kind="logits", rows=13, vocab=151936, hist=2048, bias=40, allowed="few", repeat=1.05, frequency=0.2, presence=0.1),
        dict(name="logits_rows64", kind="logits", rows=64, vocab=152064, hist=4093, bias=300, allowed="most", repeat=1.2, frequency=0.1, presence=0.3),
    ]


HEADS = [(14, 2, 64), (28, 4, 128), (4, 2, 64), (16, 16, 32), (6, 2, 96)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["heads", "cache", "attn", "attn", "logits"])
    h, kv, d = rng.choice(HEADS)
    if kind == "heads":
        tree = rng.random() < 0.5
        return dict(kind=kind, tokens=_log(rng, 1, 64 if tree else 4096), n_past=_log(rng, 1, 131000) - 1, heads=h, kv_heads=kv, dim=d,
                    n_dims=rng.choice([d, d, d // 2]), norm=rng.random() < 0.7, tree=tree)
    if kind == "cache":
        slots = rng.random() < 0.5
        return dict(kind=kind, tokens=_log(rng, 1, 64 if slots else 4096), n_past=_log(rng, 1, 4001) - 1, kv_heads=kv, dim=d, slots=slots)
    if kind == "attn":
        tokens = _log(rng, 1, 64)
        # no more score-value products than the largest listed case
        most = min(32700, 64 * 14 * 64 * 32700 // (tokens * h * d))
        return dict(kind=kind, tokens=tokens, n_past=_log(rng, 1, most) - 1, heads=h, kv_heads=kv, dim=d,
                    cache=rng.choice(["q8_0", "q8_0", "f32"]), tree=rng.random() < 0.6)
    return dict(kind=kind, rows=_log(rng, 1, 64), vocab=rng.choice([151936, 152064, 2048, _log(rng, 257, 150000)]), hist=_log(rng, 1, 4093) - 1,
                bias=rng.choice([0, rng.randint(1, 300)]), allowed=rng.choice(["", "few", "most"]), repeat=rng.choice([1.0, 1.05, 1.3]),
                frequency=rng.choice([0.0, 0.15]), presence=rng.choice([0.0, 0.4]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _parents(n, r):
    """A random draft tree: token i hangs below an earlier token, or (-1) below the cached text."""
    return [-1 if i == 0 or r.random() < 0.1 else int(r.integers(max(0, i - 8), i)) for i in range(n)]


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _mask_words(parents):
    """[n][ceil(n / 32)] words: bit j of row i where token j is token i or one of its ancestors."""
    n = len(parents)
    bits = np.zeros((n, (n + 31) // 32 * 32), dtype=np.uint32)
    for i, p in enumerate(parents):
        if p >= 0:
            bits[i] = bits[p]
        bits[i, i] = 1
    words = (bits.reshape(n, -1, 32) << np.arange(32, dtype=np.uint32)).sum(-1, dtype=np.uint32)
    return words.view(np.int32)


def _kv(shape, g):
    """Key / value rows: normal values, a few channels with an offset (as biased projections give)."""
    x = torch.randn(shape, generator=g, device="cuda")
    off = torch.randn(shape[-2:], generator=g, device="cuda") * 6
    return x + off * (torch.rand(shape[-2:], generator=g, device="cuda") < 0.06)


def _quantise(x):
    """Rows [n][kv_heads][dim] -> (int8 [kv_heads][n][dim], fp16 [kv_heads][n][dim / 32])."""
    b = x.transpose(0, 1).reshape(x.shape[1], x.shape[0], -1, BLOCK)
    d = (b.abs().amax(-1, keepdim=True) / 127).clamp(max=65504.0).half()
    f = d.float()
    q = torch.where(f > 0, torch.round(b / torch.where(f > 0, f, torch.ones_like(f))).clamp(-127, 127), torch.zeros_like(b))
    return q.to(torch.int8).flatten(-2), d.squeeze(-1)


def _pack(q, d):
    """The cache buffer: the int8 plane, then the fp16 plane."""
    return torch.cat([q.contiguous().view(torch.uint8).flatten(), d.contiguous().view(torch.uint8).flatten()])


def _planes(buf, kv_heads, n_ctx, dim):
    n = kv_heads * n_ctx * dim
    return buf[:n].view(torch.int8).view(kv_heads, n_ctx, dim), buf[n:].view(torch.float16).view(kv_heads, n_ctx, dim // BLOCK)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    st = dict(case)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    if case["kind"] == "heads":
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        qkv = torch.randn((t, (h + 2 * kv) * d), generator=g, device="cuda") * 2
        st["q"] = qkv[:, : h * d].view(t, h, d)
        st["k"] = qkv[:, h * d : (h + kv) * d].view(t, kv, d)
        st["wq"] = 1 + 0.3 * torch.randn(d, generator=g, device="cuda") if case["norm"] else None
        st["wk"] = 1 + 0.3 * torch.randn(d, generator=g, device="cuda") if case["norm"] else None
        st["pos"] = dev(np.array([case["n_past"] + x for x in _depths(_parents(t, r))], dtype=np.int32)) if case["tree"] else None
    elif case["kind"] == "cache":
        t, past, kv, d = case["tokens"], case["n_past"], case["kv_heads"], case["dim"]
        st["n_ctx"] = past + t
        for x in "kv":
            q, s = _quantise(_kv((st["n_ctx"], kv, d), g))
            st["cache_" + x] = _pack(q, s)
            st[x] = _kv((t, kv, d), g)
        if case["slots"]:
            s = past + np.arange(t)
            s[r.random(t) < 0.3] = -1
            st["slots"] = dev(s.astype(np.int32))
        else:
            st["slots"] = None
    elif case["kind"] == "attn":
        t, past, h, kv, d = case["tokens"], case["n_past"], case["heads"], case["kv_heads"], case["dim"]
        st["n_ctx"] = past + t + 37  # rows behind the last drafted token are not read
        st["q"] = torch.randn((t, h, d), generator=g, device="cuda") * 1.5
        for x in "kv":
            rows = _kv((st["n_ctx"], kv, d), g)
            st["cache_" + x] = _pack(*_quantise(rows)) if case["cache"] == "q8_0" else rows
        st["mask"] = dev(_mask_words(_parents(t, r))) if case["tree"] else None
    else:
        n, v = case["rows"], case["vocab"]
        st["logits"] = torch.randn((n, v), generator=g, device="cuda") * 3
        hist = np.minimum(r.zipf(1.3, (n, case["hist"])) * 7919 % v, v - 1).astype(np.int32) if case["hist"] else np.zeros((n, 0), np.int32)
        for i in range(1, n):  # shorter histories are padded
            hist[i, case["hist"] - int(r.integers(0, case["hist"] // 4 + 1)):] = -1
        st["hist"] = dev(hist)
        st["bias_ids"] = dev(r.choice(v, min(v, case["bias"]), replace=False).astype(np.int32)) if case["bias"] else None
        st["bias"] = dev(r.normal(0, 4, st["bias_ids"].numel()).astype(np.float32)) if case["bias"] else None
        st["allowed_words"] = None
        if case["allowed"]:
            words = (v + 31) // 32
            bits = torch.randint(-(2**31), 2**31, (n, words), generator=g, device="cuda", dtype=torch.int64)
            for _ in range(5):  # one bit in 64 is left, or one in 64 is taken out
                bits &= torch.randint(-(2**31), 2**31, (n, words), generator=g, device="cuda", dtype=torch.int64)
            st["allowed_words"] = (bits if case["allowed"] == "few" else ~bits).to(torch.int32)
    return st


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _plain_heads(st):
    n, half = st["n_dims"], st["n_dims"] // 2
    t = st["q"].shape[0]
    pos = st["pos"] if st["pos"] is not None else st["n_past"] + torch.arange(t, device="cuda")
    freq = torch.pow(torch.tensor(1e6, dtype=torch.float64, device="cuda"), -2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / n)
    a = pos.double()[:, None, None] * freq
    c, s = torch.cos(a).float(), torch.sin(a).float()
    out = []
    for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        lo, hi = x[..., :half], x[..., half:n]
        out.append(torch.cat([lo * c - hi * s, lo * s + hi * c, x[..., n:]], -1))
    return out


def _plain_cache(st):
    kv, d, n_ctx, past, t = st["kv_heads"], st["dim"], st["n_ctx"], st["n_past"], st["tokens"]
    out = []
    for x in "kv":
        q, s = _planes(st["cache_" + x], kv, n_ctx, d)
        nq, ns = _quantise(st[x])
        at = torch.where(st["slots"] < 0, n_ctx, st["slots"]).long() if st["slots"] is not None else past + torch.arange(t, device="cuda")
        # (a skipped token goes to a row behind the last)
        q = torch.cat([q, q[:, :1]], 1).index_copy(1, at, nq)[:, :n_ctx]
        s = torch.cat([s, s[:, :1]], 1).index_copy(1, at, ns)[:, :n_ctx]
        out.append((q.float().unflatten(-1, (-1, BLOCK)) * s.float()[..., None]).flatten(-2).transpose(0, 1).contiguous())
    return out


def _rows(st, x, n, dtype):
    """Cache rows [0, n) as [kv_heads][n][dim] values."""
    if st["cache"] == "f32":
        return st["cache_" + x][:n].transpose(0, 1).to(dtype)
    q, s = _planes(st["cache_" + x], st["kv_heads"], st["n_ctx"], st["dim"])
    return (q[:, :n].to(dtype).unflatten(-1, (-1, BLOCK)) * s[:, :n].to(dtype)[..., None]).flatten(-2)


def _plain_attn(st):
    t, past, h, kv, d = st["tokens"], st["n_past"], st["heads"], st["kv_heads"], st["dim"]
    rep, n = h // kv, past + t
    k, v = _rows(st, "k", n, torch.float32), _rows(st, "v", n, torch.float32)
    q = st["q"].view(t, kv, rep, d).permute(1, 0, 2, 3).reshape(kv, t * rep, d)
    s = torch.matmul(q, k.transpose(1, 2)).view(kv, t, rep, n) * (1.0 / math.sqrt(d))
    j = torch.arange(t, device="cuda")
    if st["mask"] is not None:
        seen = ((st["mask"][:, j // 32] >> (j % 32)) & 1) != 0
    else:
        seen = j[None, :] <= j[:, None]
    s[..., past:].masked_fill_(~seen[:, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1)
    o = torch.matmul(p.view(kv, t * rep, n), v).view(kv, t, rep, d) / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    return o.permute(1, 0, 2, 3).reshape(t, h, d)


def _allowed_bits(words, v):
    j = torch.arange(v, device="cuda")
    return ((words[:, j // 32] >> (j % 32)) & 1) != 0


def _plain_logits(st):
    x, v = st["logits"], st["vocab"]
    n = x.shape[0]
    if st["hist"].shape[1]:
        ids = torch.where((st["hist"] < 0) | (st["hist"] >= v), v, st["hist"]).long()  # padding counts behind the last token
        c = torch.zeros((n, v + 1), dtype=torch.int32, device="cuda").scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.int32))[:, :v]
        y = torch.where(x > 0, x / st["repeat"], x * st["repeat"]) - (c.float() * st["frequency"] + st["presence"])
        x = torch.where(c > 0, y, x)
    if st["bias"] is not None:
        x = x + torch.zeros(v, device="cuda").index_add_(0, st["bias_ids"].long(), st["bias"])
    if st["allowed_words"] is not None:
        x = torch.where(_allowed_bits(st["allowed_words"], v), x, torch.full_like(x, -math.inf))
    x = x.clone() if x is st["logits"] else x
    top = x.amax(-1, keepdim=True)
    j = torch.arange(v, device="cuda", dtype=torch.int32)
    token = torch.where((x == top) & (x > -math.inf), j, v).amin(-1)
    return x, torch.where(token == v, -1, token).to(torch.int32)


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _own_heads(st, mc):
    return mc.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], 1e-6, st["n_past"], st["n_dims"], 1e6, pos=st["pos"])


def _own_cache(st, mc):
    kv, d, n_ctx = st["kv_heads"], st["dim"], st["n_ctx"]
    mc.kv_append_q8_0(st["k"], st["v"], st["cache_k"], st["cache_v"], n_ctx, st["n_past"], slots=st["slots"])
    return mc.kv_read_q8_0(st["cache_k"], st["cache_v"], kv, d, n_ctx, 0, n_ctx)


def _own_attn(st, mc):
    t, kv, past, scale = st["tokens"], st["kv_heads"], st["n_past"], 1.0 / math.sqrt(st["dim"])
    if "scratch" not in st:  # the workspace that a program keeps for its steps
        st["scratch"] = mc.attention_tree_scratch(st["heads"], kv, past + t, t, st["dim"])
    if st["cache"] == "f32":
        return mc.attention_tree(st["q"], st["cache_k"], st["cache_v"], kv, past, scale, mask=st["mask"], scratch=st["scratch"])
    return mc.attention_tree_q8_0(st["q"], st["cache_k"], st["cache_v"], kv, st["n_ctx"], past, scale, mask=st["mask"], scratch=st["scratch"])


def _own_logits(st, mc):
    return mc.logits_process(st["logits"], hist=st["hist"], repeat=st["repeat"], frequency=st["frequency"], presence=st["presence"],
                             bias_ids=st["bias_ids"], bias=st["bias"], allowed=st["allowed_words"])


_PLAIN = {"heads": _plain_heads, "cache": _plain_cache, "attn": _plain_attn, "logits": _plain_logits}
_OWN = {"heads": _own_heads, "cache": _own_cache, "attn": _own_attn, "logits": _own_logits}


def run(state):
    if own:
        return _OWN[state["kind"]](state, _binding())
    return _PLAIN[state["kind"]](state)


def work(case):
    if case["kind"] == "heads":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 8 * n + 4 * case["tokens"], "flops": 8 * n}
    if case["kind"] == "cache":
        new, rows = (2 * m * case["kv_heads"] * case["dim"] for m in (case["tokens"], case["n_past"] + case["tokens"]))
        return {"bytes": new * (4 + 34 / 32) + rows * (34 / 32 + 4), "flops": 4 * new + rows}
    if case["kind"] == "attn":
        n = case["n_past"] + case["tokens"]
        per = 34 / 32 if case["cache"] == "q8_0" else 4
        return {"bytes": 2 * n * case["kv_heads"] * case["dim"] * per + 8 * case["tokens"] * case["heads"] * case["dim"],
                "flops": 4 * n * case["tokens"] * case["heads"] * case["dim"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": 8 * n + (n / 8 if case["allowed"] else 0) + 4 * case["rows"] * (case["hist"] + 1) + 8 * case["bias"], "flops": n}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_heads(st):
    n, half = st["n_dims"], st["n_dims"] // 2
    t = st["q"].shape[0]
    pos = st["pos"].double() if st["pos"] is not None else torch.arange(st["n_past"], st["n_past"] + t, device="cuda").double()
    turn = torch.exp(torch.arange(half, device="cuda").double() * (-2.0 * math.log(1e6) / n))
    z = torch.polar(torch.ones((t, half), dtype=torch.float64, device="cuda"), pos[:, None] * turn)[:, None]
    out = []
    for x, w in ((st["q"].double(), st["wq"]), (st["k"].double(), st["wk"])):
        if w is not None:
            x = w.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6)
        y = torch.complex(x[..., :half].contiguous(), x[..., half:n].contiguous()) * z
        out.append(torch.cat([y.real, y.imag, x[..., n:]], -1))
    return out


def _exact_cache(st):
    kv, d, n_ctx, past, t = st["kv_heads"], st["dim"], st["n_ctx"], st["n_past"], st["tokens"]
    slots = st["slots"].tolist() if st["slots"] is not None else list(range(past, past + t))
    src = [i for i, s in enumerate(slots) if s >= 0]
    dst = [slots[i] for i in src]
    out = []
    for x in "kv":
        q, s = _planes(st["cache_" + x], kv, n_ctx, d)
        rows = (q.double() * s.double().repeat_interleave(BLOCK, -1)).transpose(0, 1).clone()
        new = st[x][src].double().reshape(len(src), kv, d // BLOCK, BLOCK)
        step = (new.abs().amax(-1, keepdim=True) / 127.0).half().double()
        val = torch.where(step > 0, (new / step.clamp(min=1e-30)).round().clamp(-127, 127) * step, torch.zeros_like(new))
        rows[dst] = val.reshape(len(src), kv, d)
        out.append(rows)
    return out


def _exact_attn(st):
    t, past, h, kv, d = st["tokens"], st["n_past"], st["heads"], st["kv_heads"], st["dim"]
    n = past + t
    seen = torch.ones((t, n), dtype=torch.bool, device="cuda")
    if st["mask"] is None:
        seen[:, past:] = torch.ones((t, t), device="cuda").tril().bool()
    else:
        words = st["mask"].cpu().numpy().view(np.uint32)
        seen[:, past:] = torch.tensor([[bool(words[i, j // 32] >> (j % 32) & 1) for j in range(t)] for i in range(t)], device="cuda")
    k, v = _rows(st, "k", n, torch.float64), _rows(st, "v", n, torch.float64)
    out = torch.empty((t, h, d), dtype=torch.float64, device="cuda")
    for i in range(h):
        x = st["q"][:, i].double() @ k[i // (h // kv)].t() / math.sqrt(d)
        p = torch.softmax(x.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
        out[:, i] = p @ v[i // (h // kv)]
    return out


def _exact_logits(st):
    x, v = st["logits"].double(), st["vocab"]
    for i in range(x.shape[0]):
        ids, counts = torch.unique(st["hist"][i][(st["hist"][i] >= 0) & (st["hist"][i] < v)].long(), return_counts=True)
        y = x[i, ids]
        x[i, ids] = y * torch.where(y > 0, 1.0 / st["repeat"], st["repeat"]) - counts * st["frequency"] - st["presence"]
    if st["bias"] is not None:
        x[:, st["bias_ids"].long()] += st["bias"].double()
    if st["allowed_words"] is not None:
        bits = np.unpackbits(st["allowed_words"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :v]
        x.masked_fill_(torch.from_numpy(bits == 0).cuda(), -math.inf)
    return x, None


def exact(case, seed):
    return {"heads": _exact_heads, "cache": _exact_cache, "attn": _exact_attn, "logits": _exact_logits}[case["kind"]](prepare(case, seed))

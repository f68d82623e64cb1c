"""Timed cases of speculative decoding over a key/value cache, each operator in its plain form and as the framework's call.

  cache      keys and values of new tokens are written to an INT8 cache (one scale per head and position) and read back
  attention  n new rows, one token or a tree of drafted ones, attend to a bfloat16 or INT8 cache that already holds their own
             keys and values
  verify     drafted tokens against the target's probabilities, from given random numbers: the accepted rows and the next token
  keep       the accepted rows of a tree move together in the caches of all layers

A case is a dict of plain values; `draw` gives further cases of the same ranges.  The plain forms are elementary torch operations in
float32, in float64 where a comparison decides a token.  `exact` restates every operator in float64, apart from them."""
import math
import random
from types import SimpleNamespace

import torch

own = False

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # one generated token: its keys and values go into the cache of a layer
        dict(name="cache token", op="cache", kv_heads=8, dim=128, context=1500, tokens=1, read="new", layout="heads"),
        # a prompt is written; its attention reads what the cache holds
        dict(name="cache prompt 2048", op="cache", kv_heads=8, dim=128, context=0, tokens=2048, read="all", layout="heads"),
        # a short portion after a long conversation: everything before it is read back
        dict(name="cache portion 333 of 30000", op="cache", kv_heads=16, dim=128, context=29667, tokens=333, read="all", layout="tokens"),
        # one token of an ordinary conversation, bfloat16 cache: the smallest call
        dict(name="attention token bf16 1500", op="attention", heads=16, kv_heads=8, dim=128, context=1500, tokens=1, cache="bf16", mask="chain"),
        # one token of a very long document
        dict(name="attention token int8 65537", op="attention", heads=32, kv_heads=8, dim=128, context=65537, tokens=1, cache="int8", mask="chain"),
        # an ordinary tree of drafts
        dict(name="attention tree 21 int8 6001", op="attention", heads=16, kv_heads=8, dim=128, context=6001, tokens=21, cache="int8", mask="tree"),
        # the largest tree over the longest context
        dict(name="attention tree 64 bf16 100003", op="attention", heads=32, kv_heads=8, dim=128, context=100003, tokens=64, cache="bf16", mask="tree"),
        # greedy check of a short chain
        dict(name="verify greedy 5", op="verify", vocab=32000, tokens=5, branch=1, temperature=0.0, logits="bf16", probs=False),
        # a sampled tree of a deterministic draft (its likeliest continuations)
        dict(name="verify tree 21", op="verify", vocab=50304, tokens=21, branch=3, temperature=0.7, logits="f32", probs=False),
        # the largest tree and vocabulary, children drawn from the draft's own probabilities
        dict(name="verify tree 64 with probabilities", op="verify", vocab=151936, tokens=64, branch=4, temperature=1.0, logits="bf16", probs=True),
        # the accepted path of a chain with a few side branches, 16 layers
        dict(name="keep 3 of 16", op="keep", layers=16, kv_heads=16, dim=128, context=700, tokens=16, kept=3),
        # the deepest path of the largest tree, 28 layers
        dict(name="keep 9 of 64", op="keep", layers=28, kv_heads=8, dim=128, context=4001, tokens=64, kept=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cache", "cache", "attention", "attention", "attention", "attention", "verify", "verify", "verify", "keep"])
    dim = rng.choice([64, 128])
    if op == "cache":
        tokens = rng.choice([1, _log(rng, 2, 4096)])
        return dict(op=op, kv_heads=rng.choice([1, 2, 4, 8, 16]), dim=dim, context=rng.choice([0, _log(rng, 1, 25000)]), tokens=tokens,
                    read=rng.choice(["new", "all"]), layout=rng.choice(["heads", "tokens"]))
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8] if kv_heads < 8 else [1, 2, 4])
        tokens = rng.choice([1, _log(rng, 2, 64)])
        return dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, context=0 if rng.random() < 0.05 else _log(rng, 1, 90000), tokens=tokens,
                    cache=rng.choice(["bf16", "int8"]), mask=rng.choice(["chain", "tree", "tree", "gaps"]))
    if op == "verify":
        tokens = _log(rng, 2, 64)
        return dict(op=op, vocab=_log(rng, 1000, 150000), tokens=tokens, branch=rng.choice([1, 2, 3, 4]), temperature=rng.choice([0.0, 0.6, 1.0, 1.3]),
                    logits=rng.choice(["bf16", "f32"]), probs=rng.random() < 0.5)
    tokens = _log(rng, 4, 64)
    return dict(op=op, layers=rng.randint(1, 28), kv_heads=rng.choice([1, 2, 4, 8]), dim=dim, context=_log(rng, 1, 4000), tokens=tokens,
                kept=rng.randint(1, max(1, tokens // 2)))


# ---- inputs -------------------------------------------------------------------------------------------------------------------

def _tree(rng, n, branch):
    """parents of n rows, row 0 the root: a row continues a recent one more often than an old one, up to `branch` children each."""
    parents, children = [-1], [0] * n
    for i in range(1, n):
        free = [j for j in range(i) if children[j] < branch]
        p = free[max(0, len(free) - 1 - int(rng.expovariate(0.6)))]
        parents.append(p)
        children[p] += 1
    return parents


def _mask(parents):
    """Bits of the rows that each row sees: its ancestors and itself."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return bits


def _signed(bits):
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def _quantized(x):
    """INT8 codes and float32 scale of every vector x [.., d]: s = amax / 127, code = rint(x (1 / s))."""
    x = x.float()
    amax = x.abs().amax(-1)
    s = amax / torch.full_like(amax, 127.0)
    inv = torch.where(s > 0, torch.ones_like(s) / s, torch.zeros_like(s))
    return torch.round(x * inv[..., None]).clamp(-127, 127).to(torch.int8), s


def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, op = case["tokens"], case["op"]

    def normal(*shape, std=1.0, dtype=F32):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def vectors(heads, rows, d):
        """Keys or values: channels of unequal size, as trained models have them."""
        return (normal(heads, rows, d) * torch.exp(0.4 * normal(heads, 1, d))).to(BF)

    if op == "cache":
        hk, d, T = case["kv_heads"], case["dim"], case["context"]
        cap = T + n + 37
        k, v = vectors(hk, n, d), vectors(hk, n, d)
        if case["layout"] == "tokens":      # [tokens, heads, d] in memory, as a projection leaves them
            k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
        cache = SimpleNamespace(offset=T, capacity=cap)
        for name in ("k", "v"):
            setattr(cache, name, torch.randint(-127, 128, (hk, cap, d), generator=g, device="cuda", dtype=torch.int8))
            setattr(cache, name + "s", torch.rand((hk, cap), generator=g, device="cuda") * 0.05)
        return dict(case=case, k=k, v=v, cache=cache)
    if op == "attention":
        H, hk, d, T = case["heads"], case["kv_heads"], case["dim"], case["context"]
        cap = T + n + 100
        k, v = vectors(hk, cap, d), vectors(hk, cap, d)
        q = normal(H, n, d, std=1.5, dtype=BF)
        if case["cache"] == "int8":
            (kc, ks), (vc, vs) = _quantized(k), _quantized(v)
            cache = SimpleNamespace(k=kc, ks=ks, v=vc, vs=vs, offset=T, capacity=cap)
        else:
            k[:, T + n:], v[:, T + n:] = float("nan"), float("nan")      # rows never written: whatever memory held
            cache = SimpleNamespace(k=k, v=v, offset=T, capacity=cap)
        mask = None
        if case["mask"] != "chain":
            bits = _mask(_tree(rng, n, 3))
            if case["mask"] == "gaps":       # rows that are not part of a tree: some see drafted rows anywhere, some none
                bits = [rng.getrandbits(n) if rng.random() < 0.8 else 0 for _ in range(n)]
            mask = torch.tensor(_signed(bits), dtype=torch.int64, device="cuda")
        return dict(case=case, q=q, cache=cache, mask=mask, scale=d ** -0.5)
    if op == "verify":
        V, branch = case["vocab"], case["branch"]
        parents = [-1] + list(range(n - 1)) if branch == 1 else _tree(rng, n, branch)
        # target and draft agree on what is likely, as a small model of the same family does
        common = normal(n, V, std=2.0) + 9.0 * (torch.rand((n, V), generator=g, device="cuda") < 8.0 / V)
        logits = (common + normal(n, V, std=0.5)).to(BF if case["logits"] == "bf16" else F32)
        draft = torch.softmax((common + normal(n, V, std=0.5)).double(), -1).float()
        up = torch.tensor([max(p, 0) for p in parents], device="cuda")
        rank = [sum(parents[j] == p for j in range(i)) for i, p in enumerate(parents)]
        if case["probs"]:                    # children drawn from the draft's probabilities, independently
            pick = torch.rand((n, 1), generator=g, device="cuda", dtype=F64)
            cdf = torch.cumsum(draft.double(), -1)[up]
            tokens = torch.searchsorted(cdf, pick * cdf[:, -1:]).clamp(max=V - 1).view(-1)
        else:                                # the draft's likeliest continuations
            top = torch.topk(draft, branch, -1).indices
            tokens = top[up, torch.tensor(rank, device="cuda")]
        above = torch.tensor([[b >> j & 1 > 0 for j in range(n)] for b in _mask(parents)], device="cuda")      # the tree, as its attention masks it
        return dict(case=case, above=above, logits=logits, tokens=tokens.contiguous(), parents=torch.tensor(parents, dtype=torch.int32, device="cuda"),
                    u=torch.rand(n, generator=g, device="cuda"), probs=draft if case["probs"] else None)
    hk, d, T, kept = case["kv_heads"], case["dim"], case["context"], case["kept"]
    caches = [SimpleNamespace(k=vectors(hk, T + n + 5, d), v=vectors(hk, T + n + 5, d), offset=T, capacity=T + n + 5) for _ in range(case["layers"])]
    path = [0] + sorted(rng.sample(range(kept, n), min(kept - 1, n - kept)))
    rows = torch.tensor(path + [-1] * (n - len(path)), dtype=torch.int32, device="cuda")
    return dict(case=case, caches=caches, rows=rows)


# ---- one pass -----------------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return {"cache": _run_cache, "attention": _run_attention, "verify": _run_verify, "keep": _run_keep}[case["op"]](state, case)


def _framework():
    import importlib
    return importlib.import_module("mxfp4-int8-m5_b200")


def _run_cache(s, case):
    c, k, v, n = s["cache"], s["k"], s["v"], case["tokens"]
    first = 0 if case["read"] == "all" else c.offset
    if own:
        P = _framework()
        P.sc_cache.kv_append(k, v, c)
        return P.sc_cache.kv_read(c, first, c.offset + n)
    for x, codes, scales in ((k, c.k, c.ks), (v, c.v, c.vs)):
        codes[:, c.offset:c.offset + n], scales[:, c.offset:c.offset + n] = _quantized(x)
    return tuple((codes[:, first:c.offset + n].float() * scales[:, first:c.offset + n, None]).to(BF) for codes, scales in ((c.k, c.ks), (c.v, c.vs)))


def _run_attention(s, case):
    q, c, mask = s["q"], s["cache"], s["mask"]
    if own:
        return _framework().sc_cache.cache_attention(q, c, s["scale"], mask)
    H, n, d = q.shape
    hk, T = c.k.shape[0], c.offset
    k, v = c.k[:, :T + n].float(), c.v[:, :T + n].float()
    if case["cache"] == "int8":
        k, v = k * c.ks[:, :T + n, None], v * c.vs[:, :T + n, None]
    scores = torch.matmul(q.float().view(hk, H // hk * n, d), k.transpose(1, 2)).mul_(s["scale"]).view(hk, H // hk, n, T + n)
    i = torch.arange(n, device=q.device)
    seen = i[None, :] <= i[:, None] if mask is None else (mask[:, None] >> i[None, :] & 1) > 0
    scores[..., T:].masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(hk, H // hk * n, T + n), v).view(hk, H // hk, n, d) / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(2, 0, 1, 3).reshape(n, H * d).to(BF)


def _run_verify(s, case):
    logits, tokens, parents, u, probs = s["logits"], s["tokens"], s["parents"], s["u"], s["probs"]
    if own:
        return tuple(_framework().sc_draft.verify_draft(logits, tokens, parents, u, case["temperature"], probs))
    n, V = logits.shape
    at = torch.arange(n, device=u.device)
    up = parents.long()
    if case["temperature"] == 0.0:
        best = logits.argmax(-1)
        taken = torch.where(up >= 0, tokens == best[up.clamp(min=0)], up < 0)
        same = (up[:, None] == up[None, :]) & taken[None, :] & (at[None, :] < at[:, None])
        taken &= ~same.any(-1)               # the first of equal siblings
        p = None
    else:
        x = logits.double() / case["temperature"]
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        q = None if probs is None else probs.double()
        rank = ((up[:, None] == up[None, :]) & (at[None, :] < at[:, None])).sum(-1)
        taken, done = up < 0, torch.zeros(n, dtype=torch.bool, device=u.device)
        for r in range(case["branch"]):      # all nodes' r-th children at a time: a child is tested on what its siblings left
            child = torch.full((n + 1,), -1, dtype=torch.long, device=u.device)
            child[torch.where((rank == r) & (up >= 0), up, n)] = at
            child = child[:n]
            tested = (child >= 0) & ~done
            c = child.clamp(min=0)
            token = tokens[c][:, None]
            proposed = torch.ones(n, dtype=F64, device=u.device) if q is None else q.gather(1, token)[:, 0]
            yes = tested & (u[c].double() * proposed < p.gather(1, token)[:, 0])
            taken[torch.where(yes, c, torch.zeros_like(c))] = True
            done |= yes
            left = p.scatter(1, token, 0.0) if q is None else (p - q).clamp(min=0.0)
            z = left.sum(-1, keepdim=True)
            p = torch.where((tested & ~yes)[:, None] & (z > 0), left / z, p)
    # on the path: a row whose ancestors and itself are all taken
    path = ~(s["above"] & ~taken[None, :]).any(-1)
    count = path.sum().to(torch.int32).view(1)
    rows = torch.sort(torch.where(path, at, at + n)).values
    last = rows.gather(0, count.long() - 1)
    rows = torch.where(rows < n, rows, torch.full_like(rows, -1)).to(torch.int32)
    if p is None:
        return rows, count, best.gather(0, last)
    cdf = torch.cumsum(p.index_select(0, last)[0], 0)
    token = (cdf <= u[0].double() * cdf[-1]).sum().clamp(max=V - 1).view(1)
    return rows, count, token


def _run_keep(s, case):
    T, n = case["context"], case["tokens"]
    if own:
        _framework().sc_cache.kv_keep(s["caches"], s["rows"], T)
    else:
        rows = s["rows"].long()
        at = torch.arange(n, device=rows.device)
        source = T + torch.where(rows >= 0, rows, at)
        for c in s["caches"]:
            for x in (c.k, c.v):
                x[:, T:T + n] = x.index_select(1, source)
    return [x[:, T:T + n] for c in s["caches"] for x in (c.k, c.v)]


# ---- the least work of a pass -------------------------------------------------------------------------------------------------

def work(case):
    n = case["tokens"]
    if case["op"] == "cache":
        hk, d, T = case["kv_heads"], case["dim"], case["context"]
        old = T if case["read"] == "all" else 0       # new rows are in hand when they are read back
        return {"bytes": 2 * hk * (2 * n * d + n * (d + 4) + old * (d + 4) + (old + n) * 2 * d), "flops": 4 * hk * (old + 2 * n) * d}
    if case["op"] == "attention":
        H, hk, d, T = case["heads"], case["kv_heads"], case["dim"], case["context"]
        row = 2 * d if case["cache"] == "bf16" else d + 4
        return {"bytes": 2 * hk * (T + n) * row + 4 * H * n * d + 8 * n, "flops": 4 * H * n * (T + n) * d}
    if case["op"] == "verify":
        V = case["vocab"]
        e = 2 if case["logits"] == "bf16" else 4
        return {"bytes": n * V * (e + (4 if case["probs"] else 0)), "flops": n * V * (1 if case["temperature"] == 0.0 else 6 if case["probs"] else 4)}
    return {"bytes": case["layers"] * 2 * case["kv_heads"] * 2 * case["kept"] * case["dim"] * 2, "flops": 0}


# ---- the operators in float64 -------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cache":
        c, n = s["cache"], case["tokens"]
        out = []
        for x, codes, scales in ((s["k"], c.k, c.ks), (s["v"], c.v, c.vs)):
            x = x.to(F64)
            step = x.abs().max(dim=2, keepdim=True).values / 127
            new = torch.where(step > 0, torch.round(x / torch.where(step > 0, step, 1.0)) * step, 0.0)
            old = codes[:, :c.offset].to(F64) * scales[:, :c.offset].to(F64).unsqueeze(2)
            out.append(torch.cat([old, new], 1) if case["read"] == "all" else new)
        return tuple(out)
    if case["op"] == "attention":
        q, c, mask = s["q"].to(F64), s["cache"], s["mask"]
        H, n, d = q.shape
        T, group = c.offset, H // c.k.shape[0]
        bits = [(1 << i + 1) - 1 for i in range(n)] if mask is None else mask.tolist()
        hidden = torch.tensor([[not b >> j & 1 for j in range(n)] for b in bits], device="cuda")
        out = torch.zeros((n, H, d), dtype=F64, device="cuda")
        for h in range(H):
            key, value = c.k[h // group, :T + n].to(F64), c.v[h // group, :T + n].to(F64)
            if case["cache"] == "int8":
                key, value = key * c.ks[h // group, :T + n, None].to(F64), value * c.vs[h // group, :T + n, None].to(F64)
            a = q[h] @ key.T * s["scale"]
            a[:, T:] = a[:, T:].masked_fill(hidden, -math.inf)
            out[:, h] = torch.nan_to_num(torch.softmax(a, 1), nan=0.0) @ value
        return out.reshape(n, H * d)
    if case["op"] == "verify":
        logits, tokens, parents, u = s["logits"].to(F64), s["tokens"].tolist(), s["parents"].tolist(), s["u"].tolist()
        n, V = logits.shape
        temp = case["temperature"]
        node, rows = 0, [0]
        p = torch.softmax(logits[0] / temp, 0) if temp else None
        for c in range(1, n):                # ascending rows: a row's children and later siblings come after it
            if parents[c] != node:
                continue
            x = tokens[c]
            if temp == 0.0:
                good = x == int(logits[node].argmax())
            else:
                good = u[c] * (float(s["probs"][node, x]) if case["probs"] else 1.0) < float(p[x])
            if good:
                node = c
                rows.append(c)
                p = torch.softmax(logits[c] / temp, 0) if temp else None
            elif temp:
                if case["probs"]:
                    left = torch.relu(p - s["probs"][node].to(F64))
                else:
                    left = p.clone()
                    left[x] = 0.0
                p = left / left.sum() if float(left.sum()) > 0 else p
        if temp == 0.0:
            token = int(logits[node].argmax())
        else:
            cdf = torch.cumsum(p, 0)
            token = min(V - 1, int(torch.searchsorted(cdf, cdf[-1] * u[0], right=True)))
        return (torch.tensor(rows + [-1] * (n - len(rows)), dtype=torch.int32, device="cuda"), torch.tensor([len(rows)], dtype=torch.int32, device="cuda"),
                torch.tensor([token], dtype=torch.int64, device="cuda"))
    T, n = case["context"], case["tokens"]
    rows = [r for r in s["rows"].tolist() if r >= 0]
    out = []
    for c in s["caches"]:
        for x in (c.k, c.v):
            y = x[:, T:T + n].to(F64)
            out.append(torch.cat([y[:, rows], y[:, len(rows):]], 1))
    return out

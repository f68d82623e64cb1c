"""GPU: INT8 caches and draft trees through the W4A8 decoders: the fused write against its two steps, rows of a tree against the same tokens one after the other,
speculative generation against the model's own choices, the engine."""
import importlib
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def mod(scmx, n):
    return importlib.import_module(scmx.__name__ + "." + n)


# ---- keys and values into an INT8 cache ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("full,acc", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (8, 2, 128), (3, 1, 256), (4, 4, 128), (4, 2, 32)])
@pytest.mark.parametrize("L", [1, 7, 130])
def test_fused_write_equals_its_steps(scmx, full, acc, hq, hk, d, L):
    S, HM, C = scmx.sc_kernels, scmx.host_model, scmx.sc_cache
    if full:
        hk = hq
    g = torch.Generator(device="cuda").manual_seed(L + d)
    ntot = (hq + 2 * hk) * d
    if acc:
        src = torch.randint(-200000, 200000, (L, ntot), generator=g, device="cuda", dtype=torch.int32)
        xs, ws = torch.rand(L, generator=g, device="cuda") * 1e-3 + 1e-4, torch.rand(ntot, generator=g, device="cuda") * 1e-2 + 1e-3
    else:
        src, xs, ws = (torch.randn((L, ntot), generator=g, device="cuda") * 3).to(BF), None, None
    if not acc:
        src[0, -d:] = 0.0                            # a value of zeros
        src[L // 2, (hq + hk) * d + 1] = float("nan")
    qn, kn = ((1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(BF) for n in ((hq * d, hk * d) if full else (d, d)))
    inv, off = S.rope_inv_freq(d, 1e4), 5
    rope = (inv, off, S.rope_table(inv, 64))
    rows = torch.randint(0, 9, (L,), generator=g, device="cuda", dtype=torch.int32)
    for row_pos in (None, rows):
        got, want = HM.QuantKVCache(hk, d, L + 9), HM.QuantKVCache(hk, d, L + 9)
        for c in (got, want):
            for t in (c.k, c.v, c.ks, c.vs):
                t.fill_(3)
            c.offset = off
        q, k, v = S._qkv_norm(src, xs, ws, qn, kn, 1e-6, L, hq, hk, d, full, rope, got, None, row_pos)
        assert k is None and v is None
        q2, k2, v2 = S._qkv_norm(src, xs, ws, qn, kn, 1e-6, L, hq, hk, d, full, rope, None, None, row_pos)
        C.kv_append(k2, v2, want)
        assert torch.equal(q, q2) and torch.equal(got.k, want.k) and torch.equal(got.v, want.v) and torch.equal(got.ks, want.ks)
        assert torch.equal(got.vs.isnan(), want.vs.isnan()) and torch.equal(got.vs.nan_to_num(), want.vs.nan_to_num())
        if d >= 64:                                  # the position on the device
            dev = HM.QuantKVCache(hk, d, L + 9)
            for t in (dev.k, dev.v, dev.ks, dev.vs):
                t.fill_(3)
            q3, _, _ = S._qkv_norm(src, xs, ws, qn, kn, 1e-6, L, hq, hk, d, full, (inv, 0, rope[2]), dev, torch.tensor([off], dtype=torch.int32, device="cuda"), row_pos)
            assert torch.equal(q3, q) and torch.equal(dev.k, want.k) and torch.equal(dev.v, want.v) and torch.equal(dev.ks, want.ks)


@pytest.mark.parametrize("full", [False, True])
@pytest.mark.parametrize("d,quant", [(32, False), (64, False), (64, True), (128, False), (128, True)])
def test_rows_outside_the_cache_are_dropped(scmx, full, d, quant):
    """A position on the device before the cache's first row or past its last: rows inside are written, nothing else is, and queries are as ever.  The caches are cut
    out of the middle of larger buffers."""
    S, hq, hk, L, cap = scmx.sc_kernels, 4, 4, 5, 8
    g = torch.Generator(device="cuda").manual_seed(d)
    y = torch.randn((L, (hq + 2 * hk) * d), generator=g, device="cuda").to(BF)
    qn, kn = (torch.ones(hq * d if full else d, dtype=BF, device="cuda") for _ in range(2))
    inv = S.rope_inv_freq(d, 1e4)

    def cache():
        c, whole = scmx.host_model.KVCache(hk, d, 1), []
        for name, shape, dt in (("k", (hk, cap, d), torch.int8 if quant else BF), ("v", (hk, cap, d), torch.int8 if quant else BF)) + (
                (("ks", (hk, cap), torch.float32), ("vs", (hk, cap), torch.float32)) if quant else ()):
            n = hk * cap * (d if len(shape) == 3 else 1)
            whole.append(torch.full((3 * n,), 3, dtype=dt, device="cuda"))
            setattr(c, name, whole[-1][n:2 * n].view(shape))
        return c, whole
    for at in (0, 3, 4, 6, 8, 9, -1, -4, -5, -8, 2 ** 31 - 1, -2 ** 31):
        c, whole = cache()
        q, _, _ = S._qkv_norm(y, None, None, qn, kn, 1e-6, L, hq, hk, d, full, (inv, 0), c, torch.tensor([at], dtype=torch.int32, device="cuda"))
        assert torch.isfinite(q).all()
        alone = scmx.host_model.KVCache(hk, d, L)
        q0, k, v = S._qkv_norm(y, None, None, qn, kn, 1e-6, L, hq, hk, d, full, (inv, 0), alone)
        inside = [i for i in range(L) if 0 <= at + i < cap]
        want, whole2 = cache()
        if inside and quant:                         # values do not turn: they tell which rows were written
            want.offset = at + inside[0]
            scmx.sc_cache.kv_append(k[:, inside], v[:, inside], want)
        elif inside:
            want.v[:, at + inside[0]:at + inside[0] + len(inside)] = v[:, inside]
        assert torch.equal(c.v, want.v) and (not quant or torch.equal(c.vs, want.vs))
        rows = [at + i for i in inside]
        rest = [r for r in range(cap) if r not in rows]
        assert (c.k[:, rest] == 3).all() and (not quant or (c.ks[:, rest] == 3).all())
        for t in whole:                              # in front of the cache and behind it
            n = t.numel() // 3
            assert (t[:n] == 3).all() and (t[2 * n:] == 3).all()


def test_rows_turn_where_they_are_told(scmx):
    """row_pos 0 .. L - 1 is no row_pos; the same position for all rows turns them alike."""
    S, HM = scmx.sc_kernels, scmx.host_model
    g = torch.Generator(device="cuda").manual_seed(1)
    y = torch.randn((6, 4 * 128), generator=g, device="cuda").to(BF)
    w, inv = torch.ones(128, dtype=BF, device="cuda"), S.rope_inv_freq(128, 1e4)
    for table in ((), (S.rope_table(inv, 8),)):      # from the table, and beyond its end
        a, b = HM.KVCache(1, 128, 40), HM.KVCache(1, 128, 40)
        a.offset = b.offset = 3
        want = S.qkv_headnorm_y(y, w, w, 1e-6, 6, 2, 1, 128, rope=(inv, 3, *table), cache=a)
        got = S.qkv_headnorm_y(y, w, w, 1e-6, 6, 2, 1, 128, rope=(inv, 3, *table), cache=b, row_pos=torch.arange(6, dtype=torch.int32, device="cuda"))
        assert all(torch.equal(x[:, -6:], z[:, -6:]) for x, z in zip(got, want))
        same = S.qkv_headnorm_y(y[:1].expand(6, -1).contiguous(), w, w, 1e-6, 6, 2, 1, 128, rope=(inv, 3, *table), cache=b,
                                row_pos=torch.full((6,), 4, dtype=torch.int32, device="cuda"))
        assert all(torch.equal(same[0][:, i], same[0][:, 0]) for i in range(6))


# ---- whole models -------------------------------------------------------------------------------------------------------------

def build(scmx, kind, seed=3, **kw):
    HM = scmx.host_model
    if kind == "qwen3":
        FQ = mod(scmx, "fused_qwen3")
        model = HM.CausalLM(HM.ModelArgs(1024, 2048, 2, 8, 2, 128, 1e-6, 1e6, 512, True)).init_random(seed, 0.05).cuda()
        fused = FQ.FusedQwen3(model, FQ.pack_model(model, on_device=True), **kw)
        return fused, mod(scmx, "decode").DecodeQwen3(fused) if fused.epilogue == "gemm" else None
    FO = mod(scmx, "fused_olmoe")
    model = HM.CausalLM(HM.ModelArgs(512, 256, 2, 4, 4, 128, 1e-5, 1e4, 512, False, 8, 2, False, "olmoe")).init_random(seed, 0.05).cuda()
    fused = FO.FusedOlmoe(model, FO.pack_olmoe(model, on_device=True))
    return fused, mod(scmx, "decode").DecodeOlmoe(fused)


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("kind,kw", [("qwen3", {}), ("qwen3", dict(epilogue="row")), ("qwen3", dict(resident=True)), ("qwen3", dict(fuse_rope=False)), ("olmoe", {})])
@pytest.mark.parametrize("dtype", [None, torch.int8])
def test_rows_of_a_tree_are_their_paths(scmx, kind, kw, dtype):
    """Every row's logits are those of its path read as a prompt: the rows quantize alike, attention differs by roundings of its weights (2^-8 a weight, averaged
    over positions and layers, and the INT8 codes that they turn: a few percent of a logit at the most)."""
    fused, _ = build(scmx, kind, **kw)
    D = scmx.sc_draft
    rng = random.Random(5)
    prompt = torch.tensor([[rng.randrange(512) for _ in range(45)]], device="cuda")
    tree = D.DraftTree([-1, 0, 0, 1, 1, 3, 2, 6, 7])
    tokens = [rng.randrange(512) for _ in range(len(tree))]
    cache = fused.make_cache(80, dtype)
    fused.hidden(prompt, cache)
    got = fused.logits(fused.hidden(torch.tensor([tokens], device="cuda"), cache, tree))[0]
    assert all(c.offset == 45 for c in cache)
    for i in (0, 2, 5, 8):
        path, j = [], i
        while j >= 0:
            path.insert(0, tokens[j])
            j = tree.list[j]
        other = fused.make_cache(80, dtype)
        fused.hidden(prompt, other)
        want = fused.logits(fused.hidden(torch.tensor([path], device="cuda"), other))[0, -1]
        assert rel(got[i], want) < 0.05, (i, rel(got[i], want))
    scmx._lib.check_status()


@pytest.mark.parametrize("kind,kw", [("qwen3", {}), ("qwen3", dict(resident=True)), ("qwen3", dict(resident=True, epilogue="row")), ("olmoe", {})])
def test_a_prompt_beside_a_drafted_pass(scmx, kind, kw, monkeypatch):
    """A tree belongs to the call that was given it: a prompt and other trees that are read while a pass over a tree is under way, as from another thread, are
    what they are alone, and so is the pass.  (Models without buffers of weights, which take one pass at a time.)"""
    fused, _ = build(scmx, kind, **kw)
    C, D = scmx.sc_cache, scmx.sc_draft
    ids = torch.randint(0, 512, (1, 7), generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
    trees = [None, D.DraftTree([-1] + [0] * 6), D.DraftTree(list(range(-1, 6)))]

    def read(tree):
        cache = fused.make_cache(40)
        h = fused.hidden(ids, cache, tree)
        return h, cache[0].offset, cache[1].k[:, :7].clone()
    alone = [read(tree) for tree in trees]
    assert [offset for _, offset, _ in alone] == [7, 0, 0] and not torch.equal(alone[1][0], alone[2][0])
    inside, real, started = [], C.cache_attention, []

    def attention(*args, **kw):
        if not started:
            started.append(1)
            inside.extend(read(tree) for tree in trees)
        return real(*args, **kw)
    monkeypatch.setattr(C, "cache_attention", attention)
    for i in (1, 2):
        started.clear()
        inside.clear()
        outer = read(trees[i])
        assert len(inside) == 3
        for got, want in zip([outer] + inside, [alone[i]] + alone):
            assert torch.equal(got[0], want[0]) and got[1] == want[1] and torch.equal(got[2], want[2])


@pytest.mark.parametrize("kind", ["qwen3", "olmoe"])
def test_int8_cache_steps(scmx, kind):
    """Steps on an INT8 cache: near the bfloat16 cache's (a code is off by at most 1 / 254 of its vector's largest value), and the captured ones the same as the others."""
    fused, decoder = build(scmx, kind)
    ids = torch.randint(0, 512, (1, 60), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    plain, quant, again = fused.make_cache(100), fused.make_cache(100, torch.int8), fused.make_cache(100, torch.int8)
    a, b = (fused.logits(fused.hidden(ids, c)[:, -1:]) for c in (plain, quant))
    fused.hidden(ids, again)
    assert rel(b, a) < 0.1
    tok = a[:, -1].argmax(-1, keepdim=True)
    x, y = decoder.step(tok, plain), decoder.step(tok, quant)
    assert rel(y, x) < 0.1 and quant[0].offset == 61
    quant[0].offset, quant[1].offset = 60, 60
    steps, t = [], tok
    for _ in range(12):
        t = decoder.step(t, quant)[:, -1].argmax(-1, keepdim=True)
        steps.append(int(t))
    assert decoder.generate(tok, again, 12).tolist() == steps and again[0].offset == 72
    assert torch.equal(again[1].k[:, :72], quant[1].k[:, :72]) and torch.equal(again[1].vs[:, :72], quant[1].vs[:, :72])
    decoder.check_status() if kind == "qwen3" else None
    scmx._lib.check_status()


# Most that a chosen token's logit may be below the largest, in units of the logits' spread.  The rows' logits are within 0.05 of the spread of the prompt's (the
# bound of test_rows_of_a_tree_are_their_paths, a root mean square); of some 10^4 nearly normal errors the largest is 4 such units, and a choice is
# turned by two errors, its own and the largest logit's: 2 * 4 * 0.05.  A token that is not the model's is about 3 below.
MARGIN = 0.4


def margins(fused, prompt, tokens, dtype):
    """How far the model's logit of each generated token is below its largest, reading them as one prompt; in units of the logits' spread."""
    cache = fused.make_cache(len(prompt) + len(tokens) + 1, dtype)
    logits = fused.logits(fused.hidden(torch.tensor([prompt + tokens], device="cuda"), cache))[0, len(prompt) - 1:-1].double()
    return ((logits.amax(-1) - logits.gather(1, torch.tensor(tokens, device="cuda")[:, None])[:, 0]) / logits.std(-1)).max().item()


@pytest.mark.parametrize("kind", ["qwen3", "olmoe"])
@pytest.mark.parametrize("dtype", [None, torch.int8])
def test_drafted_generation_is_the_models(scmx, kind, dtype):
    """Greedy generation with drafts: every token is the model's own choice (its logit among the largest, up to what roundings turn), whatever is drafted; a draft that
    knows the continuation is accepted whole."""
    fused, decoder = build(scmx, kind)
    DEC = mod(scmx, "decode")
    rng = random.Random(1)
    prompt = [rng.randrange(512) for _ in range(12)] * 3
    known = []

    def oracle_draft(text, most):
        """A wrong row beside the right ones."""
        chain = [text[-1]] + known[len(text) - len(prompt):][:min(most, 7) - 1]
        if len(chain) + 1 <= most and len(chain) > 1:
            return chain + [(chain[1] + 1) % 512], list(range(-1, len(chain) - 1)) + [0]
        return chain, list(range(-1, len(chain) - 1))

    def run(propose, n=24):
        cache = fused.make_cache(len(prompt) + n, dtype)                # no room behind the last token
        first = int(fused.logits(fused.hidden(torch.tensor([prompt], device="cuda"), cache)[:, -1:]).argmax())
        passes = []
        d = DEC.DecodeDraft(fused, lambda text, most: (passes.append(1), propose(text, most))[1])
        out = d.generate(torch.tensor([[first]], device="cuda"), cache, n, prompt).tolist()
        assert cache[0].offset == len(prompt) + n and len(out) == n
        return [first] + out, len(passes)
    text, passes = run(lambda text, most: ([text[-1]], [-1]))            # nothing drafted: a token a pass
    assert passes == 24 and margins(fused, prompt, text, dtype) < MARGIN
    known[:] = text
    again, passes = run(oracle_draft)
    assert margins(fused, prompt, again, dtype) < MARGIN
    if again == text:
        assert passes <= 6                                               # 24 tokens, 7 at a time
    looked, passes = run(DEC.LookupDraft())
    assert margins(fused, prompt, looked, dtype) < MARGIN and passes <= 24
    wild, _ = run(lambda text, most: ([text[-1]] + [rng.randrange(512) for _ in range(min(most, 9) - 1)], [-1] + [0] * (min(most, 9) - 1)))
    assert margins(fused, prompt, wild, dtype) < MARGIN
    scmx._lib.check_status()


@pytest.mark.parametrize("kind", ["qwen3", "olmoe"])
@pytest.mark.parametrize("dtype", [None, torch.int8])
def test_lookup_of_a_known_continuation(scmx, kind, dtype):
    """A text that has the continuation in it: LookupDraft proposes it, and tokens of it are accepted: a pass adds one token and the accepted ones, so as many passes as
    tokens would mean that none was.  (How many are depends on choices that roundings turn: the prompt repeats a token, and a random model has near ties there.)"""
    fused, _ = build(scmx, kind)
    DEC = mod(scmx, "decode")
    prompt = [474] * 30

    def run(propose, before):
        cache, passes = fused.make_cache(len(prompt) + 24, dtype), []
        first = int(fused.logits(fused.hidden(torch.tensor([prompt], device="cuda"), cache)[:, -1:]).argmax())
        d = DEC.DecodeDraft(fused, lambda text, most: (passes.append(1), propose(text, most))[1])
        return [first] + d.generate(torch.tensor([[first]], device="cuda"), cache, 24, before + prompt).tolist(), len(passes)
    text, passes = run(lambda text, most: ([text[-1]], [-1]), [])
    assert passes == 24
    again, passes = run(DEC.LookupDraft(), prompt + text)
    assert margins(fused, prompt, again, dtype) < MARGIN and passes < 24


@pytest.mark.parametrize("kind", ["qwen3", "olmoe"])
@pytest.mark.parametrize("dtype", [None, torch.int8])
def test_replayed_passes(scmx, kind, dtype):
    """Passes of as many rows are replays from the second one on.  Trees, tokens and positions change between them: the rows that stay in the first layer's cache, which
    no attention has touched, are those of a pass launch by launch, and every token is the model's choice."""
    fused, _ = build(scmx, kind)
    DEC = mod(scmx, "decode")
    rng = random.Random(3)
    prompt = [rng.randrange(512) for _ in range(30)]
    caches = [fused.make_cache(110, dtype) for _ in range(2)]
    for c in caches:
        fused.hidden(torch.tensor([prompt], device="cuda"), c)
    drawn = {}

    def propose(text, most):
        if len(text) not in drawn:
            n = min(most, rng.choice([1, 6, 6, 6, 17]))
            drawn[len(text)] = [text[-1]] + [rng.randrange(512) for _ in range(n - 1)], [-1] + [rng.randrange(i) for i in range(1, n)]
        return drawn[len(text)]
    d, plain = DEC.DecodeDraft(fused, propose), DEC.DecodeDraft(fused, propose)
    plain._captured = lambda *a: None
    text, out = prompt + [7], []
    tensors = lambda c: (c.k, c.v) + ((c.ks, c.vs) if dtype else ())      # noqa: E731
    layer = lambda c, n: [t[:, :n] for t in tensors(c[0])]                # noqa: E731
    while len(text) < 80:
        new = d.step(text, caches[0])
        plain.step(text, caches[1])
        n = len(text)
        assert all(torch.equal(x, y) for x, y in zip(layer(caches[0], n), layer(caches[1], n)))
        text, out = text + new, out + new
        for x, y in zip(*caches):                                 # the same text whatever rounding chose
            for a, b in zip(tensors(x), tensors(y)):
                b.copy_(a)
            y.offset = x.offset
    replayed = [k for k, g in d._graphs[2].items() if g is not None]
    assert (6, 0.0) in replayed and caches[0][0].offset == len(text) - 1
    assert margins(fused, prompt + [7], out, dtype) < MARGIN
    # the end of the cache, another cache, and a draft of too many rows
    rest = d.generate(torch.tensor([[text[-1]]], device="cuda"), caches[0], 110 - caches[0][0].offset, text[:-1])
    assert caches[0][0].offset == 110 and rest.numel() == 110 - len(text) + 1
    with pytest.raises(AssertionError, match="capacity"):
        d.step(text + rest.tolist(), caches[0])
    for c in caches[1]:
        c.offset = len(prompt)
    drawn.clear()
    again = d.generate(torch.tensor([[7]], device="cuda"), caches[1], 20, prompt).tolist()
    assert margins(fused, prompt + [7], again, dtype) < MARGIN
    wide = DEC.DecodeDraft(fused, lambda t, most: ([t[-1]] * (most + 1), [-1] + [0] * most))
    with pytest.raises(ValueError, match="draft"):
        wide.step([1, 2], caches[1])
    scmx._lib.check_status()


def test_sampled_generation_repeats_with_its_generator(scmx):
    fused, _ = build(scmx, "qwen3")
    DEC = mod(scmx, "decode")
    prompt = list(range(5, 25)) * 2
    out = []
    for _ in range(2):
        cache = fused.make_cache(100, torch.int8)
        fused.hidden(torch.tensor([prompt], device="cuda"), cache)
        out.append(DEC.DecodeDraft(fused).generate(torch.tensor([[7]], device="cuda"), cache, 20, prompt, 0.8, torch.Generator(device="cuda").manual_seed(4)).tolist())
    assert out[0] == out[1] and all(0 <= t < 512 for t in out[0])


@pytest.mark.parametrize("dtype", [None, torch.int8])
def test_replays_follow_the_caches_tensors(scmx, dtype):
    """After captured passes a layer's tensors are replaced, then the layer in the list, then the whole list by one of the same layers: passes write to what the cache holds now and to
    nothing else.  (Everything replaced stays alive here.)"""
    fused, _ = build(scmx, "qwen3")
    HM, d = scmx.host_model, mod(scmx, "decode").DecodeDraft(fused, lambda text, most: ([text[-1], 3, 5], [-1, 0, 0]))
    cache, text = fused.make_cache(80, dtype), list(range(20))
    names = ("k", "v", "ks", "vs") if dtype else ("k", "v")
    for c in cache:
        for name in names:
            getattr(c, name).zero_()
    fused.hidden(torch.tensor([text], device="cuda"), cache)
    text.append(7)
    for _ in range(3):
        text += d.step(text, cache)
    captured = d._graphs[2][3, 0.0]
    assert captured is not None
    old = []

    def check(c):
        """Two passes (launched, captured) and a replay: the old tensors stay as they are, the new ones have the rows."""
        first = c[1].offset
        before = [t.clone() for t in old]
        for _ in range(3):
            for name in names:
                getattr(c[1], name)[:, c[1].offset:].zero_()
            text.extend(d.step(text, c))
        assert all(torch.equal(a, b) for a, b in zip(before, old))
        assert all((getattr(c[1], name)[:, first:c[1].offset] != 0).any(-1).all() for name in ("k", "v"))
    for name in names:                               # a layer's tensors
        old.append(getattr(cache[1], name))
        setattr(cache[1], name, old[-1].clone())
    check(cache)
    assert d._graphs[2][3, 0.0] is not captured
    layer = type(cache[1])(cache[1].k.shape[0], cache[1].k.shape[2], 80)      # the layer
    for name in names:
        old.append(getattr(cache[1], name))
        getattr(layer, name).copy_(old[-1])
    layer.offset, cache[1] = cache[1].offset, layer
    check(cache)
    captured = d._graphs[2][3, 0.0]
    check(list(cache))                               # the list alone: the same cache
    assert d._graphs[2][3, 0.0] is captured
    scmx._lib.check_status()


def test_caches_that_take_turns_keep_their_passes(scmx):
    """Two texts in turn through one DecodeDraft: each cache's pass is captured once and replayed, with the tokens that each text gets alone; a cache that is given up is not
    kept alive, and the least recently read of many gives its passes up."""
    import gc
    import weakref
    fused, _ = build(scmx, "qwen3")
    DEC = mod(scmx, "decode")
    propose = lambda text, most: ([text[-1], 3, 5], [-1, 0, 0])      # noqa: E731
    prompts = [list(range(20)), list(range(100, 130))]

    def start(prompt):
        cache = fused.make_cache(80)
        fused.hidden(torch.tensor([prompt], device="cuda"), cache)
        return cache
    want = []
    for prompt in prompts:
        alone, cache, text = DEC.DecodeDraft(fused, propose), start(prompt), prompt + [7]
        for _ in range(6):
            text += alone.step(text, cache)
        want.append(text)
    d, caches, texts, captured = DEC.DecodeDraft(fused, propose), [start(p) for p in prompts], [p + [7] for p in prompts], [[], []]
    for _ in range(6):
        for i in (0, 1):
            texts[i] += d.step(texts[i], caches[i])
            captured[i].append(d._graphs[2][3, 0.0])
    assert texts == want
    for seen in captured:
        assert seen[0] is None and seen[1] is not None and all(x is seen[1] for x in seen[1:])
    layer = weakref.ref(caches[0][0])
    caches[0] = None
    gc.collect()
    assert layer() is None
    d.step(texts[1], caches[1])
    assert len(d._kept) == 1
    more = [start(prompts[0]) for _ in range(d.CACHES)]
    for cache in more:
        d.step(prompts[0] + [7], cache)
    assert len(d._kept) == d.CACHES and all(e[0][0]() is c[0] for e, c in zip(d._kept, more))
    scmx._lib.check_status()


def test_replayed_passes_refuse_what_the_first_refuses(scmx):
    """Random numbers of another type or place, at a pass launch by launch, at the one that is captured and at a replay."""
    fused, _ = build(scmx, "qwen3")
    d = mod(scmx, "decode").DecodeDraft(fused, lambda text, most: ([text[-1], 3], [-1, 0]))
    cache, text = fused.make_cache(60), list(range(20))
    fused.hidden(torch.tensor([text], device="cuda"), cache)
    text.append(7)
    for _ in range(4):
        good = torch.rand(64, device="cuda")
        for u in (good.cpu(), good.double(), good.to(BF)):
            with pytest.raises(TypeError, match="random numbers"):
                d.step(text, cache, 0.8, u)
        text += d.step(text, cache, 0.8, good)
    assert d._graphs[2][2, 0.8] is not None
    scmx._lib.check_status()


def test_engine_with_drafts(scmx):
    fused, decoder = build(scmx, "qwen3")
    R, E, DEC = mod(scmx, "registry"), mod(scmx, "engine"), mod(scmx, "decode")
    bundle = R.Bundle("qwen3", fused, decoder, 512, scmx._lib.check_status)
    prompt = list(range(40, 70)) * 2
    for dtype in (None, torch.int8):
        engine = E.Engine(bundle, 128, cache_dtype=dtype)
        plain = engine.generate(prompt, 20)
        drafted = engine.generate(prompt, 20, draft=DEC.LookupDraft())
        assert len(plain) == len(drafted) == 20 and not engine.live
        assert engine.pool.free[0][0].k.dtype == (torch.int8 if dtype else BF)
        for text in (plain, drafted):
            assert margins(fused, prompt, text, dtype) < MARGIN
    bundle.check_status()

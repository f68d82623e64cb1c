"""CPU: refusals of the cache and draft calls, before anything is launched, and the host side of draft trees."""
import ctypes
from types import SimpleNamespace

import pytest
import torch


def test_trees(scmx):
    D = scmx.sc_draft
    parents = [-1, 0, 0, 1, 3, 2]
    assert D.draft_mask(parents, device="cpu").tolist() == [1, 3, 5, 11, 27, 37]
    assert D.draft_depths(parents) == [0, 1, 1, 2, 3, 2]
    chain = D.draft_mask([-1] + list(range(63)), device="cpu")
    assert chain[62].item() == 2 ** 63 - 1 and chain[63].item() == -1          # all 64 bits
    for bad in ([], [0], [-1, 1], [-1, -1], [-1, 0, 5], [-1] + [0] * 64):
        with pytest.raises(ValueError):
            D.check_tree(bad)


def test_cpu_tensors_are_refused(scmx):
    C, D = scmx.sc_cache, scmx.sc_draft
    c = scmx.host_model.QuantKVCache(2, 64, 16, device="cpu")
    k = torch.zeros((2, 3, 64), dtype=torch.bfloat16)
    for call in (lambda: C.kv_append(k, k, c), lambda: C.kv_read(c, 0, 2), lambda: C.cache_attention(k, c, 1.0),
                 lambda: C.kv_keep([c], torch.zeros(3, dtype=torch.int32)), lambda: c.update_and_fetch(k, k),
                 lambda: D.verify_draft(torch.zeros(3, 9), torch.zeros(3, dtype=torch.long), torch.zeros(3, dtype=torch.int32), torch.zeros(3))):
        with pytest.raises(TypeError):
            call()
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(TypeError):
            C.cache_attention(k, SimpleNamespace(k=torch.zeros(2, 4, 64, dtype=dtype), v=torch.zeros(2, 4, 64, dtype=dtype), offset=0), 1.0)


P = ctypes.c_void_p(1 << 20)          # never read: every call below is refused on the host


def _refused(scmx, name, args, text):
    rc = getattr(scmx._lib.lib(), name)(*args)
    assert rc < 0 and text in scmx._lib.lib().scmx_last_error_string().decode(), scmx._lib.lib().scmx_last_error_string()


def test_entry_points_refuse(scmx):
    def append(k=P, khs=64, krs=64, L=3, hk=2, d=64, pos=0, dev=None, cap=16, codes=P):
        return (k, khs, krs, P, 64, 64, L, hk, d, pos, dev, cap, codes, P, P, P, None)
    for kw, text in ((dict(k=None), "null"), (dict(d=24), "head size"), (dict(d=272), "head size"), (dict(d=0), "head size"), (dict(pos=14), "rows 14"),
                     (dict(pos=-1), "rows -1"), (dict(krs=12), "16-byte"), (dict(k=ctypes.c_void_p((1 << 20) + 8)), "16-byte"), (dict(hk=0), "hk=0"),
                     (dict(L=-1), "L=-1"), (dict(codes=ctypes.c_void_p((1 << 20) + 4)), "16-byte")):
        _refused(scmx, "scmx_kv_append", append(**kw), text)
    assert scmx._lib.lib().scmx_kv_append(*append(L=0)) == 0
    for start, n, hk, d, text in ((0, 17, 2, 64, "rows 0"), (-1, 2, 2, 64, "rows -1"), (0, 2, 0, 64, "rows"), (0, 2, 2, 20, "head size")):
        _refused(scmx, "scmx_kv_read", (P, P, P, P, start, n, hk, d, 16, P, P, None), text)
    layers = (ctypes.c_void_p * 8)()
    for n, pos, d, text in ((0, 0, 64, "0 rows"), (65, 0, 64, "65 rows"), (4, 13, 64, "rows 13"), (4, 0, 40, "head size"), (4, 0, 64, "layer 0")):
        _refused(scmx, "scmx_kv_keep", (layers, 2, P, n, pos, None, 2, d, 16, 0, None), text)

    def attn(q=P, qhs=64, qrs=64, int8=0, ks=None, n=3, pos=0, cap=100, hq=4, hk=2, d=64, scratch=P, size=1 << 20):
        return (q, qhs, qrs, P, P, ks, ks, int8, None, n, pos, None, cap, hq, hk, d, 1.0, P, scratch, size, P, None)
    for kw, text in ((dict(q=None), "null"), (dict(int8=1), "null"), (dict(n=0), "0 rows"), (dict(n=65), "65 rows"), (dict(d=96), "head size"), (dict(hq=5), "hq=5"),
                     (dict(hk=0), "hk=0"), (dict(pos=98), "rows 98"), (dict(pos=-1), "rows -1"), (dict(cap=2), "rows"), (dict(qhs=66), "aligned"),
                     (dict(q=ctypes.c_void_p((1 << 20) + 2)), "aligned"), (dict(pos=50000, cap=90000, size=8), "scratch"), (dict(pos=50000, cap=90000, scratch=None), "scratch")):
        _refused(scmx, "scmx_cache_attn", attn(**kw), text)
    assert scmx._lib.lib().scmx_cache_attn_scratch(5000, 3, 5, 2, 64) == 0

    def check(n=3, V=100, ld=100, u=P, t=1.0, probs=None, ldp=0, size=1 << 20, tokens=P):
        return (P, 1, ld, tokens, P, u, t, probs, ldp, n, V, P, P, P, P, size, None)
    for kw, text in ((dict(n=0), "0 rows"), (dict(n=65), "65 rows"), (dict(V=0), "0 logits"), (dict(ld=99), "99"), (dict(probs=P, ldp=99), "99"), (dict(t=-1.0), "temperature"),
                     (dict(t=float("nan")), "temperature"), (dict(t=float("inf")), "temperature"), (dict(t=1e-42), "temperature"), (dict(t=4e-39), "temperature"), (dict(u=None), "random"),
                     (dict(size=8), "scratch"), (dict(tokens=None), "null")):
        _refused(scmx, "scmx_verify", check(**kw), text)


def test_no_tokens_are_appended(scmx):
    """Tensors of no elements have no address: nothing is launched, whatever the pointers; sizes are checked all the same."""
    append = lambda L, d=64, pos=0: (None, 0, 64, None, 0, 64, L, 2, d, pos, None, 16, P, P, P, P, None)      # noqa: E731
    assert scmx._lib.lib().scmx_kv_append(*append(0)) == 0 and scmx._lib.lib().scmx_kv_append(*append(0, pos=16)) == 0
    _refused(scmx, "scmx_kv_append", append(1), "null")
    _refused(scmx, "scmx_kv_append", append(0, pos=17), "rows 17")
    _refused(scmx, "scmx_kv_append", append(0, d=24), "head size")


def test_scratch_of_the_attention(scmx):
    """Ranges whose CTAs are a cluster need none, nor does a single range; a second launch needs a state of every query row and range.  Heads and positions on both sides of the
    borders, for a device of 148 multiprocessors."""
    size = scmx._lib.lib().scmx_cache_attn_scratch
    if torch.cuda.is_available() and torch.cuda.get_device_properties(0).multi_processor_count != 148:
        return
    state = (128 + 2) * 4
    assert size(60, 1, 16, 8, 128) == 0 and size(60, 1, 400, 400, 128) == 0                      # one range
    assert size(1000, 1, 15, 15, 128) == 0 and size(1000, 1, 16, 16, 128) == 16 * 9 * 8 * state   # clusters of eight that run at once, or 148 / 16 ranges
    assert size(500, 21, 32, 32, 128) == 0 and size(500, 21, 33, 33, 128) == 33 * 4 * 32 * state   # clusters of four
    assert size(8192, 1, 16, 8, 128) == 0 and size(8193, 1, 16, 8, 128) == 8 * 18 * 8 * state      # INT8, few rows
    assert size(6144, 21, 8, 8, 128) == 0 and size(6145, 21, 8, 8, 128) == 8 * 18 * 32 * state     # tcgen05
    assert size(2000, 64, 16, 8, 128) == 8 * 16 * 128 * state                                      # 128 rows: a tile without copies


def test_lookup_draft(scmx):
    import importlib
    L = importlib.import_module(scmx.__name__ + ".decode").LookupDraft
    text = [1, 2, 3, 4, 5, 9, 1, 2, 3, 4, 6, 7, 1, 2, 3]
    rows, parents = L(match=3, length=3, places=2)(text, 64)
    assert rows == [3, 4, 6, 7, 5, 9] and parents == [-1, 0, 1, 2, 1, 4]          # the latest place first, the shared beginning once
    scmx.sc_draft.check_tree(parents)
    assert L(length=3)(text, 3) == ([3, 4, 6], [-1, 0, 1])
    assert L()(text, 1) == ([3], [-1]) and L()([5], 8) == ([5], [-1]) and L()([1, 2, 3], 8) == ([3], [-1])
    assert L(match=1, length=2, places=1)([4, 4, 4], 8) == ([4, 4], [-1, 0])


def test_caches_of_models(scmx):
    HM = scmx.host_model
    model = HM.CausalLM(HM.ModelArgs(64, 64, 2, 2, 1, 32, 1e-6, 1e6, 16, True))
    plain, quant = HM.make_prompt_cache(model, 8), HM.make_prompt_cache(model, 8, dtype=torch.int8)
    assert all(type(c) is HM.KVCache for c in plain) and all(type(c) is HM.QuantKVCache for c in quant)
    assert quant[0].k.shape == (1, 8, 32) and quant[0].ks.shape == (1, 8) and quant[0].carried() == []
    with pytest.raises(ValueError):
        HM.make_prompt_cache(model, 8, dtype=torch.float16)
    cfg = {"architecture": "Sebesun", "vocab": 8, "width": 8, "norm": {"eps": 1e-5}, "layers": [
        {"type": "retention", "mixer": {"heads": 1, "dim": 8, "vdim": 8, "decay": [0.9]}, "mlp": None}]}
    hybrid = HM.HybridLM(HM.HybridArgs.from_config(cfg), device="cpu", dtype=torch.float32)
    with pytest.raises(ValueError):
        HM.make_prompt_cache(hybrid, 8, dtype=torch.int8)
    assert len(HM.make_prompt_cache(hybrid, 8, dtype=torch.float32)) == 1


def test_drafts_are_checked(scmx):
    """What a proposal or the random numbers may get wrong is refused on the host, before anything is launched."""
    import importlib
    from types import SimpleNamespace as N
    DD = importlib.import_module(scmx.__name__ + ".decode").DecodeDraft
    d, cache = DD.__new__(DD), [N(offset=4, capacity=8)]
    d.f = N(args=N(vocab_size=16))
    chain = lambda n: list(range(-1, n - 1))                # noqa: E731
    for tokens, parents in (([3, 16], [-1, 0]), ([3, -1], [-1, 0]), ([4, 1], [-1, 0]), ([3, 1], [-1]), ([3], [-1, 0]), ([3, 1], [-1, 1]), ([3] * 5, chain(5)), ([], [])):
        d.propose = lambda text, most: (tokens, parents)
        with pytest.raises(ValueError):
            d.step([1, 3], cache)
    with pytest.raises(ValueError):
        d.step([1, 17], cache)                              # the text's last token itself
    d.propose = lambda text, most: ([3, 2, 1], chain(3))
    for u in (None, torch.zeros(2), torch.zeros(1), torch.zeros(3, 1)):
        with pytest.raises(ValueError, match="temperature"):
            d.step([1, 3], cache, 0.5, u)
    with pytest.raises(AssertionError):
        d.step([1, 3], [N(offset=8, capacity=8)])


def test_entry_points_run_as_a_script():
    """Everything that build() and smoke() call is defined above the lines that run them when the file is the program."""
    import ast
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "__graft_entry__.py")
    body = ast.parse(open(path).read()).body
    guard = next(i for i, node in enumerate(body) if isinstance(node, ast.If) and "__main__" in ast.unparse(node.test))
    defined = {node.name for node in body[:guard] if isinstance(node, ast.FunctionDef)}
    later = {node.name for node in body[guard:] if isinstance(node, ast.FunctionDef)}
    called = {node.func.id for f in body for node in ast.walk(f) if isinstance(node, ast.Call) and isinstance(node.func, ast.Name)}
    assert {"build", "smoke"} <= defined and not called & later


def test_engine_keeps_nothing_of_a_call_that_ends_early(scmx):
    """A proposal that raises, a draft that is refused, a decoder that fails: the request is gone, its cache back in the pool, and the next call starts anew.  A model
    that reads no drafts is refused before its prompt is read."""
    import importlib
    from types import SimpleNamespace as N
    E = importlib.import_module(scmx.__name__ + ".engine")

    class Cache:
        def __init__(self):
            self.offset, self.capacity = 0, 32

        def reset(self):
            self.offset = 0
    read = []

    def hidden(ids, cache):
        read.append((cache[0].offset, ids.shape[1]))
        cache[0].offset += ids.shape[1]
        return torch.zeros(1, ids.shape[1], 4)

    def fail(*a):
        raise RuntimeError("decoder")
    args = N(num_attention_heads=4, num_key_value_heads=2, head_dim=64, vocab_size=8)
    prefill = N(args=args, inv_freq=torch.zeros(1), make_cache=lambda capacity: [Cache()], hidden=hidden, logits=lambda h: torch.zeros(*h.shape[:2], 8))
    engine = E.Engine(N(prefill=prefill, decode=N(generate=fail)), 32, device="cpu")

    def gone(text, most):
        raise KeyError("proposal")
    for draft, error in ((gone, KeyError), (lambda text, most: ([text[-1], 9], [-1, 0]), ValueError), (None, RuntimeError)):
        for _ in range(2):
            with pytest.raises(error):
                engine.generate([1, 2, 3], 4, draft=draft)
            assert not engine.live and len(engine.pool.free) == 1 and read.pop() == (0, 3)
    prefill.args = N(layers=[])                             # a hybrid decoder
    other = E.Engine(N(prefill=prefill, decode=None), 32, device="cpu")
    with pytest.raises(ValueError, match="drafts"):
        other.generate([1, 2, 3], 4, draft=gone)
    assert not other.live and not read


def test_random_numbers_are_checked_in_every_pass(scmx):
    """Numbers of another type or device are refused before any pass, a captured one too, which would take them through a copy."""
    import importlib
    from types import SimpleNamespace as N
    DD = importlib.import_module(scmx.__name__ + ".decode").DecodeDraft
    d, cache = DD.__new__(DD), [N(offset=4, capacity=8)]
    d.f, d.dev, d.propose = N(args=N(vocab_size=16)), torch.device("cpu"), lambda text, most: ([3, 2], [-1, 0])
    taken = []
    d._captured = lambda tokens, parents, cache, u, temperature: taken.append(u) or torch.tensor([0, -1, 5])
    for u in (torch.zeros(64, dtype=torch.float64), torch.zeros(64, dtype=torch.bfloat16), torch.zeros(64, device="meta"), torch.zeros(64, dtype=torch.long)):
        with pytest.raises(TypeError, match="random numbers"):
            d.step([1, 3], cache, 0.5, u)
    assert not taken and cache[0].offset == 4
    assert d.step([1, 3], cache, 0.5, torch.arange(128.0)[::2]) == [5]
    assert taken[0].tolist() == [0.0, 2.0] and taken[0].is_contiguous() and cache[0].offset == 5
    assert d.step([1, 3], cache, 0.0, torch.zeros(1, dtype=torch.float64)) == [5] and taken[1] is None      # greedy: not read

"""GPU: INT8 key/value cache, attention of drafted rows, verification of drafts and the move of accepted rows, against plain float64."""
import math
import random
from types import SimpleNamespace

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -8           # most that a rounding to bfloat16 is off, relative


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def quantized(x):
    """s = amax / 127, zero below 2^-126 where 1 / s overflows, code = rint(x (1 / s)) in IEEE float32."""
    x = x.float().cpu().numpy()
    s = np.abs(x).max(-1) / np.float32(127)
    s = np.where(s < np.float32(2.0 ** -126), np.float32(0), s)
    qi = np.where(s > 0, np.float32(1) / np.where(s > 0, s, np.float32(1)), np.float32(0)).astype(np.float32)
    return torch.from_numpy(np.rint(x * qi[..., None]).astype(np.int8)).cuda(), torch.from_numpy(s.astype(np.float32)).cuda()


def quant_cache(scmx, hk, cap, d, offset, fill=99):
    c = scmx.host_model.QuantKVCache(hk, d, cap)
    for t in (c.k, c.v):
        t.fill_(fill)
    for t in (c.ks, c.vs):
        t.fill_(float(fill))
    c.offset = offset
    return c


# ---- the INT8 cache -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hk,L,d,offset,layout", [(1, 1, 16, 0, "heads"), (8, 1, 128, 5, "heads"), (3, 7, 64, 2, "tokens"), (2, 300, 128, 11, "tokens"),
                                                  (5, 33, 80, 0, "heads"), (1, 130, 256, 7, "heads"), (4, 19, 48, 3, "odd")])
def test_append_and_read(scmx, hk, L, d, offset, layout):
    g = gen(hk * 1000 + L)
    cap = offset + L + 3

    def vectors():
        x = torch.randn((hk, L, d), generator=g, device="cuda") * torch.exp(torch.randn((hk, L, 1), generator=g, device="cuda") * 3)
        if layout == "tokens":
            return x.to(BF).transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "odd":           # rows that do not start on 16-byte boundaries
            return torch.nn.functional.pad(x.to(BF), (1, 0))[:, :, 1:]
        return x.to(BF)
    k, v = vectors(), vectors()
    k[0, 0], v[-1, -1] = 0.0, 0.0
    k[0, L // 2, 3] = 1e-38           # far below the rest
    c = quant_cache(scmx, hk, cap, d, offset)
    scmx.sc_cache.kv_append(k, v, c)
    assert c.offset == offset
    for x, codes, scales in ((k, c.k, c.ks), (v, c.v, c.vs)):
        q, s = quantized(x)
        assert torch.equal(codes[:, offset:offset + L], q) and torch.equal(scales[:, offset:offset + L], s)
        for rows in (slice(0, offset), slice(offset + L, cap)):      # nothing else is written
            assert (codes[:, rows] == 99).all() and (scales[:, rows] == 99).all()
    c.offset += L
    for got, codes, scales in zip(scmx.sc_cache.kv_read(c, offset), (c.k, c.v), (c.ks, c.vs)):
        assert torch.equal(got, (codes[:, offset:offset + L].float() * scales[:, offset:offset + L, None]).to(BF))
    whole = scmx.sc_cache.kv_read(c)
    assert whole[0].shape == (hk, offset + L, d) and torch.equal(whole[1][:, offset:], scmx.sc_cache.kv_read(c, offset)[1])
    assert scmx.sc_cache.kv_read(c, 2, 2)[0].shape == (hk, 0, d)


def test_append_of_no_tokens(scmx):
    c = quant_cache(scmx, 2, 6, 64, 3)
    none = torch.empty((2, 0, 64), dtype=BF, device="cuda")
    for dev in (None, torch.tensor([2], dtype=torch.int32, device="cuda")):
        scmx.sc_cache.kv_append(none, none, c, dev)
    assert (c.k == 99).all() and (c.vs == 99).all()
    k, v = c.update_and_fetch(none, none)
    assert c.offset == 3 and k.shape == v.shape == (2, 3, 64)


def test_append_takes_its_position_from_the_device(scmx):
    k, v = (torch.randn((2, 4, 64), generator=gen(i), device="cuda").to(BF) for i in (1, 2))
    for at in (0, 3, 6, 8, -2, 2 ** 31 - 1, -2 ** 31):
        c, want = quant_cache(scmx, 2, 8, 64, 0), quant_cache(scmx, 2, 8, 64, 0)
        scmx.sc_cache.kv_append(k, v, c, torch.tensor([at], dtype=torch.int32, device="cuda"))
        rows = [i for i in range(4) if 0 <= at + i < 8]               # rows outside the cache are dropped
        if rows:
            want.offset = at + rows[0]
            scmx.sc_cache.kv_append(k[:, rows], v[:, rows], want)
        assert all(torch.equal(getattr(c, n), getattr(want, n)) for n in ("k", "v", "ks", "vs"))


def test_append_of_values_that_are_not_numbers(scmx):
    x = torch.randn((1, 6, 64), generator=gen(3), device="cuda").to(BF)
    x[0, 1, 5], x[0, 2, 0], x[0, 3, 63] = float("nan"), float("inf"), float("-inf")
    x[0, 4] = 1e-37                    # 1 / s would overflow
    c = quant_cache(scmx, 1, 6, 64, 0)
    scmx.sc_cache.kv_append(x, x, c)
    c.offset = 6
    k, v = scmx.sc_cache.kv_read(c)
    assert torch.isnan(k[0, 1:4]).all() and torch.isnan(v[0, 1:4]).all()
    assert (k[0, 4] == 0).all() and torch.isfinite(k[0, [0, 5]]).all()
    assert ((k[0, 5].float() - x[0, 5].float()).abs() <= x[0, 5].abs().max().float() * (0.5 / 127 * (1 + 1e-5) + U)).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("layers,hk,d,n,rows", [(1, 1, 64, 1, [0]), (3, 2, 128, 9, [0, 2, 5, 8, -1, -1, -1, -1, -1]), (70, 3, 64, 64, None), (2, 4, 256, 64, None),
                                                (2, 2, 16, 5, [4, 3, 2, 1, 0]), (1, 2, 80, 4, [0, 0, 3, 77])])
def test_keep(scmx, int8, layers, hk, d, n, rows):
    g, rng = gen(n), random.Random(n + d)
    rows = rows or sorted(rng.sample(range(n), n // 3)) + [-1] * (n - n // 3)
    pos, cap = 6, 6 + n + 2
    caches = []
    for _ in range(layers):
        c = quant_cache(scmx, hk, cap, d, pos) if int8 else scmx.host_model.KVCache(hk, d, cap)
        for t in ((c.k, c.v, c.ks, c.vs) if int8 else (c.k, c.v)):
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda"))
        caches.append(c)
    caches[0].offset = pos
    names = ("k", "v", "ks", "vs") if int8 else ("k", "v")
    before = [[getattr(c, m).clone() for m in names] for c in caches]
    index = torch.arange(cap, device="cuda")
    index[pos:pos + n] = torch.tensor([pos + (r if 0 <= r < n else j) for j, r in enumerate(rows)], device="cuda")
    scmx.sc_cache.kv_keep(caches, torch.tensor(rows, dtype=torch.int32, device="cuda"))
    for c, old in zip(caches, before):
        for m, t in zip(names, old):
            assert torch.equal(getattr(c, m), t[:, index])
    dev = torch.tensor([pos], dtype=torch.int32, device="cuda")
    again = [SimpleNamespace(**{m: t for m, t in zip(names, old)}, offset=0) for old in before]
    scmx.sc_cache.kv_keep(again, torch.tensor(rows, dtype=torch.int32, device="cuda"), pos_dev=dev)
    assert all(torch.equal(getattr(a, m), getattr(c, m)) for a, c in zip(again, caches) for m in names)
    dev.fill_(cap - n + 1)                                             # not inside the cache: nothing happens
    scmx.sc_cache.kv_keep(again, torch.tensor(rows[::-1], dtype=torch.int32, device="cuda"), pos_dev=dev)
    assert all(torch.equal(getattr(a, m), getattr(c, m)) for a, c in zip(again, caches) for m in names)


@pytest.mark.parametrize("int8", [False, True])
def test_keep_refuses_a_cache_that_is_listed_twice(scmx, int8):
    make = lambda: quant_cache(scmx, 2, 12, 64, 3) if int8 else scmx.host_model.KVCache(2, 64, 12)      # noqa: E731
    a, b, rows = make(), make(), torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda")
    shared = SimpleNamespace(k=a.k, v=b.v, offset=3)
    mirror = SimpleNamespace(k=b.k, v=b.k, offset=3)
    if int8:
        for c in (shared, mirror):
            c.ks, c.vs = a.ks, b.vs
    for caches in ([a, a], [a, b, a], [a, shared], [mirror]):
        with pytest.raises(ValueError, match="twice"):
            scmx.sc_cache.kv_keep(caches, rows, pos=3)
    scmx.sc_cache.kv_keep([a, b], rows, pos=3)


# ---- attention ----------------------------------------------------------------------------------------------------------------

def attention_case(scmx, hq, hk, n, T, d, int8, seed=0, extra=5, std=1.5):
    g = gen(seed)
    cap = T + n + extra
    k, v = (torch.randn((hk, cap, d), generator=g, device="cuda").to(BF) for _ in range(2))
    q = (torch.randn((hq, n, d), generator=g, device="cuda") * std).to(BF)
    if int8:
        c = quant_cache(scmx, hk, cap, d, T)
        (c.k, c.ks), (c.v, c.vs) = quantized(k), quantized(v)
    else:
        c = scmx.host_model.KVCache(hk, d, cap)
        c.k.copy_(k)
        c.v.copy_(v)
        c.k[:, T + n:], c.v[:, T + n:] = float("nan"), float("nan")
        c.offset = T
    return q, c


def bits_of(mask, n):
    return [(1 << i + 1) - 1 for i in range(n)] if mask is None else [b & (1 << n) - 1 for b in mask.tolist()]


def attention_oracle(q, c, scale, mask, T=None, weight=U):
    """float64 output, and how far a kernel's may be off: weights and outputs are rounded to bfloat16 once (U each; weight: what a weight may be off), scores are float32 sums of d
    products (an error of (d + 8) 2^-24 sum |q k| scale changes a weight by twice that), sums of weights and outputs float32."""
    hq, n, d = q.shape
    hk, T = c.k.shape[0], c.offset if T is None else T
    out, tol = torch.zeros((n, hq, d), dtype=F64, device="cuda"), torch.zeros((n, hq, d), dtype=F64, device="cuda")
    int8 = c.k.dtype == torch.int8
    seen = torch.ones((n, T + n), dtype=torch.bool, device="cuda")
    seen[:, T:] = torch.tensor([[b >> j & 1 > 0 for j in range(n)] for b in bits_of(mask, n)], device="cuda").view(n, n)
    for h in range(hq):
        k, v = c.k[h // (hq // hk), :T + n].to(F64), c.v[h // (hq // hk), :T + n].to(F64)
        if int8:
            k, v = k * c.ks[h // (hq // hk), :T + n, None].to(F64), v * c.vs[h // (hq // hk), :T + n, None].to(F64)
        s = (q[h].to(F64) @ k.T * scale).masked_fill(~seen, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, 1), nan=0.0)
        size = ((q[h].to(F64).abs() @ k.abs().T) * abs(scale)).masked_fill(~seen, 0.0).amax(1, keepdim=True)
        weighted = p @ torch.where(torch.isfinite(v), v, 0.0).abs()
        out[:, h] = p @ torch.where(torch.isfinite(v), v, 0.0)
        tol[:, h] = (weight * weighted + U * out[:, h].abs()) * (1 + U) + weighted * (2 * (d + 8) * 2.0 ** -24 * size + (T + n) ** 0.5 * 2.0 ** -22)
    return out.reshape(n, hq * d), tol.reshape(n, hq * d)


def check_attention(got, q, c, scale, mask, T=None):
    want, tol = attention_oracle(q, c, scale, mask, T)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"off by {(off / tol.clamp(min=1e-30)).max().item():.3g} of the tolerance"


def random_parents(rng, n):
    return [-1] + [rng.randrange(max(0, i - 5), i) for i in range(1, n)]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk,n,T", [(1, 1, 1, 0), (2, 2, 1, 1), (16, 8, 1, 15), (16, 8, 1, 16), (16, 8, 5, 127), (8, 1, 64, 128), (6, 2, 13, 129),
                                       (4, 4, 16, 1000), (32, 8, 1, 5000), (16, 8, 21, 777), (8, 2, 64, 4097), (7, 1, 3, 300), (3, 3, 64, 0), (40, 2, 9, 63)])
def test_attention_of_a_tree(scmx, int8, d, hq, hk, n, T):
    q, c = attention_case(scmx, hq, hk, n, T, d, int8, seed=n + T)
    scale = d ** -0.5
    mask = scmx.sc_draft.draft_mask(random_parents(random.Random(n), n))
    check_attention(scmx.sc_cache.cache_attention(q, c, scale, mask), q, c, scale, mask)
    check_attention(scmx.sc_cache.cache_attention(q, c, scale), q, c, scale, None)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hq,hk,n", [(15, 15, 1), (16, 16, 1), (20, 20, 7), (16, 16, 21), (33, 33, 21), (4, 4, 21), (8, 8, 33), (2, 1, 12)])
@pytest.mark.parametrize("T", [20, 250, 500, 1100, 2047, 4100, 6150, 8200])
def test_attention_on_both_sides_of_the_clusters_borders(scmx, int8, hq, hk, n, T):
    """One range, clusters of two, four and eight, clusters that would not run at once, and two launches; the position on the host, and on the device in a larger cache,
    which cuts it by its capacity."""
    d, at = 64 if T == 500 else 128, max(T - n, 0)                       # T positions with the new rows
    q, c = attention_case(scmx, hq, hk, n, at, d, int8, seed=T + hk)
    mask = scmx.sc_draft.draft_mask(random_parents(random.Random(n), n))
    check_attention(scmx.sc_cache.cache_attention(q, c, 0.09, mask), q, c, 0.09, mask)
    if T >= 4100:
        for pos in (at, T // 3, 3, 0):
            check_attention(scmx.sc_cache.cache_attention(q, c, 0.09, mask, torch.tensor([pos], dtype=torch.int32, device="cuda")), q, c, 0.09, mask, T=pos)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("int8,hq,hk,n,T", [(False, 8, 4, 1, 900), (False, 4, 4, 11, 10000), (False, 2, 1, 8, 40), (True, 8, 4, 1, 900), (True, 2, 2, 16, 10000), (True, 16, 2, 3, 2500),
                                            (True, 16, 2, 7, 400), (True, 8, 2, 30, 7000), (True, 8, 1, 20, 9000), (True, 4, 1, 64, 5000)])
def test_weights_keep_their_bits(scmx, int8, d, hq, hk, n, T):
    """Weights over INT8 are float16 (half a step is 2^-12 of one, the maximum's exponential, the scale's log2 and reciprocal 2^-20 together), those of up to 16
    query rows over bfloat16 two bfloat16 (2^-16): 2^-11 and 2^-15 with room for it, where one bfloat16 is 2^-8."""
    q, c = attention_case(scmx, hq, hk, n, T, d, int8, seed=3 * n + T)
    mask = scmx.sc_draft.draft_mask(random_parents(random.Random(n), n))
    want, tol = attention_oracle(q, c, d ** -0.5, mask, weight=2.0 ** -11 if int8 else 2.0 ** -15)
    off = (scmx.sc_cache.cache_attention(q, c, d ** -0.5, mask).double() - want).abs()
    assert (off <= tol).all(), f"off by {(off / tol).max().item():.3g} of the tolerance"


@pytest.mark.parametrize("hq,hk,n,T", [(4, 2, 1, 700), (4, 4, 12, 9000), (8, 2, 7, 300), (4, 1, 20, 3000), (4, 1, 64, 1200)])
def test_scales_of_all_sizes(scmx, hq, hk, n, T):
    """Values whose scales differ by 2^60, among them zeros and the smallest and largest that kv_append writes.  A weight below 2^-14 has a float16 step of 2^-24, 2^-30 of
    the largest weight's 2^6 at least: half of it for every position, times 127 codes and the largest p s."""
    q, c = attention_case(scmx, hq, hk, n, T, 128, True, seed=n)
    g = gen(9)
    c.vs.mul_(2.0 ** torch.randint(-30, 31, c.vs.shape, generator=g, device="cuda").float())
    gone = torch.rand(c.vs.shape, generator=g, device="cuda") < 0.05
    c.vs[gone] = 0.0
    c.v[gone] = 0
    for size in (None, 2.0 ** -126, 2.0 ** 120 / 127):
        if size is not None:
            c.vs.copy_(torch.where(gone, 0.0, size))
        want, tol = attention_oracle(q, c, 0.09, None, weight=2.0 ** -11)
        if size is None:
            tol += (T + n) * 2.0 ** -31 * 127 * c.vs.double().amax()
        else:
            tol += 2.0 ** -126                                        # an output below the normal numbers
        off = (scmx.sc_cache.cache_attention(q, c, 0.09).double() - want).abs()
        assert (off <= tol).all(), f"{size}: off by {(off / tol).max().item():.3g} of the tolerance"


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hq,hk,n,T", [(4, 2, 3, 40), (8, 2, 7, 300), (8, 2, 30, 129), (8, 1, 20, 1000), (8, 2, 40, 2500), (4, 4, 64, 0)])
def test_scales_of_zero_and_below(scmx, int8, hq, hk, n, T):
    """A scale of 0 is the mean of what a row sees, also where tiles hide positions; the smallest positive one is next to it; a negative one turns the order round."""
    q, c = attention_case(scmx, hq, hk, n, T, 128, int8, seed=n)
    mask = scmx.sc_draft.draft_mask(random_parents(random.Random(n), n))
    nothing = mask & ~(1 << torch.arange(n, device="cuda"))                # the first row of an empty cache sees nothing
    for scale in (0.0, -0.0, 1e-45, 1e-38, -1e-20, -0.1):
        for m in (None, mask, nothing):
            check_attention(scmx.sc_cache.cache_attention(q, c, scale, m), q, c, scale, m)


@pytest.mark.parametrize("hq,hk,n,T,at", [(2, 2, 1, 2000, 1000), (2, 2, 1, 2000, 0), (4, 2, 6, 9000, 5000), (8, 2, 20, 2000, 1500), (8, 1, 40, 3000, 2)])
def test_values_of_zeros_with_the_largest_score(scmx, hq, hk, n, T, at):
    """A vector of zeros that takes nearly all of a row's weight leaves the others their bits: the output, small as it is, keeps its relative error (a float16 weight's half
    step 2^-12, the maximum's exponential, log2 and reciprocal: 2^-11 of the weighted magnitudes)."""
    g = gen(n)
    q, c = attention_case(scmx, hq, hk, n, T, 128, True, seed=n)
    along = torch.nn.functional.normalize(torch.randn((hk, 1, 128), generator=g, device="cuda"), dim=-1)
    k, v = (torch.randn((hk, c.k.shape[1], 128), generator=g, device="cuda") for _ in range(2))
    k = 0.1 * (k - (k * along).sum(-1, keepdim=True) * along)            # no other key points there
    for powers in (0, 16, 20, 24, 28, 32, 50, 80):
        k[:, at], v[:, at] = along[:, 0] * powers * math.log(2), 0.0
        (c.k, c.ks), (c.v, c.vs) = quantized(k.to(BF)), quantized(v.to(BF))
        q = (along.repeat_interleave(hq // hk, 0) * 10 + 0.3 * torch.randn((hq, n, 128), generator=g, device="cuda")).to(BF)
        want, tol = attention_oracle(q, c, 0.1, None, weight=2.0 ** -11)
        off = (scmx.sc_cache.cache_attention(q, c, 0.1).double() - want).abs()
        assert (off <= tol).all(), f"{powers}: off by {(off / tol).max().item():.3g} of the tolerance"


@pytest.mark.parametrize("hq,hk,n,T", [(2, 2, 3, 0), (8, 2, 4, 0), (4, 4, 9, 7), (4, 2, 2, 16), (2, 1, 6, 300), (8, 2, 30, 0), (8, 2, 30, 100), (4, 1, 64, 700), (4, 4, 20, 3)])
def test_scales_in_masked_places(scmx, hq, hk, n, T):
    """Over INT8, new rows that no row sees hold any scale, and one that only its own row sees is 2^93 above or below all others: every other row is as without them.  Its own row is
    what its scale makes it.  (A float16 weight: as in test_scales_of_all_sizes, with the largest scale that a row sees.)"""
    rng = random.Random(n + T)
    odd = n // 2
    for value, alone in ((1e30, False), (1e-30, False), (2.0 ** -126, False), (float("nan"), False), (float("inf"), False), (1e28, True), (1e-28, True)):
        q, c = attention_case(scmx, hq, hk, n, T, 128, True, seed=n)
        bits = [(rng.getrandbits(n) | 1 << i) & ~(1 << odd) for i in range(n)]
        bits[odd] = 1 << odd if alone else bits[odd] | (1 << (odd + 1) % n)
        mask = torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], device="cuda")
        others = [i for i in range(n) if not (alone and i == odd)]
        amax = torch.cat((c.vs[:, :T + odd], c.vs[:, T + odd + 1:T + n]), 1).amax().double()
        for rows in ([odd], [odd] + [j for j in range(n) if not any(b >> j & 1 for b in bits)]):
            if alone:
                c.vs[:, T + odd] = value
                want, tol = attention_oracle(q, c, 0.09, mask, weight=2.0 ** -11)
            else:
                want, tol = attention_oracle(q, c, 0.09, mask, weight=2.0 ** -11)
                c.vs[:, [T + j for j in rows]] = value
                c.ks[:, [T + j for j in rows]] = float("nan")
            got = scmx.sc_cache.cache_attention(q, c, 0.09, mask)
            off = (got.double() - want).abs()
            assert torch.isfinite(got).all()
            assert (off[others] <= tol[others] + (T + n) * 2.0 ** -31 * 127 * amax).all(), f"{value}: off by {(off / tol)[others].max().item():.3g} of the tolerance"
            if alone:
                assert (off[odd] <= tol[odd] + (T + n) * 2.0 ** -31 * 127 * max(amax, value)).all(), f"{value}: its own row"
            else:
                c.vs[:, [T + j for j in rows]], c.ks[:, [T + j for j in rows]] = 0.01, 0.01


@pytest.mark.parametrize("hq,hk,n,T,first", [(2, 2, 4, 1, 1e-7), (2, 2, 4, 1, 1e5), (8, 2, 22, 1, 1e-7), (4, 4, 64, 1, 1e-7), (4, 4, 64, 2, 1e6), (1, 1, 12, 300, 1e-7), (4, 1, 20, 300, 1e-7)])
def test_zeros_count_beside_values_of_all_sizes(scmx, hq, hk, n, T, first):
    """The first position's scale is far from the others', which are 2^40 apart among themselves, and a third of the vectors are zeros: those have no value but their weight, and it
    stays in the sum.  (The tolerance of test_scales_of_all_sizes.)"""
    q, c = attention_case(scmx, hq, hk, n, T, 128, True, seed=n)
    g = gen(4)
    c.vs.mul_(2.0 ** torch.randint(-20, 21, c.vs.shape, generator=g, device="cuda").float())
    gone = torch.rand(c.vs.shape, generator=g, device="cuda") < 0.33
    c.vs[gone] = 0.0
    c.v[gone] = 0
    c.vs[:, 0], c.v[:, 0] = first, 1
    for scale in (0.09, 1e-3, 0.0):
        want, tol = attention_oracle(q, c, scale, None, weight=2.0 ** -11)
        off = (scmx.sc_cache.cache_attention(q, c, scale).double() - want).abs()
        assert (off <= tol + (T + n) * 2.0 ** -31 * 127 * c.vs.double().amax()).all(), f"off by {(off / tol).max().item():.3g} of the tolerance"


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hq,hk,n,T", [(8, 8, 4, 0), (8, 2, 40, 0), (4, 1, 64, 0), (4, 1, 3, 200), (8, 2, 64, 1)])
def test_rows_that_see_nothing(scmx, int8, hq, hk, n, T):
    q, c = attention_case(scmx, hq, hk, n, T, 128, int8)
    rng = random.Random(n)
    mask = torch.tensor([0 if i % 3 == 0 else rng.getrandbits(63) for i in range(n)], dtype=torch.int64, device="cuda")      # bits beyond n are ignored
    got = scmx.sc_cache.cache_attention(q, c, 0.1, mask)
    check_attention(got, q, c, 0.1, mask)
    if T == 0:
        assert (got[::3] == 0).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n,T", [(5, 0), (33, 100), (64, 1000), (17, 3)])
def test_masked_rows_that_are_not_numbers_stay_out(scmx, int8, n, T):
    """Drafted rows whose keys or values are NaN or infinite reach the rows that see them and no others."""
    q, c = attention_case(scmx, 8, 2, n, T, 128, int8, seed=5)
    bad = [1, n // 2, n - 1]
    parents = random_parents(random.Random(1), n)
    mask = scmx.sc_draft.draft_mask(parents)
    bits = bits_of(mask, n)
    want, tol = attention_oracle(q, c, 0.1, mask)
    for j, value in zip(bad, (float("nan"), float("inf"), float("-inf"))):
        if int8:
            c.vs[:, T + j] = value
            c.ks[:, T + j] = float("nan")
        else:
            c.v[:, T + j, 7::9] = value
            c.k[:, T + j, 3] = value
    got = scmx.sc_cache.cache_attention(q, c, 0.1, mask)
    for i in range(n):
        if any(bits[i] >> j & 1 for j in bad):
            assert not torch.isfinite(got[i]).all()
        else:
            assert torch.isfinite(got[i]).all() and ((got[i].double() - want[i]).abs() <= tol[i]).all()


@pytest.mark.parametrize("int8", [False, True])
def test_values_beyond_32_bit_offsets(scmx, int8):
    """A cache whose last head starts past 2^31 elements."""
    hk, d, T, n = 9, 128, 40, 3
    cap = (1 << 31) // (d * (hk - 1)) + 64
    c = quant_cache(scmx, hk, cap, d, 0) if int8 else SimpleNamespace(k=torch.zeros((hk, cap, d), dtype=BF, device="cuda"), v=torch.zeros((hk, cap, d), dtype=BF, device="cuda"))
    assert (hk - 1) * cap * d > 1 << 31
    c.offset = cap - n - 7
    T = c.offset
    g = gen(1)
    k, v = (torch.randn((hk, n, d), generator=g, device="cuda").to(BF) for _ in range(2))
    if int8:
        c.ks.zero_()
        c.vs.zero_()
        scmx.sc_cache.kv_append(k, v, c)
        kq, ks = quantized(k)
        assert torch.equal(c.k[:, T:T + n], kq) and torch.equal(c.ks[:, T:T + n], ks)
        kr, vr = scmx.sc_cache.kv_read(c, T, T + n)
    else:
        c.k[:, T:T + n], c.v[:, T:T + n], kr, vr = k, v, k, v
    q = (40 * kr[:, :1]).expand(hk, n, d).contiguous()        # every row's weight falls on the first new row: all other scores are zero or far below
    got = scmx.sc_cache.cache_attention(q, c, 1.0).view(n, hk, d)
    want = vr[:, 0][None].float()
    assert ((got.float() - want).abs() <= want.abs() * 2 * U + 1e-6).all()


def test_queries_of_any_strides(scmx):
    q, c = attention_case(scmx, 8, 2, 6, 100, 64, True)
    want = scmx.sc_cache.cache_attention(q, c, 0.2)
    rows = q.transpose(0, 1).contiguous().transpose(0, 1)                                   # [n, hq, d] in memory
    wide = torch.nn.functional.pad(q, (4, 0))[:, :, 4:]
    odd = torch.nn.functional.pad(q, (1, 0))[:, :, 1:]
    for x in (rows, wide, odd):
        assert torch.equal(scmx.sc_cache.cache_attention(x, c, 0.2), want)


@pytest.mark.parametrize("hk,L", [(1, 1), (1, 5), (2, 1), (2, 5)])
@pytest.mark.parametrize("first", [1, 2, 4])
def test_views_that_start_off_a_boundary(scmx, hk, L, first):
    """Contiguous views whose first element is not on a 16-byte boundary, and vectors cut out of wider rows."""
    d, T = 64, 30

    def off(x):
        flat = torch.empty(x.numel() + first, dtype=BF, device="cuda")
        flat[first:] = x.reshape(-1)
        return flat[first:].view_as(x), torch.nn.functional.pad(x, (first, 3))[:, :, first:first + d]
    q, c = attention_case(scmx, 2 * hk, hk, L, T, d, True, seed=L)
    want = scmx.sc_cache.cache_attention(q, c, 0.2)
    for x in off(q):
        assert torch.equal(x, q) and torch.equal(scmx.sc_cache.cache_attention(x, c, 0.2), want)
    k, v = (torch.randn((hk, L, d), generator=gen(i), device="cuda").to(BF) for i in range(2))
    scmx.sc_cache.kv_append(k, v, c)
    for x, y in zip(off(k), off(v)):
        other = quant_cache(scmx, hk, c.k.shape[1], d, T)
        scmx.sc_cache.kv_append(x, y, other)
        for name in ("k", "v", "ks", "vs"):
            assert torch.equal(getattr(other, name)[:, T:T + L], getattr(c, name)[:, T:T + L])


@pytest.mark.parametrize("int8", [False, True])
def test_attention_reads_its_position_from_the_device(scmx, int8):
    q, c = attention_case(scmx, 8, 4, 7, 900, 128, int8, extra=200)
    dev = torch.tensor([900], dtype=torch.int32, device="cuda")
    check_attention(scmx.sc_cache.cache_attention(q, c, 0.1, pos_dev=dev), q, c, 0.1, None)
    dev.fill_(33)
    c.offset = 10 ** 9                 # not read
    check_attention(scmx.sc_cache.cache_attention(q, c, 0.1, pos_dev=dev), q, c, 0.1, None, T=33)
    for at in (-5, 10 ** 6):           # positions that are none are taken as the nearest that is
        dev.fill_(at)
        scmx.sc_cache.cache_attention(q, c, 0.1, pos_dev=dev)
    torch.cuda.synchronize()


@pytest.mark.parametrize("int8", [False, True])
def test_two_graphs_side_by_side(scmx, int8):
    """Two captured calls share no workspace: replayed on two streams at once they give what each gives alone, at every position."""
    cases = [attention_case(scmx, 16, 8, 9, 3000 + 500 * i, 128, int8, seed=i) for i in range(2)]
    mask = scmx.sc_draft.draft_mask(random_parents(random.Random(3), 9))
    devs = [torch.tensor([c.offset], dtype=torch.int32, device="cuda") for _, c in cases]
    streams, graphs, outs = [torch.cuda.Stream() for _ in cases], [], []
    for (q, c), dev, s in zip(cases, devs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            scmx.sc_cache.cache_attention(q, c, 0.1, mask, dev)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(scmx.sc_cache.cache_attention(q, c, 0.1, mask, dev))
            graphs.append(g)
    for T in (2000, 1, 2999):
        for dev in devs:
            dev.fill_(T)
        torch.cuda.synchronize()
        for _ in range(20):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for (q, c), out, dev in zip(cases, outs, devs):
            assert torch.equal(out, scmx.sc_cache.cache_attention(q, c, 0.1, mask, dev))
            check_attention(out, q, c, 0.1, mask, T=T)


def test_one_row_agrees_with_the_decode_attention(scmx):
    q, c = attention_case(scmx, 16, 8, 1, 2000, 128, False)
    old = scmx.sc_kernels.DecodeAttention(16, 8, 128)(q, c, 128 ** -0.5, n_pos=2001)
    want, tol = attention_oracle(q, c, 128 ** -0.5, None)
    assert ((old.double() - want).abs() <= tol).all()
    check_attention(scmx.sc_cache.cache_attention(q, c, 128 ** -0.5), q, c, 128 ** -0.5, None)


# ---- verification -------------------------------------------------------------------------------------------------------------

def verify_oracle(logits, tokens, parents, u, temp, probs):
    """The walk in float64, one row at a time -> (rows, token, how near a test came to its border, relative to its sides, and how near u[0] came to an
    edge of the token's interval)."""
    logits, n, V = logits.double().cpu(), *logits.shape
    probs = None if probs is None else probs.double().cpu()
    node, rows, near = 0, [0], math.inf
    soft = lambda r: torch.softmax(logits[r] / temp, 0) if temp else None      # noqa: E731
    p = soft(0)
    for c in range(1, n):
        if parents[c] != node:
            continue
        x = tokens[c]
        inside = 0 <= x < V
        if temp == 0:
            good = x == int(logits[node].argmax())
        else:
            a, b = u[c] * (1.0 if probs is None or not inside else float(probs[node, x])), float(p[x]) if inside else 0.0
            good = a < b
            near = min(near, abs(a - b) / max(a, b)) if max(a, b) > 0 else near
        if good:
            node = c
            rows.append(c)
            p = soft(c)
        elif temp:
            left = p.clone()
            if probs is not None:
                left = (p - probs[node]).clamp(min=0)
            elif inside:
                left[x] = 0
            p = left / left.sum() if left.sum() > 0 else p
    if temp == 0:
        return rows, int(logits[node].argmax()), math.inf, math.inf
    cdf = torch.cumsum(p, 0)
    t = min(V - 1, int(torch.searchsorted(cdf, cdf[-1] * u[0], right=True)))
    edge = min(float((cdf[t] - cdf[-1] * u[0]).abs()), float((cdf[t - 1] - cdf[-1] * u[0]).abs()) if t else math.inf)
    return rows, t, near, edge


def verify_case(n, V, seed, branch, dtype, draft, spread=2.0, apart=0.5):
    g, rng = gen(seed), random.Random(seed)
    common = torch.randn((n, V), generator=g, device="cuda") * spread
    logits = (common + apart * torch.randn((n, V), generator=g, device="cuda")).to(dtype)
    q = torch.softmax((common + apart * torch.randn((n, V), generator=g, device="cuda")).double(), -1).float()
    parents = [-1] + [rng.randrange(max(0, i - branch), i) for i in range(1, n)]
    if draft:
        tokens = [0] + [int(torch.multinomial(q[parents[i]].double(), 1, generator=g)) for i in range(1, n)]
    else:
        top = torch.topk(q, min(n, V), -1).indices
        tokens = [0] + [int(top[parents[i], sum(p == parents[i] for p in parents[:i])]) for i in range(1, n)]
    u = torch.rand(n, generator=g, device="cuda")
    return logits, tokens, parents, u, q if draft else None


def verify(scmx, logits, tokens, parents, u, temp, probs):
    rows, count, token = scmx.sc_draft.verify_draft(logits, torch.tensor(tokens, device="cuda"), torch.tensor(parents, dtype=torch.int32, device="cuda"), u, temp, probs)
    rows = rows.tolist()
    m = int(count)
    assert all(r == -1 for r in rows[m:])
    return rows[:m], int(token)


def check_verify(scmx, logits, tokens, parents, u, temp, probs):
    """Acceptance compares float32 weights with their sums (each relative error below 1e-5), the token float64 sums of up to 262145 weights (below 1e-10): where the
    oracle's own distances are smaller, either answer is right -> whether the inputs decided all."""
    rows, token, near, edge = verify_oracle(logits, tokens, parents, u.double().tolist(), temp, probs)
    got = verify(scmx, logits, tokens, parents, u, temp, probs)
    if near > 1e-5:
        assert got[0] == rows
        if edge > 1e-10:
            assert got[1] == token
            return True
    return False


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("temp", [0.0, 0.7, 1.0, 5.0])
@pytest.mark.parametrize("n,V,branch", [(1, 1, 1), (1, 1000, 1), (2, 2, 1), (5, 33, 1), (8, 1001, 3), (21, 32000, 4), (64, 5003, 9), (64, 700, 64)])
def test_verify(scmx, n, V, branch, temp, draft, dtype):
    cases = [verify_case(n, V, 100 * seed + n, branch, dtype, draft) for seed in range(6)]
    assert sum(check_verify(scmx, *case[:4], temp, case[4]) for case in cases) >= 5


def test_verify_of_a_large_vocabulary(scmx):
    for seed in range(3):
        logits, tokens, parents, u, q = verify_case(9, 262145, seed, 2, BF, True, apart=0.2)
        assert check_verify(scmx, logits, tokens, parents, u, 1.0, q) and check_verify(scmx, logits.float(), tokens, parents, u, 0.8, None)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("temp", [0.6, 0.7, 1.3])
def test_verified_token_at_the_edges_of_its_interval(scmx, temp, dtype):
    """Random numbers within 2e-8 of an edge of the cumulative probabilities, and 1e-10 at least (what float64 sums of so many weights may be off): temperatures that
    are no float32 numbers are taken as they are."""
    V, g = 151936, gen(5)
    logits = (torch.randn((1, V), generator=g, device="cuda") * 2 + 9 * (torch.rand((1, V), generator=g, device="cuda") < 8 / V)).to(dtype)
    cdf = torch.cumsum(torch.softmax(logits[0].double() / temp, -1), 0)
    cdf /= cdf[-1].clone()
    u = cdf.float()
    near = (u.double() - cdf).abs()
    for draft in (None, torch.zeros((1, V), device="cuda")):
        some = ((near > 1e-10) & (near < 2e-8)).nonzero()[:, 0]
        some = some[:: max(1, len(some) // 60)].tolist()
        assert len(some) >= 50
        for i in some:
            want = int(torch.searchsorted(cdf, u[i:i + 1].double(), right=True))
            t = float((cdf[want] - u[i].double()).abs()), float((cdf[want - 1] - u[i].double()).abs()) if want else 1.0
            if min(t) > 1e-10:
                assert verify(scmx, logits, [0], [-1], u[i:i + 1].clone(), temp, draft) == ([0], want)


def test_verify_reads_strided_rows(scmx):
    logits, tokens, parents, u, q = verify_case(6, 1003, 4, 2, F32, True)
    want = verify(scmx, logits, tokens, parents, u, 1.0, q)
    for pad in (1, 5, 8):
        assert verify(scmx, torch.nn.functional.pad(logits, (0, pad))[:, :1003], tokens, parents, u, 1.0, torch.nn.functional.pad(q, (0, pad + 1))[:, :1003]) == want
        assert verify(scmx, torch.nn.functional.pad(logits, (pad, 0))[:, pad:], tokens, parents, u, 1.0, q) == want


def test_verify_corner_cases(scmx):
    V, inf = 50, float("inf")
    logits = torch.zeros((4, V), device="cuda")
    parents = [-1, 0, 0, 0]
    # greedy: the lowest of equal logits; -0 equals 0
    logits[:, 7], logits[:, 9] = 3.0, 3.0
    assert verify(scmx, logits, [0, 9, 7, 7], parents, None, 0.0, None) == ([0, 2], 7)
    # masked logits: -inf and the type's lowest value are never taken
    logits[:] = -inf
    logits[:, 11] = torch.finfo(torch.float32).min
    logits[:, 13] = 0.0
    u = torch.tensor([0.999, 0.0, 0.0, 0.0], device="cuda")
    assert verify(scmx, logits, [0, 11, 12, 13], parents, u, 1.0, None) == ([0, 3], 13)
    assert verify(scmx, logits.to(BF), [0, 11, 12, 13], parents, u, 1.0, None) == ([0, 3], 13)
    # nothing to choose from, and values that are no numbers: no row but the first, some token of the vocabulary
    for value in (-inf, float("nan"), inf):
        logits[:] = value
        rows, token = verify(scmx, logits, [0, 1, 2, 3], parents, u + 0.0005, 1.0, None)
        assert rows == [0] and token == 0
        rows, token = verify(scmx, logits, [0, 1, 2, 3], parents, u + 0.0005, 1.0, torch.full((4, V), 1 / V, device="cuda"))
        assert rows == [0] and token == 0
    # tokens outside the vocabulary are rejected; parents that are no earlier rows are never reached
    logits[:] = 0.0
    assert verify(scmx, logits, [0, -1, V, 2 ** 40], parents, u * 0, 1.0, None) == ([0], 0)
    assert verify(scmx, logits, [0, 1, 2, 3], [-1, 1, 77, -9], u * 0, 1.0, None) == ([0], 0)
    # the same token twice: its second row is tested on what the first left, which is nothing
    assert verify(scmx, logits, [0, 5, 5, 5], parents, torch.tensor([0.0, 0.5, 0.0, 0.0], device="cuda"), 1.0, None) == ([0], 0)
    # the draft's probabilities are the target's: every child is accepted, and u at its largest gives the last token
    q = torch.softmax(logits, -1)
    top = torch.full((4,), 1 - 2.0 ** -24, device="cuda")
    assert verify(scmx, logits, [0, 5, 6, 7], [-1, 0, 1, 2], top, 1.0, q) == ([0, 1, 2, 3], V - 1)
    # a draft that proposes what the target excludes
    logits[:, :25] = -inf
    q = torch.zeros((4, V), device="cuda")
    q[:, :25] = 1 / 25
    assert verify(scmx, logits, [0, 5, 6, 7], parents, u * 0, 1.0, q) == ([0], 25)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [50304, 262145])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_logit_that_is_no_number(scmx, value, V, dtype):
    """One NaN or +inf in a long row leaves it no probabilities, wherever it is: children are rejected, the token is 0; other rows are as ever."""
    logits = torch.randn((3, V), generator=gen(1), device="cuda").to(dtype)
    u = torch.tensor([0.7, 0.0, 0.0], device="cuda")
    for draft in (None, torch.full((3, V), 1 / V, device="cuda")):
        ok = verify(scmx, logits, [0, 5, 9], [-1, 0, 1], u, 1.0, draft)
        assert ok[0] == [0, 1, 2] and ok[1] > 0
        for at in (0, 7000, V // 2, V - 1):
            for row in range(3):
                bad = logits.clone()
                bad[row, at] = value
                rows, token = verify(scmx, bad, [0, 5, 9], [-1, 0, 1], u, 1.0, draft)
                assert rows == list(range(row + 1)) and token == 0


@pytest.mark.parametrize("draft", [False, True])
def test_verified_tokens_follow_the_target(scmx, draft):
    """The first token after the root has the target's distribution, accepted or not: 4000 trials, chi-square with 7 degrees of freedom below 35 (p = 1e-5)."""
    V, trials = 8, 4000
    g = gen(11)
    logits = torch.randn((4, V), generator=g, device="cuda") * 1.5
    q = torch.softmax(torch.randn((4, V), generator=g, device="cuda"), -1)
    p = torch.softmax(logits[0].double(), -1).cpu().numpy()
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    tokens = torch.multinomial(q[0], 3 * trials, replacement=True, generator=g).view(trials, 3)
    if not draft:
        tokens[:] = torch.tensor([2, 5, 1], device="cuda")
    tokens = torch.cat([torch.zeros((trials, 1), dtype=torch.long, device="cuda"), tokens], 1)
    u = torch.rand((trials, 4), generator=g, device="cuda")
    first = []
    for t in range(trials):
        rows, count, token = scmx.sc_draft.verify_draft(logits, tokens[t], parents, u[t], 1.0, q if draft else None)
        first.append(torch.where(count > 1, tokens[t][rows[1:2].clamp(min=0).long()], token))
    seen = np.bincount(torch.cat(first).cpu().numpy(), minlength=V)
    assert ((seen - trials * p) ** 2 / (trials * p)).sum() < 35


def test_verify_from_a_graph(scmx):
    cases = [verify_case(12, 3001, s, 3, BF, True) for s in range(4)]
    logits, tokens, _, u, q = [torch.empty_like(x) if torch.is_tensor(x) else x for x in cases[0]]
    tok, par = torch.zeros(12, dtype=torch.long, device="cuda"), torch.zeros(12, dtype=torch.int32, device="cuda")

    def put(case):
        for a, b in zip((logits, tok, par, u, q), case):
            a.copy_(b if torch.is_tensor(b) else torch.tensor(b))
    put(cases[0])
    scmx.sc_draft.verify_draft(logits, tok, par, u, 1.0, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = scmx.sc_draft.verify_draft(logits, tok, par, u, 1.0, q)
    for case in cases:
        put(case)
        graph.replay()
        rows, count, token = out
        assert (rows.tolist()[:int(count)], int(token)) == verify(scmx, *case[:4], 1.0, case[4])


# ---- a step of speculative decoding -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("int8", [False, True])
def test_a_step_of_all_of_them(scmx, int8):
    """Append the rows of a tree, attend, verify, keep the accepted rows: the cache then holds what one token after the other would have left."""
    C, D = scmx.sc_cache, scmx.sc_draft
    hq, hk, d, T, n, V = 8, 2, 64, 150, 11, 500
    q, c = attention_case(scmx, hq, hk, n, T, d, int8, extra=20)
    g = gen(2)
    parents = random_parents(random.Random(4), n)
    k, v = (torch.randn((hk, n, d), generator=g, device="cuda").to(BF) for _ in range(2))
    if int8:
        C.kv_append(k, v, c)
    else:
        c.k[:, T:T + n], c.v[:, T:T + n] = k, v
    mask = D.draft_mask(parents)
    o = C.cache_attention(q, c, 0.125, mask)
    check_attention(o, q, c, 0.125, mask)
    logits = o.float() @ torch.randn((hq * d, V), generator=g, device="cuda") * 0.2
    tokens = logits.argmax(-1)[torch.tensor([max(p, 0) for p in parents], device="cuda")]      # every first child is right
    rows, count, token = D.verify_draft(logits, tokens, torch.tensor(parents, dtype=torch.int32, device="cuda"), temperature=0)
    want, last, _, _ = verify_oracle(logits, tokens.tolist(), parents, None, 0, None)
    m = int(count)
    assert rows.tolist()[:m] == want and m > 2 and int(token) == last
    C.kv_keep([c], rows)
    c.offset += m
    path = torch.tensor(want, device="cuda")
    chain = quant_cache(scmx, hk, T + n, d, T) if int8 else scmx.host_model.KVCache(hk, d, T + n)
    for name in ("k", "v", "ks", "vs") if int8 else ("k", "v"):
        getattr(chain, name)[:, :T] = getattr(c, name)[:, :T]
    chain.offset = T
    if int8:
        C.kv_append(k[:, path], v[:, path], chain)
    else:
        chain.k[:, T:T + m], chain.v[:, T:T + m] = k[:, path], v[:, path]
    for name in ("k", "v", "ks", "vs") if int8 else ("k", "v"):
        assert torch.equal(getattr(chain, name)[:, :T + m], getattr(c, name)[:, :T + m])
    # the path's rows, as a chain, attend to the same
    check_attention(C.cache_attention(q[:, path], chain, 0.125), q[:, path], chain, 0.125, None)

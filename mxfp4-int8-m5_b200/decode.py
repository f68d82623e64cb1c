"""Batch-1 decode (token generation) with W4A8 GEMVs that read the packed 4-bit weights directly: the torch counterpart of
the reference's DecodeQwen3 / DecodeOlmoe (e2e/decode.py:29-165) over libscmx.  The linears compute the same function as
the prefill path (same INT8 activations, exact integer totals, same epilogues).

Attention at L = 1 is the library's own decode-attention kernel (attention="kernel"), which reads the sequence length on
the device, or torch's (attention="torch").  With the kernel, a whole step - embedding, every layer, output head, argmax,
position counter - is captured in one CUDA graph (`generate`) and replayed per token; the reference reaches the same end
by mx.compile'ing the halves of a step (e2e/decode.py:31-33).

fuse_prologue selects where the per-token INT8 of a GEMV input is computed in the reference (inside the GEMV or in a row
kernel); here both forms run the row kernel followed by the GEMV and give the same values, so the argument only keeps the
signature.

persistent=True (DecodeQwen3) runs all layers of a step as ONE cooperative kernel (scmx_decode_step): rows travel between
the phases of a layer as packets instead of across kernel boundaries, each CTA re-quantizes the activations it needs in
shared memory, and weights stream ahead of the phases.  Same bits as the chain of kernels; used where its limits
hold (head size 128, widths multiples of 1024 up to 6144, shares of rows that fit the multiprocessors) and attention="kernel".

DecodeDraft takes several tokens a step: a tree of drafted tokens runs through the prompt path as rows behind the cache's end, the target's probabilities
decide which of them are kept (speculative decoding).  The caches of all W4A8 decoders may be INT8 (make_cache(dtype=torch.int8)).

DecodeHybrid is the same for hybrid decoders (fused_hybrid.FusedHybrid): GEMVs on bfloat16 or float32 weights with the mixers'
one-token kernels between them, float32 activations."""
import ctypes
import weakref

import numpy as np
import torch

from . import _lib
from . import sc_cache as C
from . import sc_decode as G
from . import sc_draft as D
from . import sc_kernels as S
from . import hybrid_mixers as MX
from . import sc_mixers as X
from . import sc_moe as M_


class _Decoder:
    _mk = None                                                # persistent-kernel state, built per cache

    def __init__(self, fused, head, attention):
        self.f, self.model, self.args = fused, fused.model, fused.args
        self.head = G.head_product(fused.model if head == "model" else head)
        a = self.args
        hq, hk, d = a.num_attention_heads, a.num_key_value_heads, a.head_dim
        if attention == "kernel" and not S.DecodeAttention.supports(hq, hk, d):
            attention = "torch"
        self.attention = attention
        self.attn = S.DecodeAttention(hq, hk, d, fused.inv_freq.device) if attention == "kernel" else None
        self._graph = None

    @property
    def replayable(self):
        """Whether a step reads its position on the device, so that one captured graph serves every position."""
        return self.attn is not None

    def _attend(self, at, c, q, k, v, pos_dev):
        if k is None:                                         # an INT8 cache
            if self.attn is not None and C.attention_supported(q.shape[0], *c.k.shape[::2]):
                return C.cache_attention(q, c, at.scale, pos_dev=pos_dev)
            assert pos_dev is None, "a device-side position needs attention='kernel'"
            return self.f.sdpa(q, *C.kv_read(c, 0, c.offset + 1), at.scale, False)
        if self.attn is not None:
            return self.attn(q, c, at.scale, n_pos=None if pos_dev is not None else c.offset + 1, pos_dev=pos_dev)
        assert pos_dev is None, "a device-side position needs attention='kernel'"
        return self.f.sdpa(q, k, v, at.scale, False)

    @torch.no_grad()
    def step(self, tok, cache):
        """tok int [1, 1] -> logits [1, 1, V]; appends one position to the cache."""
        logits = self._step(tok, cache, None)
        for c in cache:
            c.offset += 1
        return logits

    @torch.no_grad()
    def generate(self, tok, cache, n):
        """Greedy decoding of n tokens after `tok` (int [1, 1]) from one captured CUDA graph replayed n times.
        Returns int64 [n]; the cache advances by n positions."""
        assert self.replayable, "graph decoding needs attention='kernel'"
        dev = tok.device
        if self._graph is None or self._graph[0] is not cache:
            offsets = [c.offset for c in cache]
            # the warm-up run below writes the cache row at `pos`: point it at the row the first real step overwrites
            tok_buf = tok.reshape(1, 1).to(torch.long).clone()
            pos = torch.full((1,), offsets[0], dtype=torch.int32, device=dev)
            count = torch.zeros(1, dtype=torch.int32, device=dev)
            chosen = torch.empty(cache[0].capacity, dtype=torch.long, device=dev)
            for c in cache:
                c.offset = 0                                   # rows and rotary positions come from `pos` on the device
            s = torch.cuda.Stream(device=dev)
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                kept = [(t, t.clone()) for c in cache for t in c.carried()]
                logits = self._step(tok_buf, cache, pos)       # warm-up outside the capture (lazy initialisations)
                self._select(logits, tok_buf, pos, count, chosen)
                for t, old in kept:                            # recurrent states must not see the warm-up token
                    t.copy_(old)
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    logits = self._step(tok_buf, cache, pos)
                    self._select(logits, tok_buf, pos, count, chosen)
            torch.cuda.current_stream().wait_stream(s)
            for c, o in zip(cache, offsets):
                c.offset = o
            self._graph = (cache, g, tok_buf, pos, count, chosen, logits, self._mk)
        # the layer table, scratch and status word that the graph names live as long as it does, whatever cache was stepped on since
        _, g, tok_buf, pos, count, chosen, _, self._mk = self._graph
        start = cache[0].offset
        assert start + n <= cache[0].capacity, "KV cache capacity exceeded"
        tok_buf.copy_(tok.reshape(1, 1))
        pos.fill_(start)
        count.zero_()
        for _ in range(n):
            g.replay()
        out = chosen[:n].clone()
        for c in cache:
            c.offset = start + n
        return out


    _call = staticmethod(_lib.call)      # the library that the decoder's kernels are in

    def _select(self, logits, tok, pos, count, chosen):
        """The next token (greedy) as the step's input and in the list of chosen ones, and the step's counters, in one kernel."""
        row = logits[:, -1].reshape(-1)
        if row.dtype not in (torch.bfloat16, torch.float32):      # a head of its own
            tok.copy_(row.argmax(-1, keepdim=True).view_as(tok))
            chosen.index_copy_(0, count.long(), tok.view(1))
            count.add_(1)
            pos.add_(1)
            return
        self._call("scmx_select_token", _lib.ptr(row), int(row.dtype == torch.float32), row.numel(), _lib.ptr(tok), _lib.ptr(pos), _lib.ptr(count),
                   _lib.ptr(chosen), chosen.numel(), _lib.stream())


class DecodeQwen3(_Decoder):
    """Built from a FusedQwen3 with epilogue="gemm" (gate/up rows interleaved for the SwiGLU epilogue)."""

    def __init__(self, fused, head="model", compiled=True, fuse_prologue=None, act_tile=None, attention="kernel",
                 persistent=True):
        assert fused.epilogue == "gemm"
        super().__init__(fused, head, attention)
        a = self.args
        fits = lambda n: n % 1024 == 0 and n <= 6144  # noqa: E731
        self.persistent = bool(persistent and self.attn is not None and a.head_dim == 128 and fits(a.hidden_size)
                               and fits(a.intermediate_size) and fits(a.num_attention_heads * a.head_dim)
                               and a.num_attention_heads <= 32 and fused.fmt == type(fused.fmt)()
                               and (not torch.cuda.is_available() or self._shares_fit(a, self.attn.nsplit, _lib.sm_count())))

    @staticmethod
    def _shares_fit(a, nsplit, n_sm):
        """Whether the one-kernel step takes n_sm multiprocessors, as a partition of the device may have fewer: each has rows of every product, at most
        384 of one, and there is one for every query head and every split of a key/value head (scmx_decode_step)."""
        hq, hk, d = a.num_attention_heads, a.num_key_value_heads, a.head_dim
        groups = [n // 4 for n in ((hq + 2 * hk) * d, 2 * a.intermediate_size, a.hidden_size)]
        return max(hk * nsplit, hq) <= n_sm <= min(groups) and 4 * -(-max(groups) // n_sm) <= 384

    def _persistent_state(self, cache):
        """Layer table (device pointers of the packed weights, norms and this cache's tensors) and scratch buffers."""
        if self._mk is not None and self._mk["cache"] is cache:
            return self._mk
        f, a = self.f, self.args
        dev = f.inv_freq.device
        table = (_lib.ScmxDecodeLayer * len(f.layers))()
        for i, (layer, ws) in enumerate(f.layers):
            t, at, c = table[i], layer.self_attn, cache[i]
            for j, g in enumerate(("qkv", "o", "gu", "down")):
                t.codes[j], t.bcodes[j], t.wscale[j] = ws[g].codes.data_ptr(), ws[g].bcodes.data_ptr(), ws[g].wscale.data_ptr()
            t.ln_in, t.ln_post = layer.input_layernorm.weight.data_ptr(), layer.post_attention_layernorm.weight.data_ptr()
            t.q_norm, t.k_norm = at.q_norm.weight.data_ptr(), at.k_norm.weight.data_ptr()
            t.k_cache, t.v_cache = c.k.data_ptr(), c.v.data_ptr()
        raw = np.frombuffer(ctypes.string_at(ctypes.addressof(table), ctypes.sizeof(table)), dtype=np.uint8).copy()
        size = _lib.lib().scmx_decode_step_scratch(a.hidden_size, a.intermediate_size, a.num_attention_heads, a.num_key_value_heads, a.head_dim, self.attn.nsplit)
        self._mk = dict(cache=cache, table=torch.from_numpy(raw).to(dev), scratch=torch.zeros(size, dtype=torch.uint8, device=dev),
                        status=torch.zeros(1, dtype=torch.int32, device=dev),
                        pos=torch.zeros(1, dtype=torch.int32, device=dev))
        return self._mk

    def check_status(self):
        """Raises if a wait of the persistent kernel timed out (synchronizes)."""
        if self._mk is not None:
            st = int(self._mk["status"].item())
            if st:
                raise _lib.ScmxError(f"persistent decode kernel: {_lib.describe_status(st)}")

    def _step_persistent(self, tok, cache, pos_dev):
        f, a = self.f, self.args
        mk = self._persistent_state(cache)
        if pos_dev is None:
            pos_dev = mk["pos"]
            pos_dev.fill_(cache[0].offset)
        hq, hk, d = a.num_attention_heads, a.num_key_value_heads, a.head_dim
        h = self.model.model.embed_tokens(tok)[0].clone()     # [1, D]; the kernel updates it in place
        _lib.call("scmx_decode_step", _lib.ptr(mk["table"]), len(f.layers), a.hidden_size, a.intermediate_size, hq, hk, d,
                  float(f.eps), float(f.layers[0][0].self_attn.scale), _lib.ptr(f.inv_freq), _lib.ptr(f.rope_cs),
                  f.rope_cs.shape[0], cache[0].k.shape[1], _lib.ptr(pos_dev), _lib.ptr(h), _lib.ptr(mk["scratch"]), self.attn.nsplit,
                  _lib.ptr(mk["status"]), _lib.stream())
        xn = S.rmsnorm_quant_n(h, self.model.model.norm.weight, f.eps, 1)[2]
        return self.head(xn[None])

    def _step(self, tok, cache, pos_dev):
        f, a = self.f, self.args
        S.set_format(f.fmt)
        if self.persistent and cache[0].k.dtype == torch.bfloat16:      # an INT8 cache takes the chain of kernels
            return self._step_persistent(tok, cache, pos_dev)
        hq, hk, d, eps = a.num_attention_heads, a.num_key_value_heads, a.head_dim, f.eps
        h = self.model.model.embed_tokens(tok)[0]             # [1, D]
        for i, (layer, ws) in enumerate(f.layers):
            at, c = layer.self_attn, cache[i]
            w = ws["qkv"]
            y = G.gemv(h, w.codes, w.bcodes, None, w.wscale, w.N, 1, pro=2, nw=layer.input_layernorm.weight, eps=eps)
            q, k, v = S.qkv_headnorm_y(y[None], at.q_norm.weight, at.k_norm.weight, eps, 1, hq, hk, d,
                                       rope=(f.inv_freq, c.offset, f.rope_cs), cache=c, pos_dev=pos_dev)
            o = self._attend(at, c, q, k, v, pos_dev)
            wo, wg, wd = ws["o"], ws["gu"], ws["down"]
            h = G.gemv(o, wo.codes, wo.bcodes, None, wo.wscale, wo.N, 2, res=h, pro=1)[None]
            act = G.gemv(h, wg.codes, wg.bcodes, None, wg.wscale, wg.N, 3, pro=2, nw=layer.post_attention_layernorm.weight,
                         eps=eps)
            h = G.gemv(act[None], wd.codes, wd.bcodes, None, wd.wscale, wd.N, 2, res=h, pro=1)[None]
        xn = S.rmsnorm_quant_n(h, self.model.model.norm.weight, eps, 1)[2]
        return self.head(xn[None])


class DecodeOlmoe(_Decoder):
    """Built from a FusedOlmoe: the expert GEMVs gather the top-k experts' rows themselves."""

    def __init__(self, fused, head="model", compiled=True, fuse_prologue=False, o_tile=None, attention="kernel"):
        super().__init__(fused, head, attention)
        assert not self.args.norm_topk_prob
        self.pos = torch.arange(self.args.num_experts_per_tok, dtype=torch.int32, device=fused.inv_freq.device)

    def _step(self, tok, cache, pos_dev):
        f, a = self.f, self.args
        H, d, D, eps = a.num_attention_heads, a.head_dim, a.hidden_size, f.eps
        F2, k = 2 * a.intermediate_size, a.num_experts_per_tok
        h = self.model.model.embed_tokens(tok)[0]
        row = out = None
        for i, (layer, ws, ex) in enumerate(f.layers):
            at, c = layer.self_attn, cache[i]
            w, wo = ws["qkv"], ws["o"]
            if row is None:
                y = G.gemv(h, w.codes, w.bcodes, None, w.wscale, 3 * H * d, 1, pro=2, nw=layer.input_layernorm.weight, eps=eps)
            else:
                y = G.gemv(row[0], w.codes, w.bcodes, row[1], w.wscale, 3 * H * d, 1)
            q, kk, v = S.qkv_fullnorm_y(y[None], at.q_norm.weight, at.k_norm.weight, eps, 1, H, d,
                                        rope=(f.inv_freq, c.offset, f.rope_cs), cache=c, pos_dev=pos_dev)
            o = self._attend(at, c, q, kk, v, pos_dev)
            h = G.gemv(o, wo.codes, wo.bcodes, None, wo.wscale, D, 2, res=h, pro=1)[None]
            pn = layer.post_attention_layernorm.weight
            xq, xs, inds, scores = f.norm_route_token(layer, h)
            e = inds.reshape(-1)
            (cg, bg, sg), (cd, bd, sd) = ex["gu"], ex["down"]
            act = G.gemv(xq, cg, bg, xs, sg, F2, 3, eidx=e, xstride=0)            # [k, F]
            yd = G.gemv(act, cd, bd, None, sd, D, 1, eidx=e, xstride=1, pro=1)    # [k, D], per-row INT8 in the prologue
            # the sum of the experts' rows and the norm that follows: the next layer's INT8 row, or the output head's row
            last = i + 1 == len(f.layers)
            nn = self.model.model.norm.weight if last else f.layers[i + 1][0].input_layernorm.weight
            if D <= 8192:
                h, *row, out = M_.combine_norm(yd, self.pos, scores, h, nn, eps, quant=not last, normed=last)
            else:
                h = M_.moe_combine(yd, self.pos, scores, h, pn, eps, 1, quant=False)[0]
        return self.head((S.rmsnorm_quant_n(h, self.model.model.norm.weight, eps, 1)[2] if out is None else out)[None])


class LookupDraft:
    """Drafts without a model: continuations of earlier places of the text that end in the same tokens.  A call takes the tokens so far and the most rows that may
    be drafted, and returns (tokens, parents) of a tree whose row 0 is the last token: up to `places` latest places that share the last `match` (or
    fewer) tokens, `length` tokens from each, equal beginnings shared."""

    def __init__(self, match=3, length=8, places=2):
        assert match >= 1 and length >= 1 and places >= 1
        self.match, self.length, self.places = match, length, places

    def __call__(self, text, most):
        rows, parents, children = [text[-1]], [-1], {}
        last = text[-1]
        ends = [i for i in range(len(text) - 1, 0, -1) if text[i - 1] == last]      # behind each earlier place of the last token, the latest first
        for m in range(min(self.match, len(text) - 1), 0, -1):
            tail, found = text[-m:], 0
            for e in ends:
                if e < m or text[e - m:e] != tail:
                    continue
                at = 0
                for t in text[e:e + self.length]:
                    nxt = children.get((at, t))
                    if nxt is None:
                        if len(rows) >= most:
                            return rows, parents
                        nxt = children[at, t] = len(rows)
                        rows.append(t)
                        parents.append(at)
                    at = nxt
                found += 1
                if found == self.places:
                    break
            if found:
                break
        return rows, parents


def _reference(x):
    """A weak reference, or a strong one to what has none (a SimpleNamespace)."""
    try:
        return weakref.ref(x)
    except TypeError:
        return lambda: x


class DecodeDraft:
    """Speculative decoding over a FusedQwen3 or FusedOlmoe: `propose` drafts a tree of tokens, one pass of the model reads all its rows, and verify_draft
    keeps a path of them and draws the token after it, distributed as the model alone would draw (greedy at temperature 0).

    propose(tokens so far, most rows) -> (tokens, parents) or (tokens, parents, probs): sc_draft.DraftTree's lists with row 0 the last token, and probs float32
    [rows, vocabulary] on the device where children were drawn from them (row i: what row i's children were drawn from).

    Where the model reads that many rows on digit planes (nothing beside the current stream, no buffers of its own), the second pass of as many rows
    over a cache is captured and later ones are replays (of up to 8 caches that take turns): the launches of a pass over 28 layers take the host 4.5 ms."""

    CACHES = 8            # caches that are read in turn keep their captured passes

    def __init__(self, fused, propose=None):
        a = fused.args
        if not hasattr(a, "num_key_value_heads"):
            raise ValueError(f"drafts are read by FusedQwen3 and FusedOlmoe, not by {type(fused).__name__}")
        if not C.attention_supported(a.num_attention_heads, a.num_key_value_heads, a.head_dim):
            raise ValueError(f"attention of drafted rows: head size {a.head_dim} (64 or 128)")
        self.f, self.propose = fused, propose or LookupDraft()
        self.dev = fused.inv_freq.device
        self._graphs, self._kept = None, []                       # of the cache read last, and of others: (layers, where their tensors are, {(rows, temperature): captured pass}, memory pool)

    @torch.no_grad()
    def read(self, tokens, tree, cache):
        """Logits [n, V] after every row of a tree (tokens int64 [n]); its rows are behind the cache's end."""
        h = self.f.hidden(tokens.view(1, -1), cache, tree)
        return self.f.logits(h)[0]

    def _pass(self, tok, tree, cache, u, temperature, probs):
        """A tree read, verified and its accepted rows moved -> int64 [n + 1]: the accepted rows (padded with -1), and the token after them."""
        logits = self.read(tok, tree, cache)
        rows, _, token = D.verify_draft(logits, tok, tree.parents, u, temperature, probs)
        C.kv_keep(cache, rows, pos_dev=tree.pos)
        return torch.cat((rows.long(), token))

    def _captured(self, tokens, parents, cache, u, temperature):
        """_pass as a replay, or None where it runs launch by launch."""
        n, f, a = len(tokens), self.f, self.f.args
        if not f._f4(n) or (cache[0].k.dtype == torch.int8 and a.num_attention_heads + 2 * a.num_key_value_heads > 96):
            return None
        known, pool = self._passes(cache)
        key = (n, float(temperature))
        if key not in known:
            known[key] = None
            return None
        values = torch.tensor([*tokens, *D.mask_bits(parents), *parents, *D.draft_depths(parents), cache[0].offset], dtype=torch.int64)
        if known[key] is None:
            known[key] = self._capture(parents, cache, temperature, values.to(self.dev), u, pool)
        g, inputs, numbers, out = known[key][:4]
        inputs.copy_(values)
        if numbers is not None:
            numbers.copy_(u)
        g.replay()
        return out

    def _passes(self, cache):
        """The captured passes over a cache and their memory pool.  They name its layers' tensors: others in their place, or other layers in the list, are another cache."""
        where = [(c.k.shape, *(t.data_ptr() for t in ((c.k, c.v, c.ks, c.vs) if c.k.dtype == torch.int8 else (c.k, c.v)))) for c in cache]
        same = lambda e: e[1] == where and all(r() is c for r, c in zip(e[0], cache))      # noqa: E731
        entry = next((e for e in self._kept if same(e)), None)
        self._kept = [e for e in self._kept if e is not entry and all(r() is not None for r in e[0])]      # a cache that is gone takes its passes along
        if entry is None or len(entry[2]) >= 128:                                                          # (128: temperatures that keep changing)
            entry = (tuple(map(_reference, cache)), where, {}, torch.cuda.graph_pool_handle())
        self._kept = self._kept[1 - self.CACHES:] + [entry]
        self._graphs = entry
        return self._graphs[2:]

    def _capture(self, parents, cache, temperature, inputs, u, pool):
        """(graph, its inputs int64 [4 n + 1]: tokens, mask, parents, depths, position; its random numbers; its result; what it reads).  The warm-up is this very pass."""
        n = len(parents)
        tree, ints, out = D.DraftTree(parents, self.dev), torch.empty(2 * n + 1, dtype=torch.int32, device=self.dev), torch.empty(n + 1, dtype=torch.int64, device=self.dev)
        tok, tree.mask, (tree.parents, tree.depths, tree.pos) = inputs[:n], inputs[n:2 * n], ints.split((n, n, 1))
        numbers = None if u is None else u.clone()

        def run():
            ints.copy_(inputs[2 * n:])
            out.copy_(self._pass(tok, tree, cache, numbers, temperature, None))

        offsets = [c.offset for c in cache]
        s = torch.cuda.Stream(device=self.dev)
        s.wait_stream(torch.cuda.current_stream())
        for c in cache:
            c.offset = 0                                          # rows and rotary positions come from the position on the device
        try:
            with torch.cuda.stream(s):
                run()
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s, pool=pool):
                    run()
        finally:
            for c, o in zip(cache, offsets):
                c.offset = o
        torch.cuda.current_stream().wait_stream(s)
        return g, inputs, numbers, out, tree, ints

    @torch.no_grad()
    def step(self, text, cache, temperature=0.0, u=None, most=D.MAX_ROWS):
        """One pass: text (list of ids, the last one not in the cache yet) -> the tokens that it adds, at least one.  u float32 [64] on the model's device: random numbers in [0, 1)."""
        assert cache[0].offset + 1 <= cache[0].capacity, "KV cache capacity exceeded"
        most = max(1, min(most, D.MAX_ROWS, cache[0].capacity - cache[0].offset))
        tokens, parents, *probs = self.propose(text, most)
        tokens, parents = [int(t) for t in tokens], D.check_tree(parents)
        n = len(tokens)
        if n != len(parents) or n > most or tokens[0] != text[-1]:
            raise ValueError(f"a draft of {n} tokens and {len(parents)} parents: as many of both, {most} at most, the first token the text's last")
        if not all(0 <= t < self.f.args.vocab_size for t in tokens):
            raise ValueError(f"drafted tokens {tokens}: 0 .. {self.f.args.vocab_size - 1}")
        if temperature and (u is None or u.dim() != 1 or u.numel() < n):
            raise ValueError(f"temperature {temperature}: 0, or random numbers for {n} rows")
        if temperature and (u.dtype != torch.float32 or u.device != self.dev):      # here: a replay would copy them, rounded, from wherever they are
            raise TypeError(f"random numbers {u.dtype} on {u.device}: float32 on {self.dev}")
        u = u[:n].contiguous() if temperature else None
        probs = probs[0] if probs else None
        out = self._captured(tokens, parents, cache, u, temperature) if probs is None else None
        if out is None:
            out = self._pass(torch.tensor(tokens, dtype=torch.int64, device=self.dev), D.DraftTree(parents, self.dev), cache, u, temperature, probs)
        *path, last = out.tolist()
        path = [r for r in path if r >= 0]
        for c in cache:
            c.offset += len(path)
        return [tokens[r] for r in path[1:]] + [last]

    @torch.no_grad()
    def generate(self, tok, cache, n, text=(), temperature=0.0, generator=None):
        """n tokens after `tok` (int [1, 1]), as _Decoder.generate; text: the tokens before it, which proposals may look into.  Returns int64 [n]; the cache advances
        by n positions.  temperature > 0 draws from `generator` (torch.Generator on the device, or None)."""
        assert cache[0].offset + n <= cache[0].capacity, "KV cache capacity exceeded"
        text = list(text) + [int(tok)]
        start, have = cache[0].offset, len(text)
        while len(text) - have < n:
            left = n - (len(text) - have)
            u = torch.rand(D.MAX_ROWS, device=self.dev, generator=generator) if temperature else None
            text += self.step(text, cache, temperature, u, left)      # a pass of `left` rows adds at most as many tokens
        assert cache[0].offset == start + n
        return torch.tensor(text[have:], dtype=torch.int64, device=self.dev)


def _row(row, in_parts):
    """A row for its reader: as it is left, or joined."""
    return row if in_parts or not isinstance(row, X.RowParts) else row.joined()


class DecodeHybrid(_Decoder):
    """Built from a FusedHybrid.  Activations of a step are float32 vectors in buffers that live with the decoder."""
    replayable = True
    _call = staticmethod(_lib.mcall)

    def __init__(self, fused):
        self.f, self.model, self.args, self._graph = fused, fused.model, fused.args, None
        dev, a = fused.model.device, self.args
        f32 = lambda *s: torch.empty(s, dtype=torch.float32, device=dev)    # noqa: E731
        # the residual row: a product that joins it reads one buffer and writes the other
        self.x, self.y = (f32(1, a.hidden_size), f32(1, a.hidden_size)), f32(1, a.hidden_size)
        if not a.design.prenorm:     # the embedding's and every layer's result, for the depth average
            self.xs = f32(len(a.layers) + 1, 1, a.hidden_size)
        own = {}
        for ly in fused.layers:
            if ly not in own:
                own[ly] = ly.mixer.buffers(dev)
                if ly.w_up is not None:
                    own[ly]["u"] = f32(ly.w_up.N // (2 if ly.act.code == 2 else 1))
        self.bufs = [own[ly] for ly in fused.layers]

    def _mix(self, ly, b, x, c, pos_dev):
        x = _row(x, MX.reads_parts(ly.mixer))
        return ly.mixer.w_o.vec(ly.mixer.step(self.f, x, c, b, pos_dev), out=self.y.view(-1))

    def _step(self, tok, cache, pos_dev):
        f = self.f
        f.ensure_positions(cache[0].capacity)
        assert pos_dev is not None or cache[0].offset < cache[0].capacity, "KV cache capacity exceeded"
        row = (self._prenorm if self.args.design.prenorm else self._postnorm)(tok.view(-1), cache, pos_dev)
        return f.head.vec(_row(row, X.reads_parts(f.head)))[None, None]

    def _prenorm(self, tok, cache, pos_dev):
        f, (x, spare), y, mult = self.f, self.x, self.y, self.args.residual_mult
        f.embed(tok, cache, x)
        nl = len(f.layers)
        row = X.RowParts(x, None, f.layers[0].norm1 if nl else f.final_norm, mult, f.eps, None)
        for i, (ly, b, c) in enumerate(zip(f.layers, self.bufs, cache)):
            after = f.layers[i + 1].norm1 if i + 1 < nl else f.final_norm
            self._mix(ly, b, row, c, pos_dev)
            row, x, spare = X.RowParts(x, y, after if ly.w_up is None else ly.norm2, mult, f.eps, spare), spare, x
            if ly.w_up is not None:
                ly.feed_forward_vec(_row(row, ly.feed_reads_parts()), b["u"], y.view(-1))
                row, x, spare = X.RowParts(x, y, after, mult, f.eps, spare), spare, x
        return row

    def _postnorm(self, tok, cache, pos_dev):
        f, y, nl = self.f, self.y, len(self.f.layers)
        f.embed(tok, cache, self.xs[0])
        x, row, turn = self.xs[0], self.xs[0].view(-1), 0
        if nl == 0:
            return X.norm_rows(x, f.final_norm, f.eps, torch.float32).view(-1)
        for i, (ly, b, c) in enumerate(zip(f.layers, self.bufs, cache)):
            self._mix(ly, b, row, c, pos_dev)
            last = i + 1 == nl
            norm = ly.norm1
            if ly.w_up is not None:
                row, x, turn = X.RowParts(x, y, norm, 1.0, f.eps, self.x[turn], ()), self.x[turn], 1 - turn
                ly.feed_forward_vec(_row(row, ly.feed_reads_parts()), b["u"], y.view(-1))
                norm = ly.norm2
            row = X.RowParts(x, y, norm, 1.0, f.eps, self.x[turn], (self.xs, ly.dwa, not last), f.final_norm if last else None)
            x, turn = self.x[turn], 1 - turn
        return row

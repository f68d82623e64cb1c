"""Trees of drafted tokens: their attention masks, and the check of the drafts against the target's probabilities.

A tree of n rows is a list of parents: row 0 is the last chosen token (parent -1), row c continues row parents[c] < c.  The rows of
a chain are -1, 0, 1, .."""
import torch

from . import _lib
from .sc_cache import MAX_ROWS


def check_tree(parents):
    """The list of parents; raises if it is no tree of 1 .. 64 rows."""
    parents = [int(p) for p in parents]
    if not 1 <= len(parents) <= MAX_ROWS or parents[0] != -1 or any(not 0 <= p < i for i, p in enumerate(parents) if i):
        raise ValueError(f"parents {parents}: 1 .. {MAX_ROWS} rows, the first -1, every other an earlier row")
    return parents


def mask_bits(parents):
    """draft_mask's entries as a list."""
    bits = []
    for i, p in enumerate(check_tree(parents)):
        bits.append((bits[p] if i else 0) | 1 << i)
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def draft_mask(parents, device="cuda"):
    """int64 [n]: bit j of entry i is set where j is row i's ancestor or i itself (sc_cache.cache_attention)."""
    return torch.tensor(mask_bits(parents), dtype=torch.int64, device=device)


def draft_depths(parents):
    """How many rows are above each row: its position counted from row 0's."""
    out = []
    for i, p in enumerate(check_tree(parents)):
        out.append(out[p] + 1 if i else 0)
    return out


class DraftTree:
    """A tree's parents, and what the kernels read of it, on the device: parents int32 [n], mask (draft_mask) and depths int32 [n] (draft_depths).  pos, if set: one
    device int32, the cache row of the tree's first row; it is added to the caches' offsets where keys are written, and read in their place by
    the attention, so that a captured pass can be replayed (caches at offset 0 then)."""
    __slots__ = ("list", "parents", "mask", "depths", "pos")

    def __init__(self, parents, device="cuda"):
        self.pos = None
        self.list = check_tree(parents)
        self.mask = draft_mask(self.list, device)
        self.parents, self.depths = torch.tensor([self.list, draft_depths(self.list)], dtype=torch.int32, device=device).unbind()

    def __len__(self):
        return len(self.list)


_LOGITS, _PROBS = (torch.bfloat16, torch.float32), (torch.float32,)


def _rows(x, what, dtypes):
    if x.dim() != 2 or x.dtype not in dtypes:
        raise ValueError(f"{what} {tuple(x.shape)} {x.dtype}: [rows, vocabulary], {' or '.join(map(str, dtypes))}")
    return x if x.stride(1) == 1 and x.stride(0) >= x.shape[1] else x.contiguous()


def verify_draft(logits, tokens, parents, u=None, temperature=1.0, probs=None):
    """Which drafted rows the target accepts, and the token after them -> (rows int32 [n]: the accepted ones, first 0, then -1; count int32
    [1]; token int64 [1]), all on the device.

    logits [n, V], bfloat16 or float32: the target's after every row; tokens int64 [n], parents int32 [n].  At a node, p = softmax(logits /
    temperature), children are tested in ascending order: c is accepted if u[c] q(x) < p(x) for its token x; a rejected one leaves
    p <- max(p - q, 0) / Z.  q: probs[node] (float32 [n, V]; the children were drawn from it independently), or, without probs, 1
    at the child's token and 0 elsewhere.  At the path's end the token is the first whose cumulative p exceeds u[0].  u float32 [n], uniform in [0, 1).
    So the accepted tokens and the last one are distributed as if the target had chosen each of them.
    temperature 0: greedy (the lowest index of equal logits, a NaN the largest), u and probs are not read.  By temperature a row with a NaN or +inf, or nothing but -inf, has
    no probabilities: its children are rejected, and the token after it is 0."""
    logits = _rows(logits, "logits", _LOGITS)
    n, V = logits.shape
    if not 1 <= n <= MAX_ROWS:
        raise ValueError(f"{n} rows (1 .. {MAX_ROWS})")
    if tokens.dtype != torch.int64 or tokens.numel() != n or parents.dtype != torch.int32 or parents.numel() != n:
        raise ValueError(f"tokens {tuple(tokens.shape)} {tokens.dtype}, parents {tuple(parents.shape)} {parents.dtype}: int64 and int32 [{n}]")
    _lib.require_here(tokens, parents)
    _lib.require_here(logits, contiguous=False)
    numbers = drafts = None
    ldp = 0
    if temperature != 0:
        if u is None or not temperature > 0:
            raise ValueError(f"temperature {temperature}: 0, or positive with random numbers")
        _lib.require_here(u)
        if u.dtype != torch.float32 or u.numel() != n:
            raise ValueError(f"random numbers {tuple(u.shape)} {u.dtype}: float32 [{n}]")
        numbers = u.data_ptr()
        if probs is not None:
            probs = _rows(probs, "probs", _PROBS)
            _lib.require_here(probs, contiguous=False)
            if probs.shape != logits.shape:
                raise ValueError(f"probs {tuple(probs.shape)} for logits {tuple(logits.shape)}")
            drafts, ldp = probs.data_ptr(), max(probs.stride(0), V)
    rows, count, token = parents.new_empty(n), parents.new_empty(1), tokens.new_empty(1)
    size = _lib.lib().scmx_verify_scratch(n, V)
    scratch = tokens.new_empty(size // 8)
    _lib.call("scmx_verify", logits.data_ptr(), logits.dtype == torch.float32, max(logits.stride(0), V), tokens.data_ptr(), parents.data_ptr(), numbers,
              temperature, drafts, ldp, n, V, rows.data_ptr(), count.data_ptr(), token.data_ptr(), scratch.data_ptr(), size, _lib.stream())
    return rows, count, token

"""Key ranges of the common attention masks for `ops.range_attention`: row i sees the keys
lo[i] <= j < hi[i].  Each function returns int32 tensors on `device`; they are plain tensors, so a
caller may also build or update them in place (a captured graph reads them at every replay)."""
from __future__ import annotations

import torch


def _out(*ts, device):
    return tuple(t.to(torch.int32).contiguous().to(device) for t in ts)


def document_ranges(lengths, device, *, block=0, prefix=None, window=0):
    """(lo, hi), each [sum(lengths)], for documents packed one after the other.

    block 0: every token of a document sees the whole document; block n: its own block of n tokens
    and the earlier ones (1 = causal order, tokens per latent frame = frame-causal).  prefix (one
    number, or one per document): the first `prefix` tokens of a document are seen by all of it.
    window w > 0: keys more than w - 1 tokens before the row (without a block also after it) are
    not seen, the prefix included."""
    n = [int(x) for x in lengths]
    if any(x < 0 for x in n) or block < 0 or window < 0:
        raise ValueError("document_ranges: lengths, block and window must be >= 0")
    pre = [0 if prefix is None else int(prefix)] * len(n) if not hasattr(prefix, "__len__") else [int(x) for x in prefix]
    if len(pre) != len(n) or any(x < 0 for x in pre):
        raise ValueError("document_ranges: prefix must be one number >= 0 or one per document")
    count = torch.tensor(n, dtype=torch.int64)
    end = count.cumsum(0)
    start = (end - count).repeat_interleave(count)
    pre = torch.tensor(pre, dtype=torch.int64).repeat_interleave(count)
    end = end.repeat_interleave(count)
    i = torch.arange(start.numel())
    hi = end
    if block:
        hi = torch.minimum(torch.maximum(start + ((i - start) // block + 1) * block, start + pre), end)
    lo = start
    if window:
        lo = torch.maximum(start, i - window + 1)
        if not block:
            hi = torch.minimum(end, i + window)
    return _out(lo, hi, device=device)


def padded_ranges(lengths, q_len, device):
    """(lo, hi), each [len(lengths), q_len]: row i < lengths[b] sees the keys 0 .. lengths[b] - 1,
    the padded rows behind see nothing (and come out as zeros)."""
    n = torch.as_tensor(lengths, dtype=torch.int64).cpu()[:, None]
    if bool((n < 0).any()) or bool((n > q_len).any()):
        raise ValueError("padded_ranges: lengths must lie in 0..q_len")
    hi = torch.where(torch.arange(q_len)[None] < n, n, torch.zeros_like(n))
    return _out(torch.zeros_like(hi), hi, device=device)


def cache_ranges(kv_lens, q_len, *, window=0):
    """(lo, hi, pos), each [B, q_len], for queries that are the last q_len tokens of caches holding
    kv_lens[b] keys (int32 tensor [B] on the device), in causal order; window w > 0: the last w keys
    only.  All on the tensor's device, without waiting for it."""
    if q_len < 0 or window < 0:
        raise ValueError("cache_ranges: q_len and window must be >= 0")
    pos = kv_lens.to(torch.int32)[:, None] - q_len + torch.arange(q_len, dtype=torch.int32, device=kv_lens.device)[None]
    hi = pos + 1
    lo = (hi - window).clamp_min(0) if window else torch.zeros_like(hi)
    return lo.contiguous(), hi.contiguous(), pos.contiguous()

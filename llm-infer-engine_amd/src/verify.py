"""Verification of drafted tokens: which of a draft's tokens the target model keeps,
and the token after them.

The reference draws one token a step on the host (src/sampler.py:4-33).  A step over
several drafted tokens (Llama3.forward with a ``PagedKVCache`` and
``return_all_logits=True``) has the target's logits after each of them;
``verify_drafts`` keeps the longest prefix that rejection sampling accepts and
draws the next token, such that the tokens kept are distributed as the target's
own, whatever proposed them.  It runs on the device (mi_verify_drafts, no host
sync) from random numbers that the caller draws.
"""
from __future__ import annotations

import torch

from . import _lib
from .paged import _device_of, _per_row


def verify_drafts(target_logits, draft_tokens, accept_u=None, sample_u=None, *,
                  draft_logits=None, temperature: float = 1.0, draft_lens=None):
    """(tokens [B, S + 1] int64, accepted [B] int64) of S drafted tokens per row.

    target_logits: [B, S + 1, V], row i the target's logits after the first i drafts;
    draft_tokens: [B, S] int64; accept_u [B, S] and sample_u [B]: fp32 random numbers
    in [0, 1).  draft_logits: [B, S, V] that the drafts were drawn from at this
    temperature (None: drafts that were looked up, each with probability 1).

    With p_i and q_i the softmax of target and draft logits over ``temperature``,
    draft i is accepted iff accept_u[i] * q_i(x_i) < p_i(x_i) and all before it were.
    tokens holds the accepted drafts, then the least token j with cumsum(w)[j] >
    sample_u * sum(w), then -1; w = max(p_n - q_n, 0) for a refused draft n (p_n if
    that is 0 everywhere), p_n where none was refused.  temperature 0 is greedy: a draft
    is accepted iff it is the first largest target logit, and no random numbers or
    draft logits are read.  draft_lens (device int64 [B]): a row's first
    draft_lens[b] drafts count.  NaN logits count as -inf; a row of -inf alone
    refuses its draft and gives -1, as does no token of the vocabulary.
    """
    what = "verify_drafts"
    if target_logits.dim() != 3 or draft_tokens.dim() != 2:
        raise ValueError(f"{what}: target_logits must be [B, S + 1, V] and draft_tokens [B, S], got "
                         f"{tuple(target_logits.shape)} and {tuple(draft_tokens.shape)}")
    B, S = draft_tokens.shape
    V = target_logits.shape[2]
    if target_logits.shape[:2] != (B, S + 1):
        raise ValueError(f"{what}: target_logits {tuple(target_logits.shape)} must have {S + 1} rows "
                         f"for each of the {B} rows of drafts")
    if S < 1 or V < 1:
        raise ValueError(f"{what}: needs at least one draft and one token, got S={S}, V={V}")
    if draft_tokens.dtype != torch.int64:
        raise TypeError(f"{what}: draft_tokens must have dtype torch.int64, got {draft_tokens.dtype}")
    temperature = float(temperature)
    if not (temperature == 0.0 or 1e-3 <= temperature <= 1e6):
        raise ValueError(f"{what}: temperature must be 0 or between 1e-3 and 1e6, got {temperature}")
    greedy = temperature == 0.0
    code = _lib.dtype_code(target_logits.dtype)
    if greedy:
        draft_logits = accept_u = sample_u = None
    else:
        for t, shape, name in ((accept_u, (B, S), "accept_u"), (sample_u, (B,), "sample_u")):
            if t is None:
                raise ValueError(f"{what}: {name} is needed at temperature {temperature}")
            if tuple(t.shape) != shape or t.dtype != torch.float32:
                raise ValueError(f"{what}: {name} must be float32 {shape}, got {t.dtype} "
                                 f"{tuple(t.shape)}")
    if draft_logits is not None:
        if draft_logits.shape != (B, S, V):
            raise ValueError(f"{what}: draft_logits must be {(B, S, V)}, got "
                             f"{tuple(draft_logits.shape)}")
        if draft_logits.dtype != target_logits.dtype:
            raise TypeError(f"{what}: draft_logits dtype {draft_logits.dtype} must match "
                            f"target_logits {target_logits.dtype}")
    index = _device_of(what, *[t for t in (target_logits, draft_tokens, accept_u, sample_u,
                                           draft_logits) if t is not None])
    draft_lens = _per_row(draft_lens, B, index, "draft_lens", what)
    if target_logits.stride(2) != 1:
        target_logits = target_logits.contiguous()
    if draft_logits is not None and draft_logits.stride(2) != 1:
        draft_logits = draft_logits.contiguous()
    if sample_u is not None and sample_u.stride(0) != 1:
        sample_u = sample_u.contiguous()
    lib = _lib.load()
    # (int64, on the device: tokens, counts and the workspace's 8-byte words)
    tokens, accepted = draft_tokens.new_empty((B, S + 1)), draft_tokens.new_empty((B,))
    if B == 0:
        return tokens, accepted
    ts, xs = target_logits.stride(), draft_tokens.stride()
    ds = (0, 0) if draft_logits is None else draft_logits.stride()
    us = (0, 0) if accept_u is None else accept_u.stride()
    with _lib.on_device(index):
        n = lib.mi_verify_drafts_workspace(B, S, V)
        ws = draft_tokens.new_empty((n // 8 + 1,))
        st = lib.mi_verify_drafts(
            target_logits.data_ptr(), _lib.ptr(draft_logits), draft_tokens.data_ptr(),
            _lib.ptr(accept_u), _lib.ptr(sample_u), _lib.ptr(draft_lens), tokens.data_ptr(),
            accepted.data_ptr(), ws.data_ptr(), n, B, S, V, ts[0], ts[1], ds[0], ds[1],
            xs[0], xs[1], us[0], us[1], temperature, code, torch._C._cuda_getCurrentRawStream(index))
    if st:
        _lib.check(st, what)
    return tokens, accepted

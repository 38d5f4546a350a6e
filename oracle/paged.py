"""CPU restatement of the paged KV cache: append, attention over it, and the
verification of drafted tokens.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  No counterpart in the
reference; the definitions are those of include/miattn.h.  Rotation in fp32 as
oracle.rope.rotate, everything else in 64 bits, in plain loops.
"""
from __future__ import annotations

import math

import torch

from . import rope

E4M3 = torch.float8_e4m3fn
MIN_EXP = -120


def page_scale(a: float) -> float:
    """Least power of two >= 2^-120 with a <= 448 * it."""
    e = MIN_EXP
    if a > 0:
        _, x = math.frexp(a / 448.0)     # a / 448 = f 2^x, 1/2 <= f < 1
        e = max(e, x - 1 if math.ldexp(1.0, x - 1) * 448.0 >= a else x)
    return math.ldexp(1.0, e)


def to_e4m3(x: torch.Tensor, scale: float) -> torch.Tensor:
    """fp32 x / scale as e4m3; NaN for what is not finite."""
    y = (x.double() / scale).float()
    return torch.where(torch.isfinite(y), y, torch.full_like(y, math.nan)).to(E4M3)


def _largest(x: torch.Tensor) -> float:
    f = torch.isfinite(x)
    return float(x[f].abs().max()) if bool(f.any()) else 0.0


def append(k, v, scales, table, start, lens, xk, xv, cos, sin):
    """Copies of the pages k [n, H, P, D], v [n, H, D, P] (and scales) after the append of
    xk, xv [B, H, S, D]: start, lens lists of ints."""
    k, v = k.clone(), v.clone()
    scales = None if scales is None else scales.clone()
    B, H, S, D = xk.shape
    P, slots = k.shape[2], table.shape[1]
    for b in range(B):
        places: dict[int, list[tuple[int, int]]] = {}
        for s in range(min(S, max(0, lens[b]))):
            pos = start[b] + s
            if 0 <= pos < slots * P:
                places.setdefault(pos // P, []).append((pos % P, s))
        for slot, toks in places.items():
            page = int(table[b, slot])
            if not 0 <= page < k.shape[0]:
                continue
            off = [o for o, _ in toks]
            s = [t for _, t in toks]
            rows = [min(max(start[b] + t, 0), cos.shape[0] - 1) for t in s]
            kr = rope.rotate(xk[b][:, s].float(), cos[rows], sin[rows])      # fp32, [H, m, D]
            vr = xv[b][:, s].float()
            for h in range(H):
                if scales is None:
                    k[page, h, off] = kr[h].to(k.dtype)
                    v[page, h][:, off] = vr[h].to(v.dtype).T
                    continue
                for c, (x, part) in enumerate(((kr[h], k[page, h]), (vr[h], v[page, h].T))):
                    sc = page_scale(_largest(x))
                    if off[0] > 0:
                        old = float(scales[page, h, c])
                        sc = max(sc, old)
                        part[:off[0]] = to_e4m3(part[:off[0]].float() * (old / sc), 1.0)
                    part[off] = to_e4m3(x, sc)
                    scales[page, h, c] = sc
    return k, v, scales


def values(k, v, scales):
    """The pages' entries in 64 bits, V as [n, H, P, D]."""
    k, v = k.double(), v.double().transpose(2, 3)
    if scales is not None:
        k = k * scales[..., 0, None, None].double()
        v = v * scales[..., 1, None, None].double()
    return k, v


def attend(q, k, v, scales, table, seq_lens, query_lens=None, sm_scale=None):
    """out, lse, and per output sum_j p_j |v_j| (what rounding errors of p scale with) and
    per row the largest sum_d |q_d k_d| * scale (what errors of a score scale with)."""
    B, H, S, D = q.shape
    Hkv, P = k.shape[1], k.shape[2]
    kd, vd = values(k, v, scales)
    scale = D ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros((B, H, S, D), dtype=torch.float64)
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64)
    mass, reach = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        n = S if query_lens is None else min(S, max(0, query_lens[b]))
        for s in range(n):
            vis = min(max(0, seq_lens[b] - n + s + 1), table.shape[1] * P)
            keys = [(int(table[b, j // P]), j % P) for j in range(vis)]
            keys = [(p, o) for p, o in keys if 0 <= p < k.shape[0]]
            if not keys:
                continue
            pages, offs = (torch.tensor(x) for x in zip(*keys))
            for h in range(H):
                kk, vv = kd[pages, h // (H // Hkv), offs], vd[pages, h // (H // Hkv), offs]
                qq = q[b, h, s].double()
                z = (kk @ qq) * scale
                lse[b, h, s] = torch.logsumexp(z, 0)
                p = torch.exp(z - lse[b, h, s])
                out[b, h, s] = p @ vv
                mass[b, h, s] = p @ vv.abs()
                reach[b, h, s] = ((kk.abs() @ qq.abs()) * scale).max()
    return out, lse, mass, reach


def _probs(x, temperature):
    x = x.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    x = x.clamp(max=torch.finfo(torch.float32).max)
    if float(x.max()) == -math.inf:
        return torch.zeros_like(x)
    return torch.softmax(x / temperature, -1)


def verify(target, draft, drafted, u, r, lens, temperature):
    """tokens [B, S + 1], accepted [B] (see include/miattn.h, mi_verify_drafts)."""
    B, S = drafted.shape
    V = target.shape[2]
    tokens = torch.full((B, S + 1), -1, dtype=torch.int64)
    accepted = torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        n = S if lens is None else min(S, max(0, lens[b]))
        k, refused = 0, False
        while k < n and not refused:
            x = int(drafted[b, k])
            if temperature == 0.0:
                t = target[b, k].double().nan_to_num(nan=-math.inf, posinf=torch.finfo(torch.float32).max,
                                                     neginf=-math.inf)
                ok = float(t.max()) > -math.inf and x == int((t == t.max()).nonzero()[0])
            elif not 0 <= x < V:
                ok = False
            else:
                q = 1.0 if draft is None else float(_probs(draft[b, k], temperature)[x])
                ok = float(u[b, k]) * q < float(_probs(target[b, k], temperature)[x])
            refused = not ok
            k += ok
        accepted[b] = k
        tokens[b, :k] = drafted[b, :k]
        if temperature == 0.0:
            t = target[b, k].double().nan_to_num(nan=-math.inf, posinf=torch.finfo(torch.float32).max,
                                                 neginf=-math.inf)
            if float(t.max()) > -math.inf:
                tokens[b, k] = int((t == t.max()).nonzero()[0])
            continue
        p = _probs(target[b, k], temperature)
        w = p
        if refused:
            if draft is not None:
                q = _probs(draft[b, k], temperature)
            else:
                q = torch.zeros_like(p)
                if 0 <= int(drafted[b, k]) < V:
                    q[int(drafted[b, k])] = 1.0
            w = (p - q).clamp(min=0.0)
            w = w if float(w.sum()) > 0 else p
        c = torch.cumsum(w, 0)
        if float(c[-1]) > 0:
            over = (c > float(r[b]) * c[-1]).nonzero()
            tokens[b, k] = int(over[0]) if len(over) else int((w > 0).nonzero()[-1])
    return tokens, accepted

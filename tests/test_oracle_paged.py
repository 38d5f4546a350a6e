"""CPU: pins the paged oracle to independent statements -- the dense oracle, e4m3's own
table of values, brute force -- and shows that planted mistakes are seen."""
import math

import pytest
import torch

from helpers import randn
from oracle import attention as ora
from oracle import paged as opaged
from oracle import rope as orope

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("a,e", [(448.0, 0), (448.5, 1), (224.0, -1), (224.01, 0), (1.0, -8),
                                 (0.0, -120), (2.0 ** -140, -120), (3.4e38, 120), (0.875 * 2, -8 + 0)])
def test_page_scale(a, e):
    s = opaged.page_scale(a)
    assert s == 2.0 ** e
    assert a <= 448 * s and (e == -120 or a > 448 * s / 2)


def test_e4m3_rounds_to_the_nearest_value_ties_to_even():
    codes = torch.arange(256, dtype=torch.uint8)
    vals = codes.view(E4M3).float()
    vals = vals[torch.isfinite(vals)].unique()
    x = torch.cat((randn((4000,), 1, torch.float32) * 100, (vals[1:] + vals[:-1]) / 2, vals))
    x = x.clamp(-448, 448)
    got = opaged.to_e4m3(x, 1.0).float()
    d = (vals[None] - x[:, None]).abs()
    assert torch.equal((got - x).abs(), d.min(1).values)
    mid = (vals[1:] + vals[:-1]) / 2
    even = opaged.to_e4m3(mid, 1.0).view(torch.uint8)
    assert not (even & 1).any()
    assert torch.isnan(opaged.to_e4m3(torch.tensor([math.inf, -math.inf, math.nan]), 1.0).float()).all()


def _dense(B, H, T, D, P, seed):
    """Dense k, v [B, H, T, D] and the same as pages."""
    k, v = randn((B, H, T, D), seed), randn((B, H, T, D), seed + 1)
    slots = T // P
    table = torch.randperm(B * slots, generator=torch.Generator().manual_seed(seed)).reshape(B, slots).int()
    kp, vp = torch.empty(B * slots, H, P, D, dtype=k.dtype), torch.empty(B * slots, H, D, P, dtype=k.dtype)
    for b in range(B):
        for s in range(slots):
            kp[table[b, s]] = k[b, :, s * P:(s + 1) * P]
            vp[table[b, s]] = v[b, :, s * P:(s + 1) * P].transpose(1, 2)
    return k, v, kp, vp, table


def test_attend_equals_the_dense_oracle():
    k, v, kp, vp, table = _dense(2, 2, 64, 16, 16, 3)
    q = randn((2, 4, 1, 16), 5)
    out, lse, _, _ = opaged.attend(q, kp, vp, None, table, [64, 64])
    ref, rlse = ora.decode(q, k, v)
    assert float((out.float() - ref).abs().max()) < 1e-5
    assert float((lse[:, :, 0].float() - rlse).abs().max()) < 1e-5
    # a whole prompt at once is the causal prefill
    q = randn((2, 4, 64, 16), 6)
    out, lse, _, _ = opaged.attend(q, kp, vp, None, table, [64, 64])
    ref, rlse = ora.prefill(q, k, v)
    assert float((out.float() - ref).abs().max()) < 1e-5
    # a planted mistake: one key too many for every token
    wrong, _, _, _ = opaged.attend(q[:, :, :4], kp, vp, None, table, [5, 5])
    assert float((wrong.float() - ref[:, :, :4]).abs().max()) > 1e-2


def test_append_in_the_activations_type_equals_the_dense_append():
    B, H, T, D, P, S = 2, 2, 64, 16, 16, 9
    k, v, kp, vp, table = _dense(B, H, T, D, P, 8)
    xk, xv = randn((B, H, S, D), 10), randn((B, H, S, D), 11)
    cos, sin = orope.cos_sin(orope.freqs_cis(D, T), torch.bfloat16)
    ck, cv = orope.rope_kv_append(k[None], v[None], 0, xk, xv, cos[12:12 + S], sin[12:12 + S],
                                  start_pos=12)
    rk, rv, _ = opaged.append(kp, vp, None, table, [12, 12], [S, S], xk, xv, cos, sin)
    for b in range(B):
        for s in range(T // P):
            assert torch.equal(rk[table[b, s]], ck[0, b, :, s * P:(s + 1) * P])
            assert torch.equal(rv[table[b, s]].transpose(1, 2), cv[0, b, :, s * P:(s + 1) * P])


def test_append_in_8_bits_is_within_half_a_step():
    """Every new entry is within 2^-4 of its value or half the least step, at the page's scale."""
    B, H, D, P, S = 1, 2, 16, 16, 16
    k = torch.zeros(1, H, P, D).to(E4M3)
    xk, xv = randn((B, H, S, D), 12), randn((B, H, S, D), 13)
    cos, sin = orope.cos_sin(orope.freqs_cis(D, P), torch.bfloat16)
    rk, rv, sc = opaged.append(k, k.transpose(2, 3).contiguous(), torch.zeros(1, H, 2),
                               torch.zeros(1, 1, dtype=torch.int32), [0], [S], xk, xv, cos, sin)
    kd, vd = opaged.values(rk, rv, sc)
    want = orope.rotate(xk.float(), cos, sin).double()[0]
    for got, x, c in ((kd[0], want, 0), (vd[0], xv[0].double(), 1)):
        step = 2.0 ** -10 * sc[0, :, c].double()[:, None, None]
        assert bool(((got - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, step)).all())


def test_verify_by_hand():
    """Two tokens: p = (3/4, 1/4), q = (1/4, 3/4)."""
    ln3 = math.log(3.0)
    t = torch.tensor([[[ln3, 0.0], [0.0, ln3]]], dtype=torch.float64)
    d = torch.tensor([[[0.0, ln3]]], dtype=torch.float64)
    x = torch.tensor([[1]])
    for u, r, want, n in ((0.32, 0.2, [1, 0], 1), (0.32, 0.3, [1, 1], 1), (0.34, 0.99, [0, -1], 0)):
        got, k = opaged.verify(t, d, x, torch.tensor([[u]]), torch.tensor([r]), None, 1.0)
        assert got.tolist() == [want] and k.tolist() == [n]
    got, k = opaged.verify(t, None, x, torch.tensor([[0.26]]), torch.tensor([0.9]), None, 1.0)
    assert got.tolist() == [[0, -1]] and k.tolist() == [0]
    got, k = opaged.verify(t, None, torch.tensor([[0]]), None, None, None, 0.0)
    assert got.tolist() == [[0, 1]] and k.tolist() == [1]

"""GPU: the paged KV cache -- append with RoPE, and attention over the pages -- against
the 64-bit CPU oracle.

The append's entries, scales and rotated queries are compared bit for bit: the rotation
is fp32 with each product and the sum rounded, and one rounding to what the pages hold.

Attention tolerances, from the arithmetic: with A = sum_j p_j |v_j| of an output and R the
largest sum_d |q_d k_d| * scale of its row,
  scores   a dot of D fp32 products and sums is off by at most (D + 4) 2^-24 R (4: the
           scale, the page's scale, its product with log2 e and the softmax's subtraction);
           2^x and the sums over keys add 2^-21 (hardware exp2 to 1 ulp, at most a few
           hundred keys here), relative to p, in the numerator and in the sum below it;
  p        the matrix-core path feeds p as two 16-bit parts: off by 2^-16 p at most;
  output   half a step of its type, relative to the value.
"""
import math

import pytest
import torch

from helpers import randn
from oracle import paged as opaged
from oracle import rope as orope

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn


def tables(D, n, dtype):
    fc = orope.freqs_cis(D, n)
    return orope.cos_sin(fc, dtype)


def make_pages(n, H, P, D, dtype, store, seed):
    """Pages k, v (and scales) on the CPU as earlier appends left them."""
    k, v = randn((n, H, P, D), seed, F32), randn((n, H, D, P), seed + 1, F32)
    k[..., ::7] *= 5.0
    if store == "same":
        return k.to(dtype), v.to(dtype), None
    sc = torch.empty(n, H, 2)
    k8, v8 = torch.empty_like(k, dtype=E4M3), torch.empty_like(v, dtype=E4M3)
    for i in range(n):
        for h in range(H):
            for c, (x, o) in enumerate(((k, k8), (v, v8))):
                sc[i, h, c] = opaged.page_scale(float(x[i, h].abs().max()))
                o[i, h] = opaged.to_e4m3(x[i, h], float(sc[i, h, c]))
    return k8, v8, sc


def on(dev, *ts):
    return tuple(None if t is None else t.to(dev) for t in ts)


def bits(t):
    return t.cpu().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def cache_of(dev, k, v, sc, dtype):
    from src.paged import PagedKVCache
    return PagedKVCache.from_pages(*(None if t is None else t.to(dev).contiguous() for t in (k, v, sc)),
                                   dtype=dtype)


def table_of(B, slots, n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(n, generator=g)[:B * slots].reshape(B, slots).int()


# ------------------------------------------------------------------ append

APPEND = [
    # dtype, store, Hq, Hkv, D, P, S, start, lens, model layout
    (BF16, "same", 8, 2, 64, 16, 1, [0, 15, 16, 37], None, True),
    (BF16, "e4m3", 8, 2, 64, 16, 1, [0, 15, 16, 37], None, True),
    (F16, "e4m3", 6, 2, 128, 32, 5, [0, 29, 31, 64], [5, 5, 1, 0], True),
    (F16, "same", 6, 2, 128, 32, 5, [3, 29, 31, 64], [5, 4, 0, 2], False),
    (BF16, "e4m3", 4, 4, 256, 64, 70, [0, 63], None, True),
    (BF16, "same", 4, 4, 32, 128, 131, [1, 126], [131, 77], True),
    (F32, "same", 4, 2, 24, 16, 33, [7, 0], None, True),
    (F32, "e4m3", 4, 2, 24, 16, 33, [7, 0], [33, 20], False),
    (BF16, "e4m3", 3, 1, 6, 256, 9, [250, 3], None, False),
    (F16, "same", 2, 1, 2, 16, 3, [15, 14], None, True),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x) for x in c[:7]))
@pytest.mark.parametrize("wide_tables", [False, True])
def test_append_matches_oracle_bitwise(dev, case, wide_tables):
    from src.paged import rope_and_paged_update
    dtype, store, Hq, Hkv, D, P, S, start, lens, model = case
    B = len(start)
    slots = (max(start) + S + P - 1) // P + 1
    n = B * slots + 2
    k, v, sc = make_pages(n, Hkv, P, D, dtype, store, 5)
    table = table_of(B, slots, n, 6)
    shape = (lambda h: (B, S, h, D)) if model else (lambda h: (B, h, S, D))
    turn = (lambda t: t.transpose(1, 2)) if model else (lambda t: t)
    xq, xk, xv = (turn(randn(shape(h), 7 + i, dtype)) for i, h in enumerate((Hq, Hkv, Hkv)))
    xk = xk * 3
    cos, sin = tables(D, slots * P, F32 if wide_tables else dtype)
    cache = cache_of(dev, k, v, sc, dtype)
    dxq = xq.to(dev)
    q = rope_and_paged_update(*on(dev, xk, xv, cos, sin), cache, 0, table.to(dev),
                              torch.tensor(start, device=dev), xq=dxq,
                              query_lens=None if lens is None else torch.tensor(lens, device=dev))
    torch.cuda.synchronize()
    rk, rv, rs = opaged.append(k, v, sc, table, start, lens or [S] * B, xk, xv, cos, sin)
    assert torch.equal(bits(cache.k[0]), bits(rk))
    assert torch.equal(bits(cache.v[0]), bits(rv))
    if sc is not None:
        assert torch.equal(cache.scales[0].cpu(), rs)
    assert q.stride() == dxq.stride()
    for b in range(B):
        ref = orope.rotate(xq[b], cos[start[b]:start[b] + S], sin[start[b]:start[b] + S])
        assert torch.equal(bits(q[b]), bits(ref))


@pytest.mark.parametrize("store", ["same", "e4m3"])
def test_append_token_by_token_with_growing_values(dev, store):
    """A page filled one token at a time, values growing and shrinking: the scale only
    grows, and older entries follow it."""
    from src.paged import rope_and_paged_update
    B, H, D, P, slots = 2, 2, 32, 16, 3
    n = B * slots
    k, v, sc = make_pages(n, H, P, D, BF16, store, 20)
    table = table_of(B, slots, n, 21)
    cos, sin = tables(D, slots * P, BF16)
    cache = cache_of(dev, k, v, sc, BF16)
    dtab, dcos, dsin = on(dev, table, cos, sin)
    mult = [1.0, 0.01, 30.0, 1e-3, 1e4, 0.0, 2.0, 1e6] * 6
    for t in range(40):
        xk, xv = (randn((B, H, 1, D), 30 + 2 * t + i) * mult[t + i] for i in range(2))
        start = [t, t + 5]
        rope_and_paged_update(*on(dev, xk, xv), dcos, dsin, cache, 0, dtab,
                              torch.tensor(start, device=dev))
        k, v, sc = opaged.append(k, v, sc, table, start, [1, 1], xk, xv, cos, sin)
    torch.cuda.synchronize()
    assert torch.equal(bits(cache.k[0]), bits(k)) and torch.equal(bits(cache.v[0]), bits(v))
    if sc is not None:
        assert torch.equal(cache.scales[0].cpu(), sc)


@pytest.mark.parametrize("S", [1, 20])
def test_append_scale_borders_zeros_and_values_that_are_not_finite(dev, S):
    """448 times a power of two is held by that power; the next value needs the next one;
    all-zero pages take the least scale; infinities and NaN become NaN and have no
    say in the scale."""
    from src.paged import rope_and_paged_update
    H, D, P = 6, 16, 32
    xk = torch.zeros(1, H, S, D)
    xk[0, 0, S - 1, 3] = 448.0
    xk[0, 1, S - 1, 3] = 450.0
    xk[0, 2, S - 1, 3] = -448.0 * 2.0 ** -30
    xk[0, 3, 0] = math.inf
    xk[0, 4, 0, 2] = math.nan
    xk[0, 4, 0, 5] = 7.0
    xv = xk.flip(3).clone()
    xk, xv = xk.to(BF16), xv.to(BF16)
    cos, sin = torch.ones(P, D // 2, dtype=BF16), torch.zeros(P, D // 2, dtype=BF16)
    k, v, sc = make_pages(2, H, P, D, BF16, "e4m3", 40)
    cache = cache_of(dev, k, v, sc, BF16)
    table = torch.tensor([[1]], dtype=torch.int32)
    rope_and_paged_update(*on(dev, xk, xv, cos, sin), cache, 0, table.to(dev), 0)
    rk, rv, rs = opaged.append(k, v, sc, table, [0], [S], xk, xv, cos, sin)
    torch.cuda.synchronize()
    nan = torch.isnan(rk.float())
    assert torch.equal(torch.isnan(cache.k[0].float().cpu()), nan)
    assert torch.equal(bits(cache.k[0])[~nan], bits(rk)[~nan])
    nan = torch.isnan(rv.float())
    assert torch.equal(torch.isnan(cache.v[0].float().cpu()), nan)
    assert torch.equal(bits(cache.v[0])[~nan], bits(rv)[~nan])
    assert torch.equal(cache.scales[0].cpu(), rs)
    assert rs[1, 0, 0] == 1.0 and rs[1, 1, 0] == 2.0 and rs[1, 2, 0] == 2.0 ** -30
    assert rs[1, 5, 0] == 2.0 ** -120


@pytest.mark.parametrize("store", ["same", "e4m3"])
def test_append_writes_only_places_that_exist(dev, store):
    """Positions before 0 and behind the slots, table entries that are no page: not written."""
    from src.paged import rope_and_paged_update
    H, D, P, S = 2, 16, 16, 20
    k, v, sc = make_pages(8, H, P, D, F16, store, 50)
    table = torch.tensor([[3, -1, 5], [8, 2, 7], [0, 1, 6], [4, 2 ** 31 - 1, -2 ** 31], [4, 4, 4]],
                         dtype=torch.int32)
    start = [10, 10, 40, -7, 2 ** 60]
    B = len(start)
    xk, xv = randn((B, H, S, D), 51, F16), randn((B, H, S, D), 52, F16)
    cos, sin = tables(D, 30, F16)          # fewer rows than positions: the last row serves the rest
    cache = cache_of(dev, k, v, sc, F16)
    xq = randn((B, H, S, D), 53, F16, dev)
    for st in (start, [-2 ** 62, 48, 2 ** 62, -20, 47]):
        q = rope_and_paged_update(*on(dev, xk, xv, cos, sin), cache, 0, table.to(dev),
                                  torch.tensor(st, device=dev), xq=xq)
        k, v, sc = opaged.append(k, v, sc, table, st, [S] * B, xk, xv, cos, sin)
        torch.cuda.synchronize()
        assert torch.equal(bits(cache.k[0]), bits(k)) and torch.equal(bits(cache.v[0]), bits(v))
        if sc is not None:
            assert torch.equal(cache.scales[0].cpu(), sc)
        for b in range(B):
            rows = [min(max(st[b] + s, 0), 29) for s in range(S)]
            assert torch.equal(bits(q[b]), bits(orope.rotate(xq[b].cpu(), cos[rows], sin[rows])))


def test_append_layers_int_start_empty_calls_and_odd_strides(dev):
    from src.config import ModelArgs
    from src.paged import PagedKVCache, rope_and_paged_update
    args = ModelArgs(dim=4 * 32, n_layers=3, n_heads=4, n_kv_heads=2, device=str(dev))
    cache = PagedKVCache(args, 5, 16, dtype=BF16, kv_dtype=E4M3)
    assert cache.k.shape == (3, 5, 2, 16, 32) and cache.v.shape == (3, 5, 2, 32, 16)
    table = torch.tensor([[4, 2]], dtype=torch.int32)
    cos, sin = tables(32, 32, BF16)
    # k and v inside wider rows that are not 16-byte aligned, v with a strided head dim
    wide = randn((1, 2, 18, 40), 60)
    xk, xv = wide[..., 3:35], randn((1, 2, 18, 64), 61)[..., ::2]
    dk = wide.to(dev)[..., 3:35]
    dv = randn((1, 2, 18, 64), 61, device=dev)[..., ::2]
    assert rope_and_paged_update(dk, dv, *on(dev, cos, sin), cache, -2, table.to(dev), 9) is None
    z = torch.zeros(5, 2, 16, 32).to(E4M3)
    rk, rv, rs = opaged.append(z, z.transpose(2, 3).contiguous(), torch.zeros(5, 2, 2), table, [9], [18],
                               xk, xv, cos, sin)
    torch.cuda.synchronize()
    assert torch.equal(bits(cache.k[1]), bits(rk)) and torch.equal(bits(cache.v[1]), bits(rv))
    assert torch.equal(cache.scales[1].cpu(), rs)
    assert not bits(cache.k[0]).any() and not bits(cache.k[2]).any()
    before = bits(cache.k)
    q = rope_and_paged_update(dk[:, :, :0], dv[:, :, :0], *on(dev, cos, sin), cache, 0, table.to(dev), 0,
                              xq=dk[:, :, :0])
    assert q.shape == (1, 2, 0, 32)
    assert rope_and_paged_update(dk[:0], dv[:0], *on(dev, cos, sin), cache, 0, table.to(dev)[:0],
                                 0) is None
    assert torch.equal(bits(cache.k), before)
    cache.reset()
    assert not bits(cache.k).any() and not cache.scales.any()


# --------------------------------------------------------------- attention

def tolerance(ref, mass, reach, D, dtype):
    score = (D + 4) * 2.0 ** -24 * reach[..., None] + 2.0 ** -21
    return torch.finfo(dtype).eps / 2 * ref.abs() + (2 * score + 2.0 ** -16) * mass + 1e-30


def lse_tolerance(ref, reach, D):
    return (D + 4) * 2.0 ** -24 * reach + 2.0 ** -21 + 2.0 ** -22 * ref.abs()


def check_attend(dev, q, k, v, sc, table, seq_lens, query_lens=None, *, dtype, view=None, **kw):
    """view: the layout the call gets q in (a function of q on the device)."""
    from src.paged import paged_flash_attention
    cache = cache_of(dev, k, v, sc, dtype)
    dq = q.to(dev) if view is None else view(q.to(dev))
    out, lse = paged_flash_attention(
        dq, cache, 0, table.to(dev), torch.tensor(seq_lens, device=dev), return_lse=True,
        query_lens=None if query_lens is None else torch.tensor(query_lens, device=dev), **kw)
    torch.cuda.synchronize()
    assert out.stride() == dq.stride() and out.dtype == dtype
    ref, rlse, mass, reach = opaged.attend(q, k, v, sc, table, seq_lens, query_lens,
                                           kw.get("sm_scale"))
    got, glse = out.double().cpu(), lse.double().cpu()
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), bad)
    off = ((got - ref).abs() / tolerance(ref, mass, reach, q.shape[3], dtype))[~bad]
    assert not off.numel() or float(off.max()) <= 1.0, float(off.max())
    empty = rlse == -math.inf
    assert torch.equal(glse == -math.inf, empty)
    fine = ~empty & ~torch.isnan(rlse)
    assert torch.equal(torch.isnan(glse), torch.isnan(rlse))
    off = ((glse - rlse).abs() / lse_tolerance(rlse, reach, q.shape[3]))[fine]
    assert not off.numel() or float(off.max()) <= 1.0, float(off.max())
    return out


ATTEND = [
    # dtype, store, Hq, Hkv, D, P, S, seq_lens, query_lens
    (BF16, "e4m3", 8, 2, 64, 16, 1, [1, 17, 64, 200, 0], None),
    (F16, "e4m3", 8, 2, 64, 16, 1, [1, 17, 64, 200, 0], None),
    (BF16, "same", 8, 2, 64, 16, 1, [1, 17, 64, 200, 0], None),
    (BF16, "e4m3", 6, 2, 128, 64, 1, [63, 129, 300], None),
    (F16, "same", 6, 2, 128, 64, 1, [63, 129, 300], None),
    (BF16, "e4m3", 6, 2, 128, 64, 4, [4, 129, 300], [4, 3, 0]),
    (F16, "e4m3", 6, 2, 128, 32, 5, [2, 65, 97], [5, 1, 5]),
    (BF16, "same", 4, 1, 128, 32, 9, [9, 33, 70], None),
    (F16, "same", 16, 1, 64, 128, 3, [128, 131], None),
    (BF16, "e4m3", 40, 2, 64, 256, 2, [255, 100], None),
    (BF16, "e4m3", 3, 3, 256, 64, 2, [77, 64], None),
    (F16, "same", 2, 2, 256, 16, 3, [77, 64], None),
    (BF16, "same", 4, 2, 192, 32, 2, [90], None),
    (BF16, "e4m3", 8, 2, 64, 64, 33, [33, 150], [33, 20]),
    (F16, "same", 4, 2, 128, 16, 70, [100, 70], None),
    (BF16, "e4m3", 4, 2, 128, 64, 140, [190], None),
    (BF16, "same", 4, 2, 96, 32, 2, [50, 3], None),
    (BF16, "e4m3", 4, 2, 80, 16, 3, [50, 3], None),
    (F32, "same", 4, 2, 64, 16, 3, [50, 97], None),
    (F32, "e4m3", 4, 2, 6, 32, 2, [50, 97], [1, 2]),
    (F32, "same", 4, 2, 32, 64, 1, [65, 1], None),
    (F32, "e4m3", 4, 2, 64, 64, 11, [50, 97], [11, 2]),
    (F32, "same", 8, 2, 128, 32, 1, [1, 17, 64, 200, 0], None),
    (F32, "e4m3", 6, 2, 128, 16, 4, [4, 129, 300], [4, 3, 0]),
    (F32, "same", 4, 2, 256, 64, 5, [77, 64], None),
    (F32, "e4m3", 16, 1, 256, 256, 2, [77, 300], None),
    (F32, "same", 4, 1, 64, 16, 70, [100, 70], None),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(str(x) for x in c[:7]))
@pytest.mark.parametrize("splits", [None, 1, 7, 16])
def test_attend_matches_oracle(dev, case, splits):
    dtype, store, Hq, Hkv, D, P, S, lens, qlens = case
    B = len(lens)
    slots = max((max(lens) + P - 1) // P, 1)
    n = B * slots + 1
    k, v, sc = make_pages(n, Hkv, P, D, dtype, store, 70)
    q = randn((B, Hq, S, D), 72, dtype)
    check_attend(dev, q, k, v, sc, table_of(B, slots, n, 73), lens, qlens, dtype=dtype,
                 num_splits=splits)


# rows long enough to be divided: several parts a row, parts of several rows, empty rows
LONG = [
    (BF16, "e4m3", 4, 2, 64, 64, 1, [2100, 70, 0, 1300], None),
    (F16, "e4m3", 3, 1, 128, 16, 2, [65, 0, 1900, 3], [2, 0, 2, 1]),
    (BF16, "same", 4, 2, 128, 32, 1, [1, 1601, 64], None),
    (F16, "same", 2, 2, 64, 128, 4, [1500, 1024], None),
    (BF16, "e4m3", 2, 2, 256, 256, 1, [700, 1], None),
    (BF16, "e4m3", 20, 1, 64, 64, 2, [900, 1, 1200], None),
    (F16, "same", 10, 1, 128, 64, 5, [1100, 30], [5, 3]),
    (F32, "same", 4, 2, 128, 16, 1, [1600, 1, 0, 700], None),
    (F32, "e4m3", 20, 1, 64, 64, 2, [900, 1, 1200], None),
    (F32, "same", 2, 2, 64, 256, 3, [1200, 1030], [3, 1]),
    (F32, "e4m3", 2, 1, 256, 32, 1, [1500], None),
    (F32, "same", 3, 3, 48, 16, 1, [1100, 0, 300], None),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(str(x) for x in c[:7]))
@pytest.mark.parametrize("splits", [None, 2, 5, 9, 64])
def test_attend_divided_rows_match_oracle(dev, case, splits):
    dtype, store, Hq, Hkv, D, P, S, lens, qlens = case
    B, slots = len(lens), (max(lens) + P - 1) // P
    n = B * slots + 1
    k, v, sc = make_pages(n, Hkv, P, D, dtype, store, 75)
    table = table_of(B, slots, n, 76)
    _dirty(k, v, sc, table, lens, P)
    check_attend(dev, randn((B, Hq, S, D), 77, dtype), k, v, sc, table, lens, qlens, dtype=dtype,
                 num_splits=splits)


def test_attend_one_long_row_among_many(dev):
    """140 rows, three of them long, around the ends of its 64s: the list of keys is held 64
    rows at a time."""
    B, P, slots = 140, 64, 40
    k, v, sc = make_pages(100, 1, P, 64, F16, "e4m3", 78)
    table = torch.randint(0, 100, (B, slots), generator=torch.Generator().manual_seed(79)).int()
    lens = [(7 * i) % 90 for i in range(B)]
    lens[64], lens[127], lens[139] = 2500, 2300, 2048
    for splits in (None, 6, 200):
        check_attend(dev, randn((B, 2, 1, 64), 74, F16), k, v, sc, table, lens, dtype=F16, num_splits=splits)


@pytest.mark.parametrize("dtype,store,D", [(BF16, "same", 64), (F16, "e4m3", 128), (F32, "same", 128), (F32, "same", 48)])
@pytest.mark.parametrize("step", [0.05, 3.0, -3.0])
def test_attend_scores_that_rise_and_fall(dev, dtype, store, D, step):
    """Scores that grow by less than a step's worth, by much more, and that fall: the running
    maximum moves late, in every step, and once."""
    P, L = 16, 400
    k, v, sc = make_pages(L // P + 1, 1, P, D, dtype, store, 126)
    table = torch.arange(L // P + 1, dtype=torch.int32)[None]
    at = torch.arange((L // P + 1) * P, dtype=torch.float32).view(-1, 1, P, 1) * step
    k = (k.float() * 0.01 if store == "same" else torch.zeros(k.shape))
    k[..., :1] += (at if store == "same" else (at / 8).clamp(-400, 400))
    k = k.to(dtype if store == "same" else E4M3)
    q = randn((1, 2, 3, D), 127, dtype).abs()
    q[0, 1, 2, 0] = 0.0
    check_attend(dev, q, k, v, sc, table, [L], dtype=dtype)


def _dirty(k, v, sc, table, lens, P):
    """NaN behind every row's keys and in pages that are nobody's."""
    used = set()
    for b, n in enumerate(lens):
        for slot in range(table.shape[1]):
            page, m = int(table[b, slot]), n - slot * P
            if not 0 <= page < k.shape[0]:
                continue
            used.add(page)
            if m < P:
                k[page, :, max(m, 0):] = math.nan
                v[page, :, :, max(m, 0):] = math.nan
                if sc is not None and m <= 0:
                    sc[page] = math.nan
    for page in set(range(k.shape[0])) - used:
        k[page], v[page] = math.nan, math.nan


@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (F32, 32), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("S", [1, 3])
def test_attend_reads_no_key_behind_the_last(dev, store, dtype, D, S):
    P, lens = 16, [1, 15, 16, 49, 100, 0]
    B, slots = len(lens), 9
    n = B * slots + 2
    k, v, sc = make_pages(n, 2, P, D, dtype, store, 80)
    table = table_of(B, slots, n, 81)
    _dirty(k, v, sc, table, lens, P)
    out = check_attend(dev, randn((B, 4, S, D), 82, dtype), k, v, sc, table, lens, [S, S, 1, S, S, 1],
                       dtype=dtype)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (BF16, 128), (F32, 32), (F32, 128)])
@pytest.mark.parametrize("S,lens", [(5, [70, 66]), (40, [64, 90]), (5, [1470, 1026])])
def test_attend_a_nan_reaches_only_tokens_that_see_it(dev, store, dtype, D, S, lens):
    """A NaN value at a newer token's position: the tokens before it stay finite, those from
    it on are NaN; a NaN in K likewise."""
    P, B = 32, 2
    slots = (max(lens) + P - 1) // P
    k, v, sc = make_pages(B * slots, 2, P, D, dtype, store, 90)
    table = table_of(B, slots, B * slots, 91)
    for b, (back, what) in enumerate(((2, "v"), (3, "k"))):
        j = lens[b] - back
        page = int(table[b, j // P])
        if what == "v":
            v[page, 1, 5, j % P] = math.nan
        else:
            k[page, 0, j % P, 5] = math.nan
    out = check_attend(dev, randn((B, 4, S, D), 92, dtype), k, v, sc, table, lens, dtype=dtype)
    assert bool(torch.isfinite(out[0, :, :S - 2]).all()) and bool(torch.isfinite(out[0, :2]).all())
    assert bool(torch.isnan(out[0, 2:, S - 2:, 5]).all())
    assert bool(torch.isfinite(out[0, 2:, S - 2:, 6]).all())
    assert bool(torch.isfinite(out[1, :, :S - 3]).all()) and bool(torch.isnan(out[1, :2, S - 3:]).all())


@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F32, 64), (F32, 40)])
def test_attend_skips_entries_that_are_no_page(dev, store, dtype, D):
    P, lens = 16, [80, 80, 10 ** 12, -5, 64]
    B, slots = len(lens), 5
    k, v, sc = make_pages(30, 2, P, D, dtype, store, 100)
    table = table_of(B, slots, 30, 101)
    table[0, 1], table[0, 4], table[1, 0] = -1, 30, 2 ** 31 - 1
    table[4] = -2 ** 31
    out = check_attend(dev, randn((B, 4, 2, D), 102, dtype), k, v, sc, table, lens, dtype=dtype)
    assert not out[3].any() and not out[4].any()


@pytest.mark.parametrize("dtype,store,D", [(BF16, "e4m3", 64), (F16, "same", 128), (F32, "same", 64)])
def test_attend_layouts_and_scale(dev, dtype, store, D):
    """q as a view of [B, S, H, D] projections, inside wider unaligned rows, and with a
    strided head dim; a scale of its own."""
    P, lens = 32, [40, 90]
    k, v, sc = make_pages(6, 2, P, D, dtype, store, 110)
    table = table_of(2, 3, 6, 111)
    q = randn((2, 4, 3, D), 112, dtype)

    def model(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def wider(t):
        w = torch.zeros((2, 4, 3, D + 13), dtype=dtype, device=dev)
        w[..., 3:D + 3] = t
        return w[..., 3:D + 3]

    for view in (model, None):
        check_attend(dev, q, k, v, sc, table, lens, dtype=dtype, view=view, sm_scale=0.3)
    from src.paged import paged_flash_attention
    cache = cache_of(dev, k, v, sc, dtype)
    args = (cache, 0, table.to(dev), torch.tensor(lens, device=dev))
    plain = paged_flash_attention(q.to(dev), *args)
    spread = torch.zeros((2, 4, 3, 2 * D), dtype=dtype, device=dev)
    spread[..., ::2] = q.to(dev)
    for x in (wider(q.to(dev)), spread[..., ::2]):
        assert torch.equal(paged_flash_attention(x, *args), plain)


@pytest.mark.parametrize("sm_scale", [0.0, -0.1, float("nan"), float("inf")])
def test_attend_refuses_scales(dev, sm_scale):
    from src.paged import paged_flash_attention
    cache = cache_of(dev, *make_pages(2, 2, 16, 64, BF16, "same", 118), BF16)
    with pytest.raises(ValueError, match="sm_scale"):
        paged_flash_attention(randn((1, 4, 1, 64), 119, device=dev), cache, 0,
                              torch.zeros((1, 2), dtype=torch.int32, device=dev),
                              torch.ones(1, dtype=torch.int64, device=dev), sm_scale=sm_scale)


@pytest.mark.parametrize("exp", [-120, 90])
def test_attend_pages_of_extreme_scales(dev, exp):
    """Pages whose scales are near the ends of what a page can have (K and V; the other is
    ordinary): scores that vanish, values near fp32's ends."""
    k, v, sc = make_pages(6, 2, 32, 64, BF16, "e4m3", 115)
    q, table, lens = randn((2, 4, 2, 64), 116), table_of(2, 3, 6, 117), [90, 65]
    for which in ((0, 1) if exp < 0 else (1,)):
        s = sc.clone()
        s[..., which] = 2.0 ** exp
        check_attend(dev, q, k, v, s, table, lens, dtype=BF16)


@pytest.mark.parametrize("dtype,store,D", [(BF16, "same", 64), (F16, "e4m3", 128), (F32, "same", 128), (BF16, "e4m3", 80)])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("sign", [-1, 1])
def test_attend_scores_of_any_size(dev, dtype, store, D, splits, sign):
    """All scores are finite, between 1e19 and 1e37 in size: one key (the first of the negative, the
    last of the positive) has the largest, by so much that it has all the weight."""
    from src.paged import paged_flash_attention
    P, L = 16, 600
    n = (L + P - 1) // P
    k, v, sc = make_pages(n, 1, P, D, dtype, store, 128)
    size = 30000.0 if dtype == F16 else 1e17
    at = torch.arange(n * P, dtype=torch.float32).view(n, 1, P)
    k = torch.zeros(k.shape)
    if store == "same":
        k[..., 0] = sign * torch.where(at == (0 if sign < 0 else L - 1), 0.5 if sign < 0 else 2000.0, 1.0 + at) \
            * (size / 1000)
        k = k.to(dtype)
    else:
        k[..., 0] = sign * torch.where(at == (0 if sign < 0 else L - 1), 0.5 if sign < 0 else 4.0, 1.0)
        sc[..., 0] = 2.0 ** 45
        k = k.to(E4M3)
    q = torch.zeros(1, 2, 1, D)
    q[..., 0] = size
    sm_scale = 1e5 if dtype == F16 else 1.0
    out, lse = paged_flash_attention(q.to(dtype).to(dev), cache_of(dev, k, v, sc, dtype), 0,
                                     torch.arange(n, dtype=torch.int32, device=dev)[None],
                                     torch.tensor([L], device=dev), sm_scale=sm_scale,
                                     return_lse=True, num_splits=splits)
    key = 0 if sign < 0 else L - 1
    page, off = key // P, key % P
    want = v[page, 0, :, off].double() * (1.0 if sc is None else float(sc[page, 0, 1]))
    assert torch.equal(out[0, :, 0].cpu(), want.to(dtype).expand(2, D))
    score = float(q.to(dtype)[0, 0, 0, 0]) * float(k[page, 0, off, 0]) * sm_scale
    score *= 1.0 if sc is None else float(sc[page, 0, 0])
    assert score * sign > 1e19 and float(((lse.double().cpu() - score) / score).abs().max()) < 1e-6


def test_attend_rows_share_pages(dev):
    """Rows with the same first pages (a shared prefix), and a page twice in one row."""
    k, v, sc = make_pages(8, 2, 16, 128, F16, "e4m3", 113)
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5], [6, 6, 6, 0]], dtype=torch.int32)
    check_attend(dev, randn((3, 4, 2, 128), 114, F16), k, v, sc, table, [60, 49, 50], dtype=F16)


@pytest.mark.parametrize("B,splits", [(70, None), (130, 300), (200, 3)])
def test_attend_many_rows(dev, B, splits):
    """More rows than a wave has lanes, most of them empty or short."""
    P, slots = 16, 6
    k, v, sc = make_pages(40, 1, P, 64, BF16, "e4m3", 123)
    g = torch.Generator().manual_seed(124)
    table = torch.randint(0, 40, (B, slots), generator=g).int()
    lens = [0 if i % 3 == 0 else (5 * i) % (P * slots + 1) for i in range(B)]
    check_attend(dev, randn((B, 2, 1, 64), 125), k, v, sc, table, lens, dtype=BF16, num_splits=splits)


def test_attend_empty_calls(dev):
    from src.paged import paged_flash_attention
    k, v, sc = make_pages(4, 2, 16, 64, BF16, "e4m3", 120)
    cache = cache_of(dev, k, v, sc, BF16)
    table = torch.zeros((2, 2), dtype=torch.int32, device=dev)
    q = randn((2, 4, 0, 64), 121, device=dev)
    out, lse = paged_flash_attention(q, cache, 0, table, torch.tensor([1, 2], device=dev), return_lse=True)
    assert out.shape == q.shape and lse.shape == (2, 4, 0)
    out = paged_flash_attention(randn((0, 4, 1, 64), 121, device=dev), cache, 0, table[:0],
                                torch.zeros(0, dtype=torch.int64, device=dev))
    assert out.shape == (0, 4, 1, 64)
    # table of one row of slots, lengths in int32: converted
    out = paged_flash_attention(randn((2, 4, 1, 64), 121, device=dev), cache, 0, table,
                                torch.tensor([0, 0], device=dev, dtype=torch.int32))
    assert not out.any()


@pytest.mark.parametrize("store", ["same", "e4m3"])
def test_attend_long_cache_offsets_pass_32_bits(dev, store):
    """Pages whose byte offsets (and, in 8 bits, entry numbers) pass 2^32; the row's pages
    lie at both ends."""
    from src.paged import PagedKVCache, paged_flash_attention, rope_and_paged_update
    H, P, D = 8, 256, 128
    per = H * P * D                                    # 2^18 entries a page
    n = (2 ** 32 // per + 8) // (1 if store == "e4m3" else 2) + 8
    kd = E4M3 if store == "e4m3" else BF16
    k = torch.zeros((n, H, P, D), dtype=kd, device=dev)
    v = torch.zeros((n, H, D, P), dtype=kd, device=dev)
    sc = None if store == "same" else torch.ones((n, H, 2), device=dev)
    cache = PagedKVCache.from_pages(k, v, sc, dtype=BF16)
    assert k.numel() * k.element_size() > 2 ** 32
    table = torch.tensor([[n - 1, 0, n - 2]], dtype=torch.int32, device=dev)
    S = 600
    xk, xv = randn((1, H, S, D), 130, device=dev), randn((1, H, S, D), 131, device=dev)
    cos, sin = on(dev, *tables(D, S, BF16))
    rope_and_paged_update(xk, xv, cos, sin, cache, 0, table, 0)
    q = randn((1, H, 2, D), 132)
    out = paged_flash_attention(q.to(dev), cache, 0, table, torch.tensor([S], device=dev))
    torch.cuda.synchronize()
    pick = torch.tensor([n - 1, 0, n - 2], device=dev)
    raw = (lambda t: t.view(torch.uint8)[pick].view(kd).cpu()) if sc is not None else (lambda t: t[pick].cpu())
    small = (raw(k), raw(v), None if sc is None else sc[pick].cpu())
    rk, rv, rs = opaged.append(torch.zeros((3, H, P, D), dtype=kd), torch.zeros((3, H, D, P), dtype=kd),
                               None if sc is None else torch.ones(3, H, 2), torch.tensor([[0, 1, 2]]),
                               [0], [S], xk.cpu(), xv.cpu(), cos.cpu(), sin.cpu())
    assert torch.equal(bits(small[0]), bits(rk)) and torch.equal(bits(small[1]), bits(rv))
    ref, _, mass, reach = opaged.attend(q, rk, rv, rs, torch.tensor([[0, 1, 2]]), [S])
    off = (out.double().cpu() - ref).abs() / tolerance(ref, mass, reach, D, BF16)
    assert float(off.max()) <= 1.0


# --------------------------------------------------------- graphs, streams

@pytest.mark.parametrize("dtype,store", [(BF16, "e4m3"), (F16, "same")])
def test_captured_step_follows_its_inputs(dev, dtype, store):
    """Append and attention captured as one step, two such graphs replayed in turn over
    one cache while lengths, counts and tables change, eager work between: each replay
    equals the eager step."""
    from src.paged import PagedKVCache, paged_flash_attention, rope_and_paged_update
    B, Hq, Hkv, S, D, P, slots = 3, 8, 2, 2, 64, 16, 6
    n = B * slots
    pages = make_pages(n, Hkv, P, D, dtype, store, 140)
    cache, twin = (cache_of(dev, *pages, dtype) for _ in range(2))
    cos, sin = on(dev, *tables(D, slots * P, dtype))
    table = table_of(B, slots, n, 141).to(dev)
    start = torch.zeros(B, dtype=torch.int64, device=dev)
    count = torch.full((B,), S, dtype=torch.int64, device=dev)
    xq, xk, xv = (torch.zeros((B, h, S, D), dtype=dtype, device=dev) for h in (Hq, Hkv, Hkv))

    def step(c):
        q = rope_and_paged_update(xk, xv, cos, sin, c, 0, table, start, query_lens=count, xq=xq)
        return paged_flash_attention(q, c, 0, table, start + count, query_lens=count, return_lse=True)

    step(twin)
    twin = cache_of(dev, *pages, dtype)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(cache))
        graphs.append(g)
    for t in range(6):
        for i, x in enumerate((xq, xk, xv)):
            x.copy_(randn(x.shape, 150 + 3 * t + i, dtype, dev))
        start.copy_(torch.tensor([3 * t, 15 + t, 40 + 5 * t]))
        count.copy_(torch.tensor([2, 1 + t % 2, t % 3 if t % 3 < 3 else 2]))
        if t == 3:
            perm = table_of(B, slots, n, 142).to(dev)
            table.copy_(perm)
        graphs[t % 2].replay()
        out, lse = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(outs[t % 2][0], out) and torch.equal(outs[t % 2][1], lse), t
        assert torch.equal(bits(cache.k), bits(twin.k)) and torch.equal(bits(cache.v), bits(twin.v))


def test_captured_attention_of_divided_rows(dev):
    """Two graphs over rows whose lengths move between empty, short and long: divided or
    by row, whichever the lengths of the replay call for."""
    from src.paged import paged_flash_attention
    B, P, D, slots = 3, 64, 64, 40
    cache = cache_of(dev, *make_pages(B * slots, 2, P, D, BF16, "e4m3", 170), BF16)
    table = table_of(B, slots, B * slots, 171).to(dev)
    q = randn((B, 4, 1, D), 172, device=dev)
    lens = torch.full((B,), 100, dtype=torch.int64, device=dev)
    call = (lambda: paged_flash_attention(q, cache, 0, table, lens, return_lse=True))
    call()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for i, now in enumerate(([2500, 3, 0], [0, 0, 0], [900, 900, 900], [1, 2560, 2559], [64, 65, 63])):
        lens.copy_(torch.tensor(now))
        q.copy_(randn(q.shape, 173 + i))
        graphs[i % 2].replay()
        ref = call()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2][0], ref[0]) and torch.equal(outs[i % 2][1], ref[1]), now


def test_calls_on_two_streams_at_once(dev):
    from src.paged import paged_flash_attention
    P, D, lens = 64, 128, [3000, 777]
    k, v, sc = make_pages(100, 2, P, D, BF16, "e4m3", 160)
    cache = cache_of(dev, k, v, sc, BF16)
    table = table_of(2, 48, 100, 161).to(dev)
    sl = torch.tensor(lens, device=dev)
    qs = [randn((2, 8, 1, D), 162 + i, device=dev) for i in range(2)]
    ref = [paged_flash_attention(q, cache, 0, table, sl) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in qs]
    outs = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged_flash_attention(qs[i], cache, 0, table, sl))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert torch.equal(o, ref[i])

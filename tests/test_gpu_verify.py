"""GPU: verification of drafted tokens against the 64-bit CPU oracle, token for token.

The kernel's shares are fp64 to 1e-12; a token can differ from the oracle's only where
the drawn number falls within about 1e-11 of a border between two tokens, which the
seeded numbers here do not (their distance to the nearest border is checked).
"""
import math

import pytest
import torch

from helpers import randn
from oracle import paged as opaged

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def case(B, S, V, dtype, seed, *, model=True, temperature=1.0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    target = torch.randn((B, S + 1, V), generator=g) * scale
    draft = (target[:, :S] + torch.randn((B, S, V), generator=g)).to(dtype)
    t = temperature or 1.0
    x = torch.multinomial(torch.softmax(draft.float() / t, -1).reshape(B * S, V), 1, generator=g)
    u, r = torch.rand((B, S), generator=g), torch.rand((B,), generator=g)
    return target.to(dtype), draft if model else None, x.reshape(B, S), u, r


def run(dev, target, draft, x, u, r, lens=None, temperature=1.0):
    from src.verify import verify_drafts
    t, n = verify_drafts(target.to(dev), x.to(dev), None if u is None else u.to(dev),
                         None if r is None else r.to(dev),
                         draft_logits=None if draft is None else draft.to(dev),
                         temperature=temperature,
                         draft_lens=None if lens is None else torch.tensor(lens, device=dev))
    torch.cuda.synchronize()
    return t.cpu(), n.cpu()


def same(dev, target, draft, x, u, r, lens=None, temperature=1.0):
    got, n = run(dev, target, draft, x, u, r, lens, temperature)
    ref, rn = opaged.verify(target, draft, x, u, r, lens, temperature)
    assert torch.equal(n, rn) and torch.equal(got, ref)
    return got, n


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,S,V", [(1, 1, 1), (3, 2, 7), (5, 4, 1000), (4, 3, 8184), (4, 3, 8185),
                                   (2, 5, 32003), (2, 7, 128256), (9, 1, 20001)])
@pytest.mark.parametrize("model", [True, False])
def test_matches_oracle(dev, dtype, B, S, V, model):
    same(dev, *case(B, S, V, dtype, B + V, model=model))


@pytest.mark.parametrize("temperature", [0.0, 0.05, 0.6, 1.7, 50.0])
@pytest.mark.parametrize("model", [True, False])
def test_temperatures(dev, temperature, model):
    t, d, x, u, r = case(6, 4, 5001, BF16, 11, model=model, temperature=temperature)
    if temperature == 0.0:   # some drafts that are the largest logit, first of equals
        x[:, :2] = t[:, :2].float().argmax(-1)
        u = r = None
    same(dev, t, d, x, u, r, temperature=temperature)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_rows_with_fewer_drafts(dev, temperature):
    t, d, x, u, r = case(6, 4, 3001, F16, 12)
    u *= 0.3                                      # most drafts accepted
    got, n = same(dev, t, d, x, u, r, lens=[4, 0, 1, 9, -3, 2], temperature=temperature)
    assert n[1] == 0 and n[4] == 0 and bool((got[1, 1:] == -1).all())


def test_everything_accepted_and_everything_refused(dev):
    t, _, x, u, r = case(4, 3, 999, BF16, 13)
    d = t[:, :3].clone()                          # q = p: every draft accepted
    _, n = same(dev, t, d, x, u, r)
    assert bool((n == 3).all())
    d = t[:, :3].clone()
    t[:, 0].scatter_(1, x[:, :1], -math.inf)      # the first draft has no mass
    got, n = same(dev, t, d, x, torch.zeros_like(u), r)
    assert bool((n == 0).all()) and bool((got[:, 1:] == -1).all())


def test_ties_take_the_least_token(dev):
    t = torch.zeros((3, 2, 20000), dtype=BF16)
    t[1, :, 9000:9003] = 2.0
    t[2, :, -1] = 1.0
    x = torch.tensor([[0], [9001], [19999]])
    got, n = same(dev, t, None, x, None, None, temperature=0.0)
    assert n.tolist() == [1, 0, 1] and got.tolist() == [[0, 0], [9000, -1], [19999, 19999]]


def test_borders_of_the_sum(dev):
    """Equal shares in exact numbers: the token after a border starts exactly there."""
    V = 4096
    t = torch.zeros((6, 2, V), dtype=F32)
    x = torch.zeros((6, 1), dtype=torch.int64)
    r = torch.tensor([0.0, 0.25, 0.25 - 2.0 ** -13, 1.0 - 2.0 ** -24, 0.5, 0.75])
    got, n = run(dev, t, None, x, torch.zeros(6, 1), r, lens=[0] * 6)
    assert got[:, 0].tolist() == [0, 1024, 1023, V - 1, 2048, V * 3 // 4]


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logits_that_are_not_finite(dev, dtype):
    t, d, x, u, r = case(8, 2, 9000, dtype, 14)
    t[0, 0] = -math.inf                           # no mass: refused, no token
    t[1, 0, ::2] = math.nan
    t[2, 0, 100:] = -math.inf                     # a filtered row
    d[3, 0, 5] = math.nan
    t[4, 1] = math.nan
    t[5, 0, 77] = math.inf
    t[6, 2, :] = -math.inf
    d[7, 0] = -math.inf
    x[5, 0] = 77
    u *= 0.2
    got, n = same(dev, t, d, x, u, r)
    assert n[0] == 0 and got[0, 0] == -1
    same(dev, t, None, x, u, r)
    same(dev, t, None, x, None, None, temperature=0.0)


def test_drafts_that_are_no_token(dev):
    t, d, x, u, r = case(4, 2, 500, BF16, 15)
    x[0, 0], x[1, 0], x[2, 1], x[3, 0] = -1, 500, 2 ** 40, -2 ** 63
    u[:] = 0.0
    for draft in (d, None):
        _, n = same(dev, t, draft, x, u, r)
        assert n.tolist()[:2] == [0, 0] and n[2] <= 1 and n[3] == 0
    x[0, 0] = -1
    same(dev, t, None, x, None, None, temperature=0.0)


def test_strides(dev):
    """Logits and drafts as slices of wider tensors, rows of different alignment."""
    from src.verify import verify_drafts
    t, d, x, u, r = case(3, 3, 4001, BF16, 16)
    ref = opaged.verify(t, d, x, u, r, None, 1.0)
    wide = torch.zeros((3, 6, 4100), dtype=BF16, device=dev)
    wide[:, 1:5, 7:4008] = t.to(dev)
    dw = torch.zeros((3, 3, 4001 * 2), dtype=BF16, device=dev)
    dw[..., ::2] = d.to(dev)
    xw = torch.zeros((3, 9), dtype=torch.int64, device=dev)
    xw[:, ::3] = x.to(dev)
    uw = u.to(dev).T.contiguous().T
    rw = torch.stack((r, r), 1).to(dev)[:, 0]
    for dd in (d.to(dev), dw[..., ::2]):
        got, n = verify_drafts(wide[:, 1:5, 7:4008], xw[:, ::3], uw, rw, draft_logits=dd)
        assert torch.equal(got.cpu(), ref[0]) and torch.equal(n.cpu(), ref[1])


def test_drawn_tokens_follow_the_target(dev):
    """Many rows of the same logits with their own random numbers: the token in the first
    place is distributed as the target's, whatever the draft.  Each share's count is within
    5 standard deviations."""
    V, B = 12, 20000
    g = torch.Generator().manual_seed(17)
    t = torch.randn((1, 2, V), generator=g).expand(B, 2, V).contiguous()
    d = (2.0 * torch.randn((1, 1, V), generator=g)).expand(B, 1, V).contiguous()
    x = torch.multinomial(torch.softmax(d[:1, 0], -1).expand(B, V), 1, generator=g)
    got, n = run(dev, t, d, x, torch.rand((B, 1), generator=g), torch.rand((B,), generator=g))
    p = torch.softmax(t[0, 0].double(), -1)
    count = torch.bincount(got[:, 0], minlength=V).double()
    assert float(((count - B * p).abs() / (B * p * (1 - p)).sqrt()).max()) < 5.0
    assert 0 < int(n.sum()) < B


def test_captured_calls(dev):
    """Two captured graphs replayed in turn at changing inputs equal the eager call."""
    from src.verify import verify_drafts
    t, d, x, u, r = (y.to(dev) for y in case(4, 3, 9001, BF16, 18))
    lens = torch.full((4,), 3, dtype=torch.int64, device=dev)
    call = (lambda: verify_drafts(t, x, u, r, draft_logits=d, draft_lens=lens, temperature=0.9))
    call()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for i in range(4):
        for dst, src in zip((t, d, x, u, r), case(4, 3, 9001, BF16, 19 + i)):
            dst.copy_(src)
        lens.copy_(torch.tensor([3, i % 4, 2, 1]))
        graphs[i % 2].replay()
        ref = call()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2][0], ref[0]) and torch.equal(outs[i % 2][1], ref[1])

"""GPU: a model step over the paged cache -- append, attention of one or several tokens,
draft verification -- as a serving program runs them together.

With fp32 weights, cache and activations every product is summed in fp32 in another
order than in the dense path: a relative 2^-24 a term, growing with the longest sum (512
terms: the FFN) and through 2 layers.  Logits agree to 1e-4 of their scale, the bar that
the fp32 oracle is held to against an independent model; bf16 logits to 2e-2 of it, the
bar of the dense path."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def small(dev, dtype=F32, quantized=False, **kw):
    from src.config import ModelArgs
    args = ModelArgs(**{**dict(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=1000,
                               hidden_dim=512, max_batch_size=4, max_seq_len=160, device=str(dev)), **kw})
    if quantized:
        from src.model_quantized import build_random_quantized
        return args, build_random_quantized(args, seed=0, device=dev)
    from src.model import Llama3
    torch.manual_seed(0)
    return args, Llama3(args).to(dev, dtype).eval()


def paged_cache(args, dtype, kv_dtype=None, page=16, pages=50):
    from src.paged import PagedKVCache
    return PagedKVCache(args, pages, page, dtype=dtype, kv_dtype=kv_dtype)


def shuffled(B, slots, pages, dev, seed=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:B * slots].reshape(B, slots).int().to(dev)


def prompt(B, S, vocab, dev, seed=1):
    return torch.randint(0, vocab, (B, S), generator=torch.Generator().manual_seed(seed)).to(dev)


def close(a, b, frac):
    scale = float(b.float().abs().max())
    err = float((a.float() - b.float()).abs().max())
    print(f"max|a - b| = {err:.3e} of scale {scale:.3f}")
    assert err < frac * scale


@pytest.mark.parametrize("dtype,quantized,frac", [(F32, False, 1e-4), (BF16, False, 2e-2), (BF16, True, 2e-2)])
@torch.no_grad()
def test_paged_steps_equal_dense_steps(dev, dtype, quantized, frac):
    """A prompt, single tokens and a group of tokens over both caches."""
    from src.kv_cache import KVCache
    args, model = small(dev, dtype, quantized)
    B, S = 3, 37
    dense, cache = KVCache(args, dtype=dtype), paged_cache(args, dtype)
    table = shuffled(B, 10, 50, dev)
    tok = prompt(B, S + 6, args.vocab_size, dev)
    a = model(tok[:, :S], kv_cache=dense, return_all_logits=True)
    b = model(tok[:, :S], kv_cache=cache, page_table=table, return_all_logits=True)
    close(b, a, frac)
    last = [model(tok[:, S + i:S + i + 1], start_pos=S + i, kv_cache=dense) for i in range(6)]
    for i in range(2):
        close(model(tok[:, S + i:S + i + 1], start_pos=S + i, kv_cache=cache, page_table=table), last[i], frac)
    b = model(tok[:, S + 2:], start_pos=S + 2, kv_cache=cache, page_table=table, return_all_logits=True)
    close(b, torch.cat(last[2:], 1), frac)


@torch.no_grad()
def test_ragged_rows_equal_rows_alone(dev):
    """Rows of different lengths in one padded call, then one token each at their own
    positions: each row's logits are those of the row alone."""
    args, model = small(dev)
    lens, more = [29, 1, 16, 7], 2
    B, S = len(lens), max(lens)
    tok = prompt(B, S + more, args.vocab_size, dev)
    cache = paged_cache(args, F32)
    table = shuffled(B, 3, 50, dev)
    count = torch.tensor(lens, device=dev)
    got = [model(tok[:, :S], kv_cache=cache, page_table=table, query_lens=count)]
    for i in range(more):
        nxt = tok[torch.arange(B, device=dev), count + i][:, None]
        got.append(model(nxt, kv_cache=cache, page_table=table, start_positions=count + i))
    for b, n in enumerate(lens):
        alone = paged_cache(args, F32)
        t1 = shuffled(1, 3, 50, dev, seed=9)
        for i in range(more + 1):
            row = tok[b:b + 1, :n] if i == 0 else tok[b:b + 1, n + i - 1:n + i]
            ref = model(row, start_pos=0 if i == 0 else n + i - 1, kv_cache=alone, page_table=t1)
            close(got[i][b:b + 1], ref, 1e-4)


@pytest.mark.parametrize("kv_dtype", [F32, E4M3])
@torch.no_grad()
def test_speculative_greedy_loop_gives_the_greedy_tokens(dev, kv_dtype):
    """Greedy decoding by drafts: every round appends the last token and 3 drafts (some
    right, some wrong), attends, verifies, and goes back behind the refused ones.  The
    tokens are those of one-token greedy steps (the top logits are apart by more than the
    difference between the two forms, which is checked).  With 8-bit pages a refused
    token may have raised its page's scale, so there the drafts are all right."""
    from src.verify import verify_drafts
    args, model = small(dev)
    B, S, n_new, k = 2, 21, 24, 3
    tok = prompt(B, S, args.vocab_size, dev)
    table = shuffled(B, 6, 50, dev)
    cache = paged_cache(args, F32, kv_dtype)
    logits, nxt = model(tok, kv_cache=cache, page_table=table, greedy=True)
    plain, gaps = [nxt], []
    for i in range(n_new + k):
        logits, nxt = model(nxt, start_pos=S + i, kv_cache=cache, page_table=table, greedy=True)
        top = logits[:, 0].topk(2).values
        gaps.append(float((top[:, 0] - top[:, 1]).min() / logits.abs().max()))
        plain.append(nxt)
    plain = torch.cat(plain, 1)
    assert min(gaps) > 2e-4, "the seed's tokens are too close to compare"

    cache = paged_cache(args, F32, kv_dtype)
    _, nxt = model(tok, kv_cache=cache, page_table=table, greedy=True)
    out = [[int(t)] for t in nxt[:, 0]]
    pos = torch.full((B,), S, dtype=torch.int64, device=dev)
    last, rounds = nxt, 0
    while min(map(len, out)) < n_new:
        drafts = torch.stack([plain[b, len(out[b]):len(out[b]) + k] for b in range(B)])
        if kv_dtype is F32:   # one wrong token at a place that moves
            drafts[:, rounds % (k + 1):rounds % (k + 1) + 1] += 1
            drafts %= args.vocab_size
        logits = model(torch.cat((last, drafts), 1), kv_cache=cache, page_table=table,
                       start_positions=pos, return_all_logits=True)
        tokens, n = verify_drafts(logits, drafts, temperature=0.0)
        for b in range(B):
            out[b] += tokens[b, :int(n[b]) + 1].tolist()
        last = tokens.gather(1, n[:, None])
        pos += n + 1
        rounds += 1
        if min(map(len, out)) + k + 1 > plain.shape[1]:
            break
    assert rounds < n_new - 1
    for b in range(B):
        m = min(len(out[b]), n_new)
        assert out[b][:m] == plain[b, :m].tolist()


@torch.no_grad()
def test_captured_paged_step(dev):
    """A model step of 1 token captured once follows its device positions and table."""
    args, model = small(dev, BF16)
    B, S = 2, 19
    tok = prompt(B, S + 5, args.vocab_size, dev)
    caches = [paged_cache(args, BF16, E4M3) for _ in range(2)]
    table = shuffled(B, 4, 50, dev)
    for c in caches:
        model(tok[:, :S], kv_cache=c, page_table=table)
    pos = torch.full((B,), S, dtype=torch.int64, device=dev)
    step = tok[:, S:S + 1].clone()
    spare = paged_cache(args, BF16, E4M3)
    model(step, kv_cache=spare, page_table=table, start_positions=pos)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = model(step, kv_cache=caches[0], page_table=table, start_positions=pos)
    for i in range(5):
        step.copy_(tok[:, S + i:S + i + 1])
        pos.fill_(S + i)
        g.replay()
        ref = model(step, kv_cache=caches[1], page_table=table, start_positions=pos)
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i
        assert torch.equal(caches[0].k.view(torch.uint8), caches[1].k.view(torch.uint8))


@torch.no_grad()
def test_refused_calls(dev):
    from src.cuda_graph import CUDAGraphDecodeRunner
    from src.kv_cache import KVCache
    args, model = small(dev)
    cache, tok = paged_cache(args, F32), prompt(1, 3, args.vocab_size, dev)
    table = shuffled(1, 2, 50, dev)
    with pytest.raises(ValueError, match="page_table"):
        model(tok, kv_cache=cache)
    for start in (-1, args.max_seq_len - 2):
        with pytest.raises(ValueError, match="positions"):
            model(tok, start, kv_cache=cache, page_table=table)
    with pytest.raises(ValueError, match="seq_lens"):
        model(tok, kv_cache=cache, page_table=table, seq_lens=torch.ones(1, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError, match="scatter_positions"):
        model(tok, kv_cache=cache, page_table=table, use_cuda_graph=True,
              scatter_positions=torch.arange(3, device=dev))
    with pytest.raises(ValueError, match="PagedKVCache"):
        model(tok, kv_cache=KVCache(args, dtype=F32), page_table=table)
    with pytest.raises(ValueError, match="KVCache"):
        CUDAGraphDecodeRunner(model, args, cache, str(dev))

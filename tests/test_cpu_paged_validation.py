"""CPU: argument checks of the paged cache, its append and attention, and the draft
verification: refused before anything launches (Python entry points and the C ABI)."""
import pytest
import torch

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
P = 1 << 20          # a non-null, aligned address that is never read


def args(**over):
    from src.config import ModelArgs
    return ModelArgs(**{**dict(dim=128, n_layers=2, n_heads=4, n_kv_heads=2, device="cpu"), **over})


def cache(**kw):
    from src.paged import PagedKVCache
    return PagedKVCache(args(), 6, 16, **{"dtype": BF16, **kw})


def test_cache_shapes():
    c = cache()
    assert c.k.shape == (2, 6, 2, 16, 32) and c.v.shape == (2, 6, 2, 32, 16) and c.scales is None
    c = cache(kv_dtype=E4M3)
    assert c.k.dtype == E4M3 and c.scales.shape == (2, 6, 2, 2) and c.scales.dtype == torch.float32
    from src.paged import PagedKVCache
    one = PagedKVCache.from_pages(c.k[0], c.v[0], c.scales[0], dtype=BF16)
    assert one.n_layers == 1 and one.k.data_ptr() == c.k.data_ptr()


@pytest.mark.parametrize("kw,exc", [
    (dict(page_size=24), ValueError), (dict(page_size=8), ValueError), (dict(num_pages=0), ValueError),
    (dict(dtype=torch.float64), TypeError), (dict(kv_dtype=torch.int8), TypeError),
    (dict(kv_dtype=torch.float16), TypeError),
])
def test_cache_refusals(kw, exc):
    from src.paged import PagedKVCache
    with pytest.raises(exc):
        PagedKVCache(args(), **{"num_pages": 4, "page_size": 16, "dtype": BF16, **kw})
    with pytest.raises(ValueError, match="head_dim"):
        PagedKVCache(args(n_heads=1, dim=264, n_kv_heads=1), 4, 16, dtype=BF16)


def test_from_pages_refusals():
    from src.paged import PagedKVCache
    k, v = torch.zeros(4, 2, 16, 32, dtype=BF16), torch.zeros(4, 2, 32, 16, dtype=BF16)
    with pytest.raises(ValueError, match="transposed"):
        PagedKVCache.from_pages(k, k)
    with pytest.raises(ValueError, match="scales"):
        PagedKVCache.from_pages(k, v, torch.ones(4, 2, 2))
    with pytest.raises(ValueError, match="scales"):
        PagedKVCache.from_pages(k.to(E4M3), v.to(E4M3), dtype=BF16)
    with pytest.raises(ValueError, match="scales"):
        PagedKVCache.from_pages(k.to(E4M3), v.to(E4M3), torch.ones(4, 2), dtype=BF16)
    with pytest.raises(ValueError, match="contiguous"):
        PagedKVCache.from_pages(k, k.transpose(2, 3))
    with pytest.raises(TypeError):
        PagedKVCache.from_pages(k, v.float())


def update(**over):
    from src.paged import rope_and_paged_update
    a = dict(xk=torch.zeros(1, 2, 3, 32, dtype=BF16), xv=torch.zeros(1, 2, 3, 32, dtype=BF16),
             rope_cos=torch.zeros(9, 16, dtype=BF16), rope_sin=torch.zeros(9, 16, dtype=BF16),
             cache=cache(), layer_idx=0, page_table=torch.zeros(1, 2, dtype=torch.int32), start_pos=0)
    return rope_and_paged_update(**{**a, **over})


@pytest.mark.parametrize("over,exc,msg", [
    ({}, ValueError, "CUDA"),
    (dict(layer_idx=2), ValueError, "layer_idx"),
    (dict(xv=torch.zeros(1, 2, 2, 32, dtype=BF16)), ValueError, "match"),
    (dict(xk=torch.zeros(1, 4, 3, 32, dtype=BF16), xv=torch.zeros(1, 4, 3, 32, dtype=BF16)), ValueError, "fit"),
    (dict(xk=torch.zeros(1, 2, 3, 32), xv=torch.zeros(1, 2, 3, 32)), TypeError, "dtype"),
    (dict(xq=torch.zeros(1, 3, 3, 32, dtype=BF16)), ValueError, "divisible"),
    (dict(xq=torch.zeros(1, 4, 2, 32, dtype=BF16)), ValueError, "xq"),
    (dict(xq=torch.zeros(1, 4, 3, 32)), TypeError, "q dtype"),
    (dict(rope_cos=torch.zeros(9, 8, dtype=BF16), rope_sin=torch.zeros(9, 8, dtype=BF16)), ValueError, "cos/sin"),
    (dict(rope_cos=torch.zeros(9, 16, dtype=torch.float16), rope_sin=torch.zeros(9, 16, dtype=torch.float16)),
     TypeError, "cos/sin"),
])
def test_update_refusals(over, exc, msg):
    with pytest.raises(exc, match=msg):
        update(**over)


@pytest.mark.parametrize("over,exc,msg", [
    ({}, ValueError, "CUDA"),
    (dict(q=torch.zeros(1, 4, 32, dtype=BF16)), ValueError, "rank-4"),
    (dict(q=torch.zeros(1, 4, 1, 64, dtype=BF16)), ValueError, "head_dim"),
    (dict(q=torch.zeros(1, 3, 1, 32, dtype=BF16)), ValueError, "divisible"),
    (dict(q=torch.zeros(1, 4, 1, 32)), TypeError, "dtype"),
])
def test_attention_refusals(over, exc, msg):
    from src.paged import paged_flash_attention
    a = dict(q=torch.zeros(1, 4, 1, 32, dtype=BF16), cache=cache(), layer_idx=0,
             page_table=torch.zeros(1, 2, dtype=torch.int32), seq_lens=torch.ones(1, dtype=torch.int64))
    with pytest.raises(exc, match=msg):
        paged_flash_attention(**{**a, **over})


def test_row_and_table_checks():
    from src import paged
    dev = -1   # the device index of host tensors
    with pytest.raises(ValueError, match="shape"):
        paged._per_row(torch.zeros(2, dtype=torch.int64), 3, dev, "seq_lens", "f")
    with pytest.raises(TypeError, match="integers"):
        paged._per_row(torch.zeros(3), 3, dev, "seq_lens", "f")
    assert paged._per_row(torch.ones(3, dtype=torch.int32), 3, dev, "seq_lens", "f").dtype == torch.int64
    assert paged._per_row(torch.arange(6)[::2], 3, dev, "x", "f").tolist() == [0, 2, 4]
    with pytest.raises(TypeError, match="int32"):
        paged._table(torch.zeros(3, 2, dtype=torch.int64), 3, dev, "f")
    with pytest.raises(ValueError, match="shape"):
        paged._table(torch.zeros(3, 0, dtype=torch.int32), 3, dev, "f")


@pytest.mark.parametrize("over,exc,msg", [
    ({}, ValueError, "CUDA"),
    (dict(target_logits=torch.zeros(2, 3, 9)), ValueError, "rows"),
    (dict(draft_tokens=torch.zeros(2, 3, dtype=torch.int32)), TypeError, "int64"),
    (dict(draft_tokens=torch.zeros(2, 0, dtype=torch.int64), target_logits=torch.zeros(2, 1, 9)), ValueError, "one draft"),
    (dict(accept_u=None), ValueError, "accept_u"),
    (dict(sample_u=torch.zeros(3)), ValueError, "sample_u"),
    (dict(accept_u=torch.zeros(2, 3, dtype=torch.float64)), ValueError, "accept_u"),
    (dict(temperature=-1.0), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(temperature=1e-9), ValueError, "temperature"),
    (dict(draft_logits=torch.zeros(2, 4, 9)), ValueError, "draft_logits"),
    (dict(draft_logits=torch.zeros(2, 3, 9, dtype=BF16)), TypeError, "draft_logits"),
    (dict(target_logits=torch.zeros(2, 4, 9, dtype=torch.float64)), TypeError, "dtype"),
])
def test_verify_refusals(over, exc, msg):
    from src.verify import verify_drafts
    a = dict(target_logits=torch.zeros(2, 4, 9), draft_tokens=torch.zeros(2, 3, dtype=torch.int64),
             accept_u=torch.zeros(2, 3), sample_u=torch.zeros(2))
    a.update(over)
    with pytest.raises(exc, match=msg):
        verify_drafts(a.pop("target_logits"), a.pop("draft_tokens"), **a)


# ------------------------------------------------------------------ C ABI

def c_append(**o):
    from src import _lib
    a = dict(xq=None, xk=P, xv=P, cos=P, sin=P, qo=None, kp=P, vp=P, sc=None, pt=P, first=0, start=None,
             lens=None, rows=64, B=1, Hq=4, Hkv=2, S=1, D=64, pages=8, page=16, slots=4, dtype=0,
             cdtype=0, store=0)
    a.update(o)
    return _lib.load().mi_rope_paged_append(
        a["xq"], a["xk"], a["xv"], a["cos"], a["sin"], a["qo"], a["kp"], a["vp"], a["sc"], a["pt"],
        a["first"], a["start"], a["lens"], a["rows"], a["B"], a["Hq"], a["Hkv"], a["S"], a["D"],
        a["pages"], a["page"], a["slots"], *[64] * 12, 4, 32, 32, a["dtype"], a["cdtype"], a["store"],
        None)


def c_attn(**o):
    from src import _lib
    a = dict(q=P, kp=P, vp=P, sc=None, pt=P, sl=P, ql=None, part=None, n=0, out=P, lse=None, B=1, Hq=4,
             Hkv=2, S=1, D=64, pages=8, page=16, slots=4, splits=1, dtype=0, store=0, scale=0.125)
    a.update(o)
    return _lib.load().mi_paged_attn(
        a["q"], a["kp"], a["vp"], a["sc"], a["pt"], a["sl"], a["ql"], a["part"], a["n"], a["out"],
        a["lse"], a["B"], a["Hq"], a["Hkv"], a["S"], a["D"], a["pages"], a["page"], a["slots"],
        a["splits"], *[64] * 6, 4, a["scale"], a["dtype"], a["store"], None)


SHARED = [
    ({"kp": None}, -1, "null"), ({"dtype": 5}, -1, "dtype"), ({"store": 2}, -1, "store"),
    ({"store": 1}, -1, "scales"), ({"Hq": 3}, -1, "divisible"), ({"D": 258}, -2, "head_dim"),
    ({"page": 24}, -2, "page_size"), ({"page": 512}, -2, "page_size"), ({"slots": 0}, -1, "shape"),
    ({"pages": 0}, -1, "shape"), ({"slots": 1 << 40}, -2, "range"), ({"B": 1 << 40}, -2, "range"),
    ({"B": -1}, -1, "shape"),
]


@pytest.mark.parametrize("over,code,msg", SHARED + [
    ({"xq": P}, -1, "null"), ({"D": 63}, -1, "even"), ({"cdtype": 1}, -1, "cos/sin"),
    ({"rows": 0}, -1, "cos/sin"), ({"B": 1 << 20, "S": 1 << 20}, -2, "too many"),
])
def test_c_append_refusals(over, code, msg):
    from src import _lib
    assert c_append(**over) == code
    assert msg in _lib.last_error()


@pytest.mark.parametrize("over,code,msg", SHARED + [
    ({"sl": None}, -1, "null"), ({"splits": 0}, -1, "num_splits"), ({"splits": 65537}, -1, "num_splits"),
    ({"splits": 2}, -1, "workspace"), ({"splits": 2, "part": P, "n": 2 * 2 * 2 * 16 * 66 - 1}, -1, "workspace"),
    ({"splits": 2, "part": P + 4, "n": 1 << 30}, -1, "workspace"), ({"splits": 2, "dtype": 2, "part": P, "n": 2 * 4 * 66 - 1}, -1, "workspace"),
    ({"B": 1 << 20, "slots": 1 << 22}, -2, "too many"),
    ({"scale": 0.0}, -1, "sm_scale"), ({"scale": -1.0}, -1, "sm_scale"), ({"scale": float("nan")}, -1, "sm_scale"),
    ({"scale": float("inf")}, -1, "sm_scale"), ({"kp": P + 8}, -1, "aligned"), ({"B": 1 << 20, "S": 1 << 20}, -2, "too many"),
])
def test_c_attention_refusals(over, code, msg):
    from src import _lib
    assert c_attn(**over) == code
    assert msg in _lib.last_error()


def test_c_empty_calls_launch_nothing():
    assert c_append(B=0) == 0 and c_append(S=0) == 0 and c_attn(B=0) == 0 and c_attn(S=0) == 0


@pytest.mark.parametrize("over,code,msg", [
    ({"t": None}, -1, "null"), ({"u": None}, -1, "null"), ({"n": 7}, -1, "workspace"),
    ({"ws": P + 4}, -1, "workspace"), ({"dtype": 9}, -1, "dtype"), ({"V": 0}, -1, "shape"),
    ({"S": 0}, -2, "drafts"), ({"S": 129}, -2, "drafts"), ({"B": 60000}, -2, "drafts"),
    ({"temp": -0.5}, -1, "temperature"), ({"temp": float("nan")}, -1, "temperature"),
    ({"temp": float("inf")}, -1, "temperature"),
])
def test_c_verify_refusals(over, code, msg):
    from src import _lib
    a = dict(t=P, d=P, x=P, u=P, r=P, lens=None, out=P, acc=P, ws=P, n=1 << 30, B=2, S=3, V=1000,
             temp=1.0, dtype=0)
    a.update(over)
    st = _lib.load().mi_verify_drafts(
        a["t"], a["d"], a["x"], a["u"], a["r"], a["lens"], a["out"], a["acc"], a["ws"], a["n"], a["B"],
        a["S"], a["V"], *[1000] * 4, 3, 1, 3, 1, a["temp"], a["dtype"], None)
    assert st == code and msg in _lib.last_error()


def test_workspace_and_split_questions_take_any_shape():
    from src import _lib
    lib = _lib.load()
    assert lib.mi_verify_drafts_workspace(0, 1, 10) == 0
    assert lib.mi_verify_drafts_workspace(2, 3, 1000) > 0
    for shape in ((0, 4, 2, 1, 64, 16, 4), (1, 4, 2, 1, 64, 0, 4), (1, 4, 2, 1, 64, 16, 1 << 62),
                  (1 << 40, 4, 2, 1, 64, 16, 4)):
        assert lib.mi_paged_attn_splits(*shape, 0, 1) == 1
    for shape in ((0, 4, 2, 1, 64, 5), (1, 4, 2, 1, 64, 1), (1, 4, 3, 1, 64, 5), (1, 4, 2, 1, 512, 5)):
        assert lib.mi_paged_attn_workspace(*shape, 0) == 0

"""Refusals of the E4M3 cache operators that need no GPU, and the 64-bit
oracle against brute force."""
import ctypes

import pytest
import torch

import kv8util
from oracle import kv8 as ok
from test_abi import test_struct_layout_matches_header as check_layout
from wam_ops import _lib
from wam_ops.kv8 import Kv8Cache


@pytest.mark.parametrize("cname,pyname", [
    ("wamb_kv8_cache", "Kv8CacheArgs"), ("wamb_kv8_seqs", "Kv8SeqsArgs"), ("wamb_kv8_write_args", "Kv8WriteArgs"),
    ("wamb_kv8_attention_args", "Kv8AttentionArgs"), ("wamb_kv8_evict_args", "Kv8EvictArgs")])
def test_struct_layout(tmp_path, cname, pyname):
    check_layout(tmp_path, cname, pyname)


def _cache(a, **kw):
    c = a.cache
    c.k8, c.v8, c.k_scale, c.v_scale, c.pages, c.heads, c.page = 0x1000, 0x2000, 0x3000, 0x4000, 10, 2, 64
    s = a.seqs
    s.batch, s.tokens, s.table_width, s.table, s.lens = 2, 1, 4, 0x5000, 0x6000
    for k, v in kw.items():
        part, name = k.split("_", 1)
        setattr({"c": c, "s": s, "a": a}[part], name, v)
    return a


def _write(**kw):
    a = _lib.Kv8WriteArgs()
    a.k, a.v = 0x7000, 0x8000
    a.k_stride[:] = a.v_stride[:] = (256, 256, 128)
    return _cache(a, **kw)


def _attention(**kw):
    a = _lib.Kv8AttentionArgs()
    a.q, a.out, a.q_heads, a.scale = 0x7000, 0x8000, 4, 0.1
    a.q_stride[:] = a.out_stride[:] = (512, 512, 128)
    a.lse, a.weights, a.weights_cap = 0x9000, 0xa000, 256
    return _cache(a, **kw)


def _evict(**kw):
    a = _lib.Kv8EvictArgs()
    a.weights, a.weights_cap, a.max_len, a.new_table, a.new_width = 0x7000, 256, 256, 0x8000, 2
    a.heavy, a.recent, a.kept, a.new_weights, a.new_lens = 60, 60, 0x9000, 0xa000, 0xb000
    return _cache(a, **kw)


COMMON = [({"c_k8": None}, 1), ({"c_v_scale": None}, 1), ({"c_k8": 0x1008}, 3), ({"c_page": 48}, 2), ({"c_page": 0}, 2),
          ({"c_pages": 0}, 2), ({"c_heads": 0}, 2), ({"c_pages": 1 << 30}, 2), ({"s_batch": -1}, 2),
          ({"s_batch": 40000}, 2), ({"s_tokens": -1}, 2), ({"s_table_width": 0}, 2), ({"s_table_width": 1 << 30}, 2),
          ({"s_table": None}, 1), ({"s_lens": None}, 1)]


@pytest.mark.parametrize("make,call", [(_write, "wamb_kv8_write"), (_attention, "wamb_kv8_attention"),
                                       (_attention, "wamb_kv8_weights"), (_evict, "wamb_kv8_evict")])
@pytest.mark.parametrize("kw,code", COMMON)
def test_common_refusals(make, call, kw, code):
    lib = _lib.load()
    assert getattr(lib, call)(make(**kw), None) == code
    assert lib.wamb_last_error()


@pytest.mark.parametrize("kw,code", [({"a_k": None}, 1), ({"a_v": 0x8008}, 3), ({"a_x_is_f32": 2}, 1)])
def test_write_refusals(kw, code):
    assert _lib.load().wamb_kv8_write(_write(**kw), None) == code


def test_stride_refusals():
    lib = _lib.load()
    for field in ("k_stride", "v_stride"):
        a = _write()
        getattr(a, field)[1] = 132
        assert lib.wamb_kv8_write(a, None) == 3
    for field in ("q_stride", "out_stride"):
        a = _attention()
        getattr(a, field)[0] = 516
        assert lib.wamb_kv8_attention(a, None) == 3


@pytest.mark.parametrize("kw,code", [({"a_q": None}, 1), ({"a_q": 0x7008}, 3), ({"a_q_heads": 3}, 2), ({"a_q_heads": 0}, 2),
                                     ({"a_causal": 2}, 1), ({"a_scale": 0.0}, 1), ({"a_scale": float("nan")}, 1),
                                     ({"a_scale": float("inf")}, 1), ({"s_tokens": 1 << 29}, 2)])
@pytest.mark.parametrize("call", ["wamb_kv8_attention", "wamb_kv8_weights"])
def test_attention_refusals(call, kw, code):
    assert getattr(_lib.load(), call)(_attention(**kw), None) == code


def test_weights_and_out_refusals():
    lib = _lib.load()
    assert lib.wamb_kv8_attention(_attention(a_out=None), None) == 1
    assert lib.wamb_kv8_attention(_attention(a_out=0x8008), None) == 3
    assert lib.wamb_kv8_weights(_attention(a_weights=None), None) == 1
    assert lib.wamb_kv8_weights(_attention(a_lse=None), None) == 1
    assert lib.wamb_kv8_weights(_attention(a_weights_cap=255), None) == 2


@pytest.mark.parametrize("kw,code", [({"a_heavy": -1}, 1), ({"a_recent": -1}, 1), ({"a_new_width": 0}, 2),
                                     ({"a_new_width": 1 << 30}, 2), ({"a_recent": 100}, 2), ({"a_max_len": 257}, 2),
                                     ({"a_weights": None}, 1), ({"a_new_table": None}, 1), ({"a_kept": None}, 1),
                                     ({"a_new_lens": None}, 1), ({"a_new_weights": 0x7000}, 1), ({"a_weights_cap": 255}, 2)])
def test_evict_refusals(kw, code):
    assert _lib.load().wamb_kv8_evict(_evict(**kw), None) == code


def test_null_and_empty():
    lib = _lib.load()
    for f in (lib.wamb_kv8_write, lib.wamb_kv8_attention, lib.wamb_kv8_weights, lib.wamb_kv8_evict):
        assert f(None, None) == 1
    assert lib.wamb_kv8_write(_write(s_batch=0, s_table=None, s_lens=None, a_k=None), None) == 0
    assert lib.wamb_kv8_write(_write(s_tokens=0, a_k=None), None) == 0
    assert lib.wamb_kv8_attention(_attention(s_tokens=0, a_q=None), None) == 0
    assert lib.wamb_kv8_evict(_evict(s_batch=0), None) == 0
    assert lib.wamb_kv8_attention_workspace_bytes(None) == 0


def test_handle_refuses_tensors():
    k = torch.zeros(3, 2, 64, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones(3, 2)
    for bad in ((k, k, s, s),                                                   # not on a GPU
                (k[:, :, :50], k[:, :, :50], s, s), (k[..., :64], k[..., :64], s, s), (k, k[:2], s, s),
                (k.view(torch.uint8), k, s, s), (k.transpose(0, 1), k.transpose(0, 1), s, s), (k, k, s.double(), s),
                (k, k, s, s[:2])):
        with pytest.raises(ValueError):
            Kv8Cache(*bad)


# ------------------------------------------------------------------ oracle
def test_oracle_rounds_like_torch():
    x = torch.cat([torch.linspace(-500, 500, 4001), torch.linspace(-0.05, 0.05, 4001),
                   torch.tensor([0.0, 448.0, 464.0, 2.0 ** -10, 3 * 2.0 ** -10, float("nan")])]).double()
    want = x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(ok.round_e4m3(x).nan_to_num(999.0), want.nan_to_num(999.0))


def test_oracle_scale():
    for a in (0.0, 1.0, 447.9, 448.0, 448.1, 3e38, float("inf"), 1e-30, 2.0 ** -33, 7.0):
        s = ok.block_scale(a)
        assert s == 2.0 ** -40 or 448 * s / 2 < min(a, 3.4028235e38)
        assert min(a, 448 * 2.0 ** 119) <= 448 * s          # larger magnitudes saturate


def test_oracle_attention_and_weights_are_softmax():
    g = torch.Generator().manual_seed(0)
    table, _, pages = kv8util.tables(1, 3, 1, g)
    k8, v8, ks, vs = kv8util.cache(pages, 2, 16, g, "cpu")
    q = torch.randn(1, 5, 4, 128, generator=g).bfloat16()
    out, lse, _, _ = ok.attention(q, k8, v8, ks, vs, table, [37], causal=True)
    k, v = ok.sequence(k8, ks, table[0], 37), ok.sequence(v8, vs, table[0], 37)
    mask = torch.ones(5, 37, dtype=torch.bool).tril(32)
    for h in range(4):
        s = (q[0, :, h].double() @ k[h // 2].T / 128 ** 0.5).masked_fill(~mask, float("-inf"))
        assert torch.allclose(out[0, :, h], torch.softmax(s, 1) @ v[h // 2], atol=1e-12)
        assert torch.allclose(lse[0, :, h], torch.logsumexp(s, 1), atol=1e-12)
    w, _ = ok.weights(q, k8, ks, table, [37], lse, torch.zeros(1, 2, 48), causal=True)
    assert torch.allclose(w.sum(2), torch.full((1, 2), 10.0, dtype=torch.float64))
    assert (w[:, :, 37:] == 0).all()


def test_oracle_keep():
    assert ok.keep([1.0, 3.0, 3.0, 0.0, 9.0, 9.0], 6, 2, 1) == [1, 4, 5]
    assert ok.keep([1.0, 3.0, 3.0, 0.0, 9.0], 4, 2, 1) == [1, 2, 3]
    assert ok.keep([1.0, float("nan"), 0.0], 3, 1, 0) == [1]
    assert ok.keep([1.0, 2.0], 2, 0, 5) == [0, 1]


@pytest.mark.parametrize("make,call", [(_write, "wamb_kv8_write"), (_attention, "wamb_kv8_attention"),
                                       (_attention, "wamb_kv8_weights"), (_evict, "wamb_kv8_evict")])
def test_refuses_more_positions_than_tiles_can_count(make, call):
    """2^30 cached positions and one new token: 32-bit tile ends behind them must not wrap."""
    lib = _lib.load()
    assert getattr(lib, call)(make(s_table_width=1 << 24, s_tokens=1), None) == 2
    assert b"2^30" in lib.wamb_last_error()


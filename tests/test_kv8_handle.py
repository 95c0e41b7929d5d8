"""Argument checks of the handle (wam_ops.kv8.Kv8Cache) that need no GPU: they
run on a handle whose tensors are on the CPU and whose library calls are
recorded."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from wam_ops import _lib
from wam_ops.kv8 import Kv8Cache

PAGE, HEADS, PAGES = 16, 2, 12


@pytest.fixture
def cache():
    """(handle, list of the calls that passed its checks)."""
    c = object.__new__(Kv8Cache)
    code = torch.zeros(PAGES, HEADS, PAGE, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.ones(PAGES, HEADS)
    c.k8, c.v8, c.k_scale, c.v_scale = code, code.clone(), scale, scale.clone()
    c.device, c.pages, c.heads, c.page = torch.device("cpu"), PAGES, HEADS, PAGE
    c._c = _lib.Kv8CacheArgs(code.data_ptr(), c.v8.data_ptr(), scale.data_ptr(), c.v_scale.data_ptr(), PAGES, HEADS, PAGE)
    c._lib, c._scratch = _lib.load(), {}
    calls = []
    c._call = lambda fn, args, *rest: calls.append(args)
    return c, calls


TABLE = torch.arange(8, dtype=torch.int32).view(2, 4)
LENS = torch.tensor([40, 20], dtype=torch.int32)
NEW = torch.tensor([[8, 9], [10, 11]], dtype=torch.int32)


def _inputs():
    q = torch.randn(2, 3, HEADS, 128).bfloat16()
    return q, torch.zeros(2, 3, HEADS), torch.rand(2, HEADS, 64)


def test_the_calls_pass_without_gradients(cache):
    c, calls = cache
    q, lse, w = _inputs()
    c.write(q, q, TABLE, LENS)
    c.attention(q, TABLE, LENS)
    c.weights(q, TABLE, LENS, lse, base=w, out=w)
    c.evict(TABLE, LENS, w, NEW, heavy=20, recent=10)
    assert len(calls) == 4


def _refused(c, calls, name):
    """Each call with its input `name` replaced by mark(input)."""
    q, lse, w = _inputs()

    def use(mark):
        m = {n: mark(t) if n == name else t for n, t in (("q", q), ("k", q), ("v", q.clone()), ("out", torch.empty_like(q)),
                                                         ("lse", lse), ("base", w), ("wout", w.clone()), ("w", w))}
        if name in ("k", "v"):
            return c.write(m["k"], m["v"], TABLE, LENS)
        if name in ("q", "out"):
            return c.attention(m["q"], TABLE, LENS, out=m["out"])
        if name == "lse_out":
            return c.attention(q, TABLE, LENS, lse=mark(lse))
        if name in ("lse", "base", "wout"):
            return c.weights(q, TABLE, LENS, m["lse"], base=m["base"], out=m["wout"])
        return c.evict(TABLE, LENS, m["w"], NEW, heavy=20, recent=10)
    return use


NAMES = ["k", "v", "q", "out", "lse_out", "lse", "base", "wout", "w"]


@pytest.mark.parametrize("name", NAMES)
def test_leaves_are_refused(cache, name):
    """A result without a graph, or a leaf written in place, would be silent."""
    c, calls = cache
    use = _refused(c, calls, name)
    with pytest.raises(RuntimeError, match="inference-only"):
        use(lambda t: t.clone().requires_grad_())
    assert not calls
    with torch.no_grad():
        use(lambda t: t.clone().requires_grad_())
    assert len(calls) == 1


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(cache, name):
    """Forward-mode derivatives would be dropped."""
    c, calls = cache
    use = _refused(c, calls, name)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="inference-only"):
            use(lambda t: fwd.make_dual(t.clone(), torch.ones_like(t)))
        assert not calls
        use(lambda t: t)
    assert len(calls) == 1


def test_in_place_sum_of_a_leaf_is_refused(cache):
    c, calls = cache
    q, lse, w = _inputs()
    w.requires_grad_()
    with pytest.raises(RuntimeError, match="inference-only"):
        c.weights(q, TABLE, LENS, lse, base=w, out=w)
    assert not calls


@pytest.mark.parametrize("heavy,recent,max_len", [(2 ** 32 + 5, 10, None), (20, 2 ** 32, None), (2 ** 31, 0, None),
                                                  (20, -2 ** 32, None), (20, 10, 2 ** 64 + 30)])
def test_evict_refuses_numbers_that_would_wrap(cache, heavy, recent, max_len):
    """2^32 'keep all' would be taken as 0, and the latest tokens dropped."""
    c, calls = cache
    w = _inputs()[2]
    with pytest.raises(ValueError, match="heavy, recent"):
        c.evict(TABLE, LENS, w, NEW, heavy=heavy, recent=recent, max_len=max_len)
    assert not calls


def test_evict_takes_the_largest_numbers(cache):
    c, calls = cache
    w = _inputs()[2]
    c.evict(TABLE, LENS, w, NEW, heavy=2 ** 31 - 1, recent=2 ** 31 - 1, max_len=30)
    assert (calls[0].heavy, calls[0].recent, calls[0].max_len) == (2 ** 31 - 1, 2 ** 31 - 1, 30)


def test_sizes_that_would_wrap_are_refused(cache):
    """Expanded inputs can have more rows than 32 bits count."""
    c, calls = cache
    k = torch.zeros(1, 1, HEADS, 128).bfloat16().expand(1, 2 ** 32 + 1, HEADS, 128)
    with pytest.raises(ValueError, match="2\\^31"):
        c.write(k, k, TABLE[:1], LENS[:1])
    q = torch.zeros(1, 1, 1, 128).bfloat16().expand(1, 1, 2 ** 32 + HEADS, 128)
    with pytest.raises(ValueError, match="2\\^31"):
        c.weights(q, TABLE[:1], LENS[:1], torch.zeros(1, 1, HEADS))
    assert not calls

"""The E4M3 KV cache operators (wam_ops.kv8) against their definitions in 64 bits.

Codes, scales, kept positions and lengths are compared exactly; attention and
weights within the bounds that oracle/kv8.py derives from the roundings that
the documentation names.
"""
import math

import pytest
import torch

import kv8util
from oracle import kv8 as ok
from wam_ops import _lib
from wam_ops.kv8 import Kv8Cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _setup(B, H, P, lens, seed, extra=0, spare=2, spread=0.7, poison=True):
    g = torch.Generator().manual_seed(seed)
    width = max(1, -(-(max(lens) + extra) // P))
    table, free, pages = kv8util.tables(B, width, spare, g, DEV)
    k8, v8, ks, vs = kv8util.cache(pages, H, P, g, DEV, spread)
    if poison:
        for c, s in ((k8, ks), (v8, vs)):
            kv8util.poison(c, s, table.cpu(), lens)
    return Kv8Cache(k8, v8, ks, vs), table, free, _i32(lens), g


def _close(x, ref, tol, what):
    x = x.double()
    same = (x == ref) | (x.isnan() & ref.isnan())
    bad = ~same & ~((x - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {((x - ref).abs() - tol)[bad].max()} over the bound"


# ------------------------------------------------------------------ write
def _check_write(c, k, v, table, lens, counts=None):
    want = ok.write(c.k8, c.v8, c.k_scale, c.v_scale, k, v, table, lens, counts)
    c.write(k, v, table, lens, counts)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    for got, ref in zip((ok.values(c.k8), ok.values(c.v8), c.k_scale.double(), c.v_scale.double()), want):
        assert torch.equal(got.nan_to_num(999.0), ref.nan_to_num(999.0))


@pytest.mark.parametrize("B,H,P,T,lens,dtype", [
    (1, 1, 16, 1, [0], "bf16"), (3, 2, 16, 1, [15, 16, 17], "bf16"), (2, 3, 64, 1, [63, 1], "fp32"),
    (2, 2, 32, 37, [5, 64], "bf16"), (3, 5, 64, 130, [0, 63, 100], "bf16"), (2, 1, 128, 300, [127, 1], "fp32"),
    (1, 24, 64, 64, [64], "bf16"), (4, 2, 16, 333, [0, 1, 16, 31], "fp32"),
])
def test_write(cuda_device, B, H, P, T, lens, dtype):
    c, table, _, n, g = _setup(B, H, P, lens, T, extra=T)
    dt = torch.float32 if dtype == "fp32" else torch.bfloat16
    k, v = (torch.exp(torch.randn(B, T, H, 1, generator=g)).mul(torch.randn(B, T, H, 128, generator=g)).to(DEV, dt)
            for _ in range(2))
    _check_write(c, k, v, table, n)


def test_write_counts_leave_the_rest(cuda_device):
    c, table, _, n, g = _setup(4, 2, 32, [0, 31, 40, 7], 1, extra=70)
    k = torch.randn(4, 70, 2, 128, generator=g).to(DEV, torch.bfloat16)
    _check_write(c, k, k.flip(0).contiguous(), table, n, _i32([70, 0, 1, 33]))


def test_write_reads_strided_rows(cuda_device):
    """K and V inside one projection output, and heads that are a slice of more."""
    c, table, _, n, g = _setup(2, 3, 16, [3, 20], 2, extra=20)
    qkv = torch.randn(2, 20, 3, 7, 128, generator=g).to(DEV, torch.bfloat16)
    _check_write(c, qkv[:, :, 1, 2:5], qkv[:, :, 2, 4:7], table, n)
    _check_write(c, qkv[:, ::2, 0, ::3], qkv[:, ::2, 1, ::3], table, n)
    t = torch.randn(2, 3, 20, 128, generator=g).to(DEV, torch.bfloat16)
    _check_write(c, t.transpose(1, 2), t.transpose(1, 2), table, n)
    one = torch.randn(1, 1, 3, 128, generator=g).to(DEV)
    _check_write(c, one.expand(2, 20, 3, 128), one.expand(2, 20, 3, 128), table, n)


@pytest.mark.parametrize("P", [16, 64])
def test_write_extreme_values(cuda_device, P):
    """Zeros, tiny and huge blocks, borders of the scale, infinities and NaN."""
    c, table, _, n, g = _setup(1, 1, P, [0], 3, extra=12 * P)
    x = torch.randn(1, 12 * P, 1, 128, generator=g)
    r = x[0, :, 0].view(12, P, 128)
    for i, f in enumerate((0.0, 1e-38, 1e-12, 2.0 ** -40, 1e30, 3e38)):
        r[i] *= f
    r[2, 0, 0] = 448.0 * 2.0 ** -39
    r[3, 0, :2] = torch.tensor([448.0, 449.0])
    r[4, 0, 0] = math.inf
    r[5, 1, 3] = -math.inf
    r[6, 2, 5] = math.nan
    r[7].fill_(math.nan)
    r[8] = torch.linspace(-448, 448, P * 128).view(P, 128)          # every rounding, ties among them
    r[9] = torch.linspace(-2.0 ** -5, 2.0 ** -5, P * 128).view(P, 128)
    r[9, 0, 0] = 448.0
    _check_write(c, x.to(DEV), (-x).to(DEV), table, n)


def test_write_token_by_token_grows_scales(cuda_device):
    """Appends of one token: a page's codes follow its growing scale."""
    c, table, _, n, g = _setup(2, 2, 16, [0, 5], 4, extra=40)
    for i in range(40):
        x = torch.randn(2, 1, 2, 128, generator=g) * 2.0 ** torch.randint(-3, 6, (1,), generator=g)
        _check_write(c, x.to(DEV, torch.bfloat16), (x * 3).to(DEV, torch.bfloat16), table, n)
        n += 1


def test_write_nothing(cuda_device):
    c, table, _, n, g = _setup(2, 2, 16, [0, 5], 4)
    before = c.k8.view(torch.uint8).clone()
    c.write(torch.zeros(2, 0, 2, 128, device=DEV), torch.zeros(2, 0, 2, 128, device=DEV), table, n)
    c.write(*(torch.zeros(2, 1, 2, 128, device=DEV),) * 2, table, n, _i32([0, 0]))
    assert torch.equal(before, c.k8.view(torch.uint8))


# -------------------------------------------------------------- attention
def _check_attention(c, q, table, lens, counts=None, causal=False, scale=None, out=None):
    n = lens.cpu()
    ref, rlse, tol, ltol = ok.attention(q, c.k8, c.v8, c.k_scale, c.v_scale, table, n, counts, causal, scale)
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full(q.shape[:3], 7.0, device=DEV)
    o, z = c.attention(q, table, lens, counts, causal, scale, out=out, lse=lse, return_lse=True)
    assert o is out and z is lse
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    behind = ref.isnan()                              # rows past counts: as they were
    assert (out[behind] == 7.0).all() and (lse[rlse.isnan()] == 7.0).all()
    _close(out.masked_fill(behind, 0.0), ref.nan_to_num(0.0), tol, "out")
    gone = rlse.isnan()
    _close(lse.masked_fill(gone, 0.0), rlse.masked_fill(gone, 0.0), ltol, "lse")
    return out, lse


def _q(g, *shape, gain=2.0):
    return (gain * torch.randn(*shape, generator=g)).to(DEV, torch.bfloat16)


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500]


@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (3, 5), (17, 1), (40, 3), (130, 1), (257, 2)])
def test_attention_ragged(cuda_device, P, T, G):
    """Lengths from none to several tiles, few to many rows; what lies behind
    a sequence is NaN."""
    c, table, _, n, g = _setup(len(LENS), 2, P, LENS, 10 * T + G)
    _check_attention(c, _q(g, len(LENS), T, 2 * G, 128), table, n)


@pytest.mark.parametrize("P,T,G", [(16, 1, 2), (64, 7, 2), (64, 33, 1), (128, 140, 2), (32, 300, 1)])
def test_attention_causal_and_counts(cuda_device, P, T, G):
    """Rows that see nothing (fewer positions than rows), padded rows."""
    lens = [0, 1, 5, 64, 130, 300, 471]
    counts = [T, 1, T, max(1, T // 2), 0, T - T // 3, T]
    c, table, _, n, g = _setup(len(lens), 3, P, lens, T)
    q = _q(g, len(lens), T, 3 * G, 128)
    _check_attention(c, q, table, n, causal=True)
    _check_attention(c, q, table, n, counts=_i32(counts), causal=True)
    _check_attention(c, q, table, n, counts=_i32(counts))


@pytest.mark.parametrize("T", [1, 9, 70])
def test_attention_strides_scale_and_shared_pages(cuda_device, T):
    c, table, _, n, g = _setup(2, 2, 32, [150, 150], 6, poison=False)
    qkv = _q(g, 2, T, 3, 8, 128)
    out = torch.full((2, 4, T, 256), 7.0, dtype=torch.bfloat16, device=DEV)
    view = out.transpose(1, 2)[..., 128:]
    _check_attention(c, qkv[:, :, 1, 2:6], table, n, scale=0.31, out=view)
    assert (out[..., :128] == 7.0).all()
    both = table[:1].expand(2, -1).contiguous()       # candidates over one history
    _check_attention(c, qkv[:, :, 0, ::2], both, n)


@pytest.mark.parametrize("T", [1, 40])
def test_attention_extreme_scales(cuda_device, T):
    """Values and scores over many binades: blocks of V that differ by 2^40,
    peaked rows, rows of zeros, general scales; the maximum grows late."""
    c, table, _, n, g = _setup(3, 2, 16, [200, 333, 90], 7, spread=2.5)
    c.v_scale[table[0].long()] *= 2.0 ** torch.randint(-20, 20, (table.shape[1], 2), generator=g).to(DEV)
    c.k_scale[table[1].long()] *= 1.37                  # no power of two
    c.v_scale[table[1].long()] *= 0.83
    q = _q(g, 3, T, 4, 128, gain=3.0)
    q[:, :, 1] = 0.0
    q[:, :, 2] *= torch.linspace(0.001, 30, 128, device=DEV).bfloat16()
    q[0, :, 3] *= 2.0 ** 100
    q[1, :, 3] *= 2.0 ** -100
    c.k8.view(torch.uint8)[table[2, 0].long()] &= 0x87      # the first keys are tiny: the maximum moves later
    _check_attention(c, q[:, :, :3].repeat_interleave(2, 2)[:, :, :4].contiguous(), table, n)
    q[0, :, 3] *= 2.0 ** -100
    _check_attention(c, q, table, n, scale=0.02)


@pytest.mark.parametrize("T", [1, 40])
def test_attention_nan_row_stays_its_own(cuda_device, T):
    """A query of NaN or infinity makes its own row NaN and no other."""
    c, table, _, n, g = _setup(1, 1, 64, [100], 8)
    q = _q(g, 1, T, 3, 128)
    clean = c.attention(q, table, n)
    q[0, T - 1, 1, 5] = math.nan
    q[0, T - 1, 2, 9] = math.inf
    out = c.attention(q, table, n)
    assert out[0, T - 1, 1:].isnan().all()
    keep = torch.ones(T, 3, dtype=torch.bool)
    keep[T - 1, 1:] = False
    assert torch.equal(out[0][keep], clean[0][keep])


@pytest.mark.parametrize("B,H,G,T,L", [(1, 1, 1, 1, 40000), (1, 1, 8, 2, 9000), (2, 3, 1, 1, 7777), (1, 2, 2, 200, 5000)])
def test_attention_long(cuda_device, B, H, G, T, L):
    """One item over many CTAs: partials are joined."""
    lens = [L - 13 * b for b in range(B)]
    c, table, _, n, g = _setup(B, H, 128, lens, L, poison=False)
    q = _q(g, B, T, H * G, 128)
    out, lse = _check_attention(c, q, table, n)
    again, lse2 = c.attention(q, table, n, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("T", [1, 20])
def test_cache_beyond_32_bit_offsets(cuda_device, T):
    """Pages whose codes lie more than 4 GB into the cache."""
    H, P = 4, 128
    pages = 70000                                    # 4.6 GB for K and for V
    c = Kv8Cache.empty(pages, H, P, DEV)
    g = torch.Generator().manual_seed(9)
    table = _i32([[69999, 33000, 65600], [1, 69998, 69000]])
    n = _i32([0, 0])
    k, v = (torch.randn(2, 300, H, 128, generator=g).to(DEV, torch.bfloat16) for _ in range(2))
    c.write(k, v, table, n)
    n += 300
    small = Kv8Cache.empty(6, H, P, DEV)
    near = _i32([[0, 1, 2], [3, 4, 5]])
    small.write(k, v, near, n - 300)
    ids = table.flatten().long()
    assert torch.equal(c.k8.view(torch.uint8)[ids], small.k8.view(torch.uint8))
    assert torch.equal(c.v8.view(torch.uint8)[ids], small.v8.view(torch.uint8))
    q = _q(g, 2, T, H, 128)
    for a, b in zip(c.attention(q, table, n, return_lse=True), small.attention(q, near, n, return_lse=True)):
        assert torch.equal(a, b)
    lse = small.attention(q, near, n, return_lse=True)[1]
    assert torch.equal(c.weights(q, table, n, lse), small.weights(q, near, n, lse))
    new = _i32([[69997], [68000]])
    w = torch.rand(2, H, 3 * P, generator=g).to(DEV)
    kept, _, _ = c.evict(table, n, w, new, heavy=60, recent=20)
    small2 = Kv8Cache.empty(8, H, P, DEV)
    for a, b in ((small2.k8, small.k8), (small2.v8, small.v8)):
        a.view(torch.uint8)[:6] = b.view(torch.uint8)
    small2.k_scale[:6], small2.v_scale[:6] = small.k_scale, small.v_scale
    kept2, _, _ = small2.evict(near, n, w, _i32([[6], [7]]), heavy=60, recent=20)
    assert torch.equal(kept, kept2)
    assert torch.equal(c.v8.view(torch.uint8)[new.flatten().long()], small2.v8.view(torch.uint8)[6:])


# ---------------------------------------------------------------- weights
def _check_weights(c, q, table, lens, cap, counts=None, causal=False, scale=None, inplace=False, base=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    _, lse, _, _ = ok.attention(q, c.k8, c.v8, c.k_scale, c.v_scale, table, lens.cpu(), counts, causal, scale)
    lse = lse.float().to(DEV)                         # NaN behind counts: not read
    w0 = torch.rand(q.shape[0], c.heads, cap, generator=g).to(DEV) if base else torch.zeros(q.shape[0], c.heads, cap, device=DEV)
    ref, tol = ok.weights(q, c.k8, c.k_scale, table, lens.cpu(), lse, w0, counts, causal, scale)
    out = w0 if inplace else torch.full_like(w0, 7.0)
    got = c.weights(q, table, lens, lse, base=w0 if base else None, out=out, counts=counts, causal=causal, scale=scale)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    assert got is out
    _close(out, ref, tol, "weights")


@pytest.mark.parametrize("P", [16, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (3, 5), (17, 1), (40, 3), (130, 1), (257, 2)])
def test_weights_ragged(cuda_device, P, T, G):
    c, table, _, n, g = _setup(len(LENS), 2, P, LENS, 11 * T + G)
    q = _q(g, len(LENS), T, 2 * G, 128)
    cap = table.shape[1] * P
    _check_weights(c, q, table, n, cap + 3)
    _check_weights(c, q, table, n, cap, inplace=True)
    _check_weights(c, q, table, n, cap, base=False)


@pytest.mark.parametrize("P,T,G", [(16, 1, 2), (64, 7, 2), (64, 33, 1), (128, 140, 2), (32, 300, 1)])
def test_weights_causal_and_counts(cuda_device, P, T, G):
    lens = [0, 1, 5, 64, 130, 300, 471]
    counts = _i32([T, 1, T, max(1, T // 2), 0, T - T // 3, T])
    c, table, _, n, g = _setup(len(lens), 3, P, lens, T)
    q = _q(g, len(lens), T, 3 * G, 128)
    cap = table.shape[1] * P
    _check_weights(c, q, table, n, cap, causal=True)
    _check_weights(c, q, table, n, cap, counts=counts, causal=True)
    _check_weights(c, q, table, n, cap, counts=counts, scale=0.2)


# ------------------------------------------------------------------ evict
def _check_evict(c, table, free, n, w, heavy, recent, width=None):
    P = c.page
    most = min(heavy + recent, int(n.max()))
    width = max(1, -(-most // P)) if width is None else width
    B = table.shape[0]
    new = free[:B * width].view(B, width).contiguous()
    want = ok.evict(c.k8, c.v8, c.k_scale, c.v_scale, table, n.cpu(), w, new, heavy, recent)
    got = c.evict(table, n, w, new, heavy=heavy, recent=recent, max_len=int(n.max()))
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    assert torch.equal(got[0].cpu(), want[0])
    assert torch.equal(got[1].cpu().nan_to_num(99.0), want[1].nan_to_num(99.0))
    assert torch.equal(got[2].cpu(), want[2])
    for a, b in zip((ok.values(c.k8), ok.values(c.v8), c.k_scale.double(), c.v_scale.double()), want[3:]):
        assert torch.equal(a.nan_to_num(999.0), b.nan_to_num(999.0))


@pytest.mark.parametrize("B,H,P,lens,heavy,recent", [
    (1, 1, 16, [1], 1, 0), (2, 2, 16, [40, 3], 10, 7), (3, 1, 64, [0, 64, 65], 20, 20), (2, 3, 128, [300, 131], 0, 130),
    (2, 2, 32, [500, 77], 64, 0), (1, 2, 16, [100], 90, 90), (1, 1, 64, [5000], 1000, 333),
])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_evict(cuda_device, B, H, P, lens, heavy, recent, kind):
    spare = B * max(1, -(-min(heavy + recent, max(lens)) // P))
    c, table, free, n, g = _setup(B, H, P, lens, heavy, spare=spare, poison=False)
    w = torch.rand(B, H, table.shape[1] * P + 5, generator=g)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "odd":
        w = w - 0.5
        w[:, :, ::7] = 0.0
        w[:, :, 1::7] = -0.0
        w[:, :, 2::11] = math.inf
        w[:, :, 3::13] = -math.inf
        w[:, :, 5::17] = math.nan
    _check_evict(c, table, free, n, w.to(DEV), heavy, recent)


def test_evict_keeps_outliers_out_of_new_scales(cuda_device):
    """An outlier token that is evicted does not set its neighbours' scale."""
    c, table, free, n, g = _setup(1, 1, 16, [0], 5, extra=32, spare=1, poison=False)
    x = torch.randn(1, 32, 1, 128, generator=g)
    x[0, 3] *= 1000.0
    c.write(x.to(DEV), x.to(DEV), table, n)
    n += 32
    w = torch.ones(1, 1, 32, device=DEV)
    w[0, 0, 3] = 0.0
    _check_evict(c, table, free, n, w, 10, 6)
    assert float(c.k_scale[free[0].long(), 0]) < 1.0


# ------------------------------------------------------- used together
def test_rollout_of_all_four(cuda_device):
    """A rollout: chunks and single tokens are written, attended to and
    weighed, and the history is cut, against the same steps in 64 bits on a
    cache that holds the kernels' own codes."""
    B, H, G, P, width = 2, 2, 2, 16, 12
    g = torch.Generator().manual_seed(21)
    table, free, pages = kv8util.tables(B, width, B * 6, g, DEV)
    c = Kv8Cache.empty(pages, H, P, DEV)
    n = _i32([0, 0])
    w = torch.zeros(B, H, width * P, device=DEV)
    for t in (50, 1, 1, 33, 1, 40):
        k, v = (torch.randn(B, t, H, 128, generator=g).to(DEV, torch.bfloat16) for _ in range(2))
        q = _q(g, B, t, H * G, 128)
        _check_write(c, k, v, table, n)
        n += t
        _, lse = _check_attention(c, q, table, n, causal=True)
        ref, tol = ok.weights(q, c.k8, c.k_scale, table, n.cpu(), lse, w, causal=True)
        c.weights(q, table, n, lse, base=w, out=w, causal=True)
        _close(w, ref, tol, "weights")
    total = w.sum((1, 2)).cpu()
    rows = 126 * H * G
    assert ((total - rows).abs() <= 1e-4 * rows).all()   # every row gave away one unit
    new = free.view(B, 6)
    want = ok.evict(c.k8, c.v8, c.k_scale, c.v_scale, table, n.cpu(), w, new, 50, 30)
    kept, w2, n2 = c.evict(table, n, w, new, heavy=50, recent=30)
    assert torch.equal(kept.cpu(), want[0]) and torch.equal(n2.cpu(), want[2])
    q = _q(g, B, 1, H * G, 128)
    _check_attention(c, q, new, n2)


def test_graph_replay_with_other_lengths(cuda_device):
    """One captured step (write, attention, weights) replays as lengths grow;
    a second graph of the same cache has scratch of its own."""
    B, H, P = 2, 2, 16
    c, table, _, n, g = _setup(B, H, P, [3, 100], 31, extra=64, poison=False)
    n2 = n.clone()
    x = torch.empty(B, 1, H, 128, device=DEV, dtype=torch.bfloat16)
    q = torch.empty_like(x)
    w = torch.zeros(B, H, table.shape[1] * P, device=DEV)

    def step(lens):
        c.write(x, x, table, lens)
        lens += 1
        out, lse = c.attention(q, table, lens, return_lse=True)
        c.weights(q, table, lens, lse, base=w, out=w)
        return out

    x.copy_(torch.randn(B, 1, H, 128, generator=g))
    q.copy_(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(n2)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for lens in (n, n2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(lens)
        graphs.append((gr, out, lens))
    n.copy_(_i32([3, 100]))
    for i in range(20):
        x.copy_(torch.randn(B, 1, H, 128, generator=g))
        q.copy_(torch.randn(B, 1, H, 128, generator=g) * 2)
        gr, out, lens = graphs[0]
        gr.replay()
        ref, _, tol, _ = ok.attention(q, c.k8, c.v8, c.k_scale, c.v_scale, table, lens.cpu())
        _close(out, ref, tol, "replay")
    assert n.tolist() == [23, 120]
    n2.copy_(n)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    want = c.attention(q, table, n)
    torch.cuda.synchronize()
    # Attention alone, twice at once: the scratch is each graph's own.
    pair = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = c.attention(q, table, n)
        pair.append((gr, out))
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(a):
            pair[0][0].replay()
        with torch.cuda.stream(b):
            pair[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(pair[0][1], want) and torch.equal(pair[1][1], want)


def test_two_streams_at_once(cuda_device):
    c, table, _, n, g = _setup(2, 4, 64, [3000, 1500], 33, poison=False)
    qs = [_q(g, 2, t, 4, 128) for t in (1, 3, 40, 200)]
    want = [c.attention(q, table, n) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [None] * len(qs)
    for _ in range(5):
        for i, (q, s) in enumerate(zip(qs, streams)):
            with torch.cuda.stream(s):
                got[i] = c.attention(q, table, n)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ------------------------------------------------- reported by the device
def test_bad_pages_and_lengths_are_reported(cuda_device):
    """The kernels check every page id, length and count before they use it."""
    c, table, free, n, g = _setup(2, 2, 16, [40, 20], 41, poison=False)
    q, many = _q(g, 2, 1, 2, 128), _q(g, 2, 40, 2, 128)
    w = torch.zeros(2, 2, table.shape[1] * 16, device=DEV)
    lse = torch.zeros(2, 1, 2, device=DEV)

    def bad(f):
        f()
        torch.cuda.synchronize()
        assert _lib.device_status() == 5

    for value in (c.pages, -1, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 0] = value
        bad(lambda: c.attention(q, t, n))
        bad(lambda: c.attention(many, t, n))
        bad(lambda: c.weights(q, t, n, lse))
        bad(lambda: c.write(q, q, t, n - 20))
        bad(lambda: c.evict(t, n, w, free[:2].view(2, 1).contiguous(), heavy=4, recent=4))
    for value in (-1, 10 ** 9):
        m = n.clone()
        m[0] = value
        bad(lambda: c.attention(q, table, m))
        bad(lambda: c.attention(many, table, m))
        bad(lambda: c.weights(q, table, m, lse))
        bad(lambda: c.write(q, q, table, m))
        bad(lambda: c.attention(q, table, n, counts=_i32([1, value])))
    full = _i32([table.shape[1] * 16, 0])
    bad(lambda: c.write(q, q, table, full))                       # no room behind the table
    bad(lambda: c.evict(table, n, w, table[:, :1].contiguous(), heavy=4, recent=4))   # onto itself
    c.attention(q, table, n)
    assert _lib.device_status() == 0


def test_evict_refuses_a_new_page_named_twice(cuda_device):
    """Two blocks would write it: the sequence keeps nothing, the other one is served."""
    c, table, free, n, g = _setup(2, 2, 16, [200, 150], 47, spare=6, poison=False)
    w = torch.rand(2, 2, table.shape[1] * 16, generator=g).to(DEV)
    new = free[:6].view(2, 3).contiguous()
    new[0, 2] = new[0, 0]
    before = c.k8[new[0].long()].view(torch.uint8).clone()
    kept, weights, lens = c.evict(table, n, w, new, heavy=30, recent=10)
    torch.cuda.synchronize()
    assert _lib.device_status() == 5
    assert lens.tolist() == [0, 40]
    assert (kept[0] == -1).all() and (weights[0] == 0).all()
    assert torch.equal(c.k8[new[0].long()].view(torch.uint8), before)
    for h in range(2):
        assert kept[1, h, :40].tolist() == list(ok.keep(w[1, h].cpu(), 150, 30, 10))
    # A repeat behind the pages that receive rows does no harm.
    new = free[:6].view(2, 3).contiguous()
    new[:, 2] = new[:, 0]
    _, _, lens = c.evict(table, n, w, new, heavy=20, recent=10)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0 and lens.tolist() == [30, 30]


# ------------------------------------------------- refusals of the handle
def test_handle_refuses_gradients_and_expanded_outputs(cuda_device):
    c, table, free, n, g = _setup(2, 2, 16, [40, 20], 43)
    q = _q(g, 2, 3, 4, 128)
    leaf = q.clone().requires_grad_()
    for f in (lambda: c.attention(leaf, table, n), lambda: c.write(q[:, :, :2], leaf[:, :, :2], table, n)):
        with pytest.raises(RuntimeError, match="inference-only"):
            f()
    with pytest.raises(ValueError, match="expanded"):
        c.attention(q, table, n, out=q.new_empty(1, 3, 4, 128).expand(2, 3, 4, 128))
    with torch.no_grad():
        got = c.attention(leaf, table, n)
    assert torch.equal(got, c.attention(q, table, n))


def test_strides_of_single_entries_are_free(cuda_device):
    """One token's stride, or one sequence's, may be any number."""
    c, table, free, n, g = _setup(1, 2, 16, [40], 44)
    q = _q(g, 1, 1, 4, 128)
    odd = torch.as_strided(q, (1, 1, 4, 128), (3, 5, 128, 1))
    out = torch.empty_like(q)
    c.attention(odd, table, n, out=torch.as_strided(out, (1, 1, 4, 128), (7, 1, 128, 1)))
    assert torch.equal(out, c.attention(q, table, n))


# ------------------------------------------- many tiles behind one another
@pytest.mark.parametrize("B,H,G,T,L,causal", [(1, 2, 1, 880, 4400, False), (2, 1, 2, 700, 3000, True), (3, 2, 1, 100, 2500, False)])
def test_weights_many_tiles(cuda_device, B, H, G, T, L, causal):
    """Units of one to eleven query tiles in one CTA's share (the
    exponentials fall behind the loads by several tiles)."""
    c, table, _, n, g = _setup(B, H, 64, [L - 300 * b for b in range(B)], T, poison=False)
    counts = _i32([T - 256 * b if T > 600 else T for b in range(B)])
    _check_weights(c, _q(g, B, T, H * G, 128), table, n, table.shape[1] * 64, counts=counts, causal=causal)


@pytest.mark.parametrize("L,heavy,kind", [(9000, 700, "equal"), (40000, 12345, "random"), (40000, 3, "two"), (12000, 11999, "bin")])
def test_evict_long_heads(cuda_device, L, heavy, kind):
    """More keys than shared memory holds, than its list of one bin, and all keys equal."""
    c, table, free, n, g = _setup(1, 1, 128, [L], heavy, spare=-(-(heavy + 5) // 128), poison=False)
    w = torch.rand(1, 1, table.shape[1] * 128, generator=g)
    if kind == "equal":
        w.fill_(0.75)
    elif kind == "two":
        w = (w > 0.5).float()
    elif kind == "bin":
        w = 1.0 + w * 1e-4
    _check_evict(c, table, free, n, w.to(DEV), heavy, 5)

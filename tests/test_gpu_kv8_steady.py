"""The E4M3 cache kernels with many units of work for each CTA: rings that
wrap, maxima that move inside a share, several items and segments in a CTA,
pairs of key tiles. Every case asserts that it has them, from the device's SM
count, so that another size cannot empty it."""
import threading

import pytest
import torch

from oracle import kv8 as ok
from wam_ops import _lib
from wam_ops.kv8 import Kv8Cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def _make(B, H, P, lens, seed, rise=0.0):
    """Random codes, scales of their own for each block; with `rise` the keys
    are positive and their scales grow along a sequence (general factors)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    width = -(-max(lens) // P)
    pages = B * width + 2
    table = torch.randperm(pages, generator=g, device=DEV)[:B * width].to(torch.int32).view(B, width).contiguous()
    codes = []
    for i in range(2):
        x = torch.randn(pages, H, P, 128, generator=g, device=DEV) * 60
        codes.append((x.abs() if rise and i == 0 else x).to(E4M3))
    ks, vs = (2.0 ** torch.randint(-8, -4, (pages, H), generator=g, device=DEV).float() for _ in range(2))
    if rise:
        at = torch.linspace(0.02, 1.0, width, device=DEV)[None, :, None].expand(B, width, H)
        ks[table.flatten().long()] = (at * rise).reshape(B * width, H)
    return Kv8Cache(codes[0], codes[1], ks, vs), table, torch.tensor(lens, dtype=torch.int32, device=DEV), g


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _units(lens, H, T, rows, tile, causal):
    """128-key units of a call whose query tiles hold `tile` of a head's rows (group 1 where causal)."""
    total = 0
    for n in lens:
        for r in range(0, rows, tile):
            seen = n if not causal else max(0, min(n, n - T + min(rows, r + tile)))
            total += max(1, -(-seen // 128)) * H
    return total


def _close(x, ref, tol, what):
    bad = ~((x.double() - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off"


def _attention(c, q, table, n, causal):
    ref, rlse, tol, ltol = ok.attention(q, c.k8, c.v8, c.k_scale, c.v_scale, table, n.cpu(), causal=causal)
    out, lse = c.attention(q, table, n, causal=causal, return_lse=True)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    _close(lse, rlse, ltol, "lse")
    _close(out, ref, tol, "out")


def _weights(c, q, table, n, causal):
    lse = ok.attention(q, c.k8, c.v8, c.k_scale, c.v_scale, table, n.cpu(), causal=causal)[1].float()
    base = torch.rand(q.shape[0], c.heads, table.shape[1] * c.page, device=DEV)
    ref, tol = ok.weights(q, c.k8, c.k_scale, table, n.cpu(), lse, base, causal=causal)
    got = c.weights(q, table, n, lse, base=base, causal=causal)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    _close(got, ref, tol, "weights")


def _q(g, *shape, rise):
    x = torch.randn(*shape, generator=g, device=DEV)
    return ((x.abs() if rise else x) * 0.5).to(torch.bfloat16)


# Scores grow to about 0.09 x 128 x 48 x 0.4 x rise at the last key: 20, and
# 900 (several times the 2^8 that moves a maximum, in one share of units).
RISES = [0.0, 0.09, 4.0]


@pytest.mark.parametrize("rise", RISES)
@pytest.mark.parametrize("B,H,G,T,P,lens", [
    (8, 8, 4, 1, 64, [24000 - 1300 * b for b in range(8)]),
    (2, 4, 1, 5, 16, [160001, 77]),
    (64, 8, 2, 3, 128, [700 + 61 * b for b in range(64)]),      # several items a share
])
def test_few_rows(cuda_device, B, H, G, T, P, lens, rise):
    c, table, n, g = _make(B, H, P, lens, 61, rise)
    assert _units(lens, H, T, T * G, 16, False) > 8 * 4 * _sms()
    q = _q(g, B, T, H * G, 128, rise=rise)
    _attention(c, q, table, n, False)
    _weights(c, q, table, n, False)


@pytest.mark.parametrize("rise", RISES)
@pytest.mark.parametrize("B,H,T,P,lens,causal", [
    (8, 24, 300, 64, [1100 - 77 * b for b in range(8)], False),  # segments of two halves and of one, in turn
    (8, 24, 300, 16, [1100 - 77 * b for b in range(8)], True),
    (16, 24, 100, 128, [900 - 31 * b for b in range(16)], False),
    (2, 2, 40, 64, [60000, 41003], True),
    (2, 2, 200, 32, [60000, 43007], False),
])
def test_many_rows(cuda_device, B, H, T, P, lens, causal, rise):
    c, table, n, g = _make(B, H, P, lens, 62, rise)
    assert _units(lens, H, T, T, 256, causal) > 9 * _sms()
    _attention(c, _q(g, B, T, H, 128, rise=rise), table, n, causal)


@pytest.mark.parametrize("B,H,T,P,lens,causal", [
    (8, 8, 100, 64, [3500 - 99 * b for b in range(8)], False),
    (8, 8, 300, 16, [3500 - 99 * b for b in range(8)], True),
    (2, 2, 140, 128, [60000, 41003], False),
    (16, 24, 17, 32, [700 - 13 * b for b in range(16)], True),
])
def test_weights_of_many_rows(cuda_device, B, H, T, P, lens, causal):
    """Pairs of key tiles and single ones, whose rings wrap several times."""
    c, table, n, g = _make(B, H, P, lens, 63)
    assert _units(lens, H, T, T, 1 << 30, causal) > 6 * _sms()
    _weights(c, _q(g, B, T, H, 128, rise=0.0), table, n, causal)


def test_calls_from_other_threads(cuda_device):
    """One handle, four threads, a stream each: the results are those of one thread."""
    c, table, n, g = _make(4, 4, 64, [3000, 1500, 77, 1], 64)
    qs = [_q(g, 4, t, 4, 128, rise=0.0) for t in (1, 7, 33, 150)]
    want = [c.attention(q, table, n, return_lse=True) for q in qs]
    want_w = [c.weights(q, table, n, w[1]) for q, w in zip(qs, want)]
    got, got_w = [None] * 4, [None] * 4
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = c.attention(qs[i], table, n, return_lse=True)
                got_w[i] = c.weights(qs[i], table, n, got[i][1])
        torch.cuda.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])
        assert torch.equal(got_w[i], want_w[i])

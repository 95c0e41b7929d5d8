"""Attention and weights over the E4M3 cache for queries whose channels are of
very unequal size, where the cache is zero in the large channel: what counts
are the small ones.

Up to 16 query rows the kernels hold a query in f16 scaled by its row (exact
over 28 binades), above in an E4M3 and an E5M2 value: an element is off by at
most 2^-14 when its row's largest is scaled into (224, 448], and by nothing
when it is then at least 2^-6. fp32 sums of 128 products are off
by at most 130 roundings of their sum of magnitudes (a tensor core may
truncate: 2^-23 each), and a score takes a few more roundings of its own size.
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
SCALE = 0.01
N = 300


def _case(T, seed, factor):
    """One sequence and head; row t: channel 3 is large, the others positive of size 2^-(t % 15) times its 2^-9."""
    g = torch.Generator().manual_seed(seed)
    table, _, pages = kv8util.tables(1, -(-N // 64), 2, g, DEV)
    k8, v8, ks, vs = kv8util.cache(pages, 1, 64, g, "cpu", spread=0.0)
    code = (torch.rand(pages, 1, 64, 128, generator=g) * 300 + 100).to(torch.float8_e4m3fn)
    raw = code.view(torch.uint8)
    raw[..., 3] = 0
    c = Kv8Cache(code.to(DEV), v8.to(DEV), torch.ones_like(ks).to(DEV), vs.to(DEV))
    e = torch.exp2(-(torch.arange(T) % 15).float())
    q = (1 + torch.rand(1, T, 1, 128, generator=g)) * e[None, :, None, None]
    q[..., 3] = 448.0
    return c, table, torch.tensor([N], dtype=torch.int32, device=DEV), (q * factor).to(DEV, torch.bfloat16)


def _scores(c, table, q, scale):
    """[T, N] scores in 64 bits, and the bound of a kernel's error in them."""
    k = ok.sequence(c.k8, c.k_scale, table[0], N)[0]
    x = q[0, :, 0].double()
    s, mag = x @ k.T * scale, x.abs() @ k.abs().T * scale
    err = mag * (130 * 2.0 ** -23) + s.abs() * 2.0 ** -21
    if x.shape[0] > 16:
        top = x.abs().amax(1, keepdim=True)
        n = torch.ceil(torch.log2(top / 448.0))          # the row's largest is in (224, 448] times 2^n
        lost = (x.abs() < torch.exp2(n - 6)).double()
        err = err + torch.exp2(n - 14) * (lost @ k.abs().T) * scale
    return s, err


@pytest.mark.parametrize("T", [1, 15, 16, 17, 60, 128, 200])
@pytest.mark.parametrize("factor", [1.0, 2.0 ** -20])
def test_small_channels_beside_a_large_one(cuda_device, T, factor):
    c, table, n, q = _case(T, T, factor)
    scale = SCALE / factor
    s, err = _scores(c, table, q, scale)
    z = torch.logsumexp(s, 1)
    out, lse = c.attention(q, table, n, scale=scale, return_lse=True)
    e = err.amax(1)
    assert ((lse[0, :, 0].double() - z).abs() <= e + 2.0 ** -20 + z.abs() * 2.0 ** -22).all()
    v = ok.sequence(c.v8, c.v_scale, table[0], N)[0]
    p = torch.exp(s - z[:, None])
    # P in f16 and its steps below f16's range, as in the oracle's attention.
    top = 2 * p.amax(1, keepdim=True) * v.abs().amax()
    tol = (2.0 ** -11 + 2.0 ** -20 + 2 * e[:, None]) * (p @ v.abs()) + N * 2.0 ** -30 * top + 2.0 ** -8 * (p @ v).abs()
    assert ((out[0, :, 0].double() - p @ v).abs() <= tol).all()
    w = c.weights(q, table, n, z.float().view(1, T, 1).contiguous(), scale=scale)
    z32 = z.float().double()[:, None]
    want = torch.exp(s - z32)
    rel = err + z32.abs() * 2.0 ** -22 + 2.0 ** -20 + T * 2.0 ** -24
    assert ((w[0, 0, :N].double() - want.sum(0)).abs() <= (want * rel).sum(0) + want.sum(0) * 2.0 ** -23 + 1e-30).all()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def test_sixteen_rows_and_seventeen_agree(cuda_device):
    """The two kernels' results for the same rows differ by their bounds only."""
    c, table, n, q = _case(17, 5, 1.0)
    few = c.attention(q[:, :16].contiguous(), table, n, scale=SCALE, return_lse=True)[1]
    many = c.attention(q, table, n, scale=SCALE, return_lse=True)[1]
    _, err = _scores(c, table, q, SCALE)
    z = few[0, :, 0].double()
    assert ((many[0, :16, 0].double() - z).abs() <= 2 * (err.amax(1)[:16] + 2.0 ** -20 + z.abs() * 2.0 ** -22)).all()
    assert math.isfinite(float(many.sum()))

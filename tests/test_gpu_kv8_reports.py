"""What the E4M3 cache operators do with sequences whose lengths, counts or
pages are out of range: the error word says so, and nothing that the caller
holds is lost."""
import pytest
import torch

import kv8util
from wam_ops import _lib
from wam_ops.kv8 import Kv8Cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _setup(B, H, P, width, seed, spare=4):
    g = torch.Generator().manual_seed(seed)
    table, free, pages = kv8util.tables(B, width, spare, g, DEV)
    return Kv8Cache(*kv8util.cache(pages, H, P, g, DEV)), table, free, g


def _state(c):
    return [t.view(torch.uint8).clone() for t in (c.k8, c.v8, c.k_scale, c.v_scale)]


def _reported():
    torch.cuda.synchronize()
    return _lib.device_status() == 5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,counts", [([-1, 20], None), ([-2 ** 31, 20], None), ([49, 20], None), ([2 ** 31 - 1, 20], None),
                                         ([40, 20], [4, 5]), ([40, 20], [-1, 5]), ([46, 20], None), ([48, 20], [1, 5])])
def test_write_leaves_a_reported_sequence_as_it_was(cuda_device, lens, counts, dtype):
    """A length or count out of range, or rows that do not fit the table: the
    sequence's pages keep their codes and scales; the other sequence is written."""
    T = 3
    c, table, free, g = _setup(2, 2, 16, 3, 51)
    x = (50 * torch.randn(2, T, 2, 128, generator=g)).to(DEV, dtype)     # large: scales would grow
    before = _state(c)
    bad = counts is not None and not 0 <= counts[1] <= T
    c.write(x, 2 * x, table, _i32(lens), None if counts is None else _i32(counts))
    assert _reported()
    after = _state(c)
    touched = table[0].long() if not bad else table.flatten().long()
    for a, b in zip(before, after):
        assert torch.equal(a[touched], b[touched])
    if not bad:
        ids = table[1].long()
        assert not torch.equal(before[0][ids], after[0][ids])


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("lens,counts", [([-1, 20], None), ([10 ** 9, 20], None), ([40, 20], [-3, 1]), ([40, 20], [99, 1])])
def test_running_weights_of_a_reported_sequence_stay(cuda_device, T, lens, counts):
    """weights(base=w, out=w) adds nothing for a sequence whose length or count is out of range."""
    c, table, free, g = _setup(2, 2, 16, 3, 52)
    q = torch.randn(2, T, 2, 128, generator=g).to(DEV, torch.bfloat16)
    lse = torch.zeros(2, T, 2, device=DEV)
    w = torch.rand(2, 2, 48, generator=g).to(DEV)
    before = w.clone()
    c.weights(q, table, _i32(lens), lse, base=w, out=w, counts=None if counts is None else _i32(counts))
    assert _reported()
    assert torch.equal(w[0], before[0])
    assert not torch.equal(w[1], before[1])


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("lens,counts", [([-1, 20], None), ([10 ** 9, 20], None), ([40, 20], [99, 1])])
def test_attention_of_a_reported_sequence_sees_nothing(cuda_device, T, lens, counts):
    """Rows of a sequence whose length is out of range are answered like those
    of an empty one (0 and -inf); a count out of range leaves them as they were."""
    c, table, free, g = _setup(2, 2, 16, 3, 53)
    q = torch.randn(2, T, 2, 128, generator=g).to(DEV, torch.bfloat16)
    out = torch.full_like(q, 7.0)
    lse = torch.full((2, T, 2), 7.0, device=DEV)
    c.attention(q, table, _i32(lens), None if counts is None else _i32(counts), out=out, lse=lse)
    assert _reported()
    if counts is None:
        assert (out[0] == 0).all() and (lse[0] == -float("inf")).all()
    else:
        assert (out[0] == 7.0).all() and (lse[0] == 7.0).all()
    assert (lse[1, 0] != 7.0).all()


@pytest.mark.parametrize("T", [17, 40, 150])
def test_tensor_core_weights_report_bad_pages_and_lengths(cuda_device, T):
    c, table, free, g = _setup(2, 2, 16, 12, 54)
    n = _i32([190, 77])
    q = torch.randn(2, T, 2, 128, generator=g).to(DEV, torch.bfloat16)
    lse = torch.zeros(2, T, 2, device=DEV)
    for value in (c.pages, -1, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 2] = value
        c.weights(q, t, n, lse)
        assert _reported()
    for value in (-1, 193, 10 ** 9):
        m = n.clone()
        m[0] = value
        c.weights(q, table, m, lse)
        assert _reported()
        c.weights(q, table, n, lse, counts=_i32([1, value if value != 193 else T + 1]))
        assert _reported()
    c.weights(q, table, n, lse)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def test_evict_of_a_length_out_of_range_keeps_nothing(cuda_device):
    c, table, free, g = _setup(2, 2, 16, 6, 56, spare=4)
    w = torch.rand(2, 2, 96, generator=g).to(DEV)
    for value in (-1, 97, 2 ** 31 - 1):
        kept, nw, lens = c.evict(table, _i32([value, 50]), w, free.view(2, 2), heavy=20, recent=10)
        assert _reported()
        assert lens.tolist() == [0, 30] and (kept[0] == -1).all() and (nw[0] == 0).all()

"""Evictions that new pages cannot hold."""
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


def _reported():
    torch.cuda.synchronize()
    return _lib.device_status() == 5


def test_evict_reports_a_length_beyond_max_len(cuda_device):
    """max_len let the host accept two new pages; one sequence has grown past
    it since. It would lose its tail: it keeps nothing and is reported, the
    other one is served."""
    c, table, free, g = _setup(2, 2, 16, 6, 55, spare=4)
    new = free.view(2, 2)
    w = torch.rand(2, 2, 96, generator=g).to(DEV)
    for heavy, recent in ((60, 20), (0, 90), (90, 0)):
        before = c.k8.view(torch.uint8)[new[0].long()].clone()
        kept, nw, lens = c.evict(table, _i32([33, 30]), w, new, heavy=heavy, recent=recent, max_len=32)
        assert _reported()
        assert lens.tolist() == [0, 30]
        assert (kept[0] == -1).all() and (nw[0] == 0).all()
        assert torch.equal(c.k8.view(torch.uint8)[new[0].long()], before)
        for h in range(2):
            assert kept[1, h, :30].tolist() == list(range(30))
        kept, nw, lens = c.evict(table, _i32([32, 30]), w, new, heavy=heavy, recent=recent, max_len=32)
        torch.cuda.synchronize()
        assert _lib.device_status() == 0 and lens.tolist() == [32, 30]

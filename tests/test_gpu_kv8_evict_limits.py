"""Evictions that new pages cannot hold, and page ids that are alike."""
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


def test_evict_tells_colliding_page_ids_apart(cuda_device):
    """Page ids that are equal modulo the overlap filter's 262144 bits are
    different pages; ids that are equal are found among them."""
    P, n, far = 16, 100, 262144
    pages = 2 * far + 64
    c = Kv8Cache.empty(pages, 1, P, DEV)                  # 1.1 GB for K and for V
    g = torch.Generator().manual_seed(57)
    table = _i32([[3, far + 4, 2 * far + 5, 6, far + 7, 8, 9]])
    k = torch.randn(1, n, 1, 128, generator=g).to(DEV, torch.bfloat16)
    c.write(k, k, table, _i32([0]))
    w = torch.rand(1, 1, 7 * P, generator=g).to(DEV)
    fresh = [far + 3, 4, 5, 2 * far + 6]                  # each collides with an old page
    for new, good in ((fresh, True), ([10, far + 10, 2 * far + 10, 11], True), ([10, 2 * far + 11, far + 12, far + 12], False),
                      ([far + 3, 4, far + 7, 11], False), ([10, 11, 12, 2 * far + 5], False)):
        kept, _, lens = c.evict(table, _i32([n]), w, _i32([new]), heavy=40, recent=20)
        torch.cuda.synchronize()
        assert _lib.device_status() == (0 if good else 5)
        assert lens.tolist() == [60 if good else 0]
        if good:
            assert kept[0, 0, :60].tolist() == list(ok.keep(w[0, 0].cpu(), n, 40, 20))


def test_evict_time_does_not_depend_on_where_the_pages_lie(cuda_device):
    """Ids that collide in the overlap filter cost passes over the tables, not
    a comparison of all pairs: 4096 new pages against 16384 old ones are 67
    million (seven times the time). Twice the time of distinct ids is allowed."""
    P, far, old, fresh = 16, 262144, 16384, 4096
    c = Kv8Cache.empty(2 * far + 16, 1, P, DEV)
    w = torch.rand(1, 1, old * P, device=DEV)
    n = _i32([old * P])
    table = torch.arange(old, dtype=torch.int32, device=DEV)[None].contiguous()

    def ms(new):
        new = new.to(torch.int32)[None].contiguous()
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            _, _, lens = c.evict(table, n, w, new, heavy=fresh * P - 100, recent=100)
            b.record()
            torch.cuda.synchronize()
            assert lens.tolist() == [fresh * P]
            times.append(a.elapsed_time(b))
        return min(times[1:])

    distinct = ms(torch.arange(old, old + fresh, device=DEV))
    collide = ms(torch.arange(far, far + fresh, device=DEV))
    print(f"evict with distinct ids {distinct:.3f} ms, colliding {collide:.3f} ms")
    assert _lib.device_status() == 0
    assert collide <= 2 * distinct


def test_evict_onto_a_page_that_is_none_keeps_nothing(cuda_device):
    """Rows for it would be lost although `kept` lists them."""
    c, table, free, g = _setup(2, 2, 16, 6, 58, spare=4)
    w = torch.rand(2, 2, 96, generator=g).to(DEV)
    for value in (c.pages, -1, 2 ** 31 - 1, -2 ** 31):
        for at in (0, 1):
            new = free.view(2, 2).clone()
            new[0, at] = value
            before = c.k8.view(torch.uint8)[free.long()].clone()
            kept, nw, lens = c.evict(table, _i32([90, 50]), w, new, heavy=20, recent=10)
            assert _reported()
            assert lens.tolist() == [0, 30] and (kept[0] == -1).all() and (nw[0] == 0).all()
            assert torch.equal(c.k8.view(torch.uint8)[free[:2].long()], before[:2])
            new[1, 1] = value
            new[0] = free[:2]
            kept, nw, lens = c.evict(table, _i32([90, 50]), w, new, heavy=10, recent=5)
            torch.cuda.synchronize()
            assert _lib.device_status() == 0 and lens.tolist() == [15, 15]      # a page that receives nothing may be any

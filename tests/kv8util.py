"""Seeded E4M3 caches and ragged page tables for the kv8 tests."""
import torch

from oracle import kv8 as ok

E4M3 = torch.float8_e4m3fn


def tables(B, width, spare, gen, device="cpu"):
    """(table [B, width], free page ids, page count): distinct shuffled pages."""
    pages = B * width + spare
    ids = torch.randperm(pages, generator=gen).to(torch.int32)
    return ids[:B * width].view(B, width).contiguous().to(device), ids[B * width:].to(device), pages


def cache(pages, H, P, gen, device, spread=0.7, nan_tail=None):
    """Random codes whose blocks have unequal power-of-two scales."""
    out = []
    for _ in range(2):
        x = torch.randn(pages, H, P, 128, generator=gen) * torch.exp(spread * torch.randn(pages, H, 1, 1, generator=gen))
        s = torch.tensor([[ok.block_scale(x[p, h].abs().max()) for h in range(H)] for p in range(pages)])
        out += [(x / s[:, :, None, None]).clamp(-448, 448).to(E4M3).to(device), s.to(device)]
    k8, ks, v8, vs = out
    return k8, v8, ks, vs


def poison(codes, scale, table, lens):
    """NaN codes in every row that no sequence holds (tails of last pages, free pages)."""
    P = codes.shape[2]
    live = torch.zeros(codes.shape[0], P, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            live[int(table[b, p // P]), p % P] = True
    raw = codes.view(torch.uint8)
    raw[~live[:, None, :, None].expand(raw.shape).to(raw.device)] = 0x7f
    used = live.any(1)
    scale[~used.to(scale.device)] = float("nan")

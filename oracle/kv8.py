"""The E4M3 KV cache operators from their definitions, in 64 bits.

Loops over sequences, heads and pages; cache tensors are torch tensors
(float8_e4m3fn codes, fp32 scales) on any device. attention and weights also
return how far a kernel that rounds where the documentation says may be off.
"""
import math

import torch

D = 128
E4M3 = torch.float8_e4m3fn


def _code_values(device):
    """The 256 values of E4M3 by code, in 64 bits."""
    return torch.arange(256, dtype=torch.uint8).view(E4M3).to(torch.float64).to(device)


def values(codes):
    return _code_values(codes.device)[codes.view(torch.uint8).long()]


def round_e4m3(x):
    """Nearest E4M3 value (ties to the even code), saturating; NaN stays."""
    grid = torch.arange(127, dtype=torch.uint8).view(E4M3).to(torch.float64).to(x.device)   # 0 .. 448
    a = x.abs().clamp(max=448.0).nan_to_num(0.0)
    hi = torch.searchsorted(grid, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - grid[lo], grid[hi] - a
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.where(x.isnan(), x, torch.copysign(grid[pick], x))


def block_scale(amax):
    """2^n, n the smallest whole number in [-40, 119] with amax <= 448 * 2^n."""
    n = -40
    amax = min(float(amax), torch.finfo(torch.float32).max)
    while n < 119 and amax > 448.0 * 2.0 ** n:
        n += 1
    return 2.0 ** n


def _amax(x):
    x = x.abs()
    x = x[~x.isnan()]
    return float(x.max()) if x.numel() else 0.0


def write(k8, v8, k_scale, v_scale, k, v, table, lens, counts=None):
    """The cache after the write, as (k codes, v codes) values in 64 bits and scales."""
    out = []
    P = k8.shape[2]
    for codes, scale, x in ((k8, k_scale, k), (v8, v_scale, v)):
        c, s = values(codes), scale.double().clone()
        for b in range(x.shape[0]):
            n, t = int(lens[b]), x.shape[1] if counts is None else int(counts[b])
            for page in range(n // P, (n + t - 1) // P + 1 if t else 0):
                lo, hi = max(n, page * P), min(n + t, page * P + P)
                pid, held = int(table[b, page]), lo - page * P
                for h in range(x.shape[2]):
                    rows = x[b, lo - n:hi - n, h].double()
                    new = block_scale(_amax(rows))
                    if held:
                        old = float(s[pid, h])
                        if new > old:
                            c[pid, h, :held] = round_e4m3(c[pid, h, :held] * (old / new))
                        new = max(new, old)
                    c[pid, h, held:held + hi - lo] = round_e4m3(rows / new)
                    s[pid, h] = new
        out += [c, s]
    return out[0], out[2], out[1], out[3]


def sequence(codes, scale, table, n):
    """[H, n, D] values of the first n positions of one sequence."""
    P = codes.shape[2]
    ids = table[:-(-n // P)].long() if n else table[:0].long()
    x = values(codes[ids].contiguous().view(torch.uint8)) * scale[ids].double()[:, :, None, None] if n else \
        torch.zeros(0, codes.shape[1], P, D, dtype=torch.float64, device=codes.device)
    return x.transpose(0, 1).reshape(codes.shape[1], -1, D)[:, :n]


def _rows(q, k, n, t, causal, scale):
    """Scores [t, n] (-inf where hidden) of one head and the bound of their error.

    The products are summed in fp32 (128 terms: at most 130 roundings of the
    sum of magnitudes, a tensor core may truncate: 2^-23 each); a query may be
    held in an E4M3 and an E5M2 piece, off by at most 2^-14 when its row's
    largest magnitude is at least 224; the score meets its factors, the log-sum-exp
    or the maximum in a few more fp32 roundings of numbers of its own size.
    """
    s = q @ k.T * scale
    mag = q.abs() @ k.abs().T * scale
    piece = q.abs().amax(1, keepdim=True) / 224.0 * 2.0 ** -14 * (k.abs().sum(1)[None] * scale)
    err = mag * (130 * 2.0 ** -23) + piece + s.abs() * 2.0 ** -21
    if causal:
        hidden = torch.arange(n, device=q.device)[None] > n - t + torch.arange(t, device=q.device)[:, None]
        s = s.masked_fill(hidden, -math.inf)
        err = err.masked_fill(hidden, 0.0)
    return s, err


def attention(q, k8, v8, k_scale, v_scale, table, lens, counts=None, causal=False, scale=None):
    """(out, lse, bound of |out - bf16 result|, bound of |lse - result|), NaN past counts."""
    B, T, Hq, _ = q.shape
    H = k8.shape[1]
    scale = D ** -0.5 if scale is None else scale
    dev = q.device
    out = torch.full((B, T, Hq, D), math.nan, dtype=torch.float64, device=dev)
    lse = torch.full((B, T, Hq), math.nan, dtype=torch.float64, device=dev)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        n, t = int(lens[b]), T if counts is None else int(counts[b])
        if t == 0:
            continue
        k, v = sequence(k8, k_scale, table[b], n), sequence(v8, v_scale, table[b], n)
        for h in range(Hq):
            kk, vv = k[h // (Hq // H)], v[h // (Hq // H)]
            s, err = _rows(q[b, :t, h].double(), kk, n, t, causal, scale)
            z = torch.logsumexp(s, 1) if n else torch.full((t,), -math.inf, dtype=torch.float64, device=dev)
            p = torch.exp(s - z[:, None]).masked_fill(s == -math.inf, 0.0)
            out[b, :t, h] = p @ vv
            lse[b, :t, h] = z
            # P is held in f16 (2^-11 of itself) after an exponential that is
            # off by 2^-21; below f16's normal range its steps are at most 2^-30
            # of the largest p vs, against codes of at most 448 (448 vs is less
            # than twice the block's largest value); the result is rounded to bf16.
            e = err.amax(1, keepdim=True) if n else torch.zeros(t, 1, dtype=torch.float64, device=dev)
            top = 2 * p.amax(1, keepdim=True) * vv.abs().amax() if n else 0.0
            tol[b, :t, h] = (2.0 ** -11 + 2.0 ** -20 + 2 * e) * (p @ vv.abs()) + n * 2.0 ** -30 * top + \
                2.0 ** -8 * out[b, :t, h].abs() + 1e-37
            ltol[b, :t, h] = e[:, 0] + 2.0 ** -20 + z.abs().nan_to_num(0.0, 0.0, 0.0) * 2.0 ** -22
    return out, lse, tol, ltol


def weights(q, k8, k_scale, table, lens, lse, base, counts=None, causal=False, scale=None):
    """(weights, bound of their error)."""
    B, T, Hq, _ = q.shape
    H = k8.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = base.double().clone()
    tol = out.abs() * 2.0 ** -23 + 1e-37
    for b in range(B):
        n, t = int(lens[b]), T if counts is None else int(counts[b])
        if n == 0 or t == 0:
            continue
        k = sequence(k8, k_scale, table[b], n)
        for h in range(Hq):
            s, err = _rows(q[b, :t, h].double(), k[h // (Hq // H)], n, t, causal, scale)
            z = lse[b, :t, h].double()[:, None]
            w = torch.exp(s - z).masked_fill(s == -math.inf, 0.0)
            # fp32 sums over the rows: at most t * group roundings.
            rel = err + z.abs().nan_to_num(0.0, 0.0, 0.0) * 2.0 ** -22 + 2.0 ** -20 + t * (Hq // H) * 2.0 ** -24
            out[b, h // (Hq // H), :n] += w.sum(0)
            tol[b, h // (Hq // H), :n] += (w * rel).sum(0) + w.sum(0) * 2.0 ** -23
    return out, tol


def keep(w, n, heavy, recent):
    """Kept positions of one (sequence, head), ascending, by a plain sort."""
    old = max(0, n - recent)
    rank = sorted(range(old), key=lambda i: (0 if math.isnan(w[i]) else 1, -w[i] if not math.isnan(w[i]) else 0.0, i))
    return sorted(rank[:heavy]) + list(range(old, n))


def evict(k8, v8, k_scale, v_scale, table, lens, w, new_table, heavy, recent):
    """(kept, new weights, new lens, k values, v values, k scales, v scales)."""
    B, H = table.shape[0], k8.shape[1]
    P = k8.shape[2]
    width = new_table.shape[1] * P
    kept = torch.full((B, H, width), -1, dtype=torch.int32)
    new_w = torch.zeros(B, H, width)
    new_lens = torch.zeros(B, dtype=torch.int32)
    wc = w.cpu()
    res = []
    for codes, scale in ((k8, k_scale), (v8, v_scale)):
        c, s = values(codes), scale.double().clone()
        old_c, old_s = c.clone(), s.clone()
        for b in range(B):
            n = int(lens[b])
            for h in range(H):
                pos = keep(wc[b, h].tolist(), n, heavy, recent)
                kept[b, h, :len(pos)] = torch.tensor(pos, dtype=torch.int32)
                new_w[b, h, :len(pos)] = wc[b, h, pos]
                new_lens[b] = len(pos)
                for a in range(-(-len(pos) // P)):
                    at = torch.tensor(pos[a * P:(a + 1) * P])
                    ids = table[b].cpu()[at // P].long()
                    x = old_c[ids, h, at % P] * old_s[ids, h][:, None]
                    pid = int(new_table[b, a])
                    new = block_scale(_amax(x))
                    c[pid, h, :len(at)] = round_e4m3(x / new)
                    s[pid, h] = new
        res += [c, s]
    return kept, new_w, new_lens, res[0], res[2], res[1], res[3]

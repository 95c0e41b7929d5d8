"""Cases of the 8-bit KV cache operators: write, attention, attention weights, eviction.

The cache is paged: `k8`, `v8` are [pages, heads, page, 128] E4M3 with one
power-of-two fp32 scale per (page, head); position p of sequence b is row
p % page of page table[b, p // page]. `run` computes each operator in plain
torch operations in 32 bits, or, with `own` set, through
wam_ops.kv8.Kv8Cache.
"""
import math
import sys
from pathlib import Path

import torch

own = False

D = 128
SCALE_MIN, SCALE_MAX = -40, 119     # exponents of a block scale
E4M3 = torch.float8_e4m3fn


def listed():
    def case(name, op, batch, heads, ctx, rows=0, group=1, page=64, causal=False, dtype="bf16", heavy=0, recent=0):
        return dict(name=name, op=op, batch=batch, heads=heads, ctx=ctx, rows=rows, group=group, page=page,
                    causal=causal, dtype=dtype, heavy=heavy, recent=recent)
    return [
        # one new token of each of 8 rollouts: a launch-bound append into half-filled pages
        case("write_token", "write", 8, 24, 1530, rows=1),
        # a whole 880-token chunk of 8 rollouts behind 3520 tokens of history
        case("write_chunk", "write", 8, 24, 3520, rows=880),
        # fp32 K/V of an odd chunk into small pages, starting inside a page
        case("write_odd_fp32", "write", 3, 12, 777, rows=333, page=16, dtype="fp32"),
        # one query token over a short ragged history: latency
        case("attn_token_short", "attention", 2, 12, 509, rows=1),
        # one token of 8 sequences with long ragged histories, 4 query heads on each cached head
        case("attn_token_long", "attention", 8, 8, 32768, rows=1, group=4),
        # candidate verification: 32 action tokens against 3520 tokens of history, causal, odd lengths
        case("attn_verify", "attention", 4, 24, 3551, rows=32, causal=True),
        # an 880-token chunk of 8 rollouts over history and itself
        case("attn_chunk", "attention", 8, 24, 4400, rows=880),
        # weights of one decoded token over long histories
        case("weights_token", "weights", 8, 8, 32768, rows=1, group=4),
        # weights of one 880-token chunk of one rollout
        case("weights_chunk", "weights", 1, 24, 4400, rows=880),
        # a rollout's history cut to half: 1760 heavy tokens and the last chunk
        case("evict_chunk", "evict", 1, 24, 4400, heavy=1760, recent=880),
        # long histories of 8 sequences cut to a quarter, odd counts
        case("evict_long", "evict", 8, 8, 32768, heavy=6001, recent=2047),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "attention", "attention", "weights", "evict"])
    c = dict(op=op, batch=_spread(rng, 1, 8), heads=rng.choice([1, 2, 5, 8, 12, 24]), ctx=1, rows=0, group=1,
             page=rng.choice([16, 32, 64, 128]), causal=rng.random() < 0.5, dtype="bf16", heavy=0, recent=0)
    if op == "write":
        c["rows"] = _spread(rng, 1, 900)
        c["ctx"] = _spread(rng, 1, 4000)
        c["causal"], c["dtype"] = False, rng.choice(["bf16", "fp32"])
    elif op in ("attention", "weights"):
        few = rng.random() < 0.5
        c["group"] = rng.choice([1, 2, 3, 4, 8]) if few else rng.choice([1, 1, 2])
        c["rows"] = rng.choice([1, 1, 2, 3]) if few else _spread(rng, 20, 900)
        c["ctx"] = max(_spread(rng, 1, 32768 if few else 4400), c["rows"])
        if c["heads"] * c["batch"] * c["ctx"] > 8 * 8 * 32768:
            c["heads"] = 8
        if c["rows"] * c["group"] * c["heads"] * c["batch"] * c["ctx"] > 8 * 24 * 880 * 4400:
            c["group"] = 1
    else:
        c["ctx"] = _spread(rng, 1, 32768)
        c["heads"] = min(c["heads"], 8) if c["ctx"] > 4400 else c["heads"]
        keep = rng.randint(1, max(1, c["ctx"]))
        c["recent"] = rng.randint(0, keep)
        c["heavy"] = keep - c["recent"]
        c["causal"] = False
    return c


def _lens(c):
    """Ragged lengths: the first sequence is the longest, the last about half of it (at least the query rows)."""
    return [max(1, c["rows"] if c["op"] != "write" else 0, c["ctx"] - c["ctx"] * b // (2 * c["batch"]))
            for b in range(c["batch"])]


def _block_scale(amax):
    """The smallest power of two s in [2^-40, 2^119] with amax <= 448 s."""
    m, e = torch.frexp(amax.clamp(max=torch.finfo(torch.float32).max))
    n = torch.where(m <= 0.875, e - 9, e - 8)
    n = torch.where(amax > 0, n, torch.full_like(n, SCALE_MIN)).clamp(SCALE_MIN, SCALE_MAX)
    return ((n.to(torch.int32) + 127) << 23).view(torch.float32)


def _e4m3(x):
    return x.clamp(-448.0, 448.0).to(E4M3).view(torch.uint8)


def _float(codes):
    return codes.view(E4M3).to(torch.float32)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = _lens(c)
    P, B, H = c["page"], c["batch"], c["heads"]
    new = c["rows"] if c["op"] == "write" else 0
    width = -(-(max(lens) + new) // P)
    keep = min(c["heavy"] + c["recent"], max(lens))
    width2 = -(-keep // P) if c["op"] == "evict" else 0
    pages = B * (width + width2) + 3                     # a few pages belong to nobody
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = order[:B * width].view(B, width).contiguous()
    gain = torch.exp(0.3 * torch.randn(H, 1, D, generator=g, device="cuda"))   # channels of unequal size

    def cached():
        # tokens of unequal magnitude: blocks get different scales
        x = torch.randn(pages, H, P, D, generator=g, device="cuda")
        x *= gain * torch.exp(0.5 * torch.randn(pages, H, P, 1, generator=g, device="cuda"))
        s = _block_scale(x.abs().amax((2, 3)))
        return _e4m3(x / s[:, :, None, None]).view(E4M3), s

    k8, k_scale = cached()
    v8, v_scale = cached()
    st = dict(case=c, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              k8=k8, v8=v8, k_scale=k_scale, v_scale=v_scale)
    if c["op"] == "write":
        dt = torch.float32 if c["dtype"] == "fp32" else torch.bfloat16
        for n in ("k", "v"):
            x = torch.randn(B, c["rows"], H, D, generator=g, device="cuda") * gain.view(H, D)
            st[n] = (x * torch.exp(0.5 * torch.randn(B, c["rows"], H, 1, generator=g, device="cuda"))).to(dt)
    elif c["op"] in ("attention", "weights"):
        q = torch.randn(B, c["rows"], H * c["group"], D, generator=g, device="cuda")
        st["q"] = q.to(torch.bfloat16)
        if c["op"] == "weights":
            st["lse"] = _attention(st, False)[1]
            st["base"] = torch.rand(B, H, width * P, generator=g, device="cuda") * 2
    else:
        w = torch.rand(B, H, width * P, generator=g, device="cuda").pow(4) * 8
        w = torch.where(torch.rand(B, H, width * P, generator=g, device="cuda") < 0.2,
                        w.to(torch.bfloat16).to(torch.float32), w)       # some equal weights
        st["weights"] = w
        st["new_table"] = order[B * width:B * (width + width2)].view(B, width2).contiguous()
    return st


# ------------------------------------------------------------- plain forms
def _write_one(codes, scale, x, table, lens):
    """New rows x [B, T, H, D] at positions lens[b] + t of one of K / V, in place."""
    B, T, H, _ = x.shape
    P = codes.shape[2]
    n = (T + P - 2) // P + 1                                       # pages a sequence can touch
    j = (lens // P).long()[:, None] + torch.arange(n, device=x.device)               # [B, n]
    t = j[:, :, None] * P + torch.arange(P, device=x.device) - lens[:, None, None]   # [B, n, P]
    is_new, is_old = (t >= 0) & (t < T), t < 0
    touched = is_new.any(2)
    pid = table.long().gather(1, j.clamp(max=table.shape[1] - 1))
    rows = torch.arange(B, device=x.device)[:, None, None]
    vals = x[rows, t.clamp(0, T - 1)].to(torch.float32).permute(0, 1, 3, 2, 4)       # [B, n, H, P, D]
    new = is_new[:, :, None, :, None]
    s = _block_scale(torch.where(new, vals.abs(), torch.zeros_like(vals)).amax((3, 4)))
    s_old = scale[pid]
    s = torch.where(is_old.any(2)[:, :, None], torch.maximum(s, s_old), s)
    old = codes.view(torch.uint8)[pid]
    moved = _e4m3(_float(old) * (s_old / s)[..., None, None])
    out = torch.where(new, _e4m3(vals / s[..., None, None]), torch.where(is_old[:, :, None, :, None], moved, old))
    codes.view(torch.uint8)[pid[touched]] = out[touched]
    scale[pid[touched]] = s[touched]


def _keys(codes, scale, table):
    """[B, H, width * page, D] fp32 values of the cached rows."""
    t = table.long()
    x = _float(codes.view(torch.uint8)[t]) * scale[t][..., None, None]               # [B, W, H, P, D]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _scores(st):
    """Scaled scores [B, H, T * G, L] fp32, -inf where a key is not visible."""
    c, q = st["case"], st["q"]
    B, T, _, _ = q.shape
    H, G = c["heads"], c["group"]
    rows = q.to(torch.float32).view(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    s = rows @ _keys(st["k8"], st["k_scale"], st["table"]).transpose(2, 3)
    s *= D ** -0.5
    j = torch.arange(s.shape[3], device=q.device)
    last = st["lens"].long()[:, None].expand(B, T) - 1                                # last visible key of a row
    if c["causal"]:
        last = last - (T - 1) + torch.arange(T, device=q.device)
    hidden = (j > last[:, :, None]).repeat_interleave(G, 1)                          # [B, T * G, L]
    return s.masked_fill_(hidden[:, None], -math.inf)


def _rows_out(x, st):
    B, T, Hq, _ = st["q"].shape
    H = st["case"]["heads"]
    return x.view(B, H, T, Hq // H, -1).permute(0, 2, 1, 3, 4).reshape(B, T, Hq, -1)


def _attention(st, values=True):
    p = _scores(st)
    m = p.amax(3, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = p.sub_(m).exp_()
    total = p.sum(3, keepdim=True)
    lse = _rows_out((m + total.log()).view(*p.shape[:3], 1), st).squeeze(3).contiguous()
    if not values:
        return None, lse
    live = (torch.arange(p.shape[3], device=p.device) < st["lens"][:, None])[:, None, :, None]
    v = _keys(st["v8"], st["v_scale"], st["table"]).masked_fill(~live, 0.0)
    o = (p @ v) / total.clamp(min=torch.finfo(torch.float32).tiny)
    return _rows_out(o, st).to(torch.bfloat16).contiguous(), lse


def _weights(st):
    c, q = st["case"], st["q"]
    B, T, Hq, _ = q.shape
    lse = st["lse"].view(B, T, c["heads"], c["group"]).permute(0, 2, 1, 3).reshape(B, c["heads"], T * c["group"], 1)
    p = _scores(st).sub_(lse).exp_()
    return st["base"] + p.sum(2)


def _evict(st):
    c, lens, w = st["case"], st["lens"].long(), st["weights"]
    B, H, L = w.shape
    dev, P = w.device, c["page"]
    keep = c["heavy"] + c["recent"]
    kept = (lens).clamp(max=keep)                                                     # [B]
    j = torch.arange(L, device=dev)
    rank = w.masked_fill((j >= (lens - c["recent"])[:, None])[:, None], math.inf)
    rank = rank.masked_fill((j >= lens[:, None])[:, None], -math.inf)
    order = rank.sort(dim=2, descending=True, stable=True).indices                    # ties: lowest position first
    width = st["new_table"].shape[1] * P
    at = torch.arange(width, device=dev)
    valid = (at < kept[:, None])[:, None].expand(B, H, width)                          # [B, H, width]
    order = torch.nn.functional.pad(order, (0, max(0, width - L)))[:, :, :width]
    pos = order.masked_fill(~valid, L).sort(dim=2).values                             # kept positions in order
    src = pos.masked_fill(~valid, 0)
    new_w = w.gather(2, src).masked_fill(~valid, 0.0)
    page = st["table"].long().gather(1, (src // P).flatten(1)).view(B, H, width)
    head = torch.arange(H, device=dev)[None, :, None].expand_as(page)
    dst = st["new_table"].long()
    used = valid.view(B, H, -1, P).any(3)[:, 0]                                       # [B, W2] pages that receive rows
    for codes, scale in ((st["k8"], st["k_scale"]), (st["v8"], st["v_scale"])):
        x = _float(codes.view(torch.uint8)[page, head, src % P]) * scale[page, head][..., None]
        x = x.masked_fill(~valid[..., None], 0.0).view(B, H, -1, P, D)
        s = _block_scale(x.abs().amax((3, 4)))                                        # [B, H, W2]
        put = _e4m3(x / s[..., None, None]).permute(0, 2, 1, 3, 4)                    # [B, W2, H, P, D]
        stale = codes.view(torch.uint8)[dst]
        put = torch.where(valid.view(B, H, -1, P).permute(0, 2, 1, 3)[..., None], put, stale)
        codes.view(torch.uint8)[dst[used]] = put[used]
        scale[dst[used]] = s.permute(0, 2, 1)[used]
    return pos.masked_fill(~valid, -1).to(torch.int32), new_w, kept.to(torch.int32)


def _cache(st):
    """The handle that a program keeps for its cache tensors."""
    if "cache" not in st:
        package = str(Path(__file__).resolve().parents[1] / "wam-egale_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from wam_ops.kv8 import Kv8Cache
        st["cache"] = Kv8Cache(st["k8"], st["v8"], st["k_scale"], st["v_scale"])
    return st["cache"]


def run(st):
    c = st["case"]
    tensors = [st["k8"], st["v8"], st["k_scale"], st["v_scale"]]
    if c["op"] == "write":
        if own:
            _cache(st).write(st["k"], st["v"], st["table"], st["lens"])
        else:
            _write_one(st["k8"], st["k_scale"], st["k"], st["table"], st["lens"])
            _write_one(st["v8"], st["v_scale"], st["v"], st["table"], st["lens"])
        return tensors
    if c["op"] == "attention":
        if own:
            return list(_cache(st).attention(st["q"], st["table"], st["lens"], causal=c["causal"], return_lse=True))
        return list(_attention(st))
    if c["op"] == "weights":
        if own:
            return [_cache(st).weights(st["q"], st["table"], st["lens"], st["lse"], base=st["base"],
                                       causal=c["causal"])]
        return [_weights(st)]
    if own:
        return [*_cache(st).evict(st["table"], st["lens"], st["weights"], st["new_table"], heavy=c["heavy"],
                                  recent=c["recent"]), *tensors]
    return [*_evict(st), *tensors]


def work(case):
    c, lens = case, _lens(case)
    B, H, P = c["batch"], c["heads"], c["page"]
    if c["op"] == "write":
        n = B * c["rows"] * H * D * 2
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": n * (size + 1), "flops": 2 * n}
    if c["op"] == "evict":
        kept = sum(min(n, c["heavy"] + c["recent"]) for n in lens)
        return {"bytes": H * (4 * sum(lens) + kept * (2 * 2 * D + 8)), "flops": H * sum(lens)}
    rows = c["rows"] * c["group"]
    # (query row, key) pairs that are visible
    pairs = sum(rows * n - (c["group"] * c["rows"] * (c["rows"] - 1) // 2 if c["causal"] else 0) for n in lens)
    if c["op"] == "attention":
        return {"bytes": H * (sum(lens) * 2 * D + B * rows * (2 * 2 * D + 4)), "flops": 4 * D * H * pairs}
    width = -(-max(lens) // P) * P
    return {"bytes": H * (sum(lens) * D + B * rows * (2 * D + 4) + 8 * B * width), "flops": 2 * D * H * pairs}


# ------------------------------------------------------ the definition in 64 bits
def _scale64(amax):
    """2^n, n the smallest whole number in [-40, 119] with amax <= 448 * 2^n."""
    a = amax.double()
    n = torch.ceil(torch.log2((a / 448.0).clamp(min=2.0 ** -60)))
    n = torch.where(448.0 * torch.exp2(n - 1) >= a, n - 1, n)
    n = torch.where(448.0 * torch.exp2(n) < a, n + 1, n)
    return torch.exp2(n.clamp(SCALE_MIN, SCALE_MAX))


def _sequence64(codes, scale, table, n):
    """[H, n, D] values of a sequence's first n positions."""
    P = codes.shape[2]
    ids = table[:-(-n // P)].long()
    x = codes[ids].to(torch.float64) * scale[ids].double()[:, :, None, None]
    return x.transpose(0, 1).reshape(x.shape[1], -1, D)[:, :n]


def exact(case, seed):
    c, st = case, prepare(case, seed)
    lens, P, H, G = _lens(c), c["page"], c["heads"], c["group"]
    codes = [st[n].to(torch.float64) for n in ("k8", "v8")] if c["op"] in ("write", "evict") else []
    scales = [st[n].double() for n in ("k_scale", "v_scale")]
    if c["op"] == "write":
        for b, n in enumerate(lens):
            for a in range(n // P, (n + c["rows"] - 1) // P + 1):
                lo, hi = max(n, a * P), min(n + c["rows"], (a + 1) * P)
                pid = int(st["table"][b, a])
                for code, scale, x in zip(codes, scales, (st["k"], st["v"])):
                    x = x[b, lo - n:hi - n].double().transpose(0, 1)                # [H, rows, D]
                    s, held = _scale64(x.abs().amax((1, 2))), lo - a * P
                    if held:
                        s = torch.maximum(s, scale[pid])
                        code[pid, :, :held] *= (scale[pid] / s)[:, None, None]
                    code[pid, :, held:hi - a * P] = x / s[:, None, None]
                    scale[pid] = s
        return [*codes, *scales]
    if c["op"] == "evict":
        w = st["weights"].double()
        width = st["new_table"].shape[1] * P
        pos = torch.full((c["batch"], H, width), -1, dtype=torch.int64, device=w.device)
        new_w = torch.zeros(c["batch"], H, width, dtype=torch.float64, device=w.device)
        kept = [min(n, c["heavy"] + c["recent"]) for n in lens]
        fresh = [[t.clone() for t in codes], [t.clone() for t in scales]]
        for b, n in enumerate(lens):
            old = max(0, n - c["recent"])
            best = torch.argsort(w[b, :, :old], dim=1, descending=True, stable=True)[:, :max(0, kept[b] - (n - old))]
            late = torch.arange(old, n, device=w.device).expand(H, n - old)
            p = torch.cat([best, late], 1).sort(dim=1).values                        # [H, kept]
            pos[b, :, :kept[b]] = p
            new_w[b, :, :kept[b]] = w[b].gather(1, p)
            for i in range(2):
                x = _sequence64(codes[i], scales[i], st["table"][b], n)
                x = x.gather(1, p[:, :, None].expand(-1, -1, D))
                for a in range(-(-kept[b] // P)):
                    y = x[:, a * P:(a + 1) * P]
                    s = _scale64(y.abs().amax((1, 2)))
                    pid = int(st["new_table"][b, a])
                    fresh[0][i][pid, :, :y.shape[1]] = y / s[:, None, None]
                    fresh[1][i][pid] = s
        return [pos.to(torch.int32), new_w, torch.tensor(kept, dtype=torch.int32, device=w.device), *fresh[0], *fresh[1]]
    q = st["q"].double()
    B, T, Hq, _ = q.shape
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    acc = st["base"].double().clone() if c["op"] == "weights" else None
    for b, n in enumerate(lens):
        see = torch.ones(T, n, dtype=torch.bool, device=q.device)
        if c["causal"]:
            see = see.tril(n - T)
        k, v = (_sequence64(st[t], s, st["table"][b], n) for t, s in (("k8", scales[0]), ("v8", scales[1])))
        for h in range(Hq):
            s = (q[b, :, h] @ k[h // G].T / math.sqrt(D)).masked_fill(~see, -math.inf)
            if c["op"] == "weights":
                acc[b, h // G, :n] += torch.exp(s - st["lse"][b, :, h].double()[:, None]).sum(0)
            else:
                lse[b, :, h] = torch.logsumexp(s, 1)
                out[b, :, h] = torch.exp(s - lse[b, :, h, None]).nan_to_num(0.0) @ v[h // G]
    return [acc] if c["op"] == "weights" else [out, lse]

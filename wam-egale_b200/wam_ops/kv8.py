"""A paged KV cache held in E4M3 with a scale for each block of tokens and
head: write, attention, attention weights and eviction (the C ABI's
wamb_kv8_* entry points, include/wamb.h).

    cache = Kv8Cache.empty(pages, heads, page=64, device="cuda")
    cache.write(k, v, table, lens)                  # rows at positions lens[b] + t
    lens += k.shape[1]
    out, lse = cache.attention(q, table, lens, return_lse=True)
    cache.weights(q, table, lens, lse, base=w, out=w)       # w: running sum per position
    kept, w, lens = cache.evict(table, lens, w, new_table, heavy=1760, recent=880)

Page tables and lengths are int32 device tensors that the caller owns (page
ids may come from any allocator); they are read on the device, so calls can
be captured in a CUDA graph and replayed while they change. Calls run on the
current stream of the cache's device and synchronise nothing. Bad page ids
and lengths are reported by _lib.device_status() (code 5).
"""
import math

import torch
from torch.autograd import forward_ad

from . import _lib

HEAD_DIM = 128
PAGES = (16, 32, 64, 128)
INT32_MAX = 2 ** 31 - 1      # the C ABI's sizes; a larger number would wrap without a word


def _inference_only(t):
    """Refuses a tensor whose derivatives, backward or forward, a call would drop (or a leaf that it would write)."""
    if (t.requires_grad and torch.is_grad_enabled()) or \
            (forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None):
        raise RuntimeError("Kv8Cache is inference-only; use no_grad/inference_mode")


class Kv8Cache:
    """Handle over the four cache tensors: k8, v8 [pages, heads, page, 128]
    float8_e4m3fn, k_scale, v_scale [pages, heads] fp32, contiguous."""

    def __init__(self, k8, v8, k_scale, v_scale):
        if k8.dim() != 4 or k8.shape[3] != HEAD_DIM or k8.shape[2] not in PAGES or v8.shape != k8.shape:
            raise ValueError("k8, v8 must be [pages, heads, page, 128] with page 16, 32, 64 or 128")
        pages, heads, page = k8.shape[:3]
        for name, t in (("k8", k8), ("v8", v8)):
            if t.dtype != torch.float8_e4m3fn or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous float8_e4m3fn")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or not t.is_contiguous() or t.shape != (pages, heads):
                raise ValueError(f"{name} must be contiguous fp32 [pages, heads]")
        self.device = k8.device
        if self.device.type != "cuda" or any(t.device != self.device for t in (v8, k_scale, v_scale)):
            raise ValueError("the cache tensors must be on one CUDA device")
        self.k8, self.v8, self.k_scale, self.v_scale = k8, v8, k_scale, v_scale
        self.pages, self.heads, self.page = pages, heads, page
        self._c = _lib.Kv8CacheArgs(k8.data_ptr(), v8.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads,
                                    page)
        self._lib = _lib.load()
        self._scratch = {}     # bytes that a call's shape needs

    @classmethod
    def empty(cls, pages, heads, page=64, device="cuda"):
        """A cache of zeros."""
        code = torch.zeros(2, pages, heads, page, HEAD_DIM, dtype=torch.uint8, device=device)
        scale = torch.ones(2, pages, heads, dtype=torch.float32, device=device)
        k8, v8 = code.view(torch.float8_e4m3fn)
        return cls(k8, v8, scale[0], scale[1])

    # ------------------------------------------------------------- checks
    def _ints(self, name, t, shape):
        if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or t.device != self.device:
            raise ValueError(f"{name} must be a contiguous int32 tensor {list(shape)} on {self.device}")
        return t.data_ptr()

    def _seqs(self, seqs, batch, tokens, table, lens, counts):
        shape = table.shape
        if len(shape) != 2 or shape[0] != batch:
            raise ValueError(f"table must be [batch {batch}, width]")
        if tokens > INT32_MAX:
            raise ValueError(f"{tokens} tokens: sizes are below 2^31")
        seqs.batch, seqs.tokens, seqs.table_width = batch, tokens, shape[1]
        seqs.table = self._ints("table", table, shape)
        seqs.lens = self._ints("lens", lens, (batch,))
        if counts is not None:
            seqs.counts = self._ints("counts", counts, (batch,))

    def _rows(self, name, t, heads=None, dtypes=(torch.bfloat16,)):
        """Strides of [batch, tokens, heads, 128] with rows of 128 contiguous values."""
        b, s = t.shape, t.stride()
        if len(b) != 4 or b[3] != HEAD_DIM or t.dtype not in dtypes or t.device != self.device:
            raise ValueError(f"{name} must be [batch, tokens, heads, 128] {' or '.join(map(str, dtypes))} on {self.device}")
        if heads is not None and b[2] != heads:
            raise ValueError(f"{name} has {b[2]} heads, the cache {heads}")
        _inference_only(t)
        if s[3] != 1:
            raise ValueError(f"{name} must have unit stride along the head dim")
        # The stride of a single entry may be anything; the C ABI is told 0.
        return s[0] if b[0] > 1 else 0, s[1] if b[1] > 1 else 0, s[2] if b[2] > 1 else 0

    def _weight(self, name, t, batch, width):
        if t.dtype != torch.float32 or t.dim() != 3 or t.shape[:2] != (batch, self.heads) or not t.is_contiguous() \
                or t.device != self.device or t.shape[2] < width * self.page:
            raise ValueError(f"{name} must be contiguous fp32 [batch {batch}, heads {self.heads}, >= {width * self.page}]"
                             f" on {self.device}")
        _inference_only(t)
        return t.data_ptr()

    def _call(self, fn, args, workspace_bytes=None, shape=None):
        """fn(args) on the current stream of the cache's device, with scratch
        of its own from that stream's (or the captured graph's) pool."""
        index = self.device.index
        if torch._C._cuda_getDevice() != index:
            with torch.cuda.device(self.device):
                return self._call(fn, args, workspace_bytes, shape)
        if workspace_bytes is not None:
            n = self._scratch.get(shape)
            if n is None:
                n = self._scratch[shape] = workspace_bytes(args)
            if n:
                ws = self.k_scale.new_empty((n + 3) // 4)
                args.workspace, args.workspace_bytes = ws.data_ptr(), n
        rc = fn(args, torch._C._cuda_getCurrentRawStream(index))
        if rc:
            _lib.check(rc)

    # ---------------------------------------------------------- operators
    def write(self, k, v, table, lens, counts=None):
        """Rows t < counts[b] (all without `counts`) of k, v [batch, tokens,
        heads, 128] (bf16 or fp32, any strides that are multiples of 8 elements) go to
        positions lens[b] + t. A page that already holds positions keeps the
        larger of its scale and the new rows'; its codes follow. `lens` is not
        changed."""
        a = _lib.Kv8WriteArgs()
        a.cache = self._c
        dtypes = (torch.bfloat16, torch.float32)
        a.k_stride[:] = self._rows("k", k, self.heads, dtypes)
        a.v_stride[:] = self._rows("v", v, self.heads, dtypes)
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("k and v must have one shape and dtype")
        self._seqs(a.seqs, k.shape[0], k.shape[1], table, lens, counts)
        a.k, a.v, a.x_is_f32 = k.data_ptr(), v.data_ptr(), int(k.dtype == torch.float32)
        self._call(self._lib.wamb_kv8_write, a)

    def _attention_args(self, q, table, lens, counts, causal, scale):
        a = _lib.Kv8AttentionArgs()
        a.cache = self._c
        a.q_stride[:] = self._rows("q", q)
        batch, tokens, heads, _ = q.shape
        if heads == 0 or heads % self.heads:
            raise ValueError(f"q has {heads} heads, no multiple of the cache's {self.heads}")
        if heads > INT32_MAX:
            raise ValueError(f"{heads} query heads: sizes are below 2^31")
        scale = HEAD_DIM ** -0.5 if scale is None else float(scale)
        if not (scale > 0 and math.isfinite(scale)):
            raise ValueError("scale must be positive and finite")
        self._seqs(a.seqs, batch, tokens, table, lens, counts)
        a.q, a.q_heads, a.causal, a.scale = q.data_ptr(), heads, int(bool(causal)), scale
        return a

    def attention(self, q, table, lens, counts=None, causal=False, scale=None, out=None, lse=None, return_lse=False):
        """softmax(scale q k^T) v of q [batch, tokens, q_heads, 128] bf16 over
        the first lens[b] positions (causal: row t of counts[b] sees positions
        <= lens[b] - counts[b] + t); q_heads is a multiple of the cache's heads.
        Returns out (bf16 like q) or (out, lse [batch, tokens, q_heads] fp32).
        A row without visible positions gives 0 and -inf; rows past counts[b]
        of `out` and `lse` are left as they were."""
        a = self._attention_args(q, table, lens, counts, causal, scale)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape:
            raise ValueError("out must be shaped like q")
        elif any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise ValueError("out must not be an expanded tensor")
        a.out_stride[:] = self._rows("out", out)
        a.out = out.data_ptr()
        if lse is None and return_lse:
            lse = self.k_scale.new_empty((a.seqs.batch, a.seqs.tokens, a.q_heads))
        if lse is not None:
            a.lse = self._lse(lse, q)
        self._call(self._lib.wamb_kv8_attention, a, self._lib.wamb_kv8_attention_workspace_bytes, ("attention", q.shape))
        return (out, lse) if return_lse else out

    def _lse(self, lse, q):
        if lse.dtype != torch.float32 or lse.shape != q.shape[:3] or not lse.is_contiguous() or lse.device != self.device:
            raise ValueError("lse must be contiguous fp32 [batch, tokens, q_heads]")
        _inference_only(lse)
        return lse.data_ptr()

    def weights(self, q, table, lens, lse, base=None, out=None, counts=None, causal=False, scale=None):
        """base + the attention weight that each cached position received from
        the rows of q, summed over them and over the query heads of a cached
        head: fp32 [batch, heads, capacity], capacity >= table width * page
        (that without `base` and `out`). `lse` is attention's, for the same
        arguments; out=base adds in place."""
        a = self._attention_args(q, table, lens, counts, causal, scale)
        batch, width = q.shape[0], table.shape[1]
        a.lse = self._lse(lse, q)
        if base is not None:
            a.base = self._weight("base", base, batch, width)
        if out is None:
            shape = base.shape if base is not None else (batch, self.heads, width * self.page)
            out = self.k_scale.new_empty(shape)
        a.weights = self._weight("out", out, batch, width)
        if base is not None and base.shape != out.shape:
            raise ValueError("base and out must have one shape")
        a.weights_cap = out.shape[2]
        self._call(self._lib.wamb_kv8_weights, a, self._lib.wamb_kv8_weights_workspace_bytes, ("weights", q.shape))
        return out

    def evict(self, table, lens, weights, new_table, heavy, recent, max_len=None):
        """Keeps, for each sequence and cached head, the last `recent` positions
        and the `heavy` earlier ones with the largest weights (ties: the lowest
        positions), and moves their rows, in order, to the pages of new_table
        (int32 [batch, new_width]; pages that no live table names, each once). Returns
        (kept [batch, heads, new_width * page] int32 old positions, -1 behind
        the last; their weights, 0 behind the last; new lengths int32 [batch]).
        max_len: an upper bound of lens (default: the table's capacity);
        min(heavy + recent, max_len) tokens must fit the new pages. A sequence
        that would keep more than they hold keeps nothing and is reported."""
        batch = lens.shape[0] if lens.dim() == 1 else -1
        a = _lib.Kv8EvictArgs()
        a.cache = self._c
        self._seqs(a.seqs, batch, 0, table, lens, None)
        if new_table.dim() != 2 or new_table.shape[0] != batch:
            raise ValueError(f"new_table must be [batch {batch}, new_width]")
        a.new_table = self._ints("new_table", new_table, new_table.shape)
        a.new_width = new_table.shape[1]
        a.weights = self._weight("weights", weights, batch, table.shape[1])
        a.weights_cap = weights.shape[2]
        heavy, recent = int(heavy), int(recent)
        max_len = table.shape[1] * self.page if max_len is None else int(max_len)
        if max(abs(heavy), abs(recent)) > INT32_MAX or abs(max_len) > 2 ** 62:
            raise ValueError(f"heavy, recent and max_len ({heavy}, {recent}, {max_len}) must be below 2^31, 2^31 and 2^62")
        a.heavy, a.recent, a.max_len = heavy, recent, max_len
        shape = (batch, self.heads, a.new_width * self.page)
        kept, new_lens = table.new_empty(shape), table.new_empty(batch)
        new_weights = weights.new_empty(shape)
        a.kept, a.new_weights, a.new_lens = kept.data_ptr(), new_weights.data_ptr(), new_lens.data_ptr()
        self._call(self._lib.wamb_kv8_evict, a)
        return kept, new_weights, new_lens

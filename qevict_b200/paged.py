"""Paged KV cache: full-context K/V of many sequences in pages of one pool.

For prompts that arrive in chunks and for full-cache decode, beside the
Sticky layout (which keeps a selected part of one prompt).  Four operators of
the native library, each an ordinary kernel launch on the current stream of its
tensors' device, none of which synchronises:

  qk_norm_rope     per-head norm and rotation of query and key heads
  paged_append     the same, with the new keys and values written into pages
  paged_gather     pages read back into contiguous rows [tokens, heads, head_dim]
                   (as model.prefill_attention takes them)
  paged_attention  chunks of new tokens, from one token to whole prompts,
                   over the pages

What a call writes (outputs, and the pool of paged_append) may not share memory
with anything else of the call: refused, but for the in-place outputs that are
named below.

A prompt collected in pages goes to a Sticky layer as the model's own prompt does:
model.prefill_attention over its rotated queries and the rows read back gives the
column sums, and StickyLayerState.prefill takes those with K and V transposed to
[batch, heads, tokens, head_dim].

PagedKVCache holds a pool and calls them.  Pools are [pages, kv_heads,
page_size, head_dim] in the model's dtype or INT8 with one fp32 scale per row
([pages, kv_heads, page_size]; not negative, value scales of one sequence up to
2^49, ones below 2^-60 may count as that); token j of sequence b lives in page
block_table[b, j // page_size] at offset j % page_size.
"""

import ctypes
import math

import torch

from . import _native as N

_INT_MAX = 2 ** 31 - 1
_DTYPES = {torch.float32: N.QV_F32, torch.bfloat16: N.QV_BF16, torch.float16: N.QV_F16}


def rope_table(max_pos, rot_dim, theta=10000.0, scaling=None, device="cuda"):
    """The fp32 rotation table [max_pos, rot_dim]: cos | sin, angles in 64 bits.

    scaling (long contexts), a dict with "type" and "factor" f:
      linear  positions divided by f
      ntk     theta * f^(r / (r - 2)): the slowest pair turns f times slower, the fastest as before
      llama3  frequencies divided by f where the wavelength is above
              original_max_position / low_freq_factor, kept where below
              original_max_position / high_freq_factor, blended between
      yarn    divided by f below beta_slow turns over original_max_position, kept above
              beta_fast, a linear ramp over the pairs between; cos and sin times
              attention_factor (default 0.1 ln f + 1)"""
    if max_pos <= 0 or rot_dim < 8 or rot_dim % 8:
        raise N.QevictError("rope_table: max_pos > 0 and rot_dim a positive multiple of 8 are needed")
    dev = torch.device(device)
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=dev)
    mult = 1.0
    if scaling is None:
        inv = theta ** (-i / rot_dim)
    else:
        kind, f = scaling["type"], float(scaling["factor"])
        if kind == "ntk":
            theta = theta * f ** (rot_dim / (rot_dim - 2))
        inv = theta ** (-i / rot_dim)
        if kind == "linear":
            inv = inv / f
        elif kind == "llama3":
            lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
            turns = float(scaling["original_max_position"]) * inv / (2 * math.pi)
            keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
            inv = inv / f * (1 - keep) + inv * keep
        elif kind == "yarn":
            orig = float(scaling["original_max_position"])

            def pair(turns):   # the (fractional) pair that turns this often over the original length
                return rot_dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo = max(math.floor(pair(float(scaling.get("beta_fast", 32)))), 0)
            hi = min(math.ceil(pair(float(scaling.get("beta_slow", 1)))), rot_dim - 1)
            ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            inv = inv * (1 - ramp) + inv / f * ramp
            mult = float(scaling.get("attention_factor") or 0.1 * math.log(f) + 1.0)
        elif kind != "ntk":
            raise N.QevictError(f"rope_table: unknown scaling type {kind!r}")
    a = torch.arange(max_pos, dtype=torch.float64, device=dev)[:, None] * inv
    return (torch.cat([a.cos(), a.sin()], 1) * mult).float()


# Checks format their message only when they fail: a decode step's calls are
# short enough for the host's time per call to count.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # current_stream(dev).cuda_stream, 2 us sooner


def _bad(name, expected, x):
    return N.QevictError(f"{name}: expected {expected}, got {tuple(x.shape)} {x.dtype} on {x.device}")


def _heads(name, x, tokens, dim, dtype, dev):
    """A [tokens, heads, head_dim] tensor whose heads are contiguous within a token (a view of a
    packed projection will do); returns (tokens, heads, token stride)."""
    if x.ndim != 3 or x.dtype is not dtype or x.device != dev:
        raise _bad(name, f"[tokens, heads, {dim}] {dtype} on {dev}", x)
    n, h, d = x.shape
    st, sh, sd = x.stride()
    if d != dim or n != (n if tokens is None else tokens) or n > _INT_MAX:
        raise _bad(name, f"[{'tokens' if tokens is None else tokens}, heads, {dim}]", x)
    if sd != 1 or (sh != dim and h != 1):
        raise N.QevictError(f"{name}: a token's heads must be contiguous, got strides {(st, sh, sd)}")
    return n, h, st if n > 1 else h * dim


def _apart(name, out, *reads, inplace=None):
    """Refuse an output that shares memory with a tensor that the call reads.  It may take the place of `inplace`, of the
    same shape and contiguous, where the caller's kernel reads each row in the block that writes it, before it does."""
    a = out.data_ptr()
    z = a + out.numel() * out.element_size()
    if a == z:
        return
    if inplace is not None and not (inplace.data_ptr() == a and inplace.is_contiguous()):
        reads += (inplace,)
    for x in reads:
        b = x.data_ptr()
        if b >= z or not x.numel():
            continue
        if b < a and b + x.element_size() * (sum((d - 1) * s for d, s in zip(x.shape, x.stride())) + 1) <= a:
            continue
        raise N.QevictError(f"{name} shares memory with another tensor of the call")


def _vector(name, x, shape, dtype, dev):
    if x.dtype is not dtype or x.shape != shape or x.device != dev or not x.is_contiguous():
        raise _bad(name, f"a contiguous {shape} {dtype} tensor on {dev}", x)


def _launch(dev, name, *args):
    """Call a native entry point on the current stream of `dev`."""
    fn = getattr(N.lib(), name)
    i = dev.index
    if torch.cuda.current_device() == i:
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(i))
    if rc:
        N.check(rc, name)


def _pool(k_pages, v_pages, k_scale, v_scale, dtype, err):
    """The native descriptor of a pool (checked), with its device, heads, page size and head_dim."""
    code = _DTYPES.get(dtype)
    if code is None:
        raise N.QevictError(f"dtype {dtype} is not one of fp32, bf16, fp16")
    if not k_pages.is_cuda:
        raise N.QevictError("pages must be on a CUDA device")
    dev, shape, pt = k_pages.device, k_pages.shape, k_pages.dtype
    if (len(shape) != 4 or v_pages.shape != shape or v_pages.dtype is not pt or v_pages.device != dev
            or not k_pages.is_contiguous() or not v_pages.is_contiguous()):
        raise _bad("pages", "k and v contiguous [pages, kv_heads, page_size, head_dim] of one type and device; v", v_pages)
    P, H, S, D = shape
    if S not in _PAGE_SIZES or not 8 <= D <= 256 or D % 8:
        _pool_sizes(S, D)
    ks = vs = None
    if pt is torch.int8:
        if k_scale is None or v_scale is None:
            raise N.QevictError("INT8 pages need k_scale and v_scale")
        _vector("k_scale", k_scale, (P, H, S), torch.float32, dev)
        _vector("v_scale", v_scale, (P, H, S), torch.float32, dev)
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    elif pt is not dtype:
        raise N.QevictError(f"pages of {pt} do not go with {dtype} rows")
    elif k_scale is not None or v_scale is not None:
        raise N.QevictError("k_scale and v_scale go with INT8 pages only")
    if err is not None:
        _vector("err", err, (1,), torch.int32, dev)
        err = err.data_ptr()
    c = N.QvPagedCache(k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, err, P, H, S, D, code, 0 if ks is None else 8)
    return c, dev, H, S, D


_PAGE_SIZES = (16, 32, 64, 128)


def _pool_sizes(page_size, head_dim):
    if page_size not in _PAGE_SIZES:
        raise N.QevictError(f"page_size {page_size} is not 16, 32, 64 or 128")
    _head_dim(head_dim)


def _head_dim(D):
    if not 8 <= D <= 256 or D % 8:
        raise N.QevictError(f"head_dim {D} is not a multiple of 8 up to 256")


def _turn(tokens, dim, dtype, dev, positions, table, q_weight, k_weight):
    """Checked rotation and norm weights: (q_weight, k_weight, table, max_pos, rot_dim, positions), pointers or None."""
    if q_weight is not None:
        _vector("q_weight", q_weight, (dim,), dtype, dev)
        q_weight = q_weight.data_ptr()
    if k_weight is not None:
        _vector("k_weight", k_weight, (dim,), dtype, dev)
        k_weight = k_weight.data_ptr()
    if table is None:
        return q_weight, k_weight, None, 0, 0, None
    if table.ndim != 2 or table.dtype is not torch.float32 or table.device != dev or not table.is_contiguous():
        raise _bad("table", f"a contiguous [max_pos, rot_dim] fp32 tensor on {dev} (rope_table)", table)
    max_pos, rot = table.shape
    if max_pos > _INT_MAX:
        raise _bad("table", "fewer positions", table)
    if not 8 <= rot <= dim or rot % 8:
        raise N.QevictError(f"table: rot_dim {rot} is not a multiple of 8 up to head_dim {dim}")
    if positions is None:
        raise N.QevictError("a rotation needs positions")
    _vector("positions", positions, (tokens,), torch.int32, dev)
    return q_weight, k_weight, table.data_ptr(), max_pos, rot, positions.data_ptr()


def qk_norm_rope(q, k, positions=None, table=None, *, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                 out=None):
    """RMS norm (where a weight is given) and rotation (where a table is) of each query and key head.

    q [T, q_heads, D], k [T, kv_heads, D], heads contiguous within a token, tokens on 16-byte boundaries;
    positions [T] int32; table from rope_table, its rot_dim the part of the head that turns, in pairs
    (i, i + rot_dim/2), or (2i, 2i+1) with interleaved.  Returns contiguous (q, k), or fills out=(q_out, k_out),
    which may be q and k themselves where those are contiguous.  A position outside the table gives NaN.  (qv_qk_norm_rope)"""
    dt, dev = q.dtype, q.device
    code = _DTYPES.get(dt)
    if not q.is_cuda or code is None or q.ndim != 3:
        raise _bad("q", "a [tokens, heads, head_dim] fp32, bf16 or fp16 CUDA tensor", q)
    D = q.shape[2]
    if not 8 <= D <= 256 or D % 8:
        _head_dim(D)
    T, Hq, qs = _heads("q", q, None, D, dt, dev)
    _, H, ks = _heads("k", k, T, D, dt, dev)
    qw, kw, tab, max_pos, rot, pos = _turn(T, D, dt, dev, positions, table, q_weight, k_weight)
    if out is None:
        qo, ko = q.new_empty(T, Hq, D), q.new_empty(T, H, D)
    else:
        qo, ko = out
        _vector("out[0]", qo, (T, Hq, D), dt, dev)
        _vector("out[1]", ko, (T, H, D), dt, dev)
        _apart("out[0]", qo, k, ko, inplace=q)
        _apart("out[1]", ko, q, inplace=k)
    _launch(dev, "qv_qk_norm_rope", T, Hq, H, D, code, q.data_ptr(), qs, k.data_ptr(), ks, qw, kw, eps, tab, max_pos,
            rot, bool(interleaved), pos, qo.data_ptr(), ko.data_ptr())
    return qo, ko


def paged_append(q, k, v, slots, positions, table, k_pages, v_pages, *, k_scale=None, v_scale=None, q_weight=None,
                 k_weight=None, eps=1e-6, interleaved=False, q_out=None, err=None):
    """qk_norm_rope with the keys and the values v [T, kv_heads, D] written into the pool: token t to slots[t]
    (int64, page * page_size + offset; negative: not written).  Returns the queries (q_out may be q where that is
    contiguous).  INT8 pages get scale = max|row| / 127 and code = rint(row / scale) of the fp32 row.  A slot must
    appear at most once per call; err collects device errors (PagedKVCache.read_error).  (qv_paged_append)"""
    dt = q.dtype
    c, dev, H, _, D = _pool(k_pages, v_pages, k_scale, v_scale, dt, err)
    T, Hq, qs = _heads("q", q, None, D, dt, dev)
    _, kh, ks = _heads("k", k, T, D, dt, dev)
    _, vh, vs = _heads("v", v, T, D, dt, dev)
    if kh != H or vh != H:
        raise N.QevictError(f"k and v must have the pool's {H} heads, got {kh} and {vh}")
    _vector("slots", slots, (T,), torch.int64, dev)
    qw, kw, tab, max_pos, rot, pos = _turn(T, D, dt, dev, positions, table, q_weight, k_weight)
    if q_out is None:
        q_out = q.new_empty(T, Hq, D)
    else:
        _vector("q_out", q_out, (T, Hq, D), dt, dev)
        _apart("q_out", q_out, k, v, inplace=q)
    _launch(dev, "qv_paged_append", ctypes.byref(c), T, Hq, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, qw,
            kw, eps, tab, max_pos, rot, bool(interleaved), pos, slots.data_ptr(), q_out.data_ptr())
    return q_out


def _tables(block_table, kv_lens, cu, dev):
    if (block_table.ndim != 2 or block_table.dtype is not torch.int32 or block_table.device != dev
            or not block_table.is_contiguous()):
        raise _bad("block_table", f"a contiguous [batch, max_pages] int32 tensor on {dev}", block_table)
    B, width = block_table.shape
    if not width:
        raise _bad("block_table", "pages", block_table)
    _vector("kv_lens", kv_lens, (B,), torch.int32, dev)
    _vector("cumulative lengths", cu, (B + 1,), torch.int32, dev)
    return B, width


def paged_gather(k_pages, v_pages, block_table, kv_lens, cu_kv, total, *, k_scale=None, v_scale=None, dtype=None,
                 out=None, err=None):
    """The cached rows as contiguous (k, v) [total, kv_heads, D] in dtype (default: the pages' own; INT8 pages
    need it): the first kv_lens[b] tokens of sequence b from row cu_kv[b] on, cu_kv [batch + 1] ascending int32;
    rows of no sequence are left as they were (out) or undefined.  (qv_paged_gather)"""
    dt = k_pages.dtype if dtype is None else dtype
    c, dev, H, _, D = _pool(k_pages, v_pages, k_scale, v_scale, dt, err)
    B, width = _tables(block_table, kv_lens, cu_kv, dev)
    if not 0 <= total <= _INT_MAX:
        raise N.QevictError(f"total {total} is not a number of rows")
    if out is None:
        ko = torch.empty(total, H, D, dtype=dt, device=dev)
        vo = torch.empty_like(ko)
    else:
        ko, vo = out
        _vector("out[0]", ko, (total, H, D), dt, dev)
        _vector("out[1]", vo, (total, H, D), dt, dev)
        _apart("out[0]", ko, k_pages, vo, v_pages)
        _apart("out[1]", vo, k_pages, v_pages)
    _launch(dev, "qv_paged_gather", ctypes.byref(c), B, block_table.data_ptr(), width, kv_lens.data_ptr(),
            cu_kv.data_ptr(), total, ko.data_ptr(), vo.data_ptr())
    return ko, vo


def paged_attention(q, k_pages, v_pages, block_table, kv_lens, cu_q, *, k_scale=None, v_scale=None, causal=True,
                    scale=None, max_q=None, max_kv=None, out=None, err=None):
    """Attention of chunks of new tokens over the pool.

    q [T, q_heads, D] (heads contiguous within a token), D 64 or 128, q_heads a multiple (up to 16 times) of
    kv_heads; sequence b's new tokens are rows cu_q[b] .. cu_q[b+1] (int32 [batch + 1]) and the last of its
    kv_lens[b] (int32 [batch]) cached tokens; block_table int32 [batch, max_pages].  Causal: each token sees the
    keys up to its own.  A row that sees no key gives 0; rows of no chunk are left as they were (out) or
    undefined.  max_q / max_kv: upper bounds of the chunk and cached lengths, which size the launch (default:
    T, and all that the block table can hold); a captured call serves any lengths below them, fastest where they
    are close: pass max_q=1 for a decode batch (without it more than 16 rows per kv head run as prompts do), and
    max_kv near the longest.  out may be q where that is contiguous.  scale (positive) defaults to D^-1/2.
    (qv_paged_attention)"""
    dt = q.dtype
    c, dev, H, S, D = _pool(k_pages, v_pages, k_scale, v_scale, dt, err)
    if D != 64 and D != 128:
        raise N.QevictError(f"head_dim {D} is not 64 or 128")
    T, Hq, qs = _heads("q", q, None, D, dt, dev)
    if Hq % H or Hq // H > 16:
        raise N.QevictError(f"{Hq} query heads are not 1 to 16 times the pool's {H}")
    B, width = _tables(block_table, kv_lens, cu_q, dev)
    max_q = T if max_q is None else min(max_q, T)
    max_kv = width * S if max_kv is None else max_kv
    if max_q < 0 or not 0 <= max_kv <= width * S or max_kv > 1 << 30:
        raise N.QevictError(f"max_q {max_q} and max_kv {max_kv} must be lengths, max_kv at most the block table's {width * S} and 2^30")
    if out is None:
        out = q.new_empty(T, Hq, D)
    else:
        _vector("out", out, (T, Hq, D), dt, dev)
        _apart("out", out, inplace=q)
    cp = ctypes.byref(c)
    wsb = N.lib().qv_paged_attention_workspace_bytes(cp, B, Hq, T, max_q, max_kv)
    # from torch's allocator at each call: a captured graph gets one of its own
    ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
    _launch(dev, "qv_paged_attention", cp, B, Hq, block_table.data_ptr(), width, kv_lens.data_ptr(), cu_q.data_ptr(),
            T, max_q, max_kv, q.data_ptr(), qs, D ** -0.5 if scale is None else scale, bool(causal),
            out.data_ptr(), ws.data_ptr() if wsb else None, wsb)
    return out


class PagedKVCache:
    """A pool of pages for one layer, and the operators on it.

    bits = 16 keeps pages in dtype, 8 in INT8 with fp32 row scales (fp32 pools: 32 or 8).  Which pages a
    sequence owns is the caller's: block_table [batch, max_pages] int32 on the pool's device."""

    def __init__(self, pages, kv_heads, head_dim, page_size=64, dtype=torch.bfloat16, bits=None, device="cuda"):
        if dtype not in _DTYPES:
            raise N.QevictError(f"dtype {dtype} is not one of fp32, bf16, fp16")
        full = torch.finfo(dtype).bits
        bits = full if bits is None else bits
        if bits not in (8, full):
            raise N.QevictError(f"bits {bits} is not 8 or the dtype's own {full}")
        if pages <= 0 or kv_heads <= 0:
            raise N.QevictError("a pool needs pages and heads")
        _pool_sizes(page_size, head_dim)
        self.dtype, self.page_size = dtype, page_size
        shape = (pages, kv_heads, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=torch.int8 if bits == 8 else dtype, device=device)
        self.v_pages = torch.zeros_like(self.k_pages)
        self.k_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device) if bits == 8 else None
        self.v_scale = torch.zeros_like(self.k_scale) if bits == 8 else None
        self.err = torch.zeros(1, dtype=torch.int32, device=device)

    def slots(self, block_table, seq, pos):
        """Slots of tokens at index pos [T] of sequences seq [T] (int64 [T]).  A negative pos gives -1 (append writes
        nothing); an index outside the block table, or a page that is not the pool's, gives a slot behind the
        pool (append writes nothing and raises QV_DERR_CAPACITY)."""
        B, width = block_table.shape
        pages, size = self.k_pages.shape[0], self.page_size
        pos, seq = pos.long(), seq.long()
        before = pos < 0
        if not B * width:
            return torch.full_like(pos, pages * size).masked_fill_(before, -1)
        page = pos >> size.bit_length() - 1
        outside = (page >= width) | (seq < 0) | (seq >= B)
        at = torch.add(page, seq, alpha=width).masked_fill_(outside | before, 0)
        ids = block_table.take(at).long()
        ids.masked_fill_(outside | (ids < 0), pages)           # an id above the pool's lies behind it as it is
        return torch.add(pos & size - 1, ids, alpha=size).masked_fill_(before, -1)

    def append(self, q, k, v, slots, positions=None, table=None, **kw):
        return paged_append(q, k, v, slots, positions, table, self.k_pages, self.v_pages, k_scale=self.k_scale,
                            v_scale=self.v_scale, err=self.err, **kw)

    def gather(self, block_table, kv_lens, cu_kv, total, **kw):
        return paged_gather(self.k_pages, self.v_pages, block_table, kv_lens, cu_kv, total, k_scale=self.k_scale,
                            v_scale=self.v_scale, dtype=self.dtype, err=self.err, **kw)

    def attend(self, q, block_table, kv_lens, cu_q, **kw):
        return paged_attention(q, self.k_pages, self.v_pages, block_table, kv_lens, cu_q, k_scale=self.k_scale,
                               v_scale=self.v_scale, err=self.err, **kw)

    def read_error(self):
        """The device error word (a synchronisation): bits QV_DERR_TABLE, QV_DERR_CAPACITY, QV_DERR_TIMEOUT."""
        return int(self.err.item())

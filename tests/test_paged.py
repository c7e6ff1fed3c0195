"""Paged KV cache: norm + rotation, append, read-back and attention against
their definitions in 64 bits.

Bounds: a result rounded to a type t is off by eps(t)/2 of its value; what the
kernels do in fp32 before that adds a few 2^-24 of the terms' magnitudes, which
each bound below spells out.
"""

import ctypes
import math

import pytest
import torch

from qevict_b200 import _native as N
from qevict_b200 import paged

DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TINY = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -149}   # half a subnormal step


def half(dt):
    return torch.finfo(dt).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rand(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * std


# ------------------------------------------------------------------ definitions
def ref_heads(x, w, eps, table, pos, interleaved):
    """Norm and rotation in 64 bits: (value, magnitude of the terms it sums)."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    y, mag = x.clone(), x.abs()
    if table is not None:
        r = table.shape[1]
        c, s = table[pos.long()].double()[:, None].chunk(2, -1)
        i = torch.arange(r // 2, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        both = x[..., a].abs() + x[..., b].abs()
        mag = mag.clone()
        mag[..., a], mag[..., b] = both, both
    return y, mag


def close_rows(got, ref, mag, dt):
    # fp32 steps: the mean of squares (pairwise, below 16 ulp), rsqrt, two products, two of the rotation: 2^-19 of the terms
    bound = ref.abs() * half(dt) * 1.001 + mag * 2.0 ** -19 + TINY[dt]
    assert got.dtype == dt
    assert bool(((got.double() - ref).abs() <= bound).all()), float(((got.double() - ref).abs() / bound).max())


def ref_attention(q, ks, vs, causal=True, scale=None):
    """q [n, Hq, D]; ks, vs [L, H, D] in 64 bits -> (out, sum of p |v|, largest |q||k| scale)."""
    n, Hq, D = q.shape
    L, H = ks.shape[:2]
    scale = D ** -0.5 if scale is None else scale
    q = q.double().view(n, H, Hq // H, D)
    if L == 0:
        z = torch.zeros(n, Hq, D, dtype=torch.float64, device=q.device)
        return z, z, 0.0
    x = torch.einsum("nhgd,lhd->hgnl", q, ks) * scale
    if causal:
        seen = torch.arange(L, device=q.device)[None] <= torch.arange(L - n, L, device=q.device)[:, None]
        x = x.masked_fill(~seen, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    out = torch.einsum("hgnl,lhd->nhgd", p, vs).reshape(n, Hq, D)
    mag = torch.einsum("hgnl,lhd->nhgd", p, vs.abs()).reshape(n, Hq, D)
    big = float(q.norm(dim=-1).max() * ks.norm(dim=-1).max()) * abs(scale)
    return out, mag, big


def attention_bound(out, mag, big, L, D, dt, vmax):
    """The output's rounding; each probability's rounding to the type (with the value scale of an INT8 row in it);
    fp32 logits (D terms of size up to |q||k|, an exponent's error is relative to p) and sums over L keys; and, in
    fp16, probabilities below its smallest normal: half a step of 2^-24 each against a sum of at least 1."""
    delta = 2.0 ** -24 * (2 * (D + 8) * big + L + 64)
    b = out.abs() * half(dt) * 1.001 + mag * (half(dt) + delta) * 1.01 + TINY[dt]
    return b + (L * 2.0 ** -25 * vmax if dt == FP16 else 0.0)


class Pool:
    """A pool with `lens` tokens per sequence in pages of random order; every slot that no sequence owns holds
    NaN (in INT8 pools its scale), and the block table's unused entries ids outside the pool."""

    def __init__(self, g, lens, H, D, page, dt, q8, extra=3, std=1.0):
        need = [-(-n // page) for n in lens]
        P, B = sum(need) + extra, len(lens)
        self.cache = paged.PagedKVCache(P, H, D, page, dt, bits=8 if q8 else None, device=DEV)
        c = self.cache
        ids = torch.randperm(P, generator=g, device=DEV)[: sum(need)].tolist()
        width = max(1, max(need, default=1))
        bt = torch.full((B, width), -7, dtype=torch.int32)
        bt[:, 1::2] = 2 ** 31 - 1
        for b in range(B):
            for i in range(need[b]):
                bt[b, i] = ids.pop()
        self.bt = bt.to(DEV)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.ks, self.vs = [], []
        for x in (c.k_pages, c.v_pages):
            x.fill_(127 if q8 else math.nan)
        if q8:
            c.k_scale.fill_(math.nan)
            c.v_scale.fill_(math.nan)
        for b, n in enumerate(lens):
            pos = torch.arange(n, device=DEV)
            sl = c.slots(self.bt, torch.full_like(pos, b), pos)
            pg, off = sl // page, sl % page
            for x, sc, keep in ((c.k_pages, c.k_scale, self.ks), (c.v_pages, c.v_scale, self.vs)):
                rows = rand(g, n, H, D, std=std)
                if q8:
                    s = rows.abs().amax(-1) / 127
                    code = (rows / s[..., None]).round()
                    x[pg, :, off] = code.to(torch.int8)
                    sc[pg, :, off] = s
                    keep.append(code.double() * s.double()[..., None])
                else:
                    x[pg, :, off] = rows.to(dt)
                    keep.append(rows.to(dt).double())


def cu(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)


def check_attention(g, q_lens, kv_lens, Hq, H, D, page, dt, q8, causal=True, scale=None, std=1.0, qstd=1.0, **kw):
    pool = Pool(g, kv_lens, H, D, page, dt, q8, std=std)
    T = sum(q_lens)
    qkv = rand(g, T + 2, Hq + 2 * H, D, std=qstd).to(dt)    # two rows of padding behind the last sequence
    q = qkv[:, :Hq]
    out = torch.full((T + 2, Hq, D), 7.0, dtype=dt, device=DEV)
    got = pool.cache.attend(q, pool.bt, pool.lens, cu(q_lens), causal=causal, scale=scale, out=out, **kw)
    assert got is out and pool.cache.read_error() == 0
    assert bool((out[T:] == 7).all())
    at = 0
    for b, n in enumerate(q_lens):
        if n:
            o, mag, big = ref_attention(q[at:at + n], pool.ks[b], pool.vs[b], causal, scale)
            vmax = float(pool.vs[b].abs().max()) if kv_lens[b] else 0.0
            bound = attention_bound(o, mag, big, kv_lens[b], D, dt, vmax)
            d = (out[at:at + n].double() - o).abs()
            assert bool((d <= bound).all()), (b, n, kv_lens[b], float((d / bound).max()))
        at += n
    return pool, q, out


# ------------------------------------------------------------------ CPU: tables, refusals
@pytest.mark.parametrize("scaling,hf", [
    (None, None),
    (dict(type="linear", factor=4.0), dict(rope_type="linear", factor=4.0)),
    (dict(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position=8192),
     dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
          original_max_position_embeddings=8192)),
    (dict(type="yarn", factor=16.0, original_max_position=4096),
     dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)),
])
def test_rope_table_against_transformers(scaling, hf):
    from transformers import LlamaConfig
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding
    theta, D, n = 500000.0, 128, 4096
    rp = dict(hf or dict(rope_type="default"), rope_theta=theta)
    conf = LlamaConfig(hidden_size=D * 2, num_attention_heads=2, head_dim=D, rope_theta=theta, rope_scaling=rp,
                       rope_parameters=rp, max_position_embeddings=65536)
    cos, sin = LlamaRotaryEmbedding(conf)(torch.zeros(1), torch.arange(n)[None])
    t = paged.rope_table(n, D, theta, scaling, device="cpu")
    # theirs multiplies fp32 frequencies (three roundings) by the position: an angle off by 2^-22 of itself
    bound = (2.0 ** -22 * torch.arange(n)[:, None] + 2.0 ** -22) * 1.5
    assert bool(((t[:, : D // 2] - cos[0, :, : D // 2]).abs() <= bound).all())
    assert bool(((t[:, D // 2:] - sin[0, :, : D // 2]).abs() <= bound).all())


def test_rope_table_ntk_keeps_the_fastest_pair_and_stretches_the_slowest():
    f, D, theta = 8.0, 64, 10000.0
    a = paged.rope_table(3, D, theta, device="cpu").double()
    b = paged.rope_table(3, D, theta, dict(type="ntk", factor=f), device="cpu").double()
    assert torch.equal(a[:, 0], b[:, 0])
    slow = theta ** (-(D - 2) / D)
    assert abs(float(torch.asin(b[1, -1])) - slow / f) <= slow * 2.0 ** -23
    with pytest.raises(N.QevictError):
        paged.rope_table(3, D, theta, dict(type="other", factor=f), device="cpu")
    with pytest.raises(N.QevictError):
        paged.rope_table(3, 12, theta, device="cpu")


def test_python_refusals_without_a_gpu():
    x = torch.zeros(2, 4, 64)
    with pytest.raises(N.QevictError):
        paged.qk_norm_rope(x, x)
    pages = torch.zeros(2, 1, 16, 64)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(N.QevictError):
        paged.paged_append(x, x, x, i, None, None, pages, pages)
    with pytest.raises(N.QevictError):
        paged.paged_gather(pages, pages, i, i[0], i[0], 0)
    with pytest.raises(N.QevictError):
        paged.paged_attention(x, pages, pages, i, i[0], i[0])
    for bad in (dict(bits=4), dict(dtype=torch.float64), dict(page_size=48), dict(pages=0), dict(head_dim=20)):
        with pytest.raises(N.QevictError):
            paged.PagedKVCache(**{**dict(pages=2, kv_heads=1, head_dim=64, page_size=16, device="cpu"), **bad})


FAKE = 1 << 20   # an aligned address that no refused call touches


def cache_desc(**kw):
    d = dict(k=FAKE, v=FAKE, k_scale=None, v_scale=None, err=None, pages=4, kv_heads=2, page_size=16, head_dim=64,
             dtype=N.QV_BF16, bits=0)
    d.update(kw)
    return N.QvPagedCache(*d.values())


BAD_CACHES = [dict(k=None), dict(v=FAKE + 8), dict(pages=0), dict(kv_heads=0), dict(page_size=48), dict(head_dim=60),
              dict(head_dim=264), dict(dtype=3), dict(bits=4), dict(bits=8)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_native_refuses_bad_caches(bad):
    L, c = N.lib(), ctypes.byref(cache_desc(**bad))
    assert L.qv_paged_gather(c, 1, FAKE, 1, FAKE, FAKE, 1, FAKE, FAKE, None) == N.QV_EINVAL
    assert L.qv_paged_append(c, 1, 2, FAKE, 128, FAKE, 128, FAKE, 128, None, None, 0.0, None, 0, 0, 0, None, FAKE,
                             FAKE, None) == N.QV_EINVAL
    assert L.qv_paged_attention(c, 1, 2, FAKE, 1, FAKE, FAKE, 1, 1, 16, FAKE, 128, 1.0, 1, FAKE, None, 0,
                                None) == N.QV_EINVAL
    assert L.qv_paged_attention_workspace_bytes(c, 1, 2, 1, 1, 16) == 0


def test_native_refuses_bad_arguments():
    L, c = N.lib(), ctypes.byref(cache_desc())

    def attn(batch=1, heads=4, bt=FAKE, width=2, lens=FAKE, cuq=FAKE, total=1, mq=1, mkv=32, q=FAKE, qs=256, out=FAKE,
             ws=None, wsb=0, cache=c):
        return L.qv_paged_attention(cache, batch, heads, bt, width, lens, cuq, total, mq, mkv, q, qs, 1.0, 1, out, ws,
                                    wsb, None)
    for bad in (dict(batch=-1), dict(heads=3), dict(heads=34), dict(heads=0), dict(bt=None), dict(width=0),
                dict(lens=None), dict(cuq=None), dict(total=-1), dict(mq=-1), dict(mkv=-1), dict(mkv=33), dict(q=None),
                dict(q=FAKE + 2), dict(qs=255), dict(qs=260), dict(out=None), dict(out=FAKE + 8),
                dict(cache=ctypes.byref(cache_desc(head_dim=96)))):
        assert attn(**bad) == N.QV_EINVAL, bad
    assert attn(batch=0) == attn(total=0) == attn(mq=0) == N.QV_OK
    for scale in (0.0, -0.125, math.inf, math.nan):
        assert L.qv_paged_attention(c, 1, 4, FAKE, 2, FAKE, FAKE, 1, 1, 32, FAKE, 256, scale, 1, FAKE, None, 0,
                                    None) == N.QV_EINVAL
    assert L.qv_paged_gather(ctypes.byref(cache_desc(bits=8, k_scale=FAKE, v_scale=FAKE + 4)), 1, FAKE, 1, FAKE, FAKE,
                             1, FAKE, FAKE, None) == N.QV_EINVAL
    # a call that needs a workspace and gets none, or too little
    need = L.qv_paged_attention_workspace_bytes(c, 1, 4, 1, 1, 32768)
    assert need > 0
    assert attn(width=4096, mkv=32768) == N.QV_ESPACE
    assert attn(width=4096, mkv=32768, ws=FAKE, wsb=need - 1) == N.QV_ESPACE
    assert attn(width=4096, mkv=32768, ws=FAKE + 4, wsb=need) == N.QV_EINVAL

    def rope(T=1, Hq=2, H=1, D=64, dt=N.QV_BF16, q=FAKE, qs=128, k=FAKE, ks=64, qw=None, table=FAKE, mp=8, rot=64,
             pos=FAKE, qo=FAKE, ko=FAKE):
        return L.qv_qk_norm_rope(T, Hq, H, D, dt, q, qs, k, ks, qw, None, 0.0, table, mp, rot, 0, pos, qo, ko, None)
    for bad in (dict(T=-1), dict(Hq=0), dict(H=0), dict(D=4), dict(D=260), dict(D=60), dict(dt=7), dict(q=None),
                dict(q=FAKE + 4), dict(qs=100), dict(qs=132), dict(k=None), dict(ks=32), dict(qw=FAKE + 2), dict(mp=0),
                dict(rot=12), dict(rot=72), dict(rot=0), dict(pos=None), dict(qo=None), dict(ko=None),
                dict(ko=FAKE + 8), dict(table=FAKE + 4)):
        assert rope(**bad) == N.QV_EINVAL, bad
    assert rope(T=0) == N.QV_OK
    assert rope(qo=FAKE, ko=FAKE) == N.QV_EINVAL         # one buffer for both
    assert L.qv_paged_append(c, 1, 2, FAKE, 128, FAKE, 128, FAKE, 128, None, None, 0.0, None, 0, 0, 0, None, None,
                             FAKE, None) == N.QV_EINVAL
    assert L.qv_paged_append(c, 1, 2, FAKE, 128, FAKE, 128, None, 128, None, None, 0.0, None, 0, 0, 0, None, FAKE,
                             FAKE, None) == N.QV_EINVAL
    assert L.qv_paged_gather(c, 1, FAKE, 0, FAKE, FAKE, 1, FAKE, FAKE, None) == N.QV_EINVAL
    assert L.qv_paged_gather(c, 1, FAKE, 1, FAKE, FAKE, 1, FAKE, FAKE + 8, None) == N.QV_EINVAL
    assert L.qv_paged_gather(c, 0, None, 0, None, None, 0, None, None, None) == N.QV_OK


# ------------------------------------------------------------------ norm + rotation
@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,H,D,rot,norm,dt", [
    (1, 32, 8, 128, 128, False, BF16), (3, 5, 1, 64, 64, True, FP16), (7, 4, 4, 128, 64, True, BF16),
    (2, 3, 1, 128, 8, False, FP32), (5, 20, 4, 256, 256, True, FP32), (9, 2, 2, 80, 40, True, BF16),
    (4, 2, 2, 80, 80, False, FP16), (6, 7, 1, 96, 24, True, FP32), (257, 33, 3, 64, 32, True, BF16),
    (2, 1, 1, 8, 8, True, FP32), (3, 70, 2, 256, 200, False, BF16), (4, 4, 2, 64, 0, True, FP16)])
def test_qk_norm_rope(T, Hq, H, D, rot, norm, dt, interleaved):
    g = gen(T * 1000 + D + rot)
    qkv = rand(g, T, (Hq + 2 * H) * D).to(dt)
    q, k, _ = (x.view(T, -1, D) for x in qkv.split([Hq * D, H * D, H * D], 1))
    table = paged.rope_table(5000, rot, 10000.0) if rot else None
    pos = torch.randint(0, 5000, (T,), generator=g, device=DEV, dtype=torch.int32) if rot else None
    qw = rand(g, D).to(dt) if norm else None
    kw = rand(g, D).to(dt) if norm and T != 7 else None      # one case with a query weight alone
    before = qkv.clone()
    qo, ko = paged.qk_norm_rope(q, k, pos, table, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved)
    assert torch.equal(qkv, before) and qo.is_contiguous() and ko.is_contiguous()
    close_rows(qo, *ref_heads(q, qw, 1e-5, table, pos, interleaved), dt)
    close_rows(ko, *ref_heads(k, kw, 1e-5, table, pos, interleaved), dt)
    # in place, where the inputs are contiguous
    qc, kc = q.contiguous(), k.contiguous()
    a, b = paged.qk_norm_rope(qc, kc, pos, table, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved,
                              out=(qc, kc))
    assert a is qc and b is kc and torch.equal(a, qo) and torch.equal(b, ko)


@pytest.mark.gpu
def test_qk_norm_rope_edges():
    g = gen(3)
    table = paged.rope_table(16, 32)
    q, k = rand(g, 4, 2, 64).to(BF16), rand(g, 4, 1, 64).to(BF16)
    # a position outside the table shows as NaN in what turns, and nowhere else
    pos = torch.tensor([0, 16, -1, 15], dtype=torch.int32, device=DEV)
    qo, ko = paged.qk_norm_rope(q, k, pos, table)
    for x in (qo, ko):
        assert bool(x[1:3, :, :32].isnan().all()) and not bool(x[1:3, :, 32:].isnan().any())
        assert not bool(x[[0, 3]].isnan().any())
    # rows do not touch one another: a NaN row and an infinite one stay where they are; a zero row gives zero
    q[1, 0], q[2, 1], q[3] = math.nan, math.inf, 0
    w = torch.ones(64, dtype=BF16, device=DEV)
    qo, _ = paged.qk_norm_rope(q, k, torch.zeros(4, dtype=torch.int32, device=DEV), table, q_weight=w, k_weight=w)
    assert bool(qo[1, 0].isnan().all()) and not bool(qo[1, 1].isnan().any()) and not bool(qo[2, 0].isnan().any())
    assert bool((qo[3] == 0).all())
    e = torch.empty(0, 2, 64, dtype=BF16, device=DEV)
    qo, ko = paged.qk_norm_rope(e, e, pos[:0], table)
    assert qo.shape == (0, 2, 64) and ko.shape == (0, 2, 64)
    for bad in (dict(q=q.float()), dict(k=k[:3]), dict(positions=pos.long()), dict(positions=pos[:2]),
                dict(table=table.double()), dict(q=q.transpose(1, 2)), dict(q_weight=w.float()), dict(q_weight=w[:32]),
                dict(out=(q, q)), dict(positions=None), dict(table=paged.rope_table(16, 128))):
        with pytest.raises(N.QevictError):
            paged.qk_norm_rope(**{**dict(q=q, k=k, positions=pos, table=table), **bad})


# ------------------------------------------------------------------ append and read-back
@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens,Hq,H,D,page,rot,norm,interleaved,dt", [
    ([1], 32, 8, 128, 64, 128, False, False, BF16), ([5, 1, 33, 0, 16], 6, 2, 64, 16, 32, True, True, FP16),
    ([130, 7], 4, 4, 128, 128, 64, True, False, BF16), ([40, 3, 64], 20, 4, 256, 32, 256, False, True, BF16),
    ([17, 90], 3, 1, 80, 16, 40, True, False, FP32), ([1] * 70, 5, 5, 64, 32, 0, True, False, FP32)])
def test_append_and_gather(lens, Hq, H, D, page, rot, norm, interleaved, dt, q8):
    g = gen(sum(lens) + D)
    T = sum(lens)
    pool = Pool(g, lens, H, D, page, dt, q8)
    c = pool.cache
    for x in (c.k_pages, c.v_pages):
        x.fill_(5)
    qkv = rand(g, T, (Hq + 2 * H) * D, std=3.0).to(dt)
    q, k, v = (x.view(T, -1, D) for x in qkv.split([Hq * D, H * D, H * D], 1))
    table = paged.rope_table(300, rot) if rot else None
    pos = torch.randint(0, 300, (T,), generator=g, device=DEV, dtype=torch.int32) if rot else None
    w = rand(g, D).to(dt) if norm else None
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), pool.lens.long())
    at = torch.arange(T, device=DEV) - cu(lens).long()[seq]
    slots = c.slots(pool.bt, seq, at)
    skipped = torch.zeros(T, dtype=torch.bool, device=DEV)
    if T > 4:
        skipped[2] = True
        slots[2] = -1
    order = torch.randperm(T, generator=g, device=DEV)      # tokens of a call come in any order
    qo = c.append(q[order], k[order], v[order], slots[order], None if pos is None else pos[order], table, q_weight=w,
                  k_weight=w, interleaved=interleaved)
    assert c.read_error() == 0
    rq, mq = ref_heads(q, w, 1e-6, table, pos, interleaved)
    close_rows(qo, rq[order], mq[order], dt)
    # slots that were not written keep what they held
    used = torch.zeros(c.k_pages.shape[0] * page, dtype=torch.bool, device=DEV)
    used[slots[~skipped]] = True
    flat = c.k_pages.transpose(1, 2).reshape(-1, H, D), c.v_pages.transpose(1, 2).reshape(-1, H, D)
    for x in flat:
        assert bool((x[~used] == 5).all())
    total = T + 3
    out = tuple(torch.full((total, H, D), 9.0, dtype=dt, device=DEV) for _ in range(2))
    ko, vo = c.gather(pool.bt, pool.lens, cu(lens), total, out=out)
    assert c.read_error() == 0 and bool((ko[T:] == 9).all()) and bool((vo[T:] == 9).all())
    rk, mk = ref_heads(k, w, 1e-6, table, pos, interleaved)
    for got, ref, mag in ((ko, rk, mk), (vo, v.double(), v.double().abs())):
        got, ref, mag = got[:T][~skipped], ref[~skipped], mag[~skipped]
        if not q8:
            close_rows(got, ref, mag, dt)
        else:
            # half a step of max|row| / 127 (the step and the ratio in fp32), then the type's rounding
            step = ref.abs().amax(-1, keepdim=True) / 127
            bound = step * (0.5 + 127 * 2.0 ** -18) + got.double().abs() * half(dt) * 1.001 + mag * 2.0 ** -18 + TINY[dt]
            assert bool(((got.double() - ref).abs() <= bound).all())
    if q8:   # the stored codes and scales are what the read-back returns, exactly
        kf, vf = (x.transpose(1, 2).reshape(-1, H, D)[slots[~skipped]] for x in (c.k_pages, c.v_pages))
        s = c.k_scale.transpose(1, 2).reshape(-1, H)[slots[~skipped]]
        assert torch.equal((kf.float() * s[..., None]).to(dt), ko[:T][~skipped])
        assert int(kf.abs().max()) == 127


@pytest.mark.gpu
def test_append_edges():
    g = gen(8)
    c = paged.PagedKVCache(3, 1, 64, 16, BF16, bits=8)
    q, k, v = (rand(g, 6, 1, 64).to(BF16) for _ in range(3))
    k[1], k[2], k[3], k[4] = 0, math.nan, math.inf, 1e-38     # a zero row, two that are not finite, a tiny one
    k[2, 0, 1:], k[3, 0, 1:] = 1, 1
    c.append(q, k, v, torch.arange(6, device=DEV))
    bt = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    n = torch.tensor([6], dtype=torch.int32, device=DEV)
    ko, vo = c.gather(bt, n, cu([6]), 6)
    assert bool((ko[1] == 0).all()) and bool(ko[2].isnan().all()) and bool(ko[3].isnan().all())
    assert bool(((ko[4].double() - k[4].double()).abs() <= 1e-38 * (0.5 / 127 + half(BF16)) * 1.01).all())
    assert not bool(ko[[0, 1, 4, 5]].isnan().any()) and not bool(vo.isnan().any()) and c.read_error() == 0
    # a slot behind the pool, a position outside the table
    c.append(q[:1], k[:1], v[:1], torch.tensor([48], device=DEV))
    assert c.read_error() == N.QV_DERR_CAPACITY
    c.err.zero_()
    c.append(q[:1], k[:1], v[:1], torch.tensor([7], device=DEV), torch.tensor([9], dtype=torch.int32, device=DEV),
             paged.rope_table(9, 64))
    assert c.read_error() == N.QV_DERR_TABLE
    c.err.zero_()
    # read-back: a page id outside the pool, a length above the block table
    out = tuple(torch.full((20, 1, 64), 4.0, dtype=BF16, device=DEV) for _ in range(2))
    for page in (-1, 3, 2 ** 31 - 1):
        c.gather(torch.tensor([[page]], dtype=torch.int32, device=DEV), n, cu([6]), 20, out=out)
        assert c.read_error() == N.QV_DERR_TABLE and bool((out[0] == 4).all())
        c.err.zero_()
    c.gather(bt, torch.tensor([20], dtype=torch.int32, device=DEV), cu([20]), 20, out=out)
    assert c.read_error() == N.QV_DERR_CAPACITY and bool((out[0][16:] == 4).all()) and not bool((out[0][:2] == 4).all())
    e = torch.empty(0, 1, 64, dtype=BF16, device=DEV)
    assert c.append(e, e, e, torch.empty(0, dtype=torch.int64, device=DEV)).shape == (0, 1, 64)
    with pytest.raises(N.QevictError):
        c.append(q, k, v, torch.arange(6, device=DEV, dtype=torch.int32))
    with pytest.raises(N.QevictError):
        c.append(q, k[:, :, :32], v, torch.arange(6, device=DEV))
    with pytest.raises(N.QevictError):
        c.append(q, k.expand(6, 2, 64), v, torch.arange(6, device=DEV))
    with pytest.raises(N.QevictError):
        paged.paged_gather(c.k_pages, c.v_pages, bt, n, cu([6]), 6, dtype=BF16)       # INT8 pages without scales


# ------------------------------------------------------------------ attention
SHAPES = [   # q_lens, kv_lens, Hq, H, D, page
    ([1], [1], 4, 1, 64, 16),
    ([1], [2000], 32, 8, 128, 64),                                     # one decode step, keys split over blocks
    ([1, 1, 1, 0, 1, 1], [63, 64, 65, 12, 1, 700], 8, 2, 128, 32),     # decode of a ragged batch
    ([1, 1], [5000, 3], 16, 1, 64, 128),
    ([2, 3, 1], [300, 3, 129], 5, 1, 128, 16),                         # a few tokens each
    ([16, 1, 4], [1000, 1, 90], 1, 1, 64, 16),
    ([40, 0, 7], [40, 5, 900], 12, 4, 128, 64),
    ([130], [130], 4, 4, 64, 32),                                      # a whole prompt
    ([257, 64, 1, 33], [1025, 64, 500, 34], 8, 2, 128, 16),            # chunks and single tokens in one batch
    ([100], [3000], 15, 5, 64, 128),                                   # few tiles over long keys
    ([5, 64], [0, 20], 8, 1, 64, 16),                                  # more new tokens than cached: rows that see nothing
    ([300, 200], [300, 1999], 3, 1, 128, 64),
    ([513], [640], 16, 8, 128, 128),
    ([9, 70], [200, 1500], 16, 1, 128, 32),                            # groups that do not divide a tile's rows
    ([33, 2], [33, 700], 14, 2, 64, 16),
    ([60], [260], 11, 1, 128, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,q8", [(BF16, False), (FP16, False), (FP32, False), (BF16, True), (FP16, True), (FP32, True)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(shape, dt, q8):
    q_lens, kv_lens, Hq, H, D, page = SHAPES[shape]
    g = gen(100 + shape)
    check_attention(g, q_lens, kv_lens, Hq, H, D, page, dt, q8, max_q=max(q_lens), max_kv=max(kv_lens))
    if shape in (2, 6, 8):
        # every key seen by every row; a scale of its own; bounds left to their defaults
        check_attention(g, q_lens, kv_lens, Hq, H, D, page, dt, q8, causal=False, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,q8", [(BF16, False), (FP16, True), (FP32, False)])
@pytest.mark.parametrize("most", [1, 7])
def test_attention_many_sequences(most, dt, q8):
    """More sequences than a block has threads, some with nothing new, lengths over two orders of magnitude."""
    r = torch.Generator().manual_seed(most)
    B = 700
    q_lens = torch.randint(0, most + 1, (B,), generator=r)
    kv_lens = torch.maximum(q_lens, (2.0 ** (9 * torch.rand(B, generator=r))).long())
    q_lens[5], kv_lens[5] = most, 900
    check_attention(gen(41), q_lens.tolist(), kv_lens.tolist(), 4, 1, 64, 16, dt, q8, max_q=most, max_kv=900)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,q8", [(BF16, False), (FP16, False), (BF16, True), (FP16, True), (FP32, False)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [900]), ([300], [900])])
def test_attention_large_and_growing_logits(q_lens, kv_lens, dt, q8):
    g = gen(7)
    # logits of up to +-200: the maximum moves by far more than the exponent's range from tile to tile
    check_attention(g, q_lens, kv_lens, 8, 2, 128, 32, dt, q8, std=4.0, qstd=6.0)
    # values far from 1
    check_attention(g, q_lens, kv_lens, 8, 2, 64, 32, dt, q8, std=3e-3)
    if dt != FP16:
        check_attention(g, q_lens, kv_lens, 8, 2, 64, 32, dt, q8, std=1e4, qstd=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,q8", [(BF16, False), (FP16, False), (FP32, False), (BF16, True), (FP16, True), (FP32, True)])
@pytest.mark.parametrize("n", [1, 150])
def test_attention_rising_and_falling_logits(n, dt, q8):
    """Logits that climb by several hundred along the keys, so that every tile's maximum is far above the last
    one's, and the same keys falling."""
    L, D, page = 1200, 128, 64
    g = gen(17)
    pool = Pool(g, [L, L], 1, D, page, dt, q8)
    c = pool.cache
    u = torch.nn.functional.normalize(rand(g, D), dim=-1)
    for b in range(2):
        pos = torch.arange(L, device=DEV)
        size = (pos if b == 0 else L - 1 - pos).float() / L * 40
        rows = (size[:, None, None] * u + 0.05 * rand(g, L, 1, D))
        sl = c.slots(pool.bt, torch.full_like(pos, b), pos)
        if q8:
            s = rows.abs().amax(-1) / 127
            code = (rows / s[..., None]).round()
            c.k_pages[sl // page, :, sl % page], c.k_scale[sl // page, :, sl % page] = code.to(torch.int8), s
            pool.ks[b] = code.double() * s.double()[..., None]
        else:
            c.k_pages[sl // page, :, sl % page] = rows.to(dt)
            pool.ks[b] = rows.to(dt).double()
    q = (u * 120 + 0.05 * rand(g, 2 * n, 4, D)).to(dt)      # logits up to 40 * 120 / sqrt(128) = 424
    out = c.attend(q, pool.bt, pool.lens, cu([n, n]), max_q=n)
    assert c.read_error() == 0
    for b in range(2):
        o, mag, big = ref_attention(q[b * n:(b + 1) * n], pool.ks[b], pool.vs[b])
        bound = attention_bound(o, mag, big, L, D, dt, float(pool.vs[b].abs().max()))
        assert bool(((out[b * n:(b + 1) * n].double() - o).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("n", [1, 150])
def test_attention_int8_zero_and_uneven_rows(n, dt):
    """INT8 rows of zeros (a scale of 0) in K and in V, and value scales over ten orders of magnitude."""
    L, D, page = 400, 64, 32
    g = gen(19)
    pool = Pool(g, [L], 1, D, page, dt, True)
    c = pool.cache
    pos = torch.arange(L, device=DEV)
    sl = c.slots(pool.bt, torch.zeros_like(pos), pos)
    pg, off = sl // page, sl % page
    for x, sc, keep, every in ((c.k_pages, c.k_scale, pool.ks, 7), (c.v_pages, c.v_scale, pool.vs, 5)):
        zero = pos % every == 3
        factor = torch.ones(L, device=DEV) if x is c.k_pages else 10.0 ** (-10 * torch.rand(L, generator=g, device=DEV))
        x[pg[zero], :, off[zero]] = 0
        s = torch.where(zero, 0.0, sc[pg, 0, off] * factor)
        sc[pg, 0, off] = s
        keep[0] = x[pg, :, off].double() * s.double()[:, None, None]
    q = rand(g, n, 4, D).to(dt)
    out = c.attend(q, pool.bt, pool.lens, cu([n]), max_q=n)
    o, mag, big = ref_attention(q, pool.ks[0], pool.vs[0])
    # P carries the value scale: what rounds to 0 in fp16 is half a step of 2^-24 of the largest P times its scale
    bound = attention_bound(o, mag, big, L, D, dt, float(pool.vs[0].abs().max()))
    assert bool(((out.double() - o).abs() <= bound).all())
    # every value row zero: zero, whatever the logits
    c.v_scale[pg, 0, off] = 0
    c.v_pages[pg, :, off] = 0
    assert bool((c.attend(q, pool.bt, pool.lens, cu([n]), max_q=n) == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt,size", [(BF16, 2.0 ** 40), (BF16, 2.0 ** -40), (FP16, 2.0 ** 13), (FP16, 2.0 ** -14),
                                     (FP32, 2.0 ** 40), (FP32, 2.0 ** -40)])
@pytest.mark.parametrize("n", [1, 150])
def test_attention_int8_zero_rows_beside_large_and_small_values(n, dt, size):
    """INT8 value rows of zeros beside rows of any size: their probabilities count in the sum all the same."""
    L, D, page = 400, 64, 32
    g = gen(29)
    pool = Pool(g, [L], 1, D, page, dt, True)
    c = pool.cache
    pos = torch.arange(L, device=DEV)
    sl = c.slots(pool.bt, torch.zeros_like(pos), pos)
    pg, off = sl // page, sl % page
    zero = pos % 3 == 1
    c.v_pages[pg[zero], :, off[zero]] = 0
    c.v_scale[pg, 0, off] = torch.where(zero, 0.0, c.v_scale[pg, 0, off] * size)
    pool.vs[0] = c.v_pages[pg, :, off].double() * c.v_scale[pg, :, off].double()[..., None]
    q = rand(g, n, 4, D).to(dt)
    out = c.attend(q, pool.bt, pool.lens, cu([n]), max_q=n)
    o, mag, big = ref_attention(q, pool.ks[0], pool.vs[0])
    bound = attention_bound(o, mag, big, L, D, dt, float(pool.vs[0].abs().max()))
    assert bool(((out.double() - o).abs() <= bound).all()), float(((out.double() - o).abs() / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
def test_attention_rows_that_are_not_finite(n, dt, q8):
    """A NaN key shows in every row that sees it, a NaN query row in itself alone; other sequences and heads keep
    their bits."""
    g = gen(23)
    H, G, D, page, L = 2, 4, 128, 64, 300
    pool = Pool(g, [L, L], H, D, page, dt, q8)
    c = pool.cache
    q = rand(g, 2 * n, H * G, D).to(dt)
    kw = dict(max_q=n, max_kv=L)
    want = c.attend(q, pool.bt, pool.lens, cu([n, n]), **kw)
    bad = q.clone()
    bad[n, 1, 5] = math.nan
    got = c.attend(bad, pool.bt, pool.lens, cu([n, n]), **kw)
    assert bool(got[n, 1].isnan().all())
    keep = torch.ones(2 * n, H * G, dtype=torch.bool, device=DEV)
    keep[n, 1] = False
    assert torch.equal(got[keep], want[keep])
    # the first key of sequence 1, head 0
    page0 = int(pool.bt[1, 0])
    if q8:
        c.k_scale[page0, 0, 0] = math.nan
    else:
        c.k_pages[page0, 0, 0, 3] = math.nan
    got = c.attend(q, pool.bt, pool.lens, cu([n, n]), **kw)
    assert bool(got[n:, :G].isnan().all())
    assert torch.equal(got[:n], want[:n]) and torch.equal(got[n:, G:], want[n:, G:])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 200])
def test_attention_bad_tables_stay_inside(n):
    g = gen(11)
    pool, q, out = check_attention(g, [n, n], [400, 300], 8, 2, 128, 64, BF16, False)
    c, good = pool.cache, out.clone()
    bt = pool.bt.clone()
    for bad in (-1, c.k_pages.shape[0], 2 ** 31 - 1):
        bt[1, 2] = bad
        c.k_pages.nan_to_num_(0.0), c.v_pages.nan_to_num_(0.0)
        got = c.attend(q[: 2 * n], bt, pool.lens, cu([n, n]))
        assert c.read_error() == N.QV_DERR_TABLE
        assert torch.equal(got[:n], good[:n])               # the other sequence is right
        c.err.zero_()
    # a length above max_kv is cut to it (and what it then reaches of the shorter sequence's table lies outside the
    # pool); rows past max_q are left as they were
    out = torch.full((2 * n, 8, 128), 3.0, dtype=BF16, device=DEV)
    c.attend(q[: 2 * n], pool.bt, pool.lens + 100000, cu([n, n]), out=out)
    assert c.read_error() == N.QV_DERR_CAPACITY | N.QV_DERR_TABLE
    c.err.zero_()
    if n > 1:
        out.fill_(3.0)
        c.attend(q[: 2 * n], pool.bt, pool.lens, cu([n, n]), out=out, max_q=n - 1)
        assert c.read_error() == N.QV_DERR_CAPACITY and bool((out[n - 1] == 3).all()) and bool((out[-1] == 3).all())
        assert torch.equal(out[: n - 1], good[: n - 1])
        c.err.zero_()
    # cumulative lengths outside the rows, negative lengths
    c.attend(q[: 2 * n], pool.bt, pool.lens, torch.tensor([-5, n, 10 ** 6], dtype=torch.int32, device=DEV))
    c.attend(q[: 2 * n], pool.bt, -pool.lens, cu([n, n]))
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_attention_refusals():
    g = gen(12)
    pool = Pool(g, [20], 2, 64, 16, BF16, False)
    q = rand(g, 3, 4, 64).to(BF16)
    ok = dict(q=q, block_table=pool.bt, kv_lens=pool.lens, cu_q=cu([3]))
    pool.cache.attend(**ok)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.cpu()), dict(cu_q=cu([3]).long()),
                dict(cu_q=cu([3])[:1]), dict(kv_lens=pool.lens.repeat(2)), dict(block_table=pool.bt.long()),
                dict(block_table=pool.bt[0]), dict(max_kv=33), dict(max_kv=-1), dict(max_q=-1),
                dict(out=torch.empty(3, 4, 32, dtype=BF16, device=DEV)), dict(q=q.transpose(0, 1)), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)):
        with pytest.raises(N.QevictError):
            pool.cache.attend(**{**ok, **bad})
    two = torch.empty(20, 2, 64, dtype=BF16, device=DEV)
    with pytest.raises(N.QevictError):
        pool.cache.gather(pool.bt, pool.lens, cu([20]), 20, out=(two, two))
    with pytest.raises(N.QevictError):
        paged.qk_norm_rope(two, two.clone(), out=(two, two))
    small = paged.PagedKVCache(2, 2, 96, 16, BF16)
    with pytest.raises(N.QevictError):
        small.attend(rand(g, 3, 4, 96).to(BF16), pool.bt, pool.lens, cu([3]))
    e = torch.empty(0, 4, 64, dtype=BF16, device=DEV)
    assert pool.cache.attend(e, pool.bt, pool.lens, cu([0])).shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,q8", [(BF16, False), (BF16, True), (FP32, False)])
def test_attention_offsets_past_32_bits(dt, q8):
    """Pages whose elements lie behind 2^31 elements (and, in 16 bits, 2^32 bytes) of the pool."""
    H, D, page = 8, 128, 128
    per = H * page * D
    P = 2 ** 31 // per + 4
    c = paged.PagedKVCache(P, H, D, page, dt, bits=8 if q8 else None)
    g = gen(5)
    bt = torch.tensor([[P - 1, P - 3], [0, P - 2]], dtype=torch.int32, device=DEV)
    lens = [200, 256]
    T = sum(lens)
    q, k, v = (rand(g, T, n, D).to(dt) for n in (2 * H, H, H))
    seq = torch.repeat_interleave(torch.arange(2, device=DEV), torch.tensor(lens, device=DEV))
    pos = torch.arange(T, device=DEV) - cu(lens).long()[seq]
    c.append(q, k, v, c.slots(bt, seq, pos))
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ko, vo = c.gather(bt, n, cu(lens), T)
    if not q8:
        assert torch.equal(ko, k) and torch.equal(vo, v)
    for ql in ([1, 1], [200, 150]):
        rows = torch.cat([q[:ql[0]], q[200:200 + ql[1]]])
        out = c.attend(rows, bt, n, cu(ql))
        at = 0
        for b in range(2):
            lo, hi = (0, 200) if b == 0 else (200, 456)
            kb, vb = ko[lo:hi].double(), vo[lo:hi].double()
            o, mag, big = ref_attention(rows[at:at + ql[b]], kb, vb)
            # INT8: the read-back used here is itself rounded to the type (K: an exponent's error of |q||k| half)
            more = mag * half(dt) * (1 + 2 * big) if q8 else 0.0
            bound = attention_bound(o, mag, big, lens[b], D, dt, float(vb.abs().max())) + more
            assert bool(((out[at:at + ql[b]].double() - o).abs() <= bound).all())
            at += ql[b]
    assert c.read_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [3000, 10, 700]), ([70, 1, 200], [2500, 900, 200])])
def test_attention_graph_streams_and_repeats(q_lens, kv_lens, q8):
    """The same bits eagerly, twice, in two captured graphs replayed at once, and on another stream; a replay with
    other lengths below the captured bounds."""
    g = gen(21)
    pool, q, out = check_attention(g, q_lens, kv_lens, 8, 2, 128, 64, BF16, q8)
    c, cq, T = pool.cache, cu(q_lens), sum(q_lens)
    kw = dict(max_q=max(q_lens), max_kv=max(kv_lens))
    want = c.attend(q[:T], pool.bt, pool.lens, cq, **kw)
    assert torch.equal(c.attend(q[:T], pool.bt, pool.lens, cq, **kw), want)
    lens = pool.lens.clone()
    graphs, outs = [], [torch.zeros_like(want), torch.zeros_like(want)]
    for o in outs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            c.attend(q[:T], pool.bt, lens, cq, out=o, **kw)
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    lens.copy_(torch.clamp(pool.lens // 2, min=max(0, 1)))
    lens[0] = pool.lens[0] - 1000
    graphs[0].replay()
    assert torch.equal(outs[0], c.attend(q[:T], pool.bt, lens, cq, **kw)) and not torch.equal(outs[0], want)
    with torch.cuda.stream(streams[0]):
        streams[0].wait_stream(torch.cuda.current_stream())
        again = c.attend(q[:T], pool.bt, pool.lens, cq, **kw)
    torch.cuda.synchronize()
    assert torch.equal(again, want) and c.read_error() == 0


# ------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_chunked_prompt_then_decode(bits):
    """Two prompts served as a program would: ragged chunks rotated, written and attended together, then single
    tokens, from packed projections; each step against 64 bits on what the pool holds; at the end the pool is
    read back and the framework's own prompt attention on it gives the same prompt outputs."""
    from qevict_b200.model import prefill_attention
    Hq, H, D, page, dt = 8, 2, 128, 32, BF16
    g = gen(33)
    lens, steps = [200, 131], 4
    qkv = [rand(g, n + steps, Hq + 2 * H, D).to(dt) for n in lens]
    w = (1 + rand(g, D, std=0.1)).to(dt)
    table = paged.rope_table(512, D, 500000.0, dict(type="llama3", factor=8.0, low_freq_factor=1.0,
                                                    high_freq_factor=4.0, original_max_position=128))
    c = paged.PagedKVCache(16, H, D, page, dt, bits=bits)
    bt = torch.randperm(16, generator=g, device=DEV).int()[:14].view(2, 7).contiguous()
    done, outs, rot = [0, 0], [[], []], [[], []]
    plan = [(64, 50), (100, 1), (36, 80)] + [(1, 1)] * steps
    for take in plan:
        rows = torch.cat([qkv[b][done[b]:done[b] + take[b]] for b in range(2)])
        seq = torch.repeat_interleave(torch.arange(2, device=DEV), torch.tensor(take, device=DEV))
        pos = torch.cat([torch.arange(done[b], done[b] + take[b], device=DEV) for b in range(2)])
        q, k, v = rows[:, :Hq], rows[:, Hq:Hq + H], rows[:, Hq + H:]
        qr = c.append(q, k, v, c.slots(bt, seq, pos), pos.int(), table, q_weight=w, k_weight=w)
        done = [done[b] + take[b] for b in range(2)]
        n = torch.tensor(done, dtype=torch.int32, device=DEV)
        o = c.attend(qr, bt, n, cu(take), max_q=max(take), max_kv=max(done))
        kk, vv = c.gather(bt, n, cu(done), sum(done))
        at = 0
        for b in range(2):
            lo = 0 if b == 0 else done[0]
            kb, vb = kk[lo:lo + done[b]].double(), vv[lo:lo + done[b]].double()
            ref, mag, big = ref_attention(qr[at:at + take[b]], kb, vb)
            more = mag * half(dt) * (1 + 2 * big) if bits == 8 else 0.0
            bound = attention_bound(ref, mag, big, done[b], D, dt, float(vb.abs().max())) + more
            assert bool(((o[at:at + take[b]].double() - ref).abs() <= bound).all())
            outs[b].append(o[at:at + take[b]])
            rot[b].append(qr[at:at + take[b]])
            at += take[b]
    assert c.read_error() == 0
    # the rotated keys in the pool are the formula's
    if bits == 16:
        for b in range(2):
            lo = 0 if b == 0 else done[0]
            close_rows(kk[lo:lo + done[b]], *ref_heads(qkv[b][:, Hq:Hq + H], w, 1e-6, table,
                                                       torch.arange(done[b], device=DEV), False), dt)
    n0 = lens[0]
    po, _ = prefill_attention(torch.cat(rot[0])[None, :n0].contiguous(), kk[None, :n0].contiguous(),
                              vv[None, :n0].contiguous())
    mine = torch.cat(outs[0])[:n0].double()
    # the prompt lane rounds each logit twice to bf16 (the reference's arithmetic): an exponent's error of a logit's
    # own size, up to |q||k| D^-1/2, and its probabilities once more
    kb, vb = kk[:n0].double(), vv[:n0].double()
    ref, mag, big = ref_attention(torch.cat(rot[0])[:n0], kb, vb)
    bound = attention_bound(ref, mag, big, n0, D, dt, float(vb.abs().max())) * 2 + mag * half(dt) * (2 * 2 * big + 2)
    assert bool(((po[0].double() - mine).abs() <= bound).all())


def test_native_refuses_lengths_past_2_30():
    L, c = N.lib(), ctypes.byref(cache_desc())
    big = (1 << 30) + 1
    assert L.qv_paged_attention_workspace_bytes(c, 1, 2, 1, 1, big) == 0
    assert L.qv_paged_attention(c, 1, 2, FAKE, 1 << 27, FAKE, FAKE, 1, 1, big, FAKE, 128, 1.0, 1, FAKE, FAKE, 1 << 40,
                                None) == N.QV_EINVAL


@pytest.mark.gpu
def test_numbers_past_32_bits_are_not_cut():
    g = gen(41)
    pool = Pool(g, [20], 2, 64, 16, BF16, False)
    q = rand(g, 3, 4, 64).to(BF16)
    want = pool.cache.attend(q, pool.bt, pool.lens, cu([3]))
    assert torch.equal(pool.cache.attend(q, pool.bt, pool.lens, cu([3]), max_q=2 ** 32), want)
    with pytest.raises(N.QevictError):
        pool.cache.attend(q, pool.bt, pool.lens, cu([3]), max_kv=2 ** 32 + 20)
    two = torch.empty(20, 2, 64, dtype=BF16, device=DEV)
    with pytest.raises(N.QevictError):
        pool.cache.gather(pool.bt, pool.lens, cu([20]), 2 ** 32 + 20)
    with pytest.raises(N.QevictError):
        pool.cache.gather(pool.bt, pool.lens, cu([20]), 2 ** 32 + 20, out=(two, two.clone()))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,q8", [(BF16, False), (BF16, True), (FP16, False), (FP32, False)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [700, 20]), ([1], [5000]), ([200, 1, 40], [900, 30, 40])])
def test_outputs_in_place_and_overlapping(q_lens, kv_lens, dt, q8):
    """An output in its input's place gives the same bits; any other overlap is refused."""
    g = gen(43)
    pool = Pool(g, kv_lens, 2, 128, 32, dt, q8)
    c, n = pool.cache, sum(q_lens)
    buf = rand(g, 3 * n, 8, 128).to(dt)
    q = buf[:n]
    kw = dict(block_table=pool.bt, kv_lens=pool.lens, cu_q=cu(q_lens), max_q=max(q_lens))
    want = c.attend(q, **kw)
    mine = q.clone()
    assert c.attend(mine, out=mine, **kw) is mine and torch.equal(mine, want)
    with pytest.raises(N.QevictError):
        c.attend(buf.view(-1, 128)[4:4 + 8 * n].view(n, 8, 128), out=q, **kw)
    with pytest.raises(N.QevictError):       # a strided view of the rows it would write over
        c.attend(buf[::2][:n], out=q, **kw) if n > 1 else c.attend(q, out=q[:, :4], **kw)
    k, v = buf[n:2 * n], buf[2 * n:]
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    table = paged.rope_table(n, 128)
    want = paged.qk_norm_rope(q, k, pos, table)
    for out in ((k, q), (q, q), (v, v), (q, buf.view(-1, 128)[4:4 + 8 * n].view(n, 8, 128))):
        with pytest.raises(N.QevictError):
            paged.qk_norm_rope(q, k, pos, table, out=out)
    a, b = q.clone(), k.clone()
    paged.qk_norm_rope(a, b, pos, table, out=(a, b))
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    slots = torch.full((n,), -1, dtype=torch.int64, device=DEV)
    kk = torch.zeros(n, 2, 128, dtype=dt, device=DEV)
    vv = torch.zeros(8 * n, 128, dtype=dt, device=DEV)
    with pytest.raises(N.QevictError):
        c.append(q, kk, vv.view(4 * n, 2, 128)[:n], slots, pos, table, q_out=vv.view(n, 8, 128))
    a = q.clone()
    assert torch.equal(c.append(a, kk, kk, slots, pos, table, q_out=a), want[0])
    with pytest.raises(N.QevictError):
        c.gather(pool.bt, pool.lens, cu(kv_lens), n, out=(vv[:2 * n].view(n, 2, 128), vv[1:1 + 2 * n].view(n, 2, 128)))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,q8", [(BF16, False), (FP16, False), (BF16, True), (FP16, True)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,G,causal", [(20, 4, True), (40, 4, True), (33, 1, False), (129, 1, True), (8, 8, True)])
def test_attention_moving_reference_of_one_and_two_row_tiles(n, G, causal, D, dt, q8):
    """Logits that climb by 10 (base 2) or more from key tile to key tile, for one row tile alone, two of unlike key
    counts, and a second one of a single row; and a chunk longer than its sequence, whose first rows see nothing."""
    L, page = 1500, 32
    g = gen(47)
    lens = [L, L - 700, n // 2]
    pool = Pool(g, lens, 1, D, page, dt, q8)
    c = pool.cache
    u = torch.nn.functional.normalize(rand(g, D), dim=-1)
    for b, m in enumerate(lens):
        pos = torch.arange(m, device=DEV)
        rows = (pos.float() / L * 20)[:, None, None] * u + 0.05 * rand(g, m, 1, D)
        sl = c.slots(pool.bt, torch.full_like(pos, b), pos)
        if q8:
            s = rows.abs().amax(-1) / 127
            code = (rows / s[..., None]).round()
            c.k_pages[sl // page, :, sl % page], c.k_scale[sl // page, :, sl % page] = code.to(torch.int8), s
            pool.ks[b] = code.double() * s.double()[..., None]
        else:
            c.k_pages[sl // page, :, sl % page] = rows.to(dt)
            pool.ks[b] = rows.to(dt).double()
    q = (u * 120 + 0.05 * rand(g, 3 * n, G, D)).to(dt)
    out = c.attend(q, pool.bt, pool.lens, cu([n, n, n]), max_q=n, causal=causal)
    assert c.read_error() == 0
    for b, m in enumerate(lens):
        o, mag, big = ref_attention(q[b * n:(b + 1) * n], pool.ks[b], pool.vs[b], causal)
        bound = attention_bound(o, mag, big, m, D, dt, float(pool.vs[b].abs().max()))
        assert bool(((out[b * n:(b + 1) * n].double() - o).abs() <= bound).all()), b


# ------------------------------------------------------------------ buffers that share memory
def at(n):
    """The n-th of a row of addresses a GB apart, which no refused call touches."""
    return FAKE + (n << 30)


@pytest.mark.parametrize("q8", [False, True])
def test_native_gather_refuses_outputs_on_what_it_reads(q8):
    L = N.lib()
    c = cache_desc(k=at(1), v=at(2), err=at(9), pages=4, kv_heads=1, page_size=16, head_dim=64, bits=8 if q8 else 0,
                   k_scale=at(3) if q8 else None, v_scale=at(4) if q8 else None)

    def gather(ko, vo, bt=at(5), lens=at(6), cu_kv=at(7)):
        return L.qv_paged_gather(ctypes.byref(c), 2, bt, 2, lens, cu_kv, 20, ko, vo, None)
    pool, rows = 4 * 16 * 64 * (1 if q8 else 2), 20 * 64 * 2
    for base, size in [(at(1), pool), (at(2), pool), (at(5), 16), (at(6), 8), (at(7), 12), (at(9), 4)] + (
            [(at(3), 256), (at(4), 256)] if q8 else []):
        # at its first byte, at its last 16, and ending on its first 16
        for o in (base, base + (size - 1) // 16 * 16, base - rows + 16):
            assert gather(o, at(20)) == N.QV_EINVAL
            assert gather(at(20), o) == N.QV_EINVAL
    for o in (at(20), at(20) + rows - 16, at(20) - rows + 16):
        assert gather(at(20), o) == N.QV_EINVAL


def test_an_output_is_only_in_place_where_the_call_says_so():
    """The pool's memory as a row list (one KV head), from its first byte or elsewhere."""
    pool = torch.zeros(4, 1, 16, 64)
    out = pool.view(-1, 1, 64)[:20]
    for o in (out, pool.view(-1, 1, 64)[1:21], pool.view(-1, 1, 64)[44:]):
        with pytest.raises(N.QevictError):
            paged._apart("out", o, pool, torch.zeros(20, 1, 64))
    q = torch.zeros(20, 1, 64)
    paged._apart("out", q, pool, inplace=q)
    with pytest.raises(N.QevictError):
        paged._apart("out", q, q, inplace=q)
    with pytest.raises(N.QevictError):
        paged._apart("out", q[:10], pool, inplace=q[::2])
    paged._apart("out", q[10:], q[:10], inplace=pool)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
def test_gather_refuses_outputs_on_its_pool(q8):
    g = gen(53)
    pool = Pool(g, [20, 9], 1, 64, 16, BF16, q8)
    c, free = pool.cache, torch.empty(29, 1, 64, dtype=BF16, device=DEV)
    before = [x.clone() for x in (c.k_pages, c.v_pages)]
    for x in (c.k_pages, c.v_pages) + ((c.k_scale, c.v_scale) if q8 else ()):
        rows = x.view(-1).view(BF16)[: x.numel() * x.element_size() // 128 * 64].view(-1, 1, 64)
        for n in (29, 1):
            o = rows[:n] if len(rows) >= n else rows
            lens, total = torch.full_like(pool.lens, len(o) // 2), len(o)
            for out in ((o, free[:total]), (free[:total], o)):
                with pytest.raises(N.QevictError):
                    c.gather(pool.bt, lens, cu([total // 2, total // 2]), total, out=out)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, (c.k_pages, c.v_pages)))


def around(base, size, rows):
    """Addresses of `rows` bytes that meet [base, base + size) at its first byte, its last 16, and from below."""
    return [base, base + (size - 1) // 16 * 16, base - rows + 16]


@pytest.mark.parametrize("dt", [N.QV_F32, N.QV_BF16])
@pytest.mark.parametrize("q8", [False, True])
def test_native_attention_refuses_written_buffers_on_others(q8, dt):
    L, e = N.lib(), 4 if dt == N.QV_F32 else 2
    c = cache_desc(k=at(1), v=at(2), err=at(9), pages=4, kv_heads=2, page_size=16, head_dim=64, dtype=dt,
                   bits=8 if q8 else 0, k_scale=at(3) if q8 else None, v_scale=at(4) if q8 else None)
    cp, T, row = ctypes.byref(c), 3, 4 * 64
    need = L.qv_paged_attention_workspace_bytes(cp, 2, 4, T, 1, 32 * 1024)

    def attn(out=at(20), ws=at(30), qs=row):
        return L.qv_paged_attention(cp, 2, 4, at(5), 2048, at(6), at(7), T, 1, 32 * 1024, at(8), qs, 1.0, 1, out, ws,
                                    need, None)
    pool = 4 * 2 * 16 * 64 * (1 if q8 else e)
    reads = [(at(1), pool), (at(2), pool), (at(5), 2 * 2048 * 4), (at(6), 8), (at(7), 12), (at(9), 4)] + (
        [(at(3), 512), (at(4), 512)] if q8 else [])
    assert need > 0
    for base, size in reads:
        for o in around(base, size, T * row * e):
            assert attn(out=o) == N.QV_EINVAL
        for o in around(base, size, need):
            assert attn(ws=o) == N.QV_EINVAL
    for o in around(at(8), T * row * e, need):
        assert attn(ws=o) == N.QV_EINVAL
    assert attn(ws=at(20)) == attn(ws=at(20) + T * row * e - 16) == N.QV_EINVAL
    # queries: in their place only where they are contiguous, not shifted
    assert attn(out=at(8) + 16) == attn(out=at(8) - 16) == attn(out=at(8), qs=2 * row) == N.QV_EINVAL


@pytest.mark.parametrize("q8", [False, True])
def test_native_head_kernels_refuse_written_buffers_on_others(q8):
    L, T, D, H, Hq = N.lib(), 3, 64, 1, 2
    qb, kb = T * Hq * D * 2, T * H * D * 2
    reads = [(at(11), kb), (at(12), D * 2), (at(13), D * 2), (at(14), 8 * D * 4), (at(15), T * 4)]   # k, weights, table, positions

    def rope(qo=at(20), ko=at(21), qs=Hq * D, ks=H * D):
        return L.qv_qk_norm_rope(T, Hq, H, D, N.QV_BF16, at(10), qs, at(11), ks, at(12), at(13), 0.0, at(14), 8, D, 0,
                                 at(15), qo, ko, None)
    for base, size in reads:
        assert all(rope(qo=o) == N.QV_EINVAL for o in around(base, size, qb))
        if base != at(11):
            assert all(rope(ko=o) == N.QV_EINVAL for o in around(base, size, kb))
    assert all(rope(ko=o) == N.QV_EINVAL for o in around(at(10), qb, kb) + around(at(20), qb, kb))
    assert rope(qo=at(10) + 16) == rope(qo=at(10), qs=2 * Hq * D) == N.QV_EINVAL
    assert rope(ko=at(11) + 16) == rope(ko=at(11), ks=2 * H * D) == N.QV_EINVAL

    def append(qo=at(20), qs=Hq * D, values=at(16), **kw):
        d = dict(k=at(1), v=at(2), err=at(9), pages=4, kv_heads=H, page_size=16, head_dim=D, bits=8 if q8 else 0,
                 k_scale=at(3) if q8 else None, v_scale=at(4) if q8 else None)
        c = cache_desc(**{**d, **kw})
        return L.qv_paged_append(ctypes.byref(c), T, Hq, at(10), qs, at(11), H * D, values, H * D, at(12), at(13), 0.0,
                                 at(14), 8, D, 0, at(15), at(17), qo, None)
    reads += [(at(16), kb), (at(17), T * 8), (at(9), 4)]      # v, slots, the error word
    pool = 4 * H * 16 * D * (1 if q8 else 2)
    scales = [("k_scale", at(3)), ("v_scale", at(4))] if q8 else []
    for base, size in reads + [(at(1), pool), (at(2), pool)] + [(b, 256) for _, b in scales]:
        assert all(append(qo=o) == N.QV_EINVAL for o in around(base, size, qb))
    assert append(qo=at(10) + 16) == append(qo=at(10), qs=2 * Hq * D) == N.QV_EINVAL
    # the pool on what the call reads, and its parts on one another
    for base, size in reads + [(at(10), qb)]:
        for name, n in [("k", pool), ("v", pool)] + [(s, 256) for s, _ in scales]:
            assert all(append(**{name: o}) == N.QV_EINVAL for o in around(base, size, n)), (base, name)
    assert append(values=at(2) + 32) == append(k=at(2)) == append(k=at(2) + pool - 16) == N.QV_EINVAL
    if q8:
        assert append(k_scale=at(4)) == append(k_scale=at(1)) == append(v_scale=at(2) + pool - 16) == N.QV_EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
def test_outputs_on_the_pool_and_shared_pools_are_refused(q8):
    g = gen(59)
    pool = Pool(g, [20], 1, 64, 16, BF16, q8)
    c, T = pool.cache, 3
    q, k, v = rand(g, T, 4, 64).to(BF16), rand(g, T, 1, 64).to(BF16), rand(g, T, 1, 64).to(BF16)
    slots = torch.arange(T, device=DEV)
    on = [x.view(-1).view(BF16)[: T * 4 * 64].view(T, 4, 64) for x in (c.k_pages, c.v_pages)]
    before = [x.clone() for x in (c.k_pages, c.v_pages)]
    for o in on:
        with pytest.raises(N.QevictError):
            c.attend(q, pool.bt, pool.lens, cu([T]), out=o)
        with pytest.raises(N.QevictError):
            c.append(q, k, v, slots, q_out=o)
        with pytest.raises(N.QevictError):       # queries read from the pool that the call writes
            c.append(o, k, v, slots)
    with pytest.raises(N.QevictError):
        paged.paged_append(q, k, v, slots, None, None, c.k_pages, c.k_pages, k_scale=c.k_scale, v_scale=c.v_scale)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, (c.k_pages, c.v_pages)))
    # what may share: reads alone (one tensor for keys and values), and outputs in their input's place
    paged.paged_attention(q, c.k_pages, c.k_pages, pool.bt, pool.lens, cu([T]), k_scale=c.k_scale, v_scale=c.k_scale)
    packed = torch.cat([q, k, v], 1)[:1]
    want = c.append(packed[:, :4].clone(), packed[:, 4:5], packed[:, 5:], slots[:1])
    got = c.append(packed[:, :4], packed[:, 4:5], packed[:, 5:], slots[:1], q_out=packed[:, :4])
    assert got.data_ptr() == packed.data_ptr() and torch.equal(got, want)


# ------------------------------------------------------------------ slots
def test_slots_of_indices_outside_the_table():
    """Indices before a sequence are skipped (they do not wrap to the block table's last page); those behind the
    table, of no sequence, or on a page that is not the pool's lie behind the pool."""
    c = paged.PagedKVCache(5, 1, 64, 16, BF16, device="cpu")
    bt = torch.tensor([[3, 1, -1], [0, 5, 2 ** 31 - 1]], dtype=torch.int32)
    pos = torch.tensor([0, 17, 31, 32, 47, 48, -1, -48, -49, 2 ** 31, 0, 16, 40, 3, 3, -5], dtype=torch.int64)
    seq = torch.tensor([0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 1, 1, 1, 2, -1, 9], dtype=torch.int32)
    want = [48, 17, 31, 80, 80, 80, -1, -1, -1, 80, 0, 80, 80, 80, 80, -1]      # 80: anything from there on

    def slots(*args):
        got = c.slots(*args)
        assert got.dtype == torch.int64
        return got.clamp(max=80).tolist()
    assert slots(bt, seq, pos) == want
    assert slots(bt, seq[:9], pos[:9].int()) == want[:9]
    assert slots(bt[:, :0], seq[:8], pos[:8]) == [80] * 6 + [-1] * 2
    assert slots(bt, seq[:0], pos[:0]) == []
    # a view of a wider table
    assert slots(bt[:, :2], seq[:4], pos[:4]) == [48, 17, 31, 80]


@pytest.mark.gpu
def test_append_of_a_padded_batch_through_slots():
    g = gen(61)
    c = paged.PagedKVCache(3, 2, 64, 16, BF16)
    bt = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    q, k, v = (rand(g, 4, 2, 64).to(BF16) for _ in range(3))
    seq, pos = torch.zeros(4, dtype=torch.int64, device=DEV), torch.tensor([-1, 20, -7, 3], device=DEV)
    c.append(q, k, v, c.slots(bt, seq, pos))
    assert c.read_error() == 0
    used = torch.zeros(3, 16, dtype=torch.bool, device=DEV)
    used[0, 4] = used[2, 3] = True
    assert torch.equal(c.k_pages[0, :, 4], k[1]) and torch.equal(c.v_pages[2, :, 3], v[3])
    for x in (c.k_pages, c.v_pages):
        assert bool((x.transpose(1, 2)[~used] == 0).all())
    c.append(q, k, v, c.slots(bt, seq, pos + 32))            # one behind the table
    assert c.read_error() == N.QV_DERR_CAPACITY


# ------------------------------------------------------------------ INT8 codes
def codes(x):
    """Codes and scales of rows [..., D] as promised, on the host: IEEE fp32 divisions, ties to even."""
    x = x.float().cpu()
    s = x.abs().amax(-1) / torch.tensor(127.0)
    return (x / s[..., None]).round().to(torch.int8), s


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_int8_codes_are_those_of_the_quotient(D, dt):
    """Rows as they are (no norm, no rotation), with elements on and beside ties: the code is rint(row / scale)."""
    g = gen(67)
    T, H = 700, 2          # (44 pages hold them)
    x = rand(g, T, 2 * H, D) * torch.exp2(torch.randint(-12, 5, (T, 2 * H, 1), generator=g, device=DEV).float())
    s = x.abs().amax(-1, keepdim=True) / torch.tensor(127.0, device=DEV)
    top = x.abs() == x.abs().amax(-1, keepdim=True)
    # half of the rows: every element but the largest as near to a tie as the type allows, then an ulp to either side
    tie = (torch.randint(-126, 126, x.shape, generator=g, device=DEV) + 0.5) * s
    step = torch.randint(-1, 2, x.shape, generator=g, device=DEV) * 2.0 ** -23 * tie
    x = torch.where(top | (torch.arange(T, device=DEV) % 2 == 0)[:, None, None], x, tie + step).to(dt)
    if dt == FP32:      # the reciprocal's product alone gives other codes here
        c, sc = codes(x)
        assert int(((x.cpu() * (1 / sc[..., None])).round() != c).sum()) > 0
    c = paged.PagedKVCache(T // 16 + 1, H, D, 16, dt, bits=8)
    order = torch.randperm(T, generator=g, device=DEV)
    c.append(x[:, :H], x[:, :H], x[:, H:], order)
    for pages, scales, rows in ((c.k_pages, c.k_scale, x[:, :H]), (c.v_pages, c.v_scale, x[:, H:])):
        want, ws = codes(rows)
        assert torch.equal(scales.transpose(1, 2).reshape(-1, H)[order].cpu(), ws)
        assert torch.equal(pages.transpose(1, 2).reshape(-1, H, D)[order].cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("n", [1, 150])
def test_attention_int8_negative_value_scale_is_not_another_row(n, dt):
    """A pool filled by someone else: a negative value scale is honoured or shows as NaN, in the rows that see it."""
    L, D, page = 400, 64, 32
    g = gen(71)
    pool = Pool(g, [L], 1, D, page, dt, True)
    c, key = pool.cache, L - 2
    pg, off = int(pool.bt[0, key // page]), key % page
    c.v_scale[pg, 0, off] *= -1
    pool.vs[0][key] *= -1
    q = rand(g, n, 4, D).to(dt)
    out = c.attend(q, pool.bt, pool.lens, cu([n]), max_q=n)
    o, mag, big = ref_attention(q, pool.ks[0], pool.vs[0])
    bound = attention_bound(o, mag, big, L, D, dt, float(pool.vs[0].abs().max()))
    assert bool((((out.double() - o).abs() <= bound) | out.isnan()).all())


# ------------------------------------------------------------------ cumulative lengths
@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 600])
def test_gather_reports_rows_that_do_not_hold_a_sequence(B):
    """Sequences cut by the next one's rows or by the rows there are raise the error word; the rows that exist are read."""
    g = gen(73)
    lens = [5] * B
    pool = Pool(g, lens, 1, 64, 16, BF16, False)
    c, total = pool.cache, 5 * B
    ok = cu(lens)
    want, _ = c.gather(pool.bt, pool.lens, ok, total)
    assert c.read_error() == 0
    c.gather(pool.bt, pool.lens, torch.cat([ok[:1], ok[1:] + 2]), total + 2)       # a gap is no fault
    assert c.read_error() == 0

    def reported(lens, cu_kv, total):
        c.err.zero_()
        k, _ = c.gather(pool.bt, lens, cu_kv, total, out=tuple(torch.zeros(total, 1, 64, dtype=BF16, device=DEV) for _ in range(2)))
        assert c.read_error() == N.QV_DERR_CAPACITY
        return k
    assert torch.equal(reported(pool.lens, ok, total - 1), want[:-1])              # fewer rows than tokens
    more = pool.lens.clone()
    more[B - 1] += 1
    assert torch.equal(reported(more, ok, total), want)                            # a length past its rows
    for i, d in ((0, -1), (B, -1), (1, -6)):
        bad = ok.clone()
        bad[i] += d
        reported(pool.lens, bad, total)
    less = pool.lens.clone()
    less[0] = -1
    reported(less, ok, total)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("dt", [BF16, FP32])
def test_attention_reports_chunks_outside_the_rows(n, dt):
    g = gen(79)
    pool = Pool(g, [100, 90], 1, 64, 16, dt, False)
    c, q, ok = pool.cache, rand(g, 2 * n, 4, 64).to(dt), cu([n, n])
    want = c.attend(q, pool.bt, pool.lens, ok, max_q=n)
    assert c.read_error() == 0
    for i, d in ((0, -1), (2, 1), (1, n + 1)):
        bad = ok.clone()
        bad[i] += d
        got = c.attend(q, pool.bt, pool.lens, bad, max_q=n)
        assert c.read_error() == N.QV_DERR_CAPACITY
        if i == 2:
            assert torch.equal(got[:n], want[:n])        # the other sequence is right
        c.err.zero_()


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_fp16_keeps_probabilities_down_to_2_31(shape, q8):
    """The fp16 kernels set a row's reference 2^7 below a maximum, so the largest P is at least 2^7 at the end, and what
    rounds at fp16's smallest step (2^-24) is off by 2^-25 / 2^7 of the sum for each key.  With INT8 pages P = p vs
    and the sum is of P / vs: at least 2^7 / (largest scale), each key's product with a code of up to 127 off by 127 2^-25: the
    same 2^-32 of the largest |v| (127 times its scale)."""
    q_lens, kv_lens, Hq, H, D, page = SHAPES[shape]
    pool, q, out = check_attention(gen(200 + shape), q_lens, kv_lens, Hq, H, D, page, FP16, q8, max_q=max(q_lens))
    at = 0
    for b, n in enumerate(q_lens):
        if n and kv_lens[b]:
            o, mag, big = ref_attention(q[at:at + n], pool.ks[b], pool.vs[b])
            vmax = float(pool.vs[b].abs().max())
            bound = attention_bound(o, mag, big, kv_lens[b], D, FP32, vmax) + o.abs() * half(FP16) * 1.001 + (
                mag * half(FP16) * 1.01 + TINY[FP16] + kv_lens[b] * 2.0 ** -32 * vmax)
            d = (out[at:at + n].double() - o).abs()
            assert bool((d <= bound).all()), (b, n, kv_lens[b], float((d / bound).max()))
        at += n


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_prompt_in_pages_to_a_sticky_layer(bits):
    """A prompt that came in ragged chunks is read back and becomes a Sticky layer's prompt, which then decodes across
    evictions: the same bits as the layer built from the rows that the pool holds, without pages."""
    from qevict_b200.layer_state import StickyLayerState
    from qevict_b200.model import prefill_attention
    Hq, H, D, page, dt, om, sink, S, steps = 8, 2, 128, 32, BF16, 32, 32, 32 + 32 * 15, 70
    g = gen(83)
    qkv = rand(g, S + steps, Hq + 2 * H, D).to(dt)
    table = paged.rope_table(1024, D, 500000.0)
    pos = torch.arange(S + steps, device=DEV, dtype=torch.int32)
    qr, kr = paged.qk_norm_rope(qkv[:, :Hq], qkv[:, Hq:Hq + H], pos, table)
    v = qkv[:, Hq + H:].contiguous()
    c = paged.PagedKVCache(20, H, D, page, dt, bits=bits)
    bt = torch.randperm(20, generator=g, device=DEV).int()[: S // page].view(1, -1).contiguous()
    queries, at = [], 0
    for n in (200, 1, 150, S - 351):
        rows = slice(at, at + n)
        slots = c.slots(bt, torch.zeros_like(pos[rows]), pos[rows])
        queries.append(c.append(qkv[rows, :Hq], qkv[rows, Hq:Hq + H], qkv[rows, Hq + H:], slots, pos[rows], table))
        at += n
    q = torch.cat(queries)
    k1, v1 = c.gather(bt, torch.tensor([S], dtype=torch.int32, device=DEV), cu([S]), S)
    assert c.read_error() == 0 and torch.equal(q, qr[:S])
    if bits == 16:
        k2, v2 = kr[:S], v[:S]
    else:   # the rows as the pool holds them, by hand
        def held(pages, scales):
            ids = bt[0].long()
            x = pages[ids].float() * scales[ids][..., None]
            return x.transpose(1, 2).reshape(S, H, D).to(dt)
        k2, v2 = held(c.k_pages, c.k_scale), held(c.v_pages, c.v_scale)
    outs = []
    for kk, vv in ((k1, v1), (k2, v2)):
        _, colsum = prefill_attention(q[None], kk[None].contiguous(), vv[None].contiguous())
        layer = StickyLayerState(1, H, Hq // H, D, om, sink, 64, 2, 3, 32, 8, dt)
        layer.prefill(kk[None].transpose(1, 2), vv[None].transpose(1, 2), colsum)
        outs.append(torch.stack([layer.step(qr[i].view(1, Hq, D), kr[i].view(1, H, D), v[i].view(1, H, D))
                                 for i in range(S, S + steps)]))
        assert layer.read_error() == 0
        ids, _ = layer.view_sticky(0)
        outs.append(ids)
    assert torch.equal(outs[0], outs[2]) and bool(outs[0].isfinite().all())
    assert torch.equal(torch.as_tensor(outs[1]), torch.as_tensor(outs[3]))


@pytest.mark.gpu
def test_attention_from_several_threads():
    """Four host threads at once, each on a stream of its own, over one pool: the bits of the calls made alone."""
    import threading
    g = gen(89)
    pool = Pool(g, [900, 40, 333], 2, 128, 32, BF16, True)
    jobs = []
    for n in (1, 2, 3, 33):
        q = rand(g, 3 * n, 8, 128).to(BF16)
        jobs.append((q, cu([n] * 3), n, pool.cache.attend(q, pool.bt, pool.lens, cu([n] * 3), max_q=n)))
    torch.cuda.synchronize()
    got, faults = [[] for _ in jobs], []

    def work(i):
        try:
            q, c, n, _ = jobs[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got[i].append(pool.cache.attend(q, pool.bt, pool.lens, c, max_q=n))
                torch.cuda.current_stream().synchronize()
        except Exception as e:     # noqa: BLE001 -- reported by the thread that runs the test
            faults.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not faults and pool.cache.read_error() == 0
    for (_, _, _, want), outs in zip(jobs, got):
        assert len(outs) == 50 and all(torch.equal(o, want) for o in outs)


ORIG = dict(low_freq_factor=1.0, high_freq_factor=4.0, original_max_position=8192)


@pytest.mark.parametrize("theta,rot", [(10000.0, 64), (500000.0, 128), (1000.0, 8)])
@pytest.mark.parametrize("scaling", [None, dict(type="linear", factor=3.0), dict(type="ntk", factor=4.0),
                                     dict(type="llama3", factor=8.0, **ORIG),
                                     dict(type="yarn", factor=16.0, original_max_position=4096),
                                     dict(type="yarn", factor=4.0, original_max_position=8192, beta_fast=16, beta_slow=2,
                                          attention_factor=1.25)])
def test_rope_table_is_the_formula(theta, rot, scaling):
    """Every pair at a few positions against the formulas one number at a time in 64 bits.  An entry is rounded once
    (half a step of a number below 2 mult); 64-bit frequencies are off by a few 2^-53, so an angle of up to 2^17 by 2^-33."""
    t = paged.rope_table(131072, rot, theta, scaling, device="cpu")
    kind = scaling["type"] if scaling else None
    f = scaling["factor"] if scaling else 1.0
    mult = 1.0
    if kind == "yarn":
        mult = scaling.get("attention_factor", 0.1 * math.log(f) + 1)
    worst = (0.0,)
    for i in range(rot // 2):
        base = theta * f ** (rot / (rot - 2)) if kind == "ntk" else theta
        w = base ** (-2 * i / rot)
        if kind == "linear":
            w /= f
        elif kind == "llama3":
            wave = 2 * math.pi / w
            if wave > 8192 / 1.0:
                w /= f
            elif wave >= 8192 / 4.0:
                smooth = (8192 / wave - 1.0) / (4.0 - 1.0)
                w = (1 - smooth) * w / f + smooth * w
        elif kind == "yarn":
            orig = scaling["original_max_position"]
            at = [rot * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(theta))
                  for n in (scaling.get("beta_fast", 32), scaling.get("beta_slow", 1))]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
            share = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            w = w * (1 - share) + w / f * share
        for p in (0, 1, 2, 77, 4095, 8192, 100003, 131071):
            for j, want in ((i, math.cos(p * w)), (rot // 2 + i, math.sin(p * w))):
                d = abs(float(t[p, j]) - want * mult)
                worst = max(worst, (d, p, i, float(t[p, j]), want * mult))
    assert worst[0] <= mult * (2.0 ** -24 + 2.0 ** -32), worst     # (difference, position, pair, entry, formula)

"""Measured cases of the paged-cache operators.

Four operators: the norm and rotation of query and key heads (`rope`), the
same with the new keys and values written into a paged cache (`append`),
reading a paged cache back into contiguous rows (`gather`), and attention of
chunks of new tokens over the paged cache (`attend`).  `run` computes them in
plain torch, or through the framework's entry points where `own` is set.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}


# --------------------------------------------------------------------- cases
def listed():
    """Head counts and lengths are those of the repository's workloads (a
    Llama-3-8B layer: 32 query / 8 KV heads of 128; a Llama-2-7B MHA layer:
    32 heads; the 4096-token fp32 layer; 32768- and 131072-token contexts)."""
    return [
        # the rotation of one decode step, batch 1: launch latency
        dict(name="rope_step", op="rope", tokens=1, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False,
             norm=False, dtype="bf16", max_pos=40960),
        # a prompt of an MHA layer: interleaved pairs on half of the head, normed queries and keys, an odd length
        dict(name="rope_prompt", op="rope", tokens=16383, heads=32, kv_heads=32, dim=128, rot=64, interleaved=True,
             norm=True, dtype="fp16", max_pos=40960),
        # one decode step of 64 sequences: rotate and write the new token of each
        dict(name="append_step", op="append", seqs=64, tokens=64, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, norm=False, dtype="bf16", pages="bf16", page=64, max_pos=40960),
        # ragged chunks written in 8 bits with normed heads, and the sequences read back
        dict(name="append_int8", op="append", seqs=7, tokens=8191, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, norm=True, dtype="bf16", pages="int8", page=32, max_pos=40960),
        # a few short 8-bit sequences read back
        dict(name="gather_short", op="gather", seqs=5, tokens=1001, kv_heads=8, dim=64, dtype="fp16", pages="int8",
             page=16),
        # a whole long context read back
        dict(name="gather_long", op="gather", seqs=1, tokens=131072, kv_heads=8, dim=128, dtype="bf16", pages="bf16",
             page=64),
        # one decode step over a 32768-token context, batch 1
        dict(name="attend_one", op="attend", seqs=1, chunk=1, context=32768, heads=32, kv_heads=8, dim=128,
             dtype="bf16", pages="bf16", page=64, ragged=False),
        # one decode step of 64 sequences of uneven length over 8-bit pages
        dict(name="attend_batch_int8", op="attend", seqs=64, chunk=1, context=8192, heads=32, kv_heads=8, dim=128,
             dtype="bf16", pages="int8", page=64, ragged=True),
        # the first chunk of a prompt is the whole prompt
        dict(name="attend_prompt", op="attend", seqs=1, chunk=8192, context=8192, heads=32, kv_heads=8, dim=128,
             dtype="bf16", pages="bf16", page=64, ragged=False),
        # chunks of four prompts in flight, contexts of uneven length, 8-bit pages
        dict(name="attend_chunks_int8", op="attend", seqs=4, chunk=512, context=16384, heads=32, kv_heads=8, dim=128,
             dtype="bf16", pages="int8", page=32, ragged=True),
        # chunks and single tokens in one batch, some sequences empty, small heads
        dict(name="attend_mixed", op="attend", seqs=17, chunk=300, context=4000, heads=64, kv_heads=8, dim=64,
             dtype="fp16", pages="fp16", page=16, ragged=True),
        # the fp32 layer: the last chunk of a 4096-token prompt
        dict(name="attend_fp32", op="attend", seqs=1, chunk=256, context=4096, heads=32, kv_heads=8, dim=128,
             dtype="fp32", pages="fp32", page=64, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "gather", "attend", "attend", "attend"])
    if op == "attend":
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 32, 128), (16, 2, 128), (40, 8, 128), (12, 4, 128),
                                           (64, 8, 64), (15, 5, 64), (8, 1, 64)])
    else:
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 32, 128), (16, 2, 128), (40, 8, 128), (64, 8, 64),
                                           (15, 5, 64), (8, 1, 64), (20, 4, 256), (32, 32, 80)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    if op in ("rope", "append"):
        case.update(rot=rng.choice([dim, dim, dim // 2, 32]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.5, max_pos=40960, tokens=_log(rng, 1, 8192))
    if op == "append":
        case["seqs"] = min(case["tokens"], _log(rng, 1, 64))
    if op == "gather":
        del case["heads"]
        case.update(seqs=_log(rng, 1, 64), tokens=_log(rng, 64, 65536))
    if op in ("append", "gather", "attend"):
        # fp32 rows are appended as they are: a code next to a rounding border is not fixed by 32 bits
        pages = [dtype] if op == "append" and dtype == "fp32" else [dtype, "int8"]
        case.update(pages=rng.choice(pages), page=rng.choice([16, 32, 64, 128]))
    if op == "attend":
        seqs = _log(rng, 1, 48)
        chunk = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        context = _log(rng, 16, 32768)
        # no costlier than the largest listed case: scores and gathered rows are bounded
        top = 4e8 if dtype == "fp32" else 2e9
        while seqs * chunk * context * heads > top and seqs > 1:
            seqs = (seqs + 1) // 2
        while seqs * chunk * context * heads > top:
            chunk = (chunk + 1) // 2
        while seqs * context * kv_heads * dim > 5e8:
            seqs = (seqs + 1) // 2
        case.update(seqs=seqs, chunk=min(chunk, context), context=context, ragged=seqs > 1)
    return case


# ---------------------------------------------------------------- inputs
def _split(total, parts, gen):
    """`parts` uneven lengths of at least 1 that sum to `total`."""
    w = torch.rand(parts, generator=gen) + 0.1
    lens = (w / w.sum() * (total - parts)).long() + 1
    lens[0] += total - int(lens.sum())
    return lens


def _lengths(case):
    """(new tokens, cached tokens with them) of each sequence: they go by the case alone, the values by the seed."""
    n = case["seqs"]
    gen = torch.Generator().manual_seed(1000003 * n + case.get("context", 0) + case.get("tokens", 0))
    if case["op"] in ("append", "gather"):
        lens = _split(case["tokens"], n, gen) if n <= case["tokens"] else torch.zeros(n, dtype=torch.long)
        if n > case["tokens"]:
            lens[: case["tokens"]] = 1
        return lens, lens
    kv = torch.full((n,), case["context"])
    q = torch.full((n,), case["chunk"])
    if case["ragged"]:
        # one sequence is the longest, the others are spread below it
        kv[1:] = (torch.rand(n - 1, generator=gen) * case["context"]).long() + 1
        if case["chunk"] > 1:
            q[1:] = (torch.rand(n - 1, generator=gen) * case["chunk"]).long() + 1
            q[2::4] = 1                     # single tokens among the chunks
            q[3::8] = 0                     # sequences with nothing new
        q = torch.minimum(q, kv)
    return q, kv


def _table(case, dev):
    """cos | sin of every position, angles in 64 bits, frequencies stretched for
    long contexts: wavelengths over the trained length are slowed 8 times."""
    r = case["rot"]
    inv = 500000.0 ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64) / r)
    inv = torch.where(2 * math.pi / inv > 8192, inv / 8, inv)
    a = torch.arange(case["max_pos"], device=dev, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(case, seed):
    dev, dt = "cuda", DTYPES[case["dtype"]]
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    H, D, op = case["kv_heads"], case["dim"], case["op"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * std

    # a few channels of the keys carry large values, as in trained models
    gain = torch.where(torch.rand(H, D, generator=gen, device=dev) < 0.04, 4.0, 1.0)
    s = dict(case=case)
    if op in ("rope", "append"):
        T, Hq = case["tokens"], case["heads"]
        qkv = normal(T, Hq + 2 * H, D)
        qkv[:, Hq:Hq + H] *= gain
        qkv = qkv.to(dt).view(T, (Hq + 2 * H) * D)      # one packed projection; q, k, v are views of it
        s["q"], s["k"], s["v"] = (x.view(T, -1, D) for x in qkv.split([Hq * D, H * D, H * D], 1))
        s["table"] = _table(case, dev)
        s["qw"] = (1 + normal(D, std=0.1)).to(dt) if case["norm"] else None
        s["kw"] = (1 + normal(D, std=0.1)).to(dt) if case["norm"] else None
    if op == "rope":
        start = int(torch.randint(0, case["max_pos"] - case["tokens"] + 1, (1,), generator=host))
        s["positions"] = torch.arange(start, start + case["tokens"], device=dev, dtype=torch.int32)
        return s

    page = case["page"]
    q_lens, kv_lens = _lengths(case)
    pages = (kv_lens + page - 1) // page
    total = int(pages.sum())
    n_pages = total + total // 4 + 1                    # a pool with free pages, used in random order
    order = torch.randperm(n_pages, generator=host)[:total].to(torch.int32)
    width = max(1, int(pages.max()))
    block = torch.zeros(case["seqs"], width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages.tolist()):
        block[b, :n] = order[at:at + n]
        at += n
    s["block"] = block.to(dev)
    s["kv_lens"] = kv_lens.to(torch.int32).to(dev)
    zero = torch.zeros(1, dtype=torch.long)
    s["cu_q"] = torch.cat([zero, q_lens.cumsum(0)]).to(torch.int32).to(dev)
    s["cu_kv"] = torch.cat([zero, kv_lens.cumsum(0)]).to(torch.int32).to(dev)
    s["max_q"], s["max_kv"] = int(q_lens.max()), int(kv_lens.max())
    s["total_q"], s["total_kv"] = int(q_lens.sum()), int(kv_lens.sum())

    s["ks"] = s["vs"] = None
    if op == "append":
        pt = torch.int8 if case["pages"] == "int8" else dt
        s["kp"] = torch.zeros(n_pages, H, page, D, device=dev, dtype=pt)
        s["vp"] = torch.zeros_like(s["kp"])
        if case["pages"] == "int8":
            s["ks"] = torch.zeros(n_pages, H, page, device=dev)
            s["vs"] = torch.zeros_like(s["ks"])
        seq = torch.repeat_interleave(torch.arange(case["seqs"]), kv_lens)
        pos = torch.arange(s["total_kv"]) - torch.cat([zero, kv_lens.cumsum(0)])[seq]
        # where each sequence stands: its earlier tokens are in pages that this pool does not show
        start = (torch.rand(case["seqs"], generator=host) * (case["max_pos"] - s["max_kv"])).long()
        s["positions"] = (pos + start[seq]).to(torch.int32).to(dev)
        s["slots"] = (block[seq, pos // page].long() * page + pos % page).to(dev)
        return s

    for n, std in (("k", 1.0), ("v", 0.5)):
        x = normal(n_pages, H, page, D, std=std)
        if n == "k":
            x *= gain[:, None, :]
        if case["pages"] == "int8":
            sc = x.abs().amax(-1) / 127
            s[n + "p"], s[n + "s"] = (x / sc[..., None]).round().to(torch.int8), sc
        else:
            s[n + "p"] = x.to(dt)
    if op == "attend":
        s["q"] = normal(s["total_q"], case["heads"], D).to(dt)
    return s


# ---------------------------------------------------------------- plain forms
def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()


def _rotated(x, s):
    r, row = s["case"]["rot"], s["table"][s["positions"].long()][:, None]
    c, n = row[..., : r // 2], row[..., r // 2:]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if s["case"]["interleaved"] else (x[..., : r // 2], x[..., r // 2: r])
    a, b = a * c - b * n, b * c + a * n
    y = torch.stack([a, b], -1).flatten(-2) if s["case"]["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([y, x[..., r:]], -1)


def _write(x, pages, scales, s):
    page = s["case"]["page"]
    pg, off = s["slots"] // page, s["slots"] % page
    if scales is None:
        pages[pg, :, off] = x.to(pages.dtype)
    else:
        sc = x.abs().amax(-1) / 127
        pages[pg, :, off] = torch.where(sc[..., None] > 0, x / sc[..., None], 0.0).round().to(torch.int8)
        scales[pg, :, off] = sc


def _rows(pages, scales, pg, off):
    x = pages[pg, :, off].float()
    return x if scales is None else x * scales[pg, :, off][..., None]


def _plain_gather(s):
    page, dt = s["case"]["page"], DTYPES[s["case"]["dtype"]]
    t = torch.arange(s["total_kv"], device="cuda")
    seq = torch.searchsorted(s["cu_kv"].long(), t, right=True) - 1
    pos = t - s["cu_kv"].long()[seq]
    pg, off = s["block"].long()[seq, pos // page], pos % page
    return [_rows(s["kp"], s["ks"], pg, off).to(dt), _rows(s["vp"], s["vs"], pg, off).to(dt)]


def _plain_attend(s):
    case = s["case"]
    page, H, D, B, dt = case["page"], case["kv_heads"], case["dim"], case["seqs"], DTYPES[case["dtype"]]
    G = case["heads"] // H
    j = torch.arange(s["max_kv"], device="cuda")
    live = j[None] < s["kv_lens"][:, None]
    pg, off = s["block"].long()[:, j // page], (j % page)[None].expand(B, -1)
    k = _rows(s["kp"], s["ks"], pg, off)                # [B, kv, H, D]
    v = torch.where(live[..., None, None], _rows(s["vp"], s["vs"], pg, off), 0.0)
    cu = s["cu_q"].long()
    i = torch.arange(s["max_q"], device="cuda")
    q = s["q"][(cu[:-1, None] + i).clamp(max=s["total_q"] - 1)].float().view(B, -1, H, G, D)
    first = s["kv_lens"].long() - (cu[1:] - cu[:-1])    # position of each chunk's first token
    seen = (j[None, None] <= (first[:, None] + i)[..., None]) & live[:, None]
    x = q.permute(0, 2, 3, 1, 4).reshape(B, H, -1, D) @ k.permute(0, 2, 3, 1)
    x = (x.view(B, H, G, -1, s["max_kv"]) / math.sqrt(D)).masked_fill_(~seen[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    x /= x.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (x.view(B, H, -1, s["max_kv"]) @ v.permute(0, 2, 1, 3)).view(B, H, G, -1, D).permute(0, 3, 1, 2, 4)
    t = torch.arange(s["total_q"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    return o[seq, t - cu[seq]].reshape(-1, H * G, D).to(dt)


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from qevict_b200 import paged
        if op == "rope":
            return list(paged.qk_norm_rope(s["q"], s["k"], s["positions"], s["table"], q_weight=s["qw"],
                                           k_weight=s["kw"], interleaved=case["interleaved"]))
        if op == "append":
            q = paged.paged_append(s["q"], s["k"], s["v"], s["slots"], s["positions"], s["table"], s["kp"], s["vp"],
                                   k_scale=s["ks"], v_scale=s["vs"], q_weight=s["qw"], k_weight=s["kw"],
                                   interleaved=case["interleaved"])
            if case["pages"] != "int8":
                return [q, s["kp"], s["vp"]]
            return [q, *paged.paged_gather(s["kp"], s["vp"], s["block"], s["kv_lens"], s["cu_kv"], s["total_kv"],
                                           k_scale=s["ks"], v_scale=s["vs"], dtype=DTYPES[case["dtype"]])]
        if op == "gather":
            return list(paged.paged_gather(s["kp"], s["vp"], s["block"], s["kv_lens"], s["cu_kv"], s["total_kv"],
                                           k_scale=s["ks"], v_scale=s["vs"], dtype=DTYPES[case["dtype"]]))
        return paged.paged_attention(s["q"], s["kp"], s["vp"], s["block"], s["kv_lens"], s["cu_q"], k_scale=s["ks"],
                                     v_scale=s["vs"], max_q=s["max_q"], max_kv=s["max_kv"])
    if op in ("rope", "append"):
        q, k = _rotated(_normed(s["q"], s["qw"]), s), _rotated(_normed(s["k"], s["kw"]), s)
        if op == "rope":
            return [q.to(s["q"].dtype), k.to(s["q"].dtype)]
        _write(k, s["kp"], s["ks"], s)
        _write(s["v"].float(), s["vp"], s["vs"], s)
        kv = _plain_gather(s) if case["pages"] == "int8" else [s["kp"], s["vp"]]
        return [q.to(s["q"].dtype), *kv]
    return _plain_gather(s) if op == "gather" else _plain_attend(s)


# ---------------------------------------------------------------- work
def work(case):
    op, D, H = case["op"], case["dim"], case["kv_heads"]
    e = BYTES[case["dtype"]]
    # one head's row in the pages
    row = D * BYTES[case["pages"]] + (4 if case["pages"] == "int8" else 0) if "pages" in case else 0
    if op == "gather":
        return {"bytes": 2 * case["tokens"] * H * (row + D * e), "flops": 0}
    if op == "attend":
        q, kv = (x.double() for x in _lengths(case))
        pairs = float((q * kv - q * (q - 1) / 2).sum())             # a chunk's token sees the keys up to its own
        live = float(kv[q > 0].sum())
        return {"bytes": 2 * live * H * row + 2 * float(q.sum()) * case["heads"] * D * e,
                "flops": 4 * D * case["heads"] * pairs}
    T, Hq = case["tokens"], case["heads"]
    b = 2 * T * (Hq + H) * D * e + T * (case["rot"] + 1) * 4
    if op == "append":      # values in, keys and values into the pages (no keys out), slots; 8-bit pages are read back
        b += T * H * 2 * row + 8 * T
        b += 2 * T * H * (row + D * e) if case["pages"] == "int8" else 0
    return {"bytes": b, "flops": T * (Hq + H) * (3 * case["rot"] + (4 * D if case["norm"] else 0))}


# ---------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op, D = case["op"], case["dim"]

    def heads(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        r = case["rot"]
        y, h = x.clone(), r // 2
        for i in range(h):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + h)
            c = s["table"][s["positions"].long(), i].double()[:, None]
            n = s["table"][s["positions"].long(), h + i].double()[:, None]
            y[..., a] = x[..., a] * c - x[..., b] * n
            y[..., b] = x[..., a] * n + x[..., b] * c
        return y

    def sequence(pages, scales, b):
        """The cached rows of sequence b, [tokens, heads, dim]."""
        n = int(s["kv_lens"][b])
        ids = s["block"][b, : -(-n // case["page"])].long()
        x = pages[ids].double()
        if scales is not None:
            x = x * scales[ids].double()[..., None]
        return x.transpose(1, 2).reshape(-1, pages.shape[1], D)[:n]

    if op == "rope":
        return [heads(s["q"], s["qw"]), heads(s["k"], s["kw"])]
    if op == "append":
        out = [heads(s["q"], s["qw"])]
        for x, pages in ((heads(s["k"], s["kw"]), s["kp"]), (s["v"].double(), s["vp"])):
            if case["pages"] == "int8":
                step = x.abs().amax(-1, keepdim=True) / 127
                out.append(torch.round(x / step).nan_to_num(0.0) * step)
            else:
                y = pages.double().transpose(1, 2).reshape(-1, pages.shape[1], D)
                y[s["slots"]] = x
                out.append(y.view(pages.shape[0], case["page"], -1, D).transpose(1, 2))
        return out
    if op == "gather":
        return [torch.cat([sequence(s["kp"], s["ks"], b) for b in range(case["seqs"])]),
                torch.cat([sequence(s["vp"], s["vs"], b) for b in range(case["seqs"])])]
    G = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["total_q"], case["heads"], D, dtype=torch.float64, device="cuda")
    for b in range(case["seqs"]):
        lo, hi, n = int(s["cu_q"][b]), int(s["cu_q"][b + 1]), int(s["kv_lens"][b])
        if hi == lo:
            continue
        k, v = sequence(s["kp"], s["ks"], b), sequence(s["vp"], s["vs"], b)
        later = torch.arange(n, device="cuda")[None] > torch.arange(n - (hi - lo), n, device="cuda")[:, None]
        for h in range(case["heads"]):
            x = s["q"][lo:hi, h].double() @ k[:, h // G].T / D ** 0.5
            out[lo:hi, h] = torch.softmax(x.masked_fill(later, -math.inf), -1) @ v[:, h // G]
    return out

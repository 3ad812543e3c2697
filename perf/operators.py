"""Timed workloads of the operators that carry a chunk of tokens over a paged cache.

A serving step takes the new tokens of every sequence (one token, a few, or a long chunk of a prompt; the
numbers differ from sequence to sequence) through four operators in each layer:

* ``norm_rope``  per-head RMS norms of queries and keys with the rotary embedding (``ops.qk_norm_rope``);
* ``append``     the same for a fused projection row, its keys and values written into the pages of the cache
                 and, where the cache keeps them, the pages' key bounds brought up to date (``ops.paged_append``);
* ``chunk``      causal attention of the new tokens over the pages (``ops.paged_chunk_attn``);
* ``select``     the pages that a cheap score picks for each query, and attention over those alone
                 (``ops.paged_block_select`` with ``ops.paged_sparse_decode`` or ``ops.paged_chunk_attn``).

``listed()`` names twelve passes, ``draw(rng)`` gives further ones of the same ranges.  ``prepare`` makes the
inputs on the GPU from a seed, ``run`` is one pass, ``work`` the bytes and operations that a pass cannot do
without, and ``exact`` its results in float64 from the definitions.

Lengths are texts: ``"16384x3,700"`` is three sequences of 16384 and one of 700.  ``q_lens`` counts each
sequence's new tokens, ``kv_lens`` its tokens with them.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 1e6
BLOCK = 64      # queries of a chunk that share one selection
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # A decode step's queries and keys before an unpaged cache: eight sequences, one token each.
        dict(name="norm_rope_tokens", kind="norm_rope", N=8, Hq=32, Hkv=8, D=128, dtype="bf16", norm=True,
             far=40000),
        # A prompt of odd length in fp16 with the head counts of a small model, rotation without norms.
        dict(name="norm_rope_small_heads", kind="norm_rope", N=1499, Hq=14, Hkv=2, D=64, dtype="fp16", norm=False,
             far=2000),
        # The whole prompt of the long benchmark, 32K tokens.
        dict(name="norm_rope_prompt", kind="norm_rope", N=32768, Hq=32, Hkv=8, D=128, dtype="bf16", norm=True,
             far=32768),
        # A decode step of 64 sequences of different lengths, one fused projection row each, bounds kept.
        dict(name="append_tokens", kind="append", q_lens="1x64", kv_lens="2048x20,1777x20,64,65,1,1999x21", page=64,
             Hq=32, Hkv=8, D=128, dtype="bf16", norm=True, bounds=True),
        # Chunks of uneven prompts, some over a cached prefix, one sequence without new tokens, small pages.
        dict(name="append_ragged", kind="append", q_lens="2048,1,0,513,4096,77,300,1024",
             kv_lens="2048,4000,500,3001,4096,1234,316,5000", page=16, Hq=32, Hkv=8, D=128, dtype="bf16", norm=True,
             bounds=True),
        # Drafts of four tokens checked in one pass, eight sequences of 4K cached tokens.
        dict(name="chunk_drafts", kind="chunk", q_lens="4x8", kv_lens="4096x3,4001x5", page=64, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # A mixed batch: two prompts start, two go on, four sequences decode.
        dict(name="chunk_mixed", kind="chunk", q_lens="1024,700,512,333,1x4", kv_lens="1024,700,8192,5333,9000x2,16000,77",
             page=64, Hq=32, Hkv=8, D=128, dtype="bf16"),
        # Small pages, head dim 64, seven query heads to a KV head, fp16.
        dict(name="chunk_small_pages", kind="chunk", q_lens="999,2,0,1501", kv_lens="999,3000,100,4007", page=16, Hq=14,
             Hkv=2, D=64, dtype="fp16"),
        # The last 8K tokens of a 32K prompt that is taken chunk by chunk.
        dict(name="chunk_long", kind="chunk", q_lens="8192", kv_lens="32768", page=64, Hq=32, Hkv=8, D=128, dtype="bf16"),
        # One long sequence decodes over the 16 best of its pages.
        dict(name="select_one", kind="select", q_lens="1", kv_lens="32001", page=64, Hq=32, Hkv=8, D=128, dtype="bf16",
             top_k=16, sink=1, recent=2),
        # The decode benchmark's batch, 64 sequences of 16K tokens, 11 scored pages and 3 fixed ones each.
        dict(name="select_batch", kind="select", q_lens="1x64", kv_lens="16384x64", page=64, Hq=32, Hkv=8, D=128,
             dtype="bf16", top_k=11, sink=1, recent=2),
        # A chunk of 4K tokens after 28K cached ones, each block of 64 queries over its 48 best pages.
        dict(name="select_chunk", kind="select", q_lens="4096", kv_lens="32700", page=64, Hq=32, Hkv=8, D=128,
             dtype="bf16", top_k=48, sink=1, recent=2),
    ]


def _loguniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _text(lens):
    return ",".join(str(x) for x in lens)


def draw(rng):
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (8, 8), (16, 2), (14, 2), (12, 4), (9, 3), (8, 1), (40, 8)])
    base = dict(Hq=Hq, Hkv=Hkv, D=rng.choice([128, 128, 64]), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    kind = rng.choice(["norm_rope", "append", "chunk", "chunk", "select", "select"])
    if kind == "norm_rope":
        n = _loguniform(rng, 1, 32768 * 40 // (Hq + Hkv) if Hq + Hkv > 40 else 32768)
        return dict(kind=kind, N=n, norm=rng.random() < 0.7, far=_loguniform(rng, n + 1, 131072), **base)
    page = rng.choice([16, 32, 64, 64, 128])
    if kind == "append":
        B = _loguniform(rng, 1, 64)
        one = rng.random() < 0.4
        q_lens, kv_lens = [], []
        for _ in range(B):
            t = 1 if one else rng.choice([0, 1, _loguniform(rng, 1, 8192 // B)])
            q_lens.append(t)
            kv_lens.append(t + rng.choice([0, _loguniform(rng, 1, 4000), _loguniform(rng, 1, 4000)]))
        if not any(q_lens):
            q_lens[0], kv_lens[0] = 1, kv_lens[0] + 1
        return dict(kind=kind, q_lens=_text(q_lens), kv_lens=_text(kv_lens), page=page, norm=rng.random() < 0.7,
                    bounds=rng.random() < 0.6, **base)
    one = kind == "select" and rng.random() < 0.5
    if one:
        B = _loguniform(rng, 1, 64)
        kv_lens = [_loguniform(rng, 1, 16384) for _ in range(B)]
        q_lens = [1] * B
    else:
        B = _loguniform(rng, 1, 12)
        q_lens = [rng.choice([0, 1, _loguniform(rng, 1, 4096 // B), _loguniform(rng, 1, 4096 // B)]) for _ in range(B)]
        if not any(q_lens):
            q_lens[0] = 5
        kv_lens = [t + rng.choice([0, _loguniform(rng, 1, 16384 // (1 + B // 4))]) for t in q_lens]
    case = dict(kind=kind, q_lens=_text(q_lens), kv_lens=_text(kv_lens), page=page, **base)
    if kind == "select":
        case.update(top_k=rng.randint(1, 2048 // page), sink=rng.choice([0, 1, 1, 2]), recent=rng.choice([1, 2, 3]))
    return case


# ---- inputs -------------------------------------------------------------------------------------

def _lens(text):
    out = []
    for part in text.split(","):
        n, _, times = part.partition("x")
        out += [int(n)] * (int(times) if times else 1)
    return out


def _blocks(n):
    return -(-n // BLOCK)


def _randn(g, *shape, dtype, scale=1.0):
    x = torch.randn(*shape, generator=g, device=DEV, dtype=dtype)
    return x.mul_(scale) if scale != 1.0 else x


def _inv_freq(D):
    return (1.0 / THETA ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).to(torch.float32).to(DEV)


def _norm_weight(g, case, dtype):
    if not case["norm"]:
        return None
    return (1.0 + 0.3 * torch.randn(case["D"], generator=g, device=DEV)).to(dtype)


def _bounds_of(pages, lens, table, page):
    """[P, Hkv, 2, D]: minimum and maximum of the keys of each page, over the slots that hold tokens."""
    P = pages.size(0)
    used = torch.zeros(P, dtype=torch.long, device=DEV)
    for b, n in enumerate(lens):
        nb = -(-n // page)
        if nb:
            fill = torch.full((nb,), page, device=DEV)
            fill[-1] = n - (nb - 1) * page
            used[table[b, :nb].long()] = fill
    keep = (torch.arange(page, device=DEV)[None] < used[:, None])[:, None, :, None]
    inf = torch.finfo(pages.dtype).max
    lo = torch.where(keep, pages, inf).amin(2)
    hi = torch.where(keep, pages, -inf).amax(2)
    none = (used == 0)[:, None, None]
    return torch.stack([lo.masked_fill(none, 0), hi.masked_fill(none, 0)], dim=2)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    st = dict(case=case)
    if case["kind"] == "norm_rope":
        N = case["N"]
        st["q"] = _randn(g, N, Hq, D, dtype=dtype, scale=2.0)
        st["k"] = _randn(g, N, Hkv, D, dtype=dtype, scale=2.0)
        start = case["far"] - N
        st["positions"] = torch.arange(start, start + N, device=DEV)
        if N <= 64:                                       # single tokens of sequences of different lengths
            st["positions"] = torch.randint(0, case["far"], (N,), generator=g, device=DEV)
        st["inv_freq"] = _inv_freq(D)
        st["qw"], st["kw"] = _norm_weight(g, case, dtype), _norm_weight(g, case, dtype)
        return st
    q_lens, kv_lens, page = _lens(case["q_lens"]), _lens(case["kv_lens"]), case["page"]
    B, N = len(q_lens), sum(q_lens)
    max_blocks = max(1, -(-max(kv_lens) // page))
    need = [-(-n // page) for n in kv_lens]
    P = sum(need) + 2                                     # two pages belong to nobody
    order = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(B, max_blocks, dtype=torch.int32, device=DEV)
    at = 0
    for b, nb in enumerate(need):
        table[b, :nb] = order[at:at + nb]
        at += nb
    # Keys of one page are alike, as neighbouring tokens' are: a direction of the page plus noise.
    k_pages = _randn(g, P, Hkv, page, D, dtype=dtype, scale=0.7)
    k_pages += _randn(g, P, Hkv, 1, D, dtype=dtype, scale=0.7)
    st.update(q_lens=q_lens, kv_lens_host=kv_lens, N=N, table=table, k_pages=k_pages,
              v_pages=_randn(g, P, Hkv, page, D, dtype=dtype),
              kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device=DEV),
              cu=torch.tensor([sum(q_lens[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV))
    if case["kind"] == "append":
        qkv = _randn(g, N, (Hq + 2 * Hkv) * D, dtype=dtype, scale=2.0)
        st["q"], st["k"], st["v"] = (x.view(N, -1, D) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
        st["inv_freq"] = _inv_freq(D)
        st["qw"], st["kw"] = _norm_weight(g, case, dtype), _norm_weight(g, case, dtype)
        old = [n - t for n, t in zip(kv_lens, q_lens)]
        st["bounds"] = _bounds_of(k_pages, old, table, page) if case["bounds"] else None
    else:
        st["q"] = _randn(g, N, Hq, D, dtype=dtype)
        if case["kind"] == "select":
            st["bounds"] = _bounds_of(k_pages, kv_lens, table, page)
            st["tokens_only"] = all(t == 1 for t in q_lens)
    return st


# ---- one pass -----------------------------------------------------------------------------------

def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from sparseattentioninfer_amd import ops
    case = st["case"]
    kind = case["kind"]
    if kind == "norm_rope":
        return ops.qk_norm_rope(st["q"], st["k"], st["positions"], st["inv_freq"], q_weight=st["qw"], k_weight=st["kw"],
                                eps=EPS)
    if kind == "append":
        q_out = ops.paged_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["cu"], st["kv_lens"],
                                 inv_freq=st["inv_freq"], k_weight=st["kw"], eps=EPS, k_bounds=st["bounds"], q=st["q"],
                                 q_weight=st["qw"])
        return [x for x in (q_out, st["k_pages"], st["v_pages"], st["bounds"]) if x is not None]
    if kind == "chunk":
        return ops.paged_chunk_attn(st["q"], st["k_pages"], st["v_pages"], st["table"], st["cu"], st["kv_lens"])
    pick = dict(page=case["page"], top_k=case["top_k"], sink=case["sink"], recent=case["recent"])
    if st["tokens_only"]:
        sel, sel_off = ops.paged_block_select(st["q"], st["bounds"], st["table"], st["kv_lens"], **pick)
        out = ops.paged_sparse_decode(st["q"], st["k_pages"], st["v_pages"], st["table"], st["kv_lens"], sel, sel_off,
                                      num_splits=0)
    else:
        sel, sel_off = ops.paged_block_select(st["q"], st["bounds"], st["table"], st["kv_lens"], cu_seqlens=st["cu"],
                                              **pick)
        out = ops.paged_chunk_attn(st["q"], st["k_pages"], st["v_pages"], st["table"], st["cu"], st["kv_lens"],
                                   sel=sel, sel_off=sel_off)
    return sel, sel_off, out


def _plain_norm_rope(x, w, positions, inv_freq):
    """[N, H, D] -> the normed and rotated heads, rounded once."""
    f = x.float()
    if w is not None:
        f = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + EPS) * w.float()
    angle = positions.double()[:, None] * inv_freq.double()[None]           # far positions: 64 bits
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = f.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(x.dtype)


def _token_index(st):
    """(sequence, position) of every new token."""
    seq = torch.cat([torch.full((t,), b) for b, t in enumerate(st["q_lens"])]).long().to(DEV)
    pos = torch.cat([torch.arange(n - t, n) for t, n in zip(st["q_lens"], st["kv_lens_host"])]).to(DEV)
    return seq, pos


def _cached(st, pool, b, n):
    """[Hkv, n, D] float32: the first n cached tokens of sequence b."""
    page = st["case"]["page"]
    nb = -(-n // page)
    x = pool[st["table"][b, :nb].long()].float()                            # [nb, Hkv, page, D]
    return x.permute(1, 0, 2, 3).reshape(x.size(1), nb * page, -1)[:, :n]


def _plain_attention(st, keep=None):
    """[N, Hq, D]; keep[b]: [blocks, Hkv, pages] retained pages of sequence b's query blocks."""
    case, q = st["case"], st["q"]
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    G = case["Hq"] // Hkv
    out = torch.zeros_like(q)
    at = 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        if t == 0:
            continue
        k, v = _cached(st, st["k_pages"], b, n), _cached(st, st["v_pages"], b, n)
        step = max(BLOCK, (1 << 28) // (Hkv * G * n) // BLOCK * BLOCK)
        for r0 in range(0, t, step):
            r1 = min(t, r0 + step)
            x = q[at + r0:at + r1].float().view(r1 - r0, Hkv, G, D).permute(1, 0, 2, 3).reshape(Hkv, -1, D)
            s = torch.matmul(x, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(D)).view(Hkv, r1 - r0, G, n)
            seen = torch.arange(n, device=DEV)[None] <= torch.arange(n - t + r0, n - t + r1, device=DEV)[:, None]
            if keep is None:
                seen = seen[None, :, None]
            else:
                rows = keep[b][torch.arange(r0, r1, device=DEV) // BLOCK]    # [rows, Hkv, pages]
                seen = (seen[:, None] & rows.repeat_interleave(page, dim=2)[:, :, :n]).transpose(0, 1)[:, :, None]
            s.masked_fill_(~seen, -math.inf)
            m = s.amax(-1, keepdim=True)
            s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
            total = s.sum(-1, keepdim=True)
            o = torch.matmul(s.view(Hkv, -1, n), v).view(Hkv, r1 - r0, G, D) / total.clamp_min(1e-37)
            out[at + r0:at + r1] = o.permute(1, 0, 2, 3).reshape(r1 - r0, -1, D).to(q.dtype)
        at += t
    return out


def _block_limits(case, t, n):
    """First and last position of each of the query blocks of t new tokens that end a sequence of n."""
    first = torch.arange(n - t, n, BLOCK, device=DEV)
    return first, (first + BLOCK).clamp_max(n) - 1


def _keep_mask(case, score, first, last):
    """[rows, Hkv, pages] kept pages from their scores; row r's queries are at first[r] .. last[r]."""
    page, pages = case["page"], score.size(2)
    pg = torch.arange(pages, device=DEV)
    lo = (first // page - case["recent"] + 1).clamp_min(0)[:, None]
    end = (last // page)[:, None]
    fixed = ((pg < case["sink"]) | (pg >= lo)) & (pg <= end)                # [rows, pages]
    free = (pg >= case["sink"]) & (pg < lo)
    score = score.masked_fill(~free[:, None], -math.inf)
    order = score.sort(dim=2, descending=True, stable=True).indices[..., :case["top_k"]]
    best = torch.zeros_like(score, dtype=torch.bool).scatter_(2, order, True)
    return (best & free[:, None]) | fixed[:, None]


def _width(case, tokens_only):
    span = 1 if tokens_only else (BLOCK + case["page"] - 2) // case["page"] + 1
    return case["sink"] + case["top_k"] + case["recent"] - 1 + span


def _lists(keep, width):
    """Kept pages as ascending lists, padded with zeros, and their (0, length)."""
    pages = keep.size(2)
    idx = torch.where(keep, torch.arange(pages, device=DEV), pages).sort(dim=2).values
    if pages < width:
        idx = torch.cat([idx, idx.new_full((*idx.shape[:2], width - pages), pages)], dim=2)
    count = keep.sum(2)
    idx = idx[..., :width]
    off = torch.stack([torch.zeros_like(count), count], dim=2)
    return idx.masked_fill(idx >= pages, 0).to(torch.int32), off.to(torch.int32)


def _pooled(st, x):
    """Sums over groups of query heads of the positive and of the negative parts, 64 bits (a page's rank may
    hang on the last bits of its score): [rows, Hkv, D] each for x [rows, queries, Hq, D]."""
    case = st["case"]
    x = x.double().view(x.size(0), -1, case["Hkv"], case["Hq"] // case["Hkv"], case["D"])
    return x.clamp_min(0).sum((1, 3)), x.clamp_max(0).sum((1, 3))


def _plain_select(st):
    case = st["case"]
    page = case["page"]
    width = _width(case, st["tokens_only"])
    if st["tokens_only"]:
        pos, neg = _pooled(st, st["q"][:, None])
        bounds = st["bounds"][st["table"].long()].double()                  # [B, pages, Hkv, 2, D]
        lo, hi = bounds[:, :, :, 0].transpose(1, 2), bounds[:, :, :, 1].transpose(1, 2)
        score = (hi * pos[:, :, None]).sum(-1) + (lo * neg[:, :, None]).sum(-1)
        last = st["kv_lens"].long() - 1
        keep = _keep_mask(case, score, last, last)
        sel, off = _lists(keep, width)
        # attention over the lists
        B, Hkv, D, G = len(st["q_lens"]), case["Hkv"], case["D"], case["Hq"] // case["Hkv"]
        phys = st["table"].long()[:, None].expand(B, Hkv, -1).gather(2, sel.long())
        head = torch.arange(Hkv, device=DEV)[None, :, None]
        k, v = (p[phys, head].float().view(B, Hkv, width * page, D) for p in (st["k_pages"], st["v_pages"]))
        at = (sel.long() * page)[..., None] + torch.arange(page, device=DEV)
        live = torch.arange(width, device=DEV) < off[..., 1:2]
        seen = ((at <= last[:, None, None, None]) & live[..., None]).view(B, Hkv, 1, -1)
        q = st["q"].float().view(B, Hkv, G, D)
        s = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D))
        s = s.masked_fill(~seen, -math.inf)
        p = (s - s.amax(-1, keepdim=True)).exp()
        out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        return sel, off, out.view(B, case["Hq"], D).to(st["q"].dtype)
    B, N = len(st["q_lens"]), st["N"]
    rows = N // BLOCK + B
    sel = torch.zeros(rows, case["Hkv"], width, dtype=torch.int32, device=DEV)
    off = torch.zeros(rows, case["Hkv"], 2, dtype=torch.int32, device=DEV)
    keeps, at, row = [], 0, 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        if t == 0:
            keeps.append(None)
            continue
        nb = _blocks(t)
        x = torch.zeros(nb * BLOCK, case["Hq"], case["D"], device=DEV, dtype=st["q"].dtype)
        x[:t] = st["q"][at:at + t]
        pos, neg = _pooled(st, x.view(nb, BLOCK, case["Hq"], case["D"]))
        bounds = st["bounds"][st["table"][b, :-(-n // page)].long()].double().permute(2, 1, 3, 0)   # [2, Hkv, D, pages]
        score = torch.matmul(pos.transpose(0, 1), bounds[1]) + torch.matmul(neg.transpose(0, 1), bounds[0])
        keep = _keep_mask(case, score.transpose(0, 1), *_block_limits(case, t, n))
        sel[row:row + nb], off[row:row + nb] = _lists(keep, width)
        keeps.append(keep)
        at, row = at + t, row + nb
    return sel, off, _plain_attention(st, keeps)


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "norm_rope":
        return (_plain_norm_rope(st["q"], st["qw"], st["positions"], st["inv_freq"]),
                _plain_norm_rope(st["k"], st["kw"], st["positions"], st["inv_freq"]))
    if kind == "append":
        seq, pos = _token_index(st)
        q = _plain_norm_rope(st["q"], st["qw"], pos, st["inv_freq"])
        k = _plain_norm_rope(st["k"], st["kw"], pos, st["inv_freq"])
        page = case["page"]
        phys, slot = st["table"][seq, pos // page].long(), pos % page
        st["k_pages"][phys, :, slot] = k
        st["v_pages"][phys, :, slot] = st["v"]
        out = [q, st["k_pages"], st["v_pages"]]
        if st["bounds"] is not None:
            end = st["kv_lens"].long()[seq]
            fill = (end - pos // page * page).clamp_max(page)               # tokens of each written page
            keys = st["k_pages"][phys]                                      # [N, Hkv, page, D]
            keep = (torch.arange(page, device=DEV) < fill[:, None])[:, None, :, None]
            top = torch.finfo(keys.dtype).max
            st["bounds"][phys, :, 0] = torch.where(keep, keys, top).amin(2)
            st["bounds"][phys, :, 1] = torch.where(keep, keys, -top).amax(2)
            out.append(st["bounds"])
        return out
    if kind == "chunk":
        return _plain_attention(st)
    return _plain_select(st)


# ---- bytes and operations -----------------------------------------------------------------------

def _visible(case):
    """Sum over new tokens of the keys that each sees."""
    return sum(t * (n - t) + t * (t + 1) // 2 for t, n in zip(_lens(case["q_lens"]), _lens(case["kv_lens"])))


def _selected(case):
    """(keys that the queries see, pages in the lists, pages that are scored, rows) for one KV head."""
    page, tokens_only = case["page"], all(t == 1 for t in _lens(case["q_lens"]))
    seen = listed_pages = scored = rows = 0
    for t, n in zip(_lens(case["q_lens"]), _lens(case["kv_lens"])):
        for r in range(0, t, BLOCK):
            first, last = n - t + r, min(n - t + r + BLOCK, n) - 1
            lo = max(0, first // page - case["recent"] + 1)
            free = max(0, lo - case["sink"])
            head = min(case["sink"], lo)
            tail = last // page - max(lo, 0) + 1
            full = min(free, case["top_k"]) + head
            rows += 1
            scored += free if free > case["top_k"] else 0
            listed_pages += full + tail
            m = last - first + 1
            seen += m * (full * page + first - lo * page) + m * (m + 1) // 2
    return seen, listed_pages, scored, rows, tokens_only


def work(case):
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "norm_rope":
        n = case["N"] * (Hq + Hkv) * D
        return dict(bytes=4 * n + 8 * case["N"], flops=(8 if case["norm"] else 3) * n)
    q_lens, kv_lens, page = _lens(case["q_lens"]), _lens(case["kv_lens"]), case["page"]
    N = sum(q_lens)
    if case["kind"] == "append":
        n = N * (Hq + 2 * Hkv) * D
        extra = 0
        if case["bounds"]:
            for t, m in zip(q_lens, kv_lens):
                if t:
                    touched = (m - 1) // page - (m - t) // page + 1
                    extra += Hkv * 2 * D * 2 * (touched + ((m - t) % page > 0))
        return dict(bytes=4 * n + extra, flops=(8 if case["norm"] else 3) * N * (Hq + Hkv) * D)
    io = 4 * N * Hq * D
    if case["kind"] == "chunk":
        return dict(bytes=io + sum(n for t, n in zip(q_lens, kv_lens) if t) * Hkv * D * 4,
                    flops=4 * Hq * D * _visible(case))
    seen, listed_pages, scored, rows, tokens_only = _selected(case)
    # K and V of the listed pages: a single token's lists share nothing; blocks of queries share the cache.
    kv = listed_pages if tokens_only else min(listed_pages, sum(-(-n // page) for n in kv_lens))
    bounds = scored if tokens_only else min(scored, sum(-(-n // page) for n in kv_lens))
    return dict(bytes=io + Hkv * (kv * page * D * 4 + bounds * D * 4 + 4 * listed_pages),
                flops=4 * Hq * D * seen + 4 * Hkv * D * scored)


# ---- the definitions in float64 -----------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"norm_rope": _exact_norm_rope, "append": _exact_append, "chunk": _exact_chunk,
                "select": _exact_select}[case["kind"]](st)


def _exact_rotate(x, w, positions, inv_freq):
    z = x.double()
    if w is not None:
        z = z / (torch.linalg.vector_norm(z, dim=-1, keepdim=True).square() / z.size(-1) + EPS).sqrt() * w.double()
    half = z.size(-1) // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                       torch.outer(positions.double(), inv_freq.double()))
    z = torch.complex(z[..., :half], z[..., half:]) * turn[:, None]
    return torch.cat([z.real, z.imag], dim=-1)


def _exact_norm_rope(st):
    return tuple(_exact_rotate(st[x], st[x + "w"], st["positions"], st["inv_freq"]) for x in "qk")


def _exact_append(st):
    case = st["case"]
    page = case["page"]
    kp, vp = st["k_pages"].double(), st["v_pages"].double()
    bounds = None if st["bounds"] is None else st["bounds"].double()
    qs, at = [], 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        p = torch.arange(n - t, n, device=DEV)
        qs.append(_exact_rotate(st["q"][at:at + t], st["qw"], p, st["inv_freq"]))
        k = _exact_rotate(st["k"][at:at + t], st["kw"], p, st["inv_freq"])
        v = st["v"][at:at + t].double()
        at += t
        for lb in range((n - t) // page, -(-n // page)) if t else ():
            s0, s1 = max(0, n - t - lb * page), min(page, n - lb * page)
            r0 = lb * page + s0 - (n - t)
            pg = int(st["table"][b, lb])
            kp[pg, :, s0:s1] = k[r0:r0 + s1 - s0].transpose(0, 1)
            vp[pg, :, s0:s1] = v[r0:r0 + s1 - s0].transpose(0, 1)
            if bounds is not None:
                bounds[pg, :, 0] = kp[pg, :, :s1].min(dim=1).values
                bounds[pg, :, 1] = kp[pg, :, :s1].max(dim=1).values
    out = [torch.cat(qs), kp, vp]
    return out if bounds is None else out + [bounds]


def _exact_rows(q, k, v, ok):
    """Attention of rows q [R, D] over keys with visibility ok [R, L]."""
    logit = (q @ k.t()) / math.sqrt(q.size(1))
    logit = torch.where(ok, logit, -math.inf)
    lse = torch.logsumexp(logit, dim=1, keepdim=True)
    return torch.nan_to_num((logit - lse).exp(), nan=0.0) @ v


def _exact_attention(st, lists=None):
    case = st["case"]
    Hq, Hkv, page = case["Hq"], case["Hkv"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        if t == 0:
            continue
        j = torch.arange(n, device=DEV)
        phys, slot = st["table"][b].long()[j // page], j % page
        for h in range(Hq):
            g = h // (Hq // Hkv)
            k, v = st["k_pages"][phys, g, slot].double(), st["v_pages"][phys, g, slot].double()
            for r0 in range(0, t, 1024):
                r1 = min(t, r0 + 1024)
                ok = j[None] <= torch.arange(n - t + r0, n - t + r1, device=DEV)[:, None]
                if lists is not None:
                    ok &= lists[b][torch.arange(r0, r1, device=DEV) // BLOCK, g][:, j // page]
                out[at + r0:at + r1, h] = _exact_rows(st["q"][at + r0:at + r1, h].double(), k, v, ok)
        at += t
    return out


def _exact_chunk(st):
    return _exact_attention(st)


def _exact_select(st):
    case = st["case"]
    page, Hkv, G = case["page"], case["Hkv"], case["Hq"] // case["Hkv"]
    sink, recent, top_k = case["sink"], case["recent"], case["top_k"]
    if case["Hkv"] * sum(t * G * n // page for t, n in zip(st["q_lens"], st["kv_lens_host"])) * case["D"] > 1 << 37:
        return None
    rows, lists, at = [], {}, 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        pages = -(-n // page)
        lists[b] = torch.zeros(_blocks(t), Hkv, pages, dtype=torch.bool, device=DEV)
        lo_hi = st["bounds"][st["table"][b, :pages].long()].double()         # [pages, Hkv, 2, D]
        for i in range(_blocks(t)):
            r0, r1 = i * BLOCK, min(t, (i + 1) * BLOCK)
            first, last = n - t + r0, n - t + r1 - 1
            begin = max(0, first // page - recent + 1)
            q = st["q"][at + r0:at + r1].double().view(r1 - r0, Hkv, G, -1)
            score = torch.zeros(Hkv, pages, dtype=torch.float64, device=DEV)
            for g in range(Hkv):
                x = q[:, g].reshape(-1, 1, q.size(-1))                       # every query of the block
                step = max(1, (1 << 26) // (x.size(0) * x.size(2)))
                for p0 in range(0, pages, step):
                    e = lo_hi[p0:p0 + step, g]
                    score[g, p0:p0 + step] = torch.maximum(x * e[None, :, 0], x * e[None, :, 1]).sum(-1).sum(0)
            free = torch.arange(min(sink, begin), begin, device=DEV)
            for g in range(Hkv):
                rank = score[g, free].neg().argsort(stable=True)[:top_k]
                lists[b][i, g, free[rank]] = True
            lists[b][i, :, begin:last // page + 1] = True
            lists[b][i, :, :min(sink, last // page + 1)] = True
            rows.append(lists[b][i])
        at += t
    width = _width(case, st["tokens_only"])
    total = len(rows) if st["tokens_only"] else st["N"] // BLOCK + len(st["q_lens"])
    sel = torch.zeros(total, Hkv, width, dtype=torch.int32, device=DEV)
    off = torch.zeros(total, Hkv, 2, dtype=torch.int32, device=DEV)
    for i, kept in enumerate(rows):
        for g in range(Hkv):
            ids = kept[g].nonzero().flatten()
            sel[i, g, :len(ids)] = ids.to(torch.int32)
            off[i, g, 1] = len(ids)
    return sel, off, _exact_attention(st, lists)

"""Timed workloads of the operators on a paged cache that is held in 4 bits.

A cache of long contexts is read whole for every new token, so its bytes bound decoding.  Held in 4 bits with a
scale and a minimum per 32 dims it takes 3.2 times fewer.  Four operators work on it:

* ``append``  norms, rotation, quantisation and the write of a chunk's keys and values, one launch
              (``ops.paged_append_q4``), and the chunk read back as the values that the cache now stands for, which
              is what a model's own attention of a prompt goes on with (``ops.paged_read_q4``);
* ``read``    whole sequences read back into contiguous tensors (``ops.paged_read_q4``);
* ``chunk``   causal attention of packed new tokens over every page or over lists of them
              (``ops.paged_chunk_attn_q4``);
* ``decode``  one new token per sequence over lists of pages or over every page (``ops.paged_sparse_decode_q4``).

The form of a page: for each KV head one block of ``page * D * 5 / 8`` bytes.  32 dims of a token's head are a group,
held as ``m + s c`` with ``m`` its smallest value, ``s`` a fifteenth of its range (toward zero to the element type) and
``c = floor((x - m) / s + 1/2)``, at most 15.  First the codes.  Keys: ``D / 2`` bytes a token, of which byte
``4 ((D / 32) q + g) + e`` holds dims ``32 g + 8 q + e`` (low four bits) and ``32 g + 8 q + 4 + e`` (high), ``e < 4``.
Values: byte ``2 D (t // 4) + (D / 8) i + 4 g + t % 4`` holds dims ``32 g + i`` (low) and ``32 g + 16 + i`` (high) of token
``t``, ``i < 16``.  Then ``s`` and ``m`` of group ``g`` and token ``t`` as a pair of the element type, ``[D / 32, page, 2]``.

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
BLOCK = 64      # queries of a chunk that share one list of pages
GROUP = 32      # dims that share a scale
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # A decode step of 64 sequences of different lengths, one projection row each, bounds kept.
        dict(name="append_tokens", kind="append", q_lens="1x64", kv_lens="2048x20,1777x20,64,65,1,1999x21", page=64,
             Hq=32, Hkv=8, D=128, dtype="bf16", norm=True, bounds=True),
        # Chunks of uneven prompts, some over a cached prefix, one sequence without new tokens, small pages.
        dict(name="append_ragged", kind="append", q_lens="2048,1,0,513,4096,77,300,1024",
             kv_lens="2048,4000,500,3001,4096,1234,316,5000", page=16, Hq=32, Hkv=8, D=128, dtype="bf16", norm=True,
             bounds=False),
        # A short odd sequence with the head counts of a small model, read back for other code.
        dict(name="read_short", kind="read", kv_lens="333", page=16, Hq=14, Hkv=2, D=64, dtype="fp16"),
        # A batch of long contexts read back whole, one of them empty.
        dict(name="read_batch", kind="read", kv_lens="16384x3,9001,0,12345", page=64, Hq=32, Hkv=8, D=128, dtype="bf16"),
        # Drafts of four tokens checked in one pass, eight sequences of 4K cached tokens.
        dict(name="chunk_drafts", kind="chunk", q_lens="4x8", kv_lens="4096x3,4001x5", page=64, Hq=32, Hkv=8, D=128,
             dtype="bf16", keep=0),
        # A mixed batch: two prompts start, two go on, four sequences decode; fp16.
        dict(name="chunk_mixed", kind="chunk", q_lens="1024,700,512,333,1x4", kv_lens="1024,700,8192,5333,9000x2,16000,77",
             page=64, Hq=32, Hkv=8, D=128, dtype="fp16", keep=0),
        # A chunk of 4K tokens after 28K cached ones, each block of 64 queries over 51 of the pages.
        dict(name="chunk_selected", kind="chunk", q_lens="4096", kv_lens="32700", page=64, Hq=32, Hkv=8, D=128,
             dtype="bf16", keep=51),
        # The last 8K tokens of a 32K prompt that is taken chunk by chunk.
        dict(name="chunk_long", kind="chunk", q_lens="8192", kv_lens="32768", page=64, Hq=32, Hkv=8, D=128, dtype="bf16",
             keep=0),
        # A few short conversations with a small model: every page, small pages, seven query heads to a KV head.
        dict(name="decode_short", kind="decode", kv_lens="512x4,300,77,1,0", page=16, Hq=14, Hkv=2, D=64, dtype="fp16",
             keep=0),
        # One long sequence over its whole cache.
        dict(name="decode_one", kind="decode", kv_lens="32001", page=64, Hq=32, Hkv=8, D=128, dtype="bf16", keep=0),
        # The decode benchmark's batch, 64 sequences of 16K tokens, 14 pages kept of each.
        dict(name="decode_batch", kind="decode", kv_lens="16384x64", page=64, Hq=32, Hkv=8, D=128, dtype="bf16", keep=14),
        # Uneven long sequences over their whole caches, five query heads to a KV head.
        dict(name="decode_ragged", kind="decode", kv_lens="16000x6,777,9001x20,12345,64,30000", page=64, Hq=40, Hkv=8,
             D=128, dtype="bf16", keep=0),
    ]


def _loguniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _text(lens):
    return ",".join(str(x) for x in lens)


def draw(rng):
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (8, 8), (16, 2), (14, 2), (12, 4), (9, 3), (8, 1), (40, 8), (16, 1)])
    case = dict(kind=rng.choice(["append", "append", "read", "chunk", "chunk", "decode", "decode"]),
                page=rng.choice([16, 32, 48, 64, 64, 128]), Hq=Hq, Hkv=Hkv, D=rng.choice([128, 128, 64]),
                dtype=rng.choice(["bf16", "bf16", "fp16"]))
    kind, page = case["kind"], case["page"]
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
        case.update(q_lens=_text(q_lens), kv_lens=_text(kv_lens), norm=rng.random() < 0.7, bounds=rng.random() < 0.5)
    elif kind == "read":
        B = _loguniform(rng, 1, 32)
        case.update(kv_lens=_text([rng.choice([0, 1, _loguniform(rng, 1, 65536 // B)]) for _ in range(B - 1)]
                                  + [_loguniform(rng, 1, 65536 // B)]))
    elif kind == "decode":
        B = _loguniform(rng, 1, 64)
        kv_lens = [rng.choice([_loguniform(rng, 1, 16384), _loguniform(rng, 1, 1000)]) for _ in range(B)]
        case.update(kv_lens=_text(kv_lens), keep=rng.choice([0, rng.randint(1, 2048 // page)]))
    else:
        B = _loguniform(rng, 1, 12)
        q_lens = [rng.choice([0, 1, _loguniform(rng, 1, 4096 // B), _loguniform(rng, 1, 4096 // B)]) for _ in range(B)]
        if not any(q_lens):
            q_lens[0] = 5
        kv_lens = [t + rng.choice([0, _loguniform(rng, 1, 16384 // (1 + B // 4))]) for t in q_lens]
        case.update(q_lens=_text(q_lens), kv_lens=_text(kv_lens), keep=rng.choice([0, 0, rng.randint(2, 4096 // page)]))
    return case


# ---- inputs -------------------------------------------------------------------------------------

def _lens(text):
    out = []
    for part in text.split(","):
        n, _, times = part.partition("x")
        out += [int(n)] * (int(times) if times else 1)
    return out


def _new(case):
    """New tokens of each sequence: those of a chunk, one to a decoded sequence (none where it has no token), the whole
    of what is read."""
    if case["kind"] == "decode":
        return [min(n, 1) for n in _lens(case["kv_lens"])]
    return _lens(case["kv_lens" if case["kind"] == "read" else "q_lens"])


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
    return (1.0 + 0.1 * torch.randn(case["D"], generator=g, device=DEV)).to(dtype)


def _pool(g, P, case, dtype, alike):
    """A pool of pages [P, Hkv, bytes] with the codes of random keys or values, a part of the pages at a time.  Those of
    one page are alike, as neighbouring tokens' are: a direction of the page plus noise."""
    Hkv, page, D, kind = case["Hkv"], case["page"], case["D"], "k" if alike else "v"
    pool = torch.empty(P, Hkv, page * D * 5 // 8, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 25) // (Hkv * page * D))
    for p0 in range(0, P, step):
        n = min(P, p0 + step) - p0
        x = _randn(g, n, Hkv, page, D, dtype=dtype, scale=0.7 if alike else 1.0)
        if alike:
            x += _randn(g, n, Hkv, 1, D, dtype=dtype, scale=0.7)
        code, stats = _quantised(x)
        view_c, view_s = _views(pool[p0:p0 + n], page, D, dtype)[kind == "v"::2]
        view_c.copy_(_bytes_k(code) if alike else _bytes_v(code).unflatten(2, (page // 4, 4)).permute(0, 1, 2, 4, 5, 3))
        view_s.copy_(stats.transpose(2, 3))
    return pool


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    q_lens, kv_lens = _new(case), _lens(case["kv_lens"])
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
    st = dict(case=case, dtype=dtype, q_lens=q_lens, kv_lens_host=kv_lens, N=N, table=table,
              k_pages=_pool(g, P, case, dtype, True), v_pages=_pool(g, P, case, dtype, False),
              kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device=DEV),
              cu=torch.tensor([sum(q_lens[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV))
    if case["kind"] == "append":
        # Projections of normed states: bell-shaped with short tails.
        qkv = _randn(g, N, (Hq + 2 * Hkv) * D, dtype=dtype).clamp_(-2.0, 2.0)
        st["q"], st["k"], st["v"] = (x.view(N, -1, D) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
        st["inv_freq"] = _inv_freq(D)
        st["qw"], st["kw"] = _norm_weight(g, case, dtype), _norm_weight(g, case, dtype)
        st["bounds"] = None
        if case["bounds"]:
            old = torch.zeros(P, dtype=torch.long, device=DEV)                  # tokens that a page held before
            for b, (t, n) in enumerate(zip(q_lens, kv_lens)):
                nb = -(-(n - t) // page)
                old[table[b, :nb].long()] = (n - t - page * torch.arange(nb, device=DEV)).clamp_max(page)
            k = _values_k(_views(st["k_pages"], page, D, dtype), ...).to(dtype)  # [P, Hkv, page, D]
            none = (torch.arange(page, device=DEV) >= old[:, None])[:, None, :, None]
            ends = torch.stack([k.masked_fill(none, 60000.0).amin(2), k.masked_fill(none, -60000.0).amax(2)], 2)
            st["bounds"] = ends.masked_fill((old == 0)[:, None, None, None], 0.0)
    elif case["kind"] != "read":
        rows = B if case["kind"] == "decode" else N
        st["q"] = _randn(g, rows, Hq, D, dtype=dtype)
        st["sel"] = st["off"] = None
        if case["keep"]:
            st["sel"], st["off"] = _lists(g, case, q_lens, kv_lens, max_blocks)
    return st


def _lists(g, case, q_lens, kv_lens, max_blocks):
    """Ascending lists of up to ``keep`` pages, the last ones of the queries among them, zero-padded, for each block of
    queries (a decoded sequence is one block) and KV head, and their (0, length)."""
    page, Hkv, width = case["page"], case["Hkv"], case["keep"]
    decode = case["kind"] == "decode"
    last = torch.tensor([min(n - t + r + BLOCK, n) - 1 for t, n in zip(q_lens, kv_lens)
                         for r in range(0, 1 if decode else t, BLOCK)], device=DEV)
    rows = len(q_lens) if decode else sum(q_lens) // BLOCK + len(q_lens)
    end = torch.full((rows,), -1, dtype=torch.long, device=DEV)
    end[:last.numel()] = torch.div(last, page, rounding_mode="floor")
    pg = torch.arange(max_blocks, device=DEV)
    rank = torch.rand(rows, Hkv, max_blocks, generator=g, device=DEV)
    rank += (pg >= (end - BLOCK // page)[:, None])[:, None]
    rank.masked_fill_((pg > end[:, None])[:, None], -1.0)
    best = rank.topk(min(width, max_blocks), dim=2)
    idx = torch.where(best.values >= 0, best.indices, max_blocks).sort(dim=2).values
    count = (idx < max_blocks).sum(2)
    idx = torch.nn.functional.pad(idx.masked_fill(idx == max_blocks, 0), (0, width - idx.size(2)))
    return idx.to(torch.int32), torch.stack([torch.zeros_like(count), count], dim=2).to(torch.int32)


# ---- one pass -----------------------------------------------------------------------------------

def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from sparseattentioninfer_amd import ops
    case = st["case"]
    kind = case["kind"]
    cache = (st["k_pages"], st["v_pages"], st["table"])
    if kind == "decode":
        return ops.paged_sparse_decode_q4(st["q"], *cache, st["kv_lens"], st["sel"], st["off"])
    if kind == "chunk":
        return ops.paged_chunk_attn_q4(st["q"], *cache, st["cu"], st["kv_lens"], sel=st["sel"], sel_off=st["off"])
    back = dict(rows=st["N"], head_dim=case["D"], dtype=st["dtype"])
    if kind == "read":
        return ops.paged_read_q4(*cache, st["cu"], st["kv_lens"], **back)
    q_out = ops.paged_append_q4(st["k"], st["v"], *cache, st["cu"], st["kv_lens"], inv_freq=st["inv_freq"],
                                k_weight=st["kw"], eps=EPS, k_bounds=st["bounds"], q=st["q"], q_weight=st["qw"])
    k, v = ops.paged_read_q4(*cache, st["cu"], st["kv_lens"], **back)
    return [x for x in (q_out, k, v, st["bounds"]) if x is not None]


def _quantised(x):
    """Codes of x [..., D] (uint8) and the groups' (scale, minimum) [..., D / 32, 2] of x's type.  Values next to the
    border of two codes: 64 bits."""
    f = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    s = (hi - lo) / 15
    t = s.to(x.dtype)
    # toward zero: one step of the type down where the nearest is larger (as an integer, a positive value's bits)
    t = torch.where(t.double() > s, (t.view(torch.int16) - 1).view(x.dtype), t)
    code = torch.floor((f - lo) / torch.where(t == 0, 1.0, t.double()) + 0.5).clamp_(0, 15)
    code = torch.where(t == 0, 0.0, code)
    return code.to(torch.uint8).flatten(-2), torch.cat([t, lo.to(x.dtype)], dim=-1)


def _bytes_k(code):
    """[..., D] codes -> [..., D / 2] bytes of keys."""
    c = code.unflatten(-1, (-1, 4, 2, 4)).transpose(-4, -3)                     # [..., q, g, half, e]
    return (c[..., 0, :] | c[..., 1, :] << 4).flatten(-3)


def _bytes_v(code):
    """[..., D] codes -> [..., 16, D / 32] bytes of values of one token."""
    c = code.unflatten(-1, (-1, 2, 16))                                         # [..., g, half, i]
    return (c[..., 0, :] | c[..., 1, :] << 4).transpose(-1, -2)


def _views(pool, page, D, dtype):
    """Views of a pool: key bytes [P, Hkv, page, D / 2], value bytes [P, Hkv, page / 4, 16, D / 32, 4], and (scale,
    minimum) [P, Hkv, D / 32, page, 2], twice."""
    codes, stats = pool[..., :page * D // 2], pool[..., page * D // 2:].view(dtype)
    stats = stats.unflatten(-1, (D // GROUP, page, 2))
    return codes.unflatten(-1, (page, -1)), codes.unflatten(-1, (page // 4, 16, D // GROUP, 4)), stats, stats


def _scaled(code, stats):
    """m + s c in 32 bits: codes [..., D], stats [..., D / 32, 2]."""
    s = stats.float()
    return (code.float().unflatten(-1, (-1, GROUP)) * s[..., :1] + s[..., 1:]).flatten(-2)


def _values_k(views, at):
    """float32 keys [..., D] of pages (and heads, slots) `at`: an index of the views' leading dims, or ... for all."""
    b = views[0][at]
    c = torch.stack([b & 15, b >> 4], dim=-1).unflatten(-2, (4, -1, 4))         # [..., q, g, e, half]
    c = c.movedim(-3, -4).transpose(-1, -2).flatten(-4)
    return _scaled(c, views[2][at].transpose(-3, -2))


def _values_v(views, at):
    b = views[1][at].movedim(-1, -3).flatten(-4, -3)                            # [..., page, 16, g]
    c = torch.stack([b & 15, b >> 4], dim=-1).permute(*range(b.dim() - 2), -2 % (b.dim() + 1), -1 % (b.dim() + 1),
                                                      -3 % (b.dim() + 1)).flatten(-3)
    return _scaled(c, views[3][at].transpose(-3, -2))


def _plain_norm_rope(x, w, positions, inv_freq):
    """[N, H, D] -> the normed and rotated heads, rounded once.  In 64 bits: angles of far positions, and keys whose
    codes lie next to a border."""
    f = x.double()
    if w is not None:
        f = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
    angle = positions.double()[:, None] * inv_freq.double()[None]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = f.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(x.dtype)


def _token_index(st):
    """(page, slot) and position of every new token."""
    page = st["case"]["page"]
    n = (st["cu"][1:] - st["cu"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), n, output_size=st["N"])
    pos = torch.arange(st["N"], device=DEV) - st["cu"][seq] + st["kv_lens"][seq] - n[seq]
    return st["table"][seq, pos // page].long(), pos % page, pos


def _plain_read(st):
    """[N, Hkv, D] keys and values of the new tokens, of the element type."""
    case, dtype = st["case"], st["dtype"]
    page, D = case["page"], case["D"]
    phys, slot, _ = _token_index(st)
    kb, _, ks, _ = _views(st["k_pages"], page, D, dtype)
    _, vb, _, vs = _views(st["v_pages"], page, D, dtype)
    b = kb[phys, :, slot]                                                       # [N, Hkv, D / 2]
    c = torch.stack([b & 15, b >> 4], dim=-1).unflatten(2, (4, -1, 4)).permute(0, 1, 3, 2, 5, 4).flatten(2)
    k = _scaled(c, ks[phys, :, :, slot])
    b = vb[phys, :, slot // 4, :, :, slot % 4]                                  # [N, Hkv, 16, D / 32]
    c = torch.stack([b & 15, b >> 4], dim=-1).permute(0, 1, 3, 4, 2).flatten(2)
    return k.to(dtype), _scaled(c, vs[phys, :, :, slot]).to(dtype)


def _plain_append(st):
    case, dtype, bounds = st["case"], st["dtype"], st["bounds"]
    page, D = case["page"], case["D"]
    phys, slot, pos = _token_index(st)
    q = _plain_norm_rope(st["q"], st["qw"], pos, st["inv_freq"])
    kb, _, ks, _ = _views(st["k_pages"], page, D, dtype)
    _, vb, _, vs = _views(st["v_pages"], page, D, dtype)
    code, ks[phys, :, :, slot] = _quantised(_plain_norm_rope(st["k"], st["kw"], pos, st["inv_freq"]))
    kb[phys, :, slot] = _bytes_k(code)
    code, vs[phys, :, :, slot] = _quantised(st["v"])
    vb[phys, :, slot // 4, :, :, slot % 4] = _bytes_v(code)
    k, v = _plain_read(st)
    if bounds is None:
        return [q, k, v]
    # a page whose first slot is written gets fresh bounds, another has the new keys merged into its own
    fresh = phys[slot == 0]
    bounds[fresh, :, 0], bounds[fresh, :, 1] = math.inf, -math.inf
    at = phys[:, None, None].expand_as(k)
    bounds[:, :, 0] = bounds[:, :, 0].scatter_reduce(0, at, k, "amin")
    bounds[:, :, 1] = bounds[:, :, 1].scatter_reduce(0, at, k, "amax")
    return [q, k, v, bounds]


def _softmax_rows(s, seen):
    """exp of scores [..., n] against their largest, 0 where a key is not seen, and the sums."""
    s = s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    return s, s.sum(-1, keepdim=True).clamp_min(1e-37)


def _plain_chunk(st):
    case, q, dtype = st["case"], st["q"], st["dtype"]
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    G = case["Hq"] // Hkv
    kviews, vviews = _views(st["k_pages"], page, D, dtype), _views(st["v_pages"], page, D, dtype)
    out = torch.zeros_like(q)
    at = row = 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        if t == 0:
            continue
        pages = st["table"][b, :-(-n // page)].long()
        k, v = (x.transpose(0, 1).flatten(1, 2)[:, :n] for x in (_values_k(kviews, pages), _values_v(vviews, pages)))
        k = k.transpose(1, 2).contiguous()
        keep = None
        if st["sel"] is not None:
            sel, off = (x[row:row + _blocks(t)].long() for x in (st["sel"], st["off"]))
            live = torch.arange(sel.size(2), device=DEV) < off[..., 1:]
            keep = torch.zeros(*sel.shape[:2], pages.numel() + 1, dtype=torch.bool, device=DEV)
            keep.scatter_(2, torch.where(live, sel, pages.numel()), True)
            row += _blocks(t)
        step = max(BLOCK, (1 << 28) // (Hkv * G * n) // BLOCK * BLOCK)
        for r0 in range(0, t, step):
            r1 = min(t, r0 + step)
            x = q[at + r0:at + r1].float().view(r1 - r0, Hkv, G, D).permute(1, 0, 2, 3).reshape(Hkv, -1, D)
            s = torch.matmul(x, k).mul_(1.0 / math.sqrt(D)).view(Hkv, r1 - r0, G, n)
            seen = (torch.arange(n, device=DEV) <= torch.arange(n - t + r0, n - t + r1, device=DEV)[:, None])[None, :, None]
            if keep is not None:
                rows = keep[torch.arange(r0, r1, device=DEV) // BLOCK]          # [rows, Hkv, pages]
                seen = seen & rows[..., :-1].repeat_interleave(page, dim=2)[:, :, :n].transpose(0, 1)[:, :, None]
            p, total = _softmax_rows(s, seen)
            o = torch.matmul(p.view(Hkv, -1, n), v).view(Hkv, r1 - r0, G, D) / total
            out[at + r0:at + r1] = o.permute(1, 0, 2, 3).reshape(r1 - r0, -1, D).to(q.dtype)
        at += t
    return out


def _plain_decode(st):
    case, q, dtype = st["case"], st["q"], st["dtype"]
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    kviews, vviews = _views(st["k_pages"], page, D, dtype), _views(st["v_pages"], page, D, dtype)
    B = q.size(0)
    head = torch.arange(Hkv, device=DEV)[:, None]
    out = torch.empty_like(q)
    width = st["table"].size(1) if st["sel"] is None else st["sel"].size(2)
    step = max(1, (1 << 27) // (width * Hkv * page * D))                        # sequences at a time
    for b0 in range(0, B, step):
        part = slice(b0, min(B, b0 + step))
        lens = st["kv_lens"][part].long()
        if st["sel"] is None:
            lb = torch.arange(width, device=DEV).expand(lens.numel(), Hkv, width)
            live = lb * page < lens[:, None, None]
        else:
            lb = st["sel"][part].long()
            live = torch.arange(width, device=DEV) < st["off"][part][..., 1:]
        phys = st["table"][part].long()[:, None].expand(-1, Hkv, -1).gather(2, lb)
        k, v = (f(w, (phys, head)).flatten(2, 3) for f, w in ((_values_k, kviews), (_values_v, vviews)))
        seen = ((lb * page)[..., None] + torch.arange(page, device=DEV) < lens[:, None, None, None]) & live[..., None]
        x = q[part].float().unflatten(1, (Hkv, -1))
        s = torch.matmul(x, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(D))
        p, total = _softmax_rows(s, seen.flatten(2)[:, :, None])
        out[part] = (torch.matmul(p, v) / total).flatten(1, 2).to(q.dtype)
    return out


def _run_plain(st):
    return {"append": _plain_append, "read": _plain_read, "chunk": _plain_chunk, "decode": _plain_decode}[st["case"]["kind"]](st)


# ---- bytes and operations -----------------------------------------------------------------------

def work(case):
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    q_lens, kv_lens = _new(case), _lens(case["kv_lens"])
    N = sum(q_lens)
    head = D * 5 // 8                                                           # bytes of a token's head in the cache
    if case["kind"] == "read":
        return dict(bytes=2 * N * Hkv * (head + 2 * D), flops=4 * N * Hkv * D)
    if case["kind"] == "append":
        # q in and out, k and v in, their codes out; then codes in and k and v out
        n = N * (4 * Hq * D + 2 * Hkv * (2 * D + head) + 2 * Hkv * (2 * D + head))
        if case["bounds"]:
            n += sum(4 * Hkv * D * ((m - 1) // page - (m - t) // page + 1 + ((m - t) % page > 0))
                     for t, m in zip(q_lens, kv_lens) if t)
        return dict(bytes=n, flops=N * D * ((8 if case["norm"] else 3) * (Hq + Hkv) + 12 * Hkv))
    keys = pairs = ids = 0            # cached tokens read; (query, key) pairs; list entries
    for t, n in zip(q_lens, kv_lens):
        if not case["keep"]:
            keys += n if t else 0
            pairs += t * (n - t) + t * (t + 1) // 2
            continue
        lists = 0
        for r in range(0, t, BLOCK):
            m = min(t - r, BLOCK)
            last = n - t + r + m
            pages = min(case["keep"], -(-last // page))
            lists += pages
            pairs += m * max(1, pages * page - (-last % page) - m) + m * (m + 1) // 2
        keys += min(lists * page, n)
        ids += lists
    return dict(bytes=4 * (N if case["kind"] == "chunk" else len(kv_lens)) * Hq * D + 2 * Hkv * keys * head + 4 * Hkv * ids,
                flops=4 * Hq * D * pairs)


# ---- the definitions in float64 -----------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"append": _exact_append, "read": _exact_read, "chunk": _exact_chunk, "decode": _exact_decode}[case["kind"]](st)


def _exact_cached(st, name, b, g, j):
    """Keys or values of positions j of sequence b, KV head g, byte by byte from the form of a page: [len(j), D]."""
    page, D = st["case"]["page"], st["case"]["D"]
    block = st[name][st["table"][b].long()[torch.div(j, page, rounding_mode="floor")], g]
    t, d = (j % page)[:, None], torch.arange(D, device=DEV)[None]
    group, within = d // 32, d % 32
    if name == "k_pages":
        byte = t * (D // 2) + 4 * ((D // 32) * (within // 8) + group) + within % 4
        high = within % 8 >= 4
    else:
        byte = t // 4 * (2 * D) + (D // 8) * (within % 16) + 4 * group + t % 4
        high = within >= 16
    c = block.gather(1, byte).long()
    c = torch.where(high, c // 16, c % 16).double()
    stat = block[:, page * D // 2:].contiguous().view(st["dtype"]).double()
    return stat.gather(1, 2 * (group * page + t)) * c + stat.gather(1, 2 * (group * page + t) + 1)


def _exact_read(st):
    N, Hkv, D = st["N"], st["case"]["Hkv"], st["case"]["D"]
    out = [torch.empty(N, Hkv, D, dtype=torch.float64, device=DEV) for _ in "kv"]
    at = 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        for g in range(Hkv if t else 0):
            for o, name in zip(out, ("k_pages", "v_pages")):
                o[at:at + t, g] = _exact_cached(st, name, b, g, torch.arange(n - t, n, device=DEV))
        at += t
    return out


def _exact_rotate(x, w, positions, inv_freq):
    z = x.double()
    if w is not None:
        z = z / (torch.linalg.vector_norm(z, dim=-1, keepdim=True).square() / z.size(-1) + EPS).sqrt() * w.double()
    half = z.size(-1) // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                       torch.outer(positions.double(), inv_freq.double()))
    z = torch.complex(z[..., :half], z[..., half:]) * turn[:, None]
    return torch.cat([z.real, z.imag], dim=-1)


def _exact_held(x, dtype):
    """What the cache holds of x [N, H, D], whose elements are of the type."""
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    x = x.to(dtype).double()
    bits = {torch.bfloat16: 8, torch.float16: 11}[dtype]
    least = {torch.bfloat16: -133, torch.float16: -24}[dtype]                   # exponent of the smallest step
    for d in range(0, x.size(-1), 32):
        part = x[..., d:d + 32]
        low = part.min(dim=-1, keepdim=True).values
        width = (part.max(dim=-1, keepdim=True).values - low) / 15
        unit = torch.exp2((torch.frexp(width).exponent - bits).clamp_min(least).double())
        width = (width / unit).trunc() * unit
        steps = torch.where(width > 0, (part - low) / width, 0.0)
        steps = steps.floor() + (steps - steps.floor() >= 0.5)
        out[..., d:d + 32] = low + width * steps.clamp_max(15)
    return out


def _exact_append(st):
    page, dtype = st["case"]["page"], st["dtype"]
    bounds = None if st["bounds"] is None else st["bounds"].double()
    qs, ks, at = [], [], 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        p = torch.arange(n - t, n, device=DEV)
        qs.append(_exact_rotate(st["q"][at:at + t], st["qw"], p, st["inv_freq"]))
        k = _exact_held(_exact_rotate(st["k"][at:at + t], st["kw"], p, st["inv_freq"]), dtype)
        ks.append(k)
        at += t
        for lb in range((n - t) // page, -(-n // page)) if t and bounds is not None else ():
            first = lb * page - (n - t)
            new = k[max(0, first):first + page]
            pg = int(st["table"][b, lb])
            ends = [new.min(dim=0).values, new.max(dim=0).values]
            if first < 0:
                ends = [torch.minimum(ends[0], bounds[pg, :, 0]), torch.maximum(ends[1], bounds[pg, :, 1])]
            bounds[pg] = torch.stack(ends, dim=1)
    out = [torch.cat(qs), torch.cat(ks), _exact_held(st["v"].double(), dtype)]
    return out if bounds is None else out + [bounds]


def _exact_rows(q, k, v, ok):
    """Attention of rows q [R, D] over keys with visibility ok [R, L]; 0 for a row that sees none."""
    logit = (q @ k.t()) / math.sqrt(q.size(1))
    logit = torch.where(ok, logit, -math.inf)
    lse = torch.logsumexp(logit, dim=1, keepdim=True)
    return torch.nan_to_num((logit - lse).exp(), nan=0.0) @ v


def _exact_chunk(st):
    case = st["case"]
    Hq, Hkv, page = case["Hq"], case["Hkv"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    at = row = 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["kv_lens_host"])):
        j = torch.arange(n, device=DEV)
        for g in range(Hkv if t else 0):
            k, v = (_exact_cached(st, name, b, g, j) for name in ("k_pages", "v_pages"))
            for r0 in range(0, t, 1024):
                r1 = min(t, r0 + 1024)
                ok = j[None] <= torch.arange(n - t + r0, n - t + r1, device=DEV)[:, None]
                if st["sel"] is not None:
                    listed_pages = torch.zeros(_blocks(r1 - r0), -(-n // page), dtype=torch.bool, device=DEV)
                    for i in range(_blocks(r1 - r0)):
                        r = row + r0 // BLOCK + i
                        listed_pages[i, st["sel"][r, g, :int(st["off"][r, g, 1])].long()] = True
                    ok &= listed_pages[torch.arange(r1 - r0, device=DEV) // BLOCK][:, j // page]
                for h in range(g * Hq // Hkv, (g + 1) * Hq // Hkv):
                    out[at + r0:at + r1, h] = _exact_rows(st["q"][at + r0:at + r1, h].double(), k, v, ok)
        at, row = at + t, row + _blocks(t)
    return out


def _exact_decode(st):
    case = st["case"]
    Hq, Hkv, page = case["Hq"], case["Hkv"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["kv_lens_host"]):
        for g in range(Hkv if n else 0):
            j = torch.arange(n, device=DEV)
            if st["sel"] is not None:
                ids = st["sel"][b, g, :int(st["off"][b, g, 1])].long()
                j = (ids[:, None] * page + torch.arange(page, device=DEV)).flatten()
                j = j[j < n]
            k, v = (_exact_cached(st, name, b, g, j) for name in ("k_pages", "v_pages"))
            rows = slice(g * Hq // Hkv, (g + 1) * Hq // Hkv)
            out[b, rows] = _exact_rows(st["q"][b, rows].double(), k, v, torch.ones((), dtype=torch.bool, device=DEV))
    return out

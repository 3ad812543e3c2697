"""Plain float64 forms of the chunk operators, on the CPU, and ragged paged inputs for their tests."""
from __future__ import annotations

import math

import torch

BLOCK = 64


def half_step(dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def randn(*shape, seed, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


class Ragged:
    """A paged cache of random tokens with a shuffled table, and the lengths of a call, on the CPU."""

    def __init__(self, q_lens, kv_lens, *, page, Hkv, D, dtype=torch.bfloat16, seed=0, extra_cols=1, pad_rows=0,
                 poison=True):
        self.q_lens, self.lens, self.page, self.Hkv, self.D, self.dtype = q_lens, kv_lens, page, Hkv, D, dtype
        B = len(q_lens)
        need = [-(-n // page) for n in kv_lens]
        P = sum(need) + 2
        g = torch.Generator().manual_seed(seed)
        order = torch.randperm(P, generator=g)
        self.table = torch.zeros(B, max(1, max(need)) + extra_cols, dtype=torch.int32)
        at = 0
        for b, nb in enumerate(need):
            self.table[b, :nb] = order[at:at + nb].to(torch.int32)
            at += nb
        self.k_pages = randn(P, Hkv, page, D, seed=seed + 1, dtype=dtype)
        self.v_pages = randn(P, Hkv, page, D, seed=seed + 2, dtype=dtype)
        if poison:      # slots that hold no token: a kernel that lets them in shows NaN
            held = torch.zeros(P, page, dtype=torch.bool)
            for b, n in enumerate(kv_lens):
                for lb in range(need[b]):
                    held[self.table[b, lb].item(), :min(page, n - lb * page)] = True
            for pool in (self.k_pages, self.v_pages):
                pool.masked_fill_(~held[:, None, :, None], math.nan)
        self.cu = torch.tensor([sum(q_lens[:b]) for b in range(B + 1)], dtype=torch.int32)
        self.kv_lens = torch.tensor(kv_lens, dtype=torch.int32)
        self.N = sum(q_lens) + pad_rows

    def rows(self):
        """(sequence, first packed row, new tokens, tokens in all)."""
        at = 0
        for b, (t, n) in enumerate(zip(self.q_lens, self.lens)):
            yield b, at, t, n
            at += t

    def cached(self, pool, b, n):
        nb = -(-n // self.page)
        x = pool[self.table[b, :nb].long()].double()
        return x.permute(1, 0, 2, 3).reshape(self.Hkv, nb * self.page, self.D)[:, :n]

    def gpu(self, *names):
        return [getattr(self, x).cuda() for x in names]


def rotate(x, w, positions, inv_freq, eps):
    """float64 norm and rotation of [N, H, D]; also the sum of the magnitudes of each output's two terms."""
    f = x.double()
    if w is not None:
        f = f / (f.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if inv_freq is None:
        return f, f.abs()
    ang = positions.double()[..., None] * inv_freq.double()
    c, s = ang.cos()[..., None, :], ang.sin()[..., None, :]
    a, b = f.chunk(2, dim=-1)
    y = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return y, torch.cat([a.abs() + b.abs()] * 2, dim=-1)


def assert_rotated(got, want, terms, what):
    """One rounding of the result, and fp32 arithmetic before it: the square mean over D terms, its root, two
    products by a weight and the norm, the rotation's two products and sum and cos and sin, each relative 2^-24
    of the two terms it works on, together below 2^-20 of them."""
    got, h = got.double().cpu(), half_step(got.dtype)
    err = (got - want).abs()
    tol = (h * want.abs() + 2.0 ** -20 * terms) * (1 + h) + torch.finfo(torch.float16).tiny * 2.0 ** -10
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {(err - tol).max():.3e} past the bound"


def attention(r: Ragged, q, sel=None, sel_off=None):
    """float64 attention of the packed queries, the bound of its error, and which rows belong to a sequence."""
    Hq = q.size(1)
    G = Hq // r.Hkv
    want = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(want)
    live = torch.zeros(q.size(0), dtype=torch.bool)
    blk0 = 0
    slop = torch.zeros_like(want)
    for b, at, t, n in r.rows():
        if t == 0:
            continue
        live[at:at + t] = True
        k, v = r.cached(r.k_pages, b, n), r.cached(r.v_pages, b, n)
        for i in range(t):
            p = n - t + i
            if p < 0:
                continue
            for g in range(r.Hkv):
                ok = torch.arange(n) <= p
                if sel is not None:
                    lo, hi = sel_off[blk0 + i // BLOCK, g].tolist()
                    pages = torch.zeros(-(-n // r.page), dtype=torch.bool)
                    pages[sel[blk0 + i // BLOCK, g, lo:hi].long()] = True
                    ok &= pages.repeat_interleave(r.page)[:n]
                if not ok.any():
                    continue
                x = q[at + i, g * G:(g + 1) * G].double()
                kk, vv = k[g, ok], v[g, ok]
                w = torch.softmax(x @ kk.T / math.sqrt(r.D), dim=-1)
                want[at + i, g * G:(g + 1) * G] = w @ vv
                mag[at + i, g * G:(g + 1) * G] = w @ vv.abs()
                if q.dtype == torch.float16:     # probabilities below 2^-14 of the reference: steps of 2^-24
                    slop[at + i, g * G:(g + 1) * G] = kk.size(0) * 2.0 ** -25 * vv.abs().max()
        blk0 += -(-t // BLOCK)
    # Each probability is rounded once (half a step of it), the output once more.  Scores are fp32 sums of D
    # products, off by at most D 2^-24 of sum |q k| scale < 16 here, so probabilities by 2 * 16 * D 2^-24 relative.
    h = half_step(q.dtype)
    tol = (h * mag + 32 * r.D * 2.0 ** -24 * mag + slop) * (1 + h) + h * want.abs() * (1 + h) + 1e-7
    return want, tol, live


def select(r: Ragged, q, bounds, *, top_k, sink, recent, tokens):
    """(sel, sel_off) by the definition: for every list the sum over its queries of the bound of q . k."""
    G = q.size(1) // r.Hkv
    lists = []
    for b, at, t, n in (((b, b, 1, n) for b, n in enumerate(r.lens)) if tokens else r.rows()):
        for r0 in range(0, t, BLOCK):
            first, last = n - t + r0, n - t + min(t, r0 + BLOCK) - 1
            x = q[at + r0:at + min(t, r0 + BLOCK)].double().view(-1, r.Hkv, G, r.D)
            pages = last // r.page + 1 if last >= 0 else 0
            lo = min(pages, max(0, max(first, 0) // r.page - recent + 1))
            per_head = []
            for g in range(r.Hkv):
                free = list(range(min(sink, lo), lo))
                e = bounds[r.table[b, free].long(), g].double()                 # [free, 2, D]
                xx = x[:, g].reshape(-1, 1, r.D)
                score = torch.maximum(xx * e[None, :, 0], xx * e[None, :, 1]).sum(-1).sum(0)
                best = sorted(range(len(free)), key=lambda i: (-score[i].item(), i))[:top_k]
                per_head.append(sorted(list(range(min(sink, lo))) + [free[i] for i in best] + list(range(lo, pages))))
            lists.append(per_head)
    N, B = q.size(0), len(r.lens)
    rows = B if tokens else N // BLOCK + B
    span = 1 if tokens else (BLOCK + r.page - 2) // r.page + 1
    sel = torch.zeros(rows, r.Hkv, sink + top_k + recent - 1 + span, dtype=torch.int32)
    off = torch.zeros(rows, r.Hkv, 2, dtype=torch.int32)
    for i, per_head in enumerate(lists):
        for g, pages in enumerate(per_head):
            sel[i, g, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            off[i, g, 1] = len(pages)
    return sel, off


def bounds_of(r: Ragged):
    """[P, Hkv, 2, D] over the slots that hold tokens; pages without any: zeros."""
    out = torch.zeros(r.k_pages.size(0), r.Hkv, 2, r.D, dtype=r.dtype)
    for b, n in enumerate(r.lens):
        for lb in range(-(-n // r.page)):
            pg = r.table[b, lb].item()
            k = r.k_pages[pg, :, :min(r.page, n - lb * r.page)]
            out[pg, :, 0], out[pg, :, 1] = k.amin(1), k.amax(1)
    return out

"""Attention over a 4-bit cache in float64 and how far the kernels may be from it, row by row and dim by dim: bounds that the
weights and the cache at hand give, so that a wrong weight shows whatever the values' size or offset."""
from __future__ import annotations

import math

import torch

from tests.chunk_reference import half_step, randn
from tests.q4_reference import Q4Ragged, pack, places, stats_of, unpack

F32 = 2.0 ** -24


def cache_of(q_lens, kv_lens, *, page, Hkv, D, dtype, seed, k_offset=0.0, v_offset=0.0, k_scale=1.0, v_scale=1.0, pad_rows=0):
    """A ragged cache whose keys and values have an offset and a scale of their own."""
    r = Q4Ragged(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=seed, pad_rows=pad_rows)
    hold = r.held[:, None, :, None]
    for name, pool, scale, offset in (("k", r.k4, k_scale, k_offset), ("v", r.v4, v_scale, v_offset)):
        x = (randn(*r.k_pages.shape, seed=seed + ord(name), dtype=torch.float32) * scale + offset).to(dtype)
        fresh, values = pack(x, name == "v"), name == "v"
        byte = _bytes(page, D, values)                                          # [page, bytes of a token]
        for p in range(pool.size(0)):
            for t in r.held[p].nonzero().flatten().tolist():
                pool[p, :, byte[t]] = fresh[p, :, byte[t]]
        back = unpack(pool, page, D, dtype, values)
        setattr(r, name + "_pages", torch.where(hold, back, math.nan))
    return r


def _bytes(page, D, values):
    byte, _ = places(page, D, values)
    stats = page * D // 2 + 4 * (torch.arange(D // 32)[None] * page + torch.arange(page)[:, None])
    return torch.cat([byte, *(stats + i for i in range(4))], dim=1)


def _spread(x):
    """[P, Hkv, page, D / 32] -> [P, Hkv, page, D]."""
    return x.double().repeat_interleave(32, dim=-1)


def forms(r, q, sel=None, sel_off=None, *, codes: bool, scale=None):
    """(want, tol, seen) of rows: float64 attention over m + s c and the bound of a kernel that multiplies codes (``codes``)
    or over m + s c rounded to the element type and that of one that multiplies those; seen counts each row's keys.

    With w the weights and o the output, a relative error e_j of each weight moves o by sum w_j e_j (v_j - o).  e_j: the score's
    fp32 sum of at most 2 D + 16 terms, of magnitudes that add up to a_j, is off by (2 D + 16) 2^-24 a_j; the argument of the
    exponential, (score - reference) log2 e, by 2^-22 of the largest score for its scale, product and difference, and the
    hardware's 2^x by 2^-22.  Codes: p s is rounded to bf16, by 2^-8 of it, and meets |c - 7.5| <= 7.5 (fp16: the rest is
    rounded to bf16 and added, so 2^-16 of it meets c <= 15).  Else p is rounded to the element type and meets v, in fp16 to steps of 2^-24 where it is
    small.  Sums over n keys and the merges are fp32: n + 128 roundings of the magnitudes.  The output is rounded once."""
    h, dt = half_step(r.dtype), r.dtype
    scale = r.D ** -0.5 if scale is None else scale
    G = q.size(1) // r.Hkv
    round_ = (lambda x: x) if codes else (lambda x: x.float().to(dt).double())
    kp, vp = round_(r.k_pages), round_(r.v_pages)
    (ks, km), (vs, vm) = (tuple(_spread(x) for x in stats_of(p, r.page, r.D, dt)) for p in (r.k4, r.v4))
    want = torch.zeros(q.shape, dtype=torch.float64)
    tol, seen = torch.zeros_like(want), torch.zeros(q.shape[:2], dtype=torch.int64)
    blk0 = 0
    for b, at, t, n in r.rows():
        if t == 0:
            continue
        k, v, ks_, km_, vs_, vm_ = (r.cached(x, b, n) for x in (kp, vp, ks, km, vs, vm))
        for i in range(t):
            p = n - t + i
            for g in range(r.Hkv):
                ok = torch.arange(n) <= p
                if sel is not None:
                    lo, hi = sel_off[blk0 + i // 64, g].tolist()
                    pages = torch.zeros(-(-n // r.page), dtype=torch.bool)
                    pages[sel[blk0 + i // 64, g, lo:hi].long()] = True
                    ok &= pages.repeat_interleave(r.page)[:n]
                heads = slice(g * G, (g + 1) * G)
                seen[at + i, heads] = int(ok.sum())
                if not ok.any():
                    continue
                x, kk, vv = q[at + i, heads].double(), k[g, ok], v[g, ok]
                score = x @ kk.T * scale
                w = torch.softmax(score, dim=-1)                                # [G, n]
                o = w @ vv
                if codes:
                    a = x.abs() @ (15 * ks_[g, ok] + km_[g, ok].abs()).T * scale
                else:
                    a = x.abs() @ kk.abs().T * scale
                e = ((2 * r.D + 16) * F32 * a + (score.abs().amax(-1, keepdim=True) + 1) * 2.0 ** -22)
                weights = torch.stack([(w[y, :, None] * e[y, :, None] * (vv - o[y]).abs()).sum(0) for y in range(x.size(0))])
                count = int(ok.sum()) + 128
                if codes:
                    ws = w @ vs_[g, ok]
                    step = 2.0 ** -8 * 7.5 * ws if dt == torch.bfloat16 else 2.0 ** -16 * 15 * ws
                    sums = count * F32 * (w @ vm_[g, ok].abs() + 22.5 * ws)
                else:
                    mag = w @ vv.abs()
                    step = h * mag + (count * 2.0 ** -25 * vv.abs().max() if dt == torch.float16 else 0.0)
                    sums = count * F32 * mag
                inner = 1.01 * (weights + step + sums)      # second order: e and the steps are below 2^-7 of it
                want[at + i, heads] = o
                tol[at + i, heads] = inner + h * (o.abs() + inner) + torch.finfo(torch.float16).tiny * 2.0 ** -10
        blk0 += -(-t // 64)
    return want, tol, seen


def good_rows(got, bounds):
    """[N, Hq]: rows within one of the bounds."""
    ok = None
    for want, tol, _ in bounds:
        row = ((got.double().cpu() - want).abs() <= tol).all(-1)
        ok = row if ok is None else ok | row
    return ok


def wrong_outputs(r, bounds):
    """Outputs that no bound may pass: nothing, nine tenths, the mean of all outputs, another head's."""
    want = bounds[0][0]
    out = dict(zeros=torch.zeros_like(want), tenth=0.9 * want, mean=want.mean().expand_as(want).clone())
    if want.size(1) > 1:
        out["heads"] = want.roll(1, dims=1)
    return out


# What the keys and values of the tests are like, each with an offset and a scale of its own.
VALUES = [dict(), dict(k_offset=6.0), dict(k_offset=-40.0, k_scale=3.0), dict(v_offset=3.0), dict(k_offset=6.0, v_offset=-2.0),
          dict(v_scale=30.0), dict(v_scale=1e-4, k_scale=2.0), dict(k_scale=3.0), dict(k_scale=3.0, v_scale=30.0, v_offset=-60.0)]
DECODES = [[300, 77, 40], [1200, 9, 641]]                        # tokens of each sequence
CHUNKS = [([3, 1, 2], [300, 90, 200]),                           # up to 12 rows of a KV head
          ([6, 14], [260, 333]), ([70], [300])]                  # 24 and 56; 280

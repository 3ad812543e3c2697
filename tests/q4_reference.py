"""The 4-bit form of a paged cache, byte by byte in float64 on the CPU, and ragged inputs held in it."""
from __future__ import annotations

import copy

import torch

from tests.chunk_reference import Ragged, attention

GROUP = 32


def cut(x: torch.Tensor, dtype) -> torch.Tensor:
    """float64 x >= 0 toward zero to ``dtype``."""
    t = x.to(dtype)
    return torch.where(t.double() > x, (t.view(torch.int16) - 1).view(dtype), t)


def quantise(x: torch.Tensor):
    """Codes [..., D] of x (of the element type), and the groups' scale and minimum [..., D / 32], of the type."""
    f = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = f.amin(-1), f.amax(-1)
    s = cut((hi - lo) / 15, x.dtype)
    s = torch.where(s.double() < 2.0 ** -126, torch.zeros_like(s), s)
    d = s.double()[..., None]
    code = torch.where(d == 0, torch.zeros_like(f), torch.floor((f - lo[..., None]) / torch.where(d == 0, 1.0, d) + 0.5).clamp(0, 15))
    bad = ~torch.isfinite(f).all(-1)
    s = s.masked_fill(bad, float("nan"))
    m = lo.to(x.dtype).masked_fill(bad, float("nan"))
    return code.nan_to_num(0.0).to(torch.int64).flatten(-2), s, m


def value_of(code, s, m):
    """m + s c in float64 (exact for the types' exponents at hand)."""
    return (m.double()[..., None] + s.double()[..., None] * code.unflatten(-1, (-1, GROUP)).double()).flatten(-2)


def places(page: int, D: int, values: bool):
    """Byte of the block and shift of the code of each (token, dim)."""
    t, d = torch.arange(page)[:, None], torch.arange(D)[None]
    g, w = d // GROUP, d % GROUP
    if values:
        return t // 4 * (2 * D) + 4 * ((D // 32) * (w % 16) + g) + t % 4, (4 * (w // 16)).expand(page, D)
    word, e = (D // 32) * (w // 8) + g, w % 8
    return t * (D // 2) + 4 * word + e % 4, (4 * (e // 4)).expand(page, D)


def pack(x: torch.Tensor, values: bool) -> torch.Tensor:
    """[..., page, D] of the element type -> [..., block bytes] uint8."""
    page, D = x.shape[-2:]
    code, s, m = quantise(x)
    byte, shift = places(page, D, values)
    out = torch.zeros(*x.shape[:-2], page * D // 2, dtype=torch.int64)
    out.scatter_add_(-1, byte.flatten().expand(*x.shape[:-2], -1), (code << shift).flatten(-2))
    stats = torch.stack([s, m], dim=-1).transpose(-3, -2).contiguous()          # [..., g, page, 2]
    return torch.cat([out.to(torch.uint8), stats.view(torch.uint8).flatten(-3)], dim=-1)


def stats_of(pool: torch.Tensor, page: int, D: int, dtype):
    """(scale, minimum) [..., page, D / 32] of the blocks, of the type."""
    st = pool[..., page * D // 2:].contiguous().view(dtype).unflatten(-1, (D // GROUP, page, 2)).transpose(-3, -2)
    return st[..., 0], st[..., 1]


def codes_of(pool: torch.Tensor, page: int, D: int, values: bool) -> torch.Tensor:
    byte, shift = places(page, D, values)
    got = pool[..., :page * D // 2].long().gather(-1, byte.flatten().expand(*pool.shape[:-1], -1)).unflatten(-1, (page, D))
    return (got >> shift) & 15


def unpack(pool: torch.Tensor, page: int, D: int, dtype, values: bool) -> torch.Tensor:
    """[..., block bytes] -> float64 [..., page, D]."""
    return value_of(codes_of(pool, page, D, values), *stats_of(pool, page, D, dtype))


class Q4Ragged(Ragged):
    """A ragged paged cache whose pools ``k4, v4`` hold ``k_pages, v_pages`` in 4 bits; these become what is read back, in
    float64.  Slots without a token: codes of all ones and NaN scales."""

    def __init__(self, q_lens, kv_lens, *, page, Hkv, D, dtype=torch.bfloat16, seed=0, extra_cols=1, pad_rows=0, offset=0.0):
        super().__init__(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=seed, extra_cols=extra_cols,
                         pad_rows=pad_rows, poison=False)
        self.k_pages += offset
        self.v_pages += offset
        self.k4, self.v4 = pack(self.k_pages, False), pack(self.v_pages, True)
        self.held = torch.zeros(self.k4.size(0), page, dtype=torch.bool)
        for b, n in enumerate(kv_lens):
            for lb in range(-(-n // page)):
                self.held[self.table[b, lb].item(), :min(page, n - lb * page)] = True
        for pool, values in ((self.k4, False), (self.v4, True)):
            byte, _ = places(page, D, values)
            stats = page * D // 2 + 4 * (torch.arange(D // GROUP)[None] * page + torch.arange(page)[:, None])
            bytes_of = torch.cat([byte, *(stats + i for i in range(4))], dim=1)   # [page, ...]
            for p, t in (~self.held).nonzero().tolist():
                pool[p, :, bytes_of[t]] = 0xFF
        self.k_pages, self.v_pages = (unpack(p, page, D, dtype, v) for p, v in ((self.k4, False), (self.v4, True)))


def rounded(r: Q4Ragged) -> Q4Ragged:
    """The same cache with its keys and values rounded to the element type, as kernels that multiply those take them."""
    out = copy.copy(r)
    out.k_pages, out.v_pages = (x.float().to(r.dtype).double() for x in (r.k_pages, r.v_pages))
    return out


def assert_attention(got, r: Q4Ragged, q, sel=None, sel_off=None, what="", scores=0.0):
    """Rows of attention over a 4-bit cache against float64: over m + s c, or over that rounded to the element type.
    ``scores``: the largest sum |q k| scale where that passes the 16 that attention()'s bound counts; a score is off by
    D 2^-24 of it, a probability by twice that."""
    got = got.double().cpu()
    worst, ok = None, None
    for form in (r, rounded(r)):
        want, tol, live = attention(form, q, sel, sel_off)
        tol = tol + q4_slack(r, q) + 2 * r.D * 2.0 ** -24 * scores * form.v_pages.nan_to_num(0.0).abs().max()
        over = ((got - want).abs() - tol).nan_to_num(float("inf")).amax(-1)     # [N, Hq]
        good = over <= 0
        ok = good if ok is None else ok | good
        worst = over if worst is None else torch.minimum(worst, over)
    assert ok[live].all(), f"{what}: {int((~ok[live]).sum())} of {ok[live].numel()} rows, worst {worst[live].max():.3e} past the bound"
    return live


def q4_slack(r: Q4Ragged, q) -> float:
    """What kernels that multiply codes and scale the sums add to attention()'s bound.  A probability times its scale is
    rounded to bf16 once and meets |c - 7.5| <= 7.5: half a step of s 7.5, with s the largest.  A score is the fp32 sum of
    s sum q c and m sum q over the groups: at most D 2^-24 of sum |q| (15 s + |m|) scale, twice that in a probability, of
    values no larger than the largest."""
    held = r.held[:, None, :, None].expand(-1, r.Hkv, -1, r.D // GROUP)
    smax, mmax, vmax = 0.0, 0.0, 0.0
    for pool in (r.k4, r.v4):
        s, m = stats_of(pool, r.page, r.D, r.dtype)
        if held.any():
            smax, mmax = s[held].double().max().item(), m[held].double().abs().max().item()
    if held.any():
        vmax = r.v_pages[r.held[:, None, :, None].expand_as(r.v_pages)].abs().max().item()
    qsum = q.double().abs().sum(-1).max().item() / r.D ** 0.5
    return 7.5 * smax * 2.0 ** -9 + 2 * r.D * 2.0 ** -24 * qsum * (15 * smax + mmax) * vmax

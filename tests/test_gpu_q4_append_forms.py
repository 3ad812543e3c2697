"""``paged_append_q4`` with positions of the caller's, and groups at the edges of the form's arithmetic."""
import math

import pytest
import torch

from sparseattentioninfer_amd import ops
from tests.chunk_reference import assert_rotated, randn, rotate
from tests.q4_reference import Q4Ragged, codes_of, quantise, stats_of, value_of

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[q4-append]", *msg, flush=True)


def _one(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
@pytest.mark.parametrize("bounds", [False, True])
def test_positions_that_are_given(D, dtype, bounds):
    """Angles follow the given positions and places the lengths: the tokens' own places give the bytes of a call without them,
    others those of an unpaged rotation by them that is then stored as it is."""
    _say("positions", D, dtype, bounds)
    Hq, Hkv, page = 4, 2, 32
    r = Q4Ragged([70, 0, 1, 33], [130, 40, 90, 33], page=page, Hkv=Hkv, D=D, dtype=dtype, seed=4, pad_rows=3)
    q, k, v = (randn(r.N, h, D, seed=s, dtype=dtype).cuda() for s, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    kw, qw = ((randn(D, seed=s, dtype=dtype, scale=0.2) + 1) for s in (5, 6))
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).float()
    places = torch.zeros(r.N, dtype=torch.int64)
    for _, at, t, n in r.rows():
        places[at:at + t] = torch.arange(n - t, n)
    other = torch.randint(0, 100_000, (r.N,), generator=torch.Generator().manual_seed(9))

    def run(k_in, **opts):
        pools = [r.k4.clone().cuda(), r.v4.clone().cuda()]
        bd = torch.zeros(r.k4.size(0), Hkv, 2, D, dtype=dtype, device="cuda") if bounds else None
        out = torch.full((r.N, Hq, D), 7.0, dtype=dtype, device="cuda")
        ops.paged_append_q4(k_in, v, *pools, *r.gpu("table", "cu", "kv_lens"), k_bounds=bd, q=q, q_out=out, **opts)
        return [*pools, out, *([bd] if bounds else [])]

    rope = dict(inv_freq=inv.cuda(), k_weight=kw.cuda(), q_weight=qw.cuda())
    for a, b in zip(run(k, **rope), run(k, positions=places.cuda(), **rope)):
        assert torch.equal(a, b)
    wide = torch.full((r.N, 3), -1, dtype=torch.int64)
    wide[:, 1] = other
    got = run(k, positions=wide.cuda()[:, 1], **rope)                          # every third element
    plain = run(k, positions=other.cuda(), **rope)
    for a, b in zip(got, plain):
        assert torch.equal(a, b)
    q_rot, k_rot = ops.qk_norm_rope(q, k, other.cuda(), inv.cuda(), k_weight=kw.cuda(), q_weight=qw.cuda())
    stored = run(k_rot)
    n = sum(r.q_lens)
    assert torch.equal(got[0], stored[0]) and torch.equal(got[1], stored[1])
    assert torch.equal(got[2][:n], q_rot[:n]) and (got[2][n:] == 7.0).all()
    if bounds:
        assert torch.equal(got[3], stored[3])
    for x, w, have in ((q, qw, got[2]), (k, kw, k_rot)):
        want, terms = rotate(x.cpu()[:n], w, other[:n], inv, 1e-6)
        assert_rotated(have[:n], want, terms, "rotation by positions")


def _store(x, page=16):
    """x [N, 1, D] stored as it is: (pools, read back keys and values)."""
    N, _, D = x.shape
    nb = -(-N // page)
    pools = [torch.zeros(nb, 1, ops.q4_block_bytes(page, D), dtype=torch.uint8, device="cuda") for _ in "kv"]
    table, cu, lens = torch.arange(nb, dtype=torch.int32, device="cuda")[None], _one(0, N), _one(N)
    ops.paged_append_q4(x.cuda(), x.cuda(), *pools, table, cu, lens)
    return pools, ops.paged_read_q4(*pools, table, cu, lens, rows=N, head_dim=D, dtype=x.dtype)


@pytest.mark.parametrize("D", [64, 128])
def test_scales_among_the_smallest_values(D):
    """fp16 groups whose range is a few of the type's steps of 2^-24, so that the scale is one of few subnormal values; bf16
    groups around a scale of 2^-126.  Codes, scales and minima by the definition; every value within half a step or, past
    the code 15, what 15 steps leave of the range."""
    for dtype, unit in ((HF, 2.0 ** -24), (BF, 2.0 ** -133)):
        _say("smallest", D, dtype)
        g = torch.Generator().manual_seed(3)
        ranges = [0, 1, 7, 14, 15, 16, 20, 29, 30, 31, 44, 45, 100, 400, 449, 450, 1000, 1919, 1920, 1921, 2000, 1 << 14]
        x = torch.zeros(len(ranges), 1, D, dtype=torch.float64)
        for i, n in enumerate(ranges):
            steps = torch.randint(0, n + 1, (D // 32, 32), generator=g)
            steps[:, 5], steps[:, 20] = 0, n
            x[i, 0] = (steps - (0, n // 2, 3)[i % 3]).flatten() * unit
        x = x.to(dtype)
        code, s, m = quantise(x)
        pools, back = _store(x)
        for pool, got, values in zip(pools, back, (False, True)):
            rows = lambda t: t.cpu().transpose(1, 2).flatten(0, 1)[:len(ranges)]      # [N, 1, ...]
            assert torch.equal(rows(codes_of(pool.cpu(), 16, D, values)), code)
            for have, want in zip(stats_of(pool.cpu(), 16, D, dtype), (s, m)):
                assert torch.equal(rows(have).double(), want.double())
            f = x.double().unflatten(-1, (-1, 32))
            span = f.amax(-1, keepdim=True) - f.amin(-1, keepdim=True)
            err = (value_of(code, s, m) - x.double()).abs().unflatten(-1, (-1, 32))
            sd = s.double()[..., None]
            assert (err <= torch.maximum(sd / 2, span - 15 * sd)).all()
            assert (span - 15 * sd <= 15 * (unit if dtype == HF else 2.0 ** -126)).all()
            assert torch.equal(got.cpu().double(), value_of(code, s, m).to(dtype).double())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_values_beside_ties(dtype):
    """Quotients (x - m) / s less than 2^-20 of themselves below a tie between two codes: either neighbour may be taken, so a value
    is off by half a step and 2^-20 of 15 steps at most."""
    _say("ties", dtype)
    x = torch.zeros(8, 1, 128, dtype=torch.float64)
    for i in range(8):
        m = -(i + 0.5)                          # s = 1: x = 0 would be a tie
        x[i] = m + torch.arange(128).remainder(16).double()
        x[i, 0, 1::32] = -2.0 ** -24
        x[i, 0, 2::32] = 2.0 ** -24
        x[i, 0, 3::32] = 0.0
        x[i, 0, 4::32], x[i, 0, 5::32] = m, m + 15
    x = x.to(dtype)
    code, s, m = quantise(x)
    assert (s == 1).all()
    pools, back = _store(x)
    for pool, got, values in zip(pools, back, (False, True)):
        have = codes_of(pool.cpu(), 16, 128, values).transpose(1, 2).flatten(0, 1)[:8]
        err = (value_of(have, s, m) - x.double()).abs()
        assert (err <= 0.5 + 15 * 2.0 ** -20).all()
        assert (have - code).abs().max() <= 1
        assert torch.equal(have[..., 2::32], code[..., 2::32]) and torch.equal(have[..., 3::32], code[..., 3::32])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_ranges_beside_a_scale(dtype):
    """Ranges less than 2^-24 of themselves below 15 times a value of the type, which fp32 rounds up to that: its scale or the next
    smaller one may be taken, and nothing is read back past the group's largest."""
    _say("ranges", dtype)
    x = torch.zeros(8, 1, 128, dtype=torch.float64)
    for i in range(8):
        t = 0.0 if i == 7 else 2.0 ** -(18 + i)
        x[i] = torch.arange(128).remainder(15).double()
        x[i, 0, 0::32], x[i, 0, 1::32] = t, 15.0
        x[i, 0][x[i, 0] < t] = t
    x = x.to(dtype)
    _, s, m = quantise(x)
    below = (torch.tensor(1.0, dtype=dtype).view(torch.int16) - 1).view(dtype).item()
    assert (s[:7] == below).all() and (s[7] == 1).all()
    pools, back = _store(x)
    for pool, got, values in zip(pools, back, (False, True)):
        have, hm = (t.transpose(1, 2).flatten(0, 1)[:8] for t in stats_of(pool.cpu(), 16, 128, dtype))
        assert torch.equal(hm, m) and ((have == s) | (have == 1)).all() and (have[:2] == s[:2]).all()
        code = codes_of(pool.cpu(), 16, 128, values).transpose(1, 2).flatten(0, 1)[:8]
        err = (value_of(code, have, hm) - x.double()).abs().unflatten(-1, (-1, 32))
        hd = have.double()[..., None]
        span = (x.double().unflatten(-1, (-1, 32)).amax(-1) - m.double())[..., None]
        assert (err <= torch.maximum(hd / 2, span - 15 * hd) + 15 * 2.0 ** -20).all()
        assert (got.cpu().double() <= 15).all()

"""The operators of the 4-bit paged cache where sizes, sharing and numbers are out of the ordinary."""
import pytest
import torch

from sparseattentioninfer_amd import ops
from tests.chunk_reference import attention, randn
from tests.q4_reference import Q4Ragged, assert_attention, pack, q4_slack, stats_of, unpack

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[q4-edges]", *msg, flush=True)


@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
def test_pools_past_32_bit_offsets(D, dtype):
    """Pages that begin past 2^32 bytes of the pool give what the same pages of a small pool give."""
    _say("large pools", D, dtype)
    page, Hkv, Hq, q_lens, kv_lens = 128, 4, 8, [300, 1, 5], [700, 513, 129]
    block = ops.q4_block_bytes(page, D)
    B, cols, N = 3, 6, sum(q_lens)
    many = 2 ** 32 // (Hkv * block) + 4 * B * cols
    cu = torch.tensor([0, 300, 301, 306], dtype=torch.int32, device="cuda")
    lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    small = torch.arange(B * cols, dtype=torch.int32, device="cuda").view(B, cols)
    last = many - 1 - small
    assert int(last.min()) * Hkv * block > 2 ** 32
    k, v = (randn(sum(kv_lens), Hkv, D, seed=s, dtype=dtype).cuda() for s in (1, 2))
    q = randn(N, Hq, D, seed=3, dtype=dtype).cuda()
    whole = torch.tensor([0, 700, 1213, 1342], dtype=torch.int32, device="cuda")
    got = []
    for pages, table in ((B * cols, small), (many, last)):
        pools = [torch.empty(pages, Hkv, block, dtype=torch.uint8, device="cuda") for _ in "kv"]
        ops.paged_append_q4(k, v, *pools, table, whole, lens)
        got.append((*ops.paged_read_q4(*pools, table, whole, lens, rows=sum(kv_lens), head_dim=D, dtype=dtype),
                    ops.paged_chunk_attn_q4(q, *pools, table, cu, lens),
                    ops.paged_chunk_attn_q4(q, *pools, table, cu, lens, num_splits=3),
                    ops.paged_sparse_decode_q4(q[:B], *pools, table, lens)))
        torch.cuda.synchronize()
    for a, b in zip(*got):
        assert a.isfinite().all() and torch.equal(a, b)


def test_decode_of_more_steps_than_fp32_counts():
    """A sequence of more than 2^24 steps of 32 keys, all of whose pages are one.  Each of 512 workgroups' four waves adds
    up to 2^13 steps in fp32: at most 2^13 2^-24 of the sums of p |v|, of p 7.5 s and of p."""
    _say("long list")
    page, D, Hq = 128, 64, 4
    n = (2 ** 24 + 1) * 32 - 5
    k, v = (randn(1, 1, page, D, seed=s) for s in (1, 2))
    k4, v4 = pack(k, False), pack(v, True)
    q = randn(1, Hq, D, seed=3)
    table = torch.zeros(1, -(-n // page), dtype=torch.int32, device="cuda")
    out = ops.paged_sparse_decode_q4(q.cuda(), k4.cuda(), v4.cuda(), table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    kd, vd = (unpack(p, page, D, BF, values)[0, 0] for p, values in ((k4, False), (v4, True)))
    times = torch.full((page,), n // page, dtype=torch.float64)
    times[:n % page] += 1
    p = (q[0].double() @ kd.T * D ** -0.5).exp() * times
    want = (p / p.sum(-1, keepdim=True)) @ vd
    s = stats_of(v4, page, D, BF)[0].double().max().item()
    top = vd.abs().max().item()
    # the output's rounding; that of p s to bf16; sums; scores' D 2^-24 of at most 64, twice that in a probability
    tol = want.abs() * 2.0 ** -8 + 7.5 * s * 2.0 ** -9 + 4 * 2.0 ** -11 * (top + 7.5 * s) + 2 * D * 2.0 ** -24 * 64 * top
    assert ((out[0].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
def test_chunk_of_many_sequences(D, dtype):
    _say("130 sequences", D, dtype)
    q_lens = [(3 * b) % 5 for b in range(129)] + [70]
    r = Q4Ragged(q_lens, [t + (37 * b) % 90 for b, t in enumerate(q_lens)], page=32, Hkv=2, D=D, dtype=dtype, seed=8)
    q = randn(r.N, 8, D, seed=9, dtype=dtype)
    out = ops.paged_chunk_attn_q4(q.cuda(), *r.gpu("k4", "v4", "table", "cu", "kv_lens"))
    assert_attention(out, r, q, what="130 sequences")


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("t,n,D,dtype", [(3, 900, 128, BF), (90, 900, 128, BF), (3, 500, 64, HF), (70, 400, 64, BF)])
def test_nan_keys_reach_the_rows_that_see_them(t, n, D, dtype, splits):
    """The key of the second new token is NaN: rows from that token on are NaN, in its KV head.  The others are within the
    bound of the same values as without it, so within twice the bound of each other."""
    _say("nan key", t, n, D, dtype, splits)
    page = 64
    r = Q4Ragged([t, 2], [n, 333], page=page, Hkv=2, D=D, dtype=dtype, seed=12)
    q = randn(r.N, 8, D, seed=13, dtype=dtype)
    rest = r.gpu("v4", "table", "cu", "kv_lens")
    base = ops.paged_chunk_attn_q4(q.cuda(), r.k4.cuda(), *rest, num_splits=splits)
    at = n - t + 1
    byte = page * D // 2 + 4 * (page + at % page)                       # group 1
    k4 = r.k4.clone()
    k4[r.table[0, at // page].long(), 1, byte:byte + 4] = 0xFF
    got = ops.paged_chunk_attn_q4(q.cuda(), k4.cuda(), *rest, num_splits=splits)
    assert got[1:t, 4:].isnan().all()
    _, tol, _ = attention(r, q)
    bad = ~((got.double() - base.double()).cpu().abs() <= 2 * (tol + q4_slack(r, q)))
    bad[1:t, 4:] = False
    assert not bad.any()


def test_two_graphs_replayed_in_turn():
    """Two captured calls whose lists are shared by workgroups, with workspaces of their own, replayed in turn with eager calls between."""
    _say("two graphs")
    D, page, B = 128, 64, 2
    r = Q4Ragged([4, 4], [3000, 1500], page=page, Hkv=2, D=D, seed=21)
    cache, cu = r.gpu("k4", "v4", "table"), r.gpu("cu")[0]
    lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([3000, 1500], [2500, 700])]
    qs = [randn(8, 8, D, seed=30 + i).cuda() for i in range(2)]

    def call(i):
        return (ops.paged_sparse_decode_q4(qs[i][:B], *cache, lens[i]),
                ops.paged_chunk_attn_q4(qs[i], *cache, cu, lens[i], num_splits=5))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    for n in range(4):
        for i in (0, 1, 1, 0):
            qs[i].copy_(randn(8, 8, D, seed=100 * n + i))
            graphs[i].replay()
        for i in range(2):
            want = call(i)
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want):
                assert torch.equal(a, b), (n, i)

"""The division of whole caches that the 4-bit decode plans on the device, weighed again exactly on the CPU."""
import math

import pytest
import torch

from sparseattentioninfer_amd import _lib, ops

pytestmark = pytest.mark.gpu

TARGET, MIN_UNIT, START = 512, 8, 8.0      # workgroups at once, steps of one at least, what one costs in steps


def _say(*msg):
    print("[q4-plan]", *msg, flush=True)


def _units(steps, of_seq):
    """No division, and fractions of an even share."""
    even = sum(steps) * of_seq * (1.001 / TARGET)
    return [max(1, max(steps))] + [max(MIN_UNIT, math.ceil(even * f)) for f in (1.0, 0.76, 0.5, 0.381)]


def _time(unit, steps, of_seq):
    """When a division ends, in steps: with the longest workgroup where all run at once, else the mean load and half the
    longest."""
    shares = [max(1, -(-n // unit)) for n in steps]
    groups = of_seq * sum(k for k, n in zip(shares, steps) if n)
    longest = max(n / k for k, n in zip(shares, steps)) + START
    return longest if groups <= TARGET else (of_seq * sum(steps) + groups * START) / TARGET + 0.5 * longest


class _Planned:
    """Calls whose every page is page 0; the unit that the launch has planned is the workspace's first word."""

    def __init__(self, B, heads, most):
        self.B, self.heads, page = B, heads, 128
        self.pools = [torch.zeros(1, heads, ops.q4_block_bytes(page, 64), dtype=torch.uint8, device="cuda") for _ in "kv"]
        self.table = torch.zeros(B, -(-most * 32 // page), dtype=torch.int32, device="cuda")
        self.q = torch.zeros(B, heads, 64, dtype=torch.bfloat16, device="cuda")
        need = _lib.load().sa_decode_q4_workspace_bytes(B, heads, heads, 64, self.table.size(1) * page, 0, 0)
        self.ws = torch.zeros(need, dtype=torch.uint8, device="cuda")

    def unit(self, steps):
        lens = torch.tensor([32 * n for n in steps], dtype=torch.int32, device="cuda")
        ops.paged_sparse_decode_q4(self.q, *self.pools, self.table, lens, workspace=self.ws)
        return int(self.ws[:4].view(torch.int32))


def _check(planned, cases):
    wrong = []
    for steps in cases:
        unit = planned.unit(steps)
        times = [_time(u, steps, planned.heads) for u in _units(steps, planned.heads)]
        if _time(unit, steps, planned.heads) > min(times) * 1.001:
            wrong.append((max(steps), unit, round(_time(unit, steps, planned.heads), 1), round(min(times), 1)))
    assert not wrong, f"{len(wrong)} of {len(cases)} (longest list, unit taken, its time, the best): {wrong[:8]}"


def test_equal_lists():
    """256 equal lists, which uncut fill half of the chip; lengths whose fp32 reciprocal times them is more than 1 among them."""
    _say("equal lists")
    _check(_Planned(32, 8, 8192), [[n] * 32 for n in [*range(17, 1200, 5), 1535, 3070, 4071, 6137, 6139, 6140, 8142, 8165, 8167]])


@pytest.mark.parametrize("B,heads", [(1, 8), (5, 2), (28, 8), (70, 4)])
def test_uneven_lists(B, heads):
    _say("uneven lists", B, heads)
    g = torch.Generator().manual_seed(B)
    _check(_Planned(B, heads, 1000), [torch.randint(0, 1000, (B,), generator=g).tolist() for _ in range(60)])

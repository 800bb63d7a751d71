"""How exl3r_paged_attn cuts its work: the decode kernel gives every workgroup an equal part of all sequences' keys, so
a workgroup ends one sequence and begins others, and a sequence lies in one workgroup or in many.  Tolerances are those
of test_gpu_paged_attn."""
import pytest
import torch

import exl3r.ffi as ffi
from test_gpu_paged_attn import BF16, F16, build, call, compare, exact

pytestmark = pytest.mark.gpu


CUTS = [
    # lens, seq, hq, hk, hd, dtype, window, sinks, page, shared
    ([(37 * i) % 190 for i in range(300)], 1, 4, 2, 64, F16, 0, 0, 16, None),       # more segments than lanes
    ([(53 * i) % 700 for i in range(70)], 1, 3, 3, 128, BF16, 0, 0, 32, None),      # KV heads that do not divide the slots
    ([0] * 40 + [3000] + [0] * 40, 1, 4, 1, 128, F16, 0, 0, 64, None),              # one long sequence among empty ones
    ([3000, 0, 1, 2000], 1, 7, 7, 64, F16, 0, 0, 256, None),
    ([127, 128, 129, 255, 256, 257, 0], 1, 16, 2, 128, BF16, 0, 0, 128, None),      # around a unit of 128 keys
    ([2000, 5, 900], 2, 32, 2, 128, F16, 0, 0, 16, None),                           # 32 rows of a KV head
    ([2000, 5, 900], 3, 20, 2, 128, BF16, 0, 0, 4, None),                           # 30 rows, pages of 4
    ([1500, 700], 3, 16, 2, 256, F16, 0, 0, 32, None),                              # 24 rows of 256: two row tiles each
    ([1500, 700], 2, 32, 2, 256, BF16, 300, 9, 8, None),
    ([900, 700, 2500, 1], 1, 8, 8, 256, BF16, 0, 0, 64, None),
    ([600, 601], 1, 8, 1, 128, F16, 0, 0, 8, 600),                                  # a prefix on 16 rows
    ([512, 700], 1, 28, 2, 256, F16, 0, 0, 16, 512),                                # ... on 28 of 256: two row tiles
    ([512, 2700, 513], 1, 10, 1, 64, BF16, 0, 0, 16, 512),                          # ... on 30 rows
    ([2048 + 31 * i for i in range(9)], 1, 32, 4, 128, BF16, 0, 0, 256, 2048),      # ... on 72 rows
    ([2500 + 40 * i for i in range(20)], 1, 8, 2, 128, F16, 700, 3, 32, 2496),      # a window that ends inside the prefix
    ([400], 1, 600, 600, 64, F16, 0, 0, 64, None),                                  # more KV heads than workgroups wanted
]


@pytest.mark.parametrize("lens,seq,hq,hk,hd,dtype,window,sinks,page,shared", CUTS)
def test_against_float64(lens, seq, hq, hk, hd, dtype, window, sinks, page, shared):
    a = build(lens, seq, hq, hk, hd, dtype, page, shared or 0, seed=41)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = call(*a, shared=shared, window=window, sinks=sinks, err=err)
    compare(got, exact(*a, window=window, sinks=sinks), f"{len(lens)} of {seq}, {hq}/{hk} x {hd}")
    assert err.item() == 0
    again = call(*a, shared=shared, window=window, sinks=sinks)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_lengths_outside_among_many():
    """Sequences before the first position and past the table beside long ones: zeros and -inf, or what the table
    holds; the others as if those were not there."""
    lens = [300, 40, 900, 0, 77, 500] * 50
    q, kc, vc, table, sl = build(lens, 1, 8, 2, 64, BF16, 32, seed=42, poison=False)
    want = exact(q, kc, vc, table, sl)
    good = call(q, kc, vc, table, sl)
    compare(good, want, "inside")
    bad = sl.clone()
    bad[::7] = -1
    bad[3::11] = -2 ** 31
    bad[5::13] = 2 ** 31 - 1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = call(q, kc, vc, table, bad, err=err)
    assert err.item() == 1
    before = bad < 0
    assert (got[0][before] == 0).all() and (got[1][before] == -float("inf")).all()
    past = bad == 2 ** 31 - 1
    compare((got[0][past], got[1][past]), exact(q[past], kc, vc, table[past], bad[past].clamp(max=10 ** 6)), "past the table")
    same = ~before & ~past
    # (cut elsewhere: the same up to the order of sums)
    compare((got[0][same], got[1][same]), tuple(x[same] for x in want), "the others")


def test_no_row_beside_the_batch_is_written():
    q, kc, vc, table, sl = build([900, 3, 70], 1, 6, 2, 128, F16, 64, seed=43)
    big = torch.full((5, 1, 6, 128), 3.0, dtype=F16, device="cuda")
    z = torch.full((5, 1, 6), 3.0, device="cuda")
    ws = torch.empty(ffi.paged_attn_workspace_bytes(q, kc, table) + 4096, dtype=torch.uint8, device="cuda")
    ws.fill_(77)
    ffi.paged_attn(q, kc, vc, table, sl, big[1:4], lse=z[1:4], workspace=ws[:-4096])
    torch.cuda.synchronize()
    compare((big[1:4], z[1:4]), exact(q, kc, vc, table, sl), "inside")
    assert (big[0] == 3).all() and (big[4] == 3).all() and (z[0] == 3).all() and (z[4] == 3).all()
    assert (ws[-4096:] == 77).all()


def test_a_larger_workspace_from_the_whole_table():
    """One workspace, sized for the longest table, serves calls with windows and shorter tables."""
    q, kc, vc, table, sl = build([1200, 900], 1, 8, 2, 128, BF16, 64, seed=44)
    ws = torch.empty(ffi.paged_attn_workspace_bytes(q, kc, table), dtype=torch.uint8, device="cuda")
    for window in (0, 1, 100, 1000, 10 ** 6):
        out = torch.empty_like(q)
        ffi.paged_attn(q, kc, vc, table, sl, out, window=window, workspace=ws)
        torch.cuda.synchronize()
        compare((out, None), exact(q, kc, vc, table, sl, window=window), f"window {window}")


@pytest.mark.parametrize("seq", [1, 40])
@pytest.mark.parametrize("scale", [1e-40, 1e-30, 1.0, 30.0])
def test_scales(seq, scale):
    a = build([300, 7], seq, 4, 2, 64, F16, 32, seed=45, std=0.5)
    compare(call(*a, scale=scale), exact(*a, scale=scale), f"scale {scale}")


@pytest.mark.parametrize("lens,seq,hq,hk,hd,page,blocks", [
    ([3, 200, 127, 0], 1, 8, 2, 128, 64, 2),        # sequences shorter than the prefix; 128 of it
    ([100, 20], 20, 8, 2, 256, 16, 8),              # ... and rows for the other kernel
    ([255], 1, 8, 2, 64, 64, 4),                    # a batch of one whose table is all prefix
    ([200, 190], 50, 4, 1, 128, 32, 8),
])
def test_prefix_beyond_a_sequence(lens, seq, hq, hk, hd, page, blocks):
    """A prefix that some sequences have not reached, and one that fills the table."""
    shared = page * blocks
    spare = 0 if max(lens) + seq <= shared else 1
    a = build(lens, seq, hq, hk, hd, BF16, page, shared, seed=46, spare_blocks=spare, poison=False)
    compare(call(*a, shared=shared), exact(*a), f"prefix of {shared}")

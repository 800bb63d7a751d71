"""GPU parity of exl3r_paged_attn and exl3r_paged_attn_shared against the definition in 64 bits: positions from
cache_seqlens, causal, window and sinks, keys through the block table.

Tolerances, per element, from the formats.  With u half a step of the 16-bit type, w the exact weights and
W = sum_j w_j |v_j|:
  - a weight is rounded to 16 bits (u) and comes from a score with an fp32 error; a score is a sum of head_dim exact
    products, off by at most (head_dim + 2) 2^-24 scale sum_d |q_d k_d| =: d (natural units), its exponent in base 2
    and the exponential by 2^-22 + 2^-23 |s - m|: a weight is off by the relative u + e, the sum of the weights by e,
    e = 2 d + 2^-21 + 2^-22 max|s - m|;  with 2^-19 for the fp32 sums: (u + 2 e + 2^-19) W;
  - f16 weights are held as 2^6 times their ratio to a reference that is at most the row's largest weight, so below 2^-20
    of it they have, instead, an absolute error of half of f16's smallest denormal, 2^-25, over 2^6: 2^-31 sum_j |v_j|
    (the softmax's sum is at least the largest weight);
  - out is rounded once: u |out|, and by at most half its smallest denormal.
lse is off by e, its own rounding 2^-23 |lse| and the fp32 sum."""
import math

import pytest
import torch

import exl3r.ffi as ffi
from exl3r import Exl3rError

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def build(lens, seq, hq, hk, hd, dtype, page, shared=0, seed=0, spare_blocks=1, std=1.0, poison=True):
    """Random pages; every cache row that no sequence's tokens own holds NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    bsz = len(lens)
    need = [max(1, -(-(max(n, 0) + seq) // page)) for n in lens]
    common = shared // page
    need = [max(n, common) for n in need]
    width = max(need) + spare_blocks
    pages = common + sum(n - common for n in need) + 2
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((bsz, width), 0, dtype=torch.int32)
    table[:, :common] = perm[:common]
    at = common
    for b, n in enumerate(need):
        table[b, common:n] = perm[at:at + n - common]
        at += n - common
    kc = (torch.randn((pages, page, hk, hd), generator=g, device="cuda") * std).to(dtype)
    vc = torch.randn((pages, page, hk, hd), generator=g, device="cuda").to(dtype)
    if poison:
        used = torch.zeros((pages, page), dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(max(n, 0) + seq):
                used[table[b, j // page], j % page] = True
        kc[~used.cuda()] = float("nan")
        vc[~used.cuda()] = float("nan")
    q = (torch.randn((bsz, seq, hq, hd), generator=g, device="cuda") * std).to(dtype)
    return q, kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def exact(q, kc, vc, table, lens, window=0, sinks=0, scale=None, bad_pages=()):
    """(out, lse, tolerance of out, tolerance of lse) in float64, and what each visible weight adds to the bounds."""
    bsz, seq, hq, hd = q.shape
    page, hk = kc.shape[1], kc.shape[2]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    cap = table.shape[1] * page
    for b in range(bsz):
        n = int(lens[b])
        total = max(0, min(n + seq, cap))
        if total == 0:
            continue
        j = torch.arange(total, device="cuda")
        pg = table[b].long()[j // page]
        good = (pg >= 0) & (pg < kc.shape[0])
        k = kc[pg.clamp(0, kc.shape[0] - 1), j % page].double()
        v = vc[pg.clamp(0, kc.shape[0] - 1), j % page].double()
        p = n + torch.arange(seq, device="cuda")
        see = (j[None] <= p[:, None]) & good[None]
        if window > 0:
            see &= (p[:, None] - j[None] < window) | (j[None] < sinks)
        for h in range(hq):
            kh, vh = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
            qh = q[b, :, h].double()
            s = torch.where(see, (qh[:, None] * kh[None]).sum(-1) * scale, -math.inf)
            mag = torch.where(see, (qh.abs()[:, None] * kh.abs()[None]).sum(-1) * scale, 0.0).nan_to_num(0, 0, 0).amax(1)
            z = torch.logsumexp(s, 1)
            some = see.any(1)
            w = torch.where(see, torch.exp(s - z[:, None]), 0.0)
            vv = torch.where(see[:, :, None], vh[None], 0.0)
            out[b, :, h] = torch.where(some[:, None], (w[:, :, None] * vv).sum(1), 0.0)
            lse[b, :, h] = torch.where(some, z, -math.inf)
            spread = torch.where(see, s.amax(1, keepdim=True) - s, 0.0).amax(1)
            e = 2 * (hd + 2) * 2.0 ** -24 * mag + 2.0 ** -21 + 2.0 ** -22 * spread
            W = (w[:, :, None] * vv.abs()).sum(1)
            tol[b, :, h] = (u + 2 * e + 2.0 ** -19)[:, None] * W
            if q.dtype == F16:
                tol[b, :, h] += 2.0 ** -31 * vv.abs().sum(1) + 2.0 ** -25
            tol_lse[b, :, h] = e + 2.0 ** -19 + 2.0 ** -23 * z.abs()
    return out, lse, tol + u * out.abs(), tol_lse


def call(q, kc, vc, table, lens, shared=None, window=0, sinks=0, scale=None, lse=True, out=None, err=None, stream=None):
    out = torch.full_like(q, 7.0) if out is None else out
    z = torch.full(q.shape[:3], 7.0, device="cuda") if lse else None
    need = ffi.paged_attn_workspace_bytes(q, kc, table, shared or 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    if ws is not None:
        ws.view(torch.float32).fill_(float("nan"))       # the workspace needs no initial value
    if shared is None:
        ffi.paged_attn(q, kc, vc, table, lens, out, scale, window, sinks, z, ws, err, stream)
    else:
        ffi.paged_attn_shared(q, kc, vc, table, lens, out, shared, scale, window, sinks, z, ws, err, stream)
    torch.cuda.synchronize()
    return out, z


def compare(got, want, tag):
    (out, z), (eo, ez, to, tz) = got, want
    o = out.double()
    nan = torch.isnan(eo)
    assert torch.equal(torch.isnan(o), nan), f"{tag}: NaNs differ"
    inf = torch.isinf(eo)
    assert torch.equal(o[inf], eo[inf]), f"{tag}: infinities differ"
    fin = ~nan & ~inf
    ratio = ((o - eo).abs()[fin] / to[fin].clamp_min(1e-300)).max().item() if fin.any() and (to[fin] > 0).any() else 0.0
    assert ((o - eo).abs()[fin] <= to[fin]).all(), f"{tag}: {ratio} of the tolerance"
    if z is not None:
        f = torch.isfinite(ez)
        assert torch.equal(z.double()[~f & ~torch.isnan(ez)], ez[~f & ~torch.isnan(ez)]), f"{tag}: lse"
        assert ((z.double() - ez).abs()[f] <= tz[f]).all(), f"{tag}: lse off by {(z.double() - ez).abs()[f].max().item()}"
    print(f"{tag}: {ratio:.3f} of the tolerance", flush=True)


CASES = [
    # lens, seq, hq, hk, hd, dtype, window, sinks, page, shared
    ([0], 1, 8, 8, 64, F16, 0, 0, 256, None),                    # the first token of a sequence
    ([1], 1, 4, 1, 128, BF16, 0, 0, 16, None),
    ([30, 31, 32, 33, 0, 7], 1, 8, 2, 128, F16, 0, 0, 32, None),    # around a tile of 32 keys
    ([62, 63, 64, 65, 127, 128], 1, 16, 2, 256, BF16, 0, 0, 64, None),
    ([1000, 13, 517], 1, 64, 8, 128, F16, 0, 0, 256, None),
    ([1000, 13, 517], 3, 12, 4, 64, BF16, 0, 0, 16, None),        # speculative tokens, 3 heads a group
    ([2200], 1, 5, 5, 128, BF16, 0, 0, 8, None),                 # one head a group, pages of 8
    ([700], 1, 40, 1, 64, F16, 0, 0, 1, None),                   # 40 heads a group, pages of one token
    ([0], 33, 4, 2, 128, F16, 0, 0, 256, None),                  # prefill
    ([0], 129, 8, 2, 64, BF16, 0, 0, 64, None),
    ([0, 0], 257, 4, 4, 128, F16, 0, 0, 32, None),
    ([0], 515, 6, 2, 256, BF16, 0, 0, 256, None),
    ([100, 640, 3], 77, 8, 1, 128, BF16, 0, 0, 16, None),        # chunks on top of a cache
    ([300], 200, 2, 1, 256, F16, 0, 0, 128, None),
    ([700, 3, 90], 1, 8, 2, 128, F16, 64, 0, 32, None),          # windows
    ([700, 3, 90], 1, 8, 2, 128, F16, 1, 0, 16, None),           # only itself
    ([700, 3, 90], 1, 8, 2, 128, BF16, 33, 5, 16, None),
    ([900], 2, 16, 2, 64, F16, 100, 70, 256, None),              # sinks that fill more than a tile
    ([900], 2, 16, 2, 64, F16, 100, 900, 256, None),             # sinks that reach the window
    ([0], 400, 4, 2, 128, BF16, 50, 4, 64, None),                # prefill with a window
    ([0], 400, 4, 2, 256, F16, 97, 1, 16, None),
    ([250, 31], 300, 4, 1, 64, BF16, 128, 33, 8, None),
    ([64, 70, 100], 1, 8, 2, 128, F16, 0, 0, 64, 64),            # a shared prefix
    ([64, 64], 1, 8, 2, 128, F16, 0, 0, 64, 64),                 # ... with nothing but the new token after it
    ([512, 530, 900, 513, 640], 1, 16, 2, 128, BF16, 0, 0, 256, 512),
    ([512, 530, 900, 513, 640], 5, 16, 2, 128, BF16, 0, 0, 16, 512),
    ([96] * 40, 4, 8, 2, 64, F16, 0, 0, 32, 96),                 # many query rows over the prefix
    ([48, 60, 49], 37, 4, 2, 256, F16, 0, 0, 16, 48),            # a prefix that ends inside a tile
    ([24, 60, 25], 3, 4, 2, 128, BF16, 0, 0, 8, 24),
    ([300, 320, 301], 9, 8, 2, 128, F16, 40, 4, 4, 300),         # ... with windows: some see only its sinks
    ([300, 420, 301], 2, 8, 2, 64, BF16, 200, 0, 4, 300),
    ([300, 420, 301], 2, 8, 2, 64, BF16, 0, 0, 4, 0),            # an empty prefix
]


@pytest.mark.parametrize("lens,seq,hq,hk,hd,dtype,window,sinks,page,shared", CASES)
def test_against_float64(lens, seq, hq, hk, hd, dtype, window, sinks, page, shared):
    tag = f"lens{lens[:4]} seq{seq} h{hq}/{hk}x{hd} {dtype} w{window}+{sinks} page{page} shared{shared}"
    print(tag, flush=True)
    a = build(lens, seq, hq, hk, hd, dtype, page, shared or 0, seed=len(lens) + seq)
    compare(call(*a, shared=shared, window=window, sinks=sinks), exact(*a, window, sinks), tag)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("std", [0.05, 6.0])
def test_flat_and_peaked(dtype, std):
    """Scores all alike, and scores where one key takes nearly everything."""
    a = build([900, 40], 3, 8, 2, 128, dtype, 16, seed=3, std=std)
    compare(call(*a), exact(*a), f"std {std} {dtype}")
    compare(call(*a, scale=2.5), exact(*a, scale=2.5), f"std {std} {dtype} scale 2.5")


@pytest.mark.parametrize("shared", [None, 64])
@pytest.mark.parametrize("seq", [1, 40])
@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64), (BF16, 256)])
def test_nonfinite_values(dtype, hd, seq, shared):
    """Infinities and NaNs in V reach exactly the tokens that see them; in K they are a NaN score (or -inf, which is no
    weight) for those tokens."""
    n, window, sinks = 100, 60, 3
    q, kc, vc, table, lens = build([n, n], seq, 4, 2, hd, dtype, 16, shared or 0, seed=9)
    where = lambda j: (table[0, j // 16].long(), j % 16)
    for j, d, val in ((1, 3, math.inf), (20, 5, math.nan), (n - 59, 7, -math.inf), (n, 9, math.nan), (n + seq - 1, 1, math.inf),
                      (n + seq // 2, 11, math.inf), (n + seq // 2 + 1, 11, -math.inf)):
        if j < n + seq:
            pg, r = where(j)
            vc[pg, r, :, d] = val
    for w, s in ((0, 0), (window, sinks)):
        want = exact(q, kc, vc, table, lens, w, s)
        compare(call(q, kc, vc, table, lens, shared, w, s), want, f"V {dtype} seq{seq} w{w} shared{shared}")
    if seq > 1:
        pg, r = where(n + 20)
        kc[pg, r, 0, 0] = math.nan
        vc.nan_to_num_(0, 0, 0)
        out, _ = call(q, kc, vc, table, lens, shared)
        hit = torch.isnan(out).any(-1)
        want = torch.zeros_like(hit)
        want[0, 20:, :2] = True
        assert torch.equal(hit, want)


@pytest.mark.parametrize("seq,shared", [(1, None), (70, None), (2, 32)])
def test_bad_pages_and_positions(seq, shared):
    """A page outside the cache hides its keys, a position outside the table sees what the table holds, and both are
    flagged; nothing else is, and no other token changes."""
    a = q, kc, vc, table, lens = build([150, 90, 151], seq, 4, 2, 128, F16, 16, shared or 0, seed=4)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    compare(call(*a, shared=shared, err=err), exact(*a), "clean")
    assert err.item() == 0
    for bad in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
        t2 = table.clone()
        t2[1, 3] = bad
        err.zero_()
        compare(call(q, kc, vc, t2, lens, shared, err=err), exact(q, kc, vc, t2, lens), f"page {bad}")
        assert err.item() == 1
    for n in (-1, -5, -2 ** 31):
        l2 = lens.clone()
        l2[1] = n
        err.zero_()
        compare(call(q, kc, vc, table, l2, shared, err=err), exact(q, kc, vc, table, l2), f"length {n}")
        assert err.item() == 1
    t2 = table[:, :9].contiguous()         # 144 positions: sequences 0 and 2 are past them
    err.zero_()
    out, z = call(q, kc, vc, t2, lens, shared, err=err)
    want = exact(q, kc, vc, t2, lens)
    compare((out, z), want, "short table")
    assert err.item() == 1
    l2 = lens.clone()
    l2[0] = 2 ** 31 - 1
    err.zero_()
    compare(call(q, kc, vc, t2, l2, shared, err=err), exact(q, kc, vc, t2, l2.clamp(max=10 ** 6)), "largest length")
    assert err.item() == 1


def test_a_page_of_the_window_s_past_may_be_gone():
    """Pages that no token sees any more (evicted behind the window) are not looked at."""
    a = q, kc, vc, table, lens = build([1000], 2, 8, 2, 128, BF16, 16, seed=6)
    want = exact(*a, 100, 4)
    t2 = table.clone()
    t2[0, 1:50] = -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    compare(call(q, kc, vc, t2, lens, window=100, sinks=4, err=err), want, "evicted")
    assert err.item() == 0


@pytest.mark.parametrize("seq,lens", [(1, [300, 77]), (1, [5]), (90, [60, 0])])
def test_strides_and_alignment(seq, lens):
    """q and out inside wider rows, at odd element offsets, heads apart; in place; what lies between stays."""
    a = q, kc, vc, table, sl = build(lens, seq, 4, 2, 64, F16, 32, seed=8)
    want = exact(*a)
    bsz = len(lens)
    for pad, off in ((0, 1), (3, 0), (8, 8), (5, 3)):
        def wide(fill):
            flat = torch.full((bsz * seq * 4 * (64 + pad) + off + 64,), fill, dtype=F16, device="cuda")
            v = flat[off:off + bsz * seq * 4 * (64 + pad)].view(bsz, seq, 4, 64 + pad)
            return flat, v[..., :64]
        _, qv = wide(0.0)
        flat, ov = wide(5.0)
        qv.copy_(q)
        before = flat.clone()
        out, z = call(qv, kc, vc, table, sl, out=ov)
        compare((out, z), want, f"pad{pad} off{off}")
        ov.fill_(5.0)
        assert torch.equal(flat, before), "written outside out"
        call(qv, kc, vc, table, sl, out=qv)
        compare((qv, z), want, f"in place pad{pad} off{off}")


def test_sliced_batch_of_single_tokens():
    """The last token of every row of a wider activation: a batch stride of its own."""
    a = q, kc, vc, table, sl = build([200, 31, 64], 1, 8, 2, 128, BF16, 64, seed=12)
    big = torch.randn((3, 5, 8, 128), device="cuda").to(BF16)
    big[:, 4:] = q
    compare(call(big[:, 4:], kc, vc, table, sl), exact(*a), "sliced")


def test_no_lse_and_no_sequences():
    a = q, kc, vc, table, sl = build([100, 3], 1, 8, 2, 128, F16, 64, seed=13)
    out, _ = call(*a, lse=False)
    ref, _ = call(*a)
    assert torch.equal(out, ref)
    e = q[:0]
    ffi.paged_attn(e, kc, vc, table[:0], sl[:0], torch.empty_like(e))


def test_long_context_offsets():
    """A cache of more than 2^32 bytes, whose last pages are read."""
    hk, hd, page = 8, 128, 256
    pages = 2 ** 32 // (page * hk * hd * 2) + 40
    kc = torch.zeros((pages, page, hk, hd), dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    table = torch.tensor([[pages - 1, pages - 7, 3]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in table[0].tolist():
        kc[p] = torch.randn((page, hk, hd), generator=g, device="cuda").to(BF16)
        vc[p] = torch.randn((page, hk, hd), generator=g, device="cuda").to(BF16)
    q = torch.randn((1, 1, 16, hd), generator=g, device="cuda").to(BF16)
    sl = torch.tensor([600], dtype=torch.int32, device="cuda")
    compare(call(q, kc, vc, table, sl), exact(q, kc, vc, table, sl), "beyond 4 GiB")
    q = torch.randn((1, 80, 16, hd), generator=g, device="cuda").to(BF16)
    compare(call(q, kc, vc, table, sl), exact(q, kc, vc, table, sl), "beyond 4 GiB, prefill")


def test_shared_is_plain_up_to_the_order_of_sums():
    a = build([520, 700, 513, 600], 2, 16, 4, 128, F16, 256, 512, seed=21)
    want = exact(*a)
    compare(call(*a), want, "plain")
    compare(call(*a, shared=512), want, "shared")
    compare(call(*a, shared=256), want, "half of it shared")


def test_deterministic():
    a = build([3000, 1, 777], 1, 32, 8, 128, BF16, 256, seed=22)
    first, z = call(*a)
    for _ in range(3):
        out, z2 = call(*a)
        assert torch.equal(out, first) and torch.equal(z, z2)


def test_another_stream_and_two_calls_at_once():
    a = build([900, 30], 1, 16, 2, 128, F16, 256, seed=23)
    b = build([40, 800], 1, 16, 2, 128, F16, 256, seed=24)
    ra, rb = call(*a), call(*b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for x, s in ((a, s1), (b, s2)):
        ws = torch.empty(ffi.paged_attn_workspace_bytes(x[0], x[1], x[3]), dtype=torch.uint8, device="cuda")
        out = torch.empty_like(x[0])
        torch.cuda.synchronize()
        outs.append((out, ws))
        ffi.paged_attn(*x, out, workspace=ws, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], ra[0]) and torch.equal(outs[1][0], rb[0])


@pytest.mark.parametrize("shared", [None, 256])
def test_graph_replays_with_new_lengths(shared):
    """One capture serves a growing batch: the lengths and the table are read when the graph runs."""
    q, kc, vc, table, sl = build([1500, 900, 1200], 1, 16, 2, 128, BF16, 256, shared or 0, seed=25, poison=False)
    need = ffi.paged_attn_workspace_bytes(q, kc, table, shared or 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    run = (lambda: ffi.paged_attn(q, kc, vc, table, sl, out, workspace=ws)) if shared is None else \
        (lambda: ffi.paged_attn_shared(q, kc, vc, table, sl, out, shared, workspace=ws))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for k, lens in enumerate(([256, 300, 257], [1500, 900, 1200], [1501, 260, 700], [300, 299, 1400])):
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(torch.randn_like(q))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        compare((out, None), exact(q, kc, vc, table, sl), f"replay {k}")
        eager, _ = call(q, kc, vc, table, sl, shared)
        assert torch.equal(out, eager), f"replay {k} differs from the eager call"


def test_wrapper_refusals():
    q, kc, vc, table, sl = build([100, 3], 1, 8, 2, 128, F16, 64, seed=13)
    out = torch.empty_like(q)
    ok = dict(q=q, k_cache=kc, v_cache=vc, block_table=table, cache_seqlens=sl, out=out)
    for err, change in ((TypeError, dict(k_cache=kc.to(BF16))), (TypeError, dict(cache_seqlens=sl.long())),
                        (ValueError, dict(out=out[:, :, :4])), (ValueError, dict(k_cache=kc[:, ::2])),
                        (ValueError, dict(cache_seqlens=sl[:1])), (ValueError, dict(block_table=table[:, ::2])),
                        (ValueError, dict(lse=torch.empty(3, device="cuda"))), (ValueError, dict(cache_seqlens=sl.cpu())),
                        (Exl3rError, dict(scale=0.0)), (Exl3rError, dict(sinks=4)), (Exl3rError, dict(workspace=None, q=q))):
        args = {**ok, **change}
        if err is Exl3rError and "workspace" in change and not ffi.paged_attn_workspace_bytes(q, kc, table):
            continue
        with pytest.raises(err):
            ffi.paged_attn(**args)
    with pytest.raises(Exl3rError):
        ffi.paged_attn_shared(q, kc, vc, table, sl, out, 63)

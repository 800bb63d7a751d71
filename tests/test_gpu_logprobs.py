"""GPU parity of exl3r_token_logprobs against float64.

Tolerances: every term e^(x - m) is off by the relative 2^-24 |x - m| 1.45 + 2^-22 (the difference is rounded, the
exponent is scaled to base 2, one ulp for the exponential); what weighs in the sums has a small |x - m|, and terms with
|x - m| > 40 add nothing.  The fp32 sums of a lane over at most 10^5 terms in chunks and the joins add 2^-18 at most.
So ln l is off by 2^-17, a log probability by that and the rounding 2^-24 of its size; the entropy's second term by
(2^-17 + 2^-18) of itself."""
import math

import numpy as np
import pytest
import torch

import exl3r.ffi as ffi
from exl3r import Exl3rError

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def exact(x, tokens, k, n):
    d = x[:, :n].double()
    bad = torch.isnan(d).any(1) | (d == math.inf).any(1) | torch.isneginf(d).all(1)
    # against the maximum, not against the log-sum-exp: beside logits of 2^127, 64 bits hold no ln n of 8.7
    lp = d - d.amax(1, keepdim=True)
    lp = lp - torch.logsumexp(lp, 1, keepdim=True)
    lp[bad] = math.nan
    inside = (tokens >= 0) & (tokens < n)
    tl = torch.where(inside[:, None], lp.gather(1, tokens.clamp(0, n - 1)[:, None]), -math.inf)[:, 0]
    tl[bad] = math.nan
    p = torch.exp(lp)
    ent = -torch.where(p > 0, p * lp, 0.0).sum(1)
    ent[bad] = math.nan
    # the order: NaN largest, equal values by rising column
    key = torch.where(torch.isnan(d), math.inf, d)
    ids = []
    for r in range(x.shape[0]):
        order = np.lexsort((np.arange(n), -key[r].cpu().numpy(), ~torch.isnan(d[r]).cpu().numpy()))
        ids.append(torch.from_numpy(order[:k].copy()))
    ids = torch.stack(ids).to(x.device)
    return tl, ent, ids, lp.gather(1, ids)


def call(x, tokens, k, max_logit=0, err=None, stream=None):
    rows, vocab = x.shape
    lp, ent = (torch.full((rows,), 7.0, device="cuda") for _ in range(2))
    ids = torch.full((rows, k), -7, dtype=torch.int64, device="cuda") if k else None
    tl = torch.full((rows, k), 7.0, device="cuda") if k else None
    ws = torch.full((ffi.token_logprobs_workspace_bytes(rows, vocab),), 0xff, dtype=torch.uint8, device="cuda")
    ffi.token_logprobs(x, tokens, lp, ent, ids, tl, max_logit, ws, err, stream)
    torch.cuda.synchronize()
    return lp, ent, ids, tl


def close(got, want, rel, what):
    g, w = got.double(), want
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what
    inf = torch.isinf(w)
    assert torch.equal(g[inf], w[inf]), what
    f = torch.isfinite(w)
    d = (g - w).abs()[f]
    assert (d <= 2.0 ** -17 + rel * w.abs()[f]).all(), f"{what}: off by {d.max().item()}"


def check(x, tokens, k, max_logit=0, tag=""):
    n = x.shape[1] if max_logit <= 0 else min(max_logit, x.shape[1])
    lp, ent, ids, tl = call(x, tokens, k, max_logit)
    el, ee, ei, et = exact(x, tokens, k, n)
    close(lp, el, 2.0 ** -23, tag + " logprob")
    close(ent, ee, 2.0 ** -16, tag + " entropy")
    if k:
        assert torch.equal(ids, ei), tag + " top ids"
        close(tl, et, 2.0 ** -23, tag + " top logprobs")
    print(tag, "ok", flush=True)


def logits(rows, vocab, dtype, seed, std=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g, device="cuda") * std).to(DT[dtype])


def tokens_of(rows, vocab, seed):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000)
    return torch.randint(0, vocab, (rows,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 7, 7), (3, 63, 20), (2, 64, 32), (5, 65, 1), (2, 511, 0), (4, 2048, 5),
                                          (3, 2049, 32), (2, 8193, 20), (9, 32003, 20), (1, 151936, 20), (2, 152064, 32)])
def test_against_float64(rows, vocab, k, dtype):
    check(logits(rows, vocab, dtype, rows + vocab), tokens_of(rows, vocab, vocab), k, tag=f"{rows}x{vocab} {dtype} k{k}")


@pytest.mark.parametrize("rows,vocab,dtype", [(600, 4001, "f16"), (1030, 2000, "f32"), (700, 9001, "bf16"), (130, 20000, "f32")])
def test_many_rows(rows, vocab, dtype):
    check(logits(rows, vocab, dtype, 5), tokens_of(rows, vocab, 6), 4, tag=f"{rows}x{vocab} {dtype}")


@pytest.mark.parametrize("rows", [3, 600])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_ties_and_sorted_rows(rows, dtype):
    """All equal, rising, falling, signed zeros, a handful of values."""
    vocab = 5000
    x = torch.empty((rows, vocab), device="cuda")
    x[0] = 1.5
    x[1] = torch.linspace(-20, 20, vocab, device="cuda")
    x[2] = torch.linspace(20, -20, vocab, device="cuda")
    if rows > 3:
        x[3] = torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0)
        x[4:] = torch.randint(0, 4, (rows - 4, vocab), device="cuda").float()
    check(x.to(DT[dtype]), tokens_of(rows, vocab, 1), 32, tag=f"ties {rows} {dtype}")


@pytest.mark.parametrize("rows", [8, 520])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masked_infinite_and_nan(rows, dtype):
    vocab, t = 6001, DT[dtype]
    x = logits(rows, vocab, dtype, 77)
    tok = tokens_of(rows, vocab, 3)
    x[0, 10:] = -math.inf                        # a grammar leaves ten columns
    x[1] = -math.inf                             # ... or none
    x[2] = -math.inf
    x[2, 4321] = 2.0                             # ... or one
    x[3, 100:6000] = torch.finfo(t).min          # the type's lowest value as a mask
    x[4, 17] = math.nan
    x[4, 5000] = math.nan
    x[5, 55] = math.inf
    x[6] = torch.finfo(t).min
    x[7] = -1e4
    x[7, 3] = 1e4                                # all the probability on one
    tok[0], tok[2], tok[7] = 11, 4321, 3
    check(x, tok, 20, tag=f"masks {rows} {dtype}")


@pytest.mark.parametrize("max_logit", [1, 33, 64, 1000, 5999, 6000, 7000])
def test_max_logit(max_logit):
    x = logits(3, 6000, "f16", 5)
    x[:, 1000:] += 30
    x[2, 1000:] = math.nan
    tok = torch.tensor([0, 999, 5999], device="cuda")
    check(x, tok, min(max_logit, 6), max_logit, tag=f"max_logit {max_logit}") if max_logit < 1001 else \
        check(x[:2].contiguous(), tok[:2].contiguous(), 6, max_logit, tag=f"max_logit {max_logit}")


def test_tokens_outside():
    x = logits(5, 300, "f32", 5)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    lp, _, _, _ = call(x, torch.tensor([0, 299, 250, 7, 8], device="cuda"), 0, 250, err)
    assert err.item() == 0 and torch.isinf(lp).tolist() == [False, True, True, False, False]
    for bad in (-1, 300, -100, 2 ** 62, -2 ** 63):
        err.zero_()
        lp, _, _, _ = call(x, torch.tensor([1, bad, 2, 3, 4], device="cuda"), 3, 0, err)
        assert err.item() == 1 and lp[1].item() == -math.inf and torch.isfinite(lp[[0, 2, 3, 4]]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [4, 530])
def test_strides_and_alignment(rows, dtype):
    """Rows inside a wider buffer at odd offsets: the columns around them (NaN) stay out."""
    vocab, wide = 3001, 3040
    for off in (0, 1, 3):
        buf = torch.full((rows * wide + 64,), math.nan, device="cuda", dtype=DT[dtype])
        x = buf[off:off + rows * wide].view(rows, wide)[:, 5:5 + vocab]
        x.copy_(logits(rows, vocab, dtype, off))
        check(x, tokens_of(rows, vocab, off), 7, tag=f"off {off} {dtype}")


def test_optional_outputs_and_empty():
    x = logits(6, 5000, "f16", 2)
    tok = tokens_of(6, 5000, 2)
    lp, ent, ids, tl = call(x, tok, 9)
    ws = torch.empty(ffi.token_logprobs_workspace_bytes(6, 5000), dtype=torch.uint8, device="cuda")
    e2 = torch.empty(6, device="cuda")
    ffi.token_logprobs(x, None, None, e2, workspace=ws)
    l2 = torch.empty(6, device="cuda")
    ffi.token_logprobs(x, tok, l2, workspace=ws)
    i2, t2 = torch.empty((6, 9), dtype=torch.int64, device="cuda"), torch.empty((6, 9), device="cuda")
    ffi.token_logprobs(x, None, None, None, i2, t2, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(e2, ent) and torch.equal(l2, lp) and torch.equal(i2, ids) and torch.equal(t2, tl)
    ffi.token_logprobs(x[:0], tok[:0], l2[:0], e2[:0])


def test_follows_the_argmax():
    """top_ids[:, 0] is argmax_sample's index and its log probability the row's largest."""
    for rows, dtype in ((64, "f16"), (64, "f32"), (700, "bf16")):
        x = logits(rows, 20000, dtype, rows)
        ids = torch.empty(rows, dtype=torch.int64, device="cuda")
        ffi.argmax_sample(x, ids)
        lp, _, top, tl = call(x, ids, 3)
        assert torch.equal(top[:, 0], ids) and torch.equal(tl[:, 0], lp)


def test_graph_replays():
    for rows in (16, 600):
        x = logits(rows, 9001, "f16", 9)
        tok = tokens_of(rows, 9001, 9)
        lp, ent = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        ids, tl = torch.empty((rows, 20), dtype=torch.int64, device="cuda"), torch.empty((rows, 20), device="cuda")
        ws = torch.empty(ffi.token_logprobs_workspace_bytes(rows, 9001), dtype=torch.uint8, device="cuda")
        run = lambda: ffi.token_logprobs(x, tok, lp, ent, ids, tl, workspace=ws)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for k in range(3):
            x.copy_(logits(rows, 9001, "f16", 20 + k))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in (lp, ent, ids, tl)]
            for a, b in zip(got, call(x, tok, 20)):
                assert torch.equal(a, b), f"replay {k}"


def test_two_streams():
    xs = [logits(40, 30000, "f16", s) for s in (1, 2)]
    tok = tokens_of(40, 30000, 1)
    want = [call(x, tok, 5) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    bufs = []
    for x, s in zip(xs, streams):
        b = (torch.empty(40, device="cuda"), torch.empty(40, device="cuda"), torch.empty((40, 5), dtype=torch.int64, device="cuda"),
             torch.empty((40, 5), device="cuda"))
        ws = torch.empty(ffi.token_logprobs_workspace_bytes(40, 30000), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        bufs.append((b, ws))
        ffi.token_logprobs(x, tok, *b, workspace=ws, stream=s)
    torch.cuda.synchronize()
    for (b, _), w in zip(bufs, want):
        assert all(torch.equal(i, j) for i, j in zip(b, w))


def test_wrapper_refusals():
    x = logits(4, 100, "f16", 1)
    tok = tokens_of(4, 100, 1)
    lp = torch.empty(4, device="cuda")
    ws = torch.empty(ffi.token_logprobs_workspace_bytes(4, 100), dtype=torch.uint8, device="cuda")
    ids, tl = torch.empty((4, 33), dtype=torch.int64, device="cuda"), torch.empty((4, 33), device="cuda")
    for args in ((x, tok.int(), lp), (x, tok[:3], lp), (x, None, lp), (x, tok, lp.half()), (x, tok, lp, None, ids, None),
                 (x, tok, lp, None, ids.int(), tl), (x, tok.cpu(), lp)):
        with pytest.raises((ValueError, TypeError)):
            ffi.token_logprobs(*args, workspace=ws)
    for args, kw in (((x, tok, lp, None, ids, tl), dict(workspace=ws)), ((x, tok, lp), {}), ((x, tok, lp), dict(workspace=ws[:-1])),
                     ((x.long(), tok, lp), dict(workspace=ws))):
        with pytest.raises(Exl3rError):
            ffi.token_logprobs(*args, **kw)


@pytest.mark.parametrize("rows,vocab,dtype,k", [(260, 524288, "f16", 5), (257, 524289, "bf16", 0), (3, 700001, "f16", 32),
                                                (255, 4096, "f32", 3), (256, 4096, "f32", 3)])
def test_where_the_kernel_changes(rows, vocab, dtype, k):
    """The most group maxima that a row keeps in LDS and one step more, more than a lane keeps in registers, and the rows
    from which on a workgroup has one."""
    check(logits(rows, vocab, dtype, 11), tokens_of(rows, vocab, 12), k, tag=f"{rows}x{vocab} {dtype} k{k}")

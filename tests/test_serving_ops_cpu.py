"""Refusals and workspace sizes of exl3r_paged_attn(_shared) and exl3r_token_logprobs through the C ABI: every call here
fails its validation (or has nothing to do) before any HIP call."""
import pytest

import exl3r

FAKE = 0x100000   # never dereferenced
F32, F16, BF16, I64 = exl3r.F32, exl3r.F16, exl3r.BF16, exl3r.I64


def attn(shared=None, **kw):
    a = dict(q=FAKE, qts=8 * 128, qhs=128, hq=8, kc=FAKE, vc=FAKE, hk=2, page=256, pages=10, table=FAKE, blocks=4, lens=FAKE,
             dt=F16, bsz=2, seq=1, hd=128, scale=0.1, window=0, sinks=0, out=FAKE, ots=8 * 128, ohs=128, lse=None, err=None,
             ws=FAKE, wsb=1 << 40, stream=None)
    a.update(kw)
    v = list(a.values())
    lib = exl3r.load()
    return lib.exl3r_paged_attn(*v) if shared is None else lib.exl3r_paged_attn_shared(*v[:12], shared, *v[12:])


def err():
    return exl3r.load().exl3r_last_error().decode()


@pytest.mark.parametrize("shared", [None, 0, 256])
@pytest.mark.parametrize("code,what,change", [
    (exl3r.EDTYPE, "dtype", dict(dt=F32)), (exl3r.EDTYPE, "dtype", dict(dt=I64)),
    (exl3r.EINVAL, "head_dim", dict(hd=96)), (exl3r.EINVAL, "head_dim", dict(hd=512)), (exl3r.EINVAL, "shape", dict(hq=7)),
    (exl3r.EINVAL, "shape", dict(hk=0)), (exl3r.EINVAL, "shape", dict(bsz=-1)), (exl3r.EINVAL, "power of two", dict(page=48)),
    (exl3r.EINVAL, "power of two", dict(page=0)), (exl3r.EINVAL, "cache", dict(pages=0)), (exl3r.EINVAL, "cache", dict(blocks=0)),
    (exl3r.EINVAL, "scale", dict(scale=0.0)), (exl3r.EINVAL, "scale", dict(scale=-1.0)),
    (exl3r.EINVAL, "scale", dict(scale=float("nan"))), (exl3r.EINVAL, "scale", dict(scale=float("inf"))),
    (exl3r.EINVAL, "sinks", dict(sinks=-1, window=5)), (exl3r.EINVAL, "sinks", dict(sinks=4)),
    (exl3r.EINVAL, "2^31", dict(blocks=1 << 40)), (exl3r.EINVAL, "2^31", dict(bsz=1 << 40)),
    (exl3r.EINVAL, "2^31", dict(bsz=1 << 20, seq=1 << 20)),
    (exl3r.EINVAL, "non-null", dict(q=None)), (exl3r.EINVAL, "non-null", dict(kc=None)), (exl3r.EINVAL, "non-null", dict(vc=None)),
    (exl3r.EINVAL, "non-null", dict(table=None)), (exl3r.EINVAL, "non-null", dict(lens=None)),
    (exl3r.EINVAL, "non-null", dict(out=None)), (exl3r.EINVAL, "16-byte", dict(kc=FAKE + 8)),
    (exl3r.EINVAL, "strides", dict(qhs=64)), (exl3r.EINVAL, "strides", dict(ots=64)),
    (exl3r.EINVAL, "workspace", dict(ws=None)), (exl3r.EINVAL, "workspace", dict(ws=FAKE + 64)),
    (exl3r.EINVAL, "workspace", dict(wsb=16)), (exl3r.EINVAL, "workgroups", dict(bsz=1 << 24, hq=2, hk=2)),
])
def test_attention_refusals(shared, code, what, change):
    assert attn(shared, **change) == code
    assert what in err(), err()


def test_shared_len():
    for bad in (-256, 1, 100, 5 * 256, 1 << 40):
        assert attn(bad) == exl3r.EINVAL and "shared_len" in err()


def test_nothing_to_do():
    assert attn(bsz=0, q=None, kc=None, vc=None, out=None, table=None, lens=None) == exl3r.OK
    assert attn(seq=0) == exl3r.OK
    assert attn(256, bsz=0) == exl3r.OK
    assert attn(bsz=0, hd=96) == exl3r.EINVAL


def test_attention_workspace_size():
    f = exl3r.load().exl3r_paged_attn_workspace_bytes
    assert f(64, 1, 64, 8, 128, 256, 64, 0) % 256 == 0
    assert 0 < f(1, 1, 16, 8, 128, 256, 16, 0) < 1 << 20
    for bad in ((0, 1, 8, 8, 128, 256, 4, 0), (1, 1, 8, 3, 128, 256, 4, 0), (1, 1, 8, 8, 128, 256, 1 << 40, 0),
                (1 << 40, 1 << 40, 8, 8, 128, 256, 4, 0), (1, 1, 8, 8, 128, 256, 4, 1 << 40), (1, 1, 8, 8, 128, 0, 4, 0)):
        assert f(*bad) == 0
    # the partial results of the largest prefill chunk of the repository's models stay well under a gigabyte
    assert f(1, 8192, 64, 8, 128, 256, 512, 0) < 1 << 30


def logprobs(**kw):
    a = dict(x=FAKE, dt=F16, rows=4, vocab=1000, ld=1000, mask=0, tok=FAKE, lp=FAKE, ent=FAKE, k=5, ids=FAKE, tl=FAKE, err=None,
             ws=FAKE, wsb=1 << 40, stream=None)
    a.update(kw)
    return exl3r.load().exl3r_token_logprobs(*a.values())


@pytest.mark.parametrize("code,what,change", [
    (exl3r.EDTYPE, "dtype", dict(dt=I64)), (exl3r.EINVAL, "shape", dict(rows=-1)), (exl3r.EINVAL, "shape", dict(vocab=0)),
    (exl3r.EINVAL, "shape", dict(ld=999)), (exl3r.EINVAL, "shape", dict(rows=1 << 40)), (exl3r.EINVAL, "shape", dict(vocab=1 << 40)),
    (exl3r.EINVAL, "top_k", dict(k=-1)), (exl3r.EINVAL, "top_k", dict(k=33)), (exl3r.EINVAL, "top_k", dict(mask=4)),
    (exl3r.EINVAL, "non-null", dict(x=None)), (exl3r.EINVAL, "non-null", dict(lp=None)), (exl3r.EINVAL, "non-null", dict(ids=None)),
    (exl3r.EINVAL, "non-null", dict(tl=None)), (exl3r.EINVAL, "workspace", dict(ws=None)),
    (exl3r.EINVAL, "workspace", dict(ws=FAKE + 8)), (exl3r.EINVAL, "workspace", dict(wsb=0)),
])
def test_logprobs_refusals(code, what, change):
    assert logprobs(**change) == code
    assert what in err(), err()


def test_logprobs_nothing_to_do():
    assert logprobs(rows=0, x=None, tok=None, lp=None, ent=None, ids=None, tl=None, ws=None, wsb=0) == exl3r.OK
    assert logprobs(rows=0, k=40) == exl3r.EINVAL
    f = exl3r.load().exl3r_token_logprobs_workspace_bytes
    assert f(0, 5) == 0 and f(5, 0) == 0 and f(1 << 40, 5) == 0 and f(64, 151936) % 256 == 0 and f(64, 151936) > 0


@pytest.mark.parametrize("rows", [1, 64, 300])
def test_logprobs_workspace_for_fewer_columns(rows):
    """A workspace for all columns serves every max_logit: also where a wider slice makes fewer slices."""
    sizes = [exl3r.load().exl3r_token_logprobs_workspace_bytes(rows, steps * 8192) for steps in (1, 19, 64, 65, 255, 256, 257, 512, 513)]
    if rows < 256:
        assert sizes == sorted(sizes)
    else:
        assert sizes[:3] == [0, 0, 0] and sizes == sorted(sizes)


@pytest.mark.parametrize("what,change", [("2^22", dict(hk=1 << 16, hq=1 << 16)), ("scale", dict(scale=2.5e38)),
                                         ("workgroups", dict(bsz=1 << 12, seq=1 << 14, hq=16, hk=16, hd=256, qts=4096, qhs=256, ots=4096, ohs=256))])
def test_attention_size_limits(what, change):
    assert attn(**change) == exl3r.EINVAL
    assert what in err(), err()


def test_wrappers_refuse_host_tensors():
    import torch

    import exl3r.ffi as ffi

    q, kc = torch.zeros(1, 1, 4, 64).half(), torch.zeros(4, 16, 2, 64).half()
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for stream in (None, 0):
        with pytest.raises(ValueError, match="GPU"):
            ffi.paged_attn(q, kc, kc, table, lens, torch.zeros_like(q), stream=stream)
        with pytest.raises(ValueError, match="GPU"):
            ffi.paged_attn_shared(q, kc, kc, table, lens, torch.zeros_like(q), 16, stream=stream)
        with pytest.raises(ValueError, match="GPU"):
            ffi.token_logprobs(torch.zeros(2, 100), torch.zeros(2, dtype=torch.int64), torch.zeros(2), stream=stream)

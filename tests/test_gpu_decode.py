"""attention_decode against a 64-bit attention over the same cached rows.

The allowed difference is the rounding to bf16 (half a step, 2^-8 of the value) and what 32-bit sums of these
sizes can lose (serving_ref.decode_bound), computed from the inputs before the kernel runs."""
import math

import pytest
import torch

import kernelfuser_amd as kf
from kernelfuser_amd import _lib
from helpers import announce
from serving_ref import attention, held_rows

pytestmark = pytest.mark.gpu

E8M0 = torch.float8_e8m0fnu


def _batch(lens, geom, page, kind, seed, s=1, order="head", spare=1, dtype=torch.int32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    hq, hk, d = geom
    b = len(lens)
    per = -(-max(max(lens), 1) // page) + spare
    n = b * per
    shape = (n, hk, page, d) if order == "head" else (n, page, hk, d)
    rows = [torch.randn(shape, generator=g).to(torch.bfloat16) for _ in range(2)]
    rows = [r if order == "head" else r.transpose(1, 2) for r in rows]
    scales = [None, None]
    if kind == "e4m3":
        rows = [(r.float() * 64).to(torch.float8_e4m3fn) for r in rows]
        scales = [(121 + torch.randint(-1, 2, (n, hk, page), generator=g)).to(torch.uint8).view(E8M0) for _ in range(2)]
    pages = torch.randperm(n, generator=g).view(b, per).to(dtype)
    q = (spread * torch.randn(b, hq, s, d, generator=g)).to(torch.bfloat16)
    return {"q": q, "cache": (*rows, *scales), "pages": pages, "lengths": torch.tensor(lens, dtype=dtype)}


def _gpu(x, dev):
    return {k: tuple(t if t is None else t.to(dev) for t in v) if isinstance(v, tuple) else v.to(dev)
            for k, v in x.items()}


def _decode(y, **kw):
    kc, vc, ks, vs = y["cache"]
    return kf.attention_decode(y["q"], kc, vc, y["pages"], y["lengths"], ks, vs, **kw)


def _check(x, got, window=None, softcap=None, scale=None):
    got = got.cpu().double()
    kc, vc, ks, vs = x["cache"]
    for i in range(got.shape[0]):
        n = int(x["lengths"][i])
        if n == 0:
            assert bool((got[i] == 0).all())
            continue
        k, v = held_rows(kc, ks, x["pages"][i], n), held_rows(vc, vs, x["pages"][i], n)
        want, bound = attention(x["q"][i].double(), k, v, window, softcap, scale)
        off = (got[i] - want).abs() - (2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * bound + 1e-38)
        assert float(off.max()) <= 0, (i, n, float(off.max()), float((got[i] - want).abs().max()))


CASES = [  # lengths, geometry, page, kind, S, window, softcap, order, index
    ([1], (4, 4, 128), 16, "bf16", 1, None, None, "head", torch.int32),
    ([1, 2, 15, 16, 17], (4, 1, 256), 16, "bf16", 1, None, None, "head", torch.int64),
    ([31, 32, 33, 0, 127, 128, 129], (8, 2, 128), 16, "e4m3", 1, None, None, "token", torch.int32),
    ([333], (32, 8, 128), 64, "bf16", 1, None, None, "head", torch.int32),
    ([1000, 3, 0, 511], (16, 8, 256), 32, "e4m3", 1, None, None, "head", torch.int64),
    ([700, 90], (8, 4, 256), 64, "bf16", 1, 100, None, "token", torch.int32),
    ([700, 90, 5], (8, 4, 128), 128, "e4m3", 1, 1, 30.0, "head", torch.int32),
    ([300, 2, 0, 65], (6, 2, 128), 16, "bf16", 3, None, None, "head", torch.int32),
    ([300, 2, 1, 64], (16, 2, 128), 32, "e4m3", 5, 20, None, "head", torch.int64),
    ([260, 16, 17], (8, 1, 256), 64, "bf16", 16, None, 50.0, "head", torch.int32),
    ([129, 70], (64, 8, 128), 256, "bf16", 4, 64, None, "token", torch.int32),
    ([200, 31], (16, 1, 128), 16, "e4m3", 16, 33, None, "head", torch.int32),
    ([97], (40, 1, 256), 16, "bf16", 7, None, None, "head", torch.int32),
    ([513, 40], (5, 5, 128), 32, "bf16", 2, None, None, "head", torch.int32),
    ([2500, 7], (4, 2, 128), 16, "bf16", 1, None, None, "head", torch.int32),
]


@pytest.mark.parametrize("lens,geom,page,kind,s,window,softcap,order,index", CASES)
def test_decode_matches_64_bits(gpu, lens, geom, page, kind, s, window, softcap, order, index):
    announce(f"decode {lens} {geom} page={page} {kind} S={s} window={window} cap={softcap} {order} {index}")
    x = _batch(lens, geom, page, kind, 17, s, order, dtype=index)
    y = _gpu(x, gpu)
    got = _decode(y, window=window, softcap=softcap)
    torch.cuda.synchronize()
    _check(x, got, window, softcap)
    out = torch.full_like(got, float("nan"))
    assert _decode(y, window=window, softcap=softcap, out=out) is out
    assert torch.equal(out, got)  # the same bits on every call


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("b,l", [(1, 9000), (3, 5000), (40, 600)])
def test_decode_split_and_joined(gpu, b, l, kind):
    """Lengths that are split over workgroups, alone and in ragged batches; with and without a workspace."""
    announce(f"decode split b={b} l={l} {kind}")
    g = torch.Generator().manual_seed(b)
    lens = [l] + torch.randint(0, l, (b - 1,), generator=g).tolist()
    x = _batch(lens, (8, 2, 128), 64, kind, 23)
    y = _gpu(x, gpu)
    got = _decode(y)
    none = _decode(y, work=torch.empty(0, dtype=torch.uint8, device=gpu))
    few = [0] + list(range(1, b, 7))
    part = {"q": x["q"][few], "cache": x["cache"], "pages": x["pages"][few], "lengths": x["lengths"][few]}
    _check(part, got[few])
    _check(part, none[few])


def test_decode_large_scores_and_scale(gpu):
    """Scores of some hundreds: one key takes nearly everything; a scale of the caller's own."""
    announce("decode large scores")
    x = _batch([400, 37], (8, 2, 128), 16, "bf16", 31, spread=30.0)
    y = _gpu(x, gpu)
    _check(x, _decode(y))
    _check(x, _decode(y, scale=0.01), scale=0.01)
    _check(x, _decode(y, softcap=20.0), softcap=20.0)
    _check(x, _decode(y, softcap=3e4), softcap=3e4)  # hardly a cap: scores far below it keep their digits
    _check(x, _decode(y, softcap=1e12), softcap=1e12)


@pytest.mark.parametrize("b,geom,s,kind", [(70, (4, 2, 128), 1, "bf16"), (300, (2, 1, 128), 2, "e4m3"), (2, (64, 1, 128), 4, "bf16"),
                                           (3, (48, 1, 256), 3, "e4m3")])
def test_decode_many_sequences_and_many_rows(gpu, b, geom, s, kind):
    """More sequences than lanes of a wave, and more query rows than a pass takes, split sequences among them."""
    announce(f"decode b={b} {geom} S={s} {kind}")
    g = torch.Generator().manual_seed(b)
    lens = torch.randint(0, 60, (b,), generator=g).tolist()
    lens[0], lens[-1], lens[b // 2] = 1500, 700, 0
    x = _batch(lens, geom, 32, kind, 71, s)
    got = _decode(_gpu(x, gpu))
    some = sorted({0, 1, b // 2, b - 1, min(64, b - 1), min(65, b - 1)})
    part = {"q": x["q"][some], "cache": x["cache"], "pages": x["pages"][some], "lengths": x["lengths"][some]}
    _check(part, got[some])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("s,window", [(1, None), (1, 40), (4, None), (4, 40), (3, 1)])
def test_decode_does_not_see_what_is_masked(gpu, s, window, kind):
    """NaN and infinities behind each query's last key and before its window, in rows, scales and page entries, leave
    the result's bits as they are."""
    announce(f"decode garbage outside S={s} window={window} {kind}")
    lens = [100, 33, 5, 161, 0]
    x = _batch(lens, (8, 2, 128), 16, kind, 41, s, spare=2)
    clean = _decode(_gpu(x, gpu), window=window)
    _check(x, clean, window)
    kc, vc, ks, vs = (None if t is None else t.clone() for t in x["cache"])
    pages = x["pages"].clone()
    used = torch.zeros(kc.shape[0], 16, dtype=torch.bool)
    for i, n in enumerate(lens):
        lo = max(0, n - s - window + 1) if window else 0
        for j in range(lo, n):
            used[pages[i, j // 16], j % 16] = True
        first, last = lo // 16, -(-n // 16)
        pages[i, last:] = -(2 ** 31)
        pages[i, :first] = 2 ** 31 - 1
    for t in (kc, vc):
        for pg, at in (~used).nonzero().tolist():
            t[pg, :, at] = torch.tensor(math.nan if (pg + at) % 2 else (math.inf if kind == "bf16" else math.nan)).to(t.dtype)
    for t in (ks, vs):
        if t is not None:
            t.view(torch.uint8)[(~used)[:, None].expand(-1, 2, -1)] = 255
    dirty = dict(x, cache=(kc, vc, ks, vs), pages=pages)
    got = _decode(_gpu(dirty, gpu), window=window)
    assert torch.equal(got, clean)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_decode_drafted_token_does_not_reach_earlier_queries(gpu, value):
    """The last of three tokens has NaN or infinities in its K and V: the first two do not see it, the third is NaN
    (an infinite V: infinite or NaN)."""
    announce(f"decode drafted {value}")
    x = _batch([50, 3, 33], (8, 2, 128), 16, "bf16", 43, 3)
    clean = _decode(_gpu(x, gpu))
    kc, vc = x["cache"][0].clone(), x["cache"][1].clone()
    for i, n in enumerate([50, 3, 33]):
        pg, at = int(x["pages"][i, (n - 1) // 16]), (n - 1) % 16
        kc[pg, :, at] = value
        vc[pg, :, at] = value
    got = _decode(_gpu(dict(x, cache=(kc, vc, None, None)), gpu))
    assert torch.equal(got[:, :, :2], clean[:, :, :2])
    assert not torch.isfinite(got[:, :, 2]).any()
    # the same with a window that only the first query still sees through
    kc, vc = x["cache"][0].clone(), x["cache"][1].clone()
    pg, at = int(x["pages"][0, 28 // 16]), 28 % 16  # key 28: seen by query 0 (position 47, window 20), not by 1 and 2
    kc[pg, :, at] = value
    vc[pg, :, at] = value
    clean = _decode(_gpu(x, gpu), window=20)
    got = _decode(_gpu(dict(x, cache=(kc, vc, None, None)), gpu), window=20)
    assert torch.equal(got[:, :, 1:], clean[:, :, 1:]) and not torch.isfinite(got[0, :, 0]).any()


def test_decode_visible_nan_and_infinities(gpu):
    """A NaN in a visible key or value makes that head's row NaN, as the formula does; other sequences keep their bits."""
    announce("decode visible NaN")
    x = _batch([60, 60, 60], (4, 2, 128), 16, "bf16", 47)
    clean = _decode(_gpu(x, gpu))
    kc, vc = x["cache"][0].clone(), x["cache"][1].clone()
    kc[int(x["pages"][0, 1]), 0, 3, 5] = math.nan
    vc[int(x["pages"][1, 2]), 1, 7, 9] = math.inf
    got = _decode(_gpu(dict(x, cache=(kc, vc, None, None)), gpu)).cpu()
    clean = clean.cpu()
    assert torch.isnan(got[0, :2]).all() and torch.equal(got[0, 2:], clean[0, 2:])
    assert bool((got[1, 2:, 0, 9] == math.inf).all()) and torch.equal(got[1, :2], clean[1, :2])
    keep = torch.arange(128) != 9
    assert torch.equal(got[1, 2:, 0, keep], clean[1, 2:, 0, keep]) and torch.equal(got[2], clean[2])


def test_decode_wrong_lengths_and_pages(gpu):
    """Wrong indices reach their own sequence only, as NaN."""
    announce("decode wrong indices")
    x = _batch([60, 64, 20, 30, 48], (4, 2, 128), 16, "bf16", 53, spare=0)
    clean = _decode(_gpu(x, gpu)).cpu()
    x["lengths"][0] = 65
    x["lengths"][2] = -3
    x["pages"][3, 1] = x["cache"][0].shape[0]
    x["pages"][4, 0] = -1
    got = _decode(_gpu(x, gpu)).cpu()
    assert torch.equal(got[1], clean[1])
    for i in (0, 2, 3, 4):
        assert torch.isnan(got[i]).all()


def test_decode_strided_queries_and_int64_offsets(gpu):
    """q as a view of a fused projection; a cache of more than 2^32 bytes and 2^31 elements whose pages in use are its last."""
    announce("decode large cache")
    x = _batch([130, 7], (8, 2, 128), 64, "bf16", 59)
    n = x["cache"][0].shape[0]
    total = 2 ** 31 // (2 * 64 * 128) + n + 1
    big = [torch.zeros(total, 2, 64, 128, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    for t, c in zip(big, x["cache"]):
        t[total - n:] = c.to(gpu)
    wide = torch.randn(2, 1, 3 * 8 * 128, device=gpu).to(torch.bfloat16)
    wide[:, :, 1024:2048] = x["q"].to(gpu).transpose(1, 2).reshape(2, 1, 1024)
    q = wide[:, :, 1024:2048].view(2, 1, 8, 128).transpose(1, 2)
    got = kf.attention_decode(q, *big, (x["pages"] + (total - n)).to(gpu), x["lengths"].to(gpu))
    _check(x, got)
    dense = kf.cache_to_dense(*big, (x["pages"] + (total - n)).to(gpu), x["lengths"].to(gpu), 130)
    assert torch.equal(dense[0][0].cpu().double(), held_rows(x["cache"][0], None, x["pages"][0], 130))
    k = torch.randn(1, 2, 1, 128, device=gpu).to(torch.bfloat16)
    slot = torch.tensor([[total * 64 - 1]], device=gpu)
    kf.norm_rope_to_cache(None, k, k, None, torch.ones(128, dtype=torch.bfloat16, device=gpu), None, None, None, slot, *big)
    assert torch.equal(big[1][-1, :, 63], k[0, :, 0]) and float(big[0][-1, :, 63].float().abs().sum()) > 0


def test_decode_graph_replays_and_streams(gpu):
    """Captured calls (two graphs, each with its own workspace) replayed with eager calls on other streams between
    them, lengths changed in place between replays."""
    announce("decode graphs and streams")
    x = _batch([3000, 40, 0, 700], (8, 2, 128), 64, "bf16", 61)
    y = _gpu(x, gpu)
    want = _decode(y)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got = _decode(y)
        graphs.append((graph, got))
    other = torch.cuda.Stream()
    for i in range(4):
        for graph, got in graphs:
            got.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            eager = _decode(y)
        for graph, got in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, want)
        for _, got in graphs:
            assert torch.equal(got, want), i
        if i == 1:
            y["lengths"].copy_(torch.tensor([10, 3100, 5, 0], dtype=torch.int32).clamp(max=3008))
            want = _decode(y)
            torch.cuda.synchronize()


def test_decode_own_workspace_is_left_ready(gpu):
    announce("decode own workspace")
    x = _batch([4000, 100], (8, 2, 128), 64, "bf16", 67)
    y = _gpu(x, gpu)
    n = kf.attention_decode_workspace_bytes(2, 8, 2, 1, 128, x["pages"].shape[1] * 64)
    work = torch.zeros(max(n, 1), dtype=torch.uint8, device=gpu)
    want = _decode(y)
    for _ in range(3):
        assert torch.equal(_decode(y, work=work), want)
        assert int(work[:8192].sum()) == 0


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_decode_shared_pages_and_in_place(gpu, kind):
    """Sequences that share a prefix's pages, one sequence twice, one page several times in a row; out is q."""
    announce(f"decode shared pages {kind}")
    x = _batch([700, 700, 333, 64, 700], (32, 2, 128), 64, kind, seed=41, s=2)
    x["pages"][1, :8] = x["pages"][0, :8]
    x["pages"][4] = x["pages"][0]
    x["q"][4] = x["q"][0]
    x["pages"][2, :5] = 7
    y = _gpu(x, gpu)
    got = _decode(y)
    _check(x, got)
    assert _decode(y, out=y["q"]) is y["q"] and torch.equal(y["q"], got)


def test_decode_ratio_of_scale_and_cap_beyond_32_bits(gpu):
    """A cap of 1e-30 under a scale of 1e30: scores of at most 1e-30 whatever q . k is, 0 included, so every key has
    the same weight to 1e-30, as under any other scale."""
    announce("decode extreme scale over cap")
    x = _batch([40], (2, 1, 128), 16, "bf16", seed=43)
    x["q"][0, 1] = 0
    _check(x, _decode(_gpu(x, gpu), scale=1e30, softcap=1e-30), softcap=1e-30)


@pytest.mark.parametrize("geom,s,nt", [((32, 1, 128), 1, 2), ((8, 2, 128), 8, 2), ((64, 1, 128), 1, 4), ((16, 2, 128), 7, 4),
                                       ((80, 1, 128), 1, 4), ((32, 1, 256), 1, 2), ((12, 4, 256), 16, 2)])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_decode_wide_passes(gpu, geom, s, nt, kind):
    """Page tables of a large capacity, hardly used: the widest passes (32 and 64 rows; 16 in bf16 at D = 256), also
    where the rows do not fill them; split and joined, short and empty sequences.  The same rows under a small table, in narrow passes."""
    announce(f"decode wide {geom} S={s} {kind}")
    x = _batch([3000, 0, 37, 1], geom, 64, kind, seed=47, s=s)
    y = _gpu(x, gpu)
    narrow = _decode(y)
    _check(x, narrow)
    wide = dict(y, pages=torch.nn.functional.pad(y["pages"], (0, 2 ** 15), value=-1))
    with _lib.record_launches() as seen:
        got = _decode(wide)
    nt = 1 if geom[2] == 256 and kind == "bf16" else nt
    assert f"decode_kernel<{geom[2]}, {'true' if kind == 'e4m3' else 'false'}, {nt}, " in str(seen.kernels())
    _check(x, got)
    _check(x, _decode(wide, window=100, softcap=20.0), 100, 20.0)

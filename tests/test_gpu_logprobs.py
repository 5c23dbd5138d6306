"""token_logprobs against 64-bit log-softmax.

Allowed difference: 32-bit sums of V positive terms lose at most (V/64 + 64) 2^-24 of the sum in any order the kernel
uses (64 or more partial sums), a term's exponent x - m is one rounding (2^-24 of its size, weighted by its own
e^(x-m), so at most 2^-24 in total times the spread), exp and log 2^-22; the results are rounded once more.  Indices are exact."""
import math

import pytest
import torch

import kernelfuser_amd as kf
from helpers import announce
from serving_ref import logprobs

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _compare(x, ids, top, got):
    n, v = x.shape[0] if x.ndim == 2 else x.shape[0] * x.shape[1], x.shape[-1]
    x, ids = x.double().cpu().reshape(n, v), ids.cpu().reshape(n)
    want = logprobs(x, ids, top)
    u = 2.0 ** -24
    sums = (v / 64 + 64) * u + 2.0 ** -21
    for g, w, kind in zip(got, want, ("logp", "entropy", "top")):
        if g is None:
            continue
        g = g.cpu().double().reshape(w.shape)
        assert torch.equal(torch.isnan(g), torch.isnan(w)), kind
        assert torch.equal(torch.isinf(g), torch.isinf(w)), kind
        fine = torch.isfinite(w)
        # entropy: terms p (x - m) up to log V of them count as much as the sum itself
        size = w[fine].abs() + math.log(v) + 1
        off = (g[fine] - w[fine]).abs() - 2 * (sums + 4 * u) * size
        assert off.numel() == 0 or float(off.max()) <= 0, (kind, float(off.max()))
    if top:
        assert torch.equal(got[3].cpu().reshape(n, top), want[3])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,v,top", [(1, 1, 1), (1, 1, 0), (2, 7, 7), (3, 63, 1), (2, 64, 32), (5, 1001, 5), (2, 4097, 20),
                                     (1, 32000, 5), (3, 50001, 32), (300, 257, 3), (1, 131071, 20), (2, 40000, 0)])
def test_logprobs_match_64_bits(gpu, n, v, top, kind):
    announce(f"logprobs n={n} v={v} top={top} {kind}")
    g = torch.Generator().manual_seed(n * v + top)
    x = (3 * torch.randn(n, v, generator=g)).to(TYPES[kind])
    ids = torch.randint(0, v, (n,), generator=g)
    y = kf.token_logprobs(x.to(gpu), ids.to(gpu), top)
    assert (y.top_ids is None) == (top == 0)
    _compare(x, ids, top, y)
    again = kf.token_logprobs(x.to(gpu), ids.to(gpu).to(torch.int32), top)
    assert all(torch.equal(a, b) for a, b in zip(y, again) if a is not None)


@pytest.mark.parametrize("kind", list(TYPES))
def test_logprobs_rows_that_are_hard(gpu, kind):
    """Ties, zeros of both signs, mostly -infinity, ascending and descending rows, far apart and equal logits, rows
    that are no distribution, ids outside the vocabulary."""
    announce(f"logprobs hard rows {kind}")
    v, top = 20001, 20
    g = torch.Generator().manual_seed(2)
    rows = [torch.zeros(v), torch.full((v,), -3.5), torch.arange(v) / 400.0, -torch.arange(v) / 400.0,
            torch.randint(-3, 3, (v,), generator=g).float(), torch.full((v,), -math.inf), torch.randn(v, generator=g)]
    r = torch.zeros(v)
    r[::2] = -0.0
    rows.append(r)
    for keep in ([5], [19999, 20000, 3], list(range(777, 797)), list(range(0, 20001, 1000))):
        r = torch.full((v,), -math.inf)
        r[keep] = torch.randn(len(keep), generator=g)
        rows.append(r)
    for at, what in ((0, math.nan), (20000, math.nan), (777, math.inf), (3, -math.inf)):
        r = torch.randn(v, generator=g)
        r[at] = what
        rows.append(r)
    r = torch.randn(v, generator=g)
    r[12345] = 6e4
    rows.append(r)
    r = torch.full((v,), -6e4)
    r[19000:] = -5e4
    rows.append(r)
    r = torch.randn(v, generator=g)
    r[13000:13100] = 9.0  # many equal leaders next to each other
    rows.append(r)
    r = torch.randn(v, generator=g) - 20
    r[torch.arange(0, 200) * 64 + 3] = 5.0 + torch.arange(200) / 64  # leaders that one lane would read
    rows.append(r)
    x = torch.stack(rows).to(TYPES[kind])
    ids = torch.randint(0, v, (len(rows),), generator=g)
    ids[0], ids[1], ids[2] = -1, v, 2 ** 40
    _compare(x, ids, top, kf.token_logprobs(x.to(gpu), ids.to(gpu), top))
    one = [kf.token_logprobs(x[i].to(gpu), ids[i].to(gpu), top) for i in range(len(rows))]  # one row: split further
    _compare(x, ids, top, [torch.stack([o[j] for o in one]) for j in range(4)])


@pytest.mark.parametrize("kind", list(TYPES))
def test_logprobs_lowest_and_largest_values(gpu, kind):
    """Masks of the type's lowest value, whole rows of it, and logits next to the type's largest."""
    announce(f"logprobs lowest values {kind}")
    v, top, t = 9001, 8, TYPES[kind]
    low, big = torch.finfo(t).min, torch.finfo(t).max
    g = torch.Generator().manual_seed(9)
    rows = [torch.full((v,), low), torch.full((v,), big), torch.full((v,), low), torch.full((v,), low),
            torch.randn(v, generator=g), torch.full((v,), -math.inf), torch.full((v,), low)]
    rows[2][[4, 5000, 9000]] = torch.tensor([1.0, 2.0, 0.5])
    rows[3][77] = low / 2
    rows[4][100:200] = big
    rows[4][300] = low
    rows[5][8] = low
    rows[6][::3] = -math.inf
    x = torch.stack(rows).to(t)
    ids = torch.tensor([5, 6, 5000, 77, 150, 8, 1])
    _compare(x, ids, top, kf.token_logprobs(x.to(gpu), ids.to(gpu), top))
    one = [kf.token_logprobs(x[i].to(gpu), ids[i].to(gpu), top) for i in range(len(rows))]
    _compare(x, ids, top, [torch.stack([o[j] for o in one]) for j in range(4)])


def test_logprobs_views(gpu):
    """Shifted logits of a batch, rows that do not start on 16 bytes, ids with strides, vectors and empty batches."""
    announce("logprobs views")
    g = torch.Generator().manual_seed(4)
    for kind in TYPES.values():
        full = torch.randn(3, 6, 1003, generator=g).to(kind)
        tok = torch.randint(0, 1003, (3, 6), generator=g)
        x, ids = full.to(gpu)[:, :-1], tok.to(gpu)[:, 1:]
        _compare(full[:, :-1].contiguous(), tok[:, 1:], 4, kf.token_logprobs(x, ids, 4))
        wide = torch.randn(5, 3001, generator=g).to(kind)
        for off in range(1, 9):
            part = wide.to(gpu)[:, off:off + 2900]
            _compare(wide[:, off:off + 2900], tok.view(-1)[:5], 3, kf.token_logprobs(part, tok.view(-1)[:5].to(gpu), 3))
        row = kf.token_logprobs(full.to(gpu)[0, 0], tok.to(gpu)[0, 0], 2)
        assert row.logprobs.shape == () and row.top_ids.shape == (2,)
        none = kf.token_logprobs(full.to(gpu)[:, :0], tok.to(gpu)[:, :0], 2)
        assert none.logprobs.shape == (3, 0) and none.top_ids.shape == (3, 0, 2)


def test_logprobs_graph_and_streams(gpu):
    announce("logprobs graphs and streams")
    x = torch.randn(2, 60001, device=gpu)
    ids = torch.tensor([5, 60000], device=gpu)
    want = [t.clone() for t in kf.token_logprobs(x, ids, 8)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got = kf.token_logprobs(x, ids, 8)
    other = torch.cuda.Stream()
    for _ in range(3):
        for t in got:
            t.fill_(-5)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            eager = kf.token_logprobs(x, ids, 8)
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(got, want, eager):
            assert torch.equal(a, b) and torch.equal(c, b)
    n = kf.token_logprobs_workspace_bytes(2, 60001, 8)
    work = torch.zeros(max(n, 1), dtype=torch.uint8, device=gpu)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(kf.token_logprobs(x, ids, 8, work=work), want))
        assert int(work[:8192].sum()) == 0

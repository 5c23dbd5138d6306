"""The serving ops together, as a program runs them: prompt into the pages, token by token over them, log
probabilities of the answer; and the same through a HuggingFace Qwen3 model (randomly initialised).

Ops: every decoded row is held to a 64-bit attention over the rows that norm_rope prepares for the whole sequence
(the rows in the cache are the same bits), so the bound is that of one decode call.  Model: the logits of the steps
are held to those of a forward over the whole sequence with FP32 attention, no further off than the
BF16-weights arm that the prefill caller is measured with (qwen3.noise_floor_gate)."""
import pytest
import torch

import kernelfuser_amd as kf
from helpers import announce
from kernelfuser_amd import generate as gen
from kernelfuser_amd import qwen3
from serving_ref import attention, logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,kind", [(128, "bf16"), (256, "e4m3")])
def test_a_sequence_written_attended_and_read_back(gpu, d, kind):
    """A ragged batch: prompts of two lengths prefilled in one padded call (slot -1 for padding), then 40 steps."""
    announce(f"ops together d={d} {kind}")
    hq, hk, page, steps = 8, 2, 16, 40
    lens = [21, 5]
    total = max(lens) + steps
    g = torch.Generator().manual_seed(d)
    x = [torch.randn(2, total, h, d, generator=g).to(torch.bfloat16).to(gpu).transpose(1, 2) for h in (hq, hk, hk)]
    gq, gk = ((1 + 0.1 * torch.randn(d, generator=g)).to(torch.bfloat16).to(gpu) for _ in range(2))
    cos, sin = (t.to(gpu) for t in kf.rope_tables(total, d))
    per = -(-total // page)
    pages = torch.randperm(2 * per, generator=g).view(2, per).to(gpu)
    cache = kf.make_cache(2 * per, hk, page, d, gen.KINDS[kind], gpu)

    def slots(pos):
        return torch.gather(pages, 1, pos // page) * page + pos % page

    pos = torch.arange(max(lens), device=gpu).expand(2, max(lens))
    where = slots(pos)
    where[1, lens[1]:] = -1
    args = [t[:, :, : max(lens)] for t in x]
    kf.norm_rope_to_cache(*args, gq, gk, cos, sin, pos, where, *cache)
    # what the cache has to hold: every sequence's own rows at its own positions
    qn, kn = kf.norm_rope(x[0].contiguous(), x[1].contiguous(), gq, gk, cos, sin, norm_style="hf")
    k_ref, v_ref = kn.cpu(), x[2].cpu()
    if kind == "e4m3":
        from serving_ref import quantise
        (kp, ks, _), (vp, vs, _) = quantise(k_ref), quantise(v_ref)
        k_ref, v_ref = kp * ks[..., None], vp * vs[..., None]
    lengths = torch.tensor(lens, device=gpu, dtype=torch.int32)
    for i in range(steps):
        lengths += 1
        at = (lengths.long() - 1)[:, None]
        row = [torch.stack([t[b, :, lens[b] + i] for b in range(2)])[:, :, None] for t in x]
        q = kf.norm_rope_to_cache(*row, gq, gk, cos, sin, at, slots(at), *cache)
        out = kf.attention_decode(q, cache[0], cache[1], pages, lengths, cache[2], cache[3]).cpu().double()
        for b in range(2):
            n = lens[b] + i + 1
            want, bound = attention(qn[b, :, n - 1:n].cpu().double(), k_ref[b, :, :n].double(), v_ref[b, :, :n].double())
            assert float(((out[b] - want).abs() - 2.0 ** -8 * want.abs() - (1 + 2.0 ** -8) * bound).max()) <= 0, (b, i)
    dense = kf.cache_to_dense(cache[0], cache[1], pages, lengths, total, cache[2], cache[3])
    for t, ref in zip(dense, (k_ref, v_ref)):
        for b in range(2):
            n = lens[b] + steps
            assert torch.equal(t[b, :, :n].cpu().double(), ref[b, :, :n].double())
            assert bool((t[b, :, n:] == 0).all())


@pytest.fixture(scope="module")
def model(gpu):
    return qwen3.random_qwen3(layers=2, vocab=4000, device=gpu)


@pytest.mark.parametrize("kind,graph", [("bf16", False), ("bf16", True)])
def test_generation_against_whole_forwards(gpu, model, kind, graph):
    announce(f"generate {kind} graph={graph}")
    torch.manual_seed(3)
    ids = torch.randint(0, 4000, (2, 70), device=gpu)
    got = gen.generate(model, ids, 12, kind=kind, page_size=16, graph=graph)
    whole = torch.cat([ids, got["tokens"]], dim=1)
    # the steps' logits again, token by token, against forwards over the whole sequence
    s = gen.Session(model, 2, 82, kind, 16)
    steps = [s.prefill(ids)[:, -1]]
    for i in range(11):
        steps.append(s.step(got["tokens"][:, i]).clone())
    steps = torch.stack(steps, dim=1)
    arms = {}
    for arm in ("reference", "floor"):
        saved = qwen3.patch(model, arm)
        try:
            arms[arm] = qwen3.forward_logits(model, whole[:, :-1])[:, 69:]
        finally:
            qwen3.restore(saved)
    off, floor = (qwen3.quality(t, arms["reference"], whole[:, 70:]) for t in (steps, arms["floor"]))
    assert qwen3.noise_floor_gate(off, floor), (off, floor)
    want = logprobs(steps.reshape(24, -1).double().cpu(), got["tokens"].reshape(24).cpu(), 1)
    assert torch.equal(want[3].view(2, 12), got["tokens"].cpu())
    assert float((want[0].view(2, 12) - got["logprobs"].cpu().double()).abs().max()) < 1e-5
    assert float((want[1].view(2, 12) - got["entropy"].cpu().double()).abs().max()) < 1e-5


def test_generation_over_a_quantised_cache(gpu, model):
    """e4m3 keys and values: eager and captured steps give the same tokens and bits, and the cache reads back to the
    quantised rows (2^-4 of each value, half a step of e4m3, or of its row's smallest step)."""
    announce("generate e4m3")
    torch.manual_seed(5)
    ids = torch.randint(0, 4000, (3, 40), device=gpu)
    a, b = (gen.generate(model, ids, 8, kind="e4m3", graph=graph) for graph in (False, True))
    assert all(torch.equal(a[k], b[k]) for k in a)
    s8, s16 = gen.Session(model, 3, 48, "e4m3"), gen.Session(model, 3, 48, "bf16")
    for s in (s8, s16):
        s.prefill(ids)
    for layer in (0,):  # the same inputs in both only before the first attention
        for got, want in zip(s8.dense(layer), s16.dense(layer)):
            top = want.float().abs().amax(-1, keepdim=True)
            off = (got.float() - want.float()).abs()
            assert bool((off <= torch.maximum(2.0 ** -4 * want.float().abs(), 2.0 ** -10 * top)).all())


def test_session_refusals(gpu, model):
    with pytest.raises(ValueError, match="kind"):
        gen.Session(model, 1, 8, "int8")
    s = gen.Session(model, 1, 4)
    with pytest.raises(ValueError, match="max_length"):
        s.prefill(torch.zeros(1, 5, dtype=torch.long, device=gpu))
    s.prefill(torch.zeros(1, 4, dtype=torch.long, device=gpu))
    with pytest.raises(ValueError, match="max_length"):
        s.step(torch.zeros(1, dtype=torch.long, device=gpu))
    with pytest.raises(ValueError, match="new_tokens"):
        gen.generate(model, torch.zeros(1, 4, dtype=torch.long, device=gpu), 0)


def test_full_session_is_not_captured_and_windows_are_refused(gpu, model):
    """The warm-up of a capture writes the next token's rows, which a full session does not have."""
    announce("capture of a full session")
    s = gen.Session(model, 1, 4)
    s.prefill(torch.arange(4, device=gpu)[None])
    before = s.dense(0)
    with pytest.raises(ValueError, match="max_length"):
        s.capture()
    assert all(torch.equal(a, b) for a, b in zip(before, s.dense(0)))
    attention = s.attentions[0]
    kept = attention.sliding_window
    attention.sliding_window = 8
    try:
        with pytest.raises(ValueError, match="sliding window"):
            gen.Session(model, 1, 4)
    finally:
        attention.sliding_window = kept


@pytest.mark.parametrize("graph", [False, True])
def test_generation_goes_on_where_logits_are_nan(gpu, model, graph):
    """Token -1 is no row of the embedding: the model is never given it."""
    announce(f"generate with NaN logits graph={graph}")
    norm = model.model.norm.weight
    kept = norm.detach().clone()
    with torch.no_grad():
        norm.fill_(float("nan"))
    try:
        got = gen.generate(model, torch.arange(6, device=gpu).view(2, 3), 4, graph=graph)
    finally:
        with torch.no_grad():
            norm.copy_(kept)
    assert bool((got["tokens"] == -1).all())
    assert all(bool(torch.isnan(got[k]).all()) for k in ("logprobs", "entropy", "prompt_logprobs"))

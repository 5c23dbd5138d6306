"""Greedy generation with a HuggingFace Qwen3 model over the package's paged cache.

The model-level caller of the serving ops, beside the prefill caller
(``qwen3``): every ``Qwen3Attention`` keeps its projections and its output
projection.  At the prompt, ``norm_rope_to_cache`` prepares Q and K from the
projections' views and fills the layer's pages, and the prefill kernel attends;
at each later token ``norm_rope_to_cache`` and ``attention_decode`` take the
place of both.  ``token_logprobs`` picks the likeliest token from the last
position's logits, with its log probability and the distribution's entropy.
The reference has no counterpart (its model runner stops at the prefill,
src/e2_qwen3_rope_prefill.py:129-169).

    python -m kernelfuser_amd.generate --random-layers 4 --batch 4 --prompt 512 --new 64 --out r.json

Prompts of one call have one length (no padding); the pages of a sequence need
not lie together.  ``Session`` also serves programs that choose their tokens
themselves.  Its step reads and writes only tensors that it keeps, so that it can be captured
in a HIP graph (``Session.capture``).
"""
from __future__ import annotations

import argparse
import json
import time
import types
from pathlib import Path

import torch

from . import _lib
from .ops import attention_prefill
from .qwen3 import _finish, _projections, load_qwen3, random_qwen3
from .serving import attention_decode, cache_to_dense, make_cache, norm_rope_to_cache, token_logprobs

KINDS = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


class Session:
    """``batch`` sequences of up to ``max_length`` tokens: pages, lengths and one cache per layer."""

    def __init__(self, model, batch: int, max_length: int, kind: str = "bf16", page_size: int = 64):
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {sorted(KINDS)}, got {kind!r}")
        if batch < 1 or max_length < 1:
            raise ValueError("Expected batch and max_length >= 1")
        self.model, self.batch, self.max_length, self.page_size = model, batch, max_length, page_size
        self.attentions = [m for m in model.modules() if type(m).__name__ == "Qwen3Attention"]
        if not self.attentions:
            raise RuntimeError("no Qwen3Attention modules found")
        if any(getattr(m, "sliding_window", None) is not None for m in self.attentions):
            raise ValueError("layers with a sliding window are not supported (the prefill has none)")
        dev = next(model.parameters()).device
        first = self.attentions[0]
        d, hkv = first.head_dim, first.k_proj.weight.shape[0] // first.head_dim
        per = -(-max_length // page_size)
        self.caches = [make_cache(batch * per, hkv, page_size, d, KINDS[kind], dev) for _ in self.attentions]
        self.pages = torch.arange(batch * per, dtype=torch.int32, device=dev).view(batch, per)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.filled = 0  # the same on the host: every sequence of a session has the same length
        at = torch.arange(max_length, device=dev)[None]
        with torch.inference_mode():
            cos, sin = model.model.rotary_emb(torch.empty(1, dtype=torch.bfloat16, device=dev), at)
        self.cos, self.sin = cos[0].contiguous().clone(), sin[0].contiguous().clone()
        self.tokens = torch.zeros(batch, 1, dtype=torch.long, device=dev)
        self.graph = self.logits = None

    def _slots(self, positions):
        rows = torch.gather(self.pages.long(), 1, positions // self.page_size)
        return rows * self.page_size + positions % self.page_size

    def _forward(self, layer, positions, slots):
        """The patched attention of one layer: the prompt's (more than one token) or a step's."""
        cache = self.caches[layer]

        def forward(mod, hidden_states, position_embeddings=None, attention_mask=None, past_key_values=None, **kw):
            q, k, v = _projections(mod, hidden_states)
            eps = float(getattr(mod.q_norm, "variance_epsilon", 1e-6))
            prompt = q.shape[2] > 1
            kn = torch.empty(k.shape, dtype=k.dtype, device=k.device) if prompt else None
            qn = norm_rope_to_cache(q, k, v, mod.q_norm.weight, mod.k_norm.weight, self.cos, self.sin, positions, slots,
                                    *cache, norm_style="hf", eps=eps, kn=kn)
            if prompt:
                out = torch.empty_like(qn)
                attention_prefill(qn, kn, v.contiguous(), out, causal=True, fuse_q=False, scale=float(mod.scaling))
            else:
                out = attention_decode(qn, cache[0], cache[1], self.pages, self.lengths, cache[2], cache[3],
                                       scale=float(mod.scaling))
            return _finish(mod, out, hidden_states)

        return forward

    def _run(self, ids, positions):
        slots = self._slots(positions)
        saved = [(m, m.forward) for m in self.attentions]
        try:
            for i, m in enumerate(self.attentions):
                m.forward = types.MethodType(self._forward(i, positions, slots), m)
            return self.model(input_ids=ids, position_ids=positions, attention_mask=None, use_cache=False,
                              return_dict=True).logits
        finally:
            for m, old in saved:
                m.forward = old

    @torch.inference_mode()
    def prefill(self, ids):
        """Logits [B,S,V] of the prompts ``ids`` [B,S], which start the sequences anew."""
        if ids.shape[0] != self.batch or not 1 <= ids.shape[1] <= self.max_length:
            raise ValueError("Expected ids [batch, 1 .. max_length]")
        s = ids.shape[1]
        self.lengths.fill_(s)
        self.filled = s
        return self._run(ids, torch.arange(s, device=ids.device).expand(self.batch, s))

    def _step(self):
        self.lengths += 1
        return self._run(self.tokens, (self.lengths.long() - 1)[:, None])[:, -1]

    @torch.inference_mode()
    def step(self, tokens):
        """Logits [B,V] after one more token per sequence (``tokens`` [B])."""
        if self.filled >= self.max_length:
            raise ValueError("the session's max_length is reached")
        self.filled += 1
        self.tokens.copy_(tokens.view(-1, 1))
        if self.graph is None:
            return self._step()
        self.graph.replay()
        return self.logits

    @torch.inference_mode()
    def capture(self):
        """Records the step in a HIP graph; later steps replay it.  The returned logits are then
        one tensor, overwritten by the next step."""
        if self.filled >= self.max_length:
            raise ValueError("the session's max_length is reached")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warm up outside the capture; what this writes, the next step writes again
            kept = self.lengths.clone()
            self._step()
            self.lengths.copy_(kept)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            self.logits = self._step()
        self.graph = graph

    def dense(self, layer: int, max_length: int | None = None):
        """A layer's keys and values as contiguous BF16 [B,Hkv,L,D]."""
        c = self.caches[layer]
        return cache_to_dense(c[0], c[1], self.pages, self.lengths, max_length or max(self.filled, 1), c[2], c[3])


@torch.inference_mode()
def generate(model, ids, new_tokens: int, kind: str = "bf16", page_size: int = 64, graph: bool = False,
             session: Session | None = None):
    """Greedy continuation of the prompts ``ids`` [B,S]: a dict of ``tokens``,
    ``logprobs`` and ``entropy`` [B,new_tokens] and ``prompt_logprobs`` [B,S-1].
    Where the model's logits are no distribution (NaN) the token is -1, and the sequence goes on with token 0."""
    if new_tokens < 1:
        raise ValueError("new_tokens must be >= 1")
    s = session or Session(model, ids.shape[0], ids.shape[1] + new_tokens, kind, page_size)
    logits = s.prefill(ids)
    scored = token_logprobs(logits[:, :-1], ids[:, 1:])
    if graph and s.graph is None and new_tokens > 1:
        s.capture()
    last, got = logits[:, -1], []
    for i in range(new_tokens):
        best = token_logprobs(last, ids[:, -1], 1)
        got.append((best.top_ids[:, 0], best.top_logprobs[:, 0], best.entropy))
        if i + 1 < new_tokens:
            last = s.step(got[-1][0].clamp(min=0))
    tokens, logp, entropy = (torch.stack(t, dim=1) for t in zip(*got))
    return {"tokens": tokens, "logprobs": logp, "entropy": entropy, "prompt_logprobs": scored.logprobs}


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    src = ap.add_mutually_exclusive_group(required=True)
    src.add_argument("--model", help="local Qwen3 checkpoint directory")
    src.add_argument("--random-layers", type=int, help="random Qwen3-8B-shaped model with this many layers")
    ap.add_argument("--out", required=True)
    ap.add_argument("--batch", type=int, default=1)
    ap.add_argument("--prompt", type=int, default=128)
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--kind", choices=sorted(KINDS), default="bf16")
    ap.add_argument("--page-size", type=int, default=64)
    args = ap.parse_args(argv)
    model = load_qwen3(args.model) if args.model else random_qwen3(args.random_layers)
    dev = next(model.parameters()).device
    torch.manual_seed(1701)
    ids = torch.randint(0, int(model.config.vocab_size), (args.batch, args.prompt), device=dev)
    rec = {"schema": "kernelfuser-amd-generate-v1", "gpu": torch.cuda.get_device_name(0), "kind": args.kind,
           "model": args.model or f"random Qwen3-8B geometry, {args.random_layers} layers", "batch": args.batch,
           "prompt": args.prompt, "new": args.new, "runs": {}}
    for name, graph in (("eager", False), ("graph", True)):
        session = Session(model, args.batch, args.prompt + args.new, args.kind, args.page_size)
        with _lib.record_launches() as kern:
            first = generate(model, ids, args.new, graph=graph, session=session)
        torch.cuda.synchronize()
        t = time.perf_counter()
        again = generate(model, ids, args.new, graph=graph, session=session)
        torch.cuda.synchronize()
        s = time.perf_counter() - t
        rec["runs"][name] = {"seconds": s, "tokens_per_s": args.batch * args.new / s, "kernels": kern.kernels(),
                             "same_tokens": bool(torch.equal(first["tokens"], again["tokens"])),
                             "mean_logprob": float(again["logprobs"].mean())}
        print(f"{name}: {args.batch} x {args.new} tokens after {args.prompt}: {s * 1e3:.1f} ms", flush=True)
    out = Path(args.out)
    out.parent.mkdir(parents=True, exist_ok=True)
    out.write_text(json.dumps(rec, indent=1) + "\n")
    return rec


if __name__ == "__main__":
    main()

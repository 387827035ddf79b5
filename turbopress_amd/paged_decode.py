"""Greedy decoding of several sequences over a paged cache, with the decoder
operators between the packed projections.

The reference decodes one sequence over transformers' StaticCache and leaves
everything but the projections to the HF decoder
(``scripts/graph_decode_bench.py:39-118``).  ``PagedDecoder`` runs the layers of
a packed Llama, Mistral, Qwen2 or Qwen3 causal LM itself: norm and residual, projections
(``PackedTCQLinear``), norms of the heads, rotary positions and the cache's
writes, attention over each sequence's pages, and the head, in 8 bits on
request.  Its
decode step takes one token of every sequence, has no host synchronisation and
is captured in one HIP graph; sequences have lengths of their own and hold
pages only for what they have.

    python -m turbopress_amd.paged_decode --synthetic qwen3-0.6b --sequences 4
"""

from __future__ import annotations

import time

import torch
import torch.nn.functional as F
from torch import Tensor

from turbopress_amd.fp8 import fp8_linear, quantize_fp8_weight
from turbopress_amd.norm import rms_norm, rms_norm_fp8
from turbopress_amd.paged import paged_attention, rotary_append, rotary_table

__all__ = ["PagedCache", "PagedDecoder"]


class PagedCache:
    """Keys and values of `layers` decoder layers in pages, and who holds which.

    ``k[i]``, ``v[i]``: [n_pages, page_size, kv_heads, head_dim] of layer i;
    ``block_table``: int32 [sequences, width] on the device (-1: no page), which
    ``reserve`` and ``release`` rewrite in place."""

    def __init__(self, layers: int, sequences: int, max_len: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 n_pages: int | None = None, dtype: torch.dtype = torch.float16, device="cuda") -> None:
        if min(layers, sequences, max_len, kv_heads, head_dim, page_size) < 1:
            raise ValueError("layers, sequences, max_len, kv_heads, head_dim and page_size must be positive")
        self.page_size, self.max_len = page_size, max_len
        self.width = -(-max_len // page_size)
        n_pages = sequences * self.width if n_pages is None else n_pages
        shape = (layers, n_pages, page_size, kv_heads, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in "kv")
        self.block_table = torch.full((sequences, self.width), -1, dtype=torch.int32, device=device)
        self._free = list(range(n_pages - 1, -1, -1))
        self._held: list = [[] for _ in range(sequences)]

    def _check(self, sequence: int) -> None:
        if not 0 <= sequence < len(self._held):
            raise IndexError(f"sequence {sequence} outside [0, {len(self._held)})")

    def reserve(self, sequence: int, length: int) -> None:
        """Pages for `length` tokens of a sequence, beside those it holds."""
        self._check(sequence)
        if not 0 <= length <= self.max_len:
            raise ValueError(f"length {length} outside [0, {self.max_len}]")
        held = self._held[sequence]
        need = -(-length // self.page_size) - len(held)
        if need <= 0:
            return
        if need > len(self._free):
            raise RuntimeError(f"the cache is full: {need} pages needed, {len(self._free)} free")
        new = [self._free.pop() for _ in range(need)]
        at = len(held)
        held += new
        self.block_table[sequence, at:at + need] = torch.tensor(new, dtype=torch.int32).to(self.block_table.device)

    def room(self, sequence: int) -> int:
        """Tokens that the sequence's pages hold."""
        self._check(sequence)
        return min(len(self._held[sequence]) * self.page_size, self.max_len)

    def release(self, sequence: int) -> None:
        """The sequence's pages are free again."""
        self._check(sequence)
        self._free += reversed(self._held[sequence])
        self._held[sequence] = []
        self.block_table[sequence] = -1


def _rope(config) -> tuple:
    """(base, scaling, rotary share of the head) of an HF configuration."""
    params = getattr(config, "rope_parameters", None) or {}
    scaling = getattr(config, "rope_scaling", None) or (params if params.get("rope_type", "default") != "default" else None)
    if scaling is not None and scaling.get("rope_type", scaling.get("type")) in (None, "default"):
        scaling = None
    if scaling is not None and "original_max_position_embeddings" not in scaling:
        scaling = dict(scaling, original_max_position_embeddings=config.max_position_embeddings)
    base = getattr(config, "rope_theta", None) or params.get("rope_theta", 10000.0)
    share = getattr(config, "partial_rotary_factor", None) or params.get("partial_rotary_factor", 1.0)
    return float(base), scaling, float(share)


# Families whose layers are what PagedDecoder runs: projections, norms of the
# heads where there are any, halves of the heads turned, a gated MLP, two norms.
# Others with the same modules are not (layers without positions, multipliers of
# embeddings, residuals or logits, pairs in place of halves, norms elsewhere).
_FAMILIES = ("llama", "mistral", "qwen2", "qwen3")


def _windows(config, layers) -> list:
    """The sliding window of each layer's attention (0: none)."""
    if config.model_type == "mistral":  # (one for all layers, which do not name it)
        return [getattr(config, "sliding_window", None) or 0] * len(layers)
    return [getattr(layer.self_attn, "sliding_window", None) or 0 for layer in layers]


class PagedDecoder:
    """A causal LM (HF Llama, Mistral, Qwen2 or Qwen3 modules, projections packed
    or dense, fp16 or bf16; others are refused) decoding `sequences` sequences of
    up to `max_len` tokens at once.

    ``fp8_head``: the head's weights in e4m3 with a scale per 128 x 128 block,
    made of the dense ones here (half of their bytes, codes within 2^-4 of each);
    without, the model's own.  Logits are fp32 [rows, vocabulary] with it, the
    model's type without."""

    @torch.no_grad()
    def __init__(self, model, sequences: int, max_len: int, page_size: int = 64, n_pages: int | None = None,
                 fp8_head: bool = False) -> None:
        cfg = model.config
        if cfg.model_type not in _FAMILIES:
            raise ValueError(f"model_type {cfg.model_type!r}: PagedDecoder runs the layers of {', '.join(_FAMILIES)}")
        if cfg.hidden_act != "silu":
            raise ValueError(f"hidden_act {cfg.hidden_act!r}: PagedDecoder runs the gated MLP with silu")
        self.model, self.sequences = model, sequences
        body = model.model
        self.embed, self.layers, self.norm = body.embed_tokens, body.layers, body.norm
        attn = self.layers[0].self_attn
        self.windows = _windows(cfg, self.layers)
        self.head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
        self.heads, self.kv_heads = cfg.num_attention_heads, cfg.num_key_value_heads
        self.scale = getattr(attn, "scaling", self.head_dim ** -0.5)
        dev, dtype = self.embed.weight.device, self.embed.weight.dtype
        base, scaling, share = _rope(cfg)
        if share != 1:  # (these families turn whole heads, whatever it says)
            raise ValueError(f"partial_rotary_factor {share}: the heads of {cfg.model_type} turn as a whole")
        self.table = rotary_table(max_len, self.head_dim, base, scaling, device=dev)
        self.cache = PagedCache(len(self.layers), sequences, max_len, self.kv_heads, self.head_dim, page_size, n_pages,
                                dtype, dev)
        self.head = quantize_fp8_weight(model.lm_head.weight) if fp8_head else None
        # one decode step's state: the sequences' next tokens, their positions
        # (-1: no sequence) and lengths with that token
        self.tokens = torch.zeros(sequences, dtype=torch.int64, device=dev)
        self.positions = torch.full((sequences,), -1, dtype=torch.int64, device=dev)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=dev)
        self._next = [-1] * sequences  # the positions, on the host
        self._graph = None
        self._graph_logits = None

    def _norm(self, x: Tensor, norm, residual: Tensor | None = None):
        return rms_norm(x, norm.weight, norm.variance_epsilon, residual=residual)

    def _rows(self, tokens: Tensor, positions: Tensor, block_table: Tensor, sequences: Tensor | None, lengths: Tensor):
        """(output of the last layer, residual) of rows of any sequences: row r
        is token positions[r] of the sequence whose pages are block_table[r]."""
        rows = tokens.shape[0]
        h = self.embed(tokens)
        x = self._norm(h, self.layers[0].input_layernorm)
        for i, layer in enumerate(self.layers):
            at = layer.self_attn
            q = at.q_proj(x).view(rows, self.heads, self.head_dim)
            k = at.k_proj(x).view(rows, self.kv_heads, self.head_dim)
            v = at.v_proj(x).view(rows, self.kv_heads, self.head_dim)
            if getattr(at, "q_norm", None) is not None:
                q, k = self._norm(q, at.q_norm), self._norm(k, at.k_norm)
            kc, vc = self.cache.k[i], self.cache.v[i]
            q = rotary_append(q, k, v, self.table, positions, kc, vc, self.cache.block_table, sequences=sequences)
            o = paged_attention(q, kc, vc, block_table, lengths, scale=self.scale, window=self.windows[i])
            x, h = self._norm(at.o_proj(o.view(rows, -1)), layer.post_attention_layernorm, h)
            gate, up = layer.mlp.gate_proj(x), layer.mlp.up_proj(x)
            x = layer.mlp.down_proj(F.silu(gate) * up)
            if i + 1 < len(self.layers):
                x, h = self._norm(x, self.layers[i + 1].input_layernorm, h)
        return x, h

    def _logits(self, x: Tensor, h: Tensor) -> Tensor:
        if self.head is None:
            return F.linear(self._norm(x, self.norm, h)[0], self.model.lm_head.weight)
        codes, scales, _ = rms_norm_fp8(x, self.norm.weight, self.norm.variance_epsilon, residual=h)
        return fp8_linear(codes, scales, *self.head, out_dtype=torch.float32)

    @torch.inference_mode()
    def prefill(self, sequence: int, prompt: Tensor) -> Tensor:
        """Run a prompt (int64 [tokens]) into a fresh sequence; its next token is
        the greedy one.  Returns the last token's logits [1, vocabulary].

        A prompt's tokens are rows of one pass: each attends to the pages up to
        itself, which the same layer has written before.  (Every row reads its
        whole prefix: short prompts.)"""
        n = int(prompt.shape[0])
        if n < 1:
            raise ValueError("a prompt needs a token")
        self.stop(sequence)
        self.cache.reserve(sequence, n)
        dev = self.tokens.device
        pos = torch.arange(n, device=dev)
        seq = torch.full((n,), sequence, dtype=torch.int32, device=dev)
        pages = self.cache.block_table[sequence].expand(n, -1).contiguous()
        x, h = self._rows(prompt.to(dev), pos, pages, seq, (pos + 1).int())
        logits = self._logits(x[-1:], h[-1:])
        self.tokens[sequence] = logits[0].argmax()
        self.positions[sequence] = n
        self.lengths[sequence] = n + 1
        self._next[sequence] = n
        return logits

    def stop(self, sequence: int) -> None:
        """End a sequence: its pages are free, its row of the step idles."""
        self.cache.release(sequence)
        self._next[sequence] = -1
        self.positions[sequence] = -1
        self.lengths[sequence] = 0

    @torch.inference_mode()
    def _step(self) -> Tensor:
        x, h = self._rows(self.tokens, self.positions, self.cache.block_table, None, self.lengths)
        return self._logits(x, h)

    @torch.inference_mode()
    def _advance(self, logits: Tensor) -> None:
        self.tokens.copy_(logits.argmax(-1))
        live = self.positions >= 0
        self.positions += live
        self.lengths += live.int()
        self._next = [p + (p >= 0) for p in self._next]

    def step(self, graph: bool = True) -> Tensor:
        """One token of every live sequence: the logits [sequences, vocabulary]
        of ``tokens``, which become the greedy next ones.  Pages for the tokens
        have to be reserved (``cache.reserve``); where one is not, nothing is
        run and RuntimeError raised.  graph: the step is captured on first use
        and replayed (the logits are then a fixed buffer)."""
        for s, p in enumerate(self._next):
            if p >= self.cache.room(s):  # (its key and value would be dropped, and attention miss them)
                raise RuntimeError(f"no page for token {p} of sequence {s}: pages hold {self.cache.room(s)} tokens of it "
                                   f"(cache.reserve), at most {self.cache.max_len}")
        if graph and self._graph is None:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                self._step()  # (its cache writes are the ones that the step makes again)
            torch.cuda.current_stream().wait_stream(side)
            self._graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._graph):
                self._graph_logits = self._step()
        if graph:
            self._graph.replay()
            logits = self._graph_logits
        else:
            logits = self._step()
        self._advance(logits)
        return logits

    @torch.inference_mode()
    def _begin(self, prompts, n_new: int) -> tuple:
        """Prefill up to `sequences` prompts, with pages for n_new tokens of each:
        the state from which their decoding begins."""
        if len(prompts) > self.sequences:
            raise ValueError(f"{len(prompts)} prompts for {self.sequences} sequences")
        for s in range(self.sequences):
            self.stop(s)
        for s, p in enumerate(prompts):
            self.prefill(s, p)
            self.cache.reserve(s, int(p.shape[0]) + n_new - 1)  # (the last new token is not read back)
        return len(prompts), self.tokens.clone(), self.positions.clone(), self.lengths.clone(), list(self._next)

    @torch.inference_mode()
    def _decode(self, begin: tuple, n_new: int, graph: bool) -> tuple:
        """Greedy tokens from a state of ``_begin``, as often as wanted (what a
        run leaves in the cache the next one writes again before it reads it),
        and tokens/s."""
        count, tokens, positions, lengths, following = begin
        self.tokens.copy_(tokens)
        self.positions.copy_(positions)
        self.lengths.copy_(lengths)
        self._next = list(following)
        out = [self.tokens.clone()]
        start, timed = None, 0
        for i in range(1, n_new):
            if i == 2:  # (the first step may capture)
                torch.cuda.synchronize()
                start = time.perf_counter()
            self.step(graph)
            timed += i >= 2
            out.append(self.tokens.clone())
        torch.cuda.synchronize()
        rate = timed * count / (time.perf_counter() - start) if timed else float("inf")
        return torch.stack(out, 1)[:count].tolist(), rate

    def generate(self, prompts, n_new: int, graph: bool = True) -> tuple:
        """Greedy tokens (n_new per prompt) of up to `sequences` prompts, and the
        decode steps' tokens/s over all of them."""
        return self._decode(self._begin(prompts, n_new), n_new, graph)


def main(argv=None) -> int:
    """Greedy decoding of several sequences of a packed model over a paged
    cache, eager and with one captured step replayed; prints one JSON line."""
    import argparse
    import json
    import sys
    import tempfile

    from turbopress_amd.artifact import load_packed_model
    from turbopress_amd.decode_step import fuse_shared_input_projections
    from turbopress_amd.graph_decode import SYNTHETIC, synthetic_config
    from turbopress_amd.synthetic import write_synthetic_artifact

    ap = argparse.ArgumentParser(description=main.__doc__.splitlines()[0])
    src = ap.add_mutually_exclusive_group(required=True)
    src.add_argument("--artifact", help="format-v1 artifact directory")
    src.add_argument("--synthetic", choices=sorted(SYNTHETIC), help="seeded synthetic model of this shape")
    ap.add_argument("--bits", type=int, default=3)
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--prompt-len", type=int, default=40, help="of the longest; the others are shorter")
    ap.add_argument("--new-tokens", type=int, default=64)
    ap.add_argument("--page-size", type=int, default=64)
    head = ap.add_mutually_exclusive_group()
    head.add_argument("--fp8-head", action="store_true", help="the head's weights in 8 bits")
    head.add_argument("--dense-head", action="store_true", help="the head's dense weights (the default)")
    args = ap.parse_args(argv)

    def progress(msg: str) -> None:
        print(f"[paged_decode] {msg}", file=sys.stderr, flush=True)

    with tempfile.TemporaryDirectory() as tmp:
        root = args.artifact
        if args.synthetic:
            root = tmp
            write_synthetic_artifact(root, synthetic_config(args.synthetic), bits=args.bits, seed=0, log=progress)
        progress("loading the packed model")
        model, _ = load_packed_model(root, device="cuda", mode="hip")
    fuse_shared_input_projections(model)
    gen = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, model.config.vocab_size, (max(1, args.prompt_len - 7 * s),), generator=gen).cuda()
               for s in range(args.sequences)]
    decoder = PagedDecoder(model, args.sequences, args.prompt_len + args.new_tokens, args.page_size,
                           fp8_head=args.fp8_head)
    # (one prefill for both: the sums of a prompt of 17..32 tokens are not always
    # added in one order, and a near tie may fall either way)
    begin = decoder._begin(prompts, args.new_tokens)
    eager, eager_rate = decoder._decode(begin, args.new_tokens, graph=False)
    graph, graph_rate = decoder._decode(begin, args.new_tokens, graph=True)
    print(json.dumps({"model": args.synthetic or str(args.artifact), "sequences": args.sequences,
                      "prompt_lens": [int(p.shape[0]) for p in prompts], "new_tokens": args.new_tokens,
                      "head": "fp8" if args.fp8_head else "dense", "eager_tok_s": round(eager_rate, 1),
                      "graph_tok_s": round(graph_rate, 1), "greedy_tokens_match": eager == graph}), flush=True)
    return 0


if __name__ == "__main__":
    import sys
    sys.exit(main())

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

Beside that it checks drafted tokens of all sequences in one pass (``verify``, a
chain or a tree of each, accepted where they are the greedy ones), adds each
sequence's own low-rank adapter to the shared projections, cuts attention to a
window and the first tokens, and scores given texts (``score``).

    python -m turbopress_amd.paged_decode --synthetic qwen3-0.6b --sequences 4
    python -m turbopress_amd.paged_decode --synthetic qwen3-0.6b --draft 7
"""

from __future__ import annotations

import time
from collections.abc import Callable, Sequence

import torch
import torch.nn.functional as F
from torch import Tensor

from turbopress_amd.fp8 import fp8_linear, quantize_fp8_weight
from turbopress_amd.logprobs import TokenLogprobs, token_logprobs
from turbopress_amd.lora import LoraAdapters
from turbopress_amd.norm import rms_norm, rms_norm_fp8
from turbopress_amd.paged import TREE_TOKENS, paged_attention, paged_tree_attention, rotary_append, rotary_table

__all__ = ["PagedCache", "PagedDecoder", "lookup_draft"]


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

    def move(self, moves: Sequence) -> None:
        """Keys and values of cached tokens to other places of their sequence, in
        every layer: (sequence, from, to) each, all read before any is written."""
        if not moves:
            return
        for s, a, b in moves:
            if not (0 <= a < self.room(s) and 0 <= b < self.room(s)):
                raise ValueError(f"tokens {a} and {b} of sequence {s}: its pages hold {self.room(s)}")
        seq, a, b = torch.tensor(moves, dtype=torch.int64).to(self.block_table.device).unbind(1)
        at, to = (self.block_table[seq, t // self.page_size].long() for t in (a, b))
        for c in (self.k, self.v):
            c[:, to, b % self.page_size] = c[:, at, a % self.page_size]

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


def lookup_draft(history: Sequence, count: int, longest: int = 3, branches: int = 2) -> tuple:
    """Up to `count` tokens that may follow a history (a list of ints), as a tree
    ``(tokens, parents)`` (parent -1: it follows the history), found in the history
    itself: what came behind the latest `branches` occurrences of its last tokens,
    of as many of those (`longest` at most) as occur before.  None found: empty."""
    n = len(history)
    tokens, parents = [], []
    for size in range(min(longest, n - 1) if count > 0 else 0, 0, -1):
        last, starts = history[n - size:], []
        for at in range(n - size - 1, -1, -1):
            if history[at] == last[0] and history[at:at + size] == last:
                starts.append(at + size)
                if len(starts) == branches:
                    break
        for start in starts:
            node = -1
            for t in history[start:start + count]:
                known = [j for j, p in enumerate(parents) if p == node and tokens[j] == t]
                if known:
                    node = known[0]
                elif len(tokens) < count:
                    tokens.append(t)
                    parents.append(node)
                    node = len(tokens) - 1
                else:
                    break
        if starts:
            break
    return tokens, parents


def _projections(layer) -> list:
    """(name, module) of a layer's projections."""
    at, mlp = layer.self_attn, layer.mlp
    return [("self_attn.q_proj", at.q_proj), ("self_attn.k_proj", at.k_proj), ("self_attn.v_proj", at.v_proj),
            ("self_attn.o_proj", at.o_proj), ("mlp.gate_proj", mlp.gate_proj), ("mlp.up_proj", mlp.up_proj),
            ("mlp.down_proj", mlp.down_proj)]


class PagedDecoder:
    """A causal LM (HF Llama, Mistral, Qwen2 or Qwen3 modules, projections packed
    or dense, fp16 or bf16; others are refused) decoding `sequences` sequences of
    up to `max_len` tokens at once.

    ``fp8_head``: the head's weights in e4m3 with a scale per 128 x 128 block,
    made of the dense ones here (half of their bytes, codes within 2^-4 of each);
    without, the model's own.  Logits are fp32 [rows, vocabulary] with it, the
    model's type without.

    ``draft``: tokens that ``verify`` checks of each sequence at once, beside its
    next one (up to 63).  ``window``, ``sinks``: attention sees at most the last
    `window` tokens (0: as many as the model's own layers do) and, where a window
    cuts, the first `sinks` too; positions stay those in the text.  ``adapters``:
    low-rank adapters, of which each sequence has one or none (``prefill``)."""

    @torch.no_grad()
    def __init__(self, model, sequences: int, max_len: int, page_size: int = 64, n_pages: int | None = None,
                 fp8_head: bool = False, draft: int = 0, window: int = 0, sinks: int = 0,
                 adapters: LoraAdapters | None = None) -> None:
        cfg = model.config
        if not 0 <= draft < TREE_TOKENS:
            raise ValueError(f"draft must lie between 0 and {TREE_TOKENS - 1}, got {draft}")
        if window < 0 or sinks < 0:
            raise ValueError(f"window and sinks must be 0 (none) or positive, got {window} and {sinks}")
        if cfg.model_type not in _FAMILIES:
            raise ValueError(f"model_type {cfg.model_type!r}: PagedDecoder runs the layers of {', '.join(_FAMILIES)}")
        if cfg.hidden_act != "silu":
            raise ValueError(f"hidden_act {cfg.hidden_act!r}: PagedDecoder runs the gated MLP with silu")
        self.model, self.sequences = model, sequences
        body = model.model
        self.embed, self.layers, self.norm = body.embed_tokens, body.layers, body.norm
        attn = self.layers[0].self_attn
        self.windows = _windows(cfg, self.layers)
        if window:
            self.windows = [min(w or window, window) for w in self.windows]
        self.sinks = sinks
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
        self.adapters = adapters
        self.adapter_of = None  # each sequence's adapter (-1: none)
        if adapters is not None:
            shapes = {f"model.layers.{i}.{name}": (m.out_features, m.in_features)
                      for i, layer in enumerate(self.layers) for name, m in _projections(layer)}
            adapters.check(shapes, dtype, dev)
            self.adapter_of = torch.full((sequences,), -1, dtype=torch.int32, device=dev)
        # the drafted pass's state: of each new token the token, its position and
        # place in the cache (-1: none), those it sees; and the tokens before it
        self.draft = draft
        self._drafted = torch.zeros(5, sequences, 1 + draft, dtype=torch.int64, device=dev) if draft else None
        self._verify_graph = None
        self._verify_best = None

    def _norm(self, x: Tensor, norm, residual: Tensor | None = None):
        return rms_norm(x, norm.weight, norm.variance_epsilon, residual=residual)

    def _rows(self, tokens: Tensor, positions: Tensor, block_table: Tensor, sequences: Tensor | None, lengths: Tensor,
              adapters: Tensor | None = None, slots: Tensor | None = None, attend: Callable | None = None):
        """(output of the last layer, residual) of rows of any sequences: row r
        is token positions[r] of the sequence whose pages are block_table[r].
        adapters: each row's; slots: its place in the cache where that is not its
        position; attend(layer, q): attention in place of each row's own."""
        rows = tokens.shape[0]

        def project(i, name, module, x):
            y = module(x)
            return y if adapters is None else self.adapters.add(f"model.layers.{i}.{name}", y, x, adapters)

        h = self.embed(tokens)
        x = self._norm(h, self.layers[0].input_layernorm)
        for i, layer in enumerate(self.layers):
            at = layer.self_attn
            q = project(i, "self_attn.q_proj", at.q_proj, x).view(rows, self.heads, self.head_dim)
            k = project(i, "self_attn.k_proj", at.k_proj, x).view(rows, self.kv_heads, self.head_dim)
            v = project(i, "self_attn.v_proj", at.v_proj, x).view(rows, self.kv_heads, self.head_dim)
            if getattr(at, "q_norm", None) is not None:
                q, k = self._norm(q, at.q_norm), self._norm(k, at.k_norm)
            kc, vc = self.cache.k[i], self.cache.v[i]
            q = rotary_append(q, k, v, self.table, positions, kc, vc, self.cache.block_table, sequences=sequences, slots=slots)
            if attend is None:
                o = paged_attention(q, kc, vc, block_table, lengths, scale=self.scale, window=self.windows[i], sinks=self.sinks)
            else:
                o = attend(i, q)
            o = project(i, "self_attn.o_proj", at.o_proj, o.view(rows, -1))
            x, h = self._norm(o, layer.post_attention_layernorm, h)
            gate, up = project(i, "mlp.gate_proj", layer.mlp.gate_proj, x), project(i, "mlp.up_proj", layer.mlp.up_proj, x)
            x = project(i, "mlp.down_proj", layer.mlp.down_proj, F.silu(gate) * up)
            if i + 1 < len(self.layers):
                x, h = self._norm(x, self.layers[i + 1].input_layernorm, h)
        return x, h

    def _logits(self, x: Tensor, h: Tensor) -> Tensor:
        if self.head is None:
            return F.linear(self._norm(x, self.norm, h)[0], self.model.lm_head.weight)
        codes, scales, _ = rms_norm_fp8(x, self.norm.weight, self.norm.variance_epsilon, residual=h)
        return fp8_linear(codes, scales, *self.head, out_dtype=torch.float32)

    def _tree(self, i: int, q: Tensor, block_table: Tensor, lengths: Tensor, ancestors: Tensor | None, each: int) -> Tensor:
        """Attention of layer i of `each` new tokens of every sequence."""
        return paged_tree_attention(q.view(-1, each, self.heads, self.head_dim), self.cache.k[i], self.cache.v[i], block_table,
                                    lengths, ancestors, scale=self.scale, window=self.windows[i], sinks=self.sinks)

    def _prompt(self, sequence: int, prompt: Tensor, adapter: int, chunked: bool):
        """``_rows`` of a prompt in a fresh sequence."""
        n = int(prompt.shape[0])
        if n < 1:
            raise ValueError("a prompt needs a token")
        if not -1 <= adapter < (0 if self.adapters is None else self.adapters.count):
            raise ValueError(f"adapter {adapter}: there are {0 if self.adapters is None else self.adapters.count}")
        self.stop(sequence)
        self.cache.reserve(sequence, n)
        dev = self.tokens.device
        pos = torch.arange(n, device=dev)
        seq = torch.full((n,), sequence, dtype=torch.int32, device=dev)
        rows = None
        if self.adapters is not None:
            self.adapter_of[sequence] = adapter
            rows = torch.full((n,), adapter, dtype=torch.int32, device=dev)
        pages = self.cache.block_table[sequence].expand(-(-n // TREE_TOKENS) if chunked else n, -1).contiguous()
        attend = None
        if chunked:
            whole, rest = n // TREE_TOKENS, n % TREE_TOKENS
            before = torch.arange(0, n, TREE_TOKENS, dtype=torch.int32, device=dev)

            def attend(i, q):
                at = whole * TREE_TOKENS
                parts = []
                if whole:
                    parts.append(self._tree(i, q[:at], pages[:whole], before[:whole], None, TREE_TOKENS).flatten(0, 1))
                if rest:
                    parts.append(self._tree(i, q[at:], pages[whole:], before[whole:], None, rest).flatten(0, 1))
                return parts[0] if len(parts) == 1 else torch.cat(parts)

        return self._rows(prompt.to(dev), pos, pages, seq, (pos + 1).int(), rows, None, attend)

    @torch.inference_mode()
    def prefill(self, sequence: int, prompt: Tensor, adapter: int = -1, chunked: bool = False) -> Tensor:
        """Run a prompt (int64 [tokens]) into a fresh sequence; its next token is
        the greedy one.  Returns the last token's logits [1, vocabulary].
        adapter: the sequence's from here on (-1: none).

        A prompt's tokens are rows of one pass: each attends to the pages up to
        itself, which the same layer has written before.  Every row reads its
        whole prefix (short prompts), or, ``chunked``, 64 tokens at a time share
        what they read (sums in another order)."""
        n = int(prompt.shape[0])
        x, h = self._prompt(sequence, prompt, adapter, chunked)
        logits = self._logits(x[-1:], h[-1:])
        self.tokens[sequence] = logits[0].argmax()
        self.positions[sequence] = n
        self.lengths[sequence] = n + 1
        self._next[sequence] = n
        return logits

    @torch.inference_mode()
    def score(self, tokens: Tensor, top: int = 0, adapter: int = -1, sequence: int = 0) -> TokenLogprobs:
        """Log probabilities of a text's tokens (int64 [n], n >= 2), each behind
        those before it: ``token_logprobs`` of tokens[1:], n - 1 rows.  A sequence
        that stands idle lends its pages (RuntimeError where it does not)."""
        if int(tokens.shape[0]) < 2:
            raise ValueError("a text to score needs two tokens")
        if self._next[sequence] >= 0:
            raise RuntimeError(f"sequence {sequence} is decoding")
        try:
            x, h = self._prompt(sequence, tokens[:-1], adapter, True)
            return token_logprobs(self._logits(x, h), tokens[1:].to(self.tokens.device), top)
        finally:
            self.stop(sequence)

    def stop(self, sequence: int) -> None:
        """End a sequence: its pages are free, its row of the step idles."""
        self.cache.release(sequence)
        self._next[sequence] = -1
        self.positions[sequence] = -1
        self.lengths[sequence] = 0
        if self.adapters is not None:
            self.adapter_of[sequence] = -1

    @torch.inference_mode()
    def _step(self) -> Tensor:
        x, h = self._rows(self.tokens, self.positions, self.cache.block_table, None, self.lengths, self.adapter_of)
        return self._logits(x, h)

    @torch.inference_mode()
    def _advance(self, logits: Tensor) -> None:
        self.tokens.copy_(logits.argmax(-1))
        live = self.positions >= 0
        self.positions += live
        self.lengths += live.int()
        self._next = [p + (p >= 0) for p in self._next]

    @staticmethod
    @torch.inference_mode(False)  # (captures share their generator's state: made in the mode, others could not write it)
    def _capture(run: Callable) -> tuple:
        """(graph, its outputs) of a pass, which is run once before."""
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()  # (its cache writes are the ones that the pass makes again)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        return graph, out

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
            self._graph, self._graph_logits = self._capture(self._step)
        if graph:
            self._graph.replay()
            logits = self._graph_logits
        else:
            logits = self._step()
        self._advance(logits)
        return logits

    @torch.inference_mode()
    def _verify(self) -> tuple:
        """(most likely token, its log probability) behind each new token, [sequences,
        1 + draft]."""
        tokens, positions, slots, ancestors, before = self._drafted
        each = 1 + self.draft
        sequences = torch.arange(self.sequences, dtype=torch.int32, device=tokens.device)[:, None].expand(-1, each).reshape(-1)
        lengths = before[:, 0].int()
        adapters = None if self.adapters is None else self.adapter_of[:, None].expand(-1, each).reshape(-1)
        x, h = self._rows(tokens.view(-1), positions.view(-1), self.cache.block_table, sequences, lengths, adapters, slots.view(-1),
                          lambda i, q: self._tree(i, q, self.cache.block_table, lengths, ancestors, each))
        best = token_logprobs(self._logits(x, h), top=1)
        return best.top_tokens.view(-1, each), best.top_logprobs.view(-1, each)

    @torch.inference_mode()
    def verify(self, drafts: Sequence, graph: bool = True) -> list:
        """One pass over every live sequence's next token and tokens drafted behind
        it.  drafts: for each sequence ``(tokens, parents)``, up to ``draft`` of
        them, parents[j] < j the index of the one that token j follows (-1: the
        sequence's next token; ``lookup_draft``), or None.  Drafted tokens that are
        the greedy ones are accepted.  Returns for each sequence ``(tokens,
        logprobs)``: those accepted and the greedy one behind the last, which is
        then its next token; empty for one that is not live.

        Pages for all of them have to be reserved; where one is not, nothing is run
        and RuntimeError raised.  graph: as in ``step``.  (The host waits for the
        pass: what was accepted decides what is drafted next.)"""
        if not self.draft:
            raise RuntimeError("this decoder checks no drafts (PagedDecoder(draft=...))")
        if len(drafts) != self.sequences:
            raise ValueError(f"{len(drafts)} drafts for {self.sequences} sequences")
        each, nodes, following = 1 + self.draft, [], self.tokens.tolist()
        state: list = [[], [], [], [], []]  # as _drafted
        for s, (p, draft) in enumerate(zip(self._next, drafts)):
            tokens, above = ([], []) if draft is None or p < 0 else draft
            count = len(tokens)
            if count > self.draft or len(above) != count or any(not -1 <= a < j for j, a in enumerate(above)) \
                    or any(not 0 <= t < self.embed.num_embeddings for t in tokens):
                raise ValueError(f"drafts[{s}] must be up to {self.draft} tokens of the vocabulary and a parent below each, "
                                 f"got {tokens} and {above}")
            if p >= 0 and p + count >= self.cache.room(s):
                raise RuntimeError(f"no page for token {p + count} of sequence {s}: pages hold {self.cache.room(s)} tokens of it "
                                   f"(cache.reserve), at most {self.cache.max_len}")
            tokens, above = ([following[s], *tokens], [-1, *(a + 1 for a in above)]) if p >= 0 else ([], [])
            sees: list = []
            for j, a in enumerate(above):
                sees.append(1 << j | (sees[a] if a >= 0 else 0))
            pad = each - len(tokens)
            state[0].append(tokens + [0] * pad)
            state[1].append([p - 1 + bits.bit_count() for bits in sees] + [-1] * pad)
            state[2].append([p + j for j in range(len(tokens))] + [-1] * pad)
            state[3].append([bits - (bits >> 63 << 64) for bits in sees] + [0] * pad)
            state[4].append([max(p, 0)] * each)
            nodes.append((tokens, above))
        self._drafted.copy_(torch.tensor(state, dtype=torch.int64))
        if graph and self._verify_graph is None:
            self._verify_graph, self._verify_best = self._capture(self._verify)
        if graph:
            self._verify_graph.replay()
            best = self._verify_best
        else:
            best = self._verify()
        greedy, likely = best[0].tolist(), best[1].tolist()
        gained, moves = [], []
        for s, (tokens, above) in enumerate(nodes):
            if not tokens:
                gained.append(([], []))
                continue
            path = [0]
            for j in range(1, len(tokens)):
                if above[j] == path[-1] and tokens[j] == greedy[s][path[-1]]:
                    path.append(j)
            moves += [(s, self._next[s] + j, self._next[s] + d) for d, j in enumerate(path) if j != d]
            gained.append(([greedy[s][j] for j in path], [likely[s][j] for j in path]))
            self._next[s] += len(path)
        self.cache.move(moves)
        self.tokens.copy_(torch.tensor([g[0][-1] if g[0] else t for g, t in zip(gained, following)]))
        self.positions.copy_(torch.tensor(self._next))
        self.lengths.copy_(torch.tensor([p + 1 for p in self._next], dtype=torch.int32))
        return gained

    def generate_drafted(self, prompts, n_new: int, drafter: Callable = lookup_draft, graph: bool = True,
                         adapters: Sequence | None = None) -> tuple:
        """``generate`` with drafts checked: (greedy tokens, tokens/s, tokens gained
        per pass and sequence).  drafter(history, count): ``(tokens, parents)`` of
        up to `count` tokens behind a list of ints (``lookup_draft``; ValueError
        where it gives more).  Where it raises, the sequences stay as they are."""
        if not self.draft:
            raise RuntimeError("this decoder checks no drafts (PagedDecoder(draft=...))")
        return self._decode_drafted(self._begin(prompts, n_new, adapters), prompts, n_new, drafter, graph)

    def _decode_drafted(self, begin: tuple, prompts, n_new: int, drafter: Callable, graph: bool) -> tuple:
        count = self._resume(begin)
        texts = [p.tolist() + [t] for p, t in zip(prompts, self.tokens.tolist())]
        ends = [len(t) + n_new - 1 for t in texts]
        start, timed, first, passes, idle = None, 0, 0, 0, {}
        try:
            while any(len(t) < e for t, e in zip(texts, ends)):
                if passes == 1:  # (the first pass may capture)
                    torch.cuda.synchronize()
                    start, first = time.perf_counter(), timed
                drafts = []
                for s in range(self.sequences):
                    left = ends[s] - len(texts[s]) if s < count else 0
                    if s < count and not left and s not in idle:
                        idle[s], self._next[s] = self._next[s], -1  # (it has its tokens: its rows idle)
                    asked = min(self.draft, left - 1)
                    drafts.append(drafter(texts[s], asked) if left > 1 else None)
                    if drafts[-1] is not None and len(drafts[-1][0]) > asked:  # (more than n_new could come of it)
                        raise ValueError(f"the drafter gave {len(drafts[-1][0])} tokens, up to {asked} were asked for")
                passes += 1
                for s, (tokens, _) in enumerate(self.verify(drafts, graph)[:count]):
                    texts[s] += tokens
                    timed += len(tokens)
        finally:  # (also where a drafter, or verify of what it gave, raises)
            for s, p in idle.items():
                self._next[s] = self.positions[s] = p
                self.lengths[s] = p + 1
        rate = (timed - first) / (time.perf_counter() - start) if timed > first and start else float("inf")
        gain = timed / max(passes * count, 1)
        return [t[len(p):] for t, p in zip(texts, prompts)], rate, gain

    @torch.inference_mode()
    def _begin(self, prompts, n_new: int, adapters: Sequence | None = None) -> tuple:
        """Prefill up to `sequences` prompts, with pages for n_new tokens of each:
        the state from which their decoding begins."""
        if len(prompts) > self.sequences:
            raise ValueError(f"{len(prompts)} prompts for {self.sequences} sequences")
        if adapters is not None and len(adapters) != len(prompts):
            raise ValueError(f"{len(adapters)} adapters for {len(prompts)} prompts")
        for s in range(self.sequences):
            self.stop(s)
        for s, p in enumerate(prompts):
            self.prefill(s, p, -1 if adapters is None else adapters[s])
            self.cache.reserve(s, int(p.shape[0]) + n_new - 1)  # (the last new token is not read back)
        return len(prompts), self.tokens.clone(), self.positions.clone(), self.lengths.clone(), list(self._next)

    @torch.inference_mode()
    def _resume(self, begin: tuple) -> int:
        """Back to a state of ``_begin``; how many prompts it holds."""
        count, tokens, positions, lengths, following = begin
        self.tokens.copy_(tokens)
        self.positions.copy_(positions)
        self.lengths.copy_(lengths)
        self._next = list(following)
        return count

    @torch.inference_mode()
    def _decode(self, begin: tuple, n_new: int, graph: bool) -> tuple:
        """Greedy tokens from a state of ``_begin``, as often as wanted (what a
        run leaves in the cache the next one writes again before it reads it),
        and tokens/s."""
        count = self._resume(begin)
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

    def generate(self, prompts, n_new: int, graph: bool = True, adapters: Sequence | None = None) -> tuple:
        """Greedy tokens (n_new per prompt) of up to `sequences` prompts, and the
        decode steps' tokens/s over all of them.  adapters: each prompt's (-1: none)."""
        return self._decode(self._begin(prompts, n_new, adapters), n_new, graph)


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
    ap.add_argument("--draft", type=int, default=0, help="tokens drafted of each sequence, found in its own text, checked in one pass")
    ap.add_argument("--window", type=int, default=0, help="attention sees at most the last so many tokens")
    ap.add_argument("--sinks", type=int, default=0, help="first tokens that stay visible beside a window")
    ap.add_argument("--adapter", action="append", default=[], metavar="DIR",
                    help="directory of a low-rank adapter (repeatable; sequence s takes the s-th, over and over)")
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
                           fp8_head=args.fp8_head, draft=args.draft, window=args.window, sinks=args.sinks,
                           adapters=LoraAdapters.load(args.adapter, model.model.embed_tokens.weight.dtype) if args.adapter else None)
    each = [s % len(args.adapter) for s in range(args.sequences)] if args.adapter else None
    # (one prefill for both: the sums of a prompt of 17..32 tokens are not always
    # added in one order, and a near tie may fall either way)
    begin = decoder._begin(prompts, args.new_tokens, each)
    eager, eager_rate = decoder._decode(begin, args.new_tokens, graph=False)
    graph, graph_rate = decoder._decode(begin, args.new_tokens, graph=True)
    more = {}
    if args.draft:
        # (tokens of several rows are sums in another order than a row's alone: a near tie may fall either way)
        drafted, rate, gain = decoder._decode_drafted(begin, prompts, args.new_tokens, lookup_draft, True)
        more = {"draft": args.draft, "drafted_tok_s": round(rate, 1), "tokens_per_pass": round(gain, 2),
                "drafted_tokens_match": drafted == graph}
    print(json.dumps({"model": args.synthetic or str(args.artifact), "sequences": args.sequences,
                      "prompt_lens": [int(p.shape[0]) for p in prompts], "new_tokens": args.new_tokens,
                      "head": "fp8" if args.fp8_head else "dense", "eager_tok_s": round(eager_rate, 1),
                      "graph_tok_s": round(graph_rate, 1), "greedy_tokens_match": eager == graph, **more}), flush=True)
    return 0


if __name__ == "__main__":
    import sys
    sys.exit(main())

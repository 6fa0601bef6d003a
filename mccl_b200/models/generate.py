"""Answering with a decoder, token by token: keys and values stay in a paged cache, a step reads the weights and the cache once.

    generator = Generator(model, max_sequences=8, weights="w4")
    texts = generator.generate([[1, 2, 3], [4, 5]], max_new_tokens=20)

On a CUDA device a prompt goes through the operators that score whole texts, which also fill the cache, or several prompts of different lengths at once through
those of packed texts (``ops.rotary``, ``ops.packed_attention``); a step is ``ops.paged_append`` (with the
rotation of the models that have one), ``ops.paged_attention`` and, with 4-bit weights, ``ops.linear_w4``, captured as a CUDA graph per number of
sequences.  On a CPU the same math runs on the operators' plain forms.
"""
from __future__ import annotations

import contextlib
import gc
from typing import Dict, List, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F

from .. import ops
from .cache import PagedKVCache
from .decoder import _GLOBAL_FORWARD_HOOKS, Block, Decoder, Linear, Norm, _rope_tables, _stock


class Generator:
    """A snapshot of a decoder's weights with a cache for `max_sequences` sequences.  A decoder whose modules compute something else than this package's
    (derived ones with a forward of their own, forward hooks) is refused.

    weights: "bf16", or "w4" for the layers' matrices in 4 bits (`group` columns per scale; the vocabulary projection stays bf16).
    pages: of `page_size` positions; by default enough for every sequence to be `max_positions` long (by default the model's).
    window / sinks: a token sees the last `window` positions and the first `sinks` only, and pages that nobody will see are given back.
    use_graph: capture a step as a CUDA graph, once for every number of sequences that is asked for."""

    def __init__(self, model: Decoder, *, max_sequences: int = 8, max_positions: Optional[int] = None, pages: Optional[int] = None, page_size: int = 64, weights: str = "bf16",
                 group: int = 128, window: Optional[int] = None, sinks: int = 0, use_graph: bool = True):
        if weights not in ("bf16", "w4"):
            raise RuntimeError(f"Generator: weights are 'bf16' or 'w4', not '{weights}'")
        if window is not None and window < 1 or sinks < 0 or (sinks and window is None):
            raise RuntimeError(f"Generator: no window of {window} with {sinks} first positions")
        if (not isinstance(model, Decoder) or type(model).__call__ is not torch.nn.Module.__call__
                or any(getattr(type(model), name) is not getattr(Decoder, name) or name in model.__dict__ for name in ("forward", "hidden", "head_weight"))):
            raise RuntimeError("Generator: a Decoder whose forward is its own")
        for blk in model.blocks:
            if not isinstance(blk, Block) or blk.cfg != model.cfg or any(not isinstance(m, (Linear, Norm)) for m in blk.children()):
                raise RuntimeError("Generator: the decoder's layers were replaced or wrapped")
        called = [model.tok, model.ln_f, *(m for blk in model.blocks for m in (blk, *blk.children()))]
        if not isinstance(model.tok, torch.nn.Embedding) or not isinstance(model.ln_f, Norm) or not all(
                _stock(m) and "forward" not in m.__dict__ and "with_residual" not in m.__dict__ for m in called):
            raise RuntimeError("Generator: modules of the decoder have a forward of their own")
        if any(_GLOBAL_FORWARD_HOOKS) or any(m._forward_hooks or m._forward_pre_hooks for m in (model, *called)):
            raise RuntimeError("Generator: forward hooks, which a step would not call")
        cfg = self.cfg = model.cfg
        self.max_positions = max_positions or cfg.max_seq
        if cfg.pos == "learned" and self.max_positions > cfg.max_seq:
            raise RuntimeError(f"Generator: the model has {cfg.max_seq} positions, {self.max_positions} were asked for")
        self.window, self.sinks = window, sinks
        self.device = model.tok.weight.device
        per_sequence = -(-self.max_positions // page_size)
        self.cache = PagedKVCache(cfg.n_layers, cfg.n_heads, cfg.head_dim, pages=pages or max_sequences * per_sequence, max_sequences=max_sequences,
                                  max_positions=self.max_positions, page_size=page_size, device=self.device)
        self.use_graph = use_graph and self.device.type == "cuda"
        self._graphs: Dict[int, tuple] = {}
        with torch.no_grad():
            def matrix(m: Linear, quantize: bool):
                w = m.weight.detach()
                return (ops.quantize_w4(w, group) if quantize else w.to(torch.bfloat16).clone()), None if m.bias is None else m.bias.detach().clone()

            def norm(m: Norm):
                return m.weight.detach().clone(), None if m.bias is None else m.bias.detach().clone(), m.eps

            w4 = weights == "w4"
            self._layers = [{"ln1": norm(b.ln1), "qkv": matrix(b.qkv, w4), "proj": matrix(b.proj, w4), "ln2": norm(b.ln2),
                             "up": matrix(b.gate_up if cfg.act == "swiglu" else b.up, w4), "down": matrix(b.down, w4)} for b in model.blocks]
            self._ln_f = norm(model.ln_f)
            self._tok = model.tok.weight.detach().clone()
            self._pos = None if model.pos is None else model.pos.weight.detach().clone()
            self._head = model.head_weight().detach().to(torch.bfloat16).clone()
            self._rope = tuple(t.clone() for t in _rope_tables(self.max_positions, cfg.head_dim, self.device)) if cfg.pos == "rope" else None

    # ---------------------------------------------------------------------------------------------------------- layers ----
    @staticmethod
    def _linear(x, matrix, act="none", residual=None):
        w, b = matrix
        f = ops.linear_w4 if isinstance(w, ops.W4Weight) else ops.linear
        return f(x, w, b, act=act, residual=residual)

    def _mlp(self, x, layer):
        h = ops.norm(x, *layer["ln2"])
        if self.cfg.act == "swiglu":
            h = ops.swiglu(self._linear(h, layer["up"]))
        else:
            h = self._linear(h, layer["up"], act="gelu")
        return self._linear(h, layer["down"], residual=x)

    def _append(self, i, qkv, table, positions, rows, rotate_q):
        """qkv [tokens, 3, heads, head_dim] of layer i into the cache; the queries, rotated where the model rotates them and `rotate_q`."""
        q = ops.paged_append(qkv[:, 1], qkv[:, 2], self.cache.keys(i), self.cache.values(i), table, positions, rows=rows,
                             q=qkv[:, 0] if rotate_q and self._rope is not None else None, rope=self._rope)
        return qkv[:, 0] if q is None else q

    def _logits(self, x):
        return ops.linear(ops.norm(x, *self._ln_f), self._head)

    def _ids(self, tokens):
        """Tokens on the model's device.  Those on the host are looked at first; one on the device that is outside the vocabulary counts as token 0."""
        ids = torch.as_tensor(tokens, dtype=torch.int64)
        vocab = self._tok.shape[0]
        if not ids.is_cuda and ids.numel() and not (0 <= int(ids.min()) and int(ids.max()) < vocab):
            raise RuntimeError(f"Generator: tokens outside the vocabulary of {vocab}")
        return ids.to(self.device)

    def _here(self):
        """The model's device as the current one: kernels, captures and replays go to its streams, whichever device the caller is on."""
        return torch.cuda.device(self.device) if self.device.type == "cuda" else contextlib.nullcontext()

    # --------------------------------------------------------------------------------------------------------- prompts ----
    @torch.no_grad()
    def prefill(self, tokens: Sequence[int]):
        """A new sequence that begins with these tokens: (its row, the logits ``[vocab]`` behind the last one)."""
        with self._here():
            return self._prefill(tokens)

    def _prefill(self, tokens):
        ids = self._ids(tokens).reshape(-1)
        count = ids.numel()
        if count < 1 or count > self.max_positions:
            raise RuntimeError(f"Generator: a prompt of {count} tokens, 1 to {self.max_positions} are possible")
        row = self.cache.add()
        try:
            # positions behind the first window do not see all the text before them: token by token
            at_once = count if self.window is None else min(count, self.window)
            self.cache.reserve([row], [at_once])
            logits = self._whole(ids[:at_once], row)
            self.cache.set_length(row, at_once)
            for i in range(at_once, count):
                logits = self.step([row], ids[i:i + 1])[0]
        except BaseException:
            self.cache.free(row)
            raise
        return row, logits

    def _whole(self, ids, row):
        cfg, count = self.cfg, ids.numel()
        positions = torch.arange(count, dtype=torch.int32, device=self.device)
        rows = torch.full_like(positions, row)
        x = ops.embedding(ids[None], self._tok, self._pos)
        for i, layer in enumerate(self._layers):
            qkv = self._linear(ops.norm(x, *layer["ln1"]), layer["qkv"])
            self._append(i, qkv.view(count, 3, cfg.n_heads, cfg.head_dim), self.cache.table, positions, rows, False)
            a = ops.causal_attention(qkv, cfg.n_heads) if self._rope is None else ops.rope_attention(qkv, cfg.n_heads, *self._rope)
            x = self._mlp(self._linear(a, layer["proj"], residual=x), layer)
        return self._logits(x[0, -1:])[0]

    @torch.no_grad()
    def prefill_together(self, prompts: Sequence[Sequence[int]]) -> Tuple[List[int], torch.Tensor]:
        """New sequences that begin with these prompts, all of them in one pass: (their rows, the logits ``[len(prompts), vocab]`` behind each one's last token).

        With a window too: a prompt longer than it needs pages for all its positions until the pass is over (``prefill`` goes on token by token instead)."""
        with self._here():
            return self._prefill_together(prompts)

    def _prefill_together(self, prompts):
        ids = [self._ids(tokens).reshape(-1) for tokens in prompts]
        counts = [t.numel() for t in ids]
        for count in counts:
            if count < 1 or count > self.max_positions:
                raise RuntimeError(f"Generator: a prompt of {count} tokens, 1 to {self.max_positions} are possible")
        if not counts:
            return [], torch.empty(0, self._head.shape[0], dtype=torch.bfloat16, device=self.device)
        rows: List[int] = []
        try:
            for _ in counts:
                rows.append(self.cache.add())
            self.cache.reserve(rows, counts)
            logits = self._packed(torch.cat(ids), rows, counts)
            for row, count in zip(rows, counts):
                self.cache.set_length(row, count)
            if self.window is not None:
                self.cache.drop_unseen(rows, self.window, self.sinks)
        except BaseException:
            for row in rows:
                self.cache.free(row)
            raise
        return rows, logits

    def _packed(self, ids, rows, counts):
        cfg, cache, total = self.cfg, self.cache, ids.numel()
        positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in counts]).to(self.device)
        owners = torch.repeat_interleave(torch.tensor(rows, dtype=torch.int32), torch.tensor(counts)).to(self.device)
        offsets = torch.cumsum(torch.tensor([0] + counts), 0).to(torch.int32).to(self.device)
        x = ops.embedding(ids, self._tok, None if self._pos is None else F.embedding(positions.long(), self._pos))
        for i, layer in enumerate(self._layers):
            q, k, v = self._linear(ops.norm(x, *layer["ln1"]), layer["qkv"]).view(total, 3, cfg.n_heads, cfg.head_dim).unbind(1)
            if self._rope is not None:
                q, k = ops.rotary(q, k, rope=self._rope, positions=positions)
            ops.paged_append(k, v, cache.keys(i), cache.values(i), cache.table, positions, rows=owners)
            a = ops.packed_attention(q, k, v, offsets, window=self.window, sinks=self.sinks).view(total, cfg.d_model)
            x = self._mlp(self._linear(a, layer["proj"], residual=x), layer)
        return self._logits(x.index_select(0, offsets[1:].long() - 1))

    # ----------------------------------------------------------------------------------------------------------- steps ----
    @torch.no_grad()
    def step(self, rows: Sequence[int], tokens) -> torch.Tensor:
        """One more token for each of these sequences (different ones); returns the logits ``[len(rows), vocab]`` behind it."""
        with self._here():
            return self._step(list(rows), tokens)

    def _step(self, rows, tokens):
        if len(set(rows)) != len(rows):
            raise RuntimeError("Generator: a sequence twice in one step")
        ids = self._ids(tokens)
        if ids.shape != (len(rows),):
            raise RuntimeError(f"Generator: {tuple(ids.shape)} tokens for {len(rows)} sequences")
        if not rows:
            return torch.empty(0, self._head.shape[0], dtype=torch.bfloat16, device=self.device)
        cache = self.cache
        cache.reserve(rows, [cache.length(r) + 1 for r in rows])
        at = torch.tensor(rows, dtype=torch.int64).to(self.device)
        if not self.use_graph:
            logits = self._one(at, ids)
        else:
            entry = self._graphs.get(len(rows))
            if entry is None:
                entry = self._graphs[len(rows)] = self._capture(at, ids)
            graph, static_rows, static_ids, out = entry
            static_rows.copy_(at)
            static_ids.copy_(ids)
            graph.replay()
            logits = out.clone()
        cache.advance(rows, 1)
        if self.window is not None:
            cache.drop_unseen(rows, self.window, self.sinks)
        return logits

    def _capture(self, rows, ids):
        static_rows, static_ids = rows.clone(), ids.clone()
        before = self.cache.lengths.clone()
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            self._one(static_rows, static_ids)   # what is made on first use is made outside the graph
            self.cache.lengths.copy_(before)     # the replay writes the same places again
        torch.cuda.current_stream(self.device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        collecting = gc.isenabled()
        gc.disable()   # a graph that the collector destroys meanwhile, another generator's, would invalidate the capture
        try:
            with torch.cuda.graph(graph, stream=side):   # its own default is a stream of the device that captured first
                out = self._one(static_rows, static_ids)
        finally:
            if collecting:
                gc.enable()
        return graph, static_rows, static_ids, out

    def _one(self, rows, ids):
        """A step of the sequences in `rows` (int64, on the device), whose lengths it advances."""
        cfg, cache, count = self.cfg, self.cache, ids.numel()
        positions = cache.lengths.index_select(0, rows)
        lengths = positions + 1
        table = cache.table.index_select(0, rows)
        x = ops.embedding(ids, self._tok, None if self._pos is None else F.embedding(positions.long(), self._pos))
        for i, layer in enumerate(self._layers):
            qkv = self._linear(ops.norm(x, *layer["ln1"]), layer["qkv"]).view(count, 3, cfg.n_heads, cfg.head_dim)
            q = self._append(i, qkv, table, positions, None, True)
            a = ops.paged_attention(q, cache.keys(i), cache.values(i), table, lengths, window=self.window, sinks=self.sinks).view(count, cfg.d_model)
            x = self._mlp(self._linear(a, layer["proj"], residual=x), layer)
        cache.lengths.index_copy_(0, rows, lengths)
        return self._logits(x)

    # ------------------------------------------------------------------------------------------------------- sequences ----
    def fork(self, row: int, count: int = 1) -> List[int]:
        """New sequences that begin as this one (full pages are shared)."""
        return self.cache.fork(row, count)

    def free(self, row: int) -> None:
        self.cache.free(row)

    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int, temperature: float = 0.0, generator: Optional[torch.Generator] = None,
                 stop: Optional[int] = None, *, top_k: Optional[int] = None, top_p: Optional[float] = None, min_p: Optional[float] = None,
                 together: bool = False) -> List[List[int]]:
        """New tokens for each prompt: the likeliest ones (the lowest number among equals), or drawn at a temperature, with any of top_k, top_p and min_p by
        ``ops.sample``.  A sequence ends with the token `stop`, after `max_new_tokens`, or at the last position; its pages are free afterwards.
        together: all prompts go through the model in one pass (``prefill_together``)."""
        settings = {"top_k": top_k, "top_p": top_p, "min_p": min_p}
        out: List[List[int]] = [[] for _ in prompts]
        active: Dict[int, int] = {}   # row -> prompt
        logits = {}
        try:
            if together:
                rows, first = self.prefill_together(prompts)
                active = {row: i for i, row in enumerate(rows)}
                logits = dict(zip(rows, first))
            else:
                for i, prompt in enumerate(prompts):
                    row, last = self.prefill(prompt)
                    active[row], logits[row] = i, last
            while active and max_new_tokens > 0:
                rows = list(active)
                last = torch.stack([logits[r] for r in rows]).float()
                if temperature > 0 and any(v is not None for v in settings.values()):
                    uniform = torch.rand(len(rows), generator=generator, device=self.device if generator is None else generator.device).to(self.device)
                    with self._here():
                        tokens = ops.sample(last, uniform, temperature=temperature, **settings)
                    if bool((tokens < 0).any()):
                        raise RuntimeError("Generator: the logits are not finite, there is nothing to draw from")
                elif temperature > 0:
                    # (a temperature so low that logits / temperature overflows is that of the likeliest token)
                    chances = torch.softmax(last / max(temperature, 1e-30), dim=-1)
                    if not bool(torch.isfinite(chances).all()):
                        raise RuntimeError("Generator: the logits are not finite, there is nothing to draw from")
                    tokens = torch.multinomial(chances, 1, generator=generator)[:, 0]
                else:
                    tokens = last.argmax(-1)
                for row, token in zip(rows, tokens.tolist()):
                    done = out[active[row]]
                    done.append(token)
                    if token == stop or len(done) >= max_new_tokens or self.cache.length(row) >= self.max_positions:
                        del active[row]
                        self.free(row)
                left = [k for k, r in enumerate(rows) if r in active]
                rows = [rows[k] for k in left]
                if rows:
                    next_logits = self.step(rows, tokens[torch.tensor(left, device=tokens.device)])
                    logits = dict(zip(rows, next_logits))
        except BaseException:
            for row in active:
                self.free(row)
            raise
        for row in list(active):
            self.free(row)
        return out

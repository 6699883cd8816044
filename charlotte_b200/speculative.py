"""Speculative decoding of several sequences over a cache of f16 or 8-bit rows.

A step runs, for each sequence, a tree of drafted tokens through the model at
once (cache_write and tree_attention a layer, the products as in a batched
step), draws what the target keeps of it (select, then verify), and moves the
kept rows of every layer's cache together (cache_keep). Row 0 of a tree is the
sequence's last token, so a tree of one row is a plain decode step, and every
step yields one token at least.

    python -m charlotte_b200.speculative      # a small model, drafts by lookup
"""
from __future__ import annotations

import math

import numpy as np

from . import CACHE_Q8, ERROR_STEP, GATED, QKV, CharlotteError, check, lib, matmul, plan, rope_turns, run
from . import model as M
from . import synth

MOST_NODES = 64
DRAW = dict(temperature=0.0, top_k=64, top_p=1.0, min_p=0.0)   # a draw's settings where none are given


class SpeculativeDecoder:
    """`sequences` sequences of `model`, steps of up to `nodes` rows each."""

    def __init__(self, model: M.Model, sequences: int = 1, nodes: int = 16, cache: int = CACHE_Q8):
        import torch
        if not 1 <= nodes <= MOST_NODES:
            raise ValueError(f"{nodes} rows a step (1 to {MOST_NODES})")
        self.torch, self.model, self.sequences, self.nodes = torch, model, sequences, nodes
        a = self.arch = model.arch
        rows = sequences * nodes

        def f32(x):
            return None if x is None else torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()

        def weight(w):
            piece = torch.from_numpy(synth.to_piece(w.format, w.stored)).cuda()
            return w.format, w.cols, (piece, w.blocks, 0, w.rows, 0)

        def buffer(width, dtype=torch.float32):
            return torch.zeros(rows, width, dtype=dtype, device="cuda")

        self.embed = weight(model.token_embd)
        self.head = weight(model.output) if model.output is not None else self.embed
        self.output_norm, self.factors = f32(model.output_norm), f32(model.factors)
        qd, kvd = a.query_heads * a.head_dim, a.kv_heads * a.head_dim
        self.hidden, self.normed, self.out = buffer(a.hidden), buffer(a.hidden), buffer(a.hidden)
        self.q, self.k, self.v, self.att, self.act = buffer(qd), buffer(kvd), buffer(kvd), buffer(qd), buffer(a.ffn)
        self.logits = buffer(a.vocab)
        ints = dict(dtype=torch.int32, device="cuda")
        self.ids, self.live, self.lengths = torch.zeros(rows, **ints), torch.zeros(sequences, **ints), torch.zeros(sequences, **ints)
        self.masks = torch.zeros(sequences, nodes, dtype=torch.int64, device="cuda")
        self.uniforms = torch.zeros(sequences, nodes, device="cuda")
        self.candidates = torch.zeros(rows, 64, 2, **ints)
        tiles, tickets = lib().cb_select_tiles(a.vocab), lib().cb_select_tickets(a.vocab)
        self.partials, self.tickets = torch.zeros(rows * tiles * 128, **ints), torch.zeros(rows * tickets, **ints)
        self.path, self.kept = torch.zeros(sequences, nodes, **ints), torch.zeros(sequences, **ints)
        self.sampled, self.new_lengths = torch.zeros(sequences, 4, **ints), torch.zeros(sequences, **ints)

        # Layers with the same window share one allocation, so that one call keeps a step's rows of all of them.
        windows = sorted({L.window for L in model.layers})
        self.caches, at = {}, {w: 0 for w in windows}
        for w in windows:
            count = sum(L.window == w for L in model.layers)
            slots = min(w, a.context) + nodes
            shape = (count, sequences, slots, a.kv_heads, a.head_dim)
            fields = dict(format=cache, slots=slots, kv_heads=a.kv_heads, head_dim=a.head_dim)
            data = {n: torch.zeros(shape, dtype=torch.uint8 if cache == CACHE_Q8 else torch.float16, device="cuda")
                    for n in ("key", "value")}
            if cache == CACHE_Q8:
                data |= {n + "_scale": torch.zeros(count, sequences, a.kv_heads, slots, device="cuda") for n in ("key", "value")}
            self.caches[w] = (fields, data, count)

        self.layers = []
        workspace = None
        step = dict(sequences=sequences, tokens=nodes, query_heads=a.query_heads, lengths=self.lengths, nodes=self.live,
                    ancestors=self.masks)
        for L in model.layers:
            fields, data, _ = self.caches[L.window]
            here = fields | {n: x[at[L.window]] for n, x in data.items()}
            at[L.window] += 1
            turns = f32(rope_turns(L.rope_base, a.head_dim))
            write = plan("cache_write", cache=here, query=self.q, query_out=self.q, key=self.k, value=self.v,
                         query_gain=f32(L.q_norm), key_gain=f32(L.k_norm), factors=self.factors, turns=turns,
                         halves=int(a.halves), epsilon=a.epsilon, **step)
            attend = plan("tree_attention", cache=here, query=self.q, out=self.att,
                          window=L.window if L.window < a.context else 0, max_keys=a.context + nodes,
                          scale_log2e=M.attention_scale(a) * math.log2(math.e), **step)
            if workspace is None or attend.workspace.numel() > workspace.numel():
                workspace = attend.workspace
            self.layers.append(dict(
                attn_norm=f32(L.attn_norm), ffn_norm=f32(L.ffn_norm), post_attn_norm=f32(L.post_attn_norm),
                post_ffn_norm=f32(L.post_ffn_norm), qkv=[weight(w) for w in (L.q, L.k, L.v)], o=weight(L.o),
                gate_up=[weight(w) for w in (L.gate, L.up)], down=weight(L.down), write=write, attend=attend))
        for L in self.layers:   # one for all: their launches follow one another
            L["attend"].use_workspace(workspace)
        self.keeps = [plan("cache_keep", cache=fields | data, path=self.path, kept=self.kept, lengths=self.lengths,
                           new_lengths=self.new_lengths, sequences=sequences, tokens=nodes, layers=count,
                           layer_stride=data["key"][0].numel(),
                           scale_layer_stride=data["key_scale"][0].numel() if cache == CACHE_Q8 else 0)
                      for fields, data, count in self.caches.values()]

    # ---- one pass of the step's rows through the model ------------------------------

    def _product(self, weights, x, outs, **more):
        matmul(weights[0][0], weights[0][1], [w[2] for w in weights], x, outs, tokens=x.shape[0], **more)

    def _norm(self, gain, post_gain, add):
        a = self.arch
        fields = dict(hidden=self.hidden, normed=self.normed, gain=gain, width=a.hidden, tokens=self.hidden.shape[0],
                      epsilon=a.epsilon, add=int(add))
        if add:
            fields["output"] = self.out
            if post_gain is not None:
                fields["post_gain"] = post_gain
        run("norm", **fields)

    def _forward(self, logits: bool) -> None:
        a = self.arch
        fmt, _, member = self.embed
        run("gather", piece=member[0], format=fmt, blocks=member[1], width=a.hidden, row_count=a.vocab, ids=self.ids,
            tokens=self.ids.shape[0], scale=a.embed_scale, hidden=self.hidden)
        post = None
        for i, L in enumerate(self.layers):
            self._norm(L["attn_norm"], post, i > 0)
            self._product(L["qkv"], self.normed, [self.q, self.k, self.v], epilogue=QKV)
            L["write"]()
            L["attend"]()
            self._product([L["o"]], self.att, [self.out])
            self._norm(L["ffn_norm"], L["post_attn_norm"], True)
            self._product(L["gate_up"], self.normed, [self.act], epilogue=GATED, activation=a.activation)
            self._product([L["down"]], self.act, [self.out])
            post = L["post_ffn_norm"]
        if logits:
            self._norm(self.output_norm, post, True)
            self._product([self.head], self.normed, [self.logits])

    def _within_context(self, lengths, rows) -> None:
        """rows: positions past its length that each sequence needs."""
        for s, (length, n) in enumerate(zip(lengths, rows)):
            if n and length + n > self.arch.context:
                raise ValueError(f"sequence {s}: positions past the context of {self.arch.context} ({length} + {n})")

    def _in_vocabulary(self, tokens) -> None:
        """Tokens a sequence holds: a drafted one that is not the model's is refused by verification instead."""
        for t in tokens:
            if not 0 <= t < self.arch.vocab:
                raise ValueError(f"token {t} of a vocabulary of {self.arch.vocab}")

    def _set(self, trees) -> None:
        """trees: for each sequence its rows' (tokens, ancestor masks); no rows: it takes no part."""
        ids = np.zeros((self.sequences, self.nodes), np.uint32)
        masks = np.zeros((self.sequences, self.nodes), np.uint64)
        for s, (tokens, m) in enumerate(trees):
            ids[s, :len(tokens)], masks[s, :len(tokens)] = tokens, m
        put = lambda to, x: to.copy_(self.torch.from_numpy(x).view_as(to))  # noqa: E731
        put(self.ids, ids.reshape(-1).view(np.int32))
        put(self.masks, masks.view(np.int64))
        put(self.live, np.array([len(t) for t, _ in trees], np.int32))

    def _check_waits(self) -> None:
        """A CharlotteError where a bounded wait of a kernel ran out, and its results are no step's."""
        self.torch.cuda.current_stream().synchronize()
        check(lib().cb_fault_check(None))

    # ---- steps ------------------------------------------------------------------------

    def prefill(self, prompts) -> None:
        """Writes each sequence's prompt but its last token, which the first step takes as its row 0. A prompt that does
        not fit its sequence's context, and a token that is not the model's, is a ValueError, and nothing runs."""
        self._within_context(self.lengths.tolist(), [len(p) - 1 for p in prompts])
        self._in_vocabulary(t for p in prompts for t in p)
        done, start = [0] * self.sequences, self.lengths.clone()
        while any(d < len(p) - 1 for d, p in zip(done, prompts)):
            trees = []
            for s, p in enumerate(prompts):
                part = p[done[s]:min(done[s] + self.nodes, len(p) - 1)]
                trees.append((part, [(2 << i) - 1 for i in range(len(part))]))
                done[s] += len(part)
            self._set(trees)
            self._forward(logits=False)
            self.lengths += self.live
        try:
            self._check_waits()
        except CharlotteError:
            self.lengths.copy_(start)
            raise

    def step(self, trees, sampling=None, uniforms=None, draft=None, draft_sampling=None):
        """One step of each sequence's tree: (tokens, parents), row 0 the sequence's last token (parent -1) and a row
        after its parent. `sampling`, `draft_sampling`: dicts of temperature, top_k, top_p, min_p, what they leave out as
        in DRAW (greedy); `uniforms` [sequences, nodes], which a target with a temperature needs; `draft`: the drafting model's
        candidates [sequences, nodes, 64, 2] (int32, cuda), None where each drafted token was certain. Returns each
        sequence's new tokens, the last of them the next tree's row 0. A tree with a row past the context is a ValueError,
        and nothing runs; a kernel whose wait ran out and logits that are not finite are a CharlotteError, and the step
        can be taken again."""
        target = DRAW | (sampling or {})
        if target["temperature"] > 0 and uniforms is None:
            raise ValueError("a target with a temperature draws by uniform numbers, and none are given")
        masks = [(tokens, ancestors(parents)) for tokens, parents in trees]
        self._within_context(self.lengths.tolist(), [max((x.bit_count() for x in m), default=0) for _, m in masks])
        self._in_vocabulary(tokens[0] for tokens, _ in masks if len(tokens))
        self._set(masks)
        self._forward(logits=True)
        a, rows = self.arch, self.ids.shape[0]
        run("select", logits=self.logits, count=a.vocab, partials=self.partials, ticket=self.tickets,
            candidates=self.candidates, rows=rows, logits_stride=a.vocab, candidates_only=1)
        if uniforms is not None:
            self.uniforms.copy_(uniforms)
        plan("verify", candidates=self.candidates, draft_candidates=draft, ids=self.ids, uniforms=self.uniforms,
             nodes=self.live, ancestors=self.masks, path=self.path, kept=self.kept, sampled=self.sampled,
             sequences=self.sequences, tokens=self.nodes, target=target, draft=DRAW | (draft_sampling or {}))()
        for keep in self.keeps:
            keep()
        path, kept, sampled = (x.cpu().numpy() for x in (self.path, self.kept, self.sampled))
        self._check_waits()   # before the lengths, so that a failed step's rows are no entries
        if sampled[:, 1].any():
            raise CharlotteError(ERROR_STEP, f"sequences {np.flatnonzero(sampled[:, 1]).tolist()}: the first candidate of a kept row is not finite")
        self.lengths.copy_(self.new_lengths)
        return [[int(trees[s][0][i]) for i in path[s, 1:kept[s]]] + [int(sampled[s, 0])] if kept[s] else []
                for s in range(self.sequences)]

    def generate(self, prompts, count: int, drafter=None, sampling=None, seed: int = 0):
        """`count` new tokens of each prompt (at least; lists of ints), drafted by `drafter(tokens so far, rows)` ->
        (tokens, parents) of the rows after row 0, parents counted with it; rows past the context are left out. Returns
        (the new tokens, steps taken). A ValueError where a prompt and its tokens but the last do not fit the context."""
        drafter = drafter or lookup
        self._within_context([len(p) for p in prompts], [max(count - 1, 0)] * len(prompts))
        self.lengths.zero_()
        self.prefill(prompts)
        rng = np.random.default_rng(seed)
        told, steps = [list(p) for p in prompts], 0
        while any(len(t) - len(p) < count for t, p in zip(told, prompts)):
            trees = []
            for t, p in zip(told, prompts):
                if len(t) - len(p) >= count:
                    trees.append(([], []))
                    continue
                tokens, parents = drafter(t, self.nodes)
                trees.append(less_deep([t[-1], *tokens], [-1, *parents], self.arch.context - len(t) + 1))
            u = self.torch.from_numpy(rng.random((self.sequences, self.nodes), np.float32)) if sampling else None
            for t, new in zip(told, self.step(trees, sampling, u)):
                t.extend(new)
            steps += 1
        return [t[len(p):] for t, p in zip(told, prompts)], steps


def ancestors(parents) -> list[int]:
    """The rows' ancestor masks: bit j of row i's is set when row j is an ancestor of it or i itself."""
    masks = []
    for i, parent in enumerate(parents):
        if not (parent == -1 and i == 0 or 0 <= parent < i):
            raise ValueError(f"row {i} comes before its parent {parent}")
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
    return masks


def less_deep(tokens, parents, depth: int):
    """The tree's rows of a depth below `depth` (row 0's is 0): a row's descendants go with it."""
    place = {-1: -1}
    for i, m in enumerate(ancestors(parents)):
        if m.bit_count() <= depth:
            place[i] = len(place) - 1
    return [tokens[i] for i in place if i >= 0], [place[parents[i]] for i in place if i >= 0]


def lookup(told, rows: int, most: int = 3):
    """Drafts by what followed the last tokens before: up to `most` earlier places, latest first, as branches of a tree."""
    tail = told[-2:]
    tokens, parents, place = [], [], {}
    for at in range(len(told) - len(tail) - 1, -1, -1):
        if told[at:at + len(tail)] != tail:
            continue
        node = 0
        for t in told[at + len(tail):at + len(tail) + rows]:
            if (node, t) not in place:
                if len(tokens) + 1 >= rows:
                    return tokens, parents
                tokens.append(t)
                parents.append(node)
                place[node, t] = len(tokens)
            node = place[node, t]
        most -= 1
        if most == 0:
            break
    return tokens, parents


def main() -> None:
    m = M.synthesize(M.tiny("qwen3"), seed=1)
    prompts = [[5, 6, 7, 8, 9] * 4, [1, 2, 3] * 5]
    d = SpeculativeDecoder(m, sequences=2, nodes=12)
    plain, plain_steps = d.generate(prompts, 60, drafter=lambda told, rows: ([], []))
    drafted, steps = d.generate(prompts, 60)
    same = all(x[:60] == y[:60] for x, y in zip(plain, drafted))
    print(f"60 tokens of two sequences: {plain_steps} plain steps, {steps} with drafts; the same tokens: {same}")


if __name__ == "__main__":
    main()

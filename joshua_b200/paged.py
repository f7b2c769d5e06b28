"""The decoders of this package with their keys and values in pages of few bits, for batches of long sequences.

Sequences take pages from one pool as they grow and give them back when they end (`release`); until its next prompt such a sequence
rests: it takes part in steps with nothing to attend to, and what they leave for it means nothing.  Sequences that begin with the same
prompt hold its full pages in common, and a step reads and multiplies those once for all of them (`share_prompt`).  Rotary positions
come from a table (any scaling of `rope.rope_table`), the next tokens from `sampling.sample` where a sampling rule is set.

    dec = PagedLlamaDecoder(cfg, device, batch=32, max_ctx=8192, kv_type="q8_0")
    dec.share_prompt(prompt_ids)                 # or dec.prefill(ids, sequence=i) for each
    dec.sampling = dict(temperature=..., top_p=...)
    dec.uniform.uniform_(); dec.step()           # token by token

A step may be captured in a graph by the caller, its pages reserved and one step run on the stream before.  The graph keeps the
sampling rule's tensors, the penalty and the number of shared pages as they were: capture another one when they change.  Replays move
`pos` alone; prompts, steps and host calls that follow (on the stream of the replays, or behind it) begin where it stands.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import JoshuaB200Error, check
from .kv_cache import PAGE, SCRATCH_ZEROED, PagedCache
from .llama import LlamaDecoder
from .moe_decoder import MoeDecoder
from .rope import Rope, rope_table
from .sampling import sample


def _same(a, b) -> bool:
    """Equal, tensors being the same one."""
    if isinstance(a, tuple):
        return len(a) == len(b) and all(map(_same, a, b))
    return a is b or not isinstance(a, torch.Tensor) and not isinstance(b, torch.Tensor) and a == b


class _Paged:
    def __init__(self, cfg, device, batch: int = 1, max_ctx: int = 640, kv_type: str = "q8_0", n_pages: int | None = None,
                 rope: Rope | None = None, **more):
        """`n_pages`: of the pool (default: enough for every sequence to reach max_ctx); `rope`: a table of max_ctx positions
        (default: the model's theta, unscaled, half layout)."""
        self.kv_type, self.pages_per_seq = kv_type, -(-max_ctx // PAGE)
        self.shared_pages = 0                     # leading pages that all sequences have in common
        # resting sequences still bring a row to every append: to a position each of pages behind the pool
        self._places = min(PAGE, max_ctx)
        self.n_pages = batch * self.pages_per_seq if n_pages is None else n_pages
        super().__init__(cfg, device, batch=batch, max_ctx=max_ctx, **more)
        self.rope = rope or Rope(rope_table(cfg.rope_theta, cfg.head_dim, max_ctx, self.dev))
        # -1: no page.  A row never names a page that its sequence does not hold, so whatever still runs with the row of a sequence
        # that ended (a graph) raises the caches' flag instead of writing into another sequence's page.
        self.table = torch.full((batch, self.pages_per_seq), -1, dtype=torch.int32, device=self.dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=self.dev)
        self.resting = [False] * batch
        self.active = torch.ones(batch, dtype=torch.int32, device=self.dev)       # 0: rests
        self.idle_pos = torch.zeros(batch, dtype=torch.int32, device=self.dev)    # where a resting sequence's rows go
        self._seeds: dict[int, list] = {}         # recent ids given to a resting sequence
        self.free = list(range(self.n_pages))[::-1]
        self.owned = [[] for _ in range(batch)]   # page ids of each sequence, in order
        self.holders = [0] * self.n_pages         # sequences that have a page
        self.held = [0] * batch                   # positions each holds
        self._captured_by_caller = False          # then replays may have moved `pos` past `held`
        self.sampling: dict | None = None         # temperature, top_k, top_p, min_p: vectors of `batch`
        self.uniform = torch.zeros(batch, dtype=torch.float32, device=self.dev)   # numbers in [0, 1) for the next draw

    def _layer_cache(self) -> dict:
        return dict(cache=PagedCache(self.kv_type, self.cfg.kv_heads, self.cfg.head_dim, n_pages=self.n_pages + -(-self.batch // self._places),
                                     device=self.dev))

    def _attention_scratch(self) -> None:
        """One scratch for the attention of all layers; one that a caller's graph may hold stays until the decoder goes."""
        c, old = self.cfg, getattr(self, "att_scratch", [])
        need = self.layers[0]["cache"].scratch_bytes(self.batch, c.q_heads, self.shared_pages)
        if not old or old[-1].numel() < need:
            size = max(need, 2 * old[-1].numel() if old else SCRATCH_ZEROED)   # all older ones together are smaller
            self.att_scratch = [*old, torch.zeros(size, dtype=torch.uint8, device=self.dev)]

    def _index(self, sequence: int) -> int:
        if not 0 <= sequence < self.batch:
            raise JoshuaB200Error(_lib.E_INVALID, f"sequence {sequence} of {self.batch}")
        return sequence

    # ── pages ───────────────────────────────────────────────────────────
    def reserve(self, sequence: int, positions: int) -> None:
        """Pages for the first `positions` positions of a sequence.  A step takes them itself as they fill; reserve them before
        capturing one in a graph."""
        self._reserve({self._index(sequence): positions})

    def _reserve(self, positions: dict) -> None:
        """Pages for so many positions of each of these sequences, or for none of them if there are not enough."""
        wanted = 0
        for i, n in positions.items():
            if n > self.max_ctx:
                raise JoshuaB200Error(_lib.E_TOO_LARGE, f"{n} positions in a decoder of {self.max_ctx}")
            wanted += max(0, -(-n // PAGE) - len(self.owned[i]))
        if wanted > len(self.free):
            raise JoshuaB200Error(_lib.E_TOO_LARGE, f"{wanted} pages wanted, {len(self.free)} of {self.n_pages} are free")
        places, pages = [], []
        for i, n in positions.items():
            mine = self.owned[i]
            while len(mine) < -(-n // PAGE):
                places.append(i * self.pages_per_seq + len(mine))
                pages.append(self.free.pop())
                mine.append(pages[-1])
                self.holders[pages[-1]] = 1
        if pages:   # one copy for all of them, from pinned memory: the host waits for nothing
            new = torch.tensor([places, pages], dtype=torch.int64, pin_memory=True).to(self.dev, non_blocking=True)
            self.table.view(-1).scatter_(0, new[0], new[1].int())

    def _give_back(self, pages) -> None:
        for page in pages:
            self.holders[page] -= 1
            if self.holders[page] == 0:
                self.free.append(page)

    def release(self, sequence: int) -> None:
        """Ends a sequence: its pages go back (shared ones when the last sequence ends).  It rests until its next prompt, which
        begins at position 0."""
        self._give_back(self.owned[self._index(sequence)])
        self.owned[sequence], self.held[sequence] = [], 0
        self.table[sequence] = -1
        self.table[sequence, 0] = self.n_pages + sequence // self._places
        self.pos[sequence], self.active[sequence], self.idle_pos[sequence] = 0, 0, sequence % self._places
        self.resting[sequence] = True
        self._seeds.pop(sequence, None)
        self.window[sequence], self.window_state[sequence] = 0, 0   # the next prompt is another text
        if sequence == 0:
            self.shared_pages = 0   # the kernels find the common pages through the first sequence

    def _wake(self, i: int) -> None:
        """A sequence that rests, and has its pages, takes part again, from position 0."""
        if not self.resting[i]:
            return
        self.resting[i] = False
        self.pos[i], self.active[i], self.idle_pos[i] = 0, 1, 0
        self.window[i], self.window_state[i] = 0, 0   # steps have left ids there
        if i in self._seeds:
            super().seed_window(self._seeds.pop(i), i)
        self.shared_pages = 0       # it has other pages than those who share

    def reset(self, token: int = 42) -> None:
        """All sequences from position 0, none of them resting."""
        for mine in self.owned:
            self._give_back(mine)
        self.owned, self.held, self.resting = [[] for _ in self.owned], [0] * self.batch, [False] * self.batch
        self._seeds.clear()
        self.shared_pages = 0
        self.table.fill_(-1), self.active.fill_(1), self.idle_pos.zero_()
        super().reset(token)

    def seed_window(self, prompt_ids, sequence: int | None = None) -> None:
        super().seed_window(prompt_ids, sequence)
        for i in range(self.batch) if sequence is None else [range(self.batch)[sequence]]:
            if self.resting[i]:
                self._seeds[i] = [int(t) for t in prompt_ids][-64:]

    # ── a prompt ────────────────────────────────────────────────────────
    def prefill(self, token_ids, sequence: int = 0) -> None:
        """The prompt's tokens of one sequence in one pass, from where it stands; then self.logits[sequence], its sampled next
        token (self.token) and position, as `step` leaves them."""
        self._prompt(token_ids, self._index(sequence))
        self._sample_rows(slice(sequence, sequence + 1))

    def share_prompt(self, token_ids) -> None:
        """Begins all sequences with one prompt, read once: its full pages are common to all, what is left of it (less than a
        page) is copied.  Every sequence samples its own next token."""
        self._can_prompt()
        self._look()
        if any(self.held):
            raise JoshuaB200Error(_lib.E_INVALID, "sequences are under way: reset() first")
        n, others = len(token_ids), range(1, self.batch)
        full, pages = n // PAGE, -(-n // PAGE)
        # what sequences have reserved stays theirs, but for the pages in whose place the common ones stand
        wanted = max(0, pages - len(self.owned[0])) + sum(max(0, pages - max(full, len(self.owned[i]))) for i in others)
        back = sum(min(full, len(self.owned[i])) for i in others)
        if wanted > len(self.free) + back:
            raise JoshuaB200Error(_lib.E_TOO_LARGE, f"{wanted} pages wanted, {len(self.free) + back} of {self.n_pages} are free")
        self._prompt(token_ids, 0)
        common, rest = self.owned[0][:full], self.owned[0][full:]
        for i in others:
            self._give_back(self.owned[i][:full])
            for page in common:
                self.holders[page] += 1
            self.owned[i] = common + self.owned[i][full:]
            self.table[i, :full] = self.table[0, :full]
        self._reserve({i: n for i in others})
        for i in others:
            self._wake(i)
            if n % PAGE:
                for ly in self.layers:
                    ly["cache"].pages[self.owned[i][full]] = ly["cache"].pages[rest[0]]
            self.held[i] = n
        self.shared_pages = len(common)
        self._attention_scratch()
        self.pos.fill_(n - 1)
        self.logits.copy_(self.logits[0:1].expand(self.batch, -1).clone())
        self._sample_rows(slice(0, self.batch))

    def _can_prompt(self) -> None:
        if self.cfg.head_dim not in (64, 128):
            raise JoshuaB200Error(_lib.E_INVALID, "prompts need heads of 64 or 128")
        if getattr(self, "world", 1) > 1:
            raise JoshuaB200Error(_lib.E_INVALID, "prompts run on one GPU (the exchange windows are sized for decode batches)")

    def _prompt(self, token_ids, i) -> None:
        """Logits of the prompt's last token into self.logits[i]; self.pos[i] at that token."""
        self._can_prompt()
        L, c, P = _lib.lib(), self.cfg, lambda t: t.data_ptr()
        if not hasattr(self, "_layer_index"):   # the routed experts' decoder finds its layers by it
            self._layer_index = {id(ly): k for k, ly in enumerate(self.layers)}
        self._look()
        s = torch.cuda.current_stream(self.dev).cuda_stream
        ids = torch.as_tensor(token_ids, dtype=torch.int32).to(self.dev)
        S, h, start, f32 = int(ids.numel()), c.hidden, self.held[i], dict(dtype=torch.float32, device=self.dev)
        if S == 0:
            raise JoshuaB200Error(_lib.E_INVALID, "an empty prompt")
        self.reserve(i, start + S)
        self._wake(i)
        end = start + S
        pos = torch.arange(end, dtype=torch.int32, device=self.dev)
        seq = torch.full((end,), i, dtype=torch.int32, device=self.dev)
        first = pos[start:start + 1]
        x, qkv, att = torch.empty(S, h, **f32), torch.empty(S, c.qkv_rows, **f32), torch.empty(S, c.q_heads * c.head_dim, **f32)
        dense = torch.empty(2, c.kv_heads, end, c.head_dim, **f32)
        check(L.jq_embedding_dev(self.embed._h, P(ids), S, c.vocab, h, P(x), P(self.bad), s))
        for ly in self.layers:
            check(L.jq_matmul_norm_dev(ly["wqkv"]._h, S, h, c.qkv_rows, P(x), P(ly["attn_norm"]), c.eps, None, P(qkv), s))
            cache = ly["cache"]
            q = cache.append(qkv, pos[start:], self.table, n_q=c.q_heads, seq=seq[start:], rope=self.rope,
                             q_norm=ly["q_norm"] if self.qk_norm else None, k_norm=ly["k_norm"] if self.qk_norm else None, eps=c.eps)
            cache.read(pos, self.table, seq=seq, out=(dense[0], dense[1]))   # what the cache holds is what later tokens will see
            check(L.jq_attention_prefill_dev(P(q), P(dense[0]), P(dense[1]), P(first), S, c.q_heads, c.kv_heads, c.head_dim, end, P(att),
                                             P(self.bad_pos), s))
            check(L.jq_matmul_norm_dev(ly["wo"]._h, S, c.q_heads * c.head_dim, h, P(att), None, 0.0, P(x), P(x), s))
            self._ffn_prefill(ly, x, S, s)
        last = x[S - 1:S].clone()
        check(L.jq_matmul_norm_dev(self.output._h, 1, h, c.vocab, P(last), P(self.out_norm), c.eps, None, P(self.logits[i]), s))
        self.held[i] = end
        self.pos[i] = end - 1

    # ── a token of every sequence ───────────────────────────────────────
    def step(self, stream=None) -> None:
        """One token per sequence, as the dense decoder's step, on the current stream (`stream` is that one's handle or None)."""
        now = torch.cuda.current_stream(self.dev).cuda_stream
        if stream is not None and stream != now:
            raise JoshuaB200Error(_lib.E_INVALID, "a paged decoder's step runs on the current stream")
        self._advance()
        self._launches(now)

    def _advance(self) -> None:
        """Counts one position more of every sequence that does not rest, with a page for it; where there is none, nothing."""
        if torch.cuda.is_current_stream_capturing():
            self._captured_by_caller = True
            return
        self._look()
        self._reserve({i: n + 1 for i, n in enumerate(self.held) if not self.resting[i]})
        self.held = [n + (not rests) for n, rests in zip(self.held, self.resting)]

    def _look(self) -> None:
        """Positions as replays of a caller's graph left them."""
        if self._captured_by_caller:
            self.held = [0 if rests else n for n, rests in zip(self.pos.tolist(), self.resting)]

    def _launches(self, stream) -> None:
        torch.addcmul(self.idle_pos, self.pos, self.active, out=self.pos)   # resting: to its place behind the pool,
        torch.addcmul(self.active, self.pos, self.active, out=self.lens)    # and no positions to attend to; else pos + 1
        super().step(stream)

    def _attend(self, ly, s) -> None:
        c, cache = self.cfg, ly["cache"]
        cache.append(self.qkv, self.pos, self.table, n_q=c.q_heads, rope=self.rope, q_norm=ly["q_norm"] if self.qk_norm else None,
                     k_norm=ly["k_norm"] if self.qk_norm else None, eps=c.eps, out=self.q)
        cache.attend(self.q, self.lens, self.table, n_q=c.q_heads, shared_pages=self.shared_pages, out=self.attn,
                     scratch=self.att_scratch[-1])

    def _sample(self, s) -> None:
        self._sample_rows(slice(0, self.batch))

    def _sample_rows(self, rows) -> None:
        penalised = self.repetition_penalty != 1.0
        window, state = self.window[rows], self.window_state[rows]
        if self.sampling is None:   # of equal maxima the last one, however many rows
            L, P, n = _lib.lib(), lambda t: t[rows].data_ptr(), rows.stop - rows.start
            s = torch.cuda.current_stream(self.dev).cuda_stream
            if penalised:
                check(L.jq_sample_greedy_dev(P(self.logits), n, self.cfg.vocab, self.repetition_penalty, window.data_ptr(), state.data_ptr(),
                                             P(self.token), P(self.pos), self.argmax_scratch.data_ptr(), s))
            else:
                check(L.jq_argmax_dev(P(self.logits), n, self.cfg.vocab, P(self.token), P(self.pos), self.argmax_scratch.data_ptr(), s))
            return
        sample(self.logits[rows], self.uniform[rows], **{k: v[rows] for k, v in self.sampling.items()},
               repetition_penalty=self.repetition_penalty, window=window if penalised else None,
               window_state=state if penalised else None, pos=self.pos[rows], token=self.token[rows])

    def _positions_used(self) -> int:
        return 0   # each sequence's own are counted by `held`

    def _frozen(self):
        """What a captured step keeps as it was: the host call captures another one when it changes."""
        rule = self.sampling and tuple(self.sampling.items())   # the tensors themselves: a graph reads them where they are
        return self.shared_pages, self.repetition_penalty, rule

    def _capture(self, stream):
        frozen = self._frozen()
        graph = super()._capture(stream)
        self._captured_with = frozen
        return graph

    def forward_host(self, token_ids, out_logits=None):
        token_ids = torch.as_tensor(token_ids, dtype=torch.int32).reshape(self.batch)
        held = list(self.held)
        self._advance()
        self._host_calls = 0   # each sequence's own positions are the limit
        try:
            if getattr(self, "_host", None) is not None and not _same(self._captured_with, self._frozen()):
                self._host = (*self._host[:3], self._capture(self._host[0]))
            return super().forward_host(token_ids, out_logits)
        except Exception:
            self.held = held
            raise

    def check_flags(self) -> None:
        super().check_flags()
        for ly in self.layers:
            ly["cache"].check_flags()

    def cache_bytes(self) -> int:
        return sum(ly["cache"].pages.numel() for ly in self.layers)

    def step_unfused(self, stream=None) -> None:
        raise JoshuaB200Error(_lib.E_INVALID, "the separate kernels of the dense cache do not read pages")


class PagedLlamaDecoder(_Paged, LlamaDecoder):
    """`LlamaDecoder` over a paged cache."""


class PagedMoeDecoder(_Paged, MoeDecoder):
    """`MoeDecoder` over a paged cache."""

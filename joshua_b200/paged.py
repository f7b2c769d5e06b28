"""The decoders of this package with their keys and values in pages of few bits, for batches of long sequences.

Sequences take pages from one pool as they grow and give them back when they end (`release`); until its next prompt such a sequence
rests: it takes part in steps with nothing to attend to, and what they leave for it means nothing.  Sequences that begin with the same
prompt hold its full pages in common, and a step reads and multiplies those once for all of them (`share_prompt`).  Rotary positions
come from a table (any scaling of `rope.rope_table`), the next tokens from `sampling.sample` where a sampling rule is set.

    dec = PagedLlamaDecoder(cfg, device, batch=32, max_ctx=8192, kv_type="q8_0")
    dec.share_prompt(prompt_ids)                 # or dec.prefill(ids, sequence=i) for each
    dec.sampling = dict(temperature=..., top_p=...)
    dec.uniform.uniform_(); dec.step()           # token by token
    dec.extend({0: ids, 3: more}, scores=5)      # several sequences' next tokens in one pass, with their log probabilities
    dec.rewind(3, positions)                     # without the last of them (or with all: under a penalty they become recent ids)

With `attention_window` a token sees that many positions back and the first `attention_sinks`; pages that no later token sees go back to
the pool as the sequences grow, and long prompts are read in parts.

A step may be captured in a graph by the caller, its pages reserved and one step run on the stream before.  The graph keeps the
sampling rule's tensors, the penalty and the number of shared pages as they were: capture another one when they change.  Replays move
`pos` alone; prompts, steps and host calls that follow (on the stream of the replays, or behind it) begin where it stands.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import _lib
from ._lib import JoshuaB200Error, check
from .kv_cache import PAGE, SCRATCH_ZEROED, PagedCache
from .llama import LlamaDecoder
from .moe_decoder import MoeDecoder
from .rope import Rope, rope_table
from .sampling import log_probs, sample


def _same(a, b) -> bool:
    """Equal, tensors being the same one."""
    if isinstance(a, tuple):
        return len(a) == len(b) and all(map(_same, a, b))
    return a is b or not isinstance(a, torch.Tensor) and not isinstance(b, torch.Tensor) and a == b


def _by_age(window, state) -> list:
    """A row of recent ids from the oldest to the latest."""
    ids, (count, at) = window.tolist(), state.tolist()
    count = min(count, 64)
    return [ids[(at - count + k) % 64] for k in range(count)]


@dataclass
class _Given:
    """Ids that a sequence was given at positions start .. end - 1, and its recent ids (the repetition penalty's) in front of them."""
    start: int
    end: int
    ids: torch.Tensor | None   # None: a prompt's, which are not among the recent ids
    recent: tuple | list       # rows of `window` and `window_state`; a list once they were looked at
    drawn: bool                # the latest of them was drawn for `start`
    holes: list = field(default_factory=list)   # ranges of positions whose ids are not among them: prompts, tokens set by hand
    entered: bool = False      # `ids` came in behind them


class _Paged:
    attention_window = attention_sinks = 0
    prompt_rows = 2048    # of a prompt in one pass, where there is a window
    score_rows = 256      # whose logits are held at a time for their scores

    def __init__(self, cfg, device, batch: int = 1, max_ctx: int = 640, kv_type: str = "q8_0", n_pages: int | None = None,
                 rope: Rope | None = None, attention_window: int = 0, attention_sinks: int = 0, **more):
        """`n_pages`: of the pool (default: enough for every sequence to reach max_ctx); `rope`: a table of max_ctx positions
        (default: the model's theta, unscaled, half layout); `attention_window`: positions that a token sees, its own the last of them
        (0: all), besides the first `attention_sinks`."""
        if attention_window < 0 or attention_sinks < 0 or attention_sinks and not attention_window:
            raise JoshuaB200Error(_lib.E_INVALID, f"a window of {attention_window} with {attention_sinks} sinks")
        self.attention_window, self.attention_sinks = attention_window, attention_sinks
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
        self.owned = [[] for _ in range(batch)]   # page ids of each sequence, in order; None: gone back, out of the window
        self.kept_from = [0] * batch              # pages in front of it (but those of sinks) have gone back
        self.holders = [0] * self.n_pages         # sequences that have a page
        self.held = [0] * batch                   # positions each holds
        self._given: dict[int, _Given] = {}       # what it was given last, under a repetition penalty
        self._drawn = [False] * batch             # its latest recent id was drawn for its next position
        self._captured_by_caller = False          # then replays may have moved `pos` past `held`
        self.sampling: dict | None = None         # temperature, top_k, top_p, min_p: vectors of `batch`
        self.uniform = torch.zeros(batch, dtype=torch.float32, device=self.dev)   # numbers in [0, 1) for the next draw

    def _layer_cache(self) -> dict:
        return dict(cache=PagedCache(self.kv_type, self.cfg.kv_heads, self.cfg.head_dim, n_pages=self.n_pages + -(-self.batch // self._places),
                                     device=self.dev))

    def _attention_scratch(self, rows: int | None = None) -> None:
        """One scratch for the attention of all layers, of steps and of passes of so many `rows`; one that a caller's graph may hold stays
        until the decoder goes."""
        c, old = self.cfg, getattr(self, "att_scratch", [])
        cache = self.layers[0]["cache"]
        if rows or self.attention_window:
            need = cache.scratch_bytes(self.batch, c.q_heads, rows=rows or self.batch)
        else:
            need = cache.scratch_bytes(self.batch, c.q_heads, self.shared_pages)
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
        self._enter(places, pages)

    def _enter(self, places, pages) -> None:
        """Page ids into the table: one copy for all of them, from pinned memory: the host waits for nothing."""
        if pages:
            new = torch.tensor([places, pages], dtype=torch.int64, pin_memory=True).to(self.dev, non_blocking=True)
            self.table.view(-1).scatter_(0, new[0], new[1].int())

    def _trim(self, sequences) -> None:
        """Gives back the pages that no token from the sequences' next ones on sees."""
        places, pages = [], []
        for i in sequences if self.attention_window else ():
            first = max(self.kept_from[i], -(-self.attention_sinks // PAGE))
            behind = min((self.held[i] + 1 - self.attention_window) // PAGE, len(self.owned[i]))
            for k in range(first, behind):
                if self.owned[i][k] is not None:
                    places.append(i * self.pages_per_seq + k)
                    pages.append(self.owned[i][k])
                    self.owned[i][k] = None
            self.kept_from[i] = max(first, behind)
        self._enter(places, [-1] * len(places))
        self._give_back(pages)

    def _give_back(self, pages) -> None:
        for page in pages:
            if page is None:
                continue
            self.holders[page] -= 1
            if self.holders[page] == 0:
                self.free.append(page)

    def release(self, sequence: int) -> None:
        """Ends a sequence: its pages go back (shared ones when the last sequence ends).  It rests until its next prompt, which
        begins at position 0."""
        self._give_back(self.owned[self._index(sequence)])
        self.owned[sequence], self.held[sequence], self.kept_from[sequence] = [], 0, 0
        self.table[sequence] = -1
        self.table[sequence, 0] = self.n_pages + sequence // self._places
        self.pos[sequence], self.active[sequence], self.idle_pos[sequence] = 0, 0, sequence % self._places
        self.resting[sequence] = True
        self._seeds.pop(sequence, None)
        self._forget_given(sequence)
        self.window[sequence], self.window_state[sequence] = 0, 0   # the next prompt is another text
        if sequence == 0:
            self.shared_pages = 0   # the kernels find the common pages through the first sequence

    def _wake(self, i: int) -> None:
        """A sequence that rests, and has its pages, takes part again, from position 0."""
        if not self.resting[i]:
            return
        self.resting[i] = False
        self._forget_given(i)
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
        self.kept_from = [0] * self.batch
        self._seeds.clear()
        self._given, self._drawn = {}, [False] * self.batch
        self.shared_pages = 0
        self.table.fill_(-1), self.active.fill_(1), self.idle_pos.zero_()
        super().reset(token)

    def seed_window(self, prompt_ids, sequence: int | None = None) -> None:
        super().seed_window(prompt_ids, sequence)
        for i in range(self.batch) if sequence is None else [range(self.batch)[sequence]]:
            self._forget_given(i)
            if self.resting[i]:
                self._seeds[i] = [int(t) for t in prompt_ids][-64:]

    # ── a prompt ────────────────────────────────────────────────────────
    def prefill(self, token_ids, sequence: int = 0) -> None:
        """The prompt's tokens of one sequence in one pass, from where it stands; then self.logits[sequence], its sampled next
        token (self.token) and position, as `step` leaves them."""
        self._note_given({sequence: self._prompt(token_ids, self._index(sequence))})
        self._sample_rows(slice(sequence, sequence + 1))

    def share_prompt(self, token_ids) -> None:
        """Begins all sequences with one prompt, read once: its full pages are common to all, what is left of it (less than a
        page) is copied.  Every sequence samples its own next token."""
        self._can_prompt(dense=not self.attention_window)
        self._look()
        if any(self.held):
            raise JoshuaB200Error(_lib.E_INVALID, "sequences are under way: reset() first")
        n, others = len(token_ids), range(1, self.batch)
        full, pages = n // PAGE, -(-n // PAGE)
        # what sequences have reserved stays theirs, but for the pages in whose place the common ones stand
        wanted, free = sum(max(0, pages - max(full, len(self.owned[i]))) for i in others), len(self.free)
        if self.attention_window:   # pages go back while the prompt is read
            free = self._room_for_parts(0, n)
        else:
            wanted += max(0, pages - len(self.owned[0]))
        free += sum(page is not None for i in others for page in self.owned[i][:full])
        if wanted > free:
            raise JoshuaB200Error(_lib.E_TOO_LARGE, f"{wanted} pages wanted, {free} of {self.n_pages} are free")
        self._prompt(token_ids, 0)
        common, rest = self.owned[0][:full], self.owned[0][full:]
        for i in others:
            self._give_back(self.owned[i][:full])
            for page in common:
                if page is not None:
                    self.holders[page] += 1
            self.owned[i], self.kept_from[i] = common + self.owned[i][full:], self.kept_from[0]
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
        self._note_given({i: n for i in range(self.batch)})
        self._sample_rows(slice(0, self.batch))

    def extend(self, tokens: dict, scores: int | None = None):
        """The next tokens of several sequences (ids by sequence), each from where it stands, in one pass; then self.logits, the sampled
        next tokens (self.token) and positions of these sequences, as `prefill` leaves them.

        With `scores` (a number of alternatives, at most 32): by sequence, what `sampling.log_probs` gives for its tokens but the first,
        each at the position in front of it.

        The repetition penalty's recent ids take what is sampled, as with `prefill`: a prompt's are the caller's to enter (`seed_window`), drafts
        come in with `rewind`, which says how many of them stay."""
        new = {self._index(i): torch.as_tensor(ids, dtype=torch.int32).reshape(-1) for i, ids in sorted(tokens.items())}
        if not new or any(ids.numel() == 0 for ids in new.values()):
            raise JoshuaB200Error(_lib.E_INVALID, "nothing to extend, or an empty prompt")
        if len({ids.device for ids in new.values()}) > 1:
            new = {i: ids.to(self.dev) for i, ids in new.items()}
        if scores is not None and not 0 <= scores <= 32:
            raise JoshuaB200Error(_lib.E_INVALID, f"{scores} alternatives: 0 to 32")
        self._can_prompt(dense=False)
        rows = sum(ids.numel() for ids in new.values())
        if rows > 65536 or rows * self.cfg.q_heads > 2**27 or rows * (4 * self.pages_per_seq + 8) >= 2**32:
            raise JoshuaB200Error(_lib.E_TOO_LARGE, f"{rows} tokens in one pass")
        self._look()
        self._trim(new)
        x = self._pass(new)
        counts = [ids.numel() for ids in new.values()]
        given = self._scores(x, new, scores) if scores is not None else None
        ends = torch.tensor(counts).cumsum(0)
        seqs = torch.tensor(list(new), device=self.dev)
        last = x[(ends - 1).to(self.dev)].contiguous()
        self.logits[seqs] = self._head(last)
        self.pos[seqs] = torch.tensor([self.held[i] - 1 for i in new], dtype=torch.int32, device=self.dev)
        self._note_given({i: ids.numel() for i, ids in new.items()}, new)
        for i in new:
            self._sample_rows(slice(i, i + 1))
        return given

    def rewind(self, sequence: int, positions: int, token: int | None = None) -> None:
        """Forgets a sequence's tokens behind its first `positions`, drafts that were not taken: its next ones go there (`extend`, or
        `step`, which reads self.token[sequence]; `token` is written there).  Not into pages that it has in common with others, nor to where
        its window has given back what it would see.

        Under a repetition penalty the recent ids become those of the text that is left: of the drafts of the last `extend` the ones in
        front of `positions` (all of them, where that is where the sequence stands) come in, in the place of what was drawn there; what was
        drawn behind them goes out, and `token` comes in.  Where the way back leads to the first of the last ids given or beyond, or over
        more than 64 steps, what newer ids had pushed out is not brought back."""
        self._look()
        i, n = self._index(sequence), positions
        if not 0 < n <= self.held[i]:
            raise JoshuaB200Error(_lib.E_INVALID, f"{n} of {self.held[i]} positions")
        if token is not None and not 0 <= token < self.cfg.vocab:
            raise JoshuaB200Error(_lib.E_INVALID, f"token {token} of {self.cfg.vocab}")
        mine, window = self.owned[i], self.attention_window
        if n < self.held[i]:
            if n < self.shared_pages * PAGE or any(page is not None and self.holders[page] > 1 for page in mine[n // PAGE:]):
                raise JoshuaB200Error(_lib.E_INVALID, f"{n} positions end in front of pages that sequences share")
            if window and any(page is None for page in mine[max(0, n + 1 - window) // PAGE:]):
                raise JoshuaB200Error(_lib.E_INVALID, f"pages in front of position {n} have gone back")
        self._rewind_recent(i, n, token)
        if token is not None:
            self.token[i] = token
        self.held[i] = n
        self.pos[i] = n

    # ── the repetition penalty's recent ids ─────────────────────────────
    def _forget_given(self, i: int) -> None:
        self._given.pop(i, None)
        self._drawn[i] = False

    def _note_given(self, counts: dict, ids: dict | None = None) -> None:
        """Keeps the recent ids of sequences as they are in front of what is drawn next; counts: of the ids that each was given, `ids`
        (None, or at position 0: a prompt)."""
        penalised, rows = self.repetition_penalty != 1.0, list(counts)
        window, state = (t[torch.tensor(rows, device=self.dev)] for t in (self.window, self.window_state)) if penalised else (None, None)
        for k, (i, n) in enumerate(counts.items()):
            before = self._given.pop(i, None)
            if penalised:
                start, end, drawn = self.held[i] - n, self.held[i], self._drawn[i]
                text = ids[i].clone() if ids and start else None
                holes = [range(r.start, min(r.stop, start)) for r in before.holes if r.start < start] if before else []
                if before and before.ids is not None and not before.entered:
                    holes.append(range(before.start + before.drawn, before.end))
                if text is None:
                    holes.append(range(start + drawn, end))
                self._given[i] = _Given(start, end, text, (window[k], state[k]), drawn, holes)
            self._drawn[i] = penalised

    def _rewind_recent(self, i: int, n: int, token: int | None) -> None:
        given, held = self._given.get(i), self.held[i]
        if self.repetition_penalty == 1.0:
            return self._forget_given(i)
        if n == held and token is None and (given is None or given.ids is None):
            return
        if given is not None and not isinstance(given.recent, list):
            given.recent = _by_age(*given.recent)
        if given is not None and given.start < min(n, given.end) and given.ids is None and given.drawn:   # a prompt stands where it was drawn
            given.recent, given.drawn = given.recent[:-1], False
            given.holes = [*given.holes, range(given.start, given.start + 1)]
        recent = self._recent(i, n, token is None) + ([] if token is None else [token])
        super().seed_window(recent, i)
        if given is not None:
            given.entered = True
        self._drawn[i] = token is not None or n == held and self._drawn[i]
        if given is None or n < given.start:
            given = self._given[i] = _Given(n, n, None, recent[-64:], token is not None, given.holes if given else [])
        elif n < given.end:
            given.end, given.ids = n, None if given.ids is None else given.ids[:n - given.start]
        if n < held or token is not None:
            given.holes = [range(r.start, min(r.stop, n)) for r in given.holes if r.start < n] + [range(n, n + 1)] * (token is None)

    def _recent(self, i: int, n: int, whole: bool) -> list:
        """Recent ids of a sequence's first n positions, and what was drawn for the next one if it stands there (and `whole`)."""
        now, given, held, drawn = _by_age(self.window[i], self.window_state[i]), self._given.get(i), self.held[i], self._drawn[i]
        if given is not None and n < given.start:
            now, held, drawn = given.recent, given.start, given.drawn
        holes = given.holes if given else []
        if given is None or n < given.start:   # those of positions n .. held go out
            gone = sum(not any(p in r for r in holes) for p in range(n, held)) + drawn
            return now[:max(0, len(now) - gone)]
        recent = given.recent[:-1] if given.drawn else given.recent
        if given.ids is not None:
            recent = recent + given.ids[:n - given.start].tolist()
        since = [p for p in range(given.end, held + drawn) if not any(p in r for r in holes)]   # positions of the ids drawn since
        kept = sum(p < n or whole and p == n == held for p in since)
        if kept:
            recent = now[:len(now) - len(since) + kept] if len(since) > len(now) else recent + now[len(now) - len(since):][:kept]
        return recent[-64:]

    def _head(self, x):
        logits = torch.empty(x.size(0), self.cfg.vocab, dtype=torch.float32, device=self.dev)
        s = torch.cuda.current_stream(self.dev).cuda_stream
        check(_lib.lib().jq_matmul_norm_dev(self.output._h, x.size(0), self.cfg.hidden, self.cfg.vocab, x.data_ptr(), self.out_norm.data_ptr(),
                                            self.cfg.eps, None, logits.data_ptr(), s))
        return logits

    def _scores(self, x, new, top: int) -> dict:
        """Log probabilities of every sequence's tokens behind its first one, some rows' logits at a time."""
        out, row = {}, 0
        for i, ids in new.items():
            n = ids.numel()
            ids, parts = ids.to(self.dev), []
            for a in range(0, n - 1, self.score_rows):
                b = min(n - 1, a + self.score_rows)
                parts.append(log_probs(self._head(x[row + a:row + b]), ids[a + 1:b + 1], top=top))
            if not parts:
                parts.append(log_probs(self.logits[:0], ids[:0], top=top))
            out[i] = tuple(torch.cat(p) for p in zip(*parts))
            row += n
        return out

    def _pass(self, new: dict):
        """New ids of some sequences (by sequence, in order) through all layers, over the cache: [rows, hidden]."""
        L, c, P, i32 = _lib.lib(), self.cfg, lambda t: t.data_ptr(), dict(dtype=torch.int32, device=self.dev)
        if not hasattr(self, "_layer_index"):   # the routed experts' decoder finds its layers by it
            self._layer_index = {id(ly): k for k, ly in enumerate(self.layers)}
        self._reserve({i: self.held[i] + ids.numel() for i, ids in new.items()})
        for i in new:
            self._wake(i)
        counts = [new[i].numel() if i in new else 0 for i in range(self.batch)]
        S, h, f32 = sum(counts), c.hidden, dict(dtype=torch.float32, device=self.dev)
        s = torch.cuda.current_stream(self.dev).cuda_stream
        ids = torch.cat(list(new.values())).to(self.dev)
        pos = torch.cat([torch.arange(self.held[i], self.held[i] + n) for i, n in enumerate(counts)]).to(**i32)
        seq = torch.repeat_interleave(torch.arange(self.batch), torch.tensor(counts)).to(**i32)
        first = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], **i32)
        lens = torch.tensor([self.held[i] + n for i, n in enumerate(counts)], **i32)
        x, qkv, att = torch.empty(S, h, **f32), torch.empty(S, c.qkv_rows, **f32), torch.empty(S, c.q_heads * c.head_dim, **f32)
        self._attention_scratch(S)
        check(L.jq_embedding_dev(self.embed._h, P(ids), S, c.vocab, h, P(x), P(self.bad), s))
        for ly in self.layers:
            cache = ly["cache"]
            check(L.jq_matmul_norm_dev(ly["wqkv"]._h, S, h, c.qkv_rows, P(x), P(ly["attn_norm"]), c.eps, None, P(qkv), s))
            q = cache.append(qkv, pos, self.table, n_q=c.q_heads, seq=seq, rope=self.rope,
                             q_norm=ly["q_norm"] if self.qk_norm else None, k_norm=ly["k_norm"] if self.qk_norm else None, eps=c.eps)
            cache.attend_chunk(q, lens, self.table, n_q=c.q_heads, first=first, window=self.attention_window, sinks=self.attention_sinks, out=att,
                               scratch=self.att_scratch[-1])
            check(L.jq_matmul_norm_dev(ly["wo"]._h, S, c.q_heads * c.head_dim, h, P(att), None, 0.0, P(x), P(x), s))
            self._ffn_prefill(ly, x, S, s)
        for i, n in enumerate(counts):
            self.held[i] += n
        return x

    def _can_prompt(self, dense: bool = True) -> None:
        if dense and self.cfg.head_dim not in (64, 128):
            raise JoshuaB200Error(_lib.E_INVALID, "prompts need heads of 64 or 128")
        if getattr(self, "world", 1) > 1:
            raise JoshuaB200Error(_lib.E_INVALID, "prompts run on one GPU (the exchange windows are sized for decode batches)")

    def _prompt(self, token_ids, i) -> int:
        """Logits of the prompt's last token into self.logits[i]; self.pos[i] at that token.  How many there were."""
        self._can_prompt(dense=not self.attention_window)
        if self.attention_window:
            return self._prompt_in_parts(token_ids, i)
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
        return S

    def _prompt_in_parts(self, token_ids, i) -> int:
        """The same where there is a window: the dense attention of prompts has none."""
        ids = torch.as_tensor(token_ids, dtype=torch.int32).reshape(-1)
        if ids.numel() == 0:
            raise JoshuaB200Error(_lib.E_INVALID, "an empty prompt")
        self._look()
        self._room_for_parts(i, ids.numel())
        for part in ids.split(self.prompt_rows):
            self._trim([i])
            x = self._pass({i: part})
        self.logits[i] = self._head(x[-1:].clone())[0]
        self.pos[i] = self.held[i] - 1
        return ids.numel()

    def _room_for_parts(self, i, n: int) -> int:
        """Pages that are free behind all parts: what each takes and the window gives back.  Raises, before any is taken, if one does not
        fit."""
        if self.held[i] + n > self.max_ctx:
            raise JoshuaB200Error(_lib.E_TOO_LARGE, f"{self.held[i] + n} positions in a decoder of {self.max_ctx}")
        mine = [page is not None and self.holders[page] == 1 for page in self.owned[i]]   # whether it goes back to the pool
        free, held, sinks = len(self.free), self.held[i], -(-self.attention_sinks // PAGE)
        at = max(self.kept_from[i], sinks)
        while n:
            behind = min((held + 1 - self.attention_window) // PAGE, len(mine))
            if behind > at:
                free, at = free + sum(mine[at:behind]), behind
            part = min(n, self.prompt_rows)
            held, n = held + part, n - part
            more = max(0, -(-held // PAGE) - len(mine))
            if more > free:
                raise JoshuaB200Error(_lib.E_TOO_LARGE, f"{more} pages wanted, {free} of {self.n_pages} are free")
            free -= more
            mine += [True] * more
        return free

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
        self._trim(i for i in range(self.batch) if not self.resting[i])
        self._reserve({i: n + 1 for i, n in enumerate(self.held) if not self.resting[i]})
        self.held = [n + (not rests) for n, rests in zip(self.held, self.resting)]
        self._drawn = [self.repetition_penalty != 1.0 if not rests else drawn for drawn, rests in zip(self._drawn, self.resting)]

    def _look(self) -> None:
        """Positions as replays of a caller's graph left them."""
        if self._captured_by_caller:
            was, self.held = self.held, [0 if rests else n for n, rests in zip(self.pos.tolist(), self.resting)]
            self._drawn = [self.repetition_penalty != 1.0 if n != old else drawn for n, old, drawn in zip(self.held, was, self._drawn)]

    def _launches(self, stream) -> None:
        torch.addcmul(self.idle_pos, self.pos, self.active, out=self.pos)   # resting: to its place behind the pool,
        torch.addcmul(self.active, self.pos, self.active, out=self.lens)    # and no positions to attend to; else pos + 1
        super().step(stream)

    def _attend(self, ly, s) -> None:
        c, cache = self.cfg, ly["cache"]
        cache.append(self.qkv, self.pos, self.table, n_q=c.q_heads, rope=self.rope, q_norm=ly["q_norm"] if self.qk_norm else None,
                     k_norm=ly["k_norm"] if self.qk_norm else None, eps=c.eps, out=self.q)
        if self.attention_window:
            cache.attend(self.q, self.lens, self.table, n_q=c.q_heads, out=self.attn, scratch=self.att_scratch[-1],
                         window=self.attention_window, sinks=self.attention_sinks)
        else:
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

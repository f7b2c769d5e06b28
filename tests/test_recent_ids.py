"""Recent ids behind drafts, steps and ways back, in any order: the bookkeeping of the paged decoders alone, against the text itself."""
import random

import pytest
import torch

from joshua_b200.paged import _by_age, _Paged


class Ids:
    """What a decoder does with its recent ids."""

    def __init__(self):
        self.window, self.window_state = torch.zeros(1, 64, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)

    def seed_window(self, ids, sequence=None):
        tail = list(ids)[-64:]
        self.window[0] = torch.tensor(tail + [0] * (64 - len(tail)), dtype=torch.int32)
        self.window_state[0] = torch.tensor([len(tail), len(tail) % 64], dtype=torch.int32)

    def draw(self, token):
        held, at = self.window_state[0].tolist()
        self.window[0, at] = token
        self.window_state[0] = torch.tensor([min(held + 1, 64), (at + 1) % 64], dtype=torch.int32)


class Decoder(_Paged, Ids):
    def __init__(self):
        Ids.__init__(self)
        self.batch, self.dev, self.repetition_penalty = 1, "cpu", 1.3
        self.held, self.resting, self._given, self._drawn = [0], [False], {}, [False]

    def given(self, ids, prompt=False):
        self.held[0] += len(ids)
        self._note_given({0: len(ids)}, None if prompt else {0: torch.tensor(ids)})

    def back(self, n, token):
        self._rewind_recent(0, n, token)
        self.held[0] = n


@pytest.mark.parametrize("seed", range(8))
def test_any_order(seed):
    exact_ones = 0
    for r in (random.Random(1000 * seed + k) for k in range(120)):
        dec, some = Decoder(), lambda: r.randrange(1000)
        seeds = [some() for _ in range(r.choice([0, 10, 64]))]
        dec.seed_window(seeds, 0)
        first = r.randrange(1, 40)
        dec.given([some() for _ in range(first)], prompt=True)
        text = [some()]          # from position `first` on; the next position's too, if known; None: set by hand
        dec.draw(text[0])
        known = exact = True
        for _ in range(r.randrange(1, 25)):
            what, start = r.random(), dec.held[0]
            if what < 0.4:       # drafts, behind the token that is next or one set by hand
                ids = [text[-1] if known else some()] + [some() for _ in range(r.randrange(0, 6))]
                dec.given(ids)
                drawn = some()
                dec.draw(drawn)
                text = (text[:-1] if known else text) + ids
                stay, token = r.randrange(1, len(ids) + 1), some() if r.random() < 0.7 else None
                dec.back(start + stay, token)
                known = token is not None or stay == len(ids)
                text = text[:len(text) - len(ids) + stay] + ([token] if token is not None else [drawn] if known else [])
            elif what < 0.7:     # steps
                for _ in range(r.randrange(1, 20)):
                    text += [] if known else [None]
                    text.append(some())
                    dec.draw(text[-1])
                    dec.held[0], dec._drawn[0], known = dec.held[0] + 1, True, True
            else:
                n, token = max(first, start - r.randrange(0, 15)), some() if r.random() < 0.5 else None
                if n == start and token is None:
                    continue
                exact &= dec._given[0].start < n and start - dec._given[0].end < 64
                dec.back(n, token)
                known = token is not None
                text = text[:n - first] + ([token] if known else [])
            want, got = (seeds + [t for t in text if t is not None])[-64:], _by_age(dec.window[0], dec.window_state[0])
            assert got == (want if exact else want[len(want) - len(got):])
            exact_ones += exact
    assert exact_ones > 100

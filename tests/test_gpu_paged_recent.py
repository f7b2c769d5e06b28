"""The repetition penalty's recent ids when drafts are given with `extend` and taken back with `rewind`: those of the text that is left,
as if it had been taken by steps.  Ids are compared as they are; a sampled token with the likeliest one of the decoder's own logits."""
import numpy as np
import pytest

from joshua_b200._lib import JoshuaB200Error
from tests import serving_ref as ref
from tests.test_gpu_paged_decoder import ids, make

pytestmark = pytest.mark.gpu
PENALTY = 1.3


def recent(dec, i):
    """In order of age."""
    row, (count, at) = dec.window[i].tolist(), dec.window_state[i].tolist()
    return [row[(at - count + k) % 64] for k in range(count)]


def drawn_rightly(dec, i, before):
    l = ref.penalised(dec.logits[i].cpu().numpy(), PENALTY, before)
    return int(dec.token[i]) == len(l) - 1 - int(np.argmax(l[::-1]))


@pytest.mark.parametrize("seeds", [0, 40, 64])
@pytest.mark.parametrize("window", [0, 50])
def test_drafts(seeds, window):
    dec = make(3, attention_window=window)
    dec.repetition_penalty = PENALTY
    text = [ids(seeds, 10 + i) for i in range(3)]
    for i in range(3):
        dec.seed_window(text[i], i)
    rng = np.random.RandomState(seeds)

    def drew(i, behind):
        """What was sampled last is the likeliest behind these ids."""
        assert drawn_rightly(dec, i, behind[-64:])
        return int(dec.token[i])

    dec.extend({i: ids(50, i) for i in range(3)})
    for i in range(3):
        text[i].append(drew(i, text[i]))
        assert recent(dec, i) == text[i][-64:]
    for turn in range(14):
        start, new = list(dec.held), {i: [text[i][-1]] + rng.randint(0, 2048, 4).tolist() for i in range(3)}
        dec.extend(new)
        for i in range(3):
            last = drew(i, text[i])   # the drafts come in when it is said how many of them stay
            assert recent(dec, i) == (text[i] + [last])[-64:]
            if (turn + i) % 3 == 0:   # all
                dec.rewind(i, start[i] + 5)
                text[i] += new[i][1:] + [last]
            elif (turn + i) % 3 == 1:   # some, and the right one behind them
                dec.rewind(i, start[i] + 3, token=int(rng.randint(2048)))
                text[i] += new[i][1:3] + [int(dec.token[i])]
            else:   # some, and the right one with the next drafts
                dec.rewind(i, start[i] + 3)
                text[i] += new[i][1:3]
                assert recent(dec, i) == text[i][-64:]
                more = rng.randint(0, 2048, 2).tolist()
                dec.extend({i: more})
                assert recent(dec, i) == (text[i] + [drew(i, text[i])])[-64:]
                dec.rewind(i, start[i] + 4, token=7)
                text[i] += [more[0], 7]
            assert recent(dec, i) == text[i][-64:] and text[i][-1] == int(dec.token[i]) and dec.held[i] == int(dec.pos[i])
        if turn % 4 == 3:
            dec.step()
            for i in range(3):
                text[i].append(drew(i, text[i]))
                assert recent(dec, i) == text[i][-64:]
    dec.check_flags()


@pytest.mark.parametrize("graph", [False, True])
def test_steps_behind_drafts_taken_back(graph):
    import torch

    dec = make(1)
    dec.repetition_penalty = PENALTY
    text = ids(10, 1)
    dec.seed_window(text, 0)
    dec.prefill(ids(30, 2))
    text.append(int(dec.token[0]))
    dec.extend({0: [text[-1], 1, 2, 3]})
    step = dec.step
    if graph:
        dec.reserve(0, 200)
        dec.rewind(0, 33, token=4)
        dec.step()
        assert recent(dec, 0) == text + [1, 2, 4, int(dec.token[0])]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            dec.step()
        step = g.replay
        dec.rewind(0, 33)
        assert recent(dec, 0) == text + [1, 2]
        dec.extend({0: [3]})
    dec.rewind(0, 34)
    text += [1, 2, 3, int(dec.token[0])]
    assert recent(dec, 0) == text
    for _ in range(60):
        step()
        text.append(int(dec.token[0]))
        assert recent(dec, 0) == text[-64:]
    # text[11 + n - 31] stands at position n; 94 are held.  Steps are taken back, then drafts.
    for n in (90, 60, 35, 34, 33):
        dec.rewind(0, n)
        assert recent(dec, 0) == text[:n - 20][-64:], n
        if n in (60, 34):   # a token set by hand is not among them, nor does it stand in the way of the others
            dec.token[0] = 5
            step()
            after = int(dec.token[0])
            assert recent(dec, 0) == (text[:n - 20] + [after])[-64:]
    dec.extend({0: [8, 9]})
    dec.rewind(0, 34)
    text = text[:13] + [8]
    assert recent(dec, 0) == text
    # more steps than recent ids: those pushed out stay away, the rest is in order
    dec.rewind(0, 34, token=6)
    text.append(6)
    for _ in range(70):
        step()
        text.append(int(dec.token[0]))
        assert recent(dec, 0) == text[-64:]
    dec.rewind(0, 104 - 20)
    assert recent(dec, 0) == text[-64:-21]
    dec.check_flags()


def test_prompts_are_not_among_them():
    dec = make(2)
    dec.repetition_penalty = PENALTY
    dec.seed_window(ids(20, 1), 0)
    dec.prefill(ids(100, 1)), dec.extend({1: ids(90, 2)})
    assert recent(dec, 0)[:-1] == ids(20, 1) and len(recent(dec, 1)) == 1
    dec.rewind(0, 60), dec.rewind(1, 89)
    assert recent(dec, 0) == ids(20, 1) and recent(dec, 1) == []
    dec.rewind(1, 89, token=5)
    assert recent(dec, 1) == [5] and int(dec.token[1]) == 5
    dec.rewind(1, 89)
    assert recent(dec, 1) == [5]
    dec.release(1)
    dec.prefill(ids(10, 3), sequence=1)
    assert len(recent(dec, 1)) == 1 and not dec._given[1].drawn
    dec.reset()
    assert dec._given == {} and recent(dec, 0) == []


def test_without_a_penalty_there_are_none():
    dec = make(1)
    dec.extend({0: ids(20, 1)}), dec.extend({0: ids(4, 2)})
    dec.rewind(0, 22, token=9)
    assert recent(dec, 0) == [] and dec._given == {} and dec.token.tolist() == [9] and dec.held == dec.pos.tolist() == [22]
    for token in (-1, 2048):
        with pytest.raises(JoshuaB200Error):
            dec.rewind(0, 21, token=token)
    assert dec.held == [22]

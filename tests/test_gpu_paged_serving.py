"""The decoders over pages in the life of a server: sequences that end and begin again, host calls, callers' graphs, refusals.

Every decoder is compared with a twin that reached the same tokens by single steps or prompts of its own, in the same pieces, so that
the same rows go through the same kernels; page ids differ, and no result depends on them.  What is left are the sums of f32 that a
batch of another size takes in another order (1e-4 of a logit's size, as in the tests beside these).
"""
import numpy as np
import pytest

from joshua_b200._lib import JoshuaB200Error
from tests.test_gpu_paged_decoder import ids, make, near

pytestmark = pytest.mark.gpu


def whole(dec):
    """Every page is free or somebody's, none both; rows of the table name their owner's pages and no others."""
    owned = {p for mine in dec.owned for p in mine}
    assert sorted(owned | set(dec.free)) == list(range(dec.n_pages)) and not owned & set(dec.free) and len(set(dec.free)) == len(dec.free)
    for row, mine in zip(dec.table.tolist(), dec.owned):
        assert row[:len(mine)] == mine and not set(row[len(mine):]) & set(range(dec.n_pages))


def host_and_step(dec, twin, rows):
    """The same tokens by host calls and by steps."""
    import torch

    for row in rows:
        got = dec.forward_host(row)
        twin.token.copy_(torch.tensor(row, dtype=torch.int32))
        twin.step()
        near(torch.from_numpy(np.array(got)), twin.logits)


def tokens(n, batch, seed):
    return np.random.RandomState(seed).randint(0, 2048, (n, batch)).tolist()


def test_host_calls_behind_a_reset():
    """The pages of sequences that ended are others' by then."""
    dec, twin = make(2, max_ctx=256), make(2, max_ctx=256)
    dec.forward_host([1, 2])
    dec.reset()
    for d in (dec, twin):
        d.prefill(ids(130, 1), sequence=0)
        d.prefill(ids(10, 2), sequence=1)
    whole(dec)
    host_and_step(dec, twin, tokens(60, 2, 3))
    whole(dec)
    assert dec.held == [190, 70] and dec.pos.tolist() == [190, 70]
    dec.check_flags()


def test_a_prompt_behind_host_calls():
    dec, twin = make(2), make(2)
    dec.forward_host([5, 6])
    dec.reset()
    host_and_step(dec, twin, tokens(3, 2, 4))
    for d in (dec, twin):
        d.prefill(ids(70, 5), sequence=1)
    near(dec.logits[1], twin.logits[1])
    host_and_step(dec, twin, tokens(2, 2, 6))
    whole(dec)


def test_host_calls_to_the_last_position():
    dec = make(1, max_ctx=66)
    dec.prefill(ids(65, 1))
    dec.forward_host([3])
    assert dec.held == [66]
    with pytest.raises(JoshuaB200Error):
        dec.forward_host([4])
    with pytest.raises(RuntimeError):
        dec.forward_host([4, 5])       # refused before anything is counted
    dec.release(0)
    dec.prefill(ids(3, 1))
    for _ in range(63):                # the calls before the release do not count
        dec.forward_host([4])
    assert dec.held == [66] and dec.pos.tolist() == [66]
    dec.check_flags()


def test_a_released_row_names_no_page():
    dec = make(3, max_ctx=256)
    whole(dec)
    for i in range(3):
        dec.prefill(ids(100, i), sequence=i)
    dec.release(1)
    whole(dec)
    dec.prefill(ids(130, 7), sequence=1)
    whole(dec)
    dec.reset()
    whole(dec)


def test_host_calls_follow_the_shared_pages():
    """A common prompt, then prompts of each sequence's own, then a common one of another length."""
    dec, twin = make(3), make(3)
    for d in (dec, twin):
        d.share_prompt(ids(150, 1))
    host_and_step(dec, twin, tokens(2, 3, 2))
    for d in (dec, twin):
        d.reset()
        for i, n in enumerate((140, 10, 150)):
            d.prefill(ids(n, 3 + i), sequence=i)
    host_and_step(dec, twin, tokens(2, 3, 6))
    for d in (dec, twin):
        d.reset()
        d.share_prompt(ids(64, 7))
    host_and_step(dec, twin, tokens(2, 3, 8))
    dec.check_flags()


def test_host_calls_follow_the_sampling_rule():
    import torch

    dec = make(2)
    first = dict(top_k=torch.ones(2, dtype=torch.int32, device="cuda"))
    dec.sampling = first
    dec.uniform.fill_(0.999)
    logits = torch.from_numpy(np.array(dec.forward_host([1, 2])))
    assert dec.token.tolist() == logits.argmax(1).tolist()
    dec.sampling = dict(temperature=torch.full((2,), 1e4, device="cuda"))    # all ids alike: the draw tells the id
    dec.forward_host([3, 4])
    assert all(2048 * 0.998 < t for t in dec.token.tolist())
    dec.sampling["temperature"] = torch.zeros(2, device="cuda")
    logits = torch.from_numpy(np.array(dec.forward_host([5, 6])))
    assert dec.token.tolist() == logits.argmax(1).tolist()
    dec.sampling, dec.repetition_penalty = None, 1e6
    best = int(logits[0].argmax())
    dec.seed_window([best])
    dec.reset()
    dec.seed_window(list(range(2047)))       # the last 64 ids of it
    logits = torch.from_numpy(np.array(dec.forward_host([7, 8])))
    logits[:, 2047 - 64:2047] /= torch.where(logits[:, 2047 - 64:2047] > 0, 1e6, 1e-6)
    assert dec.token.tolist() == logits.argmax(1).tolist()
    assert dec.window_state.tolist() == [[64, 1]] * 2      # one id a call, the capture's own steps leave none


def test_a_step_that_finds_no_page():
    """It changes nothing, and can be tried again once pages are back."""
    prompts = [ids(64, 1), ids(70, 2), ids(64, 3)]
    dec, twin = make(3, max_ctx=256, n_pages=5), make(3, max_ctx=256)
    for i, p in enumerate(prompts):
        dec.prefill(p, sequence=i)
        twin.prefill(p, sequence=i)
    for call in (dec.step, lambda: dec.forward_host([1, 2, 3])):
        with pytest.raises(JoshuaB200Error):
            call()
        assert dec.held == [64, 70, 64] and len(dec.free) == 1 and dec.pos.tolist() == dec.held
        whole(dec)
    dec.release(1), twin.release(1)
    dec.token.copy_(twin.token)
    dec.step(), twin.step()
    assert dec.held[0] == dec.held[2] == 65
    dec.release(1)
    for d in (dec, twin):
        d.prefill(ids(20, 4), sequence=0)
    near(dec.logits[0], twin.logits[0])
    whole(dec)
    dec.check_flags()


def test_a_callers_graph_and_then_a_prompt():
    """Replays move the positions without the decoder's knowledge: what follows begins where they stand."""
    import torch

    dec, twin = make(2), make(2)
    for d in (dec, twin):
        for i in range(2):
            d.prefill(ids(60 + i, i), sequence=i)
            d.reserve(i, 200)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            dec.step()
        for row in tokens(5, 2, 9):
            dec.token.copy_(torch.tensor(row, dtype=torch.int32))
            graph.replay()
        side.synchronize()
    for row in tokens(5, 2, 9):
        twin.token.copy_(torch.tensor(row, dtype=torch.int32))
        twin.step()
    near(dec.logits, twin.logits)
    for d in (dec, twin):
        d.prefill(ids(30, 5), sequence=1)
    near(dec.logits[1], twin.logits[1])
    assert dec.pos.tolist() == twin.pos.tolist() == [65, 96]
    dec.token.copy_(twin.token)
    graph.replay(), graph.replay()
    torch.cuda.synchronize()
    dec.step()
    for _ in range(3):
        twin.step()
    near(dec.logits, twin.logits, 2e-2)      # tokens of their own now
    assert dec.pos.tolist() == twin.pos.tolist() and dec.held == twin.held


def test_a_host_call_waits_for_the_callers_stream():
    import torch

    dec = make(2)
    dec.sampling = dict(temperature=torch.full((2,), 1e4, device="cuda"))    # all ids alike: the draw tells the id
    dec.uniform.fill_(0.1)
    dec.forward_host([1, 2])
    torch.cuda._sleep(100_000_000)     # some 50 ms of work in front of the next numbers
    dec.uniform.fill_(0.9)
    dec.forward_host([1, 2])
    assert all(abs(t - 0.9 * 2048) < 10 for t in dec.token.tolist())


def test_equal_logits_in_a_prompt_as_in_a_step():
    """Without a sampling rule the last of equal maxima is taken, for one row of a batch too."""
    import torch

    from joshua_b200 import synth

    def weights(name, rows, cols, seed):
        if name != "output":
            return synth.random_weight_torch(synth.Q8_0, rows, cols, seed, torch.device("cuda", 0))
        half = synth.random_weight_torch(synth.Q8_0, rows // 2, cols, seed, torch.device("cuda", 0))
        return torch.cat([half, half])     # every id has a twin 1024 further on

    dec = make(3, weights=weights)
    dec.prefill(ids(20, 1), sequence=1)
    assert bool((dec.logits[1, :1024] == dec.logits[1, 1024:]).all())
    best = int(dec.logits[1, 1024:].argmax()) + 1024
    assert int(dec.token[1]) == best
    dec.repetition_penalty = 2.0
    dec.prefill(ids(20, 2), sequence=2)
    assert int(dec.token[2]) == int(dec.logits[2, 1024:].argmax()) + 1024 and dec.window_state.tolist() == [[0, 0], [0, 0], [1, 1]]
    dec.step()
    assert bool((dec.token >= 1024).all()) and dec.pos.tolist() == [1, 21, 21]


@pytest.mark.parametrize("ruled", [False, True])
def test_a_slot_that_is_used_again_forgets_its_ids(ruled):
    import torch

    dec, fresh = make(2), make(2)
    for d in (dec, fresh):
        d.repetition_penalty = 1e6
        if ruled:
            d.sampling = dict(top_k=torch.ones(2, dtype=torch.int32, device="cuda"))
    fresh.prefill(ids(40, 1), sequence=0)
    dec.prefill(ids(10, 2), sequence=1)
    dec.prefill(ids(40, 1), sequence=0)      # its token goes into the window
    assert int(dec.token[0]) == int(fresh.token[0])
    kept = dec.window[1].clone(), dec.window_state[1].clone()
    dec.release(0)
    dec.prefill(ids(40, 1), sequence=0)
    assert int(dec.token[0]) == int(fresh.token[0])
    assert torch.equal(dec.window[1], kept[0]) and torch.equal(dec.window_state[1], kept[1])
    dec.release(0)
    dec.seed_window([int(fresh.token[0])], sequence=0)
    dec.prefill(ids(40, 1), sequence=0)
    assert int(dec.token[0]) == int(dec.logits[0].topk(2).indices[1])
    assert torch.equal(dec.window[1], kept[0]) and torch.equal(dec.window_state[1], kept[1])


def test_sequences_that_are_not_there():
    dec = make(2)
    for i in (-1, 2, -3):
        for call in (lambda: dec.prefill(ids(5, 1), sequence=i), lambda: dec.reserve(i, 10), lambda: dec.release(i)):
            with pytest.raises(JoshuaB200Error):
                call()
    assert dec.held == [0, 0] and len(dec.free) == dec.n_pages
    dec.prefill(ids(5, 1), sequence=1)
    dec.check_flags()


def test_a_common_prompt_keeps_what_was_reserved():
    dec, plain = make(3, max_ctx=320), make(3, max_ctx=320)
    dec.reserve(0, 30), dec.reserve(1, 250), dec.reserve(2, 70)
    for d in (dec, plain):
        d.share_prompt(ids(150, 1))
        whole(d)
    assert [len(mine) for mine in dec.owned] == [3, 4, 3] and len(dec.free) == 15 - 2 - 1 - 2 - 1
    dec.step(), plain.step()
    near(dec.logits, plain.logits)
    dec.reset()
    assert len(dec.free) == 15


def test_a_common_prompt_that_does_not_fit():
    dec = make(4, max_ctx=320, n_pages=5)       # two common pages and four of the rest
    with pytest.raises(JoshuaB200Error):
        dec.share_prompt(ids(150, 1))
    assert len(dec.free) == 5 and dec.held == [0] * 4 and dec.pos.tolist() == [0] * 4
    whole(dec)
    dec.share_prompt(ids(120, 1))               # one and four
    assert dec.free == [] and dec.shared_pages == 1


@pytest.mark.parametrize("ruled", [False, True])
def test_a_sequence_rests(ruled):
    """From its release to its next prompt a sequence takes no pages and does not hinder the others."""
    import torch

    dec, twin = make(3, max_ctx=200), make(2, max_ctx=200)
    for d, at in ((dec, (0, 2)), (twin, (0, 1))):
        d.repetition_penalty = 1.3
        if ruled:
            d.sampling = dict(top_k=torch.ones(d.batch, dtype=torch.int32, device="cuda"))
        for i, n in zip(at, (100, 30)):
            d.prefill(ids(n, n), sequence=i)
    dec.prefill(ids(197, 5), sequence=1)
    dec.release(1)
    free = len(dec.free)
    for row in tokens(70, 2, 1):
        dec.token.copy_(torch.tensor([row[0], 0, row[1]], dtype=torch.int32))
        twin.token.copy_(torch.tensor(row, dtype=torch.int32))
        dec.step(), twin.step()
    near(dec.logits[::2], twin.logits, 2e-2)
    assert dec.held == [170, 0, 100] and len(dec.free) == free - 2 and dec.owned[1] == []
    dec.check_flags()
    whole(dec)
    dec.release(0), twin.release(0)
    for d, i in ((dec, 1), (twin, 0)):                # another prompt in the slot: from position 0 on
        d.seed_window([1, 2, 3], sequence=i)
        d.step()                                      # the ids given stay while it rests
        d.prefill(ids(40, 6), sequence=i)
    near(dec.logits[1], twin.logits[0])
    assert dec.held[1] == 40 and int(dec.token[1]) == int(twin.token[0]) and dec.window_state[1].tolist() == [4, 4]
    assert dec.window[1, :3].tolist() == [1, 2, 3]
    dec.release(2), dec.release(1)
    dec.step()                                        # all of them rest
    assert dec.held == [0, 0, 0] and len(dec.free) == dec.n_pages
    dec.check_flags()


def test_a_graph_and_the_host_call_leave_resting_sequences_alone():
    import torch

    dec = make(3, max_ctx=130)
    for i in range(3):
        dec.prefill(ids(20 + i, i), sequence=i)
        dec.reserve(i, 130)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        dec.step()
        with torch.cuda.graph(graph, stream=side):
            dec.step()
        side.synchronize()
    dec.release(1)
    for _ in range(100):
        graph.replay()
    torch.cuda.synchronize()
    assert dec.pos[[0, 2]].tolist() == [121, 123]
    dec.check_flags()
    for _ in range(3):
        dec.forward_host([1, 2, 3])
    assert dec.held == [124, 0, 126] and dec.owned[1] == []
    dec.check_flags()
    whole(dec)


def test_many_resting_sequences():
    """More of them than a page has positions."""
    dec = make(70, max_ctx=64)
    for i in range(1, 70):
        dec.release(i)
    dec.prefill(ids(5, 1))
    dec.step()
    assert len(dec.free) == 69 and dec.held == [6] + [0] * 69
    dec.check_flags()


def test_a_prompt_stays_common_while_others_end():
    dec, twin = make(4), make(4)
    for d in (dec, twin):
        d.share_prompt(ids(150, 1))
        d.release(2)
    assert dec.shared_pages == 2 and len(dec.free) == 20 - 2 - 3
    twin.shared_pages = 0
    for row in tokens(2, 4, 3):
        for d in (dec, twin):
            d.token.copy_(__import__("torch").tensor(row, dtype=d.token.dtype))
            d.step()
    live = [0, 1, 3]
    near(dec.logits[live], twin.logits[live])
    for d in (dec, twin):
        d.prefill(ids(30, 4), sequence=2)
        d.step()
    assert dec.shared_pages == 0
    near(dec.logits, twin.logits, 2e-2)
    dec.reset()
    dec.share_prompt(ids(150, 1))
    dec.release(0)                   # the common pages are found through the first sequence
    assert dec.shared_pages == 0
    dec.step()
    dec.check_flags()
    whole(dec)


def test_taking_pages_waits_for_nothing():
    import torch

    dec = make(4)
    for i in range(4):
        dec.prefill(ids(64, i), sequence=i)
    dec.step()
    for i in range(4):
        dec.release(i)
        dec.prefill(ids(64, i), sequence=i)
    torch.cuda.synchronize()
    torch.cuda._sleep(600_000_000)     # some 300 ms
    end = torch.cuda.Event()
    end.record()
    dec.step()                         # a page of each sequence
    assert not end.query() and dec.held == [65] * 4 and [len(mine) for mine in dec.owned] == [2] * 4
    whole(dec)
    dec.check_flags()


def test_one_scratch_for_all_layers():
    """Growing it leaves a graph of before as it was."""
    import torch

    dec, twin = make(70, max_ctx=2600), make(70, max_ctx=2600)
    for d in (dec, twin):
        for i in range(70):
            d.prefill(ids(3, i), sequence=i)
            d.reserve(i, 10)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        dec.step()                  # what a step needs on this stream is there before the capture
        with torch.cuda.graph(graph, stream=side):
            dec.step()
        side.synchronize()
    small = dec.att_scratch[-1].numel()
    for d in (dec, twin):
        d.reset()
        d.share_prompt(ids(2500, 1))
    host_and_step(dec, twin, tokens(2, 70, 2))
    assert dec.att_scratch[-1].numel() > small
    for d in (dec, twin):
        d.reset()
        for i in range(70):
            d.prefill(ids(3, i), sequence=i)
            d.reserve(i, 10)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay(), graph.replay()
        side.synchronize()
    twin.step(), twin.step()
    near(dec.logits, twin.logits)
    dec.check_flags()

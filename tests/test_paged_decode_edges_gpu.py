"""Decoding over a paged cache where something goes wrong: rows without a token,
calls that raise, steps without a page."""

import pytest
import torch

from persona import ops
from persona.engine import Request, StaticBatchEngine
from persona.sampling import BatchSampling, SamplingParams, sample_batch, sample_next_token
from test_decode_gpu import CFG, _dev, _small_model
from test_paged_decode_gpu import E4M3, _generator, _prompts

pytestmark = pytest.mark.gpu
SAMPLED = [SamplingParams(temperature=0.8, top_p=0.9), SamplingParams(temperature=1.2, top_k=30), SamplingParams()]


def _start(model, pool, prompts, params=SAMPLED, pages=40, seed=3, **kv):
    slots = torch.tensor([pool.name_to_slot["a0"], -1, pool.name_to_slot["a2"]], dtype=torch.int32)
    st = model.new_paged_state(slots, pages, 16, 160, **kv)
    sampling = BatchSampling(params, _dev())
    g = _generator(seed)
    logits, ip = model.extend(st, prompts)
    first = sample_batch(logits[ip[1:].long() - 1], sampling, generator=g)
    return model.start_decode(st, first, sampling), first.tolist(), g


def _unused(seen):
    return next(t for t in range(CFG.vocab) if t not in seen)


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("kv", [dict(), dict(kv_dtype=E4M3, kv_block=16)])
def test_a_row_without_a_token_ends_its_sequence(use_graph, kv):
    """A token whose embedding is NaN leaves its row no logit to draw from.  The
    other sequences, which take the pages over that it filled with NaN, go on as
    they do alone."""
    pool, model = _small_model()
    prompts = _prompts([20, 33, 16], 21)

    def run(end, poison=None):
        dec, first, g = _start(model, pool, prompts, **kv)
        rows = [first]
        for i in range(40):
            if i == 6 and poison is not None:
                dec.tok[1] = poison
            if i == end:
                dec.alive[1] = 0
            rows.append(model.paged_step(dec, use_graph=use_graph, generator=g).tolist())
        model.finish_decode(dec)
        return dec.st, [list(c) for c in zip(*rows)]

    st, clean = run(7)
    nan = _unused(sum(clean, sum(prompts, [])))
    model.embed[nan] = float("nan")
    ended, got = run(None, nan)
    assert got[0] == clean[0] and got[2] == clean[2]
    assert got[1][:7] == clean[1][:7] and got[1][7:] == [-1] * 34
    assert (ended.lengths, ended.pages, ended.free) == (st.lengths, st.pages, st.free)
    assert ended.lengths == [60, 0, 56]


def test_a_prompt_without_a_token_ends_at_once():
    """-1 is what ``sample_batch`` hands to ``start_decode`` then."""
    pool, model = _small_model()
    prompts = _prompts([20, 33, 16], 22)
    nan = _unused(sum(prompts, []))
    model.embed[nan] = float("nan")
    prompts[0][-1] = nan
    dec, first, g = _start(model, pool, prompts)
    assert first[0] == -1 and min(first[1:]) >= 0
    for _ in range(3):
        got = model.paged_step(dec, generator=g).tolist()
        assert got[0] == -1 and min(got[1:]) >= 0
    model.finish_decode(dec)
    assert dec.st.lengths == [0, 36, 19] and dec.st.pages[0] == []
    for bad in (CFG.vocab, -2):
        with pytest.raises(ValueError, match="outside the vocabulary"):
            model.start_decode(dec.st, torch.tensor([1, bad, 2], device=_dev()), dec.sampling)
    # a token that was put there from outside ends its sequence too, whatever it is
    dec = model.start_decode(dec.st, torch.tensor([1, 2, 3], device=_dev()), dec.sampling)
    dec.tok[1] = 1 << 40
    got = model.paged_step(dec, generator=g).tolist()
    assert got[1] == 1 << 40 and min(got[0], got[2]) >= 0
    model.finish_decode(dec)
    assert dec.st.lengths == [1, 0, 20]


def test_ragged_generation_of_a_request_without_a_token():
    pool, model = _small_model()
    eng = StaticBatchEngine(model, pool, max_batch=4, max_seq_len=256)
    prompts = _prompts([5, 40, 12], 23)
    nan = _unused(sum(prompts, []))
    reqs = [Request(f"r{i}", "a", p, slot=i, sampling=SamplingParams()) for i, p in enumerate(prompts)]
    clean = eng.run_ragged_generate(reqs, 12)
    assert nan not in sum(clean["tokens"], [])
    model.embed[nan] = float("nan")
    reqs[1].prompt = prompts[1][:-1] + [nan]
    got = eng.run_ragged_generate(reqs, 12)
    assert got["tokens"] == [clean["tokens"][0], [], clean["tokens"][2]] and got["new_tokens"] == 24
    ops.check_errors(_dev())


@pytest.mark.parametrize("params", [SamplingParams(), SamplingParams(temperature=1.0), SamplingParams(temperature=1.0, top_p=0.9),
                                    SamplingParams(temperature=1.0, top_k=5), SamplingParams(temperature=1.0, min_p=0.1),
                                    SamplingParams(temperature=0.7, top_k=5, top_p=0.9, min_p=0.1)])
def test_next_tokens_are_always_of_the_vocabulary(params):
    """``sample_next_token`` feeds the static engine's embedding."""
    logits = torch.randn(4, 300, device=_dev(), generator=_generator(2)).half()
    logits[1] = float("nan")
    logits[2] = -float("inf")
    got = sample_next_token(logits, params, generator=_generator(3)).tolist()
    assert all(0 <= t < 300 for t in got)
    assert got[1] == int(logits[1].argmax())


def test_static_generation_of_a_request_without_a_token():
    pool, model = _small_model()
    eng = StaticBatchEngine(model, pool, max_batch=4, max_seq_len=64)
    prompts = _prompts([12, 12, 12], 24)
    nan = _unused(sum(prompts, []))
    prompts[1][-1] = nan
    model.embed[nan] = float("nan")
    reqs = [Request(f"r{i}", "a", p, slot=i, sampling=SamplingParams(temperature=1.0, top_k=4)) for i, p in enumerate(prompts)]
    out = eng.run_static_generate(reqs, 6)["tokens"]
    ops.check_errors(_dev())
    assert 0 <= int(out.min()) and int(out.max()) < CFG.vocab


def _state(dec):
    return [t.tolist() for t in (dec.tok[:3], dec.alive, dec.lengths, dec.st.page_table, dec.num_free, dec.free[:int(dec.num_free)])]


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")  # (what a capture that raises leaves)
@pytest.mark.parametrize("use_graph,calls", [(False, 1), (True, 1), (True, 2)])
@pytest.mark.parametrize("behind", [True, False])
def test_a_step_that_raises_leaves_the_sequences(monkeypatch, use_graph, calls, behind):
    """The step raises on the host, before or behind its operators: the eager
    one, the warm-up before a capture, or the capture.  Made again, it gives the
    tokens of a step that never failed."""
    pool, model = _small_model()
    prompts = _prompts([20, 32, 16], 25)
    greedy = [SamplingParams()] * 3
    kv = dict(kv_dtype=E4M3, kv_block=16)
    clean, _, _ = _start(model, pool, prompts, greedy, **kv)
    want = [model.paged_step(clean, use_graph=use_graph).tolist() for _ in range(4)]
    dec, _, _ = _start(model, pool, prompts, greedy, **kv)
    if not use_graph:
        assert model.paged_step(dec, use_graph=False).tolist() == want[0]
    before, body, left = _state(dec), model._paged_body, [calls]

    def failing(d):
        left[0] -= 1
        if left[0] == 0 and not behind:
            raise RuntimeError("on the host")
        body(d)
        if left[0] == 0:
            raise RuntimeError("on the host")

    monkeypatch.setattr(model, "_paged_body", failing)
    with pytest.raises(RuntimeError, match="on the host"):
        model.paged_step(dec, use_graph=use_graph)
    monkeypatch.undo()
    assert _state(dec) == before and dec.graph is None
    for w in want[0 if use_graph else 1:]:
        assert model.paged_step(dec, use_graph=use_graph).tolist() == w
    model.finish_decode(dec)
    assert dec.st.lengths == [24, 36, 20]
    ops.check_errors(_dev())


def _leave_an_error():
    """A step that finds no page, over buffers of its own."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=_dev())  # noqa: E731
    ops.paged_plan(i32(1), i32(0), i32(0).view(1, 1), i32(0), i32(0), 16, i32(0, 0),
                   torch.zeros(1, dtype=torch.int64, device=_dev()))
    torch.cuda.synchronize()


@pytest.mark.parametrize("use_graph", [True, False])
def test_an_error_from_before_costs_no_sequence(use_graph):
    """What an earlier operator left pending is raised by the first step."""
    pool, model = _small_model()
    prompts = _prompts([20, 32, 16], 26)
    greedy = [SamplingParams()] * 3
    clean, _, _ = _start(model, pool, prompts, greedy)
    want = [model.paged_step(clean, use_graph=use_graph).tolist() for _ in range(3)]
    dec, _, _ = _start(model, pool, prompts, greedy)
    before = _state(dec)
    _leave_an_error()
    with pytest.raises(RuntimeError, match="no room for a planned step"):
        model.paged_step(dec, use_graph=use_graph)
    assert _state(dec) == before
    assert [model.paged_step(dec, use_graph=use_graph).tolist() for _ in range(3)] == want
    model.finish_decode(dec)
    assert dec.st.lengths == [23, 35, 19]


@pytest.mark.parametrize("use_graph", [True, False])
def test_a_decode_that_ended_moves_nothing(use_graph):
    """Its sequences' pages are the host's, or another decode's."""
    pool, model = _small_model()
    dec, _, _ = _start(model, pool, _prompts([20, 32, 16], 27))
    model.paged_step(dec, use_graph=use_graph)
    model.finish_decode(dec)
    st = dec.st
    st.set_length(1, 0)
    model.extend(st, [[5] * 30, [], []])
    table, k = st.page_table.clone(), [c.clone() for c in st.k_cache]
    for again in (False, True):
        other = model.start_decode(st, torch.tensor([1, 2, 3], device=_dev()), dec.sampling) if again else None
        with pytest.raises(ValueError, match="not the sequences' own"):
            model.paged_step(dec, use_graph=use_graph)
        assert st.decode is other and torch.equal(st.page_table, table)
        assert all(torch.equal(a, b) for a, b in zip(st.k_cache, k))
    model.paged_step(st.decode, use_graph=use_graph)
    model.finish_decode(st.decode)
    assert st.lengths == [52, 1, 18]


@pytest.mark.parametrize("use_graph", [True, False])
def test_a_step_without_pages_gives_no_tokens(use_graph):
    """Two sequences need a page and one is free: no token for anybody, an error
    with the next step, and the old tokens once there is room."""
    pool, model = _small_model()
    prompts, greedy = _prompts([31, 31, 14], 28), [SamplingParams()] * 3
    clean, first, _ = _start(model, pool, prompts, greedy)
    want = [first] + [model.paged_step(clean, use_graph=use_graph).tolist() for _ in range(6)]
    dec, _, _ = _start(model, pool, prompts, greedy, pages=6)
    assert model.paged_step(dec, use_graph=use_graph).tolist() == want[1]
    before = _state(dec)
    assert before[2] == [32, 32, 15] and before[0] == want[1]
    for _ in range(3):
        with pytest.raises(RuntimeError, match="no room for a planned step"):
            for _ in range(2):  # (operators of an eager step may see it before the step is through)
                assert model.paged_step(dec, use_graph=use_graph).tolist() == [-1] * 3
        assert _state(dec) == before
    dec.alive[0] = 0
    for w in want[2:]:
        assert model.paged_step(dec, use_graph=use_graph).tolist() == [want[1][0]] + w[1:]
    model.finish_decode(dec)
    assert dec.st.lengths == [0, 37, 20]


@pytest.mark.parametrize("use_graph", [True, False])
def test_ragged_generation_with_too_few_pages_raises(use_graph):
    """The loop does not wait for its steps: nothing of those behind the one
    without a page is left for later calls."""
    pool, model = _small_model()
    eng = StaticBatchEngine(model, pool, max_batch=4, max_seq_len=256)
    reqs = [Request(f"r{i}", "a", p, slot=i, sampling=SamplingParams()) for i, p in enumerate(_prompts([15, 15], 29))]
    with pytest.raises(RuntimeError, match="no room for a planned step"):
        eng.run_ragged_generate(reqs, 100, use_graph, num_pages=3)
    ops.check_errors(_dev())
    got = eng.run_ragged_generate(reqs, 10, use_graph, num_pages=4)["tokens"]
    assert [len(t) for t in got] == [10, 10]

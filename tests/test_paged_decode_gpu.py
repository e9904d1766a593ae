"""Decoding over a paged cache without the host: the captured step of the small
model (plan, write, attention, sampling) and the engine's ragged generation."""

import pytest
import torch

from persona import ops
from persona.engine import Request, StaticBatchEngine
from persona.sampling import BatchSampling, SamplingParams, sample_batch, sample_next_token, verify_drafts
from test_decode_gpu import CFG, _dev, _reference_logits, _small_model

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _prompts(lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, CFG.vocab, (n,), generator=g).tolist() for n in lens]


def _generator(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _decode(model, pool, prompts, params, steps, use_graph=True, seed=0, end=None, kv=dict(), pages=40):
    slots = torch.tensor([pool.name_to_slot["a0"], -1, pool.name_to_slot["a2"]], dtype=torch.int32)
    st = model.new_paged_state(slots, pages, 16, 160, **kv)
    sampling = BatchSampling(params, _dev())
    g = _generator(seed)
    logits, ip = model.extend(st, prompts)
    tok = sample_batch(logits[ip[1:].long() - 1], sampling, generator=g)
    dec = model.start_decode(st, tok, sampling)
    out = [tok.tolist()]
    for i in range(steps):
        for b in [b for b in (end or {}) if end[b] == i]:
            dec.alive[b] = 0
        out.append(model.paged_step(dec, use_graph=use_graph, generator=g).tolist())
    model.finish_decode(dec)
    return st, [list(c) for c in zip(*out)]


@pytest.mark.parametrize("kv,bound", [(dict(), 0.03), (dict(kv_dtype=E4M3), 0.12), (dict(kv_dtype=E4M3, kv_block=16), 0.12),
                                      (dict(kv_dtype=E4M3, kv_block=4), 0.12)])
def test_greedy_tokens_are_the_reference_models(kv, bound):
    """Teacher-forced with the tokens that were drawn, every one is within the
    paged path's bound (twice: its own logit and the largest one's) of the fp32
    reference's largest logit."""
    pool, model = _small_model()
    prompts = _prompts([30, 1, 77], 5)
    st, got = _decode(model, pool, prompts, [SamplingParams()] * 3, 40, kv=kv)
    ops.check_errors(_dev())
    assert st.lengths == [70, 41, 117]
    for b, slot in enumerate([pool.name_to_slot["a0"], -1, pool.name_to_slot["a2"]]):
        seq = prompts[b] + got[b][:-1]
        ref = _reference_logits(model, pool, torch.tensor([seq], device=_dev()), [slot])[0][len(prompts[b]) - 1:]
        mine = ref.gather(1, torch.tensor(got[b], device=_dev())[:, None])[:, 0]
        assert torch.all(mine >= ref.amax(-1) - 2 * bound * ref.abs().max())


def test_graph_and_eager_steps_give_the_same_tokens():
    pool, model = _small_model()
    prompts = _prompts([3, 50, 17], 6)
    params = [SamplingParams(temperature=0.8, top_p=0.9), SamplingParams(temperature=1.2, top_k=30),
              SamplingParams(temperature=1.0, min_p=0.05, top_k=50, top_p=0.95)]
    end = {1: 7}
    a, ta = _decode(model, pool, prompts, params, 25, True, 3, end, dict(kv_dtype=E4M3, kv_block=16))
    b, tb = _decode(model, pool, prompts, params, 25, False, 3, end, dict(kv_dtype=E4M3, kv_block=16))
    assert ta == tb and (a.lengths, a.pages, a.free) == (b.lengths, b.pages, b.free)
    assert len(set(ta[1][8:])) == 1  # ended: its token stays
    assert a.lengths == [28, 0, 42] and a.pages[1] == [] and len(a.free) == 40 - 2 - 3
    _, other = _decode(model, pool, prompts, params, 25, True, 4, end, dict(kv_dtype=E4M3, kv_block=16))
    assert other != ta
    # who else is alive changes no sequence's numbers
    _, alone = _decode(model, pool, prompts, params, 25, True, 3, None, dict(kv_dtype=E4M3, kv_block=16))
    assert alone[0] == ta[0] and alone[2] == ta[2]


def test_the_host_goes_on_where_the_device_stopped():
    pool, model = _small_model()
    prompts = _prompts([20, 31, 16], 7)
    st, got = _decode(model, pool, prompts, [SamplingParams()] * 3, 10)
    held = sorted(sum(st.pages, st.free))
    assert held == list(range(40))
    logits, ip = model.extend(st, [[got[b][-1]] for b in range(3)])
    assert st.lengths == [31, 42, 27]
    for b, slot in enumerate([pool.name_to_slot["a0"], -1, pool.name_to_slot["a2"]]):
        seq = prompts[b] + got[b]
        ref = _reference_logits(model, pool, torch.tensor([seq], device=_dev()), [slot])[0][-1]
        torch.testing.assert_close(logits[b].float(), ref, rtol=0, atol=0.03 * ref.abs().max().item())
    sampling = BatchSampling([SamplingParams()] * 3, _dev())
    dec = model.start_decode(st, logits.argmax(-1), sampling)
    for call in (lambda: model.extend(st, [[1], [], []]), lambda: st.set_length(0, 3),
                 lambda: model.start_decode(st, logits.argmax(-1), sampling)):
        with pytest.raises(ValueError, match="being decoded"):
            call()
    model.paged_step(dec)
    model.finish_decode(dec)
    assert st.lengths == [32, 43, 28]
    with pytest.raises(ValueError, match="not the sequences' own"):
        model.finish_decode(dec)


def test_pages_that_run_out_stop_the_steps():
    pool, model = _small_model()
    prompts = _prompts([16, 16, 15], 8)
    with pytest.raises(RuntimeError, match="no room for a planned step"):
        _decode(model, pool, prompts, [SamplingParams()] * 3, 4, pages=4)
    ops.check_errors(_dev())


def test_ragged_generation():
    pool, model = _small_model()
    eng = StaticBatchEngine(model, pool, max_batch=4, max_seq_len=256)
    lens, budgets = [5, 40, 12, 1], [20, 3, 128, 1]
    params = [SamplingParams(max_tokens=budgets[0]), SamplingParams(temperature=0.9, top_k=1, max_tokens=budgets[1]),
              SamplingParams(temperature=1.0, top_p=0.9), SamplingParams(max_tokens=budgets[3])]
    reqs = [Request(f"r{i}", "a", p, slot=s, sampling=q) for i, (p, s, q) in
            enumerate(zip(_prompts(lens, 9), [0, -1, 1, 2], params))]
    a = eng.run_ragged_generate(reqs, 30, generator=_generator(1))
    assert [len(t) for t in a["tokens"]] == [20, 3, 30, 1] and a["new_tokens"] == 54
    b = eng.run_ragged_generate(reqs, 30, use_cuda_graph=False, generator=_generator(1))
    assert a["tokens"] == b["tokens"]
    c = eng.run_ragged_generate(reqs, 30, kv_dtype=E4M3, kv_block=16, generator=_generator(1))
    assert [len(t) for t in c["tokens"]] == [20, 3, 30, 1]
    for bad in ([], [Request("x", "a", [])], [Request("x", "a", [1], sampling=SamplingParams(max_tokens=0))]):
        with pytest.raises(ValueError, match="a prompt and a budget"):
            eng.run_ragged_generate(bad, 5)
    with pytest.raises(ValueError, match="exceed"):
        eng.run_ragged_generate(reqs[:1], 300) if budgets[0] > 256 else eng.run_ragged_generate(
            [Request("x", "a", [1] * 250)], 30)
    for kw in (dict(kv_block=16), dict(kv_dtype=E4M3, kv_block=3), dict(kv_dtype=E4M3, kv_block=32)):
        with pytest.raises(ValueError, match="kv_block"):
            eng.run_ragged_generate(reqs, 5, **kw)


def test_static_batches_with_top_k_and_min_p():
    """``sample_next_token`` with the new parameters; what it draws without them is untouched."""
    g = torch.Generator(device=_dev()).manual_seed(4)
    logits = torch.randn(64, 500, device=_dev(), generator=g) * 3
    k = sample_next_token(logits, SamplingParams(temperature=1.0, top_k=4), generator=g)
    inside = (logits > logits.topk(4).values[:, -1:]) | (logits == logits.topk(4).values[:, -1:])
    assert inside[torch.arange(64, device=_dev()), k].all() and (k != logits.argmax(-1)).any()
    m = sample_next_token(logits, SamplingParams(temperature=1.0, min_p=0.5), generator=g)
    p = torch.softmax(logits.double(), -1)
    assert torch.all(p.gather(1, m[:, None])[:, 0] >= 0.5 * p.amax(-1) * (1 - 1e-6))
    assert torch.equal(sample_next_token(logits, SamplingParams(top_k=9)), logits.argmax(-1))
    with pytest.raises(ValueError, match="temperature and top_p"):
        verify_drafts(logits, torch.zeros(64, dtype=torch.int64, device=_dev()), None,
                      torch.tensor([0, 64], dtype=torch.int32, device=_dev()), SamplingParams(temperature=1.0, top_k=3))

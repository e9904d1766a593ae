"""The small Mistral-architecture model over a paged cache: ragged chunks
against the fp32 reference of the whole network, cut-back drafts, 8-bit pages,
and speculative decoding that gives the greedy decode's tokens."""

import pytest
import torch

from persona import ops
from persona.sampling import SamplingParams, verify_drafts
from test_decode_gpu import CFG, _dev, _reference_logits, _small_model

pytestmark = pytest.mark.gpu


def _seqs(lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, CFG.vocab, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("kv_dtype,bound", [(torch.float16, 0.03), (torch.float8_e4m3fn, 0.12)])
def test_ragged_chunks_match_the_fp32_reference(kv_dtype, bound):
    """Three sequences of different lengths in three uneven chunks; logits of
    every row.  fp16: the bound of the dense path's test (0.03 of the largest
    logit).  8-bit pages: k and v are off by up to 2^-4 each, so the bound is
    that plus 2^-4 of a layer's attention for each of the two (0.03 + 0.09)."""
    pool, model = _small_model()
    slots = [pool.name_to_slot["a0"], -1, pool.name_to_slot["a2"]]
    seqs = _seqs([45, 7, 90], 1)
    cuts = [[20, 21, 45], [0, 7, 7], [64, 70, 90]]
    st = model.new_paged_state(torch.tensor(slots, dtype=torch.int32), num_pages=16, page_size=16, max_seq=128,
                               kv_dtype=kv_dtype)
    got = [[] for _ in seqs]
    at = [0, 0, 0]
    for step in range(3):
        chunks = [s[a:c[step]] for s, a, c in zip(seqs, at, cuts)]
        logits, indptr = model.extend(st, chunks)
        ip = indptr.tolist()
        for b in range(3):
            got[b].append(logits[ip[b]:ip[b + 1]].float())
        at = [c[step] for c in cuts]
    ops.check_errors(_dev())
    assert st.lengths == [45, 7, 90] and len(st.free) == 16 - 3 - 1 - 6
    for b, s in enumerate(seqs):
        ref = _reference_logits(model, pool, torch.tensor([s], device=_dev()), [slots[b]])[0]
        torch.testing.assert_close(torch.cat(got[b]), ref, rtol=0, atol=bound * ref.abs().max().item())


def test_pages_run_out_and_come_back():
    pool, model = _small_model()
    st = model.new_paged_state(torch.tensor([-1, -1], dtype=torch.int32), num_pages=3, page_size=16, max_seq=32)
    model.extend(st, [[1] * 17, [2] * 3])
    assert not st.free
    with pytest.raises(ValueError, match="no free pages"):
        model.extend(st, [[], [3] * 14])
    with pytest.raises(ValueError, match="outgrows"):
        model.extend(st, [[1] * 16, []])
    assert st.lengths == [17, 3]
    st.set_length(0, 16)
    assert len(st.free) == 1
    model.extend(st, [[], [3] * 14])
    with pytest.raises(ValueError, match="cut back"):
        st.set_length(0, 99)
    logits, indptr = model.extend(st, [[], []])
    assert logits.shape == (0, CFG.vocab) and indptr.tolist() == [0, 0, 0]


def test_speculative_decode_gives_the_greedy_tokens():
    """Drafts of mixed quality, verified greedily, against one token a step."""
    pool, model = _small_model()
    slots = torch.tensor([pool.name_to_slot["a0"], pool.name_to_slot["a1"]], dtype=torch.int32)
    prompts = _seqs([13, 29], 2)
    steps = 12

    def start():
        st = model.new_paged_state(slots, num_pages=32, page_size=16, max_seq=128)
        logits, ip = model.extend(st, prompts)
        ends = [int(i) - 1 for i in ip[1:]]
        return st, [int(logits[e].argmax()) for e in ends], logits[ends].float()

    st, last, _ = start()
    plain = [[t] for t in last]
    for _ in range(steps):
        logits, _ = model.extend(st, [[p[-1]] for p in plain])
        for b in range(2):
            plain[b].append(int(logits[b].argmax()))
    st, last, _ = start()
    spec = [[t] for t in last]
    rounds = 0
    while min(len(s) for s in spec) <= steps:
        drafts = []
        for b in range(2):
            ahead = plain[b][len(spec[b]):len(spec[b]) + 3]  # what a good draft would say
            if rounds % 3 == 2:
                ahead = [(t + 1) % CFG.vocab for t in ahead]  # and a bad one
            drafts.append(ahead)
        before = list(st.lengths)
        logits, ip = model.extend(st, [[s[-1]] + d for s, d in zip(spec, drafts)])
        judged = torch.tensor([t for d in drafts for t in d + [0]], device=_dev())
        tokens, acc = verify_drafts(logits, judged, None, ip, SamplingParams(temperature=0.0))
        for b in range(2):
            a, r0 = int(acc[b]), int(ip[b])
            assert rounds % 3 == 2 or a >= min(1, len(drafts[b]))
            spec[b] += tokens[r0:r0 + a + 1].tolist()
            st.set_length(b, before[b] + 1 + a)
        rounds += 1
    ops.check_errors(_dev())
    for b in range(2):
        assert spec[b][:steps] == plain[b][:steps]


def test_verify_drafts_probabilities():
    """temperature and top-p as in sample_next_token: tokens outside the
    nucleus are never kept or drawn."""
    g = torch.Generator(device=_dev()).manual_seed(4)
    logits = torch.randn(64, 50, device=_dev(), generator=g) * 3
    indptr = torch.arange(0, 65, 2, dtype=torch.int32, device=_dev())
    d = torch.randint(0, 50, (64,), device=_dev(), generator=g)
    params = SamplingParams(temperature=0.7, top_p=0.5)
    tokens, acc = verify_drafts(logits, d, None, indptr, params, generator=g)
    from persona.sampling import _nucleus_mask
    inside = torch.isfinite(_nucleus_mask(logits / 0.7, 0.5))
    rows = torch.arange(64, device=_dev())
    kept = tokens >= 0
    assert inside[rows[kept], tokens[kept]].all()
    assert set(acc.tolist()) <= {0, 1}

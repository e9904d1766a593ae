"""The workspace of the NF4 linears: one for all sets of weights, of a model's
layer above all, where launches of few tiles and of many follow each other."""

import ctypes

import pytest
import torch

import capi_lib
from persona import nf4, ops
from persona.adapter_pool import AdapterPool
from persona.mistral import MistralConfig, MistralLoRAModel

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
# Products of fp16 with fp16(NF4 x scale): the dequantised weight is rounded once
# more (2^-11 of it), so is y; sums in fp32.
LAYER = [[(4096, 4096), (1024, 4096), (1024, 4096)], [(4096, 4096)], [(14336, 4096), (14336, 4096)], [(4096, 14336)]]
SMALL = [[(256, 128)], [(9088, 256), (128, 256)], [(128, 4096)]]


def _weights(shapes, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    sets = []
    for group in shapes:
        qs = [nf4.quantize((torch.randn(N, K, generator=g, device=DEV) * 0.02).half()) for N, K in group]
        sets.append((qs, [nf4.dequantize(q).float() for q in qs]))
    return sets, g


def _check(x, ws, ys):
    for w, y in zip(ws, ys):
        want = x.float() @ w.t()
        bound = 2.0 ** -10 * (x.float().abs() @ w.abs().t()) + 1e-6
        err = (y.float() - want).abs()
        assert torch.all(err <= bound), (tuple(w.shape), int((~(err <= bound)).sum()), float(err.nan_to_num(9e9).max()))


@pytest.mark.parametrize("M", [1, 8, 9, 40])
@pytest.mark.parametrize("shapes", [LAYER, SMALL])
def test_linears_of_a_layer_one_after_another(M, shapes):
    """Every output column is written, whatever set of weights came before."""
    sets, g = _weights(shapes, M)
    first = None
    for _ in range(2):
        got = []
        for i, (qs, ws) in enumerate(sets):
            x = torch.randn(M, qs[0].K, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV).half()
            ys = [torch.full((M, q.N), float("nan"), dtype=torch.float16, device=DEV) for q in qs]
            nf4.linear(x, qs, outs=ys)
            _check(x, ws, ys)
            got += ys
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, got))
        first = got
    ops.check_errors(DEV)


def test_one_workspace_of_the_c_api():
    """Zeroed once and large enough for each: any sets of weights in any order."""
    lib = capi_lib.load()
    M = 8
    sets, g = _weights([[(1024, 4096), (256, 4096)], [(9088, 256), (8192, 256)], [(128, 4096)]], 3)
    calls = []
    for qs, ws in sets:
        x = torch.randn(M, qs[0].K, generator=g, device=DEV).half()
        ys = [torch.empty(M, q.N, dtype=torch.float16, device=DEV) for q in qs]
        arr = (capi_lib.Nf4Problem * len(qs))(*[
            capi_lib.Nf4Problem(q.packed.data_ptr(), q.offset.data_ptr(), x.data_ptr(), q.K, y.data_ptr(), q.N, q.N, q.K)
            for q, y in zip(qs, ys)])
        calls.append((arr, x, ws, ys, lib.persona_nf4_linear_workspace_size(arr, len(qs))))
    size = max(c[-1] for c in calls)
    ws = torch.zeros(size, dtype=torch.uint8, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for k in (0, 1, 2, 1, 0, 2, 1):
        arr, x, w, ys, _ = calls[k]
        for y in ys:
            y.fill_(float("nan"))
        capi_lib.check(lib.persona_nf4_linear(arr, len(ys), M, ws.data_ptr(), size, err.data_ptr(), st))
        _check(x, w, ys)
    assert int(err.item()) == 0


@pytest.mark.parametrize("graph", [True, False])
def test_steps_of_full_width_layers_agree_with_their_prompt(graph):
    """Single tokens (NF4 linears) against the same tokens as one chunk (more
    than 64 rows: dequantised weights), two layers of the model's own width."""
    cfg = MistralConfig(num_layers=2, vocab=512)
    pool = AdapterPool(max_slots=4, r=16, device=DEV, num_layers=2, geometry=(cfg.hidden, cfg.kv_dim, cfg.intermediate))
    g = torch.Generator(device=DEV).manual_seed(5)
    for i in range(3):
        pool.load_random_adapter(f"a{i}", generator=g)
    model = MistralLoRAModel(cfg, pool, DEV, seed=2)
    gen = torch.Generator().manual_seed(7)
    tokens = torch.randint(0, cfg.vocab, (3, 80), generator=gen)
    slots = torch.tensor([0, -1, 2], dtype=torch.int32)
    whole = model.new_paged_state(slots, 20, 16, 96)
    want = model.extend(whole, tokens.tolist())[0].view(3, 80, -1)[:, 70:].float()
    got = []
    if graph:
        st = model.new_state(slots, 96)
        model.prefill(st, tokens[:, :70].to(DEV))
        for i in range(70, 80):
            st.tok.copy_(tokens[:, i])
            model.decode_step(st)
            got.append(st.bufs["logits"].float().clone())
    else:
        st = model.new_paged_state(slots, 20, 16, 96)
        model.extend(st, tokens[:, :70].tolist())
        for i in range(70, 80):
            got.append(model.extend(st, tokens[:, i:i + 1].tolist())[0].float())
    ops.check_errors(DEV)
    torch.testing.assert_close(torch.stack(got, 1), want, rtol=0, atol=0.03 * want.abs().max().item())


def _graph(x, qs, ys):
    nf4.linear(x, qs, outs=ys)  # (kernel attributes are set outside of a capture)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        nf4.linear(x, qs, outs=ys)
    return g


def _prepare(shapes, M, seed):
    (sets, g) = _weights(shapes, seed)
    out = []
    for qs, ws in sets:
        x = torch.randn(M, qs[0].K, generator=g, device=DEV).half()
        ys = [torch.full((M, q.N), float("nan"), dtype=torch.float16, device=DEV) for q in qs]
        out.append((x, qs, ws, ys))
    return out


def test_graphs_keep_their_workspace():
    """Captured, then calls with far more tiles, then memory of all sizes taken:
    a replay writes its outputs and nothing else."""
    few, many = _prepare([[(1024, 1024)], [(1 << 21, 128)]], 8, 4)
    x, qs, ws, ys = few
    g = _graph(x, qs, ys)
    nf4.linear(many[0], many[1], outs=many[3])
    _check(many[0], many[2], many[3])
    taken = [torch.full((n << 20,), 17, dtype=torch.uint8, device=DEV) for n in (1, 2, 4, 18, 19, 20, 21, 24, 32) for _ in range(3)]
    for _ in range(3):
        ys[0].fill_(float("nan"))
        g.replay()
        _check(x, ws, ys)
    assert all(bool((t == 17).all()) for t in taken)
    # another capture in between leaves the first graph's alone
    h = _graph(*[many[i] for i in (0, 1, 3)])
    for graph, (a, _, w, b) in ((g, few), (h, many), (g, few)):
        b[0].fill_(float("nan"))
        graph.replay()
        _check(a, w, b)


@pytest.mark.parametrize("captured", [True, False])
def test_linears_on_two_streams(captured):
    """Launches that run at the same time have a workspace each."""
    calls = _prepare([[(1024, 4096)], [(4096, 1024)]], 8, 6)
    graphs = [_graph(x, qs, ys) for x, qs, _, ys in calls] if captured else None
    want = []
    for x, qs, ws, ys in calls:
        nf4.linear(x, qs, outs=ys)
        _check(x, ws, ys)
        want.append(ys[0].clone())
    streams = [torch.cuda.Stream(DEV) for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(DEV))
    for _ in range(20):
        for i, s in enumerate(streams):
            x, qs, _, ys = calls[i]
            with torch.cuda.stream(s):
                ys[0].fill_(float("nan"))
                graphs[i].replay() if captured else nf4.linear(x, qs, outs=ys)
        torch.cuda.synchronize()
        for (_, _, _, ys), w in zip(calls, want):
            assert torch.equal(ys[0], w)
    ops.check_errors(DEV)


def test_only_the_counters_have_to_be_zero():
    lib = capi_lib.load()
    lib.persona_nf4_linear_counter_offset.restype = ctypes.c_size_t
    (qs, ws), = _weights([[(2048, 4096), (128, 4096)]], 9)[0]
    x = torch.randn(5, 4096, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half()
    ys = [torch.full((5, q.N), float("nan"), dtype=torch.float16, device=DEV) for q in qs]
    arr = (capi_lib.Nf4Problem * 2)(*[
        capi_lib.Nf4Problem(q.packed.data_ptr(), q.offset.data_ptr(), x.data_ptr(), q.K, y.data_ptr(), q.N, q.N, q.K)
        for q, y in zip(qs, ys)])
    size, at = lib.persona_nf4_linear_workspace_size(arr, 2), lib.persona_nf4_linear_counter_offset()
    assert 0 < at < size and size - at >= 4 * 17
    space = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    space[at:] = 0
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        capi_lib.check(lib.persona_nf4_linear(arr, 2, 5, space.data_ptr(), size, err.data_ptr(), st))
        _check(x, ws, ys)
    assert int(err.item()) == 0 and not space[at:].any()  # left at zero again


def test_many_streams_keep_few_workspaces():
    """One launch on each of 60 streams: right everywhere, and the memory that
    stays is that of a few."""
    (x, qs, ws, ys), = _prepare([[(1024, 4096)]], 8, 12)
    outs = [torch.full_like(ys[0], float("nan")) for _ in range(60)]
    streams = [torch.cuda.Stream(DEV) for _ in outs]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(DEV)
    for _ in range(2):
        for s, y in zip(streams, outs):
            with torch.cuda.stream(s):
                nf4.linear(x, qs, outs=[y])
    torch.cuda.synchronize()
    for y in outs:
        _check(x, ws, [y])
    assert torch.cuda.memory_allocated(DEV) - before <= 8 * (21 << 20)
    ops.check_errors(DEV)

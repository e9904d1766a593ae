"""Rotary write and read back captured into a graph, on another stream than the
one that made the tensors: replays follow the device arrays."""

import pytest
import torch

import paged_ref as R
from persona import ops
from test_paged_gpu import THETA, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_captured_write_and_read(dtype, e4m3):
    made = []
    for seed in range(2):  # two graphs, under way at once
        bt = R.Batch([3, 1, 0, 40], [30, 100 + seed, 7, 0], 16, 2, 128, dtype, e4m3, seed=seed, width=16, pad=2)
        q, k, v = bt.randn(bt.rows, 8, 128), bt.randn(bt.rows, 2, 128), bt.randn(bt.rows, 2, 128)
        qo, ko, vo = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)

        def step(bt=bt, q=q, k=k, v=v, qo=qo, ko=ko, vo=vo):
            ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=qo, **bt.scales())
            ops.paged_cache_read(*bt.args(), ko, vo, **bt.scales())

        step()
        torch.cuda.synchronize()
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=s):
            step()
        made.append((bt, q, k, v, qo, ko, vo, g, s))
    half = torch.finfo(dtype).eps / 2
    for turn in range(3):
        for bt, q, k, v, qo, ko, vo, g, s in made:
            for t in (q, k, v):
                t.copy_(bt.randn(*t.shape))
            for t in (qo, ko, vo):
                t.fill_(3.0)
            if turn:  # shorter sequences, and the pages of the first and the last exchanged
                bt.len = [max(n, L - 11) for n, L in zip(bt.new, bt.len)]
                bt.lengths.copy_(torch.tensor(bt.len, dtype=torch.int32))
                bt.table[[0, 3], :2] = bt.table[[3, 0], :2]
        torch.cuda.synchronize()
        for *_, g, s in made:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        ops.check_errors(torch.device("cuda", 0))
        for bt, q, k, v, qo, ko, vo, g, s in made:
            used = sum(bt.new)
            pos = torch.cat([torch.arange(L - n, L) for n, L in zip(bt.new, bt.len)]).cuda()
            for got, x, turned in ((qo, q, True), (ko, k, True), (vo, v, False)):
                want = R.rotate(x[:used], pos, THETA) if turned else x[:used].double()
                tol = half * want.abs() + 2.0 ** -20 * x[:used].double().abs().amax(-1, keepdim=True)
                if e4m3 and got is not qo:  # half a step of a code, or half of the smallest one, of the head's largest value
                    most = want.abs().amax(-1, keepdim=True)
                    tol = tol + (2.0 ** -4 * want.abs()).maximum(2.0 ** -10 * most / 448) + 2.0 ** -19 * most + half * 2.0 ** -4 * want.abs()
                _check(got[:used], want, tol)
                assert torch.all(got[used:] == 3.0)

"""Sampling from given numbers against the definition in 64 bits: tokens are
equal, since nothing but sums of up to V terms separates the two (errors of
about 1e-14 of the sum against gaps between neighbouring sums; a number that
falls into such an error would be a matter of one row in 10^8)."""

import math

import pytest
import torch

from persona import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def plain(logits, u, t=None, k=None, p=None, m=None):
    """One row after another, on the host, in 64 bits; exact sums (math.fsum) at the nucleus' end and at the draw."""
    out = []
    B, V = logits.shape
    get = lambda x, b, none: none if x is None else float(x[b])  # noqa: E731
    for b in range(B):
        x = logits[b].double().cpu()
        x = torch.where(x.isnan(), -math.inf, x)
        T, K, P, M, U = (get(z, b, n) for z, n in ((t, 1.0), (k, 0), (p, 1.0), (m, 0.0), (u, 0)))
        order = torch.sort(x, descending=True, stable=True).indices
        top = float(x[order[0]])
        if top == -math.inf:
            out.append(-1)
            continue
        if not T > 0:
            out.append(int(order[0]))
            continue
        w = torch.where(x == top, 1.0, torch.exp((x - top) / T).nan_to_num(0.0))
        w = torch.where(x == -math.inf, 0.0, w)
        order = order[x[order] > -math.inf]
        if 0 < K < len(order):
            order = order[:int(K)]
        ws = w[order]
        if P < 1:
            cum = ws.cumsum(0)
            n = 1 + int((cum[:-1] <= max(P, 0.0) * math.fsum(ws.tolist())).sum())
            order = order[:n]
        if M > 0:
            order = order[w[order] >= min(M, 1.0)]
        kept = torch.sort(order).values
        cum = w[kept].cumsum(0)
        target = max(U, 0.0) * float(cum[-1]) if U == U else 0.0
        over = (cum > target).nonzero()
        out.append(int(kept[int(over[0])]) if len(over) else int(kept[w[kept] > 0][-1]))
    return out


def _logits(B, V, dtype, seed, spread=3.0, stride=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, stride or V, generator=g, device="cuda") * spread
    return x.to(dtype)[:, :V], torch.rand(B, generator=g, device="cuda")


def _f(*v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def _i(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _run(logits, u, **kw):
    tokens = torch.full((logits.shape[0],), -9, dtype=torch.int64, device="cuda")
    got = ops.sample_tokens(logits, u, tokens, **kw)
    assert got is tokens
    ops.check_errors(logits.device)
    return tokens.tolist()


def _both(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    got = _run(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert got == plain(logits, u, temperature, top_k, top_p, min_p)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 255, 256, 257, 2049, 5001, 32000, 50257])
def test_every_rule(dtype, V):
    B = 14
    x, u = _logits(B, V, dtype, V)
    t = _f(1, 1, 0.7, 1.3, 0, -1, 1, 0.5, 2, 1, 0.9, 1, 1, 8.0)
    k = _i(0, 1, 5, 40, 3, 0, 300, 3000, 0, -4, 50, 0, V, 2500)
    p = _f(1, 1, 0.9, 0.95, 0.5, 1, 0.3, 0.999, 0.8, 0.0, 0.9, 2.0, 0.99, 0.97)
    m = _f(0, 0, 0.05, 0, 0.1, 0, 0, 0.001, 0, 0, 0.3, 0.02, -1, 0)
    _both(x, u)
    _both(x, u, temperature=t)
    _both(x, u, temperature=t, top_k=k)
    _both(x, u, temperature=t, top_p=p)
    _both(x, u, min_p=m)
    _both(x, u, temperature=t, top_k=k, top_p=p, min_p=m)


@pytest.mark.parametrize("dtype", TYPES)
def test_flat_rows(dtype):
    """Nuclei of thousands of tokens, which no list holds; numbers at both ends."""
    x, u = _logits(6, 70001, dtype, 3, spread=0.3)
    u = _f(0.0, 0.25, 0.5, 0.75, 0.999, float(torch.finfo(torch.float32).eps))
    for p in (0.1, 0.5, 0.9, 0.99999):
        _both(x, u, top_p=_f(*[p] * 6))
    for k in (2047, 2048, 2049, 30000):
        _both(x, u, top_k=_i(*[k] * 6))
        _both(x, u, top_k=_i(*[k] * 6), top_p=_f(*[0.7] * 6), min_p=_f(0, 0.1, 0.3, 0.5, 0.9, 1.5))


@pytest.mark.parametrize("V", [300, 3000, 9000, 20000])
@pytest.mark.parametrize("t", [0.3, 1.0, 100.0, 1000.0])
def test_nuclei_that_end_anywhere(V, t):
    """fp32 logits, all different: a class of the first search holds thousands,
    or the end lies in its last one."""
    x, u = _logits(24, V, torch.float32, 5)
    T = torch.full((24,), t, device="cuda")
    for p in (0.5, 0.9, 0.99, 0.999, 0.9999999):
        _both(x, u, temperature=T, top_p=torch.full((24,), p, device="cuda"))
    for k in (V // 2, V - 1):
        _both(x, u, temperature=T, top_k=torch.full((24,), k, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("B", [1, 304])  # eight CTAs a row, and one
@pytest.mark.parametrize("t", [0.01, 1.0, 50.0])
@pytest.mark.parametrize("at", [2046.45, 2046.55, 2046.8, 2046.87, 2046.93, 2046.97, 2047.5])
def test_cuts_where_the_last_class_begins(B, t, at):
    """Tokens around 32 powers of two below the largest, where the classes of the
    first search end: the k-th one, and the end of a nucleus, among them.  The
    last kept token of a number of 1 shows the cut."""
    far = -at / 64 * math.log(2.0) * t
    one, zeros = _f(*[1.0] * B), 600
    T = torch.full((B,), t, device="cuda")

    def both(row, **kw):
        x = torch.tensor(row, dtype=torch.float32, device="cuda").expand(B, -1)
        got = _run(x, one, temperature=T, **kw)
        assert got == plain(x[:1], one[:1], T[:1], *(kw[n][:1] if n in kw else None for n in ("top_k", "top_p"))) * B
        return got[0]

    # one token there, more than a list of all would hold above it
    k = torch.full((B,), zeros + 1, dtype=torch.int32, device="cuda")
    assert both([0.0] * zeros + [far, far * 30 / 22.166], top_k=k) == zeros
    # more of them than are sorted at once, cut by their index
    k = torch.full((B,), zeros + 700, dtype=torch.int32, device="cuda")
    assert both([0.0] * zeros + [far] * 1500 + [1.4 * far] * 500, top_k=k) == zeros + 699
    # a nucleus that ends among them
    p = torch.full((B,), 1 - 2.0 ** -24, device="cuda")
    assert 0 < both([0.0] + [far] * 2000 + [1.4 * far] * 500, top_p=p) < 2501


def test_equal_logits_are_cut_by_index():
    V = 40000
    x = torch.zeros(8, V, device="cuda")
    x[4:] = -3.5
    x[6, ::3] = 1.0
    x[7, 5:9] = 2.0
    u = _f(0.0, 0.5, 0.99999, 0.3, 0.7, 0.2, 0.6, 0.9)
    for k in (1, 3, 100, 2048, 2049, 20000, V - 1):
        got = _both(x, u, top_k=_i(*[k] * 8))
        assert max(got[:6]) < k
    for p in (0.25, 0.5, 0.75, 0.3, 1e-6):  # sums of ones are exact: a border that is met keeps its token
        got = _both(x, u, top_p=_f(*[p] * 8))
    _both(x, u, top_k=_i(*[9000] * 8), top_p=_f(*[0.5] * 8))
    # -0 and 0 are equal
    y = torch.zeros(1, 100, device="cuda")
    y[0, :50] = -0.0
    assert _run(y, _f(0.9), top_k=_i(3)) == [2] and _run(y, _f(0.9), temperature=_f(0.0)) == [0]


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_rows(dtype):
    """-infinity, NaN, the type's lowest value and +infinity."""
    V = 3001
    x, u = _logits(8, V, dtype, 11)
    inf, low = float("inf"), torch.finfo(dtype).min
    x[0, :] = -inf
    x[1, :] = float("nan")
    x[2, :-1] = -inf
    x[3, ::2] = -inf
    x[4, 1::2] = float("nan")
    x[5, :] = low
    x[6, 10:] = low
    x[7, 100:103] = inf
    t, k, p = _f(*[0.8] * 8), _i(*[50] * 8), _f(*[0.9] * 8)
    for kw in ({}, dict(top_k=k), dict(top_p=p), dict(top_k=k, top_p=p, min_p=_f(*[0.1] * 8)), dict(temperature=_f(*[0.0] * 8)),
               dict(temperature=t, top_k=_i(*[2999] * 8)), dict(top_p=_f(*[0.99999] * 8))):
        got = _both(x, u, **kw)
        assert got[:3] == [-1, -1, V - 1] and got[3] % 2 == 1 and got[4] % 2 == 0 and got[6] < 10 and 100 <= got[7] < 103


def test_temperatures_at_the_ends():
    x, u = _logits(8, 9000, torch.float32, 5)
    x[:, 77] = x.max() + 1
    x[:4, 78] = torch.nextafter(x[:4, 77], torch.zeros(4, device="cuda"))
    t = _f(1e-45, 1e-30, 1e-6, 1e-3, 1e3, 1e30, float("inf"), float("nan"))
    for kw in ({}, dict(top_k=_i(*[60] * 8)), dict(top_p=_f(*[0.6] * 8)), dict(top_p=_f(*[0.9999999] * 8)),
               dict(min_p=_f(*[0.5] * 8)), dict(top_k=_i(*[5000] * 8), top_p=_f(*[0.5] * 8))):
        _both(x, u, temperature=t, **kw)


def test_weights_that_bounds_say_little_of():
    """A temperature so small that a class of the search spans weights of all
    sizes, with the end of the nucleus in the far tail: the exact steps."""
    V = 60000
    x = torch.full((2, V), 9.0, device="cuda")
    for i in range(8):  # 22 and more units of the last place below the largest
        x[:, 1 + i::9] = 10 - 2.2e-5 - i * 1e-6
    x[:, 0] = 10.0
    x[0, 100] = -3e38
    t = _f(1e-6, 1e-6)
    for p in (1 - 2.0 ** -24, 1 - 2.0 ** -18, 1 - 2.0 ** -16):
        _both(x, _f(0.3, 0.9999999), temperature=t, top_p=_f(p, p))


def test_numbers_outside_of_their_range():
    x, _ = _logits(5, 1000, torch.float16, 6)
    u = _f(-1.0, float("nan"), 1.0, 7.0, float("inf"))
    for kw in ({}, dict(top_k=_i(*[20] * 5)), dict(top_p=_f(*[0.9] * 5))):
        first = _run(x[:2], _f(0, 0), **{n: z[:2] for n, z in kw.items()})
        got = _both(x, u, **kw)
        assert got[:2] == first


def test_draws_follow_the_weights():
    """The numbers' even spread becomes the kept weights'."""
    V, B = 40, 4096
    x = torch.randn(1, V, generator=torch.Generator().manual_seed(1)).cuda()
    u = (torch.arange(B, device="cuda") + 0.5) / B
    got = torch.tensor(_run(x.expand(B, V), u.float(), top_k=_i(*[12] * B)))
    w = torch.softmax(x[0].double().cpu(), 0)
    keep = torch.sort(w, descending=True).indices[:12]
    want = torch.zeros(V, dtype=torch.float64).scatter_(0, keep, w[keep] / w[keep].sum())
    freq = torch.bincount(got, minlength=V).double() / B
    assert torch.all((freq - want).abs() <= 1.0 / B + 1e-6)  # a run of even numbers misses an interval's share by one at most


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,V,stride", [(1, 1048577, None), (300, 1031, 1040), (700, 333, None), (40, 128001, 128003), (5, 50257, 50264)])
def test_sizes_and_strides(dtype, B, V, stride):
    if dtype == torch.float32 and V > 1000000:
        V = 2097152
    x, u = _logits(B, V, dtype, 8, stride=stride)
    sub = slice(None) if B <= 5 else slice(0, B, 13)
    kw = dict(temperature=torch.full((B,), 0.9, device="cuda"), top_p=torch.full((B,), 0.9, device="cuda"))
    for more in ({}, dict(top_k=torch.full((B,), 100, dtype=torch.int32, device="cuda"))):
        got = _run(x, u, **kw, **more)
        want = plain(x[sub], u[sub], kw["temperature"], more.get("top_k"), kw["top_p"])
        assert got[sub] == want
    assert _run(x, u)[sub] == plain(x[sub], u[sub])


def test_captured_and_on_two_streams():
    x, u = _logits(20, 20000, torch.float16, 9)
    p, k = torch.full((20,), 0.9, device="cuda"), torch.full((20,), 30, dtype=torch.int32, device="cuda")
    tok = [torch.zeros(20, dtype=torch.int64, device="cuda") for _ in range(2)]
    graphs = []
    for i, kw in enumerate((dict(top_p=p), dict(top_k=k))):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.sample_tokens(x, u, tok[i], **kw)
        graphs.append(g)
    x.copy_(_logits(20, 20000, torch.float16, 10)[0])
    u.copy_(torch.rand(20, device="cuda"))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert tok[0].tolist() == plain(x, u, p=p) and tok[1].tolist() == plain(x, u, k=k)


def test_refusals():
    x, u = _logits(4, 100, torch.float16, 1)
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    bad = [((x.double(), u, tok), {}, "float32, float16 or bfloat16"), ((x[0], u, tok), {}, r"\[B, V\]"),
           ((x.t(), u, tok), {}, "unit inner stride"), ((x, u[:3], tok), {}, "u must be"), ((x, u.double(), tok), {}, "u must be"),
           ((x, u, tok.int()), {}, "tokens must be"), ((x, u.cpu(), tok), {}, "u must be"),
           ((x, u, tok), dict(temperature=u.half()), "temperature"), ((x, u, tok), dict(top_k=u), "top_k"),
           ((x, u, tok), dict(top_p=u[:2]), "top_p"), ((x, u, tok), dict(min_p=u.repeat(2)[::2]), "min_p"),
           ((x, tok.view(torch.float32)[:4], tok), {}, "overlaps"), ((x[:, :0], u, tok), {}, "vocabulary")]
    for args, kw, match in bad:
        with pytest.raises(RuntimeError, match=match):
            ops.sample_tokens(*args, **kw)
    ops.sample_tokens(x[:0], u[:0], tok[:0])
    assert tok.tolist() == [0] * 4

"""CPU checks of the paged cache operators and the draft verification: status
codes of the C ABI (every call fails validation before touching the GPU), the
torch layer's refusals, and the plain forms the GPU tests compare with."""

import ctypes

import pytest
import torch

import capi_lib
import paged_ref as R
from test_native_build import built  # noqa: F401  (fixture)

FAKE = 1 << 20  # aligned, never dereferenced: validation fails first


class Cache(ctypes.Structure):
    """persona_paged_cache (include/persona_bgmv.h)."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] +
                [(n, ctypes.c_int64) for n in ("page_stride", "head_stride", "pos_stride", "scale_page_stride",
                                               "scale_head_stride", "num_pages", "page_size", "Hkv", "D")] +
                [("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("max_pages", ctypes.c_int64),
                 ("indptr", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("B", ctypes.c_int64),
                 ("kind", ctypes.c_int)])


class Rows(ctypes.Structure):
    """persona_rows (include/persona_bgmv.h)."""
    _fields_ = [("p", ctypes.c_void_p), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


def _cache(**change):
    c = dict(k=FAKE, v=FAKE, k_scale=None, v_scale=None, page_stride=8 * 16 * 128, head_stride=16 * 128, pos_stride=128,
             scale_page_stride=128, scale_head_stride=16, num_pages=9, page_size=16, Hkv=8, D=128, page_table=FAKE,
             table_stride=4, max_pages=4, indptr=FAKE, lengths=FAKE, B=2, kind=0)
    c.update(change)
    return Cache(**c)


@pytest.fixture(scope="module")
def lib(built):  # noqa: F811
    lib = ctypes.CDLL(str(capi_lib.LIB_PATH))
    P, I, Z = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
    lib.persona_paged_rope_cache.argtypes = [P] * 5 + [I, I, ctypes.c_float, ctypes.c_int, P, P]
    lib.persona_paged_cache_read.argtypes = [P] * 3 + [I, ctypes.c_int, P, P]
    lib.persona_paged_attention.argtypes = [P] * 3 + [I, I, ctypes.c_float, I, I, ctypes.c_int, P, Z, P, P]
    lib.persona_paged_attention_workspace_size.argtypes = [I]
    lib.persona_paged_attention_workspace_size.restype = Z
    lib.persona_verify_draft.argtypes = [P, I, P, I, ctypes.c_int] + [P] * 6 + [I, I, I, P, P]
    return lib


def _attend(lib, cache=None, q=None, rows=4, Hq=32, scale=0.1, window=0, max_new=1, dtype=0, ws=FAKE, ws_bytes=1 << 40):
    cache = cache if cache is not None else _cache()
    q = q or Rows(FAKE, 32 * 128, 128)
    return lib.persona_paged_attention(ctypes.byref(cache), ctypes.byref(q), ctypes.byref(Rows(FAKE, 32 * 128, 128)), rows,
                                       Hq, scale, window, max_new, dtype, ws, ws_bytes, None, None)


def test_attention_statuses(lib):
    INVALID, SHAPE, DTYPE, ALIGN, WS = 1, 2, 3, 4, 6
    assert lib.persona_paged_attention(None, None, None, 1, 8, 0.1, 0, 1, 0, None, 0, None, None) == INVALID
    assert _attend(lib, rows=0) == 0 and _attend(lib, _cache(B=0)) == 0
    for change, want in [(dict(k=None), INVALID), (dict(page_table=None), INVALID), (dict(lengths=None), INVALID),
                         (dict(k_scale=FAKE), INVALID), (dict(kind=1), INVALID), (dict(kind=2), DTYPE),
                         (dict(D=96), SHAPE), (dict(Hkv=0), SHAPE), (dict(num_pages=0), SHAPE), (dict(page_size=0), SHAPE),
                         (dict(table_stride=3), SHAPE), (dict(pos_stride=64), SHAPE), (dict(page_stride=-8), SHAPE),
                         (dict(B=-1), SHAPE), (dict(max_pages=1 << 28, table_stride=1 << 28), SHAPE),
                         (dict(k=FAKE + 8), ALIGN), (dict(head_stride=12), ALIGN), (dict(lengths=FAKE + 2), ALIGN),
                         (dict(kind=1, k_scale=FAKE, v_scale=FAKE, pos_stride=136), ALIGN),
                         (dict(kind=1, k_scale=FAKE + 1, v_scale=FAKE), ALIGN)]:
        assert _attend(lib, _cache(**change)) == want, change
    assert _attend(lib, Hq=33) == SHAPE and _attend(lib, Hq=0) == SHAPE and _attend(lib, rows=-1) == SHAPE
    assert _attend(lib, window=-1) == SHAPE and _attend(lib, max_new=0) == SHAPE
    assert _attend(lib, scale=0.0) == SHAPE and _attend(lib, scale=-0.1) == SHAPE
    assert _attend(lib, scale=float("nan")) == SHAPE and _attend(lib, scale=float("inf")) == SHAPE
    assert _attend(lib, rows=1 << 30) == SHAPE and _attend(lib, dtype=2) == DTYPE
    assert _attend(lib, q=Rows(FAKE + 2, 4096, 128)) == ALIGN and _attend(lib, q=Rows(FAKE, 4095, 128)) == ALIGN
    assert _attend(lib, q=Rows(None, 4096, 128)) == INVALID
    assert _attend(lib, ws=None) == WS and _attend(lib, ws_bytes=64) == WS and _attend(lib, ws=FAKE + 8) == ALIGN
    assert lib.persona_paged_attention_workspace_size(96) == 0
    assert lib.persona_paged_attention_workspace_size(128) > lib.persona_paged_attention_workspace_size(64) > 0


def test_write_and_read_statuses(lib):
    r = ctypes.byref(Rows(FAKE, 4096, 128))

    def write(cache=None, q=r, rows=4, Hq=32, theta=1e6, dtype=0):
        return lib.persona_paged_rope_cache(ctypes.byref(cache or _cache()), q, r, r, r, rows, Hq, theta, dtype, None, None)

    assert write(rows=0) == 0 and write(_cache(B=0)) == 0
    assert write(Hq=0) == 2 and write(Hq=5000) == 2 and write(theta=1.0) == 2 and write(theta=float("nan")) == 2
    assert write(theta=float("inf")) == 2 and write(dtype=2) == 3 and write(q=None) == 1 and write(_cache(D=32)) == 2
    read = lambda c, k=r, rows=4: lib.persona_paged_cache_read(ctypes.byref(c), k, r, rows, 0, None, None)  # noqa: E731
    assert read(_cache(), rows=0) == 0 and read(_cache(), rows=-1) == 2 and read(_cache(), k=None) == 1
    assert read(_cache(v=FAKE + 4)) == 4


def test_verify_statuses(lib):
    def call(target=FAKE, ld=100, draft=FAKE, ldd=100, t=2, d=FAKE, ip=FAKE, ua=FAKE, us=FAKE, out=FAKE, acc=FAKE, rows=3, B=1, V=100):
        return lib.persona_verify_draft(target, ld, draft, ldd, t, d, ip, ua, us, out, acc, rows, B, V, None, None)

    assert call(B=0) == 0
    assert call(t=3) == 3 and call(t=-1) == 3
    assert call(V=0) == 2 and call(V=2097153, ld=1 << 22, ldd=1 << 22) == 2 and call(ld=99) == 2 and call(ldd=99) == 2
    assert call(rows=-1) == 2 and call(B=-1) == 2
    assert call(target=None) == 1 and call(ip=None) == 1 and call(ua=None) == 1 and call(out=None) == 1 and call(acc=None) == 1
    assert call(target=FAKE + 2) == 4 and call(d=FAKE + 4) == 4 and call(t=0, target=FAKE + 1) == 4


def test_ops_refuse_cpu_tensors(built):  # noqa: F811
    from persona import ops

    bt = R.Batch([1, 2], [3, 0], 16, 2, 128, torch.float16, device="cpu")
    q, k = bt.randn(3, 4, 128), bt.randn(3, 2, 128)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.paged_rope_cache(q, k, k, *bt.args(), 1e6)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.paged_cache_read(*bt.args(), k, k.clone())
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.paged_attention(q, *bt.args(), torch.empty_like(q), 0.1)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.verify_draft(torch.ones(3, 5), torch.zeros(3, dtype=torch.int64), None, bt.indptr, torch.rand(3), torch.rand(2),
                         torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32))


# --------------------------------------------------- the plain forms themselves
def test_plain_attention_is_softmax_attention():
    import torch.nn.functional as F

    bt = R.Batch([4, 1], [0, 9], 4, 2, 64, torch.float16, device="cpu")
    bt.fill()
    q = bt.randn(5, 4, 64)
    want, tol = R.attention(bt, q, 0.2)
    k, v = bt.get("k", 0, 0, 4), bt.get("v", 0, 0, 4)
    ref = F.scaled_dot_product_attention(q[:4].double().transpose(0, 1), k.transpose(0, 1).repeat_interleave(2, 0),
                                         v.transpose(0, 1).repeat_interleave(2, 0), is_causal=True, scale=0.2).transpose(0, 1)
    torch.testing.assert_close(want[:4], ref)
    # a 16-bit form of it lies within the bound, one that ignores the mask does not
    assert ((ref.half().double() - want[:4]).abs() <= tol[:4]).all()
    free = F.scaled_dot_product_attention(q[:4].double().transpose(0, 1), k.transpose(0, 1).repeat_interleave(2, 0),
                                          v.transpose(0, 1).repeat_interleave(2, 0), scale=0.2).transpose(0, 1)
    assert not ((free - want[:4]).abs() <= tol[:4]).all()


def test_plain_rotation_keeps_lengths_and_turns_by_the_position():
    x = torch.randn(3, 2, 128, dtype=torch.float64)
    y = R.rotate(x, torch.tensor([0, 1, 100000]), 1e6)
    torch.testing.assert_close(y[0], x[0])
    torch.testing.assert_close(y.norm(dim=-1), x.norm(dim=-1))
    a = torch.complex(x[1, 0, 0], x[1, 0, 64]) * torch.polar(torch.tensor(1.0).double(), torch.tensor(1.0).double())
    torch.testing.assert_close(torch.stack([y[1, 0, 0], y[1, 0, 64]]), torch.stack([a.real, a.imag]))


def test_plain_verification_by_hand():
    p = torch.tensor([[0.5, 0.5, 0.0], [0.2, 0.3, 0.5], [0.1, 0.1, 0.8]])
    q = torch.tensor([[0.25, 0.5, 0.25], [0.6, 0.2, 0.2], [0.0, 0.0, 0.0]])
    ip = torch.tensor([0, 3])
    d = torch.tensor([0, 0, 0])
    # first kept (0.9 * 0.25 < 0.5), second not (0.9 * 0.6 > 0.2): residual (0, .1, .3), the number 0.3 falls on token 2
    assert R.verify(p, d, q, ip, torch.tensor([0.9, 0.9, 0.0]), torch.tensor([0.3])) == ([0, 2, -1], [1])
    assert R.verify(p, d, q, ip, torch.tensor([0.9, 0.9, 0.0]), torch.tensor([0.2])) == ([0, 1, -1], [1])
    assert R.verify(p, d, q, ip, torch.tensor([0.9, 0.1, 0.0]), torch.tensor([0.15])) == ([0, 0, 1], [2])
    # a certain draft: kept while u < p; not drawn again
    assert R.verify(p, d, None, ip, torch.tensor([0.6, 0.0, 0.0]), torch.tensor([0.0])) == ([1, -1, -1], [0])


def test_page_tables_hold_at_most_2_30_positions(lib):
    """One page more is refused; the limit itself goes on to the next check
    (a workspace that is missing)."""
    for page in (1, 16, 64, 4096):
        most = (1 << 30) // page
        at = lambda n: _cache(page_size=page, max_pages=n, table_stride=n)  # noqa: E731
        assert _attend(lib, at(most + 1)) == 2 and _attend(lib, at(most), ws=None) == 6


def test_extend_refuses_token_ids_outside_the_vocabulary():
    """Before the state moves on (no model or GPU is reached)."""
    from types import SimpleNamespace

    from persona.mistral import MistralLoRAModel, PagedState

    none = [None]
    st = PagedState(slots=torch.zeros(2, dtype=torch.int32), page_size=4, page_table=torch.zeros(2, 2, dtype=torch.int32),
                    k_cache=none, v_cache=none, k_scale=none, v_scale=none, lengths=[0, 0], pages=[[], []],
                    free=list(range(4)))
    model = SimpleNamespace(cfg=SimpleNamespace(vocab=50), device=torch.device("cpu"))
    for bad in (-1, 50, 1 << 40):
        with pytest.raises(ValueError, match="outside the vocabulary"):
            MistralLoRAModel.extend(model, st, [[1, 49], [0, bad]])
    with pytest.raises(ValueError, match="one chunk"):
        MistralLoRAModel.extend(model, st, [[1]])
    assert st.lengths == [0, 0] and st.pages == [[], []] and len(st.free) == 4

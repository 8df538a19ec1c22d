"""Host-side behaviour of attention and of the rotation of queries and keys that needs no
GPU: the refusals of the Python entry points and of the C ABI (all before any launch),
and what autograd, traces and saved-tensor hooks make of them (the library stubbed)."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

import library_stub as stub
import memoryefficientclip_amd as mec
import tower_reference as ref
from memoryefficientclip_amd import _lib


class FakeCuda(torch.Tensor):
    @property
    def is_cuda(self):
        return True


def fake(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(FakeCuda)


def wide(*shape, dtype=torch.float32):
    """Of any size, without memory."""
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(shape).as_subclass(FakeCuda)


@pytest.fixture
def no_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


HEADS, KEYS = (2, 5, 4, 8), (2, 7, 2, 8)


def test_cpu_tensors_raise():
    x, p = torch.zeros(HEADS), torch.zeros(5, 1, dtype=torch.int64)
    with pytest.raises(AssertionError, match="GPU"):
        mec.attention(x, x, x)
    with pytest.raises(AssertionError, match="GPU"):
        mec.norm_rotary(x, x, p, (4,))
    with pytest.raises(TypeError, match="Tensor"):
        mec.attention([1.0], x, x)


def test_attention_refuses(no_capture):
    q, k = fake(*HEADS), fake(*KEYS)
    for shapes, message in [((HEADS[1:], KEYS, KEYS), "batch, tokens"), ((HEADS, KEYS, (2, 6, 2, 8)), "differ in shape"),
                            ((HEADS, (3, 7, 2, 8), (3, 7, 2, 8)), "same batch"),
                            ((HEADS, (2, 7, 2, 6), (2, 7, 2, 6)), "same batch"),
                            ((HEADS, (2, 7, 3, 8), (2, 7, 3, 8)), "divide"), ((HEADS, (2, 7, 0, 8), (2, 7, 0, 8)), "divide"),
                            (((2, 5, 0, 8), KEYS, KEYS), "divide"), (((2, 5, 2, 129), (2, 7, 2, 129), (2, 7, 2, 129)), "head_dim"),
                            (((2, 5, 4, 0), (2, 7, 2, 0), (2, 7, 2, 0)), "head_dim")]:
        with pytest.raises(ValueError, match=message):
            mec.attention(*(fake(*s) for s in shapes))
    with pytest.raises(ValueError, match="2\\^30"):
        mec.attention(q, wide(2, (1 << 30) + 1, 2, 8), wide(2, (1 << 30) + 1, 2, 8))
    with pytest.raises(TypeError, match="dtype"):
        mec.attention(q.double(), k.double(), k.double())
    with pytest.raises(TypeError, match="mismatch"):
        mec.attention(q, k, k.half())
    for s in (0.0, -1.0, math.inf, math.nan, 1e-31, 1e31):
        with pytest.raises(ValueError, match="scale"):
            mec.attention(q, k, k, scale=s)
    with pytest.raises(ValueError, match="query_lengths"):
        mec.attention(q, k, k, query_lengths=fake(3, dtype=torch.int32))
    with pytest.raises(TypeError, match="key_lengths"):
        mec.attention(q, k, k, key_lengths=fake(2))
    with pytest.raises(TypeError, match="mismatch"):
        mec.attention(q, k, k, query_lengths=fake(2, dtype=torch.int32), key_lengths=fake(2, dtype=torch.int64))
    with pytest.raises(AssertionError, match="GPU"):
        mec.attention(q, k, k, key_lengths=torch.zeros(2, dtype=torch.int32))


def test_norm_rotary_refuses(no_capture):
    q, k, p, w = fake(*HEADS), fake(2, 5, 2, 8), fake(5, 1, dtype=torch.int64), fake(8)
    bad = [((q, fake(2, 6, 2, 8), p, (4,)), "heads only"), ((fake(2, 5, 4, 7), fake(2, 5, 2, 7), p, (3,)), "even"),
           ((fake(2, 5, 0, 8), k, p, (4,)), "heads"), ((fake(2, 5, 4, 258), fake(2, 5, 2, 258), p, (129,)), "256"),
           ((q, k, p, (3,)), "pairs"), ((q, k, p, ()), "axes"), ((q, k, p, (5, -1)), "pairs"), ((q, k, p, (2, 2)), "positions"),
           ((q, k, fake(6, 1, dtype=torch.int64), (4,)), "positions"), ((q, k, p, (4,), w), "needs a norm"),
           ((q, k, p, (4,), fake(7), None, 1e-6), "query_weight"), ((q, k, p, (4,), None, None, -1.0), "eps"),
           ((q, k, p, (4,), None, None, math.nan), "eps"), ((q, k, p, (4,), None, None, None, 0.0), "theta"),
           ((q, k, p, (4,), None, None, None, math.inf), "theta"), ((q, k, p, (4,), None, None, None, 1e4, w), "frequencies"),
           ((wide(1 << 16, 1 << 16, 1, 8), wide(1 << 16, 1 << 16, 1, 8), p, (4,)), "2\\^31")]
    for args, message in bad:
        with pytest.raises(ValueError, match=message):
            mec.norm_rotary(*args)
    for args, message in [((q, k, p.double(), (4,)), "positions"), ((q, k.half(), p, (4,)), "mismatch"),
                          ((q, k, p, (4,), w, w.half(), 1e-6), "weights"),
                          ((q, k, p, (4,), None, None, None, 1e4, fake(4, dtype=torch.int64)), "frequencies")]:
        with pytest.raises(TypeError, match=message):
            mec.norm_rotary(*args)


def test_graph_capture_is_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="graph capture"):
        mec.attention(fake(*HEADS), fake(*KEYS), fake(*KEYS))
    with pytest.raises(RuntimeError, match="graph capture"):
        mec.norm_rotary(fake(*HEADS), fake(*HEADS), fake(5, 1, dtype=torch.int64), (4,))


# ---- the C ABI ----

P = 4096  # (a pointer that is never followed: every call here is refused)


def heads(**change):
    h = _lib.Heads(P, 100, 10, 5)
    for name, value in change.items():
        setattr(h, name, value)
    return ctypes.byref(h)


def attention_problem(**change):
    a = _lib.Attention(2, 5, 7, 4, 2, 8, _lib.DTYPE_F32, 0, 0.5, 4, None, None)
    for name, value in change.items():
        setattr(a, name, value)
    return a


def call_attention(a, out=P, workspace=None, nbytes=0, **change):
    h = {n: heads() for n in ("q", "k", "v")}
    h.update(change)
    return _lib.load().mec_attention(None if a is None else ctypes.byref(a), h["q"], h["k"], h["v"], out, None, workspace,
                                     nbytes, None)


def call_attention_backward(a, out=P, lse=P, dq=P, dk=P, dv=P, workspace=None, nbytes=0, **change):
    h = {n: heads() for n in ("q", "k", "v", "g")}
    h.update(change)
    return _lib.load().mec_attention_backward(ctypes.byref(a), h["q"], h["k"], h["v"], out, lse, h["g"], dq, dk, dv,
                                              workspace, nbytes, None)


BAD_ATTENTION = [(dict(dtype=4), -1), (dict(batch=0), -1), (dict(queries=0), -1), (dict(keys=0), -1), (dict(heads=0), -1),
                 (dict(key_heads=0), -1), (dict(key_heads=3), -1), (dict(head_dim=0), -1), (dict(head_dim=129), -2),
                 (dict(keys=(1 << 30) + 1), -2), (dict(queries=1 << 30), -2), (dict(batch=1 << 30), -2),
                 (dict(heads=1 << 40, key_heads=1), -2), (dict(scale=0.0), -1), (dict(scale=1e-31), -1), (dict(scale=1e31), -1), (dict(scale=math.nan), -1),
                 (dict(scale=math.inf), -1), (dict(query_lengths=P, length_bytes=3), -1)]


@pytest.mark.parametrize("change,code", BAD_ATTENTION)
def test_c_abi_attention_refuses(monkeypatch, change, code):
    monkeypatch.setenv("MEC_TEST_ASSUME_CAPTURING", "1")  # (what is not refused before would be refused for this)
    a, lib = attention_problem(**change), _lib.load()
    assert call_attention(a) == code and _lib.last_error() and "captured" not in _lib.last_error()
    assert call_attention_backward(a) == code and "captured" not in _lib.last_error()
    assert lib.mec_attention_workspace_bytes(ctypes.byref(a)) == code
    assert lib.mec_attention_backward_workspace_bytes(ctypes.byref(a)) == code


def test_c_abi_attention_refuses_pointers(monkeypatch):
    monkeypatch.setenv("MEC_TEST_ASSUME_CAPTURING", "1")
    a = attention_problem()
    assert call_attention(None) == -1
    for name in ("q", "k", "v"):
        assert call_attention(a, **{name: None}) == -1
        assert call_attention(a, **{name: heads(data=None)}) == -1
        assert call_attention(a, **{name: heads(head_stride=-1)}) == -1
        assert call_attention(a, **{name: heads(token_stride=(1 << 40) + 1)}) == -1
    assert call_attention(a, out=None) == -1
    for change in (dict(out=None), dict(lse=None), dict(g=None), dict(dk=None), dict(dv=None)):
        assert call_attention_backward(a, **change) == -1
    assert "captured" not in _lib.last_error()
    # and a capture
    assert call_attention(a) == -2 and "captured" in _lib.last_error()
    assert call_attention_backward(a) == -2 and "captured" in _lib.last_error()


def rotary(**change):
    r = _lib.Rotary(2, 5, 4, 2, 8, _lib.DTYPE_F32, _lib.DTYPE_F32, 1, 0, 1e-6, 2, (2, 2), 1, 0, 1e4, P, P, P, None)
    for name, value in change.items():
        setattr(r, name, (ctypes.c_int32 * 8)(*value) if name == "sections" else value)
    return r


def call_rotary(r, q=P, k=P, **change):
    h = {n: heads() for n in ("query", "key")}
    h.update(change)
    return _lib.load().mec_norm_rotary(None if r is None else ctypes.byref(r), h["query"], h["key"], q, k, None)


def call_rotary_backward(r, dq=P, dk=P, dwq=None, dwk=None, **change):
    h = {n: heads() for n in ("query", "key", "gq", "gk")}
    h.update(change)
    return _lib.load().mec_norm_rotary_backward(ctypes.byref(r), h["query"], h["key"], h["gq"], h["gk"], dq, dk, dwq, dwk,
                                                None, 0, None)


BAD_ROTARY = [(dict(dtype=5), -1), (dict(weight_dtype=-1), -1), (dict(batch=0), -1), (dict(tokens=0), -1),
              (dict(query_heads=-1), -1), (dict(query_heads=0, key_heads=0), -1), (dict(head_dim=7), -1),
              (dict(head_dim=258, sections=(129,), axes=1), -2), (dict(axes=0), -1), (dict(axes=9), -1),
              (dict(sections=(2, 3)), -1), (dict(sections=(5, -1)), -1), (dict(positions=None), -1),
              (dict(position_type=3), -1), (dict(theta=0.0), -1), (dict(theta=math.inf), -1), (dict(eps=-1.0), -1),
              (dict(eps=math.nan), -1), (dict(batch=1 << 16, tokens=1 << 16), -2), (dict(query_heads=(1 << 16) + 1), -2)]


@pytest.mark.parametrize("change,code", BAD_ROTARY)
def test_c_abi_rotary_refuses(monkeypatch, change, code):
    monkeypatch.setenv("MEC_TEST_ASSUME_CAPTURING", "1")
    r = rotary(**change)
    assert call_rotary(r) == code and "captured" not in _lib.last_error()
    assert call_rotary_backward(r) == code and "captured" not in _lib.last_error()
    assert _lib.load().mec_norm_rotary_workspace_bytes(ctypes.byref(r)) == code


def test_c_abi_rotary_refuses_pointers(monkeypatch):
    monkeypatch.setenv("MEC_TEST_ASSUME_CAPTURING", "1")
    r = rotary()
    assert call_rotary(None) == -1
    for change in (dict(q=None), dict(k=None), dict(query=None), dict(key=heads(data=None)), dict(key=heads(batch_stride=-1))):
        assert call_rotary(r, **change) == -1
    for change in (dict(gq=None), dict(gk=None), dict(query=None), dict(key=None)):
        assert call_rotary_backward(r, **change) == -1
    plain = rotary(norm=0)
    assert call_rotary_backward(plain, dwq=P) == -1 and "weights" in _lib.last_error()
    assert call_rotary_backward(plain, dq=None) == -1
    assert call_rotary_backward(rotary(key_heads=0), dwk=P) == -1 and "gradient" in _lib.last_error()
    assert _lib.load().mec_norm_rotary_workspace_bytes(ctypes.byref(plain)) == 0


# ---- autograd, with the library stubbed ----


@pytest.fixture
def lib(monkeypatch):
    return stub.install(monkeypatch)


POSITIONS = torch.arange(5)[:, None]
OPERATORS = [lambda x: mec.attention(x, x[:, :, :2], x[:, :, 2:]),
             lambda x: mec.norm_rotary(x, x, POSITIONS, (4,))[0],
             lambda x: mec.norm_rotary(x, x, POSITIONS, (4,), None, torch.ones(8), 1e-6)[1]]
CALLS = ["mec_attention", "mec_norm_rotary", "mec_norm_rotary"]


@pytest.mark.parametrize("op", OPERATORS)
def test_second_derivatives_are_refused(lib, op):
    x = torch.randn(HEADS, requires_grad=True)
    first, = torch.autograd.grad(op(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        first.square().sum().backward()


@pytest.mark.parametrize("wanted", [False, True])
@pytest.mark.parametrize("op", OPERATORS)
def test_forward_mode_and_make_fx_are_refused(lib, op, wanted):
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(HEADS).requires_grad_(wanted)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        op(fwd.make_dual(x, torch.ones(HEADS)))
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(op)(x)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("wanted", [False, True])
@pytest.mark.parametrize("op,call", zip(OPERATORS, CALLS))
def test_traces_call_the_library_and_check(lib, op, call, wanted):
    traced = torch.jit.trace(op, torch.randn(HEADS).requires_grad_(wanted), check_trace=False)
    lib.calls.clear()
    y = torch.randn(HEADS)
    assert traced(y).shape == y.shape and len(lib.calls[call]) == 1
    lib.calls.clear()
    with pytest.raises(Exception, match="head_dim"):
        traced(torch.randn(2, 5, 4, 300))
    assert call not in lib.calls


def test_saved_tensors_that_come_back_in_other_strides(lib):
    """The backward reads q, k, v with the strides of the tensors that it gets."""
    qkv = torch.randn(2, 5, 8, 8)
    q, k, v = (t.detach().requires_grad_(True) for t in qkv.split([4, 2, 2], 2))
    with stub.copying_hooks():
        out = mec.attention(q, k, v)
    before = lib.calls["mec_attention"][0]
    torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    problem, hq, hk, hv = lib.calls["mec_attention_backward"][0][:4]
    assert before[1]._obj.token_stride == 64 and hq._obj.token_stride == 32 and hk._obj.token_stride == 16
    assert hv._obj.head_stride == 8 and problem._obj.causal == 0
    with stub.copying_hooks(lambda t: t.double() if t.dim() == 4 else t):
        out = mec.attention(q, k, v)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(out, (q, k, v), torch.ones_like(out))


def test_a_gradient_that_is_not_asked_for_is_not_made(lib):
    q, k = torch.randn(HEADS), torch.randn(KEYS)
    mec.attention(q.requires_grad_(True), k, k).sum().backward()
    args = lib.calls["mec_attention_backward"][0]
    assert args[7] is not None and args[8] is None and args[9] is None
    x, w = torch.randn(HEADS), torch.ones(8, requires_grad=True)
    mec.norm_rotary(x, x, POSITIONS, (4,), w, w, 1e-6)[0].sum().backward()
    args = lib.calls["mec_norm_rotary_backward"][0]
    # (of the keys nothing, of the queries the weight's alone)
    assert args[0]._obj.key_heads == 0 and args[5] is None and args[7] is not None and args[8] is None


# ---- the definitions ----


def test_the_definitions_gradients_are_differences():
    g = torch.Generator().manual_seed(0)
    q, do = (torch.randn(2, 6, 4, 5, generator=g, dtype=torch.float64) for _ in "qd")
    k, v = (torch.randn(2, 7, 2, 5, generator=g, dtype=torch.float64) for _ in "kv")
    how = dict(causal=True, query_lengths=torch.tensor([6, 3]), key_lengths=torch.tensor([4, 7]))
    f = lambda q, k, v: (ref.attention(q, k, v, **how)["out"][0] * do).sum()  # noqa: E731
    want = ref.attention(q, k, v, do, **how)
    h = 1e-5
    for i, name in enumerate(("dq", "dk", "dv")):
        step = torch.randn((q, k, v)[i].shape, generator=g, dtype=torch.float64)
        ends = [f(*(t + s * h * step if j == i else t for j, t in enumerate((q, k, v)))) for s in (1, -1)]
        # (h^2 of third derivatives, and 2^-53 over h)
        assert abs((ends[0] - ends[1]) / (2 * h) - (want[name][0] * step).sum()) < 1e-7
    x, dy = (torch.randn(2, 6, 3, 8, generator=g, dtype=torch.float64) for _ in "xd")
    w, p = torch.rand(8, generator=g, dtype=torch.float64) + 0.5, torch.randint(0, 50, (6, 2), generator=g)
    for interleaved in (False, True):
        f = lambda x, w: (ref.norm_rotary(x, p, (1, 3), w, 1e-6, interleaved=interleaved)["y"][0] * dy).sum()  # noqa: E731
        want = ref.norm_rotary(x, p, (1, 3), w, 1e-6, interleaved=interleaved, dy=dy)
        for i, name in enumerate(("dx", "dw")):
            step = torch.randn((x, w)[i].shape, generator=g, dtype=torch.float64)
            ends = [f(*(t + s * h * step if j == i else t for j, t in enumerate((x, w)))) for s in (1, -1)]
            assert abs((ends[0] - ends[1]) / (2 * h) - (want[name][0] * step).sum()) < 1e-7

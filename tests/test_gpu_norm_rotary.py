"""The rotation of queries and keys with the norm of each head, and its gradients,
against their definition in 64 bits."""
import pytest
import torch

import memoryefficientclip_amd as mec
import tower_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(b, n, h, hk, d, dtype, sections, positions, norm=True, wtype=None, seed=0, leaves=None, **how):
    g = torch.Generator().manual_seed(seed)
    xs = [torch.randn(b, n, x, d, generator=g).to(dtype) for x in (h, hk)]
    dys = [torch.randn(b, n, x, d, generator=g).to(dtype) for x in (h, hk)]
    ws = [(1 + 0.2 * torch.randn(d, generator=g)).to(wtype or dtype) if norm else None for _ in "qk"]
    eps = 1e-6 if norm else None
    on = [t.to(DEV) for t in xs]
    if leaves is not None:
        on = [leaves(t) for t in on]
    on = [t.requires_grad_(True) for t in on]
    won = [w if w is None else w.to(DEV).requires_grad_(True) for w in ws]
    how_on = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in how.items()}
    out = mec.norm_rotary(*on, positions.to(DEV), sections, *won, eps=eps, **how_on)
    torch.autograd.backward(out, [t.to(DEV) for t in dys])
    how = {"freq" if k == "frequencies" else k: v for k, v in how.items()}
    for name, x, dy, w, y, xl, wl in zip("qk", xs, dys, ws, out, on, won):
        want = ref.norm_rotary(x, positions, sections, w, eps, dy=dy, **how)
        assert y.dtype == dtype and y.is_contiguous()
        ref.close(name, y, *want["y"])
        ref.close("d" + name, xl.grad, *want["dx"])
        if norm:
            assert wl.grad.dtype == wl.dtype
            ref.close("dw" + name, wl.grad, *want["dw"])


def grid(height, width):
    return torch.cartesian_prod(torch.arange(height), torch.arange(width))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("d", [2, 4, 6, 16, 36, 64, 72, 80, 100, 128, 130, 256])
def test_head_dims(d, norm, interleaved, dtype):
    check(2, 15, 3, 2, d, dtype, (d // 4, d // 2 - d // 4), grid(3, 5), norm, interleaved=interleaved, seed=d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,n,h,hk", [(1, 1, 1, 1), (1, 1, 40, 3), (5, 1, 8, 2), (1, 7, 1, 16), (3, 333, 12, 12),
                                      (70, 77, 2, 1)])
def test_sizes(b, n, h, hk, dtype):
    check(b, n, h, hk, 64, dtype, (32,), torch.arange(n)[:, None] + 5, seed=n)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_positions(kind):
    """Of three axes, one with no pairs, for each batch entry, negative, far away, and fractions."""
    g = torch.Generator().manual_seed(1)
    p = torch.randint(-1000000, 1000000, (3, 20, 4), generator=g).to(kind)
    if kind == torch.float32:
        p = p / 64
    check(3, 20, 2, 2, 64, torch.float32, (10, 0, 12, 10), p, theta=100.0)
    check(3, 20, 2, 2, 64, torch.float32, (10, 0, 12, 10), p[0], theta=5e5)


def test_frequencies():
    """Given ones; a frequency of 0 leaves its pairs as they are."""
    f = ref.frequencies((16,), 10000.0)
    f[8:] = 0.0
    for kind in (torch.float64, torch.float32):
        check(2, 9, 2, 1, 32, torch.float32, (16,), torch.arange(9)[:, None], False, frequencies=f.to(kind))
    x = torch.randn(2, 9, 2, 32, device=DEV)
    y, _ = mec.norm_rotary(x, x, torch.arange(9, device=DEV)[:, None], (16,), frequencies=f.to(DEV))
    kept = torch.arange(32).remainder(16) >= 8
    assert torch.equal(y[..., kept], x[..., kept]) and not torch.equal(y, x)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    def odd(t):
        room = torch.zeros(t.numel() // t.shape[-1] * (t.shape[-1] + 3) + 1, dtype=t.dtype, device=DEV)[1:]
        return room.view(*t.shape[:-1], t.shape[-1] + 3)[..., 2:-1].copy_(t)

    first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    columns = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)  # noqa: E731
    for leaves in (odd, first, columns):
        for interleaved in (False, True):
            check(2, 21, 4, 2, 64, dtype, (16, 16), grid(3, 7), leaves=leaves, interleaved=interleaved)


@pytest.mark.parametrize("wtype", TYPES)
def test_weights_of_another_type(wtype):
    check(2, 50, 4, 2, 64, torch.bfloat16, (32,), torch.arange(50)[:, None], wtype=wtype)


def test_a_norm_without_weights_and_one_side_alone():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 30, 4, 40, generator=g)
    pos = torch.arange(30)[:, None]
    q, k = (x.to(DEV).requires_grad_(True) for _ in "qk")
    w = torch.ones(40, device=DEV, requires_grad=True)
    y, _ = mec.norm_rotary(q, k, pos.to(DEV), (20,), None, w, eps=1e-5)
    dy = torch.randn(y.shape, generator=g)
    y.backward(dy.to(DEV))
    want = ref.norm_rotary(x, pos, (20,), None, 1e-5, dy=dy)
    ref.close("y", y, *want["y"])
    ref.close("dx", q.grad, *want["dx"])
    assert k.grad is None and w.grad is None
    # the weight alone
    _, z = mec.norm_rotary(q.detach(), k.detach(), pos.to(DEV), (20,), None, w, eps=1e-5)
    z.backward(dy.to(DEV))
    ref.close("dw", w.grad, *ref.norm_rotary(x, pos, (20,), torch.ones(40), 1e-5, dy=dy)["dw"])


def test_gradients_are_differences():
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(1, 6, 2, 16, generator=g).to(DEV) for _ in "xy")
    w = (1 + 0.1 * torch.randn(16, generator=g)).to(DEV)
    pos = torch.arange(6, device=DEV)[:, None]
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]

    def f(x, w):
        return mec.norm_rotary(x, x, pos, (8,), w, w, eps=1e-6)[0]

    y = f(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    size = (y.double().abs() * dy.double().abs()).sum().detach()
    h = 2.0 ** -7
    with torch.no_grad():
        for i in range(2):
            step = torch.randn(leaves[i].shape, generator=g).to(DEV)
            ends = [(f(*(t + s * h * step if j == i else t for j, t in enumerate(leaves))).double() * dy.double()).sum()
                    for s in (1, -1)]
            want = (grads[i].double() * step.double()).sum()
            assert abs((ends[0] - ends[1]) / (2 * h) - want) <= h * h * 20 * size + 64 * ref.E * size / h


def test_the_same_bits_again():
    g = torch.Generator().manual_seed(4)
    x, dy = (torch.randn(9, 100, 6, 64, generator=g).to(DEV, torch.bfloat16) for _ in "xy")
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    runs = []
    for _ in range(3):
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        y = mec.norm_rotary(leaves[0], x, torch.arange(100, device=DEV)[:, None], (32,), leaves[1], None, eps=1e-6)[0]
        y.backward(dy)
        runs.append([y.detach(), *(t.grad for t in leaves)])
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))


def test_no_tokens():
    x = torch.zeros(2, 0, 4, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    q, k = mec.norm_rotary(x, x, torch.zeros(0, 1, device=DEV, dtype=torch.int64), (4,), w, w, eps=1e-6)
    (q.sum() + k.sum()).backward()
    assert q.shape == k.shape == x.shape and x.grad.shape == x.shape and not w.grad.any()

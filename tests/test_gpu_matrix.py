"""GPU parity of the matrix operators against plain 64-bit arithmetic: dense layer forward and backward, orthogonalisation,
optimizer step, and a training run of them together.

Tolerances are worst-case bounds of the arithmetic, element by element.  float32 products use pairs of fp16 numbers: each
factor is off by at most 2^-22 of itself (two half steps of 2^-11) and the product of the two low parts, another 2^-22, is
left out; bfloat16 products are exact.  A float32 sum of K products is off by at most K 2^-24 of the sum of magnitudes.
Results are rounded by half a step, torch.finfo(t).eps / 2."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
PAIR = {torch.float32: 3 * 2.0 ** -22, torch.bfloat16: 0.0}


@pytest.fixture(scope='module')
def mx():
    from objectdetection_amd import matrix
    return matrix


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(1000 + seed)
    return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dtype)


def act64(z, act):
    f = torch.nn.functional
    return {None: lambda t: t, 'silu': f.silu, 'gelu': f.gelu, 'relu': f.relu}[act](z)


def slope64(z, act):
    z = z.clone().requires_grad_()
    return torch.autograd.grad(act64(z, act).sum(), z)[0] if act else torch.ones_like(z)


def product_bound(a, b, dtype):
    """|error| of a b^T: a (m, k), b (n, k) in 64 bits."""
    k = a.shape[1]
    return (PAIR[dtype] + (k + 8) * 2.0 ** -24) * (a.abs() @ b.abs().t())


def close(got, ref, bound, dtype):
    got = got.double()
    assert got.shape == ref.shape
    err, allowed = (got - ref).abs(), bound + HALF[dtype] * ref.abs() + 1e-30
    assert bool(torch.isfinite(got).all())
    worst = float((err / allowed).max()) if err.numel() else 0.0
    assert worst <= 1.0, f'{worst:.3g} of the allowed error'


def forward_reference(x, w, b, act, r):
    x, w = x.double(), w.double()
    z = x @ w.t() + (b.double() if b is not None else 0)
    y = act64(z, act) + (r.double() if r is not None else 0)
    return z, y


def forward_bound(x, w, b, act, r, z, dtype):
    e = product_bound(x.double(), w.double(), dtype) + 2.0 ** -23 * z.abs()
    # no activation is steeper than 1.13; the float32 activation and the sum with r are off by a few steps
    return 1.13 * e + 16 * 2.0 ** -24 * (z.abs() + 1) + (2.0 ** -23 * r.double().abs() if r is not None else 0)


def check_linear(mx, x, w, b, act, r, backward=True):
    dtype = x.dtype
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b, r)]
    x, w, b, r = leaves
    z, y64 = forward_reference(x.detach(), w.detach(), None if b is None else b.detach(), act, None if r is None else r.detach())
    fb = forward_bound(x.detach(), w.detach(), b, act, None if r is None else r.detach(), z, dtype)
    with torch.no_grad():
        close(mx.linear(x, w, b, act, r), y64, fb, dtype)
    if not backward:
        return
    y = mx.linear(x, w, b, act, r)
    close(y.detach(), y64, fb, dtype)
    dy = randn(*y.shape, seed=77, dtype=dtype)
    wanted = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip('xwbr', leaves) if t is not None], torch.autograd.grad(y, wanted, dy)))
    x64, w64, d64 = x.detach().double(), w.detach().double(), dy.double()
    dz = d64 * slope64(z, act)
    ez = product_bound(x64, w64, dtype) + (2.0 ** -23 + HALF[dtype]) * z.abs() + 2.0 ** -23
    # slopes change by at most 0.8 per unit of z (silu 0.5, gelu 0.8); relu's jumps where z may have either sign
    edz = d64.abs() * (0.8 * ez + 16 * 2.0 ** -24 * (1 + z.abs())) if act else torch.zeros_like(dz)
    if act == 'relu':
        edz = d64.abs() * (z.abs() <= ez)
    db_bound = edz.sum(0) + (dz.shape[0] + 8) * 2.0 ** -24 * dz.abs().sum(0)
    if dtype == torch.bfloat16 and act:
        edz = edz + HALF[dtype] * (dz.abs() + edz)
    close(grads['x'], dz @ w64, product_bound(dz.abs() + edz, w64.t().contiguous(), dtype) + edz @ w64.abs(), dtype)
    close(grads['w'], dz.t().contiguous() @ x64,
          product_bound((dz.abs() + edz).t().contiguous(), x64.t().contiguous(), dtype) + edz.t().contiguous() @ x64.abs(), dtype)
    if b is not None:
        close(grads['b'], dz.sum(0), db_bound, dtype)
    if r is not None:
        assert torch.equal(grads['r'], dy)


SIZES = [(1, 1, 1), (1, 64, 40), (2, 7, 3), (3, 130, 65), (7, 129, 9), (8, 256, 130), (9, 64, 64), (17, 33, 31), (33, 8, 200),
         (64, 64, 64), (65, 200, 63), (129, 72, 257), (300, 1000, 20), (1000, 24, 300)]
# more than 4096 workgroups of eight rows and four columns: on matrix instructions in either type
SIZES += [(600, 33, 257), (2000, 7, 80), (5000, 130, 29), (700, 64, 200), (10, 40, 9001), (40001, 1, 4), (513, 255, 256),
          (1, 40001, 5), (2, 33000, 24), (9, 40000, 24)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m, k, n', SIZES)
def test_linear_against_64_bits(mx, m, k, n, dtype):
    acts = [None, 'silu', 'gelu', 'relu']
    act = acts[(m + k + n) % 4]
    x, w = randn(m, k, dtype=dtype), randn(n, k, seed=1, dtype=dtype, scale=k ** -0.5)
    check_linear(mx, x, w, randn(n, seed=2, dtype=dtype), act, randn(m, n, seed=3, dtype=dtype))
    check_linear(mx, x, w, None, acts[(m + k + n + 1) % 4], None)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('act', [None, 'silu', 'gelu', 'relu'])
def test_linear_activations(mx, act, dtype):
    for m in (5, 70):
        x, w = randn(m, 96, dtype=dtype, scale=3.0), randn(80, 96, seed=1, dtype=dtype, scale=0.2)
        check_linear(mx, x, w, randn(80, seed=2, dtype=dtype), act, randn(m, 80, seed=3, dtype=dtype))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m, k, n', [(2100, 264, 2050), (4000, 96, 4100), (50, 4000, 72), (4097, 300, 1001), (2056, 520, 2000)])
def test_linear_tiles_and_split(mx, m, k, n, dtype):
    """Sizes that reach the 128 and 256 wide tiles and the split reduction, ragged in every direction."""
    x, w = randn(m, k, dtype=dtype), randn(n, k, seed=1, dtype=dtype, scale=k ** -0.5)
    check_linear(mx, x, w, randn(n, seed=2, dtype=dtype), 'silu', randn(m, n, seed=3, dtype=dtype))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m, k, n', [(9000, 136, 520), (5001, 129, 131), (2100, 263, 2049), (70, 1500, 3001), (2500, 1030, 1033)])
def test_linear_long_reductions_backward(mx, m, k, n, dtype):
    """dW and db of many rows, dx of many outputs: one of the two products cut, or both, aligned and not."""
    x, w = randn(m, k, dtype=dtype), randn(n, k, seed=1, dtype=dtype, scale=k ** -0.5)
    b = randn(n, seed=2, dtype=dtype)
    check_linear(mx, x, w, b, 'gelu', None)
    check_linear(mx, x, w, b, None, randn(m, n, seed=3, dtype=dtype))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m', [4, 40, 3000])
def test_linear_strides_and_offsets(mx, m, dtype):
    """Slices of wider buffers, unaligned starts, transposed and expanded views."""
    k, n = 72, 48
    wide = randn(m, k + 24, dtype=dtype)
    w = randn(n, k, seed=1, dtype=dtype, scale=0.1)
    for x in (wide[:, :k], wide[:, 8:8 + k], wide[:, 3:3 + k], randn(k, m, seed=5, dtype=dtype).t(),
              randn(1, k, seed=6, dtype=dtype).expand(m, k), randn(2 * m, k, seed=7, dtype=dtype)[::2]):
        check_linear(mx, x, w, None, 'silu', None)
    check_linear(mx, wide[:, :k], randn(k, n, seed=8, dtype=dtype, scale=0.1).t(), randn(2 * n, seed=9, dtype=dtype)[::2],
                 'gelu', randn(n, m, seed=10, dtype=dtype).t())
    flat = randn(m * k + 1, seed=11, dtype=dtype)[1:].view(m, k)
    check_linear(mx, flat, w, randn(n + 1, seed=12, dtype=dtype)[1:], 'relu', randn(m * n + 1, seed=13, dtype=dtype)[1:].view(m, n))
    # a gradient without memory of its own (a sum's), and one in another order
    x = wide[:, :k].detach().requires_grad_()
    mx.linear(x, w, None, 'silu').sum().backward()
    z = x.detach().double() @ w.double().t()
    ref = slope64(z, 'silu') @ w.double()
    assert float((x.grad.double() - ref).norm() / ref.norm()) < 4 * HALF[dtype] + 1e-5


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m, k, n', [(5, 40, 24), (33, 24, 41), (3000, 72, 200), (2100, 520, 1000)])
def test_linear_entry_points_write_within_their_rows(mx, m, k, n, dtype):
    """Rows of results further apart than they are long, the residual in the place of the result: what lies between stays."""
    from objectdetection_amd import _lib
    from objectdetection_amd._lib import lib, check
    code, ztype = (0, torch.float32) if dtype == torch.float32 else (1, torch.float16)
    st = torch.cuda.current_stream().cuda_stream
    x, w, b = randn(m, k, dtype=dtype), randn(n, k, seed=1, dtype=dtype, scale=k ** -0.5), randn(n, seed=2, dtype=dtype)
    r = randn(m, n, seed=3, dtype=dtype)
    y = torch.full((m, n + 5), 7.0, dtype=dtype, device='cuda')
    z = torch.full((m, n + 3), 7.0, dtype=ztype, device='cuda')
    y[:, :n] = r
    d = _lib.LinearDesc(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), y.data_ptr(), z.data_ptr(), k, k, n + 5, n + 5, n + 3,
                        m, k, n, 1, code)
    size = lib.odamd_linear_workspace_bytes(d)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device='cuda')
    check(lib.odamd_linear_forward(d, ws.data_ptr(), size, st))
    z64, y64 = forward_reference(x, w, b, 'silu', r)
    bound = forward_bound(x, w, b, 'silu', r, z64, dtype)
    close(y[:, :n], y64, bound, dtype)
    close(z[:, :n].float(), z64, bound + (2.0 ** -11 * z64.abs() + 2.0 ** -24 if dtype == torch.bfloat16 else 0), torch.float32)
    assert bool((y[:, n:] == 7).all()) and bool((z[:, n:] == 7).all())
    dy = randn(m, n, seed=4, dtype=dtype)
    dx = torch.full((m, k + 3), 7.0, dtype=dtype, device='cuda')
    dw = torch.full((n, k + 6), 7.0, dtype=dtype, device='cuda')
    db = torch.full((n + 8,), 7.0, dtype=dtype, device='cuda')
    g = _lib.LinearGradDesc(dy.data_ptr(), z.data_ptr(), x.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                            n, n + 3, k, k, k + 3, k + 6, m, k, n, 1, code)
    size = lib.odamd_linear_backward_workspace_bytes(g)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device='cuda')
    check(lib.odamd_linear_backward(g, ws.data_ptr(), size, st))
    plain = mx._linear_backward(dy, z[:, :n].contiguous(), x, w, 1, True, True, True)
    assert torch.equal(dx[:, :k], plain[0]) and torch.equal(dw[:, :k], plain[1]) and torch.equal(db[:n], plain[2])
    assert bool((dx[:, k:] == 7).all()) and bool((dw[:, k:] == 7).all()) and bool((db[n:] == 7).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m, k, n', [(1, 72, 48), (7, 71, 45), (40, 72, 48), (3000, 72, 48), (3001, 71, 45), (2100, 520, 1000)])
def test_linear_reads_nothing_beside_its_operands(mx, m, k, n, dtype):
    """Operands in buffers that hold NaN everywhere else."""
    def island(rows, cols, seed, scale=1.0):
        sea = torch.full((rows + 4, cols + 24), float('nan'), dtype=dtype, device='cuda')
        sea[2:rows + 2, 8:cols + 8] = randn(rows, cols, seed=seed, dtype=dtype, scale=scale)
        return sea[2:rows + 2, 8:cols + 8].detach().requires_grad_()
    x, w, r = island(m, k, 0), island(n, k, 1, k ** -0.5), island(m, n, 2)
    b = island(1, n, 3)
    for act in (None, 'gelu'):
        y = mx.linear(x, w, b[0], act, r)
        grads = torch.autograd.grad(y, (x, w, b, r), island(m, n, 4).detach())
        copies = [t.detach().clone().requires_grad_() for t in (x, w, b, r)]
        y2 = mx.linear(copies[0], copies[1], copies[2][0], act, copies[3])
        grads2 = torch.autograd.grad(y2, copies, island(m, n, 4).detach().clone())
        y, y2 = y.detach(), y2.detach()
        assert torch.isfinite(y).all() and float((y - y2).norm()) <= (HALF[dtype] + 1e-5) * float(y2.norm())
        for g, h in zip(grads, grads2):
            assert torch.isfinite(g).all() and float((g - h).norm()) <= (2 * HALF[dtype] + 1e-5) * float(h.norm())


def test_linear_shapes_of_more_axes(mx):
    x, w, b = randn(2, 3, 5, 40), randn(24, 40, seed=1), randn(24, seed=2)
    y = mx.linear(x, w, b, 'silu')
    assert y.shape == (2, 3, 5, 24)
    assert torch.equal(y.view(-1, 24), mx.linear(x.view(-1, 40), w, b, 'silu'))
    one = mx.linear(x[0, 0, 0], w, b, 'silu')
    assert one.shape == (24,)
    z = x[0, 0, 0].double() @ w.double().t() + b.double()
    close(one, act64(z, 'silu'), forward_bound(x[0, 0, :1], w, b, 'silu', None, z[None], torch.float32)[0], torch.float32)
    for lead in ((0,), (2, 0)):
        x0 = torch.zeros(*lead, 40, device='cuda', requires_grad=True)
        w0 = w.clone().requires_grad_()
        y0 = mx.linear(x0, w0, b, 'silu')
        assert y0.shape == lead + (24,)
        y0.sum().backward()
        assert x0.grad.shape == x0.shape and float(w0.grad.abs().max()) == 0.0


@pytest.mark.parametrize('m', [3, 30])
def test_linear_float32_keeps_the_range(mx, m):
    """Rows of very different magnitude, the smallest and the largest: every row keeps its 22 bits."""
    k, n = 200, 50
    scale = torch.logspace(-36, 17, m, device='cuda', dtype=torch.float64)
    x = (randn(m, k).double() * scale[:, None]).float()
    w = (randn(n, k, seed=1).double() * torch.logspace(-3, 18, n, device='cuda', dtype=torch.float64)[:, None]).float()
    ref = x.double() @ w.double().t()
    close(mx.linear(x, w), ref, product_bound(x.double(), w.double(), torch.float32) + 2.0 ** -149, torch.float32)
    x[m // 2] = 0
    assert float(mx.linear(x, w)[m // 2].abs().max()) == 0.0
    # what is no number stays in its row
    x[1, 5] = float('nan')
    x[2, 7] = float('inf')
    y = mx.linear(x, w)
    assert bool(torch.isnan(y[1]).all()) and not bool(torch.isfinite(y[2]).any())
    keep = [i for i in range(m) if i not in (1, 2)]
    assert bool(torch.isfinite(y[keep]).all())


def test_linear_only_wanted_gradients(mx):
    x, w, b = randn(20, 40), randn(24, 40, seed=1), randn(24, seed=2)
    dy = randn(20, 24, seed=3)
    full = torch.autograd.grad(mx.linear(*(t.requires_grad_() for t in (x, w, b)), 'silu'), (x, w, b), dy)
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == q) for q, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(mx.linear(*leaves, 'silu'), leaves[i], dy)
        assert torch.equal(got, full[i])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m, k, n', [(3000, 40, 72), (4100, 520, 264)])
def test_linear_only_wanted_gradients_of_products(mx, m, k, n, dtype):
    """Each gradient alone takes other paths than all of them together: within two roundings and 2^-16 of each other."""
    tensors = [randn(m, k, dtype=dtype), randn(n, k, seed=1, dtype=dtype, scale=0.1), randn(n, seed=2, dtype=dtype)]
    dy = randn(m, n, seed=3, dtype=dtype)
    for act in (None, 'silu'):
        leaves = [t.detach().requires_grad_() for t in tensors]
        full = torch.autograd.grad(mx.linear(*leaves, act), leaves, dy)
        for wanted in ([0], [1], [2], [0, 1], [0, 2], [1, 2]):
            leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate(tensors)]
            got = torch.autograd.grad(mx.linear(*leaves, act), [leaves[i] for i in wanted], dy)
            for i, g in zip(wanted, got):
                assert float((g.double() - full[i].double()).norm()) <= (2 * HALF[dtype] + 2.0 ** -16) * float(full[i].double().norm())


def test_linear_keeps_the_slope_of_large_values(mx):
    """Pre-activations past float16's range: every activation is straight there, slopes are 0 and 1."""
    for dtype in (torch.float32, torch.bfloat16):
        x, w = randn(24, 8, dtype=dtype).abs() + 1, randn(40, 8, seed=1, dtype=dtype).abs() + 1
        w[::2] = -w[::2]
        x = (x * 2.0 ** 17).requires_grad_()
        dy = randn(24, 40, seed=2, dtype=dtype)
        for act in ('silu', 'gelu', 'relu'):
            dx, = torch.autograd.grad(mx.linear(x, w, None, act), x, dy)
            open_ = dy.clone()
            open_[:, ::2] = 0
            ref = open_.double() @ w.double()
            close(dx, ref, product_bound(open_.double(), w.double().t().contiguous(), dtype), dtype)


def test_linear_relu_at_any_scale(mx):
    """relu asks for the sign of the smallest pre-activations too."""
    for dtype in (torch.float32, torch.bfloat16):
        for m in (6, 3000):
            x, w, dy = randn(m, 24, dtype=dtype), randn(40, 24, seed=1, dtype=dtype), randn(m, 40, seed=2, dtype=dtype)
            grads = []
            for scale in (1.0, 2.0 ** -30):
                leaf = (x * scale).requires_grad_()
                grads.append(torch.autograd.grad(mx.linear(leaf, w * 2.0 ** -8, None, 'relu'), leaf, dy)[0])
            assert torch.equal(*grads)


def test_linear_relu_closes_the_gradient(mx):
    """Where relu is closed nothing passes, an infinity neither; other rows and columns do not see it."""
    for dtype in (torch.float32, torch.bfloat16):
        x, w = randn(30, 40, dtype=dtype).abs(), randn(24, 40, seed=1, dtype=dtype).abs()
        w[3] = -w[3]
        leaves = [x.requires_grad_(), w.requires_grad_()]
        dy = randn(30, 24, seed=2, dtype=dtype)
        dy[:, 3] = float('inf')
        dx, dw = torch.autograd.grad(mx.linear(*leaves, activation='relu'), leaves, dy)
        clean = dy.clone()
        clean[:, 3] = 0
        rx, rw = torch.autograd.grad(mx.linear(*leaves, activation='relu'), leaves, clean)
        assert torch.equal(dx, rx) and torch.equal(dw, rw) and float(dw[3].abs().max()) == 0.0


def test_linear_differentiates_once(mx):
    leaves = [t.requires_grad_() for t in (randn(20, 40), randn(24, 40, seed=1), randn(24, seed=2), randn(20, 24, seed=3))]
    first = torch.autograd.grad(mx.linear(*leaves[:3], 'silu', leaves[3]).square().sum(), leaves)
    second = torch.autograd.grad(mx.linear(*leaves[:3], 'silu', leaves[3]).square().sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match='once_differentiable'):
        second[0].sum().backward()


def test_linear_gradient_against_differences(mx):
    """float32, central differences of the 64-bit layer along random directions."""
    x, w, b = randn(33, 20), randn(17, 20, seed=1), randn(17, seed=2)
    for act in ('silu', 'gelu'):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        dy = randn(33, 17, seed=4)
        grads = torch.autograd.grad(mx.linear(*leaves, act), leaves, dy)
        for q in range(3):
            d = randn(*leaves[q].shape, seed=20 + q).double()
            h = 1e-4
            vals = []
            for s in (h, -h):
                a = [t.detach().double() for t in leaves]
                a[q] = a[q] + s * d
                vals.append(float((act64(a[0] @ a[1].t() + a[2], act) * dy.double()).sum()))
            slope, got = (vals[0] - vals[1]) / (2 * h), float((grads[q].double() * d).sum())
            size = float((grads[q].double().abs() * d.abs()).sum())
            # truncation: h^2 / 6 of a third derivative of order one per element; arithmetic: 2^-20 of the magnitudes
            assert abs(slope - got) <= (2.0 ** -20 + 100 * h * h) * size


def test_linear_refuses(mx):
    x, w = randn(4, 8), randn(6, 8, seed=1)
    for bad in (dict(x=x.half()), dict(weight=w.bfloat16()), dict(weight=w[0]), dict(weight=randn(6, 9)), dict(bias=randn(5)),
                dict(bias=randn(6).bfloat16()), dict(residual=randn(4, 5)), dict(residual=randn(1, 6)), dict(weight=w.cpu()),
                dict(activation='swish'), dict(weight=w[:, :0], x=x[:, :0]), dict(x=x[:1, :1].expand(2 ** 31, 1), weight=w[:, :1])):
        with pytest.raises(ValueError):
            mx.linear(**dict(dict(x=x, weight=w), **bad))


# ---------------------------------------------------------------------------------------------
# orthogonalisation
# ---------------------------------------------------------------------------------------------
def orth64(g, steps=5, eps=1e-7):
    a, b, c = NS
    x = g.double()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if tall else x


# A step multiplies a small singular value by 3.4445: five of them multiply the half step of float32 by 485.  Where five steps
# run on A = X X^T (bfloat16 results, the optimizer step), a half step of A is multiplied by 3.4445^2 in four of them and
# enters P / a = 1 - (4.7750 / 3.4445) A + ... of the last.
LOOSE = 4.7750 / 3.4445 * 3.4445 ** 8 * 2.0 ** -24
ORTH_TOL = {torch.float32: 3.4445 ** 5 * 2.0 ** -24, torch.bfloat16: LOOSE + 2.0 ** -8}


def check_orth(got, g, **kw):
    for i in range(g.shape[0]):
        ref = orth64(g[i], **kw)
        assert float((got[i].double() - ref).norm()) <= ORTH_TOL[g.dtype] * float(ref.norm())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('batch, rows, cols', [(1, 1, 1), (3, 1, 7), (3, 7, 1), (1, 16, 27), (1, 27, 16), (2, 33, 31), (2, 64, 64), (1, 65, 130),
                                               (3, 130, 65), (1, 128, 1152), (1, 255, 257), (5, 300, 40), (1, 1000, 333), (140, 20, 50)])
def test_orthogonalize_against_64_bits(mx, batch, rows, cols, dtype):
    g = randn(batch, rows, cols, dtype=dtype, scale=1e-3)
    check_orth(mx.orthogonalize(g), g)


def test_orthogonalize_large_tiles(mx):
    for batch, rows, cols in ((1, 2100, 2300), (6, 1050, 1100)):
        g = randn(batch, rows, cols)
        check_orth(mx.orthogonalize(g), g)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('batch, rows, cols', [(1, 70, 4000), (1, 4001, 70), (3, 129, 2049), (8, 256, 1200), (1, 257, 9000), (1, 500, 20011), (2, 1025, 4100)])
def test_orthogonalize_long_reductions(mx, batch, rows, cols, dtype):
    """Few tiles of X X^T and a long reduction: it is cut into parts."""
    g = randn(batch, rows, cols, dtype=dtype)
    got = mx.orthogonalize(g)
    check_orth(got, g)
    assert torch.equal(mx.orthogonalize(g), got)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('batch, rows, cols', [
    (3, 1, 1023), (2, 1, 1025), (1, 1, 70001), (2, 1500, 2), (40, 5, 1024), (2, 5, 4264), (1, 16, 16), (1, 16, 40000), (3, 17, 512),
    (2, 33000, 31), (2, 32, 513), (1, 32, 1030), (3, 33, 341), (2, 342, 33), (1, 48, 343), (2, 45, 9000), (5, 49, 63), (2, 64, 256),
    (300, 64, 70), (2, 257, 64), (3, 61, 1001), (1, 20000, 64)])
def test_orthogonalize_few_rows(mx, batch, rows, cols, dtype):
    """Up to 64 rows: 64-bit arithmetic, in one workgroup or in parts.  Five steps multiply a rounding by 3e4 at most, 2^-53 to
    4e-12: what is left is the rounding of the result."""
    g = randn(batch, rows, cols, dtype=dtype, scale=1e-3)
    got = mx.orthogonalize(g)
    for i in {0, batch // 2, batch - 1}:
        ref = orth64(g[i])
        assert float((got[i].double() - ref).norm()) <= (HALF[dtype] + 1e-10) * float(ref.norm())
    assert torch.equal(mx.orthogonalize(g), got)


def test_orthogonalize_few_rows_of_no_rank(mx):
    """Equal and zero rows, ten steps: directions without a singular value stay at zero (a rounding of A, 2^-53, grows by
    3.4445^2 a step and is seen under a root)."""
    g = randn(2, 40, 300)
    g[0, 7:] = g[0, 3]
    g[1, :, 50:] = 0
    g[1, 10:20] = 0
    for steps in (1, 5, 10):
        got = mx.orthogonalize(g, steps=steps)
        for i in range(2):
            ref = orth64(g[i], steps=steps)
            assert float((got[i].double() - ref).norm()) <= (2.0 ** -24 + 3.4445 ** (2 * steps) * 2.0 ** -53 * 40) * float(ref.norm())
    assert float(mx.orthogonalize(g)[1, 10:20].abs().max()) == 0.0


@pytest.mark.parametrize('rows, cols', [(30, 50), (90, 100), (90, 400), (150, 2000)])
def test_orthogonalize_more_steps(mx, rows, cols):
    """Up to two phases of five steps and a rest; a step leaves an error of a product and multiplies what came before by 3.4445
    at most, a geometric sum of 1 / (1 - 1 / 3.4445) = 1.41 times its last term."""
    g = randn(1, rows, cols)
    for steps in (1, 2, 3, 4, 6, 7, 12):
        ref, size = orth64(g[0], steps=steps), orth64(g[0], steps=steps).norm()
        grown = 3.4445 ** min(steps, 7)                 # the smallest singular values here pass one within seven steps
        assert float((mx.orthogonalize(g, steps=steps)[0].double() - ref).norm()) <= 1.41 * grown * PAIR[torch.float32] * float(size) + 1e-30
        low = g.bfloat16()
        ref = orth64(low[0], steps=steps)
        loose = LOOSE * 3.4445 ** max(0, min(steps, 7) - 5)
        assert float((mx.orthogonalize(low, steps=steps)[0].double() - ref).norm()) <= (loose + 2.0 ** -8) * float(ref.norm())


@pytest.mark.parametrize('rows, cols', [(20, 30), (100, 333)])
def test_orthogonalize_ends_of_the_range(mx, rows, cols):
    """Norms over and under float32's range, subnormal values: the norm is held in 64 bits."""
    for scale in (2.0 ** 124, 2.0 ** -128, 2.0 ** -140):
        g = randn(1, rows, cols)
        g = (g / g.abs().max()).double().mul(scale).float()
        check_orth(mx.orthogonalize(g, eps=0.0), g, eps=0.0)
    g = randn(1, rows, cols, dtype=torch.bfloat16) * 2.0 ** 123
    check_orth(mx.orthogonalize(g, eps=0.0), g, eps=0.0)


def test_orthogonalize_brings_singular_values_near_one(mx):
    g = randn(1, 96, 300)
    s = torch.linalg.svdvals(mx.orthogonalize(g)[0].cpu().double())
    assert float(s.min()) > 0.6 and float(s.max()) < 1.25


def test_orthogonalize_forms(mx):
    g = randn(4, 40, 24)
    whole = mx.orthogonalize(g)
    assert torch.equal(mx.orthogonalize(g.view(2, 2, 40, 24)).view(4, 40, 24), whole)
    assert torch.equal(mx.orthogonalize(g[2]), whole[2])
    assert torch.equal(mx.orthogonalize(g), whole)                                  # the same bits every time
    assert torch.equal(mx.orthogonalize(g.transpose(1, 2).contiguous().transpose(1, 2)), whole)
    twin = g.clone()
    assert mx.orthogonalize(twin, out=twin) is twin and torch.equal(twin, whole)    # in place
    off = torch.empty(4 * 40 * 24 + 1, device='cuda')[1:].view(4, 40, 24)           # unaligned source and result
    off.copy_(g)
    assert torch.equal(mx.orthogonalize(off, out=off), whole)
    check_orth(mx.orthogonalize(g, steps=1), g, steps=1)
    check_orth(mx.orthogonalize(g, steps=3, eps=0.5), g, steps=3, eps=0.5)
    # scale does not matter, also where squares leave float32's range
    for s in (1e-18, 1e25):
        assert float((mx.orthogonalize(g * s, eps=0.0) - mx.orthogonalize(g, eps=0.0)).norm() / whole.norm()) < 2 * ORTH_TOL[torch.float32]
    assert mx.orthogonalize(g[:0]).shape == (0, 40, 24)
    for bad in (g[0, 0], g.half(), g.cpu()):
        with pytest.raises(ValueError):
            mx.orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=40), dict(eps=-1.0), dict(out=whole[:2]), dict(out=whole.transpose(1, 2)), dict(out=whole.bfloat16())):
        with pytest.raises(ValueError):
            mx.orthogonalize(g, **kw)


def test_orthogonalize_zero_and_no_numbers(mx):
    g = randn(5, 40, 70)
    g[1] = 0
    g[2, 3, 4] = float('nan')
    g[3, 39, 69] = float('inf')
    y = mx.orthogonalize(g)
    assert float(y[1].abs().max()) == 0.0
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3]).all())
    check_orth(y[[0, 4]], g[[0, 4]])


# ---------------------------------------------------------------------------------------------
# optimizer step
# ---------------------------------------------------------------------------------------------
def muon64(p, g, m, e, matrices, lr, mu, nesterov, wd, d, gs):
    p, g, m = p.double(), g.double() * gs, m.double()
    e = None if e is None else e.double()
    for o, r, c in matrices:
        s = slice(o, o + r * c)
        m[s] = mu * m[s] + g[s]
        u = g[s] + mu * m[s] if nesterov else m[s]
        p[s] = p[s] * (1 - lr * wd) - lr * 0.2 * math.sqrt(max(r, c)) * orth64(u.view(r, c)).reshape(-1)
        if e is not None:
            e[s] = d * e[s] + (1 - d) * p[s]
    return p, m, e


@pytest.mark.parametrize('ema, nesterov', [(True, True), (False, False)])
def test_muon_step_against_64_bits(mx, ema, nesterov):
    shapes = [(16, 27), (32, 64), (1, 5), (5, 1), (33, 7), (64, 576), (130, 129), (3, 3)]
    matrices, at = [], 4
    for i, (r, c) in enumerate(shapes):
        matrices.append((at, r, c))
        at += r * c + (i % 3) * 5                       # odd offsets too, and gaps
    p, g, m = randn(at + 9, scale=0.03), randn(at + 9, seed=1, scale=1e-3), randn(at + 9, seed=2, scale=1e-3)
    e = randn(at + 9, seed=3, scale=0.03) if ema else None
    args = (0.01, 0.9, nesterov, 0.1, 0.7, 0.5)
    rp, rm, re = muon64(p, g, m, e, matrices, *args)
    p1, g1, m1, e1 = p.clone(), g.clone(), m.clone(), None if e is None else e.clone()
    mx.muon_step(p1, g1, m1, matrices, lr=0.01, momentum_decay=0.9, nesterov=nesterov, weight_decay=0.1, ema=e1, ema_decay=0.7,
                 grad_scale=0.5)
    assert torch.equal(g1, g)
    assert float((m1.double() - rm).abs().max()) <= 4 * 2.0 ** -24 * float(rm.abs().max())
    covered = torch.zeros_like(p, dtype=torch.bool)
    for o, r, c in matrices:
        s = slice(o, o + r * c)
        covered[s] = True
        step = 0.01 * 0.2 * math.sqrt(r * c) * 1.25     # Frobenius norm of the update, at most: singular values under 1.25
        allowed = LOOSE * step + 4 * 2.0 ** -24 * float(rp[s].norm())
        assert float((p1[s].double() - rp[s]).norm()) <= allowed
        if ema:
            assert float((e1[s].double() - re[s]).norm()) <= allowed + 4 * 2.0 ** -24 * float(re[s].norm())
    for new, old in ((p1, p), (m1, m)) + (((e1, e),) if ema else ()):
        assert torch.equal(new[~covered], old[~covered])                         # what lies between stays
    # the same bits again
    p2, m2 = p.clone(), m.clone()
    mx.muon_step(p2, g, m2, mx.MatrixTable(matrices), lr=0.01, momentum_decay=0.9, nesterov=nesterov, weight_decay=0.1, grad_scale=0.5)
    assert torch.equal(p2, p1) and torch.equal(m2, m1)


def test_muon_step_many_matrices(mx):
    """More matrices than one launch's table holds."""
    matrices = [(i * 64, 8, 8) for i in range(300)]
    p, g, m = randn(300 * 64), randn(300 * 64, seed=1), torch.zeros(300 * 64, device='cuda')
    rp, rm, _ = muon64(p, g, m, None, matrices, 0.1, 0.95, True, 0.0, 0.0, 1.0)
    mx.muon_step(p, g, m, matrices, lr=0.1)
    # 300 updates of norm 0.1 * 0.2 * sqrt(8 * 8) * 1.25 at most, each off by LOOSE of itself, and the roundings of p
    assert float((p.double() - rp).norm()) <= LOOSE * 0.1 * 0.2 * 8 * 1.25 * math.sqrt(300) + 4 * 2.0 ** -24 * float(rp.norm())
    assert float((m.double() - rm).abs().max()) == 0.0


def test_muon_step_long_and_short_reductions(mx):
    """One table, reductions from one chunk to many: those of the short ones have fewer parts."""
    shapes = [(96, 6000), (6000, 96), (80, 33), (33, 80), (128, 1152), (256, 256), (1, 9000), (9000, 1), (200, 2000)]
    matrices, at = [], 0
    for r, c in shapes:
        matrices.append((at, r, c))
        at += r * c + 3
    p, g, m = randn(at, scale=0.03), randn(at, seed=1, scale=1e-3), randn(at, seed=2, scale=1e-3)
    rp, rm, _ = muon64(p, g, m, None, matrices, 0.01, 0.95, True, 0.1, 0.0, 1.0)
    mx.muon_step(p, g, m, matrices, lr=0.01, weight_decay=0.1)
    for o, r, c in matrices:
        s = slice(o, o + r * c)
        step = 0.01 * 0.2 * math.sqrt(max(r, c)) * 1.25 * math.sqrt(min(r, c))
        assert float((p[s].double() - rp[s]).norm()) <= LOOSE * step + 4 * 2.0 ** -24 * float(rp[s].norm())
        assert float((m[s].double() - rm[s]).abs().max()) <= 4 * 2.0 ** -24 * float(rm[s].abs().max())


@pytest.mark.parametrize('top', [16, 32, 48, 64])
@pytest.mark.parametrize('long', [200, 5000])
def test_muon_step_few_rows(mx, top, long):
    """Tables of matrices of few rows, of different sizes, in one workgroup each and in parts; buffers between guard values."""
    shapes = [(top, top), (3, long), (long, top), (top - 3, 77), (1, 1), (9, 5), (5, 9), (long - 1, 2)]
    matrices, at = [], 1
    for r, c in shapes:
        matrices.append((at, r, c))
        at += r * c + 2
    p, g, m, e = (randn(at, seed=i, scale=s) for i, s in enumerate((0.03, 1e-3, 1e-3, 0.03)))
    for ema, nesterov in ((e, True), (None, False)):
        rp, rm, re = muon64(p, g, m, ema, matrices, 0.01, 0.95, nesterov, 0.1, 0.7, 0.5)
        p1, m1, e1 = p.clone(), m.clone(), None if ema is None else ema.clone()
        mx.muon_step(p1, g, m1, matrices, lr=0.01, nesterov=nesterov, weight_decay=0.1, ema=e1, ema_decay=0.7, grad_scale=0.5)
        inside = torch.zeros_like(p, dtype=torch.bool)
        for o, r, c in matrices:
            s = slice(o, o + r * c)
            inside[s] = True
            step = 0.01 * 0.2 * math.sqrt(r * c) * 1.25
            allowed = LOOSE * step + 4 * 2.0 ** -24 * float(rp[s].norm())
            assert float((p1[s].double() - rp[s]).norm()) <= allowed
            assert float((m1[s].double() - rm[s]).abs().max()) <= 4 * 2.0 ** -24 * float(rm[s].abs().max())
            if ema is not None:
                assert float((e1[s].double() - re[s]).norm()) <= allowed + 4 * 2.0 ** -24 * float(re[s].norm())
        for new, old in ((p1, p), (m1, m)) + (((e1, e),) if ema is not None else ()):
            assert torch.equal(new[~inside], old[~inside])


def test_muon_step_refuses(mx):
    p = randn(100)
    for bad in (dict(grad=randn(99)), dict(momentum=randn(100).bfloat16()), dict(ema=randn(100, 1)), dict(matrices=[(90, 3, 4)]),
                dict(matrices=[(0, 5, 5), (24, 2, 2)]), dict(matrices=[]), dict(steps=0), dict(eps=-1.0), dict(grad=randn(200)[::2])):
        kw = dict(dict(param=p, grad=randn(100, seed=1), momentum=randn(100, seed=2), matrices=[(0, 8, 8)], lr=0.1), **bad)
        with pytest.raises(ValueError):
            mx.muon_step(**kw)


def test_adam_over_ranges_equals_adam():
    from objectdetection_amd import matrix
    from objectdetection_amd._lib import lib, check
    n = 9000
    bufs = [randn(n, seed=i, scale=0.1).abs() for i in range(5)]
    whole = [b.clone() for b in bufs]
    part = [b.clone() for b in bufs]
    ranges = [(0, 1), (3, 2500), (2600, 1024), (3700, 5300)] + [(3624 + i, 1) for i in range(0, 60, 2)]
    a = np.array(ranges, dtype=matrix.RANGE_DTYPE)
    st = torch.cuda.current_stream().cuda_stream
    args = (0.01, 0.937, 0.999, 1e-8, 5e-4, 3, 0.9, 0.5, st)
    check(lib.odamd_adam_ema_step(*(b.data_ptr() for b in whole), n, *args))
    check(lib.odamd_adam_ema_ranges_step(*(b.data_ptr() for b in part), a.ctypes.data, len(a), *args))
    inside = torch.zeros(n, dtype=torch.bool, device='cuda')
    for o, k in ranges:
        inside[o:o + k] = True
    for w, p, b in zip(whole, part, bufs):
        assert torch.equal(p[inside], w[inside]) and torch.equal(p[~inside], b[~inside])


# ---------------------------------------------------------------------------------------------
# in use: streams, graphs, a training run
# ---------------------------------------------------------------------------------------------
def test_workspaces_hold_what_is_written(mx):
    """Every entry point with a workspace of exactly the size asked for, in the middle of a larger buffer and full of NaN, none of
    which reaches a result."""
    from objectdetection_amd import _lib
    from objectdetection_amd._lib import lib, check
    st = torch.cuda.current_stream().cuda_stream
    buf = torch.empty(200 << 20, dtype=torch.uint8, device='cuda')

    def guarded(size, call, *results):
        assert size + 8192 <= buf.numel()
        end = 4096 + size
        buf[4096:end] = 255
        buf[:4096] = 165
        buf[end:end + 4096] = 165
        check(call(buf.data_ptr() + 4096))
        assert all(bool(torch.isfinite(r).all()) for r in results if r is not None)
        assert bool((buf[:4096] == 165).all()) and bool((buf[end:end + 4096] == 165).all())

    for code, dtype in ((0, torch.float32), (1, torch.bfloat16)):
        for batch, rows, cols in ((1, 1, 1), (3, 5, 4264), (2, 3000, 16), (1, 40, 7000), (4, 64, 2000), (1, 65, 66), (2, 130, 65),
                                  (3, 129, 2049), (1, 700, 3000), (1, 1025, 1100)):
            for steps in (5, 12):
                g, out = randn(batch, rows, cols, dtype=dtype), torch.empty(batch, rows, cols, dtype=dtype, device='cuda')
                size = lib.odamd_orthogonalize_workspace_bytes(batch, rows, cols)
                guarded(size, lambda ws: lib.odamd_orthogonalize(g.data_ptr(), out.data_ptr(), batch, rows, cols, steps, 1e-7, code,
                                                                 ws, size, st), out)
        for m, k, n in ((9001, 33, 40), (3000, 1155, 101), (600, 2000, 700), (70, 1500, 3001), (10, 40, 9001)):
            x, w, dy = randn(m, k, dtype=dtype), randn(n, k, seed=1, dtype=dtype), randn(m, n, seed=2, dtype=dtype)
            y, z = torch.empty_like(dy), torch.empty(m, n, dtype=dtype if code == 0 else torch.float16, device='cuda')
            dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(n, dtype=dtype, device='cuda')
            d = _lib.LinearDesc(x.data_ptr(), w.data_ptr(), None, None, y.data_ptr(), z.data_ptr(), k, k, 0, n, n, m, k, n, 2, code)
            size = lib.odamd_linear_workspace_bytes(d)
            guarded(size, lambda ws: lib.odamd_linear_forward(d, ws, size, st), y, z)
            for outs in ((dx, dw, db), (dx, None, None), (None, dw, None), (None, None, db)):
                g = _lib.LinearGradDesc(dy.data_ptr(), z.data_ptr(), x.data_ptr(), w.data_ptr(),
                                        *(None if o is None else o.data_ptr() for o in outs), n, n, k, k, k, k, m, k, n, 2, code)
                size = lib.odamd_linear_backward_workspace_bytes(g)
                guarded(size, lambda ws: lib.odamd_linear_backward(g, ws, size, st), *outs)
    for shapes in ([(16, 27), (5, 4000), (1, 1)], [(64, 64), (3, 9000), (1, 2)], [(64, 300), (65, 70), (300, 256)], [(8, 8)] * 130):
        matrices, at = [], 0
        for r, c in shapes:
            matrices.append((at, r, c))
            at += r * c
        table = mx.MatrixTable(matrices)
        p, g, m = randn(at), randn(at, seed=1), randn(at, seed=2)
        for steps in (5, 12):
            guarded(table.workspace_bytes, lambda ws: lib.odamd_muon_ema_step(
                p.data_ptr(), g.data_ptr(), m.data_ptr(), None, table.table.ctypes.data, len(table), 0.01, 0.9, 1, 0.0, steps, 1e-7,
                0.0, 1.0, ws, table.workspace_bytes, st), p, m)


def test_calls_on_two_streams_at_once(mx):
    xs = [randn(m, 300, seed=i) for i, m in enumerate((40, 2500, 2501, 41))]
    w = randn(70, 300, seed=9)
    ref = [(mx.linear(x, w, None, 'silu'), mx.orthogonalize(x)) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 2]):
            got.append((mx.linear(x, w, None, 'silu'), mx.orthogonalize(x)))
    torch.cuda.synchronize()
    for (a, b), (c, d) in zip(ref, got):
        assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.parametrize('rows', [30, 5000])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_captured_and_replayed(mx, dtype, rows):
    """Forward, backward, orthogonalisation and optimizer step in one graph; other inputs between the replays, eager work too."""
    x, w, b, r = randn(rows, 96, dtype=dtype), randn(64, 96, seed=1, dtype=dtype), randn(64, seed=2, dtype=dtype), randn(rows, 64, seed=3, dtype=dtype)
    dy = randn(rows, 64, seed=4, dtype=dtype)
    p, g, m = randn(2000), randn(2000, seed=5), torch.zeros(2000, device='cuda')
    table = mx.MatrixTable([(0, 16, 27), (500, 30, 50)])

    def work(x, p, m):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = mx.linear(*leaves[:3], 'silu', leaves[3])
        grads = torch.autograd.grad(y, leaves, dy)
        mx.muon_step(p, g, m, table, lr=0.01)
        return (y.detach(), *grads, mx.orthogonalize(grads[1]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(x.clone(), p.clone(), m.clone())
    torch.cuda.current_stream().wait_stream(side)
    xs, ps, ms = x.clone(), p.clone(), m.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(xs, ps, ms)
    pe, me = p.clone(), m.clone()
    for turn in range(4):
        xs.copy_(randn(rows, 96, seed=50 + turn, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        ref = work(xs.clone(), pe, me)
        for a, c in zip(out, ref):
            assert torch.equal(a, c)
        assert torch.equal(ps, pe) and torch.equal(ms, me)


def test_two_graphs_at_once(mx):
    """Two captured graphs replayed on two streams at the same time: neither uses the other's workspace."""
    def work(x, w):
        return mx.linear(x, w, None, 'silu'), mx.orthogonalize(x)
    cases = [(randn(5000, 300, seed=i), randn(60, 300, seed=10 + i)) for i in range(2)]
    refs = [work(*c) for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(work(*c))
    for _ in range(3):
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, refs):
            assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_layer_trains_in_both_types(mx):
    from objectdetection_amd.model import layer
    torch.manual_seed(3)
    net = torch.nn.ModuleList([layer.linear(40, 96, 'silu'), layer.linear(96, 40)]).cuda()
    for dtype in (torch.float32, torch.bfloat16):
        x = randn(50, 40, dtype=dtype)
        net.zero_grad()
        out = net[1](net[0](x), residual=x)
        out.float().square().mean().backward()
        leaf = [p.detach().to(dtype).double().requires_grad_() for p in net.parameters()]
        z = torch.nn.functional.silu(x.double() @ leaf[0].t() + leaf[1]) @ leaf[2].t() + leaf[3] + x.double()
        ref = torch.autograd.grad(z.square().mean(), leaf)
        for p, q in zip(net.parameters(), ref):
            # five roundings to the type between the input and a gradient
            assert p.grad.dtype == torch.float32
            assert float((p.grad.double() - q).norm() / q.norm()) < 5 * HALF[dtype] + 1e-5


def test_detector_trains_with_muon():
    """train_class with --optimizer muon: one step equals the 64-bit step on the gradients the backward pass left, Adam on
    what lies between; a second trainer resumed from the saved state continues with the same bits."""
    from objectdetection_amd.train_class import train_class, synthetic_dataset, FusedMuon
    from oracle import patterns, training as otrain
    a = patterns.default_args(input_size=64, output_class=3)
    a.__dict__.update(device='cuda', batch=2, epoch=1, lr_start=0.001, lr_end_ratio=0.1, lr_end_epoch=10, warmup_ratio=0.01,
                      regularization='L2', r_value=0.0005, ema=True, distributed=False, local_rank=0, weight_path='',
                      weight_again=True, print_info=False, synthetic_images=8, save_path=None, amp=False, optimizer='muon')
    ds = synthetic_dataset(a, 4, seed=5)
    batch = ds.collate_fn([ds[0], ds[1]])
    torch.manual_seed(1)
    tc = train_class(a, dataloader=[batch] * 4, val_dataloader=[])
    assert isinstance(tc.optimizer, FusedMuon)
    tc.model.train()
    st = tc.model.train_state()
    image, screen, expend = batch[0].cuda(), batch[1], batch[2]
    tc.train_step(image, screen, expend)                    # the state has moved once: momentum is not zero
    p0, m0, v0, e0 = st.param.clone(), st.exp_avg.clone(), st.exp_avg_sq.clone(), st.ema_param.clone()
    lr, updates = tc.optimizer.param_groups[0]['lr'], st.ema_updates
    tc.train_step(image, screen, expend)
    torch.cuda.synchronize()
    matrices = [tuple(int(v) for v in e) for e in tc.optimizer.table.table.tolist()]
    d = otrain.ema_decay(updates + 1)
    rp, rm, re = muon64(p0, st.grad, m0, e0, matrices, lr, 0.95, True, 0.0005, d, 1.0)
    for o, r, c in matrices:
        s = slice(o, o + r * c)
        step = lr * 0.2 * math.sqrt(r * c) * 1.25
        allowed = LOOSE * step + 8 * 2.0 ** -24 * float(rp[s].norm())
        assert float((st.param[s].double() - rp[s]).norm()) <= allowed
        assert float((st.ema_param[s].double() - re[s]).norm()) <= allowed + 8 * 2.0 ** -24 * float(re[s].norm())
    for o, n in tc.optimizer.rest.tolist():
        s = slice(o, o + n)
        p, m, v = p0[s].cpu().clone(), m0[s].cpu().clone(), v0[s].cpu().clone()
        otrain.adam_step(p, st.grad[s].cpu(), m, v, 2, lr, weight_decay=0.0005)
        np.testing.assert_allclose(st.param[s].cpu().numpy(), p.numpy(), rtol=1e-5, atol=0.01 * lr)
    saved = {k: v.clone() if torch.is_tensor(v) else v for k, v in tc.optimizer.state_dict().items()}
    twin = train_class(a, dataloader=[batch] * 4, val_dataloader=[])
    ts = twin.model.train_state()
    for n in ('param', 'buffers', 'counters', 'ema_param', 'ema_buffers'):
        getattr(ts, n).copy_(getattr(st, n))
    ts.ema_updates = st.ema_updates
    twin.optimizer.load_state_dict(saved)
    for g, h in zip(twin.optimizer.param_groups, tc.optimizer.param_groups):
        g['lr'] = h['lr']
    twin.model.train()
    tc.train_step(image, screen, expend)
    twin.train_step(image, screen, expend)
    assert torch.equal(st.param, ts.param) and torch.equal(st.exp_avg, ts.exp_avg)

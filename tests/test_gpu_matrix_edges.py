"""GPU tests of the matrix operators at their edges, beside test_gpu_matrix.py, whose references and bounds they use."""
import math

import pytest
import torch

from .test_gpu_matrix import HALF, LOOSE, SIZES, orth64, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def mx():
    from objectdetection_amd import matrix
    return matrix


# ---------------------------------------------------------------------------------------------
# few rows, more than ten steps
# ---------------------------------------------------------------------------------------------
# X is rounded to float32 after every ten steps.  A step changes a difference of two X by at most the largest slope of
# a s + b s^3 + c s^5 where singular values are, 4.25 at 1.21 (3.4445 at zero); norms lie between 0.68 and 1.21 times the root of
# the rank, a factor of 1.78.
def rounded_after_ten(steps):
    return 1.78 * 4.25 ** (steps - 10) * (2.0 ** -24 + 1e-9)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('batch, rows, cols', [(3, 1, 7), (1, 16, 27), (5, 30, 50), (2, 40, 33), (2, 64, 200), (3, 2000, 16), (1, 33, 900), (2, 61, 1001)])
def test_few_rows_more_than_ten_steps(mx, batch, rows, cols, dtype):
    g = randn(batch, rows, cols, dtype=dtype, scale=1e-3)
    for steps in (11, 13, 14):
        got = mx.orthogonalize(g, steps=steps)
        for i in range(batch):
            ref = orth64(g[i], steps=steps)
            assert float((got[i].double() - ref).norm()) <= (HALF[dtype] + rounded_after_ten(steps)) * float(ref.norm())
        twin = g.clone()
        assert torch.equal(mx.orthogonalize(twin, steps=steps, out=twin), got)
    for steps in (20, 21, 32):
        got = mx.orthogonalize(g, steps=steps).double().cpu()
        for i in range(batch):
            s = torch.linalg.svdvals(got[i])
            assert 0.65 < float(s.min()) and float(s.max()) < 1.25


def test_few_rows_more_than_ten_steps_and_no_numbers(mx):
    g = randn(5, 40, 70)
    g[1] = 0
    g[2, 3, 4] = float('nan')
    g[3, 39, 69] = float('inf')
    for x in (g, g.bfloat16()):
        y = mx.orthogonalize(x, steps=23)
        assert float(y[1].abs().max()) == 0.0
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3]).all()) and bool(torch.isfinite(y[[0, 4]]).all())


@pytest.mark.parametrize('top, long', [(16, 200), (33, 200), (64, 5000), (5, 40000)])
def test_muon_step_of_few_rows_more_than_ten_steps(mx, top, long):
    """Tables in one workgroup a matrix and in parts, tall and wide, at odd offsets; what lies between stays."""
    shapes = [(top, top), (3, long), (long, top), (top - 3, 77), (1, 1), (5, 9), (long - 1, 2)]
    matrices, at = [], 1
    for r, c in shapes:
        matrices.append((at, r, c))
        at += r * c + 3
    p, g, m, e = (randn(at, seed=i, scale=s) for i, s in enumerate((0.03, 1e-3, 1e-3, 0.03)))
    steps = 12
    for ema, nesterov in ((e, True), (None, False)):
        rp, rm, re = p.double(), m.double(), e.double()
        p1, m1, e1 = p.clone(), m.clone(), None if ema is None else ema.clone()
        mx.muon_step(p1, g, m1, matrices, lr=0.01, nesterov=nesterov, weight_decay=0.1, ema=e1, ema_decay=0.7, grad_scale=0.5, steps=steps)
        inside = torch.zeros_like(p, dtype=torch.bool)
        for o, r, c in matrices:
            s = slice(o, o + r * c)
            inside[s] = True
            gs = g[s].double() * 0.5
            rm[s] = 0.95 * rm[s] + gs
            u = gs + 0.95 * rm[s] if nesterov else rm[s]
            o64 = orth64(u.view(r, c), steps=steps).reshape(-1)
            rp[s] = rp[s] * (1 - 0.01 * 0.1) - 0.01 * 0.2 * math.sqrt(max(r, c)) * o64
            re[s] = 0.7 * re[s] + (1 - 0.7) * rp[s]
            # X's rounding, and the three of u, which singular values of these matrices carry to one within seven steps
            step = 0.01 * 0.2 * math.sqrt(max(r, c)) * float(o64.norm())
            allowed = step * (4 * rounded_after_ten(steps) + 3.4445 ** 7 * 3 * 2.0 ** -24) + 4 * 2.0 ** -24 * float(rp[s].norm())
            assert float((p1[s].double() - rp[s]).norm()) <= allowed
            assert float((m1[s].double() - rm[s]).abs().max()) <= 4 * 2.0 ** -24 * float(rm[s].abs().max())
            if ema is not None:
                assert float((e1[s].double() - re[s]).norm()) <= allowed + 4 * 2.0 ** -24 * float(re[s].norm())
        for new, old in ((p1, p), (m1, m)) + (((e1, e),) if ema is not None else ()):
            assert torch.equal(new[~inside], old[~inside])


# ---------------------------------------------------------------------------------------------
# who else looks at the tensors
# ---------------------------------------------------------------------------------------------
@pytest.mark.filterwarnings('ignore')
def test_traced_calls_compute(mx):
    x, w, b, r = randn(30, 40), randn(24, 40, seed=1), randn(24, seed=2), randn(30, 24, seed=3)
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            layer = torch.jit.trace(lambda t, u: mx.linear(t, w, b, 'silu', u), (x, r), check_trace=False)
            orth = torch.jit.trace(lambda t: mx.orthogonalize(t), (x,), check_trace=False)
            for seed in (10, 11):
                other = randn(30, 40, seed=seed)
                assert torch.equal(layer(other, r), mx.linear(other, w, b, 'silu', r))
                assert torch.equal(orth(other), mx.orthogonalize(other))


def test_forward_mode_is_refused(mx):
    from torch.autograd import forward_ad
    x, w = randn(30, 40), randn(24, 40, seed=1)
    plain = mx.linear(x, w)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: mx.linear(dual, w), lambda: mx.orthogonalize(dual)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(mx.linear(x, w), plain)


def test_orthogonalize_is_no_part_of_a_backward_pass(mx):
    x = randn(30, 40).requires_grad_()
    with pytest.raises(RuntimeError, match='no backward pass'):
        mx.orthogonalize(x).sum().backward()
    assert torch.equal(mx.orthogonalize(x).detach(), mx.orthogonalize(x.detach()))


def test_graphs_of_operations_are_refused(mx):
    """make_fx records torch operations, and tensors without memory hold nothing: neither sees a launch."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = randn(30, 40), randn(24, 40, seed=1)
    for call in (lambda t: mx.linear(t, w), lambda t: mx.orthogonalize(t), lambda t: mx.orthogonalize(t, out=torch.empty_like(t))):
        with pytest.raises(RuntimeError, match='make_fx'):
            make_fx(call)(x)
        with pytest.raises(RuntimeError):
            make_fx(call, tracing_mode='fake')(x)
    leaf = w.clone().requires_grad_()
    y = mx.linear(x, leaf)
    with pytest.raises(RuntimeError, match='make_fx'):
        make_fx(lambda t: torch.autograd.grad(y, leaf, t))(torch.ones_like(y))


def test_a_backward_pass_sees_a_step_between(mx):
    """A weight that lies in the flat buffers: after a step over them its saved value is gone, and the backward pass says so."""
    p, g, m = randn(24 * 40), randn(24 * 40, seed=1), torch.zeros(24 * 40, device='cuda')
    x = randn(30, 40, seed=2).requires_grad_()
    y = mx.linear(x, p.view(24, 40), None, 'silu')
    mx.muon_step(p, g, m, [(0, 24, 40)], lr=0.1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    w = randn(24, 40, seed=3)
    y = mx.linear(x, w, None, 'silu')
    mx.orthogonalize(g.view(24, 40), out=w)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_a_step_over_the_flat_buffers_reaches_cached_plans(mx):
    """matrix.muon_step on a model's own buffers: the next prediction runs on the new weights."""
    from objectdetection_amd.model.yolov7 import yolov7
    from objectdetection_amd import train_engine as te
    from oracle import patterns
    net = yolov7(patterns.default_args(input_size=64, output_class=3))
    patterns.fill_state_dict(net)
    net = net.cuda().eval()
    state = net.train_state()
    image = patterns.image_batch(2, 64).cuda()
    first = net(image).clone()
    assert torch.equal(net(image), first)
    state.grad.copy_(randn(state.n))
    mx.muon_step(state.param, state.grad, state.exp_avg, te.muon_matrices(net, state), lr=0.1)
    assert not torch.equal(net(image), first)


# ---------------------------------------------------------------------------------------------
# activations, value by value: one input of weight one, z = x
# ---------------------------------------------------------------------------------------------
def value_and_slope(z, act):
    """In 64 bits, by forms that keep their digits at negative z: 1 + erf would lose those of 64 bits too by z = -8."""
    if act == 'silu':
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * torch.exp(-z) * p)
    p = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
    return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('act', ['silu', 'gelu'])
@pytest.mark.parametrize('m, n', [(4001, 1), (4001, 9), (40001, 8)])
def test_activations_keep_their_tails(mx, act, dtype, m, n):
    """Relative to the value, however small it is.  float32 products carry 22 bits of z, and a change of z by e changes the tails
    by z z e of themselves (gelu) or z e (silu); bfloat16 values of z are exact, and the activation is good to 5e-5."""
    x = torch.linspace(-12, 12, m, device='cuda').to(dtype)[:, None].requires_grad_()
    w = torch.ones(n, 1, device='cuda', dtype=dtype)
    z = x.detach().double()
    y = mx.linear(x, w, None, act)
    y64, s64 = value_and_slope(z, act)
    rough = (z * z + 16) * 2.0 ** -21 if dtype == torch.float32 else 5e-5
    assert bool(((y.detach().double() - y64).abs() <= (rough + HALF[dtype]) * y64.abs() + 1e-37).all())
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    s64 = n * s64
    # slopes are sums that cross zero between -2 and 0; in bfloat16 they are rounded twice, before the product and after it
    near = 2e-6 * n * (z.abs() < 2)
    assert bool(((dx.double() - s64).abs() <= (rough + 2 * HALF[dtype]) * s64.abs() + near + 1e-37).all())


# ---------------------------------------------------------------------------------------------
# optimizer step
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize('steps', [5, 12])
@pytest.mark.parametrize('shapes', [[(16, 27), (30, 50)], [(16, 700), (3, 5000)], [(130, 129), (16, 27)], [(65, 700), (700, 65)]])
def test_muon_step_decays_by_little(mx, shapes, steps):
    """Without a gradient a step is the decay alone, rounded once: lr weight_decay from 2e-8 (under half a step of one) to 1e-3."""
    matrices, at = [], 0
    for r, c in shapes:
        matrices.append((at, r, c))
        at += r * c
    p, zero = randn(at, scale=0.03), torch.zeros(at, device='cuda')
    for weight_decay in (2e-5, 3e-5, 5e-4, 1.0):
        got, ema = p.clone(), p.clone()
        mx.muon_step(got, zero, zero.clone(), matrices, lr=1e-3, weight_decay=weight_decay, ema=ema, steps=steps)
        ref = p.double() * (1 - 1e-3 * weight_decay)
        # half a step, and the roundings of the decay itself
        assert bool(((got.double() - ref).abs() <= 2.0 ** -24 * ref.abs() * (1 + 4e-3)).all())
        assert torch.equal(ema, got)


# ---------------------------------------------------------------------------------------------
# matrices with few directions
# ---------------------------------------------------------------------------------------------
def of_rank(rank, rows, cols, dtype=torch.float32):
    """`rank` neighbouring columns, the rest zero: A has rows - rank singular values of zero, where every rounding that is not
    symmetric would grow by 3.4445^2 a step and be seen by what lies in the other directions."""
    g = torch.zeros(1, rows, cols, device='cuda', dtype=dtype)
    g[0, :, 5:5 + rank] = randn(rows, rank, seed=rows, dtype=dtype)
    return g


@pytest.mark.parametrize('rank', [1, 3, 40])
@pytest.mark.parametrize('rows, cols', [(65, 130), (130, 300), (130, 130), (128, 2048), (256, 2304), (257, 9001), (1025, 1100)])
def test_orthogonalize_of_little_rank(mx, rows, cols, rank):
    """Phases of five steps, of two and of one; the optimizer step shows the phases of five before they are rounded to bfloat16."""
    low, g = of_rank(rank, rows, cols, torch.bfloat16), of_rank(rank, rows, cols)
    for x, tol in ((low, LOOSE + HALF[torch.bfloat16]), (g, 3.4445 ** 5 * 2.0 ** -24)):
        for y in (x, x.transpose(1, 2).contiguous()):
            ref = orth64(y[0])
            assert float((mx.orthogonalize(y)[0].double() - ref).norm()) <= tol * float(ref.norm())
    flat = g.reshape(-1).contiguous()
    p, m = torch.zeros_like(flat), torch.zeros_like(flat)
    mx.muon_step(p, flat, m, [(0, rows, cols)], lr=-5 / math.sqrt(max(rows, cols)), momentum_decay=0.0, nesterov=False)
    ref = orth64(g[0])
    assert float((p.view(rows, cols).double() - ref).norm()) <= LOOSE * float(ref.norm())


@pytest.mark.parametrize('rank', [1, 2])
@pytest.mark.parametrize('rows, cols', [(12, 300), (16, 300), (16, 4000), (30, 300), (48, 4000), (64, 300)])
def test_orthogonalize_of_few_rows_and_little_rank(mx, rows, cols, rank):
    """64 bits: a rounding of Q, 2^-53 of 3.4445^10 at most, over up to 64 directions, is under 1e-9."""
    g = of_rank(rank, rows, cols)
    for steps in range(5, 11):
        for x in (g, g.transpose(1, 2).contiguous()):
            ref = orth64(x[0], steps=steps)
            assert float((mx.orthogonalize(x, steps=steps)[0].double() - ref).norm()) <= (2.0 ** -24 + 1e-9) * float(ref.norm())


# ---------------------------------------------------------------------------------------------
# nothing is left out: sums that are exact
# ---------------------------------------------------------------------------------------------
LONG = [(2100, 264, 2050), (4000, 96, 4100), (50, 4000, 72), (4097, 300, 1001), (2056, 520, 2000), (9000, 136, 520), (5001, 129, 131),
        (2100, 263, 2049), (70, 1500, 3001), (2500, 1030, 1033), (30001, 40, 56), (64, 9001, 64), (520, 33, 20001), (257, 2049, 129)]


def whole(*shape, seed, dtype):
    """-3 .. 3 without 0: no product is zero, sums of up to 2^20 of them are exact in float32, whatever their order."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    v = torch.randint(1, 4, shape, generator=g, device='cuda') * (2 * torch.randint(0, 2, shape, generator=g, device='cuda') - 1)
    return v.to(dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m, k, n', SIZES + LONG)
def test_linear_sums_every_term(mx, m, k, n, dtype):
    """Whole numbers: the result and all gradients are exact, rounded once."""
    x, w, b, r = (whole(*s, seed=i, dtype=dtype) for i, s in enumerate(((m, k), (n, k), (n,), (m, n))))
    dy = whole(m, n, seed=9, dtype=dtype)
    z = x.double() @ w.double().t() + b.double()
    for act in (None, 'relu'):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = mx.linear(*leaves[:3], act, leaves[3])
        assert torch.equal(y.detach(), ((z.clamp(min=0) if act else z) + r.double()).to(dtype))
        dz = dy.double() * (z > 0) if act else dy.double()
        dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
        assert torch.equal(dx, (dz @ w.double()).to(dtype))
        assert torch.equal(dw, (dz.t().contiguous() @ x.double()).to(dtype))
        assert torch.equal(db, dz.sum(0).to(dtype)) and torch.equal(dr, dy)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('rows, cols', [(5, 1025), (16, 1537), (33, 1001), (64, 513), (3, 70001), (65, 130), (130, 2049), (256, 2304),
                                        (257, 9001), (1025, 1100), (70, 4001)])
def test_orthogonalize_reads_every_column(mx, rows, cols, dtype):
    """All but three neighbouring columns are zero, at the ends and where the reduction may be cut: a column left out is an error of
    order one.  A rounding of X to 22 bits grows by 3.4445 a step in the directions that have no singular value."""
    tol = 1.41 * 3.4445 ** 5 * 3 * 2.0 ** -22 + HALF[dtype]
    for at in sorted({0, 31, cols // 3 - 1, cols // 2 - 1, cols * 3 // 4 - 1, cols - 4, cols - 3}):
        g = torch.zeros(1, rows, cols, device='cuda', dtype=dtype)
        g[0, :, at:at + 3] = randn(rows, 3, seed=at, dtype=dtype)
        for x in (g, g.transpose(1, 2).contiguous()):
            got, ref = mx.orthogonalize(x)[0].double(), orth64(x[0])
            assert float((got - ref).norm()) <= tol * float(ref.norm())


# ---------------------------------------------------------------------------------------------
# operands and results of more than 2^31 elements
# ---------------------------------------------------------------------------------------------
@pytest.fixture
def room():
    """100 GB of the card's memory, given back afterwards."""
    if torch.cuda.get_device_properties(0).total_memory < 200 << 30:
        pytest.skip('a card of less memory')
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('m, k, n', [(4, 64, 4), (40, 72, 64), (3000, 64, 56), (3001, 71, 45)])
def test_linear_of_rows_far_apart(mx, room, m, k, n, dtype):
    """The last rows of x, the residual and the gradient begin past element 2^31: the same bits as close together."""
    apart = (2 ** 31 // (m - 1) // 8 + 100) * 8
    far = torch.empty((m - 1) * apart + 4096, dtype=dtype, device='cuda')
    x, r, dy = (far.as_strided((m, c), (apart, 1), at) for c, at in ((k, 0), (n, 256), (n, 512)))
    w, b = randn(n, k, seed=1, dtype=dtype, scale=k ** -0.5), randn(n, seed=2, dtype=dtype)
    for seed, t in enumerate((x, r, dy)):
        t.copy_(randn(*t.shape, seed=10 + seed, dtype=dtype))
    # close together on rows of the same alignment: the same way through the kernels
    near = torch.empty(m * 1024, dtype=dtype, device='cuda')
    copies = [near.as_strided((m, t.shape[1]), (1024, 1), at).copy_(t) for t, at in ((x, 0), (r, 256), (dy, 512))]
    results = []
    for x, r, dy in ((x, r, dy), copies):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = mx.linear(*leaves[:3], 'silu', leaves[3])
        results.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    assert all(torch.equal(a, c) for a, c in zip(*results))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_linear_of_large_results(mx, room, dtype):
    m, k, n = 2 ** 20 + 77, 16, 2056
    x, w = whole(m, k, seed=0, dtype=dtype).requires_grad_(), whole(n, k, seed=1, dtype=dtype).requires_grad_()
    y = mx.linear(x, w, None, 'relu')
    z = x[-300:].detach().double() @ w.detach().double().t()
    assert torch.equal(y[-300:].detach(), z.clamp(min=0).to(dtype))
    # exact: sums of -1 and 1 times 0 .. 3
    dy = torch.ones(1, device='cuda', dtype=dtype).expand(m, n)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(dx[-300:], ((z > 0).double() @ w.detach().double()).to(dtype))
    last = torch.zeros(k, dtype=torch.float64, device='cuda')
    for at in range(0, m, 2 ** 18):
        part = x[at:at + 2 ** 18].detach().double()
        last += ((part @ w[-1].detach().double()) > 0).double() @ part
    assert torch.equal(dw[-1], last.to(dtype))


@pytest.mark.parametrize('steps', [5, 12])
@pytest.mark.parametrize('shapes', [[(16, 27), (64, 300), (3, 9000)], [(130, 257), (16, 27), (700, 66)]])
def test_muon_step_far_into_the_buffers(mx, room, shapes, steps):
    """Matrices past element 2^31, and Adam over ranges there: the same bits as at the start of short buffers."""
    from objectdetection_amd._lib import lib, check
    import numpy as np
    matrices, at = [], 1
    for r, c in shapes:
        matrices.append((at, r, c))
        at += r * c + 3
    length = at + 100
    start = 2 ** 31 + 5
    near = [randn(length, seed=i, scale=0.01).abs() for i in range(4)]
    far = [torch.empty(start + length, device='cuda') for _ in range(4)]
    for f, t in zip(far, near):
        f[start:].copy_(t)
    mx.muon_step(*near[:3], matrices, lr=0.01, weight_decay=0.1, ema=near[3], ema_decay=0.9, steps=steps)
    mx.muon_step(*far[:3], [(o + start, r, c) for o, r, c in matrices], lr=0.01, weight_decay=0.1, ema=far[3], ema_decay=0.9, steps=steps)
    assert all(torch.equal(f[start:], t) for f, t in zip(far, near))
    stream = torch.cuda.current_stream().cuda_stream
    for bufs, o in ((near, 0), (far, start)):
        a = np.array([(o + 3, 1000), (o + length - 50, 50)], dtype=mx.RANGE_DTYPE)
        check(lib.odamd_adam_ema_ranges_step(*(t.data_ptr() for t in bufs), None, a.ctypes.data, len(a), 0.01, 0.937, 0.999, 1e-8, 5e-4, 3,
                                             0.0, 1.0, stream))
    # by their bits: the third buffer has negative values, whose root is no number
    assert all(torch.equal(f[start:].view(torch.int32), t.view(torch.int32)) for f, t in zip(far, near))


@pytest.mark.parametrize('batch, rows, cols, dtype', [(2 ** 22 + 3, 16, 32, torch.float32), (2 ** 15 + 9, 256, 256, torch.bfloat16)])
def test_orthogonalize_of_a_large_batch(mx, room, batch, rows, cols, dtype):
    g = torch.zeros(batch, rows, cols, dtype=dtype, device='cuda')
    g[:5], g[-9:] = randn(5, rows, cols, dtype=dtype), randn(9, rows, cols, seed=1, dtype=dtype)
    got = mx.orthogonalize(g)
    for i in (0, 4, batch - 9, batch - 1):
        ref = orth64(g[i])
        assert float((got[i].double() - ref).norm()) <= (LOOSE + HALF[dtype]) * float(ref.norm())
    assert float(got[5:8].abs().max()) == 0.0 and float(got[-12:-9].abs().max()) == 0.0


# ---------------------------------------------------------------------------------------------
# in use
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize('rows, cols', [(30, 50), (16, 4000), (130, 300)])
def test_many_steps_captured_and_replayed(mx, rows, cols):
    """Several phases of steps in a graph, other inputs and eager work between its replays."""
    table = mx.MatrixTable([(3, rows, cols), (rows * cols + 7, 16, 27)])
    length = table.end + 2
    g, p, m = randn(length), randn(length, seed=1), torch.zeros(length, device='cuda')
    low = randn(2, rows, cols, seed=2, dtype=torch.bfloat16)

    def work(low, p, m):
        mx.muon_step(p, g, m, table, lr=0.01, steps=12)
        return mx.orthogonalize(low, steps=12), mx.orthogonalize(low.float(), steps=23)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(low.clone(), p.clone(), m.clone())
    torch.cuda.current_stream().wait_stream(side)
    xs, ps, ms = low.clone(), p.clone(), m.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(xs, ps, ms)
    for turn in range(4):
        xs.copy_(randn(2, rows, cols, seed=60 + turn, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        ref = work(xs.clone(), p, m)
        assert all(torch.equal(a, c) for a, c in zip(out, ref))
        assert torch.equal(ps, p) and torch.equal(ms, m)


def test_compiled_callers_leave_the_calls_alone(mx):
    x, w = randn(30, 40), randn(24, 40, seed=1)
    call = torch.compile(lambda t: mx.linear(t, w, None, 'gelu') * 2, backend='eager')
    assert torch.equal(call(x), mx.linear(x, w, None, 'gelu') * 2)
    leaf, twin = (w.clone().requires_grad_() for _ in range(2))
    call = torch.compile(lambda t: (mx.linear(t, leaf, None, 'silu') * t[:, :24]).sum(), backend='eager')
    call(x).backward()
    (mx.linear(x, twin, None, 'silu') * x[:, :24]).sum().backward()
    assert torch.equal(leaf.grad, twin.grad)

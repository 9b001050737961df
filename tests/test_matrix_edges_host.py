"""Matrix operators at their edges, what the host decides: workspaces, refusals, and how they meet autograd."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from objectdetection_amd import matrix
from objectdetection_amd._lib import lib


@pytest.mark.parametrize('batch, rows, cols', [(1, 1, 10 ** 8), (4, 4, 4 * 10 ** 6), (4 * 10 ** 6, 3, 3), (1 << 20, 16, 16), (1, 64, 256),
                                               (1, 10 ** 6, 64), (7, 33, 900)])
def test_matrices_of_few_rows_take_a_copy_of_themselves(batch, rows, cols):
    """One float32 copy, and partial sums for long matrices: no padded layouts, whatever the number of steps."""
    size = batch * rows * cols * 4
    need = lib.odamd_orthogonalize_workspace_bytes(batch, rows, cols)
    most = 700 * 1024 * batch if max(rows, cols) > 256 else 0
    assert size <= need <= size + 256 + most
    if batch == 1:
        t = np.array([(0, rows, cols)], dtype=matrix.MATRIX_DTYPE)
        assert lib.odamd_muon_workspace_bytes(t.ctypes.data, 1) == need


def test_a_dense_layer_asks_for_what_it_writes():
    """bfloat16 operands that products read in place need no room for copies; from any other address they do."""
    from .test_matrix_host import P, _desc, _grad_desc
    m, k, n = 25600, 1024, 4096
    forward = dict(m=m, k=k, n=n, x_ld=k, w_ld=k, y_ld=n)
    backward = dict(m=m, k=k, n=n, dy_ld=n, z_ld=n, x_ld=k, w_ld=k, dx_ld=k, dw_ld=k)
    query = lambda **kw: lib.odamd_linear_workspace_bytes(_desc(**forward, **kw))      # noqa: E731
    assert query() == 0
    assert query(x=P + 2) == m * k * 2 and query(w=P + 2) == n * k * 2
    assert query(x=None, w=None) == query(x=P + 2, w=P + 2) == (m + n) * k * 2
    back = lambda **kw: lib.odamd_linear_backward_workspace_bytes(_grad_desc(**backward, **kw))      # noqa: E731
    sums = m // 64 * n * 4                                     # db's
    dz = m * n * 2
    for act, laid in ((0, 0), (1, dz)):
        cut = back(act=act, dx=None, dw=P) - sums - laid       # parts of dw's reduction over the rows
        assert cut < 8 * n * k * 4
        assert back(act=act, dx=P, dw=None) == sums + laid
        assert back(act=act, dx=P, dw=None, w=P + 2) == sums + laid + n * k * 2
        assert back(act=act, dx=None, x=P + 2) == sums + laid + cut + m * k * 2
    assert back(act=0, dx=P, dw=None, dy=P + 2) == sums + dz


# ---------------------------------------------------------------------------------------------
# who else looks at the tensors: forward-mode differentiation, traces, a backward pass
# ---------------------------------------------------------------------------------------------
@pytest.fixture
def on_host(monkeypatch):
    """The Python layer over host arithmetic that, like the kernels, nothing of torch sees."""
    def forward(x, weight, bias, residual, act, keep_z):
        y = x.new_empty((x.shape[0], weight.shape[0]))
        np.copyto(np.from_dlpack(y.detach()), np.from_dlpack(x.detach()) @ np.from_dlpack(weight.detach()).T)
        return y, None

    def orthogonal(x, steps, eps, out):
        np.copyto(np.from_dlpack(out.detach()), 2 * np.from_dlpack(x.detach()))
        return out
    monkeypatch.setattr(matrix, '_check_tensor', lambda *a, **kw: None)
    monkeypatch.setattr(matrix, '_linear_forward', forward)
    monkeypatch.setattr(matrix, '_orthogonalize', orthogonal)


@pytest.mark.parametrize('grad', [False, True])
def test_a_tangent_is_refused_and_not_lost(on_host, grad):
    x, w = torch.randn(3, 4), torch.randn(5, 4)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: matrix.linear(dual, w), lambda: matrix.linear(w, dual), lambda: matrix.orthogonalize(dual)):
            with pytest.raises(NotImplementedError, match='forward mode'):
                call()
        with pytest.raises(RuntimeError, match='tangent'):
            matrix.orthogonalize(dual, out=torch.empty(3, 4))
        assert torch.allclose(matrix.linear(x, w), x @ w.t())           # without a tangent as ever
        assert torch.equal(matrix.orthogonalize(x), 2 * x)
        assert torch.equal(matrix.orthogonalize(x, out=torch.empty(3, 4)), 2 * x)


@pytest.mark.filterwarnings('ignore')
@pytest.mark.parametrize('grad', [False, True])
def test_a_trace_holds_the_call(on_host, grad):
    x, w = torch.randn(3, 4), torch.randn(5, 4)
    with torch.set_grad_enabled(grad):
        layer = torch.jit.trace(lambda t: matrix.linear(t, w), (x,), check_trace=False)
        orth = torch.jit.trace(lambda t: matrix.orthogonalize(t), (x,), check_trace=False)
        other = torch.randn(3, 4)
        assert torch.allclose(layer(other), other @ w.t()) and torch.equal(orth(other), 2 * other)
        flat = torch.zeros(12)
        for write in (lambda t: matrix.orthogonalize(t, out=torch.empty(3, 4)),
                      lambda t: matrix.muon_step(flat, t.view(12), torch.zeros(12), [(0, 3, 4)], 0.1)):
            with pytest.raises(RuntimeError, match='trace does not record'):
                torch.jit.trace(write, (x,), check_trace=False)


def test_orthogonalize_raises_in_a_backward_pass(on_host):
    x = torch.randn(3, 4, requires_grad=True)
    with pytest.raises(RuntimeError, match='no backward pass'):
        (matrix.orthogonalize(x).sum() + x.sum()).backward()
    with torch.no_grad():
        assert not matrix.orthogonalize(x).requires_grad
    assert not matrix.orthogonalize(x.detach()).requires_grad
    assert not matrix.orthogonalize(x, out=torch.empty(3, 4)).requires_grad


@pytest.mark.parametrize('with_ema', [False, True])
def test_what_is_written_counts_as_written(on_host, monkeypatch, with_ema):
    """A saved tensor that a call wrote makes the backward pass raise, and plans that folded a weight fold it again."""
    from objectdetection_amd import engine
    monkeypatch.setattr(matrix, '_call', lambda *a: 0)
    generation = engine._weights_generation[0]
    x = torch.randn(3, 4, requires_grad=True)
    out = torch.randn(3, 4)
    loss = (x * out).sum()
    matrix.orthogonalize(torch.randn(3, 4), out=out)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    assert engine._weights_generation[0] > generation
    generation = engine._weights_generation[0]
    buffers = [torch.randn(12) for _ in range(4)]
    losses = [(x * b.view(3, 4)).sum() for b in buffers]
    matrix.muon_step(*buffers[:3], [(0, 3, 4)], 0.1, ema=buffers[3] if with_ema else None)
    for i, loss in enumerate(losses):
        if i == 1 or (i == 3 and not with_ema):              # the gradient is read only
            loss.backward()
        else:
            with pytest.raises(RuntimeError, match='modified by an inplace operation'):
                loss.backward()
    assert engine._weights_generation[0] > generation


def test_memory_shared_in_part_is_refused(on_host, monkeypatch):
    monkeypatch.setattr(matrix, '_call', lambda *a: 0)
    buf = torch.randn(200)
    x = buf[:96].view(8, 12)
    for start in (1, 4, 95):
        with pytest.raises(ValueError, match='shares'):
            matrix.orthogonalize(x, out=buf[start:start + 96].view(8, 12))
        with pytest.raises(ValueError, match='shares'):
            matrix.orthogonalize(buf[start:start + 96].view(8, 12), out=x)
    for out in (x, x.view(8, 12), buf[:96].view(8, 12), buf[96:192].view(8, 12)):
        assert matrix.orthogonalize(x, out=out) is out
    # what is not contiguous is copied first
    assert matrix.orthogonalize(buf[:192].view(8, 24)[:, :12], out=x) is x
    flat = [torch.randn(100) for _ in range(4)]
    for i in range(4):
        for j in range(i):
            args = list(flat)
            args[i] = args[j]
            with pytest.raises(ValueError, match='shares memory'):
                matrix.muon_step(*args[:3], [(0, 8, 12)], 0.1, ema=args[3])
    with pytest.raises(ValueError, match='momentum shares memory with param'):
        matrix.muon_step(buf[:100], flat[1], buf[99:199], [(0, 8, 12)], 0.1)
    matrix.muon_step(buf[:100], flat[1], buf[100:], [(0, 8, 12)], 0.1)


def test_a_table_of_matrices_ends_where_it_says():
    """An end past 64 bits must not come out as one before the buffer's; sizes are whole numbers."""
    for bad in ([(2 ** 63 - 10, 4, 4)], [(2 ** 62 + 1, 4, 4)], [(0, 4, 4), (2 ** 63 - 1, 1, 1)], [(2 ** 64, 4, 4)], [(2 ** 70, 4, 4)], [(0, 2.5, 4)],
                [(0.5, 2, 4)], [(float('nan'), 2, 4)], [('0', '2', '4')], [(0, None, 4)]):
        with pytest.raises(ValueError):
            matrix.MatrixTable(bad)
    t = matrix.MatrixTable([(2 ** 62, 4, 8), (0, 2 ** 15, 2 ** 16 - 2)])
    assert t.end == 2 ** 62 + 32 and len(t.gaps(2 ** 62 + 40)) == 2
    assert matrix.MatrixTable(np.array([[3, 2, 2]], np.int32)).end == 7
    assert matrix.MatrixTable((np.int64(3), 2.0, 2) for _ in range(1)).end == 7

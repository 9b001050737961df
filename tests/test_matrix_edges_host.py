"""Matrix operators at their edges, what the host decides: workspaces, refusals, and how they meet autograd."""
import numpy as np
import pytest

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

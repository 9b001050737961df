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

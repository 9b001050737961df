"""Refusals and tables of the matrix operators (dense layer, orthogonalisation, optimizer step): everything here is
decided on the host before anything is launched, so it runs without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from objectdetection_amd import _lib, matrix
from objectdetection_amd._lib import lib

E_ARG, E_ALIGN, E_WORKSPACE, E_SHAPE, E_LIMIT = -1, -2, -3, -4, -5
P = 1 << 20            # a well aligned address that is never followed


def _desc(**kw):
    d = dict(x=P, w=P, bias=None, residual=None, y=P, z=None, x_ld=64, w_ld=64, r_ld=0, y_ld=32, z_ld=0, m=16, k=64, n=32,
             act=0, dtype=1)
    d.update(kw)
    return _lib.LinearDesc(*[d[n] for n, _ in _lib.LinearDesc._fields_])


def _grad_desc(**kw):
    d = dict(dy=P, z=P, x=P, w=P, dx=P, dw=P, db=P, dy_ld=32, z_ld=32, x_ld=64, w_ld=64, dx_ld=64, dw_ld=64, m=16, k=64, n=32,
             act=1, dtype=1)
    d.update(kw)
    return _lib.LinearGradDesc(*[d[n] for n, _ in _lib.LinearGradDesc._fields_])


@pytest.mark.parametrize('change, code', [
    (dict(x=None), E_ARG), (dict(w=None), E_ARG), (dict(y=None), E_ARG), (dict(m=0), E_ARG), (dict(k=0), E_ARG),
    (dict(n=-1), E_ARG), (dict(act=4), E_ARG), (dict(act=-1), E_ARG), (dict(dtype=2), E_ARG), (dict(m=2 ** 31 - 1), E_ARG), (dict(k=2 ** 31 - 2 ** 15, x_ld=2 ** 31, w_ld=2 ** 31), E_ARG),
    (dict(x_ld=63), E_SHAPE), (dict(w_ld=63), E_SHAPE), (dict(y_ld=31), E_SHAPE), (dict(residual=P, r_ld=31), E_SHAPE),
    (dict(z=P, z_ld=31), E_SHAPE), (dict(x=P + 1), E_ALIGN), (dict(dtype=0, w=P + 2), E_ALIGN), (dict(bias=P + 1), E_ALIGN)])
def test_linear_forward_refuses(change, code):
    assert lib.odamd_linear_forward(C.byref(_desc(**change)), P, 1 << 40, None) == code


@pytest.mark.parametrize('change, code', [
    (dict(dy=None), E_ARG), (dict(z=None), E_ARG), (dict(w=None), E_ARG), (dict(x=None), E_ARG),
    (dict(dx=None, dw=None, db=None), E_ARG), (dict(m=0), E_ARG), (dict(dtype=5), E_ARG), (dict(dy_ld=31), E_SHAPE),
    (dict(z_ld=31), E_SHAPE), (dict(dx_ld=63), E_SHAPE), (dict(dw_ld=63), E_SHAPE), (dict(x_ld=63), E_SHAPE),
    (dict(w_ld=63), E_SHAPE), (dict(dw=P + 1), E_ALIGN), (dict(db=P + 1), E_ALIGN)])
def test_linear_backward_refuses(change, code):
    assert lib.odamd_linear_backward(C.byref(_grad_desc(**change)), P, 1 << 40, None) == code


def test_workspaces_are_asked_for_and_checked():
    assert lib.odamd_linear_forward(None, None, 0, None) == E_ARG
    assert lib.odamd_linear_backward(None, None, 0, None) == E_ARG
    assert lib.odamd_linear_workspace_bytes(C.byref(_desc(m=1))) == 0              # read in place, no workspace
    assert lib.odamd_linear_workspace_bytes(C.byref(_desc(dtype=0))) == 0          # so are few workgroups
    d = _desc(dtype=0, m=40000)
    need = lib.odamd_linear_workspace_bytes(C.byref(d))
    assert need >= (40000 + 32) * 64 * 4
    assert lib.odamd_linear_forward(C.byref(d), P, need - 1, None) == E_WORKSPACE
    assert lib.odamd_linear_forward(C.byref(d), None, need, None) == E_ARG
    assert lib.odamd_linear_forward(C.byref(d), P + 64, need, None) == E_ALIGN
    assert lib.odamd_linear_backward_workspace_bytes(C.byref(_grad_desc())) == 0   # a small layer takes none
    g = _grad_desc(m=40000)
    need = lib.odamd_linear_backward_workspace_bytes(C.byref(g))
    assert lib.odamd_linear_backward(C.byref(g), P, need - 1, None) == E_WORKSPACE
    assert lib.odamd_linear_backward(C.byref(g), P + 8, need, None) == E_ALIGN
    assert lib.odamd_linear_workspace_bytes(C.byref(_desc(k=0))) == 0


def test_orthogonalize_refuses():
    def call(x=P, out=P, batch=1, rows=8, cols=16, steps=5, eps=1e-7, dtype=0, ws=P, size=1 << 40):
        return lib.odamd_orthogonalize(x, out, batch, rows, cols, steps, eps, dtype, ws, size, None)
    for bad in (dict(x=None), dict(out=None), dict(ws=None), dict(batch=0), dict(rows=0), dict(cols=0), dict(steps=0),
                dict(steps=33), dict(eps=-1.0), dict(eps=float('nan')), dict(dtype=2), dict(rows=1 << 16, cols=1 << 15)):
        assert call(**bad) == E_ARG, bad
    assert call(x=P + 2) == E_ALIGN and call(out=P + 1, dtype=1) == E_ALIGN and call(ws=P + 128) == E_ALIGN
    need = lib.odamd_orthogonalize_workspace_bytes(3, 8, 16)
    assert need > 0 and call(batch=3, size=need - 1) == E_WORKSPACE
    assert lib.odamd_orthogonalize_workspace_bytes(0, 8, 16) == 0


def test_more_than_a_launch_takes_is_refused():
    """A launch has fewer than 2^32 threads."""
    huge = 1 << 62
    row = _desc(m=1, k=1, n=1 << 30, x_ld=1, w_ld=1, y_ld=1 << 30)
    assert lib.odamd_linear_forward(C.byref(row), P, huge, None) == E_LIMIT
    many = _desc(m=1 << 30, k=1, n=1, x_ld=1, w_ld=1, y_ld=1, dtype=0)
    assert lib.odamd_linear_forward(C.byref(many), P, huge, None) == E_LIMIT
    grad = _grad_desc(m=1 << 30, k=1024, n=1024, dy_ld=1024, z_ld=1024, x_ld=1024, w_ld=1024, dx_ld=1024, dw_ld=1024)
    assert lib.odamd_linear_backward(C.byref(grad), P, huge, None) == E_LIMIT
    for rows, cols in ((1, 1), (128, 128)):
        assert lib.odamd_orthogonalize(P, P, 1 << 25, rows, cols, 5, 0.0, 0, P, huge, None) == E_LIMIT


def test_muon_and_ranges_refuse():
    t = np.array([(0, 8, 16)], dtype=matrix.MATRIX_DTYPE)

    def call(table=t, n=1, param=P, ws=P, size=1 << 40, steps=5, eps=1e-7):
        return lib.odamd_muon_ema_step(param, P, P, None, table.ctypes.data if table is not None else None, n, 0.1, 0.9, 1, 0.0,
                                       steps, eps, 0.0, 1.0, ws, size, None)
    assert call(table=None) == E_ARG and call(n=0) == E_ARG and call(param=None) == E_ARG and call(ws=None) == E_ARG
    assert call(steps=0) == E_ARG and call(eps=-1.0) == E_ARG
    assert call(table=np.array([(-1, 8, 16)], dtype=matrix.MATRIX_DTYPE)) == E_ARG
    assert call(table=np.array([(0, 0, 16)], dtype=matrix.MATRIX_DTYPE)) == E_ARG
    assert call(param=P + 2) == E_ALIGN and call(ws=P + 16) == E_ALIGN
    assert call(size=lib.odamd_muon_workspace_bytes(t.ctypes.data, 1) - 1) == E_WORKSPACE
    for r in ((-1, 4), (0, 0), (0, 2 ** 31)):
        a = np.array([r], dtype=matrix.RANGE_DTYPE)
        assert lib.odamd_adam_ema_ranges_step(P, P, P, P, None, a.ctypes.data, 1, 0.1, 0.9, 0.9, 1e-8, 0.0, 1, 0.0, 1.0, None) == E_ARG
    a = np.array([(0, 4)], dtype=matrix.RANGE_DTYPE)
    assert lib.odamd_adam_ema_ranges_step(P, P, P, P, None, a.ctypes.data, 1, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 0.0, 1.0, None) == E_ARG


def test_matrix_table():
    t = matrix.MatrixTable([(40, 2, 3), (0, 4, 8)])
    assert len(t) == 2 and t.end == 46
    assert t.gaps(50) == [(32, 8), (46, 4)] and t.gaps(46) == [(32, 8)]
    assert t.workspace_bytes > 0
    for bad in ([], [(-1, 2, 2)], [(0, 0, 2)], [(0, 2, -1)], [(0, 4, 8), (31, 1, 1)], [(0, 1 << 16, 1 << 15)]):
        with pytest.raises(ValueError):
            matrix.MatrixTable(bad)


def test_python_refuses_what_does_not_fit():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ValueError, match='CUDA'):
        matrix.linear(x, w)
    with pytest.raises(ValueError, match='activation'):
        matrix.linear(x, w, activation='tanh')
    with pytest.raises(ValueError, match='CUDA'):
        matrix.orthogonalize(x)
    for p in (x, None):
        with pytest.raises(ValueError, match='CUDA'):
            matrix.muon_step(p, x, x, [(0, 4, 8)], 0.1)
    from objectdetection_amd.model import layer
    with pytest.raises(ValueError, match='activation'):
        layer.linear(8, 6, act='tanh')
    assert sorted(layer.linear(8, 6).state_dict()) == ['bias', 'weight']


def test_optimizer_choice_and_foreign_states():
    from objectdetection_amd import train_class, train_engine as te
    from objectdetection_amd.model.yolov7 import yolov7
    from objectdetection_amd.run import build_parser
    from oracle import patterns
    assert build_parser().parse_args([]).optimizer == 'adam'
    assert build_parser().parse_args(['--optimizer', 'muon']).optimizer == 'muon'
    with pytest.raises(SystemExit):
        build_parser().parse_args(['--optimizer', 'sgd'])
    net = yolov7(patterns.default_args(input_size=64, output_class=3))
    muon = train_class.FusedMuon(net, 0.001, weight_decay=5e-4)
    adam = train_class.FusedAdam(net, 0.001)
    with pytest.raises(ValueError, match='muon'):
        adam.load_state_dict(muon.state_dict())
    with pytest.raises(ValueError):
        muon.load_state_dict(adam.state_dict())
    muon.load_state_dict(muon.state_dict())
    # every convolution of a block is a matrix, the heads are not; matrices and ranges cover the flat buffer exactly once
    heads = [net.head0.output.weight, net.head1.output.weight, net.head2.output.weight]
    offsets = set(muon.table.table['offset'].tolist())
    for p in net.parameters():
        expected = p.dim() == 4 and not any(p is h for h in heads)
        assert (muon.state.offsets[id(p)] in offsets) == expected
    seen = np.zeros(muon.state.n, np.int32)
    for o, r, c in muon.table.table.tolist():
        seen[o:o + r * c] += 1
    for o, n in muon.rest.tolist():
        seen[o:o + n] += 1
    assert (seen == 1).all()
    assert te.muon_matrices(net, muon.state)[0][1:] == (16, 27)

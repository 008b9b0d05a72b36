"""Arguments that kvm_qk_norm_rope and kvm_window_append refuse by their size or type, on
the host alone: the checks come before the state is looked at."""
import ctypes as C

import pytest

from kvmem_amd import _lib as L


def _view(tokens, heads, dims, ty=L.T_F32, es=4):
    return L.View(4096, ty, dims, heads, tokens, es, es * dims, es * dims * heads)


def _window(cells=128, H=2, D=128, kt=L.T_Q8_0, vt=L.T_Q4_0, bt=64):
    w = L.Window(cells, H, D, bt, kt, vt)
    w.k, w.v, w.cell_pos = 1 << 20, 1 << 21, 1 << 22
    return w


def _rope(q, k, n_rot=64, had=0, eps=1e-6, ty=L.T_F32, base=1e6):
    r = L.RopeParams(n_rot, base, 1.0, had)
    return L.load().kvm_qk_norm_rope(None, None if q is None else C.byref(q), None if k is None else C.byref(k), None, None,
                                     eps, C.byref(r), 1 << 23, ty, 1 << 24, 1 << 25)


@pytest.mark.parametrize("code,call", [
    (L.KVM_EUNSUPPORTED, lambda: _rope(_view(2, 4, 128), _view(2, 1, 128), n_rot=20)),
    (L.KVM_EUNSUPPORTED, lambda: _rope(_view(2, 4, 128), None, n_rot=256)),
    (L.KVM_EUNSUPPORTED, lambda: _rope(_view(2, 4, 128), None, had=32)),
    (L.KVM_EUNSUPPORTED, lambda: _rope(_view(2, 4, 192), None, had=128)),
    (L.KVM_EUNSUPPORTED, lambda: _rope(_view(2, 4, 264), None)),
    (L.KVM_EUNSUPPORTED, lambda: _rope(_view(2, 4, 4), None, n_rot=0)),
    (L.KVM_EUNSUPPORTED, lambda: _rope(_view(2, 4, 128), None, ty=L.T_Q8_0)),
    (L.KVM_EUNSUPPORTED, lambda: _rope(_view(2, 4, 128, ty=L.T_Q8_0), None)),
    (L.KVM_ERANGE, lambda: _rope(_view(2 ** 31, 1, 128), None)),
    (L.KVM_ERANGE, lambda: _rope(_view(2 ** 30, 4, 128), None)),
    (L.KVM_ERANGE, lambda: _rope(_view(1, 2 ** 21, 128), None)),
    (L.KVM_EINVAL, lambda: _rope(None, None)),
    (L.KVM_EINVAL, lambda: _rope(_view(2, 4, 128), _view(3, 4, 128))),
    (L.KVM_EINVAL, lambda: _rope(_view(2, 4, 128), _view(2, 4, 64))),
])
def test_norm_rope(code, call):
    assert call() == code


def _append(windows, cell0, counts, k, v, q=None, had=-1, q_type=L.T_F32):
    n = len(windows)
    arr = (C.POINTER(L.Window) * n)(*[C.pointer(w) for w in windows])
    r = L.RopeParams(64, 1e6, 1.0, had)
    return L.load().kvm_window_append(None, arr, (C.c_uint32 * n)(*cell0), (C.c_uint32 * n)(*counts), n, C.byref(k), C.byref(v),
                                      None, 1e-6, C.byref(r), 1 << 23, None if q is None else C.byref(q), None, q_type, 1 << 24)


@pytest.mark.parametrize("code,call", [
    (L.KVM_ERANGE, lambda: _append([_window()], [125], [4], _view(4, 2, 128), _view(4, 2, 128))),
    (L.KVM_ERANGE, lambda: _append([_window()], [2 ** 32 - 1], [4], _view(4, 2, 128), _view(4, 2, 128))),
    (L.KVM_EUNSUPPORTED, lambda: _append([_window(), _window(H=4)], [0, 0], [2, 2], _view(4, 2, 128), _view(4, 2, 128))),
    (L.KVM_EUNSUPPORTED, lambda: _append([_window(), _window(kt=L.T_Q4_0)], [0, 0], [2, 2], _view(4, 2, 128), _view(4, 2, 128))),
    (L.KVM_EUNSUPPORTED, lambda: _append([_window()], [0], [4], _view(4, 2, 128), _view(4, 2, 128), had=256)),
    (L.KVM_EUNSUPPORTED, lambda: _append([_window()], [0], [4], _view(4, 2, 128, L.T_Q4_0), _view(4, 2, 128))),
    (L.KVM_EUNSUPPORTED, lambda: _append([_window()], [0], [4], _view(4, 2, 128), _view(4, 2, 128), _view(4, 4, 128), q_type=L.T_Q4_0)),
    (L.KVM_EUNSUPPORTED, lambda: _append([_window(D=64)], [0], [4], _view(4, 2, 64), _view(4, 2, 64))),
    (L.KVM_EINVAL, lambda: _append([_window()], [0], [3], _view(4, 2, 128), _view(4, 2, 128))),
    (L.KVM_EINVAL, lambda: _append([_window()], [0], [4], _view(4, 4, 128), _view(4, 2, 128))),
])
def test_append(code, call):
    assert call() == code


def test_tokens_without_a_run():
    """No run holds no tokens: views that have some are refused, as where the runs hold too few."""
    r = L.RopeParams(64, 1e6, 1.0, -1)

    def call(k, v, q):
        refs = [None if x is None else C.byref(x) for x in (k, v, q)]
        return L.load().kvm_window_append(None, None, None, None, 0, refs[0], refs[1], None, 1e-6, C.byref(r), 1 << 23, refs[2], None,
                                          L.T_F32, 1 << 24)

    none, some = _view(0, 2, 128), _view(4, 2, 128)
    assert call(none, none, none) == call(None, None, None) == call(none, none, None) == L.KVM_OK
    for views in ((some, none, None), (none, some, None), (none, none, _view(4, 8, 128)), (some, some, _view(4, 8, 128))):
        assert call(*views) == L.KVM_EINVAL

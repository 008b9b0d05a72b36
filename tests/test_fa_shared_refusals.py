"""Arguments that kvm_fa_decode_shared refuses by their size or type, on the host alone."""
import ctypes as C

import pytest

from kvmem_amd import _lib as L


def _window(cells=128, H=2, D=128, kt=L.T_Q8_0, vt=L.T_Q4_0):
    w = L.Window(cells, H, D, 64, kt, vt)
    w.k, w.v, w.cell_pos = 1 << 20, 1 << 21, 1 << 22
    return w


def _at(w, off):
    w.v += off
    return w


def _call(prefix, windows, counts, heads=8, q_type=L.T_F32, out_type=L.T_F32, scale=1.0, lanes=None):
    n = len(counts)
    arr = (C.POINTER(L.Window) * max(n, 1))(*[C.pointer(w) if w else None for w in windows])
    return L.load().kvm_fa_decode_shared(None, None if prefix is None else C.byref(prefix), arr, (C.c_uint32 * max(n, 1))(*counts), n,
                                         1 << 23, q_type, 1 << 24, heads, scale, out_type, 1 << 25)


@pytest.mark.parametrize("code,call", [
    (L.KVM_OK, lambda: _call(_window(), [], [])),
    (L.KVM_OK, lambda: _call(_window(), [None], [0])),
    (L.KVM_ERANGE, lambda: _call(_window(), [None] * 65, [1] * 65)),
    (L.KVM_ERANGE, lambda: _call(_window(), [None], [2 ** 31])),
    (L.KVM_ERANGE, lambda: _call(_window(), [None, None], [2 ** 32 - 1, 2 ** 32 - 1])),
    (L.KVM_ERANGE, lambda: _call(_window(cells=64 * 65536), [None], [1])),
    (L.KVM_EUNSUPPORTED, lambda: _call(_window(), [_window(H=4)], [1])),
    (L.KVM_EUNSUPPORTED, lambda: _call(_window(), [_window(D=256)], [1])),
    (L.KVM_EUNSUPPORTED, lambda: _call(_window(), [_window(kt=L.T_F16, vt=L.T_F16)], [1])),
    (L.KVM_EUNSUPPORTED, lambda: _call(_window(D=64), [None], [1])),
    (L.KVM_EUNSUPPORTED, lambda: _call(_window(), [None], [1], q_type=L.T_F16)),
    (L.KVM_EUNSUPPORTED, lambda: _call(_window(), [None], [1], out_type=L.T_Q8_0)),
    (L.KVM_EINVAL, lambda: _call(None, [None], [1])),
    (L.KVM_EINVAL, lambda: _call(_window(), [None], [1], heads=7)),
    (L.KVM_EINVAL, lambda: _call(_window(), [None], [1], heads=0)),
    (L.KVM_EINVAL, lambda: _call(_window(), [None], [1], scale=float("nan"))),
    (L.KVM_EINVAL, lambda: _call(_window(), [None], [1], scale=3e38)),
    (L.KVM_EINVAL, lambda: _call(_window(cells=100), [None], [1])),
    (L.KVM_EINVAL, lambda: _call(_at(_window(), 8), [None], [1])),
    (L.KVM_EINVAL, lambda: _call(_window(), [_at(_window(), 4)], [1])),
])
def test_refusals(code, call):
    assert call() == code


@pytest.mark.parametrize("counts,heads", [([2 ** 31] * 4, 2 ** 31), ([2 ** 30] * 16 + [1], 2 ** 30), ([2 ** 31], 2 ** 31)])
def test_products_past_64_bits(counts, heads):
    """Tokens times heads of a group are compared without their product, which wraps to little."""
    assert _call(_window(H=1), [None] * len(counts), counts, heads=heads) == L.KVM_ERANGE

"""kvm_qk_norm_rope and kvm_window_append: rows against the formulas in 64 bits,
window bytes against kvm_quantize_rows + kvm_window_import_rows of the same rows and
against the oracle's stage-in chain, runs that share words or cells, strides, streams,
graphs and refusals."""
import ctypes as C
import gc
import math
import weakref

import numpy as np
import pytest
import torch

import oracle as O
from kvmem_amd import api, _lib as L

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                       # half a step of fp32, relative
BASE = 1e6
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}     # half a subnormal step
TYPES = {"q8_0": (L.T_Q8_0, L.T_Q4_0), "q4_0": (L.T_Q4_0, L.T_Q4_0), "f16": (L.T_F16, L.T_F16)}


def rand(rng, shape, dtype=torch.float32, scale=1.0):
    return (torch.from_numpy(rng.standard_normal(shape).astype(np.float32)) * scale).to(dtype).cuda()


def formula(x, w, eps, pos, n_rot, hadamard, freq_scale=1.0):
    """(result, bound of the fp32 chain's error) in 64 bits: x [tokens][heads][dims]."""
    x = x.detach().cpu().double().numpy()
    D = x.shape[-1]
    mag = np.abs(x)
    ops = 0
    if eps is not None:
        e = float(np.float32(eps))
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + e)
        if w is not None:
            x = x * w.detach().cpu().double().numpy()
        mag, ops = np.abs(x), 3                          # r, x r, (x r) w
    h = n_rot // 2
    if h:
        th = O.rope_theta(BASE, freq_scale, n_rot)
        ang = (pos.cpu().numpy().astype(np.float32)[:, None] * th[None]).astype(np.float64)[:, None]
        c, s = np.cos(ang), np.sin(ang)
        a, b, am, bm = x[..., :h].copy(), x[..., h:n_rot].copy(), mag[..., :h].copy(), mag[..., h:n_rot].copy()
        x = np.concatenate([a * c - b * s, a * s + b * c, x[..., n_rot:]], -1)
        both = (am * np.abs(c) + bm * np.abs(s), am * np.abs(s) + bm * np.abs(c))
        mag = np.concatenate([*both, mag[..., n_rot:]], -1)
        ops += 3                                         # cos or sin, product, sum
    if hadamard:
        m = np.array([[1.0]])
        while m.shape[0] < hadamard:
            m = np.block([[m, m], [m, -m]])
        m /= math.sqrt(hadamard)
        shape = x.shape
        x = (x.reshape(-1, hadamard) @ m).reshape(shape)
        mag = (mag.reshape(-1, hadamard) @ np.abs(m)).reshape(shape)
        ops += 2 + int(math.log2(hadamard))              # the scale and its product, the stages
    return x, mag * ((1 + U) ** (ops + 1) - 1)


def close(got, want, bound):
    g = got.detach().cpu().double().numpy()
    lim = bound + (np.abs(want) + bound) * HALF_STEP[got.dtype] + TINY[got.dtype]
    bad = np.abs(g - want) > lim
    assert g.shape == want.shape and not bad.any(), (int(bad.sum()), float((np.abs(g - want) - lim).max()))


def layout(x, how):
    """x [tokens][heads][dims] as a view of other strides."""
    n, h, d = x.shape
    if how == "packed":
        return x.contiguous()
    if how == "joint":                                   # part of a wider row
        y = torch.zeros((n, h + 3, d), dtype=x.dtype, device=x.device)
        y[:, 1:1 + h] = x
        return y[:, 1:1 + h]
    if how == "heads_first":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "dims_first":                              # a dim's values far apart
        return x.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    if how == "odd":                                     # rows that start at any element
        y = torch.zeros((n, h * d + 1), dtype=x.dtype, device=x.device)
        y[:, 1:] = x.reshape(n, h * d)
        return y[:, 1:].unflatten(1, (h, d))
    raise ValueError(how)


ROPE_CASES = [
    # D, q heads, kv heads, tokens, n_rot, hadamard, eps, weights, in, out, layout, first position
    (256, 24, 4, 1, 64, 256, 1e-6, True, torch.bfloat16, torch.bfloat16, "joint", 261113),
    (128, 8, 2, 33, 128, 0, 1e-6, True, torch.float32, torch.float32, "packed", 0),
    (128, 8, 2, 5, 128, 128, 1e-5, False, torch.float16, torch.float16, "odd", 9),
    (64, 3, 1, 7, 32, 64, 0.0, True, torch.float32, torch.bfloat16, "heads_first", 2 ** 31 - 9),
    (256, 5, 5, 2, 0, 0, 1e-6, True, torch.bfloat16, torch.float32, "dims_first", 3),
    (192, 4, 1, 3, 48, 64, 1e-6, True, torch.float32, torch.float32, "odd", 70001),
    (96, 2, 2, 4, 96, 0, None, False, torch.float16, torch.float32, "packed", 511),
    (8, 1, 1, 3, 8, 0, 1e-6, True, torch.float32, torch.float32, "packed", 1),
    (80, 71, 3, 2, 40, 0, 1e-6, False, torch.bfloat16, torch.float16, "joint", 12345),
    (128, 64, 64, 1, 64, 64, 1e-6, True, torch.bfloat16, torch.bfloat16, "packed", 4095),
    (256, 16, 2, 1500, 256, 0, 1e-6, True, torch.bfloat16, torch.bfloat16, "joint", 1),      # several rows a wave
    (128, 1, 1, 20011, 128, 128, 1e-6, True, torch.float32, torch.float32, "packed", 7),
    (64, 2, 1, 9000, 64, 0, None, False, torch.float16, torch.float16, "heads_first", 100000),
]


@pytest.mark.parametrize("case", ROPE_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_norm_rope_equals_the_formulas(kvm_state, case):
    D, Hq, Hk, n, n_rot, had, eps, weights, tin, tout, how, pos0 = case
    rng = np.random.default_rng(D * 1000 + n)
    q, k = layout(rand(rng, (n, Hq, D), tin, 1.7), how), layout(rand(rng, (n, Hk, D), tin, 0.01), how)
    qw, kw = (rand(rng, (D,)) + 1.0 if weights else None for _ in range(2))
    pos = torch.arange(pos0, pos0 + n, dtype=torch.int64).clamp(max=2 ** 31 - 1).to(torch.int32).cuda()
    qo, ko = api.qk_norm_rope(kvm_state, q, k, pos, n_rot, BASE, hadamard_nrot=had, q_weight=qw, k_weight=kw, eps=eps,
                              out_dtype=tout)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        close(got, *formula(x, w, eps, pos, n_rot, had))


def test_norm_rope_any_positions_and_one_tensor(kvm_state):
    """Positions in no order, repeated and negative; the queries or the keys alone give
    what both give together; a frequency scale."""
    rng = np.random.default_rng(3)
    q, k = rand(rng, (6, 8, 128)), rand(rng, (6, 2, 128))
    pos = torch.tensor([5, -3, 2 ** 24 + 1, 5, 0, 17], dtype=torch.int32).cuda()
    both = api.qk_norm_rope(kvm_state, q, k, pos, 128, BASE, freq_scale=0.25, eps=1e-6)
    qo, none = api.qk_norm_rope(kvm_state, q, None, pos, 128, BASE, freq_scale=0.25, eps=1e-6)
    assert none is None and torch.equal(qo, both[0])
    none, ko = api.qk_norm_rope(kvm_state, None, k, pos, 128, BASE, freq_scale=0.25, eps=1e-6)
    assert none is None and torch.equal(ko, both[1])
    close(both[0], *formula(q, None, 1e-6, pos, 128, 0, 0.25))
    assert torch.equal(both[0][0], api.qk_norm_rope(kvm_state, q[:1], None, pos[:1], 128, BASE, freq_scale=0.25, eps=1e-6)[0][0])
    for t in (both[0][4], both[1][4]):                   # position 0 turns nothing
        x = (q if t.shape[0] == 8 else k)[4]
        close(t[None], *formula(x[None], None, 1e-6, pos[4:5], 0, 0))


def test_norm_rope_rows_without_finite_values(kvm_state):
    """A NaN or infinity stays in its own row; a row of zeros is zeros."""
    rng = np.random.default_rng(4)
    q = rand(rng, (3, 4, 128))
    clean = api.qk_norm_rope(kvm_state, q, None, torch.arange(3, dtype=torch.int32).cuda(), 128, BASE, hadamard_nrot=128, eps=1e-6)[0]
    dirty = q.clone()
    dirty[0, 1, 7], dirty[2, 3, 100], dirty[1, 2] = float("nan"), float("inf"), 0.0
    got = api.qk_norm_rope(kvm_state, dirty, None, torch.arange(3, dtype=torch.int32).cuda(), 128, BASE, hadamard_nrot=128, eps=1e-6)[0]
    keep = torch.ones((3, 4), dtype=torch.bool)
    keep[0, 1] = keep[2, 3] = keep[1, 2] = False
    assert torch.equal(got[keep.cuda()], clean[keep.cuda()])
    assert got[0, 1].isnan().any() and not got[1, 2].any()


def test_norm_rope_in_place(kvm_state):
    rng = np.random.default_rng(5)
    pos = torch.arange(70, 170, dtype=torch.int32).cuda()
    for dt in (torch.float32, torch.bfloat16):
        q, k = rand(rng, (100, 6, 128), dt), rand(rng, (100, 2, 128), dt)
        want = api.qk_norm_rope(kvm_state, q, k, pos, 64, BASE, eps=1e-6)
        api.qk_norm_rope(kvm_state, q, k, pos, 64, BASE, eps=1e-6, q_out=q, k_out=k)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_norm_rope_far_strides(kvm_state):
    """Token strides whose offsets pass 32 bits."""
    rng = np.random.default_rng(6)
    far = torch.empty(2 * 1300000000 + 2048, dtype=torch.bfloat16, device="cuda")
    q = far.as_strided((3, 8, 128), (1300000000, 128, 1))
    src = rand(rng, (3, 8, 128), torch.bfloat16)
    q.copy_(src)
    pos = torch.tensor([1, 2, 3], dtype=torch.int32).cuda()
    assert torch.equal(api.qk_norm_rope(kvm_state, q, None, pos, 64, BASE, eps=1e-6)[0],
                       api.qk_norm_rope(kvm_state, src, None, pos, 64, BASE, eps=1e-6)[0])


# ---- appends ---------------------------------------------------------------------
def filled(st, rng, cells, H, D, cache, bt=64, shadow=False, pending=False):
    """A window whose every cell holds something."""
    w = api.KVWindow(st, cells, H, D, bt, *TYPES[cache], shadow=shadow, pending=pending)
    kr, vr = (api.quantize_rows(st, t, rand(rng, (cells, H * D))) for t in TYPES[cache])
    w.import_rows(0, kr, vr, torch.arange(cells, dtype=torch.int32).cuda())
    if pending:
        w.pending_rows.zero_()
    if shadow:
        w.shadow_rows.fill_(bt)
    return w


def twin(st, w):
    """A second window with the first one's contents."""
    o = api.KVWindow(st, w.n_cells, w.n_head_kv, w.head_dim, w.block_tokens, w.k_type, w.v_type,
                     shadow=w.k_shadow is not None, pending=w.pending_rows is not None)
    for f in ("k", "v", "cell_pos", "slot_block", "slot_base", "k_shadow", "shadow_rows", "pending_rows"):
        if getattr(w, f) is not None:
            getattr(o, f).copy_(getattr(w, f))
    return o


def same(a, b):
    for f in ("k", "v", "cell_pos", "slot_block", "slot_base", "k_shadow", "shadow_rows", "pending_rows"):
        x, y = getattr(a, f), getattr(b, f)
        assert (x is None) == (y is None) and (x is None or torch.equal(x, y)), f


def by_parts(st, w, cell0, k, v, pos, n_rot, had, eps, kw):
    """The same append by the calls there were: rows in fp32, quantised, imported."""
    n, H, D = k.shape
    if had < 0:
        had = 0 if w.k_type == L.T_F16 else D
    rows = api.qk_norm_rope(st, None, k, pos, n_rot, BASE, hadamard_nrot=had, k_weight=kw, eps=eps, out_dtype=torch.float32)[1]
    w.import_rows(cell0, api.quantize_rows(st, w.k_type, rows.view(n, H * D)),
                  api.quantize_rows(st, w.v_type, v.float().reshape(n, H * D)), pos)


APPEND_CASES = [
    # D, kv heads, cache, cells, cell0, tokens, n_rot, hadamard, eps, type, layout
    (256, 4, "q8_0", 256, 61, 1, 64, -1, 1e-6, torch.bfloat16, "joint"),
    (256, 4, "q8_0", 256, 0, 256, 64, -1, 1e-6, torch.float32, "packed"),
    (256, 4, "q4_0", 256, 13, 100, 64, -1, 1e-6, torch.bfloat16, "odd"),
    (128, 2, "q4_0", 192, 191, 1, 128, 0, None, torch.float16, "heads_first"),
    (128, 2, "f16", 128, 3, 5, 128, -1, 1e-6, torch.bfloat16, "joint"),
    (128, 8, "f16", 192, 8, 120, 96, 128, 1e-6, torch.float32, "dims_first"),
    (256, 2, "f16", 64, 63, 1, 0, 0, None, torch.float16, "packed"),
    (128, 1, "q8_0", 8192, 7, 8101, 128, -1, 1e-6, torch.bfloat16, "joint"),
    (256, 4, "q8_0", 4096, 1003, 2047, 64, -1, 1e-6, torch.bfloat16, "joint"),
    (128, 8, "f16", 4096, 5, 1025, 128, -1, 1e-6, torch.bfloat16, "joint"),
    (256, 2, "f16", 4096, 1023, 2500, 64, -1, 1e-6, torch.float32, "packed"),
    (256, 4, "q4_0", 2048, 62, 1300, 64, -1, 1e-6, torch.float16, "joint"),
    (128, 70, "q8_0", 64, 30, 3, 64, -1, 1e-6, torch.bfloat16, "packed"),
    (256, 5, "q4_0", 64, 0, 9, 256, 64, None, torch.float32, "packed"),
]


@pytest.mark.parametrize("case", APPEND_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_append_equals_the_calls_in_parts(kvm_state, case):
    D, H, cache, cells, cell0, n, n_rot, had, eps, dt, how = case
    st, rng = kvm_state, np.random.default_rng(D + cells + n)
    quant = cache != "f16"
    w = filled(st, rng, cells, H, D, cache, shadow=quant, pending=True)
    o = twin(st, w)
    k, v = (layout(rand(rng, (n, H, D), dt, 2.0), how) for _ in range(2))
    if n > 2:
        v[1, 0, :64] = 0.0                               # whole blocks of zeros
        k[2, H - 1] = 0.0
    pos = torch.from_numpy(rng.integers(0, 40000, n).astype(np.int32)).cuda()
    kw = None if eps is None else rand(rng, (D,)) + 1.0
    q = rand(rng, (n, 3 * H, D), dt)
    qw = None if eps is None else rand(rng, (D,)) + 1.0
    got = api.window_append(st, [w], [cell0], [n], k, v, pos, n_rot, BASE, hadamard_nrot=had, k_weight=kw, eps=eps, q=q,
                            q_weight=qw, q_out_dtype=torch.bfloat16)
    by_parts(st, o, cell0, k, v, pos, n_rot, had, eps, kw)
    same(w, o)
    width = had if had >= 0 else D if quant else 0
    assert torch.equal(got, api.qk_norm_rope(st, q, None, pos, n_rot, BASE, hadamard_nrot=width, q_weight=qw, eps=eps,
                                             out_dtype=torch.bfloat16)[0])


@pytest.mark.parametrize("kt", ["q8_0", "q4_0"])
@pytest.mark.parametrize("D,n_rot", [(256, 64), (128, 128)])
def test_append_writes_the_stage_in_bytes(kvm_state, kt, D, n_rot):
    """A key row that comes with the values of a history row ends with the bytes that the
    oracle's stage-in chain gives that row at the same position."""
    st, rng, H, n = kvm_state, np.random.default_rng(D), 2, 128
    t = TYPES[kt][0]
    raw = O.quant(t, rng.standard_normal(n * H * D).astype(np.float32)).reshape(n, -1)
    vals = O.dequant(t, raw.reshape(-1), n * H * D).reshape(n, H, D)
    w = api.KVWindow(st, 128, H, D, 128, *TYPES[kt])
    pos0 = 30011
    api.window_append(st, [w], [0], [n], torch.from_numpy(vals).cuda(), rand(rng, (n, H, D)),
                      torch.arange(pos0, pos0 + n, dtype=torch.int32).cuda(), n_rot, BASE)
    kr, _ = w.export_rows(0, n)
    want = O.stagein_k(raw.reshape(-1), n, H, D, n_rot, D, pos0, O.rope_theta(BASE, 1.0, n_rot), k_type=t)
    assert np.array_equal(kr.cpu().numpy().reshape(-1), want)


@pytest.mark.parametrize("cache", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("D", [128, 256])
def test_rows_come_back_from_any_cells(kvm_state, cache, D):
    """Rows imported into a window come back byte for byte from any run of its cells, K or V
    alone too, and nothing beside them is written."""
    st, rng, H, n = kvm_state, np.random.default_rng(D + 1), 3, 192
    kt, vt = TYPES[cache]
    rows = [api.quantize_rows(st, t, rand(rng, (n, H * D))).view(n, -1) for t in (kt, vt)]
    w = api.KVWindow(st, n, H, D, 64, kt, vt)
    w.import_rows(0, *rows, torch.arange(n, dtype=torch.int32).cuda())
    for cell0, m in ((0, n), (0, 1), (3, 1), (5, 8), (61, 7), (63, 2), (64, 64), (7, 130), (191, 1)):
        k, v = w.export_rows(cell0, m)
        assert torch.equal(k.view(m, -1), rows[0][cell0:cell0 + m]) and torch.equal(v.view(m, -1), rows[1][cell0:cell0 + m])
        one = [torch.full((m + 2, r.shape[1]), 0x5a, dtype=torch.uint8, device="cuda") if r.dtype == torch.uint8 else
               torch.full((m + 2, r.shape[1]), 7, dtype=r.dtype, device="cuda") for r in rows]
        for which in (0, 1):
            pair = [None, None]
            pair[which] = one[which][1:].data_ptr()
            assert st.lib.kvm_window_export_rows(st.h, C.byref(w.c), cell0, m, *pair) == L.KVM_OK
        torch.cuda.synchronize()
        for r, got in zip(rows, one):
            assert torch.equal(got[1:-1], r[cell0:cell0 + m])
            assert torch.equal(got[0], got[-1]) and bool((got[0] == got[0, 0]).all()) and got[0, 0].item() in (0x5a, 7)


@pytest.mark.parametrize("cache", ["q8_0", "q4_0", "f16"])
def test_append_runs(kvm_state, cache):
    """Runs of many windows and of one: empty ones, neighbours in one 8-cell group or one
    slot, the same cells twice (the later run's rows stay), more runs than a launch has."""
    st, rng, H, D = kvm_state, np.random.default_rng(17), 2, 128
    ws = [filled(st, rng, 128, H, D, cache, bt=32, pending=True) for _ in range(45)]
    runs = [(i, int(rng.integers(0, 120)), int(rng.integers(1, 9))) for i in range(45)]
    runs += [(0, 3, 0), (0, 40, 2), (0, 42, 3), (0, 41, 2), (0, 45, 1), (1, 0, 128), (1, 5, 3), (1, 5, 3), (2, 31, 2), (2, 8, 1),
             (2, 16, 1)]
    n = sum(r[2] for r in runs)
    k, v, q = rand(rng, (n, H, D), torch.bfloat16), rand(rng, (n, H, D), torch.bfloat16), rand(rng, (n, 4, D), torch.bfloat16)
    pos = torch.from_numpy(rng.integers(0, 9000, n).astype(np.int32)).cuda()
    os_ = [twin(st, w) for w in ws]
    got = api.window_append(st, [ws[r[0]] for r in runs], [r[1] for r in runs], [r[2] for r in runs], k, v, pos, 64, BASE, eps=1e-6,
                            q=q)
    at = 0
    for i, c0, m in runs:
        if m:
            by_parts(st, os_[i], c0, k[at:at + m], v[at:at + m], pos[at:at + m], 64, -1, 1e-6, None)
        at += m
    for w, o in zip(ws, os_):
        same(w, o)
    assert torch.equal(got, api.qk_norm_rope(st, q, None, pos, 64, BASE, hadamard_nrot=0 if cache == "f16" else D, eps=1e-6)[0])


@pytest.mark.parametrize("bt", [1, 4, 64])
def test_append_counts_of_small_slots(kvm_state, bt):
    """Slots smaller than the 8-cell groups keep their own counts."""
    st, rng, H, D = kvm_state, np.random.default_rng(bt), 1, 128
    w = filled(st, rng, 64, H, D, "q8_0", bt=bt, pending=True)
    o = twin(st, w)
    k, v = rand(rng, (9, H, D)), rand(rng, (9, H, D))
    pos = torch.arange(9, dtype=torch.int32).cuda()
    api.window_append(st, [w, w, w], [2, 5, 30], [3, 2, 4], k, v, pos, 64, BASE)
    at = 0
    for c0, m in ((2, 3), (5, 2), (30, 4)):
        by_parts(st, o, c0, k[at:at + m], v[at:at + m], pos[at:at + m], 64, -1, None, None)
        at += m
    same(w, o)


def test_append_without_finite_values(kvm_state):
    """A NaN or infinity of one block leaves every other block's bytes as they are."""
    st, rng, H, D = kvm_state, np.random.default_rng(8), 2, 128
    k, v = rand(rng, (11, H, D)), rand(rng, (11, H, D))
    pos = torch.arange(11, dtype=torch.int32).cuda()
    for bad in (float("nan"), float("inf"), -float("inf")):
        w, o = (api.KVWindow(st, 64, H, D, 64) for _ in range(2))
        api.window_append(st, [o], [3], [11], k, v, pos, 0, BASE, hadamard_nrot=0)
        kd, vd = k.clone(), v.clone()
        kd[4, 1, 40], vd[4, 1, 70] = bad, bad
        api.window_append(st, [w], [3], [11], kd, vd, pos, 0, BASE, hadamard_nrot=0)
        (ka, va), (kb, vb) = w.export_rows(0, 64), o.export_rows(0, 64)
        ka, kb = (x.view(64, H, 4, 34) for x in (ka, kb))
        va, vb = (x.view(64, H, 4, 18) for x in (va, vb))
        keep = torch.ones((64, H, 4), dtype=torch.bool).cuda()
        kk, kv = keep.clone(), keep.clone()
        kk[7, 1, 1], kv[7, 1, 2] = False, False
        assert torch.equal(ka[kk], kb[kk]) and torch.equal(va[kv], vb[kv])


def test_append_long_rows_as_views(kvm_state):
    """Views whose rows hold all heads of a token (ne1 = 1) are the same rows."""
    st, rng, H, D, n = kvm_state, np.random.default_rng(9), 4, 128, 6
    k, v = rand(rng, (n, H, D)), rand(rng, (n, H, D))
    pos = torch.arange(n, dtype=torch.int32).cuda()
    a, b = (api.KVWindow(st, 64, H, D, 64) for _ in range(2))
    api.window_append(st, [a], [1], [n], k, v, pos, 64, BASE, eps=1e-6)
    api.window_append(st, [b], [1], [n], k.view(n, 1, H * D), v.view(n, 2, H * D // 2), pos, 64, BASE, eps=1e-6)
    same(a, b)


def test_append_weights_of_long_rows(kvm_state):
    """Weights have head_dim values whatever the rows of the views hold: the same with several
    heads in a row, and one value for each of a row's is refused."""
    st, rng, H, D, n = kvm_state, np.random.default_rng(28), 4, 128, 6
    k, v, q = rand(rng, (n, H, D)), rand(rng, (n, H, D)), rand(rng, (n, 2 * H, D))
    kw, qw = rand(rng, (D,)) + 1.0, rand(rng, (D,)) + 1.0
    pos = torch.arange(n, dtype=torch.int32).cuda()
    a, b = (api.KVWindow(st, 64, H, D, 64) for _ in range(2))
    want = api.window_append(st, [a], [1], [n], k, v, pos, 64, BASE, eps=1e-6, k_weight=kw, q=q, q_weight=qw)
    long = (k.view(n, 1, H * D), v.view(n, 2, H * D // 2))
    got = api.window_append(st, [b], [1], [n], *long, pos, 64, BASE, eps=1e-6, k_weight=kw, q=q.view(n, 1, 2 * H * D), q_weight=qw)
    same(a, b)
    assert torch.equal(got.view(n, 2 * H, D), want)
    for bad in ({"k_weight": torch.ones(H * D, device="cuda")}, {"q": q, "q_weight": torch.ones(H * D, device="cuda")},
                {"k_weight": torch.ones(D - 1, device="cuda")}):
        with pytest.raises(L.KvmError) as e:
            api.window_append(st, [b], [1], [n], *long, pos, 64, BASE, eps=1e-6, **bad)
        assert e.value.code == L.KVM_EINVAL
    same(a, b)


def test_prepared_calls_keep_their_windows(kvm_state):
    """A prepared append or attention holds its windows, whatever becomes of the caller's list."""
    st, rng, H, D = kvm_state, np.random.default_rng(29), 2, 128
    k, v, q = rand(rng, (1, H, D)), rand(rng, (1, H, D)), rand(rng, (1, 4, D))
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    for prepare in (lambda ws: api.prepare_window_append(st, ws, [0], [1], k, v, pos, 64, BASE),
                    lambda ws: api.prepare_fa_decode_shared(st, None, ws, [1], q, pos, 4, 0.1)):
        ws = [api.KVWindow(st, 64, H, D, 64)]
        held = weakref.ref(ws[0])
        p = prepare(ws)
        ws.clear()
        gc.collect()
        assert held() is not None
        p()
        st.sync()
        del p
        gc.collect()
        assert held() is None


@pytest.mark.parametrize("tq,tk", [(torch.bfloat16, torch.float16), (torch.float32, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("how", [("packed", "packed"), ("odd", "heads_first"), ("dims_first", "packed")])
def test_queries_and_keys_of_different_types(kvm_state, tq, tk, how):
    """Queries and keys (and values) of unlike types and strides are rows like any others."""
    st, rng, D, n = kvm_state, np.random.default_rng(30), 128, 300
    q, k, v = layout(rand(rng, (n, 7, D), tq), how[0]), layout(rand(rng, (n, 2, D), tk), how[1]), layout(rand(rng, (n, 2, D), tq), how[0])
    pos = torch.arange(n, dtype=torch.int32).cuda()
    got = api.qk_norm_rope(st, q, k, pos, 64, BASE, eps=1e-6, out_dtype=torch.float32)
    for x, y in zip((q, k), got):
        close(y, *formula(x, None, 1e-6, pos, 64, 0))
    w, o = (api.KVWindow(st, 512, 2, D, 64) for _ in range(2))
    qo = api.window_append(st, [w], [3], [n], k, v, pos, 64, BASE, eps=1e-6, q=q, q_out_dtype=torch.float32)
    by_parts(st, o, 3, k, v, pos, 64, -1, 1e-6, None)
    same(w, o)
    assert torch.equal(qo, api.qk_norm_rope(st, q, None, pos, 64, BASE, hadamard_nrot=D, eps=1e-6, out_dtype=torch.float32)[0])


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
def test_append_far_cells(kvm_state, cache):
    """Cells whose offsets pass 32 bits end as an import of the same rows leaves them."""
    st, rng, H, D, n = kvm_state, np.random.default_rng(31), 8, 256, 37
    N = 64 * 65535 if cache == "q8_0" else 2 ** 20
    w = api.KVWindow(st, N, H, D, 64, *TYPES[cache])
    k, v = rand(rng, (n, H, D)), rand(rng, (n, H, D))
    pos = torch.arange(n, dtype=torch.int32).cuda()
    at = (0, N // 2 + 5, N - n)
    for c in at:
        by_parts(st, w, c, k, v, pos, 64, -1, 1e-6, None)
    want = [w.export_rows(c, n) for c in at]
    for c in at:
        api.window_append(st, [w], [c], [n], v, k, pos, 64, BASE, eps=1e-6)
    api.window_append(st, [w] * 3, at, [n] * 3, k.repeat(3, 1, 1), v.repeat(3, 1, 1), pos.repeat(3), 64, BASE, eps=1e-6)
    for c, rows in zip(at, want):
        assert all(torch.equal(a, b) for a, b in zip(w.export_rows(c, n), rows))
        assert torch.equal(w.cell_pos[c:c + n], pos)


def test_append_on_another_stream_and_replayed(kvm_state):
    """On a stream of its own, and captured: every replay appends the rows that its inputs
    then hold, beside eager calls between the replays."""
    rng, H, D, n = np.random.default_rng(10), 4, 256, 4
    s = torch.cuda.Stream()
    st = api.State(0, stream=s.cuda_stream)
    try:
        w = api.KVWindow(st, 256, H, D, 64, pending=True)
        other = api.KVWindow(st, 256, H, D, 64)
        k, v, q = (rand(rng, (n, h, D), torch.bfloat16) for h in (H, H, 6 * H))
        pos = torch.arange(100, 100 + n, dtype=torch.int32).cuda()
        p = api.prepare_window_append(st, [w], [77], [n], k, v, pos, 64, BASE, eps=1e-6, q=q)
        r = api.prepare_qk_norm_rope(st, q, k, pos, 64, BASE, eps=1e-6)
        torch.cuda.synchronize()
        g = st.capture(lambda: (p(), r()))
        for i in range(4):
            for x in (k, v, q):
                x.copy_(rand(rng, x.shape, x.dtype))
            pos.add_(1 + i)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            o = api.KVWindow(st, 256, H, D, 64, pending=True)
            torch.cuda.synchronize()
            want = api.window_append(st, [o], [77], [n], k, v, pos, 64, BASE, eps=1e-6, q=q)
            eager = api.qk_norm_rope(st, q, k, pos, 64, BASE, eps=1e-6)
            api.window_append(st, [other], [5], [n], v, k, pos, 64, BASE)
            torch.cuda.synchronize()
            same(w, o)
            assert torch.equal(p.q_out, want) and torch.equal(r.q_out, eager[0]) and torch.equal(r.k_out, eager[1])
    finally:
        torch.cuda.synchronize()
        st.close()


def test_refusals(kvm_state):
    """What the entry points do not take is refused before anything is written."""
    st, rng, H, D = kvm_state, np.random.default_rng(11), 2, 128
    q, k, v = rand(rng, (4, 8, D)), rand(rng, (4, H, D)), rand(rng, (4, H, D))
    pos = torch.arange(4, dtype=torch.int32).cuda()
    w = filled(st, rng, 128, H, D, "q8_0")
    was = twin(st, w)

    def refused(code, fn, *a, **kw):
        with pytest.raises(L.KvmError) as e:
            fn(st, *a, **kw)
        assert e.value.code == code, e.value

    rope, app = api.qk_norm_rope, api.window_append
    refused(L.KVM_EUNSUPPORTED, rope, q, k, pos, 12, BASE)                       # n_rot not a multiple of 8
    refused(L.KVM_EUNSUPPORTED, rope, q, k, pos, 136, BASE)
    refused(L.KVM_EUNSUPPORTED, rope, q, k, pos, 64, BASE, hadamard_nrot=32)
    refused(L.KVM_EINVAL, rope, q, k, pos, 64, BASE, hadamard_nrot=-1)
    refused(L.KVM_EINVAL, rope, q, k, pos, 64, -1.0)
    refused(L.KVM_EINVAL, rope, q, k, pos, 64, BASE, eps=float("nan"))
    refused(L.KVM_EINVAL, rope, q, k[:3], pos, 64, BASE)
    refused(L.KVM_EINVAL, rope, q, k, pos[:3], 64, BASE)
    refused(L.KVM_EINVAL, rope, q, k, pos.long(), 64, BASE)
    refused(L.KVM_EINVAL, rope, q.cpu(), k, pos, 64, BASE)
    refused(L.KVM_EINVAL, rope, q, k, pos, 64, BASE, q_weight=torch.ones(D - 1).cuda())
    refused(L.KVM_EINVAL, rope, q, k, pos, 64, BASE, q_out=q[:, :, :64])
    refused(L.KVM_EINVAL, rope, q, k, pos, 64, BASE, k_out=q.view(-1)[:k.numel()].view(k.shape))
    refused(L.KVM_EINVAL, rope, q[:, :2], k, pos, 64, BASE, q_out=q.view(-1)[:k.numel()].view(k.shape))
    refused(L.KVM_EUNSUPPORTED, rope, rand(rng, (4, 2, 264)), None, pos, 64, BASE)
    refused(L.KVM_EUNSUPPORTED, rope, rand(rng, (4, 2, 20)), None, pos, 8, BASE)
    refused(L.KVM_ERANGE, app, [w], [125], [4], k, v, pos, 64, BASE)             # past the window
    refused(L.KVM_ERANGE, app, [w], [2 ** 32 - 2], [4], k, v, pos, 64, BASE)
    refused(L.KVM_EINVAL, app, [w], [0], [3], k, v, pos, 64, BASE)               # a token too many
    refused(L.KVM_EINVAL, app, [w], [0], [-1], k, v, pos, 64, BASE)
    refused(L.KVM_EINVAL, app, [w], [0], [4], k, v[:3], pos, 64, BASE)
    refused(L.KVM_EINVAL, app, [w], [0], [4], q, v, pos, 64, BASE)               # as many heads as the window
    refused(L.KVM_EINVAL, app, [w], [0, 4], [4], k, v, pos, 64, BASE)
    refused(L.KVM_EINVAL, app, [None], [0], [4], k, v, pos, 64, BASE)
    refused(L.KVM_EUNSUPPORTED, app, [w, api.KVWindow(st, 64, H, D, 64, L.T_F16, L.T_F16)], [0, 0], [2, 2], k, v, pos, 64, BASE)
    refused(L.KVM_EUNSUPPORTED, app, [w], [0], [4], k, v, pos, 64, BASE, hadamard_nrot=256)
    refused(L.KVM_EINVAL, app, [w], [0], [4], k, v, pos, 64, BASE, q=q, q_out=torch.empty_like(q[:, :4]))
    refused(L.KVM_EINVAL, app, [w], [0], [4], k, v, pos, 64, BASE, q=q[:, :2].contiguous(), q_out=v)
    st.sync()
    same(w, was)


def test_no_tokens(kvm_state):
    st = kvm_state
    w = api.KVWindow(st, 64, 2, 128, 64)
    was = twin(st, w)
    none = torch.empty((0, 2, 128), device="cuda")
    pos = torch.empty((0,), dtype=torch.int32, device="cuda")
    assert api.qk_norm_rope(st, none, none, pos, 64, BASE)[0].shape == none.shape
    api.window_append(st, [w, w], [0, 64], [0, 0], none, none, pos, 64, BASE)
    api.window_append(st, [], [], [], none, none, pos, 64, BASE)
    st.sync()
    same(w, was)

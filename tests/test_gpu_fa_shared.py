"""kvm_fa_decode_shared against softmax attention in 64 bits over the cells' values:
prefixes and conversations of many sizes, ragged token counts, every type, masks that
leave a row or a tile empty, what is not finite at cells that are not seen, streams,
graphs and refusals; and a layer's step: append, then attend."""
import math

import numpy as np
import pytest
import torch

import oracle as O
from kvmem_amd import api, _lib as L

pytestmark = pytest.mark.gpu

TYPES = {"q8_0": (L.T_Q8_0, L.T_Q4_0), "q4_0": (L.T_Q4_0, L.T_Q4_0), "f16": (L.T_F16, L.T_F16)}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def window(st, rng, cells, H, D, cache, pos, bt=64):
    """A window of random rows at the given positions, and the cells' values in 64 bits."""
    w = api.KVWindow(st, cells, H, D, bt, *TYPES[cache])
    rows, vals = [], []
    for t in TYPES[cache]:
        r = api.quantize_rows(st, t, torch.from_numpy(rng.standard_normal((cells, H * D)).astype(np.float32)).cuda())
        rows.append(r)
        vals.append(api.dequantize_rows(st, t, r, H * D).double().view(cells, H, D))
    p = torch.from_numpy(np.asarray(pos, np.int32)).cuda()
    w.import_rows(0, rows[0], rows[1], p)
    return w, vals[0], vals[1], p


def expected(q, q_pos, counts, prefix, owns, H, scale):
    """(softmax attention, bound of the f16 operands' error) in 64 bits.  prefix and owns:
    (window, K, V, positions) or None.

    Half steps of f16 are u = 2^-11.  A score's terms carry u for q and u for k (a bf16 q
    and an f16 cell none, not used): |ds| <= 2u scale sum |q k|; p changes by a factor
    exp(+-2 ds) at most against the others; p and v are rounded: u each.  So an output,
    a weighted mean, is off by (exp(2 ds) (1 + u)^3 - 1) sum p |v| / sum p at most; fp32
    sums of n terms add n 2^-24 of it.  Probabilities below f16's range lose up to 2^-25
    of the row's reference, which is within 2^8 of its maximum: 2^-17 of the largest p
    each, n of them."""
    n, Hq, D = q.shape
    G, u = Hq // H, 2.0 ** -11
    q = q.double()
    out, lim = torch.zeros((n, Hq, D), dtype=torch.float64, device="cuda"), torch.zeros((n, Hq, D), dtype=torch.float64, device="cuda")
    at = 0
    for m, own in zip(counts, owns):
        parts = [x for x in (prefix, own) if x is not None]
        for t in range(at, at + m):
            seen = [(x[3] >= 0) & (x[3] <= q_pos[t]) for x in parts]
            if not any(bool(s.any()) for s in seen):
                continue
            for h in range(H):
                k = torch.cat([x[1][s, h] for x, s in zip(parts, seen)])
                v = torch.cat([x[2][s, h] for x, s in zip(parts, seen)])
                qq = q[t, h * G:(h + 1) * G]
                s = (k @ qq.t().contiguous()).t() * scale
                e = (k.abs() @ qq.abs().t().contiguous()).t().amax(1) * abs(scale) * 2 * u
                p = torch.softmax(s, 1)
                mean = p @ v.abs()
                cells = k.shape[0]
                out[t, h * G:(h + 1) * G] = p @ v
                lim[t, h * G:(h + 1) * G] = mean * (torch.exp(2 * e)[:, None] * (1 + u) ** 3 - 1 + cells * 2.0 ** -24) \
                    + p.amax(1, keepdim=True) * v.abs().sum(0) * 2.0 ** -17
        at += m
    return out, lim


def check(got, want, lim):
    err = (got.double() - want).abs()
    bound = lim + (want.abs() + lim) * HALF_STEP[got.dtype]
    assert not bool((~(err <= bound)).any()), float((err - bound).max())
    ref = want.norm()
    if float(ref):
        # and far closer on the whole: roundings do not all point one way
        rel = float((got.double() - want).norm() / ref)
        assert rel <= 2e-3 + HALF_STEP[got.dtype], rel


def run(st, rng, H, G, D, cache, prefix_cells, prefix_pos, lanes, counts, q_dtype, out_dtype, scale=None, q_pos=None):
    """lanes: (cells, positions) or None for each."""
    scale = D ** -0.5 if scale is None else scale
    prefix = None if not prefix_cells else window(st, rng, prefix_cells, H, D, cache, prefix_pos)
    owns = [None if x is None else window(st, rng, x[0], H, D, cache, x[1]) for x in lanes]
    n = sum(counts)
    q = torch.from_numpy(rng.standard_normal((n, H * G, D)).astype(np.float32)).to(q_dtype).cuda()
    qp = torch.from_numpy(np.asarray(q_pos, np.int32)).cuda()
    got = api.fa_decode_shared(st, prefix and prefix[0], [x and x[0] for x in owns], counts, q, qp, H * G, scale, out_dtype=out_dtype)
    check(got, *expected(q, qp, counts, prefix, owns, H, scale))
    return got, prefix, owns, q, qp


def cells(n, live, first, hole=0):
    """Positions of a window's n cells: `live` from `first` on, the rest empty."""
    p = np.where(np.arange(n) < live, first + np.arange(n), -1)
    if hole:
        p[::hole] = -1
    return p


CASES = [
    # H, G, D, cache, prefix cells, live, [own cells, live], counts, q, out
    (2, 4, 128, "f16", 1024, 1000, [(256, 130), (256, 3)], [1, 1], torch.bfloat16, torch.bfloat16),
    (4, 6, 256, "q8_0", 4096, 4096, [(512, 400)] * 8, [1] * 8, torch.bfloat16, torch.bfloat16),
    (4, 6, 256, "q8_0", 2048, 1999, [(512, 500), (64, 5), (1024, 700)], [4, 1, 5], torch.float32, torch.float32),
    (1, 8, 256, "q4_0", 1984, 1961, [(192, 190), (128, 1), (64, 64), (64, 9)], [3, 0, 2, 4], torch.bfloat16, torch.float32),
    (8, 4, 128, "f16", 640, 640, [(128, 100)] * 5, [3] * 5, torch.float32, torch.float16),
    (2, 1, 256, "f16", 320, 311, [(64, 33), (64, 2)], [1, 2], torch.bfloat16, torch.float32),
    (3, 5, 128, "q8_0", 128, 65, [(64, 1), None, (64, 64)], [1, 2, 1], torch.float32, torch.bfloat16),
    (1, 1, 128, "q4_0", 64, 1, [None], [1], torch.float32, torch.float32),
    (2, 2, 128, "q8_0", 0, 0, [(64, 10), (4096, 4000)], [1, 1], torch.float32, torch.float32),
    (1, 64, 128, "f16", 256, 200, [(64, 20)] * 3, [1, 2, 1], torch.bfloat16, torch.bfloat16),
    (1, 2, 128, "q8_0", 512, 512, [(64, 20)] * 64, [1] * 64, torch.bfloat16, torch.bfloat16),
    (2, 3, 256, "q4_0", 256, 256, [(64, 40)] * 2, [40, 33], torch.bfloat16, torch.bfloat16),     # chunks, not single tokens
    (4, 6, 256, "f16", 1024, 1024, [(256, 250)] * 4, [4, 3, 2, 1], torch.bfloat16, torch.float32),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c)[:90])
def test_equals_softmax_in_64_bits(kvm_state, case):
    H, G, D, cache, pc, live, lanes, counts, qd, od = case
    rng = np.random.default_rng(pc + D + G)
    own = [x and (x[0], cells(x[0], x[1], live)) for x in lanes]
    ends = [live + (x[1] if x else 0) for x in lanes]
    qp = np.concatenate([np.arange(e - m, e) for e, m in zip(ends, counts)])
    run(kvm_state, rng, H, G, D, cache, pc, cells(pc, live, 0) if pc else None, own, counts, qd, od, q_pos=qp)


@pytest.mark.parametrize("H,D,cache", [(8, 128, "q8_0"), (4, 256, "q4_0")])
def test_few_rows_beside_many(kvm_state, H, D, cache):
    """A prefix of many rows, and conversations of one token and of many, in no order: what
    quantised windows of few rows and of many take different ways for, in one call."""
    rng, G, P = np.random.default_rng(16), 8, 2048
    counts = [1, 9, 8, 0, 20, 8, 17, 3, 16, 16, 8, 8, 8, 8]
    lanes = [(64 * (1 + i % 5), 40 + 11 * (i % 9)) for i in range(len(counts))]
    own = [None if i == 5 else (n, cells(n, min(n, m), P)) for i, (n, m) in enumerate(lanes)]
    qp = np.concatenate([P + min(n, m) - c + np.arange(c) for (n, m), c in zip(lanes, counts)])
    run(kvm_state, rng, H, G, D, cache, P, cells(P, P, 0), own, counts, torch.bfloat16, torch.float32, q_pos=qp)


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
def test_no_prefix(kvm_state, cache):
    """Conversations alone, of hundreds of rows and of few, one without cells: its tokens give
    zeros, whatever was there."""
    rng, H, G, D = np.random.default_rng(18), 4, 8, 128
    lanes, counts = [(192, 150), (4096, 4000), None, (64, 1), (640, 600)], [1, 80, 3, 1, 6]
    qp = np.concatenate([(x[1] if x else 5) - c + np.arange(c) for x, c in zip(lanes, counts)])
    got, *_ = run(kvm_state, rng, H, G, D, cache, 0, None, [x and (x[0], cells(x[0], x[1], 0)) for x in lanes], counts,
                  torch.float32, torch.bfloat16, q_pos=qp)
    assert not got[81:84].any() and bool(got[:81].any(2).all()) and bool(got[84:].any(2).all())


def test_a_window_twice(kvm_state):
    """The prefix's window as a lane's own too, and one window for two lanes: its cells count twice."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(19), 2, 4, 128
    pre, own = (window(st, rng, n, H, D, "q8_0", cells(n, n, 0)) for n in (256, 64))
    q = torch.from_numpy(rng.standard_normal((3, H * G, D)).astype(np.float32)).cuda()
    qp = torch.tensor([200, 40, 63], dtype=torch.int32, device="cuda")
    owns = [pre, own, own]
    got = api.fa_decode_shared(st, pre[0], [x[0] for x in owns], [1, 1, 1], q, qp, H * G, D ** -0.5)
    check(got, *expected(q, qp, [1, 1, 1], pre, owns, H, D ** -0.5))


def test_output_over_the_queries(kvm_state):
    """The output may be the queries' memory: they are read before it is written."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(20), 2, 4, 128
    w = window(st, rng, 512, H, D, "q8_0", cells(512, 512, 0))
    q = torch.from_numpy(rng.standard_normal((2, H * G, D)).astype(np.float32)).cuda()
    qp = torch.tensor([511, 300], dtype=torch.int32, device="cuda")
    want = api.fa_decode_shared(st, w[0], [None, None], [1, 1], q, qp, H * G, D ** -0.5)
    assert torch.equal(api.fa_decode_shared(st, w[0], [None, None], [1, 1], q, qp, H * G, D ** -0.5, out=q), want)


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
def test_long_prefix(kvm_state, cache):
    """Many tiles a wave, several looks at a piece's tiles (one kv head, one row group: all
    tiles of 524,288 cells are a few workgroups' when the chip has few)."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(2), 1, 2, 128
    n = 131072
    p = cells(n, n - 77, 0, hole=1013)
    run(st, rng, H, G, D, cache, n, p, [(64, cells(64, 3, n))], [1], torch.bfloat16, torch.float32, q_pos=[n + 2])


def test_many_tiles_a_workgroup(kvm_state):
    """More tiles a workgroup than it looks at at a time: 8 kv heads x 5 row groups x 2,048 tiles."""
    st, rng, n = kvm_state, np.random.default_rng(14), 131072
    p = rng.permutation(n)
    p[rng.random(n) < 0.01] = -1
    run(st, rng, 8, 4, 128, "q8_0", n, p, [None, None], [20, 20], torch.bfloat16, torch.float32,
        q_pos=rng.integers(n // 2, n, 40))


@pytest.mark.parametrize("cache,H,G,tokens", [("q8_0", 8, 1, 1), ("f16", 4, 1, 1), ("q8_0", 4, 8, 9)])
def test_pieces_longer_than_a_look(kvm_state, cache, H, G, tokens):
    """As many units as the chip has workgroups, so that each is a piece of its own, of more tiles
    than are looked at at a time: sixty-four conversations over the same window."""
    st, rng, D, n = kvm_state, np.random.default_rng(21), 128, 64 * 301
    p = rng.permutation(n)
    p[rng.random(n) < 0.02] = -1
    p[64 * 270:64 * 280] = -1
    w = window(st, rng, n, H, D, cache, p)
    counts = [tokens] * 64
    q = torch.from_numpy(rng.standard_normal((64 * tokens, H * G, D)).astype(np.float32)).cuda()
    qp = torch.from_numpy(rng.integers(-3, n, 64 * tokens).astype(np.int32)).cuda()
    got = api.fa_decode_shared(st, None, [w[0]] * 64, counts, q, qp, H * G, D ** -0.5)
    check(got, *expected(q, qp, counts, None, [w] * 64, H, D ** -0.5))


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
@pytest.mark.parametrize("rows", [31, 32, 33, 63, 64, 65, 96, 97, 127, 128, 129, 257])
def test_row_counts_at_the_units_edges(kvm_state, cache, rows):
    """One conversation of that many rows of a kv head, over a prefix and its own cells."""
    rng = np.random.default_rng(rows)
    run(kvm_state, rng, 1, 1, 128, cache, 192, cells(192, 190, 0), [(320, cells(320, 320, 190))], [rows], torch.bfloat16,
        torch.float32, q_pos=np.arange(510 - rows, 510))


def test_workspace_under_capture(kvm_state):
    """A capture that needs a larger workspace is refused; one captured before another call
    grew it replays on the one it had."""
    st, rng, H, D = api.State(0), np.random.default_rng(15), 1, 128
    try:
        w = window(st, rng, 256, H, D, "q8_0", cells(256, 256, 0))[0]
        big = window(st, rng, 65536, 8, D, "q8_0", cells(65536, 65536, 0))[0]
        q = torch.from_numpy(rng.standard_normal((1, 4, D)).astype(np.float32)).cuda()
        pos = torch.tensor([300], dtype=torch.int32, device="cuda")
        small = api.prepare_fa_decode_shared(st, w, [None], [1], q, pos, 4, 0.1)
        qb = torch.from_numpy(rng.standard_normal((64, 64, D)).astype(np.float32)).cuda()
        pb = torch.full((64,), 70000, dtype=torch.int32, device="cuda")
        large = api.prepare_fa_decode_shared(st, big, [None], [64], qb, pb, 64, 0.1)
        small()
        torch.cuda.synchronize()
        want = small.out.clone()
        g = st.capture(small)
        with pytest.raises(L.KvmError) as e:
            st.capture(large)
        assert e.value.code == L.KVM_ENOMEM
        torch.cuda.synchronize()
        large()
        torch.cuda.synchronize()
        for _ in range(3):
            small.out.zero_()
            g.replay()
            large()
            torch.cuda.synchronize()
            assert torch.equal(small.out, want)
    finally:
        torch.cuda.synchronize()
        st.close()


@pytest.mark.parametrize("cache,D", [("f16", 256), ("q8_0", 128)])
def test_captures_of_smaller_calls(kvm_state, cache, D):
    """After one call on a fresh state, calls of no more tokens and cells can be captured, however
    many tokens they have (fewer can ask for more pieces) and however these are spread over lanes."""
    st, H, G, n = api.State(0), 8, 8, 32768
    try:
        torch.manual_seed(26)
        w = api.KVWindow(st, n, H, D, 64, *TYPES[cache])
        w.import_rows(0, *(api.quantize_rows(st, t, torch.randn(n, H * D, device="cuda")) for t in TYPES[cache]),
                      torch.arange(n, dtype=torch.int32, device="cuda"))
        q = torch.randn(96, H * G, D, device="cuda")
        pos = torch.full((96,), n, dtype=torch.int32, device="cuda")
        full = api.prepare_fa_decode_shared(st, w, [None], [96], q, pos, H * G, D ** -0.5)
        full()
        for counts in ([64], [16], [1], [1] * 64, [40, 56], [5]):
            m = sum(counts)
            p = api.prepare_fa_decode_shared(st, w, [None] * len(counts), counts, q[:m], pos[:m], H * G, D ** -0.5)
            g = st.capture(p)
            for _ in range(2):
                p.out.zero_()
                torch.cuda.synchronize()
                g.replay()
                full()
                torch.cuda.synchronize()
                rel = float((p.out - full.out[:m]).norm() / full.out[:m].norm())
                assert rel <= 1e-3, (counts, rel)        # (two forms of 3e-4 each)
    finally:
        torch.cuda.synchronize()
        st.close()


def test_rows_that_see_little_or_nothing(kvm_state):
    """Rows whose positions lie before every cell give zeros; others see a single cell, a part
    of the prefix and none of their own, or cells in no order with holes and whole empty tiles."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(3), 2, 3, 128
    pre = rng.permutation(640).astype(np.int64) + 10
    pre[64:192] = -1
    pre[200::7] = -1
    own = [(128, np.where(np.arange(128) % 3 == 0, 700 + np.arange(128), -1)), (64, np.full(64, -1)), None]
    for cache in ("q8_0", "f16"):
        got, prefix, *_ = run(st, rng, H, G, D, cache, 640, pre, own, [3, 2, 2], torch.float32, torch.float32,
                              q_pos=[5, 11, 760, -1, 300, 2 ** 31 - 1, 9])
        assert not got[0].any() and not got[3].any() and not got[6].any()
        first = int(np.flatnonzero((pre >= 0) & (pre <= 11))[0]) if ((pre >= 0) & (pre <= 11)).sum() == 1 else None
        if first is not None:
            assert torch.equal(got[1].view(H, G, D)[:, 0], prefix[2][first].float())


@pytest.mark.parametrize("cache", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_rows_that_see_one_cell(kvm_state, cache, tokens):
    """A row that sees a single cell, of the prefix or of its own window, gives that cell's values as
    the f16 operands hold them, to fp32's roundings."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(27), 2, 3, 128
    pre, own = rng.permutation(640) + 10, np.full(128, -1)
    own[[3, 77]] = 500, 5
    prefix, mine = window(st, rng, 640, H, D, cache, pre), window(st, rng, 128, H, D, cache, own)
    counts, at = [tokens, tokens], [(prefix, int(np.flatnonzero(pre == 10)[0])), (mine, 77)]
    q = torch.from_numpy(rng.standard_normal((2 * tokens, H * G, D)).astype(np.float32)).cuda()
    qp = torch.tensor([10] * tokens + [9] * tokens, dtype=torch.int32, device="cuda")
    assert int(((pre >= 0) & (pre <= 10)).sum()) == 1 and not ((pre >= 0) & (pre <= 9)).any()
    assert int(((own >= 0) & (own <= 9)).sum()) == 1
    got = api.fa_decode_shared(st, prefix[0], [None, mine[0]], counts, q, qp, H * G, D ** -0.5).view(2, tokens, H, G, D)
    # p = exp2(fma(s, c, -fl(s c))), c = scale log2 e: 1 but for the rounding of s c, at most |s c| 2^-24
    # of the exponent, so |scale s| 2^-24 of p (2^x's derivative is ln 2 of it); exp2's own ulp, 1 / l and
    # its product add 2^-23 + 2 x 2^-24.  The f16 p is 1: values come out within that of themselves.
    for i, (w, c) in enumerate(at):
        score = (q.view(2, tokens, H, G, D)[i].double() * w[1][c][None, :, None]).abs().sum(-1) * D ** -0.5
        want = w[2][c].half().double()[None, :, None].expand(tokens, H, G, D)
        assert bool(((got[i].double() - want).abs() <= want.abs() * (1.01 * score[..., None] + 4) * 2.0 ** -24).all())


def test_empty_windows(kvm_state):
    """Nothing anywhere: zeros, whatever was there; no tokens: nothing is written."""
    st, rng = kvm_state, np.random.default_rng(4)
    got, *_ = run(st, rng, 1, 4, 128, "q8_0", 128, np.full(128, -1), [(64, np.full(64, -1))] * 2, [1, 2], torch.float32,
                  torch.float32, q_pos=[5, 6, 7])
    assert not got.any()
    w = window(st, rng, 64, 1, 128, "q8_0", cells(64, 64, 0))[0]
    none = torch.empty((0, 4, 128), device="cuda")
    pos = torch.empty((0,), dtype=torch.int32, device="cuda")
    assert api.fa_decode_shared(st, w, [None, w], [0, 0], none, pos, 4, 1.0).shape == none.shape


@pytest.mark.parametrize("scale", [0.0, -0.07, 3.0])
def test_scales(kvm_state, scale):
    """Equal weights, a negative scale, scores that grow far past the first tile's."""
    run(kvm_state, np.random.default_rng(5), 2, 4, 128, "f16", 1024, cells(1024, 1024, 0), [(128, cells(128, 100, 1024))] * 3,
        [2, 1, 1], torch.bfloat16, torch.float32, scale=scale, q_pos=[1100, 1110, 1123, 1060])


def test_scores_that_keep_growing(kvm_state):
    """Keys along the query, longer from tile to tile: every wave moves its maximum often."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(6), 1, 2, 128
    n = 2048
    q = torch.ones((1, G, D), dtype=torch.float32, device="cuda")
    k = np.ones((n, D), np.float32) * (np.arange(n)[:, None] // 64 * 0.5)
    v = rng.standard_normal((n, D)).astype(np.float32)
    w = api.KVWindow(st, n, H, D, 64, *TYPES["f16"])
    rows = [api.quantize_rows(st, L.T_F16, torch.from_numpy(x).cuda()) for x in (k, v)]
    pos = torch.from_numpy(rng.permutation(n).astype(np.int32)).cuda()
    w.import_rows(0, *rows, pos)
    kd, vd = (api.dequantize_rows(st, L.T_F16, x, D).double().view(n, H, D) for x in rows)
    qp = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = api.fa_decode_shared(st, w, [None], [1], q, qp, G, 0.3)
    check(got, *expected(q, qp, [1], (w, kd, vd, pos), [None], H, 0.3))


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_seen_is_not_used(kvm_state, cache, what):
    """NaN and infinities in empty cells, and in cells that some tokens of a unit see and others
    do not: a token's output is as if what it does not see held zeros."""
    st, H, G, D = kvm_state, 2, 3, 128
    lanes, counts = [(128, cells(128, 40, 256)), (64, cells(64, 9, 256))], [4, 3]
    qp = np.concatenate([np.arange(292, 296), np.arange(262, 265)])
    outs = []
    for bad in (False, True):
        rng = np.random.default_rng(7)
        got, prefix, owns, q, qpos = run(st, rng, H, G, D, cache, 320, cells(320, 256, 0), lanes, counts, torch.float32, torch.float32,
                                         q_pos=qp)
        if bad:
            raw = {"f16": lambda x: x.view(torch.float16), "q8_0": lambda x: x.view(torch.float16)}[cache]
            for w, empties in ((prefix[0], range(256, 320)), (owns[0][0], range(40, 128)), (owns[1][0], range(9, 64))):
                for c in empties:
                    for h in range(H):
                        _poison(w, cache, c, h, what)
            # lane 0's last token (cell 39, position 295) and lane 1's last two: later tokens' own cells
            _poison(owns[0][0], cache, 39, 1, what)
            _poison(owns[1][0], cache, 7, 0, what)
            _poison(owns[1][0], cache, 8, 0, what)
            got = api.fa_decode_shared(st, prefix[0], [x[0] for x in owns], counts, q, qpos, H * G, D ** -0.5)
        outs.append(got)
    clean, dirty = (x.view(7, H, G, D) for x in outs)
    same = torch.ones((7, H), dtype=torch.bool)
    same[3, 1] = same[5, 0] = same[6, 0] = False       # these see one
    assert torch.equal(dirty[same], clean[same])
    assert not bool(dirty[~same].isfinite().all())


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_seen_is_not_used_by_many_rows(kvm_state, cache, what):
    """The same where a window has hundreds of rows, of which some see the cell: theirs hold it,
    the others' are as if it held zeros."""
    st, H, G, D = kvm_state, 2, 7, 128
    counts, fills = [30, 21], [100, 64]
    qp = np.concatenate([256 + f - c + np.arange(c) for f, c in zip(fills, counts)])
    rng = np.random.default_rng(17)
    clean, prefix, owns, q, qpos = run(st, rng, H, G, D, cache, 320, cells(320, 256, 0), [(128, cells(128, f, 256)) for f in fills],
                                       counts, torch.float32, torch.float32, q_pos=qp)
    _poison(prefix[0], cache, 300, 0, what)             # empty
    _poison(owns[0][0], cache, 120, 1, what)
    for c in (80, 99):
        _poison(owns[0][0], cache, c, 1, what)          # lane 0's token 10 sees the first, its last token both
    _poison(owns[1][0], cache, 63, 0, what)             # lane 1's last token
    got = api.fa_decode_shared(st, prefix[0], [x[0] for x in owns], counts, q, qpos, H * G, D ** -0.5)
    same = torch.ones((51, H), dtype=torch.bool)
    same[10:30, 1] = same[50, 0] = False
    clean, dirty = (x.view(51, H, G, D) for x in (clean, got))
    assert torch.equal(dirty[same], clean[same])
    assert not bool(dirty[~same].isfinite().flatten(1).all(1).any())


def _poison(w, cache, c, h, what):
    """What is not finite into the values (and keys) of cell c, kv head h."""
    D, t, i = w.head_dim, c // 64, c % 64
    if cache == "f16":
        v = w.v.view(torch.float16).view(w.n_head_kv, -1, 64 * D)[h, t].view(D // 16, 4, 16, 2, 8)
        k = w.k.view(torch.float16).view(w.n_head_kv, -1, 64 * D)[h, t].view(4, D // 32, 4, 16, 8)
        v[:, (i & 31) >> 3, :, i >> 5, i & 7] = what
        if int(w.cell_pos[c]) < 0:
            k[i >> 4, :, :, i & 15] = what
    else:
        NB = D // 32
        vb = w.v.view(w.n_head_kv, -1, 32 * D + 128 * NB)[h, t][32 * D:].view(torch.float16).view(NB, 2, 4, 8)
        kb = w.k.view(w.n_head_kv, -1, 64 * D + 128 * NB)[h, t][64 * D:].view(torch.float16).view(4, NB, 16)
        vb[:, i >> 5, (i & 31) >> 3, i & 7] = what
        if int(w.cell_pos[c]) < 0:
            kb[i >> 4, :, i & 15] = what


def test_infinite_values_that_are_seen(kvm_state):
    """An infinite value at a cell that every row sees reaches every row, and only its dims."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(8), 1, 2, 128
    w, k, v, pos = window(st, rng, 128, H, D, "f16", cells(128, 128, 0))
    w.v.view(torch.float16).view(-1, 64 * D)[0].view(D // 16, 4, 16, 2, 8)[3, 0, 5, 0, 2] = float("inf")     # cell 2, dim 53
    q = torch.from_numpy(rng.standard_normal((2, G, D)).astype(np.float32)).cuda() * 0.1
    got = api.fa_decode_shared(st, w, [None], [2], q, torch.tensor([200, 200], dtype=torch.int32, device="cuda"), G, D ** -0.5)
    assert bool((got[..., 53] == float("inf")).all())
    got[..., 53] = 0
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_what_is_no_number_is_not_hidden(kvm_state, cache, tokens):
    """A query that holds a NaN gives NaN, in its own head and token alone; a key that does gives
    NaN to every row that sees it, also where it is all that the row sees."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(22), 2, 3, 128
    pre, own = window(st, rng, 256, H, D, cache, cells(256, 256, 10)), window(st, rng, 64, H, D, cache, cells(64, 50, 266))
    q = torch.from_numpy(rng.standard_normal((tokens + 2, H * G, D)).astype(np.float32)).cuda()
    qp = torch.full((tokens + 2,), 315, dtype=torch.int32, device="cuda")
    qp[-1] = 10                                         # one cell of the prefix
    args = (st, pre[0], [own[0], None], [tokens, 2], q, qp, H * G, D ** -0.5)
    clean = api.fa_decode_shared(*args)
    assert bool(clean.isfinite().all())
    q[0, 4, 77] = float("nan")
    got = api.fa_decode_shared(*args)
    assert bool(got[0, 4].isnan().all())
    got[0, 4] = clean[0, 4]
    assert torch.equal(got, clean)
    q[0, 4, 77] = 0.0
    k = pre[0].k.view(torch.float16).view(H, -1, 64 * D if cache == "f16" else (64 * D + 128 * (D // 32)) // 2)
    if cache == "f16":
        k[0, 0].view(4, D // 32, 4, 16, 8)[0, 1, 2, 0, 3] = float("nan")       # cell 0, kv head 0
    else:
        k[0, 0][32 * D:].view(4, D // 32, 16)[0, 1, 0] = float("nan")
    got = api.fa_decode_shared(*args).view(tokens + 2, H, G, D)
    assert bool(got[:, 0].isnan().all()) and bool(got[:, 1].isfinite().all())


def _held(st, w, pos):
    """(window, K, V, positions) in 64 bits from what the window's cells hold now."""
    rows = w.export_rows(0, w.n_cells)
    k, v = (api.dequantize_rows(st, t, r, w.n_head_kv * w.head_dim).double().view(w.n_cells, w.n_head_kv, w.head_dim)
            for t, r in zip((w.k_type, w.v_type), rows))
    return w, k, v, pos


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("counts", [[4, 3], [30, 21]])
@pytest.mark.parametrize("what", [8192.0, 20000.0, -65504.0])
def test_large_values_that_are_not_seen_are_not_used(kvm_state, cache, D, counts, what):
    """Scales that are finite but whose values are beyond f16, in empty cells and in cells that
    some rows of a unit see: the others' outputs are as if they were small, bit for bit, and
    those that see them have the finite result."""
    st, H, G = kvm_state, 2, 7
    fills, n = [100, 64], sum(counts)
    qp = np.concatenate([256 + f - c + np.arange(c) for f, c in zip(fills, counts)])
    clean, prefix, owns, q, qpos = run(st, np.random.default_rng(23), H, G, D, cache, 320, cells(320, 256, 0),
                                       [(128, cells(128, f, 256)) for f in fills], counts, torch.float32, torch.float32, q_pos=qp)
    _poison(prefix[0], cache, 300, 0, what)             # empty
    _poison(owns[0][0], cache, 120, 1, what)
    _poison(owns[0][0], cache, 99, 1, what)             # lane 0's last token
    for c in (62, 63):
        _poison(owns[1][0], cache, c, 0, what)          # lane 1's last two tokens see the first, its last both
    got = api.fa_decode_shared(st, prefix[0], [x[0] for x in owns], counts, q, qpos, H * G, D ** -0.5)
    same = torch.ones((n, H), dtype=torch.bool)
    same[counts[0] - 1, 1] = same[n - 2:, 0] = False
    assert torch.equal(got.view(n, H, G, D)[same], clean.view(n, H, G, D)[same])
    assert not bool((got == clean).view(n, H, G, D)[~same].flatten(1).all(1).any())
    check(got, *expected(q, qpos, counts, prefix, [_held(st, x[0], x[3]) for x in owns], H, D ** -0.5))


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("tokens,sharp", [(2, 1.0), (2, 5.0), (40, 1.0), (40, 5.0)])
def test_large_values_that_every_row_sees(kvm_state, cache, D, tokens, sharp):
    """The same in tiles whose every cell every row sees, also under probabilities too small for
    f16: finite values give finite outputs."""
    st, rng, H, G = kvm_state, np.random.default_rng(24), 2, 3
    w, k, v, pos = window(st, rng, 512, H, D, cache, cells(512, 512, 0))
    for c, h, what in ((77, 1, 20000.0), (200, 0, -9000.0), (450, 1, 65504.0), (451, 1, 8192.0)):
        _poison(w, cache, c, h, what)
    q = torch.from_numpy(rng.standard_normal((tokens, H * G, D)).astype(np.float32) * np.float32(sharp)).cuda()
    qp = torch.full((tokens,), 600, dtype=torch.int32, device="cuda")
    got = api.fa_decode_shared(st, w, [None], [tokens], q, qp, H * G, D ** -0.5)
    check(got, *expected(q, qp, [tokens], _held(st, w, pos), [None], H, D ** -0.5))


@pytest.mark.parametrize("cache,H,G,tokens", [("q8_0", 8, 1, 1), ("q4_0", 4, 8, 9)])
def test_large_values_in_long_pieces(kvm_state, cache, H, G, tokens):
    """The same where a piece has more tiles than are looked at at a time: in the first of them, the
    last and between, some seen by every row and some by few."""
    st, rng, D, n = kvm_state, np.random.default_rng(35), 128, 64 * 301
    p = np.arange(n)
    w, k, v, pos = window(st, rng, n, H, D, cache, p)
    for c in (3, 64 * 255 + 1, 64 * 256, 64 * 280 + 17, n - 900, n - 5):
        _poison(w, cache, c, int(rng.integers(0, H)), float(rng.choice([8192.0, -30000.0])))
    counts = [tokens] * 64
    q = torch.from_numpy(rng.standard_normal((64 * tokens, H * G, D)).astype(np.float32)).cuda()
    qp = torch.from_numpy(rng.integers(n - 1200, n, 64 * tokens).astype(np.int32)).cuda()
    got = api.fa_decode_shared(st, None, [w] * 64, counts, q, qp, H * G, D ** -0.5)
    check(got, *expected(q, qp, counts, None, [_held(st, w, pos)] * 64, H, D ** -0.5))


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("tokens", [1, 30])
def test_large_values_everywhere(kvm_state, cache, tokens):
    """Windows of nothing but values that f16 does not hold."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(36), 2, 5, 256
    w, k, v, pos = window(st, rng, 256, H, D, cache, cells(256, 250, 0))
    for c in range(256):
        for h in range(H):
            _poison(w, cache, c, h, 60000.0 * (1 if c % 3 else -1))
    q = torch.from_numpy(rng.standard_normal((tokens, H * G, D)).astype(np.float32)).cuda()
    qp = torch.from_numpy(rng.integers(100, 300, tokens).astype(np.int32)).cuda()
    got = api.fa_decode_shared(st, w, [None], [tokens], q, qp, H * G, D ** -0.5)
    check(got, *expected(q, qp, [tokens], _held(st, w, pos), [None], H, D ** -0.5))


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
@pytest.mark.parametrize("tokens", [2, 40])
def test_infinite_values_under_small_probabilities(kvm_state, cache, tokens):
    """An infinite value that every row sees is infinite in every row, however small its (positive)
    probability: some 28 nats below the row's largest here, and f16 ends at 17."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(25), 2, 3, 128
    w, k, v, pos = window(st, rng, 256, H, D, cache, cells(256, 256, 0))
    q = (-2.0 * k[100].float())[None, :, None].expand(tokens, H, G, D).reshape(tokens, H * G, D).contiguous()
    qp = torch.full((tokens,), 600, dtype=torch.int32, device="cuda")
    args = (st, w, [None], [tokens], q, qp, H * G, D ** -0.5)
    clean = api.fa_decode_shared(*args)
    _poison(w, cache, 100, 1, float("inf"))
    got = api.fa_decode_shared(*args).view(tokens, H, G, D)
    want = _held(st, w, pos)[2][100, 1].float()         # +-inf, NaN (0 times inf)
    assert torch.equal(got[:, 0], clean.view(tokens, H, G, D)[:, 0])
    assert not bool(want.isfinite().any()) and bool((want == float("inf")).any())
    assert torch.equal(got[:, 1].nan_to_num(7.0), want.nan_to_num(7.0).expand(tokens, G, D))


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_largest_window(kvm_state, cache, tokens):
    """Windows whose tiles' offsets pass 32 bits (of the most cells there can be where quantised), almost
    all of them empty: the few rows that they hold, at both ends and between."""
    st, rng, H, G, D, n = kvm_state, np.random.default_rng(32), 8, 2, 256, 70
    N = 64 * 65535 if cache == "q8_0" else 2 ** 20
    w = api.KVWindow(st, N, H, D, 64, *TYPES[cache])
    w.cell_pos.fill_(-1)
    held, at = [], (0, 64 * 12345 + 9, N - n)
    for i, c in enumerate(at):
        rows = [api.quantize_rows(st, t, torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32)).cuda()) for t in TYPES[cache]]
        p = torch.arange(1000 * i, 1000 * i + n, dtype=torch.int32).cuda()
        w.import_rows(c, *rows, p)
        held.append((*(api.dequantize_rows(st, t, r, H * D).double().view(n, H, D) for t, r in zip(TYPES[cache], rows)), p))
    part = (w, *(torch.cat([x[i] for x in held]) for i in range(3)))
    q = torch.from_numpy(rng.standard_normal((tokens, H * G, D)).astype(np.float32)).cuda()
    qp = torch.from_numpy(rng.integers(0, 3000, tokens).astype(np.int32)).cuda()
    got = api.fa_decode_shared(st, w, [None], [tokens], q, qp, H * G, D ** -0.5)
    check(got, *expected(q, qp, [tokens], part, [None], H, D ** -0.5))


def test_two_states_at_once():
    """Calls of two states on streams of their own, over the same prefix, side by side: each has its own
    pieces, and gives what it gives alone."""
    rng, H, G, D = np.random.default_rng(33), 4, 4, 128
    streams = [torch.cuda.Stream() for _ in range(2)]
    sts = [api.State(0, stream=s.cuda_stream) for s in streams]
    try:
        with torch.cuda.stream(streams[0]):
            pre = window(sts[0], rng, 8192, H, D, "q8_0", cells(8192, 8192, 0))[0]
            qs = [torch.from_numpy(rng.standard_normal((m, H * G, D)).astype(np.float32)).cuda() for m in (3, 40)]
            ps = [torch.full((x.shape[0],), 9000, dtype=torch.int32, device="cuda") for x in qs]
        torch.cuda.synchronize()
        calls = [api.prepare_fa_decode_shared(st, pre, [None], [q.shape[0]], q, p, H * G, D ** -0.5) for st, q, p in zip(sts, qs, ps)]
        want = []
        for c in calls:
            c()
            torch.cuda.synchronize()
            want.append(c.out.clone())
        torch.cuda.synchronize()
        for _ in range(20):
            for c in calls:
                c()
        torch.cuda.synchronize()
        assert all(torch.equal(c.out, x) for c, x in zip(calls, want))
    finally:
        torch.cuda.synchronize()
        for st in sts:
            st.close()


def test_two_graphs_of_one_state(kvm_state):
    """Graphs captured from one state, of many rows and of few, replayed in turn with eager calls
    between: they follow one another in its workspace."""
    rng, H, G, D = np.random.default_rng(34), 4, 6, 256
    s = torch.cuda.Stream()
    st = api.State(0, stream=s.cuda_stream)
    try:
        with torch.cuda.stream(s):
            pre, own = (window(st, rng, n, H, D, "q8_0", cells(n, n, p))[0] for n, p in ((2048, 0), (128, 2048)))
            calls = []
            for m in (40, 2, 7):
                q = torch.from_numpy(rng.standard_normal((m, H * G, D)).astype(np.float32)).cuda()
                qp = torch.full((m,), 2100, dtype=torch.int32, device="cuda")
                calls.append(api.prepare_fa_decode_shared(st, pre, [own], [m], q, qp, H * G, D ** -0.5))
            want = []
            for c in calls:
                c()
                torch.cuda.synchronize()
                want.append(c.out.clone())
        torch.cuda.synchronize()
        graphs = [st.capture(c) for c in calls[:2]]
        for _ in range(3):
            for c in calls:
                c.out.fill_(3.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                graphs[0].replay()
                calls[2]()
                graphs[1].replay()
                graphs[0].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(c.out, x) for c, x in zip(calls, want))
    finally:
        torch.cuda.synchronize()
        st.close()


def test_same_as_one_window(kvm_state):
    """A prefix and an own window give what one window with all the cells gives (kvm_fa_prefill),
    to the roundings of both."""
    st, rng, H, G, D = kvm_state, np.random.default_rng(9), 4, 6, 256
    P, n, T = 1024, 512, 6
    kv = [api.quantize_rows(st, t, torch.from_numpy(rng.standard_normal((P + n, H * D)).astype(np.float32)).cuda()) for t in TYPES["q8_0"]]
    pos = torch.arange(P + n, dtype=torch.int32).cuda()
    one, pre, own = api.KVWindow(st, P + n, H, D, 64), api.KVWindow(st, P, H, D, 64), api.KVWindow(st, n, H, D, 64)
    one.import_rows(0, *kv, pos)
    pre.import_rows(0, kv[0][:P], kv[1][:P], pos[:P])
    own.import_rows(0, kv[0][P:], kv[1][P:], pos[P:])
    q = torch.from_numpy(rng.standard_normal((T, H * G, D)).astype(np.float32)).cuda()
    qp = pos[-T:].contiguous()
    a = api.fa_prefill(st, one, q, qp, H * G, D ** -0.5)
    b = api.fa_decode_shared(st, pre, [own], [T], q, qp, H * G, D ** -0.5)
    rel = float((a - b).norm() / a.norm())
    assert rel <= 1e-3, rel                             # (two forms of 3e-4 each)


def test_order_of_lanes_and_repeats(kvm_state):
    """The same call twice gives the same bits; a lane's output does not depend on what the
    other lanes' windows hold."""
    st, H, G, D = kvm_state, 2, 4, 128
    args = dict(H=H, G=G, D=D, cache="q8_0", prefix_cells=512, prefix_pos=cells(512, 512, 0),
                lanes=[(64, cells(64, 20, 512)), (128, cells(128, 99, 512))], counts=[2, 1], q_dtype=torch.bfloat16,
                out_dtype=torch.float32, q_pos=[530, 531, 610])
    got, prefix, owns, q, qp = run(st, np.random.default_rng(10), **args)
    again = api.fa_decode_shared(st, prefix[0], [x[0] for x in owns], [2, 1], q, qp, H * G, D ** -0.5)
    assert torch.equal(got, again)
    other = window(st, np.random.default_rng(11), 64, H, D, "q8_0", cells(64, 64, 512))
    mixed = api.fa_decode_shared(st, prefix[0], [other[0], owns[1][0]], [2, 1], q, qp, H * G, D ** -0.5)
    assert torch.equal(mixed[2], got[2]) and not torch.equal(mixed[:2], got[:2])


def test_step_append_then_attend(kvm_state):
    """A layer's step of a batch: new keys, values and queries of each conversation into its window
    (norms and rotation on the way), then the shared attention, against the same from the
    cells' values; on a stream of its own, and captured and replayed with other inputs."""
    rng, H, G, D, P = np.random.default_rng(12), 2, 4, 128, 512
    s = torch.cuda.Stream()
    st = api.State(0, stream=s.cuda_stream)
    try:
        with torch.cuda.stream(s):
            prefix = window(st, rng, P, H, D, "q8_0", cells(P, P, 0))
            counts, fill = [3, 1, 2], [10, 63, 100]
            owns = [window(st, rng, 128, H, D, "q8_0", cells(128, f, P)) for f in fill]
            n = sum(counts)
            q, k, v = (torch.from_numpy(rng.standard_normal((n, h, D)).astype(np.float32)).bfloat16().cuda() for h in (H * G, H, H))
            qw, kw = torch.ones(D, device="cuda"), torch.ones(D, device="cuda") * 0.9
            pos = torch.from_numpy(np.concatenate([P + f + np.arange(m) for f, m in zip(fill, counts)]).astype(np.int32)).cuda()
            app = api.prepare_window_append(st, [x[0] for x in owns], fill, counts, k, v, pos, 64, 1e6, k_weight=kw, eps=1e-6, q=q,
                                            q_weight=qw, q_out_dtype=torch.float32)
            att = api.prepare_fa_decode_shared(st, prefix[0], [x[0] for x in owns], counts, app.q_out, pos, H * G, D ** -0.5)

            def want():
                held = []
                for w, *_ in owns:
                    kr, vr = w.export_rows(0, 128)
                    held.append((w, *(api.dequantize_rows(st, t, r, H * D).double().view(128, H, D) for t, r in
                                      ((w.k_type, kr), (w.v_type, vr))), w.cell_pos))
                return expected(app.q_out, pos, counts, prefix, held, H, D ** -0.5)

            app()
            att()
            torch.cuda.synchronize()
            check(att.out, *want())
        g = st.capture(lambda: (app(), att()))
        for i in range(3):
            with torch.cuda.stream(s):
                for x in (q, k, v):
                    x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
                torch.cuda.synchronize()
                att.out.fill_(-7.0)
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                got = att.out.clone()
                check(got, *want())
                app()
                att()
                torch.cuda.synchronize()
                assert torch.equal(att.out, got)
    finally:
        torch.cuda.synchronize()
        st.close()


def test_refusals(kvm_state):
    st, rng, H, D = kvm_state, np.random.default_rng(13), 2, 128
    w = window(st, rng, 64, H, D, "q8_0", cells(64, 64, 0))[0]
    q, pos = torch.zeros((2, 8, D), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")

    def refused(code, *a, **kw):
        with pytest.raises(L.KvmError) as e:
            api.fa_decode_shared(st, *a, **kw)
        assert e.value.code == code, e.value

    refused(L.KVM_EUNSUPPORTED, w, [api.KVWindow(st, 64, H, D, 64, *TYPES["f16"])], [2], q, pos, 8, 1.0)
    refused(L.KVM_EUNSUPPORTED, w, [api.KVWindow(st, 64, 4, D, 64)], [2], q, pos, 8, 1.0)
    refused(L.KVM_ERANGE, w, [None] * 65, [1, 1] + [0] * 63, q, pos, 8, 1.0)
    refused(L.KVM_EINVAL, None, [None], [2], q, pos, 8, 1.0)
    refused(L.KVM_EINVAL, w, [None], [3], q, pos, 8, 1.0)
    refused(L.KVM_EINVAL, w, [None, None], [2], q, pos, 8, 1.0)
    refused(L.KVM_EINVAL, w, [None], [2], q[:, :7].contiguous(), pos, 7, 1.0)
    refused(L.KVM_EINVAL, w, [None], [2], q.half(), pos, 8, 1.0)
    refused(L.KVM_EINVAL, w, [None], [2], q.cpu(), pos, 8, 1.0)
    refused(L.KVM_EINVAL, w, [None], [2], q, pos.long(), 8, 1.0)
    refused(L.KVM_EINVAL, w, [None], [2], q, pos, 8, float("nan"))
    refused(L.KVM_EINVAL, w, [None], [2], q, pos, 8, 1.0, out=torch.empty((2, 8, D), dtype=torch.float64, device="cuda"))

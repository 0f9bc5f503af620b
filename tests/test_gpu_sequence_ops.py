"""The voxel-sequence operators against their definitions in 64 bits (tests/_sequence.py says where the bounds come from)."""
import numpy as np
import pytest
import torch

from tests import _sequence as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-5


def normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def features(seed, rows, channels, dtype, layout="dense"):
    """Rows of different scale.  layout: "columns" of a wider tensor with 16-byte rows, "odd": rows two elements apart from them."""
    x = (normal(seed, rows, channels) * torch.exp(normal(seed + 1, rows, 1))).to(dtype)
    if layout == "dense":
        return x
    wide = torch.full((rows, channels + (16 if layout == "columns" else 3)), float("nan"), device=DEV, dtype=dtype)
    at = 8 if layout == "columns" else 1
    wide[:, at:at + channels] = x
    return wide[:, at:at + channels]


def live(n):
    return torch.tensor([n], dtype=torch.int32, device=DEV)


# ---- layer norm -----------------------------------------------------------------------------------------------------
def check_norm(x, weight, bias, y, mean=None, rstd=None):
    w = ref.as64(weight) if weight is not None else np.ones(x.shape[1])
    b = ref.as64(bias) if bias is not None else np.zeros(x.shape[1])
    want, limit, m, r, _ = ref.norm(ref.as64(x), w, b, EPS)
    ref.assert_within(y, want, limit + ref.half_step(y.dtype) * (np.abs(want) + limit) + ref.smallest(y.dtype), "norm")
    if mean is not None:
        ref.assert_within(mean, m, ref.U32 * ref.DEPTH * np.abs(ref.as64(x)).mean(1), "mean")
        ref.assert_within(rstd, r, ref.U32 * ref.DEPTH * r * (1 + (np.abs(ref.as64(x)).mean(1) * r) ** 2), "rstd")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(0, 16), (1, 1), (1, 16), (257, 3), (300, 24), (1000, 64), (77, 96), (513, 131),
                                           (33, 256), (65, 520), (9, 1000), (5, 1025), (6, 4096), (3, 8191), (2, 8192)])
def test_norm_and_backward(d3d, dtype, rows, channels):
    x, grad = features(1, rows, channels, dtype), normal(3, rows, channels).to(dtype)
    weight, bias = 1 + 0.2 * normal(4, channels), 0.1 * normal(5, channels)
    y, mean, rstd = d3d.layer_norm(x, weight, bias, EPS, with_stats=True)
    dx, dw, db = d3d.layer_norm_backward(grad, x, weight, mean, rstd)
    if rows == 0:
        assert y.shape == x.shape and (dw == 0).all() and (db == 0).all()
        return
    check_norm(x, weight, bias, y, mean, rstd)
    want = ref.norm_backward(ref.as64(grad), ref.as64(x), ref.as64(weight), ref.as64(mean), ref.as64(rstd))
    for got, (w, limit), what in zip((dx, dw, db), want, ("dx", "dweight", "dbias")):
        ref.assert_within(got, w, limit + ref.half_step(got.dtype) * (np.abs(w) + limit) + ref.smallest(got.dtype), what)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["dense", "columns", "odd"])
@pytest.mark.parametrize("channels", [16, 40, 200])
def test_norm_of_a_sum(d3d, dtype, layout, channels):
    rows, n = 211, 150
    x, r = features(1, rows, channels, dtype, layout), features(7, rows, channels, dtype, layout)
    grad, more = normal(3, rows, channels).to(dtype), normal(9, rows, channels).to(dtype)
    out = torch.full((rows, channels), 3.0, device=DEV, dtype=dtype)
    y, total, mean, rstd = d3d.layer_norm(x, None, None, EPS, residual=r, num_rows=live(n), with_stats=True, out=out)
    assert y is out and (out[n:] == 3).all()
    assert torch.equal(total[:n], (x.float() + r.float()).to(dtype)[:n])
    check_norm(total[:n], None, None, y[:n], mean[:n], rstd[:n])
    dx, dw, db = d3d.layer_norm_backward(grad, total, None, mean, rstd, num_rows=live(n), grad_total=more)
    g, t, m, v = (ref.as64(a[:n]) for a in (grad, total, mean, rstd))
    (wx, lx), (ww, lw), (wb, lb) = ref.norm_backward(g, t, np.ones(channels), m, v)
    wx, lx = wx + ref.as64(more[:n]), lx + ref.U32 * 2 * (np.abs(wx) + np.abs(ref.as64(more[:n])))
    ref.assert_within(dx[:n], wx, lx + ref.half_step(dtype) * (np.abs(wx) + lx) + ref.smallest(dtype), "dx")
    ref.assert_within(dw, ww, lw, "dweight")
    ref.assert_within(db, wb, lb, "dbias")


@pytest.mark.parametrize("count", [-5, 0, 1, 64, 1000])
def test_norm_counts(d3d, count):
    rows = 64
    x, w = features(1, rows, 32, torch.float16), normal(2, 32)
    out = torch.full((rows, 32), 7.0, device=DEV, dtype=torch.float16)
    d3d.layer_norm(x, w, None, EPS, num_rows=live(count), out=out)
    n = max(0, min(rows, count))
    assert (out[n:] == 7).all()
    if n:
        check_norm(x[:n], w, None, out[:n])
    _, mean, rstd = d3d.layer_norm(x, w, None, EPS, with_stats=True)
    _, dw, db = d3d.layer_norm_backward(x, x, w, mean, rstd, num_rows=live(count))
    assert torch.equal(db == 0, torch.full((32,), n == 0, device=DEV)) and (n > 0 or (dw == 0).all())


@pytest.mark.parametrize("rows,channels", [(1, 16), (7, 16), (3, 600), (1, 8192)])
@pytest.mark.parametrize("count", [0, 1, 2, 7])
def test_norm_backward_of_few_live_rows(d3d, rows, channels, count):
    """One CTA, whose sums are the parameters' gradients: those of the live rows, to the last bit."""
    n = min(rows, count)
    x, dy, w = features(1, rows, channels, torch.float32), normal(2, rows, channels), normal(3, channels)
    _, mean, rstd = d3d.layer_norm(x, w, None, EPS, with_stats=True)
    dx, dw, db = d3d.layer_norm_backward(dy, x, w, mean, rstd, num_rows=live(count))
    assert (n > 0 or not dw.any()) and (n > 0 or not db.any())
    if n:
        again = d3d.layer_norm_backward(dy[:n].clone(), x[:n].clone(), w, mean[:n].clone(), rstd[:n].clone())
        assert torch.equal(dx[:n], again[0]) and torch.equal(dw, again[1]) and torch.equal(db, again[2])
        ref.assert_within(db, ref.as64(dy[:n]).sum(0), n * ref.U32 * np.abs(ref.as64(dy[:n])).sum(0), "db")


def test_norm_rows_keep_to_themselves(d3d):
    """A row that is not finite, beside rows that share its warp; a constant row."""
    for dtype in TYPES:
        for channels in (8, 24, 64, 5, 1000):
            x = features(1, 67, channels, dtype)
            want = d3d.layer_norm(x, None, None, EPS)
            x[5, 1], x[40, channels - 1], x[66] = float("nan"), float("inf"), 2.5
            got = d3d.layer_norm(x, None, None, EPS)
            fine = torch.ones(67, dtype=torch.bool, device=DEV)
            fine[[5, 40, 66]] = False
            assert torch.equal(got[fine], want[fine])
            assert got[5].isnan().all() and got[40].isnan().all() and (got[66] == 0).all()


@pytest.mark.parametrize("dtype,mean,rows,channels", [
    (torch.float32, 1e4, 300, 64), (torch.float32, -3e4, 65, 1001), (torch.float32, 1e4, 9, 4096), (torch.float16, 200.0, 300, 64),
    (torch.float16, -200.0, 77, 131), (torch.bfloat16, 30.0, 513, 256), (torch.bfloat16, -30.0, 5, 8191)])
def test_norm_of_rows_far_from_zero(d3d, dtype, mean, rows, channels):
    """A mean far above the spread, of either sign: what a difference of two large sums, or of squares, would lose."""
    x, grad = (mean + normal(1, rows, channels)).to(dtype), normal(3, rows, channels).to(dtype)
    weight, bias = 1 + 0.2 * normal(4, channels), 0.1 * normal(5, channels)
    y, m, r = d3d.layer_norm(x, weight, bias, EPS, with_stats=True)
    check_norm(x, weight, bias, y, m, r)
    got = d3d.layer_norm_backward(grad, x, weight, m, r)
    want = ref.norm_backward(ref.as64(grad), ref.as64(x), ref.as64(weight), ref.as64(m), ref.as64(r))
    for g, (w, limit), what in zip(got, want, ("dx", "dweight", "dbias")):
        ref.assert_within(g, w, limit + ref.half_step(g.dtype) * (np.abs(w) + limit) + ref.smallest(g.dtype), what)


def test_norm_backward_is_the_same_every_time(d3d):
    x, g = features(1, 20011, 64, torch.bfloat16), features(2, 20011, 64, torch.bfloat16)
    w = normal(4, 64)
    _, mean, rstd = d3d.layer_norm(x, w, None, EPS, with_stats=True)
    first = d3d.layer_norm_backward(g, x, w, mean, rstd)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, d3d.layer_norm_backward(g, x, w, mean, rstd)))


# ---- rows in 8-bit integers -----------------------------------------------------------------------------------------
def check_quantized(x32, q, scale):
    want, s = ref.quantize(x32.cpu().numpy())
    assert np.array_equal(scale.cpu().numpy(), s, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["dense", "columns", "odd"])
@pytest.mark.parametrize("rows,channels", [(0, 16), (1, 1), (300, 24), (1000, 64), (513, 131), (6, 4096), (3, 8191)])
def test_quantize_rows(d3d, dtype, layout, rows, channels):
    x = features(1, rows, channels, dtype, layout)
    q, scale = d3d.quantize_rows(x)
    assert q.shape == x.shape and (rows <= 1 or q.stride(0) % 16 == 0)
    if rows:
        check_quantized(x.float(), q, scale)


def test_quantize_borders(d3d):
    """Values half-way between two steps, of rows whose scale is and is not a power of two, as exact fp32 numbers; rows of
    zeros, of the smallest numbers, of what is not finite."""
    halves = torch.arange(-126.5, 127.0, 0.5, device=DEV)
    rows = [halves * s for s in (1.0, 2.0 ** -20, 3.0, 0.7, 1e30, 1e-30)]
    x = torch.stack([torch.cat([r, r.abs().max()[None] * 127 / 126.5]) for r in rows])
    neighbours = torch.cat([x, torch.nextafter(x, x + x.abs()), torch.nextafter(x, x - x.abs())])
    neighbours[:, -1] = x[:, -1].repeat(3)
    special = torch.zeros((5, x.shape[1]), device=DEV)
    special[1, 3], special[2, 3], special[3, 3], special[4, 3] = 1e-42, 1.4e-36, float("inf"), float("nan")
    x = torch.cat([neighbours, special])
    q, scale = d3d.quantize_rows(x)
    check_quantized(x, q, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [24, 131, 256])
def test_norm_int8(d3d, dtype, channels):
    """The integers are those of the normed rows, give or take one where a value lies within the norm's bound of a border."""
    rows, n = 301, 290
    x, r = features(1, rows, channels, dtype), features(7, rows, channels, dtype)
    w, b = 1 + 0.2 * normal(4, channels), 0.1 * normal(5, channels)
    q, scale, total = d3d.layer_norm_int8(x, w, b, EPS, residual=r, num_rows=live(n))
    q, scale, total = q[:n], scale[:n], total[:n]
    y, limit, _, _, _ = ref.norm(ref.as64(total), ref.as64(w), ref.as64(b), EPS)
    amax = np.abs(y).max(1)
    ref.assert_within(scale, amax / 127, limit.max(1) / 127 + 2 * ref.U32 * amax / 127, "scale")
    assert (q.abs().max(1).values == 127).all()
    s = ref.as64(scale)[:, None]
    assert (np.abs(ref.as64(q) * s - y) <= s / 2 + limit + ref.U32 * 127 * s).all()
    plain, s2 = d3d.layer_norm_int8(total, w, b, EPS)  # the sum as an input gives the same
    assert torch.equal(plain, q) and torch.equal(s2, scale)


# ---- gated recurrence -----------------------------------------------------------------------------------------------
def offsets_of(kind, rows):
    r = np.random.Generator(np.random.PCG64(rows + len(kind)))
    if kind == "one":
        return [0, rows]
    if kind == "singles":
        return list(range(rows + 1))
    if kind == "few":
        return sorted([0, rows] + list(r.integers(0, rows + 1, 3)))
    if kind == "many":  # short ones, some without rows, single rows at a tile's edges
        cuts = list(r.integers(0, rows + 1, rows // 9)) + [c for c in (127, 128, 128, 129, 255, 256) if c <= rows]
        return sorted([0, rows] + cuts)
    low, high = rows // 5, rows - rows // 7  # "inside": rows in front of the first sequence and behind the last
    return sorted([low, high] + list(r.integers(low, high + 1, 4)))


def gates_like(seed, rows, channels, dtype, layout="dense"):
    """Memories from one row to thousands."""
    g = (normal(seed, rows, channels) + torch.linspace(-2, 8, channels, device=DEV)).to(dtype)
    if layout == "dense":
        return g
    wide = features(seed, rows, channels, dtype, layout)
    wide.copy_(g)
    return wide


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("kind", ["one", "few", "many", "inside", "singles"])
@pytest.mark.parametrize("rows,channels", [(1, 1), (5, 16), (128, 8), (129, 40), (300, 3), (700, 72), (1030, 24), (2500, 64)])
def test_recurrence(d3d, dtype, reverse, kind, rows, channels):
    layout = ("dense", "columns", "odd")[(rows + channels) % 3]
    x, g = features(1, rows, channels, dtype, layout), gates_like(3, rows, channels, dtype, layout)
    offs = offsets_of(kind, rows)
    seqs = len(offs) - 1
    offsets = torch.tensor(offs, dtype=torch.int32, device=DEV)
    initial = normal(5, seqs, channels) if kind != "few" else None
    grad, grad_final = normal(7, rows, channels).to(dtype), normal(8, seqs, channels) if kind != "inside" else None
    out = torch.full((rows, channels), 9.0, device=DEV, dtype=dtype)
    h, final, states = d3d.gated_recurrence(x, g, offsets, initial, reverse=reverse, with_states=True, out=out)
    assert h is out
    x64, g64 = ref.as64(x), ref.as64(g)
    i64 = ref.as64(initial) if initial is not None else None
    want, off, wfinal, foff, _, _ = ref.recurrence(x64, g64, offs, i64, reverse, dtype)
    inside = ~np.isnan(want[:, 0])
    assert (ref.as64(out)[~inside] == 9).all()
    lim = off + ref.half_step(dtype) * (np.abs(want) + off) + ref.smallest(dtype)
    ref.assert_within(ref.as64(h)[inside], want[inside], lim[inside], "h")
    ref.assert_within(final, wfinal, foff + ref.U32 * np.abs(wfinal), "final")
    plain = d3d.gated_recurrence(x, g, offsets, initial, reverse=reverse)
    assert torch.equal(plain[0][torch.from_numpy(inside).to(DEV)], h[torch.from_numpy(inside).to(DEV)])
    assert torch.equal(plain[1], final)
    got = d3d.gated_recurrence_backward(grad, x, g, offsets, states, initial, grad_final, reverse=reverse)
    back = ref.recurrence_backward(ref.as64(grad), x64, g64, offs, i64,
                                   ref.as64(grad_final) if grad_final is not None else None, reverse, dtype)
    for t, (w, o), what in zip(got, back, ("dx", "dgates", "dinitial")):
        t = ref.as64(t)
        rnd = torch.float32 if what == "dinitial" else dtype
        lim = o + ref.half_step(rnd) * (np.abs(w) + o) + ref.smallest(rnd)
        keep = inside if what != "dinitial" else slice(None)
        ref.assert_within(t[keep], w[keep], lim[keep], what)


def test_recurrence_without_rows_or_sequences(d3d):
    for dtype in TYPES:
        x = torch.empty((0, 24), dtype=dtype, device=DEV)
        zero = torch.zeros(4, dtype=torch.int32, device=DEV)
        initial = normal(1, 3, 24)
        out, final, states = d3d.gated_recurrence(x, x, zero, initial, with_states=True)
        assert out.shape == (0, 24) and torch.equal(final, initial)
        assert (d3d.gated_recurrence(x, x, zero)[1] == 0).all()
        _, _, di = d3d.gated_recurrence_backward(x, x, x, zero, states, initial, 2 * initial)
        assert torch.equal(di, 2 * initial)
        x = features(2, 9, 24, dtype)
        out = torch.full_like(x, 4.0)
        _, final = d3d.gated_recurrence(x, x, zero[:1], out=out)
        assert final.shape == (0, 24) and (out == 4).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [16, 64, 5])
def test_sequences_do_not_touch_each_other(d3d, dtype, channels):
    """Sequences that hold NaN, infinities and gates at the type's ends, beside ones that do not: the same bytes."""
    rows, offs = 900, [0, 130, 256, 256, 300, 700, 900]
    offsets = torch.tensor(offs, dtype=torch.int32, device=DEV)
    x, g = features(1, rows, channels, dtype), gates_like(2, rows, channels, dtype)
    initial, grad, gf = normal(3, 6, channels), normal(4, rows, channels).to(dtype), normal(5, 6, channels)

    def run(reverse):
        out, final, states = d3d.gated_recurrence(x, g, offsets, initial, reverse=reverse, with_states=True)
        return (out, final) + d3d.gated_recurrence_backward(grad, x, g, offsets, states, initial, gf, reverse=reverse)
    want = [[t.clone() for t in run(r)] for r in (False, True)]
    x[131], g[200], x[310], g[500] = float("nan"), float("nan"), float("inf"), torch.finfo(dtype).min
    g[600, 0], initial[4, 0], grad[299], gf[1] = torch.finfo(dtype).max, float("-inf"), float("inf"), float("nan")
    rows_ok = torch.zeros(rows, dtype=torch.bool, device=DEV)
    rows_ok[:130] = rows_ok[700:] = True
    seqs_ok = [0, 2, 5]
    for r in (False, True):
        for a, b in zip(run(r), want[r]):
            assert torch.equal(a[rows_ok], b[rows_ok]) if len(a) == rows else torch.equal(a[seqs_ok], b[seqs_ok])


def check_not_finite(got, want, limit, dtype, what):
    """Infinities and NaN where the definition, walked row by row, has them; the others within their bound."""
    got, fine = ref.as64(got), np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), what
    ref.assert_within(got[fine], want[fine], (limit + ref.half_step(dtype) * (np.abs(want) + limit) + ref.smallest(dtype))[fine], what)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("rows,channels", [(90, 8), (700, 5), (1500, 24), (1500, 72)])
def test_states_that_are_not_finite(d3d, dtype, reverse, rows, channels):
    """An infinite state stays one whatever tiles lie behind it, although the product of their gates, 0.27 and less each, is no number
    any more; opposite ones make NaN.  The same for gradients, walked the other way."""
    x, g = features(1, rows, channels, dtype), (-1 - normal(2, rows, channels).abs()).to(dtype)
    grad, offs = normal(3, rows, channels).to(dtype), [0, rows // 9, rows - rows // 9, rows]
    initial, gf = normal(4, 3, channels), normal(5, 3, channels)
    inf, a, b = float("inf"), rows // 4, rows - rows // 5
    x[a, 0], x[a, 1], x[b, 1], initial[1, 2], x[a, 3] = inf, inf, -inf, -inf, float("nan")
    grad[a, 0], grad[b, 1], grad[a, 2], gf[1, 4] = inf, -inf, inf, inf
    offsets = torch.tensor(offs, dtype=torch.int32, device=DEV)
    h, final, states = d3d.gated_recurrence(x, g, offsets, initial, reverse=reverse, with_states=True)
    got = d3d.gated_recurrence_backward(grad, x, g, offsets, states, initial, gf, reverse=reverse)
    x64, g64, i64 = ref.as64(x), ref.as64(g), ref.as64(initial)
    with np.errstate(invalid="ignore"):
        want, off, wfinal, foff, _, _ = ref.recurrence(x64, g64, offs, i64, reverse, dtype)
        back = ref.recurrence_backward(ref.as64(grad), x64, g64, offs, i64, ref.as64(gf), reverse, dtype)
        assert np.isinf(want).sum() > rows / 2 and np.isnan(want).any() and np.isinf(back[0][0]).any()
        check_not_finite(h, want, off, dtype, "h")
        check_not_finite(final, wfinal, foff, torch.float32, "final")
        for t, (w, o), what in zip(got, back, ("dx", "dgates", "dinitial")):
            check_not_finite(t, w, o, torch.float32 if what == "dinitial" else dtype, what)


def test_recurrence_gates_at_their_ends(d3d):
    """Gates so large that nothing is added or kept, also in 32 bits: the state passes unchanged or is the row."""
    x = features(1, 300, 16, torch.float32)
    offsets = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    initial = normal(2, 1, 16)
    big = torch.full_like(x, 200.0)
    out, final = d3d.gated_recurrence(x, big, offsets, initial)
    assert torch.equal(out, initial.expand(300, 16)) and torch.equal(final, initial)
    out, final = d3d.gated_recurrence(x, -big, offsets, initial)
    assert torch.equal(out, x) and torch.equal(final, x[-1:])
    inf = torch.full_like(x, float("inf"))
    assert torch.equal(d3d.gated_recurrence(x, -inf, offsets, initial)[0], x)
    assert torch.equal(d3d.gated_recurrence(x, inf, offsets, initial)[0], initial.expand(300, 16))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_recurrence_gates_at_their_ends_in_16_bits(d3d, dtype):
    """The same, for states as large as 32 bits hold; gates between have their part of such a state."""
    lowest = torch.finfo(dtype).min
    x = features(1, 300, 16, dtype)
    offsets = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    for size in (1.0, 3e38):
        initial = size * normal(2, 1, 16).sign()
        for gate in (-200.0, lowest, float("-inf")):
            g = torch.full_like(x, gate)
            out, final = d3d.gated_recurrence(x, g, offsets, initial)
            assert torch.equal(out, x) and torch.equal(final, x[-1:].float())
            one = d3d.gated_recurrence_step(x[:1], g[:1], initial)
            assert torch.equal(one[0], x[:1]) and torch.equal(one[1], x[:1].float())
            assert torch.equal(d3d.gated_recurrence(x, -g, offsets, initial)[1], initial)
            _, _, states = d3d.gated_recurrence(x, g, offsets, initial, with_states=True)
            dx, dg, di = d3d.gated_recurrence_backward(x, x, g, offsets, states, initial)
            assert torch.equal(dx, x) and not dg.any() and not di.any()
    g = (-60 - 26 * torch.rand((300, 16), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)).to(dtype)
    state, zero = 1e38 * normal(4, 300, 16), torch.zeros_like(x)
    singles = list(range(301))
    want, off, wfinal, foff, _, _ = ref.recurrence(ref.as64(zero), ref.as64(g), singles, ref.as64(state), False, dtype)
    for got in (d3d.gated_recurrence(zero, g, torch.tensor(singles, dtype=torch.int32, device=DEV), state),
                d3d.gated_recurrence_step(zero, g, state)):
        ref.assert_within(got[1], wfinal, foff + ref.U32 * np.abs(wfinal), "state")


@pytest.mark.parametrize("offs", [[5, 3], [-4, 50], [0, 500], [20, 10, 60, 0, 99], [-9, -3], [400, 600]])
def test_offsets_out_of_order_stay_inside_the_tensors(d3d, offs):
    """Nothing is said about the results; rows behind the tensors' own are not touched."""
    rows = 100
    buf = torch.full((rows + 64, 16), 5.0, device=DEV)
    x = features(1, rows, 16, torch.float32)
    offsets = torch.tensor(offs, dtype=torch.int32, device=DEV)
    for reverse in (False, True):
        out, final, states = d3d.gated_recurrence(x, x, offsets, out=buf[32:32 + rows], reverse=reverse, with_states=True)
        d3d.gated_recurrence_backward(x, x, x, offsets, states, reverse=reverse)
        torch.cuda.synchronize()
        assert (buf[:32] == 5).all() and (buf[32 + rows:] == 5).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["dense", "columns", "odd"])
@pytest.mark.parametrize("rows,channels", [(0, 8), (1, 1), (77, 24), (512, 131)])
def test_step_is_the_recurrence_of_one_row(d3d, dtype, layout, rows, channels):
    x, g = features(1, rows, channels, dtype, layout), gates_like(2, rows, channels, dtype, layout)
    state = normal(3, rows, channels)
    out, new = d3d.gated_recurrence_step(x, g, state)
    offsets = torch.arange(rows + 1, dtype=torch.int32, device=DEV)
    want, final = d3d.gated_recurrence(x, g, offsets, state)
    assert torch.equal(out, want) and torch.equal(new, final)
    again, same = d3d.gated_recurrence_step(x, g, state, state_out=state)
    assert same is state and torch.equal(state, new) and torch.equal(again, out)


@pytest.mark.parametrize("channels", [6, 14, 30, 64])
@pytest.mark.parametrize("reverse", [False, True])
def test_states_serve_inputs_of_another_alignment(d3d, channels, reverse):
    """The forward pass over columns of an odd-pitched tensor, the backward pass over dense copies: the same gradients as from
    the dense forward pass, whose tiles have another shape."""
    rows = 777
    x, g = features(1, rows, channels, torch.float16, "odd"), gates_like(2, rows, channels, torch.float16, "odd")
    xd, gd, grad = x.contiguous(), g.contiguous(), normal(3, rows, channels).half()
    offsets = torch.tensor([0, 300, 777], dtype=torch.int32, device=DEV)
    for args in ((x, g), (xd, gd)):
        _, _, states = d3d.gated_recurrence(*args, offsets, reverse=reverse, with_states=True)
        got = d3d.gated_recurrence_backward(grad, xd, gd, offsets, states, reverse=reverse)
        back = ref.recurrence_backward(ref.as64(grad), ref.as64(x), ref.as64(g), offsets.tolist(), None, None, reverse, torch.float16)
        for t, (w, o), what in zip(got, back, ("dx", "dgates", "dinitial")):
            rnd = torch.float32 if what == "dinitial" else torch.float16
            ref.assert_within(t, w, o + ref.half_step(rnd) * (np.abs(w) + o) + ref.smallest(rnd), what)


def test_gradients_against_differences(d3d):
    """fp32, along a random direction: (L(p + e d) - L(p - e d)) / 2 e for L = <out, c> against the gradients.  The gates are
    smooth on a scale of one, so with e = 2^-6 the difference is off by at most e^2 of its terms' sizes, and rounding adds
    2^-24 / e of the outputs' sizes, summed at random."""
    rows, channels, e = 333, 16, 2.0 ** -6
    x, g = (normal(s, rows, channels) for s in (1, 2))
    offsets = torch.tensor([0, 100, 100, 333], dtype=torch.int32, device=DEV)
    h0, c, cf = normal(3, 3, channels), normal(4, rows, channels), normal(5, 3, channels)
    dirs = [normal(s, *t.shape) for s, t in ((6, x), (7, g), (8, h0))]

    def loss(e):
        out, final = d3d.gated_recurrence(x + e * dirs[0], g + e * dirs[1], offsets, h0 + e * dirs[2])
        return ((out.double() * c).sum() + (final.double() * cf).sum()).item()
    _, _, states = d3d.gated_recurrence(x, g, offsets, h0, with_states=True)
    grads = d3d.gated_recurrence_backward(c, x, g, offsets, states, h0, cf)
    along = sum((a.double() * b).sum().item() for a, b in zip(grads, dirs))
    size = sum((a.double() * b).abs().sum().item() for a, b in zip(grads, dirs))
    assert abs((loss(e) - loss(-e)) / (2 * e) - along) <= 4 * e * e * size

    w, b = 1 + 0.2 * normal(9, channels), normal(10, channels)
    dirs = [normal(11, rows, channels), normal(12, channels), normal(13, channels)]
    _, mean, rstd = d3d.layer_norm(x, w, b, EPS, with_stats=True)
    grads = d3d.layer_norm_backward(c, x, w, mean, rstd)
    along = sum((p.double() * q).sum().item() for p, q in zip(grads, dirs))
    size = sum((p.double() * q).abs().sum().item() for p, q in zip(grads, dirs))

    def loss(e):
        return (d3d.layer_norm(x + e * dirs[0], w + e * dirs[1], b + e * dirs[2], EPS).double() * c).sum().item()
    assert abs((loss(e) - loss(-e)) / (2 * e) - along) <= 4 * e * e * size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["one", "many", "inside", "singles"])
@pytest.mark.parametrize("rows", [15, 16, 17, 127, 128, 129, 255, 256, 257, 512, 513])
@pytest.mark.parametrize("channels", [8, 16, 17, 32, 34, 64, 130])
def test_recurrence_where_tiles_end(d3d, dtype, kind, rows, channels):
    """A tile has 128, 256 or 512 rows, by the channels and their type; one tile takes one kernel, two take three."""
    test_recurrence(d3d, dtype, (rows + channels) % 2 == 0, kind, rows, channels)


def test_offsets_out_of_order_over_several_tiles(d3d):
    rows = 900
    buf = torch.full((rows + 64, 40), 5.0, device=DEV)
    x = features(1, rows, 40, torch.float32)
    for offs in ([500, 3], [-4, 450], [0, 5000], [200, 100, 600, 0, 990], [899, 0, 899, 1, 898]):
        offsets = torch.tensor(offs, dtype=torch.int32, device=DEV)
        for reverse in (False, True):
            out, final, states = d3d.gated_recurrence(x, x, offsets, out=buf[32:32 + rows], reverse=reverse, with_states=True)
            d3d.gated_recurrence_backward(x, x, x, offsets, states, reverse=reverse)
            torch.cuda.synchronize()
            assert (buf[:32] == 5).all() and (buf[32 + rows:] == 5).all()


def walk64(a, b):
    """h[t] = a[t] h[t-1] + b[t] from h = 0, along the rows, in 64 bits on the GPU: blocks of rows side by side, then their ends one
    after the other, then what comes into each block."""
    rows, channels = a.shape
    block = int(rows ** 0.5)
    many = -(-rows // block)
    a, b = (torch.nn.functional.pad(t, (0, 0, 0, many * block - rows)).view(many, block, channels).clone() for t in (a, b))
    for t in range(1, block):
        b[:, t] += a[:, t] * b[:, t - 1]
        a[:, t] *= a[:, t - 1]
    into = torch.zeros((many, channels), dtype=a.dtype, device=a.device)
    for t in range(1, many):
        into[t] = a[t - 1, -1] * into[t - 1] + b[t - 1, -1]
    return (b + a * into[:, None]).view(-1, channels)[:rows]


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("rows", [600001, 4300007])
def test_recurrence_of_one_sequence_over_many_tiles(d3d, reverse, rows):
    """17 channels in 16 bits go by tiles of 128 rows.  4096 tiles are what the chain over them takes at a time, 32768 what a
    dimension of the grid does.  With gates around 8 a state lasts for thousands of rows, and with means of 1 it is of the size
    of the rows, so that what comes into a tile counts.  Definition and bounds are those of tests/_sequence.py, for all rows at once."""
    channels, dtype = 17, torch.float16
    x, g, grad = ((mean + normal(seed, rows, channels)).to(dtype) for seed, mean in ((1, 1.0), (3, 8.0), (4, 1.0)))
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    initial, gf = 100 * normal(5, 1, channels), 100 * normal(6, 1, channels)
    h, final, states = d3d.gated_recurrence(x, g, offsets, initial, reverse=reverse, with_states=True)
    dx, dg, di = d3d.gated_recurrence_backward(grad, x, g, offsets, states, initial, gf, reverse=reverse)
    turn = (lambda t: t.flip(0)) if reverse else (lambda t: t)
    x, gate, grad = (turn(t).double() for t in (x, g, grad))
    f, add, k = torch.sigmoid(gate), torch.sigmoid(-gate), ref.K + ref.PER_GATE * gate.abs()
    first, last = torch.zeros_like(f), torch.zeros_like(f)
    first[0], last[-1] = f[0], f[-1]
    del gate

    def check(got, want, off, what, rnd=dtype):
        off = off + ref.half_step(rnd) * (want.abs() + off) + ref.smallest(rnd)
        assert ((got.double() - want).abs() <= off).all(), what
    want = walk64(f, add * x + first * initial)
    size = walk64(f, add * x.abs() + first * initial.abs())
    off = walk64(f, ref.U32 * k * size)
    check(turn(h), want, off, "h")
    check(final, want[-1:], off[-1:], "final", torch.float32)
    before, before_off = torch.cat([initial.double(), want[:-1]]), torch.cat([0 * off[:1], off[:-1]])
    del want, size, off
    back = lambda a, b: walk64(a.flip(0), b.flip(0)).flip(0)
    into = lambda t, end: torch.cat([t[1:], end])  # of what leaves a row: what comes into the one in front of it
    q, size = back(f, f * grad + last * gf), back(f, f * grad.abs() + last * gf.abs())
    check(di, q[:1], (e := back(f, ref.U32 * (1 + k) * size))[:1], "dinitial", torch.float32)
    delta, dsize = grad + into(q, gf.double()), grad.abs() + into(size, gf.abs().double())
    doff = into(e, 0 * e[:1]) + ref.U32 * dsize
    check(turn(dx), delta * add, add * (doff + ref.U32 * k * dsize), "dx")
    check(turn(dg), delta * (before - x) * f * add, f * add * (doff * (before - x).abs() + dsize * before_off +
                                                               ref.U32 * k * dsize * (before.abs() + x.abs())), "dgates")


# ---- streams, graphs ------------------------------------------------------------------------------------------------
def test_on_another_stream_and_in_graphs(d3d):
    """Two graphs captured one after the other and replayed in turn on new inputs, and a call on a stream of its own."""
    def inputs(seed):
        return features(seed, 3000, 64, torch.bfloat16), gates_like(seed + 5, 3000, 64, torch.bfloat16)
    offsets = torch.tensor([0, 700, 700, 3000], dtype=torch.int32, device=DEV)
    w = normal(3, 64)

    def chain(x, g, reverse):
        y, mean, rstd = d3d.layer_norm(x, w, None, EPS, with_stats=True)
        h, final, states = d3d.gated_recurrence(y, g, offsets, reverse=reverse, with_states=True)
        dy, dg, _ = d3d.gated_recurrence_backward(x, y, g, offsets, states, reverse=reverse)
        return (h, final, dg) + d3d.layer_norm_backward(dy, x, w, mean, rstd)
    x, g = inputs(1)
    want = chain(x, g, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(x, g, False)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for reverse in (False, True):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = chain(x, g, reverse)
        graphs.append((graph, outs))
    for seed in (11, 12):
        a, b = inputs(seed)
        x.copy_(a), g.copy_(b)
        for (graph, _) in graphs * 2:
            graph.replay()
        torch.cuda.synchronize()
        for (_, outs), reverse in zip(graphs, (False, True)):
            assert all(torch.equal(p, q) for p, q in zip(outs, chain(a, b, reverse)))


def test_threads_on_streams_of_their_own(d3d):
    """Four threads at once, each on its stream, with sizes of several kinds of kernel: what one thread alone gets."""
    import threading

    def chain(seed):
        rows, channels = (90, 3000, 700, 20000)[seed], (64, 32, 130, 48)[seed]
        x, g = features(seed, rows, channels, torch.bfloat16), gates_like(seed + 5, rows, channels, torch.bfloat16)
        offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=DEV)
        w = int8(seed, 96, channels)
        results = []
        for _ in range(20):
            q, s = d3d.layer_norm_int8(x, None)
            y = d3d.int8_linear(q, s, w, torch.ones(96, device=DEV), dtype=torch.bfloat16)
            h, final, states = d3d.gated_recurrence(x, g, offsets, with_states=True)
            results.append((q, y, h, final) + d3d.gated_recurrence_backward(h, x, g, offsets, states))
        torch.cuda.current_stream().synchronize()
        return results
    want, got = [chain(i)[0] for i in range(4)], [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = chain(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for results, w in zip(got, want):
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


# ---- product of 8-bit rows ------------------------------------------------------------------------------------------
def int8(seed, rows, channels, layout="dense"):
    """Any bytes, -128 among them.  layout: "columns" 16 bytes into wider rows, "odd" one byte into them."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randint(-128, 128, (rows, channels), generator=gen, device=DEV, dtype=torch.int8)
    if layout == "dense":
        return x
    pitch, at = ((channels + 47) // 16 * 16, 16) if layout == "columns" else (channels + 3, 1)
    wide = torch.full((rows, pitch), 77, dtype=torch.int8, device=DEV)
    wide[:, at:at + channels] = x
    return wide[:, at:at + channels]


def check_linear(x, s, w, ws, b, y):
    """The sum is exact; then (float) sum, times the channel's scale, times the row's plus the bias in one rounding: three half
    units of 32 bits, and half a step of the type."""
    acc = (x.double() @ w.double().T).cpu().numpy()
    scaled = acc * ref.as64(ws) * ref.as64(s)[:, None]
    want = scaled + (ref.as64(b) if b is not None else 0.0)
    limit = 3 * ref.U32 * (np.abs(scaled) + np.abs(want))
    ref.assert_within(y, want, limit + ref.half_step(y.dtype) * (np.abs(want) + limit) + ref.smallest(y.dtype), "linear")


@pytest.mark.parametrize("layout", ["dense", "columns", "odd"])
@pytest.mark.parametrize("rows", [0, 1, 2, 3, 5, 8, 17, 33, 64])
@pytest.mark.parametrize("inputs,outputs", [(1, 1), (16, 16), (40, 9), (131, 387), (512, 130), (1000, 70), (4096, 33), (2080, 2500)])
def test_linear_of_few_rows(d3d, layout, rows, inputs, outputs):
    dtype = TYPES[(rows + inputs) % 3]
    x, w = int8(1, rows, inputs, layout), int8(2, outputs, inputs, layout)
    s, ws, b = 0.01 * normal(3, rows).abs(), 0.01 * normal(4, outputs), normal(5, outputs) if rows != 2 else None
    y = d3d.int8_linear(x, s, w, ws, b, dtype=dtype)
    assert y.shape == (rows, outputs) and y.dtype == dtype
    check_linear(x, s, w, ws, b, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["dense", "columns", "odd"])
@pytest.mark.parametrize("rows,inputs,outputs", [
    (9, 16, 16), (9, 1, 1), (127, 128, 64), (128, 96, 32), (129, 131, 40), (300, 64, 192), (257, 1000, 387), (40, 4096, 520),
    (1000, 32, 1030), (20000, 48, 24), (20000, 144, 300), (9500, 640, 515), (9500, 1040, 515), (9500, 2000, 520)])
def test_linear(d3d, dtype, layout, rows, inputs, outputs):
    """One and two CTAs to a tile, one tile and several to a CTA, ends of every kind."""
    x, w = int8(1, rows, inputs, layout), int8(2, outputs, inputs, layout)
    s, ws, b = 0.01 * normal(3, rows).abs(), 0.01 * normal(4, outputs), normal(5, outputs)
    check_linear(x, s, w, ws, b, d3d.int8_linear(x, s, w, ws, b, dtype=dtype))


@pytest.mark.parametrize("rows,inputs,outputs", [
    (4000, 48, n) for n in (130, 208, 272, 336, 387, 464, 528, 592, 656, 720, 784, 848, 912, 976)] + [
    (9600, 1040, n) for n in (272, 304, 387, 496, 592, 688)])
def test_linear_by_tiles_of_every_width(d3d, rows, inputs, outputs):
    """With one CTA to a tile 48 to 256 output channels, by 16, in 32 bits; with two 96 to 256 by 32."""
    x, w = int8(1, rows, inputs), int8(2, outputs, inputs)
    s, ws, b = 0.01 * normal(3, rows).abs(), 0.01 * normal(4, outputs), normal(5, outputs)
    for dtype in (torch.float32, torch.bfloat16):
        check_linear(x, s, w, ws, b, d3d.int8_linear(x, s, w, ws, b, dtype=dtype))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 20, 100])
@pytest.mark.parametrize("layouts", [("odd", "dense"), ("columns", "odd"), ("odd", "columns")])
@pytest.mark.parametrize("inputs,outputs", [(1024, 5000), (2080, 2500), (48, 40)])
def test_linear_of_one_side_off_its_places(d3d, rows, layouts, inputs, outputs):
    dtype = TYPES[(rows + outputs) % 3]
    x, w = int8(1, rows, inputs, layouts[0]), int8(2, outputs, inputs, layouts[1])
    s, ws, b = 0.01 * normal(3, rows).abs(), 0.01 * normal(4, outputs), normal(5, outputs)
    check_linear(x, s, w, ws, b, d3d.int8_linear(x, s, w, ws, b, dtype=dtype))
    out = torch.full((rows, outputs), 7.0, device=DEV, dtype=dtype)
    d3d.int8_linear(x, s, w, ws, b, dtype=dtype, num_rows=live(rows - 1), out=out)
    assert (out[rows - 1:] == 7).all()
    if rows > 1:
        check_linear(x[:-1], s[:-1], w, ws, b, out[:-1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("outputs", [24, 20, 18, 17, 264, 260, 258, 257])
@pytest.mark.parametrize("start", [0, 1, 2, 4, 8])
def test_linear_into_places_of_every_alignment(d3d, dtype, outputs, start):
    """Rows of the result that start on 2, 4, 8 or 16 bytes; what lies around it stays as it was."""
    for rows in (100, 300):
        x, w = int8(1, rows, 80), int8(2, outputs, 80)
        s, ws, b = 0.01 * normal(3, rows).abs(), 0.01 * normal(4, outputs), normal(5, outputs)
        buf = torch.full((rows * outputs + 64,), 7.0, device=DEV, dtype=dtype)
        out = buf[start:start + rows * outputs].view(rows, outputs)
        d3d.int8_linear(x, s, w, ws, b, dtype=dtype, out=out)
        check_linear(x, s, w, ws, b, out)
        assert (buf[:start] == 7).all() and (buf[start + rows * outputs:] == 7).all()
        out.fill_(7.0)
        d3d.int8_linear(x, s, w, ws, b, dtype=dtype, out=out, num_rows=live(90))
        check_linear(x[:90], s[:90], w, ws, b, out[:90])
        assert (buf[:start] == 7).all() and (buf[start + 90 * outputs:] == 7).all()


@pytest.mark.parametrize("rows,count", [(8, 5), (8, 0), (50, 33), (50, 0), (300, 200), (300, 0), (300, -3), (20000, 19001), (20000, 40000)])
def test_linear_counts(d3d, rows, count):
    inputs = 64 if rows > 300 else 512  # few rows: a sum shared by a cluster
    x, w = int8(1, rows, inputs), int8(2, 136, inputs)
    s, ws = 0.01 * normal(3, rows).abs(), 0.01 * normal(4, 136)
    out = torch.full((rows, 136), 7.0, device=DEV, dtype=torch.float16)
    d3d.int8_linear(x, s, w, ws, num_rows=live(count), out=out)
    n = max(0, min(rows, count))
    assert (out[n:] == 7).all()
    if n:
        check_linear(x[:n], s[:n], w, ws, None, out[:n])


@pytest.fixture
def wait_limit():
    """Sets the cycles after which a bounded wait gives up; the usual second again afterwards."""
    from deploy3d_b200 import _lib
    set_to = lambda cycles: _lib.check("d3d_debug_set_wait_limit", _lib.lib().d3d_debug_set_wait_limit(cycles))
    yield set_to
    set_to(0)


def kernel_error():
    import ctypes
    from deploy3d_b200 import _lib
    code = ctypes.c_int(-1)
    _lib.check("d3d_debug_take_kernel_error", _lib.lib().d3d_debug_take_kernel_error(ctypes.byref(code)))
    return code.value


@pytest.mark.parametrize("rows,inputs,outputs,base", [
    (20000, 512, 512, 100), (128, 8192, 256, 100),      # a CTA to a tile: several tiles each, long sums
    (9600, 2048, 1024, 100), (9600, 8192, 512, 100),    # two CTAs to a tile
    (20, 200, 20000, 200), (20, 8192, 512, 200)])       # few rows: a CTA to a sum, a cluster to a sum
def test_linear_whose_wait_gives_up(d3d, wait_limit, rows, inputs, outputs, base):
    """A wait that gives up ends the launch with an error word, wherever in the kernel it happens; a launch without one is right, and
    so are those after the limit is the usual one again."""
    x, w = int8(1, rows, inputs), int8(2, outputs, inputs)
    s, ws = 0.01 * normal(3, rows).abs(), 0.01 * normal(4, outputs)
    want = d3d.int8_linear(x, s, w, ws)
    assert kernel_error() == 0
    codes = set()
    for cycles in (1, 200, 700, 2000, 6000):
        wait_limit(cycles)
        got = d3d.int8_linear(x, s, w, ws)
        code = kernel_error()
        codes.add(code)
        assert code == 0 or base < code <= base + 4
        assert code or torch.equal(got, want)
    wait_limit(0)
    assert codes - {0}, "no wait gave up"
    for _ in range(3):
        assert torch.equal(d3d.int8_linear(x, s, w, ws), want) and kernel_error() == 0


def test_linear_of_rows_that_are_not_finite(d3d):
    """A row with a NaN in it is NaN behind the product, and no other is."""
    for rows in (4, 200):
        x = features(1, rows, 64, torch.float16)
        x[2, 5] = float("inf")
        q, s = d3d.quantize_rows(x)
        y = d3d.int8_linear(q, s, int8(2, 48, 64), normal(3, 48))
        assert y[2].isnan().all() and int(y.isnan().any(1).sum()) == 1


# ---- as a block uses them -------------------------------------------------------------------------------------------
def test_a_block_over_the_voxels_of_a_scan(d3d):
    """Encoder, then norm, 8-bit projection to features and gates (columns of one tensor), the recurrence both ways, 8-bit
    projection back onto a residual: with the live count on the device throughout, captured once and replayed on a second
    scan of another size.  Every step against its definition, from what the step before left."""
    most, channels = 4000, 32
    config = torch.tensor([0, 0, 0, 0.5, 0.5, 0.5], device=DEV)
    shape = torch.empty((1, 0, 20, 40, 40), dtype=torch.int32, device=DEV)
    points, batch = torch.zeros((6000, 4), device=DEV), torch.full((6000,), -1, dtype=torch.int32, device=DEV)
    lift = normal(1, 4, channels).half()
    w, b = 1 + 0.2 * normal(2, channels), 0.1 * normal(3, channels)
    q1, s1 = d3d.quantize_rows(normal(4, 2 * channels, channels))
    q2, s2 = d3d.quantize_rows(normal(5, channels, 2 * channels))
    b1 = 0.1 * normal(6, 2 * channels)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)

    def scan(seed, n):
        pos = torch.rand((n, 3), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * torch.tensor([20.0, 20, 10], device=DEV)
        points.zero_(), batch.fill_(-1)
        points[:n, :3], points[:n, 3], batch[:n] = pos, normal(seed, n), 0

    def block():
        means, coors, count = d3d.simple_mean_encoder(points, batch, config, shape, most)
        x = means.half() @ lift
        q, sx = d3d.layer_norm_int8(x, w, b, EPS, num_rows=count)
        both = d3d.int8_linear(q, sx, q1, s1, b1, dtype=torch.float16, num_rows=count)
        offsets = torch.cat([zero, count])
        feats, gates = both[:, :channels], both[:, channels:]
        mixed = torch.zeros((most, 2 * channels), device=DEV, dtype=torch.float16)
        down, _ = d3d.gated_recurrence(feats, gates, offsets)
        up, _ = d3d.gated_recurrence(feats, gates, offsets, reverse=True)
        mixed[:, :channels], mixed[:, channels:] = down, up
        qm, sm = d3d.quantize_rows(mixed, num_rows=count)
        y = d3d.int8_linear(qm, sm, q2, s2, dtype=torch.float16, num_rows=count)
        z, total = d3d.layer_norm(y, w, b, EPS, residual=x, num_rows=count)
        return count, x, q, sx, both, down, up, mixed, qm, sm, y, z, total

    scan(11, 3000)
    block()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        outs = block()
    for seed, points_of in ((11, 3000), (12, 5500), (13, 40)):
        scan(seed, points_of)
        graph.replay()
        torch.cuda.synchronize()
        n = int(outs[0])
        assert 0 < n <= most
        x, q, sx, both, down, up, mixed, qm, sm, y, z, total = (t[:n] for t in outs[1:])
        want, limit, _, _, _ = ref.norm(ref.as64(x), ref.as64(w), ref.as64(b), EPS)
        step = ref.as64(sx)[:, None]
        assert (np.abs(ref.as64(q) * step - want) <= step / 2 + limit + ref.U32 * 127 * step).all()
        check_linear(q, sx, q1, s1, b1, both)
        for got, reverse in ((down, False), (up, True)):
            h, off, _, _, _, _ = ref.recurrence(ref.as64(both[:, :channels]), ref.as64(both[:, channels:]), [0, n], None, reverse, torch.float16)
            ref.assert_within(got, h, off + ref.half_step(got.dtype) * (np.abs(h) + off) + ref.smallest(got.dtype), "h")
        check_quantized(mixed.float(), qm, sm)
        check_linear(qm, sm, q2, s2, None, y)
        assert torch.equal(total, (y.float() + x.float()).half())
        check_norm(total, w, b, z)


def test_offsets_past_32_bits(d3d):
    """Columns of a tensor of 4.4 GB and results of as much: the last rows, a tile and a sequence of their own, are what they are
    without the rows in front of them."""
    rows, tail, channels = 512 * 4200, 128, 32
    wide = torch.zeros((rows, 1040), dtype=torch.bfloat16, device=DEV)
    wide[-tail:] = features(1, tail, 1040, torch.bfloat16)
    x, g = wide[:, 16:16 + channels], wide[:, 512:512 + channels]
    assert rows * 1040 > 2 ** 31

    def alone(t):
        return t[-tail:].clone()
    xs, gs, w = alone(x), alone(g), normal(2, channels)
    y, mean, rstd = d3d.layer_norm(x, w, None, EPS, with_stats=True)
    for a, b in zip((y, mean, rstd), d3d.layer_norm(xs, w, None, EPS, with_stats=True)):
        assert torch.equal(a[-tail:], b)
    dx = d3d.layer_norm_backward(g, x, w, mean, rstd)[0]
    assert torch.equal(dx[-tail:], d3d.layer_norm_backward(gs, xs, w, alone(mean), alone(rstd))[0])
    offsets = torch.tensor([0, rows - tail, rows], dtype=torch.int32, device=DEV)
    short = torch.tensor([0, tail], dtype=torch.int32, device=DEV)
    for reverse in (False, True):
        h, final, states = d3d.gated_recurrence(x, g, offsets, reverse=reverse, with_states=True)
        h2, final2, states2 = d3d.gated_recurrence(xs, gs, short, reverse=reverse, with_states=True)
        assert torch.equal(h[-tail:], h2) and torch.equal(final[1:], final2)
        back = d3d.gated_recurrence_backward(g, x, g, offsets, states, reverse=reverse)
        back2 = d3d.gated_recurrence_backward(gs, xs, gs, short, states2, reverse=reverse)
        assert all(torch.equal(a[-len(b):], b) for a, b in zip(back, back2))
    state = torch.zeros((rows, channels), device=DEV)
    out, _ = d3d.gated_recurrence_step(x, g, state)
    assert torch.equal(out[-tail:], d3d.gated_recurrence_step(xs, gs, alone(state))[0])
    y = d3d.layer_norm(wide, None, None, EPS)
    assert torch.equal(y[-tail:], d3d.layer_norm(alone(wide), None, None, EPS))
    del y
    q, s = d3d.quantize_rows(wide)
    q2, s2 = d3d.quantize_rows(alone(wide))
    assert torch.equal(q[-tail:], q2) and torch.equal(s[-tail:], s2)
    ones = torch.ones(1040, device=DEV)
    for weight in (int8(3, 1040, 1040), int8(3, 1040, 1040, "odd"), int8(3, 1039, 1040)):
        outs = len(weight)
        y = d3d.int8_linear(q, s, weight, ones[:outs], dtype=torch.bfloat16)
        assert torch.equal(y[-tail:], d3d.int8_linear(q2, s2, weight, ones[:outs], dtype=torch.bfloat16))
    y = d3d.int8_linear(q[:, 1:1001], s, weight[:, :1000].contiguous(), ones[:outs], dtype=torch.bfloat16)
    assert torch.equal(y[-tail:], d3d.int8_linear(q2[:, 1:1001], s2, weight[:, :1000].contiguous(), ones[:outs], dtype=torch.bfloat16))


def test_results_in_place_of_the_features(d3d):
    for dtype in TYPES:
        for channels in (24, 7, 600):
            x, g = features(1, 1500, channels, dtype), gates_like(2, 1500, channels, dtype)
            offsets = torch.tensor([0, 700, 1500], dtype=torch.int32, device=DEV)
            want, again = d3d.layer_norm(x, None, None, EPS), x.clone()
            assert d3d.layer_norm(again, None, None, EPS, out=again) is again and torch.equal(again, want)
            for reverse in (False, True):
                want, again = d3d.gated_recurrence(x, g, offsets, reverse=reverse)[0], x.clone()
                d3d.gated_recurrence(again, g, offsets, reverse=reverse, out=again)
                assert torch.equal(again, want)


def test_autograd_notices_what_was_written_over(d3d):
    """A tensor that autograd has kept and that an operator is then given as `out`: going back raises, as behind torch's own
    operators in place, and does not use the new contents.  Tensors of inference mode have no such count."""
    x, offsets = features(1, 40, 16, torch.float32), torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    q, s = d3d.quantize_rows(x)
    calls = [lambda out: d3d.layer_norm(x, None, out=out), lambda out: d3d.gated_recurrence(x, x, offsets, out=out),
             lambda out: d3d.gated_recurrence_step(x, x, x, state_out=out),
             lambda out: d3d.int8_linear(q, s, q[:16], s[:16], dtype=torch.float32, out=out)]
    for call in calls:
        a, kept = normal(2, 40, 16).requires_grad_(), normal(3, 40, 16)
        y = (a * kept).sum()
        before = kept._version
        call(kept)
        assert kept._version == before + 1
        with pytest.raises(RuntimeError):
            y.backward()
        with torch.inference_mode():
            buf = torch.empty((40, 16), device=DEV)
        call(buf)
        assert torch.equal(buf, kept) and x._version == 0


def test_refusals_on_the_gpu(d3d):
    """Shapes, types and devices that do not fit raise before anything is launched."""
    x, g = features(1, 8, 16, torch.float16), features(2, 8, 16, torch.float16)
    w, off = normal(3, 16), torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    q, s = d3d.quantize_rows(x)
    _, final, states = d3d.gated_recurrence(x, g, off, with_states=True)
    stat = normal(4, 8)
    bad = [
        (TypeError, lambda: d3d.layer_norm(x.double(), w)), (TypeError, lambda: d3d.layer_norm(None, w)),
        (ValueError, lambda: d3d.layer_norm(x[0], w)), (ValueError, lambda: d3d.layer_norm(x, w[:8])),
        (ValueError, lambda: d3d.layer_norm(x, w.half())), (ValueError, lambda: d3d.layer_norm(x, w.cpu())),
        (ValueError, lambda: d3d.layer_norm(x, w, residual=g[:4])), (ValueError, lambda: d3d.layer_norm(x, w, residual=g.float())),
        (ValueError, lambda: d3d.layer_norm(x, w, out=torch.empty(8, 32, device=DEV, dtype=torch.float16)[:, :16])),
        (ValueError, lambda: d3d.layer_norm(x, w, num_rows=torch.tensor([8], device=DEV))),
        (ValueError, lambda: d3d.layer_norm(x, w, num_rows=torch.tensor([8], dtype=torch.int32))),
        (ValueError, lambda: d3d.layer_norm(x[:, :0], None)), (TypeError, lambda: d3d.layer_norm_backward(g, x, w, None, stat)),
        (ValueError, lambda: d3d.layer_norm_backward(g, x, w, stat[:4], stat)),
        (ValueError, lambda: d3d.quantize_rows(x.cpu())), (TypeError, lambda: d3d.int8_linear(x, s, q, w[:8])),
        (ValueError, lambda: d3d.int8_linear(q, s, q[:, :8], s)), (ValueError, lambda: d3d.int8_linear(q, s[:4], q, s)),
        (TypeError, lambda: d3d.int8_linear(q, s, q, s, dtype=torch.int32)), (ValueError, lambda: d3d.int8_linear(q, s, q[:0], s[:0])),
        (ValueError, lambda: d3d.gated_recurrence(x, g[:, :8], off)), (ValueError, lambda: d3d.gated_recurrence(x, g.float(), off)),
        (ValueError, lambda: d3d.gated_recurrence(x, g, off.long())), (ValueError, lambda: d3d.gated_recurrence(x, g, off[:0])),
        (ValueError, lambda: d3d.gated_recurrence(x, g, off, initial=normal(5, 2, 16))),
        (ValueError, lambda: d3d.gated_recurrence_backward(g, x, g, off, states[:0])),
        (ValueError, lambda: d3d.gated_recurrence_step(x, g, normal(6, 8, 8))), (TypeError, lambda: d3d.gated_recurrence_step(x, g, None))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    from deploy3d_b200._lib import D3DError
    with pytest.raises(D3DError):
        d3d.layer_norm(torch.empty((2, 8193), device=DEV), None)
    with pytest.raises(D3DError):
        d3d.layer_norm(x, w, eps=-1.0)


def test_no_wait_gave_up(d3d):
    import ctypes
    from deploy3d_b200 import _lib
    code = ctypes.c_int(0)
    _lib.check("d3d_debug_take_kernel_error", _lib.lib().d3d_debug_take_kernel_error(ctypes.byref(code)))
    assert code.value == 0

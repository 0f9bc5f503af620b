"""The voxel-sequence operators in 64 bits, row by row from their definitions, with bounds for what 32-bit arithmetic may be off.

A bound follows the operator's own recursion: every operation of the kernel may be off by a few half units of the last place of
its result (U32 each; K of them cover a gate's exponential, quotient and products, or a sum's tree), and what it is off is
carried on by the same factors as the value.  A result rounded to its type is off by half a step of it on top."""
import numpy as np
import torch

U32 = 2.0 ** -24
K = 16          # half units per step of a recurrence: exp 4, quotient 4, products, sums and the composition of maps 8
# 16-bit gates g: 1 - f = t / (1 + t), t = 2^y by the hardware's exponential, y = -g log2(e) in 32 bits.  log2(e) is rounded to
# half a unit and so is y, each at most |y| U32, which moves t by ln 2 as much relatively: 2 |g| log2(e) ln 2 = 2 |g| half units
# on top of the 4 of the exponential itself.
PER_GATE = 2.0
DEPTH = 64      # half units of a sum over channels: up to 32 terms in a thread, a tree behind it, the operations around it


def half_step(dtype):
    return 0.0 if dtype == torch.float64 else torch.finfo(dtype).eps / 2


def smallest(dtype):
    """What rounding near zero may be off: half of the smallest subnormal."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def as64(t):
    return t.detach().double().cpu().numpy()


def assert_within(got, want, limit, what):
    got = as64(got) if torch.is_tensor(got) else got
    assert got.shape == want.shape, "%s: shape %s, wanted %s" % (what, got.shape, want.shape)
    same = np.isnan(got) == np.isnan(want)
    assert same.all(), "%s: NaN in %d wrong places" % (what, int((~same).sum()))
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want) - limit
        off[(got == want) | np.isnan(want)] = -1.0
    assert not (off > 0).any(), "%s: %d of %d off, worst by %.3e over its limit of %.3e (wanted %.6e)" % (
        what, int((off > 0).sum()), off.size, off.max(), limit.flat[off.argmax()] if limit.shape == off.shape else 0.0,
        want.flat[off.argmax()])


def norm(x, weight, bias, eps):
    """y, its bound before rounding, mean, rstd, hat."""
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    hat = (x - mean) * rstd
    y = hat * weight + bias
    limit = U32 * DEPTH * (np.abs(weight) * (np.abs(hat) + np.abs(x).mean(1, keepdims=True) * rstd + 1) + np.abs(bias))
    return y, limit, mean[:, 0], rstd[:, 0], hat


def norm_backward(grad, x, weight, mean, rstd):
    """(dx, bound), (dw, bound), (db, bound)."""
    hat = (x - mean[:, None]) * rstd[:, None]
    g = grad * weight
    m1, m2 = g.mean(1, keepdims=True), (g * hat).mean(1, keepdims=True)
    dx = rstd[:, None] * (g - m1 - hat * m2)
    hat_off = np.abs(x).mean(1, keepdims=True) * rstd[:, None] + np.abs(hat) + 1
    size = np.abs(g).mean(1, keepdims=True) + np.abs(g * hat).mean(1, keepdims=True)
    limit = 2 * U32 * DEPTH * rstd[:, None] * (np.abs(g) + size * (1 + np.abs(hat)) + hat_off * (np.abs(m2) + size))
    n = DEPTH + x.shape[0]
    dw, db = (grad * hat).sum(0), grad.sum(0)
    return ((dx, limit), (dw, U32 * n * (np.abs(grad) * (np.abs(hat) + hat_off)).sum(0)),
            (db, U32 * n * np.abs(grad).sum(0)))


def quantize(x32):
    """float32 rows (numpy) -> (integers, float32 scales); the quotient in 64 bits is exact to far below any border's distance."""
    amax = np.abs(x32).max(1) if x32.shape[1] else np.zeros(len(x32), np.float32)
    with np.errstate(all="ignore"):
        scale = (amax / np.float32(127)).astype(np.float32)
        fine = np.isfinite(x32).all(1)
        zero = fine & (scale < np.float32(2.0 ** -126))
        scale = np.where(fine, np.where(zero, np.float32(0), scale), np.float32(np.nan))
        q = np.rint(x32.astype(np.float64) / scale.astype(np.float64)[:, None])
    return np.where((fine & ~zero)[:, None], q, 0.0), scale


def sigmoid(g):
    with np.errstate(over="ignore"):
        return np.where(g >= 0, 1 / (1 + np.exp(-np.abs(g))), np.exp(-np.abs(g)) / (1 + np.exp(-np.abs(g))))


def half_units(gates, dtype):
    """Half units that a step of the recurrence may be off, by gate."""
    return K + (PER_GATE * np.abs(gates) if dtype != torch.float32 else 0.0 * gates)


def recurrence(x, gates, offsets, initial, reverse, dtype=torch.float32):
    """h, its bound, final, its bound, h in front of every row, its bound.  Rows outside the sequences stay NaN."""
    seqs, channels = len(offsets) - 1, x.shape[1]
    f, add, k = sigmoid(gates), sigmoid(-gates), half_units(gates, dtype)
    h, off, before, before_off = (np.full(x.shape, np.nan) for _ in range(4))
    final, final_off = np.zeros((seqs, channels)), np.zeros((seqs, channels))
    for s in range(seqs):
        c = initial[s].copy() if initial is not None else np.zeros(channels)
        size, e = np.abs(c), np.zeros(channels)
        rows = range(offsets[s], offsets[s + 1])
        for t in (reversed(rows) if reverse else rows):
            before[t], before_off[t] = c, e
            c = f[t] * c + add[t] * x[t]
            size = f[t] * size + add[t] * np.abs(x[t])
            e = f[t] * e + U32 * k[t] * size
            h[t], off[t] = c, e
        final[s], final_off[s] = c, e
    return h, off, final, final_off, before, before_off


def recurrence_backward(grad, x, gates, offsets, initial, grad_final, reverse, dtype=torch.float32):
    """(dx, bound), (dgates, bound), (dinitial, bound)."""
    seqs, channels = len(offsets) - 1, x.shape[1]
    f, add, k = sigmoid(gates), sigmoid(-gates), half_units(gates, dtype)
    _, _, _, _, before, before_off = recurrence(x, gates, offsets, initial, reverse, dtype)
    dx, dg, dx_off, dg_off = (np.full(x.shape, np.nan) for _ in range(4))
    di, di_off = np.zeros((seqs, channels)), np.zeros((seqs, channels))
    for s in range(seqs):
        q = grad_final[s].copy() if grad_final is not None else np.zeros(channels)
        size, e = np.abs(q), np.zeros(channels)
        rows = range(offsets[s], offsets[s + 1])
        for t in (rows if reverse else reversed(rows)):
            delta, dsize = grad[t] + q, np.abs(grad[t]) + size
            doff = e + U32 * dsize
            dx[t] = delta * add[t]
            dx_off[t] = add[t] * (doff + U32 * k[t] * dsize)
            dg[t] = delta * (before[t] - x[t]) * f[t] * add[t]
            dg_off[t] = f[t] * add[t] * (doff * np.abs(before[t] - x[t]) + dsize * before_off[t] +
                                         U32 * k[t] * dsize * (np.abs(before[t]) + np.abs(x[t])))
            q, size = f[t] * delta, f[t] * dsize
            e = f[t] * doff + U32 * k[t] * size
        di[s], di_off[s] = q, e
    return (dx, dx_off), (dg, dg_off), (di, di_off)

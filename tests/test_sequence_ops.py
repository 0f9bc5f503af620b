"""What the voxel-sequence operators refuse, and their formulas' gradients against differences (CPU)."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

from tests import _sequence as ref

BAD = -1
ONE = ctypes.c_void_p(4096)  # an address no refused call follows


def test_entry_points_refuse_bad_arguments(d3d):
    from deploy3d_b200 import _lib
    lib, F, I8 = _lib.lib(), _lib.D3D_HALF, _lib.D3D_INT8
    odd = ctypes.c_void_p(4097)
    norm = lambda dt=F, x=ONE, ld=16, res=None, rld=0, eps=1e-5, rows=4, ch=16, total=None, out=ONE, mean=None, rstd=None: \
        lib.d3d_layer_norm(dt, x, ld, res, rld, None, None, eps, rows, ch, None, total, out, mean, rstd, None)
    assert norm(rows=0) == 0
    assert norm(dt=I8) == -2 and norm(ch=8193, ld=8193) == -6
    for bad in (dict(x=None), dict(out=None), dict(ld=15), dict(rows=-1), dict(ch=0), dict(eps=-1.0), dict(res=ONE, rld=16),
                dict(total=ONE), dict(res=ONE, rld=3, total=ONE), dict(mean=ONE), dict(rstd=ONE), dict(x=odd), dict(out=odd)):
        assert norm(**bad) == BAD, bad
    quant = lambda dt=F, x=ONE, ld=16, rows=4, ch=16, q=ONE, qld=16, s=ONE: \
        lib.d3d_quantize_rows(dt, x, ld, rows, ch, None, q, qld, s, None)
    assert quant(rows=0) == 0 and quant(dt=I8) == -2 and quant(ch=9000, ld=9000, qld=9000) == -6
    for bad in (dict(x=None), dict(q=None), dict(s=None), dict(qld=15), dict(ld=8), dict(x=odd)):
        assert quant(**bad) == BAD, bad
    n = lib.d3d_layer_norm_backward_workspace(4, 16)
    back = lambda dt=F, g=ONE, x=ONE, m=ONE, ws=ONE, nb=n, ld=16: \
        lib.d3d_layer_norm_backward(dt, g, 16, x, ld, None, 0, None, m, ONE, 4, 16, None, ONE, None, None, ws, nb, None)
    assert back(dt=I8) == -2 and back(nb=n - 1) == -3
    for bad in (dict(g=None), dict(x=None), dict(m=None), dict(ws=None), dict(ld=2)):
        assert back(**bad) == BAD, bad
    n = lib.d3d_gated_recurrence_workspace(200, 16)
    scan = lambda dt=F, x=ONE, g=ONE, ld=16, offs=ONE, seqs=2, rows=200, ch=16, out=ONE, ws=ONE, nb=n: \
        lib.d3d_gated_recurrence(dt, x, ld, g, 16, offs, seqs, rows, ch, 0, None, out, None, None, ws, nb, None)
    assert scan(dt=I8) == -2 and scan(nb=n - 1) == -3 and scan(seqs=0) == 0
    assert scan(rows=1 << 31) == -6 and scan(ch=1 << 17, ld=1 << 17) == BAD
    for bad in (dict(x=None), dict(g=None), dict(offs=None), dict(ld=3), dict(seqs=-1), dict(rows=-1), dict(ch=0), dict(out=None),
                dict(ws=None), dict(ws=ctypes.c_void_p(4100)), dict(x=odd)):
        assert scan(**bad) == BAD, bad
    lin = lambda dt=F, x=ONE, s=ONE, w=ONE, ld=16, rows=100, k=16, n=16, out=ONE, ws=None, nb=0: \
        lib.d3d_int8_linear(dt, x, ld, s, rows, None, w, 16, ONE, None, k, n, out, ws, nb, None)
    assert lin(rows=0) == 0 and lin(dt=I8) == -2 and lin(rows=1 << 31) == -6 and lin(n=1 << 17) == -6
    for bad in (dict(x=None), dict(s=None), dict(w=None), dict(ld=15), dict(rows=-1), dict(k=0), dict(n=0), dict(out=None),
                dict(out=odd), dict(x=odd), dict(w=odd)):  # the last two: rows to be copied, and no workspace for it
        assert lin(**bad) == BAD, bad
    need = lib.d3d_int8_linear_workspace(odd, 16, 100, ONE, 16, 16, 16)
    assert need >= 100 * 16 and lin(x=odd, ws=ONE, nb=need - 1) == -3
    assert lib.d3d_int8_linear_workspace(ONE, 16, 100, ONE, 16, 16, 16) == 0 == lib.d3d_int8_linear_workspace(odd, 17, 8, odd, 17, 16, 16)
    step = lambda dt=F, x=ONE, s=ONE, ld=16, rows=4, out=ONE: \
        lib.d3d_gated_recurrence_step(dt, x, ld, ONE, 16, s, ONE, out, rows, 16, None)
    assert step(rows=0) == 0 and step(dt=I8) == -2
    for bad in (dict(x=None), dict(s=None), dict(ld=15), dict(rows=-1), dict(out=None), dict(x=odd)):
        assert step(**bad) == BAD, bad


def test_entry_points_refuse_addresses_off_their_elements(d3d):
    """Every pointer that a kernel would follow, one byte off: two-byte features, four-byte parameters, states, scales, counts."""
    from deploy3d_b200 import _lib
    lib, F = _lib.lib(), _lib.D3D_HALF
    V = ctypes.c_void_p
    odd, half = V(4097), V(4098)

    def refuses(fn, good, pointers):
        """`good` would be launched; with any of the pointers off its elements it is refused."""
        for name, size in pointers.items():
            for bad in (odd, half) if size == 4 else (odd,):
                assert fn(*dict(good, **{name: bad}).values()) == BAD, (fn.__name__, name, bad.value)
    norm = dict(dt=F, x=ONE, ld=16, res=ONE, rld=16, w=ONE, b=ONE, eps=1e-5, rows=4, ch=16, num=ONE, total=ONE, out=ONE, mean=ONE,
                rstd=ONE, st=None)
    refuses(lib.d3d_layer_norm, norm, dict(x=2, res=2, total=2, out=2, w=4, b=4, num=4, mean=4, rstd=4))
    norm8 = dict(dt=F, x=ONE, ld=16, res=ONE, rld=16, w=ONE, b=ONE, eps=1e-5, rows=4, ch=16, num=ONE, total=ONE, q=ONE, qld=16,
                 s=ONE, st=None)
    refuses(lib.d3d_layer_norm_int8, norm8, dict(x=2, res=2, total=2, w=4, b=4, num=4, s=4))
    quant = dict(dt=F, x=ONE, ld=16, rows=4, ch=16, num=ONE, q=ONE, qld=16, s=ONE, st=None)
    refuses(lib.d3d_quantize_rows, quant, dict(x=2, num=4, s=4))
    back = dict(dt=F, g=ONE, gld=16, x=ONE, ld=16, t=ONE, tld=16, w=ONE, m=ONE, r=ONE, rows=4, ch=16, num=ONE, gx=ONE, gw=ONE,
                gb=ONE, ws=ONE, nb=1 << 20, st=None)
    refuses(lib.d3d_layer_norm_backward, back, dict(g=2, x=2, t=2, gx=2, w=4, m=4, r=4, num=4, gw=4, gb=4, ws=4))
    lin = dict(dt=F, x=ONE, ld=16, s=ONE, rows=100, num=ONE, w=ONE, wld=16, ws=ONE, b=ONE, k=16, n=16, out=ONE, work=ONE, nb=1 << 20,
               st=None)
    refuses(lib.d3d_int8_linear, lin, dict(out=2, s=4, num=4, ws=4, b=4))
    for rows in (100, 200):  # one tile, several
        scan = dict(dt=F, x=ONE, ld=16, g=ONE, gld=16, offs=ONE, seqs=2, rows=rows, ch=16, rev=0, init=ONE, out=ONE, fin=ONE, states=ONE,
                    ws=ONE, nb=1 << 20, st=None)
        refuses(lib.d3d_gated_recurrence, scan, dict(x=2, g=2, out=2, offs=4, init=4, fin=4, states=4))
        back = dict(dt=F, d=ONE, dld=16, x=ONE, ld=16, g=ONE, gld=16, offs=ONE, seqs=2, rows=rows, ch=16, rev=0, states=ONE, init=ONE,
                    gf=ONE, gx=ONE, gg=ONE, gi=ONE, ws=ONE, nb=1 << 20, st=None)
        refuses(lib.d3d_gated_recurrence_backward, back, dict(d=2, x=2, g=2, gx=2, gg=2, offs=4, states=4, init=4, gf=4, gi=4))
    step = dict(dt=F, x=ONE, ld=16, g=ONE, gld=16, s=ONE, so=ONE, out=ONE, rows=4, ch=16, st=None)
    refuses(lib.d3d_gated_recurrence_step, step, dict(x=2, g=2, out=2, s=4, so=4))


def test_few_rows_off_their_places_are_copied_and_not_all_weights_read_by_bytes(d3d):
    from deploy3d_b200 import _lib
    need = lambda x, rows, w: _lib.lib().d3d_int8_linear_workspace(ctypes.c_void_p(x), 4096, rows, ctypes.c_void_p(w), 4096, 4096, 4096)
    for rows in (1, 4):
        assert need(4097, rows, 4096) == 4096 * rows      # the rows go to the workspace
        assert need(4097, rows, 4097) == need(4096, rows, 4097) == 0  # the weights are read where they are
        assert need(4096, rows, 4096) == 0
    assert need(4097, 5, 4097) == 4096 * (5 + 4096) and need(4096, 5, 4097) == 4096 * 4096


def test_kernels_read_what_may_still_be_written_by_plain_loads():
    """The kernels live while the one in front of them still writes, so none of their loads may be of the kind that takes memory
    for constant as long as the kernel lives: __ldg, or what a const __restrict__ argument allows a plain load to become."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deploy3d_b200", "csrc")
    for name in ("layer_norm.cu", "int8_linear.cu", "gated_recurrence.cu", "packed.cuh"):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(root, name)).read())
        assert "__ldg(" not in text and ".nc." not in text, name
        assert not re.search(r"const \w+\s*\*\s*__restrict__", text), name


def test_operators_refuse_what_they_cannot_run(d3d):
    x = torch.zeros((4, 16))
    with pytest.raises(ValueError):
        d3d.layer_norm(x, None)
    with pytest.raises(ValueError):
        d3d.quantize_rows(x)
    with pytest.raises(ValueError):
        d3d.gated_recurrence(x, x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        d3d.gated_recurrence_step(x, x, x)


def test_formulas_of_the_gradients_against_differences():
    """64-bit central differences of the definitions: off by e^2 of the terms and 2^-53 / e, so 1e-6 with e = 1e-5."""
    r, e = np.random.Generator(np.random.PCG64(1)), 1e-5
    x, w, b, c = r.normal(size=(7, 5)), r.normal(size=5), r.normal(size=5), r.normal(size=(7, 5))
    _, _, mean, rstd, _ = ref.norm(x, w, b, 1e-5)
    grads = [g for g, _ in ref.norm_backward(c, x, w, mean, rstd)]
    for k, p in enumerate((x, w, b)):
        d = r.normal(size=p.shape)
        args = [[q + s * e * d if i == k else q for i, q in enumerate((x, w, b))] for s in (1, -1)]
        diff = np.subtract(*[(ref.norm(*a, 1e-5)[0] * c).sum() for a in args]) / (2 * e)
        assert abs(diff - (grads[k] * d).sum()) <= 1e-6 * np.abs(grads[k] * d).sum()
    for reverse in (False, True):
        x, g, h0 = r.normal(size=(9, 3)), r.normal(size=(9, 3)), r.normal(size=(3, 3))
        offs, c, cf = [0, 4, 4, 9], r.normal(size=(9, 3)), r.normal(size=(3, 3))
        grads = [v for v, _ in ref.recurrence_backward(c, x, g, offs, h0, cf, reverse)]
        for k, p in enumerate((x, g, h0)):
            d = r.normal(size=p.shape)
            vals = []
            for s in (1, -1):
                a = [q + s * e * d if i == k else q for i, q in enumerate((x, g, h0))]
                h, _, final, _, _, _ = ref.recurrence(a[0], a[1], offs, a[2], reverse)
                vals.append((h * c).sum() + (final * cf).sum())
            assert abs((vals[0] - vals[1]) / (2 * e) - (grads[k] * d).sum()) <= 1e-6 * np.abs(grads[k] * d).sum()

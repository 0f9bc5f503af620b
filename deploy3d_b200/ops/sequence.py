"""Operators of voxel-sequence networks, which mix voxels along an order instead of through a kernel neighbourhood: layer
norm, its rows in 8-bit integers, and a gated linear recurrence.  The reference has none of them.

Features are CUDA tensors ``[rows, channels]`` in float32, float16 or bfloat16 and may be columns of a wider tensor (their
channels side by side); parameters, scales and states are float32.  Everything runs on the current stream of the features'
device.  ``num_rows``, an int32 tensor of one element on the device, says how many rows are live, as the counts of the voxel
operators do: rows behind are neither read nor written (in a tensor the call has made itself they hold nothing).  ``out``
takes the result where given: dense, of the right shape and type.  Backward passes are functions of their own; nothing here
records autograd history.
"""
import torch

from .. import _lib
from ..plugins import _TORCH2D3D

_FEATURES = (torch.float32, torch.float16, torch.bfloat16)


def _features(t, what, like=None):
    """(tensor, elements between its rows) of a feature argument; one whose channels are not side by side is copied."""
    if t.dim() != 2 or not t.is_cuda:
        raise ValueError("%s: a CUDA tensor [rows, channels] is needed; this library has no CPU path" % what)
    if t.dtype not in _FEATURES:
        raise TypeError("%s: unsupported tensor dtype %s" % (what, t.dtype))
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError("%s: shape, dtype and device of the features are needed" % what)
    rows, channels = t.shape
    if channels == 0:
        raise ValueError("%s: no channels" % what)
    step, ld = t.stride(1), t.stride(0)
    if rows <= 1:
        ld = channels
    if (step != 1 and channels > 1) or ld < channels:
        t, ld = t.contiguous(), channels
    return t, ld


def _dense(t, shape, dtype, device, what):
    """Address of an optional dense argument, None without one."""
    if t is None:
        return None
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError("%s: a dense %s tensor %s on %s is needed" % (what, dtype, list(shape), device))
    return t.data_ptr()


def _count(t, device):
    if t is None:
        return None
    if t.dtype != torch.int32 or t.numel() != 1 or t.device != device:
        raise ValueError("num_rows: an int32 tensor of one element on %s is needed" % device)
    return t.data_ptr()


def _made(out, like, what="out"):
    """`out`, or a new tensor like the features."""
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _dense(out, like.shape, like.dtype, like.device, what)
    return out


def _call(name, device, *args):
    """The C-ABI function on the current stream of the device."""
    fn = getattr(_lib.lib(), name)
    if device.index == torch.cuda.current_device():
        status = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if status != 0:
        _lib.check(name, status)


def _norm_arguments(feats, weight, bias, residual, num_rows):
    feats, ld = _features(feats, "feats")
    residual, residual_ld = (None, 0) if residual is None else _features(residual, "residual", feats)
    device, channels = feats.device, feats.shape[1]
    total = None if residual is None else torch.empty(feats.shape, dtype=feats.dtype, device=device)
    return (feats, ld, residual, residual_ld, _dense(weight, (channels,), torch.float32, device, "weight"),
            _dense(bias, (channels,), torch.float32, device, "bias"), _count(num_rows, device), total)


def layer_norm(feats, weight, bias=None, eps=1e-5, residual=None, num_rows=None, with_stats=False, out=None):
    """(t - mean) * rstd * weight + bias over the channels of each row, t = feats or feats + residual; at most 8192 channels.

    weight, bias float32 [channels] (None: 1, 0).  Returns the normed rows; with `residual` also t, rounded to the type
    and normed as rounded; with `with_stats` also mean and rstd, float32 [rows], for layer_norm_backward."""
    feats, ld, residual, residual_ld, w, b, count, total = _norm_arguments(feats, weight, bias, residual, num_rows)
    rows, channels = feats.shape
    out = _made(out, feats)
    mean = rstd = None
    if with_stats:
        mean = torch.empty(rows, dtype=torch.float32, device=feats.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=feats.device)
    _call("d3d_layer_norm", feats.device, _TORCH2D3D[feats.dtype], feats.data_ptr(), ld,
          None if residual is None else residual.data_ptr(), residual_ld, w, b, float(eps), rows, channels, count,
          None if total is None else total.data_ptr(), out.data_ptr(), None if mean is None else mean.data_ptr(),
          None if rstd is None else rstd.data_ptr())
    if residual is None and not with_stats:
        return out
    return (out,) + (() if residual is None else (total,)) + ((mean, rstd) if with_stats else ())


def layer_norm_backward(grad_out, feats, weight, mean, rstd, num_rows=None, grad_total=None):
    """Gradients (feats, weight, bias) of layer_norm.  `feats` is what was normed: with a residual the sum layer_norm returned,
    `grad_total` the gradient that sum gets elsewhere; the first result is then the gradient of both summands."""
    feats, ld = _features(feats, "feats")
    grad_out, grad_ld = _features(grad_out, "grad_out", feats)
    grad_total, total_ld = (None, 0) if grad_total is None else _features(grad_total, "grad_total", feats)
    (rows, channels), device = feats.shape, feats.device
    if mean is None or rstd is None:
        raise ValueError("mean and rstd of the forward pass are needed")
    m, r = (_dense(t, (rows,), torch.float32, device, n) for t, n in ((mean, "mean"), (rstd, "rstd")))
    grad_feats = torch.empty(feats.shape, dtype=feats.dtype, device=device)
    grads = torch.empty((2, channels), dtype=torch.float32, device=device)
    nbytes = _lib.lib().d3d_layer_norm_backward_workspace(rows, channels)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    at = grads.data_ptr()
    _call("d3d_layer_norm_backward", device, _TORCH2D3D[feats.dtype], grad_out.data_ptr(), grad_ld, feats.data_ptr(), ld,
          None if grad_total is None else grad_total.data_ptr(), total_ld,
          _dense(weight, (channels,), torch.float32, device, "weight"), m, r, rows, channels, _count(num_rows, device),
          grad_feats.data_ptr(), at, at + 4 * channels, workspace.data_ptr(), nbytes)
    return grad_feats, grads[0], grads[1]


def _int8_rows(feats):
    """8-bit rows whose pitch is a multiple of 16 bytes, which is what the products read fastest, and their scales."""
    rows, channels = feats.shape
    pitch = (channels + 15) // 16 * 16
    q = torch.empty((rows, pitch), dtype=torch.int8, device=feats.device)
    return q if pitch == channels else q[:, :channels], pitch, torch.empty(rows, dtype=torch.float32, device=feats.device)


def layer_norm_int8(feats, weight, bias=None, eps=1e-5, residual=None, num_rows=None):
    """layer_norm whose result leaves as quantize_rows would give it: (int8 rows, scales), with `residual` also the sum."""
    feats, ld, residual, residual_ld, w, b, count, total = _norm_arguments(feats, weight, bias, residual, num_rows)
    q, pitch, scales = _int8_rows(feats)
    _call("d3d_layer_norm_int8", feats.device, _TORCH2D3D[feats.dtype], feats.data_ptr(), ld,
          None if residual is None else residual.data_ptr(), residual_ld, w, b, float(eps), feats.shape[0], feats.shape[1],
          count, None if total is None else total.data_ptr(), q.data_ptr(), pitch, scales.data_ptr())
    return (q, scales) if residual is None else (q, scales, total)


def quantize_rows(feats, num_rows=None):
    """(int8 [rows, channels], float32 [rows]): scale = max |row| / 127, row / scale to the nearest integer, ties to even.  Rows
    of zeros have scale 0, rows that are not finite zeros and scale NaN.  At most 8192 channels.  The rows lie a multiple of
    16 bytes apart."""
    feats, ld = _features(feats, "feats")
    q, pitch, scales = _int8_rows(feats)
    _call("d3d_quantize_rows", feats.device, _TORCH2D3D[feats.dtype], feats.data_ptr(), ld, feats.shape[0], feats.shape[1],
          _count(num_rows, feats.device), q.data_ptr(), pitch, scales.data_ptr())
    return q, scales


def _bytes(t, what):
    """(tensor, bytes between its rows) of a matrix of 8-bit integers."""
    if t.dim() != 2 or not t.is_cuda or t.dtype != torch.int8 or t.shape[1] == 0:
        raise ValueError("%s: an int8 CUDA tensor [rows, channels] is needed" % what)
    rows, channels = t.shape
    ld = t.stride(0) if rows > 1 else (channels + 15) // 16 * 16  # nothing lies behind a single row
    if (t.stride(1) != 1 and channels > 1) or ld < channels:
        t, ld = t.contiguous(), channels
    return t, ld


def int8_linear(feats, scales, weight, weight_scales, bias=None, dtype=torch.float16, num_rows=None, out=None):
    """scales[m] * weight_scales[n] * sum_k feats[m, k] weight[n, k] + bias[n] in `dtype` [rows, outputs].

    feats int8 [rows, inputs] and scales float32 [rows], as quantize_rows and layer_norm_int8 give them; weight int8 [outputs,
    inputs], weight_scales and bias (or None) float32 [outputs].  The sum is exact.  Rows and weights that start on 16 bytes
    and lie multiples of 16 bytes apart are read as they are, others are copied first, on every call.  At most 65536
    inputs and outputs."""
    feats, ld = _bytes(feats, "feats")
    weight, weight_ld = _bytes(weight, "weight")
    device, (rows, inputs), outputs = feats.device, feats.shape, weight.shape[0]
    if weight.shape[1] != inputs or weight.device != device or outputs == 0:
        raise ValueError("weight: [outputs, %d] on %s is needed" % (inputs, device))
    if dtype not in _FEATURES:
        raise TypeError("unsupported tensor dtype %s" % dtype)
    if scales is None or weight_scales is None:
        raise ValueError("scales of the rows and of the output channels are needed")
    s, ws, b = (_dense(t, (n,), torch.float32, device, what) for t, n, what in (
        (scales, rows, "scales"), (weight_scales, outputs, "weight_scales"), (bias, outputs, "bias")))
    if out is None:
        out = torch.empty((rows, outputs), dtype=dtype, device=device)
    _dense(out, (rows, outputs), dtype, device, "out")
    nbytes = _lib.lib().d3d_int8_linear_workspace(feats.data_ptr(), ld, rows, weight.data_ptr(), weight_ld, inputs, outputs)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _call("d3d_int8_linear", device, _TORCH2D3D[dtype], feats.data_ptr(), ld, s, rows, _count(num_rows, device), weight.data_ptr(),
          weight_ld, ws, b, inputs, outputs, out.data_ptr(), workspace.data_ptr() if nbytes else None, nbytes)
    return out


def _sequences(offsets, device):
    if offsets.dim() != 1 or offsets.shape[0] < 1 or offsets.dtype != torch.int32 or offsets.device != device:
        raise ValueError("seq_offsets: an int32 tensor [sequences + 1] on %s is needed" % device)
    return (offsets if offsets.is_contiguous() else offsets.contiguous()), offsets.shape[0] - 1


def gated_recurrence(feats, gates, seq_offsets, initial=None, reverse=False, with_states=False, out=None):
    """h[t] = f[t] h[t-1] + (1 - f[t]) feats[t] with f = sigmoid(gates), channel by channel along each sequence.

    seq_offsets int32 [sequences + 1] on the device, ascending: sequence s are the rows seq_offsets[s] .. seq_offsets[s+1]-1, walked
    downwards with `reverse`; equal ones are a sequence without rows.  initial float32 [sequences, channels]: h in front of the
    first row walked (None: zeros).  Rows outside all sequences are neither read nor written.  Returns (h in the type of
    feats, h of the last row walked of every sequence in float32); with `with_states` also what the backward pass needs."""
    feats, ld = _features(feats, "feats")
    gates, gates_ld = _features(gates, "gates", feats)
    (rows, channels), device = feats.shape, feats.device
    offsets, seqs = _sequences(seq_offsets, device)
    out = _made(out, feats)
    h0 = _dense(initial, (seqs, channels), torch.float32, device, "initial")
    final = torch.empty((seqs, channels), dtype=torch.float32, device=device)
    states = None
    if with_states:
        states = torch.empty((_lib.lib().d3d_gated_recurrence_state_rows(rows), channels), dtype=torch.float32, device=device)
    nbytes = _lib.lib().d3d_gated_recurrence_workspace(rows, channels)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _call("d3d_gated_recurrence", device, _TORCH2D3D[feats.dtype], feats.data_ptr(), ld, gates.data_ptr(), gates_ld,
          offsets.data_ptr(), seqs, rows, channels, int(bool(reverse)), h0, out.data_ptr(), final.data_ptr(),
          None if states is None else states.data_ptr(), workspace.data_ptr(), nbytes)
    return (out, final, states) if with_states else (out, final)


def gated_recurrence_backward(grad_out, feats, gates, seq_offsets, states, initial=None, grad_final=None, reverse=False):
    """Gradients (feats, gates, initial) of gated_recurrence for those of its rows and (None: zeros) of its last states;
    `states` as it returned them for the same arguments.  Rows outside all sequences are not written."""
    feats, ld = _features(feats, "feats")
    gates, gates_ld = _features(gates, "gates", feats)
    grad_out, grad_ld = _features(grad_out, "grad_out", feats)
    (rows, channels), device = feats.shape, feats.device
    offsets, seqs = _sequences(seq_offsets, device)
    lib = _lib.lib()
    if states is None:
        raise ValueError("states of the forward pass are needed")
    at = _dense(states, (lib.d3d_gated_recurrence_state_rows(rows), channels), torch.float32, device, "states")
    h0 = _dense(initial, (seqs, channels), torch.float32, device, "initial")
    dl = _dense(grad_final, (seqs, channels), torch.float32, device, "grad_final")
    grad_feats, grad_gates = (torch.empty(feats.shape, dtype=feats.dtype, device=device) for _ in range(2))
    grad_initial = torch.empty((seqs, channels), dtype=torch.float32, device=device)
    nbytes = lib.d3d_gated_recurrence_workspace(rows, channels)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _call("d3d_gated_recurrence_backward", device, _TORCH2D3D[feats.dtype], grad_out.data_ptr(), grad_ld, feats.data_ptr(), ld,
          gates.data_ptr(), gates_ld, offsets.data_ptr(), seqs, rows, channels, int(bool(reverse)), at, h0, dl,
          grad_feats.data_ptr(), grad_gates.data_ptr(), grad_initial.data_ptr(), workspace.data_ptr(), nbytes)
    return grad_feats, grad_gates, grad_initial


def gated_recurrence_step(feats, gates, state, state_out=None):
    """gated_recurrence for one new row of every sequence: (h in the type of feats, h in float32).  state float32 [rows,
    channels]; `state_out` takes the new one and may be `state`."""
    feats, ld = _features(feats, "feats")
    gates, gates_ld = _features(gates, "gates", feats)
    if state is None:
        raise ValueError("state: a float32 tensor [rows, channels] is needed")
    h = _dense(state, feats.shape, torch.float32, feats.device, "state")
    out = torch.empty(feats.shape, dtype=feats.dtype, device=feats.device)
    if state_out is None:
        state_out = torch.empty(feats.shape, dtype=torch.float32, device=feats.device)
    new = _dense(state_out, feats.shape, torch.float32, feats.device, "state_out")
    _call("d3d_gated_recurrence_step", feats.device, _TORCH2D3D[feats.dtype], feats.data_ptr(), ld, gates.data_ptr(), gates_ld,
          h, new, out.data_ptr(), feats.shape[0], feats.shape[1])
    return out, state_out

"""Operators of voxel-sequence networks, which mix voxels along an order instead of through a kernel neighbourhood: layer
norm, its rows in 8-bit integers, and a gated linear recurrence.  The reference has none of them.

Features are CUDA tensors ``[rows, channels]`` in float32, float16 or bfloat16 and may be columns of a wider tensor (their
channels side by side); parameters, scales and states are float32.  Everything runs on the current stream of the features'
device.  ``num_rows``, an int32 tensor of one element on the device, says how many rows are live, as the counts of the voxel
operators do: rows behind are not written, and what they hold does not matter (in a tensor the call has made itself they hold
nothing).  ``out`` takes the result where given: dense, of the right shape and type; it may be the (dense) features themselves.
Backward passes are functions of their own: nothing here records autograd history, also where features or parameters require
gradients.
"""
import torch

from .. import _host

_NATIVE = None


def _native():
    global _NATIVE
    if _NATIVE is None:
        _NATIVE = _host.sequence()
    return _NATIVE


def layer_norm(feats, weight, bias=None, eps=1e-5, residual=None, num_rows=None, with_stats=False, out=None):
    """(t - mean) * rstd * weight + bias over the channels of each row, t = feats or feats + residual; at most 8192 channels.

    weight, bias float32 [channels] (None: 1, 0).  Returns the normed rows; with `residual` also t, rounded to the type
    and normed as rounded; with `with_stats` also mean and rstd, float32 [rows], for layer_norm_backward."""
    return (_NATIVE or _native()).layer_norm(feats, weight, bias, eps, residual, num_rows, with_stats, out)


def layer_norm_backward(grad_out, feats, weight, mean, rstd, num_rows=None, grad_total=None):
    """Gradients (feats, weight, bias) of layer_norm.  `feats` is what was normed: with a residual the sum layer_norm returned,
    `grad_total` the gradient that sum gets elsewhere; the first result is then the gradient of both summands."""
    return (_NATIVE or _native()).layer_norm_backward(grad_out, feats, weight, mean, rstd, num_rows, grad_total)


def layer_norm_int8(feats, weight, bias=None, eps=1e-5, residual=None, num_rows=None):
    """layer_norm whose result leaves as quantize_rows would give it: (int8 rows, scales), with `residual` also the sum."""
    return (_NATIVE or _native()).layer_norm_int8(feats, weight, bias, eps, residual, num_rows)


def quantize_rows(feats, num_rows=None):
    """(int8 [rows, channels], float32 [rows]): scale = max |row| / 127, row / scale to the nearest integer, ties to even.  Rows
    of zeros, or of less than 127 times the smallest normal float, have scale 0, rows that are not finite zeros and scale NaN.  At most 8192 channels.  The rows lie a multiple of
    16 bytes apart."""
    return (_NATIVE or _native()).quantize_rows(feats, num_rows)


def int8_linear(feats, scales, weight, weight_scales, bias=None, dtype=torch.float16, num_rows=None, out=None):
    """scales[m] * weight_scales[n] * sum_k feats[m, k] weight[n, k] + bias[n] in `dtype` [rows, outputs].

    feats int8 [rows, inputs] and scales float32 [rows], as quantize_rows and layer_norm_int8 give them; weight int8 [outputs,
    inputs], weight_scales and bias (or None) float32 [outputs].  The sum is exact.  Rows and weights that start on 16 bytes
    and lie multiples of 16 bytes apart are read as they are; others, but for few rows, are copied first on every call: keep
    weights of odd widths as columns of a wider tensor.  At most 65536 inputs and outputs."""
    return (_NATIVE or _native()).int8_linear(feats, scales, weight, weight_scales, bias, dtype, num_rows, out)


def gated_recurrence(feats, gates, seq_offsets, initial=None, reverse=False, with_states=False, out=None):
    """h[t] = f[t] h[t-1] + (1 - f[t]) feats[t] with f = sigmoid(gates), channel by channel along each sequence.

    seq_offsets int32 [sequences + 1] on the device, ascending: sequence s are the rows seq_offsets[s] .. seq_offsets[s+1]-1, walked
    downwards with `reverse`; equal ones are a sequence without rows.  initial float32 [sequences, channels]: h in front of the
    first row walked (None: zeros).  Rows outside all sequences are not written, and what they hold does not matter.  An
    infinite h stays infinite to the end of its sequence; behind a gate whose f is zero in float32 or an infinite row against it,
    it may be NaN instead.  Returns (h in the type of feats, h of the last row walked of every sequence in float32); with `with_states` also what the
    backward pass needs."""
    return (_NATIVE or _native()).gated_recurrence(feats, gates, seq_offsets, initial, reverse, with_states, out)


def gated_recurrence_backward(grad_out, feats, gates, seq_offsets, states, initial=None, grad_final=None, reverse=False):
    """Gradients (feats, gates, initial) of gated_recurrence for those of its rows and (None: zeros) of its last states;
    `states` as it returned them for the same arguments.  Rows outside all sequences are not written."""
    return (_NATIVE or _native()).gated_recurrence_backward(
        grad_out, feats, gates, seq_offsets, states, initial, grad_final, reverse)


def gated_recurrence_step(feats, gates, state, state_out=None):
    """gated_recurrence for one new row of every sequence: (h in the type of feats, h in float32).  state float32 [rows,
    channels]; `state_out` takes the new one and may be `state`."""
    return (_NATIVE or _native()).gated_recurrence_step(feats, gates, state, state_out)

"""Operators on tokens -- rows of features: keypoint descriptors, cells of the descriptor map, entries of a sequence -- for the transformer blocks
that refine or match what the network extracts: layer norm (forward and backward), dropout + residual + layer norm in one pass, dropout from a
counter-based generator whose mask is never stored, rotary positions (sequences, or keypoints at (x, y)).  Kernels: csrc/token.hip,
csrc/norm.hip, csrc/norm_bwd.hip.  No reference counterpart: the reference's network is convolutional and its matcher is the mutual nearest
neighbour (models/model_wrap.py:434-476).

All of them: float16, bfloat16 or float32 tensors on the GPU, any leading dimensions, rows that may start on any element (slices of wider tensors are read
in place where their rows have one distance, else copied first); sums, statistics and angles in 32 bits or more, results rounded once;
launches on the current stream; differentiable once (a second differentiation raises).  CPU tensors, mixed devices, other types or shapes raise YpError,
and so do tensors without memory of their own (wrappers such as sharded parameters) and a call that is traced (torch.jit.trace, make_fx, fake tensors:
the recording would hold the buffers without the kernels).

A captured graph replays the kernels on the same addresses: `rng` as a device tensor lets every replay draw another mask.  A backward pass may be
captured with its forward pass; leaves that an eager graph still holds must not take part in it.
"""
import importlib.machinery
import importlib.util
import ctypes as C
import math
import operator
import os
import threading

import torch

from .. import _hip

_PATH = os.path.join(os.path.dirname(_hip.LIB_PATH), "_token_autograd.so")
_ENTRIES = ("yp_last_error", "yp_layer_norm_fwd", "yp_layer_norm_bwd", "yp_layer_norm_bwd_workspace_bytes", "yp_layer_norm_max_width", "yp_dropout", "yp_rotary")
_module = None
_lock = threading.Lock()


def _load():
    lib = _hip.lib()
    if not os.path.exists(_PATH):
        raise _hip.YpError(f"{_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
    loader = importlib.machinery.ExtensionFileLoader("_token_autograd", _PATH)
    m = importlib.util.module_from_spec(importlib.util.spec_from_loader("_token_autograd", loader))
    loader.exec_module(m)
    m.init([C.cast(getattr(lib, n), C.c_void_p).value for n in _ENTRIES], _hip.YpError)
    return m


def _native():
    """The C++ side (csrc/token_autograd.cpp: checks, buffers, launches, autograd nodes), over the entry points of the library that is loaded."""
    global _module
    if _module is None:
        with _lock:
            if _module is None:
                _module = _load()
    return _module


def _state(what, p, rng):
    """rng as (seed, offset, device tensor)"""
    if isinstance(rng, torch.Tensor):
        return 0, 0, rng
    if rng is None:
        if p != 0.0:
            raise _hip.YpError(f"{what}: p > 0 needs rng = (seed, offset)")
        return 0, 0, None
    try:
        seed, offset = rng
    except TypeError:
        raise _hip.YpError(f"{what}: rng = (seed, offset), not {type(rng).__name__}") from None
    except ValueError:
        raise _hip.YpError(f"{what}: rng is two numbers") from None
    return seed, offset, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x [..., D], 1 <= D <= 16384.

    weight, bias: [D] in float32 or x's type, or None.  Gradients: x, weight, bias (the sums over the rows in fp32 and in a fixed order: the same
    inputs give the same bits)."""
    try:
        return _native().layer_norm(x, weight, bias, eps)
    except TypeError as e:
        raise _hip.YpError(f"layer_norm: {e}") from None


def dropout_add_layer_norm(x, residual, weight=None, bias=None, p=0.0, rng=None, eps=1e-5):
    """z = residual + dropout(x), y = layer_norm(z) in one pass -> (y, z): what stands between two branches of a block.

    z is one fp32 multiply-add, rounded to the tensors' type, and y is the norm of that rounded z (what the backward pass reads): z equals
    `dropout(x, p, rng, residual=residual)` and y `layer_norm(z, ...)` bit for bit.  x, residual: one shape [..., D] and type; p, rng as in `dropout`;
    weight, bias, eps as in `layer_norm`.  Gradients: x, residual, weight, bias, from the gradients of both results."""
    seed, offset, state = _state("dropout_add_layer_norm", p, rng)
    try:
        return _native().dropout_add_layer_norm(x, residual, weight, bias, p, seed, offset, state, eps)
    except TypeError as e:
        raise _hip.YpError(f"dropout_add_layer_norm: {e}") from None


def dropout(x, p, rng, residual=None):
    """x with each element dropped (0, whatever it held) at rate p and the others multiplied by 1 / (1 - p); plus `residual` where given.

    The rate is applied in steps of 1 / 65536 (the factor belongs to the applied rate).  rng: (seed, offset), two numbers below 2^64, or an int64 device
    tensor [2] of them; the same pair gives the same mask, so every call of a program takes an offset of its own.  Element i (flat, row-major)
    is kept where half i % 8 of Philox4x32-10(counter (i / 8, offset), key seed) is >= round(65536 p): the mask does not depend on
    shape, type or strides, and the backward pass draws it again instead of reading it.  Gradients: x, residual.  A tensor `rng` must hold in the
    backward pass what it held in the forward pass (autograd refuses one that was written to in place)."""
    seed, offset, state = _state("dropout", p, rng)
    try:
        return _native().dropout(x, p, seed, offset, state, residual)
    except TypeError as e:
        raise _hip.YpError(f"dropout: {e}") from None


def rotary_frequencies(dim, base=10000.0, axes=1, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0, device=None):
    """The table `rotary` takes -> (inv_freq float64 [dim / 2], scale): inv_freq[j] = base^(-2 j / dim) radians a position, once over `dim / axes` features for
    each axis.  For contexts longer than the trained ones, stretched by `factor`:
      'linear'  positions divided by factor
      'ntk'     base * factor^(dim / (dim - 2)): the slowest pair is stretched by factor, the fastest stays
      'yarn'    pairs that turn more than `fast` times over `original` positions stay, those below `slow` turns are divided by factor, a linear
                ramp over the pairs between them (from the whole pair below the one border to the whole pair above the other, which may
                lie behind the last pair: the published method's `d - 1`, d = dim / axes); scale = 0.1 ln(factor) + 1"""
    try:
        dim, axes, base, factor = operator.index(dim), operator.index(axes), float(base), float(factor)
        original, fast, slow = None if original is None else float(original), float(fast), float(slow)
    except (TypeError, ValueError, OverflowError) as e:
        raise _hip.YpError(f"rotary_frequencies: {e}") from None
    if axes not in (1, 2) or dim < 2 * axes or dim % (2 * axes):
        raise _hip.YpError(f"rotary_frequencies: {dim} features over {axes} axes")
    if scaling not in (None, "linear", "ntk", "yarn") or not 1.0 <= factor < math.inf or (scaling is None and factor != 1.0):
        raise _hip.YpError(f"rotary_frequencies: scaling {scaling!r} by {factor}")
    d = dim // axes
    # (the largest table value and, for 'ntk', the stretched base have to be numbers)
    if not 0.0 < base < math.inf or abs(math.log(base)) + (math.log(factor) * 2.0 if scaling == "ntk" else 0.0) > 700.0:
        raise _hip.YpError(f"rotary_frequencies: base {base} (stretched by {factor})")
    if scaling == "ntk":
        if d < 4:
            raise _hip.YpError("rotary_frequencies: 'ntk' needs two pairs an axis")
        base = base * factor ** (d / (d - 2))
    f = [base ** (-2.0 * j / d) for j in range(d // 2)]
    scale = 1.0
    if scaling == "linear":
        f = [v / factor for v in f]
    elif scaling == "yarn":
        if original is None or not 0.0 < original < math.inf or not math.inf > fast > slow > 0.0 or not base > 1.0:
            raise _hip.YpError("rotary_frequencies: 'yarn' needs the original length, fast > slow > 0 and a base over 1")

        def pair_of(turns):                         # the (fractional) pair that makes this many turns over the original length
            return d * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        end = pair_of(slow)
        low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(end), d - 1)
        # (j > end: the first pair of a length that it does not turn over once stands on low = 0 and yet behind the ramp)
        ramp = [1.0 if j > end else min(max((j - low) / max(high - low, 1e-3), 0.0), 1.0) for j in range(d // 2)]
        f = [v * (1.0 - r) + v / factor * r for v, r in zip(f, ramp)]
        scale = 0.1 * math.log(factor) + 1.0
    return torch.tensor(f * axes, dtype=torch.float64, device=device), scale


def rotary(q, positions, inv_freq, k=None, interleaved=False, layout="bthd", scale=1.0, inplace=False):
    """q (and k, in the same launch) with the first 2 * len(inv_freq) features of every head turned by its token's position -> q' or (q', k').

    q, k: [B, T, H, D] ('bthd') or [B, H, T, D] ('bhtd'), dense features, any other strides (slices of a joint projection are read in place);
    their head numbers may differ.  Pairs: (j, j + R / 2), or (2 j, 2 j + 1) when interleaved, R = 2 * len(inv_freq) <= D <= 1024; the rest of a head is copied.
    positions: an int (token t stands at positions + t), or a tensor of int32, int64 or float32: [T], [1, T] or [B, T]; with a last dimension of 2
    ([T, 2], [B, T, 2], keypoints at (x, y)) the first half of the pairs turns by the first, the second half by the second.  A [B, 2] tensor is [B, T = 2].
    inv_freq, scale: from `rotary_frequencies`; the table is float64 on the tensors' device and has no gradient, angles are formed in 64 bits (positions of
    10^6 keep 1e-7 of a turn).
    inplace: write into q and k (no gradients; refused where an element would be turned twice: expanded tensors, q and k that meet).  Gradients: q, k
    (turned back)."""
    if layout not in ("bthd", "bhtd"):
        raise _hip.YpError(f"rotary: layout {layout!r}")
    start = 0
    if not isinstance(positions, torch.Tensor):
        if not isinstance(positions, int) or isinstance(positions, bool) or not -(1 << 62) < positions < 1 << 62:
            raise _hip.YpError("rotary: positions as an int or a tensor")
        start, positions = positions, None
    try:
        got = _native().rotary(q, k, positions, start, inv_freq, interleaved, layout == "bhtd", scale, inplace)
    except TypeError as e:
        raise _hip.YpError(f"rotary: {e}") from None
    return got[0] if k is None else got

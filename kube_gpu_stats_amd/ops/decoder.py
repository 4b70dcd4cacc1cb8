"""The decoder block's operators as gfx950 kernels, forward and backward
(``ops/hip/attention.hip``, ``swiglu.hip``, ``add_norm.hip``).

They are what a training step runs between its plain matrix products: softmax attention,
the gated half of the feed-forward block, and the norms around a residual connection.
With them the exporter is measured under a training step whose kernels are this
package's own, with known operations and bytes (``bench.py --load train --train-ops hip``);
they stand beside the synthetic kernels of ``ops/load.py``.

Each operator comes three times:

* ``attention``, ``swiglu``, ``add_norm`` — differentiable, for a program that uses autograd;
* ``*_fwd`` — the forward pass, returning what a backward pass needs;
* ``*_bwd`` — the gradients, for loops without autograd and for captured graphs.

All of them launch on the current stream of their tensors' device (or on ``stream=``),
allocate their results and workspaces from torch's allocator on that stream, never
synchronise and keep nothing between calls, so they can be captured into a graph.  With
``stream=`` the results may be used on the current stream once it has waited for that one.
Gradients are sums in a fixed order: equal calls give equal bits.  The autograd forms
differentiate once, backwards; an argument with a forward-mode tangent is refused.  To
capture a whole autograd step, let no eager graph of the same leaves be alive (torch's own
rule); the ``*_fwd`` / ``*_bwd`` pairs have no such rule.

There is deliberately no eager fallback: on a GPU the HIP library must load, or these
functions raise.  Wrong arguments raise ``ValueError`` or ``TypeError`` before anything
is launched.
"""
from __future__ import annotations

import ctypes
import functools
import os
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ..native import build as _build

_LIB: ctypes.CDLL | None = None


def lib() -> ctypes.CDLL:
    global _LIB
    if _LIB is None:
        path = _build.decoder_lib_path()
        if not os.path.exists(path):
            _build.build_decoder()
        L = ctypes.CDLL(path)
        L.kgs_decoder_last_error.restype = ctypes.c_char_p
        for name in ("attention", "swiglu", "add_norm"):
            for way in ("fwd", "bwd"):
                getattr(L, f"kgs_{name}_{way}").argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        _LIB = L
    return _LIB


# The C structures of ops/hip/decoder.h, field by field.
_ATTENTION = struct.Struct("@13P24q9if")
_SWIGLU = struct.Struct("@9P3q4i3i3i")
_ADD_NORM = struct.Struct("@16P5q4iP2f")


def _call(entry: str, args: bytes, index: int) -> None:
    # (the raw handle: a Stream object of torch.cuda.current_stream costs 2 us)
    if getattr(_LIB or lib(), entry)(args, torch._C._cuda_getCurrentRawStream(index)) != 0:
        raise RuntimeError(lib().kgs_decoder_last_error().decode())


def _here(t, stream) -> bool:
    """Whether ``t``'s device and the wanted stream are the current ones."""
    return stream is None and t.get_device() == torch.cuda.current_device()


def _there(t, stream, call, *tensors):
    """``call()`` with ``t``'s device and ``stream`` current: allocations and launches belong there.
    On a given stream the memory of the call's ``tensors`` is not handed out again before it is
    through, that of its results not before what the current stream does with them is."""
    now = None
    if stream is not None:
        if stream.device != t.device:
            raise ValueError(f"the stream is on {stream.device}, the tensors are on {t.device}")
        for x in (t, *tensors):
            if x is not None:
                x.record_stream(stream)
        now = torch.cuda.current_stream(t.device)
    with torch.cuda.device(t.device), torch.cuda.stream(stream):
        results = call()
    if now is not None and now != stream:
        for x in results:
            for y in x if isinstance(x, tuple) else (x,):
                if y is not None:
                    y.record_stream(now)
    return results


def _no_tangents(*tensors) -> None:
    """The kernels would drop a forward-mode tangent without a word."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise TypeError("the operators have no forward-mode derivative: an argument carries a tangent")


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _vector(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _type(t, name: str, allowed: str) -> int:
    code = _TYPES.get(t.dtype)
    if code is None or code >= (3 if "float32" in allowed else 2):
        raise TypeError(f"{name} must be {allowed}, not {t.dtype}")
    return code


def _same(first, name: str, **others) -> None:
    dtype, index = first.dtype, first.get_device()
    for other, t in others.items():
        if t is None:
            continue
        if t.dtype != dtype:
            raise TypeError(f"{other} is {t.dtype}, {name} is {dtype}")
        if t.get_device() != index:
            raise ValueError(f"{other} is on {t.device}, {name} is on {first.device}")


def _kept(t, name: str, dtype, shape, index: int, maker: str) -> None:
    """What a forward pass kept, come back as it was."""
    if t is None:
        raise TypeError(f"{name} must be the tensor that {maker} returned, not None")
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{name} must be the tensor that {maker} returned: {dtype}, {tuple(shape)}, contiguous, "
                         f"not {t.dtype}, {tuple(t.shape)} on {t.device}")


def _on_gpu(t, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU, not on {t.device}")


def _shape(t, name: str, want) -> None:
    if t.shape != want:
        raise ValueError(f"{name} must have shape {tuple(want)}, not {tuple(t.shape)}")


# --------------------------------------------------------------------------- attention

# Elements from one position to the next (offsets inside a tile of 128 fit 32 bits), and workgroups of 256
# threads (a launch has under 2^32).
MAX_ROW, MAX_PIECES = 1 << 22, (1 << 24) - 8


def _heads(t):
    """``t`` [B, S, heads, D] as the kernels read it, and its strides of (B, S, heads):
    D contiguous, positions apart, 16-byte rows.  Other layouts are copied."""
    B, S, H, D = t.shape
    if t.is_contiguous() and not t.data_ptr() % 16:
        return t, (S * H * D, H * D, D)
    b, s, h, d = t.stride()
    # A dimension of one may come with any stride; rows behind the last have to lie past it.
    st = (b if B > 1 else D, s if S > 1 else D, h if H > 1 else D)
    if d == 1 and D <= st[1] <= MAX_ROW and not (t.data_ptr() % 16 or (st[0] | st[1] | st[2]) % 8):
        return t, st
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()[:3]


def _attention_checks(q, k, v, scale, lengths, back=None):
    """(B, S, H, Hk, D, type, scale) of a call's tensors; ``back``: (dout, out, lse, low)."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        for t, name in ((q, "q"), (k, "k"), (v, "v")):
            if t.dim() != 4:
                raise ValueError(f"{name} must be [batch, positions, heads, head dimension], not {tuple(t.shape)}")
    B, S, H, D = q.shape
    Hk = k.shape[2]
    dtype, index, want = q.dtype, q.get_device(), (B, S, Hk, D)
    code = _type(q, "q", "bfloat16 or float16")
    if not (k.shape == want and v.shape == want and k.dtype == dtype and v.dtype == dtype and k.get_device() == index
            and v.get_device() == index):
        _same(q, "q", k=k, v=v)
        _shape(k, "k", want)
        _shape(v, "v", want)
    if back is not None:
        dout, out, lse, low = back
        _same(q, "q", dout=dout, out=out)
        _shape(dout, "dout", (B, S, H, D))
        _shape(out, "out", (B, S, H, D))
        _kept(lse, "lse", torch.float32, (B, H, S), index, "attention_fwd")
        _kept(low, "low", torch.uint8, (B, S, H, D), index, "attention_fwd")
    if D != 128 and D != 64:
        raise ValueError(f"the head dimension must be 64 or 128, not {D}")
    if H == 0 or Hk == 0 or H % Hk:
        raise ValueError(f"{H} query heads cannot share {Hk} key heads")
    if S >= 1 << 30:
        raise ValueError(f"at most {(1 << 30) - 1} positions, not {S}")
    if H * D > MAX_ROW:
        raise ValueError(f"at most {MAX_ROW} elements a position over all heads, not {H * D}")
    if B * H * -(-S // 128) > MAX_PIECES:
        raise ValueError(f"at most {MAX_PIECES} pieces of 128 positions over batch and heads, not {B * H * -(-S // 128)}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:  # a 32-bit number, times log2 e too
        raise ValueError(f"scale must be positive, from 2^-126 to 2^126, not {scale}")
    if lengths is not None:
        if lengths.dtype != torch.int32:
            raise TypeError(f"lengths must be int32, not {lengths.dtype}")
        _shape(lengths, "lengths", (B,))
        if lengths.get_device() != index:
            raise ValueError(f"lengths is on {lengths.device}, q is on {q.device}")
    _on_gpu(q, "q")
    return B, S, H, Hk, D, code, scale


def attention(q, k, v, *, causal: bool = True, scale: float | None = None, lengths=None):
    """softmax(scale · q kᵀ) v over each sequence's own tokens; differentiable in q, k, v.

    q [B, S, H, D], k and v [B, S, Hk, D] of bfloat16 or float16, D 64 or 128, H a multiple
    of Hk (each key head serves H / Hk query heads); any strides with D contiguous and
    16-byte aligned rows are read in place, so q, k and v may be views of one projection's
    output (other layouts are copied first).  ``causal``: position i sees positions up to i.
    ``scale``: D^-½ if None.  ``lengths`` [B] int32 on the GPU: sequence b is its first
    lengths[b] positions (clamped to 0..S); nothing behind them is read, the result and the
    gradients are zero there.  Returns [B, S, H, D], contiguous.  At most 2^22 elements a
    position (H·D), and 2^24 - 8 pieces of 128 positions over batch and heads.

    A position that is masked by ``causal`` alone is multiplied by a zero probability, as in
    a plain matrix product: its v must be finite.  A key whose score is -inf has a probability
    of zero (a row that sees no other: zeros).  Gradients need finite q, k, v and dout.
    """
    _no_tangents(q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, causal, scale, lengths)
    return _attention_fwd(q, k, v, causal, scale, lengths, None, False)[0]


def attention_qkv(qkv, heads: int, *, causal: bool = True, scale: float | None = None, lengths=None):
    """``attention`` of one projection's output [B, S, heads + 2 Hk, D], the query heads
    first, then the key heads, then the value heads; differentiable, with one gradient of
    the same layout (no gradients of views to be put together)."""
    q, k, v = _split_qkv(qkv, heads)
    _no_tangents(qkv)
    if torch.is_grad_enabled() and qkv.requires_grad:
        return _AttentionQkv.apply(qkv, heads, causal, scale, lengths)
    return _attention_fwd(q, k, v, causal, scale, lengths, None, False)[0]


def _split_qkv(qkv, heads: int):
    if qkv.dim() != 4 or heads <= 0 or qkv.shape[2] <= heads or (qkv.shape[2] - heads) % 2:
        raise ValueError(f"qkv must be [batch, positions, {heads} + 2 key heads, head dimension], "
                         f"not {tuple(qkv.shape)}")
    if qkv.shape[2] * qkv.shape[3] > MAX_ROW:
        raise ValueError(f"at most {MAX_ROW} elements a position, not {qkv.shape[2] * qkv.shape[3]}")
    kv = (qkv.shape[2] - heads) // 2
    return qkv[:, :, :heads], qkv[:, :, heads:heads + kv], qkv[:, :, heads + kv:]


def attention_fwd(q, k, v, *, causal: bool = True, scale: float | None = None, lengths=None, stream=None):
    """``attention`` without autograd: (out, saved), saved for ``attention_bwd``: (lse, low), lse
    [B, H, S] float32 the base-2 logarithm of each row's sum (-inf behind a sequence's end),
    low [B, S, H, D] uint8 what rounding took from out, a signed number of 256ths of its last place."""
    _no_tangents(q, k, v)
    return _attention_fwd(q, k, v, causal, scale, lengths, stream, True)


def _attention_fwd(q, k, v, causal, scale, lengths, stream, keep):
    B, S, H, Hk, D, code, scale = _attention_checks(q, k, v, scale, lengths)
    if not _here(q, stream):
        return _there(q, stream, lambda: _attention_fwd(q, k, v, causal, scale, lengths, None, keep), k, v, lengths)
    lengths = _vector(lengths)
    (q, qs), (k, ks), (v, vs) = _heads(q), _heads(k), _heads(v)
    out = q.new_empty((B, S, H, D))
    lse = low = None
    if keep:
        lse = torch.empty(B, H, S, dtype=torch.float32, device=q.device)
        low = torch.empty(B, S, H, D, dtype=torch.uint8, device=q.device)
    if B and S:
        _call("kgs_attention_fwd",
              _ATTENTION.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0, 0, 0, 0, _ptr(lse), 0, 0,
                              _ptr(low), _ptr(lengths), *qs, *ks, *vs, S * H * D, H * D, D, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                              0, 0, B, S, H, Hk, D, code, bool(causal), 1, 0, scale), q.get_device())
    return out, (lse, low) if keep else None


@functools.lru_cache(maxsize=4096)
def _dkv_splits(B: int, S: int, H: int, Hk: int, causal: bool, D: int = 128, padded: bool = False) -> int:
    """Parts that the walk over query rows is cut into for dk and dv (a workgroup has 128 keys
    and one key head): the count with the least expected time, in steps of 32 rows.

    A CU's workgroups take one step after the other, so the walks take their sum over 256
    CUs, plus, as they end unevenly, half of a part, but not less than one part (as long as
    all are, than the parts of one CU).  Half the steps are there if causal, half of a padded
    batch is expected.  Each part writes 32-bit sums that one more launch adds up: as long as
    D / 15 steps.  2048 parts are enough to even out, and bound the workspace.  (Backward of
    1 x 16384, 8 heads on 2, causal: 2906 us in one part, 1780 us in 4 to 8; 6 x 1021, 20
    heads on 4: 239 us in one, 172 us in 3, 198 us in 6; 1 x 1024, 32 heads: 72 us in one, 79 us
    in 2.)"""
    groups = B * Hk * -(-S // 128)
    steps = (H // Hk) * -(-S // 32)
    work = groups * steps / 256 / (2 if causal else 1) / (2 if padded else 1)

    def time(splits):
        part = -(-steps // splits)
        longest = part if causal or padded else part * -(-groups * splits // 256)
        return max(longest, work + part / 2) + (4 + D / 15 * groups * splits / 256 if splits > 1 else 0)

    return min(range(1, max(1, min(16, steps, 2048 // max(1, groups))) + 1), key=time)


def attention_bwd(dout, q, k, v, out, saved, *, causal: bool = True, scale: float | None = None, lengths=None,
                  stream=None):
    """(dq, dk, dv) of ``attention`` from the gradient of its result, with ``out`` and ``saved``
    of ``attention_fwd`` and the same keywords; the probabilities are computed again."""
    _no_tangents(dout, q, k, v, out)
    return _attention_bwd(dout, q, k, v, out, *saved, causal, scale, lengths, stream, None)


def _attention_bwd(dout, q, k, v, out, lse, low, causal, scale, lengths, stream, into):
    B, S, H, Hk, D, code, scale = _attention_checks(q, k, v, scale, lengths, (dout, out, lse, low))
    if not _here(q, stream):
        return _there(q, stream, lambda: _attention_bwd(dout, q, k, v, out, lse, low, causal, scale, lengths, None, into),
                      k, v, dout, out, lse, low, lengths)
    lengths = _vector(lengths)
    (q, qs), (k, ks), (v, vs), (out, os_), (dout, gs) = _heads(q), _heads(k), _heads(v), _heads(out), _heads(dout)
    if into is None:
        into = q.new_empty((B, S, H, D)), q.new_empty((B, S, Hk, D)), q.new_empty((B, S, Hk, D))
    splits = _dkv_splits(B, S, H, Hk, bool(causal), D, lengths is not None)
    # delta, for float16 the norms of v's and dout's rows, then the parts of a split walk
    parts = splits * 2 * B * S * Hk * D if splits > 1 else 0
    rows = B * H * -(-S // 32) * 64
    if code == 1:
        rows += -(-(B * Hk * -(-S // 128) + B * H * -(-S // 32)) // 4) * 4
    if B and S:
        work = torch.empty(rows + parts, dtype=torch.float32, device=q.device)
        at = work.data_ptr()
        _call("kgs_attention_bwd",
              _ATTENTION.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(),
                              *(t.data_ptr() for t in into), lse.data_ptr(), at, at + rows * 4 if parts else 0,
                              low.data_ptr(), _ptr(lengths), *qs, *ks, *vs, *os_, *gs, *into[0].stride()[:3],
                              *into[1].stride()[:3], *into[2].stride()[:3], B, S, H, Hk, D, code, bool(causal), splits,
                              0, scale), q.get_device())
    return tuple(into)


def attention_matrix_flops(B: int, S: int, H: int, D: int) -> tuple[int, int]:
    """(forward, backward) operations that the kernels give the matrix units for causal attention
    without lengths, of any key heads: nine products where the formula has seven, whole steps
    along the diagonal and at the end.  A counter of the matrix units is held against these."""
    forward = backward = 0  # products of 32 rows x 32 keys
    for row in range(0, -(-S // 128) * 128, 32):
        last = min(row + 32, S)  # keys that any row of the wave sees
        forward += 2 * 2 * -(-last // 64)
        backward += 3 * -(-last // 32) + (4 if last <= 64 else 0) + 4 * max(0, -(-S // 32) - row // 32)
    each = 2 * 32 * 32 * D * B * H
    return forward * each, backward * each


# ------------------------------------------------------------------------------ swiglu

def _matrix(t):
    """``t`` [..., n] as rows the kernels read, and their stride: rows contiguous, apart, 16-byte
    aligned.  Other layouts are copied."""
    n = t.shape[-1]
    m = t if t.dim() == 2 else t.reshape(-1, n)
    ld = m.stride(0) if m.shape[0] > 1 else n
    if m.stride(1) == 1 and n <= ld <= 1 << 21 and not (ld % 8 or m.data_ptr() % 16):
        return m, ld
    return m.clone(memory_format=torch.contiguous_format), n


def _swiglu_checks(x, w, dh=None, saved=None):
    if x.dim() < 1 or w.dim() != 2:
        raise ValueError(f"x must be [..., width] and w [2 inner, width], not {tuple(x.shape)} and {tuple(w.shape)}")
    K, F = x.shape[-1], w.shape[0] // 2
    code, index = _type(x, "x", "bfloat16 or float16"), x.get_device()
    if w.dtype != x.dtype or w.get_device() != index or w.shape != (2 * F, K):
        _same(x, "x", w=w)
        _shape(w, "w", (2 * F, K))
    if K == 0 or F == 0 or K % 8 or F % 8 or K > 1 << 20 or F > 1 << 20:
        raise ValueError(f"width and inner must be multiples of 8, at most {1 << 20}, not {K} and {F}")
    if dh is not None:
        lead = x.shape[:-1]
        _same(x, "x", dh=dh)
        _shape(dh, "dh", (*lead, F))
        _kept(saved, "saved", torch.uint8, (*lead, 6 * F), index, "swiglu_fwd")
    T = x.numel() // K
    if T >= 1 << 30:
        raise ValueError(f"at most {(1 << 30) - 1} rows, not {T}")
    rows, inner, width = -(-T // 256), -(-2 * F // 256), -(-K // 256)
    if max(rows * inner, rows * width, inner * width) > MAX_TILES:
        raise ValueError(f"a product of {T} rows, width {K} and inner {F} has more than {MAX_TILES} tiles of 256 x 256")
    _on_gpu(x, "x")
    return T, K, F, code


# The tiles of swiglu.hip's product, rows by columns: 128 x 128, 256 x 256, and for the
# forward pass of up to 32 rows 32 x 256.
PRODUCT_TILES = (0, 1, 2)
MAX_TILES = (1 << 23) - 8  # of 256 x 256, the largest: 512 threads each, a launch has under 2^32


@functools.lru_cache(maxsize=4096)
def _product_plan(M: int, N: int, K: int, forward: bool = False) -> tuple[int, int]:
    """(tile, splits) of an [M, N] product over K: the least of the times expected, from what
    the tiles were measured at.  A step of 64 of the sum takes all workgroups that run at
    once 1.83 us with the 256 x 256 tile (one a CU), 1.10 us with 128 x 128 (two a CU; 0.74
    us if there is no more than one); with 32 x 256 it is the time of reading the weights,
    5.2 TB/s.  A round of workgroups has a start and an end of its own; the parts of a
    split sum are written and read as 32-bit numbers, at 4 TB/s, by one more launch; no
    plan is faster than reading and writing the operands once.  (2048 x 10752 over 2048:
    110 us with 256 x 256, two rounds of which the second is a third full, and 95 us with
    128 x 128; 8192 x 22016 over 4096: 1230 us and 1430 us; 5 x 22016 over 4096, weights
    from memory: 38 us with 32 x 256 in 4 parts, 54 us with 128 x 128 in 3.)"""
    floor = 2 * (M * K + N * K + M * N) / 5.2e6
    best = None
    for tile, rows, columns, at_once, around, most in ((0, 128, 128, 512, 3.5, 2 * MAX_TILES), (1, 256, 256, 256, 8.0, MAX_TILES),
                                                       (2, 32, 256, 512, 3.5, 2 * MAX_TILES)):
        if tile == 2 and not (forward and M <= 32):
            continue
        blocks = -(-M // rows) * -(-N // columns)
        for splits in (1, 2, 3, 4, 5, 6, 8, 10, 12, 16):
            steps = -(-K // 64 // splits)
            if splits > 1 and steps < 4 or blocks * splits > most:
                break
            step = (1.10 if blocks * splits > 256 else 0.74, 1.83, 1.5)[tile]
            # a step's columns come from memory once, however many row tiles share them
            step = max(step, min(blocks * splits, at_once) / -(-M // rows) * columns * 128 / 5.2e6)
            time = max(floor, -(-blocks * splits // at_once) * (steps * step + around))
            if splits > 1:
                time += 4 + 2 * splits * M * N * 4 / 4e6
            if best is None or time < best[0]:
                best = time, tile, splits
    return best[1:]


def swiglu(x, w):
    """silu(x Wgᵀ) · (x Wuᵀ) with w = [Wg; Wu]; differentiable in x and w.

    x [..., width], w [2 inner, width] (the gate's rows first) of bfloat16 or float16, width
    and inner multiples of 8; any row strides with contiguous, 16-byte aligned rows are read
    in place.  Returns [..., inner].  At most 2^20 of width and of inner, 2^30 - 1 rows and
    2^23 - 8 tiles of 256 x 256 in a product.  With a gradient wanted the two projections are
    kept for the backward pass, 24 bits of each value.  Its two products take the projections'
    gradients (silu(g) dh and its like) in the tensors' type: in float16 they have to lie in
    its range, like any gradient between two layers.
    """
    _no_tangents(x, w)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _Swiglu.apply(x, w)
    return _swiglu_fwd(x, w, None, False)[0]


def swiglu_fwd(x, w, *, stream=None):
    """``swiglu`` without autograd: (h, saved), saved [..., 6 inner] uint8 for ``swiglu_bwd``: of
    each row the upper 16 bits of the two projections, then the 8 bits below."""
    _no_tangents(x, w)
    return _swiglu_fwd(x, w, stream, True)


def _swiglu_fwd(x, w, stream, keep):
    T, K, F, code = _swiglu_checks(x, w)
    if not _here(x, stream):
        return _there(x, stream, lambda: _swiglu_fwd(x, w, None, keep), w)
    lead = x.shape[:-1]
    h = x.new_empty((*lead, F))
    saved = torch.empty((*lead, 6 * F), dtype=torch.uint8, device=x.device) if keep else None
    if T:
        (x, x_ld), (w, w_ld) = _matrix(x), _matrix(w)
        tile, splits = _product_plan(T, 2 * F, K, True)
        part = torch.empty(splits * T * 2 * F, dtype=torch.float32, device=x.device) if splits > 1 else None
        _call("kgs_swiglu_fwd",
              _SWIGLU.pack(x.data_ptr(), w.data_ptr(), h.data_ptr(), _ptr(saved), 0, 0, 0, 0, _ptr(part), x_ld, w_ld, 0,
                           T, K, F, code, tile, 0, 0, splits, 1, 1), x.get_device())
    return h, saved


def swiglu_bwd(dh, x, w, saved, *, stream=None):
    """(dx, dw) of ``swiglu`` from the gradient of its result and what ``swiglu_fwd`` saved."""
    _no_tangents(dh, x, w)
    return _swiglu_bwd(dh, x, w, saved, True, True, stream)


def _swiglu_bwd(dh, x, w, saved, want_dx, want_dw, stream):
    T, K, F, code = _swiglu_checks(x, w, dh, saved)
    if not _here(x, stream):
        return _there(x, stream, lambda: _swiglu_bwd(dh, x, w, saved, want_dx, want_dw, None), w, dh, saved)
    dx = x.new_empty(x.shape) if want_dx else None
    dw = (w.new_empty if T else w.new_zeros)(w.shape) if want_dw else None
    if T and (want_dx or want_dw):
        (x, x_ld), (w, w_ld), (dh, dh_ld) = _matrix(x), _matrix(w), _matrix(dh)
        if saved.data_ptr() % 16:
            saved = saved.clone()
        tx, sx = _product_plan(T, K, 2 * F) if want_dx else (0, 1)
        tw, sw = _product_plan(2 * F, K, T) if want_dw else (0, 1)
        # one workspace for the parts: the products follow one another on the stream
        size = max(sx * T * K if sx > 1 else 0, sw * 2 * F * K if sw > 1 else 0)
        part = torch.empty(size, dtype=torch.float32, device=x.device) if size else None
        dgu = x.new_empty((T, 2 * F))
        _call("kgs_swiglu_bwd",
              _SWIGLU.pack(x.data_ptr(), w.data_ptr(), 0, saved.data_ptr(), dh.data_ptr(), dgu.data_ptr(), _ptr(dx),
                           _ptr(dw), _ptr(part), x_ld, w_ld, dh_ld, T, K, F, code, 0, tx, tw, 1, sx, sw), x.get_device())
    return dx, dw


def swiglu_matrix_flops(T: int, K: int, F: int) -> tuple[int, int]:
    """(forward, backward) operations that the kernels give the matrix units: whole tiles, the
    sum in steps of 64."""
    def product(M, N, K, forward):
        rows, columns = ((128, 128), (256, 256), (32, 256))[_product_plan(M, N, K, forward)[0]]
        halves = 2 if forward else 1  # a forward tile has as many columns of either projection
        blocks = -(-M // rows) * -(-(N // halves) // (columns // halves))
        return 2 * blocks * rows * columns * -(-K // 64) * 64
    if T == 0:
        return 0, 0
    return product(T, 2 * F, K, True), product(T, K, 2 * F, False) + product(2 * F, K, T, False)


# ---------------------------------------------------------------------------- add_norm

MAX_NORM_WIDTH = 16384
LARGEST = torch.finfo(torch.float32).max


def _lines(t):
    """``t`` [..., C] as rows and their stride; rows that are not contiguous are copied."""
    m = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if m.stride(1) != 1 and m.shape[1] > 1:
        m = m.clone(memory_format=torch.contiguous_format)
    return m, m.stride(0)


def _add_norm_checks(residual, branch, weight, post_weight, gate, scale, eps, back=None):
    """(rows, width, type, scale) of a call's tensors; ``back``: (dstream, dout, saved).  The scale is
    rounded to the kernels' 32 bits here: whether it is 1 is asked on both sides."""
    if residual.dim() < 1:
        raise ValueError("residual must be [..., width], not a single value")
    shape, dtype, index = residual.shape, residual.dtype, residual.get_device()
    C = shape[-1]
    code, vector = _type(residual, "residual", "bfloat16, float16 or float32"), (C,)
    if not (branch.shape == shape and branch.dtype == dtype and branch.get_device() == index and weight.shape == vector
            and weight.dtype == dtype and weight.get_device() == index):
        _shape(branch, "branch", shape)
        _shape(weight, "weight", vector)
        _same(residual, "residual", branch=branch, weight=weight)
    for name, t in (("post_weight", post_weight), ("gate", gate)):
        if t is not None and (t.shape != vector or t.dtype != dtype or t.get_device() != index):
            _shape(t, name, vector)
            _same(residual, "residual", **{name: t})
    if not 0 < C <= MAX_NORM_WIDTH:
        raise ValueError(f"the width must be 1 to {MAX_NORM_WIDTH}, not {C}")
    T = residual.numel() // C
    if T >= 1 << 30:
        raise ValueError(f"at most {(1 << 30) - 1} rows, not {T}")
    if not -LARGEST <= scale <= LARGEST:
        raise ValueError(f"scale must be a finite 32-bit number, not {scale}")
    if not 0 <= eps <= LARGEST:
        raise ValueError(f"eps must be a finite 32-bit number and not negative, not {eps}")
    if back is not None:
        for name, t in zip(("dstream", "dout"), back):
            if t is not None:
                _shape(t, name, shape)
                _same(residual, "residual", **{name: t})
        _kept(back[2], "saved", torch.float32, (2, T), index, "add_norm_fwd")
    _on_gpu(residual, "residual")
    return T, C, code, ctypes.c_float(scale).value


def add_norm(residual, branch, weight, *, post_weight=None, gate=None, scale: float = 1.0, eps: float = 1e-6):
    """(stream, out): stream = residual + scale · gate · norm(branch), out = norm(stream).

    The step between two halves of a decoder block: ``branch`` (a half's result) is
    normalised by its root mean square and multiplied by ``post_weight`` (left as it is if
    None), multiplied by ``gate`` (ones if None) and ``scale``, and added to the residual
    stream, which is then normalised with ``weight`` for the next half.  residual, branch
    [..., C], weight, post_weight, gate [C], all of one type (bfloat16, float16, float32),
    C up to 16384, of any row stride.  Differentiable in all five tensors.
    """
    _no_tangents(residual, branch, weight, post_weight, gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (residual, branch, weight, post_weight, gate)):
        return _AddNorm.apply(residual, branch, weight, post_weight, gate, scale, eps)
    return _add_norm_fwd(residual, branch, weight, post_weight, gate, scale, eps, None, False)[:2]


def add_norm_fwd(residual, branch, weight, *, post_weight=None, gate=None, scale: float = 1.0, eps: float = 1e-6,
                 stream=None):
    """``add_norm`` without autograd: (stream, out, saved), saved for ``add_norm_bwd``: [2, rows]
    float32, the factors of the two norms, in the stream's memory and with it 8 more bits of
    each of a 16-bit stream's elements."""
    _no_tangents(residual, branch, weight, post_weight, gate)
    return _add_norm_fwd(residual, branch, weight, post_weight, gate, scale, eps, stream, True, True)


def _norm_room(T: int, C: int, size: int) -> tuple[int, int, int]:
    """Where saved and the low bytes begin behind a stream of T x C elements of ``size`` bytes, and the end."""
    saved = -(-T * C * size // 16) * 16
    low = saved + 8 * T
    return saved, low, low + (T * C if size == 2 else 0)


def _from_stream(x, saved, T: int, C: int) -> bool:
    """Whether ``x`` is the stream in whose memory ``saved`` is."""
    store = saved.untyped_storage()
    base = store.data_ptr()
    if x.untyped_storage().data_ptr() != base:
        return False
    at, _, end = _norm_room(T, C, x.element_size())
    if store.nbytes() != end or saved.data_ptr() != base + at:
        return False  # a program's own memory, in which it keeps both
    if x.data_ptr() != base or not x.is_contiguous():
        raise ValueError("the stream must come as add_norm_fwd returned it, its rows in their order")
    return True


def _add_norm_fwd(residual, branch, weight, post_weight, gate, scale, eps, stream, keep, together=False):
    T, C, code, scale = _add_norm_checks(residual, branch, weight, post_weight, gate, scale, eps)
    if not _here(residual, stream):
        return _there(residual, stream,
                      lambda: _add_norm_fwd(residual, branch, weight, post_weight, gate, scale, eps, None, keep, together),
                      branch, weight, post_weight, gate)
    out, low = residual.new_empty(residual.shape), 0
    if together and T:
        # (set_: tensors of one memory, not views of one another, whose versions autograd would count together)
        at, low, end = _norm_room(T, C, residual.element_size())
        room = torch.empty(end, dtype=torch.uint8, device=residual.device)
        store = room.untyped_storage()
        s = residual.new_empty(0).set_(store, 0, residual.shape)
        saved = torch.empty(0, dtype=torch.float32, device=residual.device).set_(store, at // 4, (2, T))
        low = room.data_ptr() + low if low < end else 0
    else:
        s = residual.new_empty(residual.shape)
        saved = torch.empty(2, T, dtype=torch.float32, device=residual.device) if keep else None
    if T:
        (r, r_ld), (b, b_ld) = _lines(residual), _lines(branch)
        w, pw, g = _vector(weight), _vector(post_weight), _vector(gate)
        _call("kgs_add_norm_fwd",
              _ADD_NORM.pack(r.data_ptr(), b.data_ptr(), w.data_ptr(), _ptr(pw), _ptr(g), s.data_ptr(), out.data_ptr(),
                             _ptr(saved), 0, 0, 0, 0, 0, 0, 0, 0, r_ld, b_ld, C, 0, 0, T, C, code, 0, low, scale, eps),
              r.get_device())
    return s, out, saved


@functools.lru_cache(maxsize=4096)
def _norm_parts(T: int, C: int) -> int:
    """Workgroups of the backward, each of which leaves a part of the column sums: as many as
    run at once, 16 waves a CU.  Rows up to 512 wide share a workgroup of four waves, a
    power of two of lanes with 8 elements each to a row.  Up to 8 turns are one workgroup's:
    it writes the sums itself, which saves a launch (7 x 517, all weights: a call of 18.8 us
    became one of 14.1 us)."""
    if C <= 512:
        lanes = 1 << (-(-C // 8) - 1).bit_length()
        turns, most = -(-T // (256 // lanes)), 1024
    else:
        turns, most = T, 256 * (16 // (-(-C // 512) if C <= 8192 else -(-C // 1024)))
    return 1 if turns <= 8 else min(turns, most)


def add_norm_bwd(dstream, dout, residual, branch, weight, saved, *, post_weight=None, gate=None, scale: float = 1.0,
                 eps: float = 1e-6, stream=None):
    """(dresidual, dbranch, dweight, dpost_weight, dgate) of ``add_norm`` from the gradients of
    its two results (either may be None: zero), its arguments, and ``saved`` of ``add_norm_fwd``.

    In the residual's place the stream that ``add_norm_fwd`` returned with ``saved`` does as
    well: then the residual need not be kept, and without post_weight, gate and scale the
    branch is not read either.  It has to be that tensor, or one of its memory and order, with
    that ``saved``: they lie in one memory, by which it is known, and where either is a copy
    the stream is taken for a residual.

    Without post_weight, gate and scale dbranch is dresidual, the same tensor; gradients of
    absent weights are None."""
    if dstream is None and dout is None:
        raise ValueError("one of dstream and dout must be given")
    _no_tangents(dstream, dout, residual, branch, weight, post_weight, gate)
    T, C, code, scale = _add_norm_checks(residual, branch, weight, post_weight, gate, scale, eps, (dstream, dout, saved))
    if not _here(residual, stream):
        return _there(residual, stream,
                      lambda: add_norm_bwd(dstream, dout, residual, branch, weight, saved, post_weight=post_weight,
                                           gate=gate, scale=scale, eps=eps),
                      dstream, dout, branch, weight, saved, post_weight, gate)
    dr = residual.new_empty(residual.shape)
    db = residual.new_empty(residual.shape) if post_weight is not None or gate is not None or scale != 1.0 else dr
    new = weight.new_empty if T else weight.new_zeros
    dw, dpw, dg = new((C,)), new((C,)) if post_weight is not None else None, new((C,)) if gate is not None else None
    if T:
        (r, r_ld), (b, b_ld), s, s_ld, low = _lines(residual), _lines(branch), None, 0, 0
        if _from_stream(residual, saved, T, C):
            s, s_ld, r = residual, C, None
            low = s.data_ptr() + _norm_room(T, C, s.element_size())[1] if code < 2 else 0
        ds, ds_ld = _lines(dstream) if dstream is not None else (None, 0)
        dy, dy_ld = _lines(dout) if dout is not None else (None, 0)
        w, pw, g = _vector(weight), _vector(post_weight), _vector(gate)
        parts = _norm_parts(T, C)
        work = torch.empty(parts * 2 * C, dtype=torch.float32, device=residual.device)
        _call("kgs_add_norm_bwd",
              _ADD_NORM.pack(_ptr(r), b.data_ptr(), w.data_ptr(), _ptr(pw), _ptr(g), _ptr(s), 0, saved.data_ptr(),
                             _ptr(ds), _ptr(dy), dr.data_ptr(), db.data_ptr(), dw.data_ptr(), _ptr(dpw), _ptr(dg),
                             work.data_ptr(), r_ld, b_ld, s_ld, ds_ld, dy_ld, T, C, code, parts, low, scale, eps),
              residual.get_device())
    return dr, db, dw, dpw, dg


# ---------------------------------------------------------------------------- autograd

class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, scale, lengths):
        out, saved = _attention_fwd(q, k, v, causal, scale, lengths, None, True)
        ctx.save_for_backward(q, k, v, out, *saved, lengths)
        ctx.options = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, low, lengths = ctx.saved_tensors
        grads = _attention_bwd(dout, q, k, v, out, lse, low, *ctx.options, lengths, None, None)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


class _AttentionQkv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, heads, causal, scale, lengths):
        out, saved = _attention_fwd(*_split_qkv(qkv, heads), causal, scale, lengths, None, True)
        ctx.save_for_backward(qkv, out, *saved, lengths)
        ctx.options = heads, causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, out, lse, low, lengths = ctx.saved_tensors
        heads, causal, scale = ctx.options
        grad = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        _attention_bwd(dout, *_split_qkv(qkv, heads), out, lse, low, causal, scale, lengths, None,
                       _split_qkv(grad, heads))
        return grad, None, None, None, None


class _Swiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        h, saved = _swiglu_fwd(x, w, None, True)
        ctx.save_for_backward(x, w, saved)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        return _swiglu_bwd(dh, *ctx.saved_tensors, *ctx.needs_input_grad, None)


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, weight, post_weight, gate, scale, eps):
        stream, out, saved = _add_norm_fwd(residual, branch, weight, post_weight, gate, scale, eps, None, True)
        ctx.save_for_backward(residual, branch, weight, saved, post_weight, gate)
        ctx.options = scale, eps
        ctx.set_materialize_grads(False)
        return stream, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dstream, dout):
        if dstream is None and dout is None:
            return (None,) * 7
        residual, branch, weight, saved, post_weight, gate = ctx.saved_tensors
        grads = add_norm_bwd(dstream, dout, residual, branch, weight, saved, post_weight=post_weight, gate=gate,
                             scale=ctx.options[0], eps=ctx.options[1])
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None)

"""Causal depth-wise convolution and selective state-space scan: prompts, their gradients, and one token at a time.

    causal_conv(x, weight, bias)                        [B, L, D]     y[t] = silu(bias + sum_k weight[:, k] x[t - K + 1 + k])
    selective_scan(x, dt, A, B, C, D)                   [B, L, H, P]  S[t] = exp(d[t] A) S[t-1] + d[t] x[t] B[t]^T,  y[t] = S[t] C[t] + D x[t]
    causal_conv_step / selective_scan_step              one token of every row, the state updated in place

The uni-directional counterpart of the framework's SRU layers: `return_state=True` hands back what the next call (`state=`) or the single-token form goes on
from, `lengths` (int32 [B], on the device) makes the batch a padded one - behind a row's length outputs and gradients are zero, inputs are not read and the state
stays.  fp32 or bf16 (`x`, `B`, `C`; `dt` may be fp32 next to bf16); parameters and the scan's state are fp32.  Everything is channels-last; `x`, `dt`, `B` and `C`
may be slices of wider tensors (the values of a token contiguous, rows and tokens at any pitch).  HIP kernels in csrc/ssm_*.hip, on torch's current stream; no
workspace outlives a call, so captured graphs share none.  A backward pass may be captured too, but (as with every autograd function) not while an eager graph that
holds the same leaves lives: torch ends the process.  A value that is not finite reaches the outputs that depend on it, from its token on (an infinity may
arrive as a NaN), and may reach every gradient of its row.
CUDA tensors only: no CPU fallback."""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import lib

__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1}
_FP32 = (torch.float32,)


def _raw(t):
    """a tensor that need not be contiguous, for lib.call: its address (its pitches travel next to it)"""
    return t if t is None or t.is_contiguous() else ctypes.c_void_p(t.data_ptr())


def _check(name, what, t, shape, dtypes, device):
    if isinstance(t, torch.Tensor) and t.shape == shape and t.dtype in dtypes and t.device == device:
        return  # a single token's call is host time: one look when all is well
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: {what} must be a tensor, got {type(t).__name__}")
    if t.shape != shape:
        raise ValueError(f"{name}: {what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: {what} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")
    raise ValueError(f"{name}: {what} is on {t.device}, x on {device}")


def _first(name, x, dims):
    """x's own checks: everything else is held against it"""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: x must be a tensor, got {type(x).__name__}")
    if x.dim() != dims:
        raise ValueError(f"{name}: x must have {dims} dimensions, got shape {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise ValueError(f"{name}: x must be float32 or bfloat16, got {str(x.dtype)[6:]}")


def _on_gpu(name, x):
    """the last check: the ones before it need no device"""
    if not x.is_cuda:
        raise RuntimeError(f"rtfs_net_amd.ssm.{name} runs on an MI355X HIP device only (no CPU fallback)")


def _tokens(t, dims):
    """t with its last `dims` dimensions contiguous, and its row and token pitches in elements (of [B, L, ...]); tokens further apart than the kernels' 32-bit
    offsets allow are copied together.  One token has no pitch: whatever stride torch keeps for it (a time-first tensor's is the whole batch), a dense one's is given."""
    size, one = 1, t.shape[1] == 1
    if t.stride(1) >= 1 << 23 and not one:
        t = t.contiguous()
    for n, s in zip(t.shape[:-dims - 1:-1], t.stride()[:-dims - 1:-1]):
        if n != 1 and s != size:
            t = t.contiguous()
            break
        size *= n
    return t, t.stride(0), math.prod(t.shape[-dims:]) if one else t.stride(1)


def _rows(t):
    """one token per row: t with the values of a row contiguous"""
    return t if t.is_contiguous() or t[0].is_contiguous() else t.contiguous()


def _lengths(name, lengths, B, device):
    if lengths is not None:
        _check(name, "lengths", lengths, (B,), (torch.int32,), device)
        lengths = lengths.contiguous()
    return lengths


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _through(t, shape, dtype, device):
    """what comes out of a call without tokens where `t` went in (None: zeros)"""
    return t.clone() if t is not None else torch.zeros(shape, dtype=dtype, device=device)


# ---- convolution ---------------------------------------------------------------------------------------------------------------------------------------


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, want_state):
        B, L, D = x.shape
        K = weight.shape[1]
        x, row, tok = _tokens(x, 1)
        weight, bias, state = _dense(weight), _dense(bias), _dense(state)
        y = torch.empty(B, L, D, dtype=x.dtype, device=x.device)
        if y.numel():
            last = torch.empty(B, K - 1, D, dtype=x.dtype, device=x.device) if want_state else None
            lib.call("rtfs_causal_conv_fwd", _raw(x), row, tok, weight, bias, state, lengths, y, last, B, L, D, K, int(silu), _TYPES[x.dtype])
        else:  # no token: nothing to launch, the state goes through
            last = _through(state, (B, K - 1, D), x.dtype, x.device) if want_state else None
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths = ctx.saved_tensors
        B, L, D = x.shape
        K = weight.shape[1]
        x, row, tok = _tokens(x, 1)
        dy = torch.zeros(B, L, D, dtype=x.dtype, device=x.device) if dy is None else dy.contiguous()
        dx = torch.empty(B, L, D, dtype=x.dtype, device=x.device)
        dw = torch.empty_like(weight)
        db = torch.empty_like(bias) if bias is not None else None
        ds = torch.empty_like(state) if state is not None else None
        if not x.numel():
            ds = _through(dlast, ds.shape, x.dtype, x.device) if state is not None else None
            return dx, dw.zero_(), db.zero_() if db is not None else None, ds, None, None, None
        kind = _TYPES[x.dtype]
        work = torch.empty(lib.load().rtfs_causal_conv_bwd_work_floats(D, K, kind), device=x.device)
        lib.call("rtfs_causal_conv_bwd", _raw(x), row, tok, weight, bias, state, lengths, dy, _dense(dlast), dx, ds, dw, db, work, B, L, D, K, int(ctx.silu), kind)
        return dx, dw, db, ds, None, None, None


def _conv_parameters(name, x, weight, bias, D):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 1 <= weight.shape[1] <= 8:
        raise ValueError(f"{name}: weight must be a [D, K] tensor with 1 <= K <= 8")
    if D > 1 << 24:
        raise ValueError(f"{name}: more than {1 << 24} channels")
    _check(name, "weight", weight, (D, weight.shape[1]), (torch.float32,), x.device)
    if bias is not None:
        _check(name, "bias", bias, (D,), (torch.float32,), x.device)
    return weight.shape[1]


def causal_conv(x, weight, bias=None, *, silu=True, state=None, lengths=None, return_state=False):
    """Causal depth-wise convolution over time, `silu` of it unless told otherwise.

    x [B, L, D] fp32 or bf16; weight [D, K], K <= 8, bias [D], fp32; state [B, K-1, D] of x's type: the inputs before token 0 (None: zeros); lengths int32 [B].
    -> y [B, L, D], or (y, last) with `return_state`: last [B, K-1, D], the inputs before each row's end.  Differentiable in x, weight, bias and state."""
    _first("causal_conv", x, 3)
    B, L, D = x.shape
    K = _conv_parameters("causal_conv", x, weight, bias, D)
    if state is not None:
        _check("causal_conv", "state", state, (B, K - 1, D), (x.dtype,), x.device)
    lengths = _lengths("causal_conv", lengths, B, x.device)
    _on_gpu("causal_conv", x)
    y, last = _CausalConv.apply(x, weight, bias, state, lengths, bool(silu), bool(return_state))
    return (y, last) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, silu=True):
    """One token of every row: x [B, D], state [B, K-1, D] (contiguous, x's type) moves on by it in place -> y [B, D].  For serving: no gradient."""
    _first("causal_conv_step", x, 2)
    B, D = x.shape
    K = _conv_parameters("causal_conv_step", x, weight, bias, D)
    _check("causal_conv_step", "state", state, (B, K - 1, D), (x.dtype,), x.device)
    if not state.is_contiguous():
        raise ValueError("causal_conv_step: state is updated in place and must be contiguous")
    _no_gradient("causal_conv_step", x, state, weight, bias)
    _on_gpu("causal_conv_step", x)
    y = torch.empty(B, D, dtype=x.dtype, device=x.device)
    if B and D:
        x = _rows(x)
        lib.call("rtfs_causal_conv_step", _raw(x), x.stride(0), state, _dense(weight), _dense(bias), y, B, D, K, int(bool(silu)), _TYPES[x.dtype])
        torch.autograd.graph.increment_version(state)  # written through its address
    return y


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or the form for sequences")


# ---- scan ----------------------------------------------------------------------------------------------------------------------------------------------


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, Bm, C, D, dt_bias, state, lengths, softplus, want_state):
        B, L, H, P = x.shape
        G, N = Bm.shape[2:]
        A, D, dt_bias, state = _dense(A), _dense(D), _dense(dt_bias), _dense(state)
        (x, xr, xt), (dt, tr, tt), (Bm, br, bt), (C, cr, ct) = _tokens(x, 2), _tokens(dt, 1), _tokens(Bm, 2), _tokens(C, 2)
        y = torch.empty(B, L, H, P, dtype=x.dtype, device=x.device)
        if y.numel():
            last = torch.empty(B, H, P, N, device=x.device) if want_state else None
            handle = lib.load()
            segs = handle.rtfs_ssm_scan_segments(B, L, H, P, G, N, 1)
            work = torch.empty(B * H * segs * (handle.rtfs_ssm_tile(P, N) + 1), device=x.device) if segs > 1 else None
            lib.call("rtfs_ssm_scan_fwd", _raw(x), xr, xt, _raw(dt), tr, tt, _TYPES[dt.dtype], A, _raw(Bm), br, bt, _raw(C), cr, ct, D, dt_bias, int(softplus), state,
                     lengths, y, last, work, B, L, H, P, G, N, _TYPES[x.dtype])
        else:
            last = _through(state, (B, H, P, N), torch.float32, x.device) if want_state else None
        ctx.save_for_backward(x, dt, A, Bm, C, D, dt_bias, state, lengths)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, dt, A, Bm, C, D, dt_bias, state, lengths = ctx.saved_tensors
        B, L, H, P = x.shape
        G, N = Bm.shape[2:]
        (x, xr, xt), (dt, tr, tt), (Bm, br, bt), (C, cr, ct) = _tokens(x, 2), _tokens(dt, 1), _tokens(Bm, 2), _tokens(C, 2)
        dy = torch.zeros(B, L, H, P, dtype=x.dtype, device=x.device) if dy is None else dy.contiguous()

        def new(*shape, dtype=torch.float32):
            return torch.empty(*shape, dtype=dtype, device=x.device)

        dx, ddt = new(B, L, H, P, dtype=x.dtype), new(B, L, H, dtype=dt.dtype)
        dB, dC = new(B, L, G, N, dtype=x.dtype), new(B, L, G, N, dtype=x.dtype)
        dA, dD, db = new(H), new(H) if D is not None else None, new(H) if dt_bias is not None else None
        ds = torch.empty_like(state) if state is not None else None
        if not x.numel():
            ds = _through(dlast, ds.shape, torch.float32, x.device) if state is not None else None
            return dx, ddt, dA.zero_(), dB, dC, dD.zero_() if dD is not None else None, db.zero_() if db is not None else None, ds, None, None, None
        handle = lib.load()
        segs, tile, parts, chunks = handle.rtfs_ssm_scan_segments(B, L, H, P, G, N, 2), handle.rtfs_ssm_tile(P, N), handle.rtfs_ssm_scan_bwd_parts(B, L, H, G, N), -(-L // 64)
        starts = new(2 * B * H * segs * (tile + 1)) if segs > 1 else None
        wide = new(2 * parts * B * L * G * N) if parts > 1 else None
        lib.call("rtfs_ssm_scan_bwd", _raw(x), xr, xt, _raw(dt), tr, tt, _TYPES[dt.dtype], A, _raw(Bm), br, bt, _raw(C), cr, ct, D, dt_bias, int(ctx.softplus), state,
                 lengths, dy, _dense(dlast), dx, ddt, dA, dB, dC, dD, db, ds, starts, new(B * chunks * H * tile), new(B * chunks * H * tile), wide,
                 new(B * chunks * H * 3), B, L, H, P, G, N, _TYPES[x.dtype])
        return dx, ddt, dA, dB, dC, dD, db, ds, None, None, None


def _scan_parameters(name, x, dt, A, B, C, D, dt_bias, state, lead):
    """shapes and types of a scan's arguments, `lead` = the dimensions in front of the heads"""
    H, P = x.shape[-2:]
    if not isinstance(B, torch.Tensor) or B.dim() != len(lead) + 2:
        raise ValueError(f"{name}: B must have {len(lead) + 2} dimensions")
    G, N = B.shape[-2:]
    if not 1 <= P <= 128 or not 1 <= N <= 128 or H < 1:
        raise ValueError(f"{name}: at least one head, and 1 to 128 values per head and per state row (P = {P}, N = {N}, H = {H})")
    if G < 1 or H % G:
        raise ValueError(f"{name}: {H} heads do not divide over {G} groups of B and C")
    device, kinds = x.device, (x.dtype,)
    _check(name, "dt", dt, (*lead, H), (x.dtype, torch.float32), device)
    _check(name, "B", B, (*lead, G, N), kinds, device)
    _check(name, "C", C, (*lead, G, N), kinds, device)
    _check(name, "A", A, (H,), _FP32, device)
    if D is not None:
        _check(name, "D", D, (H,), _FP32, device)
    if dt_bias is not None:
        _check(name, "dt_bias", dt_bias, (H,), _FP32, device)
    if state is not None:
        _check(name, "state", state, (lead[0], H, P, N), _FP32, device)
    if lead[0] * H >= 1 << 22:
        raise ValueError(f"{name}: {1 << 22} rows times heads, or more")
    if max(H * P, G * N) >= 1 << 23:
        raise ValueError(f"{name}: a token of {1 << 23} values, or more")
    return G, N


def selective_scan(x, dt, A, B, C, D=None, *, dt_bias=None, softplus=False, state=None, lengths=None, return_state=False):
    """Selective state-space scan with one decay rate per head:  d = dt + dt_bias, or softplus of it;  S[t] = exp(d[t] A) S[t-1] + d[t] x[t] B[t]^T;
    y[t] = S[t] C[t] + D x[t].

    x [B, L, H, P], B and C [B, L, G, N], fp32 or bf16 (head h uses group h // (H // G)); dt [B, L, H] of x's type or fp32; A, D, dt_bias [H] fp32, the rates in A
    negative for a state that decays (without softplus a step may have either sign too; what lies between two tokens of a row may grow by e^88, fp32's range);
    state [B, H, P, N] fp32 in front of token 0 (None: zeros); lengths int32 [B].  P, N <= 128, B H < 2^22, H P < 2^23.
    -> y [B, L, H, P], or (y, last) with `return_state`: last [B, H, P, N], the state behind each row's end.  Differentiable in every tensor but lengths."""
    _first("selective_scan", x, 4)
    rows, L, H, P = x.shape
    G, N = _scan_parameters("selective_scan", x, dt, A, B, C, D, dt_bias, state, (rows, L))
    lengths = _lengths("selective_scan", lengths, rows, x.device)
    _on_gpu("selective_scan", x)
    y, last = _SelectiveScan.apply(x, dt, A, B, C, D, dt_bias, state, lengths, bool(softplus), bool(return_state))
    return (y, last) if return_state else y


def selective_scan_step(x, dt, A, B, C, state, D=None, *, dt_bias=None, softplus=False):
    """One token of every row: x [B, H, P], dt [B, H], B and C [B, G, N]; state [B, H, P, N] (contiguous, fp32) is updated in place -> y [B, H, P].
    For serving: no gradient."""
    _first("selective_scan_step", x, 3)
    rows, H, P = x.shape
    if state is None:
        raise ValueError("selective_scan_step: state is updated in place and must be given")
    G, N = _scan_parameters("selective_scan_step", x, dt, A, B, C, D, dt_bias, state, (rows,))
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("selective_scan_step: state is updated in place and must be contiguous, from a 16-byte boundary on")
    _no_gradient("selective_scan_step", x, dt, A, B, C, D, dt_bias, state)
    _on_gpu("selective_scan_step", x)
    y = torch.empty(rows, H, P, dtype=x.dtype, device=x.device)
    if rows:
        x, dt, B, C = _rows(x), _rows(dt), _rows(B), _rows(C)
        lib.call("rtfs_ssm_step", _raw(x), x.stride(0), _raw(dt), dt.stride(0), _TYPES[dt.dtype], _dense(A), _raw(B), B.stride(0), _raw(C), C.stride(0), _dense(D),
                 _dense(dt_bias), int(bool(softplus)), state, y, rows, H, P, G, N, _TYPES[x.dtype])
        torch.autograd.graph.increment_version(state)  # written through its address
    return y

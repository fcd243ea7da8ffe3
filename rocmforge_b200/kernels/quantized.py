"""Python faces of the 4-bit weight path: weights in 4 bits, rows in 8 bits, and the products that read them (csrc/quantized.cu).

maeddesg/ROCmForge keeps its quantised weights as the GGUF file has them and multiplies Q4 blocks with Q8 rows while it decodes
(src/gpu/ops.rs:455-747); here weights are quantised once, when a model is made, into the layout that the kernels read.
"""
from __future__ import annotations

import functools

import torch

from . import tensor_core as tc
from ._ffi import KernelError, c_float, c_int, c_ll, c_void_p, check, dtype_code, fn, need, need_cuda, ptr, stream

W4_GROUPS = (32, 64, 128)
W4_STORE, W4_ADD, W4_PARTIAL = 0, 2, 3


@functools.lru_cache(None)
def _f(name, *argtypes):
    return fn("quantized", name, list(argtypes))


def padded_columns(K: int, group: int) -> int:
    """Columns that the stored forms of a row of ``K`` take: whole tiles of 64 and whole groups."""
    unit = max(64, group)
    return (K + unit - 1) // unit * unit


def _need_group(group, what: str) -> None:
    need(group in W4_GROUPS, f"{what}: groups of {group} (known: {W4_GROUPS})")


def _need_here(what: str, *tensors) -> None:
    """Every tensor on the current device, whose stream the launch goes to."""
    need_cuda(*tensors)
    here = torch.cuda.current_device()
    for t in tensors:
        need(t is None or t.device.index == here, f"{what}: a tensor on {None if t is None else t.device}, the current device is cuda:{here}")


class Q8Rows:
    """Activations in 8 bits: row t's number k stands for ``scales[t, k // group] * q[t, k]``.

    ``q`` int8 [T, padded_columns(K, group)] with zeros from column K on, ``scales`` float32 [T, padded columns / group]; ``dtype`` is that
    of the rows they stand for, in which ``materialize`` gives them back and a product's result comes."""

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, K: int, group: int, dtype: torch.dtype):
        _need_group(group, "Q8Rows")
        Kp = padded_columns(K, group)
        need(q.dtype == torch.int8 and q.dim() == 2 and q.shape[1] == Kp and q.is_contiguous(), f"Q8Rows: q must be int8 [T, {Kp}]")
        need(scales.dtype == torch.float32 and tuple(scales.shape) == (q.shape[0], Kp // group) and scales.is_contiguous(),
             f"Q8Rows: scales must be float32 [T, {Kp // group}]")
        need(q.device == scales.device, "Q8Rows: q and scales must be on one device")
        dtype_code(dtype)
        self.q, self.scales, self.K, self.group, self.dtype = q, scales, int(K), int(group), dtype
        self.shape = torch.Size((q.shape[0], int(K)))

    @property
    def device(self):
        return self.q.device

    def materialize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The rows as an ordinary tensor [T, K]."""
        dtype = dtype or self.dtype
        _need_here("Q8Rows.materialize", self.q, self.scales)
        T, K = self.shape
        out = torch.empty((T, K), dtype=dtype, device=self.device)
        f = _f("rf_dequantize_q8", c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p)
        check(f(dtype_code(dtype), ptr(self.q), ptr(self.scales), ptr(out), T, K, self.group, stream()), "Q8Rows.materialize")
        return out


class W4Weight:
    """A weight [N, K] in 4 bits: weight[n, k] = s[n, k // group] * q[n, k], q in -8..7.

    ``packed`` uint8 [tiles of 16 rows, blocks of 64 columns, 32, 16]: of a tile's block, entry [4 g + t, 8 r + 4 c + b] holds row g + 8 r,
    its low four bits column 32 c + 8 t + b, its high ones column 32 c + 8 t + 4 + b (two's complement).  ``scales`` bfloat16 [tiles,
    groups, 16]: entry [2 g + r] is row g + 8 r.  Rows and columns are padded with zeros.  Products read both before they wait for the
    kernel launched before them: whoever writes them with kernels of its own calls ``weights_made`` afterwards."""

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, N: int, K: int, group: int):
        _need_group(group, "W4Weight")
        need(N > 0 and K > 0, "W4Weight: an empty weight")
        Kp, tiles = padded_columns(K, group), (N + 15) // 16
        need(packed.dtype == torch.uint8 and tuple(packed.shape) == (tiles, Kp // 64, 32, 16) and packed.is_contiguous(),
             f"W4Weight: packed must be uint8 [{tiles}, {Kp // 64}, 32, 16]")
        need(scales.dtype == torch.bfloat16 and tuple(scales.shape) == (tiles, Kp // group, 16) and scales.is_contiguous(),
             f"W4Weight: scales must be bfloat16 [{tiles}, {Kp // group}, 16]")
        need(packed.device == scales.device, "W4Weight: packed and scales must be on one device")
        need(packed.data_ptr() % 16 == 0 and scales.data_ptr() % 4 == 0, "W4Weight: packed must be aligned to 16 bytes, scales to 4")
        self.packed, self.scales, self.N, self.K, self.group = packed, scales, int(N), int(K), int(group)
        self.shape = torch.Size((int(N), int(K)))

    @property
    def device(self):
        return self.packed.device

    @property
    def nbytes(self) -> int:
        return self.packed.numel() + 2 * self.scales.numel()

    @classmethod
    def from_quantized(cls, q: torch.Tensor, scales: torch.Tensor, group: int) -> "W4Weight":
        """From whole numbers ``q`` [N, K] in -8..7 and ``scales`` [N, ceil(K / group)]: weights that were quantised elsewhere, laid out
        on their device.  Scales of more than five significant bits are kept (in bfloat16); 16-bit products of many tokens then round
        the weights to bfloat16, which the scales that ``quantize_w4`` makes spare them."""
        _need_group(group, "W4Weight")
        need(q.dim() == 2 and not q.is_floating_point() and q.shape[0] > 0 and q.shape[1] > 0, "W4Weight: q must be whole numbers [N, K]")
        N, K = q.shape
        need(scales.shape == (N, (K + group - 1) // group), f"W4Weight: scales must be [{N}, {(K + group - 1) // group}]")
        need(bool(((q >= -8) & (q <= 7)).all()), "W4Weight: q must lie in -8..7")
        Np, Kp = (N + 15) // 16 * 16, padded_columns(K, group)
        full = torch.zeros((Np, Kp), dtype=torch.uint8, device=q.device)
        full[:N, :K] = (q.to(torch.int16) & 15).to(torch.uint8)
        # [tile, r, g, block, c, t, half, b] -> [tile, block, g, t, r, c, b, half]
        full = full.view(Np // 16, 2, 8, Kp // 64, 2, 4, 2, 4).permute(0, 3, 2, 5, 1, 4, 7, 6)
        packed = (full[..., 0] | (full[..., 1] << 4)).reshape(Np // 16, Kp // 64, 32, 16).contiguous()
        s = torch.zeros((Np, Kp // group), dtype=torch.bfloat16, device=q.device)
        s[:N, :scales.shape[1]] = scales
        s = s.view(Np // 16, 2, 8, Kp // group).permute(0, 3, 2, 1).reshape(Np // 16, Kp // group, 16).contiguous()
        if q.is_cuda:
            with torch.cuda.device(q.device):
                weights_made()
        return cls(packed, s, N, K, group)


def weights_made() -> None:
    """Products on the current stream may from here on read weights that the stream's last kernels have made."""
    check(_f("rf_weights_made", c_void_p)(stream()), "weights_made")


def quantize_w4(weight: torch.Tensor, group: int = 128) -> W4Weight:
    """``weight`` [N, K] (float32 or bfloat16, rows any distance apart) in 4 bits: every group's largest magnitude becomes 7.5 steps, the
    step rounded to five significant bits, so that every weight is exactly a bfloat16 number."""
    _need_here("quantize_w4", weight)
    _need_group(group, "quantize_w4")
    need(weight.dim() == 2 and weight.shape[0] > 0 and weight.shape[1] > 0 and weight.stride(1) == 1,
         "quantize_w4: the weight must be a matrix with unit inner stride")
    N, K = weight.shape
    Kp, tiles = padded_columns(K, group), (N + 15) // 16
    packed = torch.empty((tiles, Kp // 64, 32, 16), dtype=torch.uint8, device=weight.device)
    scales = torch.empty((tiles, Kp // group, 16), dtype=torch.bfloat16, device=weight.device)
    f = _f("rf_quantize_w4", c_int, c_void_p, c_ll, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p)
    check(f(dtype_code(weight.dtype), ptr(weight), weight.stride(0), ptr(packed), ptr(scales), N, K, group, stream()), f"quantize_w4 ({N}x{K})")
    return W4Weight(packed, scales, N, K, group)


def dequantize_w4(w: W4Weight, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The weights as a tensor [N, K]; products may read it at once."""
    _need_here("dequantize_w4", w.packed, w.scales)
    out = torch.empty(w.shape, dtype=dtype, device=w.device)
    f = _f("rf_dequantize_w4", c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p)
    check(f(dtype_code(dtype), ptr(w.packed), ptr(w.scales), ptr(out), w.N, w.K, w.group, stream()), f"dequantize_w4 ({w.N}x{w.K})")
    return out


def _new_rows(T: int, K: int, group: int, dtype, device) -> Q8Rows:
    Kp = padded_columns(K, group)
    return Q8Rows(torch.empty((T, Kp), dtype=torch.int8, device=device),
                  torch.empty((T, Kp // group), dtype=torch.float32, device=device), K, group, dtype)


def quantize_q8(x: torch.Tensor, group: int = 128) -> Q8Rows:
    """``x`` [T, K] (float32 or bfloat16, rows any distance apart) in 8 bits: scale = max|x| / 127 of every group, numbers to the nearest.
    A group below 2^-120 becomes zeros; one with a NaN or an infinity gets the scale NaN."""
    _need_here("quantize_q8", x)
    _need_group(group, "quantize_q8")
    need(x.dim() == 2 and x.shape[1] > 0 and x.stride(1) == 1, "quantize_q8: x must be [T, K] with unit inner stride")
    T, K = x.shape
    y = _new_rows(T, K, group, x.dtype, x.device)
    f = _f("rf_quantize_q8", c_int, c_void_p, c_ll, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p)
    check(f(dtype_code(x.dtype), ptr(x), x.stride(0), ptr(y.q), ptr(y.scales), T, K, group, stream()), f"quantize_q8 ({T}x{K})")
    return y


def add_rmsnorm_q8(h: torch.Tensor, weight: torch.Tensor, eps: float, compute_dtype: torch.dtype, group: int = 128,
                   pending: torch.Tensor | None = None, rows: torch.Tensor | None = None) -> Q8Rows:
    """``add_rmsnorm`` with its result in 8 bits: rmsnorm(h + pending) * weight, from 32 bits straight to groups of ``group`` columns.

    ``h`` [T, H] float32 is the residual stream; ``pending`` (None, a float32 stack [S, T, H] of partial sums, or a [T, H] tensor of the
    compute dtype or float32) is added into it in place.  With ``rows`` (int32 indices) only those rows are normalised and ``h`` is left
    untouched."""
    _need_here("add_rmsnorm_q8", h, weight, pending, rows)
    _need_group(group, "add_rmsnorm_q8")
    need(h.dtype == torch.float32 and h.dim() == 2 and h.is_contiguous(), "add_rmsnorm_q8: h must be [T,H] float32")
    T, H = h.shape
    need(weight.shape == (H,) and weight.dtype in (torch.float32, torch.bfloat16) and weight.is_contiguous(),
         "add_rmsnorm_q8: weight must be [H] in float32 or bfloat16")
    kind, n_pending, pstride = 0, 0, 0
    if pending is not None:
        need(pending.is_contiguous(), "add_rmsnorm_q8: pending must be contiguous")
        if pending.dtype == torch.float32 and pending.dim() == 3 and pending.shape[1:] == (T, H):
            kind, n_pending, pstride = 1, pending.shape[0], T * H
        elif pending.dtype == torch.float32 and pending.shape == (T, H):
            kind, n_pending, pstride = 1, 1, T * H
        elif pending.dtype == compute_dtype and pending.shape == (T, H):
            kind = 2
        else:
            raise KernelError(f"add_rmsnorm_q8: pending of shape {tuple(pending.shape)} / {pending.dtype} does not fit h {tuple(h.shape)}")
    n_rows = T
    if rows is not None:
        need(rows.dtype == torch.int32 and rows.dim() == 1 and rows.is_contiguous(), "add_rmsnorm_q8: rows must be 1-d int32")
        n_rows = rows.shape[0]
    y = _new_rows(n_rows, H, group, compute_dtype, h.device)
    f = _f("rf_add_rmsnorm_q8", c_int, c_void_p, c_void_p, c_int, c_int, c_ll, c_void_p, c_int, c_float, c_void_p, c_void_p, c_void_p, c_int,
           c_int, c_int, c_int, c_void_p)
    check(f(dtype_code(compute_dtype), ptr(h), ptr(pending), kind, n_pending, pstride, ptr(weight), int(weight.dtype == torch.float32), float(eps),
            ptr(y.q), ptr(y.scales), ptr(rows), n_rows, T, H, group, stream()), f"add_rmsnorm_q8 (H={H})")
    return y


_ACTIVATIONS = {"silu": 0, "relu": 1, "gelu_tanh": 2}


def swiglu_q8(gu: torch.Tensor, group: int = 128, activation: str = "silu") -> Q8Rows:
    """``swiglu`` with its result in 8 bits: act(gu[t, 2j]) * gu[t, 2j+1], from 32 bits straight to groups of ``group`` columns."""
    need(activation in _ACTIVATIONS, f"swiglu_q8: activation {activation!r} (known: {sorted(_ACTIVATIONS)})")
    _need_here("swiglu_q8", gu)
    _need_group(group, "swiglu_q8")
    need(gu.dim() == 2 and gu.is_contiguous() and gu.shape[1] % 2 == 0 and gu.shape[1] > 0, "swiglu_q8: input must be [T, 2I]")
    T, I = gu.shape[0], gu.shape[1] // 2
    y = _new_rows(T, I, group, gu.dtype, gu.device)
    f = _f("rf_swiglu_q8", c_int, c_void_p, c_int, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p)
    check(f(dtype_code(gu.dtype), ptr(gu), _ACTIVATIONS[activation], ptr(y.q), ptr(y.scales), T, I, group, stream()), f"swiglu_q8 (I={I})")
    return y


W4_FEW_TOKENS = 128      # tokens that products of 16-bit rows take straight from the 4 bits; more: the weights as 16 bits, then that product


def gemm_w4(x, w: W4Weight, bias: torch.Tensor | None = None, *, out: torch.Tensor | None = None, out_f32: bool = False,
            accumulate: bool = False, splits: int = 0) -> torch.Tensor:
    """y = x @ w.T (+ bias) with 4-bit weights, 32-bit sums.

    ``x``: ``Q8Rows`` of the weight's K and group (products inside a group are exact, in whole numbers), or a tensor [M, K] in bfloat16
    or float32.  out_f32: the result is float32 whatever the rows; accumulate: added into ``out`` (float32); splits >= 1 (8-bit rows, or
    few 16-bit ones): the float32 stack [splits, M, N] of partial sums over ranges of K (no bias)."""
    q8 = isinstance(x, Q8Rows)
    need(q8 or isinstance(x, torch.Tensor), "gemm_w4: x must be Q8Rows or a tensor")
    need(isinstance(w, W4Weight), "gemm_w4: w must be a W4Weight")
    _need_here("gemm_w4", x.q if q8 else x, w.packed, bias, out)
    if q8:
        need(x.group == w.group, f"gemm_w4: rows in groups of {x.group}, the weight in groups of {w.group}")
    else:
        need(x.dim() == 2 and x.stride(1) == 1, "gemm_w4: x must be [M, K] with unit inner stride")
    need(x.shape[1] == w.K, f"gemm_w4: inner sizes differ ({x.shape[1]} vs {w.K})")
    M, N, dt = x.shape[0], w.N, x.dtype
    dtype_code(dt)
    if bias is not None:
        need(bias.shape == (N,) and bias.dtype in (torch.float32, torch.bfloat16) and bias.is_contiguous(), "gemm_w4: bias must be [N]")
    if splits >= 1:
        need(not accumulate and out is None and bias is None, "gemm_w4: partial sums take no bias and no output tensor")
        out, mode, odt = torch.empty((splits, M, N), dtype=torch.float32, device=x.device), W4_PARTIAL, torch.float32
    else:
        mode, odt = W4_ADD if accumulate else W4_STORE, torch.float32 if out_f32 or accumulate else dt
        if out is None:
            need(not accumulate, "gemm_w4: accumulate needs an output tensor")
            out = torch.empty((M, N), dtype=odt, device=x.device)
        need(out.shape == (M, N) and out.dtype == odt and out.is_contiguous(), "gemm_w4: output must be [M, N], contiguous, of the result's dtype")
    if M == 0:
        return out
    if not q8 and (dt == torch.float32 or M > W4_FEW_TOKENS):
        need(mode != W4_PARTIAL, "gemm_w4: no partial sums of float32 rows or of many tokens")
        return _gemm_through_16_bits(x, w, bias, out, mode, odt)
    f = _f("rf_gemm_w4", c_int, c_void_p, c_void_p, c_ll, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_int, c_int, c_int,
           c_int, c_int, c_void_p)
    check(f(0 if q8 else 1, ptr(x.q if q8 else x), ptr(x.scales if q8 else None), x.q.stride(0) if q8 else x.stride(0), ptr(w.packed), ptr(w.scales),
            ptr(bias), int(bias is not None and bias.dtype == torch.float32), ptr(out), int(odt == torch.float32), mode,
            max(splits, 1), M, N, w.K, w.group, stream()), f"gemm_w4 ({M}x{N}x{w.K})")
    return out


def _gemm_through_16_bits(x, w, bias, out, mode, odt):
    """The product by the weights written out once in the rows' dtype (exactly, with scales of five significant bits)."""
    from .basic import gemm_plain
    M, K = x.shape
    full = dequantize_w4(w, x.dtype)
    if x.dtype == torch.bfloat16:
        m = tc.RESIDUAL if mode == W4_ADD else tc.F32 if odt == torch.float32 else tc.STORE
        if tc.supported(M, w.N, K, m) and x.data_ptr() % 16 == 0 and x.stride(0) % 8 == 0:
            return tc.gemm_tc(x, full, bias, mode=m, out=out)
    return gemm_plain(x, full, bias, out=out, out_f32=odt == torch.float32 and x.dtype != torch.float32, accumulate=mode == W4_ADD)

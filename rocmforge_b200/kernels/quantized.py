"""Python faces of the 4-bit weight path: weights in 4 bits, rows in 8 bits, and the products that read them (csrc/quantized.cu).

maeddesg/ROCmForge keeps its quantised weights as the GGUF file has them and multiplies Q4 blocks with Q8 rows while it decodes
(src/gpu/ops.rs:455-747); here weights are quantised once, when a model is made, into the layout that the kernels read.

The calls of a decode step are as short on the device as a launch is on the host, so the checks build no text unless they fail.
"""
from __future__ import annotations

import functools

import torch

from . import tensor_core as tc
from ._ffi import KernelError, c_float, c_int, c_ll, c_void_p, check, dtype_code, fn, need, ptr, sm_count, stream

W4_GROUPS = (32, 64, 128)
W4_MOST_SHARED = 227 * 1024
_p, _i, _n = c_void_p, c_int, c_ll
_LAUNCHERS = {
    "rf_quantize_q8": [_i, _p, _n, _p, _p, _i, _i, _i, _p],
    "rf_dequantize_q8": [_i, _p, _p, _p, _i, _i, _i, _p],
    "rf_swiglu_q8": [_i, _p, _i, _p, _p, _i, _i, _i, _p],
    "rf_add_rmsnorm_q8": [_i, _p, _p, _i, _i, _n, _p, _i, c_float, _p, _p, _p, _i, _i, _i, _i, _p],
    "rf_quantize_w4": [_i, _p, _n, _p, _p, _i, _i, _i, _p],
    "rf_dequantize_w4": [_i, _p, _p, _p, _i, _i, _i, _i, _i, _p],
    "rf_weights_made": [_p],
    "rf_gemm_w4_shared": [_i, _i, _i, _i, _i, _i, _i, _i, _i, _i],
    "rf_gemm_w4_clusters": [_i],
    "rf_gemm_w4": [_i, _p, _p, _n, _p, _p, _p, _i, _p, _i, _i, _i, _i, _i, _i, _i, _i, _i, _i, _i, _p],
}
_TC_LAUNCHERS = {
    "rf_gemm_w4_tc": [_p, _n, _p, _p, _p, _i, _p, _i, _i, _i, _i, _i, _i, _i, _i, _p, _p],
}


@functools.lru_cache(None)
def _f(name: str):
    return fn("quantized", name, _LAUNCHERS[name]) if name in _LAUNCHERS else fn("quantized_tc", name, _TC_LAUNCHERS[name])


def padded_columns(K: int, group: int) -> int:
    """Columns that the stored forms of a row of ``K`` take: whole tiles of 64 and whole groups."""
    unit = 128 if group == 128 else 64
    return (K + unit - 1) // unit * unit


def _need_group(group, what: str) -> None:
    if group not in W4_GROUPS:
        raise KernelError(f"{what}: groups of {group} (known: {W4_GROUPS})")


_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _device_for(index: int) -> int:
    """The current device (not asked where a tensor lies on the CPU)."""
    return _device() if index >= 0 else -2


def _elsewhere(what: str, index: int) -> None:
    if index < 0:
        raise KernelError(f"{what}: rocmforge_b200 kernels run on a CUDA device only; got a tensor on cpu (there is no CPU fallback)")
    raise KernelError(f"{what}: a tensor on cuda:{index}, the current device is cuda:{_device()}")


def _need_here(what: str, *tensors) -> None:
    """Every tensor on the current device, whose stream the launch goes to."""
    here = None
    for t in tensors:
        if t is not None:
            at = t.get_device()
            if here is None:
                here = _device_for(at)
            if at != here:
                _elsewhere(what, at)


class Q8Rows:
    """Activations in 8 bits: row t's number k stands for ``scales[t, k // group] * q[t, k]``.

    ``q`` int8 [T, padded_columns(K, group)] with zeros from column K on, ``scales`` float32 [T, padded columns / group]; ``dtype`` is that
    of the rows they stand for, in which ``materialize`` gives them back and a product's result comes."""

    __slots__ = ("T", "K", "group", "dtype", "index", "at", "scales_at", "_q", "_scales", "_memory")

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, K: int, group: int, dtype: torch.dtype):
        _need_group(group, "Q8Rows")
        Kp = padded_columns(K, group)
        at, index = q.data_ptr(), q.get_device()
        if not (K > 0 and q.dtype == torch.int8 and q.dim() == 2 and q.shape[1] == Kp and q.is_contiguous() and at % 16 == 0):
            raise KernelError(f"Q8Rows: q must be int8 [T, {Kp}], aligned to 16 bytes")
        T = q.shape[0]
        if not (scales.dtype == torch.float32 and scales.shape == (T, Kp // group) and scales.is_contiguous()):
            raise KernelError(f"Q8Rows: scales must be float32 [T, {Kp // group}]")
        if index != scales.get_device():
            raise KernelError("Q8Rows: q and scales must be on one device")
        dtype_code(dtype)
        self.T, self.K, self.group, self.dtype, self.index = T, K, group, dtype, index
        self._q, self._scales, self.at, self.scales_at, self._memory = q, scales, at, scales.data_ptr(), None

    @classmethod
    def empty(cls, T: int, K: int, group: int, dtype: torch.dtype, device) -> "Q8Rows":
        """Rows that a kernel is about to fill: numbers and scales in one piece of memory (an allocation is a third of a call's host time)."""
        r = cls.__new__(cls)
        Kp = padded_columns(K, group)
        r._memory = memory = torch.empty(T * Kp + 4 * T * (Kp // group), dtype=torch.int8, device=device)
        r.T, r.K, r.group, r.dtype, r.index = T, K, group, dtype, memory.get_device()
        r.at = memory.data_ptr()
        r.scales_at = r.at + T * Kp
        r._q = r._scales = None
        return r

    def _split(self) -> None:
        Kp, T = padded_columns(self.K, self.group), self.T
        self._q = self._memory[:T * Kp].view(T, Kp)
        self._scales = self._memory[T * Kp:].view(torch.float32).view(T, Kp // self.group)

    @property
    def q(self) -> torch.Tensor:
        if self._q is None:
            self._split()
        return self._q

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._split()
        return self._scales

    @property
    def shape(self):
        return torch.Size((self.T, self.K))

    @property
    def device(self):
        return (self._memory if self._q is None else self._q).device

    def materialize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The rows as an ordinary tensor [T, K]."""
        dtype = dtype or self.dtype
        code = dtype_code(dtype)
        if self.index != _device_for(self.index):
            _elsewhere("Q8Rows.materialize", self.index)
        out = torch.empty(self.T, self.K, dtype=dtype, device=self.device)
        check(_f("rf_dequantize_q8")(code, self.at, self.scales_at, out.data_ptr(), self.T, self.K, self.group, stream()), "Q8Rows.materialize")
        return out


class W4Weight:
    """A weight [N, K] in 4 bits: weight[n, k] = s[n, k // group] * q[n, k], q in -8..7.

    ``packed`` uint8 [tiles of 16 rows, blocks of 64 columns, 32, 16]: of a tile's block, entry [4 g + t, 8 r + 4 c + b] holds row g + 8 r,
    its low four bits column 32 c + 8 t + b, its high ones column 32 c + 8 t + 4 + b (two's complement).  ``scales`` bfloat16 [tiles,
    groups, 16]: entry [2 g + r] is row g + 8 r.  Rows and columns are padded with zeros.  Products read both before they wait for the
    kernel launched before them: whoever writes them with kernels of its own calls ``weights_made`` afterwards."""

    __slots__ = ("packed", "scales", "N", "K", "group", "index", "at", "scales_at")

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, N: int, K: int, group: int):
        _need_group(group, "W4Weight")
        need(N > 0 and K > 0, "W4Weight: an empty weight")
        Kp, tiles = padded_columns(K, group), (N + 15) // 16
        if not (packed.dtype == torch.uint8 and packed.shape == (tiles, Kp // 64, 32, 16) and packed.is_contiguous()):
            raise KernelError(f"W4Weight: packed must be uint8 [{tiles}, {Kp // 64}, 32, 16]")
        if not (scales.dtype == torch.bfloat16 and scales.shape == (tiles, Kp // group, 16) and scales.is_contiguous()):
            raise KernelError(f"W4Weight: scales must be bfloat16 [{tiles}, {Kp // group}, 16]")
        index, at, scales_at = packed.get_device(), packed.data_ptr(), scales.data_ptr()
        if index != scales.get_device() or at % 16 or scales_at % 16:
            raise KernelError("W4Weight: packed and scales must be on one device and aligned to 16 bytes")
        self.packed, self.scales, self.N, self.K, self.group, self.index, self.at, self.scales_at = packed, scales, N, K, group, index, at, scales_at

    @property
    def shape(self):
        return torch.Size((self.N, self.K))

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
    check(_f("rf_weights_made")(stream()), "weights_made")


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
    check(_f("rf_quantize_w4")(dtype_code(weight.dtype), ptr(weight), weight.stride(0), ptr(packed), ptr(scales), N, K, group, stream()),
          f"quantize_w4 ({N}x{K})")
    return W4Weight(packed, scales, N, K, group)


def dequantize_w4(w: W4Weight, dtype: torch.dtype = torch.bfloat16, columns: tuple[int, int] | None = None) -> torch.Tensor:
    """The weights as a tensor [N, K], or the columns [from, to) of them, ``from`` a multiple of 64; products may read it at once."""
    _need_here("dequantize_w4", w.packed)
    lo, hi = columns or (0, w.K)
    need(0 <= lo < hi <= w.K and lo % 64 == 0, "dequantize_w4: columns must lie in the weight and start at a multiple of 64")
    out = torch.empty((w.N, hi - lo), dtype=dtype, device=w.device)
    check(_f("rf_dequantize_w4")(dtype_code(dtype), ptr(w.packed), ptr(w.scales), ptr(out), w.N, w.K, lo, hi, w.group, stream()),
          "dequantize_w4")
    return out


def quantize_q8(x: torch.Tensor, group: int = 128) -> Q8Rows:
    """``x`` [T, K] (float32 or bfloat16, rows any distance apart) in 8 bits: scale = max|x| / 127 of every group, numbers to the nearest.
    A group below 2^-120 becomes zeros; one with a NaN or an infinity gets the scale NaN."""
    _need_here("quantize_q8", x)
    _need_group(group, "quantize_q8")
    need(x.dim() == 2 and x.shape[1] > 0 and x.stride(1) == 1, "quantize_q8: x must be [T, K] with unit inner stride")
    T, K = x.shape
    code = dtype_code(x.dtype)
    y = Q8Rows.empty(T, K, group, x.dtype, x.device)
    check(_f("rf_quantize_q8")(code, x.data_ptr(), x.stride(0), y.at, y.scales_at, T, K, group, stream()), "quantize_q8")
    return y


# Columns, padded, that a row of add_rmsnorm_q8 may have: a block keeps them in registers, 32 a thread.
W4_NORM_MOST = 32768


def add_rmsnorm_q8(h: torch.Tensor, weight: torch.Tensor, eps: float, compute_dtype: torch.dtype, group: int = 128,
                   pending: torch.Tensor | None = None, rows: torch.Tensor | None = None) -> Q8Rows:
    """``add_rmsnorm`` with its result in 8 bits: rmsnorm(h + pending) * weight, from 32 bits straight to groups of ``group`` columns.

    ``h`` [T, H] float32 is the residual stream; ``pending`` (None, a float32 stack [S, T, H] of partial sums, or a [T, H] tensor of the
    compute dtype or float32) is added into it in place.  With ``rows`` (int32 indices) only those rows are normalised and ``h`` is left
    untouched.  H up to ``W4_NORM_MOST``."""
    _need_here("add_rmsnorm_q8", h, weight, pending, rows)
    _need_group(group, "add_rmsnorm_q8")
    need(h.dtype == torch.float32 and h.dim() == 2 and h.is_contiguous(), "add_rmsnorm_q8: h must be [T,H] float32")
    T, H = h.shape
    w_is_f32 = weight.dtype == torch.float32
    need(weight.shape == (H,) and (w_is_f32 or weight.dtype == torch.bfloat16) and weight.is_contiguous(),
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
    code = dtype_code(compute_dtype)
    y = Q8Rows.empty(n_rows, H, group, compute_dtype, h.device)
    check(_f("rf_add_rmsnorm_q8")(code, h.data_ptr(), ptr(pending), kind, n_pending, pstride, weight.data_ptr(), w_is_f32, eps, y.at,
                                  y.scales_at, ptr(rows), n_rows, T, H, group, stream()), "add_rmsnorm_q8")
    return y


_ACTIVATIONS = {"silu": 0, "relu": 1, "gelu_tanh": 2}


def swiglu_q8(gu: torch.Tensor, group: int = 128, activation: str = "silu", dtype: torch.dtype | None = None) -> Q8Rows:
    """``swiglu`` with its result in 8 bits: act(gu[t, 2j]) * gu[t, 2j+1], from 32 bits straight to groups of ``group`` columns.  ``dtype``:
    that of the rows they stand for, where it is not gu's.  (A gate that is no number counts as 0 for "relu", as in ``swiglu``.)"""
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise KernelError(f"swiglu_q8: activation {activation!r} (known: {sorted(_ACTIVATIONS)})")
    _need_here("swiglu_q8", gu)
    _need_group(group, "swiglu_q8")
    need(gu.dim() == 2 and gu.is_contiguous() and gu.shape[1] % 2 == 0 and gu.shape[1] > 0, "swiglu_q8: input must be [T, 2I]")
    T, I = gu.shape[0], gu.shape[1] // 2
    code, dtype = dtype_code(gu.dtype), dtype or gu.dtype
    dtype_code(dtype)
    y = Q8Rows.empty(T, I, group, dtype, gu.device)
    check(_f("rf_swiglu_q8")(code, gu.data_ptr(), act, y.at, y.scales_at, T, I, group, stream()), "swiglu_q8")
    return y


# Products of up to so many tokens take rows in 8 bits where a step may choose (32 x 37,888 x 3,584: 22.1 us against 28.5 of 16-bit rows; 64 tokens:
# 39.2, 30.2; 64 x 3,584 x 18,944: 28.0, 20.2).
W4_FEW_TOKENS = 32
# 16-bit rows straight from the 4 bits: up to so many tokens (512 x 37,888 x 3,584: 147 us, 155 by the weights written out in 16 bits; 512 x 3,584 x
# 18,944: 59, 123; 1,024: 289, 239 and 120, 142).
W4_TC_MOST = 512
# 32-bit results of rows of several SUM_COLUMNS: up to so many with two of them, twice as many with more, since that other way takes a pass over
# the result for each (1,024 x 4,608 x 3,584: 40 us against 51, 2,048: 74, 68; 2,048 x 3,584 x 18,944: 273, 338; 4,096: 488, 586; 2,048 x 5,120 x
# 13,824: 260, 326)
W4_TC_MOST_F32 = 1024
# Columns that one tensor-core sum runs over where the result is 32-bit: its additions are cut, not rounded, and what is cut adds up
# (1,999 x 3,584 x 18,944 against 64 bits: one sum 1.1e-5, pieces of 6,315 2.6e-6, of 2,048 5e-7)
SUM_COLUMNS = 2048


@functools.lru_cache(None)
def w4_clusters(splits: int, device: int) -> int:
    """Clusters of ``splits`` blocks that run at once on a device, an SM a block."""
    if splits == 1:
        return sm_count(device)
    n = _f("rf_gemm_w4_clusters")(splits)
    need(n > 0, "gemm_w4: no clusters can be launched")
    return n


# What a warp of rf_gemm_w4 takes for 128 columns of its tiles, by 8-bit rows, eights of tokens and tiles a warp, as a share of what four eights
# of 8-bit rows by one tile take; half of one more a round in which warps wait for one another, one where clusters exchange their sums.  (In
# 165 cases from 1 x 896 x 896 to 128 x 3,584 x 18,944 the plans chosen by it took 1 % more than the best of all, 14 % at most.)
W4_COST = {(True, 1, 1): 0.3, (True, 2, 1): 0.55, (True, 2, 2): 0.9, (True, 4, 1): 1.0, (True, 4, 2): 1.9,
           (False, 1, 1): 0.4, (False, 2, 1): 0.5, (False, 2, 2): 1.05}


def _w4_few(q8: bool, M: int, N: int, K: int, group: int, clusters_of):
    """(cost, eights of tokens, tiles a warp, warps a tile, splits, clusters): how ``rf_gemm_w4`` shares out a product, by what the busiest
    warp takes; None where no way fits into shared memory."""
    units, rows16 = (padded_columns(K, group) // 64 + 1) // 2, (N + 15) // 16
    # tokens at once: fewer than there are only where longer rows leave no room, or (above 16) where that is faster
    for some in ((1,),) if M <= 8 else ((2,), (1,)) if M <= 16 or not q8 else ((2, 4), (1,)):
        best = None
        for eights in some:
            shares = (M + 8 * eights - 1) // (8 * eights)
            for pair in (1, 2) if eights > 1 else (1,):
                tiles = (rows16 + pair - 1) // pair
                for splits in range(1, 9):
                    clusters = max(1, clusters_of(splits) // shares)
                    for ways in (1, 2, 4, 8, 16):
                        used = min(clusters, (tiles * ways + 15) // 16)
                        if _f("rf_gemm_w4_shared")(0 if q8 else 1, M, N, K, group, eights, pair, ways, splits, used) > W4_MOST_SHARED:
                            continue
                        rounds = (tiles + used * (16 // ways) - 1) // (used * (16 // ways))
                        each = (units + splits * ways - 1) // (splits * ways) * W4_COST[q8, eights, pair]
                        cost = rounds * (each + 0.5 * (ways > 1 or splits > 1)) + (splits > 1)
                        if best is None or cost < best[0]:
                            best = cost, eights, pair, ways, splits, used
        if best is not None:
            return best
    return None


# What a block of rf_gemm_w4_tc takes, by the tokens of its tile: us for 512 columns, us beside them.
W4_TC_COST = {32: (1.48, 3.2), 64: (1.5, 3.8), 128: (1.5, 7.5)}


def _w4_tc(M: int, N: int, K: int, group: int, clusters_of):
    """(us, tokens of a tile, splits): how ``rf_gemm_w4_tc`` shares out a product of 16-bit rows."""
    stages, rows, best = (padded_columns(K, group) + 511) // 512, (N + 127) // 128, None
    for bn, (stage, beside) in W4_TC_COST.items():
        tiles = rows * ((M + bn - 1) // bn)
        for splits in range(1, 9):
            rounds = (tiles + clusters_of(splits) - 1) // clusters_of(splits)
            cost = rounds * ((stages + splits - 1) // splits * stage + beside) + 0.5 * (splits > 1)
            if best is None or cost < best[0]:
                best = cost, bn, splits
    return best


@functools.lru_cache(4096)
def w4_launch(q8: bool, M: int, N: int, K: int, group: int, clusters_of, tensor_cores: bool = True):
    """How a product is shared out, chosen from sizes alone: five numbers for ``rf_gemm_w4`` (``_w4_few``), two for ``rf_gemm_w4_tc``
    (``_w4_tc``), None where neither takes it.  16-bit rows go where less time is expected, ``rf_gemm_w4``'s cost being 1.3 us after 2.5
    (16 x 37,888 x 3,584: 21.5 us there, 28.6 on the tensor cores; 32: 38.9, 28.8; 32 x 4,608 x 3,584: 8.3, 9.5; 64: 12.5, 10.1; 32 x 896 x
    4,864: 6.2, 6.7; 128: 10.7, 8.2).  Above 128 tokens only the tensor cores are looked at, without ``tensor_cores`` never."""
    few = _w4_few(q8, M, N, K, group, clusters_of) if q8 or M <= 128 or not tensor_cores else None
    if q8 or not tensor_cores:
        return few and few[1:]
    tiled = _w4_tc(M, N, K, group, clusters_of)
    return tiled[1:] if few is None or 2.5 + 1.3 * few[0] > tiled[0] else few[1:]


def q8_rows_at_once(M: int, N: int, K: int, group: int, clusters_of):
    """How many of ``M`` rows in 8 bits one launch takes: all, or where rows are so long that they do not lie in shared memory together
    (100,000 columns and 32 rows, 140,000 and 8), the most of 16, 8, .. 1 that do; None where one does not (beyond 400,000)."""
    return next((m for m in (M, 16, 8, 4, 2, 1) if m <= M and w4_launch(True, m, N, K, group, clusters_of)), None)


@functools.lru_cache(None)
def _clusters_on(device: int):
    return functools.partial(w4_clusters, device=device)


def gemm_w4(x, w: W4Weight, bias: torch.Tensor | None = None, *, out: torch.Tensor | None = None, out_f32: bool = False,
            accumulate: bool = False, tensor_cores: bool = True) -> torch.Tensor:
    """y = x @ w.T (+ bias) with 4-bit weights, 32-bit sums.

    ``x``: ``Q8Rows`` of the weight's K and group (products inside a group are exact, in whole numbers), or a tensor [M, K] in bfloat16
    or float32.  out_f32: the result is float32 whatever the rows; accumulate: added into ``out`` (float32, apart from ``x``);
    tensor_cores: whether the tcgen05 kernels may take it (as in ``gemm_plain``).

    8-bit rows stay what they are for any number of them, though from some 40 on bfloat16 rows take less time (``W4_FEW_TOKENS``).  Few
    bfloat16 rows: a group's sum is formed before its scale, so numbers of 2^118 and more may overflow where the scaled sum would not.
    float32 rows multiply weights written out in float32: a buffer of that size for the call, and its time (37,888 x 3,584 239 us)."""
    q8 = type(x) is Q8Rows
    if not (q8 or isinstance(x, torch.Tensor)) or type(w) is not W4Weight:
        raise KernelError("gemm_w4: x must be Q8Rows or a tensor, w a W4Weight")
    dt = x.dtype
    code = dtype_code(dt)
    if q8:
        M, K, at, index, ld = x.T, x.K, x.at, x.index, padded_columns(x.K, x.group)
        if x.group != w.group:
            raise KernelError(f"gemm_w4: rows in groups of {x.group}, the weight in groups of {w.group}")
    else:
        need(x.dim() == 2 and x.stride(1) == 1, "gemm_w4: x must be [M, K] with unit inner stride")
        M, K = x.shape
        at, index, ld = x.data_ptr(), x.get_device(), x.stride(0)
    here, N = _device_for(index), w.N
    if index != here or w.index != here:
        _elsewhere("gemm_w4", w.index if index == here else index)
    if K != w.K:
        raise KernelError(f"gemm_w4: inner sizes differ ({K} vs {w.K})")
    bias_at, bias_f32 = None, False
    if bias is not None:
        bias_at, bias_f32 = bias.data_ptr(), bias.dtype == torch.float32
        need(bias.shape == (N,) and (bias_f32 or bias.dtype == torch.bfloat16) and bias.is_contiguous(), "gemm_w4: bias must be [N]")
        if bias.get_device() != here:
            _elsewhere("gemm_w4", bias.get_device())
    f32 = out_f32 or accumulate or code == 0
    if out is None:
        need(not accumulate, "gemm_w4: accumulate needs an output tensor")
        out = torch.empty(M, N, dtype=torch.float32 if f32 else dt, device=w.packed.device)
    else:
        need(out.shape == (M, N) and out.dtype == (torch.float32 if f32 else dt) and out.is_contiguous(),
             "gemm_w4: output must be [M, N], contiguous, of the result's dtype")
        if out.get_device() != here:
            _elsewhere("gemm_w4", out.get_device())
    if M == 0:
        return out
    if code == 0 and not q8:
        return _gemm_by_wide_weights(x, w, bias, out, accumulate, tensor_cores)
    on = _clusters_on(here)
    plan = w4_launch(q8, M, N, K, w.group, on, tensor_cores)
    if plan is None:
        if not q8:
            return _gemm_by_wide_weights(x, w, bias, out, accumulate, tensor_cores)
        step = q8_rows_at_once(M, N, K, w.group, on)
        if step is None:
            raise KernelError(f"gemm_w4: rows of {K} columns are too long")
        for lo in range(0, M, step):
            rows = Q8Rows(x.q[lo:lo + step], x.scales[lo:lo + step], K, x.group, dt)
            gemm_w4(rows, w, bias, out=out[lo:lo + step], out_f32=out_f32, accumulate=accumulate)
        return out
    if len(plan) == 5:
        done = _f("rf_gemm_w4")(0 if q8 else 1, at, x.scales_at if q8 else None, ld, w.at, w.scales_at, bias_at, bias_f32, out.data_ptr(), f32, accumulate,
                                *plan, M, N, K, w.group, stream())
    else:
        rows_fit = at % 16 == 0 and ld % 8 == 0 and ld >= K             # the kernels copy whole 16 bytes
        most = W4_TC_MOST_F32 * (2 if K > 2 * SUM_COLUMNS else 1) if f32 and K > SUM_COLUMNS else W4_TC_MOST
        if M > most and rows_fit and out.data_ptr() % 16 == 0 and tc.supported(M, N, K, tc.STORE):      # (its results leave by TMA too)
            return _gemm_by_wide_weights(x, w, bias, out, accumulate)
        if not rows_fit:                                 # (64 x 37,888 x 3,583 by rf_gemm_w4, which would take them: 100 us)
            x, rows = torch.empty(M, (K + 7) // 8 * 8, dtype=dt, device=x.device), x
            x[:, :K] = rows
            at, ld = x.data_ptr(), x.stride(0)
        done = _f("rf_gemm_w4_tc")(at, ld, w.at, w.scales_at, bias_at, bias_f32, out.data_ptr(), f32, accumulate,
                                   *plan, M, N, K, w.group, tc.status_word(w.packed.device).data_ptr(), stream())
    check(done, "gemm_w4" if done == 0 else f"gemm_w4 ({M}x{N}x{K}, groups of {w.group})")
    return out


def _gemm_by_wide_weights(x, w, bias, out, accumulate, tensor_cores=True):
    """The product by the weights written out in the rows' dtype (exactly, with scales of five significant bits)."""
    from .basic import gemm_plain
    K = x.shape[1]
    if x.dtype == torch.float32 or not tensor_cores:
        return gemm_plain(x, dequantize_w4(w, x.dtype), bias, out=out, out_f32=out.dtype == torch.float32, accumulate=accumulate, tensor_cores=tensor_cores)
    m = tc.RESIDUAL if accumulate else tc.F32 if out.dtype == torch.float32 else tc.STORE
    pieces = 1 if m == tc.STORE else (K + SUM_COLUMNS - 1) // SUM_COLUMNS
    step = (K + 64 * pieces - 1) // (64 * pieces) * 64
    for lo in range(0, K, step):
        hi = min(K, lo + step)
        tc.gemm_tc(x[:, lo:hi], dequantize_w4(w, x.dtype, (lo, hi)), bias if lo == 0 else None, mode=m if lo == 0 else tc.RESIDUAL, out=out)
    return out

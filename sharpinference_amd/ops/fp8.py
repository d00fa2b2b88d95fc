"""Rows, products, feed-forwards and layers of routed experts in 8-bit floating point.

A row is cut into blocks of 128 values; a block has one scale, a power of two 2^(s - 127) with the byte s from 1 to 247, the smallest with which
the block's largest finite magnitude is at most 448; its values are stored as e4m3 (``torch.float8_e4m3fn``), rounded to nearest even.
Infinities and NaN become NaN.  Weights are quantised by their rows (over k) when a program loads them, activations row by row in the call.  The matrix
instruction applies both scales and adds in float; its results are offered as bfloat16 only, since of eight products on end it cuts those that
are some 2^-13 of the largest.

``x`` of a product is a bfloat16 or float32 tensor [M, K], or rows that ``quantize_rows`` made."""
from __future__ import annotations

import contextlib
import functools
import threading
from typing import Optional, Tuple, Union

import torch

from . import ACT_SILU, KernelError, _code, _dev, _i32, _known_act_pair, _need, _ptr, _run, compute_units

FP8_BLOCK = 128                # values that share a scale
FP8_TILE = 32                  # weight rows of a stored tile
FP8_FEW_ROWS = 64              # rows of the weight-streaming kernels (csrc/fp8_few.hip kFewRows)
# tokens of a layer that takes the picks as they are (us, so and sorted by expert: one of 16 experts of 5,120 x 8,192 and one always on, 8 tokens 146 and 203, 16 222 and
# 285, 17 272 and 271, 24 305 and 291; six of 64 of 2,048 x 1,408, 8 tokens 69 and 76, 16 90 and 88, 17 121 and 96)
FP8_FEW_TOKENS = 16
FP8_FEW_PAIRS = 512            # (token, pick) pairs of the same (kFewPairs)
FP8_LAYER_COLUMNS = 32         # columns of the sum that a block takes (16 kLayerTiles)
FP8_MAX_EXPERTS = 1023         # experts of a layer, one more may be always on (kFewExperts, kMaxGroups)
FP8_MOST_K = (1 << 24) - 1     # columns of a row (kF8MostK)
FP8_TILE_REACH = (1 << 32) - 1 # bytes of codes that the loads of a tile's rows reach
# rows of bfloat16 that the weight-streaming kernels quantise where they read them, in every block, instead of in a launch ahead (us of a layer's launches, staged
# and ahead: an expert of 16 of 5,120 x 8,192 and one always on, 1 token 54.6 and 55.8, 2 73.0 and 76.3, 4 108.7 and 103.6, 8 164 and 142; six of 64 of 2,048 x 1,408, 1 token
# 26.0 and 28.1, 2 35.9 and 38.6, 4 51.7 and 49.5)
FP8_STAGED_ROWS = 2
FP8_STAGED_COLUMNS = 32768     # columns of a single product that does (5,120 x 7,168, 1 row 9.6 and 11.1; 5,120 x 202,048, 1 row 166 and 156)
FP8_STAGED_BYTES = 48 * 1024   # LDS for rows that are quantised where they are read (kStagedMost)
_F32, _BF16 = _code(torch.float32), _code(torch.bfloat16)
_X_CODES = 2                   # csrc/fp8_few.hip X_CODES


def _blocks(k: int) -> int:
    return -(-k // FP8_BLOCK)


def _scale_stride(k: int) -> int:
    return -(-_blocks(k) // 4) * 4


def _padded(n: int) -> int:
    return -(-n // FP8_TILE) * FP8_TILE


def _powers(s: torch.Tensor) -> torch.Tensor:
    """2^(s - 127) of scale bytes, exactly."""
    return (s.int() << 23).view(torch.float32)


def _device_of(t: torch.Tensor):
    """The launches of a call go to its tensors' device."""
    return _NOTHING if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


_NOTHING = contextlib.nullcontext()
# (the handle of a device's current stream without a Stream object around it: 0.1 us for 2.8)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_of(t: torch.Tensor) -> int:
    """The current stream of the tensor's device."""
    return _raw_stream(t.device.index) if _raw_stream is not None else torch.cuda.current_stream(t.device).cuda_stream


class _Scratch:
    """Buffers of one call in one allocation, by address: what a call's launches hand to one another."""

    __slots__ = ("memory", "base", "size")

    def __init__(self):
        self.memory, self.base, self.size = None, 0, 0

    def add(self, nbytes: int) -> int:
        """Offset of a further buffer of so many bytes, on a border of 256."""
        at = self.size
        self.size = at + -(-nbytes // 256) * 256
        return at

    def make(self, device) -> None:
        self.memory = torch.empty(max(self.size, 1), dtype=torch.uint8, device=device)
        self.base = self.memory.data_ptr()

    def __getitem__(self, at: int) -> int:
        return self.base + at


def _same_device(*ts) -> None:
    first = ts[0].device
    for t in ts:
        if t.device != first:
            raise KernelError("operands must live on one device")


class Fp8Rows:
    """Rows [M, K] in 8 bits: ``codes`` float8_e4m3fn [M, K up to whole blocks of 128] (zeros behind K) and ``scales`` uint8 [M, blocks up to
    a multiple of 4] (127 behind the last block).  ``values()`` gives what they stand for."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, k: int):
        _need(codes.dim() == 2 and codes.dtype == torch.float8_e4m3fn and codes.shape[1] == _blocks(k) * FP8_BLOCK,
              "Fp8Rows: codes must be float8_e4m3fn [M, K up to whole blocks]")
        _need(scales.dtype == torch.uint8 and tuple(scales.shape) == (codes.shape[0], _scale_stride(k)) and scales.device == codes.device,
              "Fp8Rows: scales must be uint8 [M, blocks up to a multiple of 4] beside the codes")
        self.codes, self.scales, self.shape = codes, scales, (codes.shape[0], int(k))

    @property
    def device(self):
        return self.codes.device

    def values(self) -> torch.Tensor:
        M, k = self.shape
        s = _powers(self.scales[:, :_blocks(k)])
        return (self.codes.float().view(M, _blocks(k), FP8_BLOCK) * s[..., None]).reshape(M, -1)[:, :k]


class Fp8Weight:
    """A matrix [N, K] (or a stack [E, N, K]) in 8 bits, in the order the kernels read it: ``codes`` uint8 [(E,) tiles of 32 rows, blocks, 4096] and
    ``scales`` uint8 [(E,) tiles, blocks / 4, 32, 4].  ``gated``: N = 2 I, gate rows then up rows, each half in tiles of its own."""

    __slots__ = ("codes", "scales", "shape", "gated")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, gated: bool):
        self.codes, self.scales, self.shape, self.gated = codes, scales, tuple(shape), bool(gated)
        lead, tiles, K = self.shape[:-2], self.stored_rows // FP8_TILE, self.shape[-1]
        _need(codes.dtype == scales.dtype == torch.uint8 and codes.device == scales.device and codes.is_contiguous() and scales.is_contiguous()
              and tuple(codes.shape) == (*lead, tiles, _blocks(K), FP8_TILE * FP8_BLOCK) and tuple(scales.shape) == (*lead, tiles, _scale_stride(K) // 4, FP8_TILE, 4),
              f"Fp8Weight: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not those of {self.shape}")

    def dim(self) -> int:
        return len(self.shape)

    @property
    def device(self):
        return self.codes.device

    @property
    def stored_rows(self) -> int:
        """Rows of one matrix as they are stored, filled up with zeros."""
        return 2 * _padded(self.shape[-2] // 2) if self.gated else _padded(self.shape[-2])

    def select(self, e: int) -> "Fp8Weight":
        """Matrix e of a stack (a view)."""
        return Fp8Weight(self.codes[e], self.scales[e], self.shape[1:], self.gated)

    def values(self) -> torch.Tensor:
        """float32 [(E,) N, K]: what the codes stand for (a copy, for tests and other kernels)."""
        if self.dim() == 3:
            return torch.stack([self.select(e).values() for e in range(self.shape[0])])
        N, K = self.shape
        R, U = self.stored_rows, _blocks(K)
        c = self.codes.view(torch.float8_e4m3fn).view(R // 32, U, 2, 2, 2, 32, 16).float().permute(0, 5, 1, 2, 4, 3, 6).reshape(R, U, FP8_BLOCK)
        s = self.scales.permute(0, 2, 1, 3).reshape(R, -1)[:, :U]
        v = (c * _powers(s)[..., None]).reshape(R, -1)[:, :K]
        return torch.cat([v[:N // 2], v[R // 2:R // 2 + N // 2]]) if self.gated else v[:N]


def _pack(codes: torch.Tensor, scales: torch.Tensor, gated: bool, dst_codes: torch.Tensor, dst_scales: torch.Tensor) -> None:
    """Matrices: codes uint8 [E, N, K], scales uint8 [E, N, blocks], into the stored order."""
    (E, N, K), U = codes.shape, scales.shape[2]
    R, U4 = dst_codes.shape[1] * FP8_TILE, dst_scales.shape[2]
    halves = ((0, 0, N // 2), (N // 2, R // 2, N // 2)) if gated else ((0, 0, N),)
    rows, bytes_ = codes.contiguous(), scales
    if R != N or K != U * FP8_BLOCK or rows.data_ptr() % 8:
        rows = codes.new_zeros(E, R, U * FP8_BLOCK)
        for src, dst, n in halves:
            rows[:, dst:dst + n, :K].copy_(codes[:, src:src + n])
    if R != N or U != U4 * 4:
        bytes_ = scales.new_full((E, R, U4 * 4), 127)
        for src, dst, n in halves:
            bytes_[:, dst:dst + n, :U].copy_(scales[:, src:src + n])
    # [tile, row, block, half, group, piece, 16] -> [tile, block, half, piece, group, row, 16], the 16 bytes as two words
    dst_codes.view(torch.int64).view(E, R // 32, U, 2, 2, 2, 32, 2).copy_(rows.view(torch.int64).view(E, R // 32, 32, U, 2, 2, 2, 2).permute(0, 1, 3, 4, 6, 5, 2, 7))
    dst_scales.copy_(bytes_.reshape(E, R // 32, 32, U4, 4).permute(0, 1, 3, 2, 4))


def _new_weight(shape, gated: bool, device) -> Fp8Weight:
    _need(len(shape) in (2, 3) and min(shape) > 0 and (len(shape) == 2 or shape[0] <= FP8_MAX_EXPERTS + 1),
          f"8-bit weights must be [N, K] or [E, N, K] with at most {FP8_MAX_EXPERTS + 1} matrices")
    N, K = shape[-2:]
    _need(not gated or N % 2 == 0, "a gated matrix holds gate rows, then as many up rows")
    _need(K <= FP8_MOST_K, f"8-bit rows have up to {FP8_MOST_K} columns")
    R = 2 * _padded(N // 2) if gated else _padded(N)
    _need(R * _blocks(K) <= 0x7fffffff, f"8-bit weights [{N}, {K}] are too large")
    lead = tuple(shape[:-2])
    return Fp8Weight(torch.empty(*lead, R // 32, _blocks(K), FP8_TILE * FP8_BLOCK, dtype=torch.uint8, device=device),
                     torch.empty(*lead, R // 32, _scale_stride(K) // 4, FP8_TILE, 4, dtype=torch.uint8, device=device), shape, gated)


def fp8_weight(codes: torch.Tensor, scales: torch.Tensor, gated: bool = False) -> Fp8Weight:
    """A stored matrix in the kernels' order: codes float8_e4m3fn [(E,) N, K] and scales uint8 [(E,) N, K / 128 rounded up], the exponent bytes
    (1 .. 254: 2^(s - 127)) of each row's blocks.  ``gated``: gate rows, then up rows of a feed-forward."""
    _need(codes.dtype == torch.float8_e4m3fn and codes.dim() in (2, 3), "fp8_weight: codes must be float8_e4m3fn [N, K] or [E, N, K]")
    _need(scales.dtype == torch.uint8 and tuple(scales.shape) == (*codes.shape[:-1], _blocks(codes.shape[-1])) and scales.device == codes.device,
          "fp8_weight: scales must be uint8, one for each row's block of 128, beside the codes")
    w = _new_weight(tuple(codes.shape), gated, codes.device)
    if codes.dim() == 2:
        _pack(codes.view(torch.uint8)[None], scales[None], gated, w.codes[None], w.scales[None])
        return w
    at_once = max(1, (1 << 30) // (w.stored_rows * _blocks(codes.shape[2]) * FP8_BLOCK))      # (matrices: what is filled up is a copy of them)
    for e in range(0, codes.shape[0], at_once):
        some = slice(e, e + at_once)
        _pack(codes[some].view(torch.uint8), scales[some], gated, w.codes[some], w.scales[some])
    return w


def empty_fp8_weight(shape, gated: bool, device) -> Fp8Weight:
    """Room for a matrix [N, K] or a stack [E, N, K], to be filled by ``quantize_into`` (its own or ``select(e)``)."""
    return _new_weight(tuple(int(n) for n in shape), gated, device)


def quantize_into(dst: Fp8Weight, w: torch.Tensor) -> None:
    """A bfloat16 or float32 matrix on the GPU, quantised (``quantize_rows`` of its rows) into dst [N, K] of its shape."""
    _need(dst.dim() == 2 and tuple(w.shape) == dst.shape and w.device == dst.device, f"quantize_into: a matrix {dst.shape} on the destination's device is wanted")
    _quantize(dst, w)


def _quantize(dst: Fp8Weight, w: torch.Tensor) -> None:
    w = w.contiguous()
    _dev(w, dst.codes)
    with _device_of(w):
        _run("sharpi_fp8_weight", w.data_ptr(), _code(w.dtype), dst.codes.data_ptr(), dst.scales.data_ptr(), 1 if w.dim() == 2 else w.shape[0], *w.shape[-2:],
             int(dst.gated), _stream_of(w))


def quantize_weight(w: torch.Tensor, gated: bool = False) -> Fp8Weight:
    """A bfloat16 or float32 matrix [(E,) N, K] on the GPU in 8 bits, in the kernels' order."""
    _need(w.is_cuda and w.dim() in (2, 3), "quantize_weight: a matrix [N, K] or a stack [E, N, K] on the GPU")
    out = _new_weight(tuple(w.shape), gated, w.device)
    _quantize(out, w)
    return out


_SWITCH = threading.local()


def feed_forwards_in_8_bits(on: bool) -> None:
    """Whether gated feed-forwards, dense and routed, keep bfloat16 matrices in 8 bits (half of the bytes of a decode step's largest reads) and run
    through ``feed_forward_fp8`` and ``experts_fp8``.  Read when weights are loaded, by the thread that loads them: it holds for the calling thread alone, so that
    engines loaded side by side have each their own."""
    _SWITCH.on = bool(on)


def feed_forwards_are_8_bits() -> bool:
    return getattr(_SWITCH, "on", False)


def _new_rows(M: int, k: int, device) -> Fp8Rows:
    q = object.__new__(Fp8Rows)
    q.codes = torch.empty((M, _blocks(k) * FP8_BLOCK), dtype=torch.float8_e4m3fn, device=device)
    q.scales = torch.empty((M, _scale_stride(k)), dtype=torch.uint8, device=device)
    q.shape = (M, k)
    return q


def quantize_rows(x: torch.Tensor, act=None) -> Fp8Rows:
    """x [M, K] (bfloat16 or float32) in 8 bits; with ``act`` (ACT_SILU, ACT_GELU_TANH or (ACT_SWISH_CLAMP, limit)) x [M, 2I] holds gate
    columns, then up columns, and the rows are act(g) * u, rounded to x's type first (what ``gated_act`` stores)."""
    _dev(x)
    _need(x.dim() == 2 and x.shape[1] > 0, "quantize_rows: x must be [M, K]")
    dt = _code(x.dtype)
    code, limit = (0, 0.0) if act is None else _known_act_pair(act)
    _need(not code or x.shape[1] % 2 == 0, "quantize_rows: a gated input is [M, 2I]")
    M, K = x.shape[0], x.shape[1] // (2 if code else 1)
    if K > FP8_MOST_K or M >= 1 << 31:
        raise KernelError(f"quantize_rows: up to {FP8_MOST_K} columns")
    out = _new_rows(M, K, x.device)
    with _device_of(x):
        _run("sharpi_fp8_rows", x.data_ptr(), dt, out.codes.data_ptr(), out.scales.data_ptr(), M, K, code, limit, _stream_of(x))
    return out


def _staged(x) -> bool:
    """Whether the weight-streaming kernels quantise these rows where they are read: a few rows of bfloat16 that fit in LDS."""
    return (isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16 and x.shape[0] <= FP8_STAGED_ROWS and x.shape[1] % 8 == 0 and x.data_ptr() % 16 == 0
            and x.shape[0] * _blocks(x.shape[1]) * (FP8_BLOCK + 1) + 16 <= FP8_STAGED_BYTES)


class _Operand:
    """The rows of a product as its kernel takes them: (address, scales' address, kind); quantised into the call's scratch memory if they are
    not codes yet and ``staged`` does not hold."""

    __slots__ = ("x", "staged", "codes_at", "scales_at")

    def __init__(self, x, scratch: _Scratch, staged: bool):
        self.x, self.staged = x, staged
        if isinstance(x, torch.Tensor) and not staged:
            M, k = x.shape
            self.codes_at, self.scales_at = scratch.add(M * _blocks(k) * FP8_BLOCK), scratch.add(M * _scale_stride(k))

    def ready(self, scratch: _Scratch, stream: int) -> Tuple[int, Optional[int], int]:
        x = self.x
        if not isinstance(x, torch.Tensor):
            return x.codes.data_ptr(), x.scales.data_ptr(), _X_CODES
        if self.staged:
            return x.data_ptr(), None, _code(x.dtype)
        codes, scales = scratch[self.codes_at], scratch[self.scales_at]
        _run("sharpi_fp8_rows", x.data_ptr(), _code(x.dtype), codes, scales, x.shape[0], x.shape[1], 0, 0.0, stream)
        return codes, scales, _X_CODES


def _rows_checked(x, k: int, who: str) -> None:
    if isinstance(x, Fp8Rows):
        _dev(x.codes, x.scales)
    else:
        _dev(x)
        _code(x.dtype)
    if len(x.shape) != 2 or x.shape[1] != k:
        raise KernelError(f"{who}: x {tuple(x.shape)} does not fit weights over {k} columns")


def linear_fp8(x: Union[torch.Tensor, Fp8Rows], w: Fp8Weight) -> torch.Tensor:
    """x [M, K] W^T in 8 bits: bfloat16 [M, N].  A few rows go by streaming the weights (one or two of bfloat16 in a launch), more in tiles (``few_rows_fp8``,
    ``tile_fp8``)."""
    _need(isinstance(w, Fp8Weight) and w.dim() == 2 and not w.gated, "linear_fp8: w must be an Fp8Weight [N, K], not gated")
    N, K = w.shape
    _rows_checked(x, K, "linear_fp8")
    M = x.shape[0]
    _same_device(w.codes, x if isinstance(x, torch.Tensor) else x.codes)
    out = torch.empty((M, N), dtype=torch.bfloat16, device=w.codes.device)
    if M == 0:
        return out
    few = few_rows_fp8(M, N)
    scratch = _Scratch()
    rows = _Operand(x, scratch, few and N <= FP8_STAGED_COLUMNS and _staged(x))
    product = None if few else _Tiled(M, N, K, scratch)
    if scratch.size:
        scratch.make(out.device)
    with _device_of(out):
        stream = _stream_of(out)
        a, scales, kind = rows.ready(scratch, stream)
        if few:
            _run("sharpi_fp8_few", a, scales, kind, w.codes.data_ptr(), w.scales.data_ptr(), w.stored_rows, out.data_ptr(), M, N, K,
                 _few_tiles(N), stream)
        else:
            product.run(a, scales, w, out, scratch, stream)
    return out


class _Tiled:
    """A product of many rows by one matrix in tiles; where these are few, shares of k go side by side and are added up behind them."""

    __slots__ = ("shape", "height", "nt", "shares", "part_at")

    def __init__(self, M: int, N: int, K: int, scratch: _Scratch):
        self.shape = (M, N, K)
        self.height, self.nt, self.shares = tile_fp8(M, N, K, False, compute_units())
        if self.shares > 1:
            self.part_at = scratch.add(self.shares * M * N * 4)

    def run(self, codes: int, scales: int, w: Fp8Weight, out: torch.Tensor, scratch: _Scratch, stream: int) -> None:
        M, N, K = self.shape
        whole = self.shares == 1
        to = out.data_ptr() if whole else scratch[self.part_at]
        _run("sharpi_fp8_tiles", codes, scales, M, w.codes.data_ptr(), w.scales.data_ptr(), w.stored_rows, to, _BF16 if whole else _F32, M, N, K,
             None, None, 1, 0, self.height, self.nt, self.shares, stream)
        if not whole:
            _run("sharpi_fp8_join", to, out.data_ptr(), M * N, self.shares, stream)


def few_rows_fp8(M: int, N: int) -> bool:
    """Whether a product of M rows goes by streaming the weights: up to 16 rows always; then while the rows' blocks of 16 times the columns are few (us,
    streamed and in tiles, K 5,120: 7,168 columns 48 rows 19 and 30, 64 rows 22 and 31; 16,384 columns 32 rows 27 and 33, 64 rows 38 and 36; 65,536 columns 16
    rows 62 and 71, 24 rows 82 and 66)."""
    return M <= 16 or (M <= FP8_FEW_ROWS and -(-M // 16) * N <= 49152)


def _few_tiles(N: int) -> int:
    """Half tiles of 16 weight rows a block takes: two where that leaves blocks for half of the compute units (us, one and two, 16 rows: 5,120 x 5,120 14.1
    and 11.8, 65,536 x 5,120 85 and 62, 4,096 x 14,336 19.4 and 23.5, 1,024 x 2,048 7.0 and 7.6)."""
    return 2 if N >= 4608 else 1


# us that a step of 64 of k takes in a tile, where it runs alone on the chip and where all compute units do, by (rows / 64, columns / 128); tiles of up to 128
# rows in pairs of blocks a unit
TILE_STEP_US = {(1, 1): (0.24, 0.36), (2, 1): (0.28, 0.39), (3, 1): (0.39, 0.41), (4, 1): (0.42, 0.53), (3, 2): (0.50, 0.60), (4, 2): (0.59, 0.75)}
PAIRED_STEP_US = {1: (0.38, 0.62), 2: (0.42, 0.86)}
TILE_END_US = 5.0


JOIN_US, JOIN_TBS = 3.0, 6.0      # adding shares up: a launch, and the rate at which they are written and read again


def _highest(K: int) -> int:
    """Rows of a tile at most, which its loads have to reach: 256, or 192 of the widest."""
    return min(256, FP8_TILE_REACH // (_blocks(K) * FP8_BLOCK) // 64 * 64)


@functools.lru_cache(maxsize=1024)
def tile_fp8(M: int, N: int, K: int, gated: bool, units: int) -> Tuple[int, int, int]:
    """(rows, columns / 128, shares of k) of the tiles of a product of many rows (gated: 256 columns, one share): those whose rounds of the chip take the
    least time."""
    def expected(height: int, nt: int, shares: int) -> float:
        steps = 2 * -(-_blocks(K) // shares)
        blocks = -(-M // height) * -(-N // (128 if gated else 128 * nt)) * shares
        tall = -(-min(M, height) // 64)
        low, full = PAIRED_STEP_US[tall] if height <= 128 else TILE_STEP_US[(tall, nt)] if (tall, nt) in TILE_STEP_US else TILE_STEP_US[(3, nt)]
        at_once = 2 * units if height <= 128 else units
        rounds, rest = divmod(blocks, at_once)
        us = rounds * (full * steps + TILE_END_US)
        if rest:
            fill = float(rest > units) if height <= 128 else rest / units        # (a unit with a pair takes as long as all of them)
            us += (low + (full - low) * fill) * steps + TILE_END_US
        return us + (JOIN_US + 8e-6 * shares * M * N / JOIN_TBS if shares > 1 else 0.0)
    choices = [(64, 2), (128, 2), (192, 2), (256, 2)] + ([] if gated else [(192, 1), (256, 1)])
    most = 1 if gated else min(8, max(1, _blocks(K) // 4))
    return min(((h, nt, s) for h, nt in choices if h <= _highest(K) for s in range(1, most + 1)), key=lambda c: expected(*c))


def grouped_tile_fp8(K: int) -> int:
    """Rows of the tiles of a layer's products at most: over a short k in pairs of blocks a unit, which fill each other's gaps at a tile's start and end (us, tiles of
    128 and of 256: 64 experts of 2 x 1,408 x 2,048, 94 rows each 108 and 119, 188 159 and 167; 128 of 2 x 768 x 2,048, 125 rows 137 and 146; 16 of 16,384 x 5,120, 38 rows
    276 and 260, 128 383 and 364; 32 of 5,760 x 2,880, 38 rows 128 and 120, 375 362 and 347).  Of 72 launches timed both ways those it
    chooses take 1.7 % more than the faster ones in the mean (always 256: 3.7 %)."""
    return 128 if K <= 2048 else _highest(K)


def _layer_checked(x, w_gate_up: Fp8Weight, w_down: Fp8Weight, dims: int, who: str):
    if not (isinstance(w_gate_up, Fp8Weight) and isinstance(w_down, Fp8Weight) and w_gate_up.dim() == w_down.dim() == dims
            and w_gate_up.gated and not w_down.gated):
        raise KernelError(f"{who}: w_gate_up must be a gated Fp8Weight and w_down a plain one, both {'[E, N, K]' if dims == 3 else '[N, K]'}")
    inner, K = w_gate_up.shape[-2] // 2, w_gate_up.shape[-1]
    if w_down.shape != (*w_gate_up.shape[:-2], w_down.shape[-2], inner):
        raise KernelError(f"{who}: w_gate_up {w_gate_up.shape} and w_down {w_down.shape} do not fit")
    _rows_checked(x, K, who)
    _same_device(w_gate_up.codes, w_down.codes, x if isinstance(x, torch.Tensor) else x.codes)
    return x.shape[0], K, inner, w_down.shape[-2]


def _few_layer(x, ids, wts, w1: Fp8Weight, w2: Fp8Weight, code: int, limit: float, on_input: bool, shared: bool, E: int) -> torch.Tensor:
    T, K, inner, N = x.shape[0], w1.shape[-1], w1.shape[-2] // 2, w2.shape[-2]
    k, also = 1 if ids is None else ids.shape[1], 1 if shared else 0
    rows, stride = T * k + also * T, -(-inner // 8) * 8
    met = min(E, T * k) + also if ids is not None else 1
    tiles = -(-N // FP8_LAYER_COLUMNS)
    shares = sum_shares(tiles, met * _blocks(inner), compute_units())
    row_blocks = 1 if T <= 16 else 2 if T <= 32 else 4
    scratch = _Scratch()
    h, counters = scratch.add(rows * stride * 2), scratch.add(tiles * 4)
    part = scratch.add(shares * tiles * FP8_LAYER_COLUMNS * row_blocks * 64 if shares > 1 else 0)
    operand = _Operand(x, scratch, _staged(x))
    if T > FP8_STAGED_ROWS:
        codes, scales_at = scratch.add(rows * _blocks(stride) * FP8_BLOCK), scratch.add(rows * _scale_stride(stride))
    scratch.make(w1.codes.device)
    out = torch.empty((T, N), dtype=torch.bfloat16, device=w1.codes.device)
    stream, ids_at = _stream_of(out), _ptr(ids)
    a, scales, kind = operand.ready(scratch, stream)
    w_in, w_out = (_ptr(wts), None) if on_input else (None, _ptr(wts))
    _run("sharpi_fp8_few_gated", a, scales, kind, w1.codes.data_ptr(), w1.scales.data_ptr(), w1.stored_rows, scratch[h], stride, ids_at, w_in,
         T, k, E, also, inner, K, code, limit, scratch[counters], tiles, stream)
    a, scales, kind = scratch[h], None, _BF16
    if T > FP8_STAGED_ROWS:
        a, scales, kind = scratch[codes], scratch[scales_at], _X_CODES
        _run("sharpi_fp8_rows", scratch[h], _BF16, a, scales, rows, stride, 0, 0.0, stream)
    _run("sharpi_fp8_few_sum", a, scales, kind, w2.codes.data_ptr(), w2.scales.data_ptr(), w2.stored_rows, out.data_ptr(), ids_at, w_out, T, k, E,
         also, N, stride, shares, scratch[part], scratch[counters], stream)
    return out


def sum_shares(tiles: int, blocks: int, units: int) -> int:
    """Shares of the blocks of k that a layer's second product is dealt to for each column tile: about two blocks a compute unit, of eight or more."""
    return max(1, min(2 * units // tiles, blocks // 8))


def feed_forward_fp8(x: Union[torch.Tensor, Fp8Rows], w_gate_up: Fp8Weight, w_down: Fp8Weight, act=ACT_SILU) -> torch.Tensor:
    """A gated feed-forward in 8 bits: h = act(g) * u with (g | u) = x W_gate_up^T, rounded to bfloat16 and quantised again, then h W_down^T: bfloat16
    [M, N].  Up to 64 rows by streaming the weights, in two launches (up to two rows of bfloat16) to four; more rows: the quantised h is the first product's
    epilogue."""
    M, K, inner, N = _layer_checked(x, w_gate_up, w_down, 2, "feed_forward_fp8")
    code, limit = _known_act_pair(act)
    with _device_of(w_down.codes):
        if M == 0:
            return torch.empty(0, N, dtype=torch.bfloat16, device=w_down.device)
        if M <= FP8_FEW_ROWS:
            return _few_layer(x, None, None, w_gate_up, w_down, code, limit, False, False, 1)
        scratch = _Scratch()
        operand = _Operand(x, scratch, False)
        codes, scales = scratch.add(M * _blocks(inner) * FP8_BLOCK), scratch.add(M * _scale_stride(inner))
        down = _Tiled(M, N, inner, scratch)
        scratch.make(w_down.codes.device)
        out = torch.empty((M, N), dtype=torch.bfloat16, device=w_down.codes.device)
        stream = _stream_of(out)
        a, a_scales, _ = operand.ready(scratch, stream)
        _run("sharpi_fp8_tiles_gated", a, a_scales, M, w_gate_up.codes.data_ptr(), w_gate_up.scales.data_ptr(), w_gate_up.stored_rows, scratch[codes],
             scratch[scales], M, inner, K, None, None, 1, 0, None, code, limit, tile_fp8(M, inner, K, True, compute_units())[0], stream)
        down.run(scratch[codes], scratch[scales], w_down, out, scratch, stream)
        return out


def experts_fp8(x: Union[torch.Tensor, Fp8Rows], ids: torch.Tensor, wts: torch.Tensor, w_gate_up: Fp8Weight, w_down: Fp8Weight, act=ACT_SILU,
                score_on_input: bool = False, shared: bool = False) -> torch.Tensor:
    """A layer of routed experts in 8 bits, whole: out[t] = sum_j wts[t, j] F_e(x[t]) over the token's picks e = ids[t, j], with F_e the gated
    feed-forward of matrix e (see ``feed_forward_fp8``); with ``score_on_input`` the pick's score multiplies g and u instead.  ``shared``: the stacks hold
    one more matrix behind the experts, whose feed-forward of every token is added.  ids int32 [T, k] and wts float32 [T, k] as the router
    gives them (``router_topk``); a pick outside 0 .. E - 1 adds nothing.  bfloat16 [T, N].

    Up to 16 tokens the picks are taken as they are and the weights streamed, in two launches (up to two rows of bfloat16) to four, the last of which adds
    the experts' outputs.  More tokens (up to 4 GB of codes) are sorted by expert; their outputs are kept in float until they are added."""
    T, K, inner, N = _layer_checked(x, w_gate_up, w_down, 3, "experts_fp8")
    _dev(ids, wts)
    _i32(ids, "ids")
    _need(ids.dim() == 2 and ids.shape[0] == T and ids.shape[1] > 0 and wts.shape == ids.shape and wts.dtype == torch.float32,
          "experts_fp8: ids must be int32 and wts float32 [T, k]")
    _same_device(w_down.codes, ids, wts)
    E, k = w_gate_up.shape[0] - (1 if shared else 0), ids.shape[1]
    if not (0 < E <= FP8_MAX_EXPERTS and k <= FP8_FEW_PAIRS and T * (k + 1) < 1 << 31):
        raise KernelError(f"experts_fp8: up to {FP8_MAX_EXPERTS} experts and {FP8_FEW_PAIRS} picks")
    code, limit = _known_act_pair(act)
    with _device_of(w_down.codes):
        if T == 0:
            return torch.empty(0, N, dtype=torch.bfloat16, device=w_down.device)
        if T <= FP8_FEW_TOKENS and T * k <= FP8_FEW_PAIRS:
            return _few_layer(x, ids, wts, w_gate_up, w_down, code, limit, score_on_input, shared, E)
        return _many_layer(x, ids, wts, w_gate_up, w_down, code, limit, score_on_input, shared, E, inner, N)


def _many_layer(x, ids, wts, w1: Fp8Weight, w2: Fp8Weight, code: int, limit: float, on_input: bool, shared: bool, E: int, inner: int, N: int) -> torch.Tensor:
    T, k = ids.shape
    n, along, dev = T * k, T if shared else 0, w1.codes.device
    # the picks sorted by expert (no plan: that is the bfloat16 product's); the always-on matrix takes the tokens behind them, in their order
    scratch = _Scratch()
    operand = _Operand(x, scratch, False)
    offsets, tokens, inv_pos, scores = scratch.add((E + 1) * 4), scratch.add(n * 4), scratch.add(n * 4), scratch.add(n * 4)
    codes, scales = scratch.add((n + along) * _blocks(inner) * FP8_BLOCK), scratch.add((n + along) * _scale_stride(inner))
    y = scratch.add((n + along) * N * 4)
    shared_y = y + n * N * 4
    scratch.make(dev)
    out = torch.empty((T, N), dtype=torch.bfloat16, device=dev)
    stream, K = _stream_of(out), w1.shape[-1]
    a, a_scales, _ = operand.ready(scratch, stream)
    _run("sharpi_moe_permute", ids.data_ptr(), wts.data_ptr(), scratch[offsets], scratch[tokens], scratch[scores], scratch[inv_pos], None, 0,
         T, k, E, 0, 1, stream)
    _run("sharpi_fp8_tiles_gated", a, a_scales, T, w1.codes.data_ptr(), w1.scales.data_ptr(), w1.stored_rows, scratch[codes], scratch[scales],
         n, inner, K, scratch[tokens], scratch[offsets], E, along, scratch[scores] if on_input else None, code, limit, grouped_tile_fp8(K), stream)
    _run("sharpi_fp8_tiles", scratch[codes], scratch[scales], n + along, w2.codes.data_ptr(), w2.scales.data_ptr(), w2.stored_rows, scratch[y], _F32, n, N, inner,
         None, scratch[offsets], E, along, grouped_tile_fp8(inner), 2, 1, stream)
    _run("sharpi_fp8_combine", scratch[y], scratch[inv_pos], ids.data_ptr(), scratch[shared_y] if shared else None, None if on_input else wts.data_ptr(),
         out.data_ptr(), T, N, k, E, stream)
    return out

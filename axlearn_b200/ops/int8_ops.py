"""Serving in 8 bits: rows of activations, products with 8-bit weights and a paged 8-bit KV cache (``csrc/int8_rows.cu``,
``csrc/int8_gemm.cu``, ``csrc/gemm_skinny.cu``, ``csrc/int8_cache.cu``).

A block of values with the largest magnitude ``A`` is held as whole numbers ``c = round(127 x / A)`` (ties to the even one), -127 to
127, and stands for ``c A / 127``.  A block with a NaN or an infinity in it stands for NaN, one whose ``A`` is below 2^-119 for zeros.

* ``quantize_rows``, ``add_rms_norm_int8``, ``swiglu_int8``: activations, a block a row (a token).
* ``quantize_weight`` / ``int8_linear``: ``x [..., K] @ w [K, N]``, a block a column of the weight (a channel); sums are integers.
* ``append_int8``: keys and values of new tokens into the cache (prompts, chunks, single tokens); a block is the tokens of a page of
  one KV head.  Its ``A`` grows as the page fills, and codes that are there are rounded to the new one, so a token that was
  followed by larger ones in its page is off by up to half a step for each time ``A`` grew.
* ``paged_decode_attention_int8``: one query token per sequence over the cache.
* ``prompt_attention_int8``, ``rope_decode_attention_int8``: what a prompt and a decoding step run, with the rotation of
  queries and keys and the append.

Attention sees what the cache stands for: steps ``c A / 127`` itself, prompts that value rounded to bf16 (2^-8 of it at most).
Serving only: operands that need a gradient, or carry a tangent, are refused.  CUDA tensors in bf16 go to the kernels, everything
else runs the plain statements, which are also the oracle in tests.  Places that a page table or a length gets wrong (a page that
the pool does not have, a position behind a table) are not touched: on the GPU they set the device's status word, which
``cuda_ops.check_status`` raises, on the host they are an ``IndexError``.  The 16-bit forms of these operations are
``cuda_ops.rms_norm``, ``cuda_ops.gemm`` and ``decode_ops``, those of 4 bits ``int4_ops``; the reference quantises inside its layers
(axlearn/common/quantized_dot_general/layers.py) and has no 8-bit cache.
"""

from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import NamedTuple, Optional, Union

import torch

from axlearn_b200.ops import cuda_ops, dispatch
from axlearn_b200.ops.int4_ops import (
    _aligned_rows,
    _no_gradient,
    _on,
    _on_kernel,
    _overlap,
    _read_places,
    _report_places,
    _rotate,
    _split_qkv,
)

Tensor = torch.Tensor

LEAST = 2.0 ** -119
MAX_ROW = 65536        # values of a row that the row kernels keep
MAX_K = 1 << 17        # products of 127 x 127 whose sums fit 32 bits
MAX_SPLITS = 1024      # of a sequence's keys
MAX_GRID = 65535       # sequences of an attention launch, and groups of eight query heads of one KV head
PAGE_UNIT = 16         # tokens of a page are a multiple of
# Entry points and the 64-bit words of their arguments (``csrc/int8.cuh``).
_WORDS = {"axb_int8_rows": "7q", "axb_int8_add_rms_norm": "9qd", "axb_gemm_skinny_int8": "12q", "axb_int8_gemm": "12q",
          "axb_int8_dense": "13q",
          "axb_int8_append": "25q", "axb_int8_rope_append": "20q", "axb_int8_decode_attn": "18qdq"}
_entries: dict = {}


def _entry(name: str) -> tuple:
    h = cuda_ops.lib()
    if name == "axb_int8_attn_scratch_floats":
        f, pack = h.axb_int8_attn_scratch_floats, None
        f.argtypes, f.restype = [ctypes.c_int] * 4, ctypes.c_int64
    else:
        f, pack = getattr(h, name), struct.Struct(_WORDS[name]).pack
        f.argtypes, f.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_int
    _entries[name] = f, pack
    return f, pack


def _call(device: int, name: str, *words) -> None:
    """Launches on the device of the operands (its index), on its current stream."""
    if device != cuda_ops.current_device():
        with torch.cuda.device(device):
            return _call(device, name, *words)
    f, pack = _entries.get(name) or _entry(name)
    return cuda_ops._check(f(pack(*words), cuda_ops.raw_stream(device)), name)  # pylint: disable=protected-access


def _status(device: int) -> int:
    word = cuda_ops._status.get(device)  # pylint: disable=protected-access
    return (cuda_ops.status_word(torch.device("cuda", device)) if word is None else word).data_ptr()


# ------------------------------------------------------------------------------------------
# Blocks.
# ------------------------------------------------------------------------------------------


def _tops(top: Tensor) -> Tensor:
    """Largest magnitudes as blocks have them: NaN where one is not finite, 0 below ``LEAST``."""
    return torch.where(torch.isfinite(top), torch.where(top < LEAST, 0.0, top), torch.nan)


def _codes(x: Tensor, top: Tensor, factor: int = 127) -> Tensor:
    """``round(factor x / top)`` of values and tops that broadcast, 0 where ``top`` is 0 or NaN (64 bits: no near tie is decided
    by a rounding ahead of it)."""
    top = top.double()
    level = x.double() * factor / torch.where(top > 0, top, 1.0)
    return torch.where(top > 0, level, 0.0).round().clamp(-127, 127).to(torch.int8)


class Int8Rows(NamedTuple):
    """Rows in 8 bits: ``codes [..., K]`` (int8) times ``scales [...]`` (fp32)."""

    codes: Tensor
    scales: Tensor


def row_values(rows: Int8Rows, dtype: torch.dtype = torch.float32) -> Tensor:
    """What rows stand for: ``[..., K]``."""
    return (rows.codes.float() * rows.scales[..., None]).to(dtype)


def _plain_rows(x: Tensor) -> Int8Rows:
    top = _tops(x.abs().amax(-1, keepdim=True).float())
    return Int8Rows(_codes(x, top), (top.double() / 127.0).float()[..., 0])


def _check_row(dim: int) -> None:
    if dim < 8 or dim % 8 or dim > MAX_ROW:
        raise ValueError(f"rows in 8 bits have a multiple of 8 values, up to {MAX_ROW}: {dim}")


def _row_operand(x: Tensor, dim: int) -> tuple[Tensor, int, int]:
    """``x [..., dim]`` as ``(tensor, rows, pitch)`` of 16-byte aligned rows; a copy where it does not lie that way."""
    rows = x.numel() // dim
    pitch = x.stride(0) if x.dim() == 2 and x.stride(1) == 1 and rows > 1 else dim if x.is_contiguous() else 0
    if pitch < dim or pitch % 8 or x.data_ptr() % 16:
        x, pitch = x.clone(memory_format=torch.contiguous_format), dim
    return x, rows, pitch


def quantize_rows(x: Tensor) -> Int8Rows:
    """``x [..., K]`` (K a multiple of 8) with every row a block."""
    _check_row(x.shape[-1])
    _no_gradient("quantize_rows", x)
    if not _on_kernel(x):
        return _plain_rows(x)
    return _launch_rows(x, x.shape[-1], False)


def swiglu_int8(gu: Tensor) -> Int8Rows:
    """``silu(gate) * up`` of ``gu [..., 2 F]`` (gate | up, as of one product) with every row a block of F values."""
    if gu.shape[-1] % 2:
        raise ValueError(f"gate and up are halves of a row: {tuple(gu.shape)}")
    _check_row(gu.shape[-1] // 2)
    _no_gradient("swiglu_int8", gu)
    if not _on_kernel(gu):
        gate, up = gu.float().chunk(2, -1)
        far = gate < -80  # 1 + exp(gate) is 1, and 1 + exp(-gate) about to be infinite
        return _plain_rows(torch.where(far, gate * torch.exp(gate), torch.nn.functional.silu(gate)) * up)
    return _launch_rows(gu, gu.shape[-1] // 2, True)


def _row_scales(x: Tensor) -> Tensor:
    """Room for a scale of each row (from a whole number, which torch takes 0.8 us faster than a tuple)."""
    shape = x.shape
    if len(shape) == 2:
        return x.new_empty(shape[0], dtype=torch.float32)
    return x.new_empty(shape[:-1], dtype=torch.float32)


def _launch_rows(x: Tensor, dim: int, gated: bool) -> Int8Rows:
    shape = x.shape[:-1]
    codes = x.new_empty(shape + (dim,), dtype=torch.int8)
    scales = _row_scales(x)
    if codes.numel():
        x, rows, pitch = _row_operand(x, x.shape[-1])
        _call(x.get_device(), "axb_int8_rows", x.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, dim, pitch, gated)
    return Int8Rows(codes, scales)


def add_rms_norm_int8(x: Tensor, residual: Optional[Tensor], scale: Tensor, eps: float, *, values: bool = False) -> tuple:
    """RMS norm of ``total = x + residual`` (of ``x``, where there is no residual) with weights ``scale [D]`` and every row a
    block: ``(Int8Rows, total)``, and with ``values`` also what the rows stand for, in ``x``'s type.  ``total`` is rounded to that
    type ahead of the norm, which is not rounded between its steps; ``scale`` is rounded to it, too."""
    d = x.shape[-1]
    _check_row(d)
    if scale.shape != (d,) or scale.device != x.device:
        raise ValueError(f"scale {tuple(scale.shape)} on {scale.device} for rows of {d} on {x.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} for x {tuple(x.shape)} {x.dtype}")
    _no_gradient("add_rms_norm_int8", x, residual, scale)
    if scale.dtype != x.dtype:
        scale = scale.to(x.dtype)
    if not _on_kernel(x):
        total = x if residual is None else x + residual
        t = total.float()
        y = t * scale.float()
        top = _tops(y.abs().amax(-1, keepdim=True))
        rows = Int8Rows(_codes(y, top), (top / 127.0 * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps))[..., 0])
        return (rows, total, row_values(rows, x.dtype)) if values else (rows, total)
    x, n, pitch = _row_operand(x, d)
    if pitch != d:
        x = x.contiguous()
    total, other = x, 0
    if residual is not None:
        residual = _aligned(residual)
        total, other = torch.empty_like(x), residual.data_ptr()
    scale = _aligned(scale)
    rows = Int8Rows(torch.empty_like(x, dtype=torch.int8), _row_scales(x))
    held = torch.empty_like(x) if values else None
    if n:
        _call(x.get_device(), "axb_int8_add_rms_norm", x.data_ptr(), other, scale.data_ptr(), total.data_ptr() if other else 0,
              rows.codes.data_ptr(), rows.scales.data_ptr(), held.data_ptr() if values else 0, n, d, eps)
    return (rows, total, held) if values else (rows, total)


def _aligned(x: Tensor) -> Tensor:
    """``x`` as a contiguous tensor at a multiple of 16 bytes."""
    if not x.is_contiguous() or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


# ------------------------------------------------------------------------------------------
# Weights.
# ------------------------------------------------------------------------------------------


class Int8Weight:
    """A matrix ``[K, N]`` in 8 bits: ``codes [N, K]`` (int8), a block for each of its columns, and ``scales [N]`` (fp32)."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: Tensor, scales: Tensor):
        shape = codes.shape
        if (len(shape) != 2 or codes.dtype is not torch.int8 or scales.dtype is not torch.float32 or scales.shape != shape[:1]
                or codes.get_device() != scales.get_device() or not codes.is_contiguous() or not scales.is_contiguous()):
            raise ValueError(f"codes {tuple(shape)} {codes.dtype} and scales {tuple(scales.shape)} {scales.dtype} are not those of an "
                             "8-bit weight: contiguous [N, K] int8 and [N] fp32")
        n, k = shape
        if k < 16 or k % 16 or k > MAX_K or n < 8 or n % 8:
            raise ValueError(f"an 8-bit weight [{k}, {n}] has rows in sixteens up to {MAX_K} and columns in eights")
        self.codes, self.scales, self.shape = codes, scales, (k, n)


def quantize_weight(w: Tensor) -> Int8Weight:
    """``w [K, N]`` (K a multiple of 16, N of 8) with every column a block."""
    if w.dim() != 2:
        raise ValueError(f"a weight is a matrix: {tuple(w.shape)}")
    rows = _plain_rows(w.detach().t())
    return Int8Weight(rows.codes.contiguous(), rows.scales.contiguous())


def dequantize_weight(w: Int8Weight, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``[K, N]``, rounded to ``dtype``."""
    return (w.codes.float() * w.scales[:, None]).to(dtype).t()


def pair_features(rows: int, n: int, sms: int = 148) -> int:
    """Features of a tile of 256 rows: 256, or 128 where that is fewer waves' time: a tile of 128 takes 0.62 of one of 256 (us
    with 128 / 256, rows x K x N: 256 x 2048 x 8192 9.9 / 12.5, 300 x 4096 x 12288 23.4 / 25.8, 333 x 2048 x 8192 12.8 / 12.6, 1024
    x 4096 x 4096 17.7 / 17.1, 8192 x 4096 x 4096 103 / 89)."""
    blocks, pairs = -(-rows // 256), sms // 2
    wide, narrow = -(-blocks * -(-n // 256) // pairs), -(-blocks * -(-n // 128) // pairs)
    return 128 if 5 * narrow < 8 * wide else 256


def few_rows(rows: int, k: int, n: int, sms: int = 148) -> bool:
    """Whether a product streams the weight past all rows, in slices of K where columns are few: up to 128 rows, and up to 96 where K is
    short and tiles of 256 rows by 128 columns are one wave (us so / in tiles: 96 x 4096 x 4096 11.9 / 11.6, 128 rows of it 13.5 /
    11.6, 128 x 4096 x 12288 15.9 / 18.7, 128 x 14336 x 4096 19.7 / 24.6)."""
    return rows <= 96 or (rows <= 128 and (k > 4096 or -(-n // 128) > sms // 2))


def int8_linear(x: Union[Tensor, Int8Rows], w: Int8Weight, *, out: Optional[Tensor] = None, accumulate: bool = False,
                dtype: Optional[torch.dtype] = None, resident: bool = False) -> Tensor:
    """``x [..., K] @ w`` with exact integer sums of the codes, times the scales of row and column in 32 bits, rounded to ``dtype``
    (that of ``x`` where it is a tensor, which is quantised by rows first; else bf16); into ``out [..., N]``, or with ``accumulate``
    added to it ahead of that rounding.  ``out`` may overlap ``x``.  ``resident``: as in ``cuda_ops.gemm``.  The kernels' output is bf16:
    for a tensor or ``dtype`` of another type the plain statement runs, on the GPU as well, which is torch's product of 64-bit copies of
    rows and weight (eight times the weight's memory, and slower by orders).  Serving only: there is no gradient."""
    k, n = w.shape
    held = isinstance(x, Int8Rows)
    codes, w_codes = x.codes if held else x, w.codes
    shape, device = codes.shape, codes.get_device()
    if shape[-1:] != (k,) or device != w_codes.get_device():
        raise ValueError(f"x {tuple(shape)} on {codes.device} and a {w.shape} weight on {w_codes.device}")
    shape = shape[:-1] + (n,)
    if held:
        if (codes.dtype is not torch.int8 or x.scales.shape != shape[:-1] or x.scales.dtype is not torch.float32
                or x.scales.get_device() != device):
            raise ValueError(f"rows in 8 bits are int8 codes and an fp32 scale for each: {codes.dtype}, {tuple(x.scales.shape)} "
                             f"{x.scales.dtype}")
        dtype = dtype or (torch.bfloat16 if out is None else out.dtype)
    else:
        dtype = dtype or x.dtype
    _no_gradient("int8_linear", x.scales if held else x, w.scales, out)
    given = out is not None
    if not given:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = codes.new_empty(shape, dtype=dtype)
    elif out.shape != shape or out.dtype != dtype or out.get_device() != device or not out.is_contiguous():
        raise ValueError(f"out {tuple(out.shape)} {out.dtype}: contiguous {tuple(shape)} {dtype} is wanted")
    w_scales = w.scales
    if not _on_kernel(out) or (not held and x.dtype is not torch.bfloat16):
        codes, scales = x if held else quantize_rows(x)
        # (Products of codes and their sums are whole numbers below 2^53.)
        sums = (codes.double() @ w_codes.double().t()).float()
        y = sums * scales[..., None] * w_scales
        return out.copy_(out.float() + y if accumulate else y)
    rows = out.numel() // n
    if rows == 0:
        return out
    if w_codes.data_ptr() % 16 or w_scales.data_ptr() % 16:
        w_codes, w_scales, resident = w_codes.clone(), w_scales.clone(), False
    few, y = few_rows(rows, k, n), out
    if not few and out.data_ptr() % 16:  # a view into a larger buffer: tiles are stored as vectors
        y = out.clone() if accumulate else torch.empty_like(out)
    if held:
        codes, scales = x
        if given and _overlap(codes, out):  # other columns' products still read x
            codes = codes.clone(memory_format=torch.contiguous_format)
        if not scales.is_contiguous() or (given and _overlap(scales, out)):
            scales = scales.clone(memory_format=torch.contiguous_format)
        codes = _aligned(codes)
        _call(device, "axb_gemm_skinny_int8" if few else "axb_int8_gemm", codes.data_ptr(), scales.data_ptr(), w_codes.data_ptr(),
              w_scales.data_ptr(), y.data_ptr(), rows, n, k, accumulate, 0 if few else pair_features(rows, n), resident, _status(device))
    else:
        _check_row(k)
        x, _, pitch = _row_operand(x, k)
        room = x.new_empty(rows * (k + 4), dtype=torch.uint8)  # codes, then scales
        _call(device, "axb_int8_dense", x.data_ptr(), pitch, room.data_ptr(), w_codes.data_ptr(), w_scales.data_ptr(), y.data_ptr(), rows, n,
              k, accumulate, 0 if few else pair_features(rows, n), resident, _status(device))
    return out if y is out else out.copy_(y)


# ------------------------------------------------------------------------------------------
# Cache.
# ------------------------------------------------------------------------------------------


class Int8Pages(NamedTuple):
    """A page pool of keys or values: ``codes [pages, Nkv, page_size, H]`` (int8) and ``tops [pages, Nkv]`` (bf16), the largest
    magnitudes of their blocks (rounded to bf16, where the values are not): a code stands for ``code * top / 127``."""

    codes: Tensor
    tops: Tensor


def int8_pages(num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device=None) -> Int8Pages:
    """A pool of zeros."""
    if head_dim not in (64, 128):
        raise ValueError(f"the 8-bit cache holds heads of 64 or 128, not {head_dim}")
    if page_size < PAGE_UNIT or page_size % PAGE_UNIT:
        raise ValueError(f"pages of the 8-bit cache hold a multiple of {PAGE_UNIT} tokens, not {page_size}")
    return Int8Pages(torch.zeros((num_pages, num_kv_heads, page_size, head_dim), dtype=torch.int8, device=device),
                     torch.zeros((num_pages, num_kv_heads), dtype=torch.bfloat16, device=device))


def _stand_for(codes: Tensor, top: Tensor) -> Tensor:
    """``codes * top / 127`` in 32 bits, both factors of 2^-7 so that the product stays in range."""
    return codes.float() * (top * 2.0 ** -7) / (127 * 2.0 ** -7)


def page_values(pages: Int8Pages, dtype: torch.dtype = torch.float32) -> Tensor:
    """What a pool (or pages of it) stands for: ``[pages, Nkv, page_size, H]``."""
    return _stand_for(pages.codes, pages.tops.float()[..., None, None]).to(dtype)


def _check_pages(k_pages: Int8Pages, v_pages: Int8Pages, page_table: Tensor, batch: int, heads: int, head_dim: int,
                 device: int) -> tuple:
    """``(pages, Nkv, page size, columns of the table)`` and where codes and tops lie, of a cache that fits; ``device``: index of the
    operands' one."""
    (kc, kt), (vc, vt) = k_pages, v_pages
    shape = kc.shape
    num_pages, nkv, page_size, held = shape if len(shape) == 4 else (0, 0, 0, 0)
    tops = (num_pages, nkv)
    if (held != head_dim or head_dim not in (64, 128) or not nkv or heads % nkv or not num_pages or not page_size
            or page_size % PAGE_UNIT or vc.shape != shape or kt.shape != tops or vt.shape != tops):
        raise ValueError(f"8-bit pages {tuple(shape)} with {tuple(kt.shape)}, {tuple(vc.shape)} with {tuple(vt.shape)} for {heads} "
                         f"heads of {head_dim} (64 or 128; a multiple of {PAGE_UNIT} tokens a page)")
    if num_pages * nkv * page_size >= 2 ** 31 - 1 - page_size:
        raise ValueError(f"8-bit pages {tuple(shape)} have 2^31 rows or more")
    at_k, at_v = kc.data_ptr(), vc.data_ptr()
    if (kc.dtype is not torch.int8 or vc.dtype is not torch.int8 or kt.dtype is not torch.bfloat16 or vt.dtype is not torch.bfloat16
            or not (kc.get_device() == vc.get_device() == kt.get_device() == vt.get_device() == device)
            or not (kc.is_contiguous() and vc.is_contiguous() and kt.is_contiguous() and vt.is_contiguous())
            or (at_k | at_v) % 16):
        raise ValueError("8-bit pages are contiguous, 16-byte aligned int8 and bf16 tensors on the operands' device")
    table = page_table.shape
    if (page_table.dtype is not torch.int32 or len(table) != 2 or table[0] != batch or page_table.get_device() != device
            or not page_table.is_contiguous()):
        raise ValueError(f"a page table is a contiguous int32 matrix of {batch} rows on the operands' device: {tuple(table)} "
                         f"{page_table.dtype}")
    return (num_pages, nkv, page_size, table[1]), (at_k, kt.data_ptr(), at_v, vt.data_ptr())


def _check_apart(pools: tuple) -> None:
    if pools[0] == pools[2] or pools[1] == pools[3]:
        raise ValueError("keys and values are appended to pools of their own")


def _check_counts(counts: Tensor, batch: int, name: str, device: int) -> None:
    if counts.dtype is not torch.int32 or counts.shape != (batch,) or not counts.is_contiguous() or counts.get_device() != device:
        raise ValueError(f"{name} is [{batch}] int32 on the operands' device: {tuple(counts.shape)} {counts.dtype}")


def _append_plain(k, v, k_pages, v_pages, page_table, start, live):
    num_pages, nkv, page_size, _ = k_pages.codes.shape
    b, t = k.shape[:2]
    device = k.device
    at = torch.arange(t, device=device)
    keep = (at < live[:, None]) if live is not None else torch.ones((b, t), dtype=torch.bool, device=device)
    begin = start.clamp(min=0).long()
    row0 = begin % page_size
    rel = row0[:, None] + at
    block, row = rel // page_size, rel % page_size                    # of each token, counted from its sequence's first
    many = (t + page_size - 2) // page_size + 1
    col = begin[:, None] // page_size + torch.arange(many, device=device)
    placed = (start >= 0)[:, None] & (col < page_table.shape[1])
    page = torch.zeros_like(col)
    if page_table.shape[1]:
        page = page_table.long().gather(1, torch.where(placed, col, 0))
    placed &= (page >= 0) & (page < num_pages)
    touched = torch.zeros((b, many), dtype=torch.int32, device=device).scatter_add_(1, block, keep.int()) > 0
    _report_places((touched & ~placed).any(), "a token's place is outside the page table, or its page outside the pool")
    page = torch.where(placed, page, 0)
    goes_on = touched[:, 0] & placed[:, 0] & (row0 > 0)               # with a block that has tokens
    write = touched & placed
    out = []
    for x, pages in ((k, k_pages), (v, v_pages)):
        size = torch.where(keep[..., None], x.abs().amax(-1).float(), 0.0)
        size = torch.where(torch.isfinite(size), size, torch.inf)
        old = torch.where(goes_on[:, None], pages.tops[page[:, 0]].float().abs(), 0.0)
        top = torch.zeros((b, many, nkv), device=device)
        top[:, 0] = torch.where(torch.isfinite(old), old, torch.inf)
        top.scatter_reduce_(1, block[..., None].expand(b, t, nkv), size, "amax")
        top = _tops(top.bfloat16().float())
        turned = _codes(pages.codes[page[:, 0]].double() * old[..., None, None].double(), top[:, 0, :, None, None], 1)
        turns = goes_on[:, None] & (top[:, 0] > 0)
        turns = turns[..., None] & (torch.arange(page_size, device=device) < row0[:, None])[:, None]
        for i in goes_on.nonzero()[:, 0].tolist():
            pages.codes[page[i, 0]] = torch.where(turns[i][..., None], turned[i], pages.codes[page[i, 0]])
        mine = top.gather(1, block[..., None].expand(b, t, nkv))[..., None]
        codes = _codes(x, mine)
        there = keep & write.gather(1, block)
        pages.codes[page.gather(1, block)[there], :, row[there]] = codes[there]
        pages.tops[page[write]] = top[write].bfloat16()
        out.append(torch.where(keep[..., None, None], _stand_for(codes, mine), 0).to(x.dtype))
    return out


def append_int8(k: Tensor, v: Tensor, k_pages: Int8Pages, v_pages: Int8Pages, page_table: Tensor, start: Tensor, *,
                live: Optional[Tensor] = None, values: bool = False) -> Optional[tuple[Tensor, Tensor]]:
    """Quantises ``k`` and ``v [B, T, Nkv, H]`` (strided views may be given) into the pages of positions ``start[b] ..`` of
    ``page_table [B, max_pages]``; ``start [B]`` and ``live [B]`` (how many of the T tokens are there; None: all) are int32.
    A page whose first token is among them starts anew; one that goes on keeps the tokens ahead of ``start``, under its new
    largest magnitude.  What a page holds behind the new tokens has no meaning; other pages do not change.  ``values``: also
    returns what the cache stands for at these tokens, ``(k, v)`` of the inputs' shape and type, zeros behind ``live``.  No two
    columns of the page table may name the same page where it is written."""
    shape, device = k.shape, k.get_device()
    b, t, nkv, h = shape
    if v.shape != shape or v.dtype is not k.dtype or v.get_device() != device:
        raise ValueError(f"k {tuple(shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} differ")
    (num_pages, held, page_size, max_pages), pools = _check_pages(k_pages, v_pages, page_table, b, nkv, h, device)
    if held != nkv:
        raise ValueError(f"pages of {held} heads for {nkv}")
    _check_apart(pools)
    _check_counts(start, b, "start", device)
    if live is not None:
        _check_counts(live, b, "live", device)
    _no_gradient("append_int8", k, v, k_pages.tops, v_pages.tops)
    if not _on_kernel(k):
        if not b or not t:
            return (k.clone(), v.clone()) if values else None
        out = _append_plain(k, v, k_pages, v_pages, page_table, start, live)
        return tuple(out) if values else None
    k, v = _aligned_rows(k), _aligned_rows(v)
    k_strides, v_strides = k.stride(), v.stride()
    out = None
    if values:
        out = (torch.empty_like(k, memory_format=torch.contiguous_format), torch.empty_like(v, memory_format=torch.contiguous_format))
    _call(device, "axb_int8_append", k.data_ptr(), v.data_ptr(), *k_strides[:3], *v_strides[:3], out[0].data_ptr() if values else 0,
          out[1].data_ptr() if values else 0, *pools, page_table.data_ptr(), start.data_ptr(), 0 if live is None else live.data_ptr(), b, t, nkv, h,
          page_size, max_pages, num_pages, _status(device))
    return out


@functools.lru_cache(maxsize=1024)
def attention_splits(batch: int, num_kv_heads: int, group: int, max_len: int, sms: int = 148) -> int:
    """KV splits of attention over the 8-bit cache, a CTA for each split, KV head and eight query heads.  Up to eight are a cluster:
    the number of 1, 2, 4 and 8 that costs least, at 0.75 us for 128 tokens of a CTA, 1.6 us for each CTA that an SM starts and 0.7 us for
    the meeting, 64 tokens or more for each, as long as all CTAs run at once, three an SM (us with 1 / 2 / 4 / 8, sequences of up to so
    many tokens, 8 KV heads: 16 x 2048 17.4 14.7 17.0 23.1, 8 x 2048 16.7 12.6 10.3 15.0, 6 x 2048 16.1 12.1 9.4 9.6, 27 x 512
    9.4 10.6 17.2, 12 x 512 7.1 7.9 7.2 13.4; 32 x 2048, all as long, 25.8 36.9).  Tables of 4096 tokens and more, where lengths differ
    by more, may take two also where that is four CTAs an SM or more (40 x 4096 49 40, 64 x 4096 61 58, all as long 59 67 and 112 97; not 32
    x 4096 41 35, 46 59), and those of more than 8192 twice as many CTAs (42 x 9600 108 85, 30 x 9600 85 69, all as long 141 146 and 98 124).
    Long sequences of few heads take as many as fill most SMs with CTAs of three times the warps, and a second launch that joins them
    (8 heads with 8 / 16 / 18 / 24: 16000 tokens 18.7 14.0 15.7, 130001 tokens 127 47.6 51.9 69; one head with 16 / 32 / 64 / 128: 60000
    tokens 26.0 18.9 19.5 24.5), but no more than leave each warp a tile of 32 keys (so / 48: one head 8208 tokens 8.5 10.4, 12000 8.9
    10.4, two heads 9.2 11.3, 9.9 11.4), and 48, which short sequences in a wide table pay for, up to 2^18 tokens (one head with 48 / 96:
    131072 tokens 21.5 20.8, 262144 32.0 26.8, a million 92 60, but 8208 10.4 14.5).  What the rule costs elsewhere: 300 tokens of 8 heads
    in a table of 16384 8.5 where one split takes 5.7; nothing at 130001 tokens of 32 heads (8 splits: 160, at the copy rate 163)."""
    ctas = max(1, batch * num_kv_heads * ((group + 7) // 8))
    if max_len > 8192 and ctas * 9 <= sms:
        return max(9, min(128 // ctas, 48 if max_len < 2 ** 18 else 96, -(-max_len // (12 * 32))))
    at_once = (6 if max_len > 8192 else 3) * sms
    best, least = 1, math.inf
    for splits in (1, 2, 4, 8):
        if splits > 1 and (splits * 64 > max_len or (splits * ctas > at_once and (splits > 2 or max_len < 4096 or splits * ctas < 4 * sms))):
            break
        cost = 0.75 / 128 * max_len / splits + 1.6 * -(-splits * ctas // sms) + (0.7 if splits > 1 else 0.0)
        if cost < least:
            best, least = splits, cost
    return best


def _attention_plain(q, k_pages, v_pages, page_table, lengths, scale):
    b, nq, h = q.shape
    num_pages, _, page_size, _ = k_pages.codes.shape
    pages, seen, bad = _read_places(page_table, lengths, page_size, num_pages)
    _report_places(bad, "a length behind the page table, or a page outside the pool")
    k, v = (page_values(Int8Pages(x.codes[pages], x.tops[pages])).transpose(1, 2).flatten(2, 3) for x in (k_pages, v_pages))
    seen = seen[:, None, :, None]
    k, v = torch.where(seen, k, 0), torch.where(seen, v, 0)
    scores = q.float().unflatten(1, (k.shape[1], -1)) @ k.transpose(2, 3) * scale
    p = torch.softmax(scores.masked_fill(~seen.transpose(2, 3), -torch.inf), -1)
    out = torch.where(seen.any(2, keepdim=True), p @ v, 0)
    return out.reshape(b, nq, h).to(q.dtype)


def _check_attention(scale: float, splits: Optional[int]) -> None:
    if not 0 < scale < 2 ** 20:
        raise ValueError(f"softmax_scale {scale} is not in (0, 2^20)")
    if splits is not None and not 1 <= splits <= MAX_SPLITS:
        raise ValueError(f"{splits} splits: 1 to {MAX_SPLITS}")


def paged_decode_attention_int8(q: Tensor, k_pages: Int8Pages, v_pages: Int8Pages, page_table: Tensor, lengths: Tensor, *,
                                softmax_scale: Optional[float] = None, splits: Optional[int] = None,
                                out: Optional[Tensor] = None, scratch: Optional[Tensor] = None) -> Tensor:
    """q ``[B, Nq, H]``; page_table ``[B, max_pages]``, lengths ``[B]`` int32 (valid tokens per sequence; 0: zeros).  Query heads
    are grouped by KV head.  ``out`` may be ``q``, or overlap it.  ``scratch``: ``attention_scratch_floats`` fp32 values, for
    more than eight splits; calls that overlap on the GPU need one each.  Queries from 2^-40 to 2^56 and
    pages' tops from 2^-40 to 2^50 keep their digits; larger ones may overflow.  Returns ``[B, Nq, H]``."""
    b, nq, h = q.shape
    device = q.get_device()
    cache, pools = _check_pages(k_pages, v_pages, page_table, b, nq, h, device)
    _check_counts(lengths, b, "lengths", device)
    scale = 1.0 / math.sqrt(h) if softmax_scale is None else softmax_scale
    _check_attention(scale, splits)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.get_device() != device or not out.is_contiguous()):
        raise ValueError(f"out {tuple(out.shape)} {out.dtype}: contiguous {tuple(q.shape)} {q.dtype} is wanted")
    _no_gradient("paged_decode_attention_int8", q, k_pages.tops, v_pages.tops, out)
    if not _on_kernel(q):
        y = _attention_plain(q, k_pages, v_pages, page_table, lengths, scale)
        return y if out is None else out.copy_(y)
    # (In place is fine: a CTA, and its cluster, has its heads' queries before it stores their output.)
    if not q.is_contiguous() or q.data_ptr() % 16 or (out is not None and q.data_ptr() != out.data_ptr() and _overlap(q, out)):
        q = q.clone(memory_format=torch.contiguous_format)
    splits, scratch = _plan_attention(q, scratch, b, nq, h, cache, splits, device)
    if out is None:
        out = torch.empty_like(q)
    _launch_attention(q, pools, page_table, lengths, -1, out, scratch, b, nq, h, cache, splits, scale, device)
    return out


def _plan_attention(like: Tensor, scratch: Optional[Tensor], b: int, nq: int, h: int, cache: tuple, splits: Optional[int],
                    device: int) -> tuple:
    """``(splits, scratch)`` of a launch; what it refuses is refused ahead of an append."""
    _, nkv, page_size, max_pages = cache
    if not nq or max(b, nkv * -(-nq // (8 * nkv))) > MAX_GRID:
        raise ValueError(f"{b} sequences, {nq} query heads for {nkv}: 1 to {MAX_GRID} groups of eight heads, up to {MAX_GRID} sequences")
    if splits is None:
        splits = attention_splits(b, nkv, nq // nkv, max_pages * page_size)
    if splits > 8:
        floats = attention_scratch_floats(b, nq, h, splits)
        if scratch is None:
            scratch = torch.empty(floats, dtype=torch.float32, device=like.device)
        elif (scratch.numel() < floats or scratch.dtype != torch.float32 or scratch.get_device() != device
              or not scratch.is_contiguous() or scratch.data_ptr() % 8):
            raise ValueError(f"scratch is {floats} contiguous fp32 values on {like.device}, 8-byte aligned")
    return splits, scratch


def _launch_attention(q, pools, page_table, lengths, limit, out, scratch, b, nq, h, cache, splits, scale, device):
    num_pages, nkv, page_size, max_pages = cache
    _call(device, "axb_int8_decode_attn", q.data_ptr(), *pools, page_table.data_ptr(), lengths.data_ptr(), out.data_ptr(),
          0 if scratch is None else scratch.data_ptr(), limit, b, nq, nkv, h, page_size, max_pages, num_pages, splits, scale,
          _status(device))


def attention_scratch_floats(batch: int, num_q_heads: int, head_dim: int, splits: int) -> int:
    """fp32 values that the parts of more than eight splits take."""
    f, _ = _entries.get("axb_int8_attn_scratch_floats") or _entry("axb_int8_attn_scratch_floats")
    return f(batch, num_q_heads, head_dim, splits)


def _check_packed(qkv: Tensor, k_pages: Int8Pages, table: Tensor, nq: int) -> tuple[int, int]:
    """``(Nkv, H)`` of a packed projection that fits the cache and the rotation table."""
    nkv, h = k_pages.codes.shape[1], k_pages.codes.shape[3]
    if qkv.shape[-1] != (nq + 2 * nkv) * h or not qkv.is_contiguous() or qkv.data_ptr() % 16:
        raise ValueError(f"a packed projection of {nq} + 2 x {nkv} heads of {h} is contiguous and 16-byte aligned: {tuple(qkv.shape)}")
    if (table.dtype != torch.float32 or table.shape[1:] != (h // 2, 2) or not len(table) or not table.is_contiguous()
            or table.device != qkv.device or table.data_ptr() % 16):
        raise ValueError(f"a rotation table is [positions, {h // 2}, 2] fp32 on {qkv.device}: {tuple(table.shape)} {table.dtype}")
    return nkv, h


def rope_decode_attention_int8(qkv: Tensor, k_pages: Int8Pages, v_pages: Int8Pages, page_table: Tensor, lengths: Tensor,
                               table: Tensor, *, num_q_heads: int, softmax_scale: float, splits: Optional[int] = None,
                               scratch: Optional[Tensor] = None) -> Tensor:
    """``qkv [B, (Nq + 2 Nkv) * H]`` of the token at position ``lengths - 1``: rotates its query and key by ``table [positions,
    H / 2, 2]`` (``decode_ops.rope_table``), appends key and value to the cache and attends to it.  Rows of length 0, and those
    behind the page table or the rotation table, append nothing and get zeros.  Returns ``[B, Nq, H]``."""
    nkv, h = _check_packed(qkv, k_pages, table, num_q_heads)
    if qkv.dim() != 2:
        raise ValueError(f"a step takes one token a sequence, [B, width]: {tuple(qkv.shape)}")
    b, device = qkv.shape[0], qkv.get_device()
    cache, pools = _check_pages(k_pages, v_pages, page_table, b, num_q_heads, h, device)
    num_pages, _, page_size, max_pages = cache
    _check_apart(pools)
    _check_counts(lengths, b, "lengths", device)
    _check_attention(softmax_scale, splits)
    _no_gradient("rope_decode_attention_int8", qkv, k_pages.tops, v_pages.tops, table)
    limit = min(table.shape[0], max_pages * page_size)
    if not _on_kernel(qkv):
        if not b:
            return qkv.new_empty((0, num_q_heads, h))
        q, k, v = (x[:, None] for x in _split_qkv(qkv, num_q_heads, nkv))
        without = lengths > limit  # a place or a rotation
        _report_places(without.any(), f"a position behind a rotation table of {table.shape[0]} or the page table")
        lengths = torch.where(without, 0, lengths)
        pos = lengths[:, None].long() - 1
        q, k = _rotate(q, table, pos), _rotate(k, table, pos)
        _append_plain(k, v, k_pages, v_pages, page_table, lengths - 1, (lengths > 0).to(torch.int32))
        return paged_decode_attention_int8(q[:, 0], k_pages, v_pages, page_table, lengths, softmax_scale=softmax_scale)
    splits, scratch = _plan_attention(qkv, scratch, b, num_q_heads, h, cache, splits, device)
    out = qkv.new_empty((b, num_q_heads, h))  # the rotated queries, then what they attend to
    _call(device, "axb_int8_rope_append", qkv.data_ptr(), out.data_ptr(), *pools, page_table.data_ptr(), lengths.data_ptr(), 0, table.data_ptr(),
          table.shape[0], b, 1, num_q_heads, nkv, h, page_size, max_pages, num_pages, _status(device))
    _launch_attention(out, pools, page_table, lengths, limit, out, scratch, b, num_q_heads, h, cache, splits, softmax_scale, device)
    return out


def prompt_attention_int8(qkv: Tensor, k_pages: Int8Pages, v_pages: Int8Pages, page_table: Tensor, table: Tensor, *,
                          num_q_heads: int, softmax_scale: float, live: Optional[Tensor] = None) -> Tensor:
    """Whole prompts from position 0: ``qkv [B, T, (Nq + 2 Nkv) * H]`` of one projection, ``live [B]`` (int32; None: T) tokens of
    each.  Rotates queries and keys by ``table``, appends keys and values to the cache and runs causal attention over what the
    cache then stands for: in ``qkv`` queries are replaced by rotated ones, keys and values by the cache's, rounded to
    ``qkv``'s type (zeros behind ``live``).  Returns ``[B, T, Nq * H]``."""
    nkv, h = _check_packed(qkv, k_pages, table, num_q_heads)
    b, t, _ = qkv.shape
    device = qkv.get_device()
    (num_pages, _, page_size, max_pages), pools = _check_pages(k_pages, v_pages, page_table, b, num_q_heads, h, device)
    _check_apart(pools)
    if table.shape[0] < t or max_pages * page_size < t:
        raise ValueError(f"{b} x {t} tokens, a rotation table of {table.shape[0]} positions, a page table {tuple(page_table.shape)}")
    if live is not None:
        _check_counts(live, b, "live", device)
    _check_attention(softmax_scale, None)
    _no_gradient("prompt_attention_int8", qkv, k_pages.tops, v_pages.tops, table)
    if not qkv.numel():
        return qkv.new_empty((b, t, num_q_heads * h))
    q, k, v = _split_qkv(qkv, num_q_heads, nkv)
    if not _on_kernel(qkv):
        pos = torch.arange(t, device=qkv.device).expand(b, t)
        q.copy_(_rotate(q, table, pos))
        start = torch.zeros(b, dtype=torch.int32, device=qkv.device)
        for x, y in zip((k, v), _append_plain(_rotate(k, table, pos), v, k_pages, v_pages, page_table, start, live)):
            x.copy_(y)
        out = dispatch.reference.attention(q, k, v, causal=True, softmax_scale=softmax_scale)
        return out.reshape(b, t, num_q_heads * h)
    from axlearn_b200.ops import decode_ops

    if max(b, num_q_heads) > MAX_GRID:
        raise ValueError(f"{b} prompts, {num_q_heads} query heads: up to {MAX_GRID} of each")
    _call(device, "axb_int8_rope_append", qkv.data_ptr(), 0, *pools, page_table.data_ptr(), 0, 0 if live is None else live.data_ptr(),
          table.data_ptr(), table.shape[0], b, t, num_q_heads, nkv, h, page_size, max_pages, num_pages, _status(device))
    with _on(qkv.device):
        return decode_ops.packed_prompt_attention(qkv, num_q_heads=num_q_heads, num_kv_heads=nkv, softmax_scale=softmax_scale)

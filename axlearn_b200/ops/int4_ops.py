"""Serving in 4 bits: products with 4-bit weights and a paged 4-bit KV cache (``csrc/int4_linear.cu``,
``csrc/int4_cache.cu``).

A group of neighbouring values shares two bf16 numbers, its smallest value ``m`` and a step ``s``, a fifteenth of its range;
a value is held as the code ``c = round((x - m) / s)`` of 0 to 15 (ties to the even code) and stands for ``m + s * c``.  A step
below the smallest normal fp32 number counts as 0.  A group with a NaN or an infinity in it, or whose range
overflows, stands for NaN.

* ``quantize_weight`` / ``int4_linear``: ``x [..., K] @ w [K, N]``, groups of 64 or 128 rows of a column.
* ``append_int4``: keys and values of new tokens into the cache (prompts, chunks, single tokens), groups of 32 dims of a head.
* ``paged_decode_attention_int4``: one query token per sequence over the cache.
* ``prompt_attention_int4``, ``rope_decode_attention_int4``: what a prompt and a decoding step run, with the rotation of
  queries and keys and the append.

Attention sees what the cache stands for: steps ``m + s * c`` itself, prompts that value rounded to bf16 (2^-8 of it at most).
Serving only: operands that need a gradient, or carry a tangent, are refused.  CUDA tensors in bf16 go to the kernels, everything
else runs the plain statements, which are also the oracle in tests.  Places that a page table or a length gets wrong (a page that
the pool does not have, a position behind a table) are not touched: on the GPU they set the device's status word, which
``cuda_ops.check_status`` raises, on the host they are an ``IndexError``.  The bf16 forms of these operations are ``cuda_ops.gemm`` and
``decode_ops``; the reference has no 4-bit form (its quantised layers: axlearn/common/quantized_dot_general/layers.py).
"""

from __future__ import annotations

import contextlib
import ctypes
import dataclasses
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad as _forward_ad

from axlearn_b200.ops import cuda_ops, dispatch

c_void_p, c_int, c_int64, c_float = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
Tensor = torch.Tensor

CACHE_GROUP = 32
_configured = False


def _lib():
    global _configured
    h = cuda_ops.lib()
    if not _configured:
        h.axb_int4_append.argtypes = [c_void_p] * 2 + [c_int64] * 6 + [c_void_p] * 9 + [c_int] * 7 + [c_void_p] * 2
        h.axb_int4_append_prompt.argtypes = [c_void_p] * 7 + [c_int] * 9 + [c_void_p] * 2
        h.axb_int4_decode_attn.argtypes = [c_void_p] * 10 + [c_int] * 9 + [c_float, c_void_p, c_void_p]
        h.axb_int4_attn_scratch_floats.argtypes = [c_int] * 4
        h.axb_int4_attn_scratch_floats.restype = c_int64
        h.axb_int4_linear.argtypes = [c_void_p] * 4 + [c_int] * 4 + [c_int64, c_int64, c_int, c_int, c_void_p]
        h.axb_int4_gemm.argtypes = [c_void_p] * 4 + [c_int] * 4 + [c_int64] * 2 + [c_int] * 3 + [c_void_p] * 2
        h.axb_int4_expand.argtypes = [c_void_p] * 3 + [c_int] * 3 + [c_void_p]
        for f in (h.axb_int4_append, h.axb_int4_append_prompt, h.axb_int4_decode_attn, h.axb_int4_linear, h.axb_int4_gemm,
                  h.axb_int4_expand):
            f.restype = c_int
        _configured = True
    return h


def _on_kernel(x: Tensor) -> bool:
    return x.is_cuda and x.dtype == torch.bfloat16 and not dispatch._flags.force_reference  # pylint: disable=protected-access


def _no_gradient(name: str, *tensors: Optional[Tensor]) -> None:
    """Refuses operands that are differentiated, backward or forward, on every device and in every type."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no gradient")
    if getattr(_forward_ad, "_current_level", 0) >= 0:  # (a name that torch does not promise: without it tangents are looked for)
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has no gradient")


def _overlap(x: Tensor, y: Tensor) -> bool:
    """Whether the memory that two tensors span has a part in common."""
    if not x.numel() or not y.numel():
        return False
    spans = []
    for t in (x, y):
        elements = 1 + sum((size - 1) * stride for size, stride in zip(t.shape, t.stride()))
        spans.append((t.data_ptr(), t.data_ptr() + elements * t.element_size()))
    return spans[0][0] < spans[1][1] and spans[1][0] < spans[0][1]


def _on(device: torch.device):
    """The device of the operands made the current one, where it is another."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _call(device: torch.device, name: str, *args) -> None:
    """Launches on the device of the operands, on its current stream."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(device, name, *args)
    rc = getattr(_lib(), name)(*args, cuda_ops._stream())  # pylint: disable=protected-access
    return cuda_ops._check(rc, name)  # pylint: disable=protected-access


# ------------------------------------------------------------------------------------------
# Groups.
# ------------------------------------------------------------------------------------------


def quantize_groups(x: Tensor, group: int) -> tuple[Tensor, Tensor]:
    """Groups along the last dim: codes ``[..., H]`` (uint8) and ``[..., H / group, 2]`` bf16 pairs (step, smallest)."""
    g = x.float().unflatten(-1, (-1, group))
    m = g.amin(-1).bfloat16()
    spread = g.amax(-1) - m.float()
    good = torch.isfinite(spread)
    s = (spread * (1.0 / 15.0)).bfloat16()
    s = torch.where(good & (s.float() >= torch.finfo(torch.float32).tiny), s, 0)
    m = torch.where(good, m, torch.nan)
    level = (g - m.float()[..., None]) / torch.where(s > 0, s.float(), torch.inf)[..., None]
    codes = level.round().clamp(0, 15).nan_to_num(0.0).to(torch.uint8)
    return codes.flatten(-2), torch.stack((s, m), -1)


def group_values(codes: Tensor, scales: Tensor) -> Tensor:
    """fp32 values ``[..., H]`` of codes ``[..., H]`` and pairs ``[..., groups, 2]``."""
    c = codes.float().unflatten(-1, (scales.shape[-2], -1))
    s, m = scales.float().unbind(-1)
    return (m[..., None] + s[..., None] * c).flatten(-2)


# ------------------------------------------------------------------------------------------
# Weights.
# ------------------------------------------------------------------------------------------


@dataclasses.dataclass(frozen=True)
class Int4Weight:
    """A matrix ``[k, n]`` in 4 bits.  ``codes [ceil(n / 16), ceil(k / 128) * 2, 512]`` (uint8) are blocks of 16 columns and 64
    rows in the order of the kernel's operands (``csrc/int4_linear.cu``), ``scales [ceil(n / 16), groups, 8, 2, 2]`` (bf16)
    run over column mod 8, column / 8 and (step, smallest)."""

    codes: Tensor
    scales: Tensor
    k: int
    n: int
    group: int

    def __post_init__(self):
        codes, scales, tiles, blocks = self.codes, self.scales, -(-self.n // 16), -(-self.k // 128) * 2
        if self.k % 8 or self.n % 8 or self.k < 8 or self.n < 8 or self.group not in (64, 128):
            raise ValueError(f"a 4-bit weight has dims that are multiples of 8 and groups of 64 or 128: {self.k, self.n, self.group}")
        if (codes.shape != (tiles, blocks, 512) or codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16
                or scales.shape != (tiles, blocks * 64 // self.group, 8, 2, 2) or codes.device != scales.device
                or not codes.is_contiguous() or not scales.is_contiguous()):
            raise ValueError(f"codes {tuple(codes.shape)} {codes.dtype} and scales {tuple(scales.shape)} {scales.dtype} are not "
                             f"those of a [{self.k}, {self.n}] weight with groups of {self.group}")

    @property
    def shape(self) -> tuple[int, int]:
        return self.k, self.n


def _pack_blocks(codes: Tensor) -> Tensor:
    """``[N, K]`` (multiples of 16 and 64) -> ``[N / 16, K / 64, 512]``."""
    n, k = codes.shape
    x = codes.reshape(n // 16, 2, 8, k // 64, 4, 4, 2, 2)    # half, column, block, lane, MMA, pair, odd
    x = x.permute(0, 3, 2, 4, 5, 7, 6, 1)
    return (x[..., 0] | (x[..., 1] << 4)).reshape(n // 16, k // 64, 512)


def _unpack_blocks(blocks: Tensor) -> Tensor:
    tiles, k64, _ = blocks.shape
    x = torch.stack((blocks & 15, blocks >> 4), -1).reshape(tiles, k64, 8, 4, 4, 2, 2, 2)
    return x.permute(0, 7, 2, 1, 3, 4, 6, 5).reshape(tiles * 16, k64 * 64)


def quantize_weight(w: Tensor, *, group: int = 128) -> Int4Weight:
    """``w [K, N]`` (K and N multiples of 8) with groups of ``group`` rows of a column; the rows behind K that fill its last
    group are zeros."""
    if w.dim() != 2:
        raise ValueError(f"a weight is a matrix: {tuple(w.shape)}")
    k, n = w.shape
    kp, np_ = -(-k // 128) * 128, -(-n // 16) * 16
    padded = torch.nn.functional.pad(w.detach().float().t(), (0, kp - k, 0, np_ - n))
    codes, scales = quantize_groups(padded, group)
    scales = scales.reshape(np_ // 16, 2, 8, kp // group, 2).permute(0, 3, 2, 1, 4).contiguous()
    return Int4Weight(_pack_blocks(codes), scales, k=k, n=n, group=group)


def dequantize_weight(w: Int4Weight, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``[K, N]``, rounded to ``dtype``; on the GPU in bf16 a transposed view of a ``[N, K]`` buffer, for the GEMM."""
    if w.codes.is_cuda and dtype == torch.bfloat16 and not dispatch._flags.force_reference:  # pylint: disable=protected-access
        out = torch.empty((w.codes.shape[0] * 16, w.codes.shape[1] * 64), dtype=dtype, device=w.codes.device)
        _call(out.device, "axb_int4_expand", w.codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(), w.n, w.k, w.group)
        return (out if out.shape == (w.n, w.k) else out[:w.n, :w.k]).t()
    tiles, groups = w.scales.shape[:2]
    scales = w.scales.permute(0, 3, 2, 1, 4).reshape(tiles * 16, groups, 2)
    return group_values(_unpack_blocks(w.codes), scales).t()[:w.k, :w.n].to(dtype)


def multiplies_codes(rows: int, n: int) -> bool:
    """Whether a product multiplies with the codes as they are: up to 8 rows, and up to 16 where columns are few enough for one
    wave of CTAs (us of 16 rows, so / with weights expanded inside the product, 4096 rows of the weight: 4096 columns 7.8 /
    8.7, 6144 columns 14.2 / 10.6, 28672 columns 27.0 / 22.8)."""
    return rows <= 8 or (rows <= 16 and n <= 4096)


def expands_inside(rows: int, n: int) -> bool:
    """Whether a product of more rows expands weights inside, for each 128 rows again; otherwise W is expanded to bf16 once and
    multiplied by the GEMM: up to 512 rows, and more while tiles of 128 x 128 are one wave.  (us inside / with the GEMM: 256 x
    [4096, 28672] 77 / 121, 512 x [4096, 22016] 97 / 113, 768 rows of it 155 / 138, 2048 x [14336, 1024] 55 / 66, 1024 x
    [4096, 4096] 40 / 35; 2048 x [1024, 1024] 11.0 / 10.0, and 12 / 27 as a call.)"""
    return rows <= 512 or -(-rows // 128) * -(-n // 128) <= 148


def linear_splits(k: int, n: int, sms: int = 148) -> int:
    """Slices of K of a product with the codes: one wave of CTAs (four fit an SM; a CTA takes 64 columns), 512 rows of the weight
    or more for each.  More than four slices pay where columns are few and K is long (us of one row with 4 / 8: [8192, 2048]
    7.6 / 6.6, [4096, 2048] 4.8 / 5.0)."""
    ctas = -(-n // 64)
    return max(1, min(8 if ctas <= 32 and k >= 8192 else 4, k // 512, 4 * sms // ctas))


def fused_plan(rows: int, k: int, n: int) -> tuple[int, int]:
    """``(warps, splits)`` of a product with weights expanded inside: 16 columns a warp make a tile, slices of K are the CTAs of a
    cluster.  Of up to 64 rows two CTAs fit an SM.  Tiles of 128 columns in one slice, or in as many as there is a CTA for
    each SM (clusters leave some idle, so 128 are counted on) with 340 rows of the weight or more; with two CTAs an SM 800 or
    more, if they fill most of it.  Tiles of 80 columns where those of 128 would be two CTAs on few SMs and one on the others.
    (us of 64 rows: [14336, 4096] in 4 / 8 slices 18.4 / 17.1, [4096, 4096] 10.2 / 11.1, [4096, 11008] in 2 / 3 19.2 / 15.5,
    [2048, 2048] in 4 / 6 7.8 / 7.0; [4096, 22016] with 8 / 5 warps 25.1 / 22.9.)"""
    tiles = -(-n // 128) * -(-rows // 128)
    splits = max(1, min(8, 128 // tiles, k // 340))
    if rows <= 64:
        if tiles > 148 and n <= 280 * 80:
            return 5, 1
        two = min(8, 264 // tiles, k // 800)
        if two * tiles >= 224:
            splits = max(splits, two)
    return 8, splits


def int4_linear(x: Tensor, w: Int4Weight, *, out: Optional[Tensor] = None, accumulate: bool = False) -> Tensor:
    """``x [..., K] @ w`` with fp32 accumulation, rounded to ``x.dtype``; into ``out [..., N]``, or with ``accumulate`` added to
    it; ``out`` may be ``x`` itself, or overlap it.  Few rows multiply with the 4-bit weights as they are
    (``multiplies_codes``), more rows with their values rounded to bf16.  Serving only: there is no gradient.  Products keep their digits for x from 2^-57 up to 2^56, weights from 2^-62 and
    steps below 2^31; sums that overflow fp32 on the way, as with an infinity in x, are NaN."""
    k, n, codes = w.k, w.n, w.codes
    device = x.device
    if x.shape[-1] != k or device != codes.device:
        raise ValueError(f"x {tuple(x.shape)} on {device} and a {w.shape} weight on {codes.device}")
    _no_gradient("int4_linear", x, w.scales, out)
    given = out is not None
    if not given:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = x.new_empty(x.shape[:-1] + (n,))
    elif out.shape != x.shape[:-1] + (n,) or out.dtype != x.dtype or out.device != device or not out.is_contiguous():
        raise ValueError(f"out {tuple(out.shape)} {out.dtype}: contiguous {tuple(x.shape[:-1]) + (n,)} {x.dtype} is wanted")
    if not _on_kernel(x):
        y = x.float() @ dequantize_weight(w, torch.float32)
        return out.copy_(out.float() + y if accumulate else y)
    if given and _overlap(x, out):  # other columns' products still read x
        x = x.clone()
    rows = x.shape[0] if x.dim() == 2 else out.numel() // n
    if rows == 0:
        return out
    ldx = x.stride(0) if x.dim() == 2 and x.stride(1) == 1 else 0
    if ldx < k or ldx % 8 or x.data_ptr() % 16:
        x, ldx = x.reshape(rows, k).contiguous(), k
        if x.data_ptr() % 16:
            x = x.clone()
    if multiplies_codes(rows, n):
        _call(device, "axb_int4_linear", x.data_ptr(), codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(), rows, n, k, w.group,
              ldx, n, 1 if accumulate else 0, linear_splits(k, n))
        return out
    if expands_inside(rows, n):
        _call(device, "axb_int4_gemm", x.data_ptr(), codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(), rows, n, k, w.group,
              ldx, n, 1 if accumulate else 0, *fused_plan(rows, k, n), cuda_ops.status_word(device).data_ptr())
        return out
    expanded = dequantize_weight(w)
    with _on(device):
        if out.data_ptr() % 16:  # a view into a larger buffer: the GEMM stores vectors
            y = out.clone() if accumulate else torch.empty_like(out)
            cuda_ops.gemm(x, expanded, out=y.view(rows, n), accumulate=accumulate)
            return out.copy_(y)
        cuda_ops.gemm(x, expanded, out=out.view(rows, n), accumulate=accumulate)
    return out


# ------------------------------------------------------------------------------------------
# Cache.
# ------------------------------------------------------------------------------------------


class Int4Pages(NamedTuple):
    """A page pool of keys or values: ``codes [pages, Nkv, page_size, H / 2]`` (uint8), ``scales [pages, Nkv, page_size, H / 32,
    2]`` (bf16; step and smallest value of every 32 dims).  A row's codes are 8 chunks; chunk r holds dims 4r .. 4r + 3 of
    every group, group by group, the lower dim in the lower half of a byte."""

    codes: Tensor
    scales: Tensor


def int4_pages(num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device=None) -> Int4Pages:
    """A pool of zeros."""
    if head_dim not in (64, 128):
        raise ValueError(f"the 4-bit cache holds heads of 64 or 128, not {head_dim}")
    shape = (num_pages, num_kv_heads, page_size)
    return Int4Pages(torch.zeros(shape + (head_dim // 2,), dtype=torch.uint8, device=device),
                     torch.zeros(shape + (head_dim // CACHE_GROUP, 2), dtype=torch.bfloat16, device=device))


def _pack_rows(codes: Tensor) -> Tensor:
    h = codes.shape[-1]
    x = codes.unflatten(-1, (h // 32, 8, 2, 2)).transpose(-4, -3)
    return (x[..., 0] | (x[..., 1] << 4)).flatten(-3)


def _unpack_rows(rows: Tensor) -> Tensor:
    groups = rows.shape[-1] // 16
    x = torch.stack((rows & 15, rows >> 4), -1).flatten(-2).unflatten(-1, (8, groups, 4))
    return x.transpose(-3, -2).flatten(-3)


def page_values(pages: Int4Pages, dtype: torch.dtype = torch.float32) -> Tensor:
    """What a pool (or rows of it) stands for: ``[pages, Nkv, page_size, H]``."""
    return group_values(_unpack_rows(pages.codes), pages.scales).to(dtype)


def _check_pages(k_pages: Int4Pages, v_pages: Int4Pages, page_table: Tensor, batch: int, heads: int, head_dim: int,
                 device: torch.device) -> tuple:
    """``(pages, Nkv, page size)`` of a cache that fits."""
    (kc, ks), (vc, vs) = k_pages, v_pages
    shape = kc.shape
    num_pages, nkv, page_size, half = shape if len(shape) == 4 else (0, 0, 0, 0)
    if (half * 2 != head_dim or head_dim not in (64, 128) or not nkv or heads % nkv or not num_pages or not page_size
            or vc.shape != shape or ks.shape != (num_pages, nkv, page_size, half // 16, 2) or vs.shape != ks.shape):
        raise ValueError(f"4-bit pages {tuple(shape)} with {tuple(ks.shape)}, {tuple(vc.shape)} with {tuple(vs.shape)} for {heads} "
                         f"heads of {head_dim} (64 or 128)")
    for codes, scales in (k_pages, v_pages):
        if (codes.dtype is not torch.uint8 or scales.dtype is not torch.bfloat16 or codes.device != device
                or scales.device != device or not codes.is_contiguous() or not scales.is_contiguous()):
            raise ValueError(f"4-bit pages are contiguous uint8 and bf16 tensors on {device}")
    if (page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[0] != batch
            or page_table.device != device or not page_table.is_contiguous()):
        raise ValueError(f"a page table is a contiguous int32 matrix of {batch} rows on {device}: {tuple(page_table.shape)} "
                         f"{page_table.dtype}")
    return num_pages, nkv, page_size


def _check_counts(counts: Tensor, batch: int, name: str, device) -> Tensor:
    if counts.dtype != torch.int32 or counts.shape != (batch,) or not counts.is_contiguous() or counts.device != device:
        raise ValueError(f"{name} is [{batch}] int32 on {device}: {tuple(counts.shape)} {counts.dtype}")
    return counts


def _report_places(bad: Tensor, what: str) -> None:
    """``bad`` (a truth value): an error on the host, the status word on the GPU."""
    if bad.is_cuda:
        word = cuda_ops.status_word(bad.device)
        word.copy_(torch.where(bad, 5, word))
    elif bool(bad):
        raise IndexError(what)


def _rotate(x: Tensor, table: Tensor, pos: Tensor) -> Tensor:
    """``x [B, T, N, H]`` with interleaved pairs turned by ``table [positions, H / 2, 2]`` (sin, cos) at ``pos [B, T]``."""
    sn, cs = table[pos.clamp(0, table.shape[0] - 1)].unbind(-1)
    sn, cs = sn[:, :, None], cs[:, :, None]
    x0, x1 = x.float().unflatten(-1, (-1, 2)).unbind(-1)
    return torch.stack((x0 * cs - x1 * sn, x1 * cs + x0 * sn), -1).flatten(-2).to(x.dtype)


def _write_places(page_table: Tensor, start: Tensor, live: Optional[Tensor], tokens: int, page_size: int, num_pages: int) -> tuple:
    """``(page, row, keep, inside)`` ``[B, T]`` of new tokens: which are there, and which of them have a place."""
    pos = start[:, None].long() + torch.arange(tokens, device=start.device)
    keep = torch.ones_like(pos, dtype=torch.bool)
    if live is not None:
        keep = torch.arange(tokens, device=start.device) < live[:, None]
    inside = keep & (pos >= 0) & (pos < page_table.shape[1] * page_size)
    if not page_table.shape[1]:
        return pos * 0, pos * 0, keep, inside
    page = page_table.long().gather(1, torch.where(inside, pos // page_size, 0))
    inside &= (page >= 0) & (page < num_pages)
    return page, pos % page_size, keep, inside


def _append_plain(k, v, k_pages, v_pages, page_table, start, live):
    num_pages, _, page_size, _ = k_pages.codes.shape
    page, row, keep, inside = _write_places(page_table, start, live, k.shape[1], page_size, num_pages)
    _report_places((keep & ~inside).any(), "a token's place is outside the page table, or its page outside the pool")
    values = []
    for x, pages in ((k, k_pages), (v, v_pages)):
        codes, scales = quantize_groups(x, CACHE_GROUP)
        pages.codes[page[inside], :, row[inside]] = _pack_rows(codes)[inside]
        pages.scales[page[inside], :, row[inside]] = scales[inside]
        values.append(torch.where(keep[..., None, None], group_values(codes, scales).to(x.dtype), 0))
    return values


def append_int4(k: Tensor, v: Tensor, k_pages: Int4Pages, v_pages: Int4Pages, page_table: Tensor, start: Tensor, *,
                live: Optional[Tensor] = None, values: bool = False) -> Optional[tuple[Tensor, Tensor]]:
    """Quantises ``k`` and ``v [B, T, Nkv, H]`` (strided views may be given) into the pages of positions ``start[b] ..`` of
    ``page_table [B, max_pages]``; ``start [B]`` and ``live [B]`` (how many of the T tokens are there; None: all) are int32.
    Nothing else in the pages changes.  ``values``: also returns what the cache stands for at these tokens, ``(k, v)`` of
    the inputs' shape and type, zeros behind ``live``.  No two sequences may own a page that is written."""
    b, t, nkv, h = k.shape
    if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} differ")
    device = k.device
    num_pages, held, page_size = _check_pages(k_pages, v_pages, page_table, b, nkv, h, device)
    if held != nkv:
        raise ValueError(f"pages of {held} heads for {nkv}")
    _check_counts(start, b, "start", device)
    if live is not None:
        _check_counts(live, b, "live", device)
    _no_gradient("append_int4", k, v, k_pages.scales, v_pages.scales)
    if not _on_kernel(k):
        out = _append_plain(k, v, k_pages, v_pages, page_table, start, live)
        return tuple(out) if values else None
    k, v = _aligned_rows(k), _aligned_rows(v)
    out = (k.new_empty((b, t, nkv, h)), k.new_empty((b, t, nkv, h))) if values else None
    _call(device, "axb_int4_append", k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3],
          out[0].data_ptr() if values else None, out[1].data_ptr() if values else None, k_pages.codes.data_ptr(),
          k_pages.scales.data_ptr(), v_pages.codes.data_ptr(), v_pages.scales.data_ptr(), page_table.data_ptr(), start.data_ptr(),
          None if live is None else live.data_ptr(), b, t, nkv, h, page_size, page_table.shape[1], num_pages,
          cuda_ops.status_word(device).data_ptr())
    return out


def _aligned_rows(x: Tensor) -> Tensor:
    """``x [B, T, N, H]`` with 16-byte aligned rows of neighbouring dims."""
    b, t, n, h = x.stride()
    if h == 1 and not (b | t | n) % 8 and not x.data_ptr() % 16:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def attention_splits(batch: int, num_kv_heads: int, group: int, max_len: int, sms: int = 148) -> int:
    """KV splits of attention over the 4-bit cache: one wave of CTAs (four fit an SM; one takes a split, a KV head and eight
    query heads), 64 tokens or more for each.  Beyond 8, which meet in a cluster, the clusters' parts are merged by a second
    launch: for long sequences, growing with the root of their length (8 heads, us with 8 / 16 / 32 / 64 splits: 4000 tokens 8.3
    9.5 8.6 10.9, 16000 tokens 24 19 14.6 16.0, 130001 tokens 151 91 52 47), and as many as clusters of 8 fit the GPU."""
    ctas = max(1, batch * num_kv_heads * ((group + 7) // 8))
    splits = max(1, min(max_len // 64, 4 * sms // ctas))
    if splits <= 8:
        return splits
    many = min((math.isqrt(max_len) // 4 + 4) // 8, 512 // ctas // 8) * 8
    return many if many >= 24 else 8


def _read_places(page_table: Tensor, lengths: Tensor, page_size: int, num_pages: int) -> tuple[Tensor, Tensor, Tensor]:
    """Pages to gather ``[B, max_pages]`` (0 where a sequence has none, or one that is not in the pool), which keys are there ``[B,
    max_pages * page_size]``, and whether a sequence needs a place that is not."""
    lengths, capacity = lengths.long()[:, None], page_table.shape[1] * page_size
    at = torch.arange(capacity, device=lengths.device)
    used = at[::page_size] < lengths
    inside = (page_table >= 0) & (page_table < num_pages)
    bad = (used & ~inside).any() | (lengths > capacity).any()
    there = used & inside
    return torch.where(there, page_table, 0).long(), there.repeat_interleave(page_size, 1) & (at < lengths), bad


def _attention_plain(q, k_pages, v_pages, page_table, lengths, scale):
    b, nq, h = q.shape
    num_pages, _, page_size, _ = k_pages.codes.shape
    pages, seen, bad = _read_places(page_table, lengths, page_size, num_pages)
    _report_places(bad, "a length behind the page table, or a page outside the pool")
    k, v = (page_values(Int4Pages(x.codes[pages], x.scales[pages])).transpose(1, 2).flatten(2, 3) for x in (k_pages, v_pages))
    seen = seen[:, None, :, None]
    k, v = torch.where(seen, k, 0), torch.where(seen, v, 0)
    scores = q.float().unflatten(1, (k.shape[1], -1)) @ k.transpose(2, 3) * scale
    p = torch.softmax(scores.masked_fill(~seen.transpose(2, 3), -torch.inf), -1)
    out = torch.where(seen.any(2, keepdim=True), p @ v, 0)
    return out.reshape(b, nq, h).to(q.dtype)


def paged_decode_attention_int4(q: Tensor, k_pages: Int4Pages, v_pages: Int4Pages, page_table: Tensor, lengths: Tensor, *,
                                softmax_scale: Optional[float] = None, splits: Optional[int] = None,
                                out: Optional[Tensor] = None, scratch: Optional[Tensor] = None) -> Tensor:
    """q ``[B, Nq, H]``; page_table ``[B, max_pages]``, lengths ``[B]`` int32 (valid tokens per sequence; 0: zeros).  Query heads
    are grouped by KV head.  ``out`` may be ``q``, or overlap it.  ``scratch``: ``attention_scratch_floats`` fp32 values, for
    more than eight splits (made a multiple of eight); calls that overlap on the GPU need one each.  Queries from 2^-40 to 2^63 keep their digits, and steps and
    smallest values in ``v_pages`` up to 2^55 over the number of tokens; sums beyond overflow.  Returns ``[B, Nq, H]``."""
    b, nq, h = q.shape
    device = q.device
    num_pages, nkv, page_size = _check_pages(k_pages, v_pages, page_table, b, nq, h, device)
    _check_counts(lengths, b, "lengths", device)
    scale = 1.0 / math.sqrt(h) if softmax_scale is None else softmax_scale
    if not 0 < scale < 2 ** 20:
        raise ValueError(f"softmax_scale {scale} is not in (0, 2^20)")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != device or not out.is_contiguous()):
        raise ValueError(f"out {tuple(out.shape)} {out.dtype}: contiguous {tuple(q.shape)} {q.dtype} is wanted")
    _no_gradient("paged_decode_attention_int4", q, k_pages.scales, v_pages.scales, out)
    if not _on_kernel(q):
        y = _attention_plain(q, k_pages, v_pages, page_table, lengths, scale)
        return y if out is None else out.copy_(y)
    # (In place is fine: a CTA, and its cluster, has its heads' queries before it stores their output.)
    if not q.is_contiguous() or q.data_ptr() % 16 or (out is not None and q.data_ptr() != out.data_ptr() and _overlap(q, out)):
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty_like(q)
    _launch_attention(q, k_pages, v_pages, page_table, lengths, None, out, scratch, b, nq, nkv, h, page_size, num_pages, splits, scale)
    return out


def _launch_attention(q, k_pages, v_pages, page_table, lengths, table, out, scratch, b, nq, nkv, h, page_size, num_pages, splits, scale):
    max_pages, device = page_table.shape[1], q.device
    if splits is None:
        splits = attention_splits(b, nkv, nq // nkv, max_pages * page_size)
    if splits > 8:
        splits = -(-splits // 8) * 8
        floats = attention_scratch_floats(b, nq, h, splits)
        if scratch is None:
            scratch = torch.empty(floats, dtype=torch.float32, device=device)
        elif (scratch.numel() < floats or scratch.dtype != torch.float32 or scratch.device != device
              or not scratch.is_contiguous() or scratch.data_ptr() % 8):
            raise ValueError(f"scratch is {floats} contiguous fp32 values on {device}, 8-byte aligned")
    _call(device, "axb_int4_decode_attn", q.data_ptr(), k_pages.codes.data_ptr(), k_pages.scales.data_ptr(), v_pages.codes.data_ptr(),
          v_pages.scales.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), None if table is None else table.data_ptr(),
          out.data_ptr(), None if scratch is None else scratch.data_ptr(), 0 if table is None else table.shape[0], b, nq, nkv, h,
          page_size, max_pages, num_pages, splits, scale, cuda_ops.status_word(device).data_ptr())


def attention_scratch_floats(batch: int, num_q_heads: int, head_dim: int, splits: int) -> int:
    """fp32 values that the parts of more than eight splits take (a multiple of eight)."""
    splits = -(-splits // 8) * 8 if splits > 8 else splits
    return _lib().axb_int4_attn_scratch_floats(batch, num_q_heads, head_dim, splits)


def _split_qkv(qkv: Tensor, nq: int, nkv: int) -> tuple[Tensor, Tensor, Tensor]:
    """``[..., (Nq + 2 Nkv) * H]`` as views ``[..., heads, H]`` of q, k and v."""
    return qkv.unflatten(-1, (nq + 2 * nkv, -1)).split((nq, nkv, nkv), -2)


def _check_packed(qkv: Tensor, k_pages: Int4Pages, table: Tensor, nq: int) -> tuple[int, int]:
    """``(Nkv, H)`` of a packed projection that fits the cache and the rotation table."""
    nkv, h = k_pages.codes.shape[1], k_pages.codes.shape[3] * 2
    if qkv.shape[-1] != (nq + 2 * nkv) * h or not qkv.is_contiguous() or qkv.data_ptr() % 16:
        raise ValueError(f"a packed projection of {nq} + 2 x {nkv} heads of {h} is contiguous and 16-byte aligned: {tuple(qkv.shape)}")
    if (table.dtype != torch.float32 or table.shape[1:] != (h // 2, 2) or not len(table) or not table.is_contiguous()
            or table.device != qkv.device or table.data_ptr() % 16):
        raise ValueError(f"a rotation table is [positions, {h // 2}, 2] fp32 on {qkv.device}: {tuple(table.shape)} {table.dtype}")
    return nkv, h


def rope_decode_attention_int4(qkv: Tensor, k_pages: Int4Pages, v_pages: Int4Pages, page_table: Tensor, lengths: Tensor,
                               table: Tensor, *, num_q_heads: int, softmax_scale: float, splits: Optional[int] = None,
                               scratch: Optional[Tensor] = None) -> Tensor:
    """``qkv [B, (Nq + 2 Nkv) * H]`` of the token at position ``lengths - 1``: rotates its query and key by ``table [positions,
    H / 2, 2]`` (``decode_ops.rope_table``), appends key and value to the cache and attends to it.  Rows of length 0, and those
    behind the page table or the rotation table, append nothing and get zeros.  Returns ``[B, Nq, H]``."""
    nkv, h = _check_packed(qkv, k_pages, table, num_q_heads)
    if qkv.dim() != 2:
        raise ValueError(f"a step takes one token a sequence, [B, width]: {tuple(qkv.shape)}")
    b, device = qkv.shape[0], qkv.device
    num_pages, _, page_size = _check_pages(k_pages, v_pages, page_table, b, num_q_heads, h, device)
    _check_counts(lengths, b, "lengths", device)
    if not 0 < softmax_scale < 2 ** 20:
        raise ValueError(f"softmax_scale {softmax_scale} is not in (0, 2^20)")
    _no_gradient("rope_decode_attention_int4", qkv, k_pages.scales, v_pages.scales, table)
    if not _on_kernel(qkv):
        q, k, v = (x[:, None] for x in _split_qkv(qkv, num_q_heads, nkv))
        without = lengths > min(table.shape[0], page_table.shape[1] * page_size)  # a place or a rotation
        _report_places(without.any(), f"a position behind a rotation table of {table.shape[0]} or the page table")
        lengths = torch.where(without, 0, lengths)
        pos = lengths[:, None].long() - 1
        q, k = _rotate(q, table, pos), _rotate(k, table, pos)
        _append_plain(k, v, k_pages, v_pages, page_table, lengths - 1, (lengths > 0).to(torch.int32))
        return paged_decode_attention_int4(q[:, 0], k_pages, v_pages, page_table, lengths, softmax_scale=softmax_scale)
    out = torch.empty((b, num_q_heads, h), dtype=qkv.dtype, device=device)
    _launch_attention(qkv, k_pages, v_pages, page_table, lengths, table, out, scratch, b, num_q_heads, nkv, h, page_size, num_pages,
                      splits, softmax_scale)
    return out


def prompt_attention_int4(qkv: Tensor, k_pages: Int4Pages, v_pages: Int4Pages, page_table: Tensor, table: Tensor, *,
                          num_q_heads: int, softmax_scale: float) -> Tensor:
    """Whole prompts from position 0: ``qkv [B, T, (Nq + 2 Nkv) * H]`` of one projection.  Rotates queries and keys by ``table``,
    appends keys and values to the cache and runs causal attention over what the cache then stands for: in ``qkv`` queries
    are replaced by rotated ones, keys and values by the cache's, rounded to ``qkv``'s type.  Returns ``[B, T, Nq * H]``."""
    nkv, h = _check_packed(qkv, k_pages, table, num_q_heads)
    b, t, width = qkv.shape
    device = qkv.device
    num_pages, _, page_size = _check_pages(k_pages, v_pages, page_table, b, num_q_heads, h, device)
    if table.shape[0] < t or page_table.shape[1] * k_pages.codes.shape[2] < t:
        raise ValueError(f"{b} x {t} tokens, a rotation table of {table.shape[0]} positions, a page table {tuple(page_table.shape)}")
    _no_gradient("prompt_attention_int4", qkv, k_pages.scales, v_pages.scales, table)
    if not qkv.numel():
        return qkv.new_empty((b, t, num_q_heads * h))
    q, k, v = _split_qkv(qkv, num_q_heads, nkv)
    if not _on_kernel(qkv):
        pos = torch.arange(t, device=qkv.device).expand(b, t)
        q.copy_(_rotate(q, table, pos))
        start = torch.zeros(b, dtype=torch.int32, device=qkv.device)
        for x, y in zip((k, v), _append_plain(_rotate(k, table, pos), v, k_pages, v_pages, page_table, start, None)):
            x.copy_(y)
        out = dispatch.reference.attention(q, k, v, causal=True, softmax_scale=softmax_scale)
        return out.reshape(b, t, num_q_heads * h)
    from axlearn_b200.ops import decode_ops

    _call(device, "axb_int4_append_prompt", qkv.data_ptr(), k_pages.codes.data_ptr(), k_pages.scales.data_ptr(),
          v_pages.codes.data_ptr(), v_pages.scales.data_ptr(), page_table.data_ptr(), table.data_ptr(), table.shape[0], b, t,
          num_q_heads, nkv, h, page_size, page_table.shape[1], num_pages, cuda_ops.status_word(device).data_ptr())
    with _on(device):
        return decode_ops.packed_prompt_attention(qkv, num_q_heads=num_q_heads, num_kv_heads=nkv, softmax_scale=softmax_scale)

"""Per-kernel entry points over the C ABI, taking and returning torch tensors.

These are the building blocks ``tt_transformer_fwd`` chains; they are exposed for stage-level
parity tests and for callers that want one fused op (e.g. a GEMM with its epilogue) on its own.
Every function launches on the current stream of the input's device and raises on any error.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib


# Longest sequence whose mask the attention kernels summarise themselves (tt_attention_masked_fwd; the header's
# TT_ATTENTION_SUMMARISE_MAX_SEQ).
ATTENTION_SUMMARISE_MAX_SEQ = 4096


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _half(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.float16 or t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA float16 tensor")
    return t.contiguous()


def _mask(m: Optional[torch.Tensor], numel: int) -> Optional[torch.Tensor]:
    if m is None:
        return None
    if m.dtype != torch.bool or m.numel() != numel:
        raise ValueError(f"mask must be bool with {numel} elements")
    return m.contiguous()


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
              valid: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    x = _half(x, "x")
    d = x.shape[-1]
    rows = x.numel() // d
    valid = _mask(valid, rows)
    y = torch.empty_like(x)
    rc = _lib.load().tt_layernorm_fwd(x.data_ptr(), _half(weight, "weight").data_ptr(),
                                      _half(bias, "bias").data_ptr(), _ptr(valid), y.data_ptr(),
                                      rows, d, eps, _stream(x))
    _lib.check(rc, "tt_layernorm_fwd")
    return y


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, epilogue: str = "bias",
           residual: Optional[torch.Tensor] = None, valid: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None, seq: int = 0) -> torch.Tensor:
    """``epilogue`` in {"bias", "gelu", "resid_masked", "masked_resid"} (see tt_linear_fwd).
    ``seq`` (rows per sequence, with ``valid``) only changes the order tiles are visited in."""
    if epilogue not in ("bias", "gelu", "resid_masked", "masked_resid"):
        raise ValueError(f"unknown epilogue {epilogue!r}")
    x = _half(x, "x")
    weight = _half(weight, "weight")
    k = x.shape[-1]
    m = x.numel() // k
    n = weight.shape[0]
    if weight.shape[1] != k:
        raise ValueError("weight must be [N, K]")
    if residual is not None:
        residual = _half(residual, "residual")
        if residual.numel() != m * n:
            raise ValueError("residual must be [M, N]")
    valid = _mask(valid, m)
    y = out if out is not None else torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    rc = _lib.load().tt_linear_fwd(x.data_ptr(), weight.data_ptr(), _half(bias, "bias").data_ptr(),
                                   _ptr(residual), _ptr(valid), y.data_ptr(), m, n, k,
                                   _lib.EPILOGUES[epilogue], 0, int(seq), 0, _stream(x))
    _lib.check(rc, "tt_linear_fwd")
    return y


def qkv_projection(x: torch.Tensor, wqkv: torch.Tensor, bqkv: torch.Tensor,
                   heads: int, valid: Optional[torch.Tensor] = None
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x [B,S,D] -> (q [B,H,S,hd], k [B,H,S,hd], vt [B,H,hd,Sp]) with Sp = S rounded up to 64.
    With ``valid`` ([B,S] bool), tokens whose mask is False get +0.0 in q, k and vt."""
    x = _half(x, "x")
    b, s, d = x.shape
    valid = _mask(valid, b * s)
    hd = d // heads
    sp = (s + 63) // 64 * 64
    plane = b * s * d
    buf = torch.empty(2 * plane + b * d * sp, dtype=torch.float16, device=x.device)
    rc = _lib.load().tt_linear_fwd(x.data_ptr(), _half(wqkv, "wqkv").data_ptr(),
                                   _half(bqkv, "bqkv").data_ptr(), None, _ptr(valid), buf.data_ptr(),
                                   b * s, 3 * d, d, _lib.EPILOGUES["qkv"], b, s, heads,
                                   _stream(x))
    _lib.check(rc, "tt_linear_fwd(qkv)")
    q = buf[:plane].view(b, heads, s, hd)
    k = buf[plane:2 * plane].view(b, heads, s, hd)
    vt = buf[2 * plane:].view(b, heads, hd, sp)
    return q, k, vt


def mask_info(mask: Optional[torch.Tensor], batch: int, seq: int, device) -> torch.Tensor:
    info = torch.empty(2 * batch, dtype=torch.int32, device=device)
    mask = _mask(mask, batch * seq)
    rc = _lib.load().tt_mask_info(_ptr(mask), info.data_ptr(), batch, seq,
                                  torch.cuda.current_stream(device).cuda_stream)
    _lib.check(rc, "tt_mask_info")
    return info


def attention(q: torch.Tensor, k: torch.Tensor, vt: torch.Tensor, mask: Optional[torch.Tensor],
              causal: bool, out: Optional[torch.Tensor] = None,
              prescaled: bool = False) -> torch.Tensor:
    """q, k [B,H,S,hd], vt [B,H,hd,Sp] (views from qkv_projection) -> ctx [B,S,H*hd].

    `out`, if given, is a contiguous fp16 [B,S,H*hd] tensor on the same device that receives ctx.
    `prescaled`: q already holds Q * hd^-1/2 * log2(e) (the forward's own Q,
    tt_attention_fwd_prescaled); otherwise the kernel applies the factor when it loads q.
    """
    b, h, s, hd = q.shape
    if k.shape != q.shape or vt.shape[:3] != (b, h, hd) or vt.shape[3] != (s + 63) // 64 * 64:
        raise ValueError("inconsistent q/k/vt shapes")
    for t, name in ((q, "q"), (k, "k"), (vt, "vt")):
        if not t.is_contiguous() or t.dtype != torch.float16:
            raise ValueError(f"{name} must be contiguous fp16")
    mask = _mask(mask, b * s)
    if out is None:
        ctx = torch.empty(b, s, h * hd, dtype=torch.float16, device=q.device)
    elif (out.shape != (b, s, h * hd) or out.dtype != torch.float16 or not out.is_contiguous()
          or out.device != q.device):
        raise ValueError("out must be a contiguous fp16 [B,S,H*hd] tensor on q's device")
    else:
        ctx = out
    if mask is not None and s <= ATTENTION_SUMMARISE_MAX_SEQ:
        rc = _lib.load().tt_attention_masked_fwd(
            q.data_ptr(), k.data_ptr(), vt.data_ptr(), mask.data_ptr(), ctx.data_ptr(), b, s, h, hd,
            int(causal), int(prescaled), _stream(q))
        _lib.check(rc, "tt_attention_masked_fwd")
        return ctx
    info = mask_info(mask, b, s, q.device) if mask is not None else None
    fn = _lib.load().tt_attention_fwd_prescaled if prescaled else _lib.load().tt_attention_fwd
    rc = fn(q.data_ptr(), k.data_ptr(), vt.data_ptr(), _ptr(mask), _ptr(info), ctx.data_ptr(), b,
            s, h, hd, int(causal), _stream(q))
    _lib.check(rc, "tt_attention_fwd")
    return ctx


# ---- attention of ragged token rows: packed prompts, and new tokens over a paged cache ----

_SEQ_DTYPES = {torch.float16: _lib.FP16, torch.bfloat16: _lib.BF16}

# The current device, and a device's current stream as an integer, without the objects around them (0.1 us instead of
# 0.3 and 2).
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name: str, args: bytes, index: int) -> None:
    """One library call with packed arguments, on the current stream of device ``index``."""
    fn = getattr(_lib.load(), name)
    if index == _current_device():
        rc = fn(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


# The small calls below take a third of their time on the host to look their tensors over, so each attribute is asked
# for once and handed on.

def _typed(t: torch.Tensor, name: str):
    """(dtype, device index) of a tensor that the others of a call have to match."""
    dtype = t.dtype
    if dtype not in _SEQ_DTYPES or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor of float16 or bfloat16")
    return dtype, t.get_device()


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, index: int):
    """(tensor, shape, pointer, row stride, head stride) of ``t`` [T, heads, head_dim] in a form the kernels read:
    adjacent features, rows and heads 16 bytes aligned (a column slice of a fused projection's output is; anything else
    is copied)."""
    shape = t.shape
    if len(shape) != 3 or t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{name} must be a [tokens, heads, head_dim] tensor of {dtype} on cuda:{index}")
    row, head, feature = t.stride()
    pointer = t.data_ptr()
    if feature != 1 or (row | head) & 7 or pointer & 15 or row >= 1 << 26:
        t = t.clone(memory_format=torch.contiguous_format)
        row, head, _ = t.stride()
        pointer = t.data_ptr()
    return t, shape, pointer, row, head


def _int32(t: torch.Tensor, name: str, size: int, index: int) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.get_device() != index or t.shape != (size,):
        raise ValueError(f"{name} must be an int32 tensor of {size} elements on cuda:{index}")
    return t if t.is_contiguous() else t.contiguous()


def _heads(heads: int, kv_heads: int, hd: int) -> None:
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} key / value heads evenly")
    if hd % 8 or not 8 <= hd <= 256:
        raise ValueError(f"head_dim {hd} is not a multiple of 8 from 8 to 256")


def _context(out: Optional[torch.Tensor], q: torch.Tensor, tokens: int, width: int) -> torch.Tensor:
    if out is None:
        return q.new_empty((tokens, width))
    if (out.shape != (tokens, width) or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous()
            or out.data_ptr() & 15):
        raise ValueError(f"out must be a contiguous, 16-byte aligned [{tokens}, {width}] tensor of {q.dtype} on "
                         f"{q.device}")
    return out


def _cache(t: torch.Tensor, name: str, shape, dtype: torch.dtype, index: int):
    """(pointer, page, token and head strides) of one half of a cache, [pages, page_size, kv_heads, head_dim] (used in
    place, so never copied)."""
    if len(shape) != 4 or t.shape != shape or t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{name} must be a [pages, page_size, kv_heads, head_dim] tensor of shape {list(shape)} and "
                         f"{dtype} on cuda:{index}")
    page, row, head, feature = t.stride()
    pointer = t.data_ptr()
    if feature != 1 or (page | row | head) & 7 or pointer & 15:
        raise ValueError(f"{name} needs adjacent features, and pages, tokens and heads 16 bytes aligned")
    return pointer, page, row, head


def _sequences(tokens: int, page_table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor],
               index: int):
    """Checks of the description of a batch over a cache; (page_table, lengths, starts, batch, pages per sequence, the
    table's row stride)."""
    shape = lengths.shape
    batch = shape[0] if len(shape) == 1 else -1
    lengths = _int32(lengths, "lengths", batch, index)
    shape = page_table.shape
    if (len(shape) != 2 or shape[0] != batch or shape[1] == 0 or page_table.dtype is not torch.int32
            or page_table.get_device() != index):
        raise ValueError(f"page_table must be an int32 tensor [{batch}, pages per sequence] on cuda:{index}")
    row, column = page_table.stride()
    if column != 1 and shape[1] > 1:
        page_table = page_table.contiguous()
        row = shape[1]
    if starts is not None:
        starts = _int32(starts, "starts", batch + 1, index)
    elif tokens != batch:
        raise ValueError(f"{tokens} tokens for {batch} sequences need starts")
    return page_table, lengths, starts, batch, shape[1], row


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, *,
                     causal: bool = True, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of whole sequences packed one behind the other: q [T, heads, head_dim], k and v
    [T, kv_heads, head_dim] -> [T, heads * head_dim].

    ``starts`` (int32 [B + 1], on the device) holds the first row of each sequence and the end of the last:
    sequence b owns rows starts[b] ... starts[b + 1] - 1 and sees its own only (with ``causal``, each token those
    up to itself).  Query head h reads key / value head h // (heads // kv_heads).  ``scale`` defaults to
    head_dim^-1/2.  float16 or bfloat16, head_dim a multiple of 8 up to 256; q, k, v may be column slices of one
    projection's output.  Rows outside every sequence are left as they are in ``out`` (arbitrary in a new tensor),
    which may not overlap the other tensors."""
    dtype, index = _typed(q, "q")
    q, (tokens, heads, hd), q_at, q_row, q_head = _rows(q, "q", dtype, index)
    k, shape, k_at, k_row, k_head = _rows(k, "k", dtype, index)
    v, v_shape, v_at, v_row, v_head = _rows(v, "v", dtype, index)
    kv_heads = shape[1]
    if shape != v_shape or shape[0] != tokens or shape[2] != hd:
        raise ValueError("k and v must have one shape, and q's number of tokens and head_dim")
    _heads(heads, kv_heads, hd)
    shape = starts.shape
    batch = shape[0] - 1 if len(shape) == 1 else -1
    if batch < 0:
        raise ValueError("starts must be an int32 tensor of B + 1 elements")
    starts = _int32(starts, "starts", batch + 1, index)
    out = _context(out, q, tokens, heads * hd)
    args = _lib.PACKED_ATTENTION
    try:
        packed = args.pack(
            args.size, q_at, k_at, v_at, starts.data_ptr(), out.data_ptr(), q_row, q_head, k_row, k_head, v_row,
            v_head, tokens, batch, heads, kv_heads, hd, causal, _SEQ_DTYPES[dtype],
            hd ** -0.5 if scale is None else scale)
    except _lib.PACK_ERRORS as e:
        raise ValueError(f"packed_attention: {e}") from None
    _call("tt_packed_attention_fwd", packed, index)
    return out


def _cache8(t: torch.Tensor, name: str, shape, index: int):
    """``_cache`` of one half of a cache in 8 bits."""
    if len(shape) != 4 or t.shape != shape or t.dtype is not torch.float8_e4m3fn or t.get_device() != index:
        raise ValueError(f"{name} must be a [pages, page_size, kv_heads, head_dim] tensor of shape {list(shape)} and "
                         f"{torch.float8_e4m3fn} on cuda:{index}")
    page, row, head, feature = t.stride()
    pointer = t.data_ptr()
    if feature != 1 or (page | row | head) & 15 or pointer & 15:
        raise ValueError(f"{name} needs adjacent features, and pages, tokens and heads 16 bytes aligned")
    return pointer, page, row, head


def _scales(k: Optional[torch.Tensor], v: Optional[torch.Tensor], pages: int, page: int, kv_heads: int, index: int):
    """(k's pointer, v's pointer, tokens per scale, strides) of the scales of a cache in 8 bits."""
    if k is None or v is None:
        raise ValueError("a cache in 8 bits needs both k_scales and v_scales")
    shape = k.shape
    blocks = shape[1] if len(shape) == 3 else 0
    if (blocks <= 0 or page % blocks or shape != (pages, blocks, kv_heads) or v.shape != shape
            or k.dtype is not torch.float8_e8m0fnu or v.dtype is not torch.float8_e8m0fnu
            or k.get_device() != index or v.get_device() != index):
        raise ValueError(f"k_scales and v_scales must be [{pages}, {page} / tokens per scale, {kv_heads}] tensors of "
                         f"{torch.float8_e8m0fnu} on cuda:{index}")
    strides = k.stride()
    if v.stride() != strides:
        raise ValueError("k_scales and v_scales must have the same strides")
    return k.data_ptr(), v.data_ptr(), page // blocks, strides


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *,
                 k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None) -> None:
    """Write the keys and values of new tokens, k and v [T, kv_heads, head_dim], into a paged cache, in place.

    k_cache and v_cache are [pages, page_size, kv_heads, head_dim] (any strides that keep features adjacent, 16-byte
    alignment and tokens less than 2^26 elements apart, e.g. both halves of one tensor, or a permuted
    [pages, kv_heads, page_size, head_dim]); page_size is a power of two from 16 on.  Position t of sequence b
    lies in page page_table[b, t // page_size] (int32 [B, n]) at t % page_size.  ``lengths`` (int32 [B]) counts the keys
    of each sequence with the new ones: the n tokens of sequence b, rows starts[b] ... starts[b + 1] - 1 (or row b alone
    without ``starts``), take positions lengths[b] - n ... lengths[b] - 1.  Tokens whose position is negative or beyond the
    table, or whose page is no page of the cache, are not written.

    With ``k_scales`` and ``v_scales`` (float8_e8m0fnu [pages, page_size / block, kv_heads], block a power of two from
    16 on, both with the same strides) the cache is in 8 bits: k_cache and v_cache are float8_e4m3fn, and a value is the
    product of both.  A block's scale is the smallest power of two that holds its tokens' largest finite magnitude, those
    among them that were dropped since the block was begun.  Where a new token is too large for the block that older ones of
    its sequence lie in, the scale grows and those are rounded to it.  Infinities and NaN become NaN, head_dim is a multiple of 16, and two sequences may not write to one
    block in one call."""
    if k_scales is not None or v_scales is not None:
        return _append8(k, v, k_cache, v_cache, page_table, lengths, starts, k_scales, v_scales)
    dtype, index = _typed(k, "k")
    k, shape, k_at, k_row, k_head = _rows(k, "k", dtype, index)
    v, v_shape, v_at, v_row, v_head = _rows(v, "v", dtype, index)
    if shape != v_shape:
        raise ValueError("k and v must have one shape")
    tokens, kv_heads, hd = shape
    _heads(kv_heads, kv_heads, hd)
    shape = (*k_cache.shape[:2], kv_heads, hd)
    k_half, v_half = _cache(k_cache, "k_cache", shape, dtype, index), _cache(v_cache, "v_cache", shape, dtype, index)
    table, lengths, starts, batch, table_pages, table_row = _sequences(tokens, page_table, lengths, starts, index)
    args = _lib.CACHE_ROWS
    try:
        packed = args.pack(
            args.size, k_at, v_at, k_half[0], v_half[0], table.data_ptr(), lengths.data_ptr(),
            0 if starts is None else starts.data_ptr(), k_row, k_head, v_row, v_head, *k_half[1:], *v_half[1:],
            table_row, tokens, batch, kv_heads, hd, shape[0], shape[1], table_pages, 0)
    except _lib.PACK_ERRORS as e:
        raise ValueError(f"cache_append: {e}") from None
    _call("tt_cache_append", packed, index)


def _append8(k, v, k_cache, v_cache, page_table, lengths, starts, k_scales, v_scales) -> None:
    dtype, index = _typed(k, "k")
    k, shape, k_at, k_row, k_head = _rows(k, "k", dtype, index)
    v, v_shape, v_at, v_row, v_head = _rows(v, "v", dtype, index)
    if shape != v_shape:
        raise ValueError("k and v must have one shape")
    tokens, kv_heads, hd = shape
    _heads(kv_heads, kv_heads, hd)
    shape = (*k_cache.shape[:2], kv_heads, hd)
    k_half, v_half = _cache8(k_cache, "k_cache", shape, index), _cache8(v_cache, "v_cache", shape, index)
    ks_at, vs_at, block, strides = _scales(k_scales, v_scales, shape[0], shape[1], kv_heads, index)
    table, lengths, starts, batch, table_pages, table_row = _sequences(tokens, page_table, lengths, starts, index)
    args = _lib.CACHE_ROWS8
    try:
        packed = args.pack(
            args.size, k_at, v_at, k_half[0], v_half[0], ks_at, vs_at, table.data_ptr(), lengths.data_ptr(),
            0 if starts is None else starts.data_ptr(), k_row, k_head, v_row, v_head, *k_half[1:], *v_half[1:],
            *strides, table_row, tokens, batch, kv_heads, hd, shape[0], shape[1], table_pages, block, _SEQ_DTYPES[dtype], 0)
    except _lib.PACK_ERRORS as e:
        raise ValueError(f"cache_append: {e}") from None
    _call("tt_cache_append8", packed, index)


def cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                    max_length: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    k_scales: Optional[torch.Tensor] = None,
                    v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens q [T, heads, head_dim] over a paged cache that holds their keys and values already
    (``cache_append``, whose arguments these are) -> [T, heads * head_dim].

    Token i of the n new ones of sequence b sees the keys at positions 0 ... lengths[b] - n + i; one that sees none
    (a length of 0 in a padded batch) gets zeros.  Without ``starts`` every sequence has one new token.
    ``max_length`` (default: what the table can hold) is the longest length the caller expects; it only decides how
    the work is split.  Keys in a page whose number is no page of the cache are not read and count as NaN.  ``out`` may
    not overlap the other tensors.

    ``k_scales`` and ``v_scales`` as in ``cache_append``: the cache is in 8 bits, read as values of q's type (rounded where
    subnormal in it, infinities past its largest)."""
    dtype, index = _typed(q, "q")
    q, (tokens, heads, hd), q_at, q_row, q_head = _rows(q, "q", dtype, index)
    shape = (*k_cache.shape[:3], hd)
    eight = k_scales is not None or v_scales is not None
    if eight:
        k_half, v_half = _cache8(k_cache, "k_cache", shape, index), _cache8(v_cache, "v_cache", shape, index)
    else:
        k_half = _cache(k_cache, "k_cache", shape, dtype, index)
        v_half = _cache(v_cache, "v_cache", shape, dtype, index)
    pages, page, kv_heads, _ = shape
    _heads(heads, kv_heads, hd)
    table, lengths, starts, batch, table_pages, table_row = _sequences(tokens, page_table, lengths, starts, index)
    out = _context(out, q, tokens, heads * hd)
    held = table_pages * page
    max_length = held if max_length is None else min(int(max_length), held)
    nbytes = _lib.cache_attention_workspace_bytes(tokens, batch, heads, kv_heads, hd, page, table_pages, max_length,
                                                  starts is None, eight)
    work = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    if eight:
        ks_at, vs_at, block, strides = _scales(k_scales, v_scales, pages, page, kv_heads, index)
        args = _lib.CACHE_ATTENTION8
        try:
            packed = args.pack(
                args.size, q_at, k_half[0], v_half[0], ks_at, vs_at, table.data_ptr(), lengths.data_ptr(),
                0 if starts is None else starts.data_ptr(), out.data_ptr(), 0 if work is None else work.data_ptr(),
                nbytes, q_row, q_head, *k_half[1:], *v_half[1:], *strides, table_row, tokens, batch, heads, kv_heads,
                hd, pages, page, table_pages, max_length, block, _SEQ_DTYPES[dtype],
                hd ** -0.5 if scale is None else scale)
        except _lib.PACK_ERRORS as e:
            raise ValueError(f"cache_attention: {e}") from None
        _call("tt_cache_attention8_fwd", packed, index)
        return out
    args = _lib.CACHE_ATTENTION
    try:
        packed = args.pack(
            args.size, q_at, k_half[0], v_half[0], table.data_ptr(), lengths.data_ptr(),
            0 if starts is None else starts.data_ptr(), out.data_ptr(), 0 if work is None else work.data_ptr(), nbytes,
            q_row, q_head, *k_half[1:], *v_half[1:], table_row, tokens, batch, heads, kv_heads, hd, pages, page,
            table_pages, max_length, _SEQ_DTYPES[dtype], hd ** -0.5 if scale is None else scale, 0)
    except _lib.PACK_ERRORS as e:
        raise ValueError(f"cache_attention: {e}") from None
    _call("tt_cache_attention_fwd", packed, index)
    return out


# ---- rotary positions ----

def rotary_frequencies(dims: int, base: float = 10000.0, *, factor: float = 1.0, scaling: str = "linear",
                       original_length: Optional[int] = None, low: float = 1.0, high: float = 4.0,
                       device=None) -> torch.Tensor:
    """Frequencies of ``rotary`` for ``dims`` turned features (an even number), in radians per position: base^(-2 i / dims)
    for pair i, float64 [dims / 2], made for contexts ``factor`` times as long as those a model was trained on:

    * ``"linear"``: all divided by ``factor`` (positions are squeezed);
    * ``"base"``: a larger base, so that the slowest pair is divided by ``factor`` and the fastest stays;
    * ``"ramp"``: pairs that turn at least ``high`` times in ``original_length`` positions stay, those that turn at most
      ``low`` times are divided by ``factor``, and those between are mixed in proportion to their turns."""
    if dims <= 0 or dims % 2 or not base > 0 or not factor >= 1:
        raise ValueError(f"rotary frequencies of {dims} features with base {base} and factor {factor}")
    pair = torch.arange(dims // 2, dtype=torch.float64)
    if scaling == "base":
        if dims > 2:
            base = base * factor ** (dims / (dims - 2))
        return (base ** (-2 * pair / dims)).to(device)
    frequencies = base ** (-2 * pair / dims)
    if scaling == "ramp":
        if not original_length or original_length <= 0 or not high > low:
            raise ValueError(f"a ramp needs the original length ({original_length}) and low < high ({low}, {high})")
        turns = original_length * frequencies / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return (keep * frequencies + (1 - keep) * frequencies / factor).to(device)
    if scaling != "linear":
        raise ValueError(f"unknown scaling {scaling!r}")
    return (frequencies / factor).to(device)


class _Rotary(torch.autograd.Function):
    """``rotary`` of an x whose gradient is asked for: the result's gradient, turned back.  Rows outside every sequence are 0 in
    a new tensor, and so is their gradient; in place they stay, and their gradient passes."""

    @staticmethod
    def forward(ctx, x, frequencies, positions, lengths, starts, interleaved, magnitude, transpose, in_place):
        ctx.save_for_backward(frequencies, positions, lengths, starts)
        ctx.how = interleaved, magnitude, transpose, in_place
        if in_place:
            ctx.mark_dirty(x)
        out = x if in_place else x.new_zeros(x.shape) if starts is not None else None
        return rotary(x, frequencies, positions, lengths=lengths, starts=starts, interleaved=interleaved,
                      magnitude=magnitude, transpose=transpose, out=out)

    @staticmethod
    def backward(ctx, grad):
        interleaved, magnitude, transpose, in_place = ctx.how
        if in_place:
            grad = grad.clone(memory_format=torch.contiguous_format)
        return _Rotary.apply(grad, *ctx.saved_tensors, interleaved, magnitude, not transpose, in_place), *[None] * 8


def rotary(x: torch.Tensor, frequencies: torch.Tensor, positions: Optional[torch.Tensor] = None, *,
           lengths: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None, interleaved: bool = False,
           magnitude: float = 1.0, transpose: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turn the heads of x [T, heads, head_dim] (float16 or bfloat16) by their tokens' positions.

    ``frequencies`` (float64 [n], on the device; ``rotary_frequencies``) turns the first 2 n features of each head, in pairs
    (i, i + n) or with ``interleaved`` (2 i, 2 i + 1), by position * frequencies[i] radians, times ``magnitude``; the
    others stay.  Positions are ``positions`` (int32 [T]), or those that ``cache_append`` gives new tokens for
    ``lengths`` and ``starts`` (there rows outside every sequence are left as they are in ``out``, arbitrary in a new
    tensor).  With ``transpose`` they are turned back: the gradient of a loss for x is ``rotary`` of its gradient for the
    result with ``transpose=True``.  Where x requires a gradient, autograd is told so.

    Queries and keys that lie side by side in a projection's output are turned in one call, as heads of one tensor.
    ``out`` is x itself (in place) or a tensor that overlaps nothing, without gradients; features are adjacent in both,
    head_dim at most 256."""
    if torch.is_grad_enabled() and (x.requires_grad or out is not None and out.requires_grad):
        if out is not None and out is not x:
            raise ValueError("rotary into another tensor has no gradient: call it without out, or under torch.no_grad()")
        return _Rotary.apply(x, frequencies, positions, lengths, starts, interleaved, magnitude, transpose, out is x)
    dtype, index = _typed(x, "x")
    shape = x.shape
    if len(shape) != 3 or shape[1] == 0:
        raise ValueError("x must be a [tokens, heads, head_dim] tensor")
    tokens, heads, hd = shape
    if out is None:
        out = x.new_empty(shape)
    elif out.shape != shape or out.dtype is not dtype or out.get_device() != index:
        raise ValueError(f"out must be a {list(shape)} tensor of {dtype} on cuda:{index}")
    row, head, feature = x.stride()
    out_row, out_head, out_feature = out.stride()
    if feature != 1 and hd > 1:
        if out is x:
            raise ValueError("in place, the features of x must be adjacent")
        x = x.contiguous()
        row, head, _ = x.stride()
    if out_feature != 1 and hd > 1:
        raise ValueError("the features of out must be adjacent")
    pairs = frequencies.shape[0] if frequencies.dim() == 1 else 0
    if pairs == 0 or frequencies.dtype is not torch.float64 or frequencies.get_device() != index:
        raise ValueError(f"frequencies must be a float64 tensor of one dimension on cuda:{index}")
    frequencies = frequencies.contiguous()
    batch = 0
    if positions is not None:
        if lengths is not None or starts is not None:
            raise ValueError("either positions or lengths and starts are given")
        positions = _int32(positions, "positions", tokens, index)
    else:
        if lengths is None:
            raise ValueError("positions or lengths are needed")
        batch = lengths.shape[0] if lengths.dim() == 1 else -1
        lengths = _int32(lengths, "lengths", batch, index)
        if starts is not None:
            starts = _int32(starts, "starts", batch + 1, index)
        elif tokens != batch:
            raise ValueError(f"{tokens} tokens for {batch} sequences need starts")
    args = _lib.ROTARY_ROWS
    try:
        packed = args.pack(
            args.size, x.data_ptr(), out.data_ptr(), frequencies.data_ptr(),
            0 if positions is None else positions.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
            0 if starts is None else starts.data_ptr(), row, head, out_row, out_head, tokens, batch, heads, hd, pairs,
            interleaved, transpose, _SEQ_DTYPES[dtype], magnitude, 0)
    except _lib.PACK_ERRORS as e:
        raise ValueError(f"rotary: {e}") from None
    _call("tt_rotary", packed, index)
    return out


# ---- pages of a cache ----

def _layout(shape, stride, size: int):
    """(bytes from a page to the next, rows of a page, bytes of a row) of a tensor [pages, ...]; rows is 1 where the tokens
    of a page are not its outermost order."""
    if len(shape) < 2 or 0 in shape:
        raise ValueError("caches must be tensors [pages, page_size or blocks of it, ...] that hold something")
    rows, row = shape[1], 1
    for n, s in zip(reversed(shape[1:]), reversed(stride[1:])):
        if n != 1 and s != row:
            row = 0
            break
        row *= n
    if not row:  # in another order: dense all the same?
        rows, row = 1, 1
        for s, n in sorted((s, n) for n, s in zip(shape[1:], stride[1:]) if n != 1):
            if s != row:
                raise ValueError("a page of a cache must be a dense piece of memory")
            row *= n
    row = row // rows * size
    step = stride[0] * size
    if shape[0] > 1 and step < rows * row:
        raise ValueError("the pages of a cache must not overlap")
    return step, rows, row


def _parts(caches: Sequence[torch.Tensor], by_tokens: bool = True):
    """(their description for the library, number of tensors, pages, page size, device index) of tensors [pages, ...] each
    of whose pages is a dense piece of memory; ``by_tokens``: parts of pages will be copied."""
    described, pages, page_size, index = [], 0, 0, -1
    pack, last = _lib.CACHE_PART.pack, None
    for t in caches:
        if not t.is_cuda:
            raise ValueError("caches must be CUDA tensors")
        shape = t.shape
        what = shape, t.stride(), t.dtype
        if what != last:  # (the halves of all layers are alike)
            step, rows, row = _layout(shape, what[1], t.element_size())
            last = what
        if not described:
            pages, page_size, index = shape[0], shape[1], t.get_device()
        elif shape[0] != pages or t.get_device() != index:
            raise ValueError(f"caches must have {pages} pages each, all on cuda:{index}")
        # (a [pages, 2, page_size, ...] tensor would pass for one of two blocks a page)
        if by_tokens and shape[1] != page_size and (page_size % shape[1] or what[2] is not torch.float8_e8m0fnu):
            raise ValueError(f"caches must be [pages, {page_size}, ...], or scales [pages, {page_size} / tokens per scale, "
                             f"...]: got {list(shape)} of {what[2]}")
        described.append(pack(t.data_ptr(), step, row, rows, 0))
    if not described:
        raise ValueError("caches holds no tensor")
    return ctypes.create_string_buffer(b"".join(described)), len(described), pages, page_size, index


def _state(page_table: torch.Tensor, lengths: torch.Tensor, uses: torch.Tensor, pages: int, index: int):
    """Checks of a cache's state; (page_table, lengths, uses, batch, columns, the table's row stride)."""
    batch = lengths.shape[0] if lengths.dim() == 1 else -1
    lengths = _int32(lengths, "lengths", batch, index)
    uses = _int32(uses, "uses", pages, index)
    shape = page_table.shape
    if (len(shape) != 2 or shape[0] != batch or shape[1] == 0 or page_table.dtype is not torch.int32
            or page_table.get_device() != index):
        raise ValueError(f"page_table must be an int32 tensor [{batch}, pages per sequence] on cuda:{index}")
    if page_table.stride(1) != 1 or page_table.stride(0) < 0:
        page_table = page_table.contiguous()
    return page_table, lengths, uses, batch, shape[1], page_table.stride(0)


def cache_fork(caches: Sequence[torch.Tensor], page_table: torch.Tensor, lengths: torch.Tensor, uses: torch.Tensor,
               parents: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Continue, fork, reorder, free, extend or shorten the sequences of a paged cache -> (page_table, lengths, uses).

    Row b of the new ``page_table`` (int32 [B, n]) and ``lengths`` (int32 [B]) is what row parents[b] was (without
    ``parents``, int32 [B]: row b itself; a number outside 0 ... B - 1: an empty sequence, whose pages are given up), with
    counts[b] tokens more or fewer (``counts``, int32 [B]; none without it), so that ``cache_append`` finds room for them.
    Lengths are cut to what a row of the table holds: for a row that would pass it, appending all of its new tokens would
    write over older ones, so a program keeps to the table or makes it wider first.
    ``uses`` (int32 [pages]) counts the rows that hold each page, and holds that the program has on one besides (a prompt
    that is kept); pages with 0 are free.  Rows hold the pages of their lengths; what the table has behind those counts
    for nothing and is -1 in the new one.

    Whole pages are shared.  A page that is taken over in part is about to be written: the first row that takes it over so
    keeps it, unless a row holds it whole or the program does, and the others get copies of their tokens in all ``caches``
    (tensors [pages, page_size, ...], and of an 8-bit cache the scales [pages, page_size / tokens per scale, ...], each of
    whose pages is a dense piece of memory: K and V of every layer, one of them first).  New pages are the free ones of
    lowest number, row by row; where they run out the table has -1, whose tokens ``cache_append`` does not write.
    Nothing is read back: a step is a call whatever it comes to, and may be captured into a graph."""
    parts, count, pages, page_size, index = _parts(caches)
    page_table, lengths, uses, batch, columns, row = _state(page_table, lengths, uses, pages, index)
    if parents is not None:
        parents = _int32(parents, "parents", batch, index)
    if counts is not None:
        counts = _int32(counts, "counts", batch, index)
    work = uses.new_empty(_lib.cache_pages_workspace_bytes(batch, columns, pages), dtype=torch.uint8)
    table, after, held = uses.new_empty((batch, columns)), uses.new_empty(batch), uses.new_empty(pages)
    args = _lib.CACHE_FORK
    packed = args.pack(
        args.size, ctypes.addressof(parts), page_table.data_ptr(), lengths.data_ptr(), uses.data_ptr(),
        0 if parents is None else parents.data_ptr(), 0 if counts is None else counts.data_ptr(), table.data_ptr(),
        after.data_ptr(), held.data_ptr(), work.data_ptr(), work.numel(), row, count, batch, columns, pages, page_size, 0)
    _call("tt_cache_fork", packed, index)
    return table, after, held


def cache_compact(caches: Sequence[torch.Tensor], page_table: torch.Tensor, lengths: torch.Tensor, uses: torch.Tensor
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Move the used pages of a cache to its low end -> (page_table, uses); arguments as in ``cache_fork``.

    Of U used pages those numbered U and above go to the free numbers below U, both in rising order, in all ``caches``;
    what lies at and above U is free afterwards.  Other tables and lists of page numbers are the caller's to renumber:
    page p is used if ``uses`` is above 0, and a page that moves keeps its count."""
    parts, count, pages, page_size, index = _parts(caches)
    page_table, lengths, uses, batch, columns, row = _state(page_table, lengths, uses, pages, index)
    work = uses.new_empty(_lib.cache_pages_workspace_bytes(batch, columns, pages), dtype=torch.uint8)
    table, held = uses.new_empty((batch, columns)), uses.new_empty(pages)
    args = _lib.CACHE_COMPACT
    packed = args.pack(
        args.size, ctypes.addressof(parts), page_table.data_ptr(), lengths.data_ptr(), uses.data_ptr(), table.data_ptr(),
        held.data_ptr(), work.data_ptr(), work.numel(), row, count, batch, columns, pages, page_size, 0)
    _call("tt_cache_compact", packed, index)
    return table, held


def cache_copy(caches: Sequence[torch.Tensor], source: torch.Tensor, target: torch.Tensor) -> None:
    """Copy pages source[i] to target[i] (int32 [N], on the device) in all ``caches`` (as in ``cache_fork``, or any others
    [pages, ...] whose pages are dense), in place.

    Pairs with a number that is no page of the cache are skipped.  No target may be given twice or be a source."""
    parts, count, pages, _, index = _parts(caches, False)
    n = source.shape[0] if source.dim() == 1 else -1
    source, target = _int32(source, "source", n, index), _int32(target, "target", n, index)
    args = _lib.CACHE_COPY
    packed = args.pack(args.size, ctypes.addressof(parts), source.data_ptr(), target.data_ptr(), count, n, pages, 0)
    _call("tt_cache_copy", packed, index)

"""Per-kernel entry points over the C ABI, taking and returning torch tensors.

These are the building blocks ``tt_transformer_fwd`` chains; they are exposed for stage-level
parity tests and for callers that want one fused op (e.g. a GEMM with its epilogue) on its own.
Every function launches on the current stream of the input's device and raises on any error.
"""

from __future__ import annotations

from typing import Optional, Tuple

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


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None) -> None:
    """Write the keys and values of new tokens, k and v [T, kv_heads, head_dim], into a paged cache, in place.

    k_cache and v_cache are [pages, page_size, kv_heads, head_dim] (any strides that keep features adjacent, 16-byte
    alignment and tokens less than 2^26 elements apart, e.g. both halves of one tensor, or a permuted [pages, kv_heads, page_size, head_dim]);
    page_size is a power of two from 16 on.  Position t of sequence b lies in page page_table[b, t // page_size]
    (int32 [B, n]) at t % page_size.  ``lengths`` (int32 [B]) counts the keys of each sequence with the new ones:
    the n tokens of sequence b, rows starts[b] ... starts[b + 1] - 1 (or row b alone without ``starts``), take
    positions lengths[b] - n ... lengths[b] - 1.  Tokens whose position is negative or beyond the table, or whose
    page is no page of the cache, are not written."""
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


def cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                    max_length: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens q [T, heads, head_dim] over a paged cache that holds their keys and values already
    (``cache_append``, whose arguments these are) -> [T, heads * head_dim].

    Token i of the n new ones of sequence b sees the keys at positions 0 ... lengths[b] - n + i; one that sees none
    (a length of 0 in a padded batch) gets zeros.  Without ``starts`` every sequence has one new token.
    ``max_length`` (default: what the table can hold) is the longest length the caller expects; it only decides how
    the work is split.  Keys in a page whose number is no page of the cache are not read and count as NaN.  ``out`` may
    not overlap the other tensors."""
    dtype, index = _typed(q, "q")
    q, (tokens, heads, hd), q_at, q_row, q_head = _rows(q, "q", dtype, index)
    shape = (*k_cache.shape[:3], hd)
    k_half, v_half = _cache(k_cache, "k_cache", shape, dtype, index), _cache(v_cache, "v_cache", shape, dtype, index)
    pages, page, kv_heads, _ = shape
    _heads(heads, kv_heads, hd)
    table, lengths, starts, batch, table_pages, table_row = _sequences(tokens, page_table, lengths, starts, index)
    out = _context(out, q, tokens, heads * hd)
    held = table_pages * page
    max_length = held if max_length is None else min(int(max_length), held)
    nbytes = _lib.cache_attention_workspace_bytes(tokens, batch, heads, kv_heads, hd, page, table_pages, max_length,
                                                  starts is None)
    work = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
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

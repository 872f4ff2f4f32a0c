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


def _rows(t: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    """``t`` [T, heads, head_dim] in a form the kernels read: adjacent features, rows and heads 16 bytes aligned
    (a column slice of a fused projection's output is; anything else is copied)."""
    if t.dim() != 3 or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be a [tokens, heads, head_dim] tensor of {like.dtype} on {like.device}")
    row, head, feature = t.stride()
    if feature != 1 or (row | head) & 7 or t.data_ptr() & 15 or row >= 1 << 26:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _int32(t: torch.Tensor, name: str, like: torch.Tensor, *shape: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != like.device or t.shape != shape:
        raise ValueError(f"{name} must be an int32 tensor of shape {list(shape)} on {like.device}")
    return t.contiguous()


def _query(q: torch.Tensor, kv_heads: int, scale: Optional[float], out: Optional[torch.Tensor]):
    """Checks of a query tensor [T, heads, head_dim]; (q, out, scale)."""
    if q.dim() != 3 or q.dtype not in _SEQ_DTYPES or q.device.type != "cuda":
        raise ValueError("q must be a CUDA [tokens, heads, head_dim] tensor of float16 or bfloat16")
    tokens, heads, hd = q.shape
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} key / value heads evenly")
    if hd % 8 or not 8 <= hd <= 256:
        raise ValueError(f"head_dim {hd} is not a multiple of 8 from 8 to 256")
    if out is None:
        out = torch.empty(tokens, heads * hd, dtype=q.dtype, device=q.device)
    elif (out.shape != (tokens, heads * hd) or out.dtype != q.dtype or out.device != q.device
          or not out.is_contiguous() or out.data_ptr() & 15):
        raise ValueError("out must be a contiguous, 16-byte aligned [tokens, heads * head_dim] tensor like q")
    return _rows(q, "q", q), out, hd ** -0.5 if scale is None else float(scale)


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor, kv_heads: int, hd: int) -> int:
    """Checks of a cache's halves [pages, page_size, kv_heads, head_dim] (used in place, so never copied)."""
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dim() != 4 or t.dtype != like.dtype or t.device != like.device or t.shape[2:] != (kv_heads, hd):
            raise ValueError(f"{name} must be a [pages, page_size, {kv_heads}, {hd}] tensor of {like.dtype} on "
                             f"{like.device}")
        page, row, head, feature = t.stride()
        if feature != 1 or (page | row | head) & 7 or t.data_ptr() & 15:
            raise ValueError(f"{name} needs adjacent features, and pages, tokens and heads 16 bytes aligned")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have one shape")
    return k_cache.shape[1]


class _on_device:
    """The device of ``t`` is the current one inside."""

    def __init__(self, t: torch.Tensor):
        self.index, self.before = t.device.index, torch.cuda.current_device()

    def __enter__(self):
        if self.index != self.before:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.index != self.before:
            torch.cuda.set_device(self.before)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, *,
                     causal: bool = True, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of whole sequences packed one behind the other: q [T, heads, head_dim], k and v
    [T, kv_heads, head_dim] -> [T, heads * head_dim].

    ``starts`` (int32 [B + 1], on the device) holds the first row of each sequence and the end of the last:
    sequence b owns rows starts[b] ... starts[b + 1] - 1 and sees its own only (with ``causal``, each token those
    up to itself).  Query head h reads key / value head h // (heads // kv_heads).  ``scale`` defaults to
    head_dim^-1/2.  float16 or bfloat16, head_dim a multiple of 8 up to 256; q, k, v may be column slices of one
    projection's output.  Rows outside every sequence are left as they are in ``out`` (arbitrary in a new tensor)."""
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError("k and v must have one shape [tokens, kv_heads, head_dim]")
    q, out, scale = _query(q, k.shape[1], scale, out)
    k, v = _rows(k, "k", q), _rows(v, "v", q)
    if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError("q, k and v must have one number of tokens and one head_dim")
    if starts.dim() != 1 or starts.shape[0] == 0:
        raise ValueError("starts must be an int32 tensor of shape [B + 1]")
    starts = _int32(starts, "starts", q, starts.shape[0])
    tokens, heads, hd = q.shape
    with _on_device(q):
        rc = _lib.load().tt_packed_attention_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), starts.data_ptr(), out.data_ptr(), tokens, starts.shape[0] - 1,
            heads, k.shape[1], hd, q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
            scale, int(causal), _SEQ_DTYPES[q.dtype], _stream(q))
    _lib.check(rc, "tt_packed_attention_fwd")
    return out


def _sequences(tokens: int, page_table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor],
               like: torch.Tensor):
    """Checks of the description of a batch over a cache; (page_table, lengths, starts)."""
    if lengths.dim() != 1 or page_table.dim() != 2:
        raise ValueError("lengths must be [B] and page_table [B, pages per sequence]")
    batch = lengths.shape[0]
    lengths = _int32(lengths, "lengths", like, batch)
    if (page_table.dtype != torch.int32 or page_table.device != like.device or page_table.shape[0] != batch
            or page_table.shape[1] == 0):
        raise ValueError(f"page_table must be an int32 tensor [{batch}, pages per sequence] on {like.device}")
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    if starts is not None:
        starts = _int32(starts, "starts", like, batch + 1)
    elif tokens != batch:
        raise ValueError(f"{tokens} tokens for {batch} sequences need starts")
    return page_table, lengths, starts


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None) -> None:
    """Write the keys and values of new tokens, k and v [T, kv_heads, head_dim], into a paged cache, in place.

    k_cache and v_cache are [pages, page_size, kv_heads, head_dim] (any strides that keep features adjacent and
    16-byte alignment, e.g. both halves of one tensor, or a permuted [pages, kv_heads, page_size, head_dim]);
    page_size is a power of two from 16 on.  Position t of sequence b lies in page page_table[b, t // page_size]
    (int32 [B, n]) at t % page_size.  ``lengths`` (int32 [B]) counts the keys of each sequence with the new ones:
    the n tokens of sequence b, rows starts[b] ... starts[b + 1] - 1 (or row b alone without ``starts``), take
    positions lengths[b] - n ... lengths[b] - 1.  Tokens whose position is negative or beyond the table, or whose
    page is no page of the cache, are not written."""
    if k.dim() != 3 or k.shape != v.shape or k.dtype not in _SEQ_DTYPES or k.device.type != "cuda":
        raise ValueError("k and v must be CUDA [tokens, kv_heads, head_dim] tensors of float16 or bfloat16")
    k, v = _rows(k, "k", k), _rows(v, "v", k)
    tokens, kv_heads, hd = k.shape
    page = _cache(k_cache, v_cache, k, kv_heads, hd)
    table, lengths, starts = _sequences(tokens, page_table, lengths, starts, k)
    with _on_device(k):
        rc = _lib.load().tt_cache_append(
            k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lengths.data_ptr(),
            _ptr(starts), tokens, lengths.shape[0], kv_heads, hd, k_cache.shape[0], page, table.shape[1], k.stride(0),
            k.stride(1), v.stride(0), v.stride(1), *k_cache.stride()[:3], *v_cache.stride()[:3], table.stride(0),
            _stream(k))
    _lib.check(rc, "tt_cache_append")


def cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                    max_length: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens q [T, heads, head_dim] over a paged cache that holds their keys and values already
    (``cache_append``, whose arguments these are) -> [T, heads * head_dim].

    Token i of the n new ones of sequence b sees the keys at positions 0 ... lengths[b] - n + i; one that sees none
    (a length of 0 in a padded batch) gets zeros.  Without ``starts`` every sequence has one new token.
    ``max_length`` (default: what the table can hold) is the longest length the caller expects; it only decides how
    the work is split.  Keys in a page whose number is no page of the cache are not read and count as NaN."""
    if k_cache.dim() != 4:
        raise ValueError("k_cache must be [pages, page_size, kv_heads, head_dim]")
    kv_heads = k_cache.shape[2]
    q, out, scale = _query(q, kv_heads, scale, out)
    tokens, heads, hd = q.shape
    page = _cache(k_cache, v_cache, q, kv_heads, hd)
    table, lengths, starts = _sequences(tokens, page_table, lengths, starts, q)
    batch = lengths.shape[0]
    held = table.shape[1] * page
    max_length = held if max_length is None else min(int(max_length), held)
    nbytes = _lib.cache_attention_workspace_bytes(tokens, batch, heads, kv_heads, hd, page, table.shape[1], max_length,
                                                  starts is None)
    work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    with _on_device(q):
        rc = _lib.load().tt_cache_attention_fwd(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lengths.data_ptr(), _ptr(starts),
            out.data_ptr(), _ptr(work), nbytes, tokens, batch, heads, kv_heads, hd, k_cache.shape[0], page,
            table.shape[1], max_length, q.stride(0), q.stride(1), *k_cache.stride()[:3], *v_cache.stride()[:3],
            table.stride(0), scale, _SEQ_DTYPES[q.dtype], _stream(q))
    _lib.check(rc, "tt_cache_attention_fwd")
    return out

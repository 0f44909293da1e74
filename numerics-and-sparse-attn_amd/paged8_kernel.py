"""A paged KV cache held in 8 bits on MI355X (gfx950): rows of K and V
quantized as they are written, read back, and attended over.

The reference builds its quantized cache once per call over a contiguous cache
(quant_kernel.py:584-622) and decodes one token of every sequence at one
length.  Serving programs append to pages shared by all sequences, with a
block table and a length per sequence, and hand over single tokens, a few
drafted ones or whole prompts.  This module is the cache for that: the three
calls of a step share their arguments, and each is one call for a ragged batch.

    cache = new_paged8_cache(num_pages)                 # 4 tensors
    write_paged8_cache(k, v, *cache, block_table, seq_lens, cu_seqlens)
    o = paged8_attention(q, *cache, block_table, seq_lens, cu_seqlens)

Tensors
  k_pages, v_pages    codes, int8 or float8_e4m3fn (kv_layout as paged_kernel's):
                      "NHD" [num_pages, page_size, N_KV_HEADS, D_HEAD],
                      "HND" [num_pages, N_KV_HEADS, page_size, D_HEAD]
  k_scales, v_scales  [num_pages, N_KV_HEADS, page_size / block_size] fp32: one
                      for block_size (16, 32, 64 or 128) tokens of a KV head; a
                      code stands for code * scale
  block_table         [B, max_blocks] int32: token t of sequence b is row
                      t % page_size of page block_table[b, t // page_size]
  seq_lens            [B] int32: each sequence's tokens with its new ones
  cu_seqlens          [B + 1] int32: the new tokens of sequence b are rows
                      cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of k, v, q, and its
                      last ones in the cache; None: one new token a sequence
Nothing is read back to the host: all three can be captured into a graph, and
replayed with other contents of these tensors.  page_size is a power of two >=
16; D_HEAD == 128.
"""

import ctypes

import torch

from constants import D_HEAD, N_KV_HEADS
import _checks
import _kvdec as K

_LAYOUTS = ("NHD", "HND")
_CODES = {torch.int8: K.I8, torch.float8_e4m3fn: K.E4M3}
_MAX_LEN = 2**30   # tokens of a block-table row, less than this
_MAX_INT = 2**31 - 1


def new_paged8_cache(num_pages, n_kv_heads=N_KV_HEADS, page_size=64, block_size=32, dtype=torch.float8_e4m3fn,
                     kv_layout="NHD", device="cuda"):
    """(k_pages, v_pages, k_scales, v_scales) of an empty cache.  int8 keeps
    values of one magnitude more exactly (steps of scale), float8_e4m3fn rows
    with a few large channels (4 bits of every value)."""
    if kv_layout not in _LAYOUTS:
        raise ValueError(f"kv_layout must be one of {_LAYOUTS}, got {kv_layout!r}")
    if dtype not in _CODES:
        raise ValueError(f"dtype must be in {[str(d) for d in _CODES]}, got {dtype}")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two >= 16, got {page_size}")
    if block_size not in (16, 32, 64, 128) or block_size > page_size:
        raise ValueError(f"block_size must be 16, 32, 64 or 128 and at most page_size, got {block_size}")
    shape = ((num_pages, page_size, n_kv_heads, D_HEAD) if kv_layout == "NHD"
             else (num_pages, n_kv_heads, page_size, D_HEAD))
    pages = [torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2)]
    scales = [torch.ones((num_pages, n_kv_heads, page_size // block_size), device=device) for _ in range(2)]
    return (*pages, *scales)


def _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, kv_layout):
    """The checked cache as the library takes it, and B."""
    if kv_layout not in _LAYOUTS:
        raise ValueError(f"kv_layout must be one of {_LAYOUTS}, got {kv_layout!r}")
    _checks.require_gpu_tensor("k_pages", k_pages, dtypes=tuple(_CODES), ndim=4, contiguous=False)
    _checks.require_gpu_tensor("v_pages", v_pages, dtypes=(k_pages.dtype,), ndim=4, contiguous=False)
    _checks.require_gpu_tensor("k_scales", k_scales, dtypes=(torch.float32,), ndim=3)
    _checks.require_gpu_tensor("v_scales", v_scales, dtypes=(torch.float32,), ndim=3)
    _checks.require_gpu_tensor("block_table", block_table, dtypes=(torch.int32,), ndim=2)
    _checks.require_same_device(("k_pages", k_pages), ("v_pages", v_pages), ("k_scales", k_scales),
                                ("v_scales", v_scales), ("block_table", block_table))
    B, max_blocks = block_table.shape
    _checks.seq_lens_tensor("seq_lens", seq_lens, B, k_pages.device)
    if cu_seqlens is not None:
        _checks.seq_lens_tensor("cu_seqlens", cu_seqlens, B + 1, k_pages.device)
    if kv_layout == "NHD":
        num_pages, page_size, KVH, D = k_pages.shape
        sp, sr, sh, _ = k_pages.stride()
    else:
        num_pages, KVH, page_size, D = k_pages.shape
        sp, sh, sr, _ = k_pages.stride()
    if D != D_HEAD:
        raise ValueError(f"k_pages must have rows of {D_HEAD} channels, got {D}")
    _checks.require_shape("v_pages", v_pages, tuple(k_pages.shape))
    _checks.row_major_rows("k_pages", k_pages)
    if k_pages.stride() != v_pages.stride():
        raise ValueError(f"k_pages and v_pages must share strides, got {k_pages.stride()} and "
                         f"{v_pages.stride()}")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two >= 16, got {page_size}")
    if (sp | sr | sh) % 16 or k_pages.data_ptr() % 16 or v_pages.data_ptr() % 16:
        raise ValueError("k_pages and v_pages must have their rows on 16-byte boundaries")
    blocks = k_scales.shape[2]
    _checks.require_shape("k_scales", k_scales, (num_pages, KVH, blocks))
    _checks.require_shape("v_scales", v_scales, (num_pages, KVH, blocks))
    if blocks < 1 or page_size % blocks or page_size // blocks not in (16, 32, 64, 128):
        raise ValueError(f"k_scales and v_scales must have a scale for each 16, 32, 64 or 128 tokens of a page of "
                         f"{page_size}, got {blocks}")
    if max_blocks * page_size >= _MAX_LEN:
        raise ValueError(f"block_table must cover fewer than {_MAX_LEN} tokens a sequence, got {max_blocks} pages")
    c = K.Paged8Cache(K.ptr(k_pages), K.ptr(v_pages), K.ptr(k_scales), K.ptr(v_scales), K.ptr(block_table),
                      K.ptr(seq_lens), num_pages, sp, sr, sh, _CODES[k_pages.dtype], KVH, D, page_size,
                      page_size // blocks, max_blocks)
    return c, B


def _rows(name, x, heads, T, dtypes, device):
    """New tokens' rows [T, heads, D_HEAD]: strides are free but for the last
    dimension; rows off 16-byte boundaries are copied to ones on them."""
    _checks.require_gpu_tensor(name, x, dtypes=dtypes, ndim=3, contiguous=False)
    _checks.require_shape(name, x, (T, heads, D_HEAD))
    if x.device != device:
        raise ValueError(f"{name} must be on {device}, got {x.device}")
    _checks.row_major_rows(name, x)
    per16 = 16 // x.element_size()
    if x.data_ptr() % 16 or x.stride(0) % per16 or x.stride(1) % per16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _one_each(B, T, cu_seqlens):
    if cu_seqlens is None and T != B:
        raise ValueError(f"without cu_seqlens every sequence has one new token: expected {B} rows, got {T}")


def write_paged8_cache(k, v, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens=None,
                       kv_layout="NHD"):
    """Quantizes the new tokens' rows k, v [T, N_KV_HEADS, D_HEAD] (fp16, bf16
    or fp32; any token and head strides, e.g. views of a fused projection) into
    their places of the cache, in place.

    The scale of a block is a power of two: the least that brings every value
    of the block into the codes' range, so quotients are exact, and codes are
    the nearest ones.  A block that gets tokens later keeps the larger of its
    scale and theirs; where it grows, the codes of its earlier tokens are
    rounded to the new one (less than one step of it in all, however often it
    grows).  A block written from its first token starts anew.  NaN and
    infinities become NaN in e4m3; in int8, which has none, they make the scale
    of their block NaN until it is written from its first token again.

    Tokens without a page (a table entry outside [0, num_pages), or a position
    past the table) are dropped; other rows of the cache keep what they hold.
    Sequences of one call must not share the pages that it writes to.
    """
    if K.host.paged8_write(k, v, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens,
                           kv_layout) is not None:
        return
    c, B = _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, kv_layout)
    _checks.require_gpu_tensor("k", k, dtypes=tuple(_checks.ATTN_DTYPES), ndim=3, contiguous=False)
    T = k.shape[0]
    k = _rows("k", k, c.KVH, T, tuple(_checks.ATTN_DTYPES), k_pages.device)
    v = _rows("v", v, c.KVH, T, (k.dtype,), k_pages.device)
    _one_each(B, T, cu_seqlens)
    if T == 0:
        return
    with torch.cuda.device(k.device):
        rc = K.lib.kvdec_paged8_write(ctypes.byref(c), K.ptr(k), K.ptr(v), _checks.ATTN_DTYPES[k.dtype], k.stride(0),
                                      k.stride(1), v.stride(0), v.stride(1), K.ptr(cu_seqlens), B, T, K.stream_of(k))
    K.check(rc, "write_paged8_cache")


def read_paged8_cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens=None, num_tokens=None,
                      dtype=torch.float16, kv_layout="NHD"):
    """The last cu_seqlens[b + 1] - cu_seqlens[b] tokens of each sequence (None:
    its last one) as rows k, v [num_tokens, N_KV_HEADS, D_HEAD] of dtype (fp16,
    bf16 or fp32): code * scale, rounded once.

    num_tokens: rows of the result; None reads cu_seqlens[B] back to the host,
    which synchronises.  Rows of no sequence, or of no page, are zeros.
    """
    out = K.host.paged8_read(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, num_tokens,
                             dtype, kv_layout)
    if out is not None:
        return out
    c, B = _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, kv_layout)
    if dtype not in _checks.ATTN_DTYPES:
        raise ValueError(f"dtype must be in {[str(d) for d in _checks.ATTN_DTYPES]}, got {dtype}")
    if num_tokens is None:
        num_tokens = B if cu_seqlens is None else int(cu_seqlens[-1].item())
    T = int(num_tokens)
    if T < 0:
        raise ValueError(f"num_tokens must be >= 0, got {T}")
    _one_each(B, T, cu_seqlens)
    k = torch.empty((T, c.KVH, D_HEAD), dtype=dtype, device=k_pages.device)
    v = torch.empty_like(k)
    if B == 0:
        k.zero_()
        v.zero_()
    elif T:
        with torch.cuda.device(k.device):
            rc = K.lib.kvdec_paged8_read(ctypes.byref(c), K.ptr(cu_seqlens), B, T, K.ptr(k), K.ptr(v),
                                         _checks.ATTN_DTYPES[dtype], K.stream_of(k))
        K.check(rc, "read_paged8_cache")
    return k, v


def paged8_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens=None, sm_scale=None,
                     window=None, sink=0, kv_layout="NHD"):
    """Causal GQA attention of the new tokens over the cache, which holds them
    already: q [T, N_HEADS, D_HEAD] (fp16 or bf16; any token and head strides),
    result [T, N_HEADS, D_HEAD] of q's dtype.  Query head h reads KV head
    h // (N_HEADS // N_KV_HEADS).

    The token at position i attends to positions <= i; with a window only to
    the window's last positions (its own among them) and the first `sink`
    ones.  Tokens that attend to nothing (a length of 0) and rows of no
    sequence give zeros; table entries outside [0, num_pages) read as keys and
    values of zero.  Scales may be any positive floats.
    """
    o = K.host.paged8_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens,
                                D_HEAD**-0.5 if sm_scale is None else sm_scale, window, sink, kv_layout)
    if o is not None:
        return o
    c, B = _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, kv_layout)
    _checks.require_gpu_tensor("q", q, dtypes=(torch.float16, torch.bfloat16), ndim=3, contiguous=False)
    T, H = q.shape[:2]
    q = _rows("q", q, H, T, (q.dtype,), k_pages.device)
    if H % c.KVH:
        raise ValueError(f"N_HEADS must be a multiple of N_KV_HEADS, got {H} and {c.KVH}")
    _one_each(B, T, cu_seqlens)
    window, sink = (None if window is None else int(window)), int(sink)
    if sink < 0 or (sink > 0 if window is None else window < 1):
        raise ValueError(f"window must be None or >= 1, and sink >= 0 (0 without a window), got {window} and {sink}")
    window, sink = min(window or 0, _MAX_INT), min(sink, _MAX_INT)   # positions end before that
    o = torch.empty((T, H, D_HEAD), dtype=q.dtype, device=q.device)
    if B == 0 or o.numel() == 0:
        return o.zero_()
    if sm_scale is None:
        sm_scale = D_HEAD**-0.5
    nbytes = K.lib.kvdec_paged8_workspace_bytes(B, T, H, c.KVH, c.max_blocks * c.page_size)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        rc = K.lib.kvdec_paged8_attention(ctypes.byref(c), K.ptr(q), K.ptr(o), _checks.ATTN_DTYPES[q.dtype],
                                          q.stride(0), q.stride(1), K.ptr(cu_seqlens), B, T, H, window, sink,
                                          float(sm_scale), K.ptr(ws), nbytes, K.stream_of(q))
    K.check(rc, "paged8_attention")
    return o

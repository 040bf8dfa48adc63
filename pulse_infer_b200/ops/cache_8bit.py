"""Kernels around the 8-bit paged cache: page maps of a step, the quantising page write, decode and prompt attention.

Format of the pages (csrc/cache_8bit.cuh): a block is 16 tokens of one kv head.  Keys are [pages, kv heads, page size, d],
values transposed within a block, [pages, kv heads, page size / 16, d, 16], both ``torch.float8_e4m3fn`` or ``torch.int8``;
scales are float32 [pages, kv heads, page size / 16], powers of two: the smallest for which the block's largest magnitude is
at most 448 (e4m3) or 127 (int8) times it, from 2^-40 to 2^40.  Head sizes 64 and 128, page sizes 16, 32, 64 and 128.

Like all kernels here they launch on torch's current stream, on the current device, and raise ``KernelError`` for what they
do not take.  The reference engine stores its cache in the activation dtype only (src/runtime/kv_cache_manager.cpp:56-76).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import kernels as _k
from .kernels import BF16, DecodeWorkspace, KernelError, _on_current_device, _Record, choose_prompt_splits

BLOCK_TOKENS = 16
E4M3, INT8 = 2, 3
CACHE_8BIT_DTYPES = {torch.float8_e4m3fn: E4M3, torch.int8: INT8}
PAGE_SIZES_8BIT = (16, 32, 64, 128)
PAGE_MAPS_MAX_SEGMENTS = 4096
_PAGE_MAPS = _Record("page_maps", "pi_page_maps", 21)
_WRITE = _Record("cache_8bit", "pi_cache_8bit_write", 24, 1, (ctypes.c_void_p,))
_READ = _Record("cache_8bit", "pi_cache_8bit_read", 14)
_DECODE = _Record("attention_8bit", "pi_attention_decode_8bit", 29, 1)


def _vector(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple | None = None) -> None:
    if t.dtype is not dtype or not t.is_contiguous() or (shape is not None and t.shape != shape):
        raise KernelError(f"'{name}' must be contiguous {dtype}{'' if shape is None else ' of shape ' + str(shape)}, got "
                          f"{t.dtype} {tuple(t.shape)}")


def _window(window: int | None) -> int:
    """0: none.  Positions are 32-bit numbers, so a longer window is one that reaches everything."""
    return min(window or 0, 2 ** 31 - 1)


def cache_8bit_usable(head_dim: int, page_size: int) -> bool:
    return head_dim in (64, 128) and page_size in PAGE_SIZES_8BIT


def cache_8bit_pools(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype, device) -> tuple:
    """(kcache, vcache, kscale, vscale) of one layer: zeros."""
    if dtype not in CACHE_8BIT_DTYPES or not cache_8bit_usable(head_dim, page_size):
        raise KernelError(f"no 8-bit pages of {dtype} for head size {head_dim} and page size {page_size}")
    blocks = page_size // BLOCK_TOKENS
    k = torch.zeros((num_pages, num_kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(dtype)
    v = torch.zeros((num_pages, num_kv_heads, blocks, head_dim, BLOCK_TOKENS), dtype=torch.uint8, device=device).view(dtype)
    scales = [torch.full((num_pages, num_kv_heads, blocks), 2.0 ** -40, dtype=torch.float32, device=device) for _ in range(2)]
    return k, v, scales[0], scales[1]


def _check_pools(kcache, vcache, kscale, vscale, head_dim: int | None = None, nkv: int | None = None) -> tuple:
    """(dtype code, pages, kv heads, page size, head size)"""
    code = CACHE_8BIT_DTYPES.get(kcache.dtype)
    if code is None or vcache.dtype is not kcache.dtype:
        raise KernelError(f"8-bit pages are float8_e4m3fn or int8, keys and values alike; got {kcache.dtype} and {vcache.dtype}")
    shape = kcache.shape
    if len(shape) != 4:
        raise KernelError(f"key pages must be [pages, kv heads, page size, d], got {tuple(shape)}")
    pages, heads, page_size, d = shape
    if d not in (64, 128) or page_size not in PAGE_SIZES_8BIT:
        raise KernelError(f"8-bit pages take head sizes 64 and 128 and page sizes {PAGE_SIZES_8BIT}, not {d} and {page_size}")
    blocks = page_size // BLOCK_TOKENS
    if vcache.shape != (pages, heads, blocks, d, BLOCK_TOKENS):
        raise KernelError(f"value pages must be [{pages}, {heads}, {blocks}, {d}, {BLOCK_TOKENS}], got {tuple(vcache.shape)}")
    scale_shape = (pages, heads, blocks)
    if (kscale.shape != scale_shape or vscale.shape != scale_shape or kscale.dtype is not torch.float32
            or vscale.dtype is not torch.float32 or not kscale.is_contiguous() or not vscale.is_contiguous()):
        raise KernelError(f"scales must be contiguous float32 {list(scale_shape)}, got {kscale.dtype} {tuple(kscale.shape)} and "
                          f"{vscale.dtype} {tuple(vscale.shape)}")
    if not kcache.is_contiguous() or not vcache.is_contiguous():
        raise KernelError("8-bit pages must be contiguous")
    if (head_dim is not None and head_dim != d) or (nkv is not None and nkv != heads):
        raise KernelError(f"the pages hold {heads} kv heads of size {d}, the call says {nkv} of size {head_dim}")
    return code, pages, heads, page_size, d


# ---- page maps ------------------------------------------------------------------------------------------------------
class PageMaps(NamedTuple):
    """What ``page_maps`` builds.  R segments, T tokens, N listed pages, W pages per row of the block table."""
    slot_map: torch.Tensor       # int64 [T]     pool slot of a token: page * page size + place in the page; -1: none
    positions: torch.Tensor      # int32 [T]
    token_seg: torch.Tensor      # int32 [T]     -1 behind the last token
    seg_off: torch.Tensor        # int32 [R + 1] first token of a segment; the last entry is their number
    page_off: torch.Tensor       # int32 [R + 1] first listed page of a segment
    page_list: torch.Tensor      # int32 [N]     pool page of a listed page, -1: none
    page_tokens: torch.Tensor    # int32 [N, 2]  the tokens [first, end) of a listed page that the segment's queries can see
    table: torch.Tensor | None   # int32 [R, W]  block table of the listed pages: places in page_list, -1: not listed
    rows: torch.Tensor           # int32 [R]     0 .. R - 1: segment r's row of ``table``


def page_maps(block_table: torch.Tensor, seg_slot: torch.Tensor, seg_start: torch.Tensor, seg_len: torch.Tensor,
              page_size: int, num_tokens: int, num_listed_pages: int = 0, window: int | None = None,
              min_tokens: int = 1, with_table: bool = True) -> PageMaps:
    """Block tables and slot maps of a step from the lengths of its requests, in one launch.  Segment r brings
    ``seg_len[r]`` tokens (0 is allowed) of the request in row ``seg_slot[r]`` of ``block_table`` (int32 [slots, W]), which
    holds ``seg_start[r]`` tokens already.  ``num_tokens`` and ``num_listed_pages`` size the outputs: the sums, or more
    (entries behind are -1), or less (what does not fit is left out).  Segments of at least ``min_tokens`` tokens list the
    pages that their queries see, from the window's first on.  ``page_size``: a power of two.  ``with_table`` False: no
    ``table`` (None), for a step that lists nothing."""
    device = _on_current_device((block_table, seg_slot, seg_start, seg_len))
    R = seg_slot.numel()
    for name, t in (("seg_slot", seg_slot), ("seg_start", seg_start), ("seg_len", seg_len)):
        _vector(name, t, torch.int32, (R,))
    _vector("block_table", block_table, torch.int32)
    if block_table.dim() != 2 or not 1 <= R <= PAGE_MAPS_MAX_SEGMENTS:
        raise KernelError(f"page_maps takes a block table [slots, pages] and 1 to {PAGE_MAPS_MAX_SEGMENTS} segments, got "
                          f"{tuple(block_table.shape)} and {R}")
    if page_size <= 0 or page_size & (page_size - 1) or num_tokens < 0 or num_listed_pages < 0 or min_tokens < 1 \
            or (window is not None and window <= 0):
        raise KernelError(f"page_maps: page_size={page_size}, num_tokens={num_tokens}, num_listed_pages={num_listed_pages}, "
                          f"window={window}, min_tokens={min_tokens}")
    slots, W = block_table.shape
    T, N = int(num_tokens), int(num_listed_pages)
    # one allocation for all of them, the 64-bit ones first
    cells = R * W if with_table else 0
    sizes = (2 * T, T, T, 2 * N, R + 1, R + 1, N, cells, R)
    total = sum(sizes)
    if total >= 2147483647:
        raise KernelError("page_maps: the maps are beyond 2^31 entries")
    flat = torch.empty(total, dtype=torch.int32, device=block_table.device)
    at, ptr = flat.data_ptr(), []
    for n in sizes:
        ptr.append(at)
        at += 4 * n
    _PAGE_MAPS(device, (block_table.data_ptr(), slots, W, seg_slot.data_ptr(), seg_start.data_ptr(), seg_len.data_ptr(), R, page_size,
                        T, N, _window(window), min(min_tokens, 2 ** 31 - 1), ptr[0], ptr[1], ptr[2], ptr[4], ptr[5], ptr[6], ptr[3],
                        ptr[7] if with_table else 0, ptr[8]))
    slot_map, positions, token_seg, page_tokens, seg_off, page_off, page_list, table, rows = flat.split_with_sizes(sizes)
    return PageMaps(slot_map.view(torch.int64), positions, token_seg, seg_off, page_off, page_list, page_tokens.view(N, 2),
                    table.view(R, W) if with_table else None, rows)


# ---- writing ----------------------------------------------------------------------------------------------------------
def qk_norm_rope_write_8bit(qkv: torch.Tensor, q_weight, k_weight, eps: float, cos, sin, adjacent_pairs: bool,
                            kcache: torch.Tensor, vcache: torch.Tensor, kscale: torch.Tensor, vscale: torch.Tensor,
                            slot_map: torch.Tensor, nq: int, nkv: int, head_dim: int, error_count: torch.Tensor,
                            q_out: torch.Tensor | None = None) -> torch.Tensor:
    """``qk_norm_rope_write`` for 8-bit pages.  qkv bfloat16 [T, (nq + 2 nkv) d] is left as it is; returns the normalised,
    rotated queries, bfloat16 [T, nq d].  Keys (rounded to bfloat16 first) and values are encoded into the blocks that
    ``slot_map`` (int64 [T], see ``page_maps``) names.  Tokens with consecutive slots in one block are encoded together; a
    run that starts at a block's first token begins the block anew, another one adds to it, raising the block's scale where
    it has to (what is there is then encoded again).  The runs of a call must lie in distinct blocks.  NaN is stored as
    zero, infinity as the largest number.  A slot outside the pool is skipped and counted, once for each of the 2 nkv heads,
    in ``error_count``.  ``q_weight``/``k_weight`` None: no per-head norm; ``cos``/``sin`` None: no rotation."""
    device = _on_current_device((qkv, q_weight, k_weight, cos, sin, kcache, vcache, kscale, vscale, slot_map, error_count, q_out))
    code, pages, _, page_size, d = _check_pools(kcache, vcache, kscale, vscale, head_dim, nkv)
    width = (nq + 2 * nkv) * d
    if qkv.dtype is not torch.bfloat16 or qkv.dim() != 2 or qkv.shape[1] != width or qkv.stride(1) != 1:
        raise KernelError(f"qkv must be bfloat16 [T, {width}] with unit stride, got {qkv.dtype} {tuple(qkv.shape)}")
    T = qkv.shape[0]
    _vector("slot_map", slot_map, torch.int64, (T,))
    _vector("error_count", error_count, torch.int32, (1,))
    has_norm = q_weight is not None
    if has_norm and (k_weight is None or q_weight.shape != (d,) or k_weight.shape != (d,) or q_weight.dtype is not k_weight.dtype or not q_weight.is_contiguous() or not k_weight.is_contiguous()):
        raise KernelError("per-head norm weights must both be contiguous, of shape (head_dim,) and one dtype")
    if (cos is None) != (sin is None):
        raise KernelError("give both rotation tables or none")
    rot_pairs = 0
    if cos is not None:
        rot_pairs = cos.shape[-1]
        for t in (cos, sin):
            if t.dtype is not torch.float32 or t.shape != (T, rot_pairs) or not t.is_contiguous():
                raise KernelError("rotation tables must be contiguous float32 [T, pairs]")
    if q_out is None:
        q_out = torch.empty((T, nq * d), dtype=torch.bfloat16, device=qkv.device)
    elif q_out.dtype != torch.bfloat16 or tuple(q_out.shape) != (T, nq * d) or not q_out.is_contiguous():
        raise KernelError(f"q_out must be contiguous bfloat16 [{T}, {nq * d}]")
    launched = ctypes.c_int(0)
    _WRITE(device, (qkv.data_ptr(), qkv.stride(0) if T > 1 else width, q_weight.data_ptr() if has_norm else 0,
                    k_weight.data_ptr() if has_norm else 0, _k._code(q_weight.dtype) if has_norm else BF16, 1 if has_norm else 0,
                    cos.data_ptr() if rot_pairs else 0, sin.data_ptr() if rot_pairs else 0, rot_pairs, 1 if adjacent_pairs else 0,
                    kcache.data_ptr(), vcache.data_ptr(), kscale.data_ptr(), vscale.data_ptr(), code, pages, page_size,
                    slot_map.data_ptr(), q_out.data_ptr(), nq, nkv, d, T, error_count.data_ptr(), eps),
           extra=(ctypes.byref(launched),), launches=0)
    _k.count_launches(launched.value)
    return q_out


def _check_copy(name: str, t: torch.Tensor, N: int, nkv: int, page_size: int, d: int) -> None:
    if t.dtype != torch.bfloat16 or t.dim() != 4 or t.shape[0] < N or tuple(t.shape[1:]) != (nkv, page_size, d) or not t.is_contiguous():
        raise KernelError(f"{name} must be contiguous bfloat16 [at least {N}, {nkv}, {page_size}, {d}]")


def pages_8bit_to_bf16(kcache: torch.Tensor, vcache: torch.Tensor, kscale: torch.Tensor, vscale: torch.Tensor,
                       page_list: torch.Tensor, page_tokens: torch.Tensor | None = None, keys: torch.Tensor | None = None,
                       values: torch.Tensor | None = None) -> tuple:
    """The pages ``page_list`` (int32 [N]) as bfloat16 keys and values [N, kv heads, page size, d], exactly.  Tokens outside
    ``page_tokens`` (int32 [N, 2], [first, end) per page) and pages outside the pool become zeros.  ``keys`` / ``values``:
    where to, if given (at least N pages; pages behind are left as they are)."""
    device = _on_current_device((kcache, vcache, kscale, vscale, page_list, page_tokens, keys, values))
    code, pages, nkv, page_size, d = _check_pools(kcache, vcache, kscale, vscale)
    N = page_list.numel()
    _vector("page_list", page_list, torch.int32, (N,))
    if page_tokens is not None:
        _vector("page_tokens", page_tokens, torch.int32, (N, 2))
    out = []
    for name, t in (("keys", keys), ("values", values)):
        if t is None:
            t = torch.empty((N, nkv, page_size, d), dtype=torch.bfloat16, device=kcache.device)
        else:
            _check_copy(name, t, N, nkv, page_size, d)
        out.append(t)
    _READ(device, (kcache.data_ptr(), vcache.data_ptr(), kscale.data_ptr(), vscale.data_ptr(), code, pages, nkv, page_size, d,
                   page_list.data_ptr(), 0 if page_tokens is None else page_tokens.data_ptr(), N, out[0].data_ptr(),
                   out[1].data_ptr()), launches=1 if N else 0)
    return out[0], out[1]


# ---- attention ----------------------------------------------------------------------------------------------------------
DECODE_8BIT_SPAN_MIN = 2      # shortest share of a CTA, in 64-key tiles and cost units
DECODE_8BIT_MAX_SEGMENTS = 1024      # of a launch (A8_MAX_SEGS in csrc/attention_8bit.cu)
DECODE_8BIT_PAIR_COST = 2     # units that a (request, kv head, eight query heads) triple counts for beside its tiles


def _check_queries(what, q, q_stride, num_tokens, nq, nkv, d, window, scale, out) -> torch.Tensor:
    if q.dtype is not torch.bfloat16 or q.dim() != 2 or q.stride(1) != 1:
        raise KernelError(f"{what} takes bfloat16 queries [tokens, width] with unit stride, got {q.dtype} {tuple(q.shape)}")
    if nq <= 0 or nkv <= 0 or nq % nkv:
        raise KernelError(f"{what}: nq={nq} must be a positive multiple of nkv={nkv}")
    rows, width = q.shape
    if width < nq * d or q_stride % 8 or (rows > 1 and q_stride != q.stride(0)) or q_stride < nq * d:
        raise KernelError(f"{what}: a query stride of {q_stride} for rows of {width} elements, {q.stride(0)} apart, with {nq} heads of "
                          f"{d} (it must be a multiple of 8)")
    if not 0 <= num_tokens <= rows:
        raise KernelError(f"{what}: {num_tokens} tokens in {rows} rows of queries")
    if not scale > 0.0 or (window is not None and window <= 0):
        raise KernelError(f"{what}: scale={scale} must be positive, window={window} positive or None")
    if out is None:
        return torch.empty((num_tokens, nq * d), dtype=torch.bfloat16, device=q.device)
    if out.dtype is not torch.bfloat16 or out.shape != (num_tokens, nq * d) or not out.is_contiguous():
        raise KernelError(f"{what}: out must be contiguous bfloat16 [{num_tokens}, {nq * d}]")
    return out


def attention_decode_8bit(q: torch.Tensor, q_stride: int, kcache: torch.Tensor, vcache: torch.Tensor, kscale: torch.Tensor,
                          vscale: torch.Tensor, block_table: torch.Tensor, seg_off: torch.Tensor, seg_slot: torch.Tensor,
                          seg_start: torch.Tensor, seg_len: torch.Tensor, num_tokens: int, num_segments: int, nq: int, nkv: int,
                          head_dim: int, window: int | None, scale: float, workspace: DecodeWorkspace | None = None,
                          out: torch.Tensor | None = None, span_min: int | None = None,
                          pair_cost: int | None = None) -> torch.Tensor:
    """Single tokens over 8-bit pages (csrc/attention_8bit.cu): segments of one token, whose keys and values - the newest
    included - are in the pages; keys of pages that are not there are left out of the softmax, and a row that sees no key becomes
    zeros.  ``q`` holds the normalised, rotated query heads of token t at element offset t * q_stride.
    Rows of segments of several tokens in ``out`` [num_tokens, nq d] are left as they are (``attention_prompt_8bit``).
    At most DECODE_8BIT_MAX_SEGMENTS segments; slices of the four seg_* tensors do for more.
    ``workspace`` (made here when missing): what CTAs leave for one another; launches that share one must not overlap."""
    device = _on_current_device((q, kcache, vcache, kscale, vscale, block_table, seg_off, seg_slot, seg_start, seg_len, out))
    code, pages, _, page_size, d = _check_pools(kcache, vcache, kscale, vscale, head_dim, nkv)
    out = _check_queries("attention_decode_8bit", q, q_stride, num_tokens, nq, nkv, d, window, scale, out)
    for name, t in (("seg_off", seg_off), ("seg_slot", seg_slot), ("seg_start", seg_start), ("seg_len", seg_len)):
        if t.dtype is not torch.int32 or not t.is_contiguous() or t.numel() < num_segments:
            raise KernelError(f"'{name}' must be contiguous int32 with {num_segments} entries")
    _vector("block_table", block_table, torch.int32)
    if block_table.dim() != 2:
        raise KernelError("the block table must be [slots, pages]")
    ws = _k._decode_workspace(workspace, d, q.device)
    bt_rows, bt_stride = block_table.shape
    _DECODE(device, (q.data_ptr(), q_stride, kcache.data_ptr(), vcache.data_ptr(), kscale.data_ptr(), vscale.data_ptr(), code, pages,
                     block_table.data_ptr(), bt_rows, bt_stride, seg_off.data_ptr(), seg_slot.data_ptr(), seg_start.data_ptr(),
                     seg_len.data_ptr(), out.data_ptr(), ws.acc.data_ptr(), ws.ml.data_ptr(), ws.count.data_ptr(), ws.ctas,
                     DECODE_8BIT_SPAN_MIN if span_min is None else span_min,
                     DECODE_8BIT_PAIR_COST if pair_cost is None else pair_cost, num_tokens, num_segments, nq, nkv, d, page_size,
                     _window(window), scale))
    return out


def attention_prompt_8bit(q: torch.Tensor, q_stride: int, kcache: torch.Tensor, vcache: torch.Tensor, kscale: torch.Tensor,
                          vscale: torch.Tensor, maps: PageMaps, seg_start: torch.Tensor, seg_len: torch.Tensor, portions: list,
                          num_tokens: int, nq: int, nkv: int, head_dim: int, window: int | None, scale: float,
                          out: torch.Tensor | None = None, keys: torch.Tensor | None = None,
                          values: torch.Tensor | None = None) -> torch.Tensor:
    """Portions of prompts (segments of more than one token) over 8-bit pages: the pages that ``maps`` lists
    (``page_maps(..., min_tokens=2)`` with the same window) are expanded to bfloat16, exactly, and the tcgen05 prompt kernel
    runs on the copies.  ``portions``: (start, length) of the segments of more than one token, on the host (a replayed recording of the
    call may meet shorter ones, not longer ones).  ``keys`` /
    ``values``: bfloat16 [listed pages, kv heads, page size, d] for the copies, made here when missing; the layers of a step
    can share them.  Rows of single-token segments in ``out`` [num_tokens, nq d] are left as they are, and segments' tokens
    behind the first ``num_tokens`` are left out.  Keys of pages that the block table or the pool does not have are left out
    of the softmax, as ``attention_decode_8bit`` leaves them out; a row that sees no key at all becomes zeros."""
    device = _on_current_device((q, kcache, vcache, kscale, vscale, seg_start, seg_len, out, keys, values, maps.page_list, maps.table))
    code, pages, _, page_size, d = _check_pools(kcache, vcache, kscale, vscale, head_dim, nkv)
    if maps.table is None:
        raise KernelError("attention_prompt_8bit needs page maps with their table")
    out = _check_queries("attention_prompt_8bit", q, q_stride, num_tokens, nq, nkv, d, window, scale, out)
    R = maps.rows.numel()
    _vector("seg_start", seg_start, torch.int32, (R,))
    _vector("seg_len", seg_len, torch.int32, (R,))
    portions = [p for p in portions if p[1] > 1]
    if not portions or num_tokens == 0:
        return out
    longest = need = 0
    for start, n in portions:
        longest = max(longest, n)
        first = max(0, start - window + 1) // page_size if window else 0
        last = (start + n - 1) // page_size
        need += last - first + 1
        if start < 0 or last >= maps.table.shape[1]:
            raise KernelError(f"a portion from {start} to {start + n - 1} is beyond a block table of {maps.table.shape[1]} pages of {page_size}")
    if maps.page_list.numel() < need or maps.token_seg.numel() < num_tokens:
        raise KernelError(f"the page maps list {maps.page_list.numel()} pages and {maps.token_seg.numel()} tokens, the portions "
                          f"have {need} and {num_tokens}")
    N, W = maps.page_list.numel(), maps.table.shape[1]
    _vector("page_list", maps.page_list, torch.int32, (N,))
    _vector("page_tokens", maps.page_tokens, torch.int32, (N, 2))
    _vector("table", maps.table, torch.int32, (R, W))
    splits = choose_prompt_splits(portions, nq // nkv, nkv, window)
    rows = num_tokens * nq * splits if splits > 1 else 0
    # the copies and the shares' scratch in one allocation: pages are multiples of 2,048 bytes, a share's row of 256
    pages_bytes = 2 * N * nkv * page_size * d
    made = (keys is None) + (values is None)
    scratch = torch.empty(made * pages_bytes + rows * (4 * d + 8), dtype=torch.uint8, device=q.device)
    at = scratch.data_ptr()
    where = []
    for name, t in (("keys", keys), ("values", values)):
        if t is None:
            where.append(at)
            at += pages_bytes
        else:
            _check_copy(name, t, N, nkv, page_size, d)
            where.append(t.data_ptr())
    _READ(device, (kcache.data_ptr(), vcache.data_ptr(), kscale.data_ptr(), vscale.data_ptr(), code, pages, nkv, page_size, d,
                   maps.page_list.data_ptr(), maps.page_tokens.data_ptr(), N, where[0], where[1]), launches=1 if N else 0)
    _k._PROMPT(device, (q.data_ptr(), q_stride, where[0], where[1], N, maps.table.data_ptr(), W, maps.seg_off.data_ptr(),
                        maps.rows.data_ptr(), seg_start.data_ptr(), seg_len.data_ptr(), out.data_ptr(), R, longest, nq, nkv, page_size,
                        _window(window), splits, at if rows else 0, at + rows * 4 * d if rows else 0, maps.token_seg.data_ptr(), num_tokens,
                        maps.page_list.data_ptr(), pages, scale), launches=2 if splits > 1 else 1, head_dim=d)
    return out

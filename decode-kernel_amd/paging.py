"""Page tables and cache writes around the decode path, on the device.

`build_page_table` turns a serving framework's per-request token-slot map (SGLang's
ReqToTokenPool.req_to_token) into the CSR page table of src/layout.md:27-138 with one
kernel launch (libdk_decode.so: dk_build_page_table), so a decode step needs no host round
trip. Tokens are assumed to sit in 16-token pages: token t of a request at slot
16 * page + t % 16, as a paged allocator with page_size 16 places them (or one with a
page_size that is a multiple of 16: each of its pages is a run of aligned 16-slot pages).

`grow_block_tables` builds a step's tables from request lengths instead: block tables extended by
the pages that the new tokens need, the page table, and the new tokens' slots and positions.
`append_kv` writes one token per sequence into a cache; `write_kv4` and `read_kv4` write and read
any tokens of a 4-bit cache by slot.
"""
from __future__ import annotations

import ctypes
import math
import sys
from typing import NamedTuple, Optional

import torch

import dk_lib
import layout
from dk_lib import DecodeArgumentError

PAGE_SIZE = 16


def page_capacity(seq_lens_sum: int, batch: int) -> int:
    """kv_indices entries that always suffice: sum(ceil(len / 16)) <= (sum + 15 B) / 16."""
    return (int(seq_lens_sum) + (PAGE_SIZE - 1) * int(batch)) // PAGE_SIZE


def _index_array(t: torch.Tensor, dev) -> torch.Tensor:
    """t on dev, contiguous, int32 or int64 (which the page-table kernel reads as it is)."""
    if t.dtype != torch.int64:
        t = t.to(device=dev, dtype=torch.int32)
    return t.to(device=dev).contiguous()


def build_page_table(req_to_token: torch.Tensor, req_pool_indices: torch.Tensor,
                     seq_lens: torch.Tensor, capacity: Optional[int] = None,
                     seq_lens_sum: Optional[int] = None, out=None):
    """(kv_indptr (B+1,), kv_indices (capacity,), kv_last_page_len (B,)) int32 on the device.

    req_to_token     : (rows, max_tokens) int32 cache slot of each request's tokens
    req_pool_indices : (B,) row of each request (int32 or int64)
    seq_lens         : (B,) tokens per request (int32 or int64)
    capacity         : size of kv_indices; default page_capacity(seq_lens_sum, B), with
                       seq_lens_sum (a host integer) required then. Entries past the
                       table's total are left uninitialised.
    out              : optional persistent (kv_indptr, kv_indices, kv_last_page_len)
                       buffers to fill in place (at least B + 1, capacity and B entries),
                       e.g. for tables a captured HIP graph reads; capacity defaults to
                       the kv_indices buffer's size then
    """
    if req_to_token.dtype != torch.int32 or req_to_token.dim() != 2:
        raise DecodeArgumentError("req_to_token must be a 2-D int32 tensor")
    if req_to_token.stride(1) != 1:
        raise DecodeArgumentError("req_to_token rows must be contiguous")
    dev = req_to_token.device
    batch = int(seq_lens.shape[0])
    if req_pool_indices.shape[0] != batch:
        raise DecodeArgumentError("req_pool_indices and seq_lens must have one entry per request")
    if out is not None:
        kv_indptr, kv_indices, kv_last = out
        if capacity is None:
            capacity = kv_indices.numel()
        if (kv_indptr.numel() < batch + 1 or kv_indices.numel() < capacity or
                kv_last.numel() < batch or
                any(t.dtype != torch.int32 or t.device != dev or not t.is_contiguous()
                    for t in out)):
            raise DecodeArgumentError("out buffers must be contiguous int32 on the table's "
                                      "device, with B + 1, capacity and B entries")
    elif capacity is None:
        if seq_lens_sum is None:
            raise DecodeArgumentError("give capacity or seq_lens_sum (a host integer)")
        capacity = page_capacity(seq_lens_sum, batch)
    rpi, lens = _index_array(req_pool_indices, dev), _index_array(seq_lens, dev)
    if out is None:
        kv_indptr = torch.empty(batch + 1, dtype=torch.int32, device=dev)
        kv_indices = torch.empty(max(int(capacity), 1), dtype=torch.int32, device=dev)
        kv_last = torch.empty(batch, dtype=torch.int32, device=dev)
    if batch == 0:
        kv_indptr[:1].zero_()
        return kv_indptr[:1], kv_indices[:0], kv_last[:0]
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        rc = dk_lib.load().dk_build_page_table_wide(
            req_to_token.data_ptr(), req_to_token.stride(0), rpi.data_ptr(),
            rpi.dtype == torch.int64, lens.data_ptr(), lens.dtype == torch.int64, batch,
            PAGE_SIZE, kv_indptr.data_ptr(), kv_indices.data_ptr(), int(capacity),
            kv_last.data_ptr(), stream)
    dk_lib.check(rc, "build_page_table")
    return kv_indptr[:batch + 1], kv_indices[:int(capacity)], kv_last[:batch]


class StepTables(NamedTuple):
    """A step's tables on the device, all int32 (see grow_block_tables)."""
    kv_indptr: torch.Tensor           # (B + 1,)
    kv_indices: torch.Tensor          # (capacity,)
    kv_last_page_len: torch.Tensor    # (B,)
    q_indptr: torch.Tensor            # (B + 1,)
    slots: torch.Tensor               # (num_tokens,)
    positions: torch.Tensor           # (num_tokens,)


def _call(dev, fn, *args) -> int:
    """fn(*args, stream) on `dev` and torch's current stream there."""
    if dev.index == torch.cuda.current_device():
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    with torch.cuda.device(dev):
        return fn(*args, torch.cuda.current_stream(dev).cuda_stream)


_NATIVE = None   # _dk_native once bound to the loaded library; False where it is not usable


def _native():
    """_dk_native with the calls of a 4-bit cache's step bound, or False (csrc/dk_native.cpp). It takes
    the plain ones, each at about the cost of its launch: grow_block_tables costs 4.7 us on the host
    against 13.1 in Python, write_kv4 3.1 against 11.1, read_kv4 3.8 against 8.9,
    extend.extend_attention_kv4 5.5 against 15.2."""
    global _NATIVE
    if _NATIVE is None:
        import attention
        decode = attention._bind_native()
        module = sys.modules.get("_dk_native")
        if module is not None and getattr(module, "decode", None) is decode and \
                hasattr(module, "extend_attention_kv4"):
            lib = dk_lib.load()
            module.bind_paging(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
                lib.dk_grow_block_tables, lib.dk_kv4_write, lib.dk_kv4_read,
                lib.dk_extend_attention_kv4, lib.dk_extend_kv4_workspace_bytes)))
            _NATIVE = module
        else:
            _NATIVE = False
    return _NATIVE


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise DecodeArgumentError(msg)


def _on_one_gpu(what: str, dev, **tensors) -> None:
    """All given tensors (None passes) lie on the GPU `dev`: the kernels address them there."""
    _need(dev.type == "cuda", f"{what} needs tensors on a GPU, got {dev}")
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise DecodeArgumentError(f"{what}: {name} must be on {dev}, got {t.device}")


def _index_vector(what: str, name: str, t, n: Optional[int] = None):
    """t, checked to be a 1-D int32 or int64 tensor (of n entries), contiguous."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    _need(t.dtype in (torch.int32, torch.int64) and t.dim() == 1,
          f"{what}: {name} must be a 1-D int32 or int64 tensor")
    _need(n is None or t.shape[0] == n, f"{what}: {name} must have {n} entries, got {t.shape[0]}")
    return t if t.is_contiguous() else t.contiguous()


def _host_int(what: str, name: str, v) -> int:
    _need(isinstance(v, int) and not isinstance(v, bool) and 0 <= v < 2 ** 31,
          f"{what}: {name} must be a host integer in [0, 2^31), got {v!r}")
    return v


def grow_block_tables(block_table: torch.Tensor, rows: torch.Tensor, cached_lens: torch.Tensor,
                      new_lens: torch.Tensor, new_pages: torch.Tensor, num_tokens: int,
                      capacity: int, out: Optional[StepTables] = None) -> StepTables:
    """The tables of a step that adds new tokens to requests, built on the GPU in one launch
    without a host read (dk_grow_block_tables).

    block_table : (rows, max_blocks) int32, written in place: entry i of a request's row is the
                  page of its tokens 16 i .. 16 i + 15
    rows        : (B,) row of each request (distinct)
    cached_lens : (B,) tokens that each request has in the cache
    new_lens    : (B,) tokens to come (1 in a decode step; 0 is fine)
    new_pages   : page ids for the blocks that the new tokens need, in request order; a host that
                  knows the lengths passes sum(ceil((cached + new) / 16) - ceil(cached / 16)) free
                  pages (more are left alone; a block past their end gets page -1, its tokens slot -1)
    num_tokens  : entries of slots and positions, at least sum(new_lens); those behind the last new
                  token get slot -1 and position 0, which write_kv4 skips
    capacity    : entries of kv_indices (those past the table's total are left as they are)
    out         : optional StepTables of at least these sizes to fill in place, e.g. tables that a
                  captured HIP graph reads; kv_indices and slots / positions may be larger

    rows, cached_lens and new_lens are int32 or int64. Returns StepTables: kv_indptr, kv_indices
    and kv_last_page_len as build_page_table's, q_indptr (the requests' new tokens), slots
    (16 * page + position % 16) and positions of the new tokens. A row outside the table, a
    negative length or one beyond 16 * max_blocks leaves a request without pages."""
    what = "grow_block_tables"
    native = _NATIVE or _native()
    if native and out is None:
        got = native.grow_block_tables(block_table, rows, cached_lens, new_lens, new_pages,
                                       num_tokens, capacity)
        if type(got) is tuple:
            return tuple.__new__(StepTables, got)
        if got is not None:
            dk_lib.check(got, what)
    for name, t in (("block_table", block_table), ("new_pages", new_pages)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and
          (block_table.stride(1) == 1 or block_table.shape[1] <= 1),
          f"{what}: block_table must be a 2-D int32 tensor of contiguous rows")
    _need(block_table.shape[0] <= 1 or block_table.stride(0) >= block_table.shape[1],
          f"{what}: the rows of block_table overlap")
    rows = _index_vector(what, "rows", rows)
    batch = rows.shape[0]
    cached_lens = _index_vector(what, "cached_lens", cached_lens, batch)
    new_lens = _index_vector(what, "new_lens", new_lens, batch)
    _need(new_pages.dtype == torch.int32 and new_pages.dim() == 1,
          f"{what}: new_pages must be a 1-D int32 tensor")
    new_pages = new_pages if new_pages.is_contiguous() else new_pages.contiguous()
    num_tokens = _host_int(what, "num_tokens", num_tokens)
    capacity = _host_int(what, "capacity", capacity)
    dev = block_table.device
    _on_one_gpu(what, dev, rows=rows, cached_lens=cached_lens, new_lens=new_lens,
                new_pages=new_pages)
    sizes = (batch + 1, capacity, batch, batch + 1, num_tokens, num_tokens)
    if out is None:
        t = StepTables(*torch.empty(sum(sizes), dtype=torch.int32, device=dev).split(sizes))
    else:
        for name, x, n in zip(StepTables._fields, out, sizes):
            _need(isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.dim() == 1 and
                  x.is_contiguous() and x.device == dev and x.shape[0] >= n,
                  f"{what}: out.{name} must be a contiguous int32 tensor of at least {n} entries "
                  f"on {dev}")
        t = StepTables(*(x[:n] for x, n in zip(out, sizes)))
    if batch == 0:
        t.kv_indptr.zero_()
        t.q_indptr.zero_()
        t.slots.fill_(-1)
        t.positions.zero_()
        return t
    i64 = torch.int64
    rc = _call(dev, dk_lib.load().dk_grow_block_tables, block_table.data_ptr(),
               block_table.stride(0), block_table.shape[0], block_table.shape[1], rows.data_ptr(),
               rows.dtype == i64, cached_lens.data_ptr(), cached_lens.dtype == i64,
               new_lens.data_ptr(), new_lens.dtype == i64, new_pages.data_ptr(),
               new_pages.shape[0], batch, t.kv_indptr.data_ptr(), t.kv_indices.data_ptr(),
               capacity, t.kv_last_page_len.data_ptr(), t.q_indptr.data_ptr(),
               t.slots.data_ptr(), t.positions.data_ptr(), num_tokens)
    dk_lib.check(rc, what)
    return t


def expand_page_table(kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                      kv_last_page_len: torch.Tensor, page_size: int, pages_mult: int,
                      num_pages: int):
    """The page table of a cache with pages of page_size = 16 * s tokens, rewritten over
    its 16-token sub-pages (dk_expand_page_table): sub-page j of page p is id
    p * pages_mult + j. Returns (kv_indptr (B+1,), kv_indices (len(kv_indices) * s,),
    kv_last_page_len (B,)) int32 on the same device; entries past the new table's total
    are left uninitialised. No host synchronisation."""
    for name, t in (("kv_indptr", kv_indptr), ("kv_indices", kv_indices),
                    ("kv_last_page_len", kv_last_page_len)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1 or \
                not t.is_contiguous():
            raise DecodeArgumentError(f"{name} must be a contiguous 1-D int32 tensor")
    if page_size <= 0 or page_size % PAGE_SIZE:
        raise DecodeArgumentError(f"page_size must be a positive multiple of 16, got {page_size}")
    if kv_indptr.shape[0] < 1 or kv_last_page_len.shape[0] != kv_indptr.shape[0] - 1:
        raise DecodeArgumentError(
            f"kv_last_page_len must have one entry per sequence (len(kv_indptr) - 1 = "
            f"{kv_indptr.shape[0] - 1}); got {kv_last_page_len.shape[0]}")
    dev = kv_indptr.device
    # the kernel reads all three tables on one GPU: host memory there would fault it
    if dev.type != "cuda" or kv_indices.device != dev or kv_last_page_len.device != dev:
        raise DecodeArgumentError(
            f"kv_indptr, kv_indices and kv_last_page_len must be on one GPU; got "
            f"{kv_indptr.device}, {kv_indices.device}, {kv_last_page_len.device}")
    batch = int(kv_indptr.shape[0]) - 1
    sub = page_size // PAGE_SIZE
    capacity = int(kv_indices.shape[0]) * sub
    out_indptr = torch.empty(batch + 1, dtype=torch.int32, device=dev)
    out_indices = torch.empty(max(capacity, 1), dtype=torch.int32, device=dev)
    out_last = torch.empty(max(batch, 0), dtype=torch.int32, device=dev)
    if batch <= 0:
        out_indptr.zero_()
        return out_indptr, out_indices[:0], out_last
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        rc = dk_lib.load().dk_expand_page_table(
            kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_last_page_len.data_ptr(), batch,
            int(page_size), int(pages_mult), int(num_pages), int(kv_indices.shape[0]),
            out_indptr.data_ptr(), out_indices.data_ptr(), capacity, out_last.data_ptr(),
            stream)
    dk_lib.check(rc, "expand_page_table")
    return out_indptr, out_indices[:capacity], out_last


def rope_inv_freq(head_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """Plain rotary frequencies theta^(-2i/head_dim), i < head_dim/2, fp32. Frequency
    scalings (Llama 3's, YaRN, ...) produce their own inv_freq and pass it instead."""
    i = torch.arange(0, head_dim, 2, dtype=torch.float64)
    return (1.0 / (theta ** (i / head_dim))).to(device=device, dtype=torch.float32)


def append_kv(q: Optional[torch.Tensor], k_new: torch.Tensor, v_new: torch.Tensor, kv_data,
              kv_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor,
              inv_freq: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
              rope_style: int = 0, k_scale: Optional[float] = None,
              v_scale: Optional[float] = None) -> None:
    """Write each sequence's new token into the paged cache (dk_append_kv), in place.

    The token's slot is the last one the page table describes (grow the table first).
    q (batch, num_q_heads, head_dim) or None is rotated in place; k_new / v_new
    (batch, num_kv_heads, head_dim) are the token's K (rotated on the way in) and V rows;
    kv_data is the combined cache or a (k_cache, v_cache) pair as for decode_attention.
    inv_freq (head_dim/2,) fp32 on the device, or None for no rotation; positions (batch,)
    int32, or None for each token's index in its sequence; rope_style 0 = rotate-half
    pairs (i, i + D/2) (Llama), 1 = interleaved pairs (2i, 2i + 1).
    A torch.float8_e4m3fn cache (q, k_new, v_new fp16 or bf16) stores each element as
    RNE(clamp(x / scale, -448, 448)) with k_scale for K and v_scale for V (None = 1), the
    scales decode_attention then takes. A 4-bit cache (layout.alloc_kv4_cache) is written as by
    write_kv4.
    """
    import attention                     # local: attention imports nothing from here
    if layout.is_kv4(kv_data):
        _need(k_scale in (None, 1.0) and v_scale in (None, 1.0),
              "append_kv: k_scale and v_scale apply to a torch.float8_e4m3fn cache only")
        return _append_kv4(q, k_new, v_new, kv_data, kv_indptr, kv_indices, kv_last_page_len,
                           inv_freq, positions, rope_style)
    kv = attention._kv_layout(kv_data)
    batch, hkv, d = k_new.shape
    kv8 = kv.dtype == attention.KV_FP8
    act = k_new.dtype if kv8 else kv.dtype          # type of q, k_new and v_new
    if kv8 and act not in (torch.float16, torch.bfloat16):
        raise DecodeArgumentError("over an fp8 cache k_new and v_new must be fp16 or bf16")
    if v_new.shape != k_new.shape or k_new.dtype != act or v_new.dtype != act:
        raise DecodeArgumentError("k_new and v_new must be (batch, num_kv_heads, head_dim) in "
                                  "the cache's dtype (fp16 / bf16 over an fp8 cache)")
    scales = []
    for name, x in (("k_scale", k_scale), ("v_scale", v_scale)):
        if not kv8:
            if x not in (None, 1.0):
                raise DecodeArgumentError(f"{name} applies to a torch.float8_e4m3fn cache only")
            continue
        x = 1.0 if x is None else float(x)
        if not math.isfinite(x) or x <= 0.0:
            raise DecodeArgumentError(f"{name} must be finite and > 0, got {x}")
        scales.append(x)
    if v_new.stride() != k_new.stride() or k_new.stride(2) != 1:
        raise DecodeArgumentError("k_new and v_new need equal strides and a unit head_dim stride")
    if hkv != kv.hkv or d != kv.d or kv.page_size != PAGE_SIZE or kv.d_stride != 1:
        raise DecodeArgumentError("k_new does not match the cache's heads / head_dim")
    if q is not None and (q.dim() != 3 or q.shape[0] != batch or q.shape[2] != d or
                          q.dtype != act or q.stride(2) != 1):
        raise DecodeArgumentError("q must be (batch, num_q_heads, head_dim) in k_new's dtype")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() != d // 2
                                 or not inv_freq.is_contiguous()):
        raise DecodeArgumentError("inv_freq must be a contiguous fp32 tensor of head_dim/2")
    if positions is not None:
        positions = positions.to(dtype=torch.int32).contiguous()
    s = dk_lib.DkStrides()
    if q is not None:
        s.q_b, s.q_h = q.stride(0), q.stride(1)
    s.kv_p, s.kv_r, s.kv_s, s.kv_h = kv.strides
    code = dk_lib.DK_F16 if act == torch.float16 else dk_lib.DK_BF16
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    lib = dk_lib.load()
    with torch.cuda.device(k_new.device):
        stream = torch.cuda.current_stream(k_new.device).cuda_stream
        args = (ptr(q), k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0), k_new.stride(1),
                kv.k.data_ptr(), ptr(kv.v), kv_indptr.data_ptr(), kv_indices.data_ptr(),
                kv_last_page_len.data_ptr(), ptr(positions), ptr(inv_freq), rope_style, batch,
                q.shape[1] if q is not None else 1, hkv, d, PAGE_SIZE, kv.num_pages,
                kv_indices.shape[0], code)
        if kv8:
            rc = lib.dk_append_kv_fp8(*args, *scales, ctypes.byref(s), stream)
        else:
            rc = lib.dk_append_kv(*args, ctypes.byref(s), stream)
    dk_lib.check(rc, "append_kv")


# ---- the 4-bit cache

_KV4_TYPES = {torch.float16: dk_lib.DK_F16, torch.bfloat16: dk_lib.DK_BF16}


def _kv4_cache(what: str, cache) -> int:
    """head_dim of a 4-bit cache, or DecodeArgumentError."""
    try:
        return layout.kv4_head_dim(cache)
    except layout.LayoutError as exc:
        raise DecodeArgumentError(f"{what}: {exc}") from None


def _kv4_rows(what: str, q, k_new, v_new, cache, inv_freq, rope_style):
    """Checks of the rows written into a 4-bit cache; (dtype code, strides, head_dim)."""
    for name, t in (("k_new", k_new), ("v_new", v_new)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    d = _kv4_cache(what, cache)
    _need(k_new.dim() == 3 and k_new.dtype in _KV4_TYPES and v_new.shape == k_new.shape and
          v_new.dtype == k_new.dtype,
          f"{what}: k_new and v_new must both be (tokens, num_kv_heads, head_dim), fp16 or bf16")
    _need(k_new.shape[1] == cache.shape[1] and k_new.shape[2] == d,
          f"{what}: k_new has {k_new.shape[1]} heads of {k_new.shape[2]}, the cache "
          f"{cache.shape[1]} of {d}")
    _need(v_new.stride() == k_new.stride() and k_new.stride(2) == 1,
          f"{what}: k_new and v_new need equal strides and a unit head_dim stride")
    if q is not None:
        _need(isinstance(q, torch.Tensor) and q.dim() == 3 and q.shape[0] == k_new.shape[0] and
              q.shape[2] == d and q.dtype == k_new.dtype and q.stride(2) == 1,
              f"{what}: q must be (tokens, num_q_heads, head_dim) in k_new's dtype")
    if inv_freq is not None:
        _need(isinstance(inv_freq, torch.Tensor) and inv_freq.dtype == torch.float32 and
              inv_freq.numel() == d // 2 and inv_freq.is_contiguous(),
              f"{what}: inv_freq must be a contiguous fp32 tensor of head_dim / 2")
    _need(rope_style in (0, 1), f"{what}: rope_style must be 0 or 1, got {rope_style!r}")
    s = dk_lib.DkStrides()
    if q is not None:
        s.q_b, s.q_h = q.stride(0), q.stride(1)
    s.kv_p, s.kv_h = cache.stride(0), cache.stride(1)
    return _KV4_TYPES[k_new.dtype], s, d


def write_kv4(k_new: torch.Tensor, v_new: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor,
              q: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
              positions: Optional[torch.Tensor] = None, rope_style: int = 0) -> None:
    """Write tokens' K and V rows into a 4-bit cache by slot, in place (dk_kv4_write): a decode
    step's tokens or a prefill's, as grow_block_tables places them.

    k_new, v_new : (tokens, num_kv_heads, head_dim) fp16 or bf16
    cache        : uint8 (num_pages, num_kv_heads, 17 * head_dim), layout.alloc_kv4_cache
    slots        : (tokens,) int32 or int64, 16 * page + token of the page; distinct; one outside the
                   cache (-1) writes nothing
    q            : (tokens, num_q_heads, head_dim) or None, rotated in place (every row)
    inv_freq     : (head_dim / 2,) fp32, or None for no rotation; positions (tokens,) int32 or int64
                   are needed with it
    rope_style   : 0 = pairs (i, i + D/2), 1 = pairs (2i, 2i + 1)

    K is rotated on the way in. Blocks of 32 dims share a power-of-two scale that puts the largest
    magnitude in [3.5, 7) of E2M1's 6; each element is the nearest code, ties to even. A block with a NaN
    or an infinity reads as NaN."""
    what = "write_kv4"
    native = _NATIVE or _native()
    if native:
        rc = native.write_kv4(k_new, v_new, cache, slots, q, inv_freq, positions, rope_style)
        if rc is not None:
            return dk_lib.check(rc, what)
    dtype, s, d = _kv4_rows(what, q, k_new, v_new, cache, inv_freq, rope_style)
    n = k_new.shape[0]
    slots = _index_vector(what, "slots", slots, n)
    if positions is not None:
        positions = _index_vector(what, "positions", positions, n)
    _need(inv_freq is None or positions is not None, f"{what}: inv_freq needs positions")
    dev = cache.device
    _on_one_gpu(what, dev, k_new=k_new, v_new=v_new, slots=slots, q=q, inv_freq=inv_freq,
                positions=positions)
    if n == 0:
        return
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rc = _call(dev, dk_lib.load().dk_kv4_write, ptr(q), k_new.data_ptr(), v_new.data_ptr(),
               k_new.stride(0), k_new.stride(1), cache.data_ptr(), slots.data_ptr(),
               slots.dtype == torch.int64, ptr(positions),
               positions is not None and positions.dtype == torch.int64, ptr(inv_freq), rope_style,
               n, 1 if q is None else q.shape[1], cache.shape[1], d, cache.shape[0], dtype,
               ctypes.byref(s))
    dk_lib.check(rc, what)


def _append_kv4(q, k_new, v_new, cache, kv_indptr, kv_indices, kv_last_page_len, inv_freq,
                positions, rope_style) -> None:
    """append_kv into a 4-bit cache (dk_kv4_append)."""
    what = "append_kv"
    dtype, s, d = _kv4_rows(what, q, k_new, v_new, cache, inv_freq, rope_style)
    n = k_new.shape[0]
    tables = []
    for name, t, m in (("kv_indptr", kv_indptr, n + 1), ("kv_indices", kv_indices, None),
                       ("kv_last_page_len", kv_last_page_len, n)):
        _need(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == 1 and
              (m is None or t.shape[0] == m),
              f"{what}: {name} must be a 1-D int32 tensor" + (f" of {m} entries" if m else ""))
        tables.append(t if t.is_contiguous() else t.contiguous())
    if positions is not None:
        positions = _index_vector(what, "positions", positions, n).to(torch.int32)
    dev = cache.device
    _on_one_gpu(what, dev, k_new=k_new, v_new=v_new, q=q, inv_freq=inv_freq, positions=positions,
                kv_indptr=kv_indptr, kv_indices=kv_indices, kv_last_page_len=kv_last_page_len)
    if n == 0:
        return
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rc = _call(dev, dk_lib.load().dk_kv4_append, ptr(q), k_new.data_ptr(), v_new.data_ptr(),
               k_new.stride(0), k_new.stride(1), cache.data_ptr(), *(t.data_ptr() for t in tables),
               ptr(positions), ptr(inv_freq), rope_style, n, 1 if q is None else q.shape[1],
               cache.shape[1], d, cache.shape[0], kv_indices.shape[0], dtype, ctypes.byref(s))
    dk_lib.check(rc, what)


def read_kv4(cache: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """The K and V rows that a 4-bit cache holds in the given slots, each (len(slots), num_kv_heads,
    head_dim) of `dtype` (dk_kv4_read): exact in bf16, in fp16 beyond 65,504 infinite. A slot
    outside the cache reads as zeros. For moving cached tokens to another cache, and for attention
    that no kernel here runs."""
    what = "read_kv4"
    native = _NATIVE or _native()
    if native and dtype in _KV4_TYPES:
        got = native.read_kv4(cache, slots, _KV4_TYPES[dtype])
        if type(got) is tuple:
            return got
        if got is not None:
            dk_lib.check(got, what)
    d = _kv4_cache(what, cache)
    _need(dtype in _KV4_TYPES, f"{what}: dtype must be fp16 or bf16, got {dtype}")
    slots = _index_vector(what, "slots", slots)
    dev = cache.device
    _on_one_gpu(what, dev, slots=slots)
    n, hkv = slots.shape[0], cache.shape[1]
    k, v = torch.empty(2, n, hkv, d, dtype=dtype, device=dev).unbind(0)
    if n == 0 or hkv == 0:
        return k, v
    rc = _call(dev, dk_lib.load().dk_kv4_read, cache.data_ptr(), cache.stride(0), cache.stride(1),
               slots.data_ptr(), slots.dtype == torch.int64, k.data_ptr(), v.data_ptr(), hkv * d, d,
               n, hkv, d, cache.shape[0], _KV4_TYPES[dtype])
    dk_lib.check(rc, what)
    return k, v

"""A KV cache held in 4 bits: written as tokens arrive, read back, and attended over without being expanded in memory.

A cached row (one token, one KV head) is cut into groups of ``group`` channels.  A group keeps its smallest value ``low``
and ``scale`` = (max - low) / 15, both rounded to the cache's 16-bit type, and 4 bits per channel:
``code = round((x - low) / scale)`` in fp32, ties to even, 0 where ``scale`` is 0; it stands for ``scale * code + low``.  A
group with an infinity or a NaN in it, or with a range beyond fp32's, reads back as NaN.  At head_dim 128 a token of one KV
head takes 136 / 144 / 160 bytes (groups of 128 / 64 / 32 channels) where 16-bit K and V take 512.

====================================  ====================================================================================
``Int4KVCache``                       pages of one layer; sequences own pages through a ``block_table [batch, max_pages]``
``kv4_append``                        K / V rows of new tokens into the cache
``kv4_qkv_prep``                      the same from the QKV projection: per-head RMSNorm and rotation on the way, q out
``kv4_read``                          cached tokens as 16-bit rows, the sequences packed one behind the other
``gqa_fwd_kv4``                       attention of the last S tokens of every sequence over its cache
``flash_attn_with_kv4cache``          the same under the argument list of ``flash_attn_with_kvcache``
====================================  ====================================================================================

GPU tensors run csrc/ops/kv4.hip, kv4_attn.hip and kv4_chunk.hip, CPU tensors a PyTorch path over the same packed layout: codes and
parameters that either writes are the same bits.  Entries of a block table that are no page of the cache are tolerated
everywhere: rows that would go there are dropped, tokens there read as zeros and are not attended.  Everything launches
on the current stream of the tensors' device, allocates nothing that outlives the call but its results, and can be
captured into a graph.  None of it has a gradient: it refuses inputs that ask for one, by a backward pass or a tangent.
"""
from __future__ import annotations

import ctypes
import dataclasses
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .. import _lib

HEAD_DIMS = (64, 128, 256)
GROUPS = (32, 64, 128)
# columns (new tokens times query heads of a KV head) of a workgroup of csrc/ops/kv4_chunk.hip, and the products of columns and
# cached tokens from which a launch goes there
CHUNK_COLUMNS = {64: 256, 128: 256, 256: 128}
CHUNK_WORK = {64: 1 << 25, 128: 1 << 25, 256: 1 << 23}

# argument types of the native calls (p pointer, i int, q long long, f float), so that plain integers can be passed; the
# stream comes last everywhere
_CACHE_ARGS = "ppppiiiii"
_SIGNATURES = {
    "tdist_kv4_append": _CACHE_ARGS + "pp" + "qqqqqq" + "ppp" + "iiiii" + "p",
    "tdist_kv4_qkv_prep": _CACHE_ARGS + "pqqppffpppq" + "pppp" + "iiiii" + "p",
    "tdist_kv4_read": _CACHE_ARGS + "pii" + "pp" + "iq" + "pp" + "qqqq" + "i" + "p",
    "tdist_kv4_attn": _CACHE_ARGS + "pqqq" + "pii" + "ppp" + "iiiiii" + "ff" + "ipi" + "p",
    "tdist_kv4_chunk": _CACHE_ARGS + "pqqq" + "pii" + "ppp" + "iiiiii" + "f" + "ipi" + "p",
}
_CTYPES = {"p": ctypes.c_void_p, "i": ctypes.c_int, "q": ctypes.c_longlong, "f": ctypes.c_float}


def _launch(name: str, device: torch.device, *args) -> None:
    """One native call on the current stream of ``device``.  (A decode step makes a few of these per layer: a token's worth of
    work on the GPU is shorter than a careless call, so streams and pointers are passed as plain integers.)"""
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _launch(name, device, *args)
    fn = getattr(_lib.hip(), name)
    if fn.argtypes is None:
        fn.argtypes = [_CTYPES[c] for c in _SIGNATURES[name]]
    code = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if code:
        _lib.check(code, name)


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


@dataclasses.dataclass(frozen=True, eq=False)
class Int4KVCache:
    """One layer's pages.  The four tensors are packed as csrc/include/tdist/kv4.hpp describes; ``kv4_read`` gives the values.

    ``k_codes [pages, kv_heads, page_size, head_dim / 2]`` and ``v_codes [pages, kv_heads, page_size / 4, 2 * head_dim]`` uint8,
    ``k_params`` / ``v_params [pages, kv_heads, head_dim / group, page_size, 2]`` (scale, low) in ``dtype``.  Checked once, here:
    the tensors keep their memory as long as the cache is used (their contents may change, by whatever means); calls refuse a cache
    whose tensors have been given other memory since (``set_``, ``resize_``, ``.data``)."""

    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_params: torch.Tensor
    v_params: torch.Tensor

    def __post_init__(self):
        k, v, kp, vp = self.k_codes, self.v_codes, self.k_params, self.v_params
        _require(k.dim() == 4 and v.dim() == 4 and kp.dim() == 5, "a 4-bit cache has 4-dimensional codes and 5-dimensional parameters")
        P, H, S, D = k.shape[0], k.shape[1], k.shape[2], k.shape[3] * 2
        _require(D in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {D}")
        _require(kp.shape[2] > 0 and D % kp.shape[2] == 0, "the groups must divide the head")
        G = D // kp.shape[2]
        _require(G in GROUPS, f"groups must be of {GROUPS} channels, got {G}")
        _require(S > 0 and S % 16 == 0, f"pages must hold a multiple of 16 tokens, got {S}")
        _require(P > 0 and 0 < H <= 16384, "a cache needs pages, and 1 .. 16384 heads")
        _require(tuple(v.shape) == (P, H, S // 4, 2 * D), f"v_codes must be {(P, H, S // 4, 2 * D)}, got {tuple(v.shape)}")
        _require(kp.shape == vp.shape == (P, H, D // G, S, 2), f"parameters must be {(P, H, D // G, S, 2)}")
        _require(k.dtype == v.dtype == torch.uint8, "codes are uint8")
        if kp.dtype not in (torch.bfloat16, torch.float16) or vp.dtype != kp.dtype:
            raise TypeError(f"a 4-bit cache stands for bf16 or fp16 rows, got {kp.dtype} / {vp.dtype}")
        for t in (k, v, kp, vp):
            _require(not t.requires_grad, "a 4-bit cache has no gradient: its tensors cannot require one")
            _require(t.device == k.device, "the four tensors of a cache live on one device")
            _require(t.is_contiguous() and t.data_ptr() % 16 == 0, "cache tensors must be contiguous and 16-byte aligned")
        where = (k.data_ptr, v.data_ptr, kp.data_ptr, vp.data_ptr)
        memory = tuple(ptr() for ptr in where)
        for name, value in dict(num_pages=P, kv_heads=H, page_size=S, head_dim=D, group=G, dtype=kp.dtype, device=k.device,
                                _where=where, _memory=memory, _native=(*memory, P, H, S, D, G)).items():
            object.__setattr__(self, name, value)

    def __reduce__(self):       # (copies and pickles are caches of their own tensors)
        return Int4KVCache, (self.k_codes, self.v_codes, self.k_params, self.v_params)

    @classmethod
    def alloc(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, group: int = 64, dtype=torch.bfloat16,
              device=None) -> "Int4KVCache":
        """An empty cache.  ``group`` trades bytes for precision: 136 / 144 / 160 bytes per token and head for 128 / 64 / 32."""
        _require(page_size > 0 and page_size % 16 == 0, f"pages must hold a multiple of 16 tokens, got {page_size}")
        _require(head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        _require(group in GROUPS and group <= head_dim, f"groups must be of {GROUPS} channels (at most head_dim), got {group}")

        def params():
            return torch.zeros(num_pages, kv_heads, head_dim // group, page_size, 2, dtype=dtype, device=device)

        return cls(torch.zeros(num_pages, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, device=device),
                   torch.zeros(num_pages, kv_heads, page_size // 4, 2 * head_dim, dtype=torch.uint8, device=device),
                   params(), params())


# ---- checks --------------------------------------------------------------------------------------------------------
def _dt(dtype: torch.dtype) -> int:
    return 0 if dtype == torch.bfloat16 else 1


def _check_data(cache: Int4KVCache, **rows: torch.Tensor) -> None:
    for name, t in rows.items():
        if t.dtype is not cache.dtype:
            raise TypeError(f"{name} must be {cache.dtype} like the cache, got {t.dtype}")
        if t.device != cache.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
        if t.requires_grad or forward_ad._current_level >= 0:
            _check_no_gradient(name, t)


def _check_no_gradient(name: str, t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"a 4-bit cache has no gradient: {name} requires one (detach it, or run under torch.no_grad())")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"a 4-bit cache has no gradient: {name} carries a tangent")


def _check_table(cache: Int4KVCache, batch: int, table: torch.Tensor) -> int:
    """The pages of a row of the table.  (Every call comes here: the cache's memory is looked at too.)"""
    k, v, kp, vp = cache._where
    if (k(), v(), kp(), vp()) != cache._memory:
        raise RuntimeError("the tensors of this cache have been given other memory since it was made: make a new Int4KVCache of them")
    shape, strides = table.shape, table.stride()
    if len(shape) == 2 and table.dtype is torch.int32 and shape[0] == batch and table.device == cache.device:
        pages = shape[1]
        if (pages <= 1 or strides[1] == 1) and pages * cache.page_size <= 2 ** 30 and strides[0] < 2 ** 31:
            return pages
    raise ValueError(f"block_table must be int32 [{batch}, max_pages] with contiguous rows of at most 2^30 tokens, less than 2^31 entries "
                     f"apart, on {cache.device}")


def _check_counts(cache: Int4KVCache, n: int, name: str, t: torch.Tensor) -> None:
    if not (t.dtype is torch.int32 and t.dim() == 1 and t.numel() == n and t.is_contiguous() and t.device == cache.device):
        raise ValueError(f"{name} must be contiguous int32 [{n}] on {cache.device}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself where the kernels can take its rows 16 bytes at a time, else a contiguous copy."""
    strides, bits = x.stride(), 0
    for s in strides[:-1]:
        bits |= s
    if strides[-1] == 1 and bits % 8 == 0 and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


# ---- the packed layout in torch: CPU path and test oracle ----------------------------------------------------------
def quantise_reference(x: torch.Tensor, group: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x [..., D] 16-bit -> codes uint8 [..., D], scale and low [..., D / group] in x's type."""
    v = x.float().unflatten(-1, (-1, group))
    low, high = v.amin(-1), v.amax(-1)
    span = high - low
    scale = torch.where(span.isfinite(), span / 15, torch.nan).to(x.dtype)
    step = scale.float().unsqueeze(-1)
    code = torch.where(step > 0, torch.round((v - low.unsqueeze(-1)) / step), 0.0).clamp(0, 15)
    return code.to(torch.uint8).flatten(-2), scale, low.to(x.dtype)


def dequantise_reference(codes: torch.Tensor, scale: torch.Tensor, low: torch.Tensor) -> torch.Tensor:
    """fp32 values [..., D]."""
    v = codes.float().unflatten(-1, (scale.shape[-1], -1))
    return (v * scale.float().unsqueeze(-1) + low.float().unsqueeze(-1)).flatten(-2)


def _pack_k(codes: torch.Tensor) -> torch.Tensor:
    """[T, H, D] codes -> [T, H, D / 2] bytes: channel (s, lg, n, odd) is nibble n + 4 odd of dword (lg, s)."""
    c = codes.unflatten(-1, (-1, 4, 4, 2))                                   # s, lg, n, odd
    c = c.movedim(-4, -3).transpose(-1, -2).flatten(-4)                      # lg, s, odd, n
    return c[..., 0::2] | c[..., 1::2] << 4


def _unpack_k(b: torch.Tensor) -> torch.Tensor:
    c = torch.stack([b & 15, b >> 4], -1).flatten(-2).unflatten(-1, (4, -1, 2, 4))
    return c.transpose(-1, -2).movedim(-4, -3).flatten(-4)


def _pack_v(codes: torch.Tensor) -> torch.Tensor:
    """[T, H, D] codes -> [T, H, 16, D / 64, 2] bytes: channel 16 (4 h + n) + c is nibble n of unit (c, h)."""
    c = codes.unflatten(-1, (-1, 4, 16)).movedim(-1, -3)                     # c, h, n
    return c[..., 0::2] | c[..., 1::2] << 4


def _unpack_v(b: torch.Tensor) -> torch.Tensor:
    return torch.stack([b & 15, b >> 4], -1).flatten(-2).movedim(-3, -1).flatten(-3)


def _places(cache: Int4KVCache, block_table, of, pos):
    """(ok, page, place in the page) of token ``pos`` of sequence ``of``."""
    ok = (pos >= 0) & (pos < block_table.shape[1] * cache.page_size)
    if block_table.shape[1] == 0:
        return ok, torch.zeros_like(pos), torch.zeros_like(pos)
    safe = torch.where(ok, pos, 0)
    page = block_table.long()[of, safe // cache.page_size]
    ok = ok & (page >= 0) & (page < cache.num_pages)
    return ok, torch.where(ok, page, 0), safe % cache.page_size


def _v_units(cache: Int4KVCache) -> torch.Tensor:
    """v_codes as [pages, heads, page / 4, 16, D / 64, token of four, 2 bytes]."""
    return cache.v_codes.view(*cache.v_codes.shape[:3], 16, cache.head_dim // 64, 4, 2)


def _store_reference(cache: Int4KVCache, k, v, of, pos, block_table) -> None:
    ok, page, off = _places(cache, block_table, of, pos)
    k, v, page, off = k[ok], v[ok], page[ok], off[ok]
    for x, params, is_v in ((k, cache.k_params, False), (v, cache.v_params, True)):
        code, scale, low = quantise_reference(x, cache.group)
        if is_v:
            _v_units(cache)[page, :, off // 4, :, :, off % 4] = _pack_v(code)
        else:
            cache.k_codes[page, :, off] = _pack_k(code)
        params[page, :, :, off] = torch.stack([scale, low], -1)


def _load_reference(cache: Int4KVCache, of, pos, block_table) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(there, k, v): fp32 values [T, H, D], zero where there is no page."""
    ok, page, off = _places(cache, block_table, of, pos)
    out = []
    for code, params in ((_unpack_k(cache.k_codes[page, :, off]), cache.k_params),
                         (_unpack_v(_v_units(cache)[page, :, off // 4, :, :, off % 4]), cache.v_params)):
        p = params[page, :, :, off]
        out.append(torch.where(ok[:, None, None], dequantise_reference(code, p[..., 0], p[..., 1]), 0.0))
    return ok, out[0], out[1]


# ---- writing -------------------------------------------------------------------------------------------------------
def kv4_append(k: torch.Tensor, v: torch.Tensor, cache: Int4KVCache, kv_offset: torch.Tensor, block_table: torch.Tensor,
               new_lens: Optional[torch.Tensor] = None) -> None:
    """Token s of ``k`` / ``v [batch, S, kv_heads, head_dim]`` becomes token ``kv_offset[b] + s`` of sequence b.

    ``kv_offset`` int32 [batch]; ``new_lens`` (int32 [batch], optional): only the first ``new_lens[b]`` rows are tokens, the
    rest padding.  Tokens without a page are dropped.  Pages that are written must belong to one sequence: two sequences
    that write the same token of a page leave a mixture."""
    if not (k.dim() == 4 and k.shape == v.shape and k.shape[2] == cache.kv_heads and k.shape[3] == cache.head_dim):
        raise ValueError(f"k and v must be [batch, S, {cache.kv_heads}, {cache.head_dim}], got {tuple(k.shape)} and {tuple(v.shape)}")
    batch, S = k.shape[:2]
    _check_data(cache, k=k, v=v)
    pages = _check_table(cache, batch, block_table)
    _check_counts(cache, batch, "kv_offset", kv_offset)
    if new_lens is not None:
        _check_counts(cache, batch, "new_lens", new_lens)
    if batch == 0 or S == 0:
        return
    if not k.is_cuda:
        step = torch.arange(S)
        live = step < (new_lens[:, None] if new_lens is not None else S)
        pos = torch.where(live, kv_offset[:, None].long() + step, -1)
        of = torch.arange(batch)[:, None].expand(batch, S)
        _store_reference(cache, k.flatten(0, 1), v.flatten(0, 1), of.flatten(), pos.flatten(), block_table)
        return
    k, v = _rows(k), _rows(v)
    _launch("tdist_kv4_append", cache.device, *cache._native, k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3],
            kv_offset.data_ptr(), _ptr(new_lens), block_table.data_ptr(), block_table.stride(0), pages, batch, S,
            _dt(cache.dtype))


def kv4_qkv_prep(qkv: torch.Tensor, q_w: Optional[torch.Tensor], k_w: Optional[torch.Tensor], q_eps: float, k_eps: float,
                 position_ids: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, cache: Int4KVCache,
                 kv_offset: torch.Tensor, total_out: torch.Tensor, block_table: torch.Tensor, num_q_heads: int) -> torch.Tensor:
    """One launch for everything between the QKV projection and attention (``elementwise.qkv_prep`` for a 4-bit cache).

    ``qkv [batch, S, (Hq + 2 Hkv) * D]`` bf16: q / k heads get their optional per-head RMSNorm (``q_w`` / ``k_w`` [D]) and the
    neox rotation at ``position_ids [batch, S]`` (``cos`` / ``sin`` fp32 [positions, D / 2]; ids outside the tables take their
    first or last row), K and V become tokens ``kv_offset[b] + s`` of the cache and ``total_out[b]`` (int32) receives
    ``kv_offset[b] + S``.  K's mean square and rotation are taken in fp64, so that a code does not depend on the order of a sum;
    Q's in fp32 on the GPU and in fp64 on the CPU, where a rounding to bf16 may fall the other way (a few in 10^5).  Returns q
    [batch, S, Hq, D]."""
    D, Hkv = cache.head_dim, cache.kv_heads
    if cache.dtype != torch.bfloat16:
        raise TypeError(f"kv4_qkv_prep writes bf16 caches, got {cache.dtype}")
    if not (qkv.dim() == 3 and num_q_heads > 0 and qkv.shape[2] == (num_q_heads + 2 * Hkv) * D):
        raise ValueError(f"qkv must be [batch, S, {(num_q_heads + 2 * Hkv) * D}], got {tuple(qkv.shape)}")
    batch, S = qkv.shape[:2]
    _check_data(cache, qkv=qkv)
    for w in (q_w, k_w):
        if w is not None:
            _check_data(cache, norm_weight=w)
            if not (w.dim() == 1 and w.shape[0] == D and w.is_contiguous()):
                raise ValueError(f"norm weights are contiguous [{D}]")
    if not (position_ids.shape == (batch, S) and position_ids.device == cache.device):
        raise ValueError(f"position_ids must be [{batch}, {S}] on {cache.device}")
    if not (cos.dtype is torch.float32 and sin.dtype is torch.float32 and cos.dim() == 2 and cos.size(1) == D // 2 and cos.size(0) > 0
            and cos.shape == sin.shape and cos.is_contiguous() and sin.is_contiguous() and cos.device == cache.device
            and sin.device == cache.device):
        raise ValueError(f"cos / sin must be contiguous fp32 [positions, {D // 2}] on {cache.device}")
    if cos.requires_grad or sin.requires_grad or forward_ad._current_level >= 0:
        _check_no_gradient("cos", cos)
        _check_no_gradient("sin", sin)
    pages = _check_table(cache, batch, block_table)
    _check_counts(cache, batch, "kv_offset", kv_offset)
    _check_counts(cache, batch, "total_out", total_out)
    if abs(total_out.data_ptr() - kv_offset.data_ptr()) < 4 * batch:
        raise ValueError("total_out is written while kv_offset is read: they must not share memory")
    if batch == 0 or S == 0:
        total_out.copy_(kv_offset)
        return qkv.new_empty(batch, S, num_q_heads, D)
    pos = position_ids
    if pos.dtype is not torch.int64 or not pos.is_contiguous():
        pos = pos.to(torch.int64).contiguous()
    if not qkv.is_cuda:
        q, k, v = qkv.unflatten(-1, (-1, D)).split([num_q_heads, Hkv, Hkv], 2)
        at = pos.clamp(0, cos.shape[0] - 1)
        c, s = cos[at].unsqueeze(2).double(), sin[at].unsqueeze(2).double()

        def prep(x, w, eps):
            if w is not None:
                inv = (1 / (x.double().square().mean(-1, keepdim=True) + torch.tensor(eps, dtype=torch.float32)).sqrt()).float()
                x = (x.float() * inv * w.float()).to(x.dtype)
            a, b = x.double().chunk(2, -1)
            return torch.cat([a * c - b * s, b * c + a * s], -1).float().to(x.dtype)

        q, k = prep(q, q_w, q_eps), prep(k, k_w, k_eps)
        kv4_append(k, v, cache, kv_offset, block_table)
        total_out.copy_(kv_offset + S)
        return q
    qkv = _rows(qkv)
    q_w, k_w = (w if w is None or w.data_ptr() % 16 == 0 else w.clone() for w in (q_w, k_w))
    q = qkv.new_empty((batch, S, num_q_heads, D))
    _launch("tdist_kv4_qkv_prep", cache.device, *cache._native, qkv.data_ptr(), *qkv.stride()[:2], _ptr(q_w), _ptr(k_w), q_eps,
            k_eps, pos.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0], q.data_ptr(), kv_offset.data_ptr(),
            total_out.data_ptr(), block_table.data_ptr(), block_table.stride(0), pages, batch, S, num_q_heads)
    return q


# ---- reading -------------------------------------------------------------------------------------------------------
def kv4_read(cache: Int4KVCache, block_table: torch.Tensor, cu_seqlens: torch.Tensor, total: int,
             starts: Optional[torch.Tensor] = None, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cached tokens as 16-bit rows: row ``cu_seqlens[b] + i`` of both results is token ``starts[b] + i`` (``i`` without
    ``starts``) of sequence b.  ``cu_seqlens`` int32 [batch + 1] ascending, ``total`` the results' rows.

    Returns (k, v) ``[total, kv_heads, head_dim]`` - what ``flash_attn_varlen_fwd`` takes.  Rows that no sequence covers are
    left as they were (``out``) or unset; tokens without a page come out as zeros.  A finite value that its group's rounded
    scale carries beyond the type's largest number comes out as that number."""
    batch = block_table.size(0) if block_table.dim() == 2 else -1
    pages = _check_table(cache, batch, block_table)
    _check_counts(cache, batch + 1, "cu_seqlens", cu_seqlens)
    if starts is not None:
        _check_counts(cache, batch, "starts", starts)
    if not 0 <= total < 2 ** 31:
        raise ValueError(f"total must be a row count, got {total}")
    shape = (int(total), cache.kv_heads, cache.head_dim)
    if out is None:
        k, v = cache.k_params.new_empty(shape), cache.k_params.new_empty(shape)
    else:
        k, v = out
        _check_data(cache, k_out=k, v_out=v)
        for t in (k, v):
            _require(tuple(t.shape) == shape, f"out must be two tensors {shape}, got {tuple(t.shape)}")
            _require(t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0,
                     "rows of out must be contiguous and 16-byte aligned")
            _require(all(n < 2 or s > 0 for n, s in zip(shape, t.stride())), "every row of out needs memory of its own")
        _require(total == 0 or k.data_ptr() != v.data_ptr(), "K and V of out must not share memory")
    if batch == 0 or total == 0:
        return k, v
    if not cache.k_codes.is_cuda:
        cu = cu_seqlens.long()
        r = torch.arange(int(total))
        r = r[(r >= cu[0]) & (r < cu[-1])]
        of = torch.searchsorted(cu, r, right=True) - 1
        pos = r - cu[of] + (starts.long()[of] if starts is not None else 0)
        _, kk, vv = _load_reference(cache, of, pos, block_table)
        most = torch.finfo(cache.dtype).max
        k[r], v[r] = kk.clamp(max=most).to(cache.dtype), vv.clamp(max=most).to(cache.dtype)
        return k, v
    _launch("tdist_kv4_read", cache.device, *cache._native, block_table.data_ptr(), block_table.stride(0), pages,
            cu_seqlens.data_ptr(), _ptr(starts), batch, int(total), k.data_ptr(), v.data_ptr(), *k.stride()[:2], *v.stride()[:2],
            _dt(cache.dtype))
    return k, v


# ---- attention -----------------------------------------------------------------------------------------------------
def attend_reference(q, cache: Int4KVCache, kv_lens, block_table, scale, soft_cap=0.0, causal=True):
    """fp32 (out [batch, S, Hq, D], natural-log LSE [batch, S, Hq]) in plain PyTorch: CPU path and test oracle."""
    batch, S, Hq, D = q.shape
    Hkv = cache.kv_heads
    room = block_table.shape[1] * cache.page_size
    out = torch.zeros(batch, S, Hq, D, dtype=torch.float32, device=q.device)
    lse = torch.full((batch, S, Hq), -math.inf, dtype=torch.float32, device=q.device)
    for b in range(batch):
        L = min(max(int(kv_lens[b]), 0), room)
        if L == 0:
            continue
        pos = torch.arange(L, device=q.device)
        there, k, v = _load_reference(cache, torch.full_like(pos, b), pos, block_table)
        seen = there.expand(S, L)
        if causal:
            seen = seen & (pos <= (L - S + torch.arange(S, device=q.device))[:, None])
        qh = q[b].float().view(S, Hkv, -1, D).permute(1, 2, 0, 3)                       # [Hkv, g, S, D]
        s = torch.matmul(qh, k.permute(1, 2, 0).unsqueeze(1).contiguous()) * scale      # [Hkv, g, S, L]
        if soft_cap > 0:
            s = soft_cap * torch.tanh(s / soft_cap)
        s = s.masked_fill(~seen, -math.inf)
        any_seen = seen.any(-1)
        p = torch.where(any_seen[:, None], torch.softmax(s, -1), 0.0)
        # a NaN reaches the queries that see its token and, through 0 * NaN, no other
        v = v.transpose(0, 1).contiguous()                                              # [Hkv, L, D]
        got = torch.matmul(p, v.nan_to_num(0.0).unsqueeze(1))
        spoilt = torch.matmul(seen.float(), v.isnan().float()) > 0                      # [Hkv, S, D]
        out[b] = got.masked_fill(spoilt.unsqueeze(1), math.nan).permute(2, 0, 1, 3).reshape(S, Hq, D)
        lse[b] = torch.logsumexp(s, -1).permute(2, 0, 1).reshape(S, Hq)
    return out, lse


def takes_chunks(batch: int, kv_heads: int, columns: int, head_dim: int, capacity: int, soft_cap: float = 0.0) -> bool:
    """Whether a launch over a bf16 cache goes to csrc/ops/kv4_chunk.hip, which unpacks for many columns at once, and only what that
    leaves to csrc/ops/kv4_attn.hip.  (fp16 caches stay with the latter: their results show the former's roundings.)

    Measured (four query heads to a KV head, microseconds there / here): one sequence of 16384, 8 heads of 128: 128 columns 40 / 34,
    256 46 / 50, 1024 98 / 147; of 4096: 512 columns 43 / 35, 1024 49 / 51, 2048 66 / 78; of 1024: 2048 columns 39 / 27; 4 x 2048:
    256 columns 38 / 36, 1024 65 / 84; 4 heads of 256: 2048: 512 columns 30 / 29, 1024 36 / 40."""
    work = batch * kv_heads * columns * capacity
    return soft_cap == 0 and 2 * columns > CHUNK_COLUMNS[head_dim] and work >= CHUNK_WORK[head_dim]


def auto_kv_splits(batch: int, kv_heads: int, columns: int, head_dim: int, capacity: int, num_cus: int = 256,
                   chunk: bool = False) -> int:
    """KV splits of a launch: ``columns`` = new tokens times query heads of a KV head, ``capacity`` = tokens of a sequence's pages.

    One round of the chip: a CU holds two workgroups, and a third round of nothing but start-up costs more than it gives.
    Measured (32 / 8 heads of 128, groups of 64, microseconds): 131072 tokens of one sequence 38.2 / 35.6 / 42.2 with 32 / 64 / 96
    splits; 16 x 4096 23.1 / 20.3 / 24.7 with 2 / 4 / 8; 64 x 4096 55.9 / 61.9 with 1 / 2.  At least 128 tokens each: 2048 tokens 9.5 /
    8.9 with 8 / 16; beyond sixteen splits 256: 8192 tokens 10.3 / 11.0 with 32 / 64.  Up to 512 tokens in one piece: 256 tokens
    6.8 / 8.3 with 1 / 2, 512 8.5 / 8.6 with 1 / 4 (640: 9.3 / 8.6 with 1 / 6), and one launch instead of two on the host, 11 / 15.
    (Measured for a decode step; not for more columns or other heads.)  The room decides and not the lengths, which the host does
    not know: 37 tokens take 6.6 us in a table of 37 and 9.3 in one of 32768, 512 8.7 and 9.0, 16 x 512 9.1 and 10.9.

    ``chunk``: of a launch that `takes_chunks`; one workgroup fills a CU there (1024 new tokens over 16384: 613 / 356 / 443 with 1 /
    2 / 3; 256 over 16384 126 / 106 / 128 with 6 / 8 / 16)."""
    if chunk:
        groups = batch * kv_heads * (-(-columns // CHUNK_COLUMNS[head_dim]))
        return max(1, min(num_cus // max(1, groups), capacity // 256, 64))
    per_group = 32 if columns > 16 and head_dim <= 128 else 16          # columns of a workgroup
    groups = batch * kv_heads * (-(-columns // per_group))
    most = 1 if capacity <= 512 else min(capacity // 128, max(16, capacity // 256), 64)
    return max(1, min(2 * num_cus // max(1, groups), most))


def gqa_fwd_kv4(q: torch.Tensor, cache: Int4KVCache, kv_lens: torch.Tensor, block_table: torch.Tensor,
                scale: Optional[float] = None, soft_cap: float = 0.0, kv_split: int = -1, causal: bool = True,
                return_lse: bool = False) -> torch.Tensor:
    """Attention of ``q [batch, S, Hq, D]`` (or ``[batch, Hq, D]`` for S = 1), the last S tokens of each sequence.

    ``kv_lens`` int32 [batch]: cached tokens, the S new ones included (more than the table has room for count as that room); with
    ``causal`` query s sees the first ``kv_lens[b] - S + s + 1`` of them.  Rows that see nothing are zero.  Scores (``scale`` times q . k) may be up to 2^27 in size: in
    fp32 they are 8 apart from there on, and a row's weights mean nothing.  Returns q's shape in q's type, or with ``return_lse``
    fp32 ``[.., D + 1]`` with the natural-log LSE last (-inf for an empty row), the form
    ``flash_decode.gqa_fwd_batch_decode_inter_rank_combine`` merges over ranks that hold parts of the sequences."""
    flat = q.dim() == 3
    q4 = q.unsqueeze(1) if flat else q
    if q4.dim() != 4 or q4.shape[3] != cache.head_dim or q4.shape[2] == 0 or q4.shape[2] % cache.kv_heads:
        raise ValueError(f"q must be [batch, S, heads, {cache.head_dim}] with a multiple of {cache.kv_heads} heads, got {tuple(q.shape)}")
    batch, S, Hq, D = q4.shape
    _check_data(cache, q=q)
    pages = _check_table(cache, batch, block_table)
    _check_counts(cache, batch, "kv_lens", kv_lens)
    scale = D ** -0.5 if scale is None else float(scale)
    if not (math.isfinite(scale) and math.isfinite(soft_cap) and soft_cap >= 0):
        raise ValueError(f"scale must be finite, soft_cap 0 (off) or positive, got {scale} and {soft_cap}")
    if soft_cap:
        soft_cap = min(max(soft_cap, 2.0 ** -126), 2.0 ** 127)       # (ordinary fp32 numbers: 0 would be off)
    if not (kv_split == -1 or 1 <= kv_split <= 65535):
        raise ValueError(f"kv_split must be -1 (automatic) or 1 .. 65535, got {kv_split}")
    if not q.is_cuda:
        out, lse = attend_reference(q4, cache, kv_lens, block_table, scale, soft_cap, causal)
        out = torch.cat([out, lse.unsqueeze(-1)], -1) if return_lse else out.to(q.dtype)
        return out.squeeze(1) if flat else out
    q4 = _rows(q4)
    columns = Hq // cache.kv_heads * S
    room = pages * cache.page_size
    chunk = cache.dtype is torch.bfloat16 and takes_chunks(batch, cache.kv_heads, columns, D, room, soft_cap)
    splits = int(kv_split) if kv_split > 0 else auto_kv_splits(batch, cache.kv_heads, columns, D, room, chunk=chunk)
    out = torch.empty((batch, S, Hq, D + 1), dtype=torch.float32, device=q.device) if return_lse else \
        torch.empty_like(q4, memory_format=torch.contiguous_format)
    part = torch.empty(batch * S * Hq * splits * (D + 1), dtype=torch.float32, device=q.device) if splits > 1 else None
    call = (*cache._native, q4.data_ptr(), *q4.stride()[:3], block_table.data_ptr(), block_table.stride(0), pages,
            kv_lens.data_ptr(), _ptr(part), out.data_ptr(), batch, S, Hq, splits, 1 if causal else 0, 2 if return_lse else 1, scale)
    flags, at_once = None, 0
    if chunk:
        at_once = CHUNK_COLUMNS[D]
        flags = torch.empty(-(-columns // at_once) * batch * splits * cache.kv_heads, dtype=torch.int32, device=q.device)
        _launch("tdist_kv4_chunk", cache.device, *call, _dt(cache.dtype), flags.data_ptr(), at_once)
    _launch("tdist_kv4_attn", cache.device, *call, soft_cap, _dt(cache.dtype), _ptr(flags), at_once)
    return out.squeeze(1) if flat else out


def flash_attn_with_kv4cache(q: torch.Tensor, cache: Int4KVCache, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                             softmax_scale: Optional[float] = None, causal: bool = True) -> torch.Tensor:
    """``flash_attn_with_kvcache`` over a 4-bit cache that already holds the new tokens: ``q [batch, S, Hq, D]`` are the last S of
    the ``cache_seqlens`` (int32 [batch]) tokens of each sequence."""
    return gqa_fwd_kv4(q, cache, cache_seqlens, block_table, scale=softmax_scale, causal=causal)

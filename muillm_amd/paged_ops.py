"""Operators over a paged 8-bit key/value cache (include/muillm_amd.h, the section of that name), in the manner of muillm_ext.py: validate,
allocate outputs with torch, hand raw pointers and the current stream to the library. Queries, keys and values are fp16 or bf16; the cache is e4m3
with one power-of-two scale per page and KV head.

A call's tokens stand one after another, those of request b in the rows offsets[b] .. offsets[b + 1] - 1 (no offsets: row b is request b's only
one). lengths[b] counts the request's tokens with the call's among them, so paged_append and paged_attention of one step take the same table,
lengths and offsets. All three live on the device: a captured step goes on as they change. Rows behind the last request are left as they were."""

from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib
from ._lib import MUI_DTYPE_BF16, MUI_DTYPE_F16, PAGED_APPEND_ARGS, PAGED_ATTENTION_ARGS, check

PAGE_TOKENS = (64, 128, 256)
HEAD_DIMS = (64, 128, 256)

_CODES = {torch.float16: MUI_DTYPE_F16, torch.bfloat16: MUI_DTYPE_BF16}
_E4M3, _F32, _F64, _I32, _I64 = torch.float8_e4m3fn, torch.float32, torch.float64, torch.int32, torch.int64


class PagedKV:
    """One layer's pages. k: e4m3 [pages, kv_heads, page / 64, dim / 64, 64, 64], the last two token and dimension; v: e4m3 [pages, kv_heads,
    page / 64, dim, 4, 4, 4], the last three g, t, i of token 16 t + 4 g + i; k_scale, v_scale: fp32 [pages, kv_heads], powers of two."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "n_pages", "kv_heads", "page", "dim", "index")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        ks, vs = k.shape, v.shape
        if len(ks) != 6 or ks[4] != 64 or ks[5] != 64 or len(vs) != 7 or vs[4] != 4 or vs[5] != 4 or vs[6] != 4:
            raise RuntimeError("k must be [pages, kv_heads, page / 64, dim / 64, 64, 64] and v [pages, kv_heads, page / 64, dim, 4, 4, 4]")
        self.n_pages, self.kv_heads, self.page, self.dim = n, h, page, dim = ks[0], ks[1], ks[2] * 64, ks[3] * 64
        if vs[0] != n or vs[1] != h or vs[2] != ks[2] or vs[3] != dim:
            raise RuntimeError(f"v has shape {tuple(vs)}, which does not go with k's {tuple(ks)}")
        if page not in PAGE_TOKENS or dim not in HEAD_DIMS:
            raise RuntimeError(f"pages hold {PAGE_TOKENS} tokens and heads {HEAD_DIMS} dimensions, not {page} and {dim}")
        self.index = at = k.get_device()
        if not (k.dtype is _E4M3 and v.dtype is _E4M3 and k_scale.dtype is _F32 and v_scale.dtype is _F32):
            raise RuntimeError("k and v must be float8_e4m3fn tensors, k_scale and v_scale float32 ones")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise RuntimeError("k, v and their scales must be contiguous")
        if v.get_device() != at or k_scale.get_device() != at or v_scale.get_device() != at:
            raise RuntimeError(f"v and the scales must be on {k.device}, as k is")
        if k_scale.shape != (n, h) or v_scale.shape != (n, h):
            raise RuntimeError("k_scale and v_scale must be [pages, kv_heads]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @property
    def device(self) -> torch.device:
        return self.k.device

    @classmethod
    def empty(cls, n_pages: int, kv_heads: int, page: int, dim: int, device) -> "PagedKV":
        """Pages of zeros."""
        if page not in PAGE_TOKENS or dim not in HEAD_DIMS:
            raise RuntimeError(f"pages hold {PAGE_TOKENS} tokens and heads {HEAD_DIMS} dimensions, not {page} and {dim}")
        k, v = (torch.zeros(n_pages * kv_heads * page * dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
        ks, vs = (torch.ones((n_pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2))
        return cls(k.view(n_pages, kv_heads, page // 64, dim // 64, 64, 64), v.view(n_pages, kv_heads, page // 64, dim, 4, 4, 4), ks, vs)

    def dense(self, pages: torch.Tensor, tokens: int):
        """(keys, values) fp32 [kv_heads, tokens, dim] of a request whose pages these are (torch operations, for a look at the cache)."""
        need = -(-tokens // self.page)
        pages = pages[:need].long()
        k = self.k.view(torch.uint8)[pages].permute(0, 1, 2, 4, 3, 5).reshape(need, self.kv_heads, self.page, self.dim)
        v = self.v.view(torch.uint8)[pages].permute(0, 1, 2, 5, 4, 6, 3).reshape(need, self.kv_heads, self.page, self.dim)
        return tuple((x.view(torch.float8_e4m3fn).float() * s[pages][..., None, None]).transpose(0, 1).reshape(self.kv_heads, -1, self.dim)[:, :tokens]
                     for x, s in ((k, self.k_scale), (v, self.v_scale)))


# (A step of small requests takes the GPU a few microseconds, so what the host does in front of it counts: the checks ask a tensor for its device's number, its
# shape and its strides once, arguments go to the library in one piece, and the stream comes as the number that it is, not as an object.)
def _call(index: int, fn, args: bytes) -> int:
    if index == torch._C._cuda_getDevice():
        return fn(torch._C._cuda_getCurrentRawStream(index), args)
    with torch.cuda.device(index):
        return fn(torch._C._cuda_getCurrentRawStream(index), args)


def _rows(x: torch.Tensor, name: str, kv: PagedKV, heads: Optional[int], dtype: torch.dtype, n_rows: int):
    """[rows, heads, dim] with whole heads: its heads and its strides between tokens and heads."""
    s = x.shape
    if x.get_device() != kv.index:
        raise RuntimeError(f"{name} must be a CUDA tensor on the cache's device")
    if x.dtype is not dtype or len(s) != 3 or s[0] != n_rows or s[2] != kv.dim or (heads is not None and s[1] != heads):
        raise RuntimeError(f"{name} has shape {tuple(s)} and type {x.dtype}, expected {dtype} [{n_rows}, {heads or 'heads'}, {kv.dim}]")
    a, b, c = x.stride()
    if c != 1:
        raise RuntimeError(f"{name}'s heads must be contiguous")
    return s[1], a, b


def _places(kv: PagedKV, table: torch.Tensor, lengths: torch.Tensor, offsets: Optional[torch.Tensor], n_rows: int):
    """(requests, pages of a row of the table, from row to row)"""
    if kv.index < 0 or table.get_device() != kv.index or lengths.get_device() != kv.index:
        raise RuntimeError("table and lengths must be CUDA tensors on the cache's device, which is one")
    s = table.shape
    if table.dtype is not _I32 or len(s) != 2 or s[1] < 1:
        raise RuntimeError("table must be int32 [requests, pages]")
    n, width = s
    step, one = table.stride()
    if one != 1 or (step < width and n > 1):
        raise RuntimeError("table's rows must be contiguous")
    if lengths.dtype is not _I64 or lengths.shape != (n,) or not lengths.is_contiguous():
        raise RuntimeError(f"lengths must be a contiguous int64 tensor [{n}]")
    if offsets is None:
        if n_rows != n:
            raise RuntimeError(f"{n_rows} rows of {n} requests need offsets")
    elif offsets.dtype is not _I64 or offsets.shape != (n + 1,) or not offsets.is_contiguous() or offsets.get_device() != kv.index:
        raise RuntimeError(f"offsets must be a contiguous int64 tensor [{n + 1}] on the cache's device")
    return n, width, step if n > 1 else width


def _dtype(x: torch.Tensor) -> int:
    code = _CODES.get(x.dtype)
    if code is None:
        raise RuntimeError(f"unsupported dtype {x.dtype}: fp16 or bf16")
    return code


def _most_tokens(max_tokens: Optional[int], offsets: Optional[torch.Tensor], n_rows: int) -> int:
    if max_tokens is None:
        return 1 if offsets is None else n_rows
    if max_tokens < 1:
        raise RuntimeError("max_tokens must be positive")
    return min(max_tokens, n_rows)


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(*sizes: int) -> int:
    return _lib.load().mui_paged_attention_scratch_bytes(*sizes)


def _over(out: torch.Tensor, x: torch.Tensor) -> bool:
    """Whether the dense `out` has bytes between the first and the last of x [rows, heads, dim]."""
    rows, heads, dim = x.shape
    if not (rows and heads and out.numel()):
        return False
    begin, size = x.data_ptr(), x.element_size()
    end = begin + size * ((rows - 1) * x.stride(0) + (heads - 1) * x.stride(1) + dim)
    return begin < out.data_ptr() + size * out.numel() and out.data_ptr() < end


def _output(out: Optional[torch.Tensor], q: torch.Tensor, in_place: bool) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.dtype is not q.dtype or out.shape != q.shape or not out.is_contiguous() or out.get_device() != q.get_device():
        raise RuntimeError("out must be a contiguous tensor of q's shape and type")
    if in_place and out.data_ptr() == q.data_ptr() and q.is_contiguous():
        return out
    if _over(out, q):
        raise RuntimeError("out must not lie over q" + (", unless it is q" if in_place else ""))
    return out


def paged_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, kv: PagedKV, table: torch.Tensor, lengths: torch.Tensor,
                 offsets: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                 interleaved: bool = False, rope_scale: float = 1.0, max_tokens: Optional[int] = None, out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotated queries [rows, heads, dim]; keys, rotated, and values go to their places in the cache. q [rows, heads, dim] (or None), k, v [rows, kv_heads,
    dim] may be slices of one projection's output (whole heads, strides of multiples of 8, 16-byte aligned).

    The first 2 * len(inv_freq) dimensions (a multiple of 16; none without inv_freq) turn by the angles position * inv_freq, fp64: as halves (i, i + n) or,
    interleaved, as pairs (2 i, 2 i + 1); rope_scale multiplies cosine and sine (frequencies of a scaled context and their factor are the caller's). Positions
    are the tokens' own unless positions (int64 [rows]) says otherwise.

    A page's scale is the smallest power of two with which its largest value fits 448, and does not fall while earlier tokens stand there; where it
    rises their codes follow. Infinities and NaN become NaN. A page that is appended to belongs to one request and stands in its row once. Tokens without a place (a table entry that is no
    page, a length beyond the table) are not written. max_tokens: at least the most new tokens of a request (default: 1 without offsets, else all rows): 1 takes
    the kernel for single tokens, others' tokens behind the first are then not appended. out may be q itself; it must not
    lie over k or v."""
    n_rows = k.shape[0]
    n, width, step = _places(kv, table, lengths, offsets, n_rows)
    code, dtype = _dtype(k), k.dtype
    _, kt, kh = _rows(k, "k", kv, kv.kv_heads, dtype, n_rows)
    _, vt, vh = _rows(v, "v", kv, kv.kv_heads, dtype, n_rows)
    heads = qt = qh = 0
    qp = op = fp = 0
    if q is not None:
        heads, qt, qh = _rows(q, "q", kv, None, dtype, n_rows)
        given, out = out, _output(out, q, True)
        if given is not None and (_over(out, k) or _over(out, v)):
            raise RuntimeError("out must not lie over k or v, which the same launch reads")
        qp, op = q.data_ptr(), out.data_ptr()
    rot = 0
    if inv_freq is not None:
        rot, fp = 2 * inv_freq.numel(), inv_freq.data_ptr()
        if inv_freq.dtype is not _F64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or inv_freq.get_device() != kv.index:
            raise RuntimeError("inv_freq must be a contiguous float64 tensor [rotated dimensions / 2] on the cache's device")
        if rot > kv.dim or rot % 16:
            raise RuntimeError(f"{rot} rotated dimensions: a multiple of 16, at most {kv.dim}")
    if positions is not None and (positions.dtype is not _I64 or positions.shape != (n_rows,) or not positions.is_contiguous() or positions.get_device() != kv.index):
        raise RuntimeError(f"positions must be a contiguous int64 tensor [{n_rows}] on the cache's device")
    if n_rows == 0:
        return out if q is not None else None
    max_tokens = _most_tokens(max_tokens, offsets, n_rows)
    args = PAGED_APPEND_ARGS.pack(qp, k.data_ptr(), v.data_ptr(), kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(), kv.v_scale.data_ptr(), table.data_ptr(),
                                  lengths.data_ptr(), 0 if offsets is None else offsets.data_ptr(), 0 if positions is None else positions.data_ptr(), fp, op,
                                  qt, qh, kt, kh, vt, vh, step,
                                  code, kv.n_pages, kv.page, width, n_rows, n, max_tokens, heads, kv.kv_heads, kv.dim, rot, 1 if interleaved else 0, rope_scale)
    check(_call(kv.index, _lib.load().mui_paged_append, args), "mui_paged_append")
    return out if q is not None else None


def paged_attention(q: torch.Tensor, kv: PagedKV, table: torch.Tensor, lengths: torch.Tensor, offsets: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    window: int = 0, keep_first: int = 0, max_tokens: Optional[int] = None, max_length: Optional[int] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[rows, heads, dim]: causal attention of q [rows, heads, dim] (rotated; whole heads, strides of multiples of 8) over the cache, which holds the
    new tokens already. scale > 0: of the scores (default dim ** -0.5). window > 0: a token sees the last `window` ones, itself among them, and the first
    keep_first of its request. A token that sees nothing gives zeros; keys on a table entry that is no page do not count.

    max_tokens: as in paged_append; max_length: at least the largest of lengths (default: what a row of the table can hold). Both size the launch: tokens and keys
    beyond what they say may be left out."""
    n_rows = q.shape[0]
    n, width, step = _places(kv, table, lengths, offsets, n_rows)
    code = _dtype(q)
    heads, qt, qh = _rows(q, "q", kv, None, q.dtype, n_rows)
    if heads == 0 or heads % kv.kv_heads:
        raise RuntimeError(f"{heads} query heads do not go with {kv.kv_heads} key heads")
    if window < 0 or keep_first < 0:
        raise RuntimeError("window and keep_first must not be negative")
    if scale is None:
        scale = kv.dim ** -0.5
    elif not scale > 0:
        raise RuntimeError("scale must be positive")
    out = _output(out, q, False)
    if n_rows == 0:
        return out
    max_tokens, window, keep_first = _most_tokens(max_tokens, offsets, n_rows), min(window, 0x7fffffff), min(keep_first, 0x7fffffff)
    most = min(width * kv.page, 0x7fffffff)
    max_length = most if max_length is None else max(1, min(max_length, most))
    nbytes = _scratch_bytes(n_rows, n, max_tokens, max_length, window, keep_first, heads, kv.kv_heads, kv.dim)
    scratch = q.new_empty(nbytes // 2) if nbytes else None
    args = PAGED_ATTENTION_ARGS.pack(q.data_ptr(), kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(), kv.v_scale.data_ptr(), table.data_ptr(), lengths.data_ptr(),
                                     0 if offsets is None else offsets.data_ptr(), 0 if scratch is None else scratch.data_ptr(), out.data_ptr(), nbytes, qt, qh, step,
                                     code, kv.n_pages, kv.page, width, n_rows, n, max_tokens, max_length, window, keep_first, heads, kv.kv_heads, kv.dim, scale)
    check(_call(kv.index, _lib.load().mui_paged_attention, args), "mui_paged_attention")
    return out

"""Trie-verification attention with a slot-order-independent node sum, and the attention of
whole prompts and of single new tokens beside it.

`fused_attn_hyb` is a drop-in for ``respect.kernels.attention.fused_attn_hyb``
(respect/kernels/attention.py:74-96): same argument names, shapes and output.
The tile keyword arguments (BM, BN, num_warps, num_stages) of the Triton
version are accepted and ignored; BNB keeps the reference's divisibility
check on the node count. The computation runs in librespect_b200.so
(rb_fused_attn_hyb): prefix keys in fixed chunks at absolute positions,
nodes one at a time in slot order, fp32 accumulation, one final cast.

`prompt_attention` (rb_prompt_attn) is causal attention over packed whole prompts;
`paged_attention` (rb_paged_attn) reads one new token's keys from a paged cache
(respect_b200.decoding.kv_pages). Both take bf16 or fp32, any number of query heads
per kv head that divides evenly, head size 128, and keep the property of the trie
kernel: what a sequence gets does not depend on what else the call carries.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from respect_b200 import _lib

_MASK_KIND = {torch.bool: _lib.RB_MASK_BOOL, torch.uint8: _lib.RB_MASK_BOOL,
              torch.bfloat16: _lib.RB_MASK_ADD_BF16, torch.float32: _lib.RB_MASK_ADD_F32}


def _unit_inner(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def attn_call(q, kp, vp, kn, vn, msk, out, sm_scale, mask_kind=None, causal_first=0):
    """Launch rb_fused_attn_hyb on explicit (possibly strided) views.

    q, out [H, M, D]; kp, vp [HK, NP, D]; kn, vn [HK, NN, D]; msk [M, NN] (bool,
    or additive bf16/fp32 where 0 means attend) or None with
    mask_kind=RB_MASK_CAUSAL.
    """
    H, M, D = q.shape
    HK, NP, _ = kp.shape
    NN = kn.shape[1]
    a = _lib.AttnArgs()
    a.dtype = _lib.dtype_code(q.dtype)
    a.H, a.M, a.D, a.HK, a.NP, a.NN = H, M, D, HK, NP, NN
    a.q, (a.sqh, a.sqm, a.sqd) = q.data_ptr(), q.stride()
    a.kp, (a.skph, a.skpn, a.skpd) = kp.data_ptr(), kp.stride()
    a.vp, (a.svph, a.svpn, a.svpd) = vp.data_ptr(), vp.stride()
    a.kn, (a.sknh, a.sknn, a.sknd) = kn.data_ptr(), kn.stride()
    a.vn, (a.svnh, a.svnn, a.svnd) = vn.data_ptr(), vn.stride()
    if msk is None:
        a.msk, a.mask_kind, a.smm, a.smn = None, _lib.RB_MASK_CAUSAL, 0, 0
    else:
        a.msk, (a.smm, a.smn) = msk.data_ptr(), msk.stride()
        a.mask_kind = _MASK_KIND[msk.dtype] if mask_kind is None else mask_kind
    a.causal_first = int(causal_first)
    a.out, (a.soh, a.som, a.sod) = out.data_ptr(), out.stride()
    a.sm_scale = float(sm_scale)
    nbytes = _lib.lib().rb_fused_attn_hyb_workspace(H, M, D, NP)
    ws = _lib.workspace(q, nbytes)
    _lib.call("rb_fused_attn_hyb", ctypes.byref(a), ws.data_ptr() if ws is not None else None,
              nbytes, _lib.stream_of(q))
    return out


def fused_attn_hyb(q, kp, vp, kn, vn, msk, sm_scale=None,
                   BM=64, BN=128, BNB=16, num_warps=4, num_stages=1):
    """q [H, M, D], kp/vp [HK, NP, D], kn/vn [HK, NN, D], msk [M, NN] bool -> [H, M, D]."""
    H, M, D = q.shape
    NN = kn.shape[1]
    assert NN % BNB == 0  # same precondition as the reference (attention.py:79)
    if sm_scale is None:
        sm_scale = D ** -0.5
    q, kp, vp, kn, vn = (_unit_inner(t) for t in (q, kp, vp, kn, vn))
    out = torch.empty_like(q)
    return attn_call(q, kp, vp, kn, vn, msk, out, sm_scale)


def _laid_out(t: torch.Tensor) -> bool:
    """Unit inner stride, everything else in whole 16-byte pieces and no dimension repeated in place."""
    *outer, inner = t.stride()
    odd = t.data_ptr() // t.element_size()
    for x in outer:
        odd |= x                     # any low bit set shows
    return inner == 1 and odd % (16 // t.element_size()) == 0 and not (0 in outer and _repeats(t))


def _repeats(t: torch.Tensor) -> bool:
    return any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape))


def _rows(t: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    """t with the layout the kernels read; a copy only if it lacks it."""
    if t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise TypeError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    return t if _laid_out(t) else t.clone(memory_format=torch.contiguous_format)


def _out(out: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError(f"out must be {tuple(q.shape)} {q.dtype} on {q.device}")
    if not _laid_out(out):
        raise ValueError("out needs a unit inner stride and rows in whole 16-byte pieces")
    return out


def _int32(t: torch.Tensor, name: str, dims: int, like: torch.Tensor) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.get_device() != like.get_device() or t.dim() != dims:
        raise TypeError(f"{name} must be an int32 tensor of {dims} dimension(s) on {like.device}")
    if (t.stride(-1) != 1 and t.shape[-1] > 1) or (dims == 2 and t.stride(0) < t.shape[1]):
        t = t.contiguous()               # rows that overlap, as of an expanded table
    return t


def _check_heads(dtype: torch.dtype, heads: int, heads_kv: int, dim: int, dim_kv: int) -> None:
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise TypeError(f"attention takes bf16 or fp32, got {dtype}")
    if dim != 128 or dim_kv != 128:
        raise ValueError("attention heads must have 128 dims")
    if heads_kv == 0 or heads == 0 or heads % heads_kv:
        raise ValueError(f"{heads} query heads do not share {heads_kv} kv heads evenly")


def prompt_attention(q, k, v, cu_seqlens, sm_scale=None, out=None):
    """Causal attention over whole prompts packed behind one another.

    q [T, H, 128], k, v [T, HK, 128] (bf16 or fp32; slices of a fused projection are
    read in place), cu_seqlens int32 [B + 1] on the same device: sequence i is tokens
    [cu_seqlens[i], cu_seqlens[i + 1]), ascending. Returns [T, H, 128]. Rows of no
    sequence are zero in a new result and left as they were in a given ``out``, which
    must not overlap q, k or v."""
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or ks != v.shape or ks[0] != qs[0]:
        raise ValueError(f"prompt_attention: q {tuple(qs)}, k {tuple(ks)}, v {tuple(v.shape)} do not fit")
    T, H, D = qs
    HK = ks[1]
    _check_heads(q.dtype, H, HK, D, ks[2])
    if H > 64 * HK:
        raise ValueError("prompt_attention: at most 64 query heads per kv head")
    cu = _int32(cu_seqlens, "cu_seqlens", 1, q)
    B = cu.numel() - 1
    if B < 0:
        raise ValueError("cu_seqlens holds one entry more than there are sequences")
    q, k, v = _rows(q, "q", q), _rows(k, "k", q), _rows(v, "v", q)
    y = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else _out(out, q)
    sq, sk, sv, so = q.stride(), k.stride(), v.stride(), y.stride()
    a = _lib.pack_prompt_args(_lib.dtype_code(q.dtype), B, T, H, HK, D, q.data_ptr(), sq[0], sq[1], k.data_ptr(), sk[0], sk[1],
                              v.data_ptr(), sv[0], sv[1], cu.data_ptr(), y.data_ptr(), so[0], so[1],
                              D ** -0.5 if sm_scale is None else sm_scale, out is None)
    _lib.launch("rb_prompt_attn", q, a)
    return y


@functools.lru_cache(maxsize=1024)
def _paged_bytes(dtype: int, B: int, H: int, HK: int, page_size: int, width: int, max_length: int) -> int:
    """Scratch of a paged call: a function of its sizes."""
    a = _lib.PagedArgs(dtype=dtype, B=B, H=H, HK=HK, D=128, page_size=page_size, width=width, ld_table=width,
                       max_length=max_length, q=16, out=16, lengths=16, table=16)
    return _lib.lib().rb_paged_attn_workspace(ctypes.byref(a))


def paged_attention(q, k_pages, v_pages, table, lengths, sm_scale=None, seqs=None, ahead=0, max_length=None, out=None):
    """Attention of one new token per sequence over a paged KV cache.

    q [B, H, 128]; k_pages, v_pages [pages, HK, page_size, 128]; table int32 [rows,
    width] (page numbers, entries outside the pool name no page and their tokens are
    left out), lengths int32 [rows]; seqs int32 [B]: the table row of each entry
    (default: its own index). Entry b reads the first ``lengths + ahead`` tokens of its
    row (``ahead`` counts tokens written but not committed yet), cut to the table's
    width and to ``max_length``, a bound on the lengths that keeps scratch and launch
    small when the table is much wider. No tokens give zeros. Returns [B, H, 128]."""
    qs, ks = q.shape, k_pages.shape
    if len(qs) != 3 or len(ks) != 4 or ks != v_pages.shape:
        raise ValueError(f"paged_attention: q {tuple(qs)}, k_pages {tuple(ks)}, v_pages {tuple(v_pages.shape)} do not fit")
    B, H, D = qs
    pages, HK, page_size, dim = ks
    _check_heads(q.dtype, H, HK, D, dim)
    table, lengths = _int32(table, "table", 2, q), _int32(lengths, "lengths", 1, q)
    rows, width = table.shape
    if lengths.numel() != rows:
        raise ValueError(f"{lengths.numel()} lengths for {rows} table rows")
    if seqs is None:
        if rows != B:
            raise ValueError(f"{rows} table rows for {B} queries: name the rows with seqs")
    else:
        seqs = _int32(seqs, "seqs", 1, q)
        if seqs.numel() != B:
            raise ValueError(f"{seqs.numel()} seqs for {B} queries")
    if ahead < 0 or (max_length is not None and max_length < 1):
        raise ValueError("ahead must not be negative, max_length must be positive")
    q, k, v = _rows(q, "q", q), _rows(k_pages, "k_pages", q), _rows(v_pages, "v_pages", q)
    y = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else _out(out, q)
    sq, sk, sv, so = q.stride(), k.stride(), v.stride(), y.stride()
    bound = max_length or 0
    dtype = _lib.dtype_code(q.dtype)
    a = _lib.pack_paged_args(dtype, B, H, HK, D, q.data_ptr(), sq[0], sq[1], k.data_ptr(), sk[0], sk[1], sk[2],
                             v.data_ptr(), sv[0], sv[1], sv[2], pages, page_size, table.data_ptr(),
                             table.stride(0) if rows > 1 else width, width, rows, lengths.data_ptr(),
                             0 if seqs is None else seqs.data_ptr(), ahead, bound, y.data_ptr(), so[0], so[1],
                             D ** -0.5 if sm_scale is None else sm_scale)
    nbytes = _paged_bytes(dtype, B, H, HK, page_size, width, bound)
    ws = _lib.scratch(q, nbytes)
    _lib.launch("rb_paged_attn", q, a, None if ws is None else ws.data_ptr(), nbytes)
    return y

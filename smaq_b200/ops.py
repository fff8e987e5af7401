"""Torch-facing wrappers of the C-ABI kernels.

Every function here takes CUDA tensors, enqueues the kernel on
``torch.cuda.current_stream()`` and returns freshly allocated outputs (or writes
into caller buffers).  CPU tensors raise ``RuntimeError``: the hot path has no
CPU implementation.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from smaq_b200 import _lib
from smaq_b200._lib import (SMAQ_BF16, SMAQ_F16, SMAQ_F32, SMAQ_KEYS_BVQ, SMAQ_KEYS_SCALAR,
                           SMAQ_LAYOUT_DECODE, SMAQ_LAYOUT_REFERENCE)

_DT = {torch.float32: SMAQ_F32, torch.bfloat16: SMAQ_BF16, torch.float16: SMAQ_F16}

MIN_HISTORY = 16
PATH_GENERAL, PATH_FUSED_BVQ, PATH_FUSED_SCALAR = 0, 1, 2   # smaq_decode_kernel_path


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DT[dt]
    except KeyError:
        raise ValueError(f"unsupported dtype {dt}; expected float32, bfloat16 or float16") from None


def _cuda(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                "smaq_b200 kernels need CUDA tensors (there is no CPU fallback); got a tensor on "
                f"{t.device}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def packed_dim(dim: int, bits: int) -> int:
    vpb = max(1, 8 // bits)
    return (dim + vpb - 1) // vpb


def _rows(x: torch.Tensor) -> torch.Tensor:
    """Contiguous ``[n_rows, D]`` view of ``(..., D)``."""
    return x.reshape(-1, x.shape[-1]).contiguous()


# --------------------------------------------------------------------- quantize
def quantize_keys_scalar(k: torch.Tensor, E: torch.Tensor, boundaries: torch.Tensor, bits: int):
    """``(..., D)`` keys -> (packed codes ``(..., ceil(D / (8//bits)))`` uint8, norms ``(...)``)."""
    _cuda(k, E, boundaries)
    lib = _lib.load()
    D = k.shape[-1]
    kr = _rows(k)
    n = kr.shape[0]
    codes = torch.empty((n, packed_dim(D, bits)), dtype=torch.uint8, device=k.device)
    norms = torch.empty((n,), dtype=k.dtype, device=k.device)
    Ef = E.to(torch.float32).contiguous()
    bf = boundaries.to(torch.float32).contiguous()
    _lib.check(lib.smaq_quantize_keys_scalar(kr.data_ptr(), dtype_code(k.dtype), n, D, Ef.data_ptr(),
                                             bf.data_ptr(), bits, codes.data_ptr(), norms.data_ptr(),
                                             _stream()), "smaq_quantize_keys_scalar")
    return codes.reshape(*k.shape[:-1], -1), norms.reshape(k.shape[:-1])


def quantize_values(v: torch.Tensor, bits: int = 2, group_size: int = 32):
    """``(..., D)`` values -> (data uint8 ``(..., D*bits/8)``, scales, zeros ``(..., D/group)``)."""
    _cuda(v)
    lib = _lib.load()
    D = v.shape[-1]
    vr = _rows(v)
    n = vr.shape[0]
    data = torch.empty((n, D * bits // 8), dtype=torch.uint8, device=v.device)
    scales = torch.empty((n, D // group_size), dtype=v.dtype, device=v.device)
    zeros = torch.empty_like(scales)
    _lib.check(lib.smaq_quantize_values(vr.data_ptr(), dtype_code(v.dtype), n, D, bits, group_size,
                                        data.data_ptr(), scales.data_ptr(), zeros.data_ptr(), _stream()),
               "smaq_quantize_values")
    lead = v.shape[:-1]
    return data.reshape(*lead, -1), scales.reshape(*lead, -1), zeros.reshape(*lead, -1)


def quantize_keys_bvq(k: torch.Tensor, E_blocks: torch.Tensor, centroids: torch.Tensor) -> torch.Tensor:
    """``(..., D)`` keys -> uint8 block indices ``(..., D / block_dim)``."""
    _cuda(k, E_blocks, centroids)
    lib = _lib.load()
    D = k.shape[-1]
    nb, nc, bd = centroids.shape
    kr = _rows(k)
    n = kr.shape[0]
    idx = torch.empty((n, nb), dtype=torch.uint8, device=k.device)
    Eb = E_blocks.to(torch.float32).contiguous()
    cf = centroids.to(torch.float32).contiguous()
    _lib.check(lib.smaq_quantize_keys_bvq(kr.data_ptr(), dtype_code(k.dtype), n, D, Eb.data_ptr(),
                                          cf.data_ptr(), bd, nc, idx.data_ptr(), _stream()),
               "smaq_quantize_keys_bvq")
    return idx.reshape(*k.shape[:-1], nb)


def append(key: Optional[torch.Tensor], value: Optional[torch.Tensor], *, n_heads: int, slot_offset: int = 0,
           slots: Optional[torch.Tensor] = None, page_size: int, key_format: int = SMAQ_KEYS_SCALAR,
           key_bits: int = 3, E: Optional[torch.Tensor] = None, boundaries: Optional[torch.Tensor] = None,
           E_blocks: Optional[torch.Tensor] = None, centroids: Optional[torch.Tensor] = None,
           key_codes: Optional[torch.Tensor] = None, key_norms: Optional[torch.Tensor] = None,
           value_bits: int = 2, group_size: int = 32, v_data: Optional[torch.Tensor] = None,
           v_scales: Optional[torch.Tensor] = None, v_zeros: Optional[torch.Tensor] = None,
           layout: int = SMAQ_LAYOUT_REFERENCE) -> None:
    """Quantize a ``[T, H, D]`` chunk of keys and/or values into store rows (see include/smaq_b200.h)."""
    _cuda(key, value, slots, E, boundaries, E_blocks, centroids, key_codes, key_norms, v_data)
    lib = _lib.load()
    ref = key if key is not None else value
    if ref is None:
        return
    a = _lib.AppendArgs()
    a.dtype = dtype_code(ref.dtype)
    a.n_tokens = ref.shape[0]
    a.n_heads = n_heads
    a.head_dim = ref.shape[-1]
    keep = []
    if key is not None:
        if key.stride(-1) != 1:
            key = key.contiguous()
        keep.append(key)
        a.k = key.data_ptr()
        a.k_stride_t, a.k_stride_h = key.stride(0), key.stride(1)
        a.key_format = key_format
        a.key_bits = key_bits
        a.key_codes = _ptr(key_codes)
        if key_format == SMAQ_KEYS_SCALAR:
            Ef = E.to(torch.float32).contiguous()
            bf = boundaries.to(torch.float32).contiguous()
            keep += [Ef, bf]
            a.E, a.boundaries = Ef.data_ptr(), bf.data_ptr()
            a.key_norms = _ptr(key_norms)
        else:
            Eb = E_blocks.to(torch.float32).contiguous()
            cf = centroids.to(torch.float32).contiguous()
            keep += [Eb, cf]
            a.E_blocks, a.centroids = Eb.data_ptr(), cf.data_ptr()
            a.block_dim = centroids.shape[2]
            a.n_centroids = centroids.shape[1]
    if value is not None:
        if value.stride(-1) != 1:
            value = value.contiguous()
        keep.append(value)
        a.v = value.data_ptr()
        a.v_stride_t, a.v_stride_h = value.stride(0), value.stride(1)
        a.value_bits = value_bits
        a.group_size = group_size
        a.v_data, a.v_scales, a.v_zeros = _ptr(v_data), _ptr(v_scales), _ptr(v_zeros)
    if slots is not None:
        slots = slots.to(torch.int64).contiguous()
        keep.append(slots)
        a.slots = slots.data_ptr()
    a.slot_offset = slot_offset
    a.page_size = page_size
    a.layout = layout
    _lib.check(lib.smaq_append(a, _stream()), "smaq_append")


# --------------------------------------------------------------------- standalone scores / attend
def _packed_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with packed rows (last dim contiguous, rows back to back within a group); a group
    stride may be anything (a capacity buffer sliced along its token dim keeps its storage)."""
    if t.stride(-1) == 1 and (t.dim() < 2 or t.shape[-2] <= 1 or t.stride(-2) == t.shape[-1]):
        return t
    return t.contiguous()


def _groups(lead: torch.Size, *ts: torch.Tensor, tail: tuple[int, ...]) -> list[torch.Tensor]:
    """Each tensor broadcast to ``lead + its own trailing dims`` and flattened to ``[G, ...]``."""
    out = []
    for t, k in zip(ts, tail):
        t = t.expand(*lead, *t.shape[t.dim() - k:])
        out.append(t.reshape(-1, *t.shape[len(lead):]))
    return out


def key_scores(query: torch.Tensor, *, key_format: int, scale: Optional[float] = None,
               key_codes: Optional[torch.Tensor] = None, key_norms: Optional[torch.Tensor] = None, key_bits: int = 3,
               E_inv: Optional[torch.Tensor] = None, centroids: Optional[torch.Tensor] = None,
               key_idx: Optional[torch.Tensor] = None, decoded_centroids: Optional[torch.Tensor] = None
               ) -> torch.Tensor:
    """``scale * q . k_hat`` of ``query [..., Q, D]`` against compressed keys (reference layout):
    scalar ``key_codes [..., N, ceil(D/(8/bits))]`` + ``key_norms [..., N]``, or block-VQ
    ``key_idx [..., N, D/bd]`` (uint8 or int64).  Leading dims broadcast.  Returns ``[..., Q, N]`` in
    the query dtype (smaq_key_scores)."""
    _cuda(query, key_codes, key_idx)
    lib = _lib.load()
    D = query.shape[-1]
    keys = key_codes if key_format == SMAQ_KEYS_SCALAR else key_idx
    lead = torch.broadcast_shapes(query.shape[:-2], keys.shape[:-2])
    N = keys.shape[-2]
    (q,) = _groups(lead, query, tail=(2,))
    q = q if q.stride(-1) == 1 else q.contiguous()
    G, Q = q.shape[0], q.shape[1]
    out = torch.empty((G, Q, N), dtype=query.dtype, device=query.device)
    a = _lib.ScoresArgs()
    a.q, a.q_dtype, a.q_stride_g, a.q_stride_q = q.data_ptr(), dtype_code(q.dtype), q.stride(0), q.stride(1)
    a.n_groups, a.n_queries, a.n_tokens, a.head_dim = G, Q, N, D
    a.key_format = key_format
    a.scale = float(1.0 if scale is None else scale)
    keep = [q]
    if key_format == SMAQ_KEYS_SCALAR:
        # rotate the few query rows once (a small fp32 GEMM) instead of in every CTA
        qr = torch.matmul(q.float(), E_inv.to(q.device, torch.float32).T).contiguous()
        keep.append(qr)
        a.q, a.q_dtype, a.q_stride_g, a.q_stride_q = qr.data_ptr(), SMAQ_F32, qr.stride(0), qr.stride(1)
        a.q_rotated = 1
        codes, norms = _groups(lead, key_codes, key_norms, tail=(2, 1))
        codes, norms = _packed_rows(codes), (norms if norms.stride(-1) == 1 else norms.contiguous())
        Ei = E_inv.to(torch.float32).contiguous()
        cf = centroids.to(torch.float32).contiguous()
        keep += [codes, norms, Ei, cf]
        a.key_codes, a.codes_stride_g = codes.data_ptr(), codes.stride(0)
        a.key_norms, a.norms_dtype, a.norms_stride_g = norms.data_ptr(), dtype_code(norms.dtype), norms.stride(0)
        a.key_bits, a.E_inv, a.centroids = key_bits, Ei.data_ptr(), cf.data_ptr()
    else:
        (idx,) = _groups(lead, key_idx, tail=(2,))
        idx = _packed_rows(idx)
        if idx.dtype not in (torch.uint8, torch.int64):
            idx = idx.to(torch.int64)
        dc = decoded_centroids.to(torch.float32).contiguous()
        keep += [idx, dc]
        a.key_idx, a.idx_is_int64, a.idx_stride_g = idx.data_ptr(), int(idx.dtype == torch.int64), idx.stride(0)
        a.block_dim, a.n_centroids, a.decoded_centroids = dc.shape[2], dc.shape[1], dc.data_ptr()
    a.out, a.out_dtype, a.out_stride_g, a.out_stride_q = out.data_ptr(), dtype_code(out.dtype), out.stride(0), \
        out.stride(1)
    _lib.check(lib.smaq_key_scores(a, _stream()), "smaq_key_scores")
    return out.reshape(*lead, Q, N)


def attend_values(weights: torch.Tensor, v_data: torch.Tensor, v_scales: torch.Tensor, v_zeros: torch.Tensor, *,
                  bits: int = 2, group_size: int = 32, head_dim: Optional[int] = None,
                  out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``weights [..., Q, N]`` applied to compressed values ``v_data [..., N, D*bits/8]`` with
    ``v_scales / v_zeros [..., N, D/group_size]`` (reference layout): ``[..., Q, D]`` in the
    weights dtype (smaq_attend_values, dequantization fused)."""
    _cuda(weights, v_data)
    lib = _lib.load()
    D = head_dim or v_data.shape[-1] * 8 // bits
    lead = torch.broadcast_shapes(weights.shape[:-2], v_data.shape[:-2])
    w, = _groups(lead, weights, tail=(2,))
    w = w if w.stride(-1) == 1 else w.contiguous()
    data, sc, zs = (_packed_rows(t) for t in _groups(lead, v_data, v_scales, v_zeros, tail=(2, 2, 2)))
    if zs.dtype != sc.dtype:
        zs = zs.to(sc.dtype)
    G, Q, N = w.shape
    out = torch.empty((G, Q, D), dtype=out_dtype or weights.dtype, device=weights.device)
    ws_bytes = int(lib.smaq_attend_workspace_size(G, Q, N, D))
    ws = torch.empty((max(ws_bytes, 16),), dtype=torch.uint8, device=weights.device)
    a = _lib.AttendArgs()
    a.w, a.w_dtype, a.w_stride_g, a.w_stride_q = w.data_ptr(), dtype_code(w.dtype), w.stride(0), w.stride(1)
    a.n_groups, a.n_queries, a.n_tokens, a.head_dim = G, Q, N, D
    a.v_data, a.data_stride_g = data.data_ptr(), data.stride(0)
    a.v_scales, a.v_zeros, a.sz_dtype, a.sz_stride_g = sc.data_ptr(), zs.data_ptr(), dtype_code(sc.dtype), sc.stride(0)
    a.value_bits, a.group_size = bits, group_size
    a.out, a.out_dtype, a.out_stride_g, a.out_stride_q = out.data_ptr(), dtype_code(out.dtype), out.stride(0), \
        out.stride(1)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _lib.check(lib.smaq_attend_values(a, _stream()), "smaq_attend_values")
    return out.reshape(*lead, Q, D)


# --------------------------------------------------------------------- calibration
def kmeans(data: torch.Tensor, n_centroids: int, n_iters: int = 20, seed: int = 42) -> torch.Tensor:
    """k-means++ + Lloyd on the device for ``data [n_blocks, n_points, dim]`` (fp32, dim <= 16):
    ``[n_blocks, n_centroids, dim]`` centroids, one ``smaq_kmeans`` call, no host round trips
    inside."""
    _cuda(data)
    lib = _lib.load()
    x = data.to(torch.float32).contiguous()
    nb, n, d = x.shape
    cent = torch.empty((nb, n_centroids, d), dtype=torch.float32, device=x.device)
    ws = torch.empty((int(lib.smaq_kmeans_workspace_size(nb, n)),), dtype=torch.uint8, device=x.device)
    _lib.check(lib.smaq_kmeans(x.data_ptr(), nb, n, d, n_centroids, n_iters, seed & (2 ** 64 - 1), cent.data_ptr(),
                               ws.data_ptr(), ws.numel(), _stream()), "smaq_kmeans")
    return cent


# --------------------------------------------------------------------- decode
def decode_workspace_bytes(batch: int, n_q_heads: int, n_kv_heads: int, head_dim: int, num_ctas: int = 0) -> int:
    return int(_lib.load().smaq_decode_workspace_size(batch, n_q_heads, n_kv_heads, head_dim, num_ctas))


def decode(q: torch.Tensor, *, n_kv_heads: int, key_format: int, key_codes: torch.Tensor,
           v_data: torch.Tensor, v_scales: torch.Tensor, v_zeros: torch.Tensor, hist_len: torch.Tensor,
           page_size: int, key_bits: int = 4, E_inv: Optional[torch.Tensor] = None,
           centroids: Optional[torch.Tensor] = None, key_norms: Optional[torch.Tensor] = None,
           value_bits: int = 2, group_size: int = 32, block_table: Optional[torch.Tensor] = None,
           hist_total: Optional[torch.Tensor] = None, recent_k: Optional[torch.Tensor] = None,
           recent_v: Optional[torch.Tensor] = None, recent_len: Optional[torch.Tensor] = None,
           scale: Optional[float] = None, min_history: int = MIN_HISTORY, out: Optional[torch.Tensor] = None,
           partial_out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
           num_ctas: int = 0, want_out: bool = True, layout: int = SMAQ_LAYOUT_REFERENCE,
           centroids_f16: Optional[torch.Tensor] = None, entry: str = "smaq_decode",
           overlap_prior: bool = False, query_path: bool = False):
    """Batched hybrid decode attention.

    ``q``: ``[B, Hq, D]``.  History streams are store rows ``[pages, Hkv, page_size, ...]``;
    ``recent_k/v``: ``[B, W, Hkv, D]`` (stride 0 on B allowed).  Returns ``out [B, Hq, D]`` in
    the query dtype (reference rounding), and/or fills ``partial_out [B, Hq, 2D+2]``.
    ``overlap_prior``: overlap the launch with the end of the previous kernel on the stream
    (programmatic dependent launch); only when that kernel writes none of the history rows,
    block table, lengths or codebooks (``smaq_decode_args.overlap_prior``).
    ``query_path``: launch nothing and return the kernel path these arguments select
    (``PATH_FUSED_BVQ``, ``PATH_FUSED_SCALAR`` or ``PATH_GENERAL``, smaq_decode_kernel_path).
    """
    _cuda(q, key_codes, v_data, hist_len, recent_k, block_table)
    lib = _lib.load()
    B, Hq, D = q.shape
    if q.stride(-1) != 1:
        q = q.contiguous()
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None and want_out and not query_path:
        out = torch.empty((B, Hq, D), dtype=q.dtype, device=q.device)
    keep = [q]
    a = _lib.DecodeArgs()
    a.q, a.q_dtype, a.q_stride_b, a.q_stride_h = q.data_ptr(), dtype_code(q.dtype), q.stride(0), q.stride(1)
    a.batch, a.n_q_heads, a.n_kv_heads, a.head_dim = B, Hq, n_kv_heads, D
    a.scale = float(scale)
    a.key_format = key_format
    a.key_bits = key_bits
    if key_format == SMAQ_KEYS_SCALAR:
        Ei = E_inv.to(torch.float32).contiguous()
        cf = centroids.to(torch.float32).contiguous()
        keep += [Ei, cf]
        a.E_inv, a.centroids = Ei.data_ptr(), cf.data_ptr()
        a.key_norms = key_norms.data_ptr()
        a.kv_dtype = dtype_code(key_norms.dtype)
    else:
        cf = centroids.to(torch.float32).contiguous()
        keep.append(cf)
        a.centroids = cf.data_ptr()
        a.block_dim = centroids.shape[2]
        a.n_centroids = centroids.shape[1]
        a.kv_dtype = dtype_code(v_scales.dtype)
    a.key_codes = key_codes.data_ptr()
    a.v_data, a.v_scales, a.v_zeros = v_data.data_ptr(), v_scales.data_ptr(), v_zeros.data_ptr()
    a.value_bits, a.group_size = value_bits, group_size
    if block_table is not None:
        bt = block_table.to(torch.int32)
        if bt.stride(-1) != 1:
            bt = bt.contiguous()
        keep.append(bt)
        a.block_table, a.bt_stride = bt.data_ptr(), bt.stride(0)
    a.page_size = page_size
    hl = hist_len.to(torch.int32).contiguous()
    keep.append(hl)
    a.hist_len = hl.data_ptr()
    if hist_total is not None:
        ht = hist_total.to(torch.int32).contiguous()
        keep.append(ht)
        a.hist_total = ht.data_ptr()
    a.min_history = min_history
    if recent_k is not None and recent_len is not None:
        if recent_k.stride(-1) != 1 or recent_v.stride(-1) != 1 or recent_k.stride() != recent_v.stride():
            recent_k, recent_v = recent_k.contiguous(), recent_v.contiguous()
        rl = recent_len.to(torch.int32).contiguous()
        keep += [recent_k, recent_v, rl]
        a.recent_k, a.recent_v = recent_k.data_ptr(), recent_v.data_ptr()
        a.recent_dtype = dtype_code(recent_k.dtype)
        a.r_stride_b, a.r_stride_t, a.r_stride_h = recent_k.stride(0), recent_k.stride(1), recent_k.stride(2)
        a.recent_len = rl.data_ptr()
    if out is not None:
        a.out, a.o_stride_b, a.o_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    if partial_out is not None:
        a.partial_out = partial_out.data_ptr()
    if entry != "smaq_decode_noalloc" and not query_path:
        need = decode_workspace_bytes(B, Hq, n_kv_heads, D, num_ctas)
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty((max(need, 256),), dtype=torch.uint8, device=q.device)
        keep.append(workspace)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    a.num_ctas = num_ctas
    a.layout = layout
    a.overlap_prior = 1 if overlap_prior else 0
    if centroids_f16 is not None:
        c16 = centroids_f16.to(torch.float16).contiguous()
        keep.append(c16)
        a.centroids_f16 = c16.data_ptr()
    if query_path:
        if out is None and partial_out is None:
            a.out = 1  # any non-null output: only the kernel choice is asked for
        st = lib.smaq_decode_kernel_path(a)
        if st < 0:
            _lib.check(-st, "smaq_decode_kernel_path")
        return st
    if entry == "smaq_decode_noalloc":
        # fixed scratch inside the library: no workspace is passed (see include/smaq_b200.h)
        a.workspace, a.workspace_bytes = None, 0
        _lib.check(lib.smaq_decode_noalloc(a, _stream()), "smaq_decode_noalloc")
        return out
    _lib.check(lib.smaq_decode(a, _stream()), "smaq_decode")
    return out


_EMPTY_STORES: dict = {}


def _empty_store(device: torch.device, n_kv_heads: int, head_dim: int, dtype: torch.dtype) -> dict:
    """One 16-row page of 4-bit scalar-key store rows (decode layout) that no decode reads: the
    history streams of a window-only decode must still be valid pointers."""
    key = (device, n_kv_heads, head_dim, dtype)
    st = _EMPTY_STORES.get(key)
    if st is None:
        H, D = n_kv_heads, head_dim
        st = dict(codes=torch.zeros((1, H, 16, packed_dim(D, 4)), dtype=torch.uint8, device=device),
                  norms=torch.zeros((1, H, 16), dtype=dtype, device=device),
                  vdata=torch.zeros((1, H, 16, D // 4), dtype=torch.uint8, device=device),
                  vsz=torch.zeros((1, H, 16, max(1, D // 32)), dtype=dtype, device=device),
                  E_inv=torch.eye(D, dtype=torch.float32, device=device),
                  centroids=torch.zeros(16, dtype=torch.float32, device=device))
        _EMPTY_STORES[key] = st
    return st


def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of a chunk over itself: ``q [n, Hq, D]``, ``k / v [n, Hkv, D]`` ->
    ``[n, Hq, D]`` in the query dtype; query head ``h`` reads KV head ``h // (Hq / Hkv)``.

    Runs as one ``smaq_decode`` over ``n`` window-only rows: row ``i`` is query token ``i`` with
    an exact window of the chunk's first ``i + 1`` tokens.  The window is the chunk itself for
    every row (batch stride 0), so K and V are neither expanded per query head nor copied per
    row; the rows of one KV head are re-read from L2 (``n^2 / 2`` row reads per head).  bf16 /
    fp16 inputs with head_dim 128 and at most 8 query heads per KV head take the tensor-core
    window of the fused scalar-key kernel while ``2 n Hkv <= 2048``, other shapes the general
    kernel."""
    _cuda(q, k, v)
    n, Hq, D = q.shape
    Hkv = k.shape[1]
    if n == 0:
        return torch.empty_like(q)
    k = k if k.stride(-1) == 1 and k.is_contiguous() else k.contiguous()
    v = v if v.is_contiguous() else v.contiguous()
    if v.dtype != k.dtype:
        v = v.to(k.dtype)
    st = _empty_store(q.device, Hkv, D, k.dtype if k.dtype != torch.float32 else torch.bfloat16)
    rows = torch.arange(1, n + 1, dtype=torch.int32, device=q.device)
    zero = torch.zeros(n, dtype=torch.int32, device=q.device)
    return decode(q, n_kv_heads=Hkv, key_format=SMAQ_KEYS_SCALAR, key_bits=4, E_inv=st["E_inv"],
                  centroids=st["centroids"], key_norms=st["norms"], key_codes=st["codes"], v_data=st["vdata"],
                  v_scales=st["vsz"], v_zeros=st["vsz"], hist_len=zero, page_size=16,
                  block_table=torch.zeros((n, 1), dtype=torch.int32, device=q.device),
                  recent_k=k.unsqueeze(0).expand(n, n, Hkv, D), recent_v=v.unsqueeze(0).expand(n, n, Hkv, D),
                  recent_len=rows, scale=scale, layout=SMAQ_LAYOUT_DECODE)


def merge_partials(partials: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    """``[R, B, Hq, 2D+2]`` fp32 partials -> ``[B, Hq, D]`` output."""
    _cuda(partials)
    lib = _lib.load()
    R, B, Hq, W = partials.shape
    D = (W - 2) // 2
    p = partials.contiguous()
    out = torch.empty((B, Hq, D), dtype=out_dtype, device=partials.device)
    _lib.check(lib.smaq_merge_partials(p.data_ptr(), R, B, Hq, D, out.data_ptr(), dtype_code(out_dtype),
                                       out.stride(0), out.stride(1), _stream()), "smaq_merge_partials")
    return out


# --------------------------------------------------------------------- exact paged step
class StepTables(NamedTuple):
    """What ``step_tables`` builds (smaq_tables_args in include/smaq_b200.h)."""
    cu_query: torch.Tensor      # [B + 1] int32, prefix sums of the query lengths
    seq_lens: torch.Tensor      # [B] int32, context + query; 0: finished or not admitted
    positions: torch.Tensor     # [num_tokens] int32
    slots: torch.Tensor         # [num_tokens] int64, page * block_size + offset; -1: no slot
    free_count: torch.Tensor    # [1] int32
    admitted: torch.Tensor      # [B] bool


def _stream_for(ref: torch.Tensor, others: tuple) -> int:
    """The current stream of ``ref``'s device, on which every other tensor (or None) must be too."""
    dev = ref.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            _cuda(ref, *others)
            raise ValueError(f"tensors are on {ref.device} and {t.device}")
    if dev < 0:
        _cuda(ref)
    if dev != torch._C._cuda_getDevice():
        raise ValueError(f"tensors are on {ref.device}, but the current device is cuda:{torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(dev)


def _addr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _int32(name: str, t: torch.Tensor, n: int) -> torch.Tensor:
    if t.shape != (n,):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({n},)")
    if t.dtype is not torch.int32:
        if t.dtype.is_floating_point or t.dtype == torch.bool:
            raise ValueError(f"{name} must be an integer tensor, got {t.dtype}")
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def step_tables(free_blocks: torch.Tensor, free_count: torch.Tensor, context_lens: torch.Tensor,
                query_lens: torch.Tensor, block_table: torch.Tensor, *, block_size: int, num_tokens: int,
                finished: Optional[torch.Tensor] = None) -> StepTables:
    """Block bookkeeping of one step in one launch (smaq_step_tables).

    ``free_blocks[:free_count]`` is the stack of free pages.  Requests marked in ``finished [B]`` give
    their pages back; then request ``b`` grows from ``context_lens[b]`` by ``query_lens[b]`` tokens and
    takes the pages it lacks, in request order while the stack lasts.  A request whose pages run out or
    that outgrows its row of ``block_table [B, M]`` is not admitted: its slots are -1 and its sequence
    length is 0.  ``free_blocks`` (int32) and ``block_table`` (int32) are updated in place, the
    new ``free_count`` is returned.  ``num_tokens``: length of ``positions`` and ``slots``; entries past
    the step's tokens get position 0 and slot -1.  Nothing is read back to the host."""
    stream = _stream_for(free_blocks, (free_count, context_lens, query_lens, block_table, finished))
    B = context_lens.shape[0]
    if free_blocks.dtype is not torch.int32 or free_blocks.dim() != 1 or not free_blocks.is_contiguous():
        raise ValueError("free_blocks must be a contiguous int32 vector (it is updated in place)")
    width = block_table.shape
    if block_table.dtype is not torch.int32 or len(width) != 2 or width[0] != B or (
            width[1] > 1 and block_table.stride(1) != 1) or (B > 1 and block_table.stride(0) < width[1]):
        raise ValueError(f"block_table must be int32 [{B}, M] with contiguous rows of their own (it is updated in place)")
    if num_tokens < 0 or block_size < 1:
        raise ValueError(f"num_tokens {num_tokens} or block_size {block_size} out of range")
    free_count = _int32("free_count", free_count, 1)
    context_lens, query_lens = _int32("context_lens", context_lens, B), _int32("query_lens", query_lens, B)
    if finished is not None:
        if finished.shape != (B,) or finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"finished must be a bool vector of length {B}")
        if not finished.is_contiguous():
            finished = finished.contiguous()
    # two buffers and the flags; the small vectors lie behind the positions
    M, T = width[1], num_tokens
    slots = free_blocks.new_empty(T, dtype=torch.int64)
    buf = free_blocks.new_empty(T + 2 * B + 2)
    positions, cu, lens, left = buf.split_with_sizes([T, B + 1, B, 1])
    admitted = free_blocks.new_empty(B, dtype=torch.bool)
    at = buf.data_ptr()
    rest = at + 4 * T
    st = _lib.load().smaq_step_tables(
        _lib.pack_tables(free_blocks.data_ptr(), free_count.data_ptr(), context_lens.data_ptr(), query_lens.data_ptr(),
                         _addr(finished), block_table.data_ptr(), max(block_table.stride(0), M), free_blocks.shape[0], T,
                         B, M, block_size, rest, rest + 4 * (B + 1), at, slots.data_ptr(), admitted.data_ptr(),
                         rest + 4 * (2 * B + 1)), stream)
    if st:
        _lib.check(st, "smaq_step_tables")
    return StepTables(cu, lens, positions, slots, left, admitted)


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0, *, linear: float = 1.0,
               ntk: float = 1.0, yarn: Optional[dict] = None, device="cuda") -> torch.Tensor:
    """``[max_positions, rotary_dim]`` fp32 rows ``cos | sin`` for ``norm_rope``, computed in fp64.

    Long contexts: ``linear`` divides positions; ``ntk`` raises the base to
    ``base * ntk ** (R / (R - 2))``; ``yarn = dict(factor, original, beta_fast=32, beta_slow=1,
    attention=None)`` interpolates between the plain and the divided frequency of each pair by the
    number of turns it makes over ``original`` positions, and multiplies the rows by
    ``attention`` (default ``0.1 ln(factor) + 1``)."""
    R = rotary_dim
    if max_positions < 1 or R < 2 or R % 2:
        raise ValueError(f"rope_table: max_positions {max_positions} or rotary_dim {rotary_dim} out of range")
    if linear <= 0 or ntk <= 0 or base <= 0:
        raise ValueError("rope_table: base and scaling factors must be positive")
    if ntk != 1.0:
        if R == 2:
            raise ValueError("rope_table: ntk scaling needs a rotary_dim above 2")
        base = base * ntk ** (R / (R - 2))
    exps = torch.arange(0, R, 2, dtype=torch.float64, device=device) / R
    freq = base ** -exps
    gain = 1.0
    if yarn is not None:
        factor, original = float(yarn["factor"]), float(yarn["original"])
        fast, slow = float(yarn.get("beta_fast", 32.0)), float(yarn.get("beta_slow", 1.0))
        if factor <= 0 or original <= 0 or fast <= slow:
            raise ValueError("rope_table: yarn needs factor, original > 0 and beta_fast > beta_slow")

        def pair(turns):  # index of the pair that makes this many turns over `original` positions
            return R * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), R - 1)
        ramp = ((torch.arange(R // 2, dtype=torch.float64, device=device) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        gain = yarn.get("attention")
        if gain is None:
            gain = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] / linear * freq
    return (torch.cat([angle.cos(), angle.sin()], 1) * gain).to(torch.float32)


def _head_rows(name: str, x: torch.Tensor, dtype: torch.dtype, T: int, D: int) -> tuple:
    """``x`` with contiguous channels, its heads, token stride and head stride."""
    shape = x.shape
    if len(shape) != 3 or shape[0] != T or shape[2] != D or x.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype} [{T}, heads, {D}], got {x.dtype} {tuple(shape)}")
    st, sh, sd = x.stride()
    if sd != 1 and D > 1:
        x = x.contiguous()
        st, sh, _ = x.stride()
    return x, shape[1], st, sh


def _vector_f32(name: str, w: torch.Tensor, n: int) -> torch.Tensor:
    if w.shape != (n,):
        raise ValueError(f"{name} has shape {tuple(w.shape)}, expected ({n},)")
    return w if w.dtype is torch.float32 and w.is_contiguous() else w.to(torch.float32).contiguous()


def _cache_pair(k_cache: torch.Tensor, v_cache: torch.Tensor, dtype: torch.dtype, D: int) -> tuple:
    """Pages, page size, heads and the page, slot and head strides of a checked pair."""
    shape, strides = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or shape != v_cache.shape or shape[3] != D:
        raise ValueError(f"caches must be [pages, page_size, kv_heads, {D}], got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)}")
    if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError(f"caches must be {dtype} like the queries, got {k_cache.dtype} and {v_cache.dtype}")
    if strides != v_cache.stride() or (D > 1 and strides[3] != 1):
        raise ValueError("caches must have the same strides and a contiguous head_dim")
    return shape[0], shape[1], shape[2], strides[0], strides[1], strides[2]


def norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, *,
              q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
              interleaved: bool = False, v: Optional[torch.Tensor] = None, k_cache: Optional[torch.Tensor] = None,
              v_cache: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None):
    """Per-head RMS norm and rotation of ``q [T, Hq, D]`` and ``k [T, Hkv, D]`` in one pass
    (smaq_norm_rope); returns ``(q_out, k_out)``.

    ``table [P, R]``: rows ``cos | sin`` (``rope_table``) read at ``positions [T]``; the first ``R``
    channels turn in pairs ``(i, i + R/2)``, or ``(2i, 2i + 1)`` with ``interleaved``, the others pass.
    ``q_weight / k_weight [D]``: norm weights, None: no norm.  Heads may be views of a fused
    projection (any token and head stride).  With ``v, k_cache, v_cache, slots`` the keys and values go
    straight to the exact cache ``[pages, page_size, Hkv, D]`` at ``slots [T]`` (a slot outside the
    cache is skipped) and ``k_out`` is None."""
    T, Hq, D = q.shape
    dt = q.dtype
    code = dtype_code(dt)
    stream = _stream_for(q, (k, positions, table, q_weight, k_weight, v, k_cache, v_cache, slots))
    q, _, qt, qh = _head_rows("q", q, dt, T, D)
    k, Hk, kt, kh = _head_rows("k", k, dt, T, D)
    positions = _int32("positions", positions, T)
    rows = table.shape
    if len(rows) != 2 or table.dtype is not torch.float32 or rows[1] > D or rows[1] % 2:
        raise ValueError(f"table must be float32 [positions, R] with an even R <= {D}, got {table.dtype} {tuple(rows)}")
    if not table.is_contiguous():
        table = table.contiguous()
    if q_weight is not None:
        q_weight = _vector_f32("q_weight", q_weight, D)
    if k_weight is not None:
        k_weight = _vector_f32("k_weight", k_weight, D)
    k_out = None
    vt = vh = pages = page_size = cp = cs = ch = 0
    if k_cache is None and v is None and v_cache is None and slots is None:
        k_out = k.new_empty((T, Hk, D))
    else:
        if k_cache is None or v is None or v_cache is None or slots is None:
            raise ValueError("a cache write needs v, k_cache, v_cache and slots together")
        v, Hv, vt, vh = _head_rows("v", v, dt, T, D)
        pages, page_size, Hc, cp, cs, ch = _cache_pair(k_cache, v_cache, dt, D)
        if Hv != Hk or Hc != Hk:
            raise ValueError(f"v has {Hv} heads and the cache {Hc}, k has {Hk}")
        if slots.shape != (T,):
            raise ValueError(f"slots has shape {tuple(slots.shape)}, expected ({T},)")
        if slots.dtype is not torch.int64 or not slots.is_contiguous():
            slots = slots.to(torch.int64).contiguous()
    q_out = q.new_empty((T, Hq, D))
    st = _lib.load().smaq_norm_rope(
        _lib.pack_norm_rope(q.data_ptr(), k.data_ptr(), _addr(v), qt, qh, kt, kh, vt, vh, positions.data_ptr(),
                            table.data_ptr(), _addr(q_weight), _addr(k_weight), _addr(slots), q_out.data_ptr(),
                            _addr(k_out), _addr(k_cache), _addr(v_cache), cp, cs, ch, T, rows[0], pages, code, Hq, Hk,
                            D, rows[1], int(interleaved), page_size, eps), stream)
    if st:
        _lib.check(st, "smaq_norm_rope")
    return q_out, k_out


def paged_decode_workspace_bytes(batch: int, n_q_heads: int, n_kv_heads: int, head_dim: int) -> int:
    return int(_lib.load().smaq_paged_decode_workspace_size(batch, n_q_heads, n_kv_heads, head_dim))


def paged_prefill_workspace_bytes(n_rows: int, batch: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                                  max_tokens: int = 2 ** 31) -> int:
    """``max_tokens``: what the block table has room for (``M * page_size``)."""
    return int(_lib.load().smaq_paged_prefill_workspace_size(n_rows, batch, n_q_heads, n_kv_heads, head_dim, max_tokens))


def _paged(name, q, k_cache, v_cache, block_table, seq_lens, cu_query, prefix_lens, scale, window, softcap, slopes,
           out, return_lse, workspace):
    if q.dim() != 3:
        raise ValueError(f"q must be [rows, heads, head_dim], got {tuple(q.shape)}")
    T, Hq, D = q.shape
    dt = q.dtype
    code = dtype_code(dt)
    stream = _stream_for(q, (k_cache, v_cache, block_table, seq_lens, cu_query, prefix_lens, slopes, out, workspace))
    qt, qh, qd = q.stride()
    if qd != 1 and D > 1:
        q = q.contiguous()
        qt, qh, _ = q.stride()
    P, page_size, Hk, cp, cs, ch = _cache_pair(k_cache, v_cache, dt, D)
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [batch, blocks], got {tuple(block_table.shape)}")
    B, M = block_table.shape
    if block_table.dtype is not torch.int32:
        block_table = block_table.to(torch.int32)
    row, col = block_table.stride()
    if (M > 1 and col != 1) or (B > 1 and row < M):  # rows that overlap, such as one row expanded over requests
        block_table = block_table.contiguous()
        row = M
    seq_lens = _int32("seq_lens", seq_lens, B)
    if Hk == 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads do not divide over {Hk} KV heads")
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if softcap is not None and not softcap > 0:
        raise ValueError(f"softcap must be positive, got {softcap}")
    if prefix_lens is not None:
        prefix_lens = _int32("prefix_lens", prefix_lens, B)
    if slopes is not None:
        slopes = _vector_f32("slopes", slopes, Hq)
    if out is None:
        out = q.new_empty((T, Hq, D))
    elif out.shape != q.shape or out.dtype is not dt or (D > 1 and out.stride(2) != 1):
        raise ValueError(f"out must be {dt} {tuple(q.shape)} with a contiguous head_dim")
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    ot, oh, _ = out.stride()
    lib = _lib.load()
    ws = ws_bytes = 0
    if cu_query is None:
        if T != B:
            raise ValueError(f"q has {T} rows for {B} requests; one row a request")
        call, need = lib.smaq_paged_decode, lib.smaq_paged_decode_workspace_size(B, Hq, Hk, D)
    else:
        cu_query = _int32("cu_query", cu_query, B + 1)
        call, need = lib.smaq_paged_prefill, lib.smaq_paged_prefill_workspace_size(T, B, Hq, Hk, D,
                                                                                     M * page_size)
    if workspace is None and need:
        workspace = q.new_empty(need, dtype=torch.uint8)
    if workspace is not None:
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    st = call(
        _lib.pack_paged(q.data_ptr(), qt, qh, k_cache.data_ptr(), v_cache.data_ptr(), cp, cs, ch,
                        block_table.data_ptr(), max(row, M), seq_lens.data_ptr(), _addr(cu_query), _addr(prefix_lens),
                        _addr(slopes), out.data_ptr(), ot, oh, _addr(lse), ws, ws_bytes, P, T, B, M, page_size, Hq, Hk,
                        D, code, min(window or 0, 2 ** 31 - 1), 1.0 / math.sqrt(D) if scale is None else scale,
                        min(softcap or 0.0, 1e38)), stream)
    if st:
        _lib.check(st, name)
    return (out, lse) if return_lse else out


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, *, scale: Optional[float] = None, window: Optional[int] = None,
                 softcap: Optional[float] = None, slopes: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, return_lse: bool = False,
                 workspace: Optional[torch.Tensor] = None):
    """Attention of one new token per request over the exact paged cache (smaq_paged_decode).

    ``q [B, Hq, D]``; caches ``[pages, page_size, Hkv, D]`` of the query dtype; ``block_table [B, M]``;
    ``seq_lens [B]`` count the new token, already written.  ``window``: the last tokens that are seen;
    ``softcap``: scores become ``c * tanh(x / c)``; ``slopes [Hq]``: ``slope * distance`` is taken off.
    A request of length 0 gives zeros.  Returns ``out [B, Hq, D]``, with ``return_lse`` also the
    natural log-sum-exp ``[B, Hq]`` (fp32).  ``workspace``: ``paged_decode_workspace_bytes`` bytes (uint8),
    allocated per call when None.  ``out`` must not overlap ``q``."""
    return _paged("smaq_paged_decode", q, k_cache, v_cache, block_table, seq_lens, None, None, scale, window, softcap,
                  slopes, out, return_lse, workspace)


def paged_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  seq_lens: torch.Tensor, cu_query: torch.Tensor, *, prefix_lens: Optional[torch.Tensor] = None,
                  scale: Optional[float] = None, window: Optional[int] = None, softcap: Optional[float] = None,
                  slopes: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                  return_lse: bool = False, workspace: Optional[torch.Tensor] = None):
    """Attention of prompt chunks over the exact paged cache (smaq_paged_prefill).

    Rows ``cu_query[b] .. cu_query[b + 1]`` of ``q [T, Hq, D]`` are request ``b``'s newest tokens (the
    last ones of its ``seq_lens[b]``, already written): row ``i`` sees tokens up to its own, the last
    ``window`` of them if given, and the first ``prefix_lens[b]`` in any case.  Requests never see one
    another.  Other arguments as ``paged_decode`` (``workspace``: ``paged_prefill_workspace_bytes``
    bytes, which are 0 for many rows); rows before ``cu_query[0]`` and
    past ``cu_query[B]`` give zeros."""
    if cu_query is None:
        raise ValueError("paged_prefill needs cu_query")
    return _paged("smaq_paged_prefill", q, k_cache, v_cache, block_table, seq_lens, cu_query, prefix_lens, scale,
                  window, softcap, slopes, out, return_lse, workspace)


# --------------------------------------------------------------------- failure detection
def decode_status(batch: int, n_kv_heads: int, workspace: Optional[torch.Tensor] = None) -> None:
    """Raise if a bounded device wait of the last ``decode`` that used ``workspace`` (``None``:
    the no-allocation scratch) ran out.  Synchronises the current stream."""
    lib = _lib.load()
    _lib.check(lib.smaq_decode_status(None if workspace is None else workspace.data_ptr(), batch, n_kv_heads,
                                      _stream()), "smaq_decode_status")


def append_status() -> None:
    """Raise if a bounded device wait of the key kernel ran out since the last check (clears it)."""
    _lib.check(_lib.load().smaq_append_status(_stream()), "smaq_append_status")


def exact_status() -> None:
    """Raise if a bounded device wait of ``paged_prefill`` or ``norm_rope`` ran out since the last check
    (clears it).  Synchronises the current stream."""
    _lib.check(_lib.load().smaq_exact_status(_stream()), "smaq_exact_status")


def exact_wait_limit(polls: Optional[int] = None) -> None:
    """Polls (4 us each) after which those waits give up, for later calls; None: the default, a second
    (smaq_exact_set_wait_limit).  Small limits are for testing that a wait that runs out is reported."""
    _lib.load().smaq_exact_set_wait_limit(-1 if polls is None else polls)


def selftest_wait_timeout(spin_limit: int = 1 << 12) -> int:
    """Run a kernel whose mbarrier wait can never complete with a ``spin_limit`` poll bound;
    returns the library status (``5`` = SMAQ_ERR_DEVICE when the timeout path works)."""
    return int(_lib.load().smaq_selftest_wait_timeout(spin_limit, _stream()))


# --------------------------------------------------------------------- decode-layout byte order
# (SMAQ_LAYOUT_DECODE, include/smaq_b200.h): same bits as the reference, permuted inside rows.
_VPERM = [4 * (k % 8) + k // 8 for k in range(32)]          # reference byte k lives at _VPERM[k]


def values_to_reference(data: torch.Tensor) -> torch.Tensor:
    """Decode-layout 2-bit value rows ``(..., 32)`` -> reference byte order."""
    return data[..., _VPERM]


def bvq_to_reference(idx: torch.Tensor) -> torch.Tensor:
    """Decode-layout block-VQ rows ``(..., 16)`` -> reference block order."""
    b = torch.arange(16, device=idx.device)
    pos = 2 * (4 * (b // 8) + b % 4) + (b // 4) % 2
    return idx[..., pos]


_SPERM = [16 * (k % 4) + k // 4 for k in range(64)]         # 3/4-bit scalar code byte k at _SPERM[k]


def scalar_codes_to_reference(codes: torch.Tensor) -> torch.Tensor:
    """Decode-layout 3/4-bit scalar key code rows ``(..., 64)`` -> reference byte order."""
    return codes[..., _SPERM]


def fp16_codebook(decoded_centroids: torch.Tensor) -> Optional[torch.Tensor]:
    """fp16 copy of a decoded codebook if it is exactly fp16-valued (enables the tensor-core
    decode kernel), else None."""
    c16 = decoded_centroids.to(torch.float16)
    return c16 if torch.equal(c16.to(decoded_centroids.dtype), decoded_centroids) else None

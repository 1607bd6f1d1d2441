"""Cross attention: queries over another sequence's keys, padded to a common length.

The second attention of an encoder-decoder layer. Every query row of batch entry ``b``
sees the first ``kv_lengths[b]`` keys (all of them without lengths); nothing is causal
and no mask is built: the kernels walk the tiles an entry has, forward (``gki_cross_fwd``)
and backward (``gki_cross_bwd``). Few query rows over long keys, a decoder's step among
them, run against slices of the keys that fill the card; in 16 bits a whole group of
heads shares each read of a key.

There is no CPU or eager fallback: a missing library raises ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DTYPE_CODE, _HEAD_DIMS, _aligned, _current_stream, _on_device, _refuse_tangents

# launch plans: (dtype, B, H, H_kv, n_q, n_kv, D) -> (slices, floats of the LSE rows, of
# the slices' states) of a forward, (parts of dK/dV, slices of dQ, floats of the row terms,
# of the parts' sums, of the slices') of a backward
_FWD_PLANS: dict = {}
_BWD_PLANS: dict = {}


def _planned(plans: dict, key: tuple, make) -> Tuple[int, ...]:
    plan = plans.get(key)
    if plan is None:
        if len(plans) >= 4096:
            plans.clear()
        plan = plans[key] = make(_lib.load(), *key)
    return plan


def _make_fwd_plan(lib, dtype, B, H, H_kv, n_q, n_kv, D) -> Tuple[int, int, int]:
    splits = int(lib.gki_cross_splits(dtype, B, H, H_kv, n_q, n_kv, D))
    states = int(lib.gki_stream_workspace_floats(B, H, n_q, D, splits))
    rows = B * H * n_q
    return splits, (rows + 63) & ~63 if states else rows, states     # the states 256-byte aligned


def _make_bwd_plan(lib, dtype, B, H, H_kv, n_q, n_kv, D) -> Tuple[int, ...]:
    slices = ctypes.c_int32()
    parts = int(lib.gki_cross_bwd_parts(dtype, B, H, H_kv, n_q, n_kv, D, ctypes.byref(slices)))
    tile = _lib.tile_sizes()["tile_n"]
    sums = B * H_kv * -(-n_kv // tile) * parts * 2 * tile * D if parts > 1 else 0
    dq_sums = B * H * n_q * D * slices.value if slices.value > 1 else 0
    return parts, slices.value, (2 * B * H * n_q + 63) & ~63, sums, dq_sums


def _check(q, k, v, kv_lengths, enable_gqa) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("Q/K/V must be 4-D [B, H, N, D] tensors")
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise ValueError("All inputs must live on a CUDA device")
    if q.device != k.device or q.device != v.device:
        raise ValueError("Q/K/V must live on one device")
    if k.shape != v.shape:
        raise ValueError("K and V must share shape")
    B, H, _, D = q.shape
    H_kv = k.shape[1]
    if k.shape[0] != B or k.shape[-1] != D or not (
            H_kv == H or (enable_gqa and H_kv > 0 and H % H_kv == 0)):
        raise ValueError("Q/K/V batch/head/dim mismatch")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in _DTYPE_CODE:
        raise ValueError(f"Q/K/V must share one dtype among float32/float16/bfloat16, got "
                         f"{q.dtype}/{k.dtype}/{v.dtype}")
    if D not in _HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {D}")
    if kv_lengths is not None:
        if kv_lengths.dtype not in (torch.int32, torch.int64) or kv_lengths.shape != (B,):
            raise ValueError(f"kv_lengths must be an int32 or int64 tensor [{B}], got {kv_lengths.dtype} "
                             f"{tuple(kv_lengths.shape)}")
        if kv_lengths.device != q.device:
            raise ValueError(f"kv_lengths must live on {q.device}")


def _forward(q, k, v, kv_lengths, scale, keep_lse=False):
    """(o, lse rows, key) of aligned inputs; key None: nothing to compute. The slices'
    states lie behind the rows, unless these are kept (``keep_lse``)."""
    B, H, n_q, D = q.shape
    n_kv = k.shape[2]
    o = torch.empty_like(q)
    if q.numel() == 0 or n_kv == 0:
        return o.zero_(), torch.zeros(B * H * n_q, dtype=torch.float32, device=q.device), None
    key = (_DTYPE_CODE[q.dtype], B, H, k.shape[1], n_q, n_kv, D)
    splits, rows, states = _planned(_FWD_PLANS, key, _make_fwd_plan)
    scratch = torch.empty(rows if keep_lse else rows + states, dtype=torch.float32, device=q.device)
    lse = scratch.data_ptr()
    ws = lse + 4 * rows if states else 0
    if keep_lse and states:
        work = torch.empty(states, dtype=torch.float32, device=q.device)
        ws = work.data_ptr()
    lib = _lib.load()
    with _on_device(q.device):
        rc = lib.gki_cross_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse, *key,
            0 if kv_lengths is None else kv_lengths.data_ptr(), scale, ws, splits,
            _current_stream(q.device))
    if rc:
        _lib.check(rc, "gki_cross_fwd")
    return o, scratch, key


class _CrossAttention(torch.autograd.Function):
    """Autograd bridge between PyTorch and the gfx950 kernels."""

    @staticmethod
    def forward(ctx, q, k, v, kv_lengths, scale):  # type: ignore[override]
        o, lse, key = _forward(q, k, v, kv_lengths, scale, keep_lse=True)
        ctx.save_for_backward(q, k, v, o, lse, kv_lengths)
        ctx.call = key, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):  # type: ignore[override]
        q, k, v, o, lse, kv_lengths = ctx.saved_tensors
        key, scale = ctx.call
        dq = torch.empty_like(q)
        keys = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]     # a frozen encoder needs neither
        dk, dv = (torch.empty_like(k), torch.empty_like(v)) if keys else (None, None)
        if key is None:
            return dq.zero_(), *((dk.zero_(), dv.zero_()) if keys else (None, None)), None, None
        do = _aligned(do if do.dtype == q.dtype else do.to(q.dtype))
        parts, slices, terms, sums, dq_sums = _planned(_BWD_PLANS, key, _make_bwd_plan)
        sums = sums if keys else 0
        scratch = torch.empty(terms + sums + dq_sums, dtype=torch.float32, device=q.device)
        delta = scratch.data_ptr()
        lib = _lib.load()
        with _on_device(q.device):
            rc = lib.gki_cross_bwd(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(), lse.data_ptr(),
                dq.data_ptr(), dk.data_ptr() if keys else 0, dv.data_ptr() if keys else 0, delta, *key,
                0 if kv_lengths is None else kv_lengths.data_ptr(), scale, parts,
                delta + 4 * terms if sums else 0, slices, delta + 4 * (terms + sums) if dq_sums else 0,
                _current_stream(q.device))
        if rc:
            _lib.check(rc, "gki_cross_bwd")
        return dq, dk, dv, None, None


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    kv_lengths: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    enable_gqa: bool = False,
) -> torch.Tensor:
    """Differentiable attention of ``q`` (``[B, H, N_Q, D]``) over another sequence's
    ``k``, ``v`` (``[B, H, N_KV, D]``), every visible key for every query.

    One dtype among fp32/fp16/bf16, ``D`` in {16, 32, 64, 128}, any ``N_Q`` and
    ``N_KV``. ``kv_lengths``: int32 or int64 ``[B]`` on the same device, the valid keys of
    each batch entry (the first ones; a value outside ``0 .. N_KV`` counts as the nearest
    of them, as the device is not asked); keys past them are not read and get zero
    gradients, an entry without keys gives zeros (and zero gradients).
    ``softmax_scale`` defaults to ``1/sqrt(D)``, any finite value is taken. Tensors that are
    not contiguous or not 16-byte aligned are copied by each call.
    ``enable_gqa``: K and V may have ``H_kv`` heads dividing Q's ``H``, as in
    ``block_sparse_attention``. Differentiable once, in reverse mode.
    """
    _check(q, k, v, kv_lengths, enable_gqa)
    scale = 1.0 / math.sqrt(q.shape[-1]) if softmax_scale is None else float(softmax_scale)
    if not math.isfinite(scale):
        raise ValueError(f"softmax_scale must be finite, got {scale}")
    if kv_lengths is not None:
        if kv_lengths.dtype != torch.int32:
            kv_lengths = kv_lengths.clamp(0, k.shape[2]).to(torch.int32)
        kv_lengths = kv_lengths.contiguous()
    _refuse_tangents(q, k, v)
    # copies of strided inputs are made here, where autograd sees them
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, kv_lengths, scale)
    return _forward(q, k, v, kv_lengths, scale)[0]

"""Tensors with a forward-mode tangent are refused, not answered without a tangent."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from gki import StreamingMaskSpec, block_sparse_attention, cross_attention, make_streaming_mask
from gki.ops import _refuse_tangents


def test_only_tangents_are_refused():
    x, y = torch.randn(3), torch.randn(3)
    _refuse_tangents(x, y)
    with forward_ad.dual_level():
        _refuse_tangents(x, y)
        dual = forward_ad.make_dual(x, torch.ones(3))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _refuse_tangents(y, dual)
        with torch.no_grad(), pytest.raises(NotImplementedError):      # tangents flow there too
            _refuse_tangents(y, dual)
        _refuse_tangents(forward_ad.unpack_dual(dual).primal)
    _refuse_tangents(x)


def _inputs(n_q):
    gen = torch.Generator(device="cuda").manual_seed(n_q)
    return [torch.randn((1, 2, n, 64), generator=gen, device="cuda") for n in (n_q, 128, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("n_q", [1, 128])
def test_cross_attention(which, n_q):
    qkv = _inputs(n_q)
    want = cross_attention(*qkv)
    with forward_ad.dual_level():
        assert torch.equal(cross_attention(*qkv), want)
        qkv[which] = forward_ad.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises(NotImplementedError):
            cross_attention(*qkv)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            cross_attention(*qkv)
        qkv[0].requires_grad_(True)
        with pytest.raises(NotImplementedError):
            cross_attention(*qkv)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("n_q", [1, 128])
def test_block_sparse_attention(which, n_q):
    qkv = _inputs(n_q)
    mask = make_streaming_mask(n_q, 128, StreamingMaskSpec(4, 64), 64, 64, device="cuda")
    call = dict(is_causal=True, sink_size=4, window_size=64)
    want = block_sparse_attention(*qkv, mask, **call)
    with forward_ad.dual_level():
        assert torch.equal(block_sparse_attention(*qkv, mask, **call), want)
        qkv[which] = forward_ad.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises(NotImplementedError):
            block_sparse_attention(*qkv, mask, **call)

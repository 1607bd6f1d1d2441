"""Cross attention's gradients where queries or incoming gradients hold infinities or NaN
(a loss scale that overflowed): keys past an entry's length still get zeros."""

from __future__ import annotations

import math

import pytest
import torch

from gki import _lib, cross_attention

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("parts", [None, 3])
def test_keys_past_the_length_get_zeros(dtype, D, parts, monkeypatch):
    from gki import cross

    if parts:
        def cut(*a):
            a[-1]._obj.value = 1
            return parts

        monkeypatch.setattr(cross, "_BWD_PLANS", {})
        monkeypatch.setattr(_lib.load(), "gki_cross_bwd_parts", cut)
    gen = torch.Generator(device=DEV).manual_seed(D)
    q, do = (torch.randn((4, 4, 150, D), generator=gen, device=DEV).to(dtype) for _ in range(2))
    k, v = (torch.randn((4, 2, 200, D), generator=gen, device=DEV).to(dtype) for _ in range(2))
    lengths = [200, 70, 1, 0]
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)

    def grads(q, do):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(cross_attention(*leaves, n, enable_gqa=True), leaves, do)

    clean = grads(q, do)
    bad_q, bad_do = q.clone(), do.clone()
    bad_q[:, 1, 7] = math.nan
    bad_do[:, 0, 3] = math.inf
    bad_do[:, 2, 149, 1] = math.nan
    for a, b in ((bad_q, do), (q, bad_do)):
        dq, dk, dv = grads(a, b)
        for i, m in enumerate(lengths):
            assert not dk[i, :, m:].any() and not dv[i, :, m:].any(), (i, m)
        assert not dk[0].isfinite().all()                      # the valid keys of such an entry show it
        # rows of dQ are those of their own query alone
        assert torch.equal(dq[:, 3], clean[0][:, 3])

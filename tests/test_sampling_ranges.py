"""Token sampling and largest log-probabilities on the CPU where logits over the
temperature are large, and refusals of types by their own code."""

import numpy as np
import pytest
import torch

import sampling_reference as reference
from test1_amd import _native
from test1_amd.sampling import sample_tokens, top_logps

SF_EDTYPE = 9003   # include/slidefsdp.h


@pytest.mark.parametrize("t", [1.0, 0.3, 1e-6, 1e-9, 1e-12, 1e-30, 1e30])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e20])
def test_finite_masks_and_low_temperatures(mask, t):
    g = torch.Generator().manual_seed(0)
    x = torch.full((3, 500), mask)
    x[0, 200:300] = torch.randn(100, generator=g) * 3
    x[1, 250:254] = torch.randn(4, generator=g)
    u = torch.rand(3, generator=g)
    top = top_logps(x, 20, temperature=t)
    for i in range(3):
        logps, ids = reference.top(x[i].double().numpy(), 20, t)
        with np.errstate(over="ignore"):   # -1e9 over 1e-30 is -infinity in fp32
            logps = logps.astype(np.float32)
        assert np.array_equal(top.ids[i].numpy(), ids) and np.allclose(top.logps[i].numpy(), logps, rtol=2e-7, atol=1e-7)
    for s in (dict(t=0.0), dict(t=t, k=20), dict(t=t, p=0.9), dict(t=t, m=0.1), dict(t=t)):
        out = sample_tokens(x, u, s["t"], s.get("k", 0), s.get("p", 1.0), s.get("m", 0.0))
        for i in range(3):
            word, logp = reference.draw(x[i].double().numpy(), float(u[i]), **s)
            assert int(out.ids[i]) == word and np.isclose(float(out.logps[i]), logp, rtol=2e-7, atol=1e-7)


def test_types_are_refused_by_their_code():
    hip, p = _native.hip(), 1 << 20   # never read
    assert hip.sf_top_logps(p, 7, 10, 2, 10, 3, 1.0, p, p, p, None) == SF_EDTYPE
    assert hip.sf_sample_tokens(p, 7, 10, 2, 10, p, 1.0, None, 0, None, 1.0, None, 0.0, None, p, p, p, None) == SF_EDTYPE
    tiles = lambda dtype: hip.sf_distill_tiles(p, 64, 300, p, 64, 2, 64, p, p, p, 4, 1.0, dtype, p, p, None, None, 0, 0, None)  # noqa: E731
    assert tiles(_native.SF_DTYPE_F32) == tiles(7) == SF_EDTYPE

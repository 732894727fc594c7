"""Drawn tokens where the weights' last digits decide: long rows of nearly equal logits far below the largest, under temperatures at which they count."""
import numpy as np
import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.9999), dict(min_p=1e-7)])
@pytest.mark.parametrize("top", [100.0, -100.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_logits_near_zero_under_a_large_one(dtype, top, settings):
    """One logit of 100, half of the others 0, half a little less than 2^-18: their differences from the largest are the same in 24 bits, their weights are
    not, by 2^-21 of themselves.  Or that little one the largest, and all others -100.

    Numbers u are taken where the token in 64 bits lies more than 0.06 of an element from the next one.  The kernel's weights may shift it by 2^20 times what a
    weight is off: 2^-31 of itself and half a unit of 2^-42 of the largest, which is 2^-24.25 of a weight of e^-13: 0.0005 + 0.0526 elements."""
    n, drop, small = 1 << 20, 13.0, 2.0 ** -18 * (1 - 2.0 ** -6)
    x = torch.zeros(n, dtype=torch.float64)
    x[n // 2:] = small
    x[0] = 100.0
    if top < 0:
        x = torch.full((n,), -100.0, dtype=torch.float64)
        x[0] = small
    x = x.to(dtype)
    t = np.float32(100.0 / drop)
    exact = x.double().numpy()
    w = np.exp((exact - exact.max()) / float(t))
    upto = np.cumsum(w)
    g = np.random.default_rng(3)
    u = g.random(4000, dtype=np.float32)
    goal = u.astype(np.float64) * upto[-1]
    if "top_p" in settings:         # of equals the first are kept: find the end of what is kept
        p = float(np.float32(settings["top_p"]))
        order = np.argsort(-exact, kind="stable")
        before = np.cumsum(w[order]) - w[order]
        kept = np.zeros_like(w)
        some = order[before < p * w.sum()]
        kept[some] = w[some]
        upto = np.cumsum(kept)
        goal = u.astype(np.float64) * upto[-1]
    at = np.searchsorted(upto, goal, side="right")
    into = (upto[at] - goal) / w[at]
    far = (at > 0) & (into > 0.06) & (into < 0.94)
    u, at = u[far][:512], at[far][:512]
    assert len(u) == 512
    got = ops.sample_rows(x.to(DEV).expand(len(u), n), torch.from_numpy(u).to(DEV), temperature=float(t), **settings)
    assert got.tolist() == at.tolist()

"""The learner-side operators at the edges of their definitions: infinite
margins and divergences, nearly sure decisions, offsets that do not ascend,
long read-ons behind a part of a window, saved-tensor hooks and forward-mode
derivatives.  Tolerances as in test_gpu_policy.py: H = 2^-24 is half a step of
a 32-bit value of 1."""
import math

import numpy as np
import pytest
import torch

from open_spiel_coup_amd import policy
from tests import policy_oracle as oracle
from tests import test_gpu_policy as base

pytestmark = pytest.mark.gpu

H, DEV = base.H, base.DEV
_np, _close = base._np, base._close


# ------------------------------------------------------------ infinite margins
@pytest.mark.parametrize("pairs,each", [(3, 4), (600, 30), (3, 400)], ids=["short-few", "short", "long"])
@pytest.mark.parametrize("eps", [0.0, 0.1])
def test_a_margin_of_plus_infinity_costs_nothing(pairs, each, eps):
    """A rejected decision of probability 0 makes its pair's margin +inf: -log sigmoid(inf) = 0, and with smoothing
    -eps log sigmoid(-inf) = inf; a chosen one makes the cost inf either way.  The other pairs lie at a margin of 0 and
    cost log 2; a sure pair's gradient is eps beta / pairs ([b = a] - p_b) in the chosen rows."""
    n = pairs * each
    x = torch.zeros(n, 3)
    mask, actions = torch.full((n,), 7, dtype=torch.int32), torch.zeros(n, dtype=torch.int8)
    off = torch.tensor([k * each // 2 for k in range(2 * pairs + 1)], device=DEV)
    x[each // 2] = torch.tensor([-math.inf, 0.0, 0.0])  # pair 0's first rejected row
    args = (actions.to(DEV), mask.to(DEV), off)
    got = policy.preference_loss_and_grad(x.to(DEV), *args, beta=0.25, label_smoothing=eps)
    assert float(got.rewards[1]) == -math.inf and bool(torch.isfinite(got.rewards[2:]).all())
    if eps:
        assert float(got.loss) == math.inf
    else:
        _close(float(got.loss), (pairs - 1) * math.log(2) / pairs, 16 * H, "loss")
    c = eps * 0.25 / pairs
    want = np.tile(c * np.array([2 / 3, -1 / 3, -1 / 3]), (each // 2, 1))
    _close(_np(got.grad[:each // 2]), want, 16 * H * c, "grad of the chosen rows")
    assert torch.isfinite(got.grad).all()
    y = x.clone()
    y[0], y[each // 2] = x[each // 2], x[0]
    assert float(policy.preference_loss(y.to(DEV), *args, beta=0.25, label_smoothing=eps).loss) == math.inf

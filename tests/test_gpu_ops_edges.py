"""What the operators say about inputs at their edges, each against values worked out here."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import gpu_util as gu
from vllm_expert_cache import ops

pytestmark = pytest.mark.gpu

DEV = gu.DEV
INF, NAN = math.inf, math.nan


# ---- routing ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("none", [-INF, NAN])
@pytest.mark.parametrize("renormalize", [True, False])
def test_a_bias_that_excludes_an_expert_leaves_the_softmax_alone(dtype, none, renormalize):
    """Experts 0 and 65 are excluded, by a bias of -infinity or NaN: their logits still count in
    the softmax of the others."""
    E, k = 70, 5
    rows = torch.zeros((4, E))
    rows[0, 0], rows[0, 3], rows[0, 65] = 3.0, 2.0, 1.0
    rows[1] = torch.arange(E) / 16.0
    rows[1, 0] = 6.0                      # most of the row's weight
    rows[2, 1:] = -INF                    # nothing but an excluded one
    rows[3, 10:60] = NAN                  # no candidates and no part of the softmax
    rows = rows.to(dtype)
    bias = torch.zeros(E)
    bias[0], bias[65], bias[7] = none, none, 0.25
    w, ids = ops.route(rows.to(DEV), k, bias=bias.to(DEV), renormalize=renormalize)
    x = rows.double().numpy()
    e = np.where(np.isnan(x), 0.0, np.exp(np.where(np.isnan(x), 0, x) - np.nanmax(x, 1)[:, None]))
    score = e / e.sum(1, keepdims=True)
    for t in range(4):
        may = [i for i in range(E) if i not in (0, 65) and x[t, i] > -INF]
        chosen = sorted(may, key=lambda i: (-(score[t, i] + float(bias[i])), i))[:k]
        want = score[t, chosen]
        if renormalize and len(chosen):
            want = want / want.sum()
        assert ids[t].tolist() == chosen + [-1] * (k - len(chosen)), t
        # made in 64 bits and rounded once
        np.testing.assert_allclose(w[t].cpu().numpy(), list(want) + [0.0] * (k - len(chosen)),
                                   rtol=1.01 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("renormalize", [True, False])
def test_all_of_the_softmax_with_an_excluded_expert(renormalize):
    """An infinite logit under a bias of -infinity: the others' scores are 0, so they come in order
    of their biases, and weights of 0 are not divided by their sum."""
    logits = torch.tensor([[1.0, INF, 2.0, 0.5], [1.0, 2000.0, 2.0, 0.5]], device=DEV)
    bias = torch.tensor([0.0, -INF, 0.0, 0.5], device=DEV)
    w, ids = ops.route(logits, 3, bias=bias, renormalize=renormalize)
    assert ids.tolist() == [[3, 0, 2]] * 2      # (exp(-1998) is 0 in 64 bits)
    assert not w.any()

"""A NaN among the logits of zmoe.functional.route, by form: whose row it is, and who is taken there."""

import math

import pytest
import torch

from helpers import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups", [1, 4])
def test_a_nan(groups, hip_device):
    from zmoe.functional import route

    z = torch.randn(6, 32, generator=gen(3)).to(hip_device)
    z[1, 9] = math.nan
    bias = torch.zeros(32, device=hip_device)
    for score in ("sigmoid", "softmax"):
        for b in (None, bias):
            idx, w = route(z, 4, b, score, groups, 2 if groups > 1 else 1)
            clean = route(z.nan_to_num(0.0), 4, b, score, groups, 2 if groups > 1 else 1)
            # ranked by logits or by sigmoids its expert is the first; a softmax of the row is NaN throughout: all equal
            first = 0 if score == "softmax" and b is not None else 9
            assert idx[1, 0] == first and (first or idx[1].tolist() == [0, 1, 2, 3])
            assert torch.isnan(w[1]).all()
            rows = [0, 2, 3, 4, 5]
            assert torch.equal(idx[rows], clean[0][rows]) and torch.equal(w[rows], clean[1][rows])

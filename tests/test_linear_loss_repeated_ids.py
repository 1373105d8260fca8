"""Distillation where a token's entries name one id more than once and some of these are left out (a logit of -inf):
the id's place in the gradient is the product's probability less the shares of those that are not.

Tolerances are those of test_linear_loss.py.
"""

import pytest
import torch

from test_linear_loss import DTYPES, WAYS, inputs, teacher, verify_kd


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [-24.0, 0.0, 24.0])
@pytest.mark.parametrize("t,v", WAYS)
def test_entries_left_out_beside_others_of_their_id(dtype, shift, t, v):
    """Before and behind the entry that has a share, near it and more than 64 entries away; all logits near `shift`,
    the student sure of some of the ids."""
    h, w, _, g = inputs(dtype, t, v, 96)
    ids, tl = teacher(t, v, 70, g)
    inf = float("inf")
    for i in range(t):
        way = i % 6
        if way == 0:
            ids[i, 2], tl[i, 2], tl[i, 5] = ids[i, 5], -inf, 6
        elif way == 1:
            ids[i, 5], tl[i, 2], tl[i, 5] = ids[i, 2], 6, -inf
        elif way == 2:
            ids[i, 1], tl[i, 1], tl[i, 69] = ids[i, 69], -inf, 6
        elif way == 3:
            ids[i, 0] = ids[i, 3] = ids[i, 68]
            tl[i, 0], tl[i, 3], tl[i, 68] = -inf, 5, 5.5
        elif way == 4:  # padding in front that names the first id
            ids[i, :5] = 0
            tl[i, :4], tl[i, 4] = -inf, 6
        else:
            ids[i, 1] = ids[i, 66]
            tl[i, 1] = tl[i, 66] = -inf
    one = ids[torch.arange(t), torch.tensor([5, 2, 69, 68, 4, 7])[torch.arange(t) % 6]]
    h, w = h.float(), w.float()
    h = h + (12 * torch.rand(t, 1, generator=g)) * w[one]
    w[:, 0], h[:, 0] = 1, shift
    verify_kd(dtype, h.to(DTYPES[dtype]), w.to(DTYPES[dtype]), ids, tl, 1.0, "none", g)

"""lm_loss (models/train_ops.py) takes a whole number as ignore_index: 0.5 would leave out id 0.
Without a GPU."""
import numpy as np
import pytest
import torch

from smsgate_amd.models import train_ops


@pytest.mark.parametrize("bad", [0.5, -100.0, None, "x"])
def test_other_values_are_refused(bad):
    h = torch.zeros(3, 16).half()
    with pytest.raises(TypeError, match="ignore_index"):
        train_ops.lm_loss(h, torch.zeros(4, 16).half(), torch.zeros(3, dtype=torch.long), ignore_index=bad)


@pytest.mark.parametrize("good", [-1, np.int64(7), np.int32(-100)])
def test_whole_numbers_pass(good):
    h = torch.zeros(3, 16).half()
    with pytest.raises(ValueError, match="same GPU"):  # the check behind
        train_ops.lm_loss(h, torch.zeros(4, 16).half(), torch.zeros(3, dtype=torch.long), ignore_index=good)

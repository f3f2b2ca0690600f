"""The model path's embedding lookup and its ids."""

import pytest
import torch

from testt_amd import model

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_ids_outside_the_table_raise():
    """A real token's id outside the table raises, as torch's embedding does; padding may hold any."""
    weights = model.ModelWeights(
        embed=torch.randn(50, 64, device=DEV).half(), layers=[],
        final_norm=torch.ones(64, device=DEV), inv_freq=model.default_inv_freq(32, 1e4, DEV))
    ids = torch.arange(12, device=DEV).view(2, 6)
    amask = torch.ones_like(ids)
    amask[1, 4:] = 0
    ids[1, 4:] = torch.tensor([50, -100], device=DEV)
    labels = torch.where(amask.bool(), ids, -100)
    loss, _ = model.forward_weights(weights, ids, amask, labels)
    assert loss.isfinite()
    for bad in (50, -1, 1 << 40):
        wrong = ids.clone()
        wrong[0, 3] = bad
        with pytest.raises(IndexError, match="ids"):
            model.forward_weights(weights, wrong, amask, labels)

"""Farthest point sampling at the batches from which a call takes a wave per frustum instead of a workgroup: the same picks
on both sides."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,batch", [(2048, 1792), (1025, 1792), (1024, 1536), (300, 1536)])
def test_both_sides_of_the_choice_pick_the_same(device, monkeypatch, n, batch):
    from fpn.tf_ops.tf_sampling import farthest_point_sample
    g = torch.Generator().manual_seed(n)
    x = torch.rand((batch, n, 3), generator=g).to(device)
    monkeypatch.delenv("FPN_FPS", raising=False)
    picks = {rows: farthest_point_sample(24, x[:rows].contiguous()).cpu().numpy() for rows in (1024, batch - 1, batch)}
    monkeypatch.setenv("FPN_FPS", "block")
    want = farthest_point_sample(24, x).cpu().numpy()
    for rows, got in picks.items():
        np.testing.assert_array_equal(got, want[:rows])

"""The token policy takes whole batches of observations: one with fewer columns would leave the last batch's in their place."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.token_policy import TokenPolicy  # noqa: E402


@pytest.mark.parametrize("shape", [(16, 11), (16, 13), (16, 16), (1, 11), (15, 12), (12,), (1, 16, 12)])
def test_other_shapes_are_refused(shape):
    policy = TokenPolicy(12, 20, 16, hidden=32, top=4)
    good = torch.randn(16, 12, device="cuda")
    policy.load_observations(good)
    held = policy.obs.clone()
    values, indices = torch.zeros(16, 4, device="cuda"), torch.arange(4, device="cuda").expand(16, 4).contiguous()
    for call in (policy.load_observations, lambda o: policy.act(o, torch.rand(16, device="cuda")),
                 lambda o: policy.distill_update(o, values, indices)):
        with pytest.raises(ValueError, match="observations must be"):
            call(torch.ones(shape, device="cuda"))
    assert torch.equal(policy.obs, held) and torch.equal(policy.obs[:, :12], good.half())
    policy.load_observations(good[3:4])
    assert torch.equal(policy.obs[:, :12], good[3:4].half().expand(16, 12))

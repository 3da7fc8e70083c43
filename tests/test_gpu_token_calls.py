"""Calls of the token operators on the GPU that a program around them makes possible."""
import pytest
import torch

import token_oracle as oracle
from token_oracle import assert_within
from pcd_reg_hregnet_amd import tokens

pytestmark = pytest.mark.gpu
F, H = torch.float32, torch.bfloat16


def normal(seed, *shape, dtype=F):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g, dtype=F).to(dtype)


@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
def test_default_type_of_the_program(dtype):
    """torch's default type has no influence: the same bits"""
    q, k, v, do = (normal(i, 2, 70, 2, 32, dtype=dtype) for i in range(4))
    f, w = normal(5, 70, 264, dtype=dtype), normal(6, 264, dtype=dtype)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, f, w)]
        out = tokens.attention(*leaves[:3], causal=True)
        y, h = tokens.gated_residual_norm(leaves[3], leaves[3], pre_norm="layer", pre_weight=leaves[4])
        return [out.detach(), h.detach(), *torch.autograd.grad([out, h], leaves, [do, f])]

    want = once()
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = once()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

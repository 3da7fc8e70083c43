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


@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("shape", [(2, 1, 129, 4, 2, 64), (2, 1, 2000, 4, 2, 64), (2, 300, 150, 4, 4, 64)],
                         ids=["one run", "eight runs", "row kernel"])
def test_a_query_that_is_nan_gives_nan(shape, train, dtype):
    """a row whose scores are NaN is NaN, not the 0 of a row without keys, however the keys are divided;
    the other rows keep their bits"""
    B, Nq, Nk, heads, key_heads, D = shape
    q, k, v = (normal(i, B, n, h, D, dtype=dtype) for i, (n, h) in enumerate(((Nq, heads), (Nk, key_heads), (Nk, key_heads))))
    bad = q.clone()
    bad[1, Nq - 1, 1] = float("nan")
    with torch.set_grad_enabled(train):
        clean, got = (tokens.attention(t.clone().requires_grad_(train), k, v, causal=True) for t in (q, bad))
    assert torch.isnan(got[1, Nq - 1, 1]).all()
    same = torch.ones(B, Nq, heads, dtype=torch.bool, device="cuda")
    same[1, Nq - 1, 1] = False
    assert torch.equal(got[same], clean[same]) and torch.isfinite(clean).all()
    one = v.clone()  # and a single value among many that is NaN reaches every row that sees it
    one[0, Nk // 2] = float("nan")
    with torch.no_grad():
        got = tokens.attention(q, k, one)
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all()

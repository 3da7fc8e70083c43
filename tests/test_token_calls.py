"""What the token operators hand to their C entries and how they answer calls around them, without a GPU:
the checks for a GPU tensor and the launches are replaced, everything before and after them runs."""
import pytest
import torch

from pcd_reg_hregnet_amd import tokens


@pytest.fixture
def launches(monkeypatch):
    """names of the entries that would have run"""
    names = []
    monkeypatch.setattr(tokens, "_check_tensor", lambda *a, **k: None)
    monkeypatch.setattr(tokens, "_launch", lambda device, name, *a: names.append(name))
    return names


def normal(*shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(dtype)


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64])
def default_dtype(request):
    old = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(old)


def test_statistics_are_float32_whatever_the_default_type(launches, default_dtype):
    """the kernels write float32 statistics: a buffer of torch's default type would be too short"""
    x = normal(2, 4, 2, 16, dtype=torch.float32)
    for t in (x, x.bfloat16()):
        lse = tokens._attn_forward((0.25, False, False, None), t, t, t, None, None, None, None, True)[4]
        assert lse.dtype == torch.float32 and lse.shape == (2, 2, 2, 4)
        leaf = t.detach().requires_grad_(True)
        _, h = tokens.gated_residual_norm(leaf, t)
        stats = [s for s in h.grad_fn.saved_tensors if s is not None and s.shape == (16, 4)]
        assert [s.dtype for s in stats] == [torch.float32]
    assert launches == ["hreg_tok_attn_fwd", "hreg_tok_block_fwd"] * 2


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_raise(launches, grad):
    """no operator returns a result that has lost its tangent"""
    x, table = normal(1, 5, 2, 16), normal(8, 2)
    kw = dict(bias=table, buckets=tokens.Buckets(8, 6))
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        bias = torch.autograd.forward_ad.make_dual(table, torch.ones_like(table))
        for call in (lambda: tokens.attention(dual, x, x), lambda: tokens.attention(x, dual, x),
                     lambda: tokens.attention(x, x, dual), lambda: tokens.attention(x, x, x, **kw | dict(bias=bias)),
                     lambda: tokens.dropout(dual, 0.5, 1), lambda: tokens.gated_residual_norm(dual, None),
                     lambda: tokens.gated_residual_norm(x, dual, p=0.1, seed=1)):
            with pytest.raises(NotImplementedError, match="forward mode"):
                call()
        # tensors without a tangent are welcome there
        assert not tokens.attention(x, x, x, **kw).requires_grad
    assert not tokens.attention(x, x, x).requires_grad


@pytest.mark.parametrize("scale", [1e300, -1e300, 3e38, float("inf"), float("nan")])
def test_scales_that_float32_does_not_hold_are_refused(launches, scale):
    x = normal(1, 5, 2, 16)
    with pytest.raises(ValueError, match="scale"):
        tokens.attention(x, x, x, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        tokens.gated_residual_norm(x, x, scale=scale)
    with pytest.raises(ValueError, match="eps"):
        tokens.gated_residual_norm(x, x, eps=scale)
    tokens.attention(x, x, x, scale=1e38)
    assert launches == ["hreg_tok_attn_fwd"]

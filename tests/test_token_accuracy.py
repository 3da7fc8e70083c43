"""The float32 tolerances of token_accuracy.py refuse what they are there to refuse: operands that lost their
last eight bits, and a product that is rounded one way.  Both are planted in the 64-bit forms."""
import pytest
import torch

import token_oracle as oracle
from token_accuracy import SHAPES, U, error, tolerance, tolerance_table


def cut(t, bits):
    """t's leading significant bits"""
    mask = ~((1 << (24 - bits)) - 1)
    return (t.view(torch.int32) & mask).view(torch.float32)


@pytest.mark.parametrize("cfg", SHAPES, ids=lambda c: "-".join(map(str, c[:7])))
def test_two_pieces_of_three_are_not_enough(cfg):
    B, Nq, Nk, H, Hk, D, causal, spec = cfg
    g = torch.Generator().manual_seed(5)
    t = [torch.randn(B, n, h, D, generator=g) for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H))]
    bias = None if spec is None else torch.randn(spec[0], H, generator=g)
    forms = [oracle.attention(q, k, v, do=do, causal=causal, bias=bias, spec=spec)
             for q, k, v, do in (t, [cut(x, 16) for x in t])]
    for n in forms[0]:
        assert error(forms[1][n][0], forms[0][n][0]) > 2 * tolerance(D), n


def test_a_product_rounded_one_way_shows_in_the_table():
    """do . v too low by 2^-26 of its magnitudes: single ds do not feel it, the sums over 10^6 pairs do"""
    g = torch.Generator().manual_seed(6)
    B, H, N, D, num, far = 4, 8, 517, 40, 32, 128
    q, k, v, do = (torch.randn(B * H, N, D, generator=g, dtype=torch.float64) for _ in range(4))
    lut = torch.tensor([oracle.bucket(num, far, True, o) for o in range(-N, N)])
    rel = torch.arange(N)[None] - torch.arange(N)[:, None] + N
    p = torch.softmax(q @ k.transpose(1, 2).contiguous() / D ** 0.5, -1)
    dp = do @ v.transpose(1, 2).contiguous()
    low = dp - 2.0 ** -26 * (do.abs() @ v.abs().transpose(1, 2).contiguous())
    delta = (p * dp).sum(-1, keepdim=True)
    ds, ds_low = p * (dp - delta), p * (low - delta)
    table = [torch.zeros(num, H, dtype=torch.float64).index_add_(0, lut[rel].reshape(-1), x.view(B, H, N * N).sum(0).T)
             for x in (ds, ds_low)]
    assert error(ds_low, ds) < 8 * U
    assert error(table[1], table[0]) > tolerance_table(D)

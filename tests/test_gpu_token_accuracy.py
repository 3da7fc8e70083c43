"""float32 attention comes as near to its 64-bit form as float32 products do: token_accuracy.py counts how near"""
import pytest
import torch

import token_oracle as oracle
from token_accuracy import SHAPES, error, tolerance, tolerance_table
from pcd_reg_hregnet_amd import tokens

pytestmark = pytest.mark.gpu


def own(q, k, v, do, bias, spec, causal):
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v) + (() if bias is None else (bias,))]
    more = {} if bias is None else dict(bias=leaves[3], buckets=tokens.Buckets(*spec))
    out = tokens.attention(*leaves[:3], causal=causal, **more)
    return dict(zip(("out", "dq", "dk", "dv", "dbias"), (out.detach(), *torch.autograd.grad(out, leaves, do))))


@pytest.mark.parametrize("cfg", SHAPES, ids=lambda c: "-".join(map(str, c[:7])))
def test_attention_float32(cfg):
    B, Nq, Nk, H, Hk, D, causal, spec = cfg
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v, do = (torch.randn(B, n, h, D, device="cuda", generator=g) for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H)))
    bias = None if spec is None else torch.randn(spec[0], H, device="cuda", generator=g)
    want = oracle.attention(q, k, v, do=do, causal=causal, bias=bias, spec=spec)
    got = own(q, k, v, do, bias, spec, causal)
    assert set(got) == set(want)
    off = {n: error(got[n], want[n][0]) for n in got}
    assert all(e <= tolerance(D) for e in off.values()), (off, tolerance(D))


def test_table_gradient_float32():
    """4 x 517 x 8 heads: about 10^6 pairs a head"""
    B, H, N, D, spec = 4, 8, 517, 40, (32, 128, True)
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v, do = (torch.randn(B, N, H, D, device="cuda", generator=g) for _ in range(4))
    bias = torch.randn(spec[0], H, device="cuda", generator=g)
    got = own(q, k, v, do, bias, spec, False)
    Q, K, V, dO = (t.double().transpose(1, 2).contiguous() for t in (q, k, v, do))
    lut = torch.tensor([oracle.bucket(*spec, o) for o in range(-N, N)], device="cuda")
    i = torch.arange(N, device="cuda")
    at = lut[i[None] - i[:, None] + N]
    p = torch.softmax(Q @ K.transpose(2, 3).contiguous() / D ** 0.5 + bias.double()[at].permute(2, 0, 1), -1)
    dp = dO @ V.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    want = torch.zeros(spec[0], H, dtype=torch.float64, device="cuda")
    want.index_add_(0, at.reshape(-1), ds.sum(0).reshape(H, -1).T.contiguous())
    assert error(got["dbias"], want) <= tolerance_table(D)
    for n, value in (("out", p @ V), ("dq", ds @ K / D ** 0.5), ("dk", ds.transpose(2, 3).contiguous() @ Q / D ** 0.5),
                     ("dv", p.transpose(2, 3).contiguous() @ dO)):
        assert error(got[n], value.transpose(1, 2)) <= tolerance(D), n

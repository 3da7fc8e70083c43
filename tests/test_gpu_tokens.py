"""Token operators on the GPU against their 64-bit forms: every bound is counted in token_oracle.py."""
import pytest
import torch

import token_oracle as oracle
from token_oracle import assert_within
from pcd_reg_hregnet_amd import tokens

pytestmark = pytest.mark.gpu
F, H = torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def leaf(t):
    return t.detach().clone().requires_grad_(True)


# ------------------------------------------------------------------------------ attention

ATTN = [  # B, Nq, Nk, heads, key heads, width, causal, key lengths, query lengths, mask, buckets (num, far, both)
    (1, 1, 1, 1, 1, 8, False, None, None, False, None),
    (2, 37, 37, 4, 2, 64, True, None, None, False, None),
    (2, 1, 200, 4, 1, 128, True, [200, 77], None, False, None),
    (1, 130, 257, 2, 2, 40, False, None, None, False, None),
    (3, 65, 33, 6, 2, 32, True, [33, 20, 1], None, False, None),
    (4, 40, 70, 2, 1, 24, False, [0, 1, 70, 500], [40, 13, 0, 1], False, None),
    (4, 40, 70, 2, 1, 72, True, [0, 1, 70, 65], [40, 13, 7, -3], True, None),
    (2, 300, 129, 2, 2, 128, False, None, None, True, (16, 20, True)),
    (1, 161, 161, 3, 3, 64, True, None, None, False, (32, 128, False)),
    (2, 50, 300, 4, 2, 16, True, [300, 211], None, False, (8, 5, False)),
    (2, 300, 50, 2, 2, 80, False, [50, 31], [300, 17], False, (4, 2, True)),
    (1, 400, 400, 1, 1, 32, True, None, None, True, (32, 100, True)),
    (1, 2, 700, 2, 1, 48, False, None, None, False, (128, 1024, True)),
    (2, 5, 1030, 8, 2, 128, True, [1030, 3], None, False, (32, 128, False)),
    (8, 40, 1000, 32, 8, 16, True, None, None, False, None),  # a group's heads in two parts
    (1, 600, 600, 6, 1, 8, False, None, [577], True, (8, 30, True)),  # in six, with a bias
    (1, 60, 5000, 8, 1, 32, True, [4801], None, True, (32, 128, False)),  # many rows a key head, few tiles
    (2, 1, 333, 40, 1, 64, True, [333, 1], None, False, (16, 40, False)),  # more heads than a tile has rows
    (1, 2, 100, 64, 2, 32, True, None, None, False, (32, 1024, True)),  # tables too large for a group
    (2, 70, 150, 4, 2, 96, True, [150, 33], None, False, None),
    (1, 140, 90, 2, 2, 56, False, None, None, True, (16, 20, True)),
    (1, 75, 75, 4, 1, 104, True, None, None, False, None),
    (2, 3, 400, 8, 2, 88, True, [400, 129], None, False, (32, 128, False)),
    (20, 130, 140, 8, 2, 48, True, None, None, False, None),  # waves with rows of their own
    (20, 130, 140, 8, 2, 88, False, None, None, True, (16, 20, True)),
]


def attn_case(seed, cfg, dtype, bias_dtype=None):
    B, Nq, Nk, Hq, Hk, D, causal, kl, ql, holes, spec = cfg
    g = gen(seed)
    s = {n: normal(g, *shape, dtype=dtype) for n, shape in (("q", (B, Nq, Hq, D)), ("k", (B, Nk, Hk, D)),
                                                            ("v", (B, Nk, Hk, D)), ("do", (B, Nq, Hq, D)))}
    kw = dict(causal=causal, k_lengths=None if kl is None else torch.tensor(kl, device="cuda", dtype=torch.int32),
              q_lengths=None if ql is None else torch.tensor(ql, device="cuda"), key_mask=None)
    if holes:
        kw["key_mask"] = torch.rand(B, Nk, device="cuda", generator=g) < 0.6
        kw["key_mask"][0] = False  # a batch entry without any key
        if B == 1:
            kw["key_mask"][0, Nk // 2:] = True
    bias = None if spec is None else normal(g, spec[0], Hq, dtype=bias_dtype or dtype)
    return s, kw, bias, spec


def run_attn(s, kw, bias, spec):
    leaves = {n: leaf(s[n]) for n in ("q", "k", "v")}
    more = {}
    if bias is not None:
        leaves["bias"] = leaf(bias)
        more = dict(bias=leaves["bias"], buckets=tokens.Buckets(*spec))
    out = tokens.attention(leaves["q"], leaves["k"], leaves["v"], **kw, **more)
    grads = torch.autograd.grad(out, list(leaves.values()), s["do"])
    return {"out": out.detach(), **{"d" + n: t for n, t in zip(leaves, grads)}}


def check_attn(got, s, kw, bias, spec, what=""):
    want = oracle.attention(s["q"], s["k"], s["v"], do=s["do"], bias=bias, spec=spec, **kw)
    for n in want:
        assert_within(got[n], want[n], f"{what} {n}")


@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
@pytest.mark.parametrize("cfg", ATTN, ids=lambda c: "-".join(map(str, c[:7])))
def test_attention(cfg, dtype):
    case = attn_case(11, cfg, dtype)
    got = run_attn(*case)
    check_attn(got, *case)
    with torch.no_grad():  # the form without a backward pass
        s, kw, bias, spec = case
        more = {} if bias is None else dict(bias=bias, buckets=tokens.Buckets(*spec))
        out = tokens.attention(s["q"], s["k"], s["v"], **kw, **more)
    assert_within(out, oracle.attention(s["q"], s["k"], s["v"], bias=bias, spec=spec, **kw)["out"], "no grad")


def test_attention_scale_and_start():
    """a scale of its own (negative too), queries at the start of their keys although causal, and at
    the end although not"""
    for scale, causal, end in ((-0.4, True, False), (0.0, False, True), (0.7, False, True)):
        s, kw, bias, spec = attn_case(5, (2, 40, 90, 2, 1, 32, causal, [90, 64], None, False, (8, 9, True)), F)
        kw |= dict(scale=scale, align_end=end)
        check_attn(run_attn(s, kw, bias, spec), s, kw, bias, spec, f"{scale}")


def test_attention_float32_table_with_bf16_rows():
    case = attn_case(7, ATTN[8], H, bias_dtype=F)
    got = run_attn(*case)
    assert got["dbias"].dtype == F
    check_attn(got, *case)


@pytest.mark.parametrize("Nq", [237, 3])
def test_attention_few_keys_bias_gradient(Nq):
    """bf16 rows, nine keys, a float32 table: p in 16 bits and out with its remainder leave 2^-15 of the
    terms of D = do . o, which the sums over rows bring down to no less than a sixteenth (8 bits of p
    would be 2^-8 of them)"""
    case = attn_case(13, (3, Nq, 9, 32, 8, 72, False, None, None, False, (64, 64, True)), H, bias_dtype=F)
    got = run_attn(*case)
    check_attn(got, *case)
    s, kw, bias, spec = case
    want = oracle.attention(s["q"], s["k"], s["v"], do=s["do"], bias=bias, spec=spec, **kw)["dbias"][0]
    assert ((got["dbias"].double() - want).norm() / want.norm()).item() < 2 ** -11


def test_attention_strides():
    """a packed projection, head-major storage, rows that are not aligned, a batch that is broadcast"""
    B, N, h, D = 2, 45, 3, 32
    for dtype in (F, H):
        g = gen(3)
        packed = normal(g, B, N, 3, h, D, dtype=dtype)
        do = normal(g, B, N, h, D, dtype=dtype)
        x = leaf(packed)
        out = tokens.attention(x[:, :, 0], x[:, :, 1], x[:, :, 2])
        dx, = torch.autograd.grad(out, x, do.transpose(0, 1).contiguous().transpose(0, 1))
        s = {"q": packed[:, :, 0], "k": packed[:, :, 1], "v": packed[:, :, 2], "do": do}
        want = oracle.attention(s["q"], s["k"], s["v"], do=do)
        for n, got in (("out", out), ("dq", dx[:, :, 0]), ("dk", dx[:, :, 1]), ("dv", dx[:, :, 2])):
            assert_within(got, want[n], n)
        major = {n: t.transpose(1, 2).contiguous().transpose(1, 2) for n, t in s.items()}
        check_attn(run_attn_views(major), s, {}, None, None, "head-major")
        odd = {}
        for n, t in s.items():  # one element past an aligned address
            buf = torch.empty(t.numel() + 1, device="cuda", dtype=dtype)
            odd[n] = buf[1:].view(t.shape).copy_(t)
        check_attn(run_attn_views(odd), s, {}, None, None, "unaligned")
        one = leaf(s["k"][:1])
        out = tokens.attention(s["q"], one.expand(B, N, h, D), s["v"])
        dk, = torch.autograd.grad(out, one, do)
        want = oracle.attention(s["q"], s["k"][:1].expand(B, N, h, D), s["v"], do=do)
        v, b = want["dk"]  # autograd adds the two entries' gradients
        assert_within(dk, (v.sum(0, keepdim=True), b.sum(0, keepdim=True) + oracle.U[dtype] * v.sum(0, keepdim=True).abs()), "dk")


def run_attn_views(s):
    leaves = [s[n].detach().requires_grad_(True) for n in "qkv"]
    out = tokens.attention(*leaves)
    return {"out": out.detach(), **{"d" + n: t for n, t in zip("qkv", torch.autograd.grad(out, leaves, s["do"]))}}


@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
@pytest.mark.parametrize("train", [True, False])
def test_attention_hidden_values(dtype, train):
    """what stands in keys and queries that do not exist or are masked has no influence, NaN and
    infinities among it; their gradients are 0"""
    s, kw, bias, spec = attn_case(9, (2, 70, 140, 2, 2, 64, True, [100, 0], [70, 50], False, (8, 6, True)), dtype)
    kw["key_mask"] = torch.ones(2, 140, dtype=torch.bool, device="cuda")
    kw["key_mask"][0, 3:9] = False
    dirty = {n: t.clone() for n, t in s.items()}
    for n, bad in (("k", float("nan")), ("v", float("inf"))):
        dirty[n][0, 100:] = bad
        dirty[n][1] = bad
        dirty[n][0, 3:9] = -bad
    for n in ("q", "do"):
        dirty[n][1, 50:] = float("nan")
    if train:
        got, clean = run_attn(dirty, kw, bias, spec), run_attn(s, kw, bias, spec)
        check_attn(got, s, kw, bias, spec)
        for n in got:
            assert torch.equal(got[n], clean[n]), n
        assert not got["dk"][1].any() and not got["dv"][0, 3:9].any() and not got["dq"][1].any() and not got["out"][1].any()
    else:
        with torch.no_grad():
            more = dict(bias=bias, buckets=tokens.Buckets(*spec))
            a, b = (tokens.attention(t["q"], t["k"], t["v"], **kw, **more) for t in (dirty, s))
        assert torch.equal(a, b) and not torch.isnan(a).any()


@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B", [2, 90])  # waves that share rows, and not
def test_attention_queries_before_the_keys(dtype, B):
    """the last of more queries than keys: what stands in those before the first key reaches nothing"""
    s, kw, _, _ = attn_case(31, (B, 203, 33, 4, 2, 16, True, None, None, False, None), dtype)
    early = 203 - 33
    s["q"][:, :early] = s["do"][:, :early] = 0
    want = oracle.attention(s["q"], s["k"], s["v"], do=s["do"], **kw)
    s["q"][:, :early], s["do"][:, :early] = float("nan"), float("inf")
    got = run_attn(s, kw, None, None)
    for n in want:
        assert_within(got[n], want[n], n)


def test_attention_lowest_and_large_scores():
    """scores far apart and a bias of the type's lowest value: no overflow, no NaN"""
    for dtype in (F, H):
        s, kw, bias, spec = attn_case(2, (1, 33, 64, 1, 1, 16, False, None, None, False, (4, 3, True)), dtype)
        s["q"] *= 30
        bias[1] = torch.finfo(dtype).min
        got = run_attn(s, kw, bias, spec)
        assert all(torch.isfinite(t).all() for t in got.values())
        bias[1] = -1e4
        check_attn(run_attn(s, kw, bias, spec), s, kw, bias, spec)


def test_attention_far_strides():
    """a cache whose elements lie beyond 2^31 elements of its start"""
    N, step = 300, 8 << 20
    store = torch.empty(N * step, dtype=H, device="cuda")
    g = gen(1)
    k, v = (store.as_strided((1, N, 1, 64), (N * step, step, 64, 1), o) for o in (0, 4096))
    k.copy_(normal(g, 1, N, 1, 64, dtype=H)), v.copy_(normal(g, 1, N, 1, 64, dtype=H))
    q = normal(g, 1, 1, 2, 64, dtype=H)
    with torch.no_grad():
        assert_within(tokens.attention(q, k, v), oracle.attention(q, k, v)["out"])
    do = normal(g, 1, 1, 2, 64, dtype=H)
    check_attn(run_attn_views({"q": q, "k": k, "v": v, "do": do}), {"q": q, "k": k, "v": v, "do": do}, {}, None, None)


def test_attention_empty():
    for shape_q, shape_k in (((0, 3, 2, 16), (0, 5, 2, 16)), ((2, 0, 2, 16), (2, 5, 2, 16)), ((2, 3, 2, 16), (2, 0, 2, 16))):
        q, k, v = (torch.ones(s, device="cuda", requires_grad=True) for s in (shape_q, shape_k, shape_k))
        bias = torch.ones(8, 2, device="cuda", requires_grad=True)
        out = tokens.attention(q, k, v, bias=bias, buckets=tokens.Buckets(8, 6))
        assert out.shape == q.shape and not out.any()
        for t, d in zip((q, k, v, bias), torch.autograd.grad(out, (q, k, v, bias), torch.ones_like(out))):
            assert d.shape == t.shape and not d.any()


def test_attention_partial_gradients():
    """gradients that are not asked for are not made, the others are the same"""
    s, kw, bias, spec = attn_case(4, ATTN[7], F)
    full = run_attn(s, kw, bias, spec)
    for wanted in ("q", "k", "v", "b"):
        t = {n: s[n].clone().requires_grad_(n == wanted) for n in "qkv"}
        b = bias.clone().requires_grad_(wanted == "b")
        out = tokens.attention(t["q"], t["k"], t["v"], **kw, bias=b, buckets=tokens.Buckets(*spec))
        x = b if wanted == "b" else t[wanted]
        assert torch.equal(torch.autograd.grad(out, x, s["do"])[0], full["dbias" if wanted == "b" else "d" + wanted])


@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
def test_attention_same_bits_twice(dtype):
    case = attn_case(8, (2, 700, 700, 4, 2, 64, True, None, None, False, (32, 64, False)), dtype)
    a = run_attn(*case)
    for _ in range(2):
        b = run_attn(*case)
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_attention_gradient_against_differences():
    """the kernel's gradient against differences of the kernel's own forward pass in one random
    direction: they may differ by what both may be off, and by what the same difference of the
    64-bit form is off its gradient"""
    s, kw, bias, spec = attn_case(21, (2, 40, 70, 4, 2, 32, True, [70, 33], None, False, (16, 20, False)), F)
    got = run_attn(s, kw, bias, spec)
    want = oracle.attention(s["q"], s["k"], s["v"], do=s["do"], bias=bias, spec=spec, **kw)
    h = 2.0 ** -5
    for n in ("q", "k", "v", "bias"):
        base = bias if n == "bias" else s[n]
        d = torch.where(torch.rand(base.shape, device="cuda", generator=gen(1)) < 0.5, 1.0, -1.0) * 0.25

        def forms(sign):
            x = base + sign * h * d
            t = {**s, n: x} if n != "bias" else s
            b = x if n == "bias" else bias
            with torch.no_grad():
                out = tokens.attention(t["q"], t["k"], t["v"], **kw, bias=b, buckets=tokens.Buckets(*spec))
            o, e = oracle.attention(t["q"], t["k"], t["v"], bias=b, spec=spec, **kw)["out"]
            do = s["do"].double()
            return (out.double() * do).sum(), (o * do).sum(), (e * do.abs()).sum()

        up, down = forms(1), forms(-1)
        own, exact, err = (up[0] - down[0]) / (2 * h), (up[1] - down[1]) / (2 * h), (up[2] + down[2]) / (2 * h)
        v, b = want["d" + n]
        inner = (got["d" + n].double() * d).sum()
        tol = err + (exact - (v * d).sum()).abs() + (b * d.abs()).sum()
        assert (own - inner).abs() <= tol, (n, own.item(), inner.item(), tol.item())


def test_attention_refusals():
    q = torch.zeros(2, 4, 4, 16, device="cuda")
    k = torch.zeros(2, 6, 2, 16, device="cuda")
    bias, buckets = torch.zeros(8, 4, device="cuda"), tokens.Buckets(8, 6)
    bad = [
        (dict(q=q[0]), "must be"), (dict(q=q.half(), k=k.half(), v=k.half()), "not supported"),
        (dict(k=k.bfloat16()), "type"), (dict(k=k[:1]), "do not fit"), (dict(v=k[:, :5]), "do not fit"),
        (dict(k=k[:, :, :, :8], v=k[:, :, :, :8]), "do not fit"), (dict(q=q[:, :, :3]), "multiple"),
        (dict(q=q[..., :12], k=k[..., :12], v=k[..., :12]), "width"), (dict(scale=float("nan")), "finite"),
        (dict(k_lengths=torch.ones(3, device="cuda", dtype=torch.int32)), "k_lengths"),
        (dict(q_lengths=torch.ones(2, device="cuda")), "q_lengths"), (dict(k_lengths=torch.ones(2, dtype=torch.int32)), "GPU"),
        (dict(k_lengths=[1, 2]), "GPU"), (dict(key_mask=torch.ones(2, 5, device="cuda", dtype=torch.bool)), "key_mask"),
        (dict(key_mask=torch.ones(2, 6, device="cuda")), "type"), (dict(bias=bias), "together"),
        (dict(buckets=buckets), "together"), (dict(bias=bias[:7], buckets=buckets), "must be"),
        (dict(bias=bias.bfloat16(), buckets=buckets), "type"), (dict(bias=bias, buckets=(8, 6)), "Buckets"),
        (dict(q=torch.zeros(2, 4, 4, 136, device="cuda"), k=torch.zeros(2, 6, 2, 136, device="cuda"),
              v=torch.zeros(2, 6, 2, 136, device="cuda")), "width")]
    for over, text in bad:
        a = dict(q=q, k=k, v=k) | over
        with pytest.raises(ValueError, match=text):
            tokens.attention(a.pop("q"), a.pop("k"), a.pop("v"), **a)
    x = q.clone().requires_grad_(True)
    g, = torch.autograd.grad(tokens.attention(x, k, k).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


# -------------------------------------------------------------------------------- dropout

@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5, 11), (1000, 255), (0, 4), (2, 4096)])
def test_dropout(shape, dtype):
    g = gen(6)
    x, dy = normal(g, *shape, dtype=dtype), normal(g, *shape, dtype=dtype)
    seed = -0x123456789ABCDEF
    for p, site in ((0.1, 0), (0.5, 7), (0.999999, 2 ** 32 - 1)):
        step = min(int(p * 65536 + 0.5), 65535)
        keep = oracle.kept(x.numel(), step, seed & (2 ** 64 - 1), site).view(shape).cuda()
        t = leaf(x)
        on_device = torch.tensor([seed], device="cuda")
        for s in (seed, on_device):
            y = tokens.dropout(t, p, s, site=site)
            dx, = torch.autograd.grad(y, t, dy)
            for got, src in ((y, x), (dx, dy)):
                want = src.double() * keep * (65536 / (65536 - step))
                # the scale's rounding, the product's and the result's
                assert_within(got, (want, want.abs() * (2 * 2.0 ** -24 + oracle.U[dtype])))
                assert torch.equal(got == 0, ~keep | (src == 0))


def test_dropout_views_and_nothing_to_drop():
    x = normal(gen(1), 40, 60)
    a, b = tokens.dropout(x.t(), 0.3, 5), tokens.dropout(x.t().contiguous(), 0.3, 5)
    assert torch.equal(a, b)  # by logical element, whatever the storage
    buf = torch.empty(2401, device="cuda", dtype=H)
    odd = buf[1:].view(40, 60).copy_(x)
    assert torch.equal(tokens.dropout(odd, 0.3, 5), tokens.dropout(odd.clone(), 0.3, 5))
    assert tokens.dropout(x, 0.0, None) is x and tokens.dropout(x, 0.5, 1, training=False) is x
    assert not torch.equal(tokens.dropout(x, 0.5, 1), tokens.dropout(x, 0.5, 2))
    assert not torch.equal(tokens.dropout(x, 0.5, 1), tokens.dropout(x, 0.5, 1, site=1))
    bad = torch.full((64,), float("nan"), device="cuda")
    y = tokens.dropout(bad, 0.5, 3)
    assert torch.equal(y == 0, ~oracle.kept(64, 32768, 3).cuda())  # what is dropped is 0


def test_dropout_share():
    """the share kept is binomial: 6 deviations; and neighbours are not tied to each other"""
    n, p = 1 << 20, 0.25
    keep = (tokens.dropout(torch.ones(n, device="cuda"), p, 99) != 0).double()
    sd = (p * (1 - p) / n) ** 0.5
    assert abs(keep.mean().item() - (1 - p)) < 6 * sd
    c = keep - keep.mean()
    for lag in (1, 2, 7, 8, 64):
        assert abs((c[lag:] * c[:-lag]).mean().item()) / (p * (1 - p)) < 6 / n ** 0.5


def test_dropout_refusals():
    x = torch.zeros(8, device="cuda")
    for a, kw, text in (((x.half(), 0.1, 1), {}, "type"), ((x, 1.0, 1), {}, "not in"), ((x, -0.1, 1), {}, "not in"),
                        ((x, float("nan"), 1), {}, "not in"), ((x, 0.1, None), {}, "seed"), ((x, 0.1, 1.5), {}, "seed"),
                        ((x, 0.1, True), {}, "seed"), ((x, 0.1, torch.zeros(2, device="cuda", dtype=torch.int64)), {}, "one value"),
                        ((x, 0.1, torch.zeros(1, device="cuda")), {}, "type"),
                        ((x, 0.1, torch.zeros(1, dtype=torch.int64)), {}, "GPU"), ((x, 0.1, 1), dict(site=-1), "site")):
        with pytest.raises(ValueError, match=text):
            tokens.dropout(*a, **kw)


# ------------------------------------------------------------------ residual, gate and norms

BLOCK = [  # shape, post, pre, gate shape, p, scale
    ((8, 16), None, "rms", None, 0.0, 1.0),
    ((3, 5, 7), "rms", "layer", (7,), 0.3, 0.5),
    ((2, 33, 256), "layer", "rms", (2, 1, 256), 0.1, 0.7),
    ((2, 70, 64), "layer", "layer", (2, 70, 64), 0.2, 1.0),
    ((1, 1, 1), "rms", "rms", (1,), 0.0, 2.0),
    ((2, 3, 1000), "rms", None, (1, 3, 1000), 0.1, 1.0),
    ((4, 300, 24), "layer", "rms", (4, 1, 24), 0.1, -1.0),
    ((2, 9, 2048), "rms", "layer", (2, 9, 1), 0.1, 1.0),
    ((3, 2, 4096), "layer", "rms", (3, 1, 4096), 0.1, 1.0),
    ((2, 3, 8192), "rms", "rms", (2, 3, 8192), 0.0, 1.0),
    ((2, 3, 8191), "layer", "layer", (8191,), 0.4, 1.0),
    ((700, 3, 129), None, "layer", (700, 1, 129), 0.5, 1.0),
    ((2100, 520), "rms", "layer", None, 0.1, 1.0),
    ((0, 16), "rms", "rms", (16,), 0.1, 1.0),
]


def block_case(cfg, dtype, param_dtype=None, seed=5):
    shape, post, pre, gate, p, scale = cfg
    g = gen(seed)
    C = shape[-1]
    t = {"x": normal(g, *shape, dtype=dtype), "f": normal(g, *shape, dtype=dtype, std=2.0) + 0.5,
         "gate": None if gate is None else normal(g, *gate, dtype=dtype)}
    pd = param_dtype or dtype
    for side, kind in (("post", post), ("pre", pre)):
        t[side + "_weight"] = None if kind is None else 1 + normal(g, C, dtype=pd, std=0.3)
        t[side + "_bias"] = normal(g, C, dtype=pd) if kind == "layer" else None
    return t, {"dy": normal(g, *shape, dtype=dtype), "dh": normal(g, *shape, dtype=dtype) if pre else None}


def run_block(t, d, cfg, seed=77):
    shape, post, pre, _, p, scale = cfg
    leaves = {n: None if a is None else leaf(a) for n, a in t.items()}
    a = dict(leaves)
    y, h = tokens.gated_residual_norm(a.pop("x"), a.pop("f"), **a, scale=scale, post_norm=post, pre_norm=pre, p=p, seed=seed,
                                      site=3, eps=1e-5)
    assert (h is None) == (pre is None)
    outs, grads = ([y], [d["dy"]]) if h is None else ([y, h], [d["dy"], d["dh"]])
    wrt = {n: v for n, v in leaves.items() if v is not None}
    got = torch.autograd.grad(outs, list(wrt.values()), grads)
    return {"y": y.detach(), "h": None if h is None else h.detach(), **{"d" + n: v for n, v in zip(wrt, got)}}


def check_block(got, t, d, cfg, seed=77):
    shape, post, pre, _, p, scale = cfg
    step = min(int(p * 65536 + 0.5), 65535)
    mask = oracle.kept(t["x"].numel(), step, seed, 3).view(shape).cuda() if step else None
    want = oracle.block(t["x"], t["f"], gate=t["gate"], scale=scale, post=post, pre=pre, step=step, mask=mask, eps=1e-5,
                        post_w=t["post_weight"], post_b=t["post_bias"], pre_w=t["pre_weight"], pre_b=t["pre_bias"],
                        gate_written_out=cfg[3] in ((1, 3, 1000), (2, 9, 1)), **d)
    names = {"dpost_w": "dpost_weight", "dpost_b": "dpost_bias", "dpre_w": "dpre_weight", "dpre_b": "dpre_bias"}
    for n, w in want.items():
        g = got.get(names.get(n, n))
        if g is None:
            assert n.endswith(("_w", "_b")), n  # a parameter that the call did not have
            continue
        assert_within(g, w, n)


@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
@pytest.mark.parametrize("cfg", BLOCK, ids=lambda c: "-".join(map(str, c)))
def test_block(cfg, dtype):
    t, d = block_case(cfg, dtype)
    if cfg[0][0] == 0:
        got = run_block(t, d, cfg)
        assert got["y"].shape == cfg[0] and not got["dgate"].any() and not got["dpre_weight"].any()
        return
    check_block(run_block(t, d, cfg), t, d, cfg)


def test_block_first_norm():
    """f None: y is x itself, h its norm"""
    for dtype in (F, H):
        for kind in ("rms", "layer"):
            cfg = ((5, 9, 96), None, kind, None, 0.0, 1.0)
            t, d = block_case(cfg, dtype)
            x, w = leaf(t["x"]), leaf(t["pre_weight"])
            y, h = tokens.gated_residual_norm(x, None, pre_norm=kind, pre_weight=w, eps=1e-5)
            assert y is x
            dx, dw = torch.autograd.grad(h, (x, w), d["dh"])
            want = oracle.block(t["x"], None, pre=kind, pre_w=t["pre_weight"], eps=1e-5, dh=d["dh"])
            for n, g in (("h", h), ("dx", dx), ("dpre_w", dw)):
                assert_within(g, want[n], f"{kind} {n}")


def test_block_float32_parameters_with_bf16_rows():
    cfg = BLOCK[2]
    t, d = block_case(cfg, H, param_dtype=F)
    got = run_block(t, d, cfg)
    assert got["dpre_weight"].dtype == F
    check_block(got, t, d, cfg)
    t["post_bias"] = t["post_bias"].bfloat16()  # of two types: each gradient has its parameter's
    got = run_block(t, d, cfg)
    assert got["dpost_bias"].dtype == H and got["dpost_weight"].dtype == F
    for n in ("dpost_bias", "dpost_weight"):
        assert torch.isfinite(got[n]).all()


def test_block_one_gradient_missing():
    cfg = BLOCK[3]
    t, d = block_case(cfg, F)
    for missing in ("dy", "dh"):
        leaves = {n: None if a is None else leaf(a) for n, a in t.items()}
        a = dict(leaves)
        y, h = tokens.gated_residual_norm(a.pop("x"), a.pop("f"), **a, scale=cfg[5], post_norm=cfg[1], pre_norm=cfg[2], p=cfg[4],
                                          seed=77, site=3, eps=1e-5)
        out, grad = (h, d["dh"]) if missing == "dy" else (y, d["dy"])
        wrt = {n: v for n, v in leaves.items() if v is not None}
        got = torch.autograd.grad(out, list(wrt.values()), grad, allow_unused=True)
        zero = {n: None if n == missing else g for n, g in d.items()}
        got = {"y": y, "h": h, **{"d" + n: torch.zeros_like(v) if g is None else g for (n, v), g in zip(wrt.items(), got)}}
        check_block(got, t, zero, cfg)


def test_block_more_threads_than_a_launch_holds():
    """2^28 and a few rows of eight channels: sixteen threads a row pass 2^32"""
    R = (1 << 28) + 3
    x = torch.ones(R, 8, device="cuda", dtype=H)
    x[-3:] = torch.tensor([2.0, 0.0, -3.0], device="cuda", dtype=H)[:, None]
    with torch.no_grad():
        _, h = tokens.gated_residual_norm(x, None)  # 1 / sqrt(1 + 1e-6) rounds to 1
    assert h[-3:, 0].tolist() == [1.0, 0.0, -1.0]
    assert bool((h[:-3] == 1).all())


def test_block_same_bits_and_views():
    cfg = BLOCK[6]
    t, d = block_case(cfg, H)
    a, b = run_block(t, d, cfg), run_block(t, d, cfg)
    assert all(torch.equal(a[n], b[n]) for n in a if a[n] is not None)
    views = {n: v.transpose(0, 1).contiguous().transpose(0, 1) if n in ("x", "f") else v for n, v in t.items()}
    c = run_block(views, {n: v.transpose(0, 1).contiguous().transpose(0, 1) for n, v in d.items()}, cfg)
    assert all(torch.equal(a[n], c[n]) for n in a if a[n] is not None)
    odd = {n: v if v is None else torch.empty(v.numel() + 1, device="cuda", dtype=H)[1:].view(v.shape).copy_(v) for n, v in t.items()}
    leaves = {n: None if v is None else v.requires_grad_(True) for n, v in odd.items()}
    args = dict(leaves)
    y, h = tokens.gated_residual_norm(args.pop("x"), args.pop("f"), **args, scale=cfg[5], post_norm=cfg[1], pre_norm=cfg[2],
                                      p=cfg[4], seed=77, site=3, eps=1e-5)
    assert torch.equal(y, a["y"]) and torch.equal(h, a["h"])


def test_block_refusals():
    x, w = torch.zeros(2, 3, 16, device="cuda"), torch.ones(16, device="cuda")
    grn = tokens.gated_residual_norm
    for a, kw, text in (((x.half(), x.half()), {}, "type"), ((x, x[:1]), {}, "fit"), ((x, x.bfloat16()), {}, "type"),
                        ((x, x), dict(pre_norm="batch"), "pre_norm"), ((x, x), dict(post_norm="x"), "post_norm"),
                        ((x, x), dict(post_weight=w), "without a norm"), ((x, x), dict(pre_weight=w[:8]), "must be"),
                        ((x, x), dict(pre_weight=w.bfloat16()), "type"), ((x, x), dict(gate=w[:3]), "broadcast"),
                        ((x, x), dict(gate=torch.ones(5, 2, 3, 16, device="cuda")), "broadcast"),
                        ((x, x), dict(gate=w.bfloat16()), "type"), ((x, x), dict(gate=torch.ones((), device="cuda")), "broadcast"),
                        ((x, None), dict(gate=w), "need f"), ((x, None), dict(p=0.1, seed=1), "need f"),
                        ((x, None), dict(pre_norm=None), "nothing to do"), ((x, x), dict(p=0.1), "seed"),
                        ((x, x), dict(p=2.0, seed=1), "not in"), ((x, x), dict(scale=float("inf")), "finite"),
                        ((x, x), dict(eps=-1.0), "eps"), ((torch.zeros(2, 8200, device="cuda"), None), {}, "channels"),
                        ((torch.zeros((), device="cuda"), None), {}, "channels")):
        with pytest.raises(ValueError, match=text):
            grn(*a, **kw)


# ------------------------------------------------------- together, on streams and in graphs

class Layer:
    """Two blocks of a pre- and post-normed network over keypoints, as a program would write them"""

    def __init__(self, C=64, heads=4, seed=1):
        g = gen(seed)
        self.heads, self.buckets = heads, tokens.Buckets(16, 24, True)
        mk = lambda *s, std=1.0, mean=0.0: (normal(g, *s, std=std) + mean).requires_grad_(True)  # noqa: E731
        self.p = {"bias": mk(16, heads, std=0.5), "gate": mk(C, std=0.2, mean=1.0)}
        for n in ("first", "post", "pre", "post2", "last"):
            self.p[n] = mk(C, std=0.1, mean=1.0)
        for n in ("qkv", "out", "up", "down"):
            self.p[n] = mk(C, 3 * C if n == "qkv" else C, std=C ** -0.5)

    def __call__(self, x, lengths, seed):
        p, (B, N, C) = self.p, x.shape
        _, h = tokens.gated_residual_norm(x, None, pre_norm="layer", pre_weight=p["first"])
        qkv = (h.reshape(-1, C) @ p["qkv"]).view(B, N, 3, self.heads, C // self.heads)
        a = tokens.attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], k_lengths=lengths, q_lengths=lengths, bias=p["bias"],
                             buckets=self.buckets)
        f = (a.reshape(-1, C) @ p["out"]).view(B, N, C)
        x, h = tokens.gated_residual_norm(x, f, gate=p["gate"], post_norm="rms", post_weight=p["post"], pre_norm="layer",
                                          pre_weight=p["pre"], p=0.1, seed=seed, site=1)
        f = tokens.dropout(torch.relu(h.reshape(-1, C) @ p["up"]), 0.2, seed, site=2) @ p["down"]
        return tokens.gated_residual_norm(x, f.view(B, N, C), scale=0.5, post_norm="rms", post_weight=p["post2"], pre_norm="rms",
                                          pre_weight=p["last"])[1]

    def plain(self, x, lengths, seed):
        """the same in 64 bits with torch's autograd"""
        p = {n: v.detach().double().requires_grad_(True) for n, v in self.p.items()}
        B, N, C = x.shape
        D = C // self.heads

        def norm(z, w, layer):
            z = z - z.mean(-1, keepdim=True) if layer else z
            return z / (z.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w

        def drop(z, step, site):
            return z * oracle.kept(z.numel(), step, seed, site).view(z.shape).cuda() * (65536 / (65536 - step))

        h = norm(x, p["first"], True)
        q, k, v = (t.squeeze(2).transpose(1, 2) for t in (h.reshape(-1, C) @ p["qkv"]).view(B, N, 3, self.heads, D).split(1, 2))
        rel = [[self.buckets.index(j - i) for j in range(N)] for i in range(N)]
        s = q @ k.transpose(2, 3) / D ** 0.5 + p["bias"][torch.tensor(rel, device="cuda")].permute(2, 0, 1)
        there = torch.arange(N, device="cuda")[None] < lengths[:, None]
        s = s.masked_fill(~there[:, None, None], float("-inf"))
        a = (torch.softmax(s, -1) @ v).transpose(1, 2) * there[:, :, None, None]
        f = (a.reshape(-1, C) @ p["out"]).view(B, N, C)
        x = x + p["gate"] * drop(norm(f, p["post"], False), 6554, 1)
        h = norm(x, p["pre"], True)
        f = drop(torch.relu(h.reshape(-1, C) @ p["up"]), 13107, 2) @ p["down"]
        return norm(x + 0.5 * norm(f.view(B, N, C), p["post2"], False), p["last"], False), p


def chain_inputs(seed=2, B=2, N=50, C=64):
    g = gen(seed)
    lengths = torch.tensor([N, N - 13], device="cuda", dtype=torch.int32)
    return normal(g, B, N, C), lengths, normal(g, B, N, C)


def test_chain_against_64_bits():
    """Seven operators in a row (torch's products between them).  Each makes its values with at most
    C + N + 64 roundings of 2^-24 in a row, and no operator here magnifies a relative error of its
    input more than 16 times (softmax: twice the largest score, about 5; norms: 2; relu: 1; the norms
    of whole tensors are compared, so single values that cancel do not count)."""
    x, lengths, do = chain_inputs()
    net = Layer()
    xs = leaf(x)
    out = net(xs, lengths, 1234)
    grads = torch.autograd.grad(out, [xs, *net.p.values()], do)
    xd = x.double().requires_grad_(True)
    ref, p = net.plain(xd, lengths, 1234)
    want = torch.autograd.grad(ref, [xd, *p.values()], do.double())
    tol = 7 * (64 + 50 + 64) * 2.0 ** -24 * 16
    for name, a, b in zip(("out", "x", *net.p), (out, *grads), (ref, *want)):
        assert (a.double() - b).norm() <= tol * b.norm(), name


def test_chain_on_another_stream():
    x, lengths, do = chain_inputs()
    net = Layer()

    def once():
        xs = leaf(x)
        out = net(xs, lengths, 5)
        return [out.detach(), *torch.autograd.grad(out, [xs, *net.p.values()], do)]

    want = once()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = once()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_chain_in_two_graphs():
    """forward and backward captured twice (two graphs, workspaces of their own), replayed in turn with
    eager work between and a new seed and input each time: every replay is the eager result's bits"""
    x, lengths, do = chain_inputs()
    net = Layer()
    static_x, seed = x.clone().requires_grad_(True), torch.tensor([1], device="cuda")

    def once(xs):
        out = net(xs, lengths, seed)
        return [out.detach(), *torch.autograd.grad(out, [xs, *net.p.values()], do)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            once(static_x)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = once(static_x)
        graphs.append((g, outs))
    for k in range(4):
        new = normal(gen(50 + k), *x.shape)
        with torch.no_grad():
            static_x.copy_(new)
        seed.fill_(1000 + k)
        want = once(leaf(new))
        torch.cuda.synchronize()
        for g, outs in graphs:
            for o in outs:
                o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), k


@pytest.mark.parametrize("dtype", [F, H], ids=["fp32", "bf16"])
def test_attention_in_a_graph(dtype):
    """wide heads, a group, a bias, lengths that change between the replays, and a token against a cache"""
    s, kw, bias, spec = attn_case(13, (2, 200, 260, 8, 2, 128, True, [260, 100], None, False, (32, 128, False)), dtype)
    leaves = [leaf(t) for t in (s["q"], s["k"], s["v"], bias)]
    lengths = kw["k_lengths"]

    def once(q, k, v, b):
        out = tokens.attention(q, k, v, causal=True, k_lengths=lengths, bias=b, buckets=tokens.Buckets(*spec))
        with torch.no_grad():
            one = tokens.attention(q[:, :1], k, v, causal=True, k_lengths=lengths, bias=b, buckets=tokens.Buckets(*spec))
        return [out.detach(), one, *torch.autograd.grad(out, [q, k, v, b], s["do"])]

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        once(*leaves)
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = once(*leaves)
    for k in range(3):
        lengths.copy_(torch.tensor([260 - 60 * k, 100 + 80 * k]))
        want = once(*(leaf(t) for t in leaves))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), k


def test_inputs_untouched():
    s, kw, bias, spec = attn_case(3, ATTN[6], H)
    before = {n: t.clone() for n, t in s.items()}
    run_attn(s, kw, bias, spec)
    assert all(torch.equal(before[n], s[n]) for n in s)

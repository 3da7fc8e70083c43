"""Measured cases of the token operators (``pcd_reg_hregnet_amd.tokens``).

Four operators: attention over token sequences with its recomputing backward pass, the
bucketed relative position bias inside it with its gradient, the dropout that stores no
mask, and the gated residual with the norms after one block and before the next.

With ``own`` false ``run`` is the plain form (elementary torch operations in 32 bits, rounded
once at the end); with ``own`` true it makes the calls a user's program makes.
"""
import math

import torch

own = False

_F = {"fp32": torch.float32, "bf16": torch.bfloat16}
_M32 = 0xFFFFFFFF
_EPS = 1e-6


# ------------------------------------------------------------------------------- cases

def _attn(name, B, Nq, Nk, H, Hk, D, dtype, causal=False, lengths=False, holes=False, buckets=0, distance=0,
          both=True, train=True):
    c = {"op": "attention", "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "causal": causal,
         "lengths": lengths, "holes": holes, "buckets": buckets, "distance": distance, "both": both, "train": train}
    return {"name": name, **c} if name else c


def _block(name, B, N, C, dtype, post, pre, gate, p):
    c = {"op": "block", "B": B, "N": N, "C": C, "dtype": dtype, "post": post, "pre": pre, "gate": gate, "p": p}
    return {"name": name, **c} if name else c


def _drop(name, B, N, C, dtype, p):
    c = {"op": "dropout", "B": B, "N": N, "C": C, "dtype": dtype, "p": p}
    return {"name": name, **c} if name else c


def listed():
    return [
        # 256 level-3 keypoints of 8 clouds attend to each other in training: launch latency counts
        _attn("self_256_fp32", 8, 256, 256, 4, 4, 64, "fp32"),
        # 1024 level-1 keypoints attend to the other cloud's 512, some of them missing or dropped
        _attn("cross_1024_fp32", 8, 1024, 512, 4, 4, 32, "fp32", lengths=True, holes=True),
        # a long causal sequence with shared key heads: the large matrix-bound training case
        _attn("causal_4096_bf16", 2, 4096, 4096, 16, 4, 128, "bf16", causal=True),
        # an odd length with a bidirectional bias, head width between tile widths
        _attn("bias_517_fp32", 4, 517, 517, 8, 8, 40, "fp32", buckets=32, distance=128),
        # the bias in an ordinary causal training step, ragged batch
        _attn("bias_2048_bf16", 4, 2048, 2048, 16, 16, 64, "bf16", causal=True, lengths=True, buckets=32,
              distance=128, both=False),
        # one new token against a long cache with shared key heads: reads the cache once
        _attn("token_32768_bf16", 8, 1, 32768, 32, 8, 128, "bf16", lengths=True, train=False),
        # the smallest serving call: latency alone
        _attn("token_129_fp32", 1, 1, 129, 4, 4, 64, "fp32", train=False),
        # a few tokens at once against ragged caches, with the bias
        _attn("tokens_8191_bf16", 16, 4, 8191, 16, 4, 64, "bf16", causal=True, lengths=True, buckets=32,
              distance=128, both=False, train=False),
        # between two blocks over 8 x 1024 keypoints of 256 channels, a gate for each cloud, training
        _block("block_256_fp32", 8, 1024, 256, "fp32", "layer", "layer", "batch", 0.1),
        # the same boundary of a wide model, a gate for each token
        _block("block_4096_bf16", 4, 4096, 4096, "bf16", "rms", "rms", "token", 0.1),
        # dropout of one small odd activation, forward and backward: latency
        _drop("drop_255_fp32", 2, 511, 255, "fp32", 0.1),
        # dropout of a large activation: bandwidth against the generator's arithmetic
        _drop("drop_8192_bf16", 8, 4096, 2048, "bf16", 0.25),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("train", "train", "bias", "token", "block", "dropout"))
    dtype = rng.choice(("fp32", "bf16"))
    if kind in ("train", "bias"):
        Hk, G = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 2, 4))
        D = rng.choice((8, 16, 32, 40, 64, 64, 72, 96, 128, 128))
        causal = rng.random() < 0.5
        Nq = _log(rng, 8, 4096)
        Nk = Nq if rng.random() < 0.6 else _log(rng, 8, 4096)
        G = G if Nq * Nk * Hk * G < 2.2e8 else 1
        B = max(1, min(_log(rng, 1, 8), int(1.0e8 // (Nq * Nk * Hk * G))))
        nb, dist = (rng.choice((16, 32, 64)), rng.choice((64, 128, 200))) if kind == "bias" else (0, 0)
        return _attn(None, B, Nq, Nk, Hk * G, Hk, D, dtype, causal, rng.random() < 0.5, rng.random() < 0.3, nb, dist,
                     not causal, True)
    if kind == "token":
        Hk, G = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 8))
        D = rng.choice((32, 64, 80, 128))
        Nk, Nq = _log(rng, 1, 40000), rng.choice((1, 1, 1, 2, 3, 5))
        B = max(1, min(_log(rng, 1, 32), int(2.0e8 // (Nk * Hk * D))))
        bias = rng.random() < 0.3
        return _attn(None, B, Nq, Nk, Hk * G, Hk, D, dtype, True, rng.random() < 0.7, False, 32 if bias else 0,
                     128 if bias else 0, False, False)
    C = _log(rng, 8, 4096)
    C = C if rng.random() < 0.3 else max(8, C // 8 * 8)
    B, N = rng.choice((1, 2, 3, 8)), _log(rng, 1, 4096)
    p = rng.choice((0.0, 0.1, 0.3)) if kind == "block" else rng.choice((0.1, 0.3, 0.5))
    if kind == "dropout":
        return _drop(None, B, N, C, dtype, p)
    return _block(None, B, N, C, dtype, rng.choice(("none", "rms", "layer")), rng.choice(("rms", "layer")),
                  rng.choice(("none", "channel", "batch", "token")), p)


# ------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _F[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(t)

    s = {"case": case}
    if case["op"] == "attention":
        B, Nq, Nk, H, Hk, D = (case[n] for n in ("B", "Nq", "Nk", "H", "Hk", "D"))
        s["q"], s["k"], s["v"] = normal(B, Nq, H, D), normal(B, Nk, Hk, D), normal(B, Nk, Hk, D)
        s["lengths"] = s["holes"] = s["bias"] = None
        if case["lengths"]:  # ragged batches: between a half and all of the keys
            s["lengths"] = torch.randint((Nk + 1) // 2, Nk + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        if case["holes"]:  # one key in eight is not there
            s["holes"] = torch.rand(B, Nk, device="cuda", generator=g) >= 0.125
        if case["buckets"]:
            s["bias"] = normal(case["buckets"], H, std=0.5)
        if case["train"]:
            s["do"] = normal(B, Nq, H, D)
            for n in ("q", "k", "v", "bias"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
        return s
    B, N, C = case["B"], case["N"], case["C"]
    s["x"] = normal(B, N, C).requires_grad_(True)
    s["dy"] = normal(B, N, C)
    s["seed"] = torch.randint(0, 1 << 62, (1,), device="cuda", generator=g, dtype=torch.int64)
    if case["op"] == "block":
        s["f"], s["dh"] = normal(B, N, C, std=2.0).requires_grad_(True), normal(B, N, C)
        shape = {"none": None, "channel": (C,), "batch": (B, 1, C), "token": (B, N, C)}[case["gate"]]
        s["gate"] = None if shape is None else normal(*shape, mean=0.5, std=0.3).requires_grad_(True)
        for side in ("post", "pre"):
            s[side + "_w"] = s[side + "_b"] = None
            if case[side] != "none":
                s[side + "_w"] = normal(C, mean=1.0, std=0.2).requires_grad_(True)
            if case[side] == "layer":
                s[side + "_b"] = normal(C, std=0.2).requires_grad_(True)
    return s


_PARAMS = ("x", "f", "gate", "post_w", "post_b", "pre_w", "pre_b")


# ---------------------------------------------------------------------- the plain forms

def _offsets(case, lengths, device):
    """position of key j minus position of query i, [B or 1][Nq][Nk]: causal queries end where their keys end"""
    i, j = torch.arange(case["Nq"], device=device), torch.arange(case["Nk"], device=device)
    rel = (j[None, :] - i[:, None])[None]
    if case["causal"]:
        n = torch.full((1,), case["Nk"], device=device) if lengths is None else lengths
        rel = rel - (n - case["Nq"])[:, None, None]
    return rel


def _buckets(case, rel):
    """bucket of each offset: exact up to half of a side, then equal steps of the logarithm"""
    nb = case["buckets"] // 2 if case["both"] else case["buckets"]
    n = rel.abs() if case["both"] else (-rel).clamp(min=0)
    exact = nb // 2
    # 64 bits, and a step of 1e-9 past the border: a power that is a whole number counts as reached
    far = torch.log(n.clamp(min=1).double() / exact) / math.log(case["distance"] / exact) * (nb - exact)
    far = (exact + (far + 1e-9).floor().long()).clamp(max=nb - 1)
    return torch.where(n < exact, n, far) + (nb * (rel > 0).long() if case["both"] else 0)


def _keep_keys(s):
    """[B or 1][1][Nq or 1][Nk]: which keys each query sees"""
    case, dev = s["case"], s["q"].device
    j = torch.arange(case["Nk"], device=dev)
    keep = torch.ones(1, 1, 1, case["Nk"], dtype=torch.bool, device=dev)
    if s["lengths"] is not None:
        keep = keep & (j[None, :] < s["lengths"][:, None])[:, None, None]
    if s["holes"] is not None:
        keep = keep & s["holes"][:, None, None]
    if case["causal"]:
        keep = keep & (_offsets(case, s["lengths"], dev) <= 0)[:, None]
    return keep


def _plain_attention(s):
    case = s["case"]
    t, G, scale = _F[case["dtype"]], case["H"] // case["Hk"], case["D"] ** -0.5
    q = s["q"].detach().float().transpose(1, 2).contiguous()
    k, v = (s[n].detach().float().transpose(1, 2).repeat_interleave(G, 1) for n in ("k", "v"))
    a = torch.matmul(q, k.transpose(2, 3)) * scale
    if s["bias"] is not None:
        bucket = _buckets(case, _offsets(case, s["lengths"], q.device))
        a = a + s["bias"].detach().float()[bucket].permute(0, 3, 1, 2)
    a = a.masked_fill(~_keep_keys(s), -math.inf)
    top = a.amax(-1, keepdim=True)
    a = torch.exp(a - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = a.sum(-1, keepdim=True)
    a = a / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(a, v)
    out = o.transpose(1, 2).to(t)
    if not case["train"]:
        return {"out": out}
    do = s["do"].float().transpose(1, 2).contiguous()
    shared = (case["B"], case["Hk"], G, case["Nk"], case["D"])
    dv = torch.matmul(a.transpose(2, 3), do).reshape(shared).sum(2)
    da = torch.matmul(do, v.transpose(2, 3))
    da = a * (da - (do * o).sum(-1, keepdim=True))
    r = {"out": out, "dv": dv.transpose(1, 2).to(t),
         "dq": (torch.matmul(da, k) * scale).transpose(1, 2).to(t),
         "dk": (torch.matmul(da.transpose(2, 3), q).reshape(shared).sum(2) * scale).transpose(1, 2).to(t)}
    if s["bias"] is not None:
        # rows upside down and one element longer each: column Nq - 1 + j - i holds one offset
        Nq, Nk = case["Nq"], case["Nk"]
        d = torch.nn.functional.pad(da.flip(2), (0, Nq)).flatten(2)[..., :Nq * (Nq + Nk - 1)]
        d = d.reshape(case["B"], case["H"], Nq, Nq + Nk - 1).sum(2, dtype=torch.float64)  # long sums
        first = _offsets(case, s["lengths"], q.device)[:, -1, :1]
        bucket = _buckets(case, first + torch.arange(Nq + Nk - 1, device=q.device))
        one = (bucket[..., None] == torch.arange(case["buckets"], device=q.device)).double()
        r["dbias"] = torch.matmul(d, one).sum(0).T.to(t)
    return r


def _philox_round(c, k0, k1):
    a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
    hi = lambda x: (x >> 32) & _M32  # noqa: E731
    return [hi(b) ^ c[1] ^ k0, b & _M32, hi(a) ^ c[3] ^ k1, a & _M32]


def _dropout_scale(x, p, seed):
    """0 where the element is dropped, 1 / (1 - p) elsewhere: 16 bits of Philox4x32-10 for each element, eight
    consecutive elements a counter; p counts in steps of 2^-16"""
    step = min(int(p * 65536 + 0.5), 65535)
    n = x.numel()
    group = torch.arange((n + 7) // 8, device=x.device)
    c = [group & _M32, group >> 32, torch.zeros_like(group), torch.zeros_like(group)]
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    c = _philox_round(c, k0, k1)
    c = _philox_round(c, (k0 + 1 * 0x9E3779B9) & _M32, (k1 + 1 * 0xBB67AE85) & _M32)
    c = _philox_round(c, (k0 + 2 * 0x9E3779B9) & _M32, (k1 + 2 * 0xBB67AE85) & _M32)
    c = _philox_round(c, (k0 + 3 * 0x9E3779B9) & _M32, (k1 + 3 * 0xBB67AE85) & _M32)
    c = _philox_round(c, (k0 + 4 * 0x9E3779B9) & _M32, (k1 + 4 * 0xBB67AE85) & _M32)
    c = _philox_round(c, (k0 + 5 * 0x9E3779B9) & _M32, (k1 + 5 * 0xBB67AE85) & _M32)
    c = _philox_round(c, (k0 + 6 * 0x9E3779B9) & _M32, (k1 + 6 * 0xBB67AE85) & _M32)
    c = _philox_round(c, (k0 + 7 * 0x9E3779B9) & _M32, (k1 + 7 * 0xBB67AE85) & _M32)
    c = _philox_round(c, (k0 + 8 * 0x9E3779B9) & _M32, (k1 + 8 * 0xBB67AE85) & _M32)
    c = _philox_round(c, (k0 + 9 * 0x9E3779B9) & _M32, (k1 + 9 * 0xBB67AE85) & _M32)
    w = torch.stack(c, 1)
    w = torch.stack([w & 0xFFFF, w >> 16], 2).reshape(-1)[:n].reshape(x.shape)
    return (w >= step) * (65536 / (65536 - step))


def _plain_dropout(s):
    case = s["case"]
    m = _dropout_scale(s["x"], case["p"], s["seed"]).float()
    t = _F[case["dtype"]]
    return {"y": (s["x"].detach().float() * m).to(t), "dx": (s["dy"].float() * m).to(t)}




def _norm(x, kind, w, b):
    """(normed x, its values before weight and bias, 1 / deviation)"""
    if kind == "none":
        return x, x, None
    c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    n = c * r
    return n * w + (b if kind == "layer" else 0), n, r


def _norm_back(d, kind, n, r, w):
    """the gradient of a norm's input"""
    if kind == "none":
        return d
    g = d * w
    g = g - n * (g * n).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if kind == "layer" else 0)
    return g * r


def _plain_block(s):
    case = s["case"]
    t = _F[case["dtype"]]
    p = {n: s[n].detach().float() for n in _PARAMS if s[n] is not None}
    post, pre, gate = case["post"], case["pre"], p.get("gate", torch.ones((), device="cuda"))
    keep = _dropout_scale(p["x"], case["p"], s["seed"]).float() if case["p"] else 1.0
    u, fn, fr = _norm(p["f"], post, p.get("post_w"), p.get("post_b"))
    y = p["x"] + 0.5 * gate * keep * u
    h, yn, yr = _norm(y, pre, p.get("pre_w"), p.get("pre_b"))
    dh = s["dh"].float()
    dx = s["dy"].float() + _norm_back(dh, pre, yn, yr, p.get("pre_w"))
    db = dx * 0.5 * keep
    du = db * gate
    r = {"y": y, "h": h, "dx": dx, "df": _norm_back(du, post, fn, fr, p.get("post_w"))}
    if case["gate"] != "none":
        r["dgate"] = {"token": lambda a: a, "batch": lambda a: a.sum(1, keepdim=True),
                      "channel": lambda a: a.sum((0, 1))}[case["gate"]](db * u)
    if post != "none":
        r["dpost_w"] = (du * fn).sum((0, 1))
    if post == "layer":
        r["dpost_b"] = du.sum((0, 1))
    r["dpre_w"] = (dh * yn).sum((0, 1))
    if pre == "layer":
        r["dpre_b"] = dh.sum((0, 1))
    return {n: a.to(t) for n, a in r.items()}


# ------------------------------------------------------------------------ one pass each

def _own(s):
    from pcd_reg_hregnet_amd import tokens

    case = s["case"]
    if case["op"] == "attention":
        more = {}
        if s["bias"] is not None:
            more = {"bias": s["bias"], "buckets": tokens.Buckets(case["buckets"], case["distance"], case["both"])}
        with torch.set_grad_enabled(case["train"]):
            out = tokens.attention(s["q"], s["k"], s["v"], causal=case["causal"], k_lengths=s["lengths"],
                                   key_mask=s["holes"], **more)
        if not case["train"]:
            return {"out": out}
        leaves = {n: s[n] for n in ("q", "k", "v", "bias") if s[n] is not None}
        grads = torch.autograd.grad(out, list(leaves.values()), s["do"])
        r = {"out": out.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}
        return {n: r[n] for n in ("out", "dv", "dq", "dk", "dbias") if n in r}
    if case["op"] == "dropout":
        y = tokens.dropout(s["x"], case["p"], s["seed"])
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    y, h = tokens.gated_residual_norm(
        s["x"], s["f"], gate=s["gate"], scale=0.5, post_norm=None if case["post"] == "none" else case["post"],
        post_weight=s["post_w"], post_bias=s["post_b"], pre_norm=case["pre"], pre_weight=s["pre_w"],
        pre_bias=s["pre_b"], eps=_EPS, p=case["p"], seed=s["seed"])
    leaves = {n: s[n] for n in _PARAMS if s[n] is not None}
    grads = torch.autograd.grad([y, h], list(leaves.values()), [s["dy"], s["dh"]])
    return {"y": y.detach(), "h": h.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "dropout": _plain_dropout,
            "block": _plain_block}[state["case"]["op"]](state)


# --------------------------------------------------------------------------------- work

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        B, Nq, Nk, H, Hk, D = (case[n] for n in ("B", "Nq", "Nk", "H", "Hk", "D"))
        n = int(Nk * 0.75) if case["lengths"] else Nk
        pairs = Nq * n
        if case["causal"]:  # queries end where their keys end
            m = min(Nq, n)
            pairs = m * (m + 1) // 2 + m * (n - m)
        q, kv, train = B * Nq * H * D * e, B * n * Hk * D * e, case["train"]
        return {"bytes": (4 if train else 2) * q + (4 if train else 2) * kv,
                "flops": (14 if train else 4) * B * H * pairs * D}
    n = case["B"] * case["N"] * case["C"]
    if case["op"] == "dropout":
        return {"bytes": 4 * n * e, "flops": 2 * n}
    # forward x, f -> y, h ; backward f, y, dy, dh -> dx, df ; a gate for each token is read twice, written once
    return {"bytes": (10 + (3 if case["gate"] == "token" else 0)) * n * e, "flops": 40 * n}


# ---------------------------------------------------------------- the definition, 64 bits

def _exact_bucket(case, o):
    """the bucket of one offset, in whole numbers: step t is reached where (n/e)^L >= (m/e)^t"""
    nb, base, n = case["buckets"], 0, max(-o, 0)
    if case["both"]:
        nb, n = nb // 2, abs(o)
        base = nb if o > 0 else 0
    e, m = nb // 2, case["distance"]
    L = nb - e
    if n < e:
        return base + n
    return base + e + sum(n ** L * e ** t >= m ** t * e ** L for t in range(1, L))


def _exact_attention(case, s):
    B, Nq, Nk, H, Hk, D = (case[n] for n in ("B", "Nq", "Nk", "H", "Hk", "D"))
    dev, train = s["q"].device, case["train"]
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    do = s["do"].double() if train else None
    lens = [Nk] * B if s["lengths"] is None else s["lengths"].tolist()
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    table = None if s["bias"] is None else s["bias"].detach().double()
    dtable = None if table is None else torch.zeros_like(table)
    low = -(Nk + Nq)
    if table is not None:
        lut = torch.tensor([_exact_bucket(case, max(-2 * case["distance"], min(2 * case["distance"], o)))
                            for o in range(low, -low + 1)], device=dev)
    for b in range(B):
        n, start = lens[b], (lens[b] - Nq if case["causal"] else 0)
        if n == 0:
            continue
        rel = torch.arange(n, device=dev)[None] - (torch.arange(Nq, device=dev)[:, None] + start)
        hidden = (rel > 0) if case["causal"] else torch.zeros_like(rel, dtype=torch.bool)
        if s["holes"] is not None:
            hidden = hidden | ~s["holes"][b, :n][None]
        none = hidden.all(1, keepdim=True)
        for h in range(H):
            kh, vh, qh = k[b, :n, h * Hk // H], v[b, :n, h * Hk // H], q[b, :, h]
            z = (qh @ kh.T) / math.sqrt(D)
            if table is not None:
                z = z + table[lut[rel - low], h]
            z = z.masked_fill(hidden, -math.inf).masked_fill(none, 0.0)
            w = torch.softmax(z, 1).masked_fill(none, 0.0).masked_fill(hidden, 0.0)
            out[b, :, h] = w @ vh
            if train:
                g = do[b, :, h]
                dv[b, :n, h * Hk // H] += w.T @ g
                gz = w * (g @ vh.T - (g * out[b, :, h]).sum(1, keepdim=True))
                dq[b, :, h] = gz @ kh / math.sqrt(D)
                dk[b, :n, h * Hk // H] += gz.T @ qh / math.sqrt(D)
                if table is not None:
                    dtable[:, h] += torch.zeros(case["buckets"], dtype=torch.float64, device=dev).index_add_(
                        0, lut[rel - low].reshape(-1), gz.reshape(-1))
    if not train:
        return {"out": out}
    r = {"out": out, "dv": dv, "dq": dq, "dk": dk}
    return r if table is None else {**r, "dbias": dtable}


def _exact_mask(case, s):
    """1 / (1 - p) or 0 for each element, the generator in numpy's unsigned words"""
    import numpy as np
    n = s["x"].numel()
    step = min(round(case["p"] * 65536), 65535)
    if step == 0:
        return torch.ones_like(s["x"], dtype=torch.float64)
    key = int(s["seed"].item())
    word = np.uint64(_M32)
    x = [np.arange((n + 7) // 8, dtype=np.uint64), np.uint64(0), np.uint64(0), np.uint64(0)]
    ks = [key & _M32, key >> 32]
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> np.uint64(32)) ^ x[1] ^ np.uint64(ks[0]), b & word,
             (a >> np.uint64(32)) ^ x[3] ^ np.uint64(ks[1]), a & word]
        ks = [(ks[0] + 0x9E3779B9) & _M32, (ks[1] + 0xBB67AE85) & _M32]
    half = np.stack([np.broadcast_to(c, x[1].shape).astype(np.uint32) for c in x], 1).view(np.uint16).reshape(-1)[:n]
    kept = torch.from_numpy(half >= step).to(s["x"].device).reshape(s["x"].shape)
    return kept.double() / (1 - step / 65536)


def _exact_block(case, s):
    # autograd in 64 bits over the definition
    p = {n: s[n].detach().double().requires_grad_(True) for n in _PARAMS if s[n] is not None}

    def norm(z, side):
        if case[side] == "none":
            return z
        if case[side] == "layer":
            z = z - z.sum(-1, keepdim=True) / z.shape[-1]
        z = z / ((z ** 2).sum(-1, keepdim=True) / z.shape[-1] + _EPS).sqrt()
        z = z * p[side + "_w"]
        return z + p[side + "_b"] if case[side] == "layer" else z

    branch = norm(p["f"], "post") * _exact_mask(case, s)
    y = p["x"] + (branch * p["gate"] if "gate" in p else branch) / 2
    h = norm(y, "pre")
    grads = torch.autograd.grad([y, h], list(p.values()), [s["dy"].double(), s["dh"].double()])
    return {"y": y.detach(), "h": h.detach(), **{"d" + n: g for n, g in zip(p, grads)}}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "block":
        return _exact_block(case, s)
    m = _exact_mask(case, s)
    return {"y": s["x"].detach().double() * m, "dx": s["dy"].double() * m}

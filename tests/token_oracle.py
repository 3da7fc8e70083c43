"""64-bit forms of the token operators with bounds of what a kernel may be off.

Each function returns values and, beside each, how far a correctly working kernel can be from it:
roundings counted one by one.  U[t] is half a step of t (2^-8 bf16, 2^-24 f32); a sum of n terms
in f32 in any order is off by at most n U of the sum of their magnitudes."""
import math

import numpy as np
import torch

F32 = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def bucket(num, far, both, o):
    """the bucket of an offset, from the definition in exact integers"""
    side, n, base = num, max(-o, 0), 0
    if both:
        side, n = num // 2, abs(o)
        base = side if o > 0 else 0
    e = side // 2
    if n < e:
        return base + n
    L = side - e
    return base + max(e + t for t in range(L) if t == 0 or n ** L * e ** t >= far ** t * e ** L)


def attention(q, k, v, *, scale=None, causal=False, align_end=None, q_lengths=None, k_lengths=None, key_mask=None,
              bias=None, spec=None, do=None, bias_dtype=None):
    """{name: (value, bound)} for out and, with do, dq dk dv (dbias), all float64; inputs as the kernel gets
    them.  Masked keys and rows are cut out before any arithmetic, so what they hold cannot matter."""
    t = q.dtype
    B, Nq, H, D = q.shape
    Nk, Hk = k.shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    align_end = causal if align_end is None else align_end
    dev = q.device
    z = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=dev)  # noqa: E731
    val = {"out": z(q)}
    if do is not None:
        val |= {"dq": z(q), "dk": z(k), "dv": z(v)}
        if bias is not None:
            val["dbias"] = z(bias)
    bound = {n: torch.zeros_like(x) for n, x in val.items()}
    u, up = U[t], (U[t] if t == torch.bfloat16 else 0.0)
    for b in range(B):
        nq = Nq if q_lengths is None else min(max(int(q_lengths[b]), 0), Nq)
        nk = Nk if k_lengths is None else min(max(int(k_lengths[b]), 0), Nk)
        start = nk - nq if align_end else 0
        keys = torch.arange(nk, device=dev)
        if key_mask is not None:
            keys = keys[key_mask[b if key_mask.shape[0] > 1 else 0, :nk]]
        if nq == 0 or len(keys) == 0:
            continue
        rel = keys[None, :] - torch.arange(nq, device=dev)[:, None] - start
        see = rel <= 0 if causal else torch.ones_like(rel, dtype=torch.bool)
        if bias is not None:
            lut = torch.tensor([[bucket(*spec, int(o)) for o in row] for row in rel.cpu()], device=dev)
        for h in range(H):
            Q = q[b, :nq, h].double()
            K, V = k[b, keys, h // G].double(), v[b, keys, h // G].double()
            s, sa = scale * Q @ K.T, abs(scale) * Q.abs() @ K.abs().T
            if bias is not None:
                w = bias[:, h].double()[lut]
                s, sa = s + w, sa + w.abs()
            s, sa = s.masked_fill(~see, -math.inf), sa.masked_fill(~see, 0.0)
            top = s.max(1, keepdim=True).values.clamp(min=-1e300)
            p = torch.exp(s - top)
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            o = p @ V
            # a score: D products and sums, scale, bias, the running maximum's changes; a
            # probability: twice that (numerator and sum), exp2, and the sum of nk terms
            ep = (4 * (D + len(keys) + 32) * F32) * (1 + sa.max(1, keepdim=True).values)
            n = (len(keys) + 16) * F32
            ob = (ep + up + n) * (p @ V.abs()) + u * o.abs()
            val["out"][b, :nq, h], bound["out"][b, :nq, h] = o, ob
            if do is None:
                continue
            dO = do[b, :nq, h].double()
            dp, dpa = dO @ V.T, dO.abs() @ V.abs().T
            delta, da = (dO * o).sum(1, keepdim=True), (dO * o).abs().sum(1, keepdim=True)
            ds = p * (dp - delta)
            g = (D + 16) * F32
            eds = p * (ep * (dpa + da) + g * (dpa + da) + (dO.abs() * ob).sum(1, keepdim=True)) + up * ds.abs()
            dq = scale * ds @ K
            val["dq"][b, :nq, h] = dq
            bound["dq"][b, :nq, h] = abs(scale) * (eds + n * ds.abs()) @ K.abs() + u * dq.abs()
            m = (nq * G + 16) * F32
            val["dk"][b, keys, h // G] += scale * ds.T @ Q
            bound["dk"][b, keys, h // G] += abs(scale) * (eds + m * ds.abs()).T @ Q.abs()
            val["dv"][b, keys, h // G] += p.T @ dO
            bound["dv"][b, keys, h // G] += ((ep + up + m) * p).T @ dO.abs()
            if bias is not None:
                N = (nq * len(keys) + 16) * F32
                val["dbias"][:, h].index_add_(0, lut.reshape(-1), ds.reshape(-1))
                # (the bias gradient sums ds before its rounding to bf16; the rounding of out that eds counts is
                # more than the kernel's D = do . o feels, which keeps what out lost)
                bound["dbias"][:, h].index_add_(0, lut.reshape(-1), (eds + N * ds.abs()).reshape(-1))
    for name in ("dk", "dv"):
        if name in val:
            bound[name] += u * val[name].abs()
    if "dbias" in val:
        bound["dbias"] += U[bias_dtype or bias.dtype] * val["dbias"].abs()
    return {n: (val[n], bound[n]) for n in val}


def philox(counter, key):
    """Philox4x32-10 on numpy words: counter four arrays, key two ints -> four uint64 arrays of 32 bits"""
    x = [np.asarray(c, dtype=np.uint64) for c in counter]
    k = [int(c) for c in key]
    low, hi = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> hi) ^ x[1] ^ np.uint64(k[0]), b & low, (a >> hi) ^ x[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return x


def kept(n, step, seed, site=0):
    """which of n elements are kept"""
    g = np.arange((n + 7) // 8, dtype=np.uint64)
    w = philox([g & np.uint64(0xFFFFFFFF), g >> np.uint64(32), np.full_like(g, site), np.zeros_like(g)],
               [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF])
    halves = np.stack([h for c in w for h in (c & np.uint64(0xFFFF), c >> np.uint64(16))], 1).reshape(-1)[:n]
    return torch.from_numpy(halves >= step)


def block(x, f, *, gate=None, scale=1.0, post=None, post_w=None, post_b=None, pre=None, pre_w=None, pre_b=None,
          eps=1e-6, step=0, mask=None, dy=None, dh=None, gate_written_out=False):
    """{name: (value, bound)} of y, h and the gradients, float64; mask: which elements are kept.

    e = (2 C + 64) F32 covers any value that is one row sum and a few operations away from its
    inputs, relative to the magnitudes it is made of."""
    t, C = x.dtype, x.shape[-1]
    u, e = U[t], (2 * C + 64) * F32
    D = lambda a: None if a is None else a.double()  # noqa: E731
    one = torch.ones((), dtype=torch.float64, device=x.device)
    m = one if mask is None else mask.double() * (65536 / (65536 - step))
    w1, b1, w2, b2 = (D(a) if a is not None else d for a, d in
                      ((post_w, one), (post_b, 0 * one), (pre_w, one), (pre_b, 0 * one)))
    mean = lambda a: a.mean(-1, keepdim=True)  # noqa: E731

    def norm(z, kind):
        c = z - mean(z) if kind == "layer" else z
        r = 1 / (mean(c * c) + eps).sqrt()
        return c * r, r

    X = D(x)
    g = one if gate is None else D(gate)
    if f is not None:
        Fv = D(f)
        n1, r1 = norm(Fv, post) if post else (Fv, one)
        # a normed value: its row's mean and deviation carry e; magnitudes |f - mean| + mean |f|
        en1 = e * (n1.abs() + mean(Fv.abs()) * r1) if post else 0 * Fv
        un = n1 * w1 + b1 if post else Fv
        eu = en1 * w1.abs() + e * (un.abs() + b1.abs() + (n1 * w1).abs()) if post else 0 * Fv
        y = X + scale * g * m * un
        ey = abs(scale) * g.abs() * m * (eu + e * un.abs()) + e * (X.abs() + y.abs())
    else:
        y, ey = X, 0 * X
    val, bound = {}, {}

    def put(name, v, err):
        val[name], bound[name] = v, err + u * v.abs()

    if f is not None:
        put("y", y, ey)
    if pre:
        n2, r2 = norm(y, pre)
        # the norm of values that are off by ey: their own error, and the row's
        en2 = r2 * ey + n2.abs() * mean(n2.abs() * r2 * ey) + (r2 * mean(ey)) + e * (n2.abs() + mean(y.abs()) * r2)
        put("h", n2 * w2 + b2, en2 * w2.abs() + e * ((n2 * w2).abs() + b2.abs()))
    if dy is None and dh is None:
        return {n: (val[n], bound[n]) for n in val}
    dx = D(dy) if dy is not None else 0 * X
    edx = e * dx.abs()
    cols = lambda a: a.reshape(-1, C).sum(0)  # noqa: E731
    R = x.numel() // C
    er = (R + 16) * F32
    if pre and dh is not None:
        H = D(dh)
        en2b = en2 + (u * y.abs() * r2 if f is not None and t == torch.bfloat16 else 0)  # y as it was rounded
        q = H * w2
        s1, s2 = mean(q * n2), mean(q)
        es1 = mean(q.abs() * en2b) + e * mean((q * n2).abs())
        d = q - n2 * s1 - (s2 if pre == "layer" else 0)
        ed = e * (q.abs() + (n2 * s1).abs() + mean(q.abs())) + en2b * s1.abs() + n2.abs() * es1
        dx = dx + r2 * d
        er2 = e + mean(n2.abs() * r2 * ey)  # the deviation's own error
        edx = edx + r2 * (ed + er2 * d.abs()) + e * (r2 * d).abs()
        put("dpre_w", cols(H * n2), cols(H.abs() * en2b) + er * cols((H * n2).abs()))
        put("dpre_b", cols(H), er * cols(H.abs()))
    put("dx", dx, edx)
    if f is not None:
        db = dx * scale * m
        edb = (edx + e * dx.abs()) * abs(scale) * m
        du, edu = db * g, edb * g.abs() + e * (db * g).abs()
        if gate is not None:
            full, efull = db * un, edb * un.abs() + db.abs() * eu + e * (db * un).abs()
            shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
            dims = [i for i, s in enumerate(shape) if s == 1 and x.shape[i] != 1]
            red = lambda a: (a.sum(dims, keepdim=True) if dims else a).reshape(gate.shape)  # noqa: E731
            k = math.prod(x.shape[i] for i in dims)
            # a gate that is written out for each element before the call gets a gradient for each
            # element, rounded to its type (u of each), and their sum outside is rounded again
            out = 2 * u * red(full.abs()) if gate_written_out else 0
            put("dgate", red(full), red(efull) + (k + 16) * F32 * red(full.abs()) + out)
        if post:
            q, eq = du * w1, edu * w1.abs() + e * (du * w1).abs()
            s1, s2 = mean(q * n1), mean(q)
            es1 = mean(eq * n1.abs() + q.abs() * en1) + e * mean((q * n1).abs())
            es2 = mean(eq) + e * mean(q.abs()) if post == "layer" else 0
            d = q - n1 * s1 - (s2 if post == "layer" else 0)
            ed = eq + n1.abs() * es1 + en1 * s1.abs() + es2 + e * (q.abs() + (n1 * s1).abs() + mean(q.abs()))
            put("df", r1 * d, r1 * ed + 2 * e * (r1 * d).abs())
            put("dpost_w", cols(du * n1), cols(edu * n1.abs() + du.abs() * en1) + er * cols((du * n1).abs()))
            put("dpost_b", cols(du), cols(edu) + er * cols(du.abs()))
        else:
            put("df", du, edu)
    return {n: (val[n], bound[n]) for n in val}


def assert_within(got, want, what=""):
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), (what, got.shape, value.shape)
    off = (got.double() - value).abs() - bound.to(got.device)
    assert not torch.isnan(got).any(), f"{what}: NaN"
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 1e-30, f"{what}: {worst:.3g} beyond its bound (largest bound {bound.max().item():.3g})"

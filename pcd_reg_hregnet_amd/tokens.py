"""Operators over token sequences on the HIP library: what a model needs to let its keypoint
descriptors attend to each other, in training and when it answers one token at a time.

* ``attention``: softmax(scale q k^T + bias) v with grouped key heads, lengths, a key mask and
  causal order; its backward pass recomputes the probabilities (nothing of size Nq x Nk is
  stored).  ``Buckets`` and a learned table give it a relative position bias by buckets, with
  the table's gradient.  One call serves training and single tokens.
* ``dropout``: from a counter-based generator, the mask made again where it is needed.
* ``gated_residual_norm``: the norm behind one block, dropout, gate and scaled residual, and the
  norm before the next block in one pass, forward and backward.

They stand beside ``train_graph``'s operators: autograd functions whose arithmetic is one or a
few C-ABI launches (csrc/tok_attn.hip, csrc/tok_elem.hip) on the current stream of the tensors'
device; no CPU fallback.  Row data is float32 or bfloat16.  Float32 products keep float32
accuracy (three exact bf16 pieces a value); sums, statistics and accumulators are float32.
Results do not depend on the order in which workgroups run.  A call can be captured in a HIP
graph: nothing is read on the host, and a seed tensor is read when the graph replays.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.TOK_F32, torch.bfloat16: _lib.TOK_BF16}
_DENSE = torch.contiguous_format
_NORMS = {None: 0, "rms": 1, "layer": 2}
_MOST = 1e38  # a scale or eps goes to the kernels as float32, some of them multiplied by log2(e)


_ENTRIES = {}


def _call(name: str, *args) -> None:
    """the C entry, bound at its first call (``_lib.load`` checks the library and the GPU then)"""
    f = _ENTRIES.get(name)
    if f is None:
        f = _ENTRIES[name] = getattr(_lib.load(), name)
    rc = f(*args)
    if rc != _lib.HREG_OK:
        raise RuntimeError(f"{name} failed: {_lib._ERRORS.get(rc, rc)} (code {rc})")


def _launch(device, name: str, *args) -> None:
    """the entry on the current stream of the tensors' device, which is current meanwhile"""
    if device.index == torch.cuda.current_device():
        _call(name, *args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            _call(name, *args, _raw_stream(device.index))


# the handle of a device's current stream without the Stream object around it (torch's own
# compiled code takes it from here): 0.3 us instead of 2.7
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


# (checks build their messages only when they fail: a call's host time is what a single token
# waits for)
def _check_tensor(fn: str, name: str, t, device=None, dtype=None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{fn}: {name} must be a GPU tensor (no CPU fallback)")
    if device is not None and t.device != device:
        raise ValueError(f"{fn}: {name} is on {t.device}, expected {device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{fn}: {name} has type {t.dtype}, expected {dtype}")


def _any_tangent(*tensors) -> bool:
    """whether forward-mode differentiation goes through one of them: no operator has that derivative, and
    an autograd function raises on such a tensor (a plain launch would return a result without it)"""
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


# the leading fields of the C structs, packed in one step (0.5 us; one by one they take 6)
_ATTN_HEAD = struct.Struct("@9if4P12q4P")  # dtype .. scale, q k v out, their strides, lse .. k_len
_BLOCK_HEAD = struct.Struct("@7i2f2IQ20P")  # dtype .. seed, seed_dev, x .. dpre_b


# --------------------------------------------------------------------- relative positions

@functools.lru_cache(maxsize=None)
def _thresholds(exact: int, side: int, far: int) -> tuple:
    """First offsets of the logarithmic buckets: the least n with (n / exact)^L >= (far /
    exact)^t for t = 1 .. L - 1, L = side - exact, in whole numbers (a float logarithm would
    decide borders by its rounding)."""
    L = side - exact
    out = []
    for t in range(1, L):
        n = max(exact, int(exact * (far / exact) ** (t / L)) - 1)
        while n ** L * exact ** t < far ** t * exact ** L:
            n += 1
        while n > exact and (n - 1) ** L * exact ** t >= far ** t * exact ** L:
            n -= 1
        out.append(n)
    return tuple(out)


@dataclass(frozen=True)
class Buckets:
    """Buckets of the offset o = key position - query position.

    ``bidirectional``: half of the buckets for o <= 0, half for o > 0; otherwise all of them for
    o <= 0, and every o > 0 is in bucket 0.  On a side with S buckets distances below S // 2 have
    one each; the others are equal steps of the logarithm up to ``max_distance``, the last one
    for everything from there on.  A plain value: a program makes it once or for each call."""
    num_buckets: int = 32
    max_distance: int = 128
    bidirectional: bool = True

    def __post_init__(self):
        n, far = self.num_buckets, self.max_distance
        if not (isinstance(n, int) and isinstance(far, int)):
            raise ValueError("Buckets: num_buckets and max_distance must be int")
        if not 2 <= n <= _lib.TOK_MAX_BUCKETS:
            raise ValueError(f"Buckets: num_buckets {n} not in 2 .. {_lib.TOK_MAX_BUCKETS}")
        if self.bidirectional and (n % 2 or n < 4):
            raise ValueError(f"Buckets: num_buckets {n} must be even and at least 4 for both directions")
        if not self._side // 2 < far <= _lib.TOK_MAX_DISTANCE:
            raise ValueError(f"Buckets: max_distance {far} not in {self._side // 2 + 1} .. {_lib.TOK_MAX_DISTANCE}")

    @property
    def _side(self) -> int:
        return self.num_buckets // 2 if self.bidirectional else self.num_buckets

    @property
    def thresholds(self) -> tuple:
        """first distances of the logarithmic buckets after the first"""
        return _thresholds(self._side // 2, self._side, self.max_distance)

    def index(self, offset: int) -> int:
        """the bucket of one offset"""
        n = abs(offset) if self.bidirectional else max(-offset, 0)
        exact = self._side // 2
        b = n if n < exact else exact + sum(n >= t for t in self.thresholds)
        return b + (self._side if self.bidirectional and offset > 0 else 0)


# ------------------------------------------------------------------------------ attention

def _rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it whose rows the kernels can read: contiguous rows in 16-byte steps"""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        n = 16 // t.element_size()
        if t.stride(-1) == 1 and all(s % n == 0 for s, m in zip(t.stride()[:-1], t.shape[:-1]) if m > 1):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _attn_args(o, q, k, v, out, lse, out_rest, q_len, k_len, key_mask, bias) -> _lib.TokAttn:
    scale, causal, align_end, buckets = o
    B, Nq, H, D = q.shape
    p = _lib.TokAttn()
    _ATTN_HEAD.pack_into(p, 0, _DTYPES[q.dtype], B, Nq, k.shape[1], H, k.shape[2], D, causal, align_end, scale, q.data_ptr(),
                         k.data_ptr(), v.data_ptr(), out.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                         *out.stride()[:3], _ptr(lse), _ptr(out_rest), _ptr(q_len), _ptr(k_len))
    if key_mask is not None:
        p.key_mask, p.mask_sb = key_mask.data_ptr(), 0 if key_mask.shape[0] == 1 else key_mask.stride(0)
    if bias is not None:
        p.bias, p.bias_dtype = bias.data_ptr(), _DTYPES[bias.dtype]
        p.num_buckets, p.max_distance, p.both = buckets.num_buckets, buckets.max_distance, buckets.bidirectional
        t = buckets.thresholds
        p.nthresh = len(t)
        p.thresh = t
    return p


def _attn_ws(p: _lib.TokAttn, backward: int, device):
    n = _lib.load(require_gpu=False).hreg_tok_attn_ws_bytes(ctypes.byref(p), backward)
    if n == 0:
        return None
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    p.ws, p.ws_bytes = ws.data_ptr(), n
    return ws


def _attn_forward(o, q, k, v, bias, q_len, k_len, key_mask, train: bool):
    q, k, v = _rows(q), _rows(k), _rows(v)
    dev = q.device
    out = torch.empty_like(q, memory_format=_DENSE)
    B, Nq, H, _ = q.shape
    lse = torch.empty(2, B, H, Nq, dtype=torch.float32, device=dev) if train else None
    rest = torch.empty_like(out) if train and q.dtype != torch.float32 else None
    p = _attn_args(o, q, k, v, out, lse, rest, q_len, k_len, key_mask, bias)
    ws = _attn_ws(p, 0, dev)  # noqa: F841 (held until the launch is queued)
    _launch(dev, "hreg_tok_attn_fwd", ctypes.byref(p))
    return q, k, v, out, lse, rest


class _TokAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, o, q_len, k_len, key_mask):
        q, k, v, out, lse, rest = _attn_forward(o, q, k, v, bias, q_len, k_len, key_mask, True)
        ctx.save_for_backward(q, k, v, bias, out, lse, rest, q_len, k_len, key_mask)
        ctx.o = o
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, bias, out, lse, rest, q_len, k_len, key_mask = ctx.saved_tensors
        need_q, need_k, need_v, need_b = ctx.needs_input_grad[:4]
        dout = _rows(dout)
        dev = q.device
        dq = torch.empty_like(q, memory_format=_DENSE) if need_q else None
        dk = torch.empty_like(k, memory_format=_DENSE) if need_k or need_v else None
        dv = torch.empty_like(v, memory_format=_DENSE) if need_k or need_v else None
        db = torch.empty_like(bias) if need_b else None
        p = _attn_args(ctx.o, q, k, v, out, lse, rest, q_len, k_len, key_mask, bias)
        p.dout = dout.data_ptr()
        p.dos_b, p.dos_n, p.dos_h, _ = dout.stride()
        p.dq, p.dk, p.dv, p.dbias = _ptr(dq), _ptr(dk), _ptr(dv), _ptr(db)
        ws = _attn_ws(p, 1, dev)  # noqa: F841
        _launch(dev, "hreg_tok_attn_bwd", ctypes.byref(p))
        return dq, dk if need_k else None, dv if need_v else None, db, None, None, None, None


def _lengths(name: str, t, B: int, device):
    if t is None:
        return None
    _check_tensor("attention", name, t, device)
    if t.dtype not in (torch.int32, torch.int64) or t.shape != (B,):
        raise ValueError(f"attention: {name} must be int32 or int64 of shape ({B},), got {t.dtype} {tuple(t.shape)}")
    if t.dtype == torch.int64:
        t = t.clamp(0, 2 ** 31 - 1).to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def attention(q, k, v, *, scale=None, causal=False, align_end=None, q_lengths=None, k_lengths=None,
              key_mask=None, bias=None, buckets=None):
    """softmax_j(scale q_i . k_j + bias[bucket, h]) v_j -> [B, Nq, H, D].

    q [B, Nq, H, D]; k, v [B, Nk, Hk, D] with H a multiple of Hk (each key head serves H // Hk
    consecutive query heads); float32 or bfloat16, D a multiple of 8 up to 128.  Any strides:
    rows that are not contiguous 16-byte aligned steps are copied first.  Batch x heads x tokens / 128
    (rounded up) stays below 2^24.  scale: D ** -0.5 by default.  Differentiable (once) in q, k, v
    and bias; forward-mode derivatives raise.

    k_lengths, q_lengths [B] int32 / int64 on the GPU (clamped to the tensors): keys and queries
    from there on do not exist.  key_mask [B or 1, Nk] bool: False keys are not seen.  Their
    values, NaN among them, have no influence.  Queries that do not exist or see no key give 0
    and take no gradient.  A key that is not finite and that any query sees may reach every query
    of its batch entry, and a query or an output gradient that is not finite every key's gradient
    unless its position is behind the lengths or, where causal, before the first key.

    Positions: key j stands at j; query i at i, or with align_end (the default where causal) at
    i + keys - queries, so that the last query stands at the last key.  causal: a query sees keys
    up to its own position.

    bias [num_buckets, H] (float32 or q's type) and ``Buckets`` add a learned bias by the offset of
    key and query.  A finite entry hides no key, however low: rows that see nothing else share themselves out
    among such keys.  With bfloat16 rows its gradient has their accuracy (about 2^-8 of it).

    bfloat16: sums are float32; the probabilities and their gradients are rounded for the products with v, k and q,
    to bfloat16 in large calls, to 16 bits in those that do not fill the card or read few rows against a cache.  So
    out and gradients are between once and one and a half times as far off as their own rounding, and a row's last
    bit may depend on the batch that it comes in."""
    _check_tensor("attention", "q", q)
    dev, dtype = q.device, q.dtype
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != dev:
            _check_tensor("attention", name, t, dev, dtype)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"attention: q, k, v must be [batch, tokens, heads, width], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if dtype not in _DTYPES:
        raise ValueError(f"attention: type {dtype} not supported (float32, bfloat16)")
    B, Nq, H, D = q.shape
    _, Nk, Hk, _ = k.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"attention: k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    if H < 1 or Hk < 1 or H % Hk:
        raise ValueError(f"attention: {H} heads are not a multiple of {Hk} key heads")
    if not 8 <= D <= 128 or D % 8:
        raise ValueError(f"attention: width {D} is not a multiple of 8 up to 128")
    scale = D ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _MOST:
        raise ValueError(f"attention: scale {scale} is not finite in float32")
    q_len, k_len = _lengths("q_lengths", q_lengths, B, dev), _lengths("k_lengths", k_lengths, B, dev)
    if key_mask is not None:
        _check_tensor("attention", "key_mask", key_mask, dev, torch.bool)
        if key_mask.dim() != 2 or key_mask.shape[0] not in (1, B) or key_mask.shape[1] != Nk:
            raise ValueError(f"attention: key_mask must be [{B} or 1, {Nk}], got {tuple(key_mask.shape)}")
        key_mask = key_mask if key_mask.stride(1) == 1 else key_mask.contiguous()
    if (bias is None) != (buckets is None):
        raise ValueError("attention: bias and buckets come together")
    if bias is not None:
        if not isinstance(buckets, Buckets):
            raise ValueError("attention: buckets must be a Buckets")
        _check_tensor("attention", "bias", bias, dev)
        if bias.dtype not in (torch.float32, dtype):
            raise ValueError(f"attention: bias has type {bias.dtype}, expected float32 or {dtype}")
        if bias.shape != (buckets.num_buckets, H):
            raise ValueError(f"attention: bias must be [{buckets.num_buckets}, {H}], got {tuple(bias.shape)}")
        bias = bias.contiguous()
    o = scale, bool(causal), bool(causal if align_end is None else align_end), buckets
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                     or (bias is not None and bias.requires_grad))) or _any_tangent(q, k, v, bias):
        return _TokAttention.apply(q, k, v, bias, o, q_len, k_len, key_mask)
    return _attn_forward(o, q, k, v, bias, q_len, k_len, key_mask, False)[3]


# -------------------------------------------------------------------------------- dropout

def _draws(fn: str, p, seed, site, device):
    """(step, seed value, seed tensor): p counts in steps of 2^-16"""
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"{fn}: p {p} not in [0, 1)")
    step = min(int(p * 65536 + 0.5), 65535)
    if not isinstance(site, int) or not 0 <= site < 2 ** 32:
        raise ValueError(f"{fn}: site must be an int of 32 bits")
    if isinstance(seed, torch.Tensor):
        _check_tensor(fn, "seed", seed, device, torch.int64)
        if seed.numel() != 1:
            raise ValueError(f"{fn}: seed must hold one value, got {tuple(seed.shape)}")
        return step, 0, seed
    if step and (not isinstance(seed, int) or isinstance(seed, bool)):
        raise ValueError(f"{fn}: p > 0 needs a seed (int or int64 GPU tensor)")
    return step, (seed or 0) & (2 ** 64 - 1), None


def _dropout(x, step, value, seed, site):
    x = x.contiguous()
    y = torch.empty_like(x)
    _launch(x.device, "hreg_tok_dropout", x.data_ptr(), y.data_ptr(), x.numel(), _DTYPES[x.dtype], step, value, _ptr(seed),
            site)
    return y


class _TokDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, step, value, seed, site):
        ctx.save_for_backward(seed)
        ctx.draws = step, value, site
        return _dropout(x, step, value, seed, site)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        step, value, site = ctx.draws
        return _dropout(dy, step, value, ctx.saved_tensors[0], site), None, None, None, None


def dropout(x, p, seed, *, site=0, training=True):
    """x with each element kept with probability 1 - p and divided by it, else 0.

    p is taken in steps of 2^-16, and the kept values are scaled by that step, so the expectation
    is x.  The choice depends on (seed, site, element number in x's logical order) alone:
    Philox4x32-10, so the backward pass, or another call, makes the same mask.  seed: an int, or an
    int64 GPU tensor of one value that is read on the device (it must keep its value until the
    backward pass).  site (32 bits) tells the places of one model apart that share a seed.
    float32 or bfloat16, any shape; training False returns x."""
    _check_tensor("dropout", "x", x)
    if x.dtype not in _DTYPES:
        raise ValueError(f"dropout: type {x.dtype} not supported (float32, bfloat16)")
    step, value, seed = _draws("dropout", p, seed, site, x.device)
    if not training or step == 0:
        return x
    return _TokDropout.apply(x, step, value, seed, site)


# ------------------------------------------------------------------ residual, gate and norms

def _block_args(o, like, param_dtype, seed, x, f, gate, post_w, post_b, pre_w, pre_b, y, h, stats, *back) -> _lib.TokBlock:
    """back: dy, dh, then the gradients of x .. pre_b"""
    scale, eps, post, pre, step, value, site, gate_rows = o
    C = like.shape[-1]
    p = _lib.TokBlock()
    dy, dh, dx, df, dgate, dpost_w, dpost_b, dpre_w, dpre_b = back or (None,) * 9
    _BLOCK_HEAD.pack_into(p, 0, _DTYPES[like.dtype], _DTYPES[param_dtype], like.numel() // C, C, gate_rows, post, pre, scale,
                          eps, step, site, value, _ptr(seed), _ptr(x), _ptr(f), _ptr(gate), _ptr(post_w), _ptr(post_b),
                          _ptr(pre_w), _ptr(pre_b), _ptr(y), _ptr(h), _ptr(stats), _ptr(dy), _ptr(dh), _ptr(dx), _ptr(df),
                          _ptr(dgate), _ptr(dpost_w), _ptr(dpost_b), _ptr(dpre_w), _ptr(dpre_b))
    return p


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, post_w, post_b, pre_w, pre_b, o, seed, param_dtype):
        dev = x.device
        y = torch.empty_like(x) if f is not None else None
        h = torch.empty_like(x) if o[3] else None
        stats = torch.empty(x.numel() // x.shape[-1], 4, dtype=torch.float32, device=dev)
        p = _block_args(o, x, param_dtype, seed, x, f, gate, post_w, post_b, pre_w, pre_b, y, h, stats)
        _launch(dev, "hreg_tok_block_fwd", ctypes.byref(p))
        ctx.save_for_backward(f, gate, post_w, post_b, pre_w, pre_b, stats, seed, x if y is None else y)
        ctx.o, ctx.param_dtype = o, param_dtype
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        f, gate, post_w, post_b, pre_w, pre_b, stats, seed, y = ctx.saved_tensors
        need = ctx.needs_input_grad
        like = [y, f, gate, post_w, post_b, pre_w, pre_b]
        if dy is None and dh is None:
            return (None,) * 10
        make = torch.empty_like if y.numel() else torch.zeros_like  # (no rows: the sums are zero)
        grads = [make(t) if n and t is not None else None for t, n in zip(like, need)]
        dy, dh = (None if g is None else g.contiguous() for g in (dy, dh))
        dev = y.device
        p = _block_args(ctx.o, y, ctx.param_dtype, seed, None, f, gate, post_w, post_b, pre_w, pre_b, y, None, stats, dy, dh,
                        *grads)
        n = _lib.load(require_gpu=False).hreg_tok_block_ws_bytes(ctypes.byref(p))
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            p.ws, p.ws_bytes = ws.data_ptr(), n
        _launch(dev, "hreg_tok_block_bwd", ctypes.byref(p))
        return (*grads, None, None, None)


_PARAMS = ("post_weight", "post_bias", "pre_weight", "pre_bias")


def _gate_of(gate, x):
    """(gate rows [n, C], rows of x a gate row serves): a gate that is constant over trailing token
    dimensions is read in place; any other broadcast is written out"""
    shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
    lead = 0
    while lead < x.dim() - 1 and shape[lead] == x.shape[lead]:
        lead += 1
    if shape[-1] != x.shape[-1] or any(n != 1 for n in shape[lead:-1]):
        return gate.expand(x.shape).contiguous(), 1
    return gate.contiguous(), max(math.prod(x.shape[lead:-1]), 1)


def gated_residual_norm(x, f, *, gate=None, scale=1.0, post_norm=None, post_weight=None, post_bias=None,
                        pre_norm="rms", pre_weight=None, pre_bias=None, eps=1e-6, p=0.0, seed=None, site=0):
    """y = x + scale * gate * dropout(post_norm(f)), h = pre_norm(y) -> (y, h).

    The boundary between two blocks: f is the output of the last one, x the residual stream, h
    the input of the next one.  x, f [..., C] float32 or bfloat16, C <= 8192.  Norms: None, "rms"
    (x / sqrt(mean x^2 + eps)) or "layer" (mean taken off first), each with an optional weight and
    bias [C] of float32 or x's type.  gate broadcasts against x ([C], [B, 1, C], [B, N, C], ...) and
    has its type.  p, seed, site: as in ``dropout``.  f None: y is x, h its norm.  pre_norm None:
    h is None.  h is made from y before y is rounded; the backward pass reads y as returned.
    Differentiable (once) in x, f, gate, weights and biases."""
    fn = "gated_residual_norm"
    _check_tensor(fn, "x", x)
    dtype, dev = x.dtype, x.device
    if dtype not in _DTYPES:
        raise ValueError(f"{fn}: type {dtype} not supported (float32, bfloat16)")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 8192:
        raise ValueError(f"{fn}: x {tuple(x.shape)} must have 1 .. 8192 channels")
    C = x.shape[-1]
    if x.numel() // C > 2 ** 30:
        raise ValueError(f"{fn}: more than 2^30 rows")
    if post_norm not in _NORMS or pre_norm not in _NORMS:
        raise ValueError(f"{fn}: post_norm {post_norm!r}, pre_norm {pre_norm!r}: each one of None, 'rms', 'layer'")
    params = [post_weight, post_bias, pre_weight, pre_bias]
    types = set()
    for name, t, norm in zip(_PARAMS, params, (post_norm, post_norm, pre_norm, pre_norm)):
        if t is None:
            continue
        _check_tensor(fn, name, t, dev)
        if norm is None:
            raise ValueError(f"{fn}: {name} without a norm")
        if t.shape != (C,):
            raise ValueError(f"{fn}: {name} must be [{C}], got {tuple(t.shape)}")
        if t.dtype not in (torch.float32, dtype):
            raise ValueError(f"{fn}: {name} has type {t.dtype}, expected float32 or {dtype}")
        types.add(t.dtype)
    step, value, seed = _draws(fn, p, seed, site, dev)
    if f is None:
        if gate is not None or post_norm is not None or step:
            raise ValueError(f"{fn}: gate, post_norm and p need f")
        if pre_norm is None:
            raise ValueError(f"{fn}: neither f nor pre_norm: nothing to do")
    else:
        _check_tensor(fn, "f", f, dev, dtype)
        if f.shape != x.shape:
            raise ValueError(f"{fn}: f {tuple(f.shape)} does not fit x {tuple(x.shape)}")
        f = f.contiguous()
    scale, eps = float(scale), float(eps)
    if not abs(scale) <= _MOST:
        raise ValueError(f"{fn}: scale {scale} is not finite in float32")
    if not 0.0 <= eps <= _MOST:
        raise ValueError(f"{fn}: eps {eps} is not a finite number >= 0 in float32")
    rows = 1
    if gate is not None:
        _check_tensor(fn, "gate", gate, dev, dtype)
        if not 1 <= gate.dim() <= x.dim() or not all(n in (1, m) for n, m in zip(gate.shape[::-1], x.shape[::-1])):
            raise ValueError(f"{fn}: gate {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}")
        gate, rows = _gate_of(gate, x)
    if len(types) > 1:
        params = [None if t is None else t.float() for t in params]
        types = {torch.float32}
    params = [None if t is None else t.contiguous() for t in params]
    o = scale, eps, _NORMS[post_norm], _NORMS[pre_norm], step, value, site, rows
    y, h = _GatedResidualNorm.apply(x.contiguous(), f, gate, *params, o, seed if step else None,
                                    types.pop() if types else torch.float32)
    return x if y is None else y, h

"""Token operators without a GPU: the buckets, the oracle against differences and the generator's
published answers, the ABI structs' layout and the argument checks of the C entries."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

import token_oracle as oracle
from pcd_reg_hregnet_amd import _lib, tokens

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("num,far,both", [(32, 128, True), (32, 128, False), (64, 200, True), (16, 64, False), (4, 2, True),
                                          (2, 2, False), (3, 7, False), (128, 1024, False), (128, 65, False), (8, 3, True)])
def test_buckets(num, far, both):
    b = tokens.Buckets(num, far, both)
    last = -1
    for n in range(0, far + 3):
        for o in (-n, n):
            assert b.index(o) == oracle.bucket(num, far, both, o), o
        assert b.index(-n) >= last  # further keys never go back a bucket
        last = b.index(-n)
    side = num // 2 if both else num
    assert b.index(-far) == side - 1 == b.index(-10 ** 9)
    assert len(b.thresholds) == side - side // 2 - 1 <= _lib.TOK_MAX_THRESH
    assert list(b.thresholds) == sorted(b.thresholds)


@pytest.mark.parametrize("args", [(1, 8, False), (130, 256, False), (7, 64, True), (2, 64, True), (32, 8, True), (32, 16, False),
                                  (32, 1025, True), (32.0, 128, True), (32, 0, True)])
def test_buckets_refused(args):
    with pytest.raises(ValueError, match="Buckets"):
        tokens.Buckets(*args)


def test_philox_published_answers():
    """the generator's known answers (Random123's test vectors for philox4x32-10)"""
    for ctr, key, want in (((0,) * 4, (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                           ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                           ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                            (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(c) for c in oracle.philox([np.array(c) for c in ctr], key)) == want


def _difference(f, x, h=1e-5):
    g = torch.zeros_like(x)
    flat, out = x.reshape(-1), g.reshape(-1)
    for i in range(flat.numel()):
        old = flat[i].item()
        flat[i] = old + h
        a = f()
        flat[i] = old - h
        out[i] = (a - f()) / (2 * h)
        flat[i] = old
    return g


@pytest.mark.parametrize("causal", [False, True])
def test_attention_oracle_against_differences(causal):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, do, bias = r(2, 3, 2, 8), r(2, 5, 1, 8), r(2, 5, 1, 8), r(2, 3, 2, 8), r(8, 2)
    oracle.U[torch.float64] = 2.0 ** -53
    kw = dict(causal=causal, k_lengths=[5, 3], key_mask=torch.tensor([[1, 1, 0, 1, 1], [1, 1, 1, 1, 1]]).bool(), bias=bias,
              spec=(8, 4, True))
    want = oracle.attention(q, k, v, do=do, **kw)
    loss = lambda: (oracle.attention(q, k, v, **kw)["out"][0] * do).sum().item()  # noqa: E731
    for name, x in (("dq", q), ("dk", k), ("dv", v), ("dbias", bias)):
        # central differences: h^2 / 6 of a third derivative (about 10 here), roundings of about 1e-15 / h
        assert (want[name][0] - _difference(loss, x)).abs().max() < 1e-8, name


@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", "rms"), (None, "layer")])
def test_block_oracle_against_differences(post, pre):
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    oracle.U[torch.float64] = 2.0 ** -53
    x, f, gate, dy, dh = r(2, 3, 5), r(2, 3, 5), r(2, 1, 5), r(2, 3, 5), r(2, 3, 5)
    w = [r(5) for _ in range(4)]
    kw = dict(gate=gate, scale=0.7, post=post, pre=pre, pre_w=w[2], pre_b=w[3], step=20000,
              mask=oracle.kept(30, 20000, 5).view(2, 3, 5), eps=0.01)
    if post:
        kw |= dict(post_w=w[0], post_b=w[1])
    want = oracle.block(x, f, dy=dy, dh=dh, **kw)
    def loss():
        r = oracle.block(x, f, **kw)
        return ((r["y"][0] * dy).sum() + (r["h"][0] * dh).sum()).item()
    pairs = [("dx", x), ("df", f), ("dgate", gate), ("dpre_w", w[2]), ("dpre_b", w[3])]
    for name, t in pairs + ([("dpost_w", w[0]), ("dpost_b", w[1])] if post else []):
        assert (want[name][0] - _difference(loss, t)).abs().max() < 1e-7, name


def test_struct_layout_matches_c():
    src = ('#include "hregnet_amd.h"\n#include <stdio.h>\n'
           'int main(){printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(hreg_tok_attn_t), offsetof(hreg_tok_attn_t, lse),'
           ' offsetof(hreg_tok_attn_t, ws_bytes), sizeof(hreg_tok_block_t), offsetof(hreg_tok_block_t, seed_dev),'
           ' offsetof(hreg_tok_block_t, ws_bytes));return 0;}')
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "t.c"), os.path.join(td, "t")
        open(c, "w").write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(REPO, "include"), c, "-o", exe])
        got = [int(v) for v in subprocess.check_output([exe]).split()]
    A, B = _lib.TokAttn, _lib.TokBlock
    assert got == [ctypes.sizeof(A), A.lse.offset, A.ws_bytes.offset, ctypes.sizeof(B), B.seed_dev.offset, B.ws_bytes.offset]


def test_packed_fields_match_the_structs():
    """the leading fields that are packed in one step end where the struct's next field starts"""
    assert tokens._ATTN_HEAD.size == _lib.TokAttn.key_mask.offset
    assert tokens._BLOCK_HEAD.size == _lib.TokBlock.ws.offset
    p = _lib.TokAttn()
    tokens._ATTN_HEAD.pack_into(p, 0, *range(9), 0.5, *range(10, 30))
    assert [getattr(p, n) for n, _ in _lib.TokAttn._fields_[:9]] == list(range(9)) and p.scale == 0.5
    assert [getattr(p, n) for n, _ in _lib.TokAttn._fields_[10:30]] == list(range(10, 30))
    b = _lib.TokBlock()
    tokens._BLOCK_HEAD.pack_into(b, 0, *range(1, 8), 0.5, 0.25, *range(10, 33))
    assert [getattr(b, n) for n, _ in _lib.TokBlock._fields_[:32]] == [*range(1, 8), 0.5, 0.25, *range(10, 33)]


def _attn(**over):
    """arguments that pass, on made-up aligned addresses (nothing is launched without a GPU: every
    case below is refused before)"""
    p = _lib.TokAttn()
    p.dtype, p.B, p.Nq, p.Nk, p.H, p.Hk, p.D, p.scale = _lib.TOK_BF16, 1, 4, 4, 2, 1, 16, 0.25
    for n in ("q", "k", "v", "out", "dout", "lse", "dq", "dk", "dv", "ws"):
        setattr(p, n, 4096)
    for n in ("qs", "ks", "vs", "os", "dos"):
        for d, step in (("b", 128), ("n", 32), ("h", 16)):
            setattr(p, f"{n}_{d}", step)
    p.ws_bytes = 1 << 20
    for n, v in over.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize("over,code", [
    (dict(dtype=2), 1), (dict(B=-1), 1), (dict(Nq=-1), 1), (dict(Nk=-1), 1), (dict(H=3, Hk=2), 1), (dict(Hk=0), 1),
    (dict(D=12), 3), (dict(D=136), 3), (dict(D=0), 3), (dict(q=None), 1), (dict(q=4098), 1), (dict(out=4100), 1),
    (dict(ks_n=36), 1), (dict(Nq=(1 << 30) + 1), 3), (dict(B=1 << 20, Nq=1 << 20), 3), (dict(B=1 << 23, Nq=1, Nk=1), 3), (dict(B=1 << 16, Nq=1, Nk=1 << 15), 3),
    (dict(bias=4096, bias_dtype=5), 1), (dict(bias=4096, num_buckets=1, max_distance=8), 1),
    (dict(bias=4096, num_buckets=7, both=1, max_distance=8), 1), (dict(bias=4096, num_buckets=32, max_distance=16), 1),
    (dict(bias=4096, num_buckets=32, max_distance=2000, nthresh=15), 3),
    (dict(bias=4096, num_buckets=256, max_distance=1000, nthresh=127), 3),
    (dict(bias=4096, num_buckets=32, max_distance=128, nthresh=3), 1)])
def test_attention_entry_refuses(over, code):
    L = _lib.load(require_gpu=False)
    for fn in (L.hreg_tok_attn_fwd, L.hreg_tok_attn_bwd):
        assert fn(ctypes.byref(_attn(**over)), None) == code
    assert L.hreg_tok_attn_fwd(None, None) == 1


@pytest.mark.parametrize("over", [dict(ws_bytes=16), dict(ws=None), dict(ws=4096 + 16), dict(dout=None), dict(dout=4100),
                                  dict(lse=None), dict(dq=4104), dict(dk=None), dict(dv=None),
                                  dict(dos_n=33)])
def test_attention_backward_entry_refuses(over):
    assert _lib.load(require_gpu=False).hreg_tok_attn_bwd(ctypes.byref(_attn(**over)), None) == 1


def _block(**over):
    p = _lib.TokBlock()
    p.dtype = p.param_dtype = _lib.TOK_F32
    p.R, p.C, p.gate_rows, p.post, p.pre = 8, 16, 1, 1, 2
    for n in ("x", "f", "y", "h", "stats", "dy", "dh", "dx", "df", "ws"):
        setattr(p, n, 4096)
    p.ws_bytes = 1 << 20
    for n, v in over.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize("over,code", [
    (dict(dtype=2), 1), (dict(param_dtype=-1), 1), (dict(R=-1), 1), (dict(C=0), 1), (dict(C=8200), 3), (dict(post=3), 1),
    (dict(pre=-1), 1), (dict(step=65536), 1), (dict(gate=4096, gate_rows=3), 1), (dict(gate=4096, gate_rows=0), 1),
    (dict(gate=4096, f=None), 1), (dict(stats=4100), 1), (dict(R=(1 << 30) + 1), 3)])
def test_block_entries_refuse(over, code):
    L = _lib.load(require_gpu=False)
    for fn in (L.hreg_tok_block_fwd, L.hreg_tok_block_bwd):
        assert fn(ctypes.byref(_block(**over)), None) == code


def test_block_entries_refuse_missing_buffers():
    L = _lib.load(require_gpu=False)
    for over in (dict(x=None), dict(y=None), dict(h=None), dict(f=None, pre=0)):
        assert L.hreg_tok_block_fwd(ctypes.byref(_block(**over)), None) == 1, over
    for over in (dict(stats=None), dict(y=None), dict(ws=None), dict(ws_bytes=8), dict(ws=4100)):
        assert L.hreg_tok_block_bwd(ctypes.byref(_block(**over)), None) == 1, over


def test_dropout_entry_refuses():
    f = _lib.load(require_gpu=False).hreg_tok_dropout
    ok = [4096, 4096, 8, _lib.TOK_F32, 100, 1, None, 0, None]
    for at, bad in ((0, None), (1, None), (2, -1), (3, 7), (4, 65536)):
        assert f(*(bad if i == at else a for i, a in enumerate(ok))) == 1, (at, bad)
    assert f(None, None, 0, _lib.TOK_F32, 100, 1, None, 0, None) == 0
    assert f(4096, 4096, 1 << 62, _lib.TOK_F32, 100, 1, None, 0, None) == 3


def test_cpu_tensors_refused():
    x = torch.zeros(1, 4, 1, 8)
    with pytest.raises(ValueError, match="GPU tensor"):
        tokens.attention(x, x, x)
    with pytest.raises(ValueError, match="GPU tensor"):
        tokens.dropout(x, 0.1, 1)
    with pytest.raises(ValueError, match="GPU tensor"):
        tokens.gated_residual_norm(x, x)

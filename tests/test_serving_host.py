"""CPU tests of the serving operators' refusals: the C entry points check their
arguments before any CUDA call, the Python layer raises ValueError on what does
not fit together and refuses CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tritonforge_b200 import _lib, kernels
from tritonforge_b200.kernels import KV4Cache

P = ctypes.c_void_p(256)  # never dereferenced: every call below is refused first


def prompt(q=P, k=P, out=P, qs=(1024, 128), ks=(256, 128), S=1, Tq=4, Tk=4, hq=8, hkv=2, d=128, dtype=_lib.BF16, ws=P,
           n=8192, cu=P, scale=0.1):
    return _lib.load().tf_prompt_attention(q, *qs, k, *ks, k, *ks, out, *qs, cu, cu, S, Tq, Tk, hq, hkv, d, 1, scale,
                                           dtype, ws, n, None)


def test_prompt_attention_refusals():
    assert prompt(hq=7) == _lib.ERR_BAD_SHAPE
    assert prompt(Tq=-1) == _lib.ERR_BAD_SHAPE
    assert prompt(S=0) == _lib.ERR_BAD_SHAPE
    assert prompt(dtype=_lib.F32) == _lib.ERR_BAD_DTYPE
    assert prompt(d=96) == _lib.ERR_UNSUPPORTED
    assert prompt(hq=258, hkv=2) == _lib.ERR_UNSUPPORTED
    assert prompt(q=None) == _lib.ERR_BAD_ARG
    assert prompt(cu=None) == _lib.ERR_BAD_ARG
    assert prompt(ws=None) == _lib.ERR_WORKSPACE
    assert prompt(n=16) == _lib.ERR_WORKSPACE
    assert prompt(qs=(1028, 128)) == _lib.ERR_UNALIGNED
    assert prompt(k=ctypes.c_void_p(264)) == _lib.ERR_UNALIGNED
    assert prompt(scale=0.0) == prompt(scale=-1.0) == prompt(scale=float("nan")) == _lib.ERR_BAD_ARG
    assert prompt(Tq=0, q=None) == _lib.OK
    assert _lib.load().tf_prompt_attention_workspace_bytes(4, 4, 1, 8, 2, 128) >= 256


def write(k=P, ks=(256, 128), c=P, cu=P, S=1, T=4, B=1, h=2, d=128, g=64, t_max=64, dtype=_lib.F16):
    return _lib.load().tf_kv4_write(k, *ks, k, *ks, c, c, c, c, cu, None, None, S, T, B, h, d, g, t_max, dtype, None)


def test_kv4_refusals():
    lib = _lib.load()
    assert write(d=96) == _lib.ERR_UNSUPPORTED
    assert write(g=32) == _lib.ERR_UNSUPPORTED
    assert write(d=64, g=128) == _lib.ERR_UNSUPPORTED
    assert write(t_max=72) == _lib.ERR_BAD_SHAPE
    assert write(B=-1) == _lib.ERR_BAD_SHAPE
    assert write(S=0) == _lib.ERR_BAD_SHAPE
    assert write(dtype=_lib.F32) == _lib.ERR_BAD_DTYPE
    assert write(c=None) == _lib.ERR_BAD_ARG
    assert write(k=None) == _lib.ERR_BAD_ARG
    assert write(cu=None) == _lib.ERR_BAD_ARG
    assert write(ks=(260, 128)) == _lib.ERR_UNALIGNED
    assert write(c=ctypes.c_void_p(260)) == _lib.ERR_UNALIGNED
    assert write(T=0, k=None) == _lib.OK
    assert lib.tf_rope_kv4_write(P, 1000, P, P, P, P, P, P, P, None, None, 1, 4, 1, 8, 2, 128, 64, 64, _lib.F16,
                                 None) == _lib.ERR_BAD_SHAPE
    assert lib.tf_rope_kv4_write(P, 1536, None, P, P, P, P, P, P, None, None, 1, 4, 1, 8, 2, 128, 64, 64, _lib.F16,
                                 None) == _lib.ERR_BAD_ARG
    assert lib.tf_rope_kv4_write(P, 1540, P, P, P, P, P, P, P, None, None, 1, 4, 1, 8, 2, 128, 64, 64, _lib.F16,
                                 None) == _lib.ERR_UNALIGNED
    assert lib.tf_kv4_read(P, P, P, P, None, 256, 128, P, 256, 128, P, None, None, 1, 4, 1, 2, 128, 64, 64, _lib.F16,
                           None) == _lib.ERR_BAD_ARG

    def attend(q=P, lens=P, B=1, hq=8, h=2, d=128, g=64, scale=0.1, ws=P, n=1 << 40):
        return lib.tf_kv4_decode_attention(q, P, P, P, P, P, lens, B, hq, h, d, g, 64, scale, _lib.BF16, ws, n, None)

    assert attend(scale=0.0) == attend(scale=-1.0) == _lib.ERR_BAD_ARG
    assert attend(ws=None) == attend(n=256) == _lib.ERR_WORKSPACE

    assert attend(hq=7) == _lib.ERR_BAD_SHAPE
    assert attend(hq=0) == _lib.ERR_BAD_SHAPE
    assert attend(B=70000) == _lib.ERR_BAD_SHAPE
    assert attend(d=80) == _lib.ERR_UNSUPPORTED
    assert attend(q=None) == _lib.ERR_BAD_ARG
    assert attend(lens=None) == _lib.ERR_BAD_ARG
    assert attend(q=ctypes.c_void_p(258)) == _lib.ERR_UNALIGNED
    assert attend(B=0) == _lib.OK


def test_kv4_read_refuses_rows_that_overlap():
    """Rows written over each other (an expanded output): no order among them."""
    def read(ks, vs, T=4, h=2):
        return _lib.load().tf_kv4_read(P, P, P, P, P, *ks, P, *vs, P, None, None, 1, T, 1, h, 128, 64, 64, _lib.F16, None)

    good = (256, 128)
    for bad in ((0, 128), (256, 0), (64, 128), (256, 64)):
        assert read(bad, good) == read(good, bad) == _lib.ERR_BAD_SHAPE
    assert read((0, 0), good) == read((0, 128), good, h=1) == read((256, 0), good, T=1) == _lib.ERR_BAD_SHAPE


def test_logprobs_refusals():
    def call(x=P, ld=100, t=P, M=2, V=100, top=3, dtype=_lib.F32, out=P, ids=P):
        return _lib.load().tf_token_logprobs(x, ld, t, M, V, top, dtype, out, out, out, ids, None)

    assert call(V=0) == _lib.ERR_BAD_SHAPE
    assert call(ld=99) == _lib.ERR_BAD_SHAPE
    assert call(M=-1) == _lib.ERR_BAD_SHAPE
    assert call(top=33) == _lib.ERR_BAD_ARG
    assert call(V=2, top=3) == _lib.ERR_BAD_ARG
    assert call(dtype=_lib.U8) == _lib.ERR_BAD_DTYPE
    assert call(x=None) == _lib.ERR_BAD_ARG
    assert call(t=None) == _lib.ERR_BAD_ARG
    assert call(ids=None) == _lib.ERR_BAD_ARG
    assert call(M=0, x=None) == _lib.OK


CU = torch.tensor([0, 4], dtype=torch.int32)


def qkv(t=4, hq=8, h=2, d=64, dtype=torch.float16):
    return torch.zeros(t, hq, d, dtype=dtype), torch.zeros(t, h, d, dtype=dtype), torch.zeros(t, h, d, dtype=dtype)


def test_prompt_attention_python_checks():
    q, k, v = qkv()
    for bad in ((q[0], k, v), (q, k, v[:3]), (q, k.float(), v), (q.float(), k.float(), v.float()),
                (q[:, :7], k, v), (q[..., :32], k, v), (q[:3], k, v)):
        with pytest.raises(ValueError):
            kernels.prompt_attention(*bad, CU)
    with pytest.raises(ValueError):
        kernels.prompt_attention(q, k, v, CU.long())
    with pytest.raises(ValueError):
        kernels.prompt_attention(q, k, v, CU, torch.tensor([0, 2, 4], dtype=torch.int32))
    with pytest.raises(ValueError):
        kernels.prompt_attention(q, k, v, CU, scale=-1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.prompt_attention(q, k, v, CU)


def cpu_cache(b=2, h=2, t=32, d=64, g=64, dtype=torch.float16):
    return KV4Cache.empty(b, h, t, d, g, dtype, device="cpu")


def test_kv4_python_checks():
    c = cpu_cache()
    assert c.layout() == (2, 2, 64, 64, 32, _lib.F16)
    assert KV4Cache.empty(1, 1, 17, 128, 64, device="cpu").k.shape[2] == 32
    for kw in (dict(head_dim=96), dict(group_size=32), dict(head_dim=64, group_size=128), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            KV4Cache.empty(**{**dict(batch=1, kv_heads=1, max_len=16, head_dim=128, device="cpu"), **kw})
    _, k, v = qkv()
    start = torch.zeros(1, dtype=torch.int32)
    for args in ((k[..., :32], v, c, CU), (k, v[:3], c, CU), (k.bfloat16(), v.bfloat16(), c, CU), (k, v, c, CU.long()),
                 (k, v, c._replace(v=c.v[:1]), CU), (k, v, c._replace(k=c.k.to(torch.int8)), CU),
                 (k, v, c._replace(k=c.k.transpose(1, 2)), CU)):
        with pytest.raises(ValueError):
            kernels.kv4_write(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.kv4_write(k, v, c, CU, start)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.kv4_read(c, CU, 4)
    q = torch.zeros(2, 14, 64, dtype=torch.float16)
    for bad in (q[:1], q[:, :7], q[..., :32], q.bfloat16()):
        with pytest.raises(ValueError):
            kernels.kv4_decode_attention(bad, c, torch.zeros(2, dtype=torch.int32))
    rows = torch.zeros(4, 12 * 64, dtype=torch.float16)
    table = torch.zeros(32, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        kernels.rope_kv4_write(rows[:, :-64], 8, table, table, c, CU)
    with pytest.raises(ValueError):
        kernels.rope_kv4_write(rows, 8, table[:16], table, c, CU)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.rope_kv4_write(rows, 8, table, table, c, CU)


def test_logprobs_python_checks():
    x, t = torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64)
    for args in ((x[0], t), (x, t[:2]), (x, t.int()), (x.long(), t), (x, t, 33), (x, t, -1), (x[:, :4], t, 5)):
        with pytest.raises(ValueError):
            kernels.token_logprobs(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.token_logprobs(x, t, 2)


def test_fused_step_refusals():
    lib = _lib.load()

    def call(qkv=P, ld=1536, cos=P, hq=8, h=2, pos=P, scale=0.1, n=1 << 40):
        return lib.tf_kv4_decode_attention_rope(qkv, ld, cos, cos, P, P, P, P, pos, P, 1, hq, h, 128, 64, 64, scale,
                                                _lib.BF16, P, n, None)

    assert call(ld=1528) == _lib.ERR_BAD_SHAPE
    assert call(ld=1540) == _lib.ERR_UNALIGNED
    assert call(hq=7) == _lib.ERR_BAD_SHAPE
    assert call(cos=None) == call(qkv=None) == call(pos=None) == call(scale=-1.0) == _lib.ERR_BAD_ARG
    assert call(n=256) == _lib.ERR_WORKSPACE
    c = cpu_cache()
    rows, table = torch.zeros(2, 12 * 64, dtype=torch.float16), torch.zeros(32, 64, dtype=torch.float16)
    pos = torch.zeros(2, dtype=torch.int32)
    for args in ((rows[:1], 8, table, table, c, pos), (rows[:, :-64], 8, table, table, c, pos),
                 (rows, 8, table[:16], table, c, pos), (rows.bfloat16(), 8, table, table, c, pos)):
        with pytest.raises(ValueError):
            kernels.kv4_decode_attention_rope(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.kv4_decode_attention_rope(rows, 8, table, table, c, pos)

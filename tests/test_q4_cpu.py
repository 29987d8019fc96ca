"""Refusals of the 4-bit and logits entry points (no GPU call is reached), and the restatements they
are tested against."""
import ctypes

import numpy as np
import pytest

from tests import q4_util as u

A, B, C, D, E = (i << 24 for i in range(1, 6))  # addresses far apart; none is ever read


def _lib():
    from vvllm_b200 import _lib

    return _lib


def _refused(status, *words):
    msg = _lib().lib().b200q8_last_error().decode()
    assert status == -1, (status, msg)
    for w in words:
        assert w in msg, msg


def test_quantize_refusals():
    L = _lib().lib()
    _refused(L.b200q8_quantize_q4(A, 4, 64, 48, B, C, None), "group")
    _refused(L.b200q8_quantize_q4(A, 4, 64, 0, B, C, None), "group")
    _refused(L.b200q8_quantize_q4(A, 4, 0, 64, B, C, None), "K == 0")
    _refused(L.b200q8_quantize_q4(A, 1 << 31, 64, 64, B, C, None), "overflow")
    for args in ((None, B, C), (A, None, C), (A, B, None)):
        _refused(L.b200q8_quantize_q4(args[0], 4, 64, 64, args[1], args[2], None), "null")
    _refused(L.b200q8_quantize_q4(A, 4, 64, 64, A + 1023, C, None), "overlap")
    _refused(L.b200q8_quantize_q4(A, 4, 64, 64, B, B + 126, None), "overlap")
    _refused(L.b200q8_quantize_q4(A + 2, 4, 64, 64, B, C, None), "aligned")
    _refused(L.b200q8_quantize_q4_bf16(A + 1, 4, 64, 64, B, C, None), "aligned")
    _refused(L.b200q8_quantize_q4_bf16(A, 4, 64, 64, B, C + 1, None), "aligned")
    assert L.b200q8_quantize_q4(None, 0, 64, 64, None, None, None) == 0


def test_dequantize_refusals():
    L = _lib().lib()
    _refused(L.b200q8_dequantize_q4(A, 2, B, C, 64, None, 4, 4, 64, None), "dtype")
    _refused(L.b200q8_dequantize_q4(A, 0, B, C, 64, None, 5, 4, 64, None), "R must be N")
    _refused(L.b200q8_dequantize_q4(A, 0, B, C, 16, D, 5, 4, 64, None), "group")
    _refused(L.b200q8_dequantize_q4(None, 0, B, C, 64, D, 5, 4, 64, None), "null")
    _refused(L.b200q8_dequantize_q4(A, 0, None, C, 64, D, 5, 4, 64, None), "null")
    _refused(L.b200q8_dequantize_q4(A, 0, A + 1024, C, 64, D, 5, 4, 64, None), "overlap")
    _refused(L.b200q8_dequantize_q4(A, 0, B, C, 64, A + 4, 5, 4, 64, None), "overlap")
    _refused(L.b200q8_dequantize_q4(A + 2, 0, B, C, 64, D, 5, 4, 64, None), "aligned")
    _refused(L.b200q8_dequantize_q4(A, 0, B, C, 64, D, 1 << 31, 4, 64, None), "overflow")
    assert L.b200q8_dequantize_q4(None, 0, None, None, 64, None, 0, 0, 64, None) == 0
    assert L.b200q8_dequantize_q4(None, 0, B, C, 64, None, 0, 4, 64, None) == -1  # all rows of a matrix of 4


def test_linear_refusals():
    L = _lib().lib()

    def call(out=A, odt=0, x=B, xdt=0, q=C, s=D, group=64, bias=None, res=None, M=2, N=4, K=64):
        return L.b200q8_linear_q4_add(out, odt, x, xdt, q, s, group, bias, res, M, N, K, None)

    _refused(call(odt=2), "dtype")
    _refused(call(xdt=-1), "dtype")
    _refused(call(group=256), "group")
    _refused(call(K=0), "K == 0")
    _refused(call(M=1 << 31), "overflow")
    _refused(call(K=1 << 31), "overflow")
    for k in ("out", "x", "q", "s"):
        _refused(call(**{k: None}), "null")
    _refused(call(x=A + 28), "inp overlaps")
    _refused(call(q=A + 31), "weights overlap")
    _refused(call(s=A + 30), "weights overlap")
    _refused(call(bias=A + 16), "bias overlaps")
    _refused(call(res=A + 4), "residual partially")
    _refused(call(x=B + 2), "aligned")
    _refused(call(s=D + 1), "aligned")
    _refused(call(out=A + 1, odt=1), "aligned")
    assert call(M=0) == 0 and call(N=0) == 0
    _refused(L.b200q8_linear_q4(A, 0, B, 0, C, D, 1, None, 1, 4, 64, None), "linear_q4:", "group")


def test_logits_refusals():
    mod = _lib()
    L, R = mod.lib(), mod._LogitRules

    def call(out=A, odt=0, os=100, x=B, xdt=0, xs=100, M=3, V=100, am=C, **rules):
        r = R(**rules)
        return L.b200q8_process_logits(out, odt, os, x, xdt, xs, M, V, ctypes.byref(r), am, None)

    _refused(call(odt=3), "dtype")
    _refused(call(V=0), "V == 0")
    _refused(call(V=1 << 31, xs=1 << 31, os=1 << 31), "overflow")
    _refused(call(M=1 << 31), "overflow")
    _refused(call(x=None), "null")
    _refused(call(out=None, am=None), "neither")
    _refused(call(xs=99), "stride")
    _refused(call(os=99), "stride")
    _refused(call(xs=1 << 41), "stride")
    _refused(call(history=D, history_count=5), "history_len")
    _refused(call(bias_ids=D, bias_count=5), "come together")
    _refused(call(bias_values=D, bias_count=5), "come together")
    _refused(call(history=D, history_count=5, history_stride=4, history_len=E), "longer")
    _refused(call(bias_ids=D, bias_values=E, bias_count=5, bias_stride=4), "longer")
    _refused(call(allowed=D, allowed_stride=3), "longer")
    _refused(call(x=B + 2), "aligned")
    _refused(call(allowed=D + 2, allowed_stride=4), "aligned")
    _refused(call(out=B + 4), "overlaps logits")
    _refused(call(out=B, odt=1, os=200), "overlaps logits")  # in place needs one type and stride
    _refused(call(am=A + 1196), "argmax overlaps")
    _refused(call(am=B), "argmax overlaps")
    _refused(call(allowed=A + 1196), "input")
    _refused(call(history=C, history_count=1, history_len=D), "input")
    assert call(M=0) == 0


def test_binding_refusals():
    """The Python calls check shapes, types and devices before any address is taken."""
    import torch

    import vvllm_b200 as v

    f, h, b, u8, i32 = torch.float32, torch.float16, torch.bfloat16, torch.uint8, torch.int32
    w, q4, sc = torch.zeros((4, 100)), torch.zeros((4, 50), dtype=u8), torch.zeros((4, 2), dtype=b)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        v.quantize_q4(w, q4, sc, 64)
    with pytest.raises(ValueError, match="group"):
        v.quantize_q4(w, q4, sc, 65)
    with pytest.raises(ValueError, match="w must be"):
        v.quantize_q4(w.half(), q4, sc, 64)
    with pytest.raises(ValueError, match="w must be"):
        v.quantize_q4_bf16(w, q4, sc, 64)
    with pytest.raises(ValueError, match="q4 must be"):
        v.quantize_q4(w, q4[:, :-1], sc, 64)
    with pytest.raises(ValueError, match="scales must be"):
        v.quantize_q4(w, q4, sc, 32)
    with pytest.raises(ValueError, match="scales must be"):
        v.quantize_q4(w, q4, sc.half(), 64)
    with pytest.raises(ValueError, match="w must be"):
        v.quantize_q4(torch.zeros((100, 4)).t(), q4, sc, 64)
    with pytest.raises(ValueError, match="rows must be"):
        v.dequantize_q4(torch.zeros((3, 100)), q4, sc, 64, rows=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="out must be"):
        v.dequantize_q4(torch.zeros((3, 100)), q4, sc, 64)
    x, out = torch.zeros((2, 100)), torch.zeros((2, 4))
    with pytest.raises(ValueError, match="out must be"):
        v.linear_q4(torch.zeros((2, 5)), x, q4, sc, 64)
    with pytest.raises(ValueError, match="bias must be"):
        v.linear_q4(out, x, q4, sc, 64, torch.zeros(3))
    with pytest.raises(ValueError, match="residual must be"):
        v.linear_q4_add(out, x, q4, sc, 64, None, torch.zeros((2, 4), dtype=h))
    with pytest.raises(ValueError, match="x must be"):
        v.linear_q4(out, torch.zeros((100, 2)).t(), q4, sc, 64)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        v.linear_q4(out, x, q4, sc, 64)
    lg = torch.zeros((2, 64))
    with pytest.raises(ValueError, match="contiguous rows"):
        v.process_logits(torch.zeros((2, 63)), lg)
    with pytest.raises(ValueError, match="contiguous rows"):
        v.process_logits(None, torch.zeros((64, 2)).t())
    with pytest.raises(ValueError, match="argmax must be"):
        v.process_logits(lg, lg, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="history must be"):
        v.process_logits(lg, lg, history=torch.zeros((2, 3)), history_len=torch.zeros(2, dtype=i32))
    with pytest.raises(ValueError, match="history must be"):
        v.process_logits(lg, lg, history=torch.zeros((3, 3), dtype=i32), history_len=torch.zeros(2, dtype=i32))
    with pytest.raises(ValueError, match="laid out"):
        v.process_logits(lg, lg, bias_ids=torch.zeros((2, 3), dtype=i32), bias_values=torch.zeros((2, 4)))
    with pytest.raises(ValueError, match="allowed needs"):
        v.process_logits(lg, lg, allowed=torch.zeros((2, 1), dtype=i32))
    with pytest.raises(ValueError, match="overlap"):
        v.process_logits(lg, lg, allowed=torch.zeros(9, dtype=i32).as_strided((2, 2), (1, 1)))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        v.process_logits(lg, lg)
    assert f == x.dtype


def test_restated_format():
    """The restatement itself: bf16 rounding against torch's, packing, and a quantization by hand."""
    import torch

    r = np.random.default_rng(0)
    x = np.ldexp(r.standard_normal(20000), r.integers(-140, 128, 20000)).astype(np.float32)
    want = torch.from_numpy(x).bfloat16().float().numpy()
    assert np.array_equal(u.round_to_bf16(x).astype(np.float32), want)
    q, s = u.quantize(np.array([[7.0, -3.5, 0.5, 1.5, -0.49, np.nan]]), 32)
    assert q.tolist() == [[7, -4, 0, 2, 0, 0]] and s.tolist() == [[1.0]]
    assert u.pack(q).tolist() == [[15 | 4 << 4, 8 | 10 << 4, 8 | 8 << 4]]
    assert u.pack(q[:, :3]).tolist() == [[15 | 4 << 4, 8 | 8 << 4]]
    out, tok = u.logits(np.array([[2.0, -2.0, 1.0, 5.0]], np.float32), np.float32,
                        history=np.array([[0, 1, 0, 2]], np.int32), history_len=np.array([4]),
                        prompt_len=np.array([2]), repetition=[2.0], presence=[0.5], frequency=[0.25],
                        bias_ids=np.array([[2, 2]], np.int32), bias_values=np.array([[9.0, 1.0]], np.float32),
                        allowed=np.array([[7]], np.int32))
    assert out.tolist() == [[1.0 - 0.25 - 0.5, -4.0, 0.5 - 0.25 - 0.5 + 1.0, -np.inf]] and tok.tolist() == [2]

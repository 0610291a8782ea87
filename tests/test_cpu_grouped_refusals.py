"""Arguments that the grouped and the four-bit products refuse.  Everything but the device is checked before the device is, so that
these need no GPU: a call that is right up to there is refused for its tensors' place alone."""
import pytest
import torch

from paracel_b200.ops.grouped import aligned, grouped_nn, grouped_nt, grouped_tn, stride_of
from paracel_b200.ops.mx4 import Mx4Matrix, mx4_dequantize, mx4_gemm_nt, mx4_grouped_nt, mx4_quantize

T, E, N, K = 12, 3, 40, 24
H = torch.bfloat16


def _args(**other):
    a = dict(X=torch.zeros(T, K, dtype=H), dY=torch.zeros(T, N, dtype=H), W=torch.zeros(E, N, K, dtype=H),
             offsets=torch.tensor([0, 3, 3, 12]), out=None, out_dtype=None)
    a.update(other)
    return a


def _nt(**o):
    a = _args(**o)
    return grouped_nt(a["X"], a["W"], a["offsets"], a["out"], a["out_dtype"])


def _nn(**o):
    a = _args(**o)
    return grouped_nn(a["dY"], a["W"], a["offsets"], a["out"], a["out_dtype"])


def _tn(**o):
    a = _args(**o)
    return grouped_tn(a["dY"], a["X"], a["offsets"], a["out"], a["out_dtype"])


@pytest.mark.parametrize("call", [_nt, _nn, _tn])
def test_right_arguments_are_refused_for_their_device_only(call):
    with pytest.raises(ValueError, match="CUDA"):
        call()
    with pytest.raises(ValueError, match="CUDA"):
        call(offsets=torch.tensor([0, 3, 3, 12], dtype=torch.int32), out_dtype=torch.float32)


@pytest.mark.parametrize("call, other, words", [
    (_nt, dict(X=torch.zeros(T, K)), "bfloat16 or float16"),
    (_nt, dict(X=torch.zeros(T, K, dtype=torch.float16)), "W must be torch.float16"),
    (_nt, dict(X=torch.zeros(T, K + 1, dtype=H)), "24 columns"),
    (_nt, dict(X=torch.zeros(K, dtype=H)), "2 dimensions"),
    (_nt, dict(W=torch.zeros(N, K, dtype=H)), "3 dimensions"),
    (_nt, dict(W=torch.zeros(E + 1, N, K, dtype=H)), "4 matrices"),
    (_nt, dict(W=torch.zeros(E, 0, K, dtype=H)), "N must be 1"),
    (_nt, dict(W=torch.zeros(E, N, 0, dtype=H), X=torch.zeros(T, 0, dtype=H)), "K must be 1"),
    (_nt, dict(offsets=torch.tensor([0.0, 3, 3, 12])), "int32 or int64"),
    (_nt, dict(offsets=torch.tensor([[0, 3, 3, 12]])), "one-dimensional"),
    (_nt, dict(offsets=torch.arange(8)[::2]), "contiguous"),
    (_nt, dict(offsets=torch.tensor([0])), "2 to 1025"),
    (_nt, dict(offsets=torch.zeros(1026, dtype=torch.int32)), "2 to 1025"),
    (_nt, dict(out=torch.zeros(T, N)), None),
    (_nt, dict(out=torch.zeros(T, N), out_dtype=H), "out must be torch.bfloat16"),
    (_nt, dict(out=torch.zeros(T + 1, N, dtype=H)), "out must be"),
    (_nt, dict(out=torch.zeros(N, T, dtype=H).T), "contiguous rows"),
    (_nt, dict(out=torch.zeros(1, N, dtype=H).expand(T, N)), "contiguous rows"),
    (_nt, dict(out=torch.zeros(T, N, dtype=torch.float16)), "out_dtype"),
    (_nt, dict(out_dtype=torch.float64), "out_dtype"),
    (_nn, dict(dY=torch.zeros(T, K, dtype=H)), "40 columns"),
    (_nn, dict(out=torch.zeros(T, N, dtype=H)), "out must be"),
    (_tn, dict(dY=torch.zeros(T + 1, N, dtype=H)), "13 rows"),
    (_tn, dict(out=torch.zeros(E, K, N, dtype=H)), "out must be"),
    (_tn, dict(out=torch.zeros(E, K, N, dtype=H).transpose(1, 2)), "contiguous"),
])
def test_grouped_refusals(call, other, words):
    with pytest.raises(ValueError, match=words or "CUDA"):
        call(**other)


def _packed(rows, cols):
    return Mx4Matrix(torch.zeros(rows, (cols + 31) // 32 * 16, dtype=torch.uint8),
                     torch.zeros((cols + 127) // 128, rows, 4, dtype=torch.uint8), cols)


@pytest.mark.parametrize("call", [
    lambda: mx4_quantize(torch.zeros(4, 32)),
    lambda: mx4_dequantize(_packed(4, 33)),
    lambda: mx4_gemm_nt(torch.zeros(4, 33, dtype=H), _packed(7, 33)),
    lambda: mx4_gemm_nt(_packed(4, 33), _packed(7, 33), out_dtype=H),
    lambda: mx4_grouped_nt(_packed(4, 33), _packed(9, 33), torch.tensor([0, 1, 1, 4])),
])
def test_right_four_bit_arguments_are_refused_for_their_device_only(call):
    with pytest.raises(ValueError, match="CUDA"):
        call()


@pytest.mark.parametrize("call, words", [
    (lambda: Mx4Matrix(torch.zeros(4, 16), torch.zeros(1, 4, 4, dtype=torch.uint8), 32), "uint8"),
    (lambda: Mx4Matrix(torch.zeros(4, 32, dtype=torch.uint8)[:, ::2], torch.zeros(1, 4, 4, dtype=torch.uint8), 32), "contiguous"),
    (lambda: Mx4Matrix(torch.zeros(65, dtype=torch.uint8)[1:].view(4, 16), torch.zeros(1, 4, 4, dtype=torch.uint8), 32), "16 bytes"),
    (lambda: Mx4Matrix(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(1, 4, 4, dtype=torch.uint8), 33), "data must be"),
    (lambda: Mx4Matrix(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 3, 4, dtype=torch.uint8), 33), "scales must be"),
    (lambda: Mx4Matrix(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 33), "scales must be"),
    (lambda: Mx4Matrix(torch.zeros(4, 0, dtype=torch.uint8), torch.zeros(0, 4, 4, dtype=torch.uint8), 0), "cols must be"),
    (lambda: mx4_quantize(torch.zeros(4, 32, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (lambda: mx4_quantize(torch.zeros(32)), "2 or 3 dimensions"),
    (lambda: mx4_quantize(torch.zeros(4, 0)), "columns"),
    (lambda: mx4_dequantize(_packed(4, 33), torch.float64), "dtype"),
    (lambda: mx4_dequantize(_packed(4, 33), out=torch.zeros(4, 32)), "out must be"),
    (lambda: mx4_dequantize(_packed(4, 33), out=torch.zeros(4, 33, dtype=H)), "out must be"),
    (lambda: mx4_gemm_nt(torch.zeros(4, 33), torch.zeros(7, 33)), "Mx4Matrix"),
    (lambda: mx4_gemm_nt(torch.zeros(4, 34), _packed(7, 33)), "34 columns"),
    (lambda: mx4_gemm_nt(torch.zeros(4, 33, dtype=torch.int32), _packed(7, 33)), "A must be"),
    (lambda: mx4_gemm_nt(torch.zeros(33), _packed(7, 33)), "A must be"),
    (lambda: mx4_gemm_nt(_packed(4, 33), _packed(0, 33)), "at least one"),
    (lambda: mx4_gemm_nt(_packed(4, 33), _packed(7, 33), out_dtype=torch.int32), "out_dtype"),
    (lambda: mx4_gemm_nt(_packed(4, 33), _packed(7, 33), out=torch.zeros(7, 4).T), "contiguous rows"),
    (lambda: mx4_grouped_nt(_packed(4, 33), _packed(7, 33), torch.tensor([0, 1, 1, 4])), "same number of rows"),
    (lambda: mx4_grouped_nt(_packed(4, 33), _packed(9, 33), None), "mx4_gemm_nt"),
    (lambda: mx4_grouped_nt(_packed(4, 33), _packed(9, 33), torch.tensor([0.0, 4.0])), "int32 or int64"),
])
def test_four_bit_refusals(call, words):
    with pytest.raises(ValueError, match=words):
        call()


def test_rows_at_multiples_of_16_bytes():
    x = torch.arange(5 * 24, dtype=torch.float32).to(H).view(5, 24)
    assert aligned(x) is x
    part = x[:, 8:16]
    assert aligned(part) is part and stride_of(part, 0, 8) == 24
    for odd in (x[:, 1:9], torch.zeros(5, 9, dtype=H), x[:, ::2], x[:1].expand(5, 24), x.T):
        y = aligned(odd)
        assert y is not odd and torch.equal(y, odd) and y.stride(0) % 8 == 0 and y.data_ptr() % 16 == 0
    one = torch.zeros(1, 9, dtype=H)
    assert aligned(one) is one and stride_of(one, 0, 16) == 16


def test_copies_of_a_four_bit_matrix_have_memory_of_their_own():
    import copy
    import pickle
    q = _packed(4, 33)
    q.data.fill_(7)
    for other in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert torch.equal(other.data, q.data) and torch.equal(other.scales, q.scales) and other.cols == 33
        assert other._data_ptr == other.data.data_ptr() != q._data_ptr and other._scales_ptr == other.scales.data_ptr()
    assert copy.copy(q).data.data_ptr() == q._data_ptr and q.nbytes() == q.data.numel() + q.scales.numel()

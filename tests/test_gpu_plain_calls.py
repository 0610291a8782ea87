"""The way through Python gives what the module of plain calls gives, to the bit: the kernels are the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,N,K", [(1, 40, 24), (60, 45, 77), (700, 264, 136), (3, 130, 1100)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_calls_through_python_give_the_same_bits(monkeypatch, T, N, K, dtype):
    from paracel_b200.ops import _calls
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt, grouped_tn
    from paracel_b200.ops.mx4 import Mx4Matrix, mx4_dequantize, mx4_gemm_nt, mx4_grouped_nt, mx4_quantize
    g = torch.Generator(device="cuda").manual_seed(1)
    E, f = 3, torch.float32
    X, dY, W = (torch.randn(*s, device="cuda", generator=g).to(dtype) for s in ((T, K), (T, N), (E, N, K)))
    off = torch.tensor([0, T // 3, T // 3, T], device="cuda")

    def run():
        q = mx4_quantize(W)
        assert isinstance(q, Mx4Matrix)
        return (grouped_nt(X, W, off), grouped_nn(dY, W, off, out_dtype=f), grouped_tn(dY, X, off), q.data.clone(), q.scales.clone(),
                mx4_dequantize(q, dtype), mx4_gemm_nt(X, q), mx4_grouped_nt(X, q, off, out_dtype=f), mx4_grouped_nt(mx4_quantize(X), q, off))

    assert not isinstance(_calls.calls(), type)          # the built module
    plain = run()
    monkeypatch.setattr(_calls, "_mod", _calls.LongWay)
    long = run()
    check_status()
    assert all(torch.equal(a, b) for a, b in zip(plain, long))

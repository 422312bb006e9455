"""Every operand of the 4-bit operators and of the gated norm, written by the kernel right before the call: tensor scales, bias,
modulation vectors, rows and packed rows, for the kernels that start before their predecessor has ended."""
import pytest
import torch

from krea_image_b200 import binding as B, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kc():
    k = ops.KreaCuda(0)
    k.set_stream(torch.cuda.current_stream())
    yield k
    k.close()


def _u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("rows", [5, 130, 700])
def test_operands_written_by_the_kernel_before(kc, rows):
    """The chain is run with other values each time, without a pause and behind a long kernel; each result has to be the one that
    the same values give with a synchronisation after every step."""
    K, N = 1032, 520
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randn(rows, K, device="cuda", generator=g)
    w = torch.randn(K, N, device="cuda", generator=g)
    bias, mul, add, gate, post = (torch.randn(n, device="cuda", generator=g) for n in (N, K, K, K, K))
    rbk = ops.fp4_row_bytes(K)
    q, s = _u8(rows, rbk), _u8(ops.fp4_scale_bytes(B.FP4_NV, rows, K))
    wq, ws = _u8(N, rbk), _u8(ops.fp4_scale_bytes(B.FP4_NV, N, K))
    xb, wb, back = torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda"), torch.zeros(K, N, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda")
    ts, wts, hts = (torch.ones(1, device="cuda") for _ in range(3))
    v = [torch.zeros_like(t) for t in (bias, mul, add, gate, post)]
    c16, c32 = torch.zeros(rows, N, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, N, device="cuda")
    res, xo, h = torch.zeros(rows, N, device="cuda"), torch.zeros(rows, K, device="cuda"), torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda")
    big = torch.zeros(64 << 20, device="cuda")

    def chain(f, wait):
        step = torch.cuda.synchronize if wait else (lambda: None)
        if not wait:
            big.add_(1.0)
        for dst, src in zip(v, (bias, mul, add, gate, post)):
            torch.mul(src, f, out=dst)
        torch.mul(w, f, out=wb)
        torch.div(wb.abs().amax().float().reshape(1), 2688, out=wts)
        step()
        kc.fp4_quantize(wb, wq, ws, N, K, N, rbk, B.FP4_NV, tensor_scale=wts, transposed=True)
        step()
        torch.mul(x, f, out=xb)
        torch.div(xb.abs().amax().float().reshape(1), 2688, out=ts)
        step()
        kc.fp4_quantize(xb, q, s, rows, K, K, rbk, B.FP4_NV, tensor_scale=ts)
        step()
        kc.fp4_dequantize(q, s, back, rows, K, rbk, K, B.FP4_NV, tensor_scale=ts)
        step()
        kc.gemm_fp4(q, s, wq, ws, c16, rows, N, K, rbk, rbk, N, B.FP4_NV, epilogue=B.EPI_BIAS_BF16, vec=v[0], a_tensor_scale=ts, w_tensor_scale=wts)
        step()
        torch.mul(bias, f + 1, out=v[0])
        step()
        kc.gemm_fp4(q, s, wq, ws, c32, rows, N, K, rbk, rbk, N, B.FP4_NV, epilogue=B.EPI_BIAS_F32, vec=v[0], a_tensor_scale=ts, w_tensor_scale=wts)
        step()
        torch.mul(x[:, :N], f, out=res)
        torch.mul(bias, f + 2, out=v[0])
        step()
        kc.gemm_fp4(q, s, wq, ws, res, rows, N, K, rbk, rbk, N, B.FP4_NV, epilogue=B.EPI_RESID_GATE, vec=v[0], a_tensor_scale=ts, w_tensor_scale=wts)
        step()
        torch.mul(ts, 3.0, out=hts)
        step()
        kc.gated_norm(x, back, xo, q, rows, K, K, K, K, rbk, post=v[4], gate=v[3], mul=v[1], add=v[2], out=B.OUT_FP4_NV, h_scales=s, h_tensor_scale=hts)
        step()
        kc.fp4_dequantize(q, s, h, rows, K, rbk, K, B.FP4_NV, tensor_scale=hts)
        step()
        kc.gated_norm(xo, h, None, back, rows, K, K, K, 0, K, gate=v[3], mul=v[1])
        return [t.clone() for t in (c16, c32, res, xo, h, back)]

    factors = [0.5, 3.0, 1.0, 0.125]
    want = [chain(f, True) for f in factors]
    got = [chain(f, False) for _ in range(4) for f in factors]
    kc.wait()
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i % 4]))
    assert not any(torch.equal(a, b) for a, b in zip(want[0], want[1]))

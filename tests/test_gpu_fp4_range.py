"""The 4-bit operators at the ends of their documented ranges, against the float64 statement in oracle/fp4_np.py: tensor scales
next to the smallest and the largest f32, and products of two that leave it."""
import numpy as np
import pytest
import torch

from krea_image_b200 import binding as B, ops
from oracle import fp4_np
from tests.test_gpu_fp4 import _dev, _f64, _operand, _quantise
from tests.test_gpu_gated_norm import _case, _run

pytestmark = pytest.mark.gpu

# 6 ts leaves the f32 range above 5.67e37, 1 / (6 ts) below 4.9e-40; 2^-149 is the smallest f32
ENDS = [3.3e38, 1e38, 6e37, 5.7e37, 5.6e37, 2.0 ** 126, 1e37, 1e-37, 2.0 ** -128, 5.1e-40, 4.8e-40, 4e-40, 2.0 ** -131, 2.0 ** -140, 1e-44, 2.0 ** -149]


@pytest.fixture(scope="module")
def kc():
    k = ops.KreaCuda(0)
    k.set_stream(torch.cuda.current_stream())
    yield k
    k.close()


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("ts", ENDS)
def test_quantise_with_tensor_scales_at_the_ends_of_f32(kc, ts, transposed):
    """Blocks with every finite bf16 magnitude as their largest (0 among them), and smaller ones all over the grid beside it."""
    mags = np.arange(0x7F80, dtype=np.int64)
    block = np.maximum(mags[:, None] - 41 * np.arange(16)[None, :], 0).astype(np.uint16)
    block[:, 1::2] |= 0x8000
    bits = block.reshape(-1, 64)
    t = float(np.float32(ts))
    assert 0 < t < np.inf
    want_q, want_s = fp4_np.quantise(_f64(bits), "nv", t)
    q, s = _quantise(kc, bits, "nv", ts, transposed)
    assert np.array_equal(s, fp4_np.lay_out_scales(want_s, "nv", 64))
    assert np.array_equal(q, fp4_np.pack(want_q, 64))


@pytest.mark.parametrize("ts,size", [(3.3e38, 2e37), (1e38, 3e37), (6e37, 1e37), (2.0 ** -131, 1e-37), (4e-40, 1e-37), (1e-44, 1e-38), (2.0 ** -149, 2.0 ** -140), (4e-40, 1.0), (1e38, 1.0)])
@pytest.mark.parametrize("rows,width", [(3, 264), (700, 1000)])
def test_norm_with_tensor_scales_at_the_ends_of_f32(kc, rows, width, ts, size):
    x, y, w, g, mul, add = _case(rows + width, rows, width, 1, False, True, True)
    mul = (mul.astype(np.float64) * size).astype(np.float32)
    mul[:, 32:64] = 0                                        # blocks of zeros
    _, q, s = _run(kc, x, y, w, g, mul, None, "nv", h_ts=ts)
    _, h, _ = _run(kc, x, y, w, g, mul, None, "bf16")
    assert np.isfinite(h).all()
    want_q, want_s = fp4_np.quantise(h, "nv", float(np.float32(ts)))
    assert np.array_equal(s, fp4_np.lay_out_scales(want_s, "nv", width))
    assert np.array_equal(q, fp4_np.pack(want_q, width))


@pytest.fixture(scope="module", params=["0", "1", "2"], ids=["by-size", "rows", "pair"])
def kt(request):
    """A handle whose product kernel is chosen by size, or one of the two for every shape."""
    with pytest.MonkeyPatch.context() as m:
        m.setenv("KREA_CUDA_FP4_TILE", request.param)
        k = ops.KreaCuda(0)
    k.set_stream(torch.cuda.current_stream())
    yield k
    k.close()


# their product below the normal f32 numbers, below the smallest one, above the largest; and two that meet in the middle
PAIRS = [(1e-30, 1e-14), (1e-14, 1e-30), (2.0 ** -70, 2.0 ** -70), (3e-39, 1e-4), (1e-25, 1e-24), (1e25, 1e20), (1e20, 3e25), (3e38, 3e-38), (2.0 ** -149, 1e38)]


@pytest.mark.parametrize("a_ts,w_ts", PAIRS)
@pytest.mark.parametrize("M,N,K", [(1, 128, 512), (40, 264, 512), (300, 520, 512), (2600, 4160, 200)])      # the last: more tiles than CTA pairs
def test_product_with_tensor_scales_whose_product_leaves_f32(kt, M, N, K, a_ts, w_ts):
    """Every block scale is 448: sums are multiples of 224^2 and below 2^24 of them, so that f32 holds them exactly, and what is
    left are two roundings, by 2^-24 or half of the smallest f32 each.  Sums of zero stay zero."""
    rng = np.random.default_rng(M + N)
    qa, qw = rng.integers(0, 16, (M, K)).astype(np.uint8), rng.integers(0, 16, (N, K)).astype(np.uint8)
    qw[::5] = 0
    sc = [np.full((r, -(-K // 16)), 0x7E, np.uint8) for r in (M, N)]
    (A, As, va), (W, Ws, vw) = (_operand(q, c, "nv", K) for q, c in zip((qa, qw), sc))
    a, w = float(np.float32(a_ts)), float(np.float32(w_ts))
    acc = va @ vw.T
    assert (np.abs(va) @ np.abs(vw).T).max() / 224 ** 2 < 2 ** 24
    c = torch.full((M, N), float("nan"), dtype=torch.float32, device="cuda")
    kt.gemm_fp4(A, As, W, Ws, c, M, N, K, A.shape[1], W.shape[1], N, B.FP4_NV, epilogue=B.EPI_F32, a_tensor_scale=_dev(np.float32([a_ts])), w_tensor_scale=_dev(np.float32([w_ts])))
    kt.wait()
    got, want = c.double().cpu().numpy(), acc * a * w
    top = float(np.finfo(np.float32).max)
    over = np.abs(want) > top * (1 + 2.0 ** -22)
    assert np.array_equal(got[over], np.sign(want[over]) * np.inf)
    rest = ~over & (np.abs(want) < top * (1 - 2.0 ** -22))
    # the first of the two roundings is carried along by the second factor: 2^-24 of the result, or half a smallest f32 times a
    # factor below 2^23 (the smaller one, where the product is too small)
    assert (np.abs(got[rest] - want[rest]) <= np.abs(want[rest]) * 2.0 ** -22 + 2.0 ** -148).all()
    assert (got[:, ::5] == 0).all()

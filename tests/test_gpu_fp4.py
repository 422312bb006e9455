"""GPU tests of the 4-bit rows (fp4_quantize, fp4_dequantize) and of the product on them (gemm_fp4) against the float64
statement in oracle/fp4_np.py."""
import os

import numpy as np
import pytest
import torch

from krea_image_b200 import binding as B, ops, synth
from oracle import fp4_np

pytestmark = pytest.mark.gpu
FMT = {"mx": B.FP4_MX, "nv": B.FP4_NV}


@pytest.fixture(scope="module")
def kc():
    k = ops.KreaCuda(0)
    k.set_stream(torch.cuda.current_stream())
    yield k
    k.close()


@pytest.fixture(scope="module", params=["by-size", "rows", "pair"])
def kp(request):
    """The handle of the product's tests: the kernel chosen by size, and each of the two forced on every shape."""
    knob = {"rows": "1", "pair": "2"}.get(request.param)
    if knob:
        os.environ["KREA_CUDA_FP4_TILE"] = knob
    try:
        k = ops.KreaCuda(0)
    finally:
        os.environ.pop("KREA_CUDA_FP4_TILE", None)
    k.set_stream(torch.cuda.current_stream())
    yield k
    k.close()


def _bits(a):
    return synth.f32_to_bf16_bits(np.ascontiguousarray(a, dtype=np.float32)).reshape(a.shape)


def _bf16(bits):
    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int16)).cuda().view(torch.bfloat16)


def _f64(bits):
    return synth.bf16_bits_to_f32(bits).astype(np.float64)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _quantise(kc, bits, fmt, ts=None, transposed=False, pad=8, qpad=16):
    """Runs the kernel on rows (given [rows, K]) inside wider buffers; returns (packed, scales) and checks what must stay."""
    rows, K = bits.shape
    src = bits.T if transposed else bits
    wide = np.full((src.shape[0], -(-src.shape[1] // 8) * 8 + pad), 0x7FC0, dtype=np.uint16)      # NaN around the rows
    wide[:, :src.shape[1]] = src
    rb = ops.fp4_row_bytes(K)
    q = torch.full((rows + 1, rb + qpad), 0xA5, dtype=torch.uint8, device="cuda")
    nb = ops.fp4_scale_bytes(FMT[fmt], rows, K)
    s = torch.full((nb + 32,), 0xA5, dtype=torch.uint8, device="cuda")
    kc.fp4_quantize(_bf16(wide), q, s, rows, K, wide.shape[1], rb + qpad, FMT[fmt], tensor_scale=None if ts is None else _dev(np.float32([ts])), transposed=transposed)
    kc.wait()
    q, s = q.cpu().numpy(), s.cpu().numpy()
    assert (q[:rows, rb:] == 0xA5).all() and (q[rows] == 0xA5).all() and (s[nb:] == 0xA5).all()
    return q[:rows, :rb], s[:nb]


def _rows(rng, rows, K):
    """Values of many sizes, with empty blocks, exact ties and the ends of the range among them."""
    x = rng.standard_normal((rows, K)) * np.exp2(rng.integers(-3, 4, (rows, K)))
    x.flat[rng.integers(0, x.size, x.size // 7)] = 0
    if K >= 16:
        x[rng.integers(0, rows), : K // 16 * 16 // 2] = 0
        ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6])
        r = rng.integers(0, rows)
        x[r, :16] = rng.choice(ties, 16) * rng.choice([-1, 1], 16)
        x[r, 0] = 6
    return _bits(x)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("fmt,ts", [("mx", None), ("nv", None), ("nv", 0.0371), ("nv", 2.0 ** -5), ("nv", 7.40625 / 2688)])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 16), (3, 31), (2, 32), (5, 33), (130, 70), (128, 256), (129, 257), (1, 6144), (300, 1000), (67, 2500), (2000, 4200), (2500, 2600)])
def test_quantise_is_exact(kc, rows, K, fmt, ts, transposed):
    bits = _rows(np.random.default_rng(rows * 31 + K), rows, K)
    t = 1.0 if ts is None else float(np.float32(ts))
    want_q, want_s = fp4_np.quantise(_f64(bits), fmt, t)
    q, s = _quantise(kc, bits, fmt, ts, transposed)
    assert np.array_equal(s, fp4_np.lay_out_scales(want_s, fmt, K))
    assert np.array_equal(q, fp4_np.pack(want_q, K))


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_quantise_every_bf16_magnitude(kc, fmt):
    """Every finite magnitude beside a block maximum of its own size class, so that each lands all over the grid."""
    mags = np.arange(0x7F80, dtype=np.uint16)
    bs = fp4_np.BLOCK[fmt]
    out = []
    for up in (0, 40, 128, 300):                          # how far (in bf16 steps) the maximum is above
        block = np.empty((len(mags), bs), dtype=np.uint16)
        block[:] = np.maximum(mags.astype(np.int64)[:, None] - 37 * np.arange(bs)[None, :], 0)
        block[:, 1] = np.minimum(mags.astype(np.int64) + up, 0x7F7F)
        block[:, 2::2] |= 0x8000
        out.append(block)
    bits = np.concatenate(out).reshape(-1, 4 * bs)
    ts = None if fmt == "mx" else 1.37e-3
    want_q, want_s = fp4_np.quantise(_f64(bits), fmt, 1.0 if ts is None else float(np.float32(ts)))
    q, s = _quantise(kc, bits, fmt, ts, pad=0, qpad=0)
    assert np.array_equal(s, fp4_np.lay_out_scales(want_s, fmt, 4 * bs))
    assert np.array_equal(q, fp4_np.pack(want_q, 4 * bs))


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("transposed", [False, True])
def test_quantise_marks_blocks_that_are_not_finite(kc, fmt, transposed):
    rng = np.random.default_rng(5)
    bits = _bits(rng.standard_normal((9, 200)))
    bits[0, 3], bits[1, 70], bits[4, 199], bits[8, 0] = 0x7F80, 0xFF80, 0x7FC1, 0xFFFF      # inf, -inf, NaN, NaN
    x = _f64(bits)
    want_q, want_s = fp4_np.quantise(x, fmt)
    q, s = _quantise(kc, bits, fmt, None, transposed)
    assert np.array_equal(s, fp4_np.lay_out_scales(want_s, fmt, 200)) and np.array_equal(q, fp4_np.pack(want_q, 200))
    out = torch.zeros((9, 200), dtype=torch.bfloat16, device="cuda")
    kc.fp4_dequantize(_dev(q), _dev(s), out, 9, 200, q.shape[1], 200, FMT[fmt])
    kc.wait()
    bad = np.isnan(out.float().cpu().numpy())
    bs = fp4_np.BLOCK[fmt]
    want = np.zeros_like(bad)
    for r, c in ((0, 3), (1, 70), (4, 199), (8, 0)):
        want[r, c // bs * bs:(c // bs + 1) * bs] = True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("fmt,ts", [("mx", None), ("nv", None), ("nv", 0.0371)])
@pytest.mark.parametrize("rows,K", [(1, 1), (4, 17), (3, 64), (131, 300), (2, 6144)])
def test_dequantise(kc, rows, K, fmt, ts):
    rng = np.random.default_rng(rows + K)
    nb = -(-K // fp4_np.BLOCK[fmt])
    q = rng.integers(0, 16, (rows, K)).astype(np.uint8)
    code = (rng.integers(0, 255, (rows, nb)) if fmt == "mx" else rng.integers(0, 127, (rows, nb))).astype(np.uint8)
    if fmt == "mx":
        code = np.clip(code, 3, 250)                      # all values are bf16 numbers
        code[0, 0] = 0                                    # 2^-127
    t = 1.0 if ts is None else float(np.float32(ts))
    want = fp4_np.values(np.pad(q, ((0, 0), (0, nb * fp4_np.BLOCK[fmt] - K))), code, fmt, K, t)
    ld = -(-K // 8) * 8 + 8
    out = torch.full((rows, ld), 7.0, dtype=torch.bfloat16, device="cuda")
    kc.fp4_dequantize(_dev(fp4_np.pack(q, K)), _dev(fp4_np.lay_out_scales(code, fmt, K)), out, rows, K, ops.fp4_row_bytes(K), ld, FMT[fmt],
                      tensor_scale=None if ts is None else _dev(np.float32([ts])))
    kc.wait()
    got = out.double().cpu().numpy()
    assert (got[:, K:] == 7.0).all()
    # without a tensor scale every value is a bf16 number; with one: f32 product (2^-24), then bf16 (2^-8)
    tol = 0.0 if ts is None else 2.0 ** -8 + 2.0 ** -23
    assert (np.abs(got[:, :K] - want) <= tol * np.abs(want)).all()


# ------------------------------------------------------------------------------------------------- product
def _codes(rng, rows, K, fmt, exact):
    nb = -(-K // fp4_np.BLOCK[fmt])
    q = rng.integers(0, 16, (rows, K)).astype(np.uint8)
    if fmt == "mx":
        code = rng.integers(126, 129, (rows, nb)) if exact else rng.integers(117, 131, (rows, nb))
    else:
        code = rng.choice([0x30, 0x38, 0x40], (rows, nb)) if exact else rng.integers(0, 127, (rows, nb))      # 0.5, 1, 2
    return q, code.astype(np.uint8)


def _operand(q, code, fmt, K, pad=0):
    p = fp4_np.pack(q, K)
    wide = np.full((p.shape[0], p.shape[1] + pad), 0x77, dtype=np.uint8)
    wide[:, :p.shape[1]] = p
    v = fp4_np.values(np.pad(q, ((0, 0), (0, code.shape[1] * fp4_np.BLOCK[fmt] - K))), code, fmt, K)
    return _dev(wide), _dev(fp4_np.lay_out_scales(code, fmt, K)), v


SHAPES = [(1, 8, 1), (1, 128, 256), (1, 136, 70), (3, 64, 31), (16, 128, 512), (17, 256, 300), (33, 200, 1024), (64, 72, 2100), (100, 520, 777), (128, 128, 256), (129, 264, 600),
          (200, 1000, 4096), (257, 512, 256), (300, 520, 200), (512, 768, 1111), (700, 1032, 2048), (1, 2048, 6144), (5, 1024, 6900)]


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_sums_are_exact_where_32_bits_hold_them(kp, M, N, K, fmt):
    """Scales of 1/2, 1 and 2: every product is a multiple of 1/16 and every partial sum stays below 2^20 (K * 36 * 4), so
    that 24 bits hold them all and the result has no rounding at all; each wrong index shows."""
    rng = np.random.default_rng(M + 3 * N + 7 * K)
    qa, ca = _codes(rng, M, K, fmt, True)
    qw, cw = _codes(rng, N, K, fmt, True)
    A, As, va = _operand(qa, ca, fmt, K, 16)
    W, Ws, vw = _operand(qw, cw, fmt, K, 32)
    assert np.abs(va).sum(1).max() * 12 < 2 ** 20
    c = torch.full((M + 1, N + 8), -3.0, dtype=torch.float32, device="cuda")
    n0 = kp.launches
    kp.gemm_fp4(A, As, W, Ws, c, M, N, K, A.shape[1], W.shape[1], N + 8, FMT[fmt], epilogue=B.EPI_F32)
    kp.wait()
    assert kp.launches - n0 == 1
    got = c.cpu().numpy()
    assert np.array_equal(got[:M, :N], (va @ vw.T).astype(np.float32))
    assert (got[M] == -3).all() and (got[:, N:] == -3).all()


def _within(got, want, bound):
    worst = np.max(np.abs(got - want) - bound)
    assert worst <= 0, f"off by {np.abs(got - want).max():.3e}, {worst:.3e} over the bound"


@pytest.mark.parametrize("epilogue", ["bf16", "f32", "bias_bf16", "bias_f32", "gelu", "swiglu", "resid", "resid_gate"])
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("M,N,K", [(1, 192, 300), (40, 320, 1500), (150, 576, 520), (600, 1088, 1000)])
def test_product_epilogues(kp, M, N, K, fmt, epilogue):
    rng = np.random.default_rng(M + N + K)
    qa, ca = _codes(rng, M, K, fmt, False)
    qw, cw = _codes(rng, N, K, fmt, False)
    A, As, va = _operand(qa, ca, fmt, K)
    W, Ws, vw = _operand(qw, cw, fmt, K)
    norm = 1.0 / np.sqrt((va ** 2).mean() * (vw ** 2).mean() * K)
    ats, wts = (None, None) if fmt == "mx" else (np.float32(norm), np.float32(0.75))
    if fmt == "mx":                                       # bring the sums to the size of 1 by whole powers of two
        step = int(np.round(np.log2(norm)))
        cw = (cw.astype(np.int64) + step).astype(np.uint8)
        Ws, vw = _dev(fp4_np.lay_out_scales(cw, fmt, K)), vw * 2.0 ** step
    alpha = 1.0 if fmt == "mx" else float(ats) * float(wts)
    acc, size = va @ vw.T * alpha, np.abs(va) @ np.abs(vw).T * alpha
    # fp32 sums of K terms in any order, truncated at worst: K steps of 2^-23 of the terms' size; two roundings of alpha
    err = size * (K * 2.0 ** -23) + np.abs(acc) * 2.0 ** -22
    vec = rng.standard_normal(N).astype(np.float32)
    x0 = rng.standard_normal((M, N)).astype(np.float32)
    half = 2.0 ** -8                                      # bf16's half step
    kind = {"resid": B.EPI_RESID_GATE, "resid_gate": B.EPI_RESID_GATE}.get(epilogue) or getattr(B, "EPI_" + epilogue.upper())
    cols = N // 2 if epilogue == "swiglu" else N
    f32 = epilogue in ("f32", "bias_f32", "resid", "resid_gate")
    c = _dev(x0) if epilogue.startswith("resid") else torch.full((M, cols), float("nan"), dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    kp.gemm_fp4(A, As, W, Ws, c, M, N, K, A.shape[1], W.shape[1], cols, FMT[fmt], epilogue=kind, vec=None if epilogue in ("bf16", "f32", "gelu", "swiglu", "resid") else _dev(vec),
                a_tensor_scale=None if ats is None else _dev(np.array([ats])), w_tensor_scale=None if wts is None else _dev(np.array([wts])))
    kp.wait()
    got = c.double().cpu().numpy()
    if epilogue.startswith("bias"):
        want = acc + vec
        bound = err + np.abs(want) * 2.0 ** -24
    elif epilogue.startswith("resid"):
        g = vec.astype(np.float64) if epilogue == "resid_gate" else 1.0
        want = x0 + g * acc
        bound = np.abs(g) * err + np.abs(want) * 2.0 ** -24
    elif epilogue == "gelu":
        want = 0.5 * acc * (1 + np.tanh(np.sqrt(2 / np.pi) * (acc + 0.044715 * acc ** 3)))
        # the slope of gelu is 1.13 at most; 1 + tanh cancels for negative values: 4 steps of 2^-24 of |x|
        bound = 1.13 * err + np.abs(acc) * 2.0 ** -21
    elif epilogue == "swiglu":
        pair, e = acc.reshape(M, -1, 2, 32), err.reshape(M, -1, 2, 32)
        g, u = pair[:, :, 0], pair[:, :, 1]
        silu = g / (1 + np.exp(-g))
        want = (silu * u).reshape(M, cols)
        # slope of silu 1.1 at most; exp2 and the reciprocal of the sigmoid are good to 2^-21
        bound = (1.1 * e[:, :, 0] * np.abs(u) + np.abs(silu) * e[:, :, 1] + np.abs(silu * u) * 2.0 ** -20).reshape(M, cols)
    else:
        want, bound = acc, err
    if not f32:
        bound = bound + np.abs(want) * half * (1 + 2.0 ** -8) + bound * half
    _within(got, want, bound)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("M,N,K", [(1, 256, 2048), (70, 264, 600), (520, 512, 768)])
def test_product_carries_what_is_not_finite(kp, M, N, K, fmt):
    """A block scale of NaN makes its row of A (its column of C, for W) NaN and nothing else; scales past the last row are
    padding that reaches no result."""
    rng = np.random.default_rng(11)
    qa, ca = _codes(rng, M, K, fmt, True)
    qw, cw = _codes(rng, N, K, fmt, True)
    nan = 255 if fmt == "mx" else 127
    ca[M // 2, 1] = nan
    cw[N - 3, 0] = nan
    A, As, va = _operand(qa, ca, fmt, K)
    W, Ws, vw = _operand(qw, cw, fmt, K)
    # NaN in the scales of rows that do not exist
    for t, rows in ((As, M), (Ws, N)):
        v = t.cpu().numpy()
        for r in range(rows, -(-rows // 128) * 128):
            v[fp4_np.scale_index(r, np.arange(-(-K // fp4_np.BLOCK[fmt])), fmt, K)] = nan
        t.copy_(_dev(v))
    c = torch.zeros((M, N), dtype=torch.float32, device="cuda")
    kp.gemm_fp4(A, As, W, Ws, c, M, N, K, A.shape[1], W.shape[1], N, FMT[fmt], epilogue=B.EPI_F32)
    kp.wait()
    got = c.cpu().numpy()
    want = (np.nan_to_num(va) @ np.nan_to_num(vw).T).astype(np.float32)
    want[M // 2, :] = np.nan
    want[:, N - 3] = np.nan
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("epilogue", ["f32", "bf16", "swiglu", "resid_gate"])
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("M,N,K", [(2600, 4160, 520), (4700, 2112, 1300)])
def test_many_tiles_a_worker(kp, M, N, K, fmt, epilogue):
    """More tiles than CTA pairs and rows beyond one wave: accumulator, ring and output boxes are used again and again.  Sums
    are exact in 32 bits (see above), so the plain epilogues are too; SwiGLU adds a sigmoid and a rounding."""
    rng = np.random.default_rng(M + N)
    qa, ca = _codes(rng, M, K, fmt, True)
    qw, cw = _codes(rng, N, K, fmt, True)
    A, As, va = _operand(qa, ca, fmt, K)
    W, Ws, vw = _operand(qw, cw, fmt, K)
    want = _dev(va) @ _dev(vw).T
    vec = torch.from_numpy(rng.integers(-3, 4, N).astype(np.float32)).cuda()
    cols = N // 2 if epilogue == "swiglu" else N
    f32 = epilogue in ("f32", "resid_gate")
    c = torch.full((M + 1, cols), 5.0, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    kind = {"f32": B.EPI_F32, "bf16": B.EPI_BF16, "swiglu": B.EPI_SWIGLU, "resid_gate": B.EPI_RESID_GATE}[epilogue]
    for _ in range(2):
        c.fill_(5.0)
        kp.gemm_fp4(A, As, W, Ws, c, M, N, K, A.shape[1], W.shape[1], cols, FMT[fmt], epilogue=kind, vec=vec if epilogue == "resid_gate" else None)
    kp.wait()
    assert (c[M] == 5).all()
    got = c[:M]
    if epilogue == "f32":
        assert torch.equal(got, want.float())
    elif epilogue == "bf16":
        assert torch.equal(got, want.float().bfloat16())
    elif epilogue == "resid_gate":                    # 3 * 2^20 + 5 in steps of 1/16: exact as well
        assert torch.equal(got, (5 + vec.double() * want).float())
    else:
        pair = want.view(M, -1, 2, 32)
        ref = (pair[:, :, 0] / (1 + torch.exp(-pair[:, :, 0])) * pair[:, :, 1]).reshape(M, cols)
        # exp2's argument -g / ln 2 is below 128 where the sigmoid is not flushed to zero (at 2^-126): its two roundings of
        # 2^-24 move the result by 128 * 2 * 2^-24 * ln 2 < 2^-16
        flushed = (pair[:, :, 0] * pair[:, :, 1]).abs().reshape(M, cols) * 2.0 ** -126
        assert ((got.double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -16) + flushed).all()


def test_refusals_reach_the_caller(kc):
    t = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    n0 = kc.launches
    for call in (lambda: kc.fp4_quantize(t, t[1024:], t[2048:], 2, 32, 30, 16), lambda: kc.fp4_dequantize(t, t[1024:], t[2048:], 2, 32, 8, 32),
                 lambda: kc.gemm_fp4(t, t[1024:], t[2048:], t[3072:], t[512:], 2, 12, 32, 16, 16, 12)):
        with pytest.raises(ops.KreaCudaError) as e:
            call()
        assert e.value.code == B.E_ARG
    with pytest.raises(ops.KreaCudaError) as e:
        kc.gemm_fp4(t, t[1024:], t[2048:], t[3072:], t[512:], 2, 128, 32, 16, 16, 128, epilogue=B.EPI_QKNORM_ROPE)
    assert e.value.code == B.E_UNSUPPORTED
    kc.fp4_quantize(None, None, None, 0, 32, 32, 16)                     # nothing to do is no error
    kc.gemm_fp4(None, None, None, None, None, 0, 8, 32, 16, 16, 8)
    assert kc.launches == n0

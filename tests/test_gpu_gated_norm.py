"""GPU tests of gated_norm (the norms either side of a sublayer boundary with its gate and residual scale) against the
float64 statement in oracle/fp4_np.py."""
import numpy as np
import pytest
import torch

from krea_image_b200 import binding as B, ops, synth
from oracle import fp4_np

pytestmark = pytest.mark.gpu
OUT = {"bf16": B.OUT_BF16, "f32": B.OUT_F32, "mx": B.OUT_FP4_MX, "nv": B.OUT_FP4_NV}
EPS = 1e-6


@pytest.fixture(scope="module")
def kc():
    k = ops.KreaCuda(0)
    k.set_stream(torch.cuda.current_stream())
    yield k
    k.close()


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _case(seed, rows, width, samples, y_f32, post, gate):
    rng = np.random.default_rng(seed)
    x = 3.0 * rng.standard_normal((rows, width)).astype(np.float32)
    y = rng.standard_normal((rows, width)).astype(np.float32)
    if not y_f32:
        y = synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(y)).reshape(y.shape)
    vec = lambda m, d: (m + d * rng.standard_normal((samples, width))).astype(np.float32)  # noqa: E731
    return x, y, vec(1, 0.3)[0] if post else None, vec(0, 0.8) if gate else None, vec(1, 0.3), vec(0, 0.2)


def _wide(a, pad, dtype=torch.float32, fill=float("nan")):
    t = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=dtype, device="cuda")
    t[:, :a.shape[1]] = _dev(a).to(dtype)
    return t


def _run(kc, x, y, post, gate, mul, add, out, *, x_scale=1.0, mod_rows=0, y_f32=False, pad=8, in_place=False, h_ts=None, eps=EPS):
    rows, width = x.shape
    X = _wide(x, pad)
    Y = None if y is None else _wide(y, pad, torch.float32 if y_f32 else torch.bfloat16)
    XO = X if in_place else torch.full((rows + 1, width + pad), -7.0, device="cuda")
    d = lambda v: None if v is None else _dev(v)  # noqa: E731
    scales = None
    if out in ("mx", "nv"):
        rb = ops.fp4_row_bytes(width)
        H = torch.full((rows + 1, rb + 16), 0xA5, dtype=torch.uint8, device="cuda")
        nb = ops.fp4_scale_bytes(B.FP4_MX if out == "mx" else B.FP4_NV, rows, width)
        scales = torch.full((nb + 16,), 0xA5, dtype=torch.uint8, device="cuda")
    else:
        H = torch.full((rows + 1, width + 8), -7.0, dtype=torch.bfloat16 if out == "bf16" else torch.float32, device="cuda")
    n0 = kc.launches
    kc.gated_norm(X, Y, XO, H, rows, width, X.shape[1], 0 if y is None else Y.shape[1], XO.shape[1], H.shape[1], post=d(post), gate=d(gate), mul=d(mul), add=d(add), x_scale=x_scale,
                  eps=eps, mod_rows=mod_rows, mod_ld=width if mod_rows else 0, y_f32=y_f32, out=OUT[out], h_scales=scales, h_tensor_scale=None if h_ts is None else _dev(np.float32([h_ts])))
    kc.wait()
    assert kc.launches - n0 == 1
    xo, h = XO.cpu().float().numpy(), H.cpu()
    if in_place:
        assert np.isnan(xo[:, width:]).all()
    else:
        assert (xo[rows] == -7).all() and (xo[:, width:] == -7).all()
    if scales is not None:
        h, s = h.numpy(), scales.cpu().numpy()
        assert (h[rows] == 0xA5).all() and (h[:, rb:] == 0xA5).all() and (s[nb:] == 0xA5).all()
        return xo[:rows, :width], h[:rows, :rb], s[:nb]
    h = h.double().numpy()
    assert (h[rows] == -7).all() and (h[:, width:] == -7).all()
    return xo[:rows, :width], h[:rows, :width], None


def _check(got_x, got_h, want_x, want_h, x, y, mul, add, width, out, r, g):
    """Bounds from the roundings: the sum of squares (32 terms a thread, five levels in a warp, 32 warps: at most 69 steps
    of 2^-24 on positive terms), halved by the square root; rsqrt 2^-22; a handful of products and sums."""
    rel_norm = 35 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -23
    size_x = np.abs(x) + np.abs(g * r)
    err_x = size_x * 4 * 2.0 ** -24 + np.abs(g * r) * rel_norm
    assert (np.abs(got_x - want_x) <= err_x).all()
    inv = 1 / np.sqrt((want_x ** 2).mean(1, keepdims=True) + EPS)
    # an error of x' moves the row's norm too: by the row's relative error at most
    row = np.sqrt((err_x ** 2).sum(1, keepdims=True) / (want_x ** 2).sum(1, keepdims=True))
    err_h = np.abs(mul) * inv * (err_x + np.abs(want_x) * (rel_norm + row)) + (np.abs(want_h) + np.abs(add)) * 3 * 2.0 ** -24
    if out == "bf16":
        err_h = err_h * (1 + 2.0 ** -8) + np.abs(want_h) * 2.0 ** -8
    assert (np.abs(got_h - want_h) <= err_h).all()


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,samples,y_f32,post,gate,x_scale", [
    (1, 8, 1, False, True, True, 1.0), (1, 6144, 1, False, False, True, 1.0), (5, 264, 1, True, True, False, 0.5), (6, 1024, 3, False, True, True, 1.0), (9, 1032, 1, True, False, False, -2.0),
    (4, 4104, 2, False, True, True, 0.25), (131, 2560, 1, False, False, True, 1.0), (3, 8200, 1, True, True, True, 1.0), (2, 16384, 1, False, True, True, 1.0), (2, 32768, 2, False, True, True, 0.7)])
def test_gated_norm(kc, rows, width, samples, y_f32, post, gate, x_scale, out):
    x, y, w, g, mul, add = _case(rows + width, rows, width, samples, y_f32, post, gate)
    per = rows // samples if samples > 1 else 0
    f = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
    want_x, want_h = fp4_np.gated_norm(f(x), f(y), f(w), f(g), f(mul), f(add), x_scale, EPS, per)
    got_x, got_h, _ = _run(kc, x, y, w, g, mul, add, out, x_scale=x_scale, mod_rows=per, y_f32=y_f32)
    at = np.arange(rows) // per if per else np.zeros(rows, dtype=int)
    r = y if w is None else y / np.sqrt((f(y) ** 2).mean(1, keepdims=True) + EPS) * w
    _check(got_x, got_h, want_x, want_h, x_scale * x, y, mul[at], add[at], width, out, r, 1.0 if g is None else g[at])


def test_without_a_sublayer_it_is_the_row_norm(kc):
    """y NULL: the same bits as rms_norm; and without h only the residual is written."""
    rng = np.random.default_rng(3)
    rows, width = 37, 6144
    x, mul, add = rng.standard_normal((rows, width)).astype(np.float32), rng.standard_normal(width).astype(np.float32), rng.standard_normal(width).astype(np.float32)
    h = torch.zeros((rows, width), device="cuda")
    kc.gated_norm(_dev(x), None, None, h, rows, width, width, 0, 0, width, mul=_dev(mul), add=_dev(add), out=B.OUT_F32)
    y = torch.zeros((rows, width), device="cuda")
    kc.rms_norm(_dev(x), _dev(mul), _dev(add), y, rows, width, width, width, 1e-6, True)
    xo = torch.zeros((rows, width), device="cuda")
    yb = torch.randn(rows, width, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    kc.gated_norm(_dev(x), yb, xo, None, rows, width, width, width, width, 0, x_scale=0.5)
    kc.wait()
    want = x.astype(np.float64) / np.sqrt((x.astype(np.float64) ** 2).mean(1, keepdims=True) + 1e-6) * mul + add
    # the two kernels add the squares in different orders: both within 35 steps of 2^-24 and rsqrt's 2^-22
    tol = np.abs(want - add) * (35 * 2.0 ** -24 + 2.0 ** -22) + (np.abs(want) + np.abs(add)) * 2.0 ** -22
    for t in (h, y):
        assert (np.abs(t.cpu().numpy() - want) <= tol).all()
    assert torch.equal(xo, torch.addcmul(yb.float(), _dev(x), torch.tensor(0.5, device="cuda")))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("out,ts", [("mx", None), ("nv", None), ("nv", 0.0031)])
@pytest.mark.parametrize("rows,width", [(1, 8), (3, 264), (128, 256), (130, 1000), (5, 4120), (70, 6144), (2, 16392)])
def test_four_bit_output_is_the_quantised_bf16_output(kc, rows, width, out, ts, in_place):
    x, y, w, g, mul, add = _case(rows * 3 + width, rows, width, 1, False, True, True)
    xo, q, s = _run(kc, x, y, w, g, mul, add, out, in_place=in_place, h_ts=ts)
    xb, h, _ = _run(kc, x, y, w, g, mul, add, "bf16", in_place=in_place)
    assert np.array_equal(xo, xb)
    want_q, want_s = fp4_np.quantise(h, out, 1.0 if ts is None else float(np.float32(ts)))
    assert np.array_equal(s, fp4_np.lay_out_scales(want_s, out, width))
    assert np.array_equal(q, fp4_np.pack(want_q, width))


def test_rows_that_are_not_finite_stay_apart(kc):
    rows, width = 6, 520
    x, y, w, g, mul, add = _case(9, rows, width, 1, False, True, True)
    clean = _run(kc, x, y, w, g, mul, add, "f32")
    x[2, 5], y[4, 100] = np.inf, np.nan
    xo, h, _ = _run(kc, x, y, w, g, mul, add, "f32")
    keep = [0, 1, 3, 5]
    assert np.array_equal(xo[keep], clean[0][keep]) and np.array_equal(h[keep], clean[1][keep])
    assert np.isinf(xo[2, 5]) and np.isnan(h[4]).all() and np.isnan(h[2, 5])
    # rows of zeros stay finite: eps keeps the norm away from a division by zero
    z = np.zeros((2, width), np.float32)
    xo, h, _ = _run(kc, z, z, w, g[:1], mul, add, "f32")
    assert (xo == 0).all() and np.allclose(h, add, atol=0)


def test_refusals_reach_the_caller(kc):
    t = torch.zeros(4096, device="cuda")
    n0 = kc.launches
    with pytest.raises(ops.KreaCudaError) as e:
        kc.gated_norm(t, t[1024:], t[2048:], t[3072:], 2, 12, 16, 16, 16, 16, mul=t[500:])
    assert e.value.code == B.E_ARG
    kc.gated_norm(None, None, None, None, 0, 8, 8, 8, 8, 8)
    assert kc.launches == n0


@pytest.mark.parametrize("pad", [4, 8])
@pytest.mark.parametrize("out", ["bf16", "f32", "mx", "nv"])
@pytest.mark.parametrize("rows,width,samples,y_f32,post", [(700, 264, 1, False, True), (900, 520, 3, True, True), (2001, 2568, 3, False, False), (61000, 16, 2, False, True), (299, 8200, 1, True, False),
                                                           (300, 12304, 2, False, True)])
def test_many_rows(kc, rows, width, samples, y_f32, post, out, pad):
    """Enough rows that a CTA takes several, samples that end within its share, and rows that start on 16 bytes but not on 32
    (pad 4) as well as on 32 (pad 8): chosen rows against float64, and 4-bit rows against the bf16 rows of the same call."""
    pad_y = 8 if pad == 4 and not y_f32 else pad        # bf16 rows start on 16 bytes all the same
    rng = np.random.default_rng(rows + width)
    per = -(-rows // samples)
    x, y = rng.standard_normal((rows, width), dtype=np.float32), rng.standard_normal((rows, width), dtype=np.float32)
    if not y_f32:
        y = synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(y)).reshape(y.shape)
    vec = lambda m, d: (m + d * rng.standard_normal((samples, width))).astype(np.float32)  # noqa: E731
    w, gate, mul, add = vec(1, .3)[0] if post else None, vec(0, .8), vec(1, .3), vec(0, .2)
    X, Y = _wide(x, pad), _wide(y, pad_y, torch.float32 if y_f32 else torch.bfloat16)
    D = [None if v is None else _dev(v) for v in (w, gate, mul, add)]

    def run(kind):
        XO = torch.full((rows, width + pad), -7.0, device="cuda")
        S = None
        if kind in ("mx", "nv"):
            H = torch.full((rows, ops.fp4_row_bytes(width) + 16), 0xA5, dtype=torch.uint8, device="cuda")
            S = torch.full((ops.fp4_scale_bytes(B.FP4_MX if kind == "mx" else B.FP4_NV, rows, width),), 0xA5, dtype=torch.uint8, device="cuda")
        else:
            H = torch.full((rows, width + 8), -7.0, dtype=torch.bfloat16 if kind == "bf16" else torch.float32, device="cuda")
        kc.gated_norm(X, Y, XO, H, rows, width, width + pad, width + pad_y, width + pad, H.shape[1], post=D[0], gate=D[1], mul=D[2], add=D[3], x_scale=0.5, eps=EPS,
                      mod_rows=per, mod_ld=width, y_f32=y_f32, out=OUT[kind], h_scales=S)
        kc.wait()
        assert (XO[:, width:] == -7).all()
        return XO[:, :width], H, S

    XO, H, S = run(out)
    picks = sorted({0, 1, 127, per - 1, min(per, rows - 1), rows // 2, rows - 129, rows - 1})
    if out in ("mx", "nv"):
        rb = ops.fp4_row_bytes(width)
        XB, HB, _ = run("bf16")
        assert torch.equal(XO, XB) and (H[:, rb:] == 0xA5).all()
        want_q, want_s = fp4_np.quantise(HB[:, :width].double().cpu().numpy(), out)
        assert np.array_equal(H[:, :rb].cpu().numpy(), fp4_np.pack(want_q, width))
        assert np.array_equal(S.cpu().numpy(), fp4_np.lay_out_scales(want_s, out, width))
        return
    assert (H[:, width:] == -7).all()
    f = lambda v: v.astype(np.float64)  # noqa: E731
    at = np.array(picks) // per
    for i, r in enumerate(picks):
        a = at[i]
        want_x, want_h = fp4_np.gated_norm(f(x[r:r + 1]), f(y[r:r + 1]), None if w is None else f(w), f(gate[a:a + 1]), f(mul[a:a + 1]), f(add[a:a + 1]), 0.5, EPS, 0)
        yr = y[r:r + 1] if w is None else y[r:r + 1] / np.sqrt((f(y[r:r + 1]) ** 2).mean(1, keepdims=True) + EPS) * w
        _check(XO[r:r + 1].cpu().numpy(), H[r:r + 1, :width].double().cpu().numpy(), want_x, want_h, 0.5 * x[r:r + 1], y[r:r + 1], mul[a:a + 1], add[a:a + 1], width, out, yr, gate[a:a + 1])

@pytest.mark.parametrize("out", ["mx", "nv"])
@pytest.mark.parametrize("rows,width,post", [(6, 8, True), (6, 264, False), (7, 520, True), (130, 1000, True), (700, 520, True), (700, 1000, False), (6, 4120, True), (700, 8200, True), (6, 8200, False), (6, 16392, True)])
def test_scales_past_the_width_stay_zero_in_rows_that_are_not_finite(kc, rows, width, post, out):
    """Rows with a NaN, with an infinity, and of zeros without an eps: the 4-bit rows are the quantised bf16 rows, and past the width
    there is nothing but zeros."""
    x, y, w, g, mul, add = _case(rows + width, rows, width, 1, False, post, True)
    x[1, 3], x[2, 5], y[4, width - 1], y[5, 0] = np.nan, np.inf, np.nan, -np.inf
    for eps in (EPS, 0.0):
        if eps == 0:
            x[3], y[3] = 0, 0
        xo, q, s = _run(kc, x, y, w, g, mul, add, out, eps=eps)
        xb, h, _ = _run(kc, x, y, w, g, mul, add, "bf16", eps=eps)
        assert np.array_equal(xo, xb, equal_nan=True) and np.isnan(h).any()
        want_q, want_s = fp4_np.quantise(h, out)
        assert np.array_equal(s, fp4_np.lay_out_scales(want_s, out, width))
        assert np.array_equal(q, fp4_np.pack(want_q, width))


@pytest.mark.parametrize("rows,width", [(3, 40), (130, 1000), (700, 2568), (400, 8200)])
def test_rows_side_by_side_in_one_buffer(kc, rows, width):
    """x beside x_out and y beside h, each pair as column slices of one buffer: the same bits as apart, nothing else written."""
    g = torch.Generator("cuda").manual_seed(rows)
    x, y = torch.randn(rows, width, device="cuda", generator=g), torch.randn(rows, width, device="cuda", generator=g).bfloat16()
    gate, mul, add = (torch.randn(width, device="cuda", generator=g) for _ in range(3))
    xo, h = torch.empty_like(x), torch.empty_like(y)
    kc.gated_norm(x, y, xo, h, rows, width, width, width, width, width, gate=gate, mul=mul, add=add)
    ld = 2 * width + 24
    a, b = torch.full((rows, ld), 9.0, device="cuda"), torch.full((rows, ld), 9.0, dtype=torch.bfloat16, device="cuda")
    for first in (0, width + 8):                           # the input before the output, and behind it
        second = width + 8 - first
        a.fill_(9.0), b.fill_(9.0)
        a[:, first:first + width], b[:, first:first + width] = x, y
        kc.gated_norm(a[:, first:], b[:, first:], a[:, second:], b[:, second:], rows, width, ld, ld, ld, ld, gate=gate, mul=mul, add=add)
        kc.wait()
        assert torch.equal(a[:, second:second + width], xo) and torch.equal(b[:, second:second + width], h)
        assert torch.equal(a[:, first:first + width], x) and torch.equal(b[:, first:first + width], y)
        assert (a[:, width:width + 8] == 9).all() and (b[:, 2 * width + 8:] == 9).all() and (a[:, 2 * width + 8:] == 9).all()

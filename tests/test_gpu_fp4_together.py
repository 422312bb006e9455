"""The 4-bit operators and the gated norm as a program uses them: a whole block of them with the attention between, in and
out of CUDA graphs, on other streams, beside one another, and at offsets beyond 32 bits."""
import numpy as np
import pytest
import torch

from krea_image_b200 import binding as B, ops, synth
from oracle import fp4_np

pytestmark = pytest.mark.gpu
FMT = {"mx": B.FP4_MX, "nv": B.FP4_NV}
NORM_OUT = {"mx": B.OUT_FP4_MX, "nv": B.OUT_FP4_NV}


@pytest.fixture(scope="module")
def kc():
    k = ops.KreaCuda(0)
    k.set_stream(torch.cuda.current_stream())
    yield k
    k.close()


def _u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8, device="cuda")


class Block:
    """A DiT block of 4-bit products: weights quantised once from input-major bf16, buffers for one number of rows."""

    def __init__(self, kc, fmt, seed, rows=300, heads=4, kv=2, ff=448):
        g = torch.Generator("cuda").manual_seed(seed)
        self.fmt, self.S, self.heads, self.kv, self.ff, self.D = fmt, rows, heads, kv, ff, heads * 128
        D, self.QC = self.D, (2 * heads + 2 * kv) * 128
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.x0 = rnd(rows, D)
        self.mods = torch.stack([1 + .2 * rnd(D), .1 * rnd(D), torch.tanh(rnd(D)), 1 + .2 * rnd(D), .1 * rnd(D), torch.tanh(rnd(D))])
        self.qn, self.kn = 1 + .2 * rnd(128), 1 + .2 * rnd(128)
        cos, sin = synth.rope_tables_axial2d(rows - 240, 15, 16)
        self.cos, self.sin = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
        self.w = {}
        for name, K, N in (("qkvg", D, self.QC), ("o", D, D), ("gu", D, 2 * ff), ("down", ff, D)):
            wt = (rnd(K, N) / K ** .5).bfloat16()
            ts = (wt.abs().amax().float() / 2688).reshape(1) if fmt == "nv" else None
            q, s = _u8(N, ops.fp4_row_bytes(K)), _u8(ops.fp4_scale_bytes(FMT[fmt], N, K))
            kc.fp4_quantize(wt, q, s, N, K, N, q.shape[1], FMT[fmt], tensor_scale=ts, transposed=True)
            self.w[name] = (q, s, ts, wt)
        self.x = torch.empty_like(self.x0)
        self.h = [(_u8(rows, ops.fp4_row_bytes(K)), _u8(ops.fp4_scale_bytes(FMT[fmt], rows, K))) for K in (D, D, D, ff)]
        bf = lambda n: torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        self.qkvg, self.ao, self.y, self.mid = bf(self.QC), bf(D), bf(D), bf(ff)
        # K is normalised into memory of the block's own: the handle's would be shared by two captured blocks
        self.kscr = _u8(kc.joint_scratch_bytes(rows, heads, heads // kv))

    def product(self, kc, h, K, w, out, epilogue=B.EPI_BF16, vec=None):
        q, s, ts, _ = self.w[w]
        kc.gemm_fp4(h[0], h[1], q, s, out, self.S, q.shape[0], K, h[0].shape[1], q.shape[1], out.shape[1], FMT[self.fmt], epilogue=epilogue, vec=vec, w_tensor_scale=ts)

    def run(self, kc):
        S, D, QC, m, f = self.S, self.D, self.QC, self.mods, FMT[self.fmt]
        kc.gated_norm(self.x0, None, self.x, self.h[0][0], S, D, D, 0, D, self.h[0][0].shape[1], mul=m[0], add=m[1], out=NORM_OUT[self.fmt], h_scales=self.h[0][1])
        self.product(kc, self.h[0], D, "qkvg", self.qkvg)
        r = self.qkvg.view(-1)
        kc.joint_attention(r, r[D:], r[D + self.kv * 128:], self.ao, S, S, self.heads, QC, QC, QC, D, self.qn, self.kn, self.cos, self.sin, 1e-6, self.heads // self.kv,
                           G=r[D + 2 * self.kv * 128:], ldg=QC, k_scratch=self.kscr, k_scratch_bytes=self.kscr.numel())
        kc.fp4_quantize(self.ao, self.h[1][0], self.h[1][1], S, D, D, self.h[1][0].shape[1], f)
        self.product(kc, self.h[1], D, "o", self.y)
        kc.gated_norm(self.x, self.y, self.x, self.h[2][0], S, D, D, D, D, self.h[2][0].shape[1], gate=m[2], mul=m[3], add=m[4], out=NORM_OUT[self.fmt], h_scales=self.h[2][1])
        self.product(kc, self.h[2], D, "gu", self.mid, B.EPI_SWIGLU)
        kc.fp4_quantize(self.mid, self.h[3][0], self.h[3][1], S, self.ff, self.ff, self.h[3][0].shape[1], f)
        self.product(kc, self.h[3], self.ff, "down", self.x, B.EPI_RESID_GATE, m[5])

    def outputs(self):
        return [self.x, self.qkvg, self.ao, self.y, self.mid] + [t for h in self.h for t in h]


def _f64(t):
    return t.double().cpu().numpy()


def _values(h, rows, K, fmt, ts=None):
    """What packed rows stand for, in float64."""
    q, s = h[0].cpu().numpy(), h[1].cpu().numpy()
    codes = np.stack([q & 15, q >> 4], -1).reshape(rows, -1)
    nb = -(-K // fp4_np.BLOCK[fmt])
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    return fp4_np.values(codes[:, :nb * fp4_np.BLOCK[fmt]], s[fp4_np.scale_index(r, b, fmt, K)], fmt, K, 1.0 if ts is None else float(ts.item()))


def _same_rows(h, bf16_rows, fmt):
    """h holds exactly the quantised form of these bf16 rows."""
    q, s = fp4_np.quantise(bf16_rows, fmt)
    K = bf16_rows.shape[1]
    assert np.array_equal(h[0].cpu().numpy(), fp4_np.pack(q, K)) and np.array_equal(h[1].cpu().numpy(), fp4_np.lay_out_scales(s, fmt, K))


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_a_block_step_by_step(kc, fmt):
    """Each step of the block against the float64 statement on what the step before really left."""
    b = Block(kc, fmt, 3)
    b.run(kc)
    kc.wait()
    S, D, ff = b.S, b.D, b.ff
    m = _f64(b.mods)
    half = 2.0 ** -8
    w = {n: _values(t[:2], t[0].shape[0], K, fmt, t[2]) for (n, t), K in zip(b.w.items(), (D, D, D, ff))}
    for n, t in b.w.items():                        # weights: the bf16 matrix, transposed and quantised
        q, s = fp4_np.quantise(_f64(t[3]).T, fmt, 1.0 if t[2] is None else float(t[2].item()))
        assert np.array_equal(t[0].cpu().numpy(), fp4_np.pack(q, q.shape[1] if q.shape[1] == t[3].shape[0] else t[3].shape[0]))
        assert np.array_equal(t[1].cpu().numpy(), fp4_np.lay_out_scales(s, fmt, t[3].shape[0]))

    def close(got, want, size, K):
        err = size * (K + 4) * 2.0 ** -23          # fp32 sums, truncated at worst
        assert (np.abs(got - want) <= err + np.abs(want) * half * (1 + half)).all()

    h0, h1, h2, h3 = (_values(h, S, K, fmt) for h, K in zip(b.h, (D, D, D, ff)))
    # the first norm: its bf16 rows, rounded again
    hb = torch.zeros(S, D, dtype=torch.bfloat16, device="cuda")
    kc.gated_norm(b.x0, None, None, hb, S, D, D, 0, 0, D, mul=b.mods[0], add=b.mods[1])
    kc.wait()
    _same_rows(b.h[0], _f64(hb), fmt)
    _, want = fp4_np.gated_norm(_f64(b.x0), None, mul=m[0:1], add=m[1:2])
    assert (np.abs(_f64(hb) - want) <= np.abs(want) * half * 1.01 + 2.0 ** -18 * (np.abs(m[0]) * 6 + np.abs(m[1]))).all()
    close(_f64(b.qkvg), h0 @ w["qkvg"].T, np.abs(h0) @ np.abs(w["qkvg"]).T, D)
    _same_rows(b.h[1], _f64(b.ao), fmt)
    close(_f64(b.y), h1 @ w["o"].T, np.abs(h1) @ np.abs(w["o"]).T, D)
    # gate and residual: one rounding of the product with the gate, one of the sum
    x1 = _f64(b.x0) + m[2] * _f64(b.y)
    xr = torch.empty_like(b.x0)
    kc.gated_norm(b.x0, b.y, xr, hb, S, D, D, D, D, D, gate=b.mods[2], mul=b.mods[3], add=b.mods[4])
    kc.wait()
    assert (np.abs(_f64(xr) - x1) <= (np.abs(x1) + np.abs(m[2] * _f64(b.y))) * 2.0 ** -23).all()
    _same_rows(b.h[2], _f64(hb), fmt)
    gu = (h2 @ w["gu"].T).reshape(S, -1, 2, 32)
    size = (np.abs(h2) @ np.abs(w["gu"]).T).reshape(S, -1, 2, 32) * (D + 4) * 2.0 ** -23
    silu = gu[:, :, 0] / (1 + np.exp(-gu[:, :, 0]))
    want = (silu * gu[:, :, 1]).reshape(S, ff)
    err = (1.1 * size[:, :, 0] * np.abs(gu[:, :, 1]) + np.abs(silu) * size[:, :, 1]).reshape(S, ff) + np.abs(want) * 2.0 ** -20
    assert (np.abs(_f64(b.mid) - want) <= err * (1 + half) + np.abs(want) * half * (1 + half)).all()
    _same_rows(b.h[3], _f64(b.mid), fmt)
    want = _f64(xr) + m[5] * (h3 @ w["down"].T)
    err = np.abs(m[5]) * (np.abs(h3) @ np.abs(w["down"]).T) * (ff + 4) * 2.0 ** -23 + (np.abs(want) + np.abs(_f64(xr))) * 2.0 ** -23
    assert (np.abs(_f64(b.x) - want) <= err).all()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_two_captured_blocks_and_eager_ones_give_the_same_bits(kc, fmt):
    blocks = [Block(kc, fmt, s, rows=r) for s, r in ((5, 300), (6, 257))]
    want = []
    for b in blocks:
        b.run(kc)
        kc.wait()
        want.append([t.clone() for t in b.outputs()])
    other = ops.KreaCuda(0)          # the attention between keeps a word of its handle: graphs that overlap have a handle each
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graphs = []
    for b, k in zip(blocks, (kc, other)):
        k.set_stream(st)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            b.run(k)
        graphs.append(g)
    kc.set_stream(torch.cuda.current_stream())
    for b in blocks:
        for t in b.outputs():
            t.zero_()
    torch.cuda.synchronize()
    for i in (0, 1, 1, 0, 1):                       # one after the other on one stream
        graphs[i].replay()
    torch.cuda.synchronize()
    for b, w in zip(blocks, want):
        assert all(torch.equal(t, v) for t, v in zip(b.outputs(), w))
    for b in blocks:
        for t in b.outputs():
            t.zero_()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):                              # and beside one another
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for b, w in zip(blocks, want):
        assert all(torch.equal(t, v) for t, v in zip(b.outputs(), w))
    blocks[0].run(kc)                               # eager again, in the same buffers
    kc.wait()
    assert all(torch.equal(t, v) for t, v in zip(blocks[0].outputs(), want[0]))
    del graphs
    other.close()


def test_two_handles_on_two_streams(kc):
    other = ops.KreaCuda(0)
    try:
        blocks = [Block(kc, "nv", 8, rows=300), Block(kc, "mx", 9, rows=300)]
        want = []
        for b in blocks:
            b.run(kc)
            kc.wait()
            want.append([t.clone() for t in b.outputs()])
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        kc.set_stream(streams[0])
        other.set_stream(streams[1])
        for _ in range(5):
            blocks[0].run(kc)
            blocks[1].run(other)
        kc.wait()
        other.wait()
        for b, w in zip(blocks, want):
            assert all(torch.equal(t, v) for t, v in zip(b.outputs(), w))
    finally:
        kc.set_stream(torch.cuda.current_stream())
        other.close()


def test_work_is_ordered_behind_other_kernels_of_the_stream(kc):
    """Operators start early behind their predecessors, whoever those are: inputs written by torch kernels, by the bf16
    operators and by one another right before the call must be the ones that are read."""
    n, D = 384, 2048
    x = torch.randn(n, D, device="cuda")
    one = torch.ones(D, device="cuda")
    w = (torch.randn(D, 512, device="cuda") / D ** .5).bfloat16()
    q, s = _u8(512, ops.fp4_row_bytes(D)), _u8(ops.fp4_scale_bytes(B.FP4_MX, 512, D))
    a, sa = _u8(n, ops.fp4_row_bytes(D)), _u8(ops.fp4_scale_bytes(B.FP4_MX, n, D))
    hb, c = torch.zeros(n, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, 512, dtype=torch.bfloat16, device="cuda")
    kc.fp4_quantize(w, q, s, 512, D, 512, q.shape[1], B.FP4_MX, transposed=True)
    big = torch.zeros(64 << 20, device="cuda")

    def chain(scale, slow):
        if slow:
            big.add_(1.0)                           # keeps the stream busy, so that everything below is queued behind it
        y = x * scale
        kc.rms_norm(y, one, None, hb, n, D, D, D, 1e-6)
        kc.fp4_quantize(hb, a, sa, n, D, D, a.shape[1], B.FP4_MX)
        kc.gemm_fp4(a, sa, q, s, c, n, 512, D, a.shape[1], q.shape[1], 512, B.FP4_MX)
        kc.gated_norm(y, c.view(-1).repeat(4).view(n, D), None, hb, n, D, D, D, 0, D, mul=one)
        kc.fp4_quantize(hb, a, sa, n, D, D, a.shape[1], B.FP4_MX)
        kc.gemm_fp4(a, sa, q, s, c, n, 512, D, a.shape[1], q.shape[1], 512, B.FP4_MX)
        return c.clone()

    scales = [0.5, 3.0, 1.0, 7.0]
    want = []
    for v in scales:
        want.append(chain(v, False))
        torch.cuda.synchronize()
    got = [chain(v, True) for v in scales for _ in range(3)]
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i // 3])


def test_offsets_beyond_32_bits(kc):
    """Rows whose first element is past 2^31, in every operator: the last rows come out like the same rows alone."""
    rows, K = 70000, 32768                         # 2.3e9 values
    src = torch.empty(rows, K, dtype=torch.bfloat16, device="cuda")
    src.normal_(generator=torch.Generator("cuda").manual_seed(4))
    q, s = _u8(rows, ops.fp4_row_bytes(K)), _u8(ops.fp4_scale_bytes(B.FP4_NV, rows, K))
    kc.fp4_quantize(src, q, s, rows, K, K, q.shape[1], B.FP4_NV)
    first, few = rows // 128 * 128, rows - rows // 128 * 128
    q1, s1 = _u8(few, q.shape[1]), _u8(ops.fp4_scale_bytes(B.FP4_NV, few, K))
    kc.fp4_quantize(src[first:], q1, s1, few, K, K, q.shape[1], B.FP4_NV)
    kc.wait()
    assert torch.equal(q[first:], q1) and torch.equal(s[-s1.numel():], s1)
    out = src                                       # the rows are no longer needed
    want = torch.zeros(few, K, dtype=torch.bfloat16, device="cuda")
    kc.fp4_dequantize(q, s, out, rows, K, q.shape[1], K, B.FP4_NV)
    kc.fp4_dequantize(q1, s1, want, few, K, q.shape[1], K, B.FP4_NV)
    kc.wait()
    assert torch.equal(out[first:], want)
    # C [140000, 16384] from 256 values of each row, and A's rows 16 KB apart
    M, N = rows, K
    w, ws = q[:N].clone(), s[: ops.fp4_scale_bytes(B.FP4_NV, N, K)].clone()
    wk, wsk = _u8(N, 128), _u8(ops.fp4_scale_bytes(B.FP4_NV, N, 256))
    kc.fp4_quantize(want.view(-1)[: 256].repeat(N).view(N, 256).contiguous(), wk, wsk, N, 256, 256, 128, B.FP4_NV)
    del w, ws
    sk = s.view(-(-rows // 128), K // 256, 2048)[:, 0].contiguous()
    c = out
    kc.gemm_fp4(q, sk, wk, wsk, c, M, N, 256, q.shape[1], 128, N, B.FP4_NV)
    c1 = torch.zeros(few, N, dtype=torch.bfloat16, device="cuda")
    kc.gemm_fp4(q1, sk[-1], wk, wsk, c1, few, N, 256, q.shape[1], 128, N, B.FP4_NV)
    kc.wait()
    assert torch.equal(c[first:], c1)
    # norm: x f32 of the same number of values, y what is in c
    x = torch.empty(rows, K, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(5))
    one = torch.ones(K, device="cuda")
    h1 = torch.zeros(few, K, dtype=torch.bfloat16, device="cuda")
    x1 = x[first:].clone()
    kc.gated_norm(x1, c1, x1, h1, few, K, K, K, K, K, gate=one, mul=one)
    h = torch.empty(rows, K, dtype=torch.bfloat16, device="cuda")
    kc.gated_norm(x, c, x, h, rows, K, K, K, K, K, gate=one, mul=one)
    kc.wait()
    assert torch.equal(x[first:], x1) and torch.equal(h[first:], h1)


def test_calls_with_extreme_sizes_are_refused_before_any_launch(kc):
    t = _u8(1 << 16)
    n0 = kc.launches
    for call in (lambda: kc.fp4_quantize(t, t[4096:], t[8192:], 1 << 31, 32, 32, 16), lambda: kc.gemm_fp4(t, t, t, t, t, 1, 8, 1 << 40, 16, 16, 8),
                 lambda: kc.gated_norm(t, None, None, t[4096:], 1.5, 8, 8, 8, 8, 8)):
        with pytest.raises(ops.KreaCudaError) as e:
            call()
        assert e.value.code == B.E_ARG
    assert kc.launches == n0


@pytest.mark.parametrize("tile", ["0", "1", "2"])
def test_products_behind_a_wait_that_ran_out_store_nothing(monkeypatch, tile):
    """An attention launch whose last K tile is never requested gives up after 5 ms; the products queued behind it must leave
    their outputs as they were, and run again once the failure has been reported."""
    monkeypatch.setenv("KREA_CUDA_FP4_TILE", tile)
    k = ops.KreaCuda(0)
    k.set_stream(torch.cuda.current_stream())
    try:
        H, T, gh, gw = 2, 128, 16, 24
        S, ld = T + gh * gw, 3 * H * 128
        rng = np.random.default_rng(78)
        x = torch.from_numpy(synth.f32_to_bf16_bits(rng.standard_normal((S, ld)).astype(np.float32)).view(np.int16)).cuda().view(torch.bfloat16).view(-1)
        one = torch.ones(128, device="cuda")
        cos, sin = (torch.from_numpy(np.ascontiguousarray(t)).cuda() for t in synth.rope_tables_axial2d(T, gh, gw))
        o = torch.zeros((S, H * 128), dtype=torch.bfloat16, device="cuda")
        runs = []
        for M, N, K, epi in ((1, 2048, 6144, B.EPI_BF16), (64, 128, 2100, B.EPI_SWIGLU), (17, 256, 300, B.EPI_RESID_GATE), (700, 1032, 2048, B.EPI_BF16), (300, 520, 200, B.EPI_RESID_GATE)):
            a, w = (torch.from_numpy(rng.integers(0, 256, (r, ops.fp4_row_bytes(K)), dtype=np.uint8)).cuda() for r in (M, N))
            sa, sw = (torch.full((ops.fp4_scale_bytes(B.FP4_NV, r, K),), 0x38, dtype=torch.uint8, device="cuda") for r in (M, N))
            c = torch.full((M, N // 2 if epi == B.EPI_SWIGLU else N), 7.0, dtype=torch.float32 if epi == B.EPI_RESID_GATE else torch.bfloat16, device="cuda")
            vec = torch.ones(N, device="cuda") if epi == B.EPI_RESID_GATE else None
            runs.append((c, lambda a=a, sa=sa, w=w, sw=sw, c=c, M=M, N=N, K=K, epi=epi, vec=vec: k.gemm_fp4(a, sa, w, sw, c, M, N, K, a.shape[1], w.shape[1], c.shape[1], B.FP4_NV, epilogue=epi, vec=vec)))
        for _, run in runs:
            run()
        k.wait()
        want = [c.clone() for c, _ in runs]
        assert all(not bool((w == 7.0).all()) for w in want)
        for c, _ in runs:
            c.fill_(7.0)
        k.set_wait_limit(0.005)
        k.test_drop_one_load(True)
        k.joint_attention(x, x[H * 128:], x[2 * H * 128:], o, S, S, H, ld, ld, ld, H * 128, one, one, cos, sin)
        k.test_drop_one_load(False)
        for _, run in runs:
            run()
        with pytest.raises(ops.KreaCudaError) as e:
            k.wait()
        assert e.value.code == B.E_DEVICE
        assert all(bool((c == 7.0).all()) for c, _ in runs)
        k.set_wait_limit(2.0)
        k.wait()
        for (c, run), w in zip(runs, want):
            run()
            k.wait()
            assert torch.equal(c, w)
    finally:
        k.close()

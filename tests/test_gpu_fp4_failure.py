"""The 4-bit product when a bounded wait has run out, in an earlier kernel of the stream or in the product itself: every CTA
gets to its normal exit with nothing under way, nothing wrong is stored, and the handle works again afterwards."""
import time

import numpy as np
import pytest
import torch

from krea_image_b200 import binding as B, ops, synth

pytestmark = pytest.mark.gpu
FMT = {"mx": B.FP4_MX, "nv": B.FP4_NV}


@pytest.fixture(params=["0", "1", "2"], ids=["by-size", "rows", "pair"])
def kt(request, monkeypatch):
    """A handle whose product kernel is chosen by size, or one of the two for every shape."""
    monkeypatch.setenv("KREA_CUDA_FP4_TILE", request.param)
    k = ops.KreaCuda(0)
    k.set_stream(torch.cuda.current_stream())
    yield k
    k.close()


class Product:
    """Random operands (scales of 1) and C filled with 7, as one call."""

    def __init__(self, seed, fmt, M, N, K, epilogue):
        g = torch.Generator("cuda").manual_seed(seed)
        self.shape, self.fmt, self.epilogue = (M, N, K), FMT[fmt], epilogue
        rb = ops.fp4_row_bytes(K)
        self.a, self.w = (torch.randint(0, 256, (r, rb), dtype=torch.uint8, device="cuda", generator=g) for r in (M, N))
        if K % 32:
            for t in (self.a, self.w):                       # what is past K has to be zero
                t[:, (K + 1) // 2:] = 0
                if K % 2:
                    t[:, K // 2] &= 15
        self.sa, self.sw = (torch.full((ops.fp4_scale_bytes(self.fmt, r, K),), 127 if fmt == "mx" else 0x38, dtype=torch.uint8, device="cuda") for r in (M, N))
        f32 = epilogue in (B.EPI_RESID_GATE, B.EPI_F32)
        self.c = torch.full((M, N // 2 if epilogue == B.EPI_SWIGLU else N), 7.0, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
        self.vec = torch.ones(N, device="cuda") if epilogue == B.EPI_RESID_GATE else None

    def run(self, k):
        M, N, K = self.shape
        k.gemm_fp4(self.a, self.sa, self.w, self.sw, self.c, M, N, K, self.a.shape[1], self.w.shape[1], self.c.shape[1], self.fmt, epilogue=self.epilogue, vec=self.vec)

    def reset(self):
        self.c.fill_(7.0)

    def untouched(self):
        return bool((self.c == 7.0).all())


class FailingAttention:
    """A launch whose last K tile is never requested (the library's test hook): it gives up after 5 ms."""

    def __init__(self):
        H, T, gh, gw = 2, 128, 16, 24
        self.H, self.S, self.ld = H, T + gh * gw, 3 * H * 128
        rng = np.random.default_rng(78)
        bits = synth.f32_to_bf16_bits(rng.standard_normal((self.S, self.ld)).astype(np.float32))
        self.x = torch.from_numpy(bits.view(np.int16)).cuda().view(torch.bfloat16).view(-1)
        self.one = torch.ones(128, device="cuda")
        self.cos, self.sin = (torch.from_numpy(np.ascontiguousarray(t)).cuda() for t in synth.rope_tables_axial2d(T, gh, gw))
        self.o = torch.zeros((self.S, H * 128), dtype=torch.bfloat16, device="cuda")

    def run(self, k):
        H, S, ld, x = self.H, self.S, self.ld, self.x
        k.set_wait_limit(0.005)
        k.test_drop_one_load(True)
        k.joint_attention(x, x[H * 128:], x[2 * H * 128:], self.o, S, S, H, ld, ld, ld, H * 128, self.one, self.one, self.cos, self.sin)
        k.test_drop_one_load(False)
        k.set_wait_limit(2.0)


# one tile, several of a long K (shared by a cluster, or many stages a pair), more tiles than workers
AFTER = [(1, 2048, 6144, B.EPI_BF16), (40, 1024, 16384, B.EPI_F32), (200, 1024, 16384, B.EPI_RESID_GATE), (700, 1032, 9000, B.EPI_BF16), (2600, 4160, 2048, B.EPI_SWIGLU),
         (2600, 4160, 520, B.EPI_RESID_GATE)]


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_products_behind_a_failure_run_to_their_normal_end(kt, fmt):
    """The products may not stop at different stages in the CTAs of a cluster: what one has asked for and the other never waits
    for would arrive after they have left, and a wait for it would take its whole limit (2 s).  All of them together take
    some milliseconds."""
    runs = [Product(i, fmt, *s) for i, s in enumerate(AFTER)]
    bad = FailingAttention()
    for r in runs:
        r.run(kt)
    kt.wait()
    want = [r.c.clone() for r in runs]
    assert not any(r.untouched() for r in runs)
    for _ in range(4):
        for r in runs:
            r.reset()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        bad.run(kt)
        for r in runs:
            r.run(kt)
        with pytest.raises(ops.KreaCudaError) as e:
            kt.wait()
        assert time.perf_counter() - t0 < 1.0
        assert e.value.code == B.E_DEVICE and "attention" in str(e.value)
        assert all(r.untouched() for r in runs)
        for r, w in zip(runs, want):
            r.run(kt)
            kt.wait()
            assert torch.equal(r.c, w)


# one tile, a cluster that shares K, rows beyond one CTA, many stages a pair, more tiles than workers
OWN = [(1, 128, 256, B.EPI_F32), (1, 2048, 6144, B.EPI_BF16), (64, 512, 2100, B.EPI_SWIGLU), (17, 256, 3000, B.EPI_RESID_GATE), (300, 520, 9000, B.EPI_RESID_GATE), (2600, 4160, 2048, B.EPI_BF16),
       (2600, 4160, 520, B.EPI_RESID_GATE)]


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("shape", OWN, ids=lambda s: "x".join(map(str, s[:3])))
def test_a_product_whose_wait_runs_out_stores_no_unfinished_sum(kt, shape, fmt):
    """Operands that are not requested as a whole (a host-set hook; nothing faults) make the wait for them run out after 5 ms: few
    rows, the last stage of K, which one CTA of a cluster has; CTA pairs, rows of A in every stage.  The sum lacks a part:
    neither that CTA nor those it shares K with may store it."""
    r = Product(11, fmt, *shape)
    r.run(kt)
    kt.wait()
    want = r.c.clone()
    assert not r.untouched()
    for _ in range(2):
        r.reset()
        torch.cuda.synchronize()
        kt.set_wait_limit(0.005)
        kt.test_drop_one_load(True)
        t0 = time.perf_counter()
        r.run(kt)
        kt.test_drop_one_load(False)
        with pytest.raises(ops.KreaCudaError) as e:
            kt.wait()
        assert time.perf_counter() - t0 < 1.0                # a few times the limit
        assert e.value.code == B.E_DEVICE and "4-bit" in str(e.value)
        assert r.untouched()
        kt.set_wait_limit(2.0)
        r.run(kt)
        kt.wait()
        assert torch.equal(r.c, want)

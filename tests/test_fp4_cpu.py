"""CPU tests of the 4-bit operators and of the gated norm: sizes, argument checks (compiled from the library's own header,
so that no refusal needs a device), layout of the ctypes mirrors, and the oracle against closed forms."""
import ctypes
import os
import re
import subprocess
import threading

import numpy as np
import pytest

from krea_image_b200 import binding as B, ops
from oracle import fp4_np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = (("krea_cuda_fp4_quantize_args", "Fp4QuantizeArgs"), ("krea_cuda_fp4_dequantize_args", "Fp4DequantizeArgs"),
           ("krea_cuda_gemm_fp4_args", "GemmFp4Args"), ("krea_cuda_gated_norm_args", "GatedNormArgs"))


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    d = tmp_path_factory.mktemp("fp4")
    src = d / "checks.cpp"
    names = ("fp4_quantize", "fp4_dequantize", "gemm_fp4", "gated_norm")
    src.write_text('#include "fp4_checks.h"\nextern "C" {\n' + "".join(
        f"const char* {n}(const krea_cuda_{n}_args* a) {{ return krea::check_{n}(a); }}\n" for n in names) + "}\n")
    so = d / "checks.so"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "krea_image_b200", "csrc"), str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    for n in names:
        getattr(lib, n).restype = ctypes.c_char_p
    return lib


def test_sizes():
    for K in (1, 16, 31, 32, 33, 255, 256, 257, 6144):
        assert ops.fp4_row_bytes(K) == fp4_np.row_bytes(K)
        for rows in (1, 127, 128, 129, 4608):
            for code, fmt in ((B.FP4_MX, "mx"), (B.FP4_NV, "nv")):
                nb = -(-K // fp4_np.BLOCK[fmt])
                assert ops.fp4_scale_bytes(code, rows, K) == len(fp4_np.lay_out_scales(np.zeros((rows, nb), np.uint8), fmt, K))
    assert ops.fp4_row_bytes(0) == 0 and ops.fp4_row_bytes(-5) == 0
    assert ops.fp4_scale_bytes(2, 4, 4) == 0 and ops.fp4_scale_bytes(0, 0, 4) == 0 and ops.fp4_scale_bytes(0, 4, -1) == 0
    # sizes whose product passes 32 bits
    assert ops.fp4_scale_bytes(B.FP4_NV, 1 << 20, 1 << 20) == 1 << 36


def test_struct_layouts(tmp_path):
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "krea_cuda.h"', "int main(void) {"]
    for cname, pyname in STRUCTS:
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in getattr(B, pyname)._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cname, pyname in STRUCTS:
        st = getattr(B, pyname)
        assert int(got[cname]) == ctypes.sizeof(st)
        for f in st._fields_:
            assert int(got[f"{cname}.{f[0]}"]) == getattr(st, f[0]).offset, (cname, f[0])


def test_null_handles():
    lib = B.load()
    for n in ("fp4_quantize", "fp4_dequantize", "gemm_fp4", "gated_norm"):
        assert getattr(lib, "krea_cuda_" + n)(None, None) == B.E_ARG


P = [1 << 32, 2 << 32, 3 << 32, 4 << 32, 5 << 32, 6 << 32, 7 << 32, 8 << 32, 9 << 32, 10 << 32]     # apart, 16-byte aligned


def _try(fn, cls, good, changes):
    """Every change to a good call must be refused; the good one itself must not."""
    a = cls(**good)
    assert fn(ctypes.byref(a)) is None
    for ch in changes:
        a = cls(**{**good, **ch})
        assert fn(ctypes.byref(a)), ch


def test_quantize_refusals(checks):
    good = dict(src=P[0], q=P[1], scales=P[2], tensor_scale=P[3], rows=5, K=70, ld=72, ldq=48, format=B.FP4_NV, transposed=0)
    _try(checks.fp4_quantize, B.Fp4QuantizeArgs, good, [
        dict(rows=-1), dict(K=-1), dict(rows=(1 << 30) + 1), dict(K=(1 << 26) + 1, ld=0x7FFFFFF8, ldq=0x7FFFFFF0), dict(format=2), dict(format=-1), dict(src=None), dict(q=None), dict(scales=None),
        dict(src=P[0] + 8), dict(q=P[1] + 4), dict(scales=P[2] + 2), dict(tensor_scale=P[3] + 2), dict(format=B.FP4_MX), dict(ld=68), dict(ld=76), dict(ldq=32),
        dict(ldq=50), dict(transposed=1, rows=80), dict(q=P[0]), dict(scales=P[0] + 16), dict(scales=P[1]), dict(scales=P[1] + 4 * 48 + 32),
        dict(tensor_scale=P[1] + 8), dict(tensor_scale=P[2])])
    for ch in (dict(rows=0, src=None), dict(K=0, q=None), dict(tensor_scale=None), dict(transposed=1, ld=8), dict(format=B.FP4_MX, tensor_scale=None)):
        assert checks.fp4_quantize(ctypes.byref(B.Fp4QuantizeArgs(**{**good, **ch}))) is None, ch


def test_dequantize_refusals(checks):
    good = dict(q=P[0], scales=P[1], tensor_scale=P[2], out=P[3], rows=5, K=70, ldq=48, ldo=72, format=B.FP4_NV)
    _try(checks.fp4_dequantize, B.Fp4DequantizeArgs, good, [
        dict(rows=-1), dict(K=-1), dict(format=7), dict(q=None), dict(scales=None), dict(out=None), dict(q=P[0] + 8), dict(scales=P[1] + 1), dict(out=P[3] + 2),
        dict(tensor_scale=P[2] + 1), dict(format=B.FP4_MX), dict(ldq=32), dict(ldq=49), dict(ldo=70), dict(ldo=64), dict(out=P[0] + 32), dict(out=P[1]), dict(out=P[2])])


def test_gemm_refusals(checks):
    good = dict(A=P[0], a_scales=P[1], W=P[2], w_scales=P[3], C=P[4], M=3, N=64, K=70, lda=48, ldw=64, ldc=64, format=B.FP4_NV, epilogue=B.EPI_BF16, vec=P[5],
                a_tensor_scale=P[6], w_tensor_scale=P[7])
    _try(checks.gemm_fp4, B.GemmFp4Args, good, [
        dict(M=-1), dict(N=-8), dict(K=-1), dict(K=0), dict(M=(1 << 30) + 1), dict(N=(1 << 30) + 8, ldc=(1 << 30) + 8), dict(K=(1 << 26) + 1, lda=0x7FFFFFF0, ldw=0x7FFFFFF0), dict(format=3), dict(A=None), dict(a_scales=None), dict(W=None), dict(w_scales=None), dict(C=None),
        dict(A=P[0] + 8), dict(a_scales=P[1] + 8), dict(W=P[2] + 8), dict(w_scales=P[3] + 8), dict(C=P[4] + 8), dict(a_tensor_scale=P[6] + 2), dict(w_tensor_scale=P[7] + 1),
        dict(format=B.FP4_MX), dict(lda=32), dict(lda=56), dict(ldw=32), dict(ldw=72), dict(N=60), dict(ldc=66), dict(ldc=56), dict(epilogue=B.EPI_SWIGLU, N=32),
        dict(epilogue=B.EPI_BIAS_BF16, vec=None), dict(epilogue=B.EPI_BIAS_F32, vec=P[5] + 4), dict(epilogue=B.EPI_RESID_GATE, vec=P[5] + 8), dict(C=P[0]), dict(C=P[2] + 64),
        dict(C=P[1]), dict(C=P[3]), dict(C=P[6]), dict(C=P[7]), dict(epilogue=B.EPI_BIAS_BF16, C=P[5] + 16), dict(epilogue=B.EPI_RESID_GATE, C=P[5])])
    for ch in (dict(M=0, A=None), dict(N=0), dict(epilogue=B.EPI_RESID_GATE, vec=None), dict(epilogue=B.EPI_SWIGLU, ldc=32), dict(C=P[5])):
        assert checks.gemm_fp4(ctypes.byref(B.GemmFp4Args(**{**good, **ch}))) is None, ch


def test_gated_norm_refusals(checks):
    good = dict(x=P[0], y=P[1], x_out=P[2], h=P[3], h_scales=P[4], h_tensor_scale=P[5], post=P[6], gate=P[7], mul=P[8], add=P[9], rows=5, width=40, ld_x=44, ld_y=40, ld_xo=40, ld_h=32,
                mod_rows=2, mod_ld=40, x_scale=1.0, eps=1e-6, y_f32=0, out=B.OUT_FP4_NV)
    _try(checks.gated_norm, B.GatedNormArgs, good, [
        dict(rows=-1), dict(rows=(1 << 30) + 1), dict(width=-8), dict(out=4), dict(out=-1), dict(x=None), dict(x_out=None, h=None), dict(width=36), dict(width=32776, ld_x=32776, ld_y=32776, ld_xo=32776, ld_h=16400),
        dict(ld_x=36), dict(ld_x=42), dict(ld_y=44), dict(ld_y=32), dict(ld_xo=36), dict(ld_xo=41), dict(y=None), dict(y=None, post=None), dict(mul=None), dict(ld_h=16), dict(ld_h=40),
        dict(h_scales=None), dict(out=B.OUT_FP4_MX), dict(out=B.OUT_BF16, ld_h=40), dict(h_tensor_scale=P[5] + 2), dict(x=P[0] + 4), dict(y=P[1] + 2), dict(x_out=P[2] + 8), dict(h=P[3] + 8),
        dict(post=P[6] + 4), dict(gate=P[7] + 4), dict(mul=P[8] + 4), dict(add=P[9] + 4), dict(h_scales=P[4] + 4), dict(mod_rows=-1), dict(mod_ld=42), dict(mod_ld=-4),
        dict(eps=-1.0), dict(eps=float("nan")), dict(x_scale=float("inf")), dict(x_scale=float("nan")), dict(x_out=P[0]), dict(x_out=P[0] + 16, ld_xo=44), dict(x_out=P[1]), dict(h=P[0]),
        dict(h=P[1] + 16), dict(h=P[2]), dict(h_scales=P[0]), dict(h_scales=P[3]), dict(h=P[6]), dict(h=P[5]), dict(x_out=P[7] + 160), dict(x_out=P[8] + 2 * 160 + 144), dict(h_scales=P[9])])
    for ch in (dict(rows=0, x=None), dict(x_out=P[0], ld_xo=44), dict(y=None, post=None, gate=None), dict(h=None, mul=None, h_scales=None), dict(out=B.OUT_F32, h_tensor_scale=None, ld_h=40),
               dict(out=B.OUT_BF16, h_tensor_scale=None, ld_h=40), dict(x_out=None), dict(y_f32=1, ld_y=44), dict(mod_rows=0, mod_ld=3), dict(eps=0.0)):
        assert checks.gated_norm(ctypes.byref(B.GatedNormArgs(**{**good, **ch}))) is None, ch


# ---- the oracle against closed forms ----
def test_oracle_grid_ties_and_saturation():
    x = np.zeros((1, 32))
    x[0, :9] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -0.25, 7.75]      # amax 7.75: scale 2^(2 - 2) = 1
    q, s = fp4_np.quantise(x, "mx")
    assert s[0, 0] == 127
    assert list(fp4_np.values(q, s, "mx", 9)[0]) == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 0.0, 6.0]
    assert q[0, 7] == 8                                                  # the sign of a value that rounds to zero stays
    x = np.zeros((1, 16))
    x[0, :4] = [6.0, 5.0, 0.3, -2.0]
    q, s = fp4_np.quantise(x, "nv")
    assert list(fp4_np.values(q, s, "nv", 4)[0]) == [6.0, 4.0, 0.5, -2.0]
    # a block's largest value decides its scale: 448 at most, and zero below half of the smallest
    q, s = fp4_np.quantise(np.full((1, 16), 1e5), "nv")
    assert s[0, 0] == 126 and fp4_np.values(q, s, "nv", 1)[0, 0] == 6 * 448
    q, s = fp4_np.quantise(np.full((1, 16), 6 * 2.0 ** -10), "nv")
    assert s[0, 0] == 0 and fp4_np.values(q, s, "nv", 1)[0, 0] == 0
    for fmt, code in (("mx", 255), ("nv", 127)):
        x = np.ones((1, 64))
        x[0, 40] = np.inf
        v = fp4_np.values(*fp4_np.quantise(x, fmt), fmt, 64)
        bs = fp4_np.BLOCK[fmt]
        bad = np.arange(64) // bs == 40 // bs
        one = 1.0 if fmt == "mx" else 6 * 0.171875              # NV: the scale is 1 / 6 rounded to e4m3
        assert np.isnan(v[0, bad]).all() and (v[0, ~bad] == one).all()


def test_oracle_e4m3_is_the_format():
    torch = pytest.importorskip("torch")
    assert np.array_equal(fp4_np.E4M3, torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())


def test_kernels_that_start_early_use_no_read_only_loads():
    """A kernel with a programmatic launch runs while the one before it may still write what it will read: the read-only path
    is not for such memory, and a compiler may move its loads above the wait for the predecessor.  The gated norm has one
    such load, in the form that is never launched that way."""
    for name in ("fp4_quant.cu", "gemm_fp4_sm100.cu", "gated_norm.cu", "fp4_block.cuh"):
        with open(os.path.join(ROOT, "krea_image_b200", "csrc", name)) as f:
            code = "\n".join(line.split("//")[0] for line in f)
        if name == "gated_norm.cu":
            assert code.count("load8<V8, !AHEAD>") == code.count("load8<") == 1      # NC is the opposite of AHEAD
            assert "stream, AHEAD && pdl," in code and code.count("launch_kernel(") == 1
            code = re.sub(r"template <bool V8, bool NC>.*?\n}\n", "", code, flags=re.S)
        for word in ("__ldg", "global.nc", "__restrict__"):
            assert word not in code, (name, word)


def test_two_threads_on_one_handle_pass_their_own_arguments():
    """The interpreter lock is given up inside a call: another thread's call of the same operator may be prepared meanwhile."""
    seen, inside, go = {}, threading.Barrier(2), threading.Event()

    def fake(_, args):
        a = ctypes.cast(args, ctypes.POINTER(B.Fp4DequantizeArgs)).contents
        if threading.current_thread() is first:      # the arguments are read only after the second call has been prepared
            inside.wait(10)
            assert go.wait(10)
        seen[threading.current_thread()] = [getattr(a, f[0]) for f in a._fields_]
        return 0

    fn = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)(fake)
    call = ops._Call(fn, B.Fp4DequantizeArgs)
    mine, other = [256, 512, 768, 1024, 5, 70, 48, 72, 1], [4096, 8192, None, 16384, 7, 32, 16, 32, 0]
    first = threading.Thread(target=lambda: call(None, *mine))
    first.start()
    inside.wait(10)
    assert call(None, *[v or 0 for v in other]) == 0
    go.set()
    first.join(10)
    assert seen[first] == mine and seen[threading.current_thread()] == other


def test_gated_norm_takes_rows_side_by_side_in_one_buffer(checks):
    """Column slices of one wide buffer have no byte in common; slices that do, and rows of another distance, are refused."""
    base = dict(x=P[0], y=P[1], x_out=P[2], h=P[3], mul=P[8], rows=5, width=40, ld_x=128, ld_y=256, ld_xo=128, ld_h=256, mod_rows=0, mod_ld=0, x_scale=1.0, eps=1e-6, y_f32=0, out=B.OUT_BF16)
    ok = lambda **ch: checks.gated_norm(ctypes.byref(B.GatedNormArgs(**{**base, **ch}))) is None  # noqa: E731
    assert ok()
    assert ok(h=P[1] + 80) and ok(h=P[1] + 256) and ok(y=P[3] + 80)             # y and h: 80 bytes of every 512
    assert ok(x_out=P[0] + 160) and ok(x_out=P[0] + 352) and ok(x=P[2] + 160)    # x and x_out: 160 bytes of every 512
    assert ok(x_out=P[1] + 80) and ok(h=P[2] + 160) and ok(h=P[0] + 160)
    assert ok(h=P[1] + 512 - 80) and ok(h=P[1] - 80) and ok(h=P[1] + 3 * 512 + 80)
    assert not ok(h=P[1] + 64) and not ok(h=P[1] + 512 - 64) and not ok(h=P[1] - 64) and not ok(h=P[1] + 4 * 512)
    assert not ok(x_out=P[0] + 144) and not ok(x_out=P[0] + 368) and not ok(x_out=P[0] + 512)
    assert not ok(h=P[1] + 80, ld_h=248) and not ok(x_out=P[0] + 160, ld_xo=124)
    assert not ok(h=P[1] + 80, ld_h=512, out=B.OUT_FP4_MX, h_scales=P[1] + 160)

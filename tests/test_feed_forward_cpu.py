"""CPU tier: what the feed-forward operators refuse, at the C ABI (before any CUDA call) and at the Python boundary."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "amd-kernels_b200", "kernels", "libhkb200.so")
i64, f32, i32 = ctypes.c_int64, ctypes.c_float, ctypes.c_int
BAD_ARG, BAD_SHAPE, BAD_ALIGN, UNSUPPORTED = -1, -2, -3, -4
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    l = ctypes.CDLL(LIB)
    l.hkb_last_error.restype = ctypes.c_char_p
    l.hkb_gemm_fp8_blockscale_gated_workspace.restype = i64
    return l


@pytest.fixture(scope="module")
def ptr():
    buf = ctypes.create_string_buffer(8192)
    base = (ctypes.addressof(buf) + 63) & ~63
    return lambda off=0, keep=buf: ctypes.c_void_p(base + off)


def test_add_norm_refusals(lib, ptr):
    def call(x=0, r=0, w=0, q=0, s=0, h=0, M=4, D=128, group=128, null=None):
        p = [ptr(o) for o in (x, r, w, q, s, h)]
        if null is not None:
            p[null] = None
        return lib.hkb_add_rmsnorm_quant_fp8(*p, i64(M), i64(D), i64(group), f32(1e-6), None)
    for k in range(6):
        assert call(null=k) == BAD_ARG and b"null" in lib.hkb_last_error()
    for M, D, group in ((4, 100, 100), (4, 0, 0), (4, -8, -8), (-1, 128, 128), (4, 32776, 32776), (4, 136, 128), (4, 256, 64), (4, 256, 0), (1 << 31, 128, 128)):
        assert call(M=M, D=D, group=group) == BAD_SHAPE, (M, D, group)
    for name in ("x", "r", "w", "h"):
        assert call(**{name: 8}) == BAD_ALIGN, name
    assert call(q=4) == BAD_ALIGN and call(s=2) == BAD_ALIGN
    assert call(M=0) == 0


def test_epilogue_refusals(lib, ptr):
    def pts(c=0, bias=0, act=0, res=0, batch=1, M=4, N=128, K=128):
        return lib.hkb_gemm_fp8_pts_epilogue(ptr(), ptr(), ptr(c), ptr(), ptr(), ptr(bias), i32(act), ptr(res), i64(batch), i64(M), i64(N), i64(K), None)

    def block(c=0, bias=0, act=0, res=0, gn=128, M=4, N=128, K=128):
        return lib.hkb_gemm_fp8_blockscale_epilogue(ptr(), ptr(), ptr(c), ptr(), ptr(), i64(gn), ptr(bias), i32(act), ptr(res), i64(M), i64(N), i64(K), None)
    for f in (pts, block):
        assert f(act=5) == BAD_ARG and f(act=-1) == BAD_ARG and b"activation" in lib.hkb_last_error()
        assert f(bias=8) == BAD_ALIGN and f(res=8) == BAD_ALIGN and f(c=8) == BAD_ALIGN
        assert f(M=0) == BAD_SHAPE and f(N=0) == BAD_SHAPE and f(K=96) == BAD_SHAPE and f(N=100) == BAD_SHAPE
    assert pts(batch=0) == BAD_SHAPE
    assert block(gn=64) == UNSUPPORTED and block(N=136) == BAD_SHAPE
    nothing = [None] * 5
    assert lib.hkb_gemm_fp8_pts_epilogue(*nothing, None, i32(0), None, i64(1), i64(4), i64(128), i64(128), None) == BAD_ARG
    assert lib.hkb_gemm_fp8_blockscale_epilogue(*nothing, i64(128), None, i32(0), None, i64(4), i64(128), i64(128), None) == BAD_ARG


def test_gated_refusals_and_workspace(lib, ptr):
    def call(a=0, b=0, c=0, cs=0, act=4, ws=0, M=4, F=128, K=128, null=()):
        p = {"a": ptr(a), "b": ptr(b), "c": ptr(c), "cs": ptr(cs), "sa": ptr(), "sb": ptr(), "ws": ptr(ws)}
        p.update((k, None) for k in null)
        return lib.hkb_gemm_fp8_blockscale_gated(p["a"], p["b"], p["c"], p["cs"], p["sa"], p["sb"], i32(act), p["ws"], i64(M), i64(F), i64(K), None)
    for k in ("a", "b", "c", "sa", "sb"):
        assert call(null=(k,)) == BAD_ARG
    assert call(act=5) == BAD_ARG and call(act=-1) == BAD_ARG
    for M, F, K in ((0, 128, 128), (4, 0, 128), (4, 192, 128), (4, 128, 64), (4, 128, 0), (4, 1 << 30, 128), (1 << 31, 128, 128)):
        assert call(M=M, F=F, K=K) == BAD_SHAPE, (M, F, K)
        assert lib.hkb_gemm_fp8_blockscale_gated_workspace(i64(M), i64(F), i64(K), i32(1)) == BAD_SHAPE
    assert call(a=8) == BAD_ALIGN and call(b=8) == BAD_ALIGN and call(c=16) == BAD_ALIGN and call(cs=2) == BAD_ALIGN
    ws = lib.hkb_gemm_fp8_blockscale_gated_workspace
    assert ws(i64(4), i64(256), i64(128), i32(0)) == 0 and ws(i64(300), i64(256), i64(128), i32(1)) == 0
    assert ws(i64(4), i64(256), i64(128), i32(1)) >= 4 * 256 * 4
    assert call(null=("ws",)) == BAD_ARG and b"workspace" in lib.hkb_last_error()
    assert call(ws=8) == BAD_ARG


# ---- Python boundary ------------------------------------------------------------------------------------

def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def f8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4M3)


def test_signatures(hk):
    d = hk.modules["fused_fp8_quant_tk"].fused_add_rmsnorm_fp8_quant_fwd.__doc__
    assert d.startswith("fused_add_rmsnorm_fp8_quant_fwd(input: object, residual: object, weight: object, output: object, scales: object, residual_out: object, eps: ")
    for gemm in (hk.gemm.a8w8_per_token, hk.gemm.a8w8_blockscale):
        assert gemm.dispatch_epilogue.__doc__.startswith(
            "dispatch_epilogue(A: object, B: object, C: object, a_scale: object, b_scale: object, bias: object = None, activation: object = 'none', residual: object = None)")
    assert hk.gemm.a8w8_blockscale.dispatch_gated.__doc__.startswith(
        "dispatch_gated(A: object, B: object, C: object, a_scale: object, b_scale: object, c_scale: object = None, activation: object = 'silu')")


def test_add_norm_checks_its_tensors(hk):
    def call(match, **over):
        a = {"input": bf(4, 256), "residual": bf(4, 256), "weight": bf(256), "output": f8(4, 256), "scales": torch.zeros(4, 2), "residual_out": bf(4, 256)}
        a.update(over)
        with pytest.raises(RuntimeError, match=match):
            hk.fused_add_rmsnorm_fp8_quant_fwd(*a.values(), 1e-6)
    call("CUDA device")
    call("CUDA device", scales=torch.zeros(4))
    call("weight: tensor is None", weight=None)
    call("residual: tensor is None", residual=None)
    call("input: dtype float32", input=torch.zeros(4, 256))
    call("residual: dtype float16", residual=torch.zeros(4, 256, dtype=torch.float16))
    call("output: dtype int8", output=torch.zeros(4, 256, dtype=torch.int8))
    call("scales: dtype bfloat16", scales=bf(4, 2))
    call("residual and residual_out", residual=bf(4, 255))
    call("residual and residual_out", residual_out=bf(5, 256))
    call("weight must have D", weight=bf(255))
    call("output must have", output=f8(4, 128))
    call("scales must have", scales=torch.zeros(4, 3))
    call("contiguous", residual=bf(256, 4).t())
    call(r"\[M, D\]", input=bf(1024))


def test_epilogue_checks_its_tensors(hk):
    def call(match, gemm=hk.gemm.a8w8_per_token, **over):
        block = gemm is hk.gemm.a8w8_blockscale
        a = {"A": f8(4, 256), "B": f8(128, 256), "C": bf(4, 128), "a_scale": torch.zeros(4, 2) if block else torch.zeros(4),
             "b_scale": torch.zeros(2, 1) if block else torch.zeros(128), "bias": bf(128), "activation": "gelu", "residual": bf(4, 128)}
        a.update(over)
        with pytest.raises(RuntimeError, match=match):
            gemm.dispatch_epilogue(*a.values())
    for gemm in (hk.gemm.a8w8_per_token, hk.gemm.a8w8_blockscale):
        call("CUDA device", gemm)
        call("CUDA device", gemm, bias=None, residual=None, activation=None)
        call("unknown activation 'swish'", gemm, activation="swish")
        call("bias must have", gemm, bias=bf(127))
        call("bias: dtype float32", gemm, bias=torch.zeros(128))
        call("residual must be", gemm, residual=bf(4, 127))
        call("residual: dtype float32", gemm, residual=torch.zeros(4, 128))
        call("contiguous", gemm, residual=bf(128, 4).t())
        call("C must be", gemm, C=bf(4, 64))
        call("a_scale must", gemm, a_scale=torch.zeros(3))
        call("must not be empty", gemm, A=f8(0, 256), C=bf(0, 128))
        call("same K", gemm, B=f8(128, 128))
    call("b_scale group size", hk.gemm.a8w8_blockscale, b_scale=torch.zeros(2, 2))
    call("2-D operands", hk.gemm.a8w8_blockscale, A=f8(2, 4, 256), B=f8(2, 128, 256), C=bf(2, 4, 128))


def test_gated_checks_its_tensors(hk):
    def call(match, **over):
        a = {"A": f8(4, 256), "B": f8(256, 256), "C": f8(4, 128), "a_scale": torch.zeros(4, 2), "b_scale": torch.zeros(2, 2), "c_scale": torch.zeros(4, 1),
             "activation": "silu"}
        a.update(over)
        with pytest.raises(RuntimeError, match=match):
            hk.gemm.a8w8_blockscale.dispatch_gated(*a.values())
    call("CUDA device")
    call("CUDA device", C=bf(4, 128), c_scale=None)
    call("C: dtype float8_e4m3fn", c_scale=None)
    call("C: dtype bfloat16", C=bf(4, 128))
    call("unknown activation", activation="swiglu")
    call("B \\[2F, K\\]", B=f8(128, 256))
    call("multiples of 128", C=f8(4, 64), B=f8(128, 256))
    call("a_scale must be", a_scale=torch.zeros(4, 1))
    call("b_scale must be", b_scale=torch.zeros(2, 1))
    call("c_scale must be", c_scale=torch.zeros(4, 2))
    call("c_scale: dtype", c_scale=bf(4, 1))
    call("same K", A=f8(4, 128))


def test_many_leading_dimensions_are_a_batch(hk):
    ones = (1,) * 10
    a, b = torch.zeros(*ones, 4, 128, dtype=E4M3), torch.zeros(*ones, 256, 128, dtype=E4M3)
    c, sa, sb = torch.zeros(*ones, 4, 256, dtype=torch.bfloat16), torch.ones(*ones, 4), torch.ones(*ones, 256)
    for call in (lambda: hk.gemm.a8w8_per_token.dispatch(a, b, c, sa, sb), lambda: hk.gemm.a8w8_per_token.dispatch_epilogue(a, b, c, sa, sb)):
        with pytest.raises(RuntimeError, match="CUDA"):         # all that is wrong with them is where they are
            call()

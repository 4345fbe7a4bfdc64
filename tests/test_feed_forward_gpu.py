"""GPU tier: the feed-forward operators (residual + RMSNorm + FP8 quantization, FP8 GEMM with bias / activation / residual, gated
GEMM) against their definitions in 64 bits on the device.

Tolerances, from the arithmetic:
  * a result rounded to bf16 is off by at most eps/2 = 2^-8 of its value, a code by at most half an e4m3 step;
  * a GEMM value: the tensor core adds K/32 products of 32 exact terms and the block-scale promotion K/128 scaled partials, each in
    fp32 with at most one unit of the last place (2^-23) of what has been summed, so at most (K/32 + 2 K/128 + 8) * 2^-23 of the sum
    of absolute products (scales and bias multiplied in are the 8);
  * an activation has a slope of at most 1.13 and is evaluated to 2^-19 of its value; from -3 down the forms of gelu, from -20 silu, to
    2^-15.7 (the exponent's rounding), but there the value is under 2^-9 |v|, so that error is under the 8 * 2^-23 |v| of the GEMM's;
  * RMSNorm: at most 136 additions per statistic (128 in a thread, 8 across lanes and warps), half of that through the square root,
    and four roundings: 2^-16 of the value.
Codes are held to the interval that the value's tolerance leaves: e4m3((y - tol) / s) <= code <= e4m3((y + tol) / s)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
EPS = 1e-6
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).bfloat16()


def quant_rows(x, group):
    """FP8 codes and scales, one per `group` columns (IEEE division on the device)."""
    v = x.float().reshape(-1, x.shape[-1] // group, group)
    s = (v.abs().amax(2, keepdim=True) / torch.tensor(448.0, device=DEV)).clamp_min(1e-10)
    return (v / s).clamp(-448, 448).to(E4M3).reshape(x.shape), s.reshape(*x.shape[:-1], -1)


def quant_tiles(w):
    N, K = w.shape
    v = w.float().view(N // 128, 128, K // 128, 128)
    s = (v.abs().amax((1, 3), keepdim=True) / torch.tensor(448.0, device=DEV)).clamp_min(1e-10)
    return (v / s).clamp(-448, 448).to(E4M3).view(N, K), s.view(N // 128, K // 128).t().contiguous()


def act64(v, name):
    if name == "relu":
        return v.clamp_min(0)
    if name == "gelu":
        return v * 0.5 * torch.special.erfc(-v * 0.5 ** 0.5)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    return v * torch.sigmoid(v) if name == "silu" else v


def act_tol(v, tol, name):
    return 1.13 * tol + act64(v, name).abs() * 2.0 ** -19


def check_bf16(got, ref, tol):
    err = (got.double() - ref).abs()
    ok = err <= ref.abs() * 2.0 ** -8 + tol * (1 + 2.0 ** -8) + 2.0 ** -133
    assert ok.all(), f"{(~ok).sum().item()} of {ok.numel()} off, worst {(err / (ref.abs() * 2.0 ** -8 + tol)).max().item():.3g} of the bound"


def check_codes(codes, scales, y, tol, group):
    """codes [M, D], scales [M, D / group] of y (64 bits) known up to tol."""
    M, D = y.shape
    yg, tg = y.view(M, D // group, group), tol.view(M, D // group, group)
    s = scales.double().view(M, D // group, 1)
    low = ((yg.abs() - tg).amax(2, keepdim=True) / 448).clamp_min(1e-10) * (1 - 2.0 ** -22)
    high = ((yg.abs() + tg).amax(2, keepdim=True) / 448).clamp_min(1e-10) * (1 + 2.0 ** -22)
    assert ((s >= low) & (s <= high)).all(), "scales"
    c = codes.view(torch.uint8).view(E4M3).double().view(M, D // group, group)
    slack = yg.abs() * 2.0 ** -21                       # the quotient itself: a reciprocal and a product in fp32
    lo = ((yg - tg - slack) / s).clamp(-448, 448).float().to(E4M3).double()
    hi = ((yg + tg + slack) / s).clamp(-448, 448).float().to(E4M3).double()
    ok = (c >= lo) & (c <= hi)
    assert ok.all(), f"{(~ok).sum().item()} of {ok.numel()} codes off"


def guarded(*shape, dtype):
    """A tensor with 64 bytes of a pattern behind it, and a check that they are still there."""
    n = 1
    for d in shape:
        n *= d
    raw = torch.full((n * dtype.itemsize + 64,), 0x5A, dtype=torch.uint8, device=DEV)
    t = raw[: n * dtype.itemsize].view(dtype).view(shape)
    t.view(torch.uint8).fill_(0xFF if dtype.itemsize == 1 else 0x7F)
    return t, lambda: bool((raw[n * dtype.itemsize:] == 0x5A).all())


# ---- residual + RMSNorm + FP8 ------------------------------------------------------------------------

def norm_case(M, D, seed, x_scale=1.0):
    g = gen(seed)
    x, r = randn(g, M, D, scale=x_scale), randn(g, M, D, scale=x_scale)
    r[:, :: max(1, D // 16)] *= 20
    return x, r, (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).bfloat16()


def check_norm(hk, x, r, w, group, out=None, eps=EPS):
    M, D = x.shape
    total = (x.float() + r.float()).bfloat16()
    q, q_ok = guarded(M, D, dtype=E4M3)
    s, s_ok = guarded(M, D // group, dtype=torch.float32)
    h, h_ok = guarded(M, D, dtype=torch.bfloat16) if out is None else (out, lambda: True)
    hk.fused_add_rmsnorm_fp8_quant_fwd(x, r, w, q, s, h, eps)
    assert torch.equal(h, total)
    t = total.double()
    y = t / ((t * t).mean(1, keepdim=True) + eps).sqrt() * w.double()
    check_codes(q, s, y, y.abs() * 2.0 ** -16, group)
    assert q_ok() and s_ok() and h_ok()


@pytest.mark.parametrize("M,D", [(1, 128), (1, 4096), (3, 8192), (37, 384), (150, 2048), (700, 1152), (2, 16384), (3, 32768), (4500, 512)])
def test_add_norm_block_scales(hk, M, D):
    check_norm(hk, *norm_case(M, D, M + D), 128)


@pytest.mark.parametrize("M,D", [(1, 8), (5, 24), (1, 4104), (2, 136), (33, 4096), (1000, 1032), (3, 16392), (2, 32760), (2, 32768), (5000, 264)])
def test_add_norm_row_scales(hk, M, D):
    check_norm(hk, *norm_case(M, D, M + D), D)


def test_add_norm_of_no_rows(hk):
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device=DEV)      # noqa: E731
    hk.fused_add_rmsnorm_fp8_quant_fwd(e(0, 256), e(0, 256), torch.ones(256, device=DEV).bfloat16(), e(0, 256, dtype=E4M3), e(0, 2, dtype=torch.float32), e(0, 256), EPS)


@pytest.mark.parametrize("group", [128, 1024])
def test_add_norm_in_place_and_on_offset_views(hk, group):
    M, D = 19, 1024
    x, r, w = norm_case(M, D, 3)
    keep = r.clone()
    h = r
    q, s = torch.empty(M, D, dtype=E4M3, device=DEV), torch.empty(M, D // group, device=DEV)
    hk.fused_add_rmsnorm_fp8_quant_fwd(x, r, w, q, s, h, EPS)            # the stream updated in place
    fresh = [torch.empty(M, D, dtype=E4M3, device=DEV), torch.empty(M, D // group, device=DEV), torch.empty_like(x)]
    hk.fused_add_rmsnorm_fp8_quant_fwd(x, keep, w, *fresh, EPS)
    assert torch.equal(h, fresh[2]) and torch.equal(q.view(torch.uint8), fresh[0].view(torch.uint8)) and torch.equal(s, fresh[1])
    x2 = x.clone()
    hk.fused_add_rmsnorm_fp8_quant_fwd(x2, keep, w, q, s, x2, EPS)       # or over the branch's output
    assert torch.equal(x2, fresh[2]) and torch.equal(q.view(torch.uint8), fresh[0].view(torch.uint8))
    off = [torch.empty(M * D + 8, dtype=torch.bfloat16, device=DEV)[8:].view(M, D).copy_(t) for t in (x, keep)]
    assert off[0].data_ptr() % 32 == 16
    check_norm(hk, off[0], off[1], w, group)                             # 16-byte chunks
    check_norm(hk, x, off[1], w, group, out=off[1])


@pytest.mark.parametrize("group", [128, 512])
def test_add_norm_zero_rows_extremes_and_non_finite(hk, group):
    M, D = 6, 512
    x, r, w = norm_case(M, D, 5)
    x[0], r[0] = 0, 0                       # scale floor, zero codes
    r[1] = -x[1]                            # cancels
    x[2], r[2] = 1e-20, 1e-20               # eps decides
    x[3, 7] = float("nan")
    r[4, 9] = float("inf")
    x[5] *= 1e15
    h, q, s = torch.empty_like(x), torch.empty(M, D, dtype=E4M3, device=DEV), torch.empty(M, D // group, device=DEV)
    hk.fused_add_rmsnorm_fp8_quant_fwd(x, r, w, q, s, h, EPS)
    total = (x.float() + r.float()).bfloat16()
    assert torch.equal(h[[0, 1, 2, 5]], total[[0, 1, 2, 5]])
    assert (q[:2].float() == 0).all() and (s[:2] == 1e-10).all()
    t = total[[2, 5]].double()
    y = t / ((t * t).mean(1, keepdim=True) + EPS).sqrt() * w.double()
    check_codes(q[[2, 5]], s[[2, 5]], y, y.abs() * 2.0 ** -16, group)
    assert q[3].float().isnan().all() and s[3].isnan().all()             # one NaN: the row's mean is NaN
    bad = 9 // group
    assert s[4, bad].isnan() and q[4].float()[9].isnan()                 # infinity: rsqrt 0, inf * 0 in its group, zeros elsewhere
    if group == 128:
        assert (s[4, 1:] == 1e-10).all() and (q[4].float()[128:] == 0).all()


# ---- GEMM with bias, activation, residual --------------------------------------------------------------

def linear_case(scales, batch, M, N, K, bias, residual, seed, gn=128):
    g = gen(seed)
    lead = (batch,) if batch > 1 else ()
    x, w = randn(g, *lead, M, K), randn(g, *lead, N, K, scale=0.05)
    if scales == "token":
        a, sa = quant_rows(x, K)
        b, sb = quant_rows(w, K)
        ad, bd = a.double() * sa.double(), b.double() * sb.double()
    else:
        a, sa = quant_rows(x, 128)
        ad = a.double() * sa.double().repeat_interleave(128, 1)
        if gn == 128:
            b, sb = quant_tiles(w)
            bd = b.double() * sb.double().t().repeat_interleave(128, 0).repeat_interleave(128, 1)
        else:
            b, s = quant_rows(w, 128)
            sb = s.t().contiguous()
            bd = b.double() * s.double().repeat_interleave(128, 1)
    v = ad @ bd.transpose(-1, -2)
    tol = (ad.abs() @ bd.abs().transpose(-1, -2)) * (K / 32 + 2 * K / 128 + 8) * 2.0 ** -23
    bi = randn(g, *lead, N) if bias else None
    re = randn(g, *lead, M, N) if residual else None
    return a, b, sa, sb, bi, re, v, tol


def check_linear(hk, scales, batch, M, N, K, bias=True, act="none", residual=True, gn=128, in_place=False, kernel=None):
    a, b, sa, sb, bi, re, v, tol = linear_case(scales, batch, M, N, K, bias, residual, M * 7 + N + K, gn)
    if bias:
        v, tol = v + bi.double().unsqueeze(-2), tol + (v.abs() + bi.double().abs().unsqueeze(-2)) * 2.0 ** -23
    ref, tol = act64(v, act), act_tol(v, tol, act)
    if residual:
        ref, tol = ref + re.double(), tol + (ref.abs() + re.double().abs()) * 2.0 ** -23
    c, c_ok = (re, lambda: True) if in_place else guarded(*v.shape, dtype=torch.bfloat16)
    gemm = hk.gemm.a8w8_per_token if scales == "token" else hk.gemm.a8w8_blockscale
    gemm.dispatch_epilogue(a, b, c, sa, sb, bi, act, re)
    if kernel:
        assert gemm.hkb_last_kernel() == kernel
    check_bf16(c, ref, tol)
    assert c_ok()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("scales,M,N", [("token", 9, 256), ("token", 130, 264), ("block", 9, 256), ("block", 130, 384)])
def test_linear_activations(hk, scales, M, N, act):
    check_linear(hk, scales, 1, M, N, 256, act=act)


@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("scales,M", [("token", 5), ("token", 200), ("block", 5), ("block", 200)])
def test_linear_optional_operands(hk, scales, M, bias, residual):
    check_linear(hk, scales, 1, M, 256, 384, bias=bias, residual=residual, act="silu")


PTS = "gemm_fp8_kernel<{},pts,epilogue{}>".format
BLOCK = "gemm_fp8_kernel<{},blockscale,epilogue{}>".format


@pytest.mark.parametrize("batch,M,N,K,kernel", [
    (1, 1, 1024, 128, "gemm_fp8_skinny_kernel<epilogue>"), (1, 64, 2064, 1024, "gemm_fp8_skinny_kernel<epilogue>"),
    (1, 5, 1024, 8192, "gemm_fp8_skinny_kernel<epilogue,split>"), (1, 64, 1040, 4224, "gemm_fp8_skinny_kernel<epilogue,split>"),
    (1, 33, 4096, 14336, "gemm_fp8_skinny_kernel<epilogue,split>"),
    (1, 16, 1032, 256, PTS(64, "")), (1, 61, 8, 256, PTS(64, "")), (3, 77, 1032, 384, PTS(64, "")), (2, 13, 520, 256, PTS(64, "")),
    (1, 16, 1032, 4096, PTS(64, ",split")), (1, 61, 1032, 4224, PTS(64, ",split")), (2, 40, 520, 4096, PTS(64, ",split")), (1, 300, 504, 8192, PTS(64, ",split")),
    (1, 127, 80000, 128, PTS(128, "")), (1, 2048, 1024, 8192, PTS(128, "")),
    (1, 300, 1024, 8192, PTS(128, ",split")), (1, 170, 1272, 9728, PTS(128, ",split")),
    (1, 1000, 9000, 256, PTS(256, "")), (1, 2049, 9480, 256, PTS(256, "")), (4, 302, 640, 13824, PTS(128, ",split")),
    (1, 4000, 4040, 2048, PTS("256", "").replace("pts", "pts,pair")), (2, 134, 9584, 4736, PTS("256", "").replace("pts", "pts,pair"))])
def test_linear_per_token_kernels(hk, batch, M, N, K, kernel):
    check_linear(hk, "token", batch, M, N, K, act="gelu_tanh", kernel=kernel)


@pytest.mark.parametrize("M,N,K,gn,kernel", [
    (1, 128, 128, 128, "gemm_fp8_blockscale_skinny_kernel<epilogue>"), (32, 1152, 896, 128, "gemm_fp8_blockscale_skinny_kernel<epilogue>"),
    (17, 28672, 256, 128, "gemm_fp8_blockscale_skinny_kernel<epilogue>"), (32, 1024, 8192, 128, "gemm_fp8_blockscale_skinny_kernel<epilogue,split>"),
    (9, 2048, 4224, 128, "gemm_fp8_blockscale_skinny_kernel<epilogue,split>"), (3, 4096, 14336, 128, "gemm_fp8_blockscale_skinny_kernel<epilogue,split>"),
    (33, 1152, 384, 128, BLOCK(128, "")), (1025, 9728, 256, 128, BLOCK(128, "")),
    (300, 128, 5248, 128, BLOCK(128, ",split")), (40, 128, 8320, 128, BLOCK(128, ",split")),
    (1025, 9728, 1024, 128, BLOCK(256, "")), (300, 4096, 14336, 128, BLOCK(256, ",split")), (600, 1024, 8320, 128, BLOCK(256, ",split")),
    (300, 14336, 4096, 128, BLOCK(256, ",split")), (2047, 8192, 8320, 128, BLOCK(256, ",split")),            # whole waves and a split rest
    (200, 256, 384, 1, BLOCK(128, "").replace("scale", "scale,gn1")), (3, 128, 128, 1, BLOCK(128, "").replace("scale", "scale,gn1"))])
def test_linear_block_scale_kernels(hk, M, N, K, gn, kernel):
    check_linear(hk, "block", 1, M, N, K, act="gelu", gn=gn, kernel=kernel)


@pytest.mark.parametrize("scales,M,N,gn", [("token", 30, 256, 0), ("token", 300, 1032, 0), ("token", 2048, 9472, 0), ("block", 30, 256, 128),
                                           ("block", 300, 256, 128), ("block", 1025, 9728, 128), ("block", 40, 256, 1)])
def test_linear_residual_in_place(hk, scales, M, N, gn):
    check_linear(hk, scales, 1, M, N, 256, act="relu", gn=gn or 128, in_place=True)


@pytest.mark.parametrize("scales,batch,M,N", [("token", 1, 40, 512), ("token", 2, 300, 1032), ("token", 1, 2048, 9472), ("block", 1, 20, 512),
                                              ("block", 1, 300, 512), ("block", 1, 1025, 9728)])
def test_linear_with_nothing_in_the_epilogue_is_the_plain_gemm(hk, scales, batch, M, N):
    a, b, sa, sb, _, _, v, _ = linear_case(scales, batch, M, N, 256, False, False, 1)
    plain, c = torch.empty(v.shape, dtype=torch.bfloat16, device=DEV), torch.empty(v.shape, dtype=torch.bfloat16, device=DEV)
    gemm = hk.gemm.a8w8_per_token if scales == "token" else hk.gemm.a8w8_blockscale
    gemm.dispatch(a, b, plain, sa, sb)
    gemm.dispatch_epilogue(a, b, c, sa, sb)
    assert torch.equal(c, plain)


def test_linear_result_on_an_offset_view(hk):
    """C 16-byte but not 32-byte aligned: the decode kernel's and the tiles' wide stores do not apply."""
    M, N, K = 24, 256, 256
    a, b, sa, sb, bi, re, v, tol = linear_case("token", 1, M, N, K, True, True, 2)
    c = torch.empty(M * N + 8, dtype=torch.bfloat16, device=DEV)[8:].view(M, N)
    re_off = torch.empty(M * N + 8, dtype=torch.bfloat16, device=DEV)[8:].view(M, N).copy_(re)
    hk.gemm.a8w8_per_token.dispatch_epilogue(a, b, c, sa, sb, bi, "none", re_off)
    ref = v + bi.double() + re.double()
    check_bf16(c, ref, tol + ref.abs() * 2.0 ** -22 + 2.0 ** -20)


def test_activations_over_the_whole_range(hk):
    """One product per value: x = code * scale through an identity weight, so the epilogue's argument is exact.  Tails, zeros,
    infinities and NaN; the result against 64 bits, relative to its own value."""
    K = N = 128
    M = 256
    v = torch.cat([torch.linspace(-30, 30, 16384), torch.linspace(-12, -3, 16384)]).to(DEV)
    b = torch.eye(N, K, device=DEV).to(E4M3)
    one = torch.ones(N, device=DEV)
    for act in ACTS:
        # sa is a row's scale: x[m, k] = 1 everywhere, the value comes in as the (fp32) row scale
        got = []
        for m0 in range(0, v.numel(), M):
            a = torch.ones(M, K, device=DEV).to(E4M3)
            c = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
            hk.gemm.a8w8_per_token.dispatch_epilogue(a, b, c, v[m0:m0 + M].contiguous(), one, None, act, None)
            got.append(c[:, 0])
        ref = act64(v.double(), act)
        err = (torch.cat(got).double() - ref).abs()
        # erfc and exp in fp32 at these arguments: a few units of 2^-23 times the argument's square (its rounding, amplified)
        assert (err <= ref.abs() * (2.0 ** -8 + 2.0 ** -12) + 2.0 ** -126).all(), act
    edge = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 3e38, -3e38, 1e-38], device=DEV)
    want = {"none": edge, "relu": torch.tensor([float("inf"), 0, float("nan"), 0, 0, 3e38, 0, 1e-38], device=DEV)}
    for act in ACTS:
        a, c = torch.ones(8, K, device=DEV).to(E4M3), torch.empty(8, N, dtype=torch.bfloat16, device=DEV)
        b0 = torch.ones(N, K, device=DEV).to(E4M3)
        hk.gemm.a8w8_per_token.dispatch_epilogue(a, b0, c, edge / K, one, None, act, None)
        got = c[:, 0].float()
        assert got[0] == float("inf") and got[2].isnan() and got[3] == 0 and got[4] == 0 and got[5] > 2.9e38
        if act in want:
            assert torch.equal(got[[1, 6]], want[act][[1, 6]].bfloat16().float())
        else:
            assert got[1].isnan() or got[1] == 0                         # -inf * 0 or its limit
            assert got[6] == 0


# ---- gated --------------------------------------------------------------------------------------------

def gated_case(M, F, K, seed):
    g = gen(seed)
    a, sa = quant_rows(randn(g, M, K), 128)
    b, sb = quant_tiles(randn(g, 2 * F, K, scale=2.0 / K ** 0.5))
    ad = a.double() * sa.double().repeat_interleave(128, 1)
    bd = b.double() * sb.double().t().repeat_interleave(128, 0).repeat_interleave(128, 1)
    v = ad @ bd.t()
    tol = (ad.abs() @ bd.abs().t()) * (K / 32 + 2 * K / 128 + 8) * 2.0 ** -23
    return a, b, sa, sb, v[:, :F], v[:, F:], tol[:, :F], tol[:, F:]


def check_gated(hk, M, F, K, act, fp8, kernel=None):
    a, b, sa, sb, gate, up, tg, tu = gated_case(M, F, K, M + F + K)
    y = act64(gate, act) * up
    t = act_tol(gate, tg, act)
    tol = t * up.abs() + act64(gate, act).abs() * tu + t * tu + y.abs() * 2.0 ** -23
    if fp8:
        c, c_ok = guarded(M, F, dtype=E4M3)
        cs, s_ok = guarded(M, F // 128, dtype=torch.float32)
        hk.gemm.a8w8_blockscale.dispatch_gated(a, b, c, sa, sb, cs, act)
        check_codes(c, cs, y, tol, 128)
    else:
        c, c_ok = guarded(M, F, dtype=torch.bfloat16)
        s_ok = c_ok
        hk.gemm.a8w8_blockscale.dispatch_gated(a, b, c, sa, sb, None, act)
        check_bf16(c, y, tol)
    if kernel:
        assert hk.gemm.a8w8_blockscale.hkb_last_kernel() == kernel
    assert c_ok() and s_ok()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [5, 140])
def test_gated_activations(hk, M, act, fp8):
    check_gated(hk, M, 256, 256, act, fp8)


DECODE = "gemm_fp8_blockscale_skinny_kernel<gated{}>".format
GATED = "gemm_fp8_kernel<{},blockscale,gated{}>".format


@pytest.mark.parametrize("M,F,K,fp8,kernel", [
    (1, 128, 128, False, DECODE("")), (1, 128, 128, True, DECODE("")), (16, 14336, 256, True, DECODE("")), (17, 1152, 1152, False, DECODE("")),
    (32, 28672, 384, True, DECODE("")), (32, 640, 2176, False, DECODE(",split")), (9, 1024, 4224, True, DECODE(",split")), (31, 128, 8192, True, DECODE(",split")),
    (33, 128, 128, True, GATED(256, "")), (33, 128, 128, False, GATED(128, "")), (257, 640, 384, False, GATED(128, "")),
    (200, 640, 4224, False, GATED(128, ",split")), (130, 1024, 8192, False, GATED(128, ",split")), (40, 128, 8320, False, GATED(128, ",split")),
    (300, 1152, 4224, True, GATED(256, ",split")), (70, 256, 2048, True, GATED(256, ",split")), (40, 128, 8320, True, GATED(256, ",split")),
    (512, 14336, 4096, True, GATED(256, ",split")), (500, 14336, 4224, False, GATED(256, ",split")),            # whole waves and a split rest
    (1025, 9600, 256, False, GATED(256, "")), (1300, 4096, 128, True, GATED(256, ""))])
def test_gated_kernels(hk, M, F, K, fp8, kernel):
    check_gated(hk, M, F, K, "silu", fp8, kernel)


def test_gated_zero_infinite_and_nan_rows(hk):
    for M, F, K in ((6, 256, 256), (70, 256, 256), (6, 256, 4096), (70, 256, 4096)):
        a, b, sa, sb, *_ = gated_case(M, F, K, 9)
        sa[0] = 0
        sa[1] = float("nan")
        sa[2, 0] = float("inf")
        c, cs = torch.empty(M, F, dtype=E4M3, device=DEV), torch.empty(M, F // 128, device=DEV)
        hk.gemm.a8w8_blockscale.dispatch_gated(a, b, c, sa, sb, cs, "silu")
        assert (c[0].float() == 0).all() and (cs[0] == 1e-10).all()
        assert c[1].float().isnan().all() and cs[1].isnan().all()
        assert not cs[2].isfinite().any()
        assert c[3:].float().isfinite().all() and cs[3:].isfinite().all()


# ---- together -------------------------------------------------------------------------------------------

class GatedLayer:
    """A pre-norm gated feed-forward layer: x = branch output, h = residual stream."""

    def __init__(self, M, D, F, seed):
        g = gen(seed)
        self.x, self.h, self.w = randn(g, M, D), randn(g, M, D), (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).bfloat16()
        self.wgu, self.sgu = quant_tiles(randn(g, 2 * F, D, scale=2 / D ** 0.5))
        self.wd, self.sd = quant_tiles(randn(g, D, F, scale=2 / F ** 0.5))
        self.q, self.qs = torch.empty(M, D, dtype=E4M3, device=DEV), torch.empty(M, D // 128, device=DEV)
        self.a, self.as_ = torch.empty(M, F, dtype=E4M3, device=DEV), torch.empty(M, F // 128, device=DEV)

    def __call__(self, hk):
        hk.fused_add_rmsnorm_fp8_quant_fwd(self.x, self.h, self.w, self.q, self.qs, self.h, EPS)
        hk.gemm.a8w8_blockscale.dispatch_gated(self.q, self.wgu, self.a, self.qs, self.sgu, self.as_, "silu")
        hk.gemm.a8w8_blockscale.dispatch_epilogue(self.a, self.wd, self.h, self.as_, self.sd, None, "none", self.h)
        return self.h

    def reference(self):
        """64 bits throughout, the activations unquantized, the stored stream rounded once."""
        def deq(w, s):
            return w.double() * s.double().t().repeat_interleave(128, 0).repeat_interleave(128, 1)
        h = (self.x.float() + self.h.float()).bfloat16().double()
        y = h / ((h * h).mean(1, keepdim=True) + EPS).sqrt() * self.w.double()
        p = y @ deq(self.wgu, self.sgu).t()
        F = p.shape[1] // 2
        return h, (act64(p[:, :F], "silu") * p[:, F:]) @ deq(self.wd, self.sd).t()


@pytest.mark.parametrize("M,D,F", [(1, 512, 1152), (24, 1024, 2048), (200, 512, 1152), (1200, 1024, 4096)])
def test_gated_layer(hk, M, D, F):
    """Against the unquantized layer.  A code is off by at most 2^-4 of its value, on average (uniform within a step) 2^-4 / sqrt(3) at
    the bottom of a binade and half of that at its top; the errors are independent, so the update, a sum over all of them, is off by
    about 2.6 % of its norm for either of the two quantizations: sqrt(2) * 2.6 % plus the gate's slope, held to 6 %."""
    layer = GatedLayer(M, D, F, M)
    h, update = layer.reference()
    got = layer(hk).double() - h
    assert (got - update).norm() <= 0.06 * update.norm() + 2.0 ** -8 * h.norm()


def test_layers_captured_replayed_and_on_two_streams(hk):
    shapes = [(24, 1024, 2048), (200, 512, 1152), (150, 512, 8192), (8, 512, 8192)]
    for M, D, F in shapes:
        eager, graphed, other = (GatedLayer(M, D, F, 1) for _ in range(3))
        start = eager.h.clone()
        eager(hk)
        graphed(hk)                                                   # warm-up outside capture
        graphed.h.copy_(start)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphed(hk)
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2):
            other(hk)
        for t in (graphed.q, graphed.a, graphed.as_, graphed.qs):
            t.view(torch.uint8).fill_(0)
        graphed.h.copy_(start)
        other.h.copy_(start)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            g.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphed.h, eager.h) and torch.equal(other.h, eager.h)
        # new inputs, same graph
        graphed.x.mul_(-0.5)
        eager.x.mul_(-0.5)
        graphed.h.copy_(start)
        eager.h.copy_(start)
        g.replay()
        eager(hk)
        torch.cuda.synchronize()
        assert torch.equal(graphed.h, eager.h)


def test_layers_on_a_side_stream_match(hk):
    a, b = GatedLayer(20, 512, 1152, 4), GatedLayer(20, 512, 1152, 4)
    want = a(hk).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b(hk)
    side.synchronize()
    assert torch.equal(b.h, want)


def test_layer_without_gate_per_token(hk):
    """add_norm (row scales) -> linear(bias, gelu) -> per-token quantizer -> linear(bias, residual)."""
    M, D, F = 150, 512, 1032
    g = gen(11)
    x, h = randn(g, M, D), randn(g, M, D)
    w = (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).bfloat16()
    w1, s1 = quant_rows(randn(g, F, D, scale=2 / D ** 0.5), D)
    F2 = 1024                                                        # the second product's K: a multiple of 128
    w2, s2 = quant_rows(randn(g, D, F2, scale=2 / F2 ** 0.5), F2)
    b1, b2 = randn(g, F), randn(g, D)
    q, qs = torch.empty(M, D, dtype=E4M3, device=DEV), torch.empty(M, 1, device=DEV)
    hk.fused_add_rmsnorm_fp8_quant_fwd(x, h, w, q, qs, h, EPS)
    total = h.double()
    c1 = torch.empty(M, F, dtype=torch.bfloat16, device=DEV)
    hk.gemm.a8w8_per_token.dispatch_epilogue(q, w1, c1, qs, s1, b1, "gelu", None)
    mid = c1[:, :F2].contiguous()
    q2, qs2 = torch.empty(M, F2, dtype=E4M3, device=DEV), torch.empty(M, 1, device=DEV)
    hk.per_token_quant_fwd(mid, q2, qs2)
    hk.gemm.a8w8_per_token.dispatch_epilogue(q2, w2, h, qs2, s2, b2, "none", h)
    y = total / ((total * total).mean(1, keepdim=True) + EPS).sqrt() * w.double()
    m = act64(y @ (w1.double() * s1.double()).t() + b1.double(), "gelu")[:, :F2]
    update = m @ (w2.double() * s2.double()).t() + b2.double()
    assert (h.double() - total - update).norm() <= 0.06 * update.norm() + 2.0 ** -8 * total.norm()

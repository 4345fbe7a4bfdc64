"""GPU tier: forms of the feed-forward operators beside those of test_feed_forward_gpu.py, with that file's references and tolerances."""
import pytest
import torch

from test_feed_forward_gpu import (DEV, E4M3, act64, act_tol, check_bf16, check_linear, check_norm, gated_case, gen, linear_case, norm_case,
                                   quant_rows)

pytestmark = pytest.mark.gpu
SPLIT = "gemm_fp8_skinny_kernel<epilogue,split>"


@pytest.mark.parametrize("M", [1, 8])
@pytest.mark.parametrize("N,K", [(16, 2048), (128, 14336), (256, 2048), (256, 8192)])
def test_narrow_layer_of_a_few_tokens_split(hk, M, N, K):
    check_linear(hk, "token", 1, M, N, K, act="silu", kernel=SPLIT)


def test_narrow_split_layers_back_to_back_and_on_two_streams(hk):
    """Narrow split calls in a chain, and two chains on streams of their own: the results of a call alone."""
    cases = []
    for M, N, K in ((1, 256, 4096), (8, 128, 8192), (8, 256, 14336), (4, 16, 2048)):
        a, b, sa, sb, bi, re, *_ = linear_case("token", 1, M, N, K, True, True, M + N)
        cases.append((a, b, sa, sb, bi, re, torch.empty_like(re)))

    def chain(outs):
        for (a, b, sa, sb, bi, re, _), c in zip(cases, outs):
            hk.gemm.a8w8_per_token.dispatch_epilogue(a, b, c, sa, sb, bi, "gelu", re)

    for a, b, sa, sb, bi, re, want in cases:
        hk.gemm.a8w8_per_token.dispatch_epilogue(a, b, want, sa, sb, bi, "gelu", re)
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[[torch.empty_like(c[6]) for c in cases] for _ in range(20)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(20):
        for s, out in zip(streams, outs):
            with torch.cuda.stream(s):
                chain(out[i])
    torch.cuda.synchronize()
    for out in outs:
        for got in out:
            assert all(torch.equal(c, case[6]) for c, case in zip(got, cases))


class Duck:
    """What the boundary needs of a tensor, and nothing else."""

    def __init__(self, t):
        self.shape, self.keep = tuple(t.shape), t

    def data_ptr(self):
        return self.keep.data_ptr()


class Named(torch.Tensor):
    """A subclass: read through the general path."""


@pytest.mark.parametrize("M", [5, 40])
@pytest.mark.parametrize("wrap", [Duck, lambda t: t.as_subclass(Named)])
def test_gated_codes_of_other_tensor_types(hk, M, wrap):
    """Operands that are not plain tensors, with and without a workspace behind the call."""
    F, K = 256, 256
    a, b, sa, sb, *_ = gated_case(M, F, K, 3)
    want = [torch.empty(M, F, dtype=E4M3, device=DEV), torch.empty(M, F // 128, device=DEV)]
    hk.gemm.a8w8_blockscale.dispatch_gated(a, b, want[0], sa, sb, want[1], "silu")
    got = [torch.empty_like(t) for t in want]
    hk.gemm.a8w8_blockscale.dispatch_gated(wrap(a), wrap(b), wrap(got[0]), wrap(sa), wrap(sb), wrap(got[1]), "silu")
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(got, want))


# ---- codes of values that are known exactly: bit for bit those of an IEEE division ------------------------

def same_codes(q, s, y, group):
    want_q, want_s = quant_rows(y, group)
    assert torch.equal(s.view_as(want_s), want_s)
    differ = (q.view(torch.uint8) != want_q.view(torch.uint8)).sum().item()
    assert differ == 0, f"{differ} of {q.numel()} codes"


@pytest.mark.parametrize("offset", [0, 8])                            # 16- and 8-element chunks
@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("D", [1024, 4096, 8192, 32768])
def test_add_norm_codes_of_exact_values(hk, D, per_row, offset):
    """h = +-1 in every column and eps = 0: the norm is 1 exactly and y = +-w.  Gains of few bits put quotients on the edge between two
    codes, where a quotient that is one unit off goes to the other side."""
    g = gen(D + offset)
    M = 8
    for bits in (3, 4, 5, 6, 8):
        w = torch.randint(0, 1 << bits, (D,), generator=g, device=DEV).bfloat16()
        h = torch.randint(0, 2, (M, D), generator=g, device=DEV) * 2.0 - 1
        def view(t):                                                  # noqa: E306
            return torch.empty(M * D + offset, dtype=torch.bfloat16, device=DEV)[offset:].view(M, D).copy_(t)
        x, r, out = view(0.25 * h), view(0.75 * h), view(torch.zeros_like(h))
        q, s = torch.empty(M, D, dtype=E4M3, device=DEV), torch.empty(M, 1 if per_row else D // 128, device=DEV)
        hk.fused_add_rmsnorm_fp8_quant_fwd(x, r, w, q, s, out, 0.0)
        same_codes(q, s, h * w.float(), D if per_row else 128)


@pytest.mark.parametrize("M,F,K,kernel", [(5, 512, 256, "gemm_fp8_blockscale_skinny_kernel<gated>"), (20, 256, 8192, "gemm_fp8_blockscale_skinny_kernel<gated,split>"),
                                          (200, 512, 256, "gemm_fp8_kernel<256,blockscale,gated>"), (70, 256, 4096, "gemm_fp8_kernel<256,blockscale,gated,split>")])
def test_gated_codes_of_exact_values(hk, M, F, K, kernel):
    """gate = 1 without activation, up = a sum of two or three small integers: y is known exactly."""
    g = gen(M + F + K)
    a, b = torch.zeros(M, K, device=DEV), torch.zeros(2 * F, K, device=DEV)
    b[:F, 2] = 1
    b[F:, 0] = 16.0 * torch.randint(0, 16, (F,), generator=g, device=DEV)
    b[F:, 1] = torch.randint(-15, 16, (F,), generator=g, device=DEV).float()
    a[:, 0] = torch.randint(-1, 2, (M,), generator=g, device=DEV).float()
    a[:, 1] = torch.randint(0, 4, (M,), generator=g, device=DEV).float()
    a[:, 2] = 1
    y = a @ b[F:].t()
    sa, sb = torch.ones(M, K // 128, device=DEV), torch.ones(K // 128, 2 * F // 128, device=DEV)
    c, cs = torch.empty(M, F, dtype=E4M3, device=DEV), torch.empty(M, F // 128, device=DEV)
    hk.gemm.a8w8_blockscale.dispatch_gated(a.to(E4M3), b.to(E4M3), c, sa, sb, cs, "none")
    assert hk.gemm.a8w8_blockscale.hkb_last_kernel() == kernel
    same_codes(c, cs, y, 128)


# ---- every norm kernel: chunks of 8 on wide rows, 3, 6 and 8 of them per thread --------------------------------

@pytest.mark.parametrize("M,D", [(3, 4232), (2500, 520), (3, 8200), (40, 12280), (2, 12296)])
def test_add_norm_row_scales_of_odd_widths(hk, M, D):
    check_norm(hk, *norm_case(M, D, M + D), D)


@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("M,D", [(5, 128), (3, 4224), (2400, 512), (7, 8192), (3, 16384), (2, 32768)])
def test_add_norm_on_views_that_start_inside_32_bytes(hk, M, D, per_row):
    x, r, w = norm_case(M, D, M + D)
    x, r = (torch.empty(M * D + 8, dtype=torch.bfloat16, device=DEV)[8:].view(M, D).copy_(t) for t in (x, r))
    check_norm(hk, x, r, w, D if per_row else 128)


# ---- split kernels: the residual stream updated in place, operands that start inside 32 bytes -------------------

PTS = "gemm_fp8_kernel<{},pts,epilogue{}>".format
BLOCK = "gemm_fp8_kernel<{},blockscale,epilogue{}>".format
BLOCK_DECODE = "gemm_fp8_blockscale_skinny_kernel<epilogue{}>".format


@pytest.mark.parametrize("scales,batch,M,N,K,kernel", [
    ("token", 1, 5, 1024, 8192, SPLIT), ("token", 1, 64, 1040, 4224, SPLIT), ("token", 1, 8, 128, 4096, SPLIT),
    ("token", 1, 61, 1032, 4224, PTS(64, ",split")), ("token", 2, 40, 520, 4096, PTS(64, ",split")), ("token", 1, 300, 1024, 8192, PTS(128, ",split")),
    ("block", 1, 9, 2048, 4224, BLOCK_DECODE(",split")), ("block", 1, 32, 1024, 8192, BLOCK_DECODE(",split")),
    ("block", 1, 300, 128, 5248, BLOCK(128, ",split")), ("block", 1, 600, 1024, 8320, BLOCK(256, ",split")),
    ("block", 1, 2047, 8192, 8320, BLOCK(256, ",split"))])                          # whole waves and a split rest
def test_linear_split_in_place(hk, scales, batch, M, N, K, kernel):
    check_linear(hk, scales, batch, M, N, K, act="silu", in_place=True, kernel=kernel)


@pytest.mark.parametrize("scales,batch,M,N,K,kernel", [
    ("token", 1, 16, 1024, 256, PTS(64, "")), ("token", 1, 60, 1024, 4096, PTS(64, ",split")), ("token", 1, 5, 1024, 8192, PTS(64, ",split")),
    ("token", 2, 77, 1032, 384, PTS(64, "")), ("token", 1, 2048, 1024, 8192, PTS(128, "")), ("token", 1, 300, 1024, 8192, PTS(128, ",split")),
    ("token", 1, 1000, 9008, 256, PTS(256, "")), ("token", 1, 4000, 4048, 2048, PTS("256", "").replace("pts", "pts,pair")),
    ("block", 1, 9, 256, 256, BLOCK_DECODE("")), ("block", 1, 9, 2048, 4224, BLOCK_DECODE(",split")), ("block", 1, 300, 256, 256, BLOCK(128, "")),
    ("block", 1, 300, 128, 5248, BLOCK(128, ",split")), ("block", 1, 1025, 9728, 1024, BLOCK(256, "")), ("block", 1, 600, 1024, 8320, BLOCK(256, ",split"))])
def test_linear_views_that_start_inside_32_bytes(hk, scales, batch, M, N, K, kernel):
    """Residual, bias and (per-token) the result 16-byte but not 32-byte aligned."""
    a, b, sa, sb, bi, re, v, tol = linear_case(scales, batch, M, N, K, True, True, M + N + K)

    def off(t):
        return torch.empty(t.numel() + 8, dtype=t.dtype, device=DEV)[8:].view(t.shape).copy_(t)
    gemm = hk.gemm.a8w8_per_token if scales == "token" else hk.gemm.a8w8_blockscale
    c = off(re) if scales == "token" else torch.empty_like(re)
    gemm.dispatch_epilogue(a, b, c, sa, sb, off(bi), "relu", off(re))
    assert gemm.hkb_last_kernel() == kernel
    ref = v + bi.double().unsqueeze(-2)
    tol = tol + (v.abs() + bi.double().abs().unsqueeze(-2)) * 2.0 ** -23
    ref, tol = act64(ref, "relu"), act_tol(ref, tol, "relu")
    ref, tol = ref + re.double(), tol + (ref.abs() + re.double().abs()) * 2.0 ** -23
    check_bf16(c, ref, tol)


# ---- activations to the accuracy that they are written for --------------------------------------------------------

@pytest.mark.parametrize("act,low,high", [("silu", -60.0, 60.0), ("gelu", -11.0, 12.0), ("gelu_tanh", -9.0, 12.0)])
def test_activations_below_the_result_s_rounding(hk, act, low, high):
    """The residual takes away the leading part: r = -bf16(ref), so the result is the rest, act(v) + r, exact in fp32 (both are within
    2^-8 of one another) and rounded to bf16.  Of a dense grid, the arguments whose value is within 2^-14 of a bf16: that rounding is
    under 2^-8 * 2^-14.  Error of the activation relative to its value, in units of 2^-23 (ex2 is good to two units, rcp to one):
      silu: the exponent's argument |v| log2(e) / 2 rounds twice, which the square doubles: |v|; the square of ex2 4; reciprocal and
        products 4;
      gelu_tanh: the same of z = 1.6 v + 0.07 v^3, and z's own five roundings (two of them of constants), each half a unit of |z|: 3 |z| + 8;
      gelu: the exponent's argument v^2 log2(e) / 4 with three roundings, doubled, 0.75 v^2; ex2 4, the fit 7.3, Horner steps and their
        argument 6, products 2."""
    K = N = 128
    v = torch.linspace(low, high, 1 << 21, dtype=torch.float64, device=DEV).float()
    ref = act64(v.double(), act)
    near = ((ref - ref.bfloat16().double()).abs() <= ref.abs() * 2.0 ** -14) & (ref.abs() >= 2.0 ** -100)
    pick = near.nonzero().flatten()
    pick = pick[torch.linspace(0, pick.numel() - 1, 32768, dtype=torch.float64, device=DEV).long()]
    v, ref = v[pick].contiguous(), ref[pick]
    lead = ref.bfloat16()
    M = v.numel()
    a, b = torch.ones(M, K, device=DEV).to(E4M3), torch.eye(N, K, device=DEV).to(E4M3)
    c = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
    res = (-lead)[:, None].expand(M, N).contiguous()
    hk.gemm.a8w8_per_token.dispatch_epilogue(a, b, c, v, torch.ones(N, device=DEV), None, act, res)
    assert torch.equal(c, c[:, :1].expand(M, N))
    w = v.double().abs()
    units = {"silu": w + 8, "gelu_tanh": 3 * (1.59577 * w + 0.0713549 * w ** 3) + 8, "gelu": 0.75 * w * w + 19.3}[act]
    rest = ref - lead.double()
    err = (c[:, 0].double() - rest).abs()
    bound = units * 2.0 ** -23 * ref.abs()
    bound = bound + (rest.abs() + bound) * 2.0 ** -8
    assert (err <= bound).all(), f"{(err > bound).sum().item()} of {M}, worst {(err / bound).max().item():.3g} of the bound"

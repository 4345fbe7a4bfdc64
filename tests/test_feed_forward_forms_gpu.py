"""GPU tier: forms of the feed-forward operators beside those of test_feed_forward_gpu.py, with that file's references and tolerances."""
import pytest
import torch

from test_feed_forward_gpu import DEV, E4M3, check_linear, gated_case, gen, linear_case, quant_rows

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

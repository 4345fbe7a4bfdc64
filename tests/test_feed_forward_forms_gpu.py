"""GPU tier: forms of the feed-forward operators beside those of test_feed_forward_gpu.py, with that file's references and tolerances."""
import pytest
import torch

from test_feed_forward_gpu import DEV, E4M3, check_linear, gated_case, linear_case

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

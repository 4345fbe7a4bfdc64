"""CPU tier: which tensors the Python boundary reads."""
import pytest
import torch

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("lead", [7, 8, 9, 62, 63, 64, 80])
def test_any_number_of_leading_dimensions_is_a_batch(hk, lead):
    ones = (1,) * lead
    a, b = torch.zeros(*ones, 4, 128, dtype=E4M3), torch.zeros(*ones, 256, 128, dtype=E4M3)
    c, sa, sb = torch.zeros(*ones, 4, 256, dtype=torch.bfloat16), torch.ones(*ones, 4), torch.ones(*ones, 256)
    for call in (hk.gemm.a8w8_per_token.dispatch, hk.gemm.a8w8_per_token.dispatch_epilogue):
        with pytest.raises(RuntimeError, match="CUDA"):         # all that is wrong with them is where they are
            call(a, b, c, sa, sb)
        with pytest.raises(RuntimeError, match="same K"):       # the last two extents are read, whatever is ahead of them
            call(a, torch.zeros(*ones, 256, 256, dtype=E4M3), c, sa, sb)

"""Table rows that no token names, and the padding row, in the embedding gradient:
zeros (with no sign) whatever the scale is, where the sort has zeroed them and
where the sums' kernel writes them."""

import pytest
import torch

import flagsparse_amd as fs

pytestmark = pytest.mark.gpu
DEV = "cuda"

# tokens, table rows, width: a short sort whose zeros end inside the table (64 MB of f32 and f16), a longer sort,
# and rows shorter than a slice
SIZES = [(5, 4400, 4096), (5, 8500, 4096), (5000, 6000, 24), (5000, 6000, 3), (300, 7, 5)]


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), 1e39, -2.0])
@pytest.mark.parametrize("n,n_rows,width", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_rows_without_tokens_are_zero(dtype, n, n_rows, width, scale):
    g = torch.Generator().manual_seed(n + n_rows)
    tokens = torch.randint(0, n_rows, (n,), generator=g)
    tokens[: n // 2] = n_rows - 2  # more than 64 of them where there are as many tokens
    tokens[tokens == 1] = 0
    grad = torch.ones((n, width), dtype=dtype)
    for padding in (None, n_rows - 2, 1):
        got = fs.flagsparse_embedding_grad(grad.to(DEV), tokens.to(DEV), n_rows, scale=scale, padding_idx=padding)
        named = torch.bincount(tokens, minlength=n_rows) > 0
        if padding is not None:
            named[padding] = False
        empty = got[~named.to(DEV)]
        assert bool((empty == 0).all()) and not bool(torch.signbit(empty).any())
        kept = got[named.to(DEV)]
        if scale == -2.0:
            counts = torch.bincount(tokens, minlength=n_rows)[named].to(DEV)
            assert torch.equal(kept, (-2.0 * counts[:, None].double()).to(dtype).expand_as(kept))
        else:
            assert not bool(torch.isfinite(kept).any())

"""f32 prompts whose rows of k and v lie more than 2^23 elements apart, as views of a larger array, against
the same rows side by side: the same bits."""
import pytest
import torch

from borch_amd import attention as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [40, 130])  # tiles split where they are used, and before
def test_f32_rows_far_apart(dev, n):
    print(f"prompt f32 far rows n={n}", flush=True)
    dim, step = 128, 2 ** 23 + 64
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, h, dim, generator=g).to(dev) for h in (4, 2, 2))
    cu = torch.tensor([0, n - 20, n], dtype=torch.int32, device=dev)
    wide = torch.empty(n * step, device=dev)
    fk = wide.as_strided((n, 2, dim), (step, dim, 1))
    fv = wide.as_strided((n, 2, dim), (step, dim, 1), 2 * dim)
    fk.copy_(k)
    fv.copy_(v)
    assert torch.equal(A.prompt_attention(q, fk, fv, cu), A.prompt_attention(q, k, v, cu))

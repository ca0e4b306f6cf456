"""prompt_attention where one token draws nearly all of the weight and has values of 0: the outputs are the sum of
many small weights, each rounded to the type.

Tolerance relative to sum_i p_i |v_i|: half a step of the type for each p (2^-11 fp16, 2^-8 bf16; all are above
fp16's least normal number, 2^-25 of the largest) and for the output, (n + 16) 2^-24 for the sums, and for the
exponents' arguments (below 32) 32 2^-24, twice."""
import pytest
import torch

from borch_amd import attention as A
from oracle import decode as D

pytestmark = pytest.mark.gpu

HALF = {"bf16": (torch.bfloat16, 2.0 ** -8), "f16": (torch.float16, 2.0 ** -11), "f32": (torch.float32, 0.0)}


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,heads,causal", [(64, 2, True), (128, 2, True), (64, 64, False), (128, 64, False)])
@pytest.mark.parametrize("lead", [4.0, 8.0, 12.0, 14.0, 17.0])
def test_a_token_that_leads(dev, kind, dim, heads, causal, lead):
    print(f"prompt {kind} dim={dim} heads={heads} causal={causal} lead={lead}", flush=True)
    dt, half = HALF[kind]
    n = 1500
    g = torch.Generator().manual_seed(dim)
    q, k = torch.zeros(n, heads, dim), torch.zeros(n, 1, dim)
    q[:, :, 7] = 1.0
    k[:, 0, 7] = -8.0 * (lead - 0.5 * torch.rand(n, generator=g))
    k[0] = 0
    v = 8.0 * torch.randn(n, 1, dim, generator=g) + 20.0
    v[0] = 0
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    cu = torch.tensor([0, n], dtype=torch.int32)
    got = A.prompt_attention(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), causal=causal, scale=0.125).cpu().double()
    rows = [1, 100, 700, n - 1]
    seen = torch.ones(n, n, dtype=torch.bool)
    seen = (seen.tril() if causal else seen)[rows]
    want, _, size = D.softmax_rows(q[rows, 0], k[:, 0], v[:, 0], seen, 0.125)
    tol = size * (2 * half + (n + 16 + 64) * 2.0 ** -24) + {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}[kind]
    for j in (0, heads - 1):
        off = (got[rows, j] - want).abs()
        assert bool((off <= tol).all()), f"off by {float((off / size).max()):.3g} of the size"

"""The decoder's attention where each low piece of its operands decides the result (oracle/pieces.py, whose bounds
test_pieces_host.py shows to fail without any one of the products)."""
import pytest
import torch

from borch_amd import attention as A
from borch_amd import kv4
from oracle import pieces as P

pytestmark = pytest.mark.gpu

H = 8  # key-value heads, each with inputs of its own
FORMS = [(90, 1), (300, 1), (300, 33)]  # tokens, query heads to a key-value head: split where used; two waves a query; one


def prompt(dev, q, k, v, **more):
    """q [n, H, 2], k [n, H, 2] in two channels of dim; the query heads repeated."""
    n, _, dim = v.shape
    group = more.pop("group")
    wide = torch.zeros(2, n, H, dim)
    wide[0][..., [3, dim - 2]], wide[1][..., [3, dim - 2]] = q, k
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    out = A.prompt_attention(wide[0].to(dev).repeat_interleave(group, 1), wide[1].to(dev), v.to(dev), cu, causal=False,
                             scale=0.125)
    assert torch.equal(out[:, ::group], out[:, group - 1::group])
    return out[:, ::group].cpu().double()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,group", FORMS)
@pytest.mark.parametrize("heavy", [(5, 40), (37, 70), (33, 2)])
def test_f32_prompt_scores(dev, dim, n, group, heavy):
    print(f"pieces prompt scores dim={dim} n={n} group={group} heavy={heavy}", flush=True)
    q, k, v = torch.empty(n, H, 2), torch.empty(n, H, 2), torch.randn(n, H, dim)
    for h in range(H):
        q[:, h], pair = P.close_scores(n, 10 * h)
        k[:, h] = -pair.sum(0)
        k[list(heavy), h] = pair
    v[heavy[0]], v[heavy[1]] = 0, 1
    got = prompt(dev, q, k, v, group=group)
    for h in range(H):
        pair, v1 = k[list(heavy), h], torch.ones(dim)
        want = P.exact(q[:, h], pair, v1, 0.125)
        tol = P.score_bound(q[:, h], pair, v1, 0.125, 20 * 2.0 ** -24) + P.WEIGHT_BOUND * want
        assert bool(((got[:, h] - want).abs() <= tol).all()), h


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,group", FORMS)
def test_f32_prompt_weights_and_values(dev, dim, n, group):
    print(f"pieces prompt weights dim={dim} n={n} group={group}", flush=True)
    heavy = (7, 45)
    q, k, v = torch.zeros(n, H, 2), torch.zeros(n, H, 2), torch.randn(n, H, dim)
    q[..., 0], k[..., 0] = 1, -1600
    v[heavy[0]] = 0
    for h in range(H):
        k[list(heavy), h, 0] = 8 * torch.round(P.rough((2,), 0.0, 2.0, h).double() * 16).float() / 16
        v[heavy[1], h] = P.rough((dim,), 1.0, 2.0, h + 50)
    got = prompt(dev, q, k, v, group=group)
    for h in range(H):
        want = P.exact(q[:, h], k[list(heavy), h], v[heavy[1], h], 0.125)
        assert bool(((got[:, h] - want).abs() <= P.WEIGHT_BOUND * want).all()), h
    # one key with all of the weight: its values to the last bit
    k[heavy[0]] = -1600
    assert torch.equal(prompt(dev, q, k, v, group=group), v[heavy[1]].double().expand(n, H, dim))


@pytest.mark.parametrize("kind,half", [("f32", 0.0), ("f16", 2.0 ** -11), ("bf16", 2.0 ** -8)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [300, 3000])  # one launch, and shares that are joined
@pytest.mark.parametrize("group", [1, 20])  # one row tile, and several
@pytest.mark.parametrize("what", ["scores", "weights"])
def test_attend(dev, kind, half, dim, n, group, what):
    print(f"pieces attend {kind} {what} dim={dim} n={n} group={group}", flush=True)
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]
    B, heavy = 16, [9, 170]
    pages = B * -(-n // 64)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(B, -1).to(dev)
    k, v = torch.zeros(B, n, 1, dim), torch.randn(B, n, 1, dim)
    if what == "scores":
        q2, pair = P.close_cached_scores(B * group, 3, dt)
        k[..., [3, dim - 2]] = -4.0
        k[:, heavy, 0, 3], k[:, heavy, 0, dim - 2] = pair[:, 0], pair[:, 1]
    else:
        q1, pair = P.near_scores(B * group, 5, dt), torch.tensor([[0.0, 0.0], [4.0, 0.0]])
        # by the other channel all others are 200 below
        q2 = torch.cat((q1.float(), torch.full((B * group, 1), 400.0)), 1).to(dt)
        k[..., dim - 2] = -4.0
        k[:, heavy, 0, 3], k[:, heavy, 0, dim - 2] = pair[:, 0], 0.0
    v[:, heavy[0]], v[:, heavy[1]] = 0.0, 1.0
    c = kv4.Cache4.zeros(pages, 1, 64, dim, dev)
    lens = torch.full((B,), n, dtype=torch.int32, device=dev)
    cu = (torch.arange(B + 1) * n).to(torch.int32).to(dev)
    c.append(k.reshape(-1, 1, dim).to(dev), v.reshape(-1, 1, dim).to(dev), table, lens, cu)
    q = torch.zeros(B * group, dim, dtype=dt)
    q[:, [3, dim - 2]] = q2
    sums = torch.zeros(B, 1, n, device=dev)
    got = c.attend(q.reshape(B, 1, group, dim).to(dev), table, lens, max_len=n, weights=sums, scale=0.125).cpu().double()
    want = P.exact(q2.float(), pair, torch.ones(dim), 0.125)
    tol = P.score_bound(q2.float(), pair, torch.ones(dim), 0.125, 4 * 2.0 ** -24) if what == "scores" else 0.0
    bound = tol + (P.PART_BOUND[kind] + half) * want
    assert bool(((got.reshape(-1, dim) - want).abs() <= bound).all())
    # what the two received, summed over the group's rows in f32
    p1 = want[:, 0].reshape(B, group).sum(1)
    tol = (tol[:, 0].reshape(B, group).sum(1) if what == "scores" else 0.0) + (33 + group) * 2.0 ** -24 * group
    assert bool(((sums[:, 0, heavy[1]].cpu().double() - p1).abs() <= tol).all())
    assert bool(((sums[:, 0, heavy[0]].cpu().double() - (group - p1)).abs() <= tol).all())

"""The bounds of test_gpu_pieces.py on the CPU: the scheme as it is keeps within them, and without any one of its
pieces' products it does not."""
import pytest
import torch

from oracle import pieces as P


def prompt_scores(drop=()):
    q, k = P.close_scores(300, 1)
    v1 = torch.ones(1)
    off = (P.prompt_f32(q, k, v1, 0.125, drop) - P.exact(q, k, v1, 0.125)).abs()
    return bool((off <= P.score_bound(q, k, v1, 0.125, 20 * 2.0 ** -24) + P.WEIGHT_BOUND * P.exact(q, k, v1, 0.125)).all())


def prompt_weights(drop=()):
    fine = True
    for seed in range(16):
        d = torch.round(P.rough((2,), 0.0, 2.0, seed).double() * 16).float() / 16
        v1 = P.rough((64,), 1.0, 2.0, seed + 50)
        q, k = torch.ones(1, 1), 8 * d[:, None]
        want = P.exact(q, k, v1, 0.125)
        fine &= bool(((P.prompt_f32(q, k, v1, 0.125, drop) - want).abs() <= P.WEIGHT_BOUND * want).all())
    return fine


def test_prompt_scheme():
    assert prompt_scores() and prompt_weights()
    for i, j in P.PROMPT_SCORES:
        assert not prompt_scores((f"s{i}{j}",)), (i, j)
    for i, j in P.PROMPT_VALUES:
        assert not prompt_weights((f"p{i}{j}",)), (i, j)


@pytest.mark.parametrize("kind,half", [("f32", 0.0), ("f16", 2.0 ** -11), ("bf16", 2.0 ** -8)])
def test_attend_scheme(kind, half):
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]

    def scores(drop=()):
        q, k = P.close_cached_scores(300, 3, dt)
        want = P.exact(q.float(), k, torch.ones(1), 0.125)
        got = P.attend(kind, q.float(), k, torch.ones(1), 0.125, drop).to(dt).double()
        tol = P.score_bound(q.float(), k, torch.ones(1), 0.125, 4 * 2.0 ** -24)
        return bool(((got - want).abs() <= tol + (P.PART_BOUND[kind] + half) * want).all())

    def weights(drop=()):
        q = P.near_scores(600, 5, dt)
        k = torch.tensor([[0.0], [4.0]])
        want = P.exact(q.float(), k, torch.ones(1), 0.125)
        got = P.attend(kind, q.float(), k, torch.ones(1), 0.125, drop).to(dt).double()
        return bool(((got - want).abs() <= (P.PART_BOUND[kind] + half) * want).all())

    assert scores() and weights()
    for i in range(1, P.Q_PIECES[kind]):
        assert not scores((f"q{i}",)), i
    for i in range(P.P_PIECES[kind]):
        assert not weights((f"p0{i}",)), i

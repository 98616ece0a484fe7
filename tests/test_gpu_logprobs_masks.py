"""Rows masked with finite values, alone and beside -inf, in the operators on next-token distributions: against the
fp64 formulas and with the tolerances of tests/test_gpu_logprobs.py."""
import pytest
import torch

from tests.test_gpu_logprobs import DT, L, NINF, check_logprobs, strided, targets_for  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ alternatives
def mixed_masks(rows, vocab, dtype, ordinary, low, lead, seed=0):
    """Rows of `ordinary` logits and `low` ones of the type's lowest value at random places from `lead` on, the others
    -inf; 1,100 elements of 7, above nearly all of them, lie between the rows and behind the last one."""
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows + vocab)
    x, _ = strided(rows, vocab, dtype, 1100)
    place = torch.rand(rows, vocab - lead, device="cuda", generator=g).argsort(1) + lead
    v = torch.full((rows, vocab), NINF, device="cuda")
    v.scatter_(1, place[:, ordinary:ordinary + low], torch.finfo(DT[dtype]).min)
    v.scatter_(1, place[:, :ordinary], torch.randn(rows, ordinary, device="cuda", generator=g) * 3)
    x.copy_(v)
    return x


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(3, 300), (1300, 400), (2400, 1000), (5, 4000), (1300, 4001), (300, 9000), (2, 140000)])
@pytest.mark.parametrize("ordinary,low,lead,k", [(10, 60, 0, 30), (20, 40, 0, 30), (1, 100, 0, 96), (40, 130, 60, 64),
                                                 (0, 200, 0, 25), (24, 24, 200, 48), (120, 1, 0, 128)])
def test_alternatives_beside_lowest_values(L, rows, vocab, ordinary, low, lead, k, dtype):
    """Fewer ordinary logits than alternatives: the others are masks of the lowest value, then -inf, by their index; none
    comes from outside the row."""
    check_logprobs(L, mixed_masks(rows, vocab, dtype, ordinary, low, lead), dtype, 1.0, k, targets_for(rows, vocab))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [3, 1300])
def test_alternatives_behind_a_long_masked_run(L, rows, dtype):
    """Masks of the lowest value in more vectors than are listed at once, behind a run of -inf."""
    for vocab, low, lead in [(3700, 2000, 1700), (8000, 6000, 1600), (30000, 20000, 9000)]:
        check_logprobs(L, mixed_masks(rows, vocab, dtype, 7, low, lead), dtype, 1.0, 40, targets_for(rows, vocab))

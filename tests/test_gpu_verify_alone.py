"""GPU checks that a sequence's verification does not depend on what stands beside it in the batch: not in the last bit
of a sum, which decides where a random number meets a border."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

from test_gpu_verify import check, problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def row_that_sums_to(target: Fraction, v: int, seed: int) -> np.ndarray:
    """v probabilities of sizes from 2^-50 to 2^-15 in no order (FP64 rounds nearly every addition of them), the last
    ones what is missing of ``target``, 24 bits each; 100 and 200 are left out."""
    g = np.random.default_rng(seed)
    row = np.exp2(g.uniform(-50.0, -15.0, v)).astype(np.float32)
    row[[100, 200, -5, -4, -3, -2, -1]] = 0.0
    left = target - sum(Fraction(float(x)) for x in row)
    for i in range(5):
        assert left >= 0
        x = np.float32(float(left))
        if Fraction(float(x)) > left:
            x = np.nextafter(x, np.float32(0))
        row[v - 5 + i] = x
        left -= Fraction(float(x))
    assert abs(left) < Fraction(1, 1 << 80)
    return row


@pytest.mark.parametrize("sampled", [True, False])
def test_a_sequence_alone_and_in_a_batch(cp, sampled):
    """A candidate that is taken where u s < p with u = p = 1/2 and s within the last bits of 1: the sum of a rejection
    decides, and beside it the border u_0 s."""
    v, kinds, batch = 32000, 12, 600
    half, tiny = Fraction(1, 2), Fraction(1, 1 << 55)
    target = torch.zeros((kinds, 3, v))
    for i in range(kinds):
        row = row_that_sums_to(half - (i % 6) * tiny, v, i)
        row[100] = 0.5                    # the second candidate's
        row[200] = 0.0 if sampled else 2.0 ** -20  # the first one's
        target[i, 0] = torch.from_numpy(row)
    target[:, 1:, 7] = 1.0
    draft = torch.zeros((kinds, 3, v))
    draft[:, 0, 200], draft[:, 0, 100] = 2.0 ** -60, 1.0  # the first candidate's rejection takes nothing but itself
    if sampled:  # r = p - q: what is left sums to the same, the second candidate's 1/2 among it
        target[:, 0, 100] = 1.5
    tokens = torch.tensor([0, 200, 100]).repeat(kinds, 1)
    parents = torch.tensor([-1, 0, 0])
    u = torch.tensor([0.5, 0.999, 0.5]).repeat(kinds, 1)

    def call(rows):
        return [x.cpu() for x in cp.cuda_verify_drafted(
            target[rows].cuda(), tokens[rows].cuda(), u[rows].cuda(), parents=parents.cuda(),
            draft_probs=draft[rows].cuda() if sampled else None)]

    alone = [torch.cat(x) for x in zip(*(call([i]) for i in range(kinds)))]
    assert len(set(alone[1].tolist())) > 1  # both sides of the border
    for n in (kinds, 3 * kinds, batch):
        rows = torch.arange(n) % kinds
        assert all(torch.equal(x, y[rows]) for x, y in zip(call(rows), alone))


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("v", [4097, 5000, 7680, 8191, 8193, 9000, 16385, 70001])
def test_rows_of_fewer_segments_than_runs_and_a_few_more(cp, sampled, v):
    """Runs that hold no segment, one, or one more than others: the definition's paths and tokens."""
    target, draft, tokens, parents, u = problem(6, 7, v, True, v, near=1.5)
    check(cp, target, tokens, u, draft if sampled else None, parents)
    one = torch.zeros((6, 7, v))  # all of a row in one element: of the first, a middle or the last segment
    for i, y in enumerate((0, 511, 512, v // 2, v - 512, v - 1)):
        one[i, :, y] = 0.75
    path, counts, nexts = check(cp, one, tokens, u, draft if sampled else None, parents)
    assert sorted(set(nexts.tolist())) == sorted({0, 511, 512, v // 2, v - 512, v - 1})

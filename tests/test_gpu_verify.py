"""GPU checks of the verification of drafted tokens: whole numbers, equal to the definition's in 64 bits."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def problem(b, t, v, tree, seed, spread=1.0, near=0.5):
    """Target and draft rows that resemble each other, tokens drawn from the parent's draft row."""
    g = torch.Generator().manual_seed(seed)
    logits = spread * torch.randn((b, t, v), generator=g)
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits + near * torch.randn((b, t, v), generator=g), -1)
    parents = (torch.rand((b, t), generator=g) * torch.arange(t)).long() if tree else (torch.arange(t) - 1).repeat(b, 1)
    parents[:, 0] = -1
    tokens = torch.zeros((b, t), dtype=torch.int64)
    for i in range(1, t):
        tokens[:, i] = torch.multinomial(draft[torch.arange(b), parents[:, i]], 1, generator=g)[:, 0]
    return target, draft, tokens, parents, torch.rand((b, t), generator=g)


def check(cp, target, tokens, uniforms, draft=None, parents=None, counts=None):
    def dev(x):
        return None if x is None else x.cuda()

    got = cp.cuda_verify_drafted(dev(target), dev(tokens), dev(uniforms), draft_probs=dev(draft), parents=dev(parents),
                                 counts=dev(counts))
    want = ref.verify(target, tokens, uniforms, draft, parents, counts)
    for x, y in zip(got, want):
        assert x.dtype == torch.int64 and x.tolist() == y
    return [x.cpu() for x in got]


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("b,t,v,tree", [
    (1, 1, 1, False), (1, 2, 2, False), (2, 1, 5, False), (3, 5, 7, True), (17, 8, 129, True), (4, 6, 511, False),
    (64, 4, 1000, False), (200, 6, 513, True), (2, 64, 4096, True), (5, 9, 32003, True), (1, 5, 50000, False),
    (2, 3, 131075, True), (3, 1024, 64, True),
])
def test_verify(cp, b, t, v, tree, sampled):
    for seed, near in ((1, 0.4), (2, 2.0)):
        target, draft, tokens, parents, u = problem(b, t, v, tree, seed, near=near)
        path, counts, _ = check(cp, target, tokens, u, draft if sampled else None, parents if tree else None)
        if sampled and b >= 17 and t > 1:  # the cases are not all of one kind
            assert len(set(counts.tolist())) > 1


def test_likeliest_candidates_of_peaked_rows(cp):
    """Trees of a row's likeliest tokens, best first: paths of many lengths, rejected siblings before accepted ones."""
    b, t, v = 50, 14, 3001
    target, draft, tokens, parents, u = problem(b, t, v, True, 23, spread=4.0)
    for i in range(1, t):
        rank = (parents[:, :i] == parents[:, i:i + 1]).sum(1)
        tokens[:, i] = draft[torch.arange(b), parents[:, i]].topk(t).indices[torch.arange(b), rank]
    path, counts, _ = check(cp, target, tokens, u, None, parents)
    assert len(set(counts.tolist())) > 3
    first = path[counts > 1, 1]
    assert (first > 1).any()


@pytest.mark.parametrize("sampled", [True, False])
def test_counts_shared_parents_and_views(cp, sampled):
    b, t, v = 7, 6, 1000
    target, draft, tokens, parents, u = problem(b, t, v, True, 5)
    counts = torch.tensor([6, 0, 1, 3, -4, 99, 2])
    check(cp, target, tokens, u, draft if sampled else None, parents, counts)
    parents = parents[0].contiguous()
    want = check(cp, target, tokens, u, draft if sampled else None, parents)
    for pad in (1, 2, 4):  # rows of a wider vocabulary, aligned to 4, 8 and 16 bytes
        p, q = (torch.nn.functional.pad(x, (pad, pad)).cuda()[..., pad:pad + v] for x in (target, draft))
        got = cp.cuda_verify_drafted(p, tokens.cuda(), u.cuda(), draft_probs=q if sampled else None,
                                     parents=parents.cuda())
        assert all(torch.equal(x.cpu(), y) for x, y in zip(got, want))
    p = target.cuda().transpose(0, 1).contiguous().transpose(0, 1)  # nodes outermost
    got = cp.cuda_verify_drafted(p, tokens.cuda(), u.cuda(), draft_probs=draft.cuda() if sampled else None,
                                 parents=parents.cuda())
    assert all(torch.equal(x.cpu(), y) for x, y in zip(got, want))


@pytest.mark.parametrize("sampled", [True, False])
def test_random_numbers_at_their_ends(cp, sampled):
    for value in (0.0, 1.0, 2.0, -1.0, float("nan"), float("inf")):
        target, draft, tokens, parents, u = problem(3, 5, 300, True, 9)
        u[:, 0] = value
        check(cp, target, tokens, u, draft if sampled else None, parents)
        u[:] = value
        check(cp, target, tokens, u, draft if sampled else None, parents)


@pytest.mark.parametrize("sampled", [True, False])
def test_rows_that_are_no_distributions(cp, sampled):
    """Zeros, one-hot rows, infinities, NaN, negative and subnormal elements, rows of nothing, and drafts of nothing."""
    b, t, v = 9, 5, 700
    target, draft, tokens, parents, u = problem(b, t, v, True, 13)
    target[0] = 0.0
    target[1] = torch.nn.functional.one_hot(tokens[1], v).float()
    target[2, :, ::2], target[2, :, 1::3] = float("inf"), float("nan")
    target[3] = -target[3]
    target[4] *= 1e-40
    draft[5] = 0.0
    draft[6, :, ::2], draft[6, :, 1::3] = float("nan"), float("-inf")
    draft[7] = target[7] * 2  # nothing is left where a child is rejected
    u[7, 1:] = 0.9
    target[8] = draft[8]
    check(cp, target, tokens, u, draft if sampled else None, parents)


@pytest.mark.parametrize("sampled", [True, False])
def test_candidates_that_repeat_or_are_none(cp, sampled):
    """Siblings of one token, tokens outside the vocabulary, parents that are none or come later."""
    b, t, v = 6, 8, 50
    target, draft, tokens, parents, u = problem(b, t, v, True, 17, spread=0.3, near=1.5)
    parents[:3] = 0
    tokens[0, 1:] = tokens[0, 1]
    tokens[1, 2], tokens[1, 4], tokens[1, 5] = -1, v, 1 << 40
    tokens[2, 1:5] = tokens[2, 5]
    parents[3, 2], parents[3, 4], parents[4, 3] = 7, -1, 1 << 40
    parents[5, 1:] = torch.arange(7) + 1  # each its own parent
    u[:3] = 0.95
    check(cp, target, tokens, u, draft if sampled else None, parents)


def test_siblings_that_hold_all_of_a_row(cp):
    """Given siblings of probabilities 2^-1, 2^-2, ...: what the last ones hold decides, however little it is.  In exact
    arithmetic s is below twice a sibling's own p, which the one half of a row does not round away."""
    for n in (2, 31, 33, 64, 65, 120):
        v = 700
        target = torch.zeros((3, n + 1, v))
        target[:, 0, :n] = 2.0 ** -torch.arange(1.0, n + 1)
        target[:, 1:, 9] = 1.0
        tokens = torch.arange(-1, n).repeat(3, 1)
        tokens[:, 0] = 0
        parents = torch.zeros(n + 1, dtype=torch.int64)
        u = torch.full((3, n + 1), 0.75)
        u[:, 0] = 0.7
        u[1, n] = 2.0  # none is left: the row stands again
        u[2, 1:] = 0.75 * (torch.arange(n) < n // 2)
        path, counts, nexts = check(cp, target, tokens, u, None, parents)
        assert counts.tolist() == [2, 1, 2] and path[:, 1].tolist() == [n, -1, n // 2 + 1]
        assert nexts.tolist() == [9, 1, 9]


@pytest.mark.parametrize("sampled", [True, False])
def test_tokens_follow_the_target(cp, sampled):
    """The first new token of 40,000 trees: within 5 standard deviations of the target's row everywhere."""
    n, v = 40000, 6
    g = torch.Generator().manual_seed(3)
    p = torch.tensor([0.05, 0.1, 0.15, 0.2, 0.22, 0.28])
    q = p.flip(0)
    tokens = torch.multinomial(q, 4 * n, replacement=True, generator=g).view(n, 4)
    if not sampled:
        tokens[:] = torch.tensor([0, 5, 4, 0])
    parents = torch.tensor([-1, 0, 0, 0])
    u = torch.rand((n, 4), generator=g)
    path, count, nexts = cp.cuda_verify_drafted(p.expand(n, 4, v).cuda(), tokens.cuda(), u.cuda(),
                                                draft_probs=q.expand(n, 4, v).cuda() if sampled else None,
                                                parents=parents.cuda())
    child = torch.gather(tokens, 1, path[:, 1:2].cpu().clamp(min=0))[:, 0]
    first = torch.where(count.cpu() > 1, child, nexts.cpu())
    share = torch.bincount(first, minlength=v) / n
    assert ((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()
    assert set(count.tolist()) == {1, 2}


def test_repeated_and_captured_calls_agree(cp):
    target, draft, tokens, parents, u = (x.cuda() for x in problem(33, 7, 20001, True, 21))
    first = cp.cuda_verify_drafted(target, tokens, u, draft_probs=draft, parents=parents)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(20):
            again = cp.cuda_verify_drafted(target, tokens, u, draft_probs=draft, parents=parents)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cp.cuda_verify_drafted(target, tokens, u, draft_probs=draft, parents=parents)
    u.copy_(1.0 - u)
    graph.replay()
    want = ref.verify(target.cpu(), tokens.cpu(), u.cpu(), draft.cpu(), parents.cpu())
    assert all(x.tolist() == y for x, y in zip(out, want))


def test_offsets_past_32_bits_and_the_longest_chain(cp):
    """More than 2^31 probabilities: one-hot rows lead down a chain of 1,024 nodes."""
    b, t, v = 2, 1024, (1 << 20) + 4
    target = torch.zeros((b, t, v), device="cuda")
    tokens = torch.randint(0, v, (b, t), generator=torch.Generator().manual_seed(1)).cuda()
    node = torch.arange(t - 1).cuda()
    for i in range(b):
        target[i, node, tokens[i, 1:]] = 1.0
        target[i, t - 1, v - 1 - i] = 0.25
    u = torch.full((b, t), 0.9).cuda()
    path, counts, nexts = cp.cuda_verify_drafted(target, tokens, u)
    assert counts.tolist() == [t, t] and nexts.tolist() == [v - 1, v - 2]
    assert torch.equal(path, torch.arange(t).cuda().expand(b, t))
    tokens[1, 700] = (tokens[1, 700] + 1) % v  # a candidate that has no probability: the row's own token is drawn
    path, counts, nexts = cp.cuda_verify_drafted(target, tokens, u)
    assert counts.tolist() == [t, 700] and nexts[1] == (tokens[1, 700] - 1) % v and (path[1, 700:] == -1).all()


def test_refusals(cp):
    target, draft, tokens, parents, u = (x.cuda() for x in problem(2, 3, 10, True, 1))

    def call(target=target, tokens=tokens, u=u, **kw):
        return cp.cuda_verify_drafted(target, tokens, u, **kw)

    for kw, text in ((dict(target=target.half()), "dtype"), (dict(target=target[0]), "rank 3"),
                     (dict(target=target.transpose(1, 2)), "contiguous in its last"), (dict(tokens=tokens.int()), "dtype"),
                     (dict(tokens=tokens[:, :2].contiguous()), "tokens must have shape"), (dict(u=u.double()), "dtype"),
                     (dict(u=u[:1]), "uniforms must have shape"), (dict(draft_probs=draft[:1]), "same shape"),
                     (dict(parents=parents[:1]), "parents must have shape"), (dict(parents=parents.cpu()), "CUDA tensor"),
                     (dict(counts=tokens[:, 0]), "counts must be contiguous")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    big = torch.zeros((1, 1025, 2)).cuda()
    with pytest.raises(RuntimeError, match="at most 1024 nodes"):
        cp.cuda_verify_drafted(big, torch.zeros((1, 1025), dtype=torch.int64).cuda(), big[..., 0].contiguous())

"""Verification of drafted tokens against the definition in 64 bits: whole numbers, so equal.

The kernel's sums are fp64 in another order than the oracle's: they differ by at most 2^-53 times the number of additions
(about 2^-40 of the whole at 151936 columns), so a drawn column could differ only where a border lies that near u C_V; with
uniforms of 24 bits that is a chance of about 10^-7 for a row, and the seeds are fixed."""

import pytest
import torch

from ckb200 import softmax, topk, verify
from helpers import guarded_empty
from oracle import serving

pytestmark = pytest.mark.gpu


def problem(seed, b, k, v, dtype, probs=True, noise=1.0):
    g = torch.Generator().manual_seed(seed)
    logits = 3 * torch.randn(b, k + 1, v, generator=g)
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :k] + noise * torch.randn(b, k, v, generator=g), -1)
    tokens = torch.multinomial(draft.flatten(0, 1), 1, generator=g).view(b, k) if k else torch.empty(b, 0, dtype=torch.int64)
    return target, tokens, torch.rand(b, k + 1, generator=g), draft.to(dtype) if probs else None


def check(target, tokens, uniforms, draft=None, counts=None):
    want = serving.verify(target, tokens, uniforms, draft, counts)
    args = [None if t is None else t.cuda() for t in (target, tokens, uniforms, draft, counts)]
    got = verify.verify_drafts(*args)
    assert torch.equal(got[1].cpu(), want[1]), "accepted"
    assert torch.equal(got[0].cpu(), want[0]), "tokens"
    return got


CASES = [(1, 4, 151936, torch.float32), (3, 5, 128256, torch.bfloat16), (7, 3, 50001, torch.float32),
         (5, 2, 50001, torch.bfloat16), (40, 6, 1000, torch.float32), (9, 0, 4096, torch.float32),
         (2, 40, 513, torch.bfloat16), (4, 3, 1, torch.float32), (6, 2, 31, torch.float32), (300, 1, 4100, torch.float32),
         (150, 2, 2048, torch.bfloat16)]


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("b,k,v,dtype", CASES)
def test_matches_the_definition(b, k, v, dtype, probs):
    target, tokens, uniforms, draft = problem(b * 31 + v, b, k, v, dtype, probs)
    check(target, tokens, uniforms, draft)
    counts = torch.arange(b) % (k + 2)  # 0 .. k + 1: the last is one too many
    check(target, tokens, uniforms, draft, counts)


def test_views_with_strides_and_guarded_outputs():
    target, tokens, uniforms, draft = problem(3, 4, 3, 1000, torch.float32)
    wide_t, wide_d = torch.rand(4, 5, 1030).cuda(), torch.rand(4, 7, 1003).cuda()  # a padded vocabulary; odd rows
    wide_t[:, 1:, :1000], wide_d[:, 2:5, 3:] = target.cuda(), draft.cuda()
    out, check_out = guarded_empty((4, 4), torch.int64)
    acc, check_acc = guarded_empty((4,), torch.int64)
    verify.verify_drafts(wide_t[:, 1:, :1000], tokens.cuda(), uniforms.cuda(), wide_d[:, 2:5, 3:], out=(out, acc))
    want = serving.verify(target, tokens, uniforms, draft)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(acc.cpu(), want[1])
    check_out()
    check_acc()
    turned = target.cuda().transpose(0, 2).contiguous().transpose(0, 2)  # the last dim is not contiguous: copied
    got = verify.verify_drafts(turned, tokens.cuda(), uniforms.cuda(), draft.cuda())
    assert torch.equal(got[0].cpu(), want[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_borders_zeros_and_odd_values(dtype):
    """Rows of few values, whose sums are exact: the border itself (u C_V equal to a running sum) goes to the next column
    with weight; columns of zeros are never drawn; refused rows without weight left draw from the target's own."""
    v = 40
    target = torch.zeros(8, 2, v, dtype=dtype)
    target[:, :, 4], target[:, :, 9], target[:, :, 39] = 0.25, 0.25, 0.5
    draft = target[:, :1].clone()
    tokens = torch.full((8, 1), 9)
    u = torch.tensor([[0.0, 0.0], [0.0, 0.25], [0.0, 0.4999], [0.0, 0.5], [0.0, 0.99999994], [1.0, 0.3], [0.0, 0.25], [0.0, 0.0]])
    draft[5] = target[5, :1]  # u = 1 refuses where p = q: nothing is left, the target's row is drawn from
    tokens[6] = 7  # the target gives it nothing
    tokens[7] = -1  # no token at all
    got = check(target, tokens, u, draft)[0].cpu()
    assert got[:, 1].tolist()[:5] == [4, 9, 9, 39, 39] and got[5].tolist() == [9, -1] and got[6, 0] == 9 and got[7, 0] == 4
    check(target, tokens, u)
    target[0] = 0  # no mass anywhere
    target[1, 1] = float("nan")
    target[2, 1, 4] = -0.25
    target[3, 0, 3] = float("nan")
    assert check(target, tokens, u, draft)[0][0].tolist() == [-1, -1]
    check(target, torch.full((8, 1), v), u, draft)  # outside the vocabulary
    huge = target.clone()
    huge[4, 1, 5] = float("inf")  # what it gives is undefined, but it stays inside the row
    got = verify.verify_drafts(huge.cuda(), tokens.cuda(), u.cuda(), draft.cuda())[0].cpu()
    assert ((got >= -1) & (got < v)).all()


def test_one_token_has_all_the_mass_at_either_end():
    for v in (5, 4096, 151936):
        for at in (0, v - 1):
            target = torch.zeros(2, 2, v)
            target[:, :, at] = 1.0
            u = torch.tensor([[0.5, 0.0], [0.5, 0.99999994]])
            got = check(target, torch.full((2, 1), (at + 1) % v), u)
            assert got[0][:, 0].tolist() == [at, at]


def test_drawn_tokens_follow_the_target():
    """One drafted token over 8 columns, 2^16 sequences: the first token of each is distributed as the target. A count's
    standard deviation is at most sqrt(2^16 / 4) = 128; six of them are allowed."""
    g = torch.Generator().manual_seed(11)
    p, q = torch.softmax(torch.randn(8, generator=g), 0), torch.softmax(torch.randn(8, generator=g), 0)
    n = 1 << 16
    tokens = torch.multinomial(q, n, replacement=True, generator=g).view(n, 1)
    got, _ = verify.verify_drafts(p.expand(n, 2, 8).cuda(), tokens.cuda(), torch.rand(n, 2, generator=g).cuda(),
                                  q.expand(n, 1, 8).cuda())
    counts = torch.bincount(got[:, 0].cpu(), minlength=8)
    assert ((counts - n * p).abs() < 6 * 128).all(), counts


def test_after_softmax_two_calls_streams_and_graphs():
    g = torch.Generator().manual_seed(12)
    logits = (3 * torch.randn(6, 4, 32000, generator=g)).cuda()
    draft_logits = logits[:, :3] + torch.randn(6, 3, 32000, generator=g).cuda()
    u = torch.rand(6, 4, generator=g).cuda()
    drafted = torch.rand(18, generator=g).cuda()
    _, _, samples = topk.topk_softmax(draft_logits.flatten(0, 1), k=50, uniforms=drafted)
    tokens = samples.view(6, 3)

    def step():
        return verify.verify_drafts(softmax.softmax(logits), tokens, u, softmax.softmax(draft_logits))

    want = serving.verify(softmax.softmax(logits).cpu(), tokens.cpu(), u.cpu(), softmax.softmax(draft_logits).cpu())
    first, second = step(), step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fourth = step()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for got in (first, second, third, fourth):
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [40, 41, 4096])  # vectors, single elements, a step for each warp
def test_draft_probabilities_that_are_nan_or_negative_count_as_zero(v, dtype):
    """At the drafted token (which is then accepted wherever the target gives it anything) and beside it (where the column
    keeps the target's own weight, no more and no less). Sums of eighths are exact."""
    target = torch.zeros(8, 2, v, dtype=dtype)
    target[:, :, 4], target[:, :, 9], target[:, :, v - 1] = 0.25, 0.25, 0.5
    draft = torch.zeros(8, 1, v, dtype=dtype)
    draft[:, 0, 4], draft[:, 0, 9], draft[:, 0, v - 1] = 0.125, 0.75, 0.125
    bad = torch.tensor([float("nan"), -0.25, float("nan"), -1.0, float("nan"), -0.5, float("-inf"), float("nan")], dtype=dtype)
    tokens = torch.full((8, 1), 9)
    u = torch.tensor([[0.99, 0.3], [0.99, 0.3], [0.5, 0.3], [0.5, 0.3], [0.5, 0.45], [0.5, 0.45], [0.5, 0.45], [0.5, 0.9]])
    draft[:2, 0, 9] = bad[:2]  # at the drafted token
    draft[2:7, 0, 4] = bad[2:7]  # beside it: w = (0.25, 0, 0.375) of 0.625 in all, so 0.3 draws column 4 and 0.45 the last
    draft[7, 0, :4] = bad[7]  # where the target has nothing
    target[6, 0, 2] = -1.0  # below zero in both
    draft[6, 0, 2] = -2.0
    got = check(target, tokens, u, draft)
    assert got[1].tolist() == [1, 1, 0, 0, 0, 0, 0, 0]
    assert got[0][:, 0].tolist() == [9, 9, 4, 4, v - 1, v - 1, v - 1, v - 1]
    p, t, u, q = problem(21, 6, 3, v, dtype)
    q[:, :, ::3] = float("nan")
    q[:, :, 1::3] *= -1.0
    check(p, t, u, q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [40, 41, 4096])
def test_an_infinite_draft_probability_takes_its_column_alone(v, dtype):
    """max(p - inf, 0) is 0, and the other columns keep theirs: w = (0, 0.125, 0.375) of 0.5."""
    target, draft = torch.zeros(4, 2, v, dtype=dtype), torch.zeros(4, 1, v, dtype=dtype)
    target[:, :, 4], target[:, :, 9], target[:, :, v - 1] = 0.25, 0.25, 0.5
    draft[:, 0, 4], draft[:, 0, 9], draft[:, 0, v - 1] = float("inf"), 0.125, 0.125
    u = torch.tensor([[0.5, 0.0], [0.5, 0.2], [0.5, 0.3], [0.5, 0.9]])
    got = check(target, torch.full((4, 1), 4), u, draft)
    assert got[0][:, 0].tolist() == [9, 9, v - 1, v - 1]

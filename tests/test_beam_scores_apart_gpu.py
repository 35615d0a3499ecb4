"""beam_select where scores are so large that the scores of different logits are one number in float64: lower beams come first, within a beam the larger logit, then the lower token."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def expected(logits, scores, n, finished=None, pad=0):
    """by sorting with those rules, one beam and token after another"""
    B, K, V = logits.shape
    z = logits.double().cpu()
    top = z.amax(-1, keepdim=True)
    total = scores.double().cpu()[..., None] + ((z - top) - torch.log(torch.exp(z - top).sum(-1, keepdim=True)))
    total = torch.where(z == float("-inf"), torch.full((), float("-inf")).double(), total)
    if finished is not None:
        only = torch.full((B, K, V), float("-inf")).double()
        only[..., pad] = scores.double().cpu()
        total = torch.where(finished.cpu()[..., None], only, total)
    found = []
    for b in range(B):
        # (a stable sort by each key in turn, the last one first)
        by_logit = torch.sort(z[b], dim=-1, descending=True, stable=True)[1]
        flat = torch.where(total[b].gather(-1, by_logit) > float("-inf"), by_logit, -1)
        order = torch.cat([torch.cat((flat[k][flat[k] >= 0], (total[b, k] == float("-inf")).nonzero()[:, 0])) + k * V for k in range(K)])
        best = torch.sort(total[b].flatten()[order], descending=True, stable=True)[1][:n]
        found.append(order[best])
    at = torch.stack(found)
    return total.flatten(1).gather(1, at), at // V, at % V


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V,n", [(50, 12), (3000, 12), (9000, 40), (40000, 128)])
@pytest.mark.parametrize("low", [float(torch.finfo(torch.float32).min), -1e30, 1e25, float("inf")])
def test_scores_next_to_which_logits_are_nothing(low, V, n, dtype):
    """beams that are masked by the type's lowest value, say, when the others have too few tokens"""
    import t2fw_amd as t2
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(3, 4, V, generator=g) * 3).to(dtype).cuda()
    logits[:, 0] = float("-inf")
    logits[:, 0, 5:8] = torch.tensor([1.0, 3.0, 2.0], device="cuda").to(dtype)
    logits[1, 2, V // 2:] = float("-inf")
    logits[2, 1, 4:] = float("-inf")
    scores = torch.full((3, 4), low, device="cuda")
    scores[:, 0] = -1.0
    want = expected(logits, scores, n)
    got = t2.beam_select(logits, scores, count=n)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    finite = want[0].abs() < 1e3
    assert torch.equal(got[0].cpu()[~finite], want[0].float()[~finite])
    assert bool(((got[0].cpu() - want[0])[finite].abs() <= 2.0 ** -19 + 2.0 ** -20).all())


def test_ended_beams_of_such_scores():
    import t2fw_amd as t2
    logits = torch.randn(1, 4, 500, generator=torch.Generator().manual_seed(0)).cuda()
    scores = torch.full((1, 4), -3e38, device="cuda")
    finished = torch.tensor([[False, True, False, True]], device="cuda")
    for n in (3, 20, 128):
        want = expected(logits, scores, n, finished, 7)
        got = t2.beam_select(logits, scores, count=n, finished=finished, pad=7)
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])


def test_one_pair_of_logits_that_float64_does_not_tell_apart():
    import t2fw_amd as t2
    logits = torch.full((1, 2, 9000), -40.0, device="cuda")
    logits[0, :, 10], logits[0, :, 3], logits[0, :, 8995] = 1e-30, 0.0, 2e-30
    scores = torch.tensor([[-12.0, -12.0]], device="cuda")
    s, k, v = t2.beam_select(logits, scores, count=6)
    assert k.tolist() == [[0, 0, 0, 1, 1, 1]] and v.tolist() == [[8995, 10, 3] * 2] and bool((s == s[0, 0]).all())

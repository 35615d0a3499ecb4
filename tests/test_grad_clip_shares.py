"""clip_grad_norm on as many elements as a model has: a workgroup's share is several pieces of 2048 elements, of several arrays, and its loop
takes eight vectors of each thread at a time.  Every element is compared; the bounds are those of test_grad_clip.py."""
import pytest
import torch

from tests.test_gated_scan import STORE, TINY

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def make(sizes, dtypes, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, generator=g, device="cuda").to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def sizes_of(count, most, seed):
    """odd sizes from a few elements to `most`, most of them large"""
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(count, generator=g)
    return [max(1, int(most * (v if i % 5 else v ** 8))) | 1 for i, v in enumerate(u.tolist())]


def check(got, before, by):
    for g, b in zip(got, before):
        want = b.double() * by
        off = (g.double() - want).abs() - ((2.0 ** -22 + STORE[g.dtype]) * want.abs() + TINY[g.dtype])
        assert bool((off <= 0).all()), float(off.max())


def norm64(ts):
    return float(torch.stack([t.double().square().sum() for t in ts]).sum().sqrt())


# elements, and the elements of a share: one table and two, all types mixed and one
@pytest.mark.parametrize("count,most,dtypes", [(40, 700000, DTYPES), (40, 1800000, DTYPES), (24, 3000000, [torch.bfloat16]), (200, 500000, DTYPES[:2]),
                                               (7, 6000000, [torch.float32])], ids=["40", "40 large", "24 of bf16", "200", "7 of float32"])
def test_shares_of_several_pieces_and_arrays(count, most, dtypes):
    import t2fw_amd as t2
    grads = make(sizes_of(count, most, seed=count), dtypes, seed=most)
    pieces = sum(-(-g.numel() // 2048) for g in grads)
    assert pieces > 2 * 1024                                 # (a launch has at most 1024 workgroups)
    before, norm = [g.clone() for g in grads], norm64(grads)
    for to in (torch.float32, torch.bfloat16):
        out = [torch.full(g.shape, float("nan"), dtype=to, device="cuda") for g in grads]
        assert abs(float(t2.clip_grad_norm(grads, 0.75, out=out)) - norm) <= 2.0 ** -23 * norm
        check(out, before, 0.75 / (norm + 1e-6))
        assert all(torch.equal(g, b) for g, b in zip(grads, before))
    # larger than any gradient's rounding, so that none becomes zero
    assert abs(float(t2.clip_grad_norm(grads, norm / 3)) - norm) <= 2.0 ** -23 * norm
    check(grads, before, norm / 3 / (norm + 1e-6))


def test_one_element_of_many_counts():
    """the norm of zeros with one element that is not, wherever it lies: nothing is left out and nothing taken twice"""
    import t2fw_amd as t2
    flat = torch.zeros(24_000_017, device="cuda", dtype=torch.bfloat16)
    cuts = [0, 3, 2051, 1_000_000, 1_000_001, 9_999_999, 17_000_000, flat.numel()]
    parts = [flat[a:b] for a, b in zip(cuts, cuts[1:])]
    g = torch.Generator().manual_seed(0)
    places = cuts[:-1] + [c - 1 for c in cuts[1:]] + torch.randint(0, flat.numel(), (60,), generator=g).tolist()
    for at in places:
        flat[at] = 3.0
        assert float(t2.grad_norm(parts)) == 3.0, at
        flat[at] = 0.0

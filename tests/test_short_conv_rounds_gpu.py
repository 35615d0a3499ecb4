"""The convolution's gradients where a workgroup goes on with several rounds of stretches, each with its share of the weights' sums.

Inputs are small whole numbers, and nothing is rounded: every product and sum is a whole number below 2^24 (of the weights' gradient, of at most B T terms of 4), results of
16 bits are below 2^8.  So all results are equal to those in whole numbers of 64 bits, whatever the order of the sums."""
import pytest
import torch

from tests.test_short_conv import check, reference, run

# (rows, steps, channels, taps): workgroups of 16 stretches before they are shared out, at least 1024 of them
SHAPES = [(23, 2003, 130, 4), (40, 1111, 129, 2), (9, 3001, 197, 8), (1, 32003, 257, 3), (1500, 33, 130, 4), (2100, 900, 3, 4), (3000, 700, 5, 5)]


def groups_of(B, T, D, taps, dtype):
    """(workgroups along rows and time, rounds of each): from how many sums the workspace has room for"""
    from t2fw_amd import _lib
    steps = 4 if taps + (3 if dtype == torch.float32 else 0) > 5 else 8
    per_row = (D + 3) // 4 if D >= 4 else D
    lanes = 16
    while lanes > 1 and lanes // 2 >= per_row:
        lanes //= 2
    stretches = B * ((T + steps - 1) // steps)
    groups = -(-stretches // (256 // lanes))
    room = _lib.load().t2fw_short_conv_backward_workspace_bytes(B, T, D, taps, 0 if dtype == torch.float32 else 2)
    now = room // (D * (taps + 1) * 4)
    return groups, now


def whole(x, w, bias, state, lengths, gy, gs):
    x, w, bias, state, gy, gs = (t.detach().cpu().long() for t in (x, w, bias, state, gy, gs))
    (B, T, D), W = x.shape, w.shape[1]
    live = (torch.arange(T)[None] < lengths.cpu()[:, None])[:, :, None]
    xs, gy = torch.cat((state, x * live), 1), gy * live
    y = sum((xs[:, j:j + T] * w[:, j] for j in range(W)), bias.expand(B, T, D)) * live
    at = (lengths.cpu()[:, None] + torch.arange(W - 1))[:, :, None].expand(-1, -1, D)
    dxs = torch.zeros_like(xs)
    for j in range(W):
        dxs[:, j:j + T] += gy * w[:, j]
    dxs.scatter_add_(1, at, gs)
    dw = torch.stack([(gy * xs[:, j:j + T]).sum((0, 1)) for j in range(W)], 1)
    return {"y": y, "last": xs.gather(1, at), "d_x": dxs[:, W - 1:] * live, "d_w": dw, "d_bias": gy.sum((0, 1)), "d_state": dxs[:, :W - 1]}


def test_the_sizes_are_those_of_several_rounds():
    partial = 0
    for s in SHAPES:
        for dtype in (torch.float32, torch.bfloat16):
            groups, now = groups_of(*s, dtype)
            rounds = -(-groups // now)
            assert rounds >= 2, (s, dtype)
            partial += groups % rounds != 0
    assert partial >= 4                                  # the last workgroup has fewer rounds than the others


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_every_stretch_counts_once(shape, dtype):
    B, T, D, W = shape
    g = torch.Generator().manual_seed(T)
    make = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g)
    x, state, gy, gs = (make(-2, 2, *s).to(dtype).cuda() for s in ((B, T, D), (B, W - 1, D), (B, T, D), (B, W - 1, D)))
    w, bias = make(-3, 3, D, W).float().cuda(), make(-3, 3, D).float().cuda()
    for lengths in (torch.full((B,), T), torch.randint(0, T + 1, (B,), generator=g)):
        got = run((x, w, bias, state), lengths.cuda(), False, gy, gs)
        want = whole(x, w, bias, state, lengths, gy, gs)
        assert int(want["d_w"].abs().max()) < 1 << 24 and int(want["d_x"].abs().max()) <= 1 << 8
        for n in want:
            assert torch.equal(got[n].cpu().double(), want[n].double()), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_with_activation(dtype):
    from tests.test_short_conv import inputs
    B, T, D, W = SHAPES[0]
    ins, gy, gs = inputs(B, T, D, W, dtype, seed=1)
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(1))
    got, ref = run(ins, lengths.cuda(), True, gy, gs), reference(*ins, lengths, True, gy, gs)
    for n in got:
        check(n, got[n], ref[n])

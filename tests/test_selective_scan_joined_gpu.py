"""The selective scan over more than 48 chunks, whose maps a launch of its own puts together: by many parts of few lanes, and by few parts of many.  Bounds as in
test_selective_scan.py; how many chunks a call has is what its workspace has room for."""
import pytest
import torch

from tests.test_selective_scan import compare, inputs


def chunks_of(B, T, D, N):
    from t2fw_amd import _lib
    lanes = 1
    while 4 * lanes < N:
        lanes *= 2
    room = _lib.load().t2fw_selective_scan_workspace_bytes(B, T, D, N)
    assert room % (B * D * (4 * lanes + 1) * 4) == 0
    return room // (B * D * (4 * lanes + 1) * 4), B * D * lanes


FEW = [(3, 1100, 9, N) for N in (1, 6, 16, 30, 64)] + [(1, 2300, 5, 16)]
# a workgroup's 16 lanes go over the end of a row, and the last one over the end of all
MANY = [(3, 1124, 1401, 1), (3, 1124, 701, 5), (3, 1124, 350, 16), (3, 1124, 171, 17), (3, 1124, 86, 40)]


def test_the_sizes_are_those_of_joined_chunks():
    for s in FEW:
        chunks, lanes = chunks_of(*s)
        assert chunks > 48 and (chunks > 128 or lanes < 16 * 256), s
    assert any(chunks_of(*s)[0] > 128 for s in FEW)
    for s in MANY:
        chunks, lanes = chunks_of(*s)
        assert 48 < chunks <= 128 and lanes >= 16 * 256, s


@pytest.mark.gpu
@pytest.mark.parametrize("shape", FEW + MANY, ids=str)
def test_joined_chunks(shape):
    B, T, D, N = shape
    assert chunks_of(*shape)[0] > 48
    p, gy, gs = inputs(*shape, torch.float32, seed=N, long=True)
    # rows that end before the first chunk, in the first, in the last, and between
    lengths = torch.tensor([T - 1, 7, 530] if B == 3 else [T - 3])
    compare(p, lengths.cuda(), True, gy, gs)
    p["state"] = None
    compare(p, None, True, gy, gs)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 1100, 9, 16), (3, 1124, 350, 16)], ids=str)
def test_joined_chunks_in_16_bits_without_a_gate_and_of_no_steps(shape):
    B, T, D, N = shape
    p, gy, gs = inputs(*shape, torch.bfloat16, seed=N, gated=False, long=True)
    got = compare(p, torch.tensor([0, T, 64]).cuda(), True, gy, gs)
    assert torch.equal(got["last"][0], p["state"][0]) and torch.equal(got["d_state"][0], gs[0])

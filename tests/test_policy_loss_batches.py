"""policy_loss on batches of training sizes: tokens counted by a launch of their own, several rows to a workgroup, masks that begin at any
address.  Loss, log probabilities and every element of the gradient; the bounds are those of test_policy_loss.py."""
import pytest
import torch

from tests.test_policy_loss import call, check, inputs, reference

pytestmark = pytest.mark.gpu


# rows past what one wave (1024), four (4096) and sixteen count themselves; more rows than the chip holds workgroups of 64 (8192), 256 (1536,
# 2048), 512 (768) and 1024 threads (256, 512 where the row is read twice)
@pytest.mark.parametrize("N,V,dtype", [(1025, 500, torch.float32), (9003, 300, torch.float16), (8500, 1500, torch.bfloat16), (4099, 9001, torch.bfloat16),
                                       (2101, 2500, torch.float32), (801, 20011, torch.bfloat16), (601, 50257, torch.bfloat16),
                                       (16397, 40, torch.float32), (301, 50257, torch.float32), (531, 70001, torch.float32)], ids=str)
def test_values_and_gradients(N, V, dtype):
    ins = inputs(N, V, dtype, seed=N)
    held = torch.zeros(N + 1, dtype=torch.bool, device="cuda")
    held[1:] = ins[5]
    ins[5] = held[1:]                                        # an odd address
    assert ins[5].data_ptr() % 2 == 1
    z = ins[0].requires_grad_(True)
    want = reference(*ins)
    loss, logp = call(ins)
    grad, = torch.autograd.grad(loss, z)
    for n, v in (("loss", loss), ("logp", logp), ("grad", grad)):
        check(n, v, want[n])
    loss, _ = call(ins)
    again, = torch.autograd.grad(loss * 0.5, z)
    check("grad", again, (want["grad"][0] * 0.5, want["grad"][1] * 0.5))


@pytest.mark.parametrize("N", [1030, 17000])
def test_every_token_of_a_mask_counts_once(N):
    """a single token, and all but one, wherever it lies: the loss of equal tokens is that of one of them"""
    import t2fw_amd as t2
    z = torch.zeros(N, 8, device="cuda")
    targets, zero = torch.zeros(N, dtype=torch.int64, device="cuda"), torch.zeros(N, device="cuda")
    old, adv = torch.full((N,), -2.0794415, device="cuda"), torch.full((N,), 0.75, device="cuda")
    for at in (0, 1, 7, 8, 511, 512, 1023, 1024, N - 2, N - 1):
        for mask in (torch.zeros(N, dtype=torch.bool, device="cuda"), torch.ones(N, dtype=torch.bool, device="cuda")):
            mask[at] = ~mask[at]
            with torch.no_grad():
                loss, _ = t2.policy_loss(z, targets, old, zero, adv, mask=mask)
            assert abs(float(loss) + 0.75) < 1e-6, at

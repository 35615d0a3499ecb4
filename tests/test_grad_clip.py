"""clip_grad_norm and grad_norm against float64.

Bounds: squares and sums are carried in double, so that the norm is off by its rounding to float32 (2^-24, and as much for the
root); a scaled gradient by the coefficient's three roundings and its own, 2^-22, and by what storing rounds."""
import pytest
import torch

from tests.test_gated_scan import STORE, TINY

DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]


def make(sizes, dtypes, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtypes[i % len(dtypes)]).cuda() for i, s in enumerate(sizes)]


def norm64(ts):
    return float(torch.sqrt(sum((t.double().cpu() ** 2).sum() for t in ts)))


def check_scaled(got, before, norm, most):
    by = min(1.0, most / (norm + 1e-6))
    for g, b in zip(got, before):
        want = b.double().cpu() * by
        off = (g.double().cpu() - want).abs() - ((2.0 ** -22 + STORE[g.dtype]) * want.abs() + TINY[g.dtype])
        assert g.shape == b.shape and bool((off <= 0).all()), float(off.max())


# a whole chunk, one element more and less, several chunks, nothing
SIZES = [(1,), (8192,), (8191,), (8193,), (0,), (3, 5, 7), (200, 333), (100001,)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtypes", [[d] for d in DTYPES] + [DTYPES], ids=str)
@pytest.mark.parametrize("most", [0.5, 1e6])
def test_in_place_and_into_other_tensors(dtypes, most):
    import t2fw_amd as t2
    grads = make(SIZES, dtypes, seed=1)
    before = [g.clone() for g in grads]
    norm = norm64(before)
    for to in DTYPES:
        out = [torch.full(g.shape, 7.0, dtype=to, device="cuda") for g in grads]
        got = t2.clip_grad_norm(grads, most, out=out)
        assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - norm) <= 2.0 ** -23 * norm
        check_scaled(out, before, norm, most)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert torch.equal(t2.grad_norm(grads), got) and all(torch.equal(a, b) for a, b in zip(grads, before))
    versions = [g._version for g in grads]
    assert torch.equal(t2.clip_grad_norm(grads, most), got)
    check_scaled(grads, before, norm, most)
    assert all(g._version > v for g, v in zip(grads, versions))
    if most > norm:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 143, 144, 145, 300])
def test_more_tensors_than_one_launch_takes(count):
    import t2fw_amd as t2
    grads = make([(1 + 37 * (i % 11),) for i in range(count)], [torch.float32, torch.bfloat16], seed=count)
    before = [g.clone() for g in grads]
    norm = norm64(before)
    assert abs(float(t2.clip_grad_norm(grads, 1.0)) - norm) <= 2.0 ** -23 * norm
    check_scaled(grads, before, norm, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
def test_parts_of_a_buffer_and_dense_tensors_of_other_orders(dtype):
    import t2fw_amd as t2
    flat = make([(50000,)], [dtype], seed=3)[0]
    parts = [flat[1:20000], flat[20003:20004], flat[20005:49999]]
    before, norm = flat.clone(), norm64(parts)
    t2.clip_grad_norm(parts, 2.0)
    check_scaled(parts, [before[1:20000], before[20003:20004], before[20005:49999]], norm, 2.0)
    assert all(torch.equal(flat[i], before[i]) for i in (0, 20000, 20002, 20004, 49999))
    turned = make([(300, 200)], [dtype], seed=4)[0].t()
    kept = turned.clone()
    t2.clip_grad_norm([turned], 1.0)
    check_scaled([turned], [kept], norm64([kept]), 1.0)
    single = t2.clip_grad_norm(kept.contiguous(), 1.0)
    assert abs(float(single) - norm64([kept])) <= 2.0 ** -23 * norm64([kept])


@pytest.mark.gpu
def test_large_small_and_not_finite_gradients():
    import t2fw_amd as t2
    big = torch.full((1000,), 1e30, device="cuda")
    assert abs(float(t2.grad_norm([big])) / (1e30 * 1000 ** 0.5) - 1) < 1e-6       # squares of 1e60
    small = torch.full((1000,), 1e-30, device="cuda")
    assert abs(float(t2.grad_norm([small])) / (1e-30 * 1000 ** 0.5) - 1) < 1e-6
    assert float(t2.grad_norm([torch.zeros(5, device="cuda")])) == 0.0
    empty = torch.zeros(0, device="cuda")
    assert float(t2.clip_grad_norm([empty], 1.0)) == 0.0
    nan = [torch.ones(10, device="cuda"), torch.tensor([float("nan")], device="cuda")]
    assert bool(torch.isnan(t2.clip_grad_norm(nan, 1.0))) and bool(torch.isnan(nan[0]).all())
    inf = [torch.ones(10, device="cuda"), torch.tensor([float("inf"), 2.0], device="cuda")]
    assert bool(torch.isinf(t2.clip_grad_norm(inf, 1.0))) and bool((inf[0] == 0).all()) and bool(torch.isnan(inf[1][0])) and float(inf[1][1]) == 0
    zero = [torch.ones(10, device="cuda")]
    t2.clip_grad_norm(zero, 0.0)
    assert bool((zero[0] == 0).all())


@pytest.mark.gpu
def test_the_same_bits_again_on_another_stream_and_in_a_graph():
    import t2fw_amd as t2
    grads = make([(777, 1000), (12345,), (64,)], [torch.bfloat16], seed=8)
    out = [torch.empty(g.shape, device="cuda") for g in grads]

    def run():
        return [t2.clip_grad_norm(grads, 0.7, out=out)] + out
    want = [t.clone() for t in run()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in run()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for seed in (1, 2, 3):
        for g, t in zip(grads, make([(777, 1000), (12345,), (64,)], [torch.bfloat16], seed=seed)):
            g.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(replayed, run()))


@pytest.mark.gpu
def test_refusals():
    import t2fw_amd as t2
    g = torch.zeros(4, 4, device="cuda")
    for args in (([g, g.cpu()], 1.0), ([g[:, :2]], 1.0), ([g.long()], 1.0), ([g], -1.0), ([g], float("nan")), ([], 1.0)):
        with pytest.raises(RuntimeError):
            t2.clip_grad_norm(*args)
    for out in ([], [g[:2]], [g.t()], [g.cpu()], [g.int()]):
        with pytest.raises(RuntimeError):
            t2.clip_grad_norm([g], 1.0, out=out)


def test_host_memory_and_bad_c_calls_are_refused():
    import ctypes
    import t2fw_amd as t2
    from t2fw_amd import _lib
    with pytest.raises(RuntimeError, match="CUDA"):
        t2.clip_grad_norm([torch.zeros(3)], 1.0)
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 64

    def clip(src=p, dst=p, n=4, types=(0, 0), most=1.0, norm=p, ws=p, size=4096):
        d = (_lib.ClipDesc * 1)(_lib.ClipDesc(src, dst, n, *types))
        return lib.t2fw_clip_grad_norm(d, 1, most, norm, ws, size, None)
    assert clip(types=(9, 0)) == 2 and clip(types=(0, 9)) == 2 and clip(types=(0, 1)) == 2 and clip(n=-1) == 3 and clip(src=None) == 1
    assert clip(src=p + 1) == 4 and clip(most=-1.0) == 3 and clip(norm=None) == 1 and clip(ws=None) == 1 and clip(size=8) == 6
    assert lib.t2fw_clip_grad_norm(None, 1, 1.0, p, p, 4096, None) == 1 and lib.t2fw_clip_grad_norm(None, -1, 1.0, p, p, 4096, None) == 3
    assert lib.t2fw_clip_workspace_bytes(None, 3) == 0 and lib.t2fw_clip_workspace_bytes(None, 0) == 8

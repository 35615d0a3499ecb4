"""beam_select against the scores in float64, sorted; reorder_beams against indexing.

A score is off by the logarithm of a sum of float32 exponentials: each off by 2^-22 (the exponential's unit, and its argument's rounding at arguments
that count, 2^-24 |z - top| e^(z - top) < 2^-25), partial sums of 64 of them in four shares by 17 u, and a factor that is off by 2^-22 like them: 25.5 u of
the sum in all, less than 2^-19, which is 2^-19 in its logarithm.  What is returned is rounded to float32.  Which candidates come, and in what order, is exact wherever no two scores are nearer than that: the tests' inputs hold scores apart, or equal."""
import pytest
import torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def reference(logits, scores, n, finished=None, pad=0):
    z = logits.double().cpu()
    B, K, V = z.shape
    top = z.amax(-1, keepdim=True)
    logp = z - top - torch.log(torch.exp(z - top).sum(-1, keepdim=True))
    total = scores.double().cpu()[..., None] + logp
    total = torch.where(torch.isnan(total), torch.full((), float("-inf")).double(), total)
    if finished is not None:
        ended = torch.full((B, K, V), float("-inf")).double()
        ended[..., pad] = scores.double().cpu()
        total = torch.where(finished.cpu()[..., None], ended, total)
    best, at = torch.sort(total.view(B, -1), dim=1, descending=True, stable=True)
    return best[:, :n], at[:, :n] // V, at[:, :n] % V


def apart(best):
    """whether a request's scores are equal or further apart than they may be off"""
    gaps = (best[:, :-1] - best[:, 1:]).nan_to_num(0, 0, 0)
    return bool(((gaps == 0) | (gaps > 2.0 ** -17)).all())


def check(logits, scores, n, finished=None, pad=0):
    import t2fw_amd as t2
    got = t2.beam_select(logits, scores, count=n, finished=finished, pad=pad)
    best, beams, tokens = reference(logits, scores, min(n + 1, logits.shape[1] * logits.shape[2]), finished, pad)
    assert apart(best), "the test's own scores are too near one another"
    best, beams, tokens = best[:, :n], beams[:, :n], tokens[:, :n]
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int64
    assert torch.equal(got[1].cpu(), beams) and torch.equal(got[2].cpu(), tokens)
    off = (got[0].double().cpu() - best).abs()
    fine = (got[0].double().cpu() == best) | (off <= 2.0 ** -19 + 2.0 ** -24 * best.abs())
    assert bool(fine.all()), float(off.nan_to_num(0).max())


def logits_of(B, K, V, dtype, seed, std=3.0):
    """Distinct logits in every beam, few of them alike between beams: random orders of evenly spaced numbers, moved by the beam"""
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, K, V, generator=g) * std
    return z.to(dtype).cuda(), (torch.randn(B, K, generator=g) * 2 - 5).cuda()


# logits of one, of fewer than candidates, of less and more than a vector, a piece and several; beams of one, odd, many
SHAPES = [(1, 1, 1, 1), (2, 3, 2, 6), (1, 4, 8000, 8), (3, 1, 100, 100), (2, 5, 257, 7), (4, 2, 8192, 4), (1, 3, 8193, 6), (2, 8, 50257, 16), (1, 16, 20000, 32),
          (3, 64, 130, 128), (64, 8, 16389, 16), (8, 64, 8300, 128), (16, 40, 5000, 96), (30, 8, 40000, 20), (1, 200, 40, 20), (2, 2, 131072, 128), (70, 4, 60, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_best_of_all(shape, dtype):
    B, K, V, n = shape
    for seed in range(100):              # of the draws the first whose scores are apart
        logits, scores = logits_of(B, K, V, dtype, seed)
        if apart(reference(logits, scores, min(n + 1, K * V))[0]):
            return check(logits, scores, n)
    pytest.fail("no such draw")


@pytest.mark.gpu
@pytest.mark.parametrize("middle,std", [(1e3, 3.0), (-9e5, 3.0), (1048575.0, 3.0), (1e6, 1e5), (-3e7, 50.0), (0.0, 1e7)])
def test_large_logits(middle, std):
    """on either side of where the exponents are taken another way; B K V such that a thread has 8, 32 and 64 logits"""
    for B, K, V in ((1, 3, 5000), (8, 8, 40000), (64, 8, 16400)):
        for seed in range(100):
            logits, scores = logits_of(B, K, V, torch.float32, seed, std)
            logits += middle
            if apart(reference(logits, scores, 9)[0]):
                check(logits, scores, 8)
                break
        else:
            pytest.fail("no such draw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V,n", [(5, 9), (700, 16), (20000, 16), (20000, 128)])
def test_equal_scores_come_by_their_index(V, n, dtype):
    import t2fw_amd as t2
    zero = torch.zeros(2, 3, V, device="cuda", dtype=dtype)
    s, k, v = t2.beam_select(zero, torch.zeros(2, 3, device="cuda"), count=n)
    at = torch.arange(n).expand(2, n)
    assert torch.equal(k.cpu(), at // V) and torch.equal(v.cpu(), at % V) and bool((s == s[:, :1]).all())
    # a few that are better, among them two that are equal; zeros of both signs
    zero[:, 1, V // 2] = 1.0
    zero[:, 2, V // 2] = 1.0
    zero[:, 0, ::2] *= -1.0
    check(zero, torch.zeros(2, 3, device="cuda"), n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_best_ones_next_to_one_another(dtype):
    """all in one thread's share, in one piece, at the ends of pieces"""
    V = 3 * 8192 + 5
    for begin in (0, 8192 - 20, 8192, 2 * 8192 + 1000, V - 40):
        logits = torch.randn(1, 2, V, generator=torch.Generator().manual_seed(begin)).to(dtype).cuda() * 0.25
        logits[0, 1, begin:begin + 40] = 10 + torch.arange(40, device="cuda").to(dtype) * 0.25
        check(logits, torch.tensor([[-1.0, -2.0]], device="cuda"), 40)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_candidates_that_cannot_be(dtype):
    inf = float("inf")
    B, K, V, n = 6, 4, 9000, 12
    logits, scores = logits_of(B, K, V, dtype, 1)
    logits[:, :, 1::2] = -inf                            # a grammar's
    logits[1, 0] = -inf                                  # a beam without any
    logits[2] = -inf                                     # a request without any
    logits[3, :, 4:] = -inf                              # fewer than candidates
    scores[4, 1:] = -inf                                 # the first step
    scores[5] = -inf
    scores[0, 2] = float("nan")
    logits[0, 3, 7::2] = torch.finfo(dtype).min          # masks of the type's lowest value
    check(logits, scores, n)
    # the first step of a vocabulary smaller than the number of candidates
    small, s = logits_of(1, 4, 3, dtype, 2)
    s = torch.tensor([[0.0, -inf, -inf, -inf]], device="cuda")
    check(small, s, 8)


@pytest.mark.gpu
def test_beams_with_nan_and_infinities_come_last():
    import t2fw_amd as t2
    for bad in (float("nan"), float("inf")):
        for V, where in ((300, 7), (20000, 15000)):
            logits, scores = logits_of(2, 3, V, torch.float32, 4)
            logits[0, 1, where] = bad
            s, k, v = t2.beam_select(logits, scores, count=6)
            keep = logits.clone()
            keep[0, 1] = float("-inf")
            best, beams, tokens = reference(keep, scores, 6)
            assert torch.equal(k.cpu(), beams) and torch.equal(v.cpu(), tokens)
            s, k, v = t2.beam_select(logits[:1, 1:2].contiguous(), scores[:1, 1:2].contiguous(), count=4)
            assert bool((s == float("-inf")).all()) and bool((k == 0).all()) and bool(((v >= 0) & (v < V)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("V,pad", [(50, 0), (50, 49), (10000, 9000), (8192, 5)])
def test_ended_beams_go_on_alone(V, pad):
    logits, scores = logits_of(4, 3, V, torch.float32, V + pad)
    logits[0, 0, 3] = float("nan")                       # of an ended beam nothing is looked at
    logits[1, 1] = float("-inf")
    finished = torch.tensor([[True, False, False], [False, True, False], [True, True, True], [False, False, False]], device="cuda")
    scores[0, 0] = -1.25
    check(torch.where(finished[..., None], torch.zeros((), device="cuda"), logits), scores, 7, finished, pad)
    import t2fw_amd as t2
    a = t2.beam_select(logits, scores, count=7, finished=finished, pad=pad)
    b = t2.beam_select(torch.where(finished[..., None], torch.zeros((), device="cuda"), logits), scores, count=7, finished=finished, pad=pad)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert float(a[0][0][a[1][0] == 0][0]) == -1.25      # as it was, not through a sum


@pytest.mark.gpu
def test_no_requests_and_defaults():
    import t2fw_amd as t2
    s, k, v = t2.beam_select(torch.zeros(0, 3, 5, device="cuda"), torch.zeros(0, 3, device="cuda"))
    assert s.shape == k.shape == v.shape == (0, 3)
    z, scores = logits_of(2, 3, 50, torch.float32, 0)
    assert all(torch.equal(a, b) for a, b in zip(t2.beam_select(z, scores), t2.beam_select(z, scores, count=3)))


# ---- reordering ---------------------------------------------------------------------------------------------------

def arrays_of(rows, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(s, generator=g, device="cuda")
    return [make(rows * 3, 8, 8).to(torch.bfloat16), make(rows, 129), torch.randint(0, 9, (rows, 33), generator=g, device="cuda"),
            make(rows, 7, 5).half(), make(rows).double(), make(rows, 3) > 0, torch.randint(0, 200, (rows, 5001), generator=g, device="cuda").to(torch.uint8),
            make(rows, 2, 9), make(rows, 0), torch.complex(make(rows, 3), make(rows, 3))]


def expected(t, beams):
    B, K = beams.shape
    at = (torch.arange(B, device="cuda")[:, None] * K + beams).flatten()
    return t.view(B * K, -1).index_select(0, at).view(t.shape) if t.numel() else t


@pytest.mark.gpu
@pytest.mark.parametrize("B,K", [(1, 1), (2, 3), (1, 4), (5, 8), (3, 5), (2, 16), (2, 17), (1, 64)])
def test_states_move_to_their_beams(B, K):
    import t2fw_amd as t2
    g = torch.Generator(device="cuda").manual_seed(B * K)
    random = torch.randint(0, K, (B, K), generator=g, device="cuda")
    for beams in (random, torch.arange(K, device="cuda").expand(B, K).contiguous(), torch.arange(K, device="cuda").flip(0).expand(B, K).contiguous(),
                  torch.full((B, K), K - 1, device="cuda")):
        arrays = arrays_of(B * K)
        want = [expected(t, beams) for t in arrays]
        outs = [torch.empty_like(t) for t in arrays]
        kept = [t.clone() for t in arrays]
        assert all(a is b for a, b in zip(t2.reorder_beams(arrays, beams, out=outs), outs))
        assert all(torch.equal(a, b) for a, b in zip(arrays, kept)) and all(torch.equal(a, b) for a, b in zip(outs, want))
        assert all(a is b for a, b in zip(t2.reorder_beams(arrays, beams), arrays))
        assert all(torch.equal(a, b) for a, b in zip(arrays, want))


@pytest.mark.gpu
def test_more_arrays_than_a_launch_and_large_ones():
    import t2fw_amd as t2
    beams = torch.randint(0, 4, (3, 4), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    arrays = [torch.randn(12, 1 + i % 7, device="cuda") for i in range(200)] + [torch.randn(12, 1 << 20, device="cuda")]
    want = [expected(t, beams) for t in arrays]
    t2.reorder_beams(arrays, beams)
    assert all(torch.equal(a, b) for a, b in zip(arrays, want))
    # one tensor; an index that is no beam
    t = torch.arange(12.0, device="cuda")
    assert t2.reorder_beams(t, torch.tensor([[1, 1, 5, -1]] * 3, device="cuda"))[0] is t
    assert t.tolist() == [1, 1, 2, 3, 5, 5, 6, 7, 9, 9, 10, 11]
    version = t._version
    t2.reorder_beams([t], beams)
    assert t._version == version + 1
    # neighbours in one buffer, at odd bytes
    buffer = torch.arange(12 * 21 + 1, device="cuda").to(torch.uint8)
    a, b = buffer[1:1 + 12 * 10].view(12, 10), buffer[1 + 12 * 10:].view(12, 11)
    want = [expected(a.contiguous(), beams), expected(b.contiguous(), beams)]
    t2.reorder_beams([a, b], beams)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and int(buffer[0]) == 0


@pytest.mark.gpu
def test_state_cache_under_beams():
    import t2fw_amd as t2
    layer = t2.FastWeightState(value_dim=64, key_dim=64)
    B, K, H = 2, 3, 2
    beams = torch.tensor([[2, 0, 0], [1, 1, 2]], device="cuda")
    ins = [torch.rand(B * K * H, 5, 64, device="cuda", dtype=torch.float16) * 0.5 for _ in range(5)]
    with torch.no_grad():
        layer(*ins)
        before = layer.state.clone()
        held = layer.state
        assert layer.reorder(beams) is layer
        assert layer.state is held and torch.equal(layer.state, expected(before, beams))
    # a state that a recorded graph still needs is left as it is
    x = ins[0].clone().requires_grad_(True)
    layer.reset()
    out = layer(x, *ins[1:])
    held, before = layer.state, layer.state.detach().clone()
    layer.reorder(beams)
    assert layer.state is not held and torch.equal(held, before) and torch.equal(layer.state, expected(before, beams))
    out.sum().backward()
    t2.FastWeightState(4, 4).reorder(beams)              # nothing kept yet


@pytest.mark.gpu
def test_captured_search_step_replays():
    import t2fw_amd as t2
    logits, scores = logits_of(3, 4, 9001, torch.bfloat16, 0)
    arrays = arrays_of(12)
    kept = [t.clone() for t in arrays]

    def step():
        for t, k in zip(arrays, kept):
            t.copy_(k)
        s, k, v = t2.beam_select(logits, scores)
        t2.reorder_beams(arrays, k)
        return s, k, v
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for seed in range(3):
        new, s = logits_of(3, 4, 9001, torch.bfloat16, 10 + seed)
        logits.copy_(new)
        scores.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        want = t2.beam_select(new, s)
        assert all(torch.equal(a, b) for a, b in zip(res, want))
        assert all(torch.equal(a, expected(k, want[1])) for a, k in zip(arrays, kept))


def bad_calls():
    import t2fw_amd as t2
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    i64 = {"dtype": torch.int64}
    x, s, b = z(2, 3, 8), z(2, 3), z(2, 3, **i64)
    t = z(6, 4)
    return {
        "logits are flat": lambda: t2.beam_select(z(6, 8), s),
        "logits apart": lambda: t2.beam_select(z(2, 8, 3).transpose(1, 2), s),
        "logits are a number": lambda: t2.beam_select(z(), s),
        "scores are a number": lambda: t2.beam_select(x, z()),
        "beams are a number": lambda: t2.reorder_beams([t], z(**i64)),
        "logits in 64 bits": lambda: t2.beam_select(x.double(), s),
        "no logits": lambda: t2.beam_select(z(2, 3, 0), s),
        "no beams": lambda: t2.beam_select(z(2, 0, 8), z(2, 0)),
        "too many beams": lambda: t2.beam_select(z(1, 257, 8), z(1, 257), count=2),
        "scores of other beams": lambda: t2.beam_select(x, z(2, 4)),
        "scores in 16 bits": lambda: t2.beam_select(x, s.half()),
        "no candidates": lambda: t2.beam_select(x, s, count=0),
        "too many candidates": lambda: t2.beam_select(z(2, 3, 800), s, count=129),
        "more candidates than there are": lambda: t2.beam_select(x, s, count=25),
        "finished are numbers": lambda: t2.beam_select(x, s, finished=b),
        "finished of other beams": lambda: t2.beam_select(x, s, finished=z(2, 4, dtype=torch.bool)),
        "pad is no token": lambda: t2.beam_select(x, s, finished=z(2, 3, dtype=torch.bool), pad=8),
        "logits with gradients": lambda: t2.beam_select(x.clone().requires_grad_(True), s),
        "logits in host memory": lambda: t2.beam_select(x.cpu(), s),
        "beams in 32 bits": lambda: t2.reorder_beams([t], b.int()),
        "beams are flat": lambda: t2.reorder_beams([t], b.view(-1)),
        "beams in host memory": lambda: t2.reorder_beams([t], b.cpu()),
        "too many beams to move": lambda: t2.reorder_beams([z(65)], z(1, 65, **i64)),
        "rows that are no beams": lambda: t2.reorder_beams([z(7, 4)], b),
        "a scalar": lambda: t2.reorder_beams([z()], b),
        "apart": lambda: t2.reorder_beams([z(4, 6).t()], b),
        "twice": lambda: t2.reorder_beams([t, t], b),
        "overlapping": lambda: t2.reorder_beams([t.view(-1)[:12], t.view(-1)[6:18]], b),
        "results that are the beams": lambda: t2.reorder_beams([z(6, **i64)], b, out=[b.view(-1)]),
        "the beams themselves": lambda: t2.reorder_beams([b.view(-1)], b),
        "results among the inputs": lambda: t2.reorder_beams([t, z(6, 4)], b, out=[z(6, 4), t]),
        "in place by out": lambda: t2.reorder_beams([t], b, out=[t]),
        "results of another type": lambda: t2.reorder_beams([t], b, out=[t.half()]),
        "results of another shape": lambda: t2.reorder_beams([t], b, out=[z(6, 2, 2)]),
        "fewer results": lambda: t2.reorder_beams([t, z(6)], b, out=[z(6, 4)]),
        "in host memory": lambda: t2.reorder_beams([t.cpu()], b),
        "with gradients": lambda: t2.reorder_beams([t.clone().requires_grad_(True)], b),
        "a negated view": lambda: t2.reorder_beams([torch._neg_view(z(6, 4))], b),
        "a conjugate": lambda: t2.reorder_beams([z(6, 4, dtype=torch.complex64).conj()], b),
    }


@pytest.mark.gpu
def test_refusals():
    for name, call in bad_calls().items():
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(name)


def test_c_abi_refusals():
    import ctypes
    from t2fw_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p(ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 64)
    def sel(B=1, K=2, V=9, n=2, pad=0, dtype=0, room=1 << 20, ptrs=None):
        return lib.t2fw_beam_select(*(ptrs or [p] * 6), B, K, V, n, pad, dtype, p, room, None)
    assert sel(dtype=3) == 2 and sel(K=0) == 3 and sel(K=257) == 3 and sel(V=0) == 3 and sel(V=1 << 32) == 3 and sel(n=0) == 3
    assert sel(n=129, V=900) == 3 and sel(n=19) == 3 and sel(pad=9) == 3 and sel(pad=-1) == 3 and sel(B=0) == 0 and sel(room=8) == 6
    for i in (0, 1, 3, 4, 5):
        ptrs = [p] * 6
        ptrs[i] = None
        assert sel(ptrs=ptrs) == 1
    assert lib.t2fw_beam_select_workspace_bytes(32, 8, 50257, 16, 2) % (32 * 8 * (16 + 16 * 8)) == 0
    desc = (_lib.ReorderDesc * 1)(_lib.ReorderDesc(p, p, 64))
    move = lambda count=1, B=1, K=2, d=desc, beams=p: lib.t2fw_beam_reorder(d, count, beams, B, K, None)
    assert move(K=0) == 3 and move(K=65) == 3 and move(B=-1) == 3 and move(count=-1) == 3 and move(d=None) == 1 and move(beams=None) == 1
    assert move(B=0) == 0 and move(count=0) == 0
    assert move(d=(_lib.ReorderDesc * 1)(_lib.ReorderDesc(None, p, 64))) == 1 and move(d=(_lib.ReorderDesc * 1)(_lib.ReorderDesc(p, p, -1))) == 3
    assert move(B=1 << 30, d=(_lib.ReorderDesc * 1)(_lib.ReorderDesc(p, p, 1 << 20))) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", [1, 5, 16, 40, 128])
def test_few_tokens_that_are_allowed(n, dtype):
    """fewer than candidates, in one piece or several, among the first tokens or the last: those that cannot be follow by their index"""
    for V in (300, 9000, 40000):
        logits, scores = logits_of(3, 2, V, dtype, V + n)
        allowed = torch.zeros(3, 2, V, dtype=torch.bool, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(n)
        for b, k, count, top in ((0, 0, n // 2, V), (0, 1, 1, 20), (1, 0, n + 3, V), (1, 1, n, min(V, 2 * n + 5)), (2, 0, 3, 8), (2, 1, 0, 1)):
            allowed[b, k, torch.randperm(top, generator=g, device="cuda")[:count]] = True
        for seed in range(100):
            logits, scores = logits_of(3, 2, V, dtype, seed)
            logits = logits.masked_fill(~allowed, float("-inf"))
            if apart(reference(logits, scores, min(n + 1, 2 * V))[0]):
                break
        check(logits, scores, n)

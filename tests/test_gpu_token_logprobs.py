"""Log probabilities of given tokens, entropy, top alternatives and gradients
(ext.token_logprobs) against the 64-bit form: types, vocabularies around the
kernels' pieces, few and many rows, strides, ties, forbidden tokens, empty
rows, NaN, graphs.

Bounds (e = 2^-24): z = x - m is off by e |z|, so exp(z) by (|z| + 1.5 |z| + 2) e
relative (the subtraction, the factor log2 e, the exponential), a sum of
positive values by at most 1.2 e V / 256 + 40 e relative (values a lane adds one
after the other, then lanes); with Z = min(max |z| that matters, 100) below
which exp(z) is nothing, l and so log l is off by A = (2.5 Z + 44) e + 1.2 e V /
256; logp by A + e (|logp| + |log l|), the entropy, a weighted mean of -logp, by
2 A (1 + Z) + 4 e (1 + log V)."""
import math

import pytest

import llm_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24
INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    import rac_amd
    rac_amd.load()
    yield
    torch.cuda.synchronize()


def make(N, V, dt, seed=0, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((N, V), generator=gen) * spread
    tok = torch.randint(0, V, (N,), generator=gen)
    tok = torch.where(torch.rand(N, generator=gen) < 0.5, x.argmax(-1), tok)
    return x.to(dt).to(DEV), tok.to(DEV)


def bounds(x, V):
    x = x.double().cpu()
    z = (x - x.amax(-1, keepdim=True)).abs().clamp(max=100).nan_to_num(100.0).amax(-1)
    A = (2.5 * z + 44) * E + 1.2 * E * V / 256
    return A, 2 * A * (1 + z) + 4 * E * (1 + math.log(V))


def verify(x, tok, top=0):
    from rac_amd import ext
    V = x.size(-1)
    res = ext.token_logprobs(x, tok, top, return_lse=True)
    lp, ent, lse, logp, p = ref.logprob_reference(x, tok)
    A, AE = bounds(x, V)
    ref.check(res[0], lp, A + E * (lp.abs().nan_to_num(0, 0, 0) + math.log(V)), "logprob")
    ref.check(res[1], ent, AE, "entropy")
    ref.check(res[-1], lse, A + 2 * E * (lse.abs().nan_to_num(0, 0, 0) + math.log(V)), "lse")
    if top:
        # equal values: the lower token first
        order = torch.sort(x.float().cpu(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(res[3].cpu(), order)
        want = logp.gather(1, order)
        want = torch.where((lse == -INF)[:, None], torch.full_like(want, -INF), want)
        ref.check(res[2], want, (A[:, None] + E * (want.abs().nan_to_num(0, 0, 0) + math.log(V))), "top")
    return res, (lp, ent, lse, logp, p)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("N,V,top", [
    (1, 1, 1), (3, 2, 2), (1, 7, 3), (5, 64, 64), (2, 65, 1), (1, 1000, 20), (4, 2047, 5), (3, 2049, 64),
    (2, 4097, 20), (7, 32000, 20), (1, 100003, 5), (1100, 300, 5), (1030, 5003, 1), (2, 8195, 0)])
def test_token_logprobs(N, V, top, dt):
    verify(*make(N, V, dt), top)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N,V", [(2, 9000), (1500, 1201)])
def test_forbidden_tokens_ties_and_empty_rows(N, V, dt):
    x, tok = make(N, V, dt)
    x[:, ::3] = -INF
    x[0, 100:200] = 11.0                       # ties across lanes and vectors, at the top
    x[0, V - 1] = 11.0
    x[1] = -INF                                # a row of nothing
    verify(x, tok, 20)
    x[0] = 0.0                                 # a row of equal values
    x[0, 1::2] = -0.0                          # zeros of either sign are equal
    verify(x, tok, 64)


@pytest.mark.parametrize("N", [1, 1100])
def test_peaked_and_ascending_rows(N):
    # one token has it all; values ascend, so that every one enters the list
    V = 3001
    x, tok = make(N, V, F32)
    x[0] = -20.0
    x[0, 17] = 30.0
    tok[0] = 17
    verify(x, tok, 5)
    x[0] = torch.linspace(-5, 5, V, device=DEV)
    verify(x, tok, 64)


@pytest.mark.parametrize("N", [2, 1100])
def test_nan_and_infinity_in_a_row(N):
    from rac_amd import ext
    for bad in (float("nan"), INF):
        x, tok = make(N, 5000, F32)
        x[1, 4321] = bad
        lp, ent, tv, ti, lse = ext.token_logprobs(x, tok, 3, return_lse=True)
        for t in (lp, ent, lse):
            assert bool(t[1].isnan()) and not bool(t[0].isnan())
        assert bool(tv[1].isnan().all()) and not bool(tv[0].isnan().any())
        dx = ext.token_logprobs_backward(x, tok, lse, ent, torch.ones_like(lp), None)
        assert bool(dx[1].isnan().all()) and not bool(dx[0].isnan().any())


def test_tokens_that_are_none_or_past_the_vocabulary():
    from rac_amd import ext
    x, tok = make(6, 300, F32)
    tok[1], tok[2], tok[3] = -1, -100, 300
    lp, ent, lse = ext.token_logprobs(x, tok, return_lse=True)
    assert float(lp[1]) == 0 and float(lp[2]) == 0 and bool(lp[3].isnan())
    assert not bool(ent.isnan().any())
    dx = ext.token_logprobs_backward(x, tok, lse, ent, torch.ones_like(lp), None)
    assert bool((dx[1:3] == 0).all()) and bool(dx[3].isnan().all()) and not bool(dx[4:].isnan().any())


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("N,V", [(1, 1), (3, 50), (2, 5001), (5, 4096), (300, 1003)])
@pytest.mark.parametrize("parts", ["both", "logprob", "entropy"])
def test_gradients(N, V, dt, parts):
    from rac_amd import ext
    x, tok = make(N, V, dt)
    if V > 10:
        x[0, ::4] = -INF
        x[0, int(tok[0])] = 1.0
    res = ext.token_logprobs(x, tok, return_lse=True)
    gen = torch.Generator().manual_seed(4)
    gl, ge = (torch.randn(N, generator=gen).to(DEV) for _ in range(2))
    gl, ge = gl if parts != "entropy" else None, ge if parts != "logprob" else None
    dx = ext.token_logprobs_backward(x, tok, res[2], res[1], gl, ge)
    _, ent, lse, logp, p = ref.logprob_reference(x, tok)
    g = gl.double().cpu() if gl is not None else torch.zeros(N, dtype=torch.float64)
    h = ge.double().cpu() if ge is not None else torch.zeros(N, dtype=torch.float64)
    hit = torch.zeros((N, V), dtype=torch.float64).scatter_(1, tok.cpu()[:, None], 1.0)
    pl = torch.where(p > 0, logp + ent[:, None], torch.zeros_like(p))
    want = g[:, None] * (hit - p) - h[:, None] * p * pl
    A, AE = bounds(x, V)
    la = logp.abs().nan_to_num(0, 0, 0).clamp(max=110)
    # p is off by the logp's bound and its exponential's, the entropy and logp by theirs
    P = (A + 2 * E * (lse.abs() + math.log(V)))[:, None] + (2.5 * la + 4) * E
    tol = p * (g.abs()[:, None] + h.abs()[:, None] * (la + ent[:, None])) * (P + 8 * E)
    tol += h.abs()[:, None] * p * (AE[:, None] + P) + (ref.half_step(dt) + 2 * E) * want.abs()
    tol += g.abs()[:, None] * hit * 2 * E + 2.0 ** -126 + (2.0 ** -25 if dt == F16 else 0.0)
    ref.check(dx, want, tol, "dx")


def test_rows_that_lie_apart():
    from rac_amd import ext
    for dt in (F32, BF16):
        x, tok = make(8, 1001, dt)
        wide = torch.full((8, 1009), float("nan"), device=DEV, dtype=dt)
        for shift in (0, 1, 3):
            wide[:, shift:shift + 1001] = x
            v = wide[:, shift:shift + 1001]
            a, b = (ext.token_logprobs(t, tok, 5, return_lse=True) for t in (x, v))
            assert torch.equal(a[3], b[3])
            verify(v, tok, 5)
            one = torch.ones_like(a[0])
            d1 = ext.token_logprobs_backward(x, tok, a[4], a[1], one, one)
            d2 = ext.token_logprobs_backward(v, tok, a[4], a[1], one, one)
            assert torch.equal(d1, d2)
    # leading dims, other token types, a transposed and a broadcast tensor
    y = x.view(2, 4, 1001)
    a = ext.token_logprobs(y, tok.view(2, 4).int(), 2)
    b = ext.token_logprobs(x, tok, 2)
    assert tuple(a[2].shape) == (2, 4, 2) and all(torch.equal(s.reshape(t.shape), t) for s, t in zip(a, b))
    assert torch.equal(ext.token_logprobs(x.t().contiguous().t(), tok)[0], b[0])
    # copies of a row of 1001 values start at other places of 16 bytes, and so sum in other orders
    verify(x[:1].expand(8, -1), tok)


def test_no_rows():
    from rac_amd import ext
    lp, ent, tv, ti = ext.token_logprobs(torch.empty((0, 10), device=DEV), torch.empty(0, device=DEV, dtype=torch.int64), 3)
    assert lp.numel() == 0 and tuple(tv.shape) == (0, 3)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_autograd(dt):
    from rac_amd import ext, rac_torch
    x, tok = make(12, 777, dt)
    leaf = x.clone().requires_grad_()
    lp, ent, tv, ti = rac_torch.rac_token_logprobs(leaf, tok, top=4)
    assert not tv.requires_grad and torch.equal(ti, ext.token_logprobs(x, tok, 4)[3])
    (0.3 * ent.sum() - lp.mean()).backward()
    r = ext.token_logprobs(x, tok, return_lse=True)
    want = ext.token_logprobs_backward(x, tok, r[2], r[1], torch.full_like(lp, -1 / 12), torch.full_like(lp, 0.3))
    assert torch.equal(leaf.grad, want)
    leaf.grad = None
    lp, _ = rac_torch.rac_token_logprobs(leaf, tok)              # one of the two only
    lp.sum().backward()
    assert torch.equal(leaf.grad, ext.token_logprobs_backward(x, tok, r[2], r[1], torch.ones_like(lp), None))


def test_gradient_against_differences():
    """Along random directions; the sums' rounding 2^-22 of values near 10
    over the step, and the step's square times a third derivative below 1."""
    from rac_amd import ext
    x, tok = make(4, 400, F32)
    r = ext.token_logprobs(x, tok, return_lse=True)
    gen = torch.Generator().manual_seed(2)
    gl, ge = (torch.randn(4, generator=gen).to(DEV) for _ in range(2))
    dx = ext.token_logprobs_backward(x, tok, r[2], r[1], gl, ge)

    def f(t):
        lp, ent = ext.token_logprobs(t, tok)
        return float((lp.double() * gl.double() + ent.double() * ge.double()).sum())

    h = 2.0 ** -6
    for _ in range(4):
        dirn = torch.randn(x.shape, generator=gen).to(DEV)
        dirn /= dirn.norm()
        diff = (f(x + h * dirn) - f(x - h * dirn)) / (2 * h)
        exact = float((dx.double() * dirn.double()).sum())
        assert abs(diff - exact) <= 8 * 10 * 2.0 ** -22 / h + 4 * h * h


def test_a_recorded_graph_replays():
    from rac_amd import ext
    for N, V in ((3, 9001), (1200, 500)):
        x, tok = make(N, V, F32)
        g = torch.ones(N, device=DEV)

        def step():
            r = ext.token_logprobs(x, tok, 5, return_lse=True)
            return (*r, ext.token_logprobs_backward(x, tok, r[4], r[1], g, g))

        step()
        torch.cuda.synchronize()
        graphs, outs = [], []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(step())
            graphs.append(graph)
        for i in range(3):
            x.copy_(make(N, V, F32, seed=20 + i)[0])
            for graph in graphs:
                graph.replay()
            torch.cuda.synchronize()
            want = step()
            for got in outs:
                assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_more_than_2_31_logits():
    from rac_amd import ext
    N, V = 17000, 131073                       # 4.5 GB in bf16, elements past 2^31
    x = torch.zeros((N, V), device=DEV, dtype=BF16)
    x[-1, V - 1] = 12.0
    tok = torch.full((N,), V - 1, device=DEV)
    lp, ent, tv, ti, lse = ext.token_logprobs(x, tok, 2, return_lse=True)
    l = math.exp(12.0) + V - 1
    tol = 2.0 ** -20 * 12                      # A at z = 12, and lse's own rounding
    assert abs(float(lp[-1]) - (12.0 - math.log(l))) < tol and abs(float(lp[0]) + math.log(V)) < tol
    assert ti[-1].tolist() == [V - 1, 0] and ti[0].tolist() == [0, 1]
    dx = ext.token_logprobs_backward(x, tok, lse, ent, torch.ones_like(lp), None)
    assert abs(float(dx[-1, V - 1]) - (1 - math.exp(12.0) / l)) < 2.0 ** -7 and float(dx[-1, 0]) < 0

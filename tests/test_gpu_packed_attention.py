"""Causal attention over packed sequences (ext.packed_attention and its
gradients) against the 64-bit form, within the bounds of llm_ref: types, head
layouts, lengths around the kernels' tiles of 32, 64 and 128 rows, strides,
masked places, rows outside the sequences, graphs and streams."""
import math

import pytest

import llm_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    import rac_amd
    rac_amd.load()
    yield
    torch.cuda.synchronize()


def cu_of(lens, start=0):
    cu = [start]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, device=DEV, dtype=torch.int32)


def make(lens, H, G, d, dt, seed=0, extra=0, start=0):
    gen = torch.Generator().manual_seed(seed)
    total = start + sum(lens) + extra
    q, k, v, g = (torch.randn((total, h, d), generator=gen) for h in (H, G, G, H))
    return [t.to(dt).to(DEV) for t in (q * 1.5, k, v, g)]


def run(q, k, v, g, cu, scale=None):
    from rac_amd import ext
    out, lse, lo = ext.packed_attention(q, k, v, cu, scale, return_lse=True, return_residual=True)
    dq, dk, dv = ext.packed_attention_backward(g, q, k, v, out, lse, cu, scale, lo)
    return dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)


def compare(got, want, tol, names=("out", "lse", "dq", "dk", "dv")):
    for n in names:
        ref.check(got[n], want[n], tol[n], n)


CASES = [
    ([1], 1, 1, 32), ([2, 1, 0, 3], 2, 1, 64), ([31, 32, 33], 4, 2, 64), ([127, 1, 128, 129], 4, 1, 64),
    ([63, 65, 64], 6, 3, 80), ([0, 0, 5, 0], 8, 8, 32), ([300, 17], 8, 2, 128), ([200], 2, 2, 96),
    ([77, 140], 3, 1, 256), ([50, 9], 2, 1, 136), ([40, 3], 4, 4, 1), ([70], 2, 1, 7), ([129], 2, 2, 33),
    ([1] * 70, 2, 1, 64), ([5, 0] * 100, 8, 2, 16),
]


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("lens,H,G,d", CASES)
def test_packed_attention_and_gradients(lens, H, G, d, dt):
    q, k, v, g = make(lens, H, G, d, dt)
    got = run(q, k, v, g, cu_of(lens))
    want, tol = ref.packed_reference(q, k, v, lens, 1 / math.sqrt(d), g)
    compare(got, want, tol)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_long_sequence(dt):
    lens = [1500]
    q, k, v, g = make(lens, 2, 1, 128, dt)
    compare(run(q, k, v, g, cu_of(lens)), *ref.packed_reference(q, k, v, lens, 1 / math.sqrt(128), g))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("d", [64, 80, 33])
def test_slices_of_a_stacked_projection(dt, d):
    lens, H, G = [100, 45], 4, 2
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn((145, (H + 2 * G) * d + 1), generator=gen).to(dt).to(DEV)
    for shift in (0, 1):                                     # 1: rows that start on no 16-byte boundary
        w = qkv[:, shift:shift + (H + 2 * G) * d].unflatten(1, (H + 2 * G, d))
        q, k, v = w[:, :H], w[:, H:H + G], w[:, H + G:]
        g = torch.randn((145, H, d), generator=gen).to(dt).to(DEV)
        compare(run(q, k, v, g, cu_of(lens)), *ref.packed_reference(q, k, v, lens, 1 / math.sqrt(d), g))


def test_strides_give_the_same_bits():
    from rac_amd import ext
    lens, H, G, d = [90, 60], 4, 2, 64
    q, k, v, g = make(lens, H, G, d, BF16)
    cu = cu_of(lens)
    a = run(q, k, v, g, cu)
    pad = torch.full((150, H + 2 * G, d + 3), float("nan"), device=DEV, dtype=BF16)
    pq, pk, pv = pad[:, :H, 1:d + 1], pad[:, H:H + G, 1:d + 1], pad[:, H + G:, 1:d + 1]
    for p, t in ((pq, q), (pk, k), (pv, v)):
        p.copy_(t)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    last_strided = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    for x in ((pq, pk, pv), heads_first, last_strided):
        b = run(*x, g, cu)
        assert all(torch.equal(a[n], b[n]) for n in a)
    g2 = g.transpose(0, 1).contiguous().transpose(0, 1)
    b = run(q, k, v, g2, cu)
    assert all(torch.equal(a[n], b[n]) for n in a)
    # one key / value head for all, given by a broadcast
    one = k[:, :1]
    wide = run(q, one.expand(-1, 4, -1), v[:, :1].expand(-1, 4, -1), g, cu)
    assert torch.equal(wide["out"], ext.packed_attention(q, one, v[:, :1], cu))


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_same_call_same_bits(dt):
    lens = [260, 130]
    q, k, v, g = make(lens, 8, 2, 64, dt)
    cu = cu_of(lens)
    a = run(q, k, v, g, cu)
    for _ in range(3):
        b = run(q, k, v, g, cu)
        assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_sequences_do_not_see_each_other(dt):
    # bits of a sequence alone and in the middle of a pack whose others hold NaN
    lens, H, G, d = [70, 99, 40], 4, 2, 64
    q, k, v, g = make(lens, H, G, d, dt)
    mid = slice(70, 169)
    alone = run(*(t[mid].contiguous() for t in (q, k, v, g)), cu_of([99]))
    for t in (q, k, v, g):
        t[:70] = float("nan")
        t[169:] = float("inf")
    packed = run(q, k, v, g, cu_of(lens))
    for n in ("out", "dq", "dk", "dv"):
        assert torch.equal(packed[n][mid], alone[n]), n
    assert torch.equal(packed["lse"][:, mid], alone["lse"])


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", ["k", "v", "q", "g"])
def test_values_a_row_does_not_see(dt, bad, which):
    """One token's key, value, query or gradient is not finite: earlier rows
    (for the keys' gradients: later keys) stay within their bounds."""
    lens, H, G, d, at = [200], 2, 1, 64, 137
    q, k, v, g = make(lens, H, G, d, dt)
    clean = {"q": q.clone(), "k": k.clone(), "v": v.clone(), "g": g.clone()}
    dict(q=q, k=k, v=v, g=g)[which][at, :, 5] = bad
    got = run(q, k, v, g, cu_of(lens))
    want, tol = ref.packed_reference(clean["q"], clean["k"], clean["v"], lens, 1 / math.sqrt(d), clean["g"])
    for n in ("out", "dq"):
        ref.check(got[n][:at], want[n][:at], tol[n][:at], n)
    ref.check(got["lse"][:, :at], want["lse"][:, :at], tol["lse"][:, :at], "lse")
    for n in ("dk", "dv"):
        # keys behind the token see its row in nothing they sum
        if which in ("q", "g"):
            ref.check(got[n][at + 1:], want[n][at + 1:], tol[n][at + 1:], n)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("heads", [2, 64])
def test_seen_and_unseen_values_that_are_not_finite(dt, heads):
    """An early token's NaN reaches the rows behind it in its own column only,
    whatever a later token, in the tiles on those rows' diagonals, holds (two
    head counts: one and four row sets to a workgroup in the longer sequence)."""
    lens, d = [700], 64
    q, k, v, g = make(lens, heads, 1, d, dt)
    v[10, 0, 7] = float("nan")
    v[650, 0, 3] = float("inf")
    k[651, 0, 5] = float("nan")
    out = run(q, k, v, g, cu_of(lens))["out"]
    clean = make(lens, heads, 1, d, dt)
    want, tol = ref.packed_reference(clean[0][:, :2], clean[1], clean[2], lens, 1 / math.sqrt(d))
    rest = [c for c in range(d) if c != 7]
    assert bool(out[10:, :, 7].isnan().all()) and not bool(out[:650, :, rest].isnan().any())
    ref.check(out[:650, :2][..., rest], want["out"][:650][..., rest], tol["out"][:650][..., rest], "out")
    g[655, :, 9] = float("nan")                      # and a late row's gradient the keys before it only
    got = run(*clean[:3], g, cu_of(lens))
    want, tol = ref.packed_reference(clean[0][:, :2], clean[1], clean[2], lens, 1 / math.sqrt(d), clean[3][:, :2])
    assert bool(got["dv"][:656, :, 9].isnan().all()) and not bool(got["dv"][656:].isnan().any())
    assert not bool(got["dv"][:, :, :9].isnan().any())
    if heads == 2:
        for n in ("dk", "dv"):
            ref.check(got[n][656:], want[n][656:], tol[n][656:], n)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_nan_reaches_what_it_should(dt):
    lens, d, at = [150], 64, 100
    q, k, v, g = make(lens, 2, 1, d, dt)
    v[at, 0, 7] = float("nan")
    got = run(q, k, v, g, cu_of(lens))
    assert bool(got["out"][at:, :, 7].isnan().all()) and not bool(got["out"][:at].isnan().any())
    assert not bool(got["out"][at:, :, :7].isnan().any())
    v[at, 0, 7] = float("inf")
    assert bool((run(q, k, v, g, cu_of(lens))["out"][at:, :, 7] == float("inf")).all())


@pytest.mark.parametrize("dt", [F32, BF16])
def test_nothing_but_nan(dt):
    lens = [300, 40]
    q, k, v, g = make(lens, 4, 2, 64, dt)
    for t in (q, k, v, g):
        t[:300] = float("nan")
    got = run(q, k, v, g, cu_of(lens))
    for n in ("out", "dq", "dk", "dv"):
        assert bool(got[n][:300].isnan().all()) and not bool(got[n][300:].isnan().any()), n


def test_scores_of_minus_infinity():
    # a key that gives every query -inf has no part; a row of nothing else is 0
    lens, d = [40], 64
    q, k, v, g = make(lens, 1, 1, d, F32)
    q[..., 0] = 1.0
    k[0, 0, 0] = -float("inf")
    got = run(q, k, v, g, cu_of(lens))
    assert bool((got["out"][0] == 0).all()) and float(got["lse"][0, 0]) == -float("inf")
    assert bool((got["dq"][0, :, 1:] == 0).all())      # of column 0: 0 times -inf
    assert not bool(got["out"].isnan().any()) and bool((got["dv"][0] == 0).all())
    rest = run(q[1:], k[1:], v[1:], g[1:], cu_of([39]))
    tol = ref.packed_reference(q[1:], k[1:], v[1:], [39], 1 / math.sqrt(d), g[1:])[1]
    for n in ("out", "dv"):
        ref.check(got[n][1:], rest[n].double().cpu(), 2 * tol[n], n)


@pytest.mark.parametrize("dt", [F32, F16])
def test_large_scores(dt):
    # scores near 1000: exponentials of their differences only
    lens, d = [65, 130], 64
    q, k, v, g = make(lens, 2, 1, d, dt)
    q, k = q * 8, k * 8
    compare(run(q, k, v, g, cu_of(lens)), *ref.packed_reference(q, k, v, lens, 1 / math.sqrt(d), g), names=("out", "lse"))


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_scale(scale):
    lens = [50, 77]
    q, k, v, g = make(lens, 2, 1, 32, F32)
    compare(run(q, k, v, g, cu_of(lens), scale), *ref.packed_reference(q, k, v, lens, scale, g))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_rows_outside_the_sequences(dt):
    from rac_amd import ext
    lens, start, extra, H, G, d = [60, 0, 33], 9, 200, 4, 2, 80
    q, k, v, g = make(lens, H, G, d, dt, extra=extra, start=start)
    for t in (q, k, v, g):
        t[:start] = float("nan")
        t[start + 93:] = float("nan")
    cu = cu_of(lens, start)
    got = run(q, k, v, g, cu)
    want, tol = ref.packed_reference(q, k, v, lens, 1 / math.sqrt(d), g, start=start)
    compare(got, want, tol, names=("out", "dq", "dk", "dv"))            # zeros outside
    kept = torch.full_like(q, 7.0)
    res = ext.packed_attention(q, k, v, cu, out=kept)
    assert res is kept and bool((kept[:start] == 7).all()) and bool((kept[start + 93:] == 7).all())
    assert torch.equal(kept[start:start + 93], got["out"][start:start + 93])


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("d", [64, 33])
def test_the_residual_of_a_rounded_output(dt, d):
    """out + residual is the output to the sums' own error: its bound without
    the output's rounding, half a step of what rounding can take away besides.
    The gradients hold their bounds without it, and with it a bound whose D has
    only the residual's error."""
    from rac_amd import ext
    lens = [90, 41]
    q, k, v, g = make(lens, 4, 2, d, dt)
    cu = cu_of(lens)
    out, lse, lo = ext.packed_attention(q, k, v, cu, return_lse=True, return_residual=True)
    want, tol = ref.packed_reference(q, k, v, lens, 1 / math.sqrt(d), g)
    u = ref.half_step(dt)
    fine = tol["out"] - u * want["out"].abs() + u * u * want["out"].abs() + 2.0 ** -25
    ref.check(out.double() + lo.double(), want["out"], fine, "out + residual")
    assert bool((lo.double().abs().cpu() <= u * 1.01 * out.double().abs().cpu() + 2.0 ** -25).all())
    without = dict(zip(("dq", "dk", "dv"), ext.packed_attention_backward(g, q, k, v, out, lse, cu)))
    compare(without, want, tol, names=("dq", "dk", "dv"))
    wide = torch.full((131, 4, d + 1), float("nan"), device=DEV, dtype=dt)[..., 1:]
    wide.copy_(lo)
    both = [ext.packed_attention_backward(g, q, k, v, out, lse, cu, residual=x) for x in (lo, wide)]
    assert all(torch.equal(a, b) for a, b in zip(*both))
    assert ext.packed_attention(q.float(), k.float(), v.float(), cu, return_residual=True)[1] is None


def test_no_sequences_and_no_rows():
    from rac_amd import ext
    q, k, v, g = make([20], 2, 1, 64, F32)
    assert bool((ext.packed_attention(q, k, v, cu_of([])) == 0).all())
    e = ext.packed_attention(q[:0], k[:0], v[:0], cu_of([0, 0]))
    assert tuple(e.shape) == (0, 2, 64)
    a = run(q[:0], k[:0], v[:0], g[:0], cu_of([0]))
    assert a["dq"].numel() == 0 and tuple(a["lse"].shape) == (2, 0)


def test_lengths_that_do_not_fit_touch_nothing_else():
    from rac_amd import ext
    q, k, v, _ = make([64], 2, 1, 64, F32)
    guard = torch.full((64 + 256, 2, 64), 3.0, device=DEV)
    ext.packed_attention(q, k, v, torch.tensor([0, 1000], device=DEV, dtype=torch.int32), out=guard[128:192])
    assert bool((guard[:128] == 3).all()) and bool((guard[192:] == 3).all())
    assert torch.equal(guard[128:192], ext.packed_attention(q, k, v, cu_of([64])))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_autograd(dt):
    from rac_amd import rac_torch
    lens, H, G, d = [90, 41], 4, 2, 64
    q, k, v, g = make(lens, H, G, d, dt)
    cu = cu_of(lens)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = rac_torch.rac_packed_attention(*leaves, cu)
    out.backward(g)
    plain = run(q, k, v, g, cu)
    assert torch.equal(out, plain["out"])
    for t, n in zip(leaves, ("dq", "dk", "dv")):
        assert torch.equal(t.grad, plain[n])
    # a broadcast key / value head gets the sum of its copies' gradients
    k1 = k[:, :1].clone().requires_grad_()
    out = rac_torch.rac_packed_attention(q, k1.expand(-1, 4, -1), v[:, :1].expand(-1, 4, -1), cu)
    (gk,) = torch.autograd.grad(out, k1, g)
    want, tol = ref.packed_reference(q, k[:, :1], v[:, :1], lens, 1 / math.sqrt(d), g)
    wide, wtol = ref.packed_reference(q, k[:, :1].expand(-1, 4, -1), v[:, :1].expand(-1, 4, -1), lens, 1 / math.sqrt(d), g)
    # four rounded parts added in the type: each within its bound, each sum half a step of at most the parts' size
    ref.check(gk, want["dk"], wtol["dk"].sum(1, keepdim=True) + 4 * ref.half_step(dt) * wide["dk"].abs().sum(1, keepdim=True)
              + tol["dk"], "dk")
    assert not rac_torch.rac_packed_attention(q, k, v, cu).requires_grad


def test_gradients_against_differences():
    """Central differences of the scalar sum(out * g) in fp32 along random
    directions: their own error is the step's square times the third
    derivative and the rounding of the sums over the step."""
    from rac_amd import ext
    lens, H, G, d = [33, 12], 2, 1, 32
    q, k, v, g = make(lens, H, G, d, F32)
    cu = cu_of(lens)
    r = run(q, k, v, g, cu)
    f = lambda a, b, c: float((ext.packed_attention(a, b, c, cu).double() * g.double()).sum())
    gen = torch.Generator().manual_seed(9)
    h = 2.0 ** -7
    for i, n in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        dirn = torch.randn(x[i].shape, generator=gen).to(DEV)
        dirn /= dirn.norm()
        lo, hi = list(x), list(x)
        lo[i], hi[i] = x[i] - h * dirn, x[i] + h * dirn
        diff = (f(*hi) - f(*lo)) / (2 * h)
        exact = float((r[n].double() * dirn.double()).sum())
        # |out| <= about 4, 45 rows of 64: rounding of out 2^-22 * |g|_1 / h; third derivative of order 10
        assert abs(diff - exact) <= 2.0 ** -22 * float(g.abs().sum()) / h + 10 * h * h, n


@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_recorded_graph_replays_with_new_lengths(dt):
    from rac_amd import ext
    H, G, d = 4, 2, 64
    q, k, v, g = make([256], H, G, d, dt)
    cu = cu_of([256, 0, 0])
    run(q, k, v, g, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(q, k, v, g, cu)
    for lens in ([100, 56, 100], [1, 254, 1], [256, 0, 0], [17, 40, 60]):
        cu.copy_(cu_of(lens))
        q.mul_(-0.75)
        graph.replay()
        torch.cuda.synchronize()
        want = run(q, k, v, g, cu)
        n = sum(lens)
        for name in ("out", "dq", "dk", "dv"):
            assert torch.equal(got[name], want[name]), (lens, name)
        assert torch.equal(got["lse"][:, :n], want["lse"][:, :n])


def test_two_streams():
    lens = [300, 211]
    sets = [make(lens, 4, 2, 64, BF16, seed=s) for s in (1, 2)]
    cu = cu_of(lens)
    want = [run(*s, cu) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(*sets[i], cu)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(a[n], b[n]) for n in a)

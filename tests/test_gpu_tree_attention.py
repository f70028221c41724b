"""Attention of a tree of drafted tokens over a cache (ext.tree_attention)
against the 64-bit form, within the bounds of llm_ref: types, head layouts,
trees, cache lengths around the kernels' tiles, strides, masked places, lengths
outside the cache, graphs and streams."""
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


def tree(T, kind, seed=0):
    if kind == "chain":
        return list(range(-1, T - 1))
    if kind == "flat":
        return [-1] * T
    gen = torch.Generator().manual_seed(seed)
    return [int(torch.randint(-1, t, (1,), generator=gen)) if t else -1 for t in range(T)]


def make(B, T, H, G, d, cap, dt, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn((B, T, H, d), generator=gen) * 1.5
    k, v = (torch.randn((B, G, cap, d), generator=gen) for _ in range(2))
    return [t.to(dt).to(DEV) for t in (q, k, v)]


def i32(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def reference(q, k, v, lens, trees, scale):
    dt = q.dtype
    q, k, v = (t.double().cpu() for t in (q, k, v))
    B, T, H, d = q.shape
    rep = H // k.size(1)
    want, tol = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        seen = ref.tree_seen(lens[b], trees[b])
        n = lens[b] + T
        for h in range(H):
            # what no token of the tree sees is none of the reference's business
            (o, _), (t, _) = ref.attention_row_sets(q[b, :, h], k[b, h // rep, :n], v[b, h // rep, :n], seen, scale, dt)
            want[b, :, h], tol[b, :, h] = o, t
    return want, tol


CASES = [
    (1, 1, 1, 1, 32, 4, [0], "flat"), (1, 1, 8, 8, 64, 64, [37], "flat"), (2, 3, 4, 2, 64, 80, [0, 77], "random"),
    (1, 24, 8, 1, 64, 300, [276], "random"), (3, 33, 4, 4, 80, 200, [1, 96, 127], "chain"),
    (2, 64, 8, 2, 128, 500, [129, 400], "random"), (1, 256, 4, 2, 64, 300, [31], "random"),
    (1, 200, 2, 1, 32, 456, [256], "chain"), (2, 5, 6, 2, 96, 130, [125, 64], "flat"), (1, 7, 4, 1, 256, 150, [128], "random"),
    (1, 40, 8, 2, 256, 170, [130], "random"), (1, 3, 2, 1, 7, 70, [60], "random"), (4, 2, 32, 4, 64, 1100, [1000, 1, 0, 600], "chain"),
    (1, 16, 16, 1, 33, 100, [70], "random"), (1, 1, 32, 4, 128, 3000, [2999], "flat"), (1, 65, 1, 1, 64, 130, [65], "random"),
]


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("B,T,H,G,d,cap,lens,kind", CASES)
def test_tree_attention(B, T, H, G, d, cap, lens, kind, dt):
    from rac_amd import ext
    q, k, v = make(B, T, H, G, d, cap, dt)
    for b in range(B):
        k[b, :, lens[b] + T:] = v[b, :, lens[b] + T:] = float("nan")       # behind the drafts: not read
    trees = [tree(T, kind, b) for b in range(B)]
    got = ext.tree_attention(q, k, v, i32(lens), i32(trees))
    ref.check(got, *reference(q, k, v, lens, trees, 1 / math.sqrt(d)), "out")


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_a_token_does_not_see(dt, bad):
    from rac_amd import ext
    B, T, H, G, d, cap, lens = 1, 40, 4, 2, 64, 400, [333]
    q, k, v = make(B, T, H, G, d, cap, dt)
    trees = [tree(T, "random", 5)]
    want, tol = reference(q, k, v, lens, trees, 1 / math.sqrt(d))
    seen = ref.tree_seen(lens[0], trees[0])
    for t in (6, 39):
        for c in (k, v):
            x, y = k.clone(), v.clone()
            (x if c is k else y)[0, :, lens[0] + t, 3] = bad
            got = ext.tree_attention(q, x, y, i32(lens), i32(trees))
            blind = ~seen[:, lens[0] + t]
            assert int(blind.sum()) > 20
            ref.check(got[:, blind], want[:, blind], tol[:, blind], "out")
            if c is v and bad != bad:
                assert bool(got[0, ~blind][..., 3].isnan().all())


def test_one_token_is_a_decode_step():
    from rac_amd import ext
    H, G, d, cap, n = 8, 2, 64, 600, 515
    q, k, v = make(1, 1, H, G, d, cap, F32)
    got = ext.tree_attention(q, k, v, i32([n]), i32([-1]))
    step = ext.decode_attention(q.view(-1), k[0], v[0], i32([n]), H, ext.attention_scale(d), 24)
    _, tol = reference(q, k, v, [n], [[-1]], 1 / math.sqrt(d))
    # the CORDIC exponential's 24 steps: 2^-20 relative to each probability, twice
    va = v[0].double().cpu().abs().amax(1).repeat_interleave(H // G, 0).view(1, 1, H, d)
    ref.check(got, step.view(1, 1, H, d).double().cpu(), 2 * tol + 2.0 ** -19 * va, "out")


def test_a_chain_is_a_prompt():
    from rac_amd import ext
    T, H, G, d = 100, 4, 2, 64
    q, k, v = make(1, T, H, G, d, T, BF16)
    got = ext.tree_attention(q, k, v, i32([0]), i32(tree(T, "chain")))
    packed = ext.packed_attention(q[0], k[0].transpose(0, 1), v[0].transpose(0, 1), i32([0, T]))
    _, tol = reference(q, k, v, [0], [tree(T, "chain")], 1 / math.sqrt(d))
    ref.check(got[0], packed.double().cpu(), 2 * tol[0], "out")


def test_lengths_outside_the_cache():
    from rac_amd import ext
    q, k, v = make(4, 3, 4, 2, 64, 50, BF16)
    got = ext.tree_attention(q, k, v, i32([-1, 47, 48, 2 ** 31 - 1]), i32([-1, 0, 1]))
    assert bool(got[0].isnan().all()) and bool(got[2].isnan().all()) and bool(got[3].isnan().all())
    want, tol = reference(q[1:2], k[1:2], v[1:2], [47], [[-1, 0, 1]], 1 / 8)
    ref.check(got[1:2], want, tol, "out")


def test_parents_that_do_not_come_before():
    # parents at or past their token, and below -1, count as -1
    from rac_amd import ext
    q, k, v = make(1, 5, 2, 1, 64, 40, F32)
    got = ext.tree_attention(q, k, v, i32([20]), i32([[0, 1000, -7, 3, 2]]))
    assert torch.equal(got, ext.tree_attention(q, k, v, i32([20]), i32([[-1, -1, -1, -1, 2]])))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_strides_and_forms_give_the_same_bits(dt):
    from rac_amd import ext
    B, T, H, G, d, cap, lens = 2, 9, 4, 2, 64, 90, [50, 81]
    q, k, v = make(B, T, H, G, d, cap, dt)
    par = i32(tree(T, "random"))
    a = ext.tree_attention(q, k, v, i32(lens), par)
    by_pos = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]          # [B, cap, G, d] storage
    assert torch.equal(a, ext.tree_attention(q, *by_pos, i32(lens), par.expand(B, T)))
    odd = [torch.full((B, G, cap, d + 1), float("nan"), device=DEV, dtype=dt)[..., 1:] for _ in range(2)]
    for o, t in zip(odd, (k, v)):
        o.copy_(t)
    assert torch.equal(a, ext.tree_attention(q, *odd, i32(lens), par))
    stacked = torch.empty((B, T, H + 3, d), device=DEV, dtype=dt)
    stacked[:, :, :H] = q
    assert torch.equal(a, ext.tree_attention(stacked[:, :, :H], k, v, i32(lens), par))
    for b in range(B):
        one = ext.tree_attention(q[b], k[b], v[b], i32(lens[b:b + 1]), par)
        _, tol = reference(q[b:b + 1], k[b:b + 1], v[b:b + 1], lens[b:b + 1], [tree(T, "random")], 1 / 8)
        ref.check(one, a[b].double().cpu(), 2 * tol[0], "one sequence")       # other splits: another order
    kept = torch.empty_like(q)
    assert ext.tree_attention(q, k, v, i32(lens), par, out=kept) is kept and torch.equal(kept, a)


def test_a_cache_past_32_bits():
    """Positions whose offsets pass 2^31 elements: a cache of 2^25 + 100
    positions of 64 values and one head (4.3 GB in bf16), the drafts at its
    end; keys far smaller than the last ones leave the rest no weight."""
    from rac_amd import ext
    cap, d, T = 2 ** 25 + 100, 64, 3
    k = torch.zeros((1, 1, cap, d), device=DEV, dtype=BF16)
    v = torch.ones((1, 1, cap, d), device=DEV, dtype=BF16)
    q = torch.ones((1, T, 1, d), device=DEV, dtype=BF16)
    n = cap - T
    k[0, 0, n:] = 8.0                         # scores 64 against 0: e^64 > 10^27 times 2^25 keys
    v[0, 0, n:] = torch.tensor([2.0, 4.0, 8.0], device=DEV, dtype=BF16)[:, None]
    got = ext.tree_attention(q, k, v, i32([n]), i32([[-1, -1, 1]]))
    assert torch.equal(got[0, :, 0, 0].float().cpu(), torch.tensor([2.0, 4.0, 6.0]))
    assert bool((got == got[..., :1]).all())


def test_a_recorded_graph_replays_with_new_lengths_and_trees():
    from rac_amd import ext
    B, T, H, G, d, cap = 2, 12, 8, 2, 64, 700
    q, k, v = make(B, T, H, G, d, cap, BF16)
    lens, par = i32([5, 600]), i32([tree(T, "random", s) for s in (1, 2)])
    ext.tree_attention(q, k, v, lens, par)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                        # two graphs of the same call: their own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ext.tree_attention(q, k, v, lens, par))
        graphs.append(g)
    for i in range(4):
        lens.copy_(i32([100 * i, 688 - i]))
        par.copy_(i32([tree(T, "random", 10 + i), tree(T, "chain")]))
        q.mul_(-1.1)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = ext.tree_attention(q, k, v, lens, par)
        assert all(torch.equal(o, want) for o in outs)


def test_two_streams():
    from rac_amd import ext
    sets = [make(2, 20, 8, 2, 128, 900, BF16, seed=s) for s in (1, 2)]
    lens, par = i32([850, 700]), i32(tree(20, "random"))
    want = [ext.tree_attention(*s, lens, par) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = ext.tree_attention(*sets[i], lens, par)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

"""The operators of packed prompts, drafted tokens and given tokens together, as
a program uses them: a decoder that verifies trees of drafted tokens and accepts
a path, and a training step of a small layer over packed sequences."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    import rac_amd
    rac_amd.load()
    yield
    torch.cuda.synchronize()


def decoders(n, cfg, t_max):
    from rac_amd.decoder import RACDecoder
    w = RACDecoder.synthetic_weights(cfg, DEV, seed=1)
    return [RACDecoder(cfg, w, t_max) for _ in range(n)]


def close(a, b):
    # the attention's order of sums and its exponential (24 CORDIC steps, 2^-20)
    # differ from step()'s; the layers' norms keep values near 1
    assert float((a - b).abs().max()) <= 2.0 ** -13 * float(b.abs().max())


@pytest.mark.parametrize("d_model,heads,kv", [(256, 4, 2), (288, 9, 3)])
def test_verify_equals_steps(d_model, heads, kv):
    from rac_amd.decoder import DecoderConfig
    cfg = DecoderConfig(d_model, heads, kv, 512, 2)
    tree, step = decoders(2, cfg, 64)
    gen = torch.Generator().manual_seed(0)
    prompt = torch.randn((20, d_model), generator=gen).to(DEV)
    drafts = torch.randn((7, d_model), generator=gen).to(DEV)
    parents = [-1, 0, 0, 1, -1, 4, 2]
    for dec in (tree, step):
        dec.forward(prompt)
    out = tree.verify(drafts, parents)
    assert tree.length == 20
    for t in range(7):
        path, u = [], t
        while u >= 0:
            path.insert(0, u)
            u = parents[u]
        for u in path:
            y = step.step(drafts[u:u + 1])
        close(out[t:t + 1], y)
        step.length = 20
        step.pos.fill_(20)
    # a path of the tree joins the cache; the next step agrees, eager and recorded
    tree.accept([0, 2, 6])
    for u in (0, 2, 6):
        step.step(drafts[u:u + 1])
    assert tree.length == step.length == 23 and int(tree.pos) == 23
    for a, b in zip(tree.k_cache + tree.v_cache, step.k_cache + step.v_cache):
        close(a[:, :23], b[:, :23])
    nxt = torch.randn((1, d_model), generator=gen).to(DEV)
    want = step.step(nxt)
    close(tree.step(nxt), want)
    tree.capture()
    again = tree.verify(drafts, parents)
    tree.accept([])
    nxt2 = torch.randn((1, d_model), generator=gen).to(DEV)
    close(tree.step(nxt2), step.step(nxt2))
    assert again.shape == drafts.shape


def test_verify_and_accept_refuse():
    from rac_amd.decoder import DecoderConfig
    (dec,) = decoders(1, DecoderConfig(256, 4, 2, 512, 1), 8)
    x = torch.randn((3, 256), device=DEV)
    for parents in ([-1, 0], [-1, 1, 0], [-2, 0, 0], [-1, 0, 3]):
        with pytest.raises(RuntimeError):
            dec.verify(x, parents)
    with pytest.raises(RuntimeError):
        dec.verify(x.double(), [-1, 0, 1])
    with pytest.raises(RuntimeError):
        dec.verify(torch.randn((9, 256), device=DEV), [-1] * 9)
    with pytest.raises(RuntimeError):
        dec.verify(x[:0], [])
    with pytest.raises(RuntimeError):
        dec.accept([0])
    dec.verify(x, [-1, 0, 0])
    for path in ([1], [0, 1, 2], [0, 3], [0, 0], [-1]):
        with pytest.raises(RuntimeError):
            dec.accept(path)
    dec.step(x[:1])
    with pytest.raises(RuntimeError):
        dec.accept([0])                                    # the step dropped the drafts
    dec.verify(x, [-1, 0, 0])
    dec.accept([0, 2])
    assert dec.length == 3
    with pytest.raises(RuntimeError):
        dec.accept([0])


def test_prompts_then_drafts_then_scores():
    """A batch of prompts in one pass, their keys and values into padded
    caches, a tree of drafts over those, its tokens scored: as one sequence
    after the other."""
    from rac_amd import ext
    H, G, d, V, cap = 4, 2, 64, 500, 80
    lens, T = [33, 7, 64], 5
    total = sum(lens)
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((total, h, d), generator=gen).to(DEV) for h in (H, G, G))
    cu = torch.tensor([0, 33, 40, 104], device=DEV, dtype=torch.int32)
    att = ext.packed_attention(q, k, v, cu)
    kc, vc = (torch.zeros((3, G, cap, d), device=DEV) for _ in range(2))
    dq, dk, dv = (torch.randn((3, T, h, d), generator=gen).to(DEV) for h in (H, G, G))
    for b, n in enumerate(lens):
        a = int(cu[b])
        for c, t, u in ((kc, k, dk), (vc, v, dv)):
            c[b, :, :n] = t[a:a + n].transpose(0, 1)
            c[b, :, n:n + T] = u[b].transpose(0, 1)
    par = torch.tensor([-1, 0, 1, 2, 3], device=DEV, dtype=torch.int32)
    out = ext.tree_attention(dq, kc, vc, cu.diff(), par)
    head = torch.randn((V, H * d), generator=gen).to(DEV) / 16
    tok = torch.randint(0, V, (3, T), generator=gen).to(DEV)
    logits = ext.linear_forward(out.flatten(2), head, torch.empty(0), mode=ext.MODE_FAST)
    lp, ent, tv, ti = ext.token_logprobs(logits, tok, top=3)
    for b, n in enumerate(lens):
        a = int(cu[b])
        # a chain of drafts behind a prompt is a longer prompt
        full = [torch.cat([x[a:a + n], y[b]]) for x, y in ((q, dq), (k, dk), (v, dv))]
        whole = ext.packed_attention(*full, torch.tensor([0, n + T], device=DEV, dtype=torch.int32))
        # sums of unit-size values over at most 69 keys and 64 columns
        tol = 200 * 2.0 ** -24 * 4
        assert float((whole[:n] - att[a:a + n]).abs().max()) <= tol
        assert float((whole[n:] - out[b]).abs().max()) <= tol
        p = torch.softmax(logits[b].double(), -1)
        assert float((lp[b].double() - p.gather(-1, tok[b, :, None])[:, 0].log()).abs().max()) <= 2.0 ** -18
        assert torch.equal(ti[b], torch.topk(logits[b], 3).indices)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_a_training_step_over_packed_sequences(dt):
    """Next-token loss with an entropy bonus through a projection, packed
    attention, a head and token_logprobs: the gradients are those of the same
    layer composed of torch operations in 64 bits, within the roundings of its
    stages' types (relative to each gradient's norm)."""
    from rac_amd import rac_torch
    H, G, d, V, dm = 4, 2, 32, 301, 96
    lens = [40, 1, 55]
    total = sum(lens)
    gen = torch.Generator().manual_seed(5)
    x = torch.randn((total, dm), generator=gen).to(dt).to(DEV)
    w = (torch.randn(((H + 2 * G) * d, dm), generator=gen) / math.sqrt(dm)).to(dt).to(DEV).requires_grad_()
    wo = (torch.randn((V, H * d), generator=gen) / math.sqrt(H * d)).to(dt).to(DEV).requires_grad_()
    tok = torch.randint(0, V, (total,), generator=gen).to(DEV)
    tok[[39, 40, 95]] = -1                                  # the last of each sequence has no next token
    cu = torch.tensor([0, 40, 41, 96], device=DEV, dtype=torch.int32)
    qkv = rac_torch.rac_linear(x, w).unflatten(1, (H + 2 * G, d))
    att = rac_torch.rac_packed_attention(qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], cu)
    logits = rac_torch.rac_linear(att.flatten(1), wo)
    lp, ent = rac_torch.rac_token_logprobs(logits, tok)
    loss = -lp.sum() / 93 - 0.01 * ent.mean()
    gw, gwo = torch.autograd.grad(loss, (w, wo))

    x8, w8, wo8 = x.double().cpu(), w.detach().double().cpu().requires_grad_(), wo.detach().double().cpu().requires_grad_()
    qkv = (x8 @ w8.T).unflatten(1, (H + 2 * G, d))
    q, k, v = qkv[:, :H], qkv[:, H:H + G].repeat_interleave(H // G, 1), qkv[:, H + G:].repeat_interleave(H // G, 1)
    i = torch.arange(total)
    doc = torch.repeat_interleave(torch.arange(3), torch.tensor(lens))
    ok = (doc[:, None] == doc) & (i[:, None] >= i)
    s = torch.einsum("thd,uhd->htu", q, k) / math.sqrt(d)
    p = torch.softmax(s.masked_fill(~ok, -math.inf), -1)
    att = torch.einsum("htu,uhd->thd", p, v).flatten(1)
    L = torch.log_softmax(att @ wo8.T, -1)
    t8 = tok.cpu()
    lp8 = torch.where(t8 >= 0, L.gather(1, t8.clamp(min=0)[:, None])[:, 0], torch.zeros(total, dtype=torch.float64))
    loss8 = -lp8.sum() / 93 - 0.01 * -(L.exp() * L).sum(-1).mean()
    gw8, gwo8 = torch.autograd.grad(loss8, (w8, wo8))
    # each of the about ten roundings to the type between loss and weight: half a step of what it rounds
    tol = 10 * torch.finfo(dt).eps / 2 if dt != torch.float32 else 200 * 2.0 ** -24
    for a, b in ((gw, gw8), (gwo, gwo8)):
        assert float((a.double().cpu() - b).norm() / b.norm()) <= tol


def test_a_backward_pass_in_a_graph():
    """Warm passes on the capturing stream, none of whose graphs live on; then
    one recorded forward and backward pass, replayed with new inputs."""
    from rac_amd import rac_torch
    H, G, d = 4, 2, 64
    cu = torch.tensor([0, 50, 130], device=DEV, dtype=torch.int32)
    q, k, v = (torch.randn((130, h, d), device=DEV).requires_grad_() for h in (H, G, G))
    g = torch.randn((130, H, d), device=DEV)

    def step():
        out = rac_torch.rac_packed_attention(q, k, v, cu)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got = step()
    for i in range(3):
        with torch.no_grad():
            q.mul_(0.9)
        g.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))

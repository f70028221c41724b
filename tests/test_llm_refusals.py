"""Arguments that the entry points of rac_llm.h and their Python forms refuse,
before any device work (no GPU needed)."""
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    import rac_amd
    return rac_amd.load()


A = 0x1000                                    # a non-null address that is never read


def packed(lib, **kw):
    a = dict(q=A, k=A, v=A, out=A, lse=A, cu=A, n=1, total=8, H=4, G=2, d=64, st=(256, 64, 128, 64, 128, 64), scale=0.125,
             dtype=0)
    a.update(kw)
    return lib.rac_packed_attention_dev(a["q"], a["k"], a["v"], a["out"], None, a["lse"], a["cu"], a["n"], a["total"], a["H"],
                                        a["G"], a["d"], *a["st"], a["scale"], 1, a["dtype"], None)


def backward(lib, **kw):
    a = dict(bufs=[A] * 12, n=1, total=8, H=4, G=2, d=64, st=(256, 64, 128, 64, 128, 64), scale=0.125, dtype=0)
    a.update(kw)
    return lib.rac_packed_attention_backward_dev(*a["bufs"], a["n"], a["total"], a["H"], a["G"], a["d"], *a["st"],
                                                 a["scale"], 1, a["dtype"], None)


def tree(lib, **kw):
    a = dict(bufs=[A] * 7, B=1, T=4, H=4, G=2, d=64, cap=100, st=[1] * 10, scale=0.125, dtype=0)
    a.update(kw)
    return lib.rac_tree_attention_dev(*a["bufs"], a["B"], a["T"], a["H"], a["G"], a["d"], a["cap"], *a["st"], a["scale"],
                                      a["dtype"], None)


def logp(lib, **kw):
    a = dict(x=A, stride=100, bufs=[A] * 7, rows=2, V=100, top=5, dtype=0)
    a.update(kw)
    return lib.rac_token_logprobs_dev(a["x"], a["stride"], *a["bufs"], a["rows"], a["V"], a["top"], a["dtype"], None)


def logp_backward(lib, **kw):
    a = dict(x=A, stride=100, bufs=[A] * 6, rows=2, V=100, dtype=0)
    a.update(kw)
    return lib.rac_token_logprobs_backward_dev(a["x"], a["stride"], *a["bufs"], a["rows"], a["V"], a["dtype"], None)


NAN, INF = float("nan"), float("inf")
HEADS = [dict(H=0), dict(G=0), dict(H=3), dict(H=-4), dict(G=-2), dict(d=0), dict(d=257), dict(scale=0.0),
         dict(scale=-1.0), dict(scale=NAN), dict(scale=INF), dict(dtype=3), dict(dtype=-1), dict(H=65536, G=1)]


@pytest.mark.parametrize("bad", HEADS)
def test_head_arguments(lib, bad):
    for f in (packed, backward, tree):
        lib.rac_clear_error()
        assert f(lib, **bad) == -2 and lib.rac_last_error() != b""


@pytest.mark.parametrize("bad", [dict(n=-1), dict(total=-1), dict(total=2 ** 30 + 1), dict(n=2 ** 30, H=4),
                                 dict(st=(-1, 64, 128, 64, 128, 64)), dict(st=(256, 64, 128, 64, 128, -64))])
def test_packed_arguments(lib, bad):
    assert packed(lib, **bad) == -2 and backward(lib, **bad) == -2


def test_more_workgroups_than_a_launch_counts(lib):
    assert packed(lib, total=2 ** 28, H=4, G=2) == -2 and packed(lib, n=2 ** 24, H=2, G=1) == -2
    assert backward(lib, total=2 ** 28, H=4, G=2) == -2
    assert tree(lib, B=65535, G=1, H=128, T=256) == -2       # 65535 x 1024 blocks of 32 rows
    assert logp(lib, rows=2 ** 24) == -2 and logp_backward(lib, rows=2 ** 24) == -2


def test_null_buffers(lib):
    for n in ("q", "k", "v", "out", "cu"):
        assert packed(lib, **{n: None}) == -1
    for i in range(12):
        if i != 4:                            # the residual may be absent
            assert backward(lib, bufs=[A] * i + [None] + [A] * (11 - i)) == -1
    for i in range(6):
        assert tree(lib, bufs=[A] * i + [None] + [A] * (6 - i)) == -1
    for i in (0, 1, 2):
        assert logp(lib, bufs=[A] * i + [None] + [A] * (6 - i)) == -1
    for i in (4, 5):                          # top buffers are needed when there are alternatives
        assert logp(lib, bufs=[A] * i + [None] + [A] * (6 - i)) == -1
    assert logp(lib, x=None) == -1 and logp_backward(lib, x=None) == -1
    for bufs in ([None, A, A, A, A, A], [A, None, A, A, A, A], [A, A, None, A, A, A], [A, A, A, None, None, A],
                 [A, A, A, A, A, None]):
        assert logp_backward(lib, bufs=bufs) == -1


@pytest.mark.parametrize("bad", [dict(B=-1), dict(B=40000), dict(T=0), dict(T=257), dict(cap=3), dict(cap=2 ** 31),
                                 dict(st=[-1] + [1] * 9), dict(st=[1] * 9 + [-1])])
def test_tree_arguments(lib, bad):
    assert tree(lib, **bad) == -2


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(rows=2 ** 31), dict(V=0), dict(V=2 ** 31, stride=2 ** 31),
                                 dict(stride=99), dict(dtype=3)])
def test_logit_arguments(lib, bad):
    assert logp(lib, **bad) == -2 and logp_backward(lib, **bad) == -2


def test_top_arguments(lib):
    assert logp(lib, top=-1) == -2 and logp(lib, top=65) == -2 and logp(lib, top=8, V=7, stride=7) == -2


def test_nothing_to_do_is_no_error(lib):
    assert packed(lib, total=0) == 0 and backward(lib, total=0) == 0 and tree(lib, B=0) == 0
    assert logp(lib, rows=0) == 0 and logp_backward(lib, rows=0) == 0


def test_workspace_sizes(lib):
    size = lib.rac_packed_attention_backward_workspace_bytes
    assert size(3, 100, 8, 8, 64) == 6400 and size(1, 0, 8, 8, 64) == 0 and size(1, 100, 8, 3, 64) == 0
    assert size(3, 101, 3, 3, 64) == 4 * 608                # the statistics, up to 16 bytes
    assert size(3, 100, 8, 2, 64) >= 6400
    assert lib.rac_tree_attention_workspace_bytes(0, 4, 4, 2, 64, 100, 0) == 0
    assert lib.rac_tree_attention_workspace_bytes(1, 300, 4, 2, 64, 1000, 0) == 0
    assert lib.rac_token_logprobs_workspace_bytes(0, 100, 0, 0) == 0
    assert lib.rac_token_logprobs_workspace_bytes(4, 32000, 65, 0) == 0


def test_header_compiles_as_c(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "rac_llm.h"\nint main(void){ return rac_token_logprobs_workspace_bytes(0, 1, 0, 0) == 0 ? 0 : 1; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-c", str(src), "-o",
                    str(tmp_path / "t.o")], check=True)


def test_python_refuses_cpu_tensors():
    from rac_amd import ext, rac_torch
    q, kv = torch.randn(5, 4, 64), torch.randn(5, 2, 64)
    cu = torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ext.packed_attention(q, kv, kv, cu)
    with pytest.raises(RuntimeError, match="ROCm device"):
        rac_torch.rac_packed_attention(q, kv, kv, cu)
    c = torch.randn(2, 9, 64)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ext.tree_attention(q, c, c, cu[:1], cu)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ext.token_logprobs(torch.randn(3, 8), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="ROCm device"):
        rac_torch.rac_token_logprobs(torch.randn(3, 8), torch.zeros(3, dtype=torch.int64))


@pytest.mark.gpu
def test_python_refuses_shapes_and_types():
    from rac_amd import ext
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    D = "cuda"
    q, kv = torch.randn(5, 4, 64, device=D), torch.randn(5, 2, 64, device=D)
    cu = torch.tensor([0, 5], dtype=torch.int32, device=D)
    bad = [(q, kv[:4], kv, cu), (q, kv[:4], kv[:4], cu), (q.half(), kv, kv, cu), (q.double(), kv.double(), kv.double(), cu),
           (q, kv, kv, cu.long()), (q, kv, kv, cu.cpu()), (q, kv, kv, cu[:0]), (q, kv, kv, cu.view(1, 2)),
           (q[:, :3], kv, kv, cu), (q[:, :, :32], kv, kv, cu), (q[0], kv[0], kv[0], cu),
           (torch.randn(5, 4, 300, device=D), torch.randn(5, 2, 300, device=D), torch.randn(5, 2, 300, device=D), cu),
           (q[:, :0], kv[:, :0], kv[:, :0], cu)]
    for args in bad:
        with pytest.raises(RuntimeError):
            ext.packed_attention(*args)
    with pytest.raises(RuntimeError):
        ext.packed_attention(q, kv, kv, cu, scale=0.0)
    for out in (q[:4].clone(), q.half(), q.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(RuntimeError):
            ext.packed_attention(q, kv, kv, cu, out=out)
    out, lse = ext.packed_attention(q, kv, kv, cu, return_lse=True)
    for g, o, l in ((q[:4], out, lse), (q.half(), out, lse), (q, out, lse[:2]), (q, out, lse.double()), (q, out[:4], lse)):
        with pytest.raises(RuntimeError):
            ext.packed_attention_backward(g, q, kv, kv, o, l, cu)
    t, c = torch.randn(1, 3, 4, 64, device=D), torch.randn(1, 2, 9, 64, device=D)
    n, par = cu[1:], torch.tensor([-1, 0, 1], dtype=torch.int32, device=D)
    bad = [(t, c, c[:, :, :8], n, par), (t, c[:, :1].expand(-1, 3, -1, -1), c[:, :1].expand(-1, 3, -1, -1), n, par),
           (t.half(), c, c, n, par), (t, c, c, n.long(), par), (t, c, c, cu, par), (t, c, c, n, par[:2]),
           (t, c, c, n, par.long()), (t, c, c, n, par.cpu()), (t, c[..., :32], c[..., :32], n, par), (t[:, :0], c, c, n, par[:0]),
           (t.expand(2, -1, -1, -1), c, c, cu, par), (t, c[:, :, :2], c[:, :, :2], n, par)]
    for args in bad:
        with pytest.raises(RuntimeError):
            ext.tree_attention(*args)
    x, tok = torch.randn(3, 8, device=D), torch.zeros(3, dtype=torch.int64, device=D)
    for args in ((x, tok[:2]), (x, tok.float()), (x.double(), tok), (x, tok.cpu()), (x[:, :0], tok), (x, tok, 9), (x, tok, -1)):
        with pytest.raises(RuntimeError):
            ext.token_logprobs(*args)
    lp, ent, lse = ext.token_logprobs(x, tok, return_lse=True)
    for args in ((lse[:2], ent, lp, None), (lse, None, lp, None), (lse, ent, lp.double(), None)):
        with pytest.raises(RuntimeError):
            ext.token_logprobs_backward(x, tok, *args)
    assert bool((ext.token_logprobs_backward(x, tok, lse, ent, None, None) == 0).all())


@pytest.mark.gpu
def test_an_output_within_an_input():
    from rac_amd import ext
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    D = "cuda"
    flat = torch.randn(5, 12, 64, device=D)
    q, k, v = flat[:, :4], flat[:, 4:8], flat[:, 8:]
    cu = torch.tensor([0, 5], dtype=torch.int32, device=D)
    plain = ext.packed_attention(q, k, v, cu)
    for t in (q.contiguous(), v.contiguous()):
        with pytest.raises(RuntimeError, match="share"):
            ext.packed_attention(t, k, t, cu, out=t)
    with pytest.raises(RuntimeError, match="share"):
        ext.packed_attention(q, k, v, cu, out=flat.view(-1)[-5 * 256:].view(5, 4, 64))
    both = torch.empty(2 * 5 * 256, device=D)                 # neighbours in one buffer are no overlap
    own = both[:1280].view(5, 4, 64).copy_(q)
    out = ext.packed_attention(own, k, v, cu, out=both[1280:].view(5, 4, 64))
    assert torch.equal(out, plain)
    t, c = torch.randn(1, 3, 4, 64, device=D), torch.randn(1, 4, 9, 64, device=D)
    par = torch.tensor([-1, 0, 1], dtype=torch.int32, device=D)
    for o in (t, c.view(-1)[:768].view(1, 3, 4, 64)):
        with pytest.raises(RuntimeError, match="share"):
            ext.tree_attention(t, c, c, cu[1:], par, out=o)

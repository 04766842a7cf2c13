"""Calls of the operators that their documentation allows, or that they have to refuse, beside the sizes of test_gpu_ops."""
import numpy as np
import pytest
import torch

from test_gpu_ops import _archive, _check, _check_project, _index, _inputs, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _library(gpu):
    return gpu


def test_tangents_are_refused_beside_a_scale_and_in_a_gradient():
    from torch.autograd import forward_ad

    from lmz_b200 import adapters, embed
    x, w, a, b, scales = _inputs(6, 64, 96, 8, 3, torch.bfloat16)
    index, dy = torch.zeros(6, dtype=torch.int32, device="cuda"), _randn(1, (6, 96), torch.bfloat16)
    table, ids = _randn(2, (5, 8), torch.float32).requires_grad_(True), torch.zeros(3, dtype=torch.int64, device="cuda")
    y, e = adapters.project(x.requires_grad_(True), w, a, b, index, scale=scales), embed.lookup(table, ids)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="tangent"):
            adapters.project(x, w, a, b, index, scale=forward_ad.make_dual(scales, torch.ones_like(scales)))
        with pytest.raises(NotImplementedError, match="tangent"):
            torch.autograd.grad(y, x, forward_ad.make_dual(dy, dy.clone()))
        with pytest.raises(NotImplementedError, match="tangent"):
            torch.autograd.grad(e, table, forward_ad.make_dual(e.detach(), e.detach().clone()))
        assert adapters.project(x, w, a, b, index, scale=scales).shape == (6, 96)


def test_one_row_of_an_archive_by_its_number():
    """Row numbers of any shape: of none, too."""
    from lmz_b200 import archive, decode
    table = _randn(71, (900, 250), torch.bfloat16, 0.02)
    ar = archive.Archive(_archive({"norm": _randn(70, (33,), torch.bfloat16), "emb": table}, mapped=True))
    for row in (7, np.int64(7), np.array(7, dtype=np.uint8), torch.tensor(7)):
        got = decode.decode_rows(ar, "emb", row)
        assert got.shape == (250,) and torch.equal(got, table[7])
    assert decode.decode_rows(ar, "emb", torch.tensor([[899], [0]])).shape == (2, 1, 250)
    with pytest.raises(IndexError):
        decode.decode_rows(ar, "emb", 900)


@pytest.mark.parametrize("n", [3, 33])
def test_rows_gradient_of_the_widest_rows(n):
    """2^24 - 1 elements of 16 bits, which move one at a time: more slices of a row than a grid has along y."""
    from lmz_b200 import embed
    dim = (1 << 24) - 1
    table = torch.zeros((2, dim), dtype=torch.float16, device="cuda").requires_grad_(True)
    ids = torch.ones(n, dtype=torch.int64, device="cuda")
    ids[1] = 0
    dy = torch.randint(-8, 9, (n, dim), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda", dtype=torch.int8).to(torch.float16)
    (got,) = torch.autograd.grad(embed.lookup(table, ids), table, dy)
    assert torch.equal(got[0], dy[1])
    want = torch.zeros(dim, device="cuda")                 # (whole numbers up to 33 * 8: exact in F16 too)
    for t in range(n):
        if t != 1:
            want += dy[t]
    assert torch.equal(got[1].float(), want)


def test_a_merge_in_place_is_noticed():
    """As any operator of torch that writes to a tensor which a gradient still needs; and a leaf is not written to."""
    from lmz_b200 import adapters
    w, a, b = _randn(50, (16, 24), torch.bfloat16), _randn(51, (4, 24), torch.bfloat16), _randn(52, (16, 4), torch.bfloat16)
    v = torch.ones_like(w).requires_grad_(True)
    y = (v * w).sum()
    adapters.merge(w, a, b, out=torch.empty_like(w))       # (leaves w alone)
    (g,) = torch.autograd.grad(y, v, retain_graph=True)
    assert torch.equal(g, w)
    adapters.merge(w, a, b, out=w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    leaf = torch.empty_like(w).requires_grad_(True)
    with pytest.raises(ValueError, match="gradient"):
        adapters.merge(w, a, b, out=leaf)
    with torch.no_grad():
        assert adapters.merge(w, a, b, out=leaf) is leaf
    with torch.inference_mode():
        out = torch.empty_like(w)
        assert torch.equal(adapters.merge(w, a, b, out=out), leaf)


def test_merged_tensors_are_checked(monkeypatch):
    from lmz_b200 import adapters, archive, decode, gpu
    w, a, b = _randn(50, (32, 64), torch.bfloat16), _randn(51, (4, 64), torch.bfloat16), _randn(52, (32, 4), torch.bfloat16)
    ar, tuned = archive.Archive(_archive({"p.weight": w})), archive.Archive(_archive({"p.lora_A.weight": a, "p.lora_B.weight": b}))
    (got,) = decode.decode_tensors(ar, ["p.weight"], adapter=tuned).values()
    assert torch.equal(got, adapters.merge(w, a, b))
    monkeypatch.setattr(gpu.library(), "lmz_gpu_ops_gave_up", lambda: 1)      # a merge whose wait has run out
    with pytest.raises(RuntimeError, match="gave up"):
        decode.decode_tensors(ar, ["p.weight"], adapter=tuned)
    (plain,) = decode.decode_tensors(ar, ["p.weight"]).values()
    assert torch.equal(plain, w)


@pytest.mark.parametrize("tokens", [1, 64, 700])
@pytest.mark.parametrize("n", [2, 5])
def test_without_an_index_only_the_first_adapter_has_gradients(tokens, n):
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(tokens, 64, 136, 8, n, torch.bfloat16)
    dy = _randn(40, (tokens, 136), torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = adapters.project(x, w, a, b, scale=scales)
    grads = torch.autograd.grad(y, leaves, dy)
    _check_project(x, w, a, b, scales, None, y.detach(), dy, grads)
    zeros = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    for g, h in zip(grads, torch.autograd.grad(adapters.project(x, w, a, b, zeros, scale=scales), leaves, dy)):
        assert torch.equal(g, h)
    assert (grads[1][1:] == 0).all() and (grads[2][1:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_graph_that_is_kept_gives_the_same_gradients_again(dtype):
    """What the gradients need of the forward pass is not used up by them."""
    from lmz_b200 import adapters
    for kind, tokens in (("runs", 300), ("mixed", 1500)):
        x, w, a, b, scales = _inputs(tokens, 392, 400, 64, 4, dtype)
        index, dy = _index(kind, tokens, 4), _randn(1, (tokens, 400), dtype)
        leaves = [t.requires_grad_(True) for t in (x, a, b)]
        y = adapters.project(x, w, a, b, index, scale=scales)
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        torch.autograd.grad(y, leaves, _randn(2, (tokens, 400), dtype, 100.0), retain_graph=True)
        for g, h in zip(first, torch.autograd.grad(y, leaves, dy)):
            assert torch.equal(g, h)


def test_f16_captured_for_any_order_of_the_tokens():
    """Which adapters' factors are taken as parts shows only on the device, too."""
    from lmz_b200 import adapters
    dtype = torch.float16
    for tokens, n in ((1500, 6), (200, 40), (1, 5)):
        x, w, a, b, scales = _inputs(tokens, 392, 400, 128, n, dtype)
        dy, index = _randn(62, (tokens, 400), dtype), _index("runs", tokens, n).long()

        def step():
            leaves = [t.detach().requires_grad_(True) for t in (x, a, b)]
            y = adapters.project(*leaves[:1], w, *leaves[1:], index, scale=scales)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

        step()
        torch.cuda.synchronize()
        graphs, outs = [], []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(step())
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in graphs]
        for kind in ("mixed", "runs", "short", "far", "off"):
            index.copy_(_index(kind, tokens, n, seed=64))
            for t in outs[0] + outs[1]:
                t.fill_(7)
            torch.cuda.synchronize()
            for graph, stream in zip(graphs, streams):     # (side by side: their workspaces are their own)
                with torch.cuda.stream(stream):
                    graph.replay()
            torch.cuda.synchronize()
            want = step()
            for out in outs:
                for g, v in zip(out, want):
                    assert torch.equal(g, v)
            _check_project(x, w, a, b, scales, index, want[0], dy, want[1:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_threads_with_streams_of_their_own(dtype):
    import threading

    from lmz_b200 import adapters, embed
    jobs, want, got = [], [], [None] * 4
    for i, (tokens, kind) in enumerate(((1, "runs"), (700, "mixed"), (300, "runs"), (64, "far"))):
        x, w, a, b, scales = _inputs(tokens, 256, 264, 16, 5, dtype, seed=30 + 10 * i)
        jobs.append((x, w, a, b, scales, _index(kind, tokens, 5), _randn(i, (tokens, 264), dtype)))

    def work(x, w, a, b, scales, index, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, a, b)]
        y = adapters.project(*leaves[:1], w, *leaves[1:], index, scale=scales)
        e = embed.lookup(w, index.clamp(0, 200))
        return (y.detach(), *torch.autograd.grad(y, leaves, dy), e, adapters.merge(w, a[0], b[0]))

    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = work(*jobs[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for w_, g_ in zip(want, got):
        for p, q in zip(w_, g_):
            assert torch.equal(p, q)
    adapters.check()


@pytest.mark.parametrize("kind", ["runs", "mixed"])
def test_project_beyond_32_bits(kind):
    """More than 2^32 elements of y and dy: the last tokens, and the factors' gradients, which sum over all of them."""
    from lmz_b200 import adapters
    tokens, inp, out, rank, n, dtype = 270_000, 64, 16_384, 8, 3, torch.bfloat16
    x, w, a, b, scales = _inputs(tokens, inp, out, rank, n, dtype)
    index = _index(kind, tokens, n)
    dy = torch.empty((tokens, out), dtype=dtype, device="cuda")
    for t0 in range(0, tokens, 30_000):
        dy[t0:t0 + 30_000] = _randn(t0, (30_000, out), dtype)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = adapters.project(x, w, a, b, index, scale=scales)
    dx, da, db = torch.autograd.grad(y, leaves, dy)
    last = slice(tokens - 300, tokens)
    wd, ad, bd = (t.detach().double() for t in (w, a, b))
    # (the bounds of _check_project for y and dx of the last tokens)
    for got, up, first, second, terms in ((y[last], x[last], ad, bd.transpose(1, 2), inp), (dx[last], dy[last], bd.transpose(1, 2), ad, out)):
        u = up.detach().double()
        want, size = (u @ wd.t(), u.abs() @ wd.abs().t()) if terms == inp else (u @ wd, u.abs() @ wd.abs())
        carried = torch.zeros_like(want)
        for i in range(n):
            at = torch.nonzero(index[last] == i).flatten()
            h, hs = float(scales[i]) * (u[at] @ first[i].t()), float(scales[i]) * (u[at].abs() @ first[i].abs().t())
            want[at] += h @ second[i]
            size[at] += hs @ second[i].abs()
            carried[at] = 2 ** -16 * (h.abs() @ second[i].abs())
        _check(got.detach(), want, size, carried, terms + rank + 8, "the last tokens")
    da_, das, db_, dbs = torch.zeros_like(ad), torch.zeros_like(ad), torch.zeros_like(bd), torch.zeros_like(bd)
    for t0 in range(0, tokens, 10_000):
        t1 = t0 + 10_000
        for i in range(n):
            at = t0 + torch.nonzero(index[t0:t1] == i).flatten()
            s, xd, dyd = float(scales[i]), x[at].detach().double(), dy[at].double()
            g, gs, h, hs = s * (dyd @ bd[i]), s * (dyd.abs() @ bd[i].abs()), s * (xd @ ad[i].t()), s * (xd.abs() @ ad[i].abs().t())
            da_[i] += g.t() @ xd
            das[i] += gs.t() @ xd.abs()
            db_[i] += dyd.t() @ h
            dbs[i] += dyd.abs().t() @ hs
    # thin products off by 2^-16 of their magnitude at most: less than 2^-16 of these sums
    _check(da, da_, das, 2 ** -16 * das, 1000, "da")
    _check(db, db_, dbs, 2 ** -16 * dbs, 1000, "db")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_stack_of_adapters_beyond_32_bits(dtype):
    from lmz_b200 import adapters
    tokens, inp, out, rank, n = 40, 16_384, 72, 64, 4200
    a = torch.zeros((n, rank, inp), dtype=dtype, device="cuda")
    used = torch.tensor([0, n - 1, n - 2, 4100], device="cuda")
    a[used] = _randn(1, (4, rank, inp), dtype, 0.01)
    b = torch.zeros((n, out, rank), dtype=dtype, device="cuda")
    b[used] = _randn(2, (4, out, rank), dtype, 0.3)
    x, w = _randn(3, (tokens, inp), dtype), _randn(4, (out, inp), dtype, 0.01)
    for pick in (torch.arange(tokens, device="cuda") // 16, torch.arange(tokens, device="cuda") % 4):
        leaf = x.detach().requires_grad_(True)
        y = adapters.project(leaf, w, a, b, used[pick])
        (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
        few = x.detach().requires_grad_(True)
        z = adapters.project(few, w, a[used], b[used], pick)
        (ez,) = torch.autograd.grad(z, few, torch.ones_like(z))
        assert torch.equal(y, z) and torch.equal(dx, ez)

"""Embedding rows and their gradient against plain 64-bit sums.

Tolerances: a rounding to type t is off by at most eps(t)/2 of the value.  Lookup: the scale's rounding to fp32 and the fp32
product, 2^-24 each, then the rounding to t.  Gradient: a sum of n fp32 terms in any order is off by at most
(n - 1) 2^-24 / (1 - (n - 1) 2^-24) of the sum of their magnitudes; then scale, product and rounding as above, and with accumulate
one more fp32 addition."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(t, v, d, dtype, spread="uniform", masked=0.0, index=torch.int64, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if spread == "one":
        idx = torch.full((t,), v // 2, device="cuda")
    elif spread == "runs":
        ray = torch.cumsum((torch.rand(t, generator=gen, device="cuda") < 0.05).long(), 0)
        idx = torch.randint(0, v, (t + 1,), generator=gen, device="cuda")[ray] if t else ray
    else:
        idx = torch.randint(0, v, (t,), generator=gen, device="cuda")
    if masked:
        idx = torch.where(torch.rand(t, generator=gen, device="cuda") < masked, torch.full_like(idx, -1), idx)
    return idx.to(index), torch.randn((t, d), generator=gen, device="cuda").to(dtype), torch.randn((v, d), generator=gen, device="cuda").to(dtype)


def plain_gradient(grad, idx, v, padding=None):
    """(sums, sums of magnitudes, terms of every row) in 64 bits."""
    idx = idx.reshape(-1).long()
    grad = grad.reshape(idx.numel(), grad.shape[-1]).double()
    keep = (idx >= 0) & (idx < v)
    if padding is not None:
        keep &= idx != padding
    idx, grad = idx[keep], grad[keep]
    out = torch.zeros((v, grad.shape[1]), dtype=torch.float64, device=grad.device)
    return out.index_add(0, idx, grad), out.index_add(0, idx, grad.abs()), torch.bincount(idx, minlength=v).double()[:, None]


def check_gradient(got, grad, idx, v, scale=1.0, padding=None, old=None):
    ref, size, n = plain_gradient(grad, idx, v, padding)
    ref, size = ref * scale, size * abs(scale)
    total = ref if old is None else ref + old.double()
    tol = (n * U * 1.01 + 2 * U) * size + half_step(got.dtype) * total.abs() * (1 + 1e-6)
    if old is not None:
        tol = tol + U * (total.abs() + size)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # below the smallest normal number the steps are 2^-24
    err = (got.double() - total).abs()
    assert bool((err <= tol).all()), f"worst {float((err - tol).max()):.3e}"
    if old is None:
        assert bool((got[(n == 0)[:, 0]] == 0).all())
    else:
        assert torch.equal(got[(n == 0)[:, 0]], old[(n == 0)[:, 0]])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,v,d", [(1, 1, 1), (1, 11500, 48), (7, 3, 5), (333, 11500, 48), (1000, 50, 771), (129, 17, 1024), (70001, 600, 48)])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_lookup(dtype, t, v, d, index):
    from landmark_b200.embedding import embedding

    idx, _, w = make(t, v, d, dtype, masked=0.2, index=index)
    for scale in (1.0, math.sqrt(d), -0.37):
        got = embedding(idx, w, scale=scale)
        ref = torch.where((idx >= 0)[:, None], w[idx.long().clamp(min=0)].double() * scale, 0.0)
        tol = (2 * U + half_step(dtype) * (1 + 1e-6)) * ref.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert got.dtype == dtype and got.shape == (t, d)
        assert bool(((got.double() - ref).abs() <= tol).all())
        if scale == 1.0:
            assert torch.equal(got, torch.where((idx >= 0)[:, None], w[idx.long().clamp(min=0)], torch.zeros_like(got)))


def test_lookup_shapes_strides_and_wrong_indices():
    from landmark_b200.embedding import embedding

    idx, _, w = make(60, 40, 96, torch.float32)
    square = idx.view(6, 10)
    assert torch.equal(embedding(square.t(), w), w[square.t()])
    assert torch.equal(embedding(idx[::3], w), w[idx[::3]])
    assert torch.equal(embedding(idx[3], w), w[idx[3]])
    assert torch.equal(embedding(idx, w[:, 7:30]), w[:, 7:30][idx])          # rows of a wider table, not 16-byte aligned
    assert torch.equal(embedding(idx, w[:, 8:40]), w[:, 8:40][idx])          # aligned
    assert torch.equal(embedding(idx % 20, w[::2]), w[::2][idx % 20])
    assert torch.equal(embedding(idx % 20, w[1::2].t().contiguous().t()), w[1::2][idx % 20])
    assert torch.equal(embedding(idx, w[:1].expand(40, 96)), w[:1].expand(60, 96))
    assert embedding(idx[:0], w).shape == (0, 96)
    wrong = torch.tensor([0, 40, -1, 39, 2 ** 40, -2 ** 40], device="cuda")
    got = embedding(wrong, w)
    assert torch.equal(got[[0, 3]], w[[0, 39]]) and bool((got[[2, 5]] == 0).all()) and bool(got[[1, 4]].isnan().all())


def test_masked_places_do_not_read_and_bad_values_stay_in_their_rows():
    from landmark_b200.embedding import embedding, embedding_backward

    idx, g, w = make(5000, 300, 48, torch.float32, masked=0.3)
    g[idx < 0] = float("nan")
    check_gradient(embedding_backward(g, idx, 300), g.nan_to_num(), idx, 300)
    g = g.nan_to_num()
    t = int((idx >= 0).nonzero()[7])
    g[t, 5] = float("inf")
    got = embedding_backward(g, idx, 300)
    assert float(got[int(idx[t]), 5]) == float("inf") and int((~got.isfinite()).sum()) == 1
    w[3] = float("nan")
    assert bool((embedding(idx, w).isnan().any(1) == (idx == 3)).all())


SIZES = [(0, 5, 48), (1, 1, 1), (1, 11500, 48), (33, 3, 5), (4095, 700, 48), (4096, 700, 48), (4097, 700, 48), (12289, 1, 3), (20000, 70001, 12),
         (5003, 5021, 771), (3000, 9000, 1028), (300, 40, 2056), (100003, 11500, 48)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,v,d", SIZES)
@pytest.mark.parametrize("spread", ["uniform", "runs", "one"])
def test_gradient(dtype, t, v, d, spread):
    from landmark_b200.embedding import embedding_backward

    idx, g, _ = make(t, v, d, dtype, spread, masked=0.1)
    got = embedding_backward(g, idx, v)
    assert got.dtype == dtype and got.shape == (v, d)
    check_gradient(got, g, idx, v)
    assert torch.equal(got, embedding_backward(g, idx.to(torch.int32), v))  # and the same bits again


# where the way of sorting, the number of blocks or the number of passes changes, and one beside it
BORDERS = [(n + k, v, d) for n, v, d in ((672, 11500, 48), (1024, 11500, 48), (2048, 11500, 48), (8192, 511, 4), (16384, 512, 4), (32768, 262143, 4), (65536, 262144, 4),
                                         (2048 * 40, 3, 1)) for k in (0, 1)]


@pytest.mark.parametrize("t,v,d", BORDERS)
@pytest.mark.parametrize("spread", ["uniform", "runs", "one"])
def test_gradient_at_borders(t, v, d, spread):
    from landmark_b200.embedding import embedding_backward

    idx, g, _ = make(t, v, d, torch.float32, spread, masked=0.02, seed=1)
    idx[:: max(1, t // 7)] = v - 1  # the last row is named
    got = embedding_backward(g, idx, v)
    check_gradient(got, g, idx, v)
    assert torch.equal(got, embedding_backward(g, idx, v))


def test_many_tokens():
    """Twenty million tokens: whole numbers, so that every sum is exact whatever its order."""
    from landmark_b200.embedding import embedding_backward

    t, v = 20_000_003, 11500
    g = torch.ones((t, 4), device="cuda")
    for idx in (torch.arange(t, device="cuda") % v, torch.arange(t, device="cuda") // 1_000_000, torch.zeros(t, dtype=torch.int64, device="cuda")):
        got = embedding_backward(g, idx, v)
        assert torch.equal(got, torch.bincount(idx, minlength=v).float()[:, None].expand(v, 4)) or float(got.max()) >= 2 ** 24
        if float(got.max()) >= 2 ** 24:  # one row: past the whole numbers that fp32 counts singly
            n = torch.bincount(idx, minlength=v).double()[:, None]
            assert bool(((got.double() - n).abs() <= n * 1000 * U).all())


@pytest.mark.parametrize("d", [1, 2, 3, 5, 255, 257, 1023, 1025, 4100])
def test_gradient_of_odd_widths(d):
    from landmark_b200.embedding import embedding_backward

    for dtype, out in ((torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)):
        for t in (700, 3000):
            idx, g, _ = make(t, 90, d, dtype, "runs", masked=0.1)
            check_gradient(embedding_backward(g, idx, 90, dtype=out), g, idx, 90)
            old = torch.randn((90, d), device="cuda").to(out)
            check_gradient(embedding_backward(g, idx, 90, scale=2.0, out=old.clone(), accumulate=True), g, idx, 90, 2.0, old=old)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_types_and_accumulation(dtype, out):
    from landmark_b200.embedding import embedding_backward

    for t, v, d in [(6001, 400, 48), (900, 400, 51)]:
        idx, g, _ = make(t, v, d, dtype, "runs", masked=0.05)
        check_gradient(embedding_backward(g, idx, v, scale=0.25, dtype=out), g, idx, v, 0.25)
        old = torch.randn((v, d), device="cuda").to(out)
        into = old.clone()
        got = embedding_backward(g, idx, v, scale=-3.7, out=into, accumulate=True)
        assert got.data_ptr() == into.data_ptr()
        check_gradient(got, g, idx, v, -3.7, old=old)
        check_gradient(embedding_backward(g, idx, v, padding_idx=int(idx.max()), dtype=out), g, idx, v, padding=int(idx.max()))


def test_gradient_masks_that_leave_nothing():
    from landmark_b200.embedding import embedding_backward

    for t in (1, 50, 9000):
        g = torch.full((t, 48), float("nan"), device="cuda")
        idx = torch.full((t,), -1, device="cuda")
        assert bool((embedding_backward(g, idx, 77) == 0).all())
        assert bool((embedding_backward(g, idx + 78, 77) == 0).all())  # past the table
        assert bool((embedding_backward(g, idx + 4, 77, padding_idx=3) == 0).all())
        old = torch.randn((77, 48), device="cuda")
        assert torch.equal(embedding_backward(g, idx, 77, out=old.clone(), accumulate=True), old)


def test_gradient_strides():
    from landmark_b200.embedding import embedding_backward

    idx, g, _ = make(3000, 200, 96, torch.float32)
    for cut in (g[:, :48], g[:, 3:40], g[:, 8:9]):
        check_gradient(embedding_backward(cut, idx, 200), cut, idx, 200)
    check_gradient(embedding_backward(g.t().contiguous().t(), idx, 200), g, idx, 200)
    check_gradient(embedding_backward(g[:1].expand(3000, 96), idx, 200), g[:1].expand(3000, 96), idx, 200)
    wide = torch.full((200, 100), 7.0, device="cuda")
    for lo in (0, 1, 4):
        wide.fill_(7.0)
        embedding_backward(g, idx, 200, out=wide[:, lo:lo + 96])
        check_gradient(wide[:, lo:lo + 96], g, idx, 200)
        assert bool((wide[:, :lo] == 7).all()) and bool((wide[:, lo + 96:] == 7).all())  # the columns beside it stay
    check_gradient(embedding_backward(g.view(30, 100, 96), idx.view(30, 100), 200), g, idx, 200)


def test_gradients_of_each_other():
    from landmark_b200.embedding import embedding, embedding_backward

    idx, g, w = make(500, 40, 24, torch.float32, masked=0.2)
    w.requires_grad_(True)
    loss = (embedding(idx, w, scale=0.5, padding_idx=7) * g).sum()
    loss.backward()
    check_gradient(w.grad, g, idx, 40, 0.5, padding=7)
    # differences: the loss is linear in w, one value of w at a time
    for row, col in ((int(idx.max()), 3), (12, 20), (7, 0)):
        delta = torch.zeros_like(w)
        delta[row, col] = 1.0
        diff = (torch.where((idx >= 0)[:, None], delta[idx.clamp(min=0)].double() * 0.5, 0.0) * g.double()).sum()
        want = 0.0 if row == 7 else float(diff)
        assert abs(float(w.grad[row, col]) - want) <= 40 * U * 500
    # the sum's own gradient is the lookup, and that one's the sum
    g2 = g.clone().requires_grad_(True)
    up = torch.randn((40, 24), device="cuda", requires_grad=True)
    (embedding_backward(g2, idx, 40, scale=0.5, padding_idx=7) * up).sum().backward(create_graph=True)
    want = torch.where(((idx >= 0) & (idx != 7))[:, None], up[idx.clamp(min=0)] * 0.5, torch.zeros_like(g))
    assert torch.equal(g2.grad, want)
    (again,) = torch.autograd.grad(g2.grad.square().sum(), up)
    ref = torch.autograd.grad(want.square().sum(), up)[0]
    assert torch.allclose(again, ref, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("t", [300, 6000, 70000])
def test_streams_and_graphs(t):
    from landmark_b200.embedding import embedding, embedding_backward

    idx, g, w = make(t, 500, 48, torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = embedding(idx, w), embedding_backward(g, idx, 500)
    torch.cuda.current_stream().wait_stream(side)
    want_a, want_b = embedding(idx, w), embedding_backward(g, idx, 500)
    assert torch.equal(a, want_a) and torch.equal(b, want_b)
    graphs = []
    for k in range(2):  # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = embedding(idx, w, scale=k + 1.0), embedding_backward(g, idx, 500, scale=k + 1.0)
        graphs.append((graph, out))
    idx2, g2, w2 = make(t, 500, 48, torch.float32, "runs", masked=0.1, seed=5)
    idx.copy_(idx2), g.copy_(g2), w.copy_(w2)
    for graph, _ in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    for k, (_, (a, b)) in enumerate(graphs):
        assert torch.equal(a, embedding(idx, w, scale=k + 1.0)) and torch.equal(b, embedding_backward(g, idx, 500, scale=k + 1.0))


def test_two_threads_at_once():
    """Calls of host threads with streams of their own do not disturb each other."""
    import threading

    from landmark_b200.embedding import embedding, embedding_backward

    jobs = [make(n, 700, 48, torch.float32, "runs", seed=n) for n in (900, 5000, 80000)]
    want = [(embedding(i, w), embedding_backward(g, i, 700)) for i, g, w in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        i, g, w = jobs[k]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not (torch.equal(embedding(i, w), want[k][0]) and torch.equal(embedding_backward(g, i, 700), want[k][1])):
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_backward_pass_under_capture_is_refused():
    from landmark_b200.embedding import embedding

    idx, g, w = make(100, 50, 48, torch.float32)
    w.requires_grad_(True)
    eager = (embedding(idx, w) * g).sum()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            (embedding(idx, w) * g).sum().backward()
    torch.cuda.synchronize()
    w.grad = None
    eager.backward()  # the context and the eager graph are as they were
    check_gradient(w.grad, g, idx, 50)


def test_offsets_past_32_bits():
    from landmark_b200.embedding import embedding, embedding_backward

    v, d = 1_100_000, 2048  # 2.25e9 values
    w = torch.zeros((v, d), dtype=torch.bfloat16, device="cuda")
    w[-3:] = torch.randn((3, d), device="cuda").bfloat16()
    idx = torch.tensor([v - 1, 0, v - 3, v - 1], device="cuda")
    assert torch.equal(embedding(idx, w), w[idx])
    g = torch.randn((4, d), device="cuda").bfloat16()
    w.fill_(1.0)
    embedding_backward(g, idx, v, out=w)
    got = w[[v - 1, 0, v - 3]].double()
    ref = torch.stack([g[0].double() + g[3].double(), g[1].double(), g[2].double()])
    assert bool(((got - ref).abs() <= 2.0 ** -8 * ref.abs() * 1.01 + 4 * U * 8).all())
    assert int(w[1:v - 3].count_nonzero()) == 0 and int(w[v - 2].count_nonzero()) == 0
    del w
    t = 1_100_000
    g = torch.ones((t, d), dtype=torch.bfloat16, device="cuda")
    idx = torch.arange(t, device="cuda") % 1000
    assert bool((embedding_backward(g, idx, 1000, dtype=torch.float32) == 1100).all())  # whole numbers: exact in fp32


@pytest.mark.parametrize("t", [2049, 2179, 2200, 2211, 2310, 4950, 9009, 33000, 65536, 65537, 100000, 1500007])
@pytest.mark.parametrize("v,d,dtype", [(0, 1, torch.float32), (0, 48, torch.float32), (0, 5, torch.float16), (131072, 48, torch.bfloat16)])
def test_every_row_is_named_once(t, v, d, dtype):
    """No token is masked and no row has two: each row's gradient is its token's row, bit for bit, in every call, and no row that is
    named is taken for one that is not (its zeros would be written beside its sum)."""
    from landmark_b200.embedding import embedding_backward

    gen = torch.Generator(device="cuda").manual_seed(t)
    rows = max(t, v)
    g = torch.randn((t, d), generator=gen, device="cuda").to(dtype)
    out = torch.empty((rows, d), dtype=dtype, device="cuda")
    for idx in (torch.arange(t, device="cuda"), torch.randperm(rows, generator=gen, device="cuda")[:t], torch.arange(rows - t, rows, device="cuda").flip(0)):
        want = torch.zeros_like(out)
        want[idx] = g
        for _ in range(5):
            assert torch.equal(embedding_backward(g, idx, rows, out=out.fill_(float("nan"))), want)


@pytest.mark.parametrize("t", [2200, 2310, 4950, 9009])
def test_named_rows_of_a_wide_table(t):
    """Uniform tokens of 2048 values against a table of many more rows: what is marked as named decides most of what is written."""
    from landmark_b200.embedding import embedding_backward

    idx, g, _ = make(t, 131072, 2048, torch.bfloat16, seed=t)
    got = embedding_backward(g, idx, 131072)
    check_gradient(got, g, idx, 131072)
    for _ in range(5):
        assert torch.equal(got, embedding_backward(g, idx, 131072))


@pytest.mark.parametrize("accumulate", [False, True])
def test_backward_over_a_written_out_is_refused(accumulate):
    from landmark_b200.embedding import embedding_backward

    idx, g, w = make(300, 40, 48, torch.float32)
    x = torch.ones((40, 48), device="cuda", requires_grad=True)
    loss = (w * x).sum()  # keeps w
    embedding_backward(g, idx, 40, out=w, accumulate=accumulate)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_forward_mode_tangents():
    """Both operators are linear: the tangent of a result is the operator's result for the tangent, with and without a backward pass as
    well, and its gradient is the other operator."""
    import torch.autograd.forward_ad as fwd

    from landmark_b200.embedding import embedding, embedding_backward

    for dtype in (torch.float32, torch.bfloat16):
        idx, g, w = make(500, 40, 24, dtype, masked=0.2)
        dw, dg = torch.randn_like(w), torch.randn_like(g)
        for grad in (False, True):
            with fwd.dual_level():
                a, b = w.clone().requires_grad_(grad), g.clone().requires_grad_(grad)
                da, db = dw.clone().requires_grad_(grad), dg.clone().requires_grad_(grad)
                out = fwd.unpack_dual(embedding(idx, fwd.make_dual(a, da), scale=0.5, padding_idx=7))
                assert torch.equal(out.primal, embedding(idx, w, scale=0.5)) and torch.equal(out.tangent, embedding(idx, dw, scale=0.5))
                total = fwd.unpack_dual(embedding_backward(fwd.make_dual(b, db), idx, 40, scale=0.5, padding_idx=7, dtype=torch.float32))
                assert torch.equal(total.primal, embedding_backward(g, idx, 40, scale=0.5, padding_idx=7, dtype=torch.float32))
                assert torch.equal(total.tangent, embedding_backward(dg, idx, 40, scale=0.5, padding_idx=7, dtype=torch.float32))
                if grad:  # the tangent's own gradient
                    (got,) = torch.autograd.grad((out.tangent * g).sum(), da)
                    assert torch.equal(got, embedding_backward(g, idx, 40, scale=0.5, padding_idx=7))
                into = torch.zeros((40, 24), dtype=dtype, device="cuda")
                with pytest.raises(RuntimeError, match="not differentiable"):
                    embedding_backward(fwd.make_dual(g, dg), idx, 40, out=into)
                with pytest.raises(RuntimeError, match="not differentiable"):
                    embedding_backward(g, idx, 40, out=fwd.make_dual(into, into.clone()), accumulate=True)
                plain = fwd.unpack_dual(embedding(idx, w))  # no tangent: none comes out
                assert plain.tangent is None and torch.equal(plain.primal, embedding(idx, w))
    with torch.no_grad(), fwd.dual_level():
        idx, g, w = make(50, 40, 24, torch.float32)
        assert fwd.unpack_dual(embedding(idx, fwd.make_dual(w, g[:40]))).tangent is not None


def test_out_that_is_read_is_refused():
    from landmark_b200.embedding import embedding_backward

    g = torch.randn((3000, 48), device="cuda")
    idx = torch.arange(3000, device="cuda") % 40
    kept = g.clone()
    for accumulate in (False, True):
        for out, rows in ((g, 3000), (g[:40], 40), (g[2960:], 40), (g.view(-1)[5:5 + 40 * 48].view(40, 48), 40)):
            with pytest.raises(ValueError, match="shares memory"):
                embedding_backward(g, idx, rows, out=out, accumulate=accumulate)
    with pytest.raises(ValueError, match="shares memory"):
        embedding_backward(g, idx, 60, out=idx.view(torch.float32)[:60 * 48].view(60, 48))
    assert torch.equal(g, kept) and torch.equal(idx, torch.arange(3000, device="cuda") % 40)
    wide = torch.randn((3000, 100), device="cuda")  # beside each other in one buffer: as it was
    kept = wide.clone()
    embedding_backward(wide[:, :48], idx, 3000, out=wide[:, 50:98])
    check_gradient(wide[:, 50:98], kept[:, :48], idx, 3000)
    assert torch.equal(wide[:, :50], kept[:, :50]) and torch.equal(wide[:, 98:], kept[:, 98:])
    got = embedding_backward(g[:1].expand(3000, 48), idx, 40, out=g[1:41])  # what is copied first may lie beside
    check_gradient(got, g[:1].expand(3000, 48), idx, 40)


def test_imaginary_parts_of_conjugates():
    """Views whose sign is still to come: read with it, refused where they are written."""
    from landmark_b200.embedding import embedding, embedding_backward

    idx, _, _ = make(500, 40, 1, torch.float32)
    z = torch.randn((500, 1), dtype=torch.complex64, device="cuda").conj()
    g, w = z.imag, z[:40].imag
    assert g.is_neg() and w.is_neg()
    assert torch.equal(embedding(idx, w), w[idx])
    check_gradient(embedding_backward(g, idx, 40), g, idx, 40)
    wide = torch.randn((500, 24), dtype=torch.complex64, device="cuda").conj().imag
    assert torch.equal(embedding(idx, wide[:40]), wide[:40][idx])
    check_gradient(embedding_backward(wide, idx, 40), wide, idx, 40)
    with pytest.raises(ValueError, match="out must"):
        embedding_backward(z.imag.clone(), idx, 40, out=w)

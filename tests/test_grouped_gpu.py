"""One matrix for each group of rows: the product and its gradients (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
import dense_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return ref.ops_of(pkg)


def _offsets(sizes, first=0):
    return torch.tensor([first] + sizes, device="cuda").cumsum(0).int()


def _weights(G, K, N, dtype, gen, transposed):
    w = torch.randn((G, N, K) if transposed else (G, K, N), device="cuda", generator=gen).to(dtype)
    return w.transpose(1, 2) if transposed else w


def _check(ops, X, W, offsets, dY):
    x, w = X.detach().requires_grad_(), W.detach().requires_grad_()
    y = ops.grouped_product(x, w, offsets)
    want, tol = ref.grouped(X, W, offsets)
    assert y.shape == want.shape and y.dtype == X.dtype and ref.outside(y.detach(), want, tol) == 0
    dx, dw = torch.autograd.grad(y, (x, w), dY)
    want, tol = ref.grouped(dY, W.transpose(1, 2), offsets)
    assert dx.shape == X.shape and ref.outside(dx, want, tol) == 0
    want, tol = ref.grouped_weight(X, dY, offsets)
    assert dw.shape == W.shape and dw.dtype == X.dtype and ref.outside(dw, want, tol) == 0
    return y, dx, dw


SIZES = [([1], 1, 1), ([0], 8, 8), ([5], 3, 2), ([64], 64, 64), ([1], 2048, 128), ([3, 0, 1, 2], 256, 512), ([17, 300, 0, 64, 1], 72, 136),
         ([129, 127, 128, 257], 64, 256), ([33] * 40, 40, 24), ([1000, 1], 264, 520), ([0, 0, 700, 0], 100, 64),
         ([63, 65, 191], 333, 131), ([2] * 70, 128, 384), ([515], 1000, 8), ([16, 48, 240, 272, 496], 320, 320)]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("sizes,K,N", SIZES)
def test_sizes_and_types(ops, type, transposed, sizes, K, N):
    gen = torch.Generator("cuda").manual_seed(K + N + len(sizes))
    R = sum(sizes)
    X = torch.randn((R, K), device="cuda", generator=gen).to(ref.TYPES[type])
    dY = torch.randn((R, N), device="cuda", generator=gen).to(ref.TYPES[type])
    _check(ops, X, _weights(len(sizes), K, N, X.dtype, gen, transposed), _offsets(sizes), dY)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("K,N", [(128, 192), (50, 30)])
@pytest.mark.parametrize("first,behind", [(0, 9), (5, 0), (70, 200), (0, 0)])
def test_rows_of_no_group(ops, type, K, N, first, behind):
    """Rows in front of the first group and behind the last one: zeros in Y and dX, nothing in dW, whatever they hold."""
    gen = torch.Generator("cuda").manual_seed(first + behind)
    sizes = [40, 0, 130, 7]
    R = first + sum(sizes) + behind
    X = torch.randn((R, K), device="cuda", generator=gen).to(ref.TYPES[type])
    dY = torch.randn((R, N), device="cuda", generator=gen).to(ref.TYPES[type])
    X[:first], dY[:first] = float("nan"), float("inf")
    X[first + sum(sizes):], dY[first + sum(sizes):] = float("inf"), float("nan")
    W = _weights(4, K, N, X.dtype, gen, False)
    y, dx, dw = _check(ops, X, W, _offsets(sizes, first), dY)
    for t in (y, dx):
        assert not t[:first].any() and not t[first + sum(sizes):].any()
    assert not dw[1].any()


@pytest.mark.parametrize("K,N", [(128, 256), (36, 20)])
def test_infinities_stay_in_their_rows_and_groups(ops, K, N):
    gen = torch.Generator("cuda").manual_seed(K)
    sizes = [20, 30, 50, 70]
    for dtype in (torch.bfloat16, torch.float32):
        X, dY = (torch.randn((170, c), device="cuda", generator=gen).to(dtype) for c in (K, N))
        W = _weights(4, K, N, dtype, gen, False)
        X[20, 3], X[49, 0], W[3, 0, 0], dY[100, N - 1] = float("nan"), float("inf"), float("inf"), float("nan")
        y = ops.grouped_product(X, W, _offsets(sizes))
        dx = ops.grouped_product(dY, W.transpose(1, 2), _offsets(sizes))
        dw = torch.ops.hpspmm.grouped_weight_grad(X, dY, _offsets(sizes), False)
        rows = torch.ones(170, dtype=torch.bool, device="cuda")
        rows[[20, 49]] = False
        rows[100:] = False
        want, tol = ref.grouped(X, W, _offsets(sizes))
        assert ref.outside(y[rows], want[rows], tol[rows]) == 0
        assert bool(torch.isnan(y[20]).all()) and not torch.isfinite(y[49]).any()
        want, tol = ref.grouped(dY[:100], W.transpose(1, 2), _offsets([20, 30, 50, 0]))
        assert ref.outside(dx[:100], want, tol) == 0 and bool(torch.isnan(dx[100]).all())
        want, tol = ref.grouped_weight(X, dY, _offsets(sizes))
        for g in (0, 2):                              # groups whose neighbours hold what spreads
            assert ref.outside(dw[g], want[g], tol[g]) == 0
        assert torch.equal(torch.isnan(dw[3]), torch.isnan(want[3]))


def test_many_groups_and_none(ops):
    gen = torch.Generator("cuda").manual_seed(1)
    sizes = torch.randint(0, 5, (3001,), generator=torch.Generator().manual_seed(2)).tolist()
    for K, N in ((64, 64), (24, 40), (7, 5)):
        for dtype in (torch.float16, torch.float32):
            X, dY = (torch.randn((sum(sizes), c), device="cuda", generator=gen).to(dtype) for c in (K, N))
            _check(ops, X, _weights(3001, K, N, dtype, gen, True), _offsets(sizes), dY)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    X = torch.randn((5, 64), device="cuda", generator=gen)
    assert not ops.grouped_product(X, X.new_empty((0, 64, 16)), none).any()
    assert torch.ops.hpspmm.grouped_weight_grad(X, X, none, False).shape == (0, 64, 64)
    for K, N in ((0, 16), (16, 0)):
        y = ops.grouped_product(X[:, :K], X.new_empty((1, K, N)), _offsets([5]))
        assert y.shape == (5, N) and not y.any()
        assert torch.ops.hpspmm.grouped_weight_grad(X[:, :K], y, _offsets([5]), True).shape == (1, K, N)
    assert ops.grouped_product(X[:0], X.new_empty((2, 64, 16)), _offsets([0, 0])).shape == (0, 16)
    assert not torch.ops.hpspmm.grouped_weight_grad(X[:0], X[:0], _offsets([0, 0]), False).any()


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_strides(ops, type):
    gen = torch.Generator("cuda").manual_seed(4)
    sizes, dtype = [100, 30, 66], ref.TYPES[type]
    big = torch.randn((400, 320), device="cuda", generator=gen).to(dtype)
    W = _weights(3, 128, 64, dtype, gen, False)
    dys = big[200:396, 100:164], big[4:200, :64], big[:196, 1:65], big[:1, :64].expand(196, 64), big[:196, :1].expand(196, 64)
    for X, dY in zip((big[:196, :128], big[:196, 8:136], big[:196, 3:131], big[::2][:196, :128], big.T[:196, 64:192]), dys):
        _check(ops, X, W, _offsets(sizes), dY)
    X, dY = big[:196, :128], big[:196, 128:192]
    for w in (W[:, :, ::2].repeat_interleave(2, 2)[:, :, :64], W[:1].expand(3, 128, 64), W.transpose(0, 1).contiguous().transpose(0, 1)):
        _check(ops, X, w, _offsets(sizes), dY)
    spaced = torch.stack([_offsets(sizes), _offsets(sizes)], 1)[:, 0]
    assert torch.equal(ops.grouped_product(X, W, spaced), ops.grouped_product(X, W, _offsets(sizes)))
    # memory that begins 2 or 4 bytes off a 16-byte boundary
    flat = torch.randn(3 * 128 * 64 + 1, device="cuda", generator=gen).to(dtype)
    _check(ops, X, flat[1:].view(3, 128, 64), _offsets(sizes), dY)
    # one matrix for all groups, from a smaller leaf: its gradient is the sum over the groups
    leaf = W[:1].clone().requires_grad_()
    ops.grouped_product(X, leaf.expand(3, 128, 64), _offsets(sizes)).backward(dY)
    parts, tol = ref.grouped_weight(X, dY, _offsets(sizes))
    want = parts.sum(0, keepdim=True)
    assert ref.outside(leaf.grad, want, tol.sum(0, keepdim=True) + 3 * ref.rounding(dtype, parts.abs().sum(0, keepdim=True))) == 0


def test_offsets_that_do_not_ascend_stay_in_bounds(ops):
    """The values are of no use, but nothing outside the operands is touched and rows that are named once are right."""
    gen = torch.Generator("cuda").manual_seed(5)
    for dtype in (torch.bfloat16, torch.float32):
        for K, N in ((128, 64), (33, 20)):
            X, dY = (torch.randn((90, c), device="cuda", generator=gen).to(dtype) for c in (K, N))
            W = _weights(3, K, N, dtype, gen, False)
            for bad in ([-5, 30, 1000, 2 ** 31 - 1], [0, 60, 20, 90], [90, 60, 30, 0], [2 ** 31 - 1, -2 ** 31, 0, 7]):
                off = torch.tensor(bad, dtype=torch.int32, device="cuda")
                y = ops.grouped_product(X, W, off)
                dw = torch.ops.hpspmm.grouped_weight_grad(X, dY, off, False)
                assert y.shape == (90, N) and dw.shape == (3, K, N)
            off = torch.tensor([-5, 30, 1000, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
            want, tol = ref.grouped(X, W, _offsets([30, 60, 0]))
            assert ref.outside(ops.grouped_product(X, W, off), want, tol) == 0


def test_same_every_time_captured_and_on_another_stream(ops):
    gen = torch.Generator("cuda").manual_seed(6)
    side = torch.cuda.Stream()
    for dtype, sizes, K, N in ((torch.bfloat16, [3, 0, 1, 9], 1024, 256), (torch.bfloat16, [300, 40, 500, 7], 256, 384),
                               (torch.float32, [100, 0, 31, 7], 60, 36)):
        R = sum(sizes) + 5
        X, dY = (torch.randn((R, c), device="cuda", generator=gen).to(dtype) for c in (K, N))
        W, off = _weights(4, K, N, dtype, gen, False), _offsets(sizes)

        def step():
            return (ops.grouped_product(X, W, off), ops.grouped_product(dY, W.transpose(1, 2), off),
                    torch.ops.hpspmm.grouped_weight_grad(X, dY, off, False))

        first = step()
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, step()))
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            held = step()
        X.mul_(2), off.copy_(_offsets(sizes[::-1]))
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))
        want, tol = ref.grouped(X, W, off)
        assert ref.outside(held[0], want, tol) == 0


def test_gradients_against_differences_and_second_derivatives(ops):
    gen = torch.Generator("cuda").manual_seed(7)
    sizes = [10, 0, 25]
    X, dY = (torch.randn((35, c), device="cuda", generator=gen).requires_grad_() for c in (20, 12))
    W = _weights(3, 20, 12, torch.float32, gen, False).requires_grad_()
    off = _offsets(sizes)
    ways = [torch.randn_like(X), torch.randn_like(W)]
    dx, dw = torch.autograd.grad(ops.grouped_product(X, W, off), (X, W), dY, create_graph=True)
    with torch.no_grad():
        for leaf, way, got in ((X, ways[0], dx), (W, ways[1], dw)):
            def f(t):
                return (ops.grouped_product(*((t, W) if leaf is X else (X, t)), off).double() * dY.double()).sum()
            # linear in each operand: exact but for the roundings of 35 x 12 sums of 20 products
            assert abs(float((f(leaf + way) - f(leaf - way)) / 2 - (got.double() * way.double()).sum())) < 35 * 12 * 20 * 2.0 ** -20
    # derivatives of the gradients, each along a random way
    a, b = (t.detach().double().requires_grad_() for t in (X, W))
    d = dY.detach().double().requires_grad_()
    y = torch.cat([a[s:e] @ b[g] for g, (s, e) in enumerate(zip(off.tolist(), off.tolist()[1:]))])
    ra, rb = torch.autograd.grad(y, (a, b), d, create_graph=True)
    for got, want, way in ((dx, ra, ways[0]), (dw, rb, ways[1])):
        g = torch.autograd.grad(got, (X, W, dY), way, retain_graph=True, allow_unused=True)
        w = torch.autograd.grad(want, (a, b, d), way.double(), retain_graph=True, allow_unused=True)
        for p, q in zip(g, w):
            assert (p is None) == (q is None)
            if q is not None:
                assert ref.outside(p, q, torch.full_like(q, 40 * 2.0 ** -23 * 40 * 16)) == 0     # 35 products of values below 4


def test_more_than_2_31_elements(ops):
    # weights: group 519 lies behind 2^31 elements
    G, K, N = 520, 2048, 2056
    W = torch.zeros((G, K, N), dtype=torch.bfloat16, device="cuda")
    W[-1] = torch.randn((K, N), device="cuda") / 45
    X = torch.randn((3, K), device="cuda").bfloat16()
    off = _offsets([1] + [0] * (G - 2) + [2])
    want, tol = ref.grouped(X[1:], W[-1:], _offsets([2]))
    y = ops.grouped_product(X, W, off)
    assert ref.outside(y[1:], want, tol) == 0 and not y[0].any()
    dw = torch.ops.hpspmm.grouped_weight_grad(X, y, off, False)
    want, tol = ref.grouped_weight(X[1:], y[1:], _offsets([2]))
    assert ref.outside(dw[-1:], want, tol) == 0 and not dw[:-1].any()
    del W, dw
    for K, dtype in ((2056, torch.bfloat16), (515, torch.float32)):        # rows
        R = (2 ** 31 + 5_000_000) // K
        X = torch.zeros((R, K), dtype=dtype, device="cuda")
        X[-70:] = torch.randn((70, K), device="cuda")
        W = _weights(2, K, 16, dtype, None, False)
        off = torch.tensor([0, R - 66, R], dtype=torch.int32, device="cuda")
        y = ops.grouped_product(X, W, off)
        want, tol = ref.grouped(X[-70:], W, _offsets([4, 66]))
        assert ref.outside(y[-70:], want, tol) == 0
        dx = ops.grouped_product(y, W.transpose(1, 2), off)
        want, tol = ref.grouped(y[-70:], W.transpose(1, 2), _offsets([4, 66]))
        assert ref.outside(dx[-70:], want, tol) == 0
        dw = torch.ops.hpspmm.grouped_weight_grad(X, y, off, True)
        want, tol = ref.grouped_weight(X[-70:], y[-70:], _offsets([4, 66]))
        assert ref.outside(dw[1], want[1], tol[1]) == 0
        del X, y, dx


def test_refusals(ops, pkg, gpu_ctx):
    X, W, off = torch.zeros((6, 8), device="cuda"), torch.zeros((2, 8, 4), device="cuda"), _offsets([3, 3])
    ops.grouped_product(X, W, off)
    for args in ((X.double(), W.double(), off), (X.half(), W, off), (X, W[0], off), (X[:, :7], W, off), (X, W, off.long()),
                 (X, W, off[:2]), (X, W, off.cpu()), (X.cpu(), W.cpu(), off.cpu()), (X, W.cpu(), off), (X[0], W, off)):
        with pytest.raises(RuntimeError, match="hpspmm"):
            ops.grouped_product(*args)
    grad = torch.ops.hpspmm.grouped_weight_grad
    for args in ((X, X[:5], off), (X, X.half(), off), (X, X, off.long()), (X, X, off[:0]), (X, X[0], off), (X, X, off[None])):
        with pytest.raises(RuntimeError, match="hpspmm"):
            grad(*args, False)
    Y = torch.zeros((6, 4), device="cuda")
    good = [6, 2, 8, 4, pkg.TYPE_F32, X.data_ptr(), 8, W.data_ptr(), 0, off.data_ptr(), Y.data_ptr()]
    gpu_ctx.grouped_product(*good)
    for at, v in ((0, -1), (1, -1), (2, -1), (3, -1), (4, 7), (5, None), (6, -1), (7, None), (9, None), (10, None), (0, 1 << 31)):
        with pytest.raises(pkg.HpspmmError):
            gpu_ctx.grouped_product(*(good[:at] + [v] + good[at + 1:]))
    good = [6, 2, 8, 4, pkg.TYPE_F32, X.data_ptr(), 8, Y.data_ptr(), 4, off.data_ptr(), W.data_ptr(), 0]
    gpu_ctx.grouped_weight_grad(*good)                # so few rows are not cut into pieces
    for at, v in ((0, -1), (4, -1), (5, None), (6, -1), (7, None), (8, -1), (9, None), (10, None), (1, 1 << 40)):
        with pytest.raises(pkg.HpspmmError):
            gpu_ctx.grouped_weight_grad(*(good[:at] + [v] + good[at + 1:]))
    with pytest.raises(pkg.HpspmmError, match="2\\^27"):
        gpu_ctx.grouped_product(6, 2, (1 << 27) + 8, 4, pkg.TYPE_BF16, X.data_ptr(), (1 << 27) + 8, W.data_ptr(), 0, off.data_ptr(),
                                Y.data_ptr())
    with pytest.raises(pkg.HpspmmError, match="2\\^27"):
        gpu_ctx.grouped_weight_grad((1 << 27) + 1, 3000, 8, 4, pkg.TYPE_BF16, X.data_ptr(), 8, Y.data_ptr(), 4, off.data_ptr(),
                                    W.data_ptr(), 0)
    size = pkg.load_library().hpspmm_grouped_weight_grad_workspace
    for dtype in (pkg.TYPE_F32, pkg.TYPE_BF16):
        assert size(0, 3, 8, 8, dtype, 0) == 0 and size(100, 3, 8, 8, dtype, 1) == 0
        assert size(-1, 3, 8, 8, dtype, 0) == -1 and size(5, 3, 8, 8, 9, 0) == -1
        need = size(20_000, 3, 64, 32, dtype, 0)
        assert 0 < need <= 20_000 * 96 * 4
    X, Y, W = torch.zeros((20_000, 64), device="cuda"), torch.zeros((20_000, 32), device="cuda"), torch.zeros((3, 64, 32), device="cuda")
    off = _offsets([10_000, 0, 10_000])
    need = size(20_000, 3, 64, 32, pkg.TYPE_F32, 0)
    space = torch.zeros(need + 256, dtype=torch.uint8, device="cuda")
    good = [20_000, 3, 64, 32, pkg.TYPE_F32, X.data_ptr(), 64, Y.data_ptr(), 32, off.data_ptr(), W.data_ptr(), 0, space.data_ptr(), need]
    gpu_ctx.grouped_weight_grad(*good)
    for at, v in ((12, None), (13, need - 1), (12, space.data_ptr() + 4)):
        with pytest.raises(pkg.HpspmmError):
            gpu_ctx.grouped_weight_grad(*(good[:at] + [v] + good[at + 1:]))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sizes,K,N", [([5000], 64, 40), ([0, 9000, 3, 2049, 0, 1024], 136, 64), ([4097, 7000], 33, 50), ([30_000, 1], 256, 264)])
def test_groups_cut_into_pieces(ops, type, sizes, K, N):
    """Few matrices and many rows: the gradient of a matrix is a sum over pieces of its group."""
    gen = torch.Generator("cuda").manual_seed(K)
    for transposed in (False, True):
        X, dY = (torch.randn((sum(sizes) + 3, c), device="cuda", generator=gen).to(ref.TYPES[type]) for c in (K, N))
        W = _weights(len(sizes), K, N, X.dtype, gen, transposed)
        _, _, first = _check(ops, X, W, _offsets(sizes), dY)
        _, _, again = _check(ops, X, W, _offsets(sizes), dY)
        assert torch.equal(first, again)
    # offsets that do not ascend want more pieces than there is room for
    n = sum(sizes)
    off = torch.tensor([0, n] * 3 + [0], dtype=torch.int32, device="cuda")
    assert torch.ops.hpspmm.grouped_weight_grad(X, dY, off, False).shape == (6, K, N)


# enough tiles for blocks of 256 rows: pairs of blocks (1024 columns), blocks by themselves (384), rows that no copy engine
# takes (odd widths)
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("sizes,K,N", [([4000, 0, 3000, 33], 256, 1024), ([300] * 40 + [1, 15, 17], 1024, 2048), ([6000, 0, 7001, 500], 72, 384),
                                       ([1500, 1, 4000, 0, 777], 70, 1031), ([511, 513, 3, 2048, 70, 900], 1024, 1100)])
def test_many_tiles(ops, type, sizes, K, N):
    gen = torch.Generator("cuda").manual_seed(N)
    R = sum(sizes) + 40
    X, dY = (torch.randn((R, c), device="cuda", generator=gen).to(ref.TYPES[type]) for c in (K, N))
    X[sum(sizes):], dY[sum(sizes):] = float("nan"), float("inf")        # rows behind the last group
    for transposed in (False, True):
        W = _weights(len(sizes), K, N, X.dtype, gen, transposed)
        y, dx, dw = _check(ops, X, W, _offsets(sizes), dY)
        assert not y[sum(sizes):].any() and not dx[sum(sizes):].any()
        again = _check(ops, X, W, _offsets(sizes), dY)
        assert all(torch.equal(a, b) for a, b in zip((y, dx, dw), again))


def test_neighbours_of_a_group_do_not_reach_its_gradient(ops):
    """Groups that end inside the 16 rows of an instruction, between groups of NaN: pairs of blocks and single ones."""
    gen = torch.Generator("cuda").manual_seed(3)
    for K, N in ((1024, 2048), (72, 384), (64, 64)):
        sizes = [37, 64, 30, 1, 50, 5, 100] * 6
        off = _offsets(sizes)
        X, dY = (torch.randn((sum(sizes), c), device="cuda", generator=gen).bfloat16() for c in (K, N))
        want, tol = ref.grouped_weight(X, dY, off)
        bounds = off.tolist()
        for g in range(1, len(sizes), 2):
            X[bounds[g]:bounds[g + 1]], dY[bounds[g]:bounds[g + 1]] = float("nan"), float("inf")
        for transposed in (False, True):
            dw = torch.ops.hpspmm.grouped_weight_grad(X, dY, off, transposed)
            assert ref.outside(dw[::2], want[::2], tol[::2]) == 0 and bool(torch.isnan(dw[1::2]).all())


def test_streams_and_threads_at_once(ops):
    """Calls of several threads, each on a stream of its own, without waiting for one another."""
    import threading
    gen = torch.Generator("cuda").manual_seed(11)
    work, errors = [], []
    for i, (K, N, dtype) in enumerate(((1024, 1024, torch.bfloat16), (50, 30, torch.float32), (2048, 128, torch.float16))):
        sizes = [30 * (i + 1), 0, 700]
        X = torch.randn((sum(sizes), K), device="cuda", generator=gen).to(dtype)
        dY = torch.randn((sum(sizes), N), device="cuda", generator=gen).to(dtype)
        W = _weights(3, K, N, dtype, gen, False)
        work.append((X, dY, W, _offsets(sizes), ref.grouped(X, W, _offsets(sizes)), ref.grouped_weight(X, dY, _offsets(sizes))))
    torch.cuda.synchronize()

    def steps(X, dY, W, off, want, want_w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(40):
                    y, dw = ops.grouped_product(X, W, off), torch.ops.hpspmm.grouped_weight_grad(X, dY, off, False)
                    if i % 10 == 9:
                        assert ref.outside(y, *want) == 0 and ref.outside(dw, *want_w) == 0
        except BaseException as e:      # noqa: B902 -- a thread's failure is the test's
            errors.append(e)

    threads = [threading.Thread(target=steps, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    assert ops.timeouts() == 0


@pytest.mark.parametrize("K", [8, 64, 120, 128, 130, 256, 328, 403, 512, 520, 777, 1000, 1024, 2049, 4096])
def test_few_rows_of_every_depth(ops, K):
    """A step of a decoder: blocks that split the depth of one tile, where it is long enough for that."""
    gen = torch.Generator("cuda").manual_seed(K)
    for dtype in (torch.float16, torch.bfloat16):
        for sizes in ([1], [3, 2], [0, 17, 0, 5], [40, 1, 60]):
            for N in (8, 22, 136):
                X, dY = (torch.randn((sum(sizes) + 2, c), device="cuda", generator=gen).to(dtype) for c in (K, N))
                for transposed in (False, True):
                    _check(ops, X, _weights(len(sizes), K, N, dtype, gen, transposed), _offsets(sizes), dY)


def test_beside_the_librarys_products(ops):
    """Kernels of another owner on the same tensor cores, on another stream: nobody waits for anybody."""
    gen = torch.Generator("cuda").manual_seed(14)
    X, W = torch.randn((3000, 1024), device="cuda", generator=gen).bfloat16(), _weights(4, 1024, 1024, torch.bfloat16, gen, False)
    off, A = _offsets([500, 10, 1490, 1000]), torch.randn((2048, 2048), device="cuda", generator=gen).bfloat16()
    want, tol = ref.grouped(X, W, off)
    want_w, tol_w = ref.grouped_weight(X, X, off)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(40):
        with torch.cuda.stream(one):
            y = ops.grouped_product(X, W, off)
            few = ops.grouped_product(X[:8], W, off // 400)
        with torch.cuda.stream(two):
            A @ A
            dw = torch.ops.hpspmm.grouped_weight_grad(X, X, off, False)
    torch.cuda.synchronize()
    assert ref.outside(y, want, tol) == 0 and ref.outside(dw, want_w, tol_w) == 0 and ops.timeouts() == 0
    want, tol = ref.grouped(X[:8], W, off // 400)
    assert ref.outside(few, want, tol) == 0


# One call of each kind of kernel: (rows of the groups, K, N).  Pairs of blocks, 256 rows to a tile, 128, 64, clusters of two to
# eight blocks, widths that no copy engine takes; the gradients come with each of them.
KINDS = [([4000, 0, 3000, 33], 256, 1024), ([6000, 0, 7001, 500], 72, 384), ([600], 1024, 1024), ([300, 9], 256, 136), ([40], 1024, 2048),
         ([16], 2048, 1024), ([3, 5], 4096, 256), ([300, 40], 333, 131), ([3], 1001, 24), ([20_000], 64, 40)]


@pytest.fixture
def waits(pkg):
    f = pkg.load_library().hpspmm_debug_grouped_waits
    yield f
    f(0, 0)


@pytest.mark.parametrize("sizes,K,N", KINDS)
def test_a_wait_that_runs_out_ends_the_call(pkg, waits, sizes, K, N):
    """Copies that never come: every block gives up, all of its warps together, and the next calls are as ever."""
    gen = torch.Generator("cuda").manual_seed(K)
    R, G = sum(sizes), len(sizes)
    X, dY = (torch.randn((R, c), device="cuda", generator=gen).bfloat16() for c in (K, N))
    W, off = _weights(G, K, N, torch.bfloat16, gen, False), _offsets(sizes)
    Y, dW = torch.empty((R, N), dtype=X.dtype, device="cuda"), torch.empty_like(W)
    need = pkg.load_library().hpspmm_grouped_weight_grad_workspace(R, G, K, N, pkg.TYPE_BF16, 0)
    space = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream().cuda_stream

    def product(ctx):
        ctx.grouped_product(R, G, K, N, pkg.TYPE_BF16, X.data_ptr(), K, W.data_ptr(), 0, off.data_ptr(), Y.data_ptr(), stream)

    def gradient(ctx):
        ctx.grouped_weight_grad(R, G, K, N, pkg.TYPE_BF16, X.data_ptr(), K, dY.data_ptr(), N, off.data_ptr(), dW.data_ptr(), 0, space.data_ptr(),
                                need, stream)

    for call, out, (want, tol) in ((product, Y, ref.grouped(X, W, off)), (gradient, dW, ref.grouped_weight(X, dY, off))):
        with pkg.Context(0) as ctx:
            assert waits(200_000, 1) == pkg.OK
            call(ctx)
            assert ctx.timeouts() > 0
            assert waits(0, 0) == pkg.OK
            seen = ctx.timeouts()
            with pytest.raises(pkg.HpspmmError, match="gave up") as e:      # told once, by the next call
                call(ctx)
            assert e.value.status == pkg.ERR_TIMEOUT
            for _ in range(3):
                call(ctx)
            assert ref.outside(out, want, tol) == 0 and ctx.timeouts() == seen


@pytest.mark.parametrize("case", ["lines", "neighbour", "deep lines", "deep"])
def test_a_wait_lasts_as_long_as_its_tile(pkg, waits, case):
    """Tiles of several milliseconds under a limit of 50 microseconds, which comes on top of the time that a tile's stages may
    take.  Gradients of one long group among many (which is not cut into pieces) at a width that no copy engine takes;
    one behind which the same block has a group that ends inside an instruction's depth; products over a long depth."""
    gen = torch.Generator("cuda").manual_seed(5)
    with pkg.Context(0) as ctx:
        assert waits(100_000, 0) == pkg.OK
        if case.startswith("deep"):
            R, K, N = 8, (1 << 20) + 1 if case == "deep lines" else 1 << 23, 8
            X, W, off = torch.randn((R, K), device="cuda", generator=gen).bfloat16(), _weights(1, K, N, torch.bfloat16, gen, False), _offsets([R])
            out, (want, tol) = torch.full((R, N), float("nan"), dtype=X.dtype, device="cuda"), ref.grouped(X, W, off)
            torch.cuda.synchronize()
            ctx.grouped_product(R, 1, K, N, pkg.TYPE_BF16, X.data_ptr(), K, W.data_ptr(), 0, off.data_ptr(), out.data_ptr())
        else:
            width = 3 if case == "lines" else 64
            sizes = [0] * 2100
            sizes[0], sizes[torch.cuda.get_device_properties(0).multi_processor_count] = 1 << 20, 5
            R, G, off = sum(sizes), len(sizes), _offsets(sizes)
            X, dY = (torch.randn((R, width), device="cuda", generator=gen).bfloat16() for _ in range(2))
            out, (want, tol) = torch.full((G, width, width), float("nan"), dtype=X.dtype, device="cuda"), ref.grouped_weight(X, dY, off)
            torch.cuda.synchronize()
            ctx.grouped_weight_grad(R, G, width, width, pkg.TYPE_BF16, X.data_ptr(), width, dY.data_ptr(), width, off.data_ptr(), out.data_ptr(), 0)
        assert ctx.timeouts() == 0 and ref.outside(out, want, tol) == 0


def test_whoever_calls_next_is_told_of_a_wait_that_ran_out(pkg, waits):
    """Every dense operator of the context, once, and with nothing done; refused arguments are refused as ever."""
    bf16 = torch.bfloat16
    X, W, off, Y = (torch.ones(s, dtype=bf16, device="cuda") for s in ((40, 64), (1, 64, 8), (1,), (40, 8)))
    off = _offsets([40])
    ids, z, teacher = torch.zeros(40, dtype=torch.int64, device="cuda"), torch.zeros((40, 8), device="cuda"), torch.zeros(40, device="cuda")
    loss, stats, out = (torch.full(s, 5.0, device="cuda") for s in ((40,), (40, 2), (40, 8)))
    space = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    p = [t.data_ptr() for t in (X, W, off, Y, ids, z, teacher, loss, stats, out, space)]
    x, w, o, y, i, zz, te, lo, st, ou, sp = p
    with pkg.Context(0) as ctx:
        def product(rows=40):
            ctx.grouped_product(rows, 1, 64, 8, pkg.TYPE_BF16, x, 64, w, 0, o, y)
        for call in (lambda: ctx.embedding_forward(40, 40, 8, pkg.TYPE_F32, i, 8, zz, 8, 1.0, ou),
                     lambda: ctx.embedding_backward(40, 40, 8, pkg.TYPE_F32, i, 8, zz, 8, 1.0, ou, sp, 1 << 20), product,
                     lambda: ctx.grouped_weight_grad(40, 1, 64, 8, pkg.TYPE_BF16, x, 64, y, 8, o, w, 0),
                     lambda: ctx.topk_distill_forward(40, 8, 1, pkg.TYPE_F32, zz, 8, i, 8, te, 1.0, lo, st),
                     lambda: ctx.topk_distill_backward(40, 8, 1, pkg.TYPE_F32, zz, 8, i, 8, te, 1.0, st, te, 1, ou)):
            waits(100_000, 1)
            product()
            waits(0, 0)
            torch.cuda.synchronize()
            before = [t.clone() for t in (loss, stats, out, W)]
            with pytest.raises(pkg.HpspmmError) as e:
                product(-1)
            assert e.value.status == pkg.ERR_INVALID
            with pytest.raises(pkg.HpspmmError, match="gave up") as e:
                call()
            assert e.value.status == pkg.ERR_TIMEOUT
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(before, (loss, stats, out, W)))
            call()
            product()
            torch.cuda.synchronize()
            assert bool((Y == 64 * W[0, 0, 0]).all())


def test_pytorch_raises_after_a_wait_that_ran_out():
    """A process of its own, whose contexts may count: a graph's replay gives up, the next call outside raises, those behind work."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import sys
sys.path[:0] = [%r, %r]
import torch
import __graft_entry__
import dense_reference as ref
pkg = __graft_entry__.load_package()
ops = ref.ops_of(pkg)
waits = pkg.load_library().hpspmm_debug_grouped_waits
X, W, off = torch.ones((40, 64), device="cuda").half(), torch.ones((1, 64, 8), device="cuda").half(), torch.tensor([0, 40], dtype=torch.int32, device="cuda")
ops.grouped_product(X, W, off)
g = torch.cuda.CUDAGraph()
waits(100_000, 1)
with torch.cuda.graph(g):
    ops.grouped_product(X, W, off)
waits(0, 0)
assert ops.timeouts() == 0
g.replay()
torch.cuda.synchronize()
try:
    ops.embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), X)
except RuntimeError as e:
    assert "gave up" in str(e) and "status 4" in str(e), e
else:
    assert False
assert bool((ops.grouped_product(X, W, off) == 64).all()) and ops.timeouts() > 0
print("well")
""" % (root, os.path.join(root, "tests"))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip().endswith("well"), out.stdout[-2000:]


def test_refusals_next_to_2_31(pkg, gpu_ctx):
    t = torch.zeros(64, device="cuda")
    off, at = _offsets([3]), t.data_ptr()
    for type in (pkg.TYPE_F32, pkg.TYPE_BF16):
        for R, K, N in ((2 ** 31 - 1025, 1, 1), (1, 2 ** 31 - 1025, 1), (1, 1, 2 ** 31 - 1025), (2 ** 31 - 2, 1, 1), (1, 1, 2 ** 31 - 2)):
            with pytest.raises(pkg.HpspmmError) as e:
                gpu_ctx.grouped_product(R, 1, K, N, type, at, K, at, 0, off.data_ptr(), at)
            assert e.value.status == pkg.ERR_UNSUPPORTED
            with pytest.raises(pkg.HpspmmError) as e:
                gpu_ctx.grouped_weight_grad(R, 1, K, N, type, at, K, at, N, off.data_ptr(), at, 0)
            assert e.value.status == pkg.ERR_UNSUPPORTED


@pytest.mark.parametrize("type", ["bf16", "f32"])
def test_nearly_2_31_rows(ops, type):
    """One column in, one out: every row is one product, rounded once, and the gradient is a sum over pieces of 14 million rows
    of which a few hold something."""
    gen = torch.Generator("cuda").manual_seed(30)
    R, dtype = 2 ** 31 - 2000, ref.TYPES[type]
    torch.cuda.empty_cache()
    X = torch.empty((R, 1), dtype=dtype, device="cuda").normal_(generator=gen)
    W = torch.tensor([[[0.7]]], device="cuda").to(dtype)
    off = torch.tensor([0, R - 3], dtype=torch.int32, device="cuda")
    y = ops.grouped_product(X, W, off)
    assert not y[R - 3:].any()
    y[R - 3:] = X[R - 3:].float().mul(W[0, 0].float()).to(dtype)
    assert all(torch.equal(b, a.float().mul(W[0, 0].float()).to(dtype)) for a, b in zip(X.split(1 << 28), y.split(1 << 28)))
    y.zero_()
    places = torch.tensor([0, 1 << 24, 10 ** 9, R // 2, R - 20_000_000, R - 5, R - 4], device="cuda")
    y[places] = torch.randn((7, 1), device="cuda", generator=gen).to(dtype)
    dw = torch.ops.hpspmm.grouped_weight_grad(X, y, off, False)
    want, tol = ref.grouped_weight(X[places], y[places], _offsets([7]))
    assert ref.outside(dw, want, tol) == 0
    del X, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("first,behind", [(0, 0), (5, 70)])
def test_more_groups_than_one_launch_has(ops, first, behind):
    """Products in 32 bits take their groups in launches of 4,224: nothing is lost between two of them, and rows of no group are
    cleared once."""
    gen = torch.Generator("cuda").manual_seed(33)
    sizes = torch.randint(0, 3, (8448,), generator=torch.Generator().manual_seed(34)).tolist()
    for at in (0, 2049, 4222, 4223, 4224, 4225, 8446, 8447):
        sizes[at] = 65 + at % 7
    R = first + sum(sizes) + behind
    X, dY = (torch.randn((R, c), device="cuda", generator=gen) for c in (20, 12))
    X[:first], X[R - behind:] = float("nan"), float("nan")
    y, dx, dw = _check(ops, X, _weights(8448, 20, 12, torch.float32, gen, False), _offsets(sizes, first), dY)
    for t in (y, dx):
        assert not t[:first].any() and not t[R - behind:].any()


def test_time_grows_with_the_groups_not_with_their_square(ops):
    """131,072 groups of a thousand rows: 118 and 175 ms when every block looked through all groups, 1 to 2 since."""
    gen = torch.Generator("cuda").manual_seed(35)
    G, R = 1 << 17, 1000
    off = torch.zeros(G + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.bincount(torch.randint(0, G, (R,), device="cuda", generator=gen), minlength=G).cumsum(0)
    X, dY = (torch.randn((R, 16), device="cuda", generator=gen) for _ in range(2))
    W = torch.randn((G, 16, 16), device="cuda", generator=gen)
    for call in (lambda: ops.grouped_product(X, W, off), lambda: torch.ops.hpspmm.grouped_weight_grad(X, dY, off, False)):
        call()
        times = []
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        assert min(times) < 25, times

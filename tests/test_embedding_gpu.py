"""Rows of a table by id and the table's gradient (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
import dense_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return ref.ops_of(pkg)


def _ids(n, rows, gen, skew=True, missing=0.1, wide=True):
    u = torch.rand(n, device="cuda", generator=gen)
    ids = ((rows ** u - 1) if skew else rows * u).long().clamp_(0, max(rows - 1, 0))
    ids[torch.rand(n, device="cuda", generator=gen) < missing] = -1
    return ids if wide else ids.int()


def _check(ops, ids, table, scale, dout):
    leaf = table.detach().requires_grad_()
    out = ops.embedding(ids, leaf, scale)
    want, tol = ref.embedding(ids, table, scale)
    assert out.shape == want.shape and out.dtype == table.dtype and ref.outside(out.detach(), want, tol) == 0
    got, = torch.autograd.grad(out, leaf, dout)
    want, tol = ref.embedding_grad(ids.reshape(-1), dout.reshape(-1, table.shape[1]), table.shape[0], scale)
    assert got.shape == table.shape and got.dtype == table.dtype and ref.outside(got, want, tol) == 0
    return got


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,rows,cols", [(1, 1, 1), (1, 50_000, 2048), (7, 3, 5), (31, 1000, 47), (257, 33, 64), (1000, 70_001, 100),
                                         (4097, 2, 130), (8191, 512, 24), (8193, 100_000, 33), (20_011, 5_003, 250),
                                         (70_001, 300_007, 16), (300_001, 1_000, 8)])
def test_sizes_and_types(ops, type, n, rows, cols):
    gen = torch.Generator("cuda").manual_seed(n + rows + cols)
    dtype = ref.TYPES[type]
    table = torch.randn((rows, cols), device="cuda", generator=gen).to(dtype)
    dout = torch.randn((n, cols), device="cuda", generator=gen).to(dtype)
    _check(ops, _ids(n, rows, gen, wide=n % 2 == 0), table, 1.0 if n % 3 == 0 else 5.657, dout)


@pytest.mark.parametrize("n,rows,cols", [(64, 40, 4096), (300, 1000, 2176), (12_000, 600, 1025), (9_000, 3, 515)])
def test_wide_rows(ops, n, rows, cols):
    gen = torch.Generator("cuda").manual_seed(cols)
    for dtype in (torch.bfloat16, torch.float32):
        table = torch.randn((rows, cols), device="cuda", generator=gen).to(dtype)
        dout = torch.randn((n, cols), device="cuda", generator=gen).to(dtype)
        _check(ops, _ids(n, rows, gen), table, 0.25, dout)


@pytest.mark.parametrize("n", [5, 3000, 40_000])
@pytest.mark.parametrize("kind", ["one id", "none", "ascending", "descending", "far outside", "two"])
def test_distributions(ops, n, kind):
    rows, cols = 700, 72
    gen = torch.Generator("cuda").manual_seed(n)
    at = torch.arange(n, device="cuda")
    ids = {"one id": torch.full_like(at, 699), "none": torch.full_like(at, -1), "ascending": at * rows // n,
           "descending": rows - 1 - at * rows // n, "two": at % 2 * 699,
           "far outside": torch.where(at % 3 == 0, at % rows, torch.where(at % 3 == 1, 2 ** 40 + at, -(2 ** 62)))}[kind]
    dtype = torch.bfloat16
    table = torch.randn((rows, cols), device="cuda", generator=gen).to(dtype)
    dout = torch.randn((n, cols), device="cuda", generator=gen).to(dtype)
    _check(ops, ids, table, 2.0, dout)


def test_no_ids_no_rows_no_columns(ops):
    table = torch.randn((9, 16), device="cuda", requires_grad=True)
    out = ops.embedding(torch.zeros((3, 0), dtype=torch.int64, device="cuda"), table)
    assert out.shape == (3, 0, 16)
    got, = torch.autograd.grad(out, table, torch.zeros_like(out))
    assert got.shape == (9, 16) and not got.any()
    ids = torch.tensor([0, -1, 5], device="cuda")
    none = torch.empty((0, 8), device="cuda", requires_grad=True)
    out = ops.embedding(ids, none)
    assert out.shape == (3, 8) and not out.any()
    assert torch.autograd.grad(out, none, torch.ones_like(out))[0].shape == (0, 8)
    flat = torch.empty((4, 0), device="cuda", requires_grad=True)
    out = ops.embedding(ids, flat)
    assert out.shape == (3, 0) and torch.autograd.grad(out, flat, out.detach())[0].shape == (4, 0)


def test_strides_and_shapes(ops):
    gen = torch.Generator("cuda").manual_seed(3)
    wide = torch.randn((50, 80), device="cuda", generator=gen)
    ids = _ids(60, 50, gen).reshape(4, 3, 5)
    dout = torch.randn((4, 3, 5, 32), device="cuda", generator=gen)
    for table in (wide[:, :32], wide[:, 3:35], wide[:, 1:65:2], wide[::2][:, 48:], wide.T[:50, :32], wide[:1, :32].expand(50, 32)):
        want, tol = ref.embedding(ids % table.shape[0], table, 1.5)
        assert ref.outside(ops.embedding(ids % table.shape[0], table, 1.5), want, tol) == 0
    table = wide[:, :32].contiguous()
    assert torch.equal(ops.embedding(ids.transpose(0, 2), table), ops.embedding(ids.transpose(0, 2).contiguous(), table))
    for d in (dout, dout.transpose(0, 1).contiguous().transpose(0, 1), dout[..., :1].expand(4, 3, 5, 32),
              dout[:1].expand(4, 3, 5, 32), torch.randn((4, 3, 5, 40), device="cuda", generator=gen)[..., 8:]):
        _check(ops, ids, table, 1.0, d)
    leaf = table.requires_grad_()
    ops.embedding(ids, leaf).sum().backward()
    want, tol = ref.embedding_grad(ids.reshape(-1), torch.ones((60, 32), device="cuda"), 50, 1.0)
    assert ref.outside(leaf.grad, want, tol) == 0


def test_infinities_stay_in_their_rows(ops):
    table = torch.randn((6, 8), device="cuda")
    table[2], table[3] = float("inf"), float("nan")
    ids = torch.tensor([0, 2, 3, 1, -1], device="cuda")
    want, tol = ref.embedding(ids, table, 2.0)
    assert ref.outside(ops.embedding(ids, table, 2.0), want, tol) == 0
    dout = torch.randn((5, 8), device="cuda")
    dout[4] = float("nan")                           # belongs to no row of the table
    dout[1, 3] = float("inf")
    leaf = table.requires_grad_()
    got, = torch.autograd.grad(ops.embedding(ids, leaf, 2.0), leaf, dout)
    want, tol = ref.embedding_grad(ids, dout, 6, 2.0)
    assert ref.outside(got, want, tol) == 0


def test_gradient_is_the_same_every_time(ops):
    gen = torch.Generator("cuda").manual_seed(8)
    for n in (5_000, 60_000):
        table = torch.randn((1000, 96), device="cuda", generator=gen).requires_grad_()
        ids = _ids(n, 1000, gen)
        dout = torch.randn((n, 96), device="cuda", generator=gen)
        first, = torch.autograd.grad(ops.embedding(ids, table), table, dout)
        for _ in range(5):
            assert torch.equal(first, torch.autograd.grad(ops.embedding(ids, table), table, dout)[0])


def test_gradient_against_differences_and_its_own_derivative(ops):
    gen = torch.Generator("cuda").manual_seed(9)
    table = torch.randn((40, 24), device="cuda", generator=gen).requires_grad_()
    ids, dout = _ids(100, 40, gen), torch.randn((100, 24), device="cuda", generator=gen).requires_grad_()
    way = torch.randn((40, 24), device="cuda", generator=gen)

    def f(t):
        return (ops.embedding(ids, t, 3.0).double() * dout.double()).sum()

    got, = torch.autograd.grad(ops.embedding(ids, table, 3.0), table, dout, create_graph=True)
    with torch.no_grad():
        slope = (f(table + way) - f(table - way)) / 2     # linear: exact but for roundings of 100 x 24 terms
        assert abs(float(slope - (got.double() * way.double()).sum())) < 100 * 24 * 3 * 16 * 2.0 ** -22
    second, = torch.autograd.grad(got, dout, way)
    want, tol = ref.embedding(ids, way, 3.0)
    assert ref.outside(second, want, tol) == 0


def test_more_than_2_31_elements(ops):
    rows, cols = 1_050_000, 2050                          # neither a multiple of 8 elements nor below 2^31
    table = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    table[-3:] = torch.arange(3 * cols, device="cuda").reshape(3, cols) % 251
    ids = torch.tensor([rows - 1, rows - 3, rows, rows - 2], device="cuda")
    out = ops.embedding(ids, table, 2.0)
    assert torch.equal(out[[0, 1, 3]], table[[rows - 1, rows - 3, rows - 2]] * 2) and not out[2].any()
    few = torch.zeros((5, cols), dtype=torch.bfloat16, device="cuda").requires_grad_()
    ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    ids[-3:] = torch.tensor([4, 0, 4], device="cuda")
    got, = torch.autograd.grad(ops.embedding(ids, few), few, table)
    assert torch.equal(got[0], table[-2]) and not got[1:4].any()
    assert torch.equal(got[4], (table[-1].float() + table[-3].float()).bfloat16())
    del table, got
    # a gradient of that many elements
    few = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda").requires_grad_()
    ids = torch.tensor([rows - 1, 0, rows - 1], device="cuda")
    dout = torch.ones((3, cols), dtype=torch.bfloat16, device="cuda")
    got, = torch.autograd.grad(ops.embedding(ids, few), few, dout)
    assert bool((got[0] == 1).all()) and bool((got[-1] == 2).all()) and not got[1:-1].any()


def test_captured_and_on_another_stream(ops):
    gen = torch.Generator("cuda").manual_seed(12)
    table = torch.randn((900, 64), device="cuda", generator=gen)
    ids, dout = _ids(12_000, 900, gen), torch.randn((12_000, 64), device="cuda", generator=gen)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):                                    # two graphs of one pool
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side, pool=graphs[0][0].pool() if graphs else None):
            out = ops.embedding(ids, table, 2.0)
            grad = torch.ops.hpspmm.embedding_backward(dout, ids, 900, 2.0)
        graphs.append((g, out, grad))
    for k in range(3):
        ids.copy_(_ids(12_000, 900, gen))
        dout.copy_(torch.randn((12_000, 64), device="cuda", generator=gen))
        torch.cuda.synchronize()
        g, out, grad = graphs[k % 2]
        g.replay()
        with torch.cuda.stream(other):
            eager = torch.ops.hpspmm.embedding_backward(dout, ids, 900, 2.0)
        torch.cuda.synchronize()
        want, tol = ref.embedding(ids, table, 2.0)
        assert ref.outside(out, want, tol) == 0
        assert torch.equal(grad, eager)
        want, tol = ref.embedding_grad(ids, dout, 900, 2.0)
        assert ref.outside(grad, want, tol) == 0


def test_refusals(ops, pkg, gpu_ctx):
    table, ids = torch.zeros((4, 8), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for args in ((ids, table.double()), (ids, table[0]), (ids.float(), table), (ids.cpu(), table), (ids, table.cpu()),
                 (ids.short(), table)):
        with pytest.raises(RuntimeError, match="hpspmm"):
            ops.embedding(*args)
    with pytest.raises(RuntimeError, match="hpspmm"):
        torch.ops.hpspmm.embedding_backward(torch.zeros((4, 8), device="cuda"), ids, 4, 1.0)
    with pytest.raises(RuntimeError, match="hpspmm"):
        torch.ops.hpspmm.embedding_backward(torch.zeros((3, 8), device="cuda"), ids, -1, 1.0)
    out, space = torch.zeros((3, 8), device="cuda"), torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = {"ids": ids.data_ptr(), "table": table.data_ptr(), "out": out.data_ptr()}
    good = [3, 4, 8, pkg.TYPE_F32, p["ids"], 8, p["table"], 8, 1.0, p["out"]]
    gpu_ctx.embedding_forward(*good)
    for at, v in ((0, -1), (1, -1), (2, -1), (3, 3), (4, None), (5, 2), (6, None), (7, 7), (9, None), (0, 1 << 31)):
        with pytest.raises(pkg.HpspmmError):
            gpu_ctx.embedding_forward(*(good[:at] + [v] + good[at + 1:]))
    need = pkg.load_library().hpspmm_embedding_backward_workspace(3, 4, 8)
    good = [3, 4, 8, pkg.TYPE_F32, p["ids"], 8, p["out"], 8, 1.0, p["table"], space.data_ptr(), need]
    assert 0 < need <= 1 << 16
    gpu_ctx.embedding_backward(*good)
    for at, v in ((0, -1), (3, -1), (5, 3), (7, -8), (9, None), (10, None), (11, need - 1)):
        with pytest.raises(pkg.HpspmmError):
            gpu_ctx.embedding_backward(*(good[:at] + [v] + good[at + 1:]))
    assert pkg.load_library().hpspmm_embedding_backward_workspace(-1, 4, 8) == -1
    with pytest.raises(pkg.HpspmmError):
        gpu_ctx.embedding_backward(*(good[:10] + [space.data_ptr() + 8, need]))


def test_one_row_of_the_gradient_for_all_positions(pkg, gpu_ctx):
    """A row stride of zero, as of a sum over the positions: read as it lies."""
    ids = torch.tensor([2, 0, 2, 5, -1, 2], dtype=torch.int32, device="cuda")
    row, dtable = torch.randn(40, device="cuda"), torch.full((4, 40), 7.0, device="cuda")
    need = pkg.load_library().hpspmm_embedding_backward_workspace(6, 4, 40)
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.embedding_backward(6, 4, 40, pkg.TYPE_F32, ids.data_ptr(), 4, row.data_ptr(), 0, 1.0, dtable.data_ptr(),
                               space.data_ptr(), need)
    torch.cuda.synchronize()
    assert torch.equal(dtable[0], row) and not dtable[1].any() and not dtable[3].any()
    assert float((dtable[2].double() - 3 * row.double()).abs().max()) <= 3 * 2.0 ** -23 * float(row.abs().max())


@pytest.mark.parametrize("type", ["f16", "f32"])
def test_a_row_of_nearly_2_31_columns(ops, type):
    torch.cuda.empty_cache()
    K, gen = 2 ** 31 - 3, torch.Generator("cuda").manual_seed(31)
    table = torch.empty((1, K), dtype=ref.TYPES[type], device="cuda").uniform_(generator=gen)
    out = ops.embedding(torch.tensor([0, -1], device="cuda"), table, 1.5)
    assert all(torch.equal(a.float().mul(1.5).to(table.dtype), b) for a, b in zip(table[0].split(1 << 28), out[0].split(1 << 28)))
    assert not any(bool(c.any()) for c in out[1].split(1 << 28))
    del table, out
    torch.cuda.empty_cache()

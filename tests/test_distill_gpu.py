"""The loss against a teacher's largest logits, its gradient, and the operators together (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
import dense_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(scope="module")
def ops(pkg):
    return ref.ops_of(pkg)


def _inputs(T, V, k, dtype, gen, missing=0.2, wide=True):
    z = (torch.randn((T, V), device="cuda", generator=gen) * 3).to(dtype)
    ids = torch.randint(0, max(V, 1), (T, k), device="cuda", generator=gen)
    ids[torch.rand((T, k), device="cuda", generator=gen) < missing] = -1
    teacher = torch.randn((T, k), device="cuda", generator=gen) * 2 + 4
    return z, ids if wide else ids.int(), teacher


def _check(ops, z, ids, teacher, tau, dloss=None):
    leaf = z.detach().requires_grad_()
    loss = ops.topk_distill_loss(leaf, ids, teacher, tau)
    want, tol = ref.distill(z, ids, teacher, tau)
    assert loss.shape == want.shape and loss.dtype == torch.float32 and ref.outside(loss.detach(), want, tol) == 0
    if dloss is None:
        dloss = torch.rand(loss.shape, device="cuda") + 0.5
    dz, = torch.autograd.grad(loss, leaf, dloss)
    want, tol = ref.distill_grad(z, ids, teacher, tau, dloss)
    assert dz.shape == z.shape and dz.dtype == z.dtype and ref.outside(dz, want, tol) == 0
    return loss.detach(), dz


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (1, 7, 3), (3, 47, 5), (2, 131_072, 64), (1, 131_073, 100), (9, 32_003, 20), (5, 4099, 1024),
                                   (700, 513, 8), (148, 10_000, 32), (2000, 40, 1), (20, 8192, 33), (300, 20_001, 7)])
def test_sizes_and_types(ops, type, T, V, k):
    gen = torch.Generator("cuda").manual_seed(T + V + k)
    z, ids, teacher = _inputs(T, V, k, ref.TYPES[type], gen, wide=T % 2 == 0)
    _check(ops, z, ids, teacher, 2.0 if k % 2 else 0.7)


@pytest.mark.parametrize("V", [29, 5000])
def test_entries_that_do_not_count(ops, V):
    gen = torch.Generator("cuda").manual_seed(1)
    z, ids, teacher = _inputs(8, V, 6, torch.float32, gen, missing=0.0)
    ids[0] = -1                                       # a row without entries
    ids[1, 2:], teacher[1, 2:] = -1, float("nan")     # whatever a padded entry holds
    ids[2, 3] = V                                     # one behind the last column
    ids[3, :4], ids[3, 4] = 2 ** 40, -(2 ** 60)
    teacher[4, 1:] = -INF                             # one entry left: p = 1
    teacher[5] = -INF                                 # none left
    teacher[6, 0] = 200.0                             # the others' shares vanish
    teacher[7] = torch.finfo(torch.float32).min       # the type's lowest value is a value: equal shares
    loss, dz = _check(ops, z, ids, teacher, 1.0)
    assert loss[0] == 0 and loss[5] == 0 and not dz[0].any() and not dz[5].any()
    loss, dz = _check(ops, z, torch.full_like(ids, -1), teacher, 1.0)
    assert not loss.any() and not dz.any()
    loss, dz = _check(ops, z, ids[:, :0], teacher[:, :0], 1.0)
    assert not loss.any() and not dz.any()


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_the_same_id_several_times(ops, type):
    gen = torch.Generator("cuda").manual_seed(2)
    z, ids, teacher = _inputs(6, 1000, 40, ref.TYPES[type], gen, missing=0.0)
    ids[0] = 999
    ids[1] = ids[1] % 3
    ids[2, ::2] = 5
    loss, dz = _check(ops, z, ids, teacher, 1.5)
    again = _check(ops, z, ids, teacher, 1.5)
    leaf = z.clone().requires_grad_()
    dloss = torch.ones(6, device="cuda")
    a, = torch.autograd.grad(ops.topk_distill_loss(leaf, ids, teacher, 1.5), leaf, dloss)
    b, = torch.autograd.grad(ops.topk_distill_loss(leaf, ids, teacher, 1.5), leaf, dloss)
    assert torch.equal(a, b) and torch.equal(loss, again[0])


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_masked_and_infinite_logits(ops, type):
    gen = torch.Generator("cuda").manual_seed(3)
    dtype = ref.TYPES[type]
    z, ids, teacher = _inputs(9, 3001, 4, dtype, gen, missing=0.0)
    z[0, 100:] = -INF                                 # masked columns
    ids[0] = torch.arange(4, device="cuda")
    z[1, 100:] = torch.finfo(dtype).min
    ids[1] = torch.arange(4, device="cuda")
    z[2, int(ids[2, 0])] = -INF                       # the teacher wants what the mask forbids: an infinite loss
    z[3] = -INF
    z[4, 17] = INF
    z[5, 2000] = float("nan")
    z[6] = torch.finfo(dtype).max
    z[7] = float("nan")
    ids[7] = -1                                       # no entries: no loss, whatever the logits
    z[8, :2999] = -INF
    ids[8] = 3000
    loss, dz = _check(ops, z, ids, teacher, 1.0, torch.ones(9, device="cuda"))
    assert torch.isinf(loss[2]) and torch.isnan(loss[[3, 4, 5]]).all() and loss[7] == 0 and not dz[7].any()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("tau", [0.05, 1.0, 30.0])
def test_temperatures_and_large_logits(ops, type, tau):
    gen = torch.Generator("cuda").manual_seed(4)
    z, ids, teacher = _inputs(40, 2000, 16, ref.TYPES[type], gen)
    # exponents of up to 50 / tau: each is within two roundings of its size, which the tolerances count for sizes of about
    # log(V); the mean of the exponents under the softmax stays that small at any temperature
    _check(ops, z, ids, teacher, tau)
    _check(ops, (z.float() + 300).to(z.dtype), ids, teacher, tau)


def test_strides_and_shapes(ops):
    gen = torch.Generator("cuda").manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        big, ids, teacher = _inputs(24, 1200, 10, dtype, gen)
        for z in (big[:, :1000], big[:, 7:1007], big[:, ::2], big[:1].expand(24, 1200), big.T.contiguous().T):
            _check(ops, z, ids % z.shape[1], teacher, 1.0)
        _check(ops, big, ids.T.contiguous().T, teacher[:, :1].expand(24, 10), 1.0)
        one, _ = _check(ops, big.reshape(2, 3, 4, 1200), ids.reshape(2, 3, 4, 10), teacher.reshape(2, 3, 4, 10), 1.0)
        assert torch.equal(one.reshape(-1), ops.topk_distill_loss(big, ids, teacher, 1.0))
        assert ops.topk_distill_loss(big[0], ids[0], teacher[0]).shape == ()
        assert torch.equal(ops.topk_distill_loss(big, ids, teacher.bfloat16()), ops.topk_distill_loss(big, ids, teacher.bfloat16().float()))
        # the gradient of a mean: one value for all rows
        leaf = big.clone().requires_grad_()
        ops.topk_distill_loss(leaf, ids, teacher).mean().backward()
        want, tol = ref.distill_grad(big, ids, teacher, 1.0, torch.full((24,), 1 / 24, device="cuda"))
        assert ref.outside(leaf.grad, want, tol) == 0
    assert ops.topk_distill_loss(big[:0], ids[:0], teacher[:0]).shape == (0,)
    leaf = big[:0].requires_grad_()
    assert torch.autograd.grad(ops.topk_distill_loss(leaf, ids[:0], teacher[:0]).sum(), leaf)[0].shape == (0, 1200)
    leaf = big[:, :0].detach().requires_grad_()
    loss = ops.topk_distill_loss(leaf, ids, teacher)
    assert not loss.any() and torch.autograd.grad(loss.sum(), leaf)[0].shape == (24, 0)


def test_gradient_against_differences(ops):
    gen = torch.Generator("cuda").manual_seed(6)
    z, ids, teacher = _inputs(4, 200, 6, torch.float32, gen)
    leaf, way, h = z.requires_grad_(), torch.randn((4, 200), device="cuda", generator=gen), 2.0 ** -6
    got, = torch.autograd.grad(ops.topk_distill_loss(leaf, ids, teacher, 1.3).sum(), leaf)
    with torch.no_grad():
        up, down = (ops.topk_distill_loss(leaf + s * h * way, ids, teacher, 1.3).double().sum() for s in (1, -1))
    # third derivatives of a log-sum-exp along a way are below 8 * (its largest value, about 4) ^ 3 / tau; roundings of the
    # losses (about 10 a row) are divided by 2 h
    room = 4 * (h * h / 6 * 8 * 64 / 1.3) + 4 * 16 * 2.0 ** -19 / (2 * h)
    assert abs(float((up - down) / (2 * h) - (got.double() * way.double()).sum())) < room


def test_no_second_derivative_and_none_of_the_teacher(ops):
    gen = torch.Generator("cuda").manual_seed(7)
    z, ids, teacher = _inputs(4, 50, 6, torch.float32, gen)
    leaf = z.requires_grad_()
    loss = ops.topk_distill_loss(leaf, ids, teacher)
    dz, = torch.autograd.grad(loss.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(dz.sum(), leaf)
    with pytest.raises(RuntimeError, match="teacher_logits"):
        ops.topk_distill_loss(leaf, ids, teacher.clone().requires_grad_())
    with torch.no_grad():
        ops.topk_distill_loss(leaf, ids, teacher.clone().requires_grad_())


def test_captured_and_on_another_stream(ops):
    gen = torch.Generator("cuda").manual_seed(8)
    side = torch.cuda.Stream()
    for T, V in ((3, 40_000), (400, 1001)):
        z, ids, teacher = _inputs(T, V, 12, torch.bfloat16, gen)
        dloss = torch.rand(T, device="cuda", generator=gen)
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            loss, stats = torch.ops.hpspmm.topk_distill(z, ids, teacher, 2.0)
            dz = torch.ops.hpspmm.topk_distill_backward(dloss, z, ids, teacher, stats, 2.0)
        for _ in range(2):
            fresh = _inputs(T, V, 12, torch.bfloat16, gen)
            for to, new in zip((z, ids, teacher), fresh):
                to.copy_(new)
            torch.cuda.synchronize()
            g.replay()
            with torch.cuda.stream(side):
                eager = torch.ops.hpspmm.topk_distill(z, ids, teacher, 2.0)
                dz2 = torch.ops.hpspmm.topk_distill_backward(dloss, z, ids, teacher, eager[1], 2.0)
            torch.cuda.synchronize()
            assert torch.equal(loss, eager[0]) and torch.equal(dz, dz2)
            want, tol = ref.distill(z, ids, teacher, 2.0)
            assert ref.outside(loss, want, tol) == 0


def test_more_than_2_31_elements(ops):
    T, V = 17_000, 131_075
    z = torch.zeros((T, V), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator("cuda").manual_seed(9)
    z[-2:] = torch.randn((2, V), device="cuda", generator=gen)
    ids = torch.full((T, 3), V - 1, device="cuda")
    teacher = torch.randn((T, 3), device="cuda", generator=gen)
    loss, stats = torch.ops.hpspmm.topk_distill(z, ids, teacher, 1.0)
    dloss = torch.ones(T, device="cuda")
    dz = torch.ops.hpspmm.topk_distill_backward(dloss, z, ids, teacher, stats, 1.0)
    for rows in (slice(T - 2, T), slice(0, 2)):
        want, tol = ref.distill(z[rows], ids[rows], teacher[rows], 1.0)
        assert ref.outside(loss[rows], want, tol) == 0
        want, tol = ref.distill_grad(z[rows], ids[rows], teacher[rows], 1.0, dloss[rows])
        assert ref.outside(dz[rows], want, tol) == 0


def test_refusals(ops, pkg, gpu_ctx):
    z, ids, teacher = torch.zeros((4, 9), device="cuda"), torch.zeros((4, 2), dtype=torch.int64, device="cuda"), torch.zeros((4, 2), device="cuda")
    ops.topk_distill_loss(z, ids, teacher, 1.0)
    for args in ((z.double(), ids, teacher, 1.0), (z, ids.float(), teacher, 1.0), (z, ids, teacher.double(), 1.0),
                 (z, ids[:3], teacher[:3], 1.0), (z, ids, teacher[:, :1], 1.0), (z, ids.cpu(), teacher, 1.0),
                 (z, ids, teacher.cpu(), 1.0), (z.cpu(), ids.cpu(), teacher.cpu(), 1.0), (z, ids, teacher, 0.0),
                 (z, ids, teacher, -1.0), (z, ids, teacher, float("nan")), (z, ids, teacher, INF), (z, ids[0], teacher[0], 1.0),
                 (z, ids[:, :1].expand(4, 1025), teacher[:, :1].expand(4, 1025), 1.0)):
        with pytest.raises(RuntimeError, match="hpspmm"):
            ops.topk_distill_loss(*args)
    loss, stats = torch.ops.hpspmm.topk_distill(z, ids, teacher, 1.0)
    back = torch.ops.hpspmm.topk_distill_backward
    for args in ((loss[:3], z, ids, teacher, stats, 1.0), (loss.double(), z, ids, teacher, stats, 1.0),
                 (loss, z, ids, teacher, stats[:3], 1.0), (loss.cpu(), z, ids, teacher, stats, 1.0), (loss, z, ids, teacher, stats, 0.0)):
        with pytest.raises(RuntimeError, match="hpspmm"):
            back(*args)
    good = [4, 9, 2, pkg.TYPE_F32, z.data_ptr(), 9, ids.data_ptr(), 8, teacher.data_ptr(), 1.0, loss.data_ptr(), stats.data_ptr()]
    gpu_ctx.topk_distill_forward(*good)
    for at, v in ((0, -1), (1, -1), (2, -1), (2, 1025), (3, 9), (4, None), (5, -1), (6, None), (7, 1), (8, None), (9, 0.0), (10, None)):
        with pytest.raises(pkg.HpspmmError):
            gpu_ctx.topk_distill_forward(*(good[:at] + [v] + good[at + 1:]))
    good = good[:10] + [stats.data_ptr(), loss.data_ptr(), 1, z.data_ptr()]
    gpu_ctx.topk_distill_backward(*good)
    for at, v in ((4, None), (8, None), (10, None), (11, None), (12, -1), (13, None), (9, -2.0)):
        with pytest.raises(pkg.HpspmmError):
            gpu_ctx.topk_distill_backward(*(good[:at] + [v] + good[at + 1:]))


def test_a_model_of_all_of_them(pkg, ops):
    """Vertices looked up, aggregated over the graph, one matrix for each type of vertex, the logits held against a teacher:
    loss and gradients of every parameter against the same model in 64 bits."""
    gen = torch.Generator("cuda").manual_seed(10)
    g = pkg.gen_rmat(9, 8, seed=3)
    M, K, V, types = g["M"], 32, 40, 5
    rp, ci, v = (torch.from_numpy(g[x]).cuda() for x in ("row_ptr", "col_idx", "vals"))
    layer = ops.TorchLayer(rp, ci, v, M, M, K)
    table = (torch.randn((300, K), device="cuda", generator=gen)).requires_grad_()
    W = (torch.randn((types, V, K), device="cuda", generator=gen) / 8).requires_grad_()
    weights = v.clone().requires_grad_()
    ids = torch.randint(-1, 300, (M,), device="cuda", generator=gen)
    kinds = torch.sort(torch.randint(0, types, (M,), device="cuda", generator=gen)).values
    offsets = torch.searchsorted(kinds, torch.arange(types + 1, device="cuda")).int()
    top = torch.randint(-1, V, (M, 6), device="cuda", generator=gen)
    teacher = torch.randn((M, 6), device="cuda", generator=gen)

    h = layer(ops.embedding(ids, table, 2.0), weights)
    loss = ops.topk_distill_loss(ops.grouped_product(h / 8, W.transpose(1, 2), offsets), top, teacher, 2.0).mean()
    got = torch.autograd.grad(loss, (table, weights, W))

    t, w, a = (x.detach().double().requires_grad_() for x in (table, W, weights))
    row = torch.repeat_interleave(torch.arange(M, device="cuda"), (rp[1:] - rp[:-1]).long())
    e = torch.where((ids >= 0)[:, None], t[ids.clamp(min=0)], 0.0) * 2.0
    h64 = torch.zeros((M, K), dtype=torch.float64, device="cuda").index_add(0, row, a[:, None] * e[ci.long()])
    z64 = torch.einsum("mk,mvk->mv", h64 / 8, w[kinds])
    p, logp, at, some = ref._teacher(z64, top, teacher, 2.0)
    logq = torch.log_softmax(z64 / 2, -1).gather(-1, at)
    want = (4 * torch.where(p > 0, p * (logp - logq), 0.0).sum(-1)).mean()
    exact = torch.autograd.grad(want, (t, a, w))
    # four stages of sums in 32 bits, up to 500 terms long: a few thousand roundings of the largest value at most
    assert abs(float(loss.detach() - want)) <= 4096 * ref.EPS32 * abs(float(want))
    for x, y in zip(got, exact):
        assert float((x.double() - y).abs().max()) <= 4096 * ref.EPS32 * float(y.abs().max())
    layer.close()


def test_the_operators_pass_through_a_tracer(ops):
    """Shape functions: fake tensors give the shapes, types and layouts of the real ones."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ids, table = torch.zeros((2, 3), dtype=torch.int64, device="cuda"), torch.zeros((7, 8), device="cuda")
    X, off = torch.zeros((6, 8), device="cuda"), torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    Wt = torch.zeros((2, 5, 8), device="cuda").transpose(1, 2)
    z, top, teacher = torch.zeros((2, 3, 9), device="cuda"), torch.zeros((2, 3, 4), dtype=torch.int32, device="cuda"), torch.zeros((2, 3, 4), device="cuda")
    o = torch.ops.hpspmm
    stats, loss = torch.zeros((6, 2), device="cuda"), torch.zeros((2, 3), device="cuda")
    calls = [(o.embedding, (ids, table, 2.0)), (o.embedding_backward, (torch.zeros((2, 3, 8), device="cuda"), ids, 7, 2.0)),
             (o.grouped_product, (X, Wt, off)), (o.grouped_weight_grad, (X, torch.zeros((6, 5), device="cuda"), off, True)),
             (o.grouped_weight_grad, (X, torch.zeros((6, 5), device="cuda"), off, False)), (o.topk_distill, (z, top, teacher, 1.0)),
             (o.topk_distill_backward, (loss, z, top, teacher, stats, 1.0))]
    for op, args in calls:
        real = op(*args)
        with FakeTensorMode() as mode:
            fake = op(*[mode.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args])
        for r, f in zip(real if isinstance(real, tuple) else (real,), fake if isinstance(fake, tuple) else (fake,)):
            assert (r.shape, r.dtype, r.stride()) == (f.shape, f.dtype, f.stride())


def test_a_captured_training_step(ops):
    """Lookup, product by group and loss with all their gradients as one graph, replayed on new inputs."""
    gen = torch.Generator("cuda").manual_seed(12)
    T, rows, K, V = 3000, 700, 64, 520
    ids, offsets = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.tensor([0, 1000, 1010, 3000], dtype=torch.int32, device="cuda")
    top, teacher = torch.zeros((T, 8), dtype=torch.int64, device="cuda"), torch.zeros((T, 8), device="cuda")
    table = torch.randn((rows, K), device="cuda", generator=gen).bfloat16().requires_grad_()
    W = (torch.randn((3, K, V), device="cuda", generator=gen) / 8).bfloat16().requires_grad_()

    def step():
        z = ops.grouped_product(ops.embedding(ids, table, 2.0), W, offsets)
        loss = ops.topk_distill_loss(z, top, teacher, 2.0).mean()
        return (loss.detach(), *torch.autograd.grad(loss, (table, W)))

    def fill():
        ids.copy_(torch.randint(-1, rows, (T,), device="cuda", generator=gen))
        top.copy_(torch.randint(-1, V, (T, 8), device="cuda", generator=gen))
        teacher.copy_(torch.randn((T, 8), device="cuda", generator=gen))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fill()
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        held = step()
    for _ in range(3):
        fill()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


def test_first_call_of_a_process_inside_a_capture():
    """Contexts and kernels are made ready there and then."""
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
ops = ref.ops_of(__graft_entry__.load_package())
ids, table = torch.tensor([1, 0, -1], device="cuda"), torch.randn((2, 64), device="cuda").bfloat16()
W, off = torch.randn((2, 64, 32), device="cuda").bfloat16(), torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
top, teacher = torch.tensor([[3], [4], [5]], device="cuda"), torch.zeros((3, 1), device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    x = ops.embedding(ids, table)
    z = ops.grouped_product(x, W, off)
    loss = ops.topk_distill_loss(z, top, teacher)
g.replay()
torch.cuda.synchronize()
want, tol = ref.grouped(x, W, off)
assert ref.outside(z, want, tol) == 0 and torch.equal(x[0], table[1]) and not x[2].any()
want, tol = ref.distill(z, top, teacher, 1.0)
assert ref.outside(loss, want, tol) == 0
print("well")
""" % (root, os.path.join(root, "tests"))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip().endswith("well"), out.stdout[-2000:]


def test_a_compiled_step_is_the_same(ops):
    """Through the tracer and PyTorch's ahead-of-time autograd: same loss, same gradients."""
    gen = torch.Generator("cuda").manual_seed(13)
    ids, top = (torch.randint(-1, n, shape, device="cuda", generator=gen) for n, shape in ((50, (300,)), (32, (300, 4))))
    table = torch.randn((50, 64), device="cuda", generator=gen).bfloat16().requires_grad_()
    W = torch.randn((2, 32, 64), device="cuda", generator=gen).bfloat16().transpose(1, 2).requires_grad_()
    offsets, teacher = torch.tensor([0, 100, 290], dtype=torch.int32, device="cuda"), torch.randn((300, 4), device="cuda", generator=gen)

    def step(ids, table, W):
        z = ops.grouped_product(ops.embedding(ids, table, 2.0), W, offsets)
        return ops.topk_distill_loss(z, top, teacher, 2.0).mean()

    first = step(ids, table, W)
    grads = torch.autograd.grad(first, (table, W))
    loss = torch.compile(step, backend="aot_eager", fullgraph=True)(ids, table, W)
    assert torch.equal(loss, first)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(loss, (table, W))))


@pytest.mark.parametrize("k", [63, 64, 65, 255, 256, 257, 1023])
def test_short_rows_and_long_teachers(ops, k):
    """Rows that a warp takes, with room for 64 or 256 entries, and rows that need a block for their entries alone."""
    gen = torch.Generator("cuda").manual_seed(k)
    for dtype in (torch.float32, torch.bfloat16):
        _check(ops, *_inputs(37, 1024, k, dtype, gen), 1.3)


@pytest.mark.parametrize("T", [1, 5, 37, 140])
def test_few_long_rows_again_and_again_on_a_busy_gpu(ops, T):
    """Clusters whose blocks find their SMs at different times, beside products on another stream: the same bits every time."""
    gen = torch.Generator("cuda").manual_seed(20 + T)
    z, ids, teacher = _inputs(T, 40_000, 9, torch.bfloat16, gen)
    A = torch.randn((2048, 2048), device="cuda", generator=gen).bfloat16()
    want, tol = ref.distill(z, ids, teacher, 1.0)
    first = torch.ops.hpspmm.topk_distill(z, ids, teacher, 1.0)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    held = []
    for _ in range(60):
        with torch.cuda.stream(two):
            A @ A
        with torch.cuda.stream(one):
            held.append(torch.ops.hpspmm.topk_distill(z, ids, teacher, 1.0))
    torch.cuda.synchronize()
    assert ref.outside(first[0], want, tol) == 0
    for loss, stats in held:
        assert torch.equal(loss, first[0]) and torch.equal(stats, first[1])


@pytest.mark.parametrize("off", [0, 1])
def test_a_row_of_nearly_2_31_columns(ops, off):
    """All logits 0 but four: the sum over the row is known, and so is every value of the gradient."""
    torch.cuda.empty_cache()
    V = 2 ** 31 - 2 - off
    z = torch.zeros(2 ** 31 - 2, dtype=torch.bfloat16, device="cuda")[off:][None]
    ids = torch.tensor([[7, V - 1, V - 2, V]], device="cuda")                 # (the last one is no column)
    logits = torch.tensor([4.0, 5.0, 3.0], dtype=torch.float64, device="cuda")
    z[0, ids[0, :3]] = logits.bfloat16()
    z[0, V // 2] = 6.0
    teacher = torch.tensor([[1.0, 0.5, 2.0, 9.0]], device="cuda")
    loss, stats = torch.ops.hpspmm.topk_distill(z, ids, teacher, 1.0)
    total = float(logits.exp().sum()) + float(torch.tensor(6.0).double().exp()) + (V - 4)
    p = torch.softmax(teacher[0, :3].double(), 0)
    want = float((p * (p.log() - (logits - torch.tensor(total).double().log().cuda()))).sum())
    assert abs(float(loss[0]) - want) <= 2.0 ** -18 * want
    dz = torch.ops.hpspmm.topk_distill_backward(torch.ones(1, device="cuda"), z, ids, teacher, stats, 1.0)[0]
    # two roundings of the exponent's parts (up to 6 of 2^-24 relative to values of up to 9), ex2, the sum, one of bf16
    room = torch.finfo(torch.bfloat16).eps / 2 * (1 + 2.0 ** -6)
    want = torch.cat((logits.exp() / total - p, torch.tensor([6.0], device="cuda").double().exp() / total))
    at = torch.cat((ids[0, :3], torch.tensor([V // 2], device="cuda")))
    assert bool(((dz[at].double() - want).abs() <= room * want.abs()).all())
    dz[at] = float(dz[0])
    assert abs(float(dz[0]) * total - 1) <= room
    assert all(bool((c == dz[0]).all()) for c in dz.split(1 << 28))
    del z, dz
    torch.cuda.empty_cache()


@pytest.mark.parametrize("V,k", [(29, 6), (5000, 6), (700, 200), (40_000, 6)])
def test_teachers_that_are_no_number_do_not_count(ops, V, k):
    """An entry counts when its logit is above -infinity, which NaN is not, whatever its id."""
    gen = torch.Generator("cuda").manual_seed(32)
    for dtype in (torch.float32, torch.bfloat16):
        z, ids, teacher = _inputs(6, V, k, dtype, gen, missing=0.0)
        teacher[0, 0] = float("nan")
        teacher[1, 1:] = float("nan")                 # one is left
        teacher[2] = float("nan")                     # none is left
        teacher[3, 1], ids[3, 2] = float("nan"), ids[3, 1]      # a column that another entry names too
        teacher[4, :2], teacher[4, 2:4] = float("nan"), -INF
        loss, dz = _check(ops, z, ids, teacher, 1.3)
        assert loss[2] == 0 and not dz[2].any() and bool(torch.isfinite(loss).all()) and bool(torch.isfinite(dz).all())


def test_statistics_on_any_4_bytes(ops, pkg, gpu_ctx):
    """They are T x 2 floats and may begin where floats may."""
    gen = torch.Generator("cuda").manual_seed(37)
    for T, V in ((5, 300), (40, 3001), (3, 40_000)):
        z, ids, teacher = _inputs(T, V, 7, torch.float32, gen)
        loss, stats = torch.ops.hpspmm.topk_distill(z, ids, teacher, 1.2)
        room = torch.full((2 * T + 3,), 7.0, device="cuda")
        odd, loss2 = room[1:2 * T + 1], torch.empty_like(loss)
        torch.cuda.synchronize()
        gpu_ctx.topk_distill_forward(T, V, 7, pkg.TYPE_F32, z.data_ptr(), V, ids.data_ptr(), 8, teacher.data_ptr(), 1.2, loss2.data_ptr(), odd.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(odd.view(T, 2), stats) and torch.equal(loss, loss2) and bool((room[[0, -2, -1]] == 7).all())
        dloss, back = torch.ones(T, device="cuda"), torch.ops.hpspmm.topk_distill_backward
        assert torch.equal(back(dloss, z, ids, teacher, odd.view(T, 2), 1.2), back(dloss, z, ids, teacher, stats, 1.2))


def test_arrays_off_their_elements_are_refused(pkg, gpu_ctx):
    """Every array of every dense operator, by one byte and by half an element: the host says no before anything is launched."""
    t = torch.zeros(4096, device="cuda")
    a, f32, bf16 = t.data_ptr(), pkg.TYPE_F32, pkg.TYPE_BF16
    calls = [(gpu_ctx.embedding_forward, [4, 4, 4, f32, a, 8, a, 4, 1.0, a], {4: 4, 6: 2, 9: 2}),
             (gpu_ctx.embedding_forward, [4, 4, 4, bf16, a, 4, a, 4, 1.0, a], {4: 2, 6: 1, 9: 1}),
             (gpu_ctx.embedding_backward, [4, 4, 4, f32, a, 8, a, 4, 1.0, a, a, 16384], {4: 4, 6: 2, 9: 2, 10: 128}),
             (gpu_ctx.embedding_backward, [4, 4, 4, bf16, a, 4, a, 4, 1.0, a, a, 16384], {4: 2, 6: 1, 9: 1}),
             (gpu_ctx.grouped_product, [4, 1, 4, 4, f32, a, 4, a, 0, a, a], {5: 2, 7: 2, 9: 2, 10: 2}),
             (gpu_ctx.grouped_product, [4, 1, 4, 4, bf16, a, 4, a, 1, a, a], {5: 1, 7: 1, 9: 2, 10: 1}),
             (gpu_ctx.grouped_weight_grad, [4, 1, 4, 4, f32, a, 4, a, 4, a, a, 0], {5: 2, 7: 2, 9: 2, 10: 2}),
             (gpu_ctx.grouped_weight_grad, [4, 1, 4, 4, bf16, a, 4, a, 4, a, a, 1], {5: 1, 7: 1, 9: 2, 10: 1}),
             (gpu_ctx.topk_distill_forward, [4, 4, 2, f32, a, 4, a, 8, a, 1.0, a, a], {4: 2, 6: 4, 8: 2, 10: 2, 11: 2}),
             (gpu_ctx.topk_distill_backward, [4, 4, 2, bf16, a, 4, a, 4, a, 1.0, a, a, 1, a], {4: 1, 6: 2, 8: 2, 10: 2, 11: 2, 13: 1})]
    for call, args, places in calls:
        for at, off in places.items():
            for by in {off, 1}:
                with pytest.raises(pkg.HpspmmError) as e:
                    call(*(args[:at] + [a + by] + args[at + 1:]))
                assert e.value.status == pkg.ERR_INVALID

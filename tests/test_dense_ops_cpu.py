"""What the dense operators by index say without a GPU: CPU tensors and bad arguments are refused, shapes are known."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
import dense_reference as ref  # noqa: E402


def test_cpu_tensors_are_refused(pkg):
    ops = ref.ops_of(pkg)
    ids, x = torch.zeros(3, dtype=torch.int64), torch.zeros((3, 4))
    off = torch.zeros(2, dtype=torch.int32)
    calls = [lambda: ops.embedding(ids, x), lambda: torch.ops.hpspmm.embedding_backward(x, ids, 5, 1.0),
             lambda: ops.grouped_product(x, torch.zeros((1, 4, 2)), off),
             lambda: torch.ops.hpspmm.grouped_weight_grad(x, x, off, False),
             lambda: ops.topk_distill_loss(x, torch.zeros((3, 2), dtype=torch.int64), torch.zeros((3, 2))),
             lambda: torch.ops.hpspmm.topk_distill_backward(x[:, 0], x, torch.zeros((3, 2), dtype=torch.int64),
                                                            torch.zeros((3, 2)), torch.zeros((3, 2)), 1.0)]
    for f in calls:
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


def test_null_contexts_are_refused(pkg):
    lib = pkg.load_library()
    i64 = ctypes.c_int64
    for name in ("embedding_forward", "embedding_backward", "grouped_product", "grouped_weight_grad", "topk_distill_forward",
                 "topk_distill_backward"):
        args = [0 if t in (i64, ctypes.c_int32, ctypes.c_size_t) else 1.0 if t is ctypes.c_float else None
                for t in pkg.PROTOTYPES["hpspmm_" + name][1]]
        assert getattr(lib, "hpspmm_" + name)(*args) == pkg.ERR_INVALID


def test_workspace_sizes(pkg):
    need = pkg.load_library().hpspmm_embedding_backward_workspace
    assert need(0, 5, 5) >= 0 and need(-1, 5, 5) == -1 and need(5, -1, 5) == -1 and need(5, 5, -1) == -1
    assert need(1 << 31, 5, 5) == -1 and need(5, 1 << 31, 5) == -1
    last = 0
    for T in (1, 100, 8192, 8193, 1 << 20, 1 << 26):      # grows with the batch, stays far below the operands
        got = need(T, 100_000, 64)
        assert got >= 8 * T and got >= last
        last = got


def test_no_block_writes_into_a_cluster_before_all_of_it_runs():
    """A block that has not started has no shared memory to write into: in every kernel that stores into another block's, a
    wait for the cluster comes first.  (Nothing else shows its absence: the blocks of a cluster mostly start together.)"""
    import glob
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hp-spmm-sddmm_b200", "csrc")
    seen = 0
    for path in sorted(glob.glob(os.path.join(csrc, "*.cu"))):
        source = re.sub(r"//[^\n]*", "", open(path).read())
        for kernel in source.split("__global__")[1:]:
            body = kernel[:kernel.index("\n}\n")]
            store = re.search(r"st\.shared::cluster", body)
            if store:
                seen += 1
                before = body[:store.start()]
                waits = [before.find(x) for x in ("cluster_wait()", "barrier.cluster.wait")]
                arrives = [before.find(x) for x in ("cluster_arrive()", "barrier.cluster.arrive")]
                assert max(waits) >= 0 and max(arrives) >= 0, path
                assert min(x for x in arrives if x >= 0) < min(x for x in waits if x >= 0), path
    assert seen == 2


def test_sizes_whose_last_tile_would_pass_2_31(pkg):
    """Rows and columns of the grouped products: what the kernels add to fill a tile has to stay below 2^31."""
    need = pkg.load_library().hpspmm_grouped_weight_grad_workspace
    most = 2 ** 31 - 1026
    for type in (pkg.TYPE_F32, pkg.TYPE_BF16):
        for out_first in (0, 1):
            assert need(most, 1, 8, 8, type, out_first) > 0 and need(5, 1, most, 8, type, out_first) == 0
            for sizes in ((most + 1, 1, 8, 8), (2 ** 31 - 2, 1, 8, 8), (5, 1, most + 1, 8), (5, 1, 8, most + 1), (5, 2 ** 20 + 1, 8, 8)):
                assert need(*sizes, type, out_first) == -1


def test_waits_are_asked_for_on_a_gpu(pkg):
    for device in ("cpu", torch.device("meta")):
        with pytest.raises(RuntimeError, match="hpspmm: waits are counted on a CUDA device"):
            ref.ops_of(pkg).timeouts(device)

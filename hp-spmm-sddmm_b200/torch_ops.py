"""PyTorch front-end of the aggregation layer and of what stands beside it: autograd over the C ABI, no PyTorch arithmetic.

    layer = TorchLayer(row_ptr, col_idx, vals, M, N, max_K)   # CUDA tensors, int32 / int32 / float32
    C = layer(H)                                              # C = A·H, differentiable in H and in vals
    C.sum().backward()                                        # dH = Aᵀ·dC (SpMM), dvals = SDDMM(dC, H)

    E = embedding(ids, table, scale)                          # rows of a table by id, differentiable in the table
    Y = grouped_product(X, W, offsets)                        # one matrix for each group of rows, differentiable in X and W
    loss = topk_distill_loss(logits, teacher_ids, teacher_logits, temperature)   # one value a row

For the layer four operators are registered under the namespace ``hpspmm`` (``layer_forward``,
``layer_backward_features``, ``layer_backward_weights``, and ``layer_backward`` for both gradients at
once) by csrc/torch_binding.cpp, with an autograd formula that chains them; the shape functions for tracing are below, so the layer can sit inside a
compiled or exported module.  The three functions have six more (csrc/torch_dense_binding.cpp): ``embedding``,
``grouped_product`` and ``topk_distill`` with their gradients.  Every operator calls libhpspmm.so on the current
CUDA stream of the input's device; a CPU tensor is rejected (there is no fallback).  PyTorch supplies
memory, streams and the autograd tape only.

The reference has no framework binding; this is the caller either side of its products
(test/test_all.cpp:63-107 issues them one at a time from a C++ driver).
"""
import itertools
import os

import torch
from torch.overrides import has_torch_function_variadic

from . import PKG_DIR, Context, Layer, load_extension

_layers = {}      # what a layer id stands for: the shapes, and what has to stay alive
_ids = itertools.count(1)

_C = load_extension("_hpspmm_torch", os.path.join(PKG_DIR, "lib", "_hpspmm_torch.so"))

layer_forward = torch.ops.hpspmm.layer_forward.default
layer_backward_features = torch.ops.hpspmm.layer_backward_features.default
layer_backward_weights = torch.ops.hpspmm.layer_backward_weights.default
layer_backward = torch.ops.hpspmm.layer_backward.default


def _entry(layer_id):
    try:
        return _layers[layer_id]
    except KeyError:
        raise RuntimeError("hpspmm: unknown or closed layer id %d" % layer_id) from None


@torch.library.register_fake("hpspmm::layer_forward")
def _(H, vals, layer_id):
    return H.new_empty((_entry(layer_id)["M"], H.shape[1]))


@torch.library.register_fake("hpspmm::layer_backward_features")
def _(dC, vals, layer_id):
    return dC.new_empty((_entry(layer_id)["N"], dC.shape[1]))


@torch.library.register_fake("hpspmm::layer_backward_weights")
def _(dC, H, layer_id):
    return dC.new_empty((_entry(layer_id)["nnz"],))


@torch.library.register_fake("hpspmm::layer_backward")
def _(dC, H, vals, layer_id):
    e = _entry(layer_id)
    return dC.new_empty((e["N"], dC.shape[1])), dC.new_empty((e["nnz"],))


class TorchLayer:
    """A sparse operand A (CSR on one GPU) as a differentiable map H -> A·H."""

    def __init__(self, row_ptr, col_idx, vals, M, N, max_K):
        for t, dt, what in ((row_ptr, torch.int32, "row_ptr"), (col_idx, torch.int32, "col_idx"),
                            (vals, torch.float32, "vals")):
            if not t.is_cuda or t.dtype != dt or not t.is_contiguous():
                raise RuntimeError("hpspmm: %s must be a contiguous CUDA %s tensor" % (what, dt))
        if row_ptr.numel() != M + 1 or col_idx.numel() != vals.numel():
            raise RuntimeError("hpspmm: CSR arrays disagree with M or with each other")
        self.M, self.N, self.nnz, self.max_K = int(M), int(N), int(vals.numel()), int(max_K)
        self.row_ptr, self.col_idx, self.vals = row_ptr, col_idx, vals
        dev = row_ptr.device
        # One context per layer.  A context owns scratch and a flag that plan building uses (also lazily, on
        # the first product of a new width class), and calls that share a context must not overlap on the
        # GPU: with a context of their own, two layers driven from different streams or threads cannot meet
        # there.  Products of ONE layer still must not overlap with each other.
        ctx = Context(dev.index if dev.index is not None else torch.cuda.current_device())
        with torch.cuda.device(dev):
            v = vals.detach()
            layer = Layer(ctx, self.M, self.N, self.nnz, row_ptr.data_ptr(), col_idx.data_ptr(), v.data_ptr(),
                          self.max_K, torch.cuda.current_stream().cuda_stream)
        self.layer_id = next(_ids)
        _layers[self.layer_id] = {"layer": layer, "ctx": ctx, "M": self.M, "N": self.N, "nnz": self.nnz,
                                  "keep": (row_ptr, col_idx)}
        _C.register_layer(self.layer_id, ctx.handle.value, layer.handle.value, self.M, self.N, self.nnz, v)

    def __call__(self, H, vals=None):
        if vals is None:
            vals = self.vals
        # tracers, tensor subclasses and function modes see the call through __torch_function__
        if (torch.compiler.is_compiling() or not isinstance(H, torch.Tensor) or not isinstance(vals, torch.Tensor)
                or has_torch_function_variadic(H, vals)):
            return layer_forward(H, vals, self.layer_id)
        return _C.layer_forward(H, vals, self.layer_id)    # the same operator without the Python dispatcher's share

    def close(self):
        e = _layers.pop(self.layer_id, None)
        if e:
            _C.forget_layer(self.layer_id)
            e["layer"].close()
            e["ctx"].close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- dense operands by index -----------------------------------------------------------------------------------

def _plain(*tensors):
    """Whether a call may skip the Python dispatcher: tracers, tensor subclasses and function modes have to see it."""
    return not (torch.compiler.is_compiling() or not all(isinstance(t, torch.Tensor) for t in tensors)
                or has_torch_function_variadic(*tensors))


@torch.library.register_fake("hpspmm::embedding")
def _(ids, table, scale):
    return table.new_empty((*ids.shape, table.shape[1]))


@torch.library.register_fake("hpspmm::embedding_backward")
def _(grad, ids, rows, scale):
    return grad.new_empty((rows, grad.shape[-1]))


@torch.library.register_fake("hpspmm::grouped_product")
def _(X, W, offsets):
    return X.new_empty((X.shape[0], W.shape[2]))


@torch.library.register_fake("hpspmm::grouped_weight_grad")
def _(X, dY, offsets, transposed):
    G, K, N = offsets.shape[0] - 1, X.shape[1], dY.shape[1]
    return X.new_empty((G, N, K)).transpose(1, 2) if transposed else X.new_empty((G, K, N))


@torch.library.register_fake("hpspmm::topk_distill")
def _(logits, teacher_ids, teacher_logits, temperature):
    loss = logits.new_empty(logits.shape[:-1], dtype=torch.float32)
    return loss, loss.new_empty((loss.numel(), 2))


@torch.library.register_fake("hpspmm::topk_distill_backward")
def _(dloss, logits, teacher_ids, teacher_logits, stats, temperature):
    return logits.new_empty(logits.shape)


def embedding(ids, table, scale=1.0):
    """``scale * table[ids]``: ids int32 or int64 of any shape, table [N, K] in float32, float16 or bfloat16.

    An id outside [0, N) (the -1 of a padded batch) gives a row of zeros and takes no part in the gradient.  The
    gradient of the table is dense, summed in 32 bits in an order that does not change from call to call.  A routed
    layer's rows by slot are such a lookup too, and their gradient such a sum."""
    if _plain(ids, table):
        return _C.embedding(ids, table, scale)
    return torch.ops.hpspmm.embedding.default(ids, table, scale)


def grouped_product(X, W, offsets):
    """``Y[r] = X[r] @ W[g]`` for the rows offsets[g] <= r < offsets[g + 1]: X [R, K], W [G, K, N], offsets [G + 1]
    ascending int32 on the GPU.  Rows of no group (behind the last one of a padded batch) become zeros.

    W may be the transpose of a contiguous [G, N, K] (``W.transpose(1, 2)`` of the weights of linear layers): it is
    read as it lies, and its gradient lies the same way.  float32, float16 or bfloat16, all of one type.

    Waits inside the 16-bit kernels are bounded; one that runs out spoils its call, which a later call reports (``timeouts``)."""
    if _plain(X, W, offsets):
        return _C.grouped_product(X, W, offsets)
    return torch.ops.hpspmm.grouped_product.default(X, W, offsets)


def topk_distill_loss(logits, teacher_ids, teacher_logits, temperature=1.0):
    """``temperature**2 * KL(teacher || student)`` of every row, the teacher known by its k largest logits: logits
    [..., V], teacher_ids (int32 or int64) and teacher_logits [..., k], k up to 1024; float32 [...] comes out.

    The teacher's softmax runs over the entries whose id lies in [0, V) and whose logit is above -inf (NaN is not); a
    row without any has loss 0 and a gradient of zeros.  Differentiable in the logits, once."""
    if _plain(logits, teacher_ids, teacher_logits):
        return _C.topk_distill(logits, teacher_ids, teacher_logits, temperature)
    return torch.ops.hpspmm.topk_distill.default(logits, teacher_ids, teacher_logits, temperature)[0]


def timeouts(device=None):
    """How many blocks of the grouped products' tensor-core kernels have given up a wait on this GPU (expected 0; what
    such a call wrote is not to be used).  Waits for the device.  The first call of these operators that finds such a product
    done raises an error by itself; after a last step, or replays of a graph, ask here."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise RuntimeError("hpspmm: waits are counted on a CUDA device, got %s" % device)
    return _C.timeouts(torch.cuda.current_device() if device.index is None else device.index)

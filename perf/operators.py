"""The operators around the sparse products that training and serving time: rows of a table by id, one matrix for each
group of rows, a loss against the largest logits of a teacher.

listed() names twelve calls over the real range of sizes, draw() gives more of the same ranges, prepare() makes what a
program holds before the call, run() is one pass, exact() the same from the definitions in 64 bits.

The operations:
  embedding  out[t] = scale * table[id[t]]; an id outside the table gives a row of zeros
  grouped    Y[r] = X[r] W[g] for the rows offsets[g] <= r < offsets[g + 1] of group g; rows of no group give zeros
  distill    tau^2 sum_j p_j (log p_j - log_softmax(z / tau)[id_j]) for every row z of logits, with p the softmax of the
             teacher's k values divided by tau over the entries whose id lies in the row; 0 where there is none
A case with "train" returns the gradients too.

Ids are drawn by rank, p(i) proportional to 1 / (i + 3), as tokens and the vertices of power-law graphs come.  Groups get
uneven shares, log-normally spread.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAME = "hp_spmm_sddmm_b200"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    """The package lies in a directory whose name has hyphens, so it is imported by path (from the working folder)."""
    if NAME not in sys.modules:
        init = os.path.join(os.getcwd(), "hp-spmm-sddmm_b200", "__init__.py")
        if not os.path.exists(init):
            init = os.path.join(ROOT, "hp-spmm-sddmm_b200", "__init__.py")
        spec = importlib.util.spec_from_file_location(NAME, init)
        mod = importlib.util.module_from_spec(spec)
        sys.modules[NAME] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module(NAME + ".torch_ops")


def _embedding(name, type, ids, rows, cols, scale, missing, train):
    """ids tokens out of a table of rows x cols; missing: the share of positions that hold -1 (padding)."""
    return {"name": name, "op": "embedding", "type": type, "ids": ids, "rows": rows, "cols": cols, "scale": scale,
            "missing": missing, "train": train}


def _grouped(name, type, rows, groups, k, n, spread, spare, out_first, train):
    """spread: of the logarithm of the groups' shares; spare: rows behind the last group; out_first: weights lie [G, n, k]."""
    return {"name": name, "op": "grouped", "type": type, "rows": rows, "groups": groups, "k": k, "n": n,
            "spread": spread, "spare": spare, "out_first": out_first, "train": train}


def _distill(name, type, rows, cols, k, tau, missing, train):
    """missing: the share of the teacher's entries that hold no id (-1)."""
    return {"name": name, "op": "distill", "type": type, "rows": rows, "cols": cols, "k": k, "tau": tau,
            "missing": missing, "train": train}


def listed():
    return [
        # one step of a decoder: a token for each of 32 sequences
        _embedding("lookup-32", "bf16", 32, 131_072, 2048, 45.25, 0.0, False),
        # a training step's tokens, lookup and gradient of a vocabulary-sized table
        _embedding("embed-train-16k", "bf16", 16_384, 131_072, 1024, 32.0, 0.0, True),
        # learned vertex features in 32 bits, an odd number of vertices and positions, padded with -1
        _embedding("embed-train-vertices", "f32", 50_003, 169_999, 100, 1.0, 0.05, True),
        # the largest: a long batch through a wide table
        _embedding("embed-train-256k", "bf16", 262_144, 262_144, 2048, 1.0, 0.02, True),
        # one step of a decoder through a routed layer: a few rows for each group, the batch padded
        _grouped("grouped-step-56", "bf16", 56, 64, 2048, 1536, 0.5, 8, False, False),
        # a prompt through a routed layer, weights [G, out, in]
        _grouped("grouped-prompt-16k", "bf16", 16_384, 32, 2048, 2816, 0.4, 0, True, False),
        # a training step of a routed layer: product and both gradients
        _grouped("grouped-train-32k", "bf16", 32_768, 8, 2048, 5632, 0.3, 0, False, True),
        # one matrix for each relation type of a graph, in 32 bits as the aggregation layers are, a few rows of padding
        _grouped("grouped-train-relations", "f32", 100_003, 47, 100, 64, 0.8, 29, False, True),
        # widths that fit no vector, in 16 bits
        _grouped("grouped-train-odd", "f16", 5_003, 13, 333, 131, 0.6, 0, False, True),
        # a training step against a teacher's 64 largest logits over a vocabulary
        _distill("distill-train-4k", "bf16", 4_096, 131_072, 64, 2.0, 0.0, True),
        # an odd vocabulary in 32 bits, teachers of different lengths
        _distill("distill-train-odd", "f32", 1_021, 32_003, 20, 1.0, 0.3, True),
        # a few positions of a sequence scored against a teacher
        _distill("distill-score-8", "f16", 8, 131_072, 100, 1.0, 0.0, False),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("embedding", "grouped", "grouped", "distill"))
    type = rng.choice(("bf16", "bf16", "f16", "f32"))
    train = rng.random() < 0.7
    if op == "embedding":
        cols = 64 * rng.randint(1, 48) if rng.random() < 0.6 else log_int(3, 3000)
        rows = log_int(500, min(400_000, 500_000_000 // cols))
        ids = log_int(1, min(400_000, 500_000_000 // cols))
        return _unnamed(_embedding(None, type, ids, rows, cols, rng.choice((1.0, 0.5, round(math.sqrt(cols), 3))),
                                   rng.choice((0.0, 0.0, 0.1, 0.4)), train))
    if op == "grouped":
        wide = type != "f32" and rng.random() < 0.7
        k, n = (64 * rng.randint(2, 48) if wide else log_int(8, 700) for _ in range(2))
        groups = log_int(1, min(200, max(2, 400_000_000 // (k * n))))
        rows = log_int(1, min(60_000, max(100, int(3e11 if wide else 2e10) // (k * n))))
        return _unnamed(_grouped(None, type, rows, groups, k, n, round(rng.uniform(0.0, 0.9), 2),
                                 rng.choice((0, 0, 7, 40)), rng.random() < 0.5, train))
    cols = 64 * rng.randint(100, 2500) if rng.random() < 0.5 else log_int(40, 160_000)
    rows = log_int(1, min(20_000, (300_000_000 if type == "f32" else 500_000_000) // cols))
    return _unnamed(_distill(None, type, rows, cols, min(cols // 2, log_int(1, 128)),
                             rng.choice((1.0, 2.0, round(rng.uniform(0.5, 4.0), 2))), rng.choice((0.0, 0.0, 0.3, 0.9)),
                             train))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


# ---- inputs --------------------------------------------------------------------------------------------------

def _by_rank(count, n, gen):
    """`count` draws of 0..n-1, i with a weight of 1 / (i + 3)."""
    edge = torch.log(torch.arange(n + 1, device="cuda", dtype=torch.float64) + 2.5)
    u = torch.rand(count, device="cuda", dtype=torch.float64, generator=gen)
    at = torch.searchsorted(edge, edge[0] + u * (edge[-1] - edge[0]), right=True) - 1
    return at.clamp_(0, n - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = TYPES[case["type"]], case["op"]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    st = dict(case)
    if op == "embedding":
        ids = _by_rank(case["ids"], case["rows"], gen)
        ids[torch.rand(case["ids"], device="cuda", generator=gen) < case["missing"]] = -1
        st["id"] = ids
        st["table"] = normal(case["rows"], case["cols"]).to(dtype).requires_grad_(case["train"])
        if case["train"]:
            st["dout"] = normal(case["ids"], case["cols"]).to(dtype)
    elif op == "grouped":
        rows, groups, k, n = (case[x] for x in ("rows", "groups", "k", "n"))
        share = torch.exp(case["spread"] * normal(groups).double())
        edge = torch.cumsum(share, 0) / share.sum()
        which = torch.searchsorted(edge, torch.rand(rows, device="cuda", dtype=torch.float64, generator=gen))
        sizes = torch.bincount(which.clamp_(max=groups - 1), minlength=groups)
        st["offsets"] = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
        st["offsets"][1:] = sizes.cumsum(0)
        st["most"] = int(sizes.max())                    # the most rows of one group: what the plain form pads to
        st["X"] = normal(rows + case["spare"], k).to(dtype).requires_grad_(case["train"])
        w = normal(groups, *((n, k) if case["out_first"] else (k, n))) / math.sqrt(k)
        st["W"] = (w.to(dtype).transpose(1, 2) if case["out_first"] else w.to(dtype)).requires_grad_(case["train"])
        if case["train"]:
            st["dY"] = normal(rows + case["spare"], n).to(dtype)
    else:
        rows, cols, k = case["rows"], case["cols"], case["k"]
        # distinct ids in every row: a stride that shares no factor with the number of columns
        step = next(s for s in range(int(cols * 0.618) + 1, 2 * cols + 2) if math.gcd(s, cols) == 1)
        first = torch.randint(cols, (rows, 1), device="cuda", generator=gen)
        ids = (first + torch.arange(k, device="cuda") * step) % cols
        ids[torch.rand((rows, k), device="cuda", generator=gen) < case["missing"]] = -1
        st["id"] = ids
        z = normal(rows, cols) * 2
        st["teacher"] = (normal(rows, k) * 2 + 6).sort(-1, descending=True).values
        st["z"] = z.to(dtype).requires_grad_(case["train"])       # the student knows nothing of the teacher yet
        if case["train"]:
            st["dloss"] = torch.full((), 1.0 / rows, device="cuda").expand(rows)    # of the mean over the rows
    return st


# ---- one pass ------------------------------------------------------------------------------------------------

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    ops = _ops()
    if st["op"] == "embedding":
        out = ops.embedding(st["id"], st["table"], st["scale"])
        if not st["train"]:
            return {"out": out}
        return {"out": out.detach(), "dtable": torch.autograd.grad(out, st["table"], st["dout"])[0]}
    if st["op"] == "grouped":
        y = ops.grouped_product(st["X"], st["W"], st["offsets"])
        if not st["train"]:
            return {"Y": y}
        dx, dw = torch.autograd.grad(y, (st["X"], st["W"]), st["dY"])
        return {"Y": y.detach(), "dX": dx, "dW": dw}
    loss = ops.topk_distill_loss(st["z"], st["id"], st["teacher"], st["tau"])
    if not st["train"]:
        return {"loss": loss}
    return {"loss": loss.detach(), "dz": torch.autograd.grad(loss, st["z"], st["dloss"])[0]}


def _run_plain(st):
    with torch.no_grad():
        return {"embedding": _plain_embedding, "grouped": _plain_grouped, "distill": _plain_distill}[st["op"]](st)


def _plain_embedding(st):
    ids, table = st["id"], st["table"]
    held = (ids >= 0) & (ids < table.shape[0])
    row = torch.where(held, ids, 0)
    out = {"out": (table[row].float() * held[:, None] * st["scale"]).to(table.dtype)}
    if st["train"]:
        d = torch.zeros(table.shape, dtype=torch.float32, device="cuda")
        d.index_add_(0, row, st["dout"].float() * held[:, None])
        out["dtable"] = (d * st["scale"]).to(table.dtype)
    return out


def _plain_grouped(st):
    X, W, off, most = st["X"], st["W"].float(), st["offsets"].long(), st["most"]
    groups = W.shape[0]
    # every group padded to the longest one, so that one batched product does them all
    at = off[:-1, None] + torch.arange(most, device="cuda")
    held = at < off[1:, None]
    at = torch.where(held, at, X.shape[0])               # a row behind the last one, of zeros, stands for none

    def padded(t):
        t = torch.cat((t.float(), t.new_zeros((1, t.shape[1]), dtype=torch.float32)))
        return t[at.view(-1)].view(groups, most, -1)

    def back(t):
        out = t.new_zeros((X.shape[0] + 1, t.shape[-1]))
        out[at.view(-1)] = t.view(-1, t.shape[-1])
        return out[:-1].to(X.dtype)

    x = padded(X)
    out = {"Y": back(torch.bmm(x, W))}
    if st["train"]:
        dy = padded(st["dY"])
        out["dX"] = back(torch.bmm(dy, W.transpose(1, 2)))
        out["dW"] = torch.bmm(x.transpose(1, 2), dy).to(X.dtype)
    return out


def _plain_distill(st):
    ids, tau = st["id"], st["tau"]
    z = st["z"].float() / tau
    held = (ids >= 0) & (ids < z.shape[1]) & (st["teacher"] > -math.inf)
    at = torch.where(held, ids, 0)
    t = torch.where(held, st["teacher"].float() / tau, torch.finfo(torch.float32).min)
    some = held.any(-1, keepdim=True)
    t = t - t.amax(-1, keepdim=True)
    e = torch.exp(t) * held
    total = e.sum(-1, keepdim=True)
    p = torch.where(some, e / total, 0.0)
    most = z.amax(-1, keepdim=True)
    lse = most + torch.log(torch.exp(z - most).sum(-1, keepdim=True))
    term = p * (t - torch.log(total) - (z.gather(1, at) - lse))
    out = {"loss": torch.where(p > 0, term, 0.0).sum(-1) * tau ** 2}
    if st["train"]:
        dz = torch.exp(z - lse) * some
        dz.scatter_add_(1, at, -p)
        out["dz"] = (dz * (st["dloss"][:, None] * tau)).to(st["z"].dtype)
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    """Bytes and operations of a pass: each input read once, each output written once."""
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "embedding":
        ids, rows, cols = case["ids"], case["rows"], case["cols"]
        p = np.diff(np.log(np.arange(rows + 1) + 2.5))
        p *= (1 - case["missing"]) / p.sum()
        hit = float((1 - (1 - p) ** ids).sum())          # expected number of rows that are read
        bytes = 8 * ids + size * cols * (hit + ids)
        if case["train"]:
            bytes += size * cols * (ids + rows)
        return {"bytes": bytes, "flops": ids * cols * (2 if case["train"] else 1)}
    if case["op"] == "grouped":
        rows, groups, k, n, all_rows = case["rows"], case["groups"], case["k"], case["n"], case["rows"] + case["spare"]
        hit = groups * (1 - (1 - 1 / groups) ** rows)
        product = 2 * rows * k * n
        bytes = size * (rows * k + hit * k * n + all_rows * n) + 4 * (groups + 1)
        if not case["train"]:
            return {"bytes": bytes, "flops": product}
        return {"bytes": bytes + size * (rows * n + all_rows * k + groups * k * n), "flops": 3 * product}
    rows, cols, k = case["rows"], case["cols"], case["k"]
    bytes = size * rows * cols + rows * (12 * k + 4)
    if not case["train"]:
        return {"bytes": bytes, "flops": 4 * rows * cols}
    # the whole row is read again: its gradient depends on the sum over all of it
    return {"bytes": bytes + 2 * size * rows * cols + 4 * rows, "flops": 8 * rows * cols}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "embedding":
            return _exact_embedding(st)
        return _exact_grouped(st) if case["op"] == "grouped" else _exact_distill(st)


def _exact_embedding(st):
    ids, table = st["id"], st["table"].double()
    rows = table.shape[0]
    longer = torch.cat((table, torch.zeros_like(table[:1])))
    out = {"out": longer[torch.where((ids < 0) | (ids >= rows), rows, ids)] * st["scale"]}
    if st["train"]:
        d = torch.zeros_like(longer)
        for part in torch.arange(ids.numel(), device="cuda").split(65_536):
            here = ids[part]
            d.index_add_(0, torch.where((here < 0) | (here >= rows), rows, here), st["dout"][part].double())
        out["dtable"] = d[:rows] * st["scale"]
    return out


def _exact_grouped(st):
    X, W, bounds = st["X"].double(), st["W"].double(), st["offsets"].tolist()
    out = {"Y": X.new_zeros((X.shape[0], W.shape[2]))}
    if st["train"]:
        dY = st["dY"].double()
        out["dX"], out["dW"] = torch.zeros_like(X), torch.zeros(W.shape, dtype=torch.float64, device="cuda")
    for g, (a, b) in enumerate(zip(bounds, bounds[1:])):
        out["Y"][a:b] = X[a:b] @ W[g]
        if st["train"]:
            out["dX"][a:b] = dY[a:b] @ W[g].T
            out["dW"][g] = X[a:b].T @ dY[a:b]
    return out


def _exact_distill(st):
    tau, rows, cols = st["tau"], st["rows"], st["cols"]
    loss, dz = [], []
    for r in range(0, rows, 1024):
        z = st["z"][r:r + 1024].double() / tau
        ids, t = st["id"][r:r + 1024], st["teacher"][r:r + 1024].double() / tau
        t = t.masked_fill((ids < 0) | (ids >= cols), -math.inf)
        none = (t == -math.inf).all(-1)
        logp = torch.log_softmax(t.masked_fill(none[:, None], 0.0), -1)
        logq = torch.log_softmax(z, -1)
        p = torch.exp(logp).masked_fill(none[:, None], 0.0)
        logp = logp.masked_fill(p == 0, 0.0)
        at = ids.clamp(0, cols - 1)
        loss.append(tau * tau * (p * (logp - logq.gather(1, at)).masked_fill(p == 0, 0.0)).sum(-1))
        if st["train"]:
            target = torch.zeros_like(z).scatter_add_(1, at, p)
            d = torch.exp(logq).masked_fill(none[:, None], 0.0) - target
            dz.append(d * tau * st["dloss"][r:r + 1024, None].double())
    return {"loss": torch.cat(loss), "dz": torch.cat(dz)} if st["train"] else {"loss": torch.cat(loss)}

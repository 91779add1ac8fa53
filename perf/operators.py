"""The operators that learn from clicks, as they are measured: pooled row lookup, its gradient, and the softmax
cross entropy of queries over a whole corpus of rows with its gradients.

A corpus is a table of document vectors, one row per docid, in float32 or bfloat16: what a vector store holds. Queries
are vectors of the same type. The cases stand for what a user of the search library does with clicks: build a query
from documents that a visitor liked (a bag of rows, weighted), score the clicked document against every document that
the filter lets through, and take the gradients that move queries, documents and weights.

With `own` false, `run` computes the operators in plain torch operations in 32 bits; with `own` true it calls the
library. `exact` computes them in 64 bits."""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_kept = {}  # one context and one workspace per process, as a user's program keeps them


# ---- cases --------------------------------------------------------------------------------


def listed():
    return [
        # one visitor's next page from three liked documents of a small shop: latency counts
        {"name": "lookup 1x3 of 10k x384 f32", "op": "lookup", "dtype": "f32", "rows": 10000, "dim": 384, "bags": 1,
         "most": 3, "weights": True},
        # the query side of a large batch: histories of up to 40 documents, some visitors without any
        {"name": "lookup 16k bags of 1M x768 bf16", "op": "lookup", "dtype": "bf16", "rows": 1000000, "dim": 768,
         "bags": 16384, "most": 40, "weights": True},
        # gradients of a small batch of plain lookups
        {"name": "lookup grad 64x5 of 10k x384 f32", "op": "lookup_grad", "dtype": "f32", "rows": 10000, "dim": 384,
         "bags": 64, "most": 5, "weights": False},
        # the same for the large batch: a few documents are in very many histories
        {"name": "lookup grad 16k bags of 1M x768 bf16", "op": "lookup_grad", "dtype": "bf16", "rows": 1000000,
         "dim": 768, "bags": 16384, "most": 40, "weights": True},
        # how likely the clicked document was, one request, a filter that keeps a tenth of the shop
        {"name": "loss 1 query 10k x384 f32 10%", "op": "loss", "dtype": "f32", "rows": 10000, "dim": 384,
         "queries": 1, "percent": 10},
        # one request over a large corpus: bound by memory
        {"name": "loss 1 query 1M x768 bf16", "op": "loss", "dtype": "bf16", "rows": 1000000, "dim": 768,
         "queries": 1, "percent": 100},
        # evaluation of held-out clicks in batches
        {"name": "loss 256 queries 1M x768 bf16", "op": "loss", "dtype": "bf16", "rows": 1000000, "dim": 768,
         "queries": 256, "percent": 100},
        # a training step on a small corpus
        {"name": "train 64 queries 10k x384 f32", "op": "train", "dtype": "f32", "rows": 10000, "dim": 384,
         "queries": 64, "percent": 100, "frozen": False},
        # a training step on a large corpus: every document vector learns
        {"name": "train 256 queries 1M x768 bf16", "op": "train", "dtype": "bf16", "rows": 1000000, "dim": 768,
         "queries": 256, "percent": 100, "frozen": False},
        # only the query side learns, long vectors, half of an odd-sized corpus is filtered out
        {"name": "train 1000 queries 200003 x1536 bf16 50%", "op": "train", "dtype": "bf16", "rows": 200003,
         "dim": 1536, "queries": 1000, "percent": 50, "frozen": True},
        # the reference's own element type
        {"name": "train 256 queries 250k x768 f32", "op": "train", "dtype": "f32", "rows": 250000, "dim": 768,
         "queries": 256, "percent": 100, "frozen": False},
        # the operators in a row, one table on both sides: histories, queries, loss, gradients of table and weights
        {"name": "step 100 bags 50k x383 f32 90%", "op": "step", "dtype": "f32", "rows": 50000, "dim": 383, "bags": 100,
         "most": 20, "percent": 90},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "loss", "train", "step"])
    dtype = rng.choice(["f32", "bf16"])
    dim = rng.choice([32, 96, 100, 128, 255, 256, 383, 384, 500, 512, 768, 768, 1000, 1024, 1536])
    rows = _log(rng, 1000, 1000000)
    if op in ("lookup", "lookup_grad"):
        return {"op": op, "dtype": dtype, "rows": rows, "dim": min(dim, 768), "bags": _log(rng, 1, 16384),
                "most": _log(rng, 1, 40), "weights": rng.random() < 0.5}
    percent = rng.choice([1, 10, 50, 90, 100])
    most = {"bf16": 256 * 1000000 * 768, "f32": 256 * 250000 * 768}[dtype]
    if op == "step":
        dtype = "f32"
        bags = _log(rng, 1, 512)
        rows = max(1000, min(rows, 200000, most // 4 // (bags * dim)))
        return {"op": op, "dtype": dtype, "rows": rows, "dim": dim, "bags": bags, "most": _log(rng, 1, 40),
                "percent": percent}
    queries = _log(rng, 1, 1024)
    rows = max(1000, min(rows, most // (queries * dim)))
    case = {"op": op, "dtype": dtype, "rows": rows, "dim": dim, "queries": queries, "percent": percent}
    if op == "train":
        case["frozen"] = rng.random() < 0.3
    return case


SCALE = 20.0  # of the logits, which are 20 x cosine: vectors have length one
POOL = 0.5  # of a bag's sum


# ---- inputs -------------------------------------------------------------------------------


def _table(case, g):
    """Rows of length one; of the rows that the filter keeps out, every other one is not a number (vectors that were
    never written), which must not be seen in any result."""
    n, d = case["rows"], case["dim"]
    t = torch.empty(n, d, dtype=TYPES[case["dtype"]], device=DEVICE)
    for a in range(0, n, 65536):
        x = torch.randn(min(65536, n - a), d, generator=g, device=DEVICE)
        t[a : a + x.shape[0]] = x / x.norm(dim=1, keepdim=True)
    return t


def _n_ids(case):
    return sum(case["most"] - i * (case["most"] + 1) // case["bags"] for i in range(case["bags"]))


def _ids(case, g, bags):
    """Bags of 0 to `most` documents, popular documents first: offsets, ids, weights."""
    sizes = case["most"] - torch.arange(bags, device=DEVICE) * (case["most"] + 1) // bags
    sizes = sizes[torch.randperm(bags, generator=g, device=DEVICE)]
    offsets = torch.zeros(bags + 1, dtype=torch.int64, device=DEVICE)
    offsets[1:] = sizes.cumsum(0)
    n = _n_ids(case)
    ids = (torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64).pow(4) * case["rows"]).long()
    ids = (ids * 2654435761) % case["rows"]  # popular documents lie anywhere
    weights = torch.rand(n, generator=g, device=DEVICE) + 0.25 if case.get("weights", True) else None
    return offsets.int(), ids.int(), weights


def _filter(case, g, table):
    if case["percent"] == 100:
        return None, None
    keep = torch.rand(case["rows"], generator=g, device=DEVICE) * 100 < case["percent"]
    keep[0] = True
    out = (~keep).nonzero().flatten()[::2]
    table[out] = float("nan")
    words = torch.zeros(-(-case["rows"] // 64) * 64, dtype=torch.int64, device=DEVICE)
    words[: case["rows"]] = keep.long()
    words = (words.view(-1, 64) << torch.arange(64, device=DEVICE)).sum(1)  # bit d & 63 of word d >> 6
    return keep, words


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    table = _table(case, g)
    s = {"case": case, "table": table}
    if case["op"] in ("lookup", "lookup_grad"):
        s["offsets"], s["ids"], s["weights"] = _ids(case, g, case["bags"])
        if case["op"] == "lookup_grad":
            s["grad_out"] = torch.randn(case["bags"], case["dim"], generator=g, device=DEVICE).to(table.dtype)
            n = s["ids"].numel()
            s["unique"] = torch.zeros(n, dtype=torch.int32, device=DEVICE)
            s["count"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
            s["grad_rows"] = torch.zeros(n, case["dim"], device=DEVICE)
        return s
    s["keep"], s["words"] = _filter(case, g, table)
    n = case["queries"] if "queries" in case else case["bags"]
    # clicked documents are candidates, but for every 50th click, whose document is filtered out or gone
    places = torch.arange(case["rows"], device=DEVICE) if s["keep"] is None else s["keep"].nonzero().flatten()
    targets = places[(torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64).square() * places.numel()).long()]
    s["targets"] = targets.int()
    if case["op"] == "step":
        # histories come from the candidates too
        s["offsets"], ids, s["weights"] = _ids(case, g, n)
        s["ids"] = places[(ids.long() * 7919) % places.numel()].int()
    else:
        noise = torch.randn(n, case["dim"], generator=g, device=DEVICE)
        q = table[targets].float() + noise / noise.norm(dim=1, keepdim=True)
        s["queries"] = (q / q.norm(dim=1, keepdim=True)).to(table.dtype)
    if n > 1:
        s["targets"][49::50] = -1  # 0xFFFFFFFF: no such document
    if case["op"] != "loss":
        s["grad_loss"] = torch.rand(n, generator=g, device=DEVICE) / n + 0.5 / n
    return s


# ---- plain forms --------------------------------------------------------------------------


def _bags(offsets, n):
    """The bag of each of n ids."""
    sizes = (offsets[1:] - offsets[:-1]).long()
    return torch.repeat_interleave(torch.arange(sizes.numel(), device=DEVICE), sizes, output_size=n)


def _plain_lookup(table, ids, offsets, weights):
    x = table[ids.long()].float()
    if weights is not None:
        x = x * weights[:, None]
    out = torch.zeros(offsets.numel() - 1, table.shape[1], device=DEVICE)
    out.index_add_(0, _bags(offsets, ids.numel()), x)
    return out * POOL


def _plain_row_grads(grad_out, ids, offsets, weights):
    """The gradient that each id hands to its row."""
    x = grad_out[_bags(offsets, ids.numel())].float() * POOL
    return x if weights is None else x * weights[:, None]


def _plain_weight_grads(table, grad_out, ids, offsets):
    return (table[ids.long()].float() * grad_out[_bags(offsets, ids.numel())].float()).sum(1) * POOL


def _plain_logits(s, queries, table):
    z = (queries @ table.T) * SCALE
    return z if s["keep"] is None else torch.where(s["keep"], z, -math.inf)


def _plain_loss(s, z):
    """Loss and log-sum-exp. The clicked document's logit is kept out of the sum, log(1 + sum of the others over it), so
    that a loss near zero keeps its digits; the vectors of one number per query are in 64 bits."""
    valid = s["targets"] >= 0
    t = s["targets"].long().clamp(min=0)[:, None]
    click = z.gather(1, t)
    others = z.scatter(1, t, torch.where(valid[:, None], -math.inf, click))
    click = click[:, 0].double()
    m = others.max(1).values
    m = torch.where(m == -math.inf, 0.0, m)
    rest = (others - m[:, None]).exp().sum(1).double().log() + m
    loss = torch.where(valid, torch.logaddexp(torch.zeros_like(rest), rest - click), 0.0)
    return loss, torch.where(valid, torch.logaddexp(rest, click), rest), valid


def _plain_train(s, queries, rows_too):
    """Loss, and gradients of queries and rows."""
    table = s["table"].float()
    if s["keep"] is not None:
        table = torch.where(s["keep"][:, None], table, 0.0)
    z = _plain_logits(s, queries, table)
    loss, lse, valid = _plain_loss(s, z)
    p = (z - lse.float()[:, None]).exp()
    del z
    t = s["targets"].long().clamp(min=0)[:, None]
    p.scatter_(1, t, torch.where(valid[:, None], torch.expm1(-loss).float()[:, None], p.gather(1, t)))
    p *= (torch.where(valid, s["grad_loss"], 0.0) * SCALE)[:, None]
    return loss.float(), lse.float(), p @ table, p.T @ queries if rows_too else None


# ---- the library --------------------------------------------------------------------------


def _library():
    if "ctx" not in _kept:
        from search_engine_amd import abi
        _kept["abi"], _kept["ctx"] = abi, abi.Context(0)
    return _kept["ctx"]


def _workspace(n):
    if _kept.get("workspace") is None or _kept["workspace"].numel() < n:
        _kept["workspace"] = torch.empty(n, dtype=torch.uint8, device=DEVICE)
    return _kept["workspace"]


def _type(t):
    return _kept["abi"].VS_F32 if t.dtype == torch.float32 else _kept["abi"].VS_BF16


def _address(t):
    return None if t is None else t.data_ptr()


def _own_lookup(s, ctx, stream):
    table, n = s["table"], s["offsets"].numel() - 1
    out = torch.empty(n, table.shape[1], dtype=table.dtype, device=DEVICE)
    ctx.lookup_device(table.data_ptr(), _type(table), table.shape[0], table.stride(0), table.shape[1],
                      s["ids"].data_ptr(), s["ids"].numel(), s["offsets"].data_ptr(), n, _address(s["weights"]),
                      POOL, out.data_ptr(), _type(out), out.stride(0), stream)
    return out


def _own_lookup_grad(s, ctx, stream, grad_out, grad_rows, unique, count):
    table, n = s["table"], s["offsets"].numel() - 1
    ws = _workspace(ctx.lookup_grad_workspace_bytes(s["ids"].numel(), table.shape[0], table.shape[1]))
    ctx.lookup_grad_device(grad_out.data_ptr(), _type(grad_out), grad_out.stride(0), table.shape[1],
                           s["ids"].data_ptr(), s["ids"].numel(), s["offsets"].data_ptr(), n, _address(s["weights"]),
                           POOL, table.shape[0], ws.data_ptr(), ws.numel(), grad_rows.data_ptr(),
                           _type(grad_rows), grad_rows.stride(0), _address(unique), _address(count), stream)


def _own_weight_grads(s, ctx, stream, grad_out):
    table = s["table"]
    out = torch.empty_like(s["weights"])
    ctx.lookup_grad_weights_device(table.data_ptr(), _type(table), table.shape[0], table.stride(0), table.shape[1],
                                   s["ids"].data_ptr(), s["ids"].numel(), s["offsets"].data_ptr(),
                                   s["offsets"].numel() - 1, POOL, grad_out.data_ptr(), _type(grad_out),
                                   grad_out.stride(0), out.data_ptr(), stream)
    return out


def _own_loss(s, ctx, stream, queries):
    table, n = s["table"], queries.shape[0]
    loss, lse = torch.empty(2, n, device=DEVICE)
    ws = _workspace(ctx.xent_workspace_bytes(n, table.shape[0], table.shape[1], _type(table)))
    ctx.xent_device(queries.data_ptr(), n, queries.stride(0), table.data_ptr(), table.shape[0], table.stride(0),
                    _type(table), table.shape[1], s["targets"].data_ptr(), _address(s["words"]), SCALE,
                    ws.data_ptr(), ws.numel(), loss.data_ptr(), lse.data_ptr(), stream)
    return loss, lse


def _own_grads(s, ctx, stream, queries, loss, lse, rows_too):
    table, n = s["table"], queries.shape[0]
    grad_queries = torch.empty_like(queries)
    grad_rows = torch.empty_like(table) if rows_too else None
    ws = _workspace(ctx.xent_workspace_bytes(n, table.shape[0], table.shape[1], _type(table)))
    ctx.xent_grad_device(queries.data_ptr(), n, queries.stride(0), table.data_ptr(), table.shape[0], table.stride(0),
                         _type(table), table.shape[1], s["targets"].data_ptr(), _address(s["words"]), SCALE,
                         loss.data_ptr(), lse.data_ptr(), s["grad_loss"].data_ptr(), ws.data_ptr(), ws.numel(),
                         grad_queries.data_ptr(), _address(grad_rows), stream)
    return grad_queries, grad_rows


def _run_own(s):
    case, ctx, stream = s["case"], _library(), torch.cuda.current_stream().cuda_stream
    if case["op"] == "lookup":
        return _own_lookup(s, ctx, stream)
    if case["op"] == "lookup_grad":
        _own_lookup_grad(s, ctx, stream, s["grad_out"], s["grad_rows"], s["unique"], s["count"])
        got = {"rows": s["grad_rows"], "ids": s["unique"], "count": s["count"]}
        if s["weights"] is not None:
            got["weights"] = _own_weight_grads(s, ctx, stream, s["grad_out"])
        return got
    if case["op"] == "loss":
        loss, lse = _own_loss(s, ctx, stream, s["queries"])
        return {"loss": loss, "lse": lse}
    queries = _own_lookup(s, ctx, stream) if case["op"] == "step" else s["queries"]
    rows_too = case["op"] == "step" or not case["frozen"]
    loss, lse = _own_loss(s, ctx, stream, queries)
    grad_queries, grad_rows = _own_grads(s, ctx, stream, queries, loss, lse, rows_too)
    got = {"loss": loss, "lse": lse, "queries": grad_queries}
    if case["op"] == "step":
        got["weights"] = _own_weight_grads(s, ctx, stream, grad_queries)
        _own_lookup_grad(s, ctx, stream, grad_queries, grad_rows, None, None)  # added to the rows' gradient
    if rows_too:
        got["rows"] = grad_rows
    return got


def run(state):
    s = state
    if own:
        return _run_own(s)
    case, table = s["case"], s["table"]
    if case["op"] == "lookup":
        return _plain_lookup(table, s["ids"], s["offsets"], s["weights"]).to(table.dtype)
    if case["op"] == "lookup_grad":
        x = _plain_row_grads(s["grad_out"], s["ids"], s["offsets"], s["weights"])
        unique, place = torch.unique(s["ids"], return_inverse=True)
        s["grad_rows"][: unique.numel()] = 0
        s["grad_rows"].index_add_(0, place, x)
        s["unique"][: unique.numel()] = unique
        s["count"].fill_(unique.numel())
        got = {"rows": s["grad_rows"], "ids": s["unique"], "count": s["count"]}
        if s["weights"] is not None:
            got["weights"] = _plain_weight_grads(table, s["grad_out"], s["ids"], s["offsets"])
        return got
    if case["op"] == "loss":
        loss, lse, _ = _plain_loss(s, _plain_logits(s, s["queries"].float(), table.float()))
        return {"loss": loss.float(), "lse": lse.float()}
    step = case["op"] == "step"
    queries = _plain_lookup(table, s["ids"], s["offsets"], s["weights"]) if step else s["queries"].float()
    rows_too = case["op"] == "step" or not case["frozen"]
    loss, lse, grad_queries, grad_rows = _plain_train(s, queries, rows_too)
    got = {"loss": loss, "lse": lse, "queries": grad_queries.to(table.dtype)}
    if case["op"] == "step":
        got["weights"] = _plain_weight_grads(table, grad_queries, s["ids"], s["offsets"])
        x = _plain_row_grads(grad_queries, s["ids"], s["offsets"], s["weights"])
        grad_rows.index_add_(0, s["ids"].long(), x)
    if rows_too:
        got["rows"] = grad_rows.to(table.dtype)
    return got


# ---- 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    wide, d, f64 = s["table"].double(), case["dim"], {"dtype": torch.float64, "device": DEVICE}
    if s.get("offsets") is not None:
        off = s["offsets"].long()
        owner = torch.searchsorted(off, torch.arange(s["ids"].numel(), device=DEVICE), right=True) - 1
        ids = s["ids"].long()
        w = (torch.ones(ids.numel(), device=DEVICE) if s["weights"] is None else s["weights"]).double() * POOL
    if case["op"] == "lookup":
        return torch.zeros(case["bags"], d, **f64).index_add_(0, owner, wide[ids] * w[:, None])
    if case["op"] == "lookup_grad":
        g = s["grad_out"].double()[owner]
        names, place = ids.unique(return_inverse=True)
        rows = torch.zeros(ids.numel(), d, **f64).index_add_(0, place, g * w[:, None])
        unique = torch.zeros(ids.numel(), dtype=torch.int32, device=DEVICE)
        unique[: names.numel()] = names.int()
        got = {"rows": rows, "ids": unique, "count": torch.tensor([names.numel()], dtype=torch.int32, device=DEVICE)}
        if s["weights"] is not None:
            got["weights"] = torch.einsum("id,id->i", wide[ids], g) * POOL
        return got
    keep = torch.ones(case["rows"], dtype=torch.bool, device=DEVICE) if s["keep"] is None else s["keep"]
    at = keep.nonzero().flatten()
    rows = wide[at]  # the candidates alone
    if case["op"] == "step":
        q = torch.zeros(case["bags"], d, **f64).index_add_(0, owner, wide[ids] * w[:, None])
    else:
        q = s["queries"].double()
    del wide
    z = torch.mm(q, rows.t()).mul_(SCALE)
    lse = torch.logsumexp(z, 1)
    clicks = s["targets"].long()
    some = (clicks >= 0).nonzero().flatten()
    column = torch.searchsorted(at, clicks[some])
    loss = torch.zeros_like(lse)
    loss[some] = lse[some] - z[some, column]
    got = {"loss": loss, "lse": lse}
    if case["op"] == "loss":
        return got
    weight = torch.zeros_like(lse)
    weight[some] = s["grad_loss"].double()[some] * SCALE
    z = z.sub_(lse[:, None]).exp_()
    z[some, column] -= 1
    z.mul_(weight[:, None])
    got["queries"] = torch.mm(z, rows)
    if case["op"] == "step" or not case["frozen"]:
        grad = torch.zeros(case["rows"], d, **f64)
        grad[at] = torch.mm(z.t(), q)
        if case["op"] == "step":
            back = got["queries"][owner]
            full = s["table"].double()
            got["weights"] = torch.einsum("id,id->i", full[ids], back) * POOL
            grad.index_add_(0, ids, back * w[:, None])
        got["rows"] = grad
    return got


# ---- what a pass cannot do without --------------------------------------------------------


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    d, rows = case["dim"], case["rows"]
    bytes_, flops = 0, 0
    if "bags" in case:
        n = _n_ids(case)
        # distinct rows of n ids whose popularity falls as the fourth power: each is read or written once
        distinct = min(n, int(rows * (1 - math.exp(-n / rows)) * 0.6) + 1)
        if case["op"] == "lookup":
            return {"bytes": distinct * d * e + n * 8 + case["bags"] * (d * e + 4), "flops": 2 * n * d}
        back = case["bags"] * d * e + distinct * d * 4 + n * 8
        if case.get("weights", True):
            back += distinct * d * e + n * 4
        if case["op"] == "lookup_grad":
            return {"bytes": back, "flops": (4 if case["weights"] else 2) * n * d}
        bytes_ += back + n * 8
        flops += 6 * n * d
    q = case.get("queries", case.get("bags"))
    seen = max(1, rows * case["percent"] // 100)
    bytes_ += seen * d * e + q * (d * e + 12) + (rows // 8 if case["percent"] < 100 else 0)
    flops += 2 * q * seen * d
    if case["op"] != "loss":
        bytes_ += q * d * e
        flops += 2 * q * seen * d
        if case["op"] == "step" or not case["frozen"]:
            bytes_ += rows * d * e
            flops += 2 * q * seen * d
    return {"bytes": bytes_, "flops": flops}

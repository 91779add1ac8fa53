"""The operators that learn from clicks as programs use them: padded batches, a few queries at a time, tables behind 4 GiB,
graphs that run beside each other."""
import math

import numpy as np
import pytest
import torch

from learn_helpers import (DEV, call_lookup, call_row_grads, call_weight_grads, call_xent, call_xent_grads, check,
                           lookup_reference, ptr, rounded, row_grads_reference, words_of, xent_reference)
from search_engine_amd import abi
from test_learn_xent_gpu import clicks, like, matrix, whole

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NONE = -1  # VS_ROW_NONE in 32 bits


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q", [3, 20, 100, 300])
def test_padding_of_a_batch_reaches_no_gradient(gpu_ctx, dtype, n_q):
    """Queries without a click hold NaN, infinities and the lowest value, and so does the gradient of their loss: they get
    gradient 0, and everything else is what it is with zeros in their place."""
    rows, dim, scale = 700, 70, 9.0
    table, queries = matrix(rows, dim, dtype, 1), matrix(n_q, dim, dtype, 2)
    g = torch.Generator(device=DEV).manual_seed(3)
    keep = torch.rand(rows, generator=g, device=DEV) < 0.6
    keep[5], keep[6] = True, False
    at = keep.nonzero().flatten()
    targets = at[torch.randint(0, at.numel(), (n_q,), generator=g, device=DEV)].int()
    targets[1::3] = NONE
    targets[2::3] = 6  # filtered out
    empty = torch.arange(n_q, device=DEV) % 3 > 0
    grad_loss = torch.rand(n_q, generator=g, device=DEV)
    for mask in (None, keep):
        clicked = torch.where(empty, -1, targets) if mask is None else targets
        words = None if mask is None else words_of(mask)
        results = []
        for fill in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
            q, c = queries.clone(), grad_loss.clone()
            q[empty], c[empty] = fill, fill
            loss, lse = call_xent(gpu_ctx, q, table, clicked, words, scale)
            assert (loss[empty] == 0).all()
            dq, dr = like(q), like(table)
            call_xent_grads(gpu_ctx, q, table, clicked, words, scale, loss, lse, c, dq, dr)
            assert (dq[empty] == 0).all()
            results.append((loss, lse[~empty], dq, dr))
        for other in results[1:]:
            for a, b in zip(results[0], other):
                assert torch.equal(a, b)
        zeros = queries.clone()
        zeros[empty] = 0
        want = xent_reference(zeros, table, clicked, mask, scale, grad_loss)
        check(results[0][2], rounded(want["queries"], dtype))
        check(results[0][3], rounded(want["rows"], dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q", [1, 2, 3, 4])
@pytest.mark.parametrize("rows,dim,percent", [(1, 5, 100), (63, 97, 50), (5000, 104, 10), (40000, 33, 90), (130, 6000, 50),
                                              (70, 8192, 100)])
def test_a_few_queries(gpu_ctx, dtype, n_q, rows, dim, percent):
    table, queries = matrix(rows, dim, dtype, 4), matrix(n_q, dim, dtype, 5)
    g = torch.Generator(device=DEV).manual_seed(6)
    keep = None if percent == 100 else torch.rand(rows, generator=g, device=DEV) * 100 < percent
    if keep is not None:
        keep[rows // 2] = True
        table[~keep] = float("nan")
    targets = torch.randint(0, rows, (n_q,), generator=g, device=DEV).int()
    targets[0] = rows // 2
    whole(gpu_ctx, queries, table, targets, keep, 6.0, None)


@pytest.mark.parametrize("dtype,t", [(abi.VS_F32, F32), (abi.VS_BF16, BF16)])
@pytest.mark.parametrize("metric", [abi.VS_ANGULAR, abi.VS_DOT])
@pytest.mark.parametrize("n_q", [1, 2, 3, 4, 9])
def test_a_few_queries_of_a_store(gpu_ctx, dtype, t, metric, n_q):
    """Documents from an id on, some removed, under a filter; the last query is padding where there is more than one."""
    rng = np.random.default_rng(7)
    base, cap, dim = 640, 400, 50
    rows = rng.standard_normal((300, dim), dtype=np.float32)
    rows[8] = 0  # no direction
    store = gpu_ctx.create_store(0x4400, dim, cap, dtype=dtype, metric=metric, docid_base=base)
    docids = base + np.sort(rng.choice(cap, 300, replace=False)).astype(np.uint32)
    store.upload(docids, rows)
    store.remove(docids[2:4])
    store.seal()
    slots = -(-cap // 64) * 64
    local = torch.from_numpy((docids - base).astype(np.int64)).to(DEV)
    table = torch.zeros(slots, dim, dtype=t, device=DEV)
    table[local] = torch.from_numpy(rows).to(DEV).to(t)
    keep = torch.zeros(slots, dtype=torch.bool, device=DEV)
    keep[local] = True
    keep[local[2:4]] = False
    filt = torch.rand(slots, generator=torch.Generator(device=DEV).manual_seed(8), device=DEV) < 0.5
    filt[local[10:19]] = True
    queries = torch.from_numpy(rng.standard_normal((n_q, dim), dtype=np.float32)).to(DEV)
    click = local[10 : 10 + n_q].clone()
    if n_q > 1:
        click[-1] = local[3]  # removed
    ws = torch.empty(store.xent_workspace_bytes(n_q), dtype=torch.uint8, device=DEV)
    loss, lse = torch.empty(2, n_q, device=DEV)
    dq = torch.empty(n_q, dim, device=DEV)
    scale = 11.0 if metric == abi.VS_ANGULAR else 0.4
    st = torch.cuda.current_stream().cuda_stream
    for mask in (None, filt):
        words = None if mask is None else words_of(mask)
        targets = (click + base).int()
        args = (n_q, dim, ptr(targets), ptr(words), scale)
        store.xent_device(ptr(queries), *args, ptr(ws), ws.numel(), ptr(loss), ptr(lse), st)
        store.xent_grad_device(ptr(queries), *args, ptr(loss), ptr(lse), None, ptr(ws), ws.numel(), ptr(dq), st)
        want = xent_reference(queries.to(t), table, click.int(), keep if mask is None else keep & mask, scale,
                              cosine=metric == abi.VS_ANGULAR)
        check(loss, want["loss"], "loss")
        check(lse, want["lse"], "lse")
        check(dq, rounded(want["queries"], F32), "gradient of the queries")
        if n_q > 1:
            padded = queries.clone()
            padded[-1] = float("nan")
            dq2 = torch.empty_like(dq)
            store.xent_device(ptr(padded), *args, ptr(ws), ws.numel(), ptr(loss), ptr(lse), st)
            store.xent_grad_device(ptr(padded), *args, ptr(loss), ptr(lse), None, ptr(ws), ws.numel(), ptr(dq2), st)
            assert torch.equal(dq, dq2) and (dq2[-1] == 0).all()
    torch.cuda.synchronize()
    store.destroy()


def test_the_list_of_candidates_of_a_large_corpus(gpu_ctx):
    """4 300 001 rows: more words of candidates than one workgroup of the list counts by itself."""
    rows, dim, n_q = 4300001, 8, 6
    table, queries = matrix(rows, dim, BF16, 9), matrix(n_q, dim, BF16, 10)
    keep = torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(11), device=DEV) < 0.2
    keep[:70000] = False
    keep[-1] = True
    table[~keep] = float("nan")
    targets = clicks(n_q, rows, None, 12)
    targets[3] = rows - 1
    whole(gpu_ctx, queries, table, targets, keep, 5.0, None)


def test_numbers_beyond_the_largest_of_bf16(gpu_ctx):
    """f32 rows with elements that bf16 would round to an infinity: where the queries are zero there, nothing of them is in
    the loss, and all of them in the queries' gradient."""
    rows, dim, scale = 600, 40, 4.0
    for n_q in (3, 30, 150):
        table, queries = matrix(rows, dim, F32, 50), matrix(n_q, dim, F32, 51)
        queries[:, 3] = 0
        table[5::7, 3] = torch.finfo(F32).max
        table[6::7, 3] = -3.3961775e38
        whole(gpu_ctx, queries, table, clicks(n_q, rows, None, 52), None, scale, torch.full((n_q,), 1e-3, device=DEV))


@pytest.mark.parametrize("metric", [abi.VS_ANGULAR, abi.VS_DOT])
@pytest.mark.parametrize("dim", [40, 41])
def test_a_large_batch_over_an_f32_store(gpu_ctx, metric, dim):
    """So many queries and rows that the tiles are the largest ones, aligned rows and others."""
    rng = np.random.default_rng(53)
    n, n_q = 40000, 256
    rows = rng.standard_normal((n, dim), dtype=np.float32)
    rows[100] = 0  # no direction
    store = gpu_ctx.create_store(0x4500, dim, n, dtype=abi.VS_F32, metric=metric)
    store.upload(np.arange(n, dtype=np.uint32), rows)
    store.remove(np.array([7, 39999], np.uint32))
    store.seal()
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[[7, 39999]] = False
    queries = torch.from_numpy(rng.standard_normal((n_q, dim), dtype=np.float32)).to(DEV)
    targets = torch.arange(n_q, device=DEV).int() * 150
    targets[0] = 7
    ws = torch.empty(store.xent_workspace_bytes(n_q), dtype=torch.uint8, device=DEV)
    loss, lse = torch.empty(2, n_q, device=DEV)
    dq = torch.empty(n_q, dim, device=DEV)
    scale = 8.0 if metric == abi.VS_ANGULAR else 0.4
    st = torch.cuda.current_stream().cuda_stream
    store.xent_device(ptr(queries), n_q, dim, ptr(targets), None, scale, ptr(ws), ws.numel(), ptr(loss), ptr(lse), st)
    store.xent_grad_device(ptr(queries), n_q, dim, ptr(targets), None, scale, ptr(loss), ptr(lse), None, ptr(ws), ws.numel(), ptr(dq), st)
    want = xent_reference(queries, torch.from_numpy(rows).to(DEV), targets, keep, scale, cosine=metric == abi.VS_ANGULAR)
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")
    check(dq, rounded(want["queries"], F32), "gradient of the queries")
    torch.cuda.synchronize()
    store.destroy()


@pytest.mark.parametrize("dtype,rows", [(BF16, 300000), (F32, 140000)])
def test_tables_beyond_4_gib(gpu_ctx, dtype, rows):
    """Rows whose byte offsets pass 32 bits (and, in bf16, element offsets 31): lookups, loss and gradients at the far end.
    The table is 1000 rows over and over, with rows of their own at its end: logits and gradients of equal rows are equal,
    so that the 64-bit form needs the distinct ones alone."""
    dim, n_q, scale, own = 8192, 6, 10.0, 40
    few = matrix(1000 + own, dim, dtype, 13)
    table = torch.empty(rows, dim, dtype=dtype, device=DEV)
    for a in range(0, rows - own, 1000):
        table[a : a + 1000] = few[: min(1000, rows - a)]
    table[-own:] = few[1000:]
    times = torch.bincount(torch.arange(rows - own, device=DEV) % 1000, minlength=1000 + own).double()
    times[1000:] = 1
    queries = matrix(n_q, dim, dtype, 14)
    targets = (rows - own + torch.arange(n_q, device=DEV)).int()  # rows of their own
    z = (queries.double() @ few.double().T) * scale
    lse = torch.logsumexp(z + times.log(), 1)
    p = torch.exp(z - lse[:, None]) * scale
    p[torch.arange(n_q), 1000 + torch.arange(n_q)] -= scale
    # as xent_reference bounds them: a product of `dim` terms of size one at most, a sum over all rows
    e = (dim + 4) * 2.0**-24 * scale + (4 + 4 * scale + rows) * 2.0**-24
    g_rel = 2 * e + 60 * 2.0**-24 * scale + (2.0**-8 if dtype == BF16 else 0)
    for n in (1, n_q):
        loss, lse_got = call_xent(gpu_ctx, queries[:n], table, targets[:n], None, scale)
        check(lse_got, (lse[:n], torch.full((n,), e + 2.0**-23 * 30, device=DEV).double()))
        check(loss, (lse[:n] - z[torch.arange(n), 1000 + torch.arange(n)], torch.full((n,), 2 * e + 2.0**-22 * 30, device=DEV).double()))
    dq, dr = torch.empty_like(queries), torch.empty_like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, None, scale, loss, lse_got, None, dq, dr)
    size = p.abs() * times
    check(dq, rounded(((p * times) @ few.double(), g_rel * (size @ few.double().abs())), dtype))
    want = rounded((p.T @ queries.double(), g_rel * (p.abs().T @ queries.double().abs())), dtype)
    check(dr[-own:], (want[0][1000:], want[1][1000:]), "the last rows' gradient")
    check(dr[rows - own - 500 : rows - own], tuple(w[(torch.arange(rows - own - 500, rows - own) % 1000).to(DEV)] for w in want))
    check(dr[:1000], (want[0][:1000], want[1][:1000]))
    # the far end, looked up and added to
    ids = (rows - 1 - torch.arange(30, device=DEV) // 2).int()
    off = torch.tensor([0, 7, 7, 30], device=DEV).int()
    out = call_lookup(gpu_ctx, table, ids, off, 3, None, 1.0, torch.empty(3, dim, dtype=dtype, device=DEV))
    near = torch.cat([few[1000:], few[1000:]])[: own]
    check(out, lookup_reference(near, ids - (rows - own), off, 3, None, 1.0, dtype))
    before = dr[-own:].double()
    call_row_grads(gpu_ctx, out, ids, off, None, 1.0, rows, dr)
    value, bound, _ = row_grads_reference(out, ids - (rows - own), off, None, 1.0, own, F32)
    check(dr[-own:], rounded((before + value, bound + 2.0**-24 * (before + value).abs()), dtype), "added at the far end")


@pytest.mark.parametrize("n,n_bags", [(1500, 5000), (2048, 2049), (2049, 1), (1, 9000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_bags_than_ids_and_one_bag_of_all(gpu_ctx, dtype, n, n_bags):
    rows, dim = 300, 20
    g = torch.Generator(device=DEV).manual_seed(15)
    ids = torch.randint(0, rows, (n,), generator=g, device=DEV).int()
    off = torch.cat([torch.zeros(1, device=DEV).long(), torch.randint(0, n + 1, (n_bags,), generator=g, device=DEV).sort().values]).int()
    off[-1] = n
    w = torch.rand(n, generator=g, device=DEV)
    grad = matrix(n_bags, dim, dtype, 16)
    dr = torch.zeros(rows, dim, device=DEV)
    call_row_grads(gpu_ctx, grad, ids, off, w, 0.5, rows, dr)
    value, bound, _ = row_grads_reference(grad, ids, off, w, 0.5, rows, F32)
    check(dr, (value, bound))
    table = matrix(rows, dim, dtype, 17)
    out = call_lookup(gpu_ctx, table, ids, off, n_bags, w, 0.5, torch.empty(n_bags, dim, device=DEV))
    check(out, lookup_reference(table, ids, off, n_bags, w, 0.5, F32))


def test_two_graphs_beside_each_other(gpu_ctx):
    """Loss and gradients of bf16 queries under a filter and of a row of ids, captured twice, each with workspaces of its
    own: replayed on two streams at once, with eager calls in between, they give the eager calls' bits."""
    rows, dim, n_q, scale = 9000, 96, 150, 8.0
    table = matrix(rows, dim, BF16, 18)
    words = words_of(torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(19), device=DEV) < 0.7)
    ids = torch.randint(0, rows, (3000,), generator=torch.Generator(device=DEV).manual_seed(20), device=DEV).int()
    off = (torch.arange(n_q + 1, device=DEV) * 20).int()
    w = torch.rand(3000, device=DEV)

    class Side:
        def __init__(self, seed):
            self.queries, self.targets = matrix(n_q, dim, BF16, seed), clicks(n_q, rows, None, seed)
            self.dq, self.dr = torch.empty_like(self.queries), torch.empty_like(table)
            self.loss, self.lse = torch.empty(2, n_q, device=DEV)
            self.dw = torch.empty(3000, device=DEV)
            self.ws = torch.empty(gpu_ctx.xent_workspace_bytes(n_q, rows, dim, abi.VS_BF16), dtype=torch.uint8, device=DEV)
            self.ws2 = torch.empty(gpu_ctx.lookup_grad_workspace_bytes(3000, rows, dim), dtype=torch.uint8, device=DEV)

        def run(self):
            st = torch.cuda.current_stream().cuda_stream
            gpu_ctx.xent_device(ptr(self.queries), n_q, dim, ptr(table), rows, dim, abi.VS_BF16, dim, ptr(self.targets), ptr(words),
                                scale, ptr(self.ws), self.ws.numel(), ptr(self.loss), ptr(self.lse), st)
            call_xent_grads(gpu_ctx, self.queries, table, self.targets, words, scale, self.loss, self.lse, None, self.dq, self.dr, self.ws)
            call_weight_grads(gpu_ctx, table, ids, off, 1.0, self.dq, self.dw)
            call_row_grads(gpu_ctx, self.dq, ids, off, w, 1.0, rows, self.dr, ws=self.ws2)

        def results(self):
            return [t.clone() for t in (self.loss, self.lse, self.dq, self.dr, self.dw)]

    sides, graphs, streams = [Side(21), Side(22)], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for side in sides:
        side.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            side.run()
        graphs.append(graph)
    for seed in range(3):
        for i, side in enumerate(sides):
            side.queries.copy_(matrix(n_q, dim, BF16, 30 + 2 * seed + i))
            side.targets.copy_(clicks(n_q, rows, None, 40 + 2 * seed + i))
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        replayed = [side.results() for side in sides]
        for side, got in zip(sides, replayed):
            side.run()
            torch.cuda.synchronize()
            for a, b in zip(got, side.results()):
                assert torch.equal(a, b)
    assert math.isfinite(float(sides[0].loss.sum()))


def test_calls_on_a_store_are_refused_under_capture(gpu_ctx):
    store = gpu_ctx.create_store(0x4600, 32, 100)
    rows = np.random.default_rng(60).standard_normal((100, 32), dtype=np.float32)
    store.upload(np.arange(100, dtype=np.uint32), rows)
    store.seal()
    ids = torch.arange(3, device=DEV).int()
    out, queries = torch.zeros(3, 32, device=DEV), torch.ones(3, 32, device=DEV)
    loss, lse = torch.zeros(2, 3, device=DEV)
    ws = torch.empty(store.xent_workspace_bytes(3), dtype=torch.uint8, device=DEV)

    def calls(st):
        yield lambda: store.lookup_device(ptr(ids), 3, None, 3, None, 1.0, ptr(out), abi.VS_F32, 32, st)
        yield lambda: store.xent_device(ptr(queries), 3, 32, ptr(ids), None, 1.0, ptr(ws), ws.numel(), ptr(loss), ptr(lse), st)
        yield lambda: store.xent_grad_device(ptr(queries), 3, 32, ptr(ids), None, 1.0, ptr(loss), ptr(lse), None, ptr(ws), ws.numel(),
                                             ptr(out), st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        queries += 1  # (something to record)
        for call in calls(torch.cuda.current_stream().cuda_stream):
            with pytest.raises(abi.VsError) as e:
                call()
            assert e.value.code == abi.VS_E_INVALID_ARG
    graph.replay()
    torch.cuda.synchronize()
    assert (queries == 2).all() and (out == 0).all()
    for call in calls(torch.cuda.current_stream().cuda_stream):
        call()
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and torch.isfinite(loss).all() and (loss != 0).any()
    store.destroy()

"""Cross entropy over a corpus and its gradients against 64-bit forms, at the sizes and masks where they can go wrong."""
import math

import numpy as np
import pytest
import torch

from learn_helpers import (DEV, TYPE, call_lookup, call_row_grads, call_weight_grads, call_xent, call_xent_grads, check,
                           ids_tensor, lookup_reference, ptr, rounded, words_of, xent_reference)
from search_engine_amd import abi

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def matrix(rows, dim, dtype, seed, pad=0, offset=0, unit=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    flat = torch.full((offset + rows * (dim + pad) + 64,), float("nan"), device=DEV, dtype=dtype)
    t = flat[offset : offset + rows * (dim + pad)].view(rows, dim + pad)[:, :dim]
    x = torch.randn(rows, dim, generator=g, device=DEV)
    t.copy_(x / x.norm(dim=1, keepdim=True) if unit else x)
    return t


def like(t):
    """A matrix of the same layout, NaN everywhere (between the rows too)."""
    base = torch.full((t.shape[0] * t.stride(0) + 64,), float("nan"), dtype=t.dtype, device=DEV)
    return base[: t.shape[0] * t.stride(0)].view(t.shape[0], t.stride(0))[:, : t.shape[1]]


def gaps_are_nan(t):
    if t.shape[1] == t.stride(0):
        return True
    return bool(torch.isnan(t.as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1))[:, t.shape[1] :]).all())


def clicks(n, rows, keep, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = torch.randint(0, rows, (n,), generator=g, device=DEV)
    if n > 2:
        t[1] = 0xFFFFFFFF
        t[2] = rows
    return t.to(torch.int32)


def whole(ctx, queries, table, targets, keep, scale, grad_loss, cosine=False):
    """Loss and both gradients through the calls, checked."""
    words = None if keep is None else words_of(keep)
    want = xent_reference(queries, table, targets, keep, scale, grad_loss)
    loss, lse = call_xent(ctx, queries, table, targets, words, scale)
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")
    dq, dr = like(queries), like(table)
    call_xent_grads(ctx, queries, table, targets, words, scale, loss, lse, grad_loss, dq, dr)
    check(dq, rounded(want["queries"], dq.dtype), "gradient of the queries")
    check(dr, rounded(want["rows"], dr.dtype), "gradient of the rows")
    assert gaps_are_nan(dq) and gaps_are_nan(dr)
    return loss, lse, dq, dr


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q,rows", [(1, 1), (1, 64), (2, 65), (3, 1000), (16, 255), (17, 256), (64, 257), (65, 2000),
                                      (128, 4096), (130, 300), (256, 1025), (257, 640), (700, 129)])
@pytest.mark.parametrize("dim", [32, 100])
def test_sizes(gpu_ctx, dtype, n_q, rows, dim):
    table, queries = matrix(rows, dim, dtype, 1), matrix(n_q, dim, dtype, 2)
    grad_loss = torch.rand(n_q, device=DEV)
    whole(gpu_ctx, queries, table, clicks(n_q, rows, None, 3), None, 8.0, grad_loss)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim,pad,offset", [(1, 0, 0), (3, 1, 0), (8, 0, 0), (8, 0, 8), (24, 0, 1), (63, 0, 0), (64, 0, 0),
                                            (64, 8, 0), (65, 7, 0), (383, 0, 0), (384, 0, 0), (768, 0, 0), (776, 0, 0),
                                            (1536, 0, 0), (2050, 0, 0), (8192, 0, 0)])
def test_dimensions_strides_and_alignment(gpu_ctx, dtype, dim, pad, offset):
    rows, n_q = 300, 20
    table, queries = matrix(rows, dim, dtype, 4, pad, offset), matrix(n_q, dim, dtype, 5, pad, offset)
    keep = torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV) < 0.7
    whole(gpu_ctx, queries, table, clicks(n_q, rows, keep, 7), keep, 5.0, None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["none", "one", "two", "half", "tenth", "last", "all", "block"])
@pytest.mark.parametrize("n_q", [1, 40, 200])
def test_filters(gpu_ctx, dtype, kind, n_q):
    """Rows that the filter keeps out hold NaN and infinities: they reach no result, and their gradient is zero."""
    rows, dim = 1500, 72
    g = torch.Generator(device=DEV).manual_seed(8)
    keep = torch.zeros(rows, dtype=torch.bool, device=DEV)
    if kind == "one":
        keep[777] = True
    elif kind == "two":
        keep[[3, 1499]] = True
    elif kind in ("half", "tenth"):
        keep = torch.rand(rows, generator=g, device=DEV) < (0.5 if kind == "half" else 0.1)
    elif kind == "last":
        keep[rows - 1] = True
    elif kind == "all":
        keep[:] = True
    elif kind == "block":
        keep[512:1024] = True
    table, queries = matrix(rows, dim, dtype, 9), matrix(n_q, dim, dtype, 10)
    out = (~keep).nonzero().flatten()
    table[out[::3]] = float("nan")
    table[out[1::3]] = float("inf")
    table[out[2::3]] = torch.finfo(dtype).min
    targets = clicks(n_q, rows, keep, 11)
    loss, lse, dq, dr = whole(gpu_ctx, queries, table, targets, keep, 12.0, torch.rand(n_q, device=DEV) - 0.5)
    assert (dr[~keep] == 0).all()
    if kind == "none":
        assert (loss == 0).all() and (lse == -math.inf).all() and (dq == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.0, 1e-3, 100.0, -30.0, 1000.0])
def test_scales(gpu_ctx, dtype, scale):
    """From a flat distribution to one document that takes all of it."""
    table, queries = matrix(500, 96, dtype, 12), matrix(33, 96, dtype, 13)
    whole(gpu_ctx, queries, table, clicks(33, 500, None, 14), None, scale, None)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_certain_click_keeps_its_digits(gpu_ctx, dtype):
    """Losses near zero: lse - z would leave nothing of them."""
    dim = 64
    table = matrix(400, dim, dtype, 15)
    targets = torch.arange(20, device=DEV).int()
    queries = table[:20].clone()
    loss, _, dq, _ = whole(gpu_ctx, queries, table, targets, None, 40.0, None)
    assert 0 < float(loss.max()) < 1e-3
    assert float(dq.float().abs().max()) > 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_rows_and_equal_clicks(gpu_ctx, dtype):
    table = matrix(300, 40, dtype, 16)
    table[:] = table[0].clone()
    queries = matrix(50, 40, dtype, 17)
    targets = torch.full((50,), 123, dtype=torch.int32, device=DEV)
    loss, *_ = whole(gpu_ctx, queries, table, targets, None, 7.0, None)
    assert (loss - math.log(300)).abs().max() < 1e-5


def test_not_a_number_stays_one(gpu_ctx):
    """A candidate row with NaN makes every loss NaN; a query with NaN its own alone."""
    table, queries = matrix(300, 64, F32, 18), matrix(5, 64, F32, 19)
    queries[3, 5] = float("nan")
    targets = torch.tensor([0, 1, 2, 3, 4], device=DEV).int()
    loss, _ = call_xent(gpu_ctx, queries, table, targets, None, 1.0)
    assert torch.isnan(loss).tolist() == [False, False, False, True, False]
    table[200, 7] = float("nan")
    loss, lse = call_xent(gpu_ctx, queries, table, targets, None, 1.0)
    assert torch.isnan(loss).all() and torch.isnan(lse).all()


def test_one_gradient_alone_and_the_same_bits_twice(gpu_ctx):
    for dtype in (F32, BF16):
        table, queries = matrix(3000, 128, dtype, 20), matrix(70, 128, dtype, 21)
        targets = clicks(70, 3000, None, 22)
        loss, lse = call_xent(gpu_ctx, queries, table, targets, None, 9.0)
        loss2, lse2 = call_xent(gpu_ctx, queries, table, targets, None, 9.0)
        assert torch.equal(loss, loss2) and torch.equal(lse, lse2)
        dq, dr = like(queries), like(table)
        call_xent_grads(gpu_ctx, queries, table, targets, None, 9.0, loss, lse, None, dq, dr)
        dq2, dr2 = like(queries), like(table)
        call_xent_grads(gpu_ctx, queries, table, targets, None, 9.0, loss, lse, None, dq2, None)
        call_xent_grads(gpu_ctx, queries, table, targets, None, 9.0, loss, lse, None, None, dr2)
        assert torch.equal(dq, dq2) and torch.equal(dr, dr2)


def test_no_queries(gpu_ctx):
    table = matrix(70, 16, F32, 23)
    queries = torch.zeros(0, 16, device=DEV)
    none = torch.zeros(0, device=DEV)
    dr = like(table)
    call_xent(gpu_ctx, queries, table, none.int(), None, 1.0)
    call_xent_grads(gpu_ctx, queries, table, none.int(), None, 1.0, none, none, None, None, dr)
    assert (dr == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_than_one_piece(gpu_ctx, dtype):
    """So many queries that the rows go by in several pieces (the weights of one piece are held at a time)."""
    n_q, rows, dim = 20000, 9001, 16
    table, queries = matrix(rows, dim, dtype, 24), matrix(n_q, dim, dtype, 25)
    keep = torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(26), device=DEV) < 0.9
    whole(gpu_ctx, queries, table, clicks(n_q, rows, keep, 27), keep, 3.0, torch.rand(n_q, device=DEV) / n_q)


def test_many_rows(gpu_ctx):
    """A corpus of 300 001 documents, one query and 260, against 64 bits."""
    for dtype in (F32, BF16):
        table = matrix(300001, 64, dtype, 28)
        for n_q in (1, 260):
            queries = matrix(n_q, 64, dtype, 29)
            keep = torch.rand(300001, generator=torch.Generator(device=DEV).manual_seed(30), device=DEV) < 0.3
            for k in (None, keep):
                whole(gpu_ctx, queries, table, clicks(n_q, 300001, k, 31), k, 6.0, None)


def test_gradients_against_differences(gpu_ctx):
    """Central differences of the 64-bit loss. Its third derivative is at most scale^3 |x|^3, so a step of 1e-3 leaves an
    error of h^2 / 6 times that, below 1e-4 of the gradients' size here; f32 gradients add their own bound."""
    rows, dim, n_q, scale, h = 40, 6, 5, 3.0, 1e-3
    table, queries = matrix(rows, dim, F32, 32), matrix(n_q, dim, F32, 33)
    targets = ids_tensor([4, 39, 2**32 - 1, 0, 7])
    c = torch.rand(n_q, device=DEV)
    loss, lse = call_xent(gpu_ctx, queries, table, targets, None, scale)
    dq, dr = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, None, scale, loss, lse, c, dq, dr)

    def total(q, r):
        return float((xent_reference(q, r, targets, None, scale)["loss"][0] * c.double()).sum())
    for i, k in ((0, 0), (1, 5), (2, 3), (4, 2)):
        e = torch.zeros(n_q, dim, dtype=torch.float64, device=DEV)
        e[i, k] = h
        diff = (total(queries.double() + e, table.double()) - total(queries.double() - e, table.double())) / (2 * h)
        assert abs(diff - float(dq[i, k])) < 1e-4
    for i, k in ((4, 0), (39, 5), (11, 3), (0, 2)):
        e = torch.zeros(rows, dim, dtype=torch.float64, device=DEV)
        e[i, k] = h
        diff = (total(queries.double(), table.double() + e) - total(queries.double(), table.double() - e)) / (2 * h)
        assert abs(diff - float(dr[i, k])) < 1e-4


# ---- in use -------------------------------------------------------------------------------------


def test_on_another_stream_and_two_calls_at_once(gpu_ctx):
    table = matrix(20000, 96, BF16, 34)
    work = []
    for i in range(4):
        s = torch.cuda.Stream()
        q, t = matrix(30 + i, 96, BF16, 35 + i), clicks(30 + i, 20000, None, 40 + i)
        ws = torch.empty(gpu_ctx.xent_workspace_bytes(30 + i, 20000, 96, abi.VS_BF16), dtype=torch.uint8, device=DEV)
        work.append((s, q, t, ws))
    torch.cuda.synchronize()
    got = []
    for s, q, t, ws in work:
        with torch.cuda.stream(s):
            loss, lse = call_xent(gpu_ctx, q, table, t, None, 6.0, ws)
            dq = like(q)
            call_xent_grads(gpu_ctx, q, table, t, None, 6.0, loss, lse, None, dq, None, ws)
            got.append((loss, dq))
    torch.cuda.synchronize()
    for (s, q, t, ws), (loss, dq) in zip(work, got):
        want = xent_reference(q, table, t, None, 6.0)
        check(loss, want["loss"])
        check(dq, rounded(want["queries"], BF16))


def test_captured_and_replayed(gpu_ctx):
    """A training step in a graph: replayed with new queries, weights and clicks, with eager work in between, every replay
    equals the eager call bit for bit."""
    rows, dim, n_bags = 4000, 64, 24
    table = matrix(rows, dim, F32, 50)
    g = torch.Generator(device=DEV).manual_seed(51)
    n = n_bags * 5
    ids = torch.randint(0, rows, (n,), generator=g, device=DEV).int()
    off = (torch.arange(n_bags + 1, device=DEV) * 5).int()
    w = torch.rand(n, generator=g, device=DEV)
    targets = torch.randint(0, rows, (n_bags,), generator=g, device=DEV).int()
    keep = torch.rand(rows, generator=g, device=DEV) < 0.8
    words = words_of(keep)
    queries, dq, dr = torch.empty(n_bags, dim, device=DEV), torch.empty(n_bags, dim, device=DEV), like(table)
    loss, lse = torch.empty(2, n_bags, device=DEV)
    dw = torch.empty(n, device=DEV)
    ws = torch.empty(gpu_ctx.xent_workspace_bytes(n_bags, rows, dim, abi.VS_F32), dtype=torch.uint8, device=DEV)
    ws2 = torch.empty(gpu_ctx.lookup_grad_workspace_bytes(n, rows, dim), dtype=torch.uint8, device=DEV)

    def step():
        st = torch.cuda.current_stream().cuda_stream
        call_lookup(gpu_ctx, table, ids, off, n_bags, w, 1.0, queries)
        gpu_ctx.xent_device(ptr(queries), n_bags, dim, ptr(table), rows, table.stride(0), abi.VS_F32, dim, ptr(targets),
                            ptr(words), 4.0, ptr(ws), ws.numel(), ptr(loss), ptr(lse), st)
        call_xent_grads(gpu_ctx, queries, table, targets, words, 4.0, loss, lse, None, dq, dr, ws)
        call_weight_grads(gpu_ctx, table, ids, off, 1.0, dq, dw)
        call_row_grads(gpu_ctx, dq, ids, off, w, 1.0, rows, dr, ws=ws2)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(4):
        g.manual_seed(60 + seed)
        w.copy_(torch.rand(n, generator=g, device=DEV))
        ids.copy_(torch.randint(0, rows, (n,), generator=g, device=DEV).int())
        targets.copy_(torch.randint(0, rows, (n_bags,), generator=g, device=DEV).int())
        graph.replay()
        torch.cuda.synchronize()
        first = [t.clone() for t in (loss, lse, dq, dr, dw)]
        step()
        torch.cuda.synchronize()
        for a, b in zip(first, (loss, lse, dq, dr, dw)):
            assert torch.equal(a, b)
    assert torch.isfinite(loss).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_training_step(gpu_ctx, dtype):
    """Histories -> queries -> loss over the filtered corpus -> gradients of table and weights, one table on both sides,
    against the same chain in 64 bits."""
    rows, dim, n_bags = 2000, 56, 30
    table = matrix(rows, dim, dtype, 70)
    g = torch.Generator(device=DEV).manual_seed(71)
    sizes = torch.randint(0, 9, (n_bags,), generator=g, device=DEV)
    off = torch.cat([torch.zeros(1, device=DEV), sizes.cumsum(0)]).int()
    n = int(off[-1])
    keep = torch.rand(rows, generator=g, device=DEV) < 0.9
    at = keep.nonzero().flatten()
    ids = at[torch.randint(0, at.numel(), (n,), generator=g, device=DEV)].int()
    targets = at[torch.randint(0, at.numel(), (n_bags,), generator=g, device=DEV)].int()
    w = torch.rand(n, generator=g, device=DEV)
    words = words_of(keep)
    queries = call_lookup(gpu_ctx, table, ids, off, n_bags, w, 0.5, torch.empty(n_bags, dim, dtype=dtype, device=DEV))
    check(queries, lookup_reference(table, ids, off, n_bags, w, 0.5, dtype))
    loss, lse = call_xent(gpu_ctx, queries, table, targets, words, 10.0)
    dq, dr = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, words, 10.0, loss, lse, None, dq, dr)
    want = xent_reference(queries, table, targets, keep, 10.0)  # of the queries as they were rounded
    check(loss, want["loss"])
    check(dq, rounded(want["queries"], dtype))
    both = dr.double()
    call_row_grads(gpu_ctx, dq, ids, off, w, 0.5, rows, dr)
    dw = call_weight_grads(gpu_ctx, table, ids, off, 0.5, dq, torch.empty(n, device=DEV))
    from learn_helpers import row_grads_reference, weight_grads_reference
    value, bound, _ = row_grads_reference(dq, ids, off, w, 0.5, rows, F32)
    check(dr, rounded((both + value, bound + 2.0**-24 * (both + value).abs()), dtype), "rows' gradient from both sides")
    check(dw, weight_grads_reference(table, dq, ids, off, 0.5))


# ---- over a store -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,t", [(abi.VS_F32, F32), (abi.VS_BF16, BF16)])
@pytest.mark.parametrize("metric", [abi.VS_ANGULAR, abi.VS_DOT])
@pytest.mark.parametrize("dim,n_q", [(96, 20), (99, 5), (384, 200)])
def test_store_loss_and_query_gradient(gpu_ctx, dtype, t, metric, dim, n_q):
    rng = np.random.default_rng(80)
    base, cap = 128, 1500
    rows = rng.standard_normal((900, dim), dtype=np.float32)
    rows[17] = 0  # no direction
    store = gpu_ctx.create_store(0x4200, dim, cap, dtype=dtype, metric=metric, docid_base=base)
    docids = base + np.sort(rng.choice(cap, 900, replace=False)).astype(np.uint32)
    store.upload(docids, rows)
    store.remove(docids[5:9])
    store.seal()
    queries = torch.from_numpy(rng.standard_normal((n_q, dim), dtype=np.float32)).to(DEV)
    queries[1] = 0
    table = torch.zeros(store_slots(cap), dim, dtype=t, device=DEV)
    local = torch.from_numpy((docids - base).astype(np.int64)).to(DEV)
    table[local] = torch.from_numpy(rows).to(DEV).to(t)
    keep = torch.zeros(table.shape[0], dtype=torch.bool, device=DEV)
    keep[local] = True
    keep[local[5:9]] = False
    filt = torch.rand(table.shape[0], device=DEV) < 0.8
    rounded_queries = queries.to(t)
    target_local = local[torch.randint(0, 900, (n_q,), device=DEV)]
    target_local[0] = local[6]  # removed
    targets = (target_local + base).int()
    if n_q > 4:
        targets[4] = 3  # before the store
        target_local[4] = 0xFFFFFFFF
    c = torch.rand(n_q, device=DEV)
    ws = torch.empty(store.xent_workspace_bytes(n_q), dtype=torch.uint8, device=DEV)
    loss, lse = torch.empty(2, n_q, device=DEV)
    dq = torch.empty(n_q, dim, device=DEV)
    scale = 15.0 if metric == abi.VS_ANGULAR else 0.3
    for mask in (None, filt):
        words = None if mask is None else words_of(mask)
        st = torch.cuda.current_stream().cuda_stream
        store.xent_device(ptr(queries), n_q, dim, ptr(targets), ptr(words), scale, ptr(ws), ws.numel(), ptr(loss), ptr(lse), st)
        store.xent_grad_device(ptr(queries), n_q, dim, ptr(targets), ptr(words), scale, ptr(loss), ptr(lse), ptr(c), ptr(ws),
                               ws.numel(), ptr(dq), st)
        torch.cuda.synchronize()
        want = xent_reference(rounded_queries, table, target_local.to(torch.int32), keep if mask is None else keep & mask, scale, c,
                              cosine=metric == abi.VS_ANGULAR)
        check(loss, want["loss"], "loss")
        check(lse, want["lse"], "lse")
        check(dq, rounded(want["queries"], F32), "gradient of the queries")
    # a search sees the same rows: the nearest document of a query is the one with the largest logit
    if metric == abi.VS_DOT and dtype == abi.VS_F32:
        ids, _ = store.search(queries[2].cpu().numpy(), 1)
        z = torch.where(keep, table.double() @ queries[2].double(), -math.inf)
        assert int(ids[0]) - base == int(z.argmax())
    store.destroy()


def store_slots(capacity):
    return -(-capacity // 64) * 64


def test_store_refusals(gpu_ctx):
    buf = torch.zeros(1 << 22, dtype=torch.uint8, device=DEV)
    p = buf.data_ptr()

    def refused(code, f, *a):
        with pytest.raises(abi.VsError) as e:
            f(*a)
        assert e.value.code == code, e.value

    s = gpu_ctx.create_store(0x4300, 64, 100)
    refused(abi.VS_E_NOT_SEALED, s.xent_device, p, 1, 64, p, None, 1.0, p, 1 << 20, p, p)
    refused(abi.VS_E_NOT_SEALED, s.lookup_device, p, 1, None, 1, None, 1.0, p, abi.VS_F32, 64)
    s.upload(np.arange(10, dtype=np.uint32), np.ones((10, 64), np.float32))
    s.seal()
    refused(abi.VS_E_DIM_MISMATCH, s.xent_device, p, 1, 63, p, None, 1.0, p, 1 << 20, p, p)
    refused(abi.VS_E_CAPACITY, s.xent_device, p, 1, 64, p, None, 1.0, p, 100, p, p)
    refused(abi.VS_E_CAPACITY, s.xent_grad_device, p, 1, 64, p, None, 1.0, p, p, None, p, 100, p)
    refused(abi.VS_E_INVALID_ARG, s.xent_grad_device, p, 1, 64, p, None, 1.0, p, p, None, p, 1 << 20, None)
    refused(abi.VS_E_INVALID_ARG, s.xent_device, None, 1, 64, p, None, 1.0, p, 1 << 20, p, p)
    refused(abi.VS_E_INVALID_ARG, s.xent_device, p, abi.VS_XENT_MAX_QUERIES + 1, 64, p, None, 1.0, p, 1 << 20, p, p)
    refused(abi.VS_E_INVALID_ARG, s.lookup_device, p, 1, None, 1, None, 1.0, p, abi.VS_F32, 63)
    s.destroy()
    for dtype, metric in ((abi.VS_F32, abi.VS_EUCLIDEAN), (abi.VS_BIN1, abi.VS_HAMMING)):
        s = gpu_ctx.create_store(0x4301, 64, 100, dtype=dtype, metric=metric)
        s.upload(np.arange(10, dtype=np.uint32), np.ones((10, 64), np.float32))
        s.seal()
        refused(abi.VS_E_INVALID_ARG, s.xent_device, p, 1, 64, p, None, 1.0, p, 1 << 20, p, p)
        s.destroy()


def test_the_types_the_helpers_know():
    assert TYPE == {F32: abi.VS_F32, BF16: abi.VS_BF16}

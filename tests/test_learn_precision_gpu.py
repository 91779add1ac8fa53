"""What the cross entropy over a corpus keeps of its numbers: weights, exponents and lengths, against tight bounds."""
import math

import numpy as np
import pytest
import torch

from learn_bounds import bounds, weight_bits
from learn_helpers import DEV, U32, call_xent, call_xent_grads, check, ptr, rounded, words_of
from search_engine_amd import abi
from test_learn_xent_gpu import clicks, like, matrix

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def steps(rows, dim, dtype, seed):
    """Elements -1/4, -1/8, 0, 1/8, 1/4: whatever order a product is summed in, nothing of it is rounded."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randint(-2, 3, (rows, dim), generator=g, device=DEV) / 8).to(dtype)


@pytest.fixture
def store_of(gpu_ctx):
    """Makes stores of rows, sealed; they go when the test ends."""
    made = []

    def make(dtype, metric, rows):
        store = gpu_ctx.create_store(0x4700 + len(made), rows.shape[1], rows.shape[0], dtype=dtype, metric=metric)
        made.append(store)
        store.upload(np.arange(rows.shape[0], dtype=np.uint32), rows)
        store.seal()
        return store
    yield make
    torch.cuda.synchronize()
    for store in made:
        store.destroy()


def store_loss_and_grad(store, queries, targets, scale, words=None):
    n_q, dim = queries.shape
    ws = torch.empty(store.xent_workspace_bytes(n_q), dtype=torch.uint8, device=DEV)
    loss, lse = torch.empty(2, n_q, device=DEV)
    dq = torch.empty(n_q, dim, device=DEV)
    st = torch.cuda.current_stream().cuda_stream
    store.xent_device(ptr(queries), n_q, dim, ptr(targets), ptr(words), scale, ptr(ws), ws.numel(), ptr(loss), ptr(lse), st)
    store.xent_grad_device(ptr(queries), n_q, dim, ptr(targets), ptr(words), scale, ptr(loss), ptr(lse), None, ptr(ws), ws.numel(), ptr(dq), st)
    torch.cuda.synchronize()
    return loss, lse, dq


@pytest.mark.parametrize("filtered", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q", [3, 40, 64, 65, 100, 300])
def test_weights_keep_their_bits(gpu_ctx, dtype, n_q, filtered):
    """A rounding of the weights to 8 bits (2^-8 of each) lies far outside of what a row's gradient may be off by, whatever the
    size of the batch."""
    rows, dim, scale = 700, 32, 8.0
    table, queries = steps(rows, dim, dtype, 1), steps(n_q, dim, dtype, 2)
    keep = torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) < 0.6 if filtered else None
    words = None if keep is None else words_of(keep)
    targets = clicks(n_q, rows, keep, 4)
    c = torch.rand(n_q, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)
    loss, lse = call_xent(gpu_ctx, queries, table, targets, words, scale)
    dq, dr = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, words, scale, loss, lse, c, dq, dr)
    want = bounds(queries, table, targets, keep, scale, c, exact_products=True, kept=weight_bits(dtype))
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")
    check(dr, rounded(want["rows"], dtype), "gradient of the rows")
    check(dq, rounded(want["queries"], dtype), "gradient of the queries")


@pytest.mark.parametrize("metric", [abi.VS_ANGULAR, abi.VS_DOT])
@pytest.mark.parametrize("dtype,t", [(abi.VS_F32, F32), (abi.VS_BF16, BF16)])
@pytest.mark.parametrize("n_q", [4, 64, 65, 300])
def test_weights_keep_their_bits_over_a_store(store_of, dtype, t, metric, n_q):
    """The gradient of a store's queries is f32, so nothing else rounds them."""
    rows, dim = 700, 32
    table, queries = steps(rows, dim, t, 6), steps(n_q, dim, F32, 7)
    queries[0, 0] = table[:, 0] = 0.25  # (no vector of zeros)
    scale = 10.0 if metric == abi.VS_ANGULAR else 8.0
    store = store_of(dtype, metric, table.float().cpu().numpy())
    targets = clicks(n_q, rows, None, 8)
    loss, lse, dq = store_loss_and_grad(store, queries, targets, scale)
    want = bounds(queries, table, targets, None, scale, cosine=metric == abi.VS_ANGULAR, exact_products=True,
                  kept=weight_bits(t))
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")
    check(dq, rounded(want["queries"], F32), "gradient of the queries")


@pytest.mark.parametrize("n_q", [5, 70, 300])
def test_an_improbable_click(store_of, n_q):
    """A clicked document far from its query: its weight, nearly one, is as large as all others together, and reaches the
    queries' gradient in f32."""
    rows, dim, scale = 640, 64, 16.0
    table, queries = steps(rows, dim, BF16, 9), steps(n_q, dim, BF16, 10)
    targets = (torch.arange(n_q, device=DEV) * 2).int()
    table[targets.long()] = -queries
    store = store_of(abi.VS_BF16, abi.VS_DOT, table.float().cpu().numpy())
    loss, lse, dq = store_loss_and_grad(store, queries.float(), targets, scale)
    want = bounds(queries, table, targets, None, scale, exact_products=True, kept=weight_bits(BF16))
    check(loss, want["loss"], "loss")
    check(dq, rounded(want["queries"], F32), "gradient of the queries")


@pytest.mark.parametrize("n_q", [1, 4, 5, 70])
@pytest.mark.parametrize("dim", [1, 4, 8])
def test_f32_products_keep_24_bits(gpu_ctx, n_q, dim):
    """So few terms that a product of planes that is missing (2^-16 of it) shows."""
    for rows in (6, 300):
        table, queries = matrix(rows, dim, F32, 11, unit=False), matrix(n_q, dim, F32, 12, unit=False)
        targets = torch.arange(n_q, device=DEV).int() % rows
        loss, lse = call_xent(gpu_ctx, queries, table, targets, None, 6.0)
        dq, dr = like(queries), like(table)
        call_xent_grads(gpu_ctx, queries, table, targets, None, 6.0, loss, lse, None, dq, dr)
        want = bounds(queries, table, targets, None, 6.0, chain=rows, share=rows)
        check(loss, want["loss"], "loss")
        check(lse, want["lse"], "lse")
        check(dq, rounded(want["queries"], F32), "gradient of the queries")
        check(dr, rounded(want["rows"], F32), "gradient of the rows")


@pytest.mark.parametrize("filtered", [False, True])
@pytest.mark.parametrize("n_q", [20, 100, 300])
def test_the_clicked_rows_weight_is_not_rounded(gpu_ctx, n_q, filtered):
    """bf16 gradients of queries in columns that the clicked documents have nearly to themselves: a weight that had been rounded
    to bf16 before, as those of the other documents are, would make two roundings where the bound has one."""
    rows, dim, scale = 700, 64, 8.0
    table, queries = steps(rows, dim, BF16, 13), steps(n_q, dim, BF16, 14)
    targets = (torch.arange(n_q, device=DEV) * 2).int()
    table[:, :32] = 0
    table[targets.long(), :32] = steps(n_q, 32, BF16, 15)
    keep = torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(16), device=DEV) < 0.5 if filtered else None
    if filtered:
        keep[targets.long()[: n_q - 3]] = True
    words = None if keep is None else words_of(keep)
    c = torch.rand(n_q, generator=torch.Generator(device=DEV).manual_seed(17), device=DEV) + 0.5
    loss, lse = call_xent(gpu_ctx, queries, table, targets, words, scale)
    dq, dr = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, words, scale, loss, lse, c, dq, dr)
    want = bounds(queries, table, targets, keep, scale, c, exact_products=True, kept=weight_bits(BF16))
    check(dq, rounded(want["queries"], BF16), "gradient of the queries")
    # (with the mistake in the 64-bit value, the clicked weights rounded, the bound is left)
    value, bound = want["queries"]
    weight = torch.expm1(-want["loss"][0]) * c * scale
    wrong = (value + (weight.bfloat16().double() - weight)[:, None] * table[targets.long()].double()).bfloat16().double()
    assert ((wrong - value).abs() > rounded((value, bound), BF16)[1]).any()
    check(dr, rounded(want["rows"], BF16), "gradient of the rows")


def exact_factor():
    """A scale near 100 whose product with log2 e is nearly a number of f32."""
    s = (64 + np.arange(1 << 16) / 1024).astype(np.float32)
    product = s * np.float32(np.log2(np.e))
    return float(s[np.argmin(np.abs(product.astype(np.float64) / (s.astype(np.float64) * np.log2(np.e)) - 1))])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q", [1, 2, 3, 4, 5, 70, 300])
def test_large_logits_lose_nothing_to_their_size(gpu_ctx, dtype, n_q):
    """Logits of hundreds, the clicked one and another equal and far above the rest: the loss is log 2, and a rounding of a
    logit before the largest is taken off (2^-24 of hundreds) would show."""
    dim, rows, scale = 8, 200, exact_factor()
    table, queries = steps(rows + n_q, dim, dtype, 18) * 8, steps(n_q, dim, dtype, 19) * 8
    targets = (rows + torch.arange(n_q, device=DEV)).int()
    table[targets.long()] = table[(queries.double() @ table[:rows].double().T).argmax(1)]
    loss, lse = call_xent(gpu_ctx, queries, table, targets, None, scale)
    want = bounds(queries, table, targets, None, scale, exact_products=True, exact_factor=True)
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")


@pytest.mark.parametrize("dtype,t", [(abi.VS_F32, F32), (abi.VS_BF16, BF16)])
@pytest.mark.parametrize("n_q", [3, 70])
@pytest.mark.parametrize("size", [1e25, 1e-25])
def test_cosines_of_long_and_short_queries(store_of, dtype, t, n_q, size):
    """Queries whose squares f32 does not hold: a cosine knows no length."""
    rows, dim, scale = 300, 40, 12.0
    table, queries = matrix(rows, dim, t, 20), (matrix(n_q, dim, F32, 21) * size).to(t).float()
    store = store_of(dtype, abi.VS_ANGULAR, table.float().cpu().numpy())
    targets = torch.arange(n_q, device=DEV).int() * 4
    loss, lse, dq = store_loss_and_grad(store, queries, targets, scale)
    want = bounds(queries, table, targets, None, scale, cosine=True, kept=weight_bits(t))
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")
    check(dq, rounded(want["queries"], F32), "gradient of the queries")


@pytest.mark.parametrize("dtype,t", [(abi.VS_F32, F32), (abi.VS_BF16, BF16)])
@pytest.mark.parametrize("metric", [abi.VS_ANGULAR, abi.VS_DOT])
@pytest.mark.parametrize("n_q", [1, 4, 70])
def test_a_documents_nan_is_no_number_in_any_loss(store_of, dtype, t, metric, n_q):
    """Whichever way a batch of this size goes, as a candidate and as the clicked document; filtered out it is in none."""
    rows, dim = 300, 40
    table = matrix(rows, dim, t, 22).float().cpu().numpy()
    table[7, 3] = np.nan
    store = store_of(dtype, metric, table)
    queries = matrix(n_q, dim, F32, 23)
    keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    keep[7] = False
    for first in (7, 100):
        targets = (first + torch.arange(n_q, device=DEV)).int()
        loss, lse, dq = store_loss_and_grad(store, queries, targets, 5.0)
        assert torch.isnan(loss).all() and torch.isnan(dq).all()
        loss, lse, dq = store_loss_and_grad(store, queries, targets, 5.0, words_of(torch.nn.functional.pad(keep, (0, 20))))
        assert torch.isfinite(lse).all() and torch.isfinite(loss).all() and torch.isfinite(dq).all()
        assert (loss[targets != 7] > 0).all() and (loss[targets == 7] == 0).all()
    assert torch.isnan(store_loss_and_grad(store, queries, torch.full((n_q,), -1, device=DEV).int(), 5.0)[1]).all()


@pytest.mark.parametrize("dtype,t", [(abi.VS_F32, F32), (abi.VS_BF16, BF16)])
@pytest.mark.parametrize("n_q", [1, 4, 5, 70])
def test_a_clicked_document_without_a_length(store_of, dtype, t, n_q):
    """Documents whose length a store keeps as infinity (its square passes f32) or as zero have cosine zero with everything, as
    in the searches' quotient; a click on one counts like any other."""
    rows, dim, scale = 300, 40, 7.0
    table, queries = matrix(rows, dim, t, 24), matrix(n_q, dim, F32, 25).to(t).float()
    as_stored = table.float().clone()
    for i in range(0, 2 * n_q + 8, 4):
        as_stored[i] *= 1e36 if i % 8 else 1e25
        as_stored[i + 1] = 0
        table[i : i + 2] = 0
    store = store_of(dtype, abi.VS_ANGULAR, as_stored.cpu().numpy())
    targets = (torch.arange(n_q, device=DEV) * 2).int()
    targets[1::2] -= 1
    loss, lse, dq = store_loss_and_grad(store, queries, targets, scale)
    want = bounds(queries, table, targets, None, scale, cosine=True, kept=weight_bits(t))
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")
    check(dq, rounded(want["queries"], F32), "gradient of the queries")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q", [4, 5, 70])
def test_a_scale_that_is_no_number(gpu_ctx, dtype, n_q):
    table, queries = matrix(300, 40, dtype, 26), matrix(n_q, 40, dtype, 27)
    loss, lse = call_xent(gpu_ctx, queries, table, clicks(n_q, 300, None, 28), None, float("nan"))
    assert torch.isnan(lse).all() and torch.isnan(loss[0])


@pytest.mark.parametrize("n_q", [3, 5, 70])
def test_long_queries_under_a_small_scale(store_of, n_q):
    """The factor of a query's products, scale over length, is below the smallest normal f32."""
    rows, dim, scale = 300, 40, 0.01
    table, queries = matrix(rows, dim, F32, 29), matrix(n_q, dim, F32, 30) * 1e37
    store = store_of(abi.VS_F32, abi.VS_ANGULAR, table.cpu().numpy())
    targets = torch.arange(n_q, device=DEV).int() * 4
    loss, lse, _ = store_loss_and_grad(store, queries, targets, scale)
    want = bounds(queries, table, targets, None, scale, cosine=True)
    # (in base 2 a factor near 1e-39 is a multiple of 2^-149: off by 2^-150 times products of up to 2^123 each)
    for got, name in ((loss, "loss"), (lse, "lse")):
        value, bound = want[name]
        check(got, (value, bound + 2 * 2.0**-27), name)


def certain(rows, n_q, dim, dtype, seed):
    """Queries with nearly all of their probability on one document, which was not clicked."""
    table, near = matrix(rows, dim, dtype, seed), torch.arange(n_q, device=DEV)
    queries = (table[near].float() * 6 + matrix(n_q, dim, F32, seed + 1) / 8).to(dtype)
    return table, queries, near, (rows - 1 - near % 90).int()


# The certain document's logit, a sum of thousands of roundings, is in lse with the weight of one and in its own weight again: what
# the roundings make of it has to be the same both times, and cancel, whichever way the loss went. So the bounds count none of
# them; nor those of the sums, of which the others are a millionth.
ALONE = dict(exact_products=True, exact_factor=True, chain=2, share=2, joins=2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q,dim", [(1, 1024), (1, 8192), (2, 6000), (3, 4096), (4, 3071), (5, 8192), (70, 8192), (130, 4096), (300, 4100)])
def test_a_certain_other_document(gpu_ctx, dtype, n_q, dim):
    rows, scale = 400, 4.0
    table, queries, near, targets = certain(rows, n_q, dim, dtype, 31)
    loss, lse = call_xent(gpu_ctx, queries, table, targets, None, scale)
    dq, dr = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, None, scale, loss, lse, None, dq, dr)
    want = bounds(queries, table, targets, None, scale, kept=weight_bits(dtype), **ALONE)
    assert float(want["loss"][0].min()) > 15
    check(dq, rounded(want["queries"], dtype), "gradient of the queries")
    value, bound = rounded(want["rows"], dtype)
    check(dr[near], (value[near], bound[near]), "gradient of the certain rows")


@pytest.mark.parametrize("dtype,t", [(abi.VS_F32, F32), (abi.VS_BF16, BF16)])
@pytest.mark.parametrize("n_q,dim", [(1, 4096), (2, 4000), (3, 4000), (4, 3001), (5, 4096), (130, 4000)])
def test_a_certain_other_document_of_a_store(store_of, dtype, t, n_q, dim):
    table, queries, near, targets = certain(400, n_q, dim, t, 33)
    store = store_of(dtype, abi.VS_DOT, table.float().cpu().numpy())
    loss, lse, dq = store_loss_and_grad(store, queries.float(), targets, 4.0)
    want = bounds(queries, table, targets, None, 4.0, kept=weight_bits(t), **ALONE)
    check(dq, rounded(want["queries"], F32), "gradient of the queries")


@pytest.mark.parametrize("n_q", [1, 4, 5, 70, 300])
@pytest.mark.parametrize("over_store", [False, True])
def test_a_certain_other_document_with_a_large_logit(gpu_ctx, store_of, n_q, over_store):
    """lse near 100 is the certain document's logit, rounded to f32 (2^-24 of 100). In its weight, nearly one, that rounding cancels
    if the logit is rounded the same way there; products are exact here, so that it is known which way. (Left out: logits so near
    to the middle between two numbers of f32 that the sum's own rounding may turn lse the other way.)"""
    rows, dim, scale = 400, 64, 25.3
    table, near = steps(rows, dim, F32, 35), torch.arange(n_q, device=DEV)
    queries = table[near] * 2
    targets = (rows - 1 - near % 90).int()
    logit = (queries.double() * table[near].double()).sum(1) * float(np.float32(scale))
    others = queries.double() @ table.double().T * scale
    others[near, near] = -math.inf
    other_way = (logit.float().double() - logit).abs() + 4 * U32 > (torch.nextafter(logit.float(), torch.full_like(logit, 1e9).float())
                                                                    - logit.float()).double() / 2
    sure = (logit - others.amax(1) > 25) & ~other_way & (targets.long() != near)
    assert int(sure.sum()) > 0.6 * n_q and float(logit.min()) > 25 and float(logit.max()) > 90
    if over_store:
        store = store_of(abi.VS_F32, abi.VS_DOT, table.cpu().numpy())
        loss, lse, dq = store_loss_and_grad(store, queries, targets, scale)
    else:
        loss, lse = call_xent(gpu_ctx, queries, table, targets, None, scale)
        dq = like(queries)
        call_xent_grads(gpu_ctx, queries, table, targets, None, scale, loss, lse, None, dq, None)
    value = scale * (table[near].double() - table[targets.long()].double())
    size = scale * (table[near].double().abs() + table[targets.long()].double().abs())
    # the weight: 8 roundings; the product with the row and the sum: 4; the click's: 4; all others: exp(-25) each at most, of
    # elements of 1/4 at most
    bound = size * 16 * U32 + rows * math.exp(-25) * scale / 4
    check(dq[sure], (value[sure], bound[sure]), "gradient of the queries")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q", [3, 64, 65, 300])
@pytest.mark.parametrize("filtered", [False, True])
def test_a_copy_of_the_clicked_document(gpu_ctx, dtype, n_q, filtered):
    """The clicked document and one that differs from it in one column share the probability: the query's gradient is their
    difference, and all that is left of the other columns is what the weights are off by (2^-8 of each, were they rounded to
    bf16)."""
    rows, dim, scale = 700, 64, 25.3
    table, near = steps(rows, dim, dtype, 36), torch.arange(n_q, device=DEV)
    queries = table[near] * 2
    queries[:, 0] = 0
    copies = rows - 1 - near
    table[copies] = table[near]
    table[copies, 0] = 0.25 - table[near, 0].abs()  # (another number than before)
    logit = (queries.double() * table[near].double()).sum(1) * scale
    others = queries.double() @ table.double().T * scale
    others[near, near] = others[near, copies] = -math.inf
    sure = logit - others.amax(1) > 25
    assert int(sure.sum()) > 0.6 * n_q
    words = None
    if filtered:
        keep = torch.ones(rows, dtype=torch.bool, device=DEV)
        keep[n_q + 5 : n_q + 40] = False
        words = words_of(keep)
    c = torch.rand(n_q, generator=torch.Generator(device=DEV).manual_seed(37), device=DEV) + 0.5
    loss, lse = call_xent(gpu_ctx, queries, table, near.int(), words, scale)
    dq, dr = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, near.int(), words, scale, loss, lse, c, dq, dr)
    half = (c.double() * scale / 2)[:, None]
    value = half * (table[copies].double() - table[near].double())
    size = half * (table[copies].double().abs() + table[near].double().abs())
    # the weights: lse's rounding and the logit's own (2^-24 of 100 and less), 8 roundings, the planes; all others exp(-25) each
    off = 2 * U32 * logit[:, None] + 16 * U32 + (0 if dtype == F32 else 2.0**-16)
    bound = size * off + rows * math.exp(-25) * c.double().max() * scale / 4
    check(dq[sure], tuple(t[sure] for t in rounded((value, bound), dtype)), "gradient of the queries")
    value, bound = half * queries.double(), half * queries.double().abs() * off + n_q * math.exp(-25) * c.double().max() * scale / 2
    check(dr[copies[sure]], tuple(t[sure] for t in rounded((value, bound), dtype)), "gradient of the copies")
    check(dr[near[sure]], tuple(t[sure] for t in rounded((-value, bound), dtype)), "gradient of the clicked rows")


@pytest.mark.parametrize("over_store", [False, True])
@pytest.mark.parametrize("n_q", [1, 5, 100])
def test_small_shares_are_not_lost_in_a_large_one(gpu_ctx, store_of, n_q, over_store):
    """The clicked document's share of a query's gradient is nearly one, each other workgroup's 0.4 of its last bit: added to it
    in f32 one after the other, all of them would be lost."""
    rows, dim, scale = 16384, 64, 8.0
    for dtype, t in ((abi.VS_F32, F32),) + (((abi.VS_BF16, BF16),) if over_store else ()):
        table, queries = torch.zeros(rows, dim, dtype=t, device=DEV), torch.zeros(n_q, dim, dtype=t, device=DEV)
        table[:, 0] = 0.4 * 256 * 2.0**-24  # (every logit is zero, each probability 1 / rows, and 64 rows or more a share)
        table[0, 0] = 1
        queries[:, 1] = 1
        targets = torch.zeros(n_q, dtype=torch.int32, device=DEV)
        if over_store:
            store = store_of(dtype, abi.VS_DOT, table.float().cpu().numpy())
            loss, lse, dq = store_loss_and_grad(store, queries.float(), targets, scale)
        else:
            loss, lse = call_xent(gpu_ctx, queries, table, targets, None, scale)
            dq = like(queries)
            call_xent_grads(gpu_ctx, queries, table, targets, None, scale, loss, lse, None, dq, None)
        want = bounds(queries, table, targets, None, scale, exact_products=True, exact_factor=True, chain=64, kept=weight_bits(t),
                      share=-(-rows * -(-n_q // 64) // 256), joins=0)
        check(dq, rounded(want["queries"], F32), "gradient of the queries")

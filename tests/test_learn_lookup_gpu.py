"""Pooled row lookup and its gradients against 64-bit forms, at the sizes where they can go wrong."""
import pytest
import torch

from learn_helpers import (DEV, bag_of_positions, call_lookup, call_row_grads, call_weight_grads, check, ids_tensor,
                           lookup_reference, row_grads_reference, weight_grads_reference)
from search_engine_amd import abi

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def table_of(rows, dim, dtype, seed, pad=0, offset=0):
    """A table inside a larger buffer of NaN: `pad` elements between rows, `offset` elements before the first."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    flat = torch.full((offset + rows * (dim + pad) + 64,), float("nan"), device=DEV, dtype=dtype)
    t = flat[offset : offset + rows * (dim + pad)].view(rows, dim + pad)[:, :dim]
    t.copy_(torch.randn(rows, dim, generator=g, device=DEV))
    return t


def bags(sizes, rows, seed, weighted=True, tail=0, head=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = head + sum(sizes) + tail
    off = torch.tensor([head] + [head + sum(sizes[: i + 1]) for i in range(len(sizes))], device=DEV).int()
    ids = torch.randint(0, rows, (n,), generator=g, device=DEV).int()
    w = torch.randn(n, generator=g, device=DEV) if weighted else None
    return ids, off, w


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("dim,pad,offset", [(1, 0, 0), (7, 0, 0), (8, 0, 0), (8, 8, 0), (8, 0, 1), (64, 1, 0), (100, 4, 4),
                                            (383, 0, 0), (384, 0, 0), (768, 0, 8), (1536, 0, 0), (8192, 0, 0)])
def test_lookup(gpu_ctx, dtype, out_dtype, dim, pad, offset):
    rows = 37
    table = table_of(rows, dim, dtype, 1, pad, offset)
    ids, off, w = bags([3, 0, 1, 5, 4, 40, 0], rows, 2, tail=3, head=2)
    ids[4], ids[9] = -1, rows  # no rows
    out = table_of(7, dim, out_dtype, 3, pad, offset)
    gap = out.as_strided((7, dim + pad), (dim + pad, 1))[:, dim:].clone()
    call_lookup(gpu_ctx, table, ids, off, 7, w, 0.75, out)
    check(out, lookup_reference(table, ids, off, 7, w, 0.75, out_dtype), "lookup")
    assert torch.isnan(out.as_strided((7, dim + pad), (dim + pad, 1))[:, dim:]).all() and torch.isnan(gap).all()


@pytest.mark.parametrize("sizes", [[1], [0], [1, 0, 0, 2], [17], [1000], [2000, 1, 3], [5000, 5000], [16] * 4, [300] * 70])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [5, 384])
def test_lookup_of_bags_of_many_sizes(gpu_ctx, sizes, dtype, dim):
    table = table_of(5000, dim, dtype, 4)
    for weighted in (False, True):
        ids, off, w = bags(sizes, 5000, 5, weighted)
        out = call_lookup(gpu_ctx, table, ids, off, len(sizes), w, 2.0, torch.empty(len(sizes), dim, device=DEV))
        check(out, lookup_reference(table, ids, off, len(sizes), w, 2.0, F32), f"lookup {sizes}")
        again = call_lookup(gpu_ctx, table, ids, off, len(sizes), w, 2.0, torch.empty(len(sizes), dim, device=DEV))
        assert torch.equal(out, again)


def test_plain_lookup_without_bags(gpu_ctx):
    table = table_of(100, 48, BF16, 6)
    ids = ids_tensor([5, 99, 100, 0, 5, 2**32 - 1])
    out = call_lookup(gpu_ctx, table, ids, None, 8, None, 1.0, torch.full((8, 48), 9.0, device=DEV, dtype=BF16))
    want = torch.zeros(8, 48, device=DEV, dtype=BF16)
    for i, r in enumerate([5, 99, None, 0, 5, None]):
        if r is not None:
            want[i] = table[r]
    assert torch.equal(out, want)  # one row times one: exact


def test_a_row_that_no_id_names_is_not_seen(gpu_ctx):
    """Row 0 holds NaN (it stands in for rows that ids without one would have): it reaches no result."""
    table = table_of(10, 64, F32, 7)
    table[0] = float("nan")
    ids = ids_tensor([3, 2**32 - 1, 4, 77, 5])
    off = torch.tensor([0, 2, 5, 5], device=DEV).int()
    out = call_lookup(gpu_ctx, table, ids, off, 3, None, 1.0, torch.empty(3, 64, device=DEV))
    check(out, lookup_reference(table, ids, off, 3, None, 1.0, F32))
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("offsets", [[0, 9, 4, 200, 3], [2**32 - 1, 0, 5, 5, 2**32 - 1]])
def test_offsets_out_of_order_stay_inside_the_ids(gpu_ctx, offsets):
    """Not allowed, and not checked (device data): nothing outside the ids is read, and the call ends."""
    table = table_of(50, 32, F32, 8)
    ids = ids_tensor(list(range(20)))
    off = ids_tensor(offsets)
    out = call_lookup(gpu_ctx, table, ids, off, 4, None, 1.0, torch.zeros(4, 32, device=DEV))
    assert torch.isfinite(out).all()
    grads = torch.zeros(50, 32, device=DEV)
    call_row_grads(gpu_ctx, torch.ones(4, 32, device=DEV), ids, off, None, 1.0, 50, grads)
    w = call_weight_grads(gpu_ctx, table, ids, off, 1.0, torch.ones(4, 32, device=DEV), torch.zeros(20, device=DEV))
    assert torch.isfinite(grads).all() and torch.isfinite(w).all()


def grad_case(n, rows, n_bags, skew, seed, weighted=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cut = torch.sort(torch.randint(0, n + 1, (n_bags - 1,), generator=g, device=DEV)).values
    off = torch.cat([torch.zeros(1, device=DEV), cut, torch.full((1,), n, device=DEV)]).int()
    ids = (torch.rand(n, generator=g, device=DEV, dtype=torch.float64).pow(skew) * rows).int()
    w = torch.randn(n, generator=g, device=DEV) if weighted else None
    return ids, off, w


GRADS = [(1, 1, 1, 1), (5, 10, 2, 1), (64, 3, 9, 1), (300, 1000, 20, 4), (2048, 1, 7, 1), (2048, 100, 300, 2),
         (2049, 1, 7, 1), (2049, 70000, 50, 1), (4097, 255, 100, 1), (4160, 256, 100, 3), (9000, 300, 5, 8),
         (70000, 5, 4000, 1), (70000, 20000000, 4000, 1), (200001, 100000, 3000, 4)]


@pytest.mark.parametrize("n,rows,n_bags,skew", GRADS)
@pytest.mark.parametrize("dtype,grad_dtype,dim", [(F32, F32, 20), (BF16, F32, 64), (BF16, BF16, 33), (F32, BF16, 3)])
def test_row_gradients(gpu_ctx, n, rows, n_bags, skew, dtype, grad_dtype, dim):
    ids, off, w = grad_case(n, rows, n_bags, skew, 9)
    g = table_of(n_bags, dim, dtype, 10)
    # compact: the named rows ascending, what lies behind them as it was
    unique = torch.full((n,), 12345678, dtype=torch.int32, device=DEV)
    count = torch.full((1,), -7, dtype=torch.int32, device=DEV)
    got = torch.full((n, dim), 5.0, dtype=grad_dtype, device=DEV)
    call_row_grads(gpu_ctx, g, ids, off, w, 0.5, rows, got, unique, count)
    names, place = torch.unique(ids.long(), return_inverse=True)
    k = names.numel()
    assert int(count) == k and torch.equal(unique[:k].long(), names)
    assert (unique[k:] == 12345678).all() and (got[k:] == 5.0).all()
    value, bound, _ = row_grads_reference(g, place, off, w, 0.5, k, grad_dtype)
    check(got[:k], (value, bound), "compact")
    # twice the same bits
    again = torch.empty_like(got)
    call_row_grads(gpu_ctx, g, ids, off, w, 0.5, rows, again, unique, count)
    assert torch.equal(again[:k], got[:k])
    # added to a table
    if rows <= 100000:
        base = table_of(rows, dim, grad_dtype, 11, pad=1)
        want = base.double()
        value, bound, named = row_grads_reference(g, ids, off, w, 0.5, rows, F32)
        before = base.clone()
        call_row_grads(gpu_ctx, g, ids, off, w, 0.5, rows, base)
        half = torch.finfo(grad_dtype).eps / 2
        check(base, (want + value, bound + half * ((want + value).abs() + bound) + 2.0**-24 * (want + value).abs()), "added")
        assert torch.equal(base[~named], before[~named])


def test_row_gradients_without_bags_and_with_ids_that_name_nothing(gpu_ctx):
    n, rows, dim = 3000, 50, 24
    g = torch.Generator(device=DEV).manual_seed(12)
    ids = torch.randint(-3, rows + 5, (n,), generator=g, device=DEV).int()
    grad = torch.randn(2500, dim, generator=g, device=DEV)  # positions from 2500 on are in no bag
    for part in (ids, ids[:900]):
        got = torch.zeros(rows, dim, device=DEV)
        call_row_grads(gpu_ctx, grad, part, None, None, 1.5, rows, got)
        value, bound, _ = row_grads_reference(grad, part, None, None, 1.5, rows, F32)
        check(got, (value, bound))


def test_no_ids_and_no_bags(gpu_ctx):
    count = torch.full((1,), 9, dtype=torch.int32, device=DEV)
    unique = torch.full((4,), 3, dtype=torch.int32, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    grads = torch.full((4, 8), 2.0, device=DEV)
    call_row_grads(gpu_ctx, torch.ones(2, 8, device=DEV), none, off, None, 1.0, 10, grads, unique, count)
    assert int(count) == 0 and (unique == 3).all() and (grads == 2).all()
    out = call_lookup(gpu_ctx, torch.ones(3, 8, device=DEV), none, off, 2, None, 1.0, torch.ones(2, 8, device=DEV))
    assert (out == 0).all()
    call_lookup(gpu_ctx, torch.ones(3, 8, device=DEV), none, None, 0, None, 1.0, torch.ones(0, 8, device=DEV))


@pytest.mark.parametrize("dtype,grad_dtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("n,rows,n_bags,dim,pad", [(1, 1, 1, 1, 0), (50, 20, 7, 100, 0), (3000, 500, 400, 384, 0),
                                                   (40000, 10, 9000, 72, 8), (333, 40, 5, 77, 1)])
def test_weight_gradients(gpu_ctx, dtype, grad_dtype, n, rows, n_bags, dim, pad):
    ids, off, _ = grad_case(n, rows, n_bags, 1, 13)
    ids[n // 2] = rows + 3
    table, g = table_of(rows, dim, dtype, 14, pad), table_of(n_bags, dim, grad_dtype, 15, pad)
    out = call_weight_grads(gpu_ctx, table, ids, off, 0.3, g, torch.full((n,), 4.0, device=DEV))
    check(out, weight_grads_reference(table, g, ids, off, 0.3), "weights")


def test_gradients_against_differences(gpu_ctx):
    """<dout, lookup(table + h)> - <dout, lookup(table - h)> over 2 h: the lookup is linear, so a difference in 64 bits of
    the reference is the gradient itself."""
    rows, dim = 12, 10
    table = table_of(rows, dim, F32, 16)
    ids, off, w = bags([2, 3, 0, 4], rows, 17)
    g = torch.randn(4, dim, device=DEV)
    grads = torch.zeros(rows, dim, device=DEV)
    call_row_grads(gpu_ctx, g, ids, off, w, 0.7, rows, grads)
    dw = call_weight_grads(gpu_ctx, table, ids, off, 0.7, g, torch.zeros(9, device=DEV))

    def f(t, ww):
        return float((lookup_reference(t, ids, off, 4, ww, 0.7, F32)[0] * g.double()).sum())
    for r, c in ((int(ids[0]), 0), (int(ids[3]), 9), (int(ids[8]), 4)):
        h = torch.zeros(rows, dim, dtype=torch.float64, device=DEV)
        h[r, c] = 0.5
        diff = f(table.double() + h, w) - f(table.double() - h, w)
        assert abs(diff - float(grads[r, c])) <= 1e-5 * (1 + abs(diff))
    for i in (0, 4, 8):
        h = torch.zeros(9, dtype=torch.float64, device=DEV)
        h[i] = 0.5
        diff = f(table, w.double() + h) - f(table, w.double() - h)
        assert abs(diff - float(dw[i])) <= 1e-5 * (1 + abs(diff))


def test_lookup_of_a_store(gpu_ctx):
    """Documents by docid from the sealed rows: removed and missing ones add nothing, unsealed changes are not seen."""
    import numpy as np
    rng = np.random.default_rng(18)
    for dtype, t in ((abi.VS_F32, F32), (abi.VS_BF16, BF16)):
        for dim in (384, 99):
            rows = rng.standard_normal((300, dim), dtype=np.float32)
            store = gpu_ctx.create_store(0x4100, dim, 1000, dtype=dtype, docid_base=640)
            store.upload(np.arange(640, 940, dtype=np.uint32), rows)
            store.remove(np.array([650, 700], np.uint32))
            store.seal()
            store.upload(np.array([941], np.uint32), rows[:1])  # not sealed
            ids = ids_tensor([640, 650, 939, 941, 0, 639, 5000, 641, 641])
            off = torch.tensor([0, 1, 4, 9], device=DEV).int()
            w = torch.tensor([1.0, 2, 3, 4, 5, 6, 7, 8, 9], device=DEV)
            out = torch.empty(3, dim, device=DEV)
            store.lookup_device(ids.data_ptr(), 9, off.data_ptr(), 3, w.data_ptr(), 0.5, out.data_ptr(), abi.VS_F32,
                                out.stride(0), torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            table = torch.zeros(1000, dim, device=DEV, dtype=t)
            table[:300] = torch.from_numpy(rows).to(DEV)
            local = ids_tensor([0, 2**32 - 1, 299] + [2**32 - 1] * 4 + [1, 1])
            check(out, lookup_reference(table, local, off, 3, w, 0.5, F32), "store lookup")
            store.destroy()


def test_bag_of_positions_reference():
    off = torch.tensor([1, 1, 3, 6], device=DEV).int()
    assert bag_of_positions(8, off, 3).tolist() == [-1, 1, 1, 2, 2, 2, -1, -1]

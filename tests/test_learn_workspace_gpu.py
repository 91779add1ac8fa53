"""Workspaces of the cross entropy: what each call asks for, that it is enough, and that it is no more than the call uses."""
import pytest
import torch

from learn_helpers import DEV, TYPE, ptr
from search_engine_amd import abi
from test_learn_precision_gpu import store_of  # noqa: F401  (a fixture)
from test_learn_xent_gpu import clicks, like, matrix

F32, BF16 = torch.float32, torch.bfloat16
GUARD = 4096


def guarded(n):
    """A workspace of n bytes, with bytes behind it that are known."""
    t = torch.full((n + GUARD,), 0x5A, dtype=torch.uint8, device=DEV)
    return t, lambda: bool((t[n:] == 0x5A).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q,rows,dim,pad", [(1, 3000, 64, 0), (4, 3000, 64, 0), (5, 3000, 64, 0), (70, 3000, 61, 0), (300, 3000, 64, 3),
                                              (3, 3000, 61, 0), (130, 100, 768, 0)])
def test_one_calls_workspace_is_enough(gpu_ctx, dtype, n_q, rows, dim, pad):
    table, queries = matrix(rows, dim, dtype, 1, pad), matrix(n_q, dim, dtype, 2)
    targets, code = clicks(n_q, rows, None, 3), TYPE[dtype]
    st = torch.cuda.current_stream().cuda_stream
    both = gpu_ctx.xent_workspace_bytes(n_q, rows, dim, code)
    need = [gpu_ctx.xent_call_workspace_bytes(n_q, ptr(table), rows, table.stride(0), code, dim, g) for g in (False, True)]
    assert need[0] < need[1] <= both
    if n_q <= 4:
        assert need[0] <= 2048 * 8 * n_q + 1024
    results = []
    for sizes in ((both, both), need):
        loss, lse = torch.empty(2, n_q, device=DEV)
        dq, dr = like(queries), like(table)
        (ws, whole), (ws2, whole2) = guarded(sizes[0]), guarded(sizes[1])
        args = (ptr(queries), n_q, queries.stride(0), ptr(table), rows, table.stride(0), code, dim, ptr(targets), None, 6.0)
        gpu_ctx.xent_device(*args, ptr(ws), sizes[0], ptr(loss), ptr(lse), st)
        gpu_ctx.xent_grad_device(*args, ptr(loss), ptr(lse), None, ptr(ws2), sizes[1], ptr(dq), ptr(dr), st)
        assert whole() and whole2()
        results.append((loss, lse, dq, dr))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    for gradients, call in ((0, lambda n: gpu_ctx.xent_device(*args, ptr(ws), n, ptr(loss), ptr(lse), st)),
                            (1, lambda n: gpu_ctx.xent_grad_device(*args, ptr(loss), ptr(lse), None, ptr(ws2), n, ptr(dq), None, st))):
        with pytest.raises(abi.VsError) as e:
            call(need[gradients] // 2)
        assert e.value.code == abi.VS_E_CAPACITY


@pytest.mark.gpu
def test_the_loss_of_one_query_takes_little(gpu_ctx):
    """A million rows: neither weights nor copies of rows are asked for; an address off by an element asks for the copies."""
    rows, dim = 1000000, 768
    for dtype, size in ((abi.VS_BF16, 2), (abi.VS_F32, 4)):
        p = 1 << 20  # (no rows are read for the question)
        assert gpu_ctx.xent_call_workspace_bytes(1, p, rows, dim, dtype, dim, False) < 20000
        assert gpu_ctx.xent_call_workspace_bytes(1, p + size, rows, dim, dtype, dim, False) < 20000
        batch = gpu_ctx.xent_call_workspace_bytes(100, p, rows, dim, dtype, dim, False)
        assert batch < 16 << 20
        assert gpu_ctx.xent_call_workspace_bytes(100, p + size, rows, dim, dtype, dim, False) > batch + (1 << 29)
        assert gpu_ctx.xent_workspace_bytes(100, rows, dim, dtype) > 1 << 30


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,t", [(abi.VS_F32, F32), (abi.VS_BF16, BF16)])
@pytest.mark.parametrize("n_q", [2, 20, 100])
@pytest.mark.parametrize("dim", [64, 61])
def test_one_calls_workspace_over_a_store(store_of, dtype, t, n_q, dim):  # noqa: F811
    rows = 1000
    table, queries = matrix(rows, dim, t, 4), matrix(n_q, dim, F32, 5)
    store = store_of(dtype, abi.VS_ANGULAR, table.float().cpu().numpy())
    targets, st = clicks(n_q, rows, None, 6), torch.cuda.current_stream().cuda_stream
    need = [store.xent_call_workspace_bytes(n_q, g) for g in (False, True)]
    both = store.xent_workspace_bytes(n_q)
    assert need[0] < need[1] <= both
    results = []
    for sizes in ((both, both), need):
        loss, lse = torch.empty(2, n_q, device=DEV)
        dq = torch.empty(n_q, dim, device=DEV)
        (ws, whole), (ws2, whole2) = guarded(sizes[0]), guarded(sizes[1])
        store.xent_device(ptr(queries), n_q, dim, ptr(targets), None, 6.0, ptr(ws), sizes[0], ptr(loss), ptr(lse), st)
        store.xent_grad_device(ptr(queries), n_q, dim, ptr(targets), None, 6.0, ptr(loss), ptr(lse), None, ptr(ws2), sizes[1], ptr(dq), st)
        assert whole() and whole2()
        results.append((loss, lse, dq))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    with pytest.raises(abi.VsError) as e:
        store.xent_device(ptr(queries), n_q, dim, ptr(targets), None, 6.0, ptr(ws), need[0] // 2, ptr(loss), ptr(lse), st)
    assert e.value.code == abi.VS_E_CAPACITY


def test_what_the_question_refuses():
    import ctypes
    n, p = ctypes.c_uint64(0), 1 << 20
    for args, part in (((None, 1, p, 0, 8, abi.VS_F32, 8, 0), "rows"), ((None, 1, p, 10, 8, abi.VS_F32, 0, 0), "dimension"),
                       ((None, 1, p, 10, 8, abi.VS_BIN1, 8, 0), "type"), ((None, 1, p, 10, 7, abi.VS_F32, 8, 1), "stride"),
                       ((None, 1, p + 2, 10, 8, abi.VS_F32, 8, 1), "aligned"), ((None, 1, None, 10, 8, abi.VS_F32, 8, 1), "null"),
                       ((None, abi.VS_XENT_MAX_QUERIES + 1, p, 10, 8, abi.VS_F32, 8, 0), "n_q"),
                       ((None, 1, p, 10, 8, abi.VS_F32, 8, 0), "null context")):
        with pytest.raises(abi.VsError) as e:
            abi._check(abi.lib.vs_xent_call_workspace_bytes(*args, ctypes.byref(n)))
        assert e.value.code == abi.VS_E_INVALID_ARG and part in e.value.message
    assert abi.lib.vs_xent_call_workspace_bytes(None, 1, p, 10, 8, abi.VS_F32, 8, 0, None) == abi.VS_E_INVALID_ARG
    assert abi.lib.vs_store_xent_call_workspace_bytes(None, 1, 0, ctypes.byref(n)) == abi.VS_E_INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q", [1, 4])
def test_a_few_queries_captured_with_what_they_need(gpu_ctx, dtype, n_q):
    """Loss and gradients in a graph, each with one call's workspace; replayed with new queries and clicks, with eager calls
    between, every replay gives the eager calls' bits."""
    rows, dim, code = 5000, 60, TYPE[dtype]
    table, queries, targets = matrix(rows, dim, dtype, 7), matrix(n_q, dim, dtype, 8), clicks(n_q, rows, None, 9)
    ws = [torch.empty(gpu_ctx.xent_call_workspace_bytes(n_q, ptr(table), rows, dim, code, dim, g), dtype=torch.uint8, device=DEV)
          for g in (False, True)]
    loss, lse = torch.empty(2, n_q, device=DEV)
    dq, dr = like(queries), like(table)

    def run():
        st = torch.cuda.current_stream().cuda_stream
        args = (ptr(queries), n_q, dim, ptr(table), rows, dim, code, dim, ptr(targets), None, 7.0)
        gpu_ctx.xent_device(*args, ptr(ws[0]), ws[0].numel(), ptr(loss), ptr(lse), st)
        gpu_ctx.xent_grad_device(*args, ptr(loss), ptr(lse), None, ptr(ws[1]), ws[1].numel(), ptr(dq), ptr(dr), st)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in range(4):
        queries.copy_(matrix(n_q, dim, dtype, 10 + seed))
        targets.copy_(clicks(n_q, rows, None, 20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        first = [t.clone() for t in (loss, lse, dq, dr)]
        run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, (loss, lse, dq, dr)))
    assert torch.isfinite(dr).all()

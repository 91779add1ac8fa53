"""Learning from a store that changes: a call sees the rows of the last seal before it, also while it is still waiting for its
stream; and calls from several threads at once return what they return one at a time."""
import threading

import numpy as np
import pytest
import torch

from learn_helpers import DEV, call_lookup, call_row_grads, call_weight_grads, call_xent, call_xent_grads, ptr
from search_engine_amd import abi
from test_learn_precision_gpu import store_of  # noqa: F401  (a fixture)
from test_learn_xent_gpu import clicks, like, matrix

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
ROWS, DIM = 2000, 48


class Calls:
    """The three calls on a store, with buffers and a stream of their own."""

    def __init__(self, store, n_q, seed):
        self.store, self.n_q, self.stream = store, n_q, torch.cuda.Stream()
        self.queries, self.targets = matrix(n_q, DIM, F32, seed), (torch.arange(n_q, device=DEV) * 3).int()
        self.ids = (torch.arange(64, device=DEV) * 17).int()
        self.out = torch.empty(8, DIM, device=DEV)
        self.off = (torch.arange(9, device=DEV) * 8).int()
        self.loss, self.lse = torch.empty(2, n_q, device=DEV)
        self.dq = torch.empty(n_q, DIM, device=DEV)
        self.ws = torch.empty(store.xent_workspace_bytes(n_q), dtype=torch.uint8, device=DEV)
        torch.cuda.synchronize()

    def lookup(self):
        self.store.lookup_device(ptr(self.ids), 64, ptr(self.off), 8, None, 1.0, ptr(self.out), abi.VS_F32, DIM, self.stream.cuda_stream)

    def learn(self):
        args = (ptr(self.queries), self.n_q, DIM, ptr(self.targets), None, 9.0)
        self.store.xent_device(*args, ptr(self.ws), self.ws.numel(), ptr(self.loss), ptr(self.lse), self.stream.cuda_stream)
        self.store.xent_grad_device(*args, ptr(self.loss), ptr(self.lse), None, ptr(self.ws), self.ws.numel(), ptr(self.dq),
                                    self.stream.cuda_stream)

    def results(self):
        self.stream.synchronize()
        return [t.clone() for t in (self.out, self.loss, self.lse, self.dq)]

    def behind_other_work(self):
        """The calls, queued behind work of some 20 ms: what the host does next, it does while they wait."""
        with torch.cuda.stream(self.stream):
            torch.cuda._sleep(40_000_000)
        self.lookup()
        self.learn()


def rows_of(seed):
    return matrix(ROWS, DIM, F32, seed).cpu().numpy()


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [abi.VS_F32, abi.VS_BF16])
@pytest.mark.parametrize("metric", [abi.VS_ANGULAR, abi.VS_DOT])
@pytest.mark.parametrize("n_q", [3, 70])
def test_a_seal_behind_a_call_that_waits(store_of, dtype, metric, n_q):  # noqa: F811
    """Rows replaced, removed and added, and sealed once and twice, before the calls have run."""
    store = store_of(dtype, metric, rows_of(1))
    calls = Calls(store, n_q, 2)
    calls.lookup()
    calls.learn()
    before = calls.results()

    def replace():
        store.upload(np.arange(0, ROWS, 2, dtype=np.uint32), 2 * rows_of(3)[::2])

    def remove_twice():
        store.remove(np.arange(1, ROWS, 3, dtype=np.uint32))
        store.seal()
        store.remove(np.arange(2, ROWS, 5, dtype=np.uint32))

    for change in (replace, remove_twice):
        calls.behind_other_work()
        change()
        store.seal()
        during = calls.results()
        assert equal(during, before)
        calls.lookup()
        calls.learn()
        after = calls.results()
        assert not equal(after, before) and all(torch.isfinite(t).all() for t in after)
        before = after


def test_a_seal_beside_a_learning_thread(store_of):  # noqa: F811
    """A writer puts one of two sets of rows into the store, over and over, while another thread learns: every call sees one
    set, whole."""
    store = store_of(abi.VS_F32, abi.VS_DOT, rows_of(4))
    ids = np.arange(ROWS, dtype=np.uint32)
    sets = [rows_of(4), rows_of(5)]
    calls = Calls(store, 20, 6)
    known = []
    for rows in sets:
        store.upload(ids, rows)
        store.seal()
        calls.lookup()
        calls.learn()
        known.append(calls.results())
    assert not equal(known[0][1:3], known[1][1:3])
    seen, stop, errors = set(), threading.Event(), []

    def learn():
        try:
            while not stop.is_set():
                calls.lookup()
                calls.learn()
                got = calls.results()
                # (the gradient's call may see another seal than the loss's: it is not compared)
                for part in (slice(0, 1), slice(1, 3)):
                    which = [i for i in (0, 1) if equal(got[part], known[i][part])]
                    assert which, "rows of two seals in one call"
                    seen.update(which)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
    thread = threading.Thread(target=learn)
    thread.start()
    for i in range(20):
        store.upload(ids, sets[i % 2])
        store.seal()
    stop.set()
    thread.join(60)
    assert not thread.is_alive()
    if errors:
        raise errors[0]
    assert seen


def test_threads_at_once(gpu_ctx, store_of):  # noqa: F811
    """Four threads, each with streams, buffers and workspaces of its own, through every call."""
    stores = [store_of(abi.VS_F32, abi.VS_ANGULAR, rows_of(7)), store_of(abi.VS_BF16, abi.VS_DOT, rows_of(8))]
    table = matrix(5000, DIM, BF16, 9)

    class Worker:
        def __init__(self, i):
            self.calls = Calls(stores[i % 2], (3, 70, 300, 9)[i], 10 + i)
            n_q = self.n_q = (70, 4, 130, 300)[i]
            self.queries, self.targets = matrix(n_q, DIM, BF16, 20 + i), clicks(n_q, 5000, None, 30 + i)
            self.ids = ((torch.arange(3000, device=DEV) * (101 + i)) % 5000).int()
            self.off = torch.linspace(0, 3000, n_q + 1, device=DEV).int()
            self.pooled, self.dq, self.dr = torch.empty(n_q, DIM, device=DEV), like(self.queries), like(table)
            self.dw = torch.empty(3000, device=DEV)
            self.ws = torch.empty(gpu_ctx.xent_workspace_bytes(n_q, 5000, DIM, abi.VS_BF16), dtype=torch.uint8, device=DEV)
            self.ws2 = torch.empty(gpu_ctx.lookup_grad_workspace_bytes(3000, 5000, DIM), dtype=torch.uint8, device=DEV)
            torch.cuda.synchronize()

        def run(self):
            with torch.cuda.stream(self.calls.stream):
                self.calls.lookup()
                self.calls.learn()
                call_lookup(gpu_ctx, table, self.ids, self.off, self.n_q, None, 1.0, self.pooled)
                self.loss, self.lse = call_xent(gpu_ctx, self.queries, table, self.targets, None, 8.0, self.ws)
                call_xent_grads(gpu_ctx, self.queries, table, self.targets, None, 8.0, self.loss, self.lse, None, self.dq, self.dr, self.ws)
                call_weight_grads(gpu_ctx, table, self.ids, self.off, 1.0, self.dq, self.dw)
                call_row_grads(gpu_ctx, self.dq, self.ids, self.off, None, 1.0, 5000, self.dr, ws=self.ws2)
                return self.calls.results() + [t.clone() for t in (self.pooled, self.loss, self.lse, self.dq, self.dr, self.dw)]
    workers = [Worker(i) for i in range(4)]
    alone = []
    for w in workers:
        alone.append(w.run())
        torch.cuda.synchronize()
    failed = []

    def again(w, want):
        try:
            for _ in range(8):
                got = w.run()
                w.calls.stream.synchronize()
                assert equal(got, want)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=again, args=a) for a in zip(workers, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads)
    if failed:
        raise failed[0]

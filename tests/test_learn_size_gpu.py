"""The cross entropy over corpora so large that a workgroup takes several tiles, of rows so long that a tile takes several
steps: every tile counts once."""
import math

import pytest
import torch

from learn_bounds import bounds, chain_of, weight_bits
from learn_helpers import DEV, call_xent, call_xent_grads, check, rounded, words_of
from test_learn_xent_gpu import gaps_are_nan, like, matrix

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def borders(rows, n_q):
    """Places where something ends or begins: of words, of tiles of 64, 128 and 256, of the tiles that a workgroup's first one
    is followed by, of the corpus; and others, until there is one for every query."""
    near = [0, 63, 64, 127, 128, 255, 256, 511, 512]
    for tile in (64, 128, 256):
        for first in (128 * tile, 256 * tile, 512 * tile):
            near += [first - 1, first, first + tile - 1, first + tile]
    last = rows // 256 * 256
    near += [rows - 1, rows - 2, rows - 64, rows - 65, last - 1, last, last - 256, last - 257, rows // 64 * 64 - 1]
    near = sorted({p for p in near if 0 <= p < rows})
    more = [p for p in ((i * 2654435761) % rows for i in range(1, 10 * n_q)) if p not in near]
    return near + more[: max(0, n_q - len(near))]


@pytest.mark.parametrize("filtered", [False, True])
@pytest.mark.parametrize("dtype,n_q,rows,dim", [
    (BF16, 100, 140000, 256), (BF16, 300, 70001, 256), (BF16, 100, 70001, 768), (BF16, 300, 140000, 768), (BF16, 40, 140000, 768),
    (BF16, 2, 140001, 200), (F32, 100, 50000, 383), (F32, 100, 50000, 384), (F32, 300, 70001, 256), (F32, 60, 140000, 256),
    (F32, 3, 100001, 100)])
def test_every_tile_counts_once(gpu_ctx, dtype, n_q, rows, dim, filtered):
    """Each query's largest logits are those of documents at borders, each with about the weight of all that are at none
    together: a tile that is lost or taken twice moves lse by 0.05 or more (two queries, 16 borders each; by 0.4 where each has
    one), and the gradients with it."""
    table, queries = matrix(rows, dim, dtype, 1), matrix(n_q, dim, dtype, 2)
    places = borders(rows, n_q)
    keep = None
    if filtered:
        keep = torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) < 0.8
        keep[places] = True
        table[~keep] = float("nan")
    n = rows if keep is None else int(keep.sum())
    scale = math.log(n)  # (the others' logits are scale times cosines of about dim^-1/2: their sum is n and a little more)
    table[places] = queries[torch.arange(len(places), device=DEV) % n_q]
    candidates = torch.arange(rows, device=DEV) if keep is None else keep.nonzero().flatten()
    targets = candidates[torch.randint(0, n, (n_q,), generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)].int()
    if n_q > 2:
        targets[1] = -1
    c = torch.rand(n_q, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)
    words = None if keep is None else words_of(keep)
    loss, lse = call_xent(gpu_ctx, queries, table, targets, words, scale)
    dq, dr = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, words, scale, loss, lse, c, dq, dr)
    # (a share of a query's gradient: the workgroups side by side are tiles of 64 queries and of 128 columns, at least)
    want = bounds(queries, table, targets, keep, scale, c, kept=weight_bits(dtype),
                  share=chain_of(n, n_q) * -(-dim // 128))
    assert float((want["lse"][1]).max()) < 5e-3
    # (with the mistake in the 64-bit value, a border's word of 64 rows lost, the bound is left)
    value, bound = want["lse"]
    for place in (places[0], places[len(places) // 2], rows - 1):
        near = torch.arange(place // 64 * 64, min(place // 64 * 64 + 64, rows), device=DEV)
        near = near if keep is None else near[keep[near]]
        share = torch.exp(queries.double() @ table[near].double().T * scale - value[:, None]).sum(1)
        assert (-torch.log1p(-share) > bound).any()
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")
    check(dq, rounded(want["queries"], dtype), "gradient of the queries")
    check(dr, rounded(want["rows"], dtype), "gradient of the rows")
    assert gaps_are_nan(dq) and gaps_are_nan(dr)
    loss2, lse2 = call_xent(gpu_ctx, queries, table, targets, words, scale)
    dq2, dr2 = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, words, scale, loss, lse, c, dq2, dr2)
    assert all(torch.equal(a, b) for a, b in ((loss, loss2), (lse, lse2), (dq, dq2), (dr, dr2)))


@pytest.mark.parametrize("filtered", [False, True])
@pytest.mark.parametrize("dtype,rows", [(BF16, 4300001), (F32, 2900003)])
def test_a_few_queries_over_more_than_one_piece(gpu_ctx, dtype, rows, filtered):
    """Weights of up to four queries, a piece of the rows at a time: documents at the pieces' borders have most of the probability."""
    n_q, dim = 3, 8
    table, queries = matrix(rows, dim, dtype, 6), matrix(n_q, dim, dtype, 7)
    piece = (1 << 30) // (64 * 2 * (3 if dtype == F32 else 2)) // 65536 * 65536
    places = torch.tensor([0, piece - 1, piece, rows - 1, piece + 7, 3, 63, 64, piece // 2], device=DEV)
    queries *= 2
    table[places] = queries[torch.arange(9, device=DEV) % n_q] * 2
    keep = None
    if filtered:
        keep = torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(8), device=DEV) < 0.98
        keep[places] = True
        table[~keep] = float("nan")
    targets = torch.tensor([5, piece + 1, rows - 2], device=DEV).int()
    if keep is not None:
        keep[targets.long()] = True
        table[targets.long()] = 0.25
    words = None if keep is None else words_of(keep)
    loss, lse = call_xent(gpu_ctx, queries, table, targets, words, 2.0)
    dq, dr = like(queries), like(table)
    call_xent_grads(gpu_ctx, queries, table, targets, words, 2.0, loss, lse, None, dq, dr)
    want = bounds(queries, table, targets, keep, 2.0, kept=weight_bits(dtype), share=chain_of(rows, n_q))
    check(loss, want["loss"], "loss")
    check(lse, want["lse"], "lse")
    check(dq, rounded(want["queries"], dtype), "gradient of the queries")
    check(dr, rounded(want["rows"], dtype), "gradient of the rows")

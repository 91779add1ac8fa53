"""64-bit forms of the operators that learn from clicks, with the bounds their results have to keep, and the calls.

Bounds are derived, not fitted. u(t) = torch.finfo(t).eps / 2 is the largest relative error of one rounding. A sum of n
products in f32 is off by at most (n + 2) u(f32) times the sum of the products' magnitudes, in any order.
"""
import torch

from search_engine_amd import abi

DEV = "cuda:0"
TYPE = {torch.float32: abi.VS_F32, torch.bfloat16: abi.VS_BF16}
U32 = torch.finfo(torch.float32).eps / 2


def u(t):
    return torch.finfo(t).eps / 2


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def ids_tensor(ids):
    """uint32 ids on the device (as int32 bits)."""
    return torch.tensor(ids, dtype=torch.int64, device=DEV).to(torch.int32)


def words_of(keep):
    """Dense candidate words of a boolean tensor."""
    n = -(-keep.numel() // 64) * 64
    bits = torch.zeros(n, dtype=torch.int64, device=keep.device)
    bits[: keep.numel()] = keep.long()
    return (bits.view(-1, 64) << torch.arange(64, device=keep.device)).sum(1)


# ---- lookup ---------------------------------------------------------------------------------


def bag_of_positions(n, offsets, n_bags):
    """The bag of each position, -1 for none."""
    p = torch.arange(n, device=DEV)
    if offsets is None:
        return torch.where(p < n_bags, p, -1)
    off = offsets.long()
    bag = torch.searchsorted(off, p, right=True) - 1
    return torch.where((p >= off[0]) & (p < off[-1]), bag.clamp(0, n_bags - 1), -1)


def lookup_reference(table, ids, offsets, n_bags, weights, scale, out_type):
    """(out, bound) in 64 bits."""
    n, (rows, d) = ids.numel(), table.shape
    bag = bag_of_positions(n, offsets, n_bags)
    use = ((ids.long() & 0xFFFFFFFF) < rows) & (bag >= 0)
    w = torch.ones(n, dtype=torch.float64, device=DEV) if weights is None else weights.double()
    x = table[ids.long()[use]].double() * w[use][:, None]
    zeros = torch.zeros(n_bags, d, dtype=torch.float64, device=DEV)
    out = zeros.index_add(0, bag[use], x) * scale
    size = zeros.index_add(0, bag[use], x.abs()) * abs(scale)
    count = torch.zeros(n_bags, dtype=torch.float64, device=DEV).index_add(0, bag[use], w[use] * 0 + 1)
    bound = (count[:, None] + 3) * U32 * size
    return out, bound + u(out_type) * (out.abs() + bound) + 1e-38


def call_lookup(ctx, table, ids, offsets, n_bags, weights, scale, out):
    ctx.lookup_device(table.data_ptr(), TYPE[table.dtype], table.shape[0], table.stride(0), table.shape[1], ptr(ids),
                      ids.numel(), ptr(offsets), n_bags, ptr(weights), scale, ptr(out), TYPE[out.dtype], out.stride(0),
                      stream())
    return out


def row_grads_reference(grad_out, ids, offsets, weights, scale, rows, out_type):
    """(dense rows, bound, rows that an id names)."""
    n, (n_bags, d) = ids.numel(), grad_out.shape
    bag = bag_of_positions(n, offsets, n_bags)
    use = ((ids.long() & 0xFFFFFFFF) < rows) & (bag >= 0)
    w = torch.ones(n, dtype=torch.float64, device=DEV) if weights is None else weights.double()
    x = grad_out.double()[bag[use]] * w[use][:, None]
    zeros = torch.zeros(rows, d, dtype=torch.float64, device=DEV)
    at = ids.long()[use]
    out = zeros.index_add(0, at, x) * scale
    size = zeros.index_add(0, at, x.abs()) * abs(scale)
    count = torch.zeros(rows, dtype=torch.float64, device=DEV).index_add(0, at, w[use] * 0 + 1)
    bound = (count[:, None] + 3) * U32 * size
    return out, bound + u(out_type) * (out.abs() + bound) + 1e-38, count > 0


def call_row_grads(ctx, grad_out, ids, offsets, weights, scale, rows, grad_rows, unique=None, count=None, ws=None):
    need = ctx.lookup_grad_workspace_bytes(ids.numel(), rows, grad_out.shape[1])
    ws = torch.empty(need, dtype=torch.uint8, device=DEV) if ws is None else ws
    ctx.lookup_grad_device(ptr(grad_out), TYPE[grad_out.dtype], grad_out.stride(0), grad_out.shape[1], ptr(ids),
                           ids.numel(), ptr(offsets), grad_out.shape[0], ptr(weights), scale, rows, ws.data_ptr(),
                           ws.numel(), ptr(grad_rows), TYPE[grad_rows.dtype], grad_rows.stride(0), ptr(unique),
                           ptr(count), stream())


def weight_grads_reference(table, grad_out, ids, offsets, scale):
    n, rows = ids.numel(), table.shape[0]
    bag = bag_of_positions(n, offsets, grad_out.shape[0])
    use = ((ids.long() & 0xFFFFFFFF) < rows) & (bag >= 0)
    x = torch.where(use[:, None], table.double()[ids.long().clamp(0, rows - 1)], 0.0)
    g = torch.where(use[:, None], grad_out.double()[bag.clamp(min=0)], 0.0)
    out = (x * g).sum(1) * scale
    return out, (table.shape[1] + 3) * U32 * (x * g).abs().sum(1) * abs(scale) + 1e-38


def call_weight_grads(ctx, table, ids, offsets, scale, grad_out, out):
    ctx.lookup_grad_weights_device(ptr(table), TYPE[table.dtype], table.shape[0], table.stride(0), table.shape[1],
                                   ptr(ids), ids.numel(), ptr(offsets), grad_out.shape[0], scale, ptr(grad_out),
                                   TYPE[grad_out.dtype], grad_out.stride(0), ptr(out), stream())
    return out


# ---- cross entropy ----------------------------------------------------------------------------


def xent_reference(queries, table, targets, keep, scale, grad_loss=None, cosine=False):
    """Values and bounds, in 64 bits: dict of (value, bound) for loss, lse, queries, rows (gradients before the rounding
    to their type; `grads_bound` adds it)."""
    q, n_rows = queries.double(), table.shape[0]
    keep = torch.ones(n_rows, dtype=torch.bool, device=DEV) if keep is None else keep
    at = keep.nonzero().flatten()
    r = table[at].double()
    depth = q.shape[1]
    qn = rn = None
    qs, rs = q, r
    if cosine:
        qn, rn = q.norm(dim=1, keepdim=True), r.norm(dim=1, keepdim=True)
        qs = torch.where(qn > 0, q / qn, 0.0)
        rs = torch.where(rn > 0, r / rn, 0.0)
    z = qs @ rs.T * scale
    # products in f32 in any order, times the factor: (depth + 2) roundings, and one for the factor; cosines: two more
    # quotients, and lengths that are off by half as many roundings as a sum of squares has, each
    zb = (depth + 4 + (depth + 8 if cosine else 0)) * U32 * (qs.abs() @ rs.abs().T) * abs(scale)
    zb = zb.amax(1) if at.numel() else torch.zeros(q.shape[0], dtype=torch.float64, device=DEV)
    t = targets.long() & 0xFFFFFFFF
    place = torch.full((n_rows + 1,), -1, dtype=torch.int64, device=DEV)
    place[at] = torch.arange(at.numel(), device=DEV)
    column = place[t.clamp(max=n_rows)]
    ok = column >= 0
    rowi = torch.arange(q.shape[0], device=DEV)
    lse = torch.logsumexp(z, 1) if at.numel() else torch.full((q.shape[0],), -float("inf"), dtype=torch.float64, device=DEV)
    others = z.clone()
    others[rowi[ok], column[ok]] = -float("inf")
    rest = torch.logsumexp(others, 1) if at.numel() else lse
    click = torch.zeros_like(lse)
    click[ok] = z[rowi[ok], column[ok]]
    loss = torch.where(ok, torch.nn.functional.softplus(rest - click, threshold=1e9), 0.0)
    loss = torch.where(torch.isnan(loss), 0.0, loss)
    # an exponential of x is off by 2 roundings and the rounding of x log2 e (|x| of up to the spread of the logits),
    # a sum of n of them by n roundings
    if at.numel():
        spread = z.amax(1) - z.amin(1)
        size = z.abs().amax(1)
    else:
        spread = size = torch.zeros_like(zb)
    e = zb + (4 + 2 * spread + at.numel()) * U32
    p_not = -torch.expm1(-loss)
    out = {
        "lse": (lse, e + 2 * U32 * size + 1e-37),
        "loss": (loss, p_not * (2 * e + 2 * U32 * size) + 2 * U32 * loss + 1e-37),
    }
    c = torch.ones_like(lse) if grad_loss is None else grad_loss.double()
    w = torch.where(ok, c, 0.0) * scale
    p = torch.exp(z - torch.where(torch.isinf(lse), 0.0, lse)[:, None])
    p[rowi[ok], column[ok]] = torch.expm1(-loss[ok])
    g = p * w[:, None]
    # relative error of a weight: that of z and of lse (twice e), a few roundings, and one to the table's type
    g_rel = 2 * e + (8 + spread) * U32 + 4 * U32 * size + (u(torch.bfloat16) if table.dtype == torch.bfloat16 else 0.0)
    # an exponential below the smallest normal f32, 2^-126, may come out as zero: an error of up to 2^-126 in a
    # probability, whatever the probability, and |w| times that in a weight (for w = 1000: 1.2e-35, where the relative
    # bound of a probability of 1e-39 would be 1e-42)
    gb = g.abs() * g_rel[:, None] + w.abs()[:, None] * 2.0**-126
    if cosine:
        gs = g * torch.where(qn > 0, 1 / qn, 0.0)
        d = gs @ rs
        db = (gb * torch.where(qn > 0, 1 / qn, 0.0)) @ rs.abs() + (at.numel() + depth + 4) * U32 * (gs.abs() @ rs.abs())
        along = torch.where(qn > 0, (d * q).sum(1, keepdim=True) / qn.square(), 0.0)
        alongb = torch.where(qn > 0, (db * q.abs()).sum(1, keepdim=True) / qn.square(), 0.0)
        alongb = alongb + torch.where(qn > 0, 4 * depth * U32 * (d * q).abs().sum(1, keepdim=True) / qn.square(), 0.0)
        dq = d - along * q
        dqb = db + alongb * q.abs() + 4 * U32 * (d.abs() + (along * q).abs())
    else:
        dq = g @ r
        dqb = gb @ r.abs() + (at.numel() + 4) * U32 * (g.abs() @ r.abs())
    out["queries"] = (dq, dqb + 1e-37)
    rows = torch.zeros(n_rows, depth, dtype=torch.float64, device=DEV)
    rb = torch.zeros_like(rows)
    rows[at] = g.T @ q
    rb[at] = gb.T @ q.abs() + (q.shape[0] + 4) * U32 * (g.abs().T @ q.abs())
    out["rows"] = (rows, rb + 1e-37)
    return out


def rounded(value_and_bound, t):
    """The bound with one rounding to type t."""
    v, b = value_and_bound
    return v, b + u(t) * (v.abs() + b)


def check(got, value_and_bound, what=""):
    v, b = value_and_bound
    got = got.double()
    same = (got == v) | (torch.isnan(got) & torch.isnan(v))
    off = torch.where(same, 0.0, (got - v).abs())
    bad = ~(off <= b)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside their bounds, worst {float((off / b)[bad].max()):.3g} times, "
        f"first at {bad.nonzero()[0].tolist()}: {float(got[bad][0])} for {float(v[bad][0])} +- {float(b[bad][0])}")


def call_xent(ctx, queries, table, targets, words, scale, ws=None):
    n, d = queries.shape
    need = ctx.xent_workspace_bytes(n, table.shape[0], d, TYPE[table.dtype])
    ws = torch.empty(need, dtype=torch.uint8, device=DEV) if ws is None else ws
    loss, lse = torch.full((2, n), 77.0, device=DEV)
    ctx.xent_device(ptr(queries), n, queries.stride(0), ptr(table), table.shape[0], table.stride(0), TYPE[table.dtype], d,
                    ptr(targets), ptr(words), scale, ws.data_ptr(), ws.numel(), ptr(loss), ptr(lse), stream())
    return loss, lse


def call_xent_grads(ctx, queries, table, targets, words, scale, loss, lse, grad_loss, grad_queries, grad_rows, ws=None):
    n, d = queries.shape
    need = ctx.xent_workspace_bytes(n, table.shape[0], d, TYPE[table.dtype])
    ws = torch.empty(need, dtype=torch.uint8, device=DEV) if ws is None else ws
    ctx.xent_grad_device(ptr(queries), n, queries.stride(0), ptr(table), table.shape[0], table.stride(0),
                         TYPE[table.dtype], d, ptr(targets), ptr(words), scale, ptr(loss), ptr(lse), ptr(grad_loss),
                         ws.data_ptr(), ws.numel(), ptr(grad_queries), ptr(grad_rows), stream())

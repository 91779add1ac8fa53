"""Tight bounds of the cross entropy over a corpus: what its sums, exponentials and weights may be off by, counted from
how the work is cut, so that a lost tile, a repeated one or a plane of bits that is missing lies outside them.

U32 = 2^-24 is one rounding to f32. To first order:
  product   depth + 8 roundings of the sum of its magnitudes (the three smallest of nine products of planes, left out, are
            below 2^-22 of it and among the 8), none where every partial sum is a whole number of some power of two and
            below 2^24 of it (`exact_products`); a cosine's row length takes depth / 2 + 2 more and its quotients 4
  exponent  the factor times log2 e 2 roundings and the product one, of |z|, or none where the factor is such that it is not
            rounded (`exact_factor`: one fma takes the product and its distance from the largest); the distance two more, and
            two where sums over it are brought together, each with the term's share of the sum
  sum       `chain` roundings: as many terms as one workgroup adds up, and 20 for the joins
  lse       all of these, and one rounding of itself
  weight    its own product and exponent, lse's error, 8 roundings; and `kept`, where it is kept to fewer bits
"""
import torch

from learn_helpers import DEV, U32


def chain_of(n_rows, n_q):
    """Candidates that a workgroup takes, at most: 256 workgroups, of which those of the same candidates (tiles of 64 queries
    or more) stand beside each other; and a tile more for what does not divide."""
    return n_rows * -(-n_q // 64) / 256 + 256


def weight_bits(dtype):
    """How far the weights of the gradients may be from their f32 values: f32 tables keep 24 bits, bf16 tables 16."""
    return 0.0 if dtype == torch.float32 else 2.0**-16


def bounds(queries, table, targets, keep, scale, grad_loss=None, cosine=False, exact_products=False, exact_factor=False, chain=None, kept=0.0,
           share=None, joins=256):
    """{loss, lse, queries, rows: (value in 64 bits, bound)}, the gradients before the rounding to their type. share: the
    candidates that one running sum of a query's gradient takes; joins: how many of those are brought together, at most."""
    n_q, depth = queries.shape
    q, n_rows = queries.double(), table.shape[0]
    keep = torch.ones(n_rows, dtype=torch.bool, device=DEV) if keep is None else keep
    at = keep.nonzero().flatten()
    r = table[at].double()
    chain = chain_of(at.numel(), n_q) if chain is None else chain
    share = at.numel() if share is None else share
    qs, rs, terms = q, r, 0 if exact_products else depth + 8
    if cosine:
        qn, rn = q.norm(dim=1, keepdim=True), r.norm(dim=1, keepdim=True)
        qs = torch.where(qn > 0, q / qn, 0.0)
        rs = torch.where(rn > 0, r / rn, 0.0)
        terms += depth / 2 + 6
    z = qs @ rs.T * scale
    zb = terms * U32 * abs(scale) * (qs.abs() @ rs.abs().T) + (0 if exact_factor else 3 * U32) * z.abs()
    column = torch.full((n_rows,), -1, dtype=torch.int64, device=DEV)
    column[at] = torch.arange(at.numel(), device=DEV)
    t = targets.long() & 0xFFFFFFFF
    column = torch.where(t < n_rows, column[t.clamp(max=n_rows - 1)], -1)
    ok, row = column >= 0, torch.arange(n_q, device=DEV)
    lse = torch.logsumexp(z, 1)
    rest = z.clone()
    rest[row[ok], column[ok]] = -float("inf")
    rest = torch.logsumexp(rest, 1)
    click, clickb = torch.zeros_like(lse), torch.zeros_like(lse)
    click[ok], clickb[ok] = z[row[ok], column[ok]], zb[row[ok], column[ok]]
    loss = torch.where(ok, torch.nn.functional.softplus(rest - click, threshold=1e9), 0.0).nan_to_num()
    e = zb.amax(1) + (4 * (torch.softmax(z, 1) * (z.amax(1, keepdim=True) - z)).sum(1) + chain + 20) * U32
    p_not = -torch.expm1(-loss)
    lossb = p_not * (e + clickb) + 2 * U32 * loss + 1e-37
    out = {"lse": (lse, e + U32 * lse.abs() + 1e-37), "loss": (loss, lossb)}
    w = torch.where(ok, torch.ones_like(lse) if grad_loss is None else grad_loss.double(), 0.0) * scale
    g = torch.exp(z - lse[:, None])
    rel = zb + 2 * U32 * (z - lse[:, None]).abs() + (e + U32 * lse.abs() + 8 * U32)[:, None]
    tiny = 2.0**-125 * (1 + w.abs())[:, None]

    def error_of(click_kept):
        b = g * (rel + kept)
        b[row[ok], column[ok]] = (torch.exp(-loss) * lossb + p_not * (4 * U32 + click_kept))[ok]
        return b * w.abs()[:, None] + tiny
    # (what a clicked row's weight is not kept to goes into the queries' gradient by itself)
    gb_queries, gb_rows = error_of(0.0), error_of(kept)
    g[row[ok], column[ok]] = torch.expm1(-loss[ok])
    g = g * w[:, None]
    if cosine:
        over = torch.where(qn > 0, 1 / qn, 0.0)
        d = (g * over) @ rs
        db = (gb_queries * over) @ rs.abs() + (share + joins + depth + 20) * U32 * ((g * over).abs() @ rs.abs())
        along = (d * q).sum(1, keepdim=True) * over.square()
        alongb = ((db * q.abs()).sum(1, keepdim=True) + (depth + 8) * U32 * (d * q).abs().sum(1, keepdim=True)) * over.square()
        out["queries"] = d - along * q, db + alongb * q.abs() + 4 * U32 * (d.abs() + (along * q).abs()) + 1e-37
        return out
    out["queries"] = g @ r, gb_queries @ r.abs() + (share + joins + 8) * U32 * (g.abs() @ r.abs()) + 1e-37
    dr, drb = torch.zeros(2, n_rows, depth, dtype=torch.float64, device=DEV)
    dr[at] = g.T @ q
    drb[at] = gb_rows.T @ q.abs() + (n_q + 8) * U32 * (g.abs().T @ q.abs()) + 1e-37
    out["rows"] = dr, drb
    return out

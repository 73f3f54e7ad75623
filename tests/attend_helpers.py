"""Attention over a window and over shared slots in 64 bits, and what its 16-bit products may be off by."""
import torch

from paged_helpers import DIM, rounding


def visible(own_slot, slots, window, sink):
    """[rows, slots]: which slots a token at `own_slot` sees."""
    j, s = torch.arange(slots), torch.as_tensor(own_slot)[:, None]
    seen = j <= s
    return seen if window is None else seen & ((j > s - window) | (j < sink))


def attend_rows(q, k, v, seen, scale=DIM ** -0.5):
    """q [rows, heads, 128], k and v [kv_heads, slots, 128] in 64 bits, seen [rows, slots] -> out, lse, what out may be off by, what lse may be.

    A probability that is rounded to 16 bits is off by half a step of it, and so is the output: u sum p|v| + u |out|.  A score is a sum of
    128 products that are cut off at 2^-23 of the sum so far, at most 128 2^-23 sum |q k| in all, and moves its probability and the sum of
    them by as much; the exponential adds 2^-22.  fp16 has no steps below 2^-24, of probabilities that go up to 2^10."""
    rows, heads, _ = q.shape
    hk = k.shape[0]
    k, v = k.repeat_interleave(heads // hk, 0), v.repeat_interleave(heads // hk, 0)
    z = torch.einsum("rhd,hsd->rhs", q, k) * scale
    z = z.masked_fill(~seen[:, None], -torch.inf)
    lse = torch.logsumexp(z, -1) if k.shape[1] else torch.full((rows, heads), -torch.inf, dtype=torch.float64)
    p = torch.where(seen[:, None] & torch.isfinite(z), torch.exp(z - torch.where(torch.isfinite(lse), lse, 0.0)[..., None]), torch.zeros_like(z))
    size = torch.einsum("rhd,hsd->rhs", q.abs(), k.abs()).masked_fill(~seen[:, None], 0.0)
    score = (size.amax(-1) if k.shape[1] else torch.zeros(rows, heads, dtype=torch.float64)) * scale * 2.0 ** -16 + 2.0 ** -22
    clean = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
    out, spread = torch.einsum("rhs,hsd->rhd", p, clean), torch.einsum("rhs,hsd->rhd", p, clean.abs())
    return out, lse, spread, score


def close(got, got_lse, want, lse, spread, score):
    """Whether out and log-sum-exp are within what `attend_rows` allows."""
    half, tiny = rounding(got.dtype)
    allowed = half * (spread + want.abs()) * 1.01 + 2 * score[..., None] * spread + tiny + 1e-8
    fine = ((got.cpu().double() - want).abs() <= allowed).all()
    if got_lse is not None:
        x, finite = got_lse.cpu().double(), torch.isfinite(lse)
        fine = fine and torch.equal(x[~finite], lse[~finite])
        fine = fine and ((x - lse).abs()[finite] <= (score + 2.0 ** -22 * lse.abs() + 1e-6)[finite]).all()
    return bool(fine)

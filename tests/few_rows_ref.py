"""What cs1_attention_paged_varlen promises for entries of few columns: the precision of the single-token call, whose bound
(decode_ref.attention) has no rounding of the probabilities to bfloat16 in it."""
import copy

import numpy as np

import decode_ref as R


def row_by_row(t, seqs, cu):
    """A table with a sequence for each row, which holds what the row sees."""
    x = copy.copy(t)
    owner = np.repeat(np.asarray(seqs), np.diff(cu))
    x.nseq, x.table = len(owner), t.table[owner]
    x.lens = np.concatenate([int(t.lens[s]) - (b - a) + 1 + np.arange(b - a) for s, a, b in zip(seqs, cu, cu[1:])]).astype(np.int32)
    return x


def attention(t, seqs, cu, q, kp, vp, gate, hk, scale):
    """Float64 result, log-sum-exp and bounds of all rows.

    Beside decode_ref.attention's: the reciprocal of the sum is off by a step (2 E32) and the gate's sigmoid by two and its
    argument's rounding, |g| E32; the two products add E32 each.  And the rounding is off by half a step of the value's own
    binade, which is E16 of the value at its lower end only."""
    x = row_by_row(t, seqs, cu)
    out, lse, tol, ltol = R.attention(x, np.arange(x.nseq), q, kp, vp, gate, hk, scale)
    g = 0.0 if gate is None else np.abs(R.f64(gate))
    err = (tol - R.E16 * np.abs(out)) / (1 + R.E16) + (8 + g) * R.E32 * np.abs(out)  # before the rounding
    size = np.maximum(np.abs(out) + err, 2.0 ** -126)
    return out, lse, err + 2.0 ** (np.floor(np.log2(size)) - 8), ltol

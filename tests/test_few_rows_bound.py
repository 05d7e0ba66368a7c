"""The bound that pins the precision of entries of few columns tells probabilities with all their bits from such that were
rounded to bfloat16: the same inputs as the GPU tests', the kernel's arithmetic in numpy."""
import numpy as np
import pytest

import decode_ref as R
import few_rows_ref as F


def emulated(x, q, kp, vp, hk, scale, parts):
    """Scores and sums in float32, the exponentials' first `parts` bfloat16 parts to the second product."""
    B, hq, dh = q.shape
    out = np.zeros((B, hq, dh))
    for r in range(B):
        j = np.arange(int(x.lens[r]))
        at = x.table[r, j // x.page], j % x.page
        for h in range(hq):
            k, v = (R.f64(np.ascontiguousarray(p[at][:, h // (hq // hk)])).astype(np.float32) for p in (kp, vp))
            s = (k @ R.f64(q[r, h]).astype(np.float32)) * np.float32(scale)
            p = np.exp(s - s.max())
            rest, kept = p.copy(), np.zeros(len(p), np.float64)
            for _ in range(parts):
                part = R.f64(R.O.f32_to_bf16(rest))
                kept += part
                rest = (rest - part).astype(np.float32)
            out[r, h] = (kept.astype(np.float32) @ v) / p.sum()
    return R.f64(R.O.f32_to_bf16(out.astype(np.float32).reshape(-1))).reshape(out.shape)


@pytest.mark.parametrize("held,new", [(20, 4), (300, 3)])
def test_bound_tells_them_apart(held, new):
    rng = np.random.default_rng(held)
    t = R.scattered(rng, 1, [held], 16)
    cu = np.array([0, new])
    q, kp, vp = R.bf16(rng, new, 8, 128), R.bf16(rng, t.npages, 16, 2, 128), R.bf16(rng, t.npages, 16, 2, 128)
    scale = 128 ** -0.5
    want, _, tol, _ = F.attention(t, [0], cu, q, kp, vp, None, 2, scale)
    x = F.row_by_row(t, [0], cu)
    off = lambda parts: np.abs(emulated(x, q, kp, vp, 2, scale, parts) - want) > tol  # noqa: E731
    assert not off(3).any()
    print(f"one part: {off(1).mean():.4f} of the outputs are outside")
    assert off(1).any()

"""Entries of few columns (rows times q heads of a kv head, up to 16) have the precision of the single-token call: within a
bound that has no rounding of the probabilities, alone, beside long entries, cut and whole."""
import numpy as np
import pytest

import decode_ref as R
import few_rows_ref as F
from gpu_helpers import say
from test_gpu_attention_chunk import Call, handle  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk,dh,most", [(16, 4, 128, 4), (16, 4, 256, 4), (24, 4, 256, 2), (4, 4, 128, 16), (16, 1, 256, 1), (10, 2, 256, 3)])
@pytest.mark.parametrize("lens", [[1, 4, 17, 20, 33, 64, 130], [300, 5, 900], [9000]], ids=str)
@pytest.mark.parametrize("company", [False, True])
def test_precision(handle, hq, hk, dh, most, lens, company):  # noqa: F811
    say(f"few rows, precision: {lens}, up to {most} rows, heads {hq}/{hk} Dh={dh}, beside a long entry: {company}")
    rng = np.random.default_rng(sum(lens) + hq + dh + company)
    t = R.scattered(rng, len(lens) + 1, lens + [200], 48)
    new = [min(n, most - i % 2 if most > 1 else 1) for i, n in enumerate(lens)]
    few = int(sum(new))
    seqs = list(range(len(lens)))
    c = Call(handle, rng, t, seqs + [len(lens)] * company, new + [100] * company, hq, hk, dh, gate=bool(len(lens) % 2))
    c.upload()
    c.launch()
    out, lse = c.results()
    gate = None if c.gate is None else c.gate[:few]
    want, wl, tol, ltol = F.attention(t, seqs, c.cu[:len(lens) + 1], c.q[:few], c.kp, c.vp, gate, hk, c.scale)
    R.close(R.f64(out[:few]), want, tol, "out")
    R.close(lse[:, :few].astype(np.float64), wl, ltol, "lse")

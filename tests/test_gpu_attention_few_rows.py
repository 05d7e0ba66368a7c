"""cs1_attention_paged_varlen for entries of few columns (rows times q heads of a kv head), alone and beside longer ones."""
import numpy as np
import pytest

import decode_ref as R
from gpu_helpers import say
from test_gpu_attention_chunk import Call, handle, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk,dh,most", [(16, 4, 128, 4), (16, 4, 256, 4), (24, 4, 256, 2), (4, 4, 128, 16), (6, 2, 128, 5), (16, 1, 256, 1),
                                           (10, 2, 256, 3), (7, 1, 128, 2), (1, 1, 256, 16)])
def test_head_layouts(handle, hq, hk, dh, most):  # noqa: F811
    """Rows up to the most that a tile holds and one more, of sequences that end around units of keys."""
    say(f"few rows: heads {hq}/{hk} Dh={dh}")
    rng = np.random.default_rng(hq + dh)
    lens = [1, 0, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 130, 257, 900]
    t = R.scattered(rng, len(lens) + 2, lens, 48)
    for top in (most, most + 1):
        new = [min(n, int(k)) for n, k in zip(lens, rng.integers(1, top + 1, len(lens)))]
        new[-1] = top
        order = rng.permutation(len(lens))
        run(Call(handle, rng, t, order, np.array(new)[order], hq, hk, dh, gate=most != 4, pad=2))


@pytest.mark.parametrize("lens,new", [([20000], [4]), ([30000, 1, 700], [4, 1, 3]), ([4000] * 43, [1 + i % 4 for i in range(43)]),
                                      ([200] * 300, [1 + i % 3 for i in range(300)]), ([9000, 300, 9000, 2], [4, 100, 3, 1]),
                                      ([500] * 70, [4 if i % 9 else 65 for i in range(70)]), ([600] * 3, [0, 0, 0])],
                         ids=lambda l: f"{len(l)}x{max(l)}")
@pytest.mark.parametrize("dh", [128, 256])
def test_lengths(handle, lens, new, dh):  # noqa: F811
    say(f"few rows: {len(lens)} sequences up to {max(lens)}, {sum(new)} rows, Dh={dh}")
    rng = np.random.default_rng(sum(lens) + dh)
    t = R.scattered(rng, len(lens), lens, 64)
    run(Call(handle, rng, t, np.arange(len(lens)), new, 8, 2, dh, max_new=4 if max(new) <= 4 else None, pad=1))


def test_padding_repeats_and_rows_before_position_0(handle):  # noqa: F811
    say("few rows: padding entries, a sequence twice, rows before position 0, rows behind max_new")
    rng = np.random.default_rng(3)
    t = R.scattered(rng, 5, [70, 0, 33, 500, 2], 16)
    for dh in (128, 256):
        c = Call(handle, rng, t, [3, -1, 0, 5, 0, 2 ** 31 - 1, 1, 4, 3], [3, 2, 4, 4, 4, 1, 3, 4, 4], 8, 2, dh, pad=5, max_new=4)
        out, l = run(c)
        for i in (1, 3, 5, 6):
            rows = slice(c.cu[i], c.cu[i + 1])
            assert (out[rows] == 0).all() and (l[:, rows] == -np.inf).all()
        assert (out[c.cu[7]:c.cu[7] + 2] == 0).all()  # sequence 4 has 2 tokens and 4 rows
        run(Call(handle, rng, t, [3, 0, 4], [9, 2, 2], 8, 2, dh, max_new=3))


@pytest.mark.parametrize("dh", [128, 256])
@pytest.mark.parametrize("kind", ["nan", "inf"])
@pytest.mark.parametrize("held", [66, 65, 200, 4])
def test_later_rows_are_not_seen(handle, dh, kind, held):  # noqa: F811
    """NaN and infinities in new tokens' keys and values: rows before them keep their bits."""
    say(f"few rows: {kind} in later rows, {held} keys, Dh={dh}")
    rng = np.random.default_rng(held)
    t = R.scattered(rng, 2, [held, 300], 16)
    c = Call(handle, rng, t, [0, 1], [4, 2], 8, 2, dh, gate=False, max_new=4)
    c.upload()
    c.launch()
    clean, cl = c.results()
    at = lambda s, p: (t.table[s, p // 16], p % 16)  # noqa: E731
    spots = [(0, held - 3, 0, 3), (0, held - 2, 1, 100), (0, held - 1, 1, dh - 1), (1, 299, 0, 0)]
    for s, p, h, d in spots:
        c.vp[at(s, p)][h, d] = {"nan": 0x7fc0, "inf": 0xff80 if d == 100 else 0x7f80}[kind]
    c.upload()
    c.launch()
    out, l = c.results()
    hit = np.zeros(out.shape, bool)
    for s, p, h, d in spots:
        hit[c.cu[s] + p - (int(t.lens[s]) - (c.cu[s + 1] - c.cu[s])):c.cu[s + 1], 4 * h:4 * h + 4, d] = True
    np.testing.assert_array_equal(out[~hit], clean[~hit])
    np.testing.assert_array_equal(l, cl)
    x = R.f64(out)
    assert np.isnan(x[hit]).all() if kind == "nan" else np.isinf(x[hit]).all()
    if kind == "inf":
        assert (x[2:4, 4:, 100] == -np.inf).all()
    c.kp[at(0, held - 1)][1, 5] = 0x7fc0
    c.upload()
    c.launch()
    again = c.results()[0]
    assert np.isnan(R.f64(again[3, 4:])).all()
    np.testing.assert_array_equal(again[:3], out[:3])

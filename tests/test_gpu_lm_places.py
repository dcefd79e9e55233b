"""Places asked for again and again: as many draws of one row as a step has room for."""
import numpy as np
import pytest

import drafts_oracle
import lm_util
from test_gpu_lm_serving import load, prompt  # noqa: F401 (load is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["plain", "mixed", "latent"])
@pytest.mark.parametrize("tokens,places", [(1, 64), (1, 65), (3, 70), (20, 200), (5, 300)])
def test_draws_of_one_row(pkg, synth, tmp_path, load, name, tokens, places):  # noqa: F811
    cfg, w, folder = lm_util.build(synth, tmp_path, name)
    m = load(folder)
    rng = np.random.default_rng(places)
    t, a = prompt(cfg, 30), m.open()
    m.step([(a, t, [])])
    other = m.open()
    m.step([(other, t[:9], [])])
    line = rng.integers(0, cfg["vocab"], tokens)
    b = m.fork(a)
    logits = m.step([(b, line, None)])[0]
    d = m.fork(other)
    single = m.step([(d, [5], None)])[0]
    for turn in range(3):                               # (a shape's second step is captured, its third replayed)
        at = np.sort(rng.integers(0, tokens, places))
        key = rng.integers(0, 2 ** 64, places + 1, dtype=np.uint64)
        c, e = m.fork(a), m.fork(other)
        got = m.sampled([(c, line, at), (e, [5], [0])], 1.0, key)
        rows = np.concatenate([logits[at], single])
        unsure = 0
        for i in range(places + 1):
            want = drafts_oracle.verify(rows[i][None], [], None, 1.0, int(key[i]))
            # rows beside other rows may go through other kernels, whose logits differ by rounding: a draw between nearly equal tokens may then be another
            z = rows[i].astype(np.float64) - np.log(drafts_oracle.waits(int(key[i]), cfg["vocab"]))
            unsure += got[i] != want[1]
            assert z.max() - z[got[i]] <= 6 * lm_util.TOL[6] * rows[i].std(), (turn, i)
        assert unsure <= 1 + 0.1 * places
        m.end(c)
        m.end(e)


def test_no_more_than_there_is_room_for(pkg, synth, tmp_path, load):  # noqa: F811
    cfg, w, folder = lm_util.build(synth, tmp_path, "plain")
    m = load(folder, max_step_rows=80)
    s = m.open()
    key = np.arange(81, dtype=np.uint64)
    with pytest.raises(pkg.CmlB200Error):
        m.sampled([(s, [1, 2], [0] * 81)], 1.0, key)
    assert pkg.lib.cml_lm_sequence_length(m.h, s) == 0
    assert len(m.sampled([(s, [1, 2], [0] * 80)], 1.0, key[:80])) == 80

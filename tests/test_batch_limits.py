"""The longest texts that a batch plan takes: host checks, no device."""
import numpy as np
import pytest

import gguf_runner_b200 as g

OK, RANGE = 0, 4


@pytest.mark.parametrize("want,kv_len", [(OK, [2 ** 31 - 1025]), (RANGE, [2 ** 31 - 1024]), (RANGE, [2 ** 31 - 1]), (RANGE, [2 ** 30, 2 ** 30 - 1024]),
                                         (OK, [2 ** 30, 2 ** 30 - 1025])])
def test_key_tiles_stay_within_32_bits(want, kv_len):
    """A page that is only read may stand for many stretches of a text; the tile behind its last key has to be a position, too."""
    table = np.zeros((len(kv_len), 2 ** 23), np.int32)
    assert g.batch_check([0] * len(kv_len), kv_len, table, page_size=256, n_pages=1) == want

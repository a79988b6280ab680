"""ud_logits_process's ranges as include/ud_layer.h states them, in any order: row i's history is tokens[a .. c), cut to the array; its
tokens in front of place b are the prompt, the others were generated."""
import itertools

import numpy as np
import pytest

import layer_ref as ref
from test_gpu_logits import compare, process

pytestmark = pytest.mark.gpu


def counted(tokens, a, b, c, V):
    """For each token whether it is in the history, and how often it was generated: place by place."""
    seen, fresh = np.zeros(V, bool), np.zeros(V)
    for place, t in enumerate(tokens):
        if a <= place < c and 0 <= t < V:
            seen[t] = True
            fresh[t] += place >= b
    return seen, fresh


@pytest.mark.parametrize("length,V", [(9, 40), (66000, 2100)])
def test_ranges_in_any_order(gpu, length, V):
    """Every order of three places, and places outside the array; short histories and ones too long for one word a token."""
    rng = np.random.default_rng(length)
    tokens = rng.integers(-1, V + 1, length).astype(np.int32)
    places = [-3, 0, 5, length // 2, length, length + 7] if length < 100 else [-3, 0, length // 3, length + 7]
    ranges = np.array(list(itertools.product(places, repeat=3)) + [(0, 5, 3), (3, 1, 7), (-2 ** 31, 4, 2 ** 31 - 1), (2, -2 ** 31, 8), (2, 2 ** 31 - 1, 8)], np.int32)
    n = len(ranges)
    x = rng.standard_normal((n, V)).astype(np.float32).astype(np.float64)
    pen = np.tile(np.array([[1.25, 0.5, 0.25]], np.float32), (n, 1))
    out, token = process(gpu, x, "f32", tokens, ranges, pen)
    want, mag = x.copy(), np.abs(x)
    for i, (a, b, c) in enumerate(ranges.tolist()):
        seen, fresh = counted(tokens, a, b, c, V)
        y = np.where(seen, np.where(x[i] > 0, x[i] / 1.25, x[i] * 1.25), x[i])
        want[i] = y - 0.25 * fresh - 0.5 * (fresh > 0)
        mag[i] = np.abs(y) + 0.25 * fresh + 0.5
    compare(out, want, mag)
    np.testing.assert_array_equal(token, ref.chosen(out))

"""GPU parity of ud_logits_process over lists too long for one word a token (more than 65,535 tokens of history, or 32,767 biases), in each
size of segment: a thread then holds up to eight pieces of its row between the two passes."""
import numpy as np
import pytest

import layer_ref as ref
from test_gpu_logits import compare, process

pytestmark = pytest.mark.gpu

# rows, vocabulary, tokens of a segment (held against the launch's own choice on the CPU)
SIZES = [(2, 9001, 2048), (130, 8000, 4096), (40, 60000, 8192), (70, 60001, 16384), (130, 32769, 32768), (257, 30000, 32768)]


@pytest.mark.parametrize("history,biases", [(70000, 20), (300, 33000), (66000, 40000)])
@pytest.mark.parametrize("n,V,segment", SIZES)
def test_long_lists(gpu, n, V, segment, history, biases):
    """Rows share one history and one list of biases; every third row sees all of them, the others less than would be long."""
    rng = np.random.default_rng([n, V, history])
    dtype = ["f32", "bf16", "f16"][n % 3]
    x = ref.stored(3 * rng.standard_normal((n, V)), dtype)[1]
    tokens = np.minimum(V - 1, (V * rng.random(history) ** 2)).astype(np.int32)
    tokens[rng.integers(0, history, history // 50)] = -1
    whole = np.arange(n) % 3 == 0
    lo = np.where(whole, 0, rng.integers(0, history // 2, n))
    hi = np.where(whole, history, lo + rng.integers(0, 200, n))
    ranges = np.stack([lo, lo + (hi - lo) // 3, hi], 1).astype(np.int32)
    pen = (np.array([1, 0, 0]) + rng.random((n, 3)) * [0.5, 1, 0.5]).astype(np.float32)
    ids = rng.integers(0, V, biases).astype(np.int32)
    values = (2 * rng.standard_normal(biases)).astype(np.float32)
    blo = np.where(whole, 0, rng.integers(0, biases // 2, n))
    br = np.stack([blo, np.where(whole, biases, blo + rng.integers(0, 9, n))], 1).astype(np.int32)
    mask = rng.random((3, V)) < 0.5
    mask_rows = (np.arange(n) % 4 - 1).astype(np.int32)
    out, token = process(gpu, x, dtype, tokens, ranges, pen, (ids, values, br), mask, mask_rows)
    want, mag = ref.logits_out(x, tokens, ranges, pen, [(ids[a:b], values[a:b]) for a, b in br], [mask[m] if m >= 0 else None for m in mask_rows])
    compare(out, want, mag)
    np.testing.assert_array_equal(token, ref.chosen(out))

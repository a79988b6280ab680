"""GPU parity of ud_logits_process under repetition penalties whose reciprocals are infinite, subnormal or short of bits: the quotient of
the definition, l / repetition, in every case."""
import numpy as np
import pytest

import layer_ref as ref
from test_gpu_logits import process

pytestmark = pytest.mark.gpu

f32 = np.float32
REPS = np.array([1e-45, 2.0 ** -149 * 12345, 1e-39, 2.0 ** -128, 2.0 ** -127 * 1.7, 2.0 ** -126, 2.0 ** -101, 0.9 * 2.0 ** -100, 3.4e38, 2.0 ** 127, 2.0 ** 126 * 1.3, 1.1 * 2.0 ** 100], f32)


@pytest.mark.parametrize("n,V", [(12, 300), (260, 20000)])
@pytest.mark.parametrize("rest", [False, True])
def test_far_repetitions(gpu, n, V, rest):
    """All tokens in the prompt, one row a repetition; rest: biases and penalties for generated tokens behind it."""
    rng = np.random.default_rng([n, V])
    rep = np.resize(REPS, n)
    # logits whose quotients lie within fp32's range, at its upper end and past it; negative ones are products
    x = rng.standard_normal((n, V)) * np.clip(rep[:, None].astype(np.float64) * np.exp2(rng.integers(-10, 140, (n, V)).astype(np.float64)), 0, 1e38)
    x[:, ::3] = -np.abs(x[:, ::3])
    x[:, 1:4] = [np.inf, -np.inf, 0]
    x = x.astype(f32).astype(np.float64)
    tokens = np.arange(V, dtype=np.int32)
    ranges = np.tile(np.array([[0, V - 50 if rest else V, V]], np.int32), (n, 1))
    pen = np.stack([rep, np.full(n, 0.5 if rest else 9), np.full(n, 0.25 if rest else 9)], 1).astype(f32)
    b = (np.array([5, V - 5], np.int32), np.array([1, 2], f32), np.tile(np.array([[0, 2]], np.int32), (n, 1))) if rest else None
    out, token = process(gpu, x, "f32", tokens, ranges, pen, b)
    with np.errstate(over="ignore"):
        want = np.where(x > 0, x / rep[:, None].astype(np.float64), x * rep[:, None].astype(np.float64)).astype(f32)
        if rest:
            want[:, V - 50:] -= f32(0.75)
            want[:, [5, V - 5]] += np.array([1, 2], f32)
    np.testing.assert_array_equal(out, want.astype(np.float64))
    np.testing.assert_array_equal(token, ref.chosen(want.astype(np.float64)))


def test_ordinary_and_far_rows_beside_each_other(gpu):
    """A far row changes no other row's bits."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, 5000)).astype(f32).astype(np.float64)
    tokens = rng.integers(0, 5000, 400).astype(np.int32)
    ranges = np.array([[0, 100, 200], [200, 300, 400]] * 2, np.int32)
    pen = np.array([[1.3, 0.5, 0.1], [0.8, 0.1, 0.2], [1e-40, 0.5, 0.1], [3e38, 0.1, 0.2]], f32)
    out, _ = process(gpu, x, "f32", tokens, ranges, pen)
    alone, _ = process(gpu, x[:2], "f32", tokens, ranges[:2], pen[:2])
    np.testing.assert_array_equal(out[:2], alone)

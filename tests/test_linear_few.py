"""CPU check: the int8 product's kernels for a few rows, whose workgroups all take the first 16 rows, are chosen for no more."""
import numpy as np

from test_linear_plan import NAMES, kernel  # noqa: F401


def test_few_rows_are_at_most_sixteen(kernel):  # noqa: F811
    rng = np.random.default_rng(2)
    sizes = [(M, N, K) for M in (1, 4, 5, 16, 17, 64) for N in (1, 16, 4096, 4097, 8192, 1 << 24) for K in (16, 2048, 2064, 8192, 131056)]
    sizes += [tuple(int(x) for x in np.exp(rng.uniform(0, [8, 16.6, 11.7]))) for _ in range(20000)]
    few = {M for M, N, K in sizes if NAMES[kernel(M, N, max(16, K // 16 * 16))].startswith("few")}
    assert few and max(few) <= 16

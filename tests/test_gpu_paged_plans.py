"""GPU parity of the windowed and prompt attention over the paged cache where their plans (csrc/paged_plan.hpp) take the paths that
small cases do not reach: MXFP4 batches taken by length with several layers of workgroups, row tiles among them; one sequence in
more than 64 splits; prompts over pages that are missing inside the range.  tests/test_paged_plans.py checks on the CPU that these
sizes get these plans."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged_window import P_STEP, PROMPT_STEP, PROMPTS, Cache, causal, check_window, close, prefill, window

pytestmark = pytest.mark.gpu

# page format, queries' type, sequences, kv heads, query heads of one, positions; the layer that the plan gives
BY_LENGTH = [("mxfp4", "bf16", 64, 6, 1, 1, 42), ("mxfp4", "bf16", 64, 8, 2, 1, 32), ("mxfp4", "f32", 50, 8, 5, 4, 32),
             ("mxfp4", "f16", 64, 6, 8, 5, 21), ("mxfp4", "f32", 48, 8, 16, 4, 16), ("bf16", "bf16", 64, 6, 7, 3, 64),
             ("f16", "f32", 64, 6, 8, 5, 64)]
# page format, queries' type, head size, query heads of the one kv head, keys; the splits that the plan gives
LONG = [("bf16", "f32", 128, 20, 32_768, 256), ("f16", "f32", 64, 1, 65_500, 256), ("mxfp4", "f32", 128, 4, 48_000, 188),
        ("mxfp4", "bf16", 64, 20, 65_530, 256), ("f16", "f16", 128, 17, 17_000, 133), ("mxfp4", "f16", 64, 33, 19_000, 75)]
SPAN = 2_100                                        # the batches' longest sequence


@pytest.mark.parametrize("fmt,dtype,n,hkv,group,M,layer", BY_LENGTH)
def test_batches_taken_by_length(gpu, fmt, dtype, n, hkv, group, M, layer):
    """More sequences than a layer: every one of them is taken once, long and short, equal ones and ones that see nothing."""
    rng = np.random.default_rng([81, n, hkv, group, M, len(fmt), len(dtype)])
    lens = [int(x) for x in rng.choice([5, 40, 64, 64, 130, 301], n)]
    for i, L in ((n - 1, SPAN), (0, 1_400), (n // 2, 900)):
        lens[i] = L
    empty = [(i, m) for i in range(3, n, 9) for m in range(M)]
    check_window(gpu, rng, fmt, dtype, group * hkv, hkv, 64, lens, M, 0, 0, empty=empty, span=SPAN)


@pytest.mark.parametrize("fmt,dtype,d,hq,keys,splits", LONG)
def test_more_splits_than_a_wave_has_lanes(gpu, fmt, dtype, d, hq, keys, splits):
    """One sequence in up to 256 splits.  Its scores are steep, so that a handful of keys make a row's output and the weight of
    each of their splits shows."""
    ud, rng = gpu, np.random.default_rng([82, d, hq, keys])
    c = Cache(ud, rng, fmt, [keys], 1, d)
    q = ref.rounded(rng.standard_normal((1, 1, hq, d)) * 3, dtype)
    ranges = np.array([[[0, keys]]])
    got = window(ud, c, q, ranges, 0, dtype)
    want = ref.attention(q[0], c.k, c.v, np.zeros(1, int), ranges[0], 0, 1, c.most * 16)
    close(got, want, c, d, dtype, P_STEP[fmt, dtype])


@pytest.mark.parametrize("fmt,dtype", PROMPTS)
@pytest.mark.parametrize("span", [None, 20_000])
def test_prompts_over_pages_that_are_not_held(gpu, fmt, dtype, span):
    """Block-table entries outside the pool inside a prompt's range, among them a window's first and last page, four in a row (a
    tile) and one of the sinks: their keys are not there.  span: keys split over workgroups."""
    ud, rng, hq, hkv, d, win, sinks = gpu, np.random.default_rng([83, len(fmt), len(dtype)]), 4, 2, 64, 300, 40
    new, past = [90, 40, 16], [400, 30, 0]
    gone = {(0, 1), (0, 6), (0, 15), (0, 20), (0, 21), (0, 22), (0, 23), (0, 30), (1, 2), (2, 0)}
    c = Cache(ud, rng, fmt, [a + b for a, b in zip(new, past)], hkv, d, keep=lambda i, b: (i, b) not in gone)
    ranges = causal(new, past, win)
    start = np.concatenate([[0], np.cumsum(new)])
    q = ref.rounded(rng.standard_normal((start[-1], hq, d)), dtype)
    assert (span is not None) == (ud.gqa_prefill_workspace_bytes(3, 146, 90, hq, hkv, d, sinks, span or 389) > 0)
    got = prefill(ud, c, q, start, ranges, sinks, dtype, span=span)
    want = ref.attention(q, c.k, c.v, np.repeat(np.arange(3), new), ranges, sinks, hkv, c.most * 16, held_keys=c.held_keys)
    assert np.any(want[4] == 0)                         # the third sequence's only page is one of them
    close(got, want, c, d, dtype, PROMPT_STEP[dtype])

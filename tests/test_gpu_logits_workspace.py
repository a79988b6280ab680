"""A workspace of ud_logits_process, made once for the largest batch, serves the smaller ones that a serving loop comes to."""
import numpy as np
import pytest

import layer_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("most,V", [(64, 131072), (300, 9000)])
def test_workspace_of_the_largest_batch(gpu, most, V):
    ud, rng = gpu, np.random.default_rng(V)
    x = rng.standard_normal((most, V)).astype(np.float32)
    logits, out, token = ud.DeviceBuffer.from_numpy(x), ud.DeviceBuffer(x.nbytes), ud.DeviceBuffer(4 * most)
    need = ud.logits_workspace_bytes(most, V)
    guarded = ud.DeviceBuffer.from_numpy(np.full(need // 8 + 64, 0x5A5A5A5A5A5A5A5A, np.uint64))

    class Ws:
        ptr, nbytes = guarded.ptr, need

    for n in (most, most - 1, most // 2, most // 2 - 1, 7, 2, 1):
        for v in (V, V - 1, V // 2, 1000):
            ud.logits_process(logits, out, n, v, token=token, workspace=Ws, ld=V, out_ld=V)
            ud.synchronize()
            np.testing.assert_array_equal(token.download(n, np.int32), ref.chosen(x[:n, :v].astype(np.float64)), err_msg="%d x %d" % (n, v))
    assert np.all(guarded.download(need // 8 + 64, np.uint64)[need // 8:] == 0x5A5A5A5A5A5A5A5A)

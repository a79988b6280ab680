"""CPU checks that ud_qk_norm_rope_append refuses outputs that share memory with its inputs: a row's heads would be read after others
had been written over them.  (No call here reaches the device; that separate and interleaved rows are taken is in
tests/test_gpu_paged_edges.py.)"""
import pytest

F32, BF16 = 0, 1
BASE, ROWS, HQ, HKV, D = 1 << 30, 5, 8, 2, 64
QW, KW, LD = HQ * D, HKV * D, (HQ + 2 * HKV) * D


def _call(ud, q, k, v, out, q_ld=LD, k_ld=LD, v_ld=LD, out_ld=LD, rows=ROWS, dtype=BF16):
    """Offsets in elements from one address."""
    size = 4 if dtype == F32 else 2
    at = lambda x: BASE + x * size  # noqa: E731
    lib = ud.load_library()
    rc = lib.ud_qk_norm_rope_append(dtype, BF16, at(q), q_ld, at(k), k_ld, at(v), v_ld, at(out), out_ld, None, None, 1e-6, None, 0x10000,
                                    None, 0x10000, 0x10000, 10, 0x10000, 8, 9, rows, HQ, HKV, D, 16, None)
    return rc, lib.ud_last_error().decode()


FAR = 1 << 22


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", [
    dict(q=0, k=QW, v=QW + KW, out=0, out_ld=QW),                   # q's place, its rows closer together (the default distance)
    dict(q=0, k=FAR, v=2 * FAR, out=0, q_ld=QW, out_ld=LD),
    dict(q=0, k=QW, v=QW + KW, out=4),                              # moved by four elements
    dict(q=4, k=FAR, v=2 * FAR, out=0),
    dict(q=0, k=QW, v=QW + KW, out=LD),                             # a row on
    dict(q=0, k=QW, v=QW + KW, out=(ROWS - 1) * LD),
    dict(q=(ROWS - 1) * LD, k=FAR, v=2 * FAR, out=0),
    dict(q=FAR, k=QW, v=QW + KW, out=0, out_ld=QW),                 # over k and v
    dict(q=FAR, k=0, v=2 * FAR, out=0),
    dict(q=FAR, k=2 * FAR, v=0, out=0),
    dict(q=FAR, k=2 * FAR, v=KW - 4, out=0, rows=1),
    dict(q=FAR, k=QW - 4, v=2 * FAR, out=0),
    dict(q=FAR, k=2 * FAR, v=0, out=KW - 4, rows=1),
    dict(q=FAR, k=2 * FAR, v=LD - 4 + 3 * LD, out=4 * LD),
])
def test_overlapping_outputs_are_refused(ud, case, dtype):
    rc, msg = _call(ud, dtype=dtype, **case)
    assert rc == -1 and msg.startswith("ud_qk_norm_rope_append: q_out overlaps"), (rc, msg)

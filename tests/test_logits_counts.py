"""logits_process takes no list without its count, which would be none of it (CPU: the call is refused before it is made)."""
import pytest


class Buf:
    ptr, nbytes = 1 << 20, 1 << 20


@pytest.mark.parametrize("kw,missing", [
    (dict(tokens=Buf, ranges=Buf, penalties=Buf), "n_tokens"), (dict(bias_ids=Buf, bias_values=Buf, bias_ranges=Buf), "n_biases"),
    (dict(mask=Buf, mask_rows=Buf), "n_masks"), (dict(mask=Buf), "n_masks"),
    (dict(tokens=Buf, n_tokens=4, ranges=Buf, mask=Buf, mask_rows=Buf), "n_masks"),
])
def test_counts_are_asked_for(ud, kw, missing):
    with pytest.raises(ud.EngineError, match=missing):
        ud.logits_process(Buf, Buf, 2, 100, **kw)


def test_counts_of_none(ud, monkeypatch):
    """An explicit 0 is none; without the arrays nothing is asked for."""
    seen = []

    class Lib:
        @staticmethod
        def ud_logits_process(*a):
            seen.append((a[9], a[14], a[18]))
            return 0

    monkeypatch.setattr(ud, "lib", lambda: Lib)
    ud.logits_process(Buf, Buf, 2, 100, tokens=Buf, n_tokens=0, ranges=Buf, bias_ids=Buf, n_biases=0, mask=Buf, n_masks=0, mask_rows=Buf)
    ud.logits_process(Buf, Buf, 2, 100)
    ud.logits_process(Buf, Buf, 2, 100, tokens=Buf, n_tokens=5, ranges=Buf, bias_ids=Buf, n_biases=6, mask=Buf, n_masks=7)
    assert seen == [(0, 0, 0), (0, 0, 0), (5, 6, 7)]

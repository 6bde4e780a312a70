"""Calls whose launch would have 2^32 threads are refused before it."""

import pytest

from aspire_amd import _lib
from aspire_amd.logits_processor import _ADJUST

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libaspire_hip.so not built")


@pytest.mark.parametrize("vocab,requests,history", [(256 * 8192, 32768, 0), (256 * 8192, 32768, 8), (512 * 4096, 65535, 0)])
def test_logits_of_2_to_the_23_workgroups(vocab, requests, history):
    at = 4096 if history else 0
    args = dict(logits=4096, st=vocab, out=4096, ost=vocab, qo=0, hist=at, hst=8, lens=at, told=0, rep=at, pres=0, freq=0, tt=0, tm=0, mst=0, bi=0, bv=0, bp=0,
                g=0, gst=0, gr=0, start=0, tokens=requests, vocab=vocab, requests=requests, dtype=0, hl=history, words=0, gn=0, be=0)
    assert _lib.lib().aspire_adjust_logits(_ADJUST.pack(*args.values()), None) == _lib.ASPIRE_ERR_INVALID
    assert "too large" in _lib.lib().aspire_last_error().decode()

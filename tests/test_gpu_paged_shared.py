"""Attention over 8-bit pages that several sequences have: their values are loaded another way than those of one."""
import numpy as np
import pytest

from tests.paged_ext_ref import SetupExt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
@pytest.mark.parametrize("heads,kv,hd,new,window", [(40, 8, 128, 1, 0), (8, 2, 256, 1, 0), (8, 2, 512, 1, 0), (8, 2, 64, 1, 0),
                                                    (8, 1, 128, 3, 0), (8, 2, 256, 5, 0), (8, 2, 128, 1, 90), (4, 1, 128, 40, 0)])
def test_shared_prefix(gpu, heads, kv, hd, new, window, dtype):
    """Sequences whose first 0, 16, 96 and 400 positions are the same pages: each as if it were alone, bit for bit, and
    within the bounds."""
    print(f"\n[case] shared prefix {dtype} hd={hd} new={new} window={window}", flush=True)
    seqs = [(new, 400 + new + 7 * s) for s in range(7)]
    st = SetupExt(gpu, seqs, heads, kv, hd, dtype, 16, window=window, seed=hd + new)
    q = (np.random.default_rng(3).standard_normal((st.rows, heads * hd)) * 1.5).astype(np.float32)
    own = st.pages.copy()
    for n in (0, 1, 6, 25):
        st.pages[1:, :n] = own[0, :n]
        st.batch.set(st.new, st.len, st.pages)
        want, tol = st.attend(q)
        got = st.run_attention(q)
        assert np.all(np.abs(got - want) <= tol)
        # the same values in pages of each sequence's own
        raw, scales = {m: st.raw[m].copy() for m in "kv"}, {m: st.scales[m].copy() for m in "kv"}
        for m in "kv":
            for s in range(1, 7):
                st.raw[m][own[s, :n]], st.scales[m][own[s, :n]] = raw[m][own[0, :n]], scales[m][own[0, :n]]
        st.upload()
        st.batch.set(st.new, st.len, own)
        assert np.array_equal(st.run_attention(q), got)
        st.raw, st.scales = raw, scales
        st.upload()

"""Attention's sums over the pages where one key outweighs the others."""
import numpy as np
import pytest

from tests.paged_ext_ref import SetupExt
from tests.paged_ref import encode

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"\n[case] {msg}", flush=True)


def put(st, k, v):
    """Sequence 0's keys and values."""
    g = st.slots(0, 0, st.len[0])
    for n, x in (("k", k), ("v", v)):
        if st.eight:
            y = st.pool[n].copy()
            y[g] = x
            st.fill(n, y)
        else:
            st.pool[n][g] = encode(x.astype(np.float32), st.dtype)
    st.upload()


@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32", "bf16", "f16"])
def test_one_key_before_many(gpu, dtype):
    """The first key weighs about as much as the 50,000 to 65,000 behind it, which are all alike, and it alone has a
    value: a row is the first key's share, 1 / (1 + pos e^-c(S)).

    A lane adds up 2048 tiles: sixteen of them, then those sums, each of 16 + 128 additions off by 2^-24 of the sum at
    most; the lanes' and the division, 4.  (All 2048 one after the other lose up to half of the sum's last place
    each, always the same way: 3e-5 of it in the mean, 8e-5 at most.)  The other keys' probability: its distance to
    the first, at most 18.1 in log2, has nine roundings (q times the scale and its factor, three sums, the cap's
    three, the distance), 9 * 18.1 * ln 2 = 113, the exponential 4."""
    say(f"one key before many: {dtype}")
    kv, G, hd, new, n = 2, 2, 64, 16384, 65536
    st = SetupExt(gpu, [(new, n)], kv * G, kv, hd, dtype, 128, cap=1000.0, max_rows=new)
    k, v = np.zeros((n, kv, hd)), np.zeros((n, kv, hd))
    k[0, :, 0], v[0] = 8.0, 1.0
    put(st, k, v)
    q = np.zeros((new, kv * G, hd), np.float32)
    q[:, :, 0] = np.random.default_rng(1).uniform(9.5, 12.5, (new, kv * G))
    got = st.run_attention(q.reshape(new, -1)).reshape(q.shape)
    s = 1000 * np.tanh(q[:, :, 0].astype(np.float64) / 1000)
    others = np.arange(n - new, n)[:, None] * np.exp(-s)
    want = 1 / (1 + others)
    tol = (16 + 128 + 4 + (113 + 4) * others * want) * 2.0 ** -24
    off = np.abs(got / want[..., None] - 1).max(-1)
    assert np.all(off <= tol), (off.max(), (off > tol).mean())

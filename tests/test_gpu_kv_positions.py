"""Decoding past an attention layer's max_seq_len, and at far positions: against
the numpy decoder of test_gpu_kv_mha.py, with its tolerance."""
import numpy as np
import pytest

import kv_model as km
import pywelvet as pw
from test_gpu_attention_masks import layer
from test_gpu_dense import rel_l2
from test_gpu_kv_mha import ALIBI, ROPE, ROPE_ALIBI, Decoder, sessions

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mask,pos,start", [(1, ROPE, 0), (3, ROPE, 0), (3, ALIBI, 0), (1, ROPE_ALIBI, 0),
                                            (1, ROPE, 200000), (3, ROPE, 200000)])
@pytest.mark.parametrize("dtype", [km.F32, km.BF16], ids=km.NAMES.get)
def test_decode_past_the_layers_max_seq_len(gpu, oracle, dtype, mask, pos, start):
    """A layer of max_seq_len 16 over a cache of 48: a windowed one (mask 3) sees
    the last 16 positions, the others all."""
    hip = pw.Hip()
    H, KVH, hd, msl, batch = 4, 2, 32, 16, 2
    Q, K, V, O, x = layer(start % 97 + mask, batch, 40, H, KVH, hd)
    x = x.reshape(batch, 40, H * hd)
    c = km.Cache(hip, dtype, H, KVH, hd, batch, 3, 16, poison=True)
    c.next[:] = start
    c.put(c.d_next, c.next)
    dec = Decoder(c, (Q, K, V, O), H, KVH, hd, pos, msl if mask == 3 else 0)
    m = sessions(batch, 1, H, KVH, hd, msl, mask, pos, (Q, K, V, O))
    dx, da, dy = (c.up(np.zeros((batch, H * hd), np.float32)) for _ in range(3))
    for t in range(40):
        c.put(dx, x[:, t])
        m.decode(c.c, c.seqs, dx, da, dy)
        want = dec.step(x[:, t], oracle).reshape(batch, H * hd)
        got = c.down(da, (batch, H * hd))
        assert rel_l2(got, want) <= 3e-6, t
        assert rel_l2(c.down(dy, (batch, H * hd)), got @ O.T) <= 5e-5
        c.c.advance(batch, c.d_lens, c.d_next, add=1)
    m.close()
    c.close()
    # a prefill keeps to it
    with pytest.raises(pw.WelvetError) as e:
        sessions(1, msl + 1, H, KVH, hd, msl, mask, pos, (Q, K, V, O))
    assert e.value.code == 1

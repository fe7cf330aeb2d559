"""Host side of the low-bit operators, on the CPU: scratch sizes, scratch of threads, sizes that 32 bits
do not hold, and the sampled loop over stand-in models."""
import ctypes

import pytest

from littlebit_b200 import _lib as L


def _attn_bytes(S, heads, kvh, d, max_seq, n, prefix):
    c = L.Kv4Cache(256, 256, 256, 256, S, kvh, max_seq, d)
    a = L.Kv4AttnArgs(cache=c, n=n, heads=heads, max_prefix=prefix, dtype=L.LBX_F32, q_ld=heads * d)
    return L.load().lbx_kv4_attn_workspace_size(ctypes.byref(a))


@pytest.mark.parametrize("S,heads,kvh,d,max_seq", [(64, 64, 8, 128, 2048), (64, 64, 8, 128, 4096), (64, 64, 8, 128, 8192),
                                                   (64, 32, 32, 128, 4096), (5, 64, 8, 64, 131072), (1, 4, 2, 64, 192),
                                                   (64, 64, 64, 128, 131072)])
def test_attention_scratch_for_the_longest_prefix_serves_every_step(S, heads, kvh, d, max_seq):
    most = 0
    for n in (1, 2, 3, 5, 7, 15, 16, 17, 31, 63, 64):
        sizes = [_attn_bytes(S, heads, kvh, d, max_seq, n, p) for p in [*range(0, max_seq - n, 61), max_seq - n]]
        assert min(sizes) > 0 and sizes == sorted(sizes), n
        assert sizes[-1] >= most  # (a chunk of fewer tokens runs in the scratch of more)
        most = sizes[-1]

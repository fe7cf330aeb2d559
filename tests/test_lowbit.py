"""The 64-bit restatement of the low-bit operators, on the CPU: the cache format's
properties, quantisation bounds, acceptance rules, and that a planted mistake is seen; and the
library's host-side refusals."""
import ctypes

import numpy as np
import pytest

from littlebit_b200 import _lib as L
from oracle import lowbit as olow


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [False, True])
def test_words_are_a_permutation_and_pack_round_trips(d, value):
    assert sorted(olow.kv4_words(d, value).tolist()) == list(range(d // 8))
    c = np.random.default_rng(0).integers(0, 16, (3, 5, d)).astype(np.uint8)
    assert np.array_equal(olow.kv4_unpack(olow.kv4_pack(c, value), value), c)


def test_quantised_values_lie_within_a_step():
    x = np.random.default_rng(1).standard_normal((200, 128)).astype(np.float32) * 5
    c, p = olow.kv4_quantize(x)
    v = olow.kv4_values(c, p)
    step = olow.bf16_value(p[..., 0]).astype(np.float64)
    # half a step; the ends moved by the bf16 rounding of least and of 15 steps
    y = x.reshape(200, 2, 64).astype(np.float64)
    slack = 2.0 ** -8 * (np.abs(y).max(-1) + 15 * step)
    assert (np.abs(v.reshape(200, 2, 64) - y).max(-1) <= step / 2 + slack).all()
    # a constant group is held to bfloat16, whatever its value
    k, p = olow.kv4_quantize(np.full((1, 64), 0.3, np.float32))
    assert (k == 0).all() and olow.kv4_values(k, p)[0, 0] == olow.bf16_value(olow.bf16_bits(np.float32(0.3)))


def test_eight_bit_codes():
    x = np.array([[0.0, 0, 0], [1, -2, 0.5], [np.nan, 1, 2], [1, np.inf, 0]], np.float32)
    q, s = olow.quantize_tokens(x)
    assert q.tolist() == [[0, 0, 0], [64, -127, 32], [0, 0, 0], [0, 0, 0]]
    assert s[0] == 0 and s[1] == np.float32(2) * np.float32(1 / 127) and np.isnan(s[2:]).all()


def test_attention_of_nothing_is_zero_and_trees_restrict():
    rng = np.random.default_rng(2)
    k, v = rng.standard_normal((1, 4, 64)), rng.standard_normal((1, 4, 64))
    q = rng.standard_normal((3, 1, 64))
    o = olow.attention(q, k, v, 0, 0.125, masks=[0, 0b10, 0b111])
    assert (o[0] == 0).all() and np.allclose(o[1, 0], v[0, 1])
    c = olow.attention(q, k, v, 0, 0.125)
    assert np.allclose(c[2], o[2]) and np.allclose(c[0, 0], v[0, 0])
    # a mistake in the mask is seen
    assert not np.allclose(olow.attention(q, k, v, 0, 0.125, masks=[1, 3, 5])[2], c[2])


def test_acceptance_rules():
    t = np.log(np.array([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]))
    d = np.log(np.array([[0.2, 0.6, 0.2]]))
    e = np.ones(3)
    assert olow.accept_sampled([1], t, d, [0.49], e, 1.0, 1)[:2] == (1, 2)   # 0.3 / 0.6
    assert olow.accept_sampled([1], t, d, [0.51], e, 1.0, 1)[:2] == (0, 0)   # only token 0 gained
    assert olow.accept_sampled([1], t, d, [0.51], e, 1.0, 0)[:2] == (0, 0)
    assert olow.accept_sampled([1], t, None, [0.31], e, 1.0, 1)[:2] == (0, 0)
    assert olow.accept_sampled([0], t, d, [0.99], e, 0.0, 1)[:2] == (1, 2)
    none = np.full((1, 3), -np.inf)
    assert olow.accept_sampled([], none, None, [], e, 1.0, 0)[:2] == (0, -1)


def test_host_side_refusals_without_a_gpu():
    lib = L.load()
    assert lib.lbx_linear_int8(None, None, 0, None) == L.LBX_EINVAL
    a = L.Int8Args(1, 1, 131073, 0, 0, 0, 256, 131073, 256, 131088, 256, None, 256, 1)
    assert lib.lbx_linear_int8(ctypes.byref(a), 256, 1 << 20, None) == L.LBX_EUNSUPPORTED
    a = L.Int8Args(1, 1, 64, 0, 0, 0, 256, 64, 264, 64, 256, None, 256, 1)
    assert lib.lbx_linear_int8(ctypes.byref(a), 256, 1 << 20, None) == L.LBX_EINVAL and "16 bytes" in L.last_error()
    a = L.Int8Args(1, 1, 64, 0, 0, 0, 256, 64, 256, 64, 256, None, 256, 1)
    assert lib.lbx_linear_int8(ctypes.byref(a), 256, 16, None) == L.LBX_EINVAL and "workspace" in L.last_error()
    assert lib.lbx_linear_int8_workspace_size(0, 1, 1) == 0
    c = L.Kv4Cache(256, 256, 256, 256, 1, 1, 64, 96)
    p = L.Kv4AppendArgs(c, 1, 0, 0, 0, None, 256, 256, 96, None)
    assert lib.lbx_kv4_append(ctypes.byref(p), None) == L.LBX_EUNSUPPORTED
    p.cache.head_dim, p.kv_ld, p.max_start = 64, 64, 64
    assert lib.lbx_kv4_append(ctypes.byref(p), None) == L.LBX_EINVAL and "max_seq" in L.last_error()
    p.cache.max_seq, p.max_start = 65, 0
    assert lib.lbx_kv4_append(ctypes.byref(p), None) == L.LBX_EINVAL and "multiple of 64" in L.last_error()
    t = L.Kv4AttnArgs(c, 1, 3, 0, 0, 0, 1.0, None, 256, 192, None, None, 256)
    t.cache.head_dim, t.cache.kv_heads = 64, 2
    assert lib.lbx_kv4_attn(ctypes.byref(t), 256, 1 << 20, None) == L.LBX_EINVAL
    assert lib.lbx_kv4_attn_workspace_size(ctypes.byref(t)) == 0
    s = L.AcceptArgs(n_seq=1, k=65, vocab=8)
    assert lib.lbx_accept_sampled(ctypes.byref(s), None) == L.LBX_EUNSUPPORTED
    s = L.AcceptArgs(n_seq=1, k=0, vocab=8, temperature=-1.0)
    assert lib.lbx_accept_sampled(ctypes.byref(s), None) == L.LBX_EINVAL


def test_struct_layouts_match_c(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    if shutil.which("gcc") is None:
        pytest.skip("gcc missing")
    hdr = Path(__file__).resolve().parent.parent / "include" / "lbx.h"
    structs = {"lbx_int8_args": L.Int8Args, "lbx_kv4_cache": L.Kv4Cache, "lbx_kv4_append_args": L.Kv4AppendArgs,
               "lbx_kv4_attn_args": L.Kv4AttnArgs, "lbx_accept_args": L.AcceptArgs}
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{hdr}"', "int main(void){"]
    for c, py in structs.items():
        src.append(f'printf("{c} %zu\\n", sizeof({c}));')
        src += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    (tmp_path / "s.c").write_text("\n".join(src + ["return 0;}"]))
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", "/usr/local/cuda/include", str(tmp_path / "s.c"), "-o", str(exe)], check=True)
    out = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, py in structs.items():
        assert int(out[c]) == ctypes.sizeof(py), c
        for f, _ in py._fields_:
            assert int(out[f"{c}.{f}"]) == getattr(py, f).offset, f"{c}.{f}"

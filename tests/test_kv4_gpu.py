"""The 4-bit KV cache: stored codes against the format's definition bit for bit,
attention against 64-bit sums over the stored values.

Tolerance of the attention, float32: a score is a sum of d products of rounded
factors, so it is off by at most (d + 8) 2^-24 sum |q k| scale; a probability by twice
that, relatively, and the result by as much of the largest value; bfloat16: the
queries are held in 16 bits of their group's largest instead (2^-16 each), and the
result is rounded to 8."""
import numpy as np
import pytest
import torch

from oracle import lowbit as olow

pytestmark = pytest.mark.gpu
THETA = 10000.0
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _bits(t):
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def _filled(S, H, T, d, seed, junk_from=None):
    """A cache of quantised random rows; slots from junk_from on hold NaN steps and any codes."""
    from littlebit_b200 import ops

    rng = np.random.default_rng(seed)
    c = ops.Kv4Cache.empty(S, H, T, d)
    T = c.shape[2]
    out = []
    for codes, par, value in ((c.k_codes, c.k_params, False), (c.v_codes, c.v_params, True)):
        x = rng.standard_normal((S, H, T, d)).astype(np.float32) * (1 + 3 * (np.arange(d) % 29 == 3))
        q, p = olow.kv4_quantize(x)
        pk = olow.kv4_pack(q, value)
        if junk_from is not None:
            p[:, :, junk_from:] = 0x7FC0
            pk[:, :, junk_from:] = 0xFF
        codes.copy_(torch.from_numpy(pk))
        par.copy_(torch.from_numpy(p.view(np.int16)).view(torch.bfloat16))
        out.append(olow.kv4_values(q, p))
    return c, out[0], out[1]


def _rope(pos, d):
    from littlebit_b200 import ops

    return ops.rope_table(torch.as_tensor(pos, dtype=torch.int32).cuda(), d, THETA)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("S,n,H,rope", [(1, 1, 1, True), (1, 1, 32, True), (1, 5, 3, True), (3, 2, 2, True), (2, 70, 5, True),
                                        (4, 1, 8, False)])
def test_append_stores_the_defined_codes(S, n, H, rope, d, dtype):
    from littlebit_b200 import ops

    g = torch.Generator().manual_seed(S * 100 + n + H)
    k = (torch.randn(S * n, H * d, generator=g) * 3).to(DT[dtype])
    v = torch.randn(S * n, H * d, generator=g).to(DT[dtype])
    v[0, :64] = 1.5       # a constant group
    v[-1, -64:] = 1e-39   # one below the least normal float
    v[0, 0] = 1.5
    start = torch.randint(0, 50, (S,), generator=g, dtype=torch.int32)
    c, kv0, vv0 = _filled(S, H, 128, d, 1)
    before = [t.clone() for t in (c.k_codes, c.k_params, c.v_codes, c.v_params)]
    pos = (start[:, None] + torch.arange(n)).reshape(-1)
    cs = _rope(pos, d) if rope else None
    ops.kv4_append(k.cuda(), v.cuda(), c, start.cuda(), 50, rope_cs=cs)
    kk = k.float().numpy().reshape(S * n, H, d)
    if rope:
        kk = olow.rotate_f32(kk, cs.cpu().numpy().reshape(S * n, 1, d // 2, 2))
    want = [(olow.kv4_quantize(kk), False), (olow.kv4_quantize(v.float().numpy().reshape(S * n, H, d)), True)]
    rk, rv = ops.kv4_read(c, start.cuda(), 50, n)
    for ((q, p), value), codes, par, b_codes, b_par, read in zip(
            want, (c.k_codes, c.v_codes), (c.k_params, c.v_params), (before[0], before[2]), (before[1], before[3]),
            (rk, rv)):
        packed = olow.kv4_pack(q, value).reshape(S, n, H, d // 2)
        vals = olow.kv4_values(q, p).reshape(S, n, H, d)
        for s in range(S):
            a = int(start[s])
            np.testing.assert_array_equal(codes[s, :, a:a + n].cpu().numpy(), packed[s].swapaxes(0, 1))
            np.testing.assert_array_equal(_bits(par[s, :, a:a + n]), p.reshape(S, n, H, d // 64, 2)[s].swapaxes(0, 1))
            # least + step * code, the product and the sum rounded to float32
            np.testing.assert_allclose(read[s].cpu().numpy(), vals[s].swapaxes(0, 1), rtol=2 ** -23, atol=2.0 ** -24 * 20)
            # nothing else was written
            assert torch.equal(codes[s, :, :a], b_codes[s, :, :a]) and torch.equal(codes[s, :, a + n:], b_codes[s, :, a + n:])
            assert torch.equal(par[s, :, :a].view(torch.int16), b_par[s, :, :a].view(torch.int16))
            assert torch.equal(par[s, :, a + n:].view(torch.int16), b_par[s, :, a + n:].view(torch.int16))


def test_append_of_nan_and_infinity():
    from littlebit_b200 import ops

    c = ops.Kv4Cache.empty(1, 2, 64, 128)
    k = torch.randn(3, 256, device="cuda")
    v = torch.randn(3, 256, device="cuda")
    k[0, 5], k[1, 70], v[2, 255] = float("nan"), float("inf"), float("-inf")
    v[0, 10], v[0, 20] = 3.3e38, -3.3e38  # a range that float32 does not hold
    ops.kv4_append(k, v, c, 0)
    rk, rv = ops.kv4_read(c, 0, None, 3)
    bad_k = torch.isnan(rk[0]).reshape(2, 3, 2, 64)
    bad_v = torch.isnan(rv[0]).reshape(2, 3, 2, 64)
    want_k, want_v = torch.zeros_like(bad_k), torch.zeros_like(bad_v)
    want_k[0, 0, 0] = want_k[0, 1, 1] = True
    want_v[1, 2, 1] = want_v[0, 0, 0] = True
    assert torch.equal(bad_k, want_k) and torch.equal(bad_v, want_v)


def _attend(q, c, prefix, heads, d, cs, mask, dtype):
    from littlebit_b200 import ops

    bound = int(max(prefix))
    return ops.attention_kv4(q.to(DT[dtype]).cuda(), c, torch.tensor(prefix, dtype=torch.int32).cuda(), bound, heads, d ** -0.5,
                             rope_cs=cs, tree_mask=mask)


def _tol(ref, kv, vv, q, d, dtype):
    qn = np.abs(q.double().numpy())
    sumqk = d * float(np.sqrt((qn ** 2).mean()) * np.sqrt((kv ** 2).mean())) * d ** -0.5
    vmax = float(np.abs(vv).max())
    if dtype == "f32":
        return 2 * (d + 8) * 2.0 ** -24 * sumqk * vmax + 1e-6 * vmax
    step = float(qn.max()) * 2.0 ** -15
    return 2 * d * step * float(np.abs(kv).mean()) * d ** -0.5 * vmax + 2.0 ** -8 * np.abs(ref)


# prefixes around the 16-slot tiles and the chunks of 128 and more; one query and many; shared heads; odd repeats
ATT = [(1, 1, 4, 4, 128, [0]), (1, 1, 4, 4, 64, [1]), (1, 1, 8, 1, 128, [15]), (1, 1, 8, 8, 128, [16]),
       (1, 1, 2, 2, 64, [127]), (1, 2, 6, 2, 128, [128]), (1, 5, 7, 1, 128, [129]), (1, 3, 16, 2, 64, [255]),
       (1, 8, 8, 2, 128, [700]), (1, 1, 64, 8, 128, [2049]), (1, 33, 4, 1, 64, [300]), (1, 64, 16, 2, 128, [1000]),
       (1, 100, 2, 2, 64, [37]), (1, 200, 8, 1, 128, [0]), (3, 1, 4, 2, 128, [5, 0, 300]), (5, 4, 8, 2, 64, [77, 1, 511, 512, 0]),
       (16, 1, 32, 32, 128, list(range(0, 480, 30)))]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S,n,heads,kvh,d,prefix", ATT)
def test_attention_matches_64_bits(S, n, heads, kvh, d, prefix, dtype):
    T = max(prefix) + n
    c, kv, vv = _filled(S, kvh, T, d, S + n + heads, junk_from=None)
    # what lies past each sequence's own tokens is stale: NaN steps and any codes
    for s in range(S):
        for t in (c.k_params, c.v_params):
            t[s, :, prefix[s] + n:] = float("nan")
    g = torch.Generator().manual_seed(n + heads)
    q = torch.randn(S * n, heads * d, generator=g).to(DT[dtype]).float()
    pos = [p + i for p in prefix for i in range(n)]
    cs = _rope(pos, d)
    out = _attend(q, c, prefix, heads, d, cs, None, dtype).double().cpu().numpy().reshape(S, n, heads, d)
    csn = cs.cpu().numpy().reshape(S, n, d // 2, 2)
    for s in range(S):
        ref = olow.attention(q.numpy().reshape(S, n, heads, d)[s], kv[s], vv[s], prefix[s], d ** -0.5, csn[s])
        tol = _tol(ref, kv, vv, q, d, dtype)
        assert (np.abs(out[s] - ref) <= tol).all(), (s, float(np.abs(out[s] - ref).max()), float(np.max(tol)))


@pytest.mark.parametrize("prefix", [0, 9, 250])
@pytest.mark.parametrize("n,d", [(2, 64), (17, 128), (26, 64), (64, 128)])
def test_tree_masks_and_rows_that_see_nothing(n, d, prefix):
    from littlebit_b200 import ops

    heads, kvh = 6, 2
    c, kv, vv = _filled(1, kvh, prefix + n, d, n)
    rng = np.random.default_rng(n)
    masks = [int(rng.integers(0, 1 << 63, dtype=np.uint64)) | (1 << i) for i in range(n)]
    masks[0] = 0                     # with no prefix, this row sees nothing
    masks[n - 1] = (1 << 64) - 1     # bits past n name no token
    md = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64).cuda()
    q = torch.randn(n, heads * d, generator=torch.Generator().manual_seed(n))
    cs = _rope([prefix + i for i in range(n)], d)
    out = _attend(q, c, [prefix], heads, d, cs, md, "f32").double().cpu().numpy().reshape(n, heads, d)
    ref = olow.attention(q.numpy().reshape(n, heads, d), kv[0], vv[0], prefix, d ** -0.5,
                         cs.cpu().numpy().reshape(n, d // 2, 2), masks)
    assert (np.abs(out - ref) <= _tol(ref, kv, vv, q, d, "f32")).all()
    if prefix == 0:
        assert (out[0] == 0).all()
    assert ops.device_error() == 0


def test_batched_and_single_calls_give_the_same_bits():
    from littlebit_b200 import ops

    S, n, heads, kvh, d = 3, 5, 16, 2, 128
    prefix = [250, 3, 700]
    c, _, _ = _filled(S, kvh, 1024, d, 4)
    q = torch.randn(S * n, heads * d, generator=torch.Generator().manual_seed(2)).cuda()
    cs = _rope([p + i for p in prefix for i in range(n)], d)
    both = _attend(q, c, prefix, heads, d, cs, None, "f32")
    for s in range(S):
        one = ops.Kv4Cache(*(t[s:s + 1] for t in (c.k_codes, c.k_params, c.v_codes, c.v_params)))
        rows = slice(s * n, (s + 1) * n)
        y = ops.attention_kv4(q[rows], one, prefix[s], None, heads, d ** -0.5, rope_cs=cs[rows])
        assert torch.equal(y.view(torch.int32), both[rows].view(torch.int32)), s
        for i in range(n):  # and each token as a step of its own
            r = slice(s * n + i, s * n + i + 1)
            y1 = ops.attention_kv4(q[r], one, prefix[s] + i, None, heads, d ** -0.5, rope_cs=cs[r])
            assert torch.equal(y1.view(torch.int32), both[r].view(torch.int32)), (s, i)
    assert torch.equal(_attend(q, c, prefix, heads, d, cs, None, "f32"), both)


def test_large_scores_keep_their_softmax():
    from littlebit_b200 import ops

    c, kv, vv = _filled(1, 1, 200, 128, 8)
    q = 40 * torch.randn(1, 128, generator=torch.Generator().manual_seed(3))
    y = ops.attention_kv4(q.cuda(), c, 199, None, 1, 128 ** -0.5).double().cpu().numpy()
    ref = olow.attention(q.numpy().reshape(1, 1, 128), kv[0], vv[0], 199, 128 ** -0.5)
    assert (np.abs(y.reshape(ref.shape) - ref) <= _tol(ref, kv, vv, q, 128, "f32")).all()


def test_visible_nan_reaches_the_result():
    from littlebit_b200 import ops

    c, _, _ = _filled(1, 1, 64, 64, 8)
    q = torch.randn(2, 64).cuda()
    clean = ops.attention_kv4(q, c, 20, None, 1, 0.125)
    c.v_params[0, 0, 21, 0, 0] = float("nan")  # the second new token's
    y = ops.attention_kv4(q, c, 20, None, 1, 0.125)
    assert torch.equal(y[0], clean[0]) and torch.isnan(y[1]).all()


def test_long_offsets_pass_32_bits():
    """A cache whose byte and value offsets pass 2^32: the last sequence is read at its own place."""
    from littlebit_b200 import ops

    S, H, T, d = 17, 32, 131072, 128  # 4.6e9 bytes of codes in each half, 9.1e9 values
    c = ops.Kv4Cache.empty(S, H, T, d)
    one, kv, vv = _filled(1, H, 192, d, 5)
    for a, b in ((c.k_codes, one.k_codes), (c.k_params, one.k_params), (c.v_codes, one.v_codes), (c.v_params, one.v_params)):
        a[S - 1, :, :192] = b[0]
    q = torch.randn(S, H * d, generator=torch.Generator().manual_seed(3)).cuda()
    prefix = torch.full((S,), 100, dtype=torch.int32, device="cuda")
    y = ops.attention_kv4(q, c, prefix, 130000, H, d ** -0.5)
    ref = ops.attention_kv4(q[S - 1:], one, 100, None, H, d ** -0.5)
    r64 = olow.attention(q[S - 1].cpu().numpy().reshape(1, H, d), kv[0], vv[0], 100, d ** -0.5)
    tol = _tol(r64, kv, vv, q[S - 1:].cpu(), d, "f32")
    assert (np.abs(y[S - 1].double().cpu().numpy().reshape(r64.shape) - r64) <= tol).all()
    assert (np.abs(ref.double().cpu().numpy().reshape(r64.shape) - r64) <= tol).all()
    k = torch.randn(S, H * d, device="cuda")
    ops.kv4_append(k, k, c, torch.full((S,), T - 1, dtype=torch.int32, device="cuda"), T - 1)
    rk, rv = ops.kv4_read(c, T - 1, None, 1)
    w, p = olow.kv4_quantize(k[S - 1].cpu().numpy().reshape(H, d))
    np.testing.assert_allclose(rv[S - 1, :, 0].cpu().numpy(), olow.kv4_values(w, p), rtol=2 ** -23, atol=1e-6)


def test_starts_out_of_range_are_told():
    from littlebit_b200 import ops

    c, _, _ = _filled(2, 1, 64, 64, 1)
    kept = c.k_codes.clone()
    x = torch.randn(2, 64, device="cuda")
    bad = torch.tensor([-1, 41], dtype=torch.int32, device="cuda")
    ops.clear_device_error()
    ops.kv4_append(x, x, c, bad, 40)
    assert ops.device_error() == 0x801 and torch.equal(c.k_codes, kept)
    ops.clear_device_error()
    rk, _ = ops.kv4_read(c, bad, 40, 2)
    assert ops.device_error() == 0x802 and torch.isnan(rk).all()
    ops.clear_device_error()
    y = ops.attention_kv4(x, c, bad, 40, 1, 1.0)
    assert ops.device_error() == 0x803 and torch.isnan(y).all()
    ops.clear_device_error()


def test_side_stream_and_graph():
    from littlebit_b200 import ops

    c, _, _ = _filled(1, 2, 512, 128, 6)
    q = torch.randn(1, 512).cuda()
    pre = torch.tensor([300], dtype=torch.int32, device="cuda")
    want = [ops.attention_kv4(q, c, p, None, 4, 0.1) for p in (300, 17)]
    out = torch.empty_like(q)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops.attention_kv4(q, c, pre, 500, 4, 0.1, out=out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ops.attention_kv4(q, c, pre, 500, 4, 0.1, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0])
    for p, w in ((17, want[1]), (300, want[0])):  # one graph at any length
        pre.fill_(p)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_refusals():
    from littlebit_b200 import ops

    c = ops.Kv4Cache.empty(1, 2, 64, 128)
    x = torch.zeros(1, 256, device="cuda")
    with pytest.raises(RuntimeError):
        ops.Kv4Cache.empty(1, 2, 64, 96)
    with pytest.raises(RuntimeError):
        ops.Kv4Cache(c.k_codes, c.k_params, c.v_codes[:, :, :32], c.v_params)
    for bad in (lambda: ops.kv4_append(x, x, c, 64), lambda: ops.kv4_append(x, x.bfloat16(), c, 0),
                lambda: ops.kv4_append(x[:, :128], x[:, :128], c, 0), lambda: ops.kv4_append(x.cpu(), x, c, 0),
                lambda: ops.kv4_append(x, x, c, torch.zeros(1, dtype=torch.int64, device="cuda"), 5),
                lambda: ops.kv4_append(x, x, c, 0, rope_cs=torch.zeros(64, device="cuda")),
                lambda: ops.kv4_read(c, 60, None, 5), lambda: ops.attention_kv4(x, c, 64, None, 2, 1.0),
                lambda: ops.attention_kv4(x, c, 0, None, 3, 1.0), lambda: ops.attention_kv4(x.half(), c, 0, None, 2, 1.0),
                lambda: ops.attention_kv4(x, c, 0, None, 2, 1.0, tree_mask=torch.zeros(2, dtype=torch.int64, device="cuda")),
                lambda: ops.attention_kv4(torch.zeros(65, 256, device="cuda"), ops.Kv4Cache.empty(1, 2, 128, 128), 0, None, 2, 1.0,
                                          tree_mask=torch.zeros(65, dtype=torch.int64, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()

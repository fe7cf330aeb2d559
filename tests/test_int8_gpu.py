"""8-bit integer product (lbx_quant_tokens, lbx_linear_int8) against 64-bit sums.

Tolerance: the integer sums are exact; the result has one rounding for the sum,
two for the token's scale and two products (5 x 2^-24 of the product), and one for
the bias sum; a bfloat16 result is the rounding of a number that near."""
import numpy as np
import pytest
import torch

from oracle import lowbit as olow

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _case(m, k, n, dtype, bias, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * (1 + 9 * (torch.rand(k, generator=g) < 0.01))
    w = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8)
    w[:, :k] = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8)
    w[:, k:] = 77  # what lies between rows is not read
    ws = torch.rand(n, generator=g) / (32 * k ** 0.5) + 1e-5
    b = torch.randn(n, generator=g) if bias else None
    return x.to(DT[dtype]), w, ws, b


def _check(y, x, w, ws, b):
    xf = x.float().numpy()
    ref = olow.linear_int8(xf, w.numpy(), ws.numpy(), None if b is None else b.numpy())
    prod = ref if b is None else ref - b.double().numpy()
    tol = 6 * 2.0 ** -24 * (np.abs(prod) + (0 if b is None else np.abs(b.double().numpy()))) + 1e-30
    got = y.double().cpu().numpy()
    if y.dtype == torch.bfloat16:  # the rounding of a number within the tolerance
        lo, hi = (torch.from_numpy(v).float().bfloat16().double().numpy() for v in (ref - tol, ref + tol))
        assert ((lo <= got) & (got <= hi)).all()
        return
    err = np.abs(got - ref)
    assert (err <= tol).all(), f"largest error over tolerance {float((err / tol).max())}"


SHAPES = [(1, 16, 1), (1, 4096, 1000), (1, 1, 7), (2, 17, 129), (3, 2056, 1030), (5, 100, 64), (8, 4096, 4096),
          (15, 640, 200), (16, 128, 128), (17, 129, 127), (31, 1000, 300), (33, 512, 640), (64, 4096, 513),
          (65, 300, 1025), (96, 2048, 256), (127, 384, 257), (128, 8192, 384), (129, 1024, 130), (200, 777, 999),
          (256, 256, 256), (257, 4096, 1000), (300, 129, 2049), (513, 640, 3000), (1000, 1000, 1000)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_int8(m, k, n, dtype):
    from littlebit_b200 import ops

    bias = (m + k + n) % 2 == 0
    x, w, ws, b = _case(m, k, n, dtype, bias, m * 7 + k + n)
    wd = w.cuda()[:, :k]
    y = ops.linear_int8(x.cuda(), wd, ws.cuda(), bias=None if b is None else b.cuda())
    assert y.dtype == x.dtype and y.shape == (m, n)
    _check(y, x, w[:, :k], ws, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 5), (3, 64), (2, 100), (7, 4096), (5, 8192), (2, 11008), (3, 28672),
                                 (2, 40000), (300, 33)])
def test_quantize_tokens_codes(m, k, dtype):
    from littlebit_b200 import ops

    g = torch.Generator().manual_seed(m + k)
    x = (torch.randn(m, k, generator=g) * 10 ** (torch.rand(m, 1, generator=g) * 8 - 4)).to(DT[dtype])
    x[0] = 0
    q, s = ops.quantize_tokens(x.cuda())
    rq, rs = olow.quantize_tokens(x.float().numpy())
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    assert q.stride(0) % 16 == 0


def test_rows_with_nan_or_infinity_stay_their_own():
    from littlebit_b200 import ops

    x, w, ws, b = _case(6, 200, 130, "f32", True, 3)
    clean = ops.linear_int8(x.cuda(), w.cuda()[:, :200], ws.cuda(), bias=b.cuda())
    x[1, 7], x[4, 0], x[5, 199] = float("nan"), float("inf"), float("-inf")
    y = ops.linear_int8(x.cuda(), w.cuda()[:, :200], ws.cuda(), bias=b.cuda())
    assert torch.isnan(y[[1, 4, 5]]).all()
    assert torch.equal(y[[0, 2, 3]], clean[[0, 2, 3]])


# long sums and few tiles (or few past whole rounds of them): K is cut over the SMs and the parts are joined
CUT = [(1, 20000, 700), (5, 28672, 500), (40, 16384, 1000), (130, 29990, 290), (300, 4992, 12631)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", CUT)
def test_sums_joined_from_parts(m, k, n, dtype):
    from littlebit_b200 import ops

    x, w, ws, b = _case(m, k, n, dtype, True, k)
    xd, wd, sd, bd = x.cuda(), w.cuda()[:, :k], ws.cuda(), b.cuda()
    y = ops.linear_int8(xd, wd, sd, bd)
    _check(y, x, w[:, :k], ws, b)
    for _ in range(3):  # whichever part comes last
        assert torch.equal(ops.linear_int8(xd, wd, sd, bd), y)
    assert torch.equal(ops.linear_int8(xd[m - 1:], wd, sd, bd)[0], y[m - 1])
    assert ops.device_error() == 0


@pytest.mark.parametrize("m", [2, 16, 40, 130, 300])
def test_a_token_does_not_depend_on_the_others(m):
    from littlebit_b200 import ops

    x, w, ws, _ = _case(m, 1040, 700, "f32", False, m)
    xd, wd, sd = x.cuda(), w.cuda()[:, :1040], ws.cuda()
    y = ops.linear_int8(xd, wd, sd)
    for i in (0, m // 2, m - 1):
        assert torch.equal(ops.linear_int8(xd[i:i + 1], wd, sd)[0], y[i]), i
    assert torch.equal(ops.linear_int8(xd, wd, sd), y)


def test_strided_rows_streams_and_types():
    from littlebit_b200 import ops

    x, w, ws, _ = _case(9, 256, 300, "f32", False, 5)
    big = torch.full((9, 300), 7.0, device="cuda")
    big[:, 3:259] = x.cuda()
    wbig = torch.zeros(300, 512, dtype=torch.int8, device="cuda")
    wbig[:, 16:272] = w[:, :256].cuda()
    out = torch.full((9, 400), -1.0, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear_int8(big[:, 3:259], wbig[:, 16:272], ws.cuda(), out=out[:, 50:350])
    torch.cuda.current_stream().wait_stream(side)
    _check(out[:, 50:350], x, w[:, :256], ws, None)
    assert (out[:, :50] == -1).all() and (out[:, 350:] == -1).all()
    y = ops.linear_int8(x.cuda(), w.cuda()[:, :256], ws.cuda(), out_dtype=torch.bfloat16)
    assert torch.equal(y, out[:, 50:350])


def test_zero_tokens_and_the_layer():
    from littlebit_b200 import ops

    x, w, ws, _ = _case(4, 64, 32, "f32", False, 5)
    assert ops.linear_int8(x.cuda()[:0], w.cuda(), ws.cuda()).shape == (0, 32)
    g = torch.Generator().manual_seed(1)
    wf = torch.randn(70, 90, generator=g)
    lin = ops.Int8Linear.from_float(wf.cuda())
    y = lin(x.cuda()[:, :64].repeat(1, 2)[:, :90].contiguous())
    ref = x[:, :64].repeat(1, 2)[:, :90].double() @ wf.double().T
    # each code is off by half a step at most: 1/254 of the row's maximum, of both factors
    xa = x[:, :64].repeat(1, 2)[:, :90]
    bound = 90 * xa.abs().amax(1, keepdim=True) * wf.abs().amax(1)[None] * 2 / 254
    assert ((y.cpu().double() - ref).abs() <= bound).all()


def test_in_a_cuda_graph():
    from littlebit_b200 import ops

    x, w, ws, _ = _case(5, 512, 640, "f32", False, 8)
    xd, wd, sd, out = x.cuda(), w.cuda(), ws.cuda(), torch.empty(5, 640, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops.linear_int8(xd, wd, sd, out=out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ops.linear_int8(xd, wd, sd, out=out)
    torch.cuda.synchronize()
    x2 = torch.randn(5, 512, generator=torch.Generator().manual_seed(9))
    xd.copy_(x2)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        _check(out, x2, w, ws, None)


def test_graphs_keep_their_workspaces():
    """Graphs captured on one stream, and eager calls there that need more, leave each other's scratch alone."""
    from littlebit_b200 import ops

    st = torch.cuda.Stream()
    cases = []
    for m, k, n in ((1, 20000, 700), (64, 16384, 1000), (130, 512, 2000)):
        x, w, ws, _ = _case(m, k, n, "f32", False, m)
        cases.append((x.cuda(), w.cuda()[:, :k], ws.cuda(), torch.empty(m, n, device="cuda")))
    want = [ops.linear_int8(x, w, s) for x, w, s, _ in cases]
    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(st):
        for x, w, s, out in cases:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):  # (no call before it on this stream)
                ops.linear_int8(x, w, s, out=out)
            graphs.append(g)
        eager = [ops.linear_int8(x, w, s) for x, w, s, _ in cases]
        junk = [torch.full((1 << 22,), 7, dtype=torch.int32, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(2):
        for (_, _, _, out), g, y, e in zip(cases, graphs, want, eager):
            out.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(st):
                g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, y) and torch.equal(e, y)
    assert all(int(j.min()) == 7 == int(j.max()) for j in junk)


def test_refusals():
    from littlebit_b200 import ops

    x, w, ws, _ = _case(4, 64, 32, "f32", False, 5)
    xd, wd, sd = x.cuda(), w.cuda(), ws.cuda()
    for bad in (lambda: ops.linear_int8(x, wd, sd), lambda: ops.linear_int8(xd.half(), wd, sd),
                lambda: ops.linear_int8(xd[:, :48], wd, sd), lambda: ops.linear_int8(xd, wd, sd[:31]),
                lambda: ops.linear_int8(xd, wd.to(torch.int32), sd), lambda: ops.linear_int8(xd, wd, sd.double()),
                lambda: ops.linear_int8(xd.T, wd, sd), lambda: ops.linear_int8(xd[None], wd, sd),
                lambda: ops.linear_int8(xd, wd, sd, bias=sd[:3]),
                lambda: ops.linear_int8(xd, wd, sd, out=torch.empty(4, 31, device="cuda")),
                lambda: ops.linear_int8(xd[:, :60].contiguous(), torch.zeros(32, 60, dtype=torch.int8, device="cuda"), sd),
                lambda: ops.linear_int8(xd[:, 1:49], wd[:, 1:49], sd),
                lambda: ops.linear_int8(torch.zeros(1, 131073, device="cuda"),
                                        torch.zeros(1, 131088, dtype=torch.int8, device="cuda")[:, :131073], sd[:1])):
        with pytest.raises(RuntimeError):
            bad()
    assert ops.device_error() == 0

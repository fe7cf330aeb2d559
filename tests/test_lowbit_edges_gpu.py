"""Edges of the low-bit operators: what a mask hides, extreme magnitudes, ties, default bounds, many row tiles."""
import numpy as np
import pytest
import torch

from oracle import lowbit as olow

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _cache(S, H, T, d, seed, scale=1.0):
    """A 4-bit cache of random rows, filled by the library, and the values it holds (float64)."""
    from littlebit_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(seed)
    c = ops.Kv4Cache.empty(S, H, T, d)
    T = c.shape[2]
    loud = 1 + 3 * (torch.arange(H * d, device="cuda") % d % 29 == 3)
    for s0 in range(0, T, 1024):
        n = min(1024, T - s0)
        k, v = (scale * torch.randn(S * n, H * d, generator=g, device="cuda") for _ in range(2))
        ops.kv4_append(k * loud, v, c, s0)
    return c


def _values(c, s, n):
    from littlebit_b200 import ops

    one = ops.Kv4Cache(*(t[s:s + 1] for t in (c.k_codes, c.k_params, c.v_codes, c.v_params)))
    k, v = ops.kv4_read(one, 0, None, n)
    return k[0].double(), v[0].double()


# a step that is not a number beside a least value that is one, and the reverse
BAD = [(float("nan"), 0.25), (float("inf"), 0.25), (float("-inf"), -1.0), (0.5, float("nan")), (0.5, float("inf")),
       (float("nan"), float("nan"))]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", BAD)
def test_stale_params_of_any_kind_reach_no_row(bad, d, dtype):
    from littlebit_b200 import ops

    heads, kvh, prefix = 8, 2, 70
    c = _cache(1, kvh, 192, d, 3)
    q = torch.randn(3, heads * d, generator=torch.Generator().manual_seed(1)).to(DT[dtype]).cuda()
    masks = torch.tensor([0b001, 0b011, 0b101], dtype=torch.int64, device="cuda")
    clean = [ops.attention_kv4(q, c, prefix, None, heads, d ** -0.5, tree_mask=m) for m in (None, masks)]
    for t in (c.k_params, c.v_params):
        t[:, :, prefix + 3:, :, 0], t[:, :, prefix + 3:, :, 1] = bad
    for m, want in zip((None, masks), clean):
        got = ops.attention_kv4(q, c, prefix, None, heads, d ** -0.5, tree_mask=m)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("half", ["k", "v"])
def test_a_slot_that_is_no_number_reaches_the_rows_that_see_it_alone(half, bad, d, dtype):
    from littlebit_b200 import ops

    heads, prefix = 3, 40
    c = _cache(1, 1, 64, d, 5)
    q = torch.randn(3, heads * d, generator=torch.Generator().manual_seed(2)).to(DT[dtype]).cuda()
    clean = ops.attention_kv4(q, c, prefix, None, heads, d ** -0.5)
    p = c.k_params if half == "k" else c.v_params
    p[0, 0, prefix + 1, :, 0], p[0, 0, prefix + 1, :, 1] = bad  # the second new token's
    y = ops.attention_kv4(q, c, prefix, None, heads, d ** -0.5)
    assert torch.equal(y[0], clean[0])
    if half == "v":
        assert torch.isnan(y[1:]).all()
    tree = ops.attention_kv4(q, c, prefix, None, heads, d ** -0.5,
                             tree_mask=torch.tensor([1, 3, 5], dtype=torch.int64, device="cuda"))
    assert torch.equal(tree[0], clean[0]) and not torch.isnan(tree[2]).any()


def test_threads_on_one_stream_keep_their_results():
    import threading

    from littlebit_b200 import ops

    d, heads = 128, 8
    g = torch.Generator().manual_seed(11)
    c = _cache(1, 2, 1024, d, 4)
    w = torch.randint(-127, 128, (700, 512), generator=g, dtype=torch.int32).to(torch.int8).cuda()
    ws = torch.rand(700, generator=g).cuda()
    xs = [torch.randn(m, 512, generator=g).cuda() for m in (1, 7, 33, 64)]
    qs = [torch.randn(n, heads * d, generator=g).cuda() for n in (1, 2, 5, 9)]
    want = [(ops.linear_int8(x, w, ws), ops.attention_kv4(q, c, 900, None, heads, 0.1)) for x, q in zip(xs, qs)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            for _ in range(150):
                y = ops.linear_int8(xs[i], w, ws)
                o = ops.attention_kv4(qs[i], c, 900, None, heads, 0.1)
                if not (torch.equal(y, want[i][0]) and torch.equal(o, want[i][1])):
                    bad.append(i)
        except BaseException as e:  # noqa: BLE001 (told below, from the main thread)
            bad.append(repr(e))

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad and ops.device_error() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1e-45, 1e-40, 1.1754943508222875e-38, 1e-37, 3.7e-37, 3.8e-37, 1e-36, 1e-30, 1e30, 3.3e38])
def test_eight_bit_codes_of_rows_of_any_magnitude(top, dtype):
    """Codes are 127 x / a wherever float32 holds 127 / a (from a = 3.74e-37 on), and 0 below: never a
    sign or a size that the row does not have."""
    from littlebit_b200 import ops

    x = torch.linspace(-1, 1, 200, dtype=torch.float64)
    rows = torch.stack([x, x.flip(0) * 0.5, -x.abs()]) * top
    rows = rows.float().to(DT[dtype])
    q, s = ops.quantize_tokens(rows.cuda())
    rq, rs = olow.quantize_tokens(rows.float().numpy())
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    f = rows.double()
    assert (q.cpu().double() * f >= 0).all()
    a = f.abs().amax(1, keepdim=True)
    held = (a > 3.75e-37) if top > 1e-38 else torch.zeros_like(a, dtype=torch.bool)
    want = torch.where(held, f / a.clamp_min(1e-300) * 127, torch.zeros_like(f))
    assert ((q.cpu().double() - want).abs() <= 0.5 + 1e-4).all()
    w = torch.ones(16, 208, dtype=torch.int8, device="cuda")[:, :200]
    y = ops.linear_int8(rows.cuda(), w, torch.ones(16, device="cuda"), out_dtype=torch.float32)
    assert (y[:, 0].cpu().double().numpy() * rq.astype(np.float64).sum(1) >= 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S", [1, 20, 40])
@pytest.mark.parametrize("T", [0.4, 1.0, 2.0])
def test_rows_of_the_lowest_number_are_uniform(T, S, dtype):
    """A row whose every logit is the type's lowest number has equal probabilities; only -inf and NaN have none."""
    from littlebit_b200 import ops

    V = 1003
    low = torch.finfo(DT[dtype]).min
    g = torch.Generator().manual_seed(S)
    e = -torch.log(torch.rand(S, V, generator=g).clamp_min(1e-30)) + 1e-30
    t = torch.full((S, 1, V), low, dtype=DT[dtype])
    _, nxt = ops.accept_sampled(None, t.cuda(), None, None, e.cuda(), T)
    assert torch.equal(nxt.cpu(), e.argmin(-1))
    # with some of them masked by -inf and NaN, among the others
    t[:, :, ::2] = float("-inf")
    t[:, :, 1::10] = float("nan")
    _, nxt = ops.accept_sampled(None, t.cuda(), None, None, e.cuda(), T)
    left = e.clone()
    left[:, ::2] = left[:, 1::10] = float("inf")
    assert torch.equal(nxt.cpu(), left.argmin(-1))
    # beside an ordinary logit they have no probability
    t[:, :, 5] = -40.0
    _, nxt = ops.accept_sampled(None, t.cuda(), None, None, e.cuda(), T)
    assert (nxt == 5).all()
    # nothing but -inf and NaN
    t[:] = float("-inf")
    t[:, :, 7] = float("nan")
    _, nxt = ops.accept_sampled(None, t.cuda(), None, None, e.cuda(), T)
    assert (nxt == -1).all()


def test_a_draft_from_a_row_of_the_lowest_number():
    """p and q uniform: the ratio is 1 and every draft is accepted; p against a q elsewhere: refused by q's excess alone."""
    from littlebit_b200 import ops

    V, low = 64, torch.finfo(torch.float32).min
    t = torch.full((2, 2, V), low)
    d = torch.full((2, 1, V), low)
    d[1, 0, 9] = 0.0                       # q is 1 at 9, p is 1/64
    u = torch.tensor([[0.999], [0.02]])    # above 1/64
    e = torch.rand(2, V, generator=torch.Generator().manual_seed(1)) + 0.1
    acc, nxt = ops.accept_sampled(torch.tensor([[3], [9]]).cuda(), t.cuda(), d.cuda(), u.cuda(), e.cuda())
    e[1, 9] = 9.0
    assert acc.tolist() == [1, 0] and nxt.cpu().tolist() == e.argmin(-1).tolist()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("at", [(3, 4), (0, 999), (500, 501), (31, 512)])
def test_zeros_of_either_sign_are_a_tie(at, dtype):
    from littlebit_b200 import ops

    t = torch.full((3, 1, 1000), -1.0, dtype=DT[dtype])
    t[0, 0, at[0]], t[0, 0, at[1]] = -0.0, 0.0
    t[1, 0, at[0]], t[1, 0, at[1]] = 0.0, -0.0
    t[2, 0, at[0]], t[2, 0, at[1]] = -0.0, -0.0
    _, nxt = ops.accept_sampled(None, t.cuda(), None, None, torch.ones(3, 1000, device="cuda"), 0.0)
    assert nxt.tolist() == [at[0]] * 3


def test_a_device_start_without_a_bound_reaches_the_whole_cache():
    from littlebit_b200 import ops

    c = ops.Kv4Cache.empty(2, 1, 64, 64)
    x = torch.randn(2 * 3, 64, device="cuda")
    at = torch.tensor([0, 61], dtype=torch.int32, device="cuda")  # the last start that three tokens fit at
    ops.clear_device_error()
    ops.kv4_append(x, x, c, at)
    k, v = ops.kv4_read(c, at, None, 3)
    y = ops.attention_kv4(x, c, at, None, 1, 0.125)
    assert ops.device_error() == 0
    w, p = olow.kv4_quantize(x.cpu().numpy().reshape(2, 3, 64))
    np.testing.assert_allclose(v[:, 0].cpu().numpy(), olow.kv4_values(w, p), rtol=2 ** -23, atol=1e-6)
    assert torch.equal(k, v)
    assert torch.equal(y, ops.attention_kv4(x, c, at, 61, 1, 0.125))
    # past the last start: told, as with a bound of the caller's
    ops.kv4_append(x, x, c, at + 1)
    assert ops.device_error() == 0x801
    ops.clear_device_error()


@pytest.mark.parametrize("max_seq", [1, 64, 100])
def test_a_draft_view_of_a_four_bit_decoder_steps_by_itself(max_seq):
    from littlebit_b200.cuda_models import _branch0_view
    from littlebit_b200.model import DecoderShape, LittleBitDecoder, synthetic_runtime_state

    shape = DecoderShape(num_hidden_layers=2, hidden_size=256, intermediate_size=512, num_attention_heads=4,
                         num_key_value_heads=2, vocab_size=512)
    ranks = {"q_proj": [64, 32], "k_proj": [32, 16], "v_proj": [32, 16], "o_proj": [64, 32],
             "gate_proj": [96, 40], "up_proj": [96, 40], "down_proj": [96, 40]}
    st = synthetic_runtime_state(shape, ranks, seed=21, unit_gain=True)
    dec = LittleBitDecoder(shape, st, device="cuda", max_seq=128, kv_bits=4)
    view = _branch0_view(dec, max_seq)
    assert view.max_seq == -(-max_seq // 64) * 64 == view.kv4[0].shape[2]
    wide = _branch0_view(dec, 128)
    ids = [5, 9, 2, 77][:max_seq]
    got, want = (x.forward_tokens(ids, 0)["logits"] for x in (view, wide))
    assert torch.equal(got, want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("exp", [-120, -60, 60, 99, 101, 110, 120])
def test_float32_queries_of_any_magnitude(exp, d):
    """Scores that far apart leave the largest one's value (or, for tiny queries, the mean), whatever the
    queries' exponent."""
    from littlebit_b200 import ops

    c = _cache(1, 1, 64, d, 9)
    kv, vv = _values(c, 0, 50)
    q = torch.randn(1, d, generator=torch.Generator().manual_seed(4)) * 2.0 ** exp
    y = ops.attention_kv4(q.cuda(), c, 49, None, 1, d ** -0.5).double()[0]
    s = (kv[0] @ q.cuda().double()[0]) * d ** -0.5
    want = torch.softmax(s, 0) @ vv[0]
    # (the two largest scores differ by far more than their rounding, 2^-18 of the largest)
    top = s.topk(2).values
    assert exp < 0 or top[0] - top[1] > 2.0 ** -12 * s.abs().max()
    assert (y - want).norm() <= 2.0 ** -18 * want.norm()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("exp", [-120, -60, 60, 95, 100])
def test_values_of_any_magnitude(exp, dtype):
    """Values up to 2^100 and down to the least normal step."""
    from littlebit_b200 import ops

    d = 64
    c = ops.Kv4Cache.empty(1, 1, 64, d)
    g = torch.Generator().manual_seed(6)
    k = torch.randn(50, d, generator=g).to(DT[dtype])
    v = (torch.randn(50, d, generator=g) * 2.0 ** exp).to(DT[dtype])
    ops.kv4_append(k.cuda(), v.cuda(), c, 0)
    kv, vv = _values(c, 0, 50)
    q = torch.randn(1, d, generator=g).to(DT[dtype])
    y = ops.attention_kv4(q.cuda(), c, 49, None, 1, d ** -0.5).double()[0]
    want = torch.softmax((kv[0] @ q.cuda().double()[0]) * d ** -0.5, 0) @ vv[0]
    tol = 2.0 ** -18 if dtype == "f32" else 2.0 ** -8
    assert (y - want).norm() <= tol * want.norm()


@pytest.mark.parametrize("exp", [-120, -60, 60, 100, 105, 110, 114])
def test_bfloat16_queries_of_any_magnitude(exp):
    """As in float32, with the rounding of the result to bfloat16 (2^-8) and of the queries to 11 bits, which for
    tiny queries is nothing and for huge ones leaves the largest score the largest."""
    from littlebit_b200 import ops

    d = 64
    c = _cache(1, 1, 64, d, 9)
    kv, vv = _values(c, 0, 50)
    q = (torch.randn(1, d, generator=torch.Generator().manual_seed(4)) * 2.0 ** exp).bfloat16()
    y = ops.attention_kv4(q.cuda(), c, 49, None, 1, d ** -0.5).double()[0]
    s = (kv[0] @ q.cuda().double()[0]) * d ** -0.5
    want = torch.softmax(s, 0) @ vv[0]
    top = s.topk(2).values
    assert exp < 0 or top[0] - top[1] > 2.0 ** -7 * s.abs().max()
    assert (y - want).norm() <= 2.0 ** -8 * want.norm()

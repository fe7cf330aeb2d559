"""Verification of sampled drafts (lbx_accept_sampled) against 64-bit softmaxes.

Accepted counts and tokens are whole numbers: they have to be equal wherever no
decision is nearer than 1e-5 (relatively) to its opposite, about a hundred times what float32
softmaxes are off by; all but a few sequences are that clear."""
import numpy as np
import pytest
import torch

from oracle import lowbit as olow

pytestmark = pytest.mark.gpu


def _inputs(S, k, V, seed, dtype=torch.float32, spread=3.0, noise=0.7, T=1.0):
    g = torch.Generator().manual_seed(seed)
    t = spread * torch.randn(S, k + 1, V, generator=g)
    d = t[:, :k] + noise * torch.randn(S, k, V, generator=g)
    t, d = t.to(dtype), d.to(dtype)
    pick = -torch.log(torch.rand(S, k, V, generator=g).clamp_min(1e-30))
    tok = (torch.softmax(d.float() / max(T, 1e-3), -1) / pick).argmax(-1) if k else torch.zeros(S, 0, dtype=torch.int64)
    u = torch.rand(S, k, generator=g)
    e = -torch.log(torch.rand(S, V, generator=g).clamp_min(1e-30)) + 1e-30
    return tok, t, d, u, e


def _check(tok, t, d, u, e, T, count=None, got=None, clear=0.9):
    from littlebit_b200 import ops

    c = lambda x: None if x is None else x.cuda()  # noqa: E731
    if got is None:
        Td = c(T) if isinstance(T, torch.Tensor) else T
        got = ops.accept_sampled(c(tok), c(t), c(d), c(u), c(e), Td, n_draft=c(count))
    acc, nxt = got[0].tolist(), got[1].tolist()
    S, k1 = t.shape[:2]
    told = 0
    for s in range(S):
        Ts = float(T[s]) if isinstance(T, torch.Tensor) else T
        n = k1 - 1 if count is None else int(count[s])
        a, b, margin = olow.accept_sampled(tok[s].numpy(), t[s].float().numpy(), None if d is None else d[s].float().numpy(),
                                           u[s].double().numpy(), e[s].double().numpy(), Ts, n)
        if margin > 1e-5:
            assert (acc[s], nxt[s]) == (a, b), (s, margin)
            told += 1
    assert told >= clear * S
    return acc, nxt


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,k,V,T", [(1, 0, 1, 1.0), (1, 0, 32000, 1.0), (1, 4, 32000, 1.0), (3, 1, 7, 0.5), (5, 8, 1000, 0.7),
                                     (33, 3, 513, 1.3), (16, 5, 4097, 1.0), (4, 2, 128256, 0.8), (2, 64, 300, 1.0),
                                     (200, 2, 65, 1.0)])
def test_matches_64_bits(S, k, V, T, dtype):
    _check(*_inputs(S, k, V, S + k + V, dtype, T=T), T)


def test_ragged_drafts_and_temperatures():
    S, k, V = 24, 6, 2000
    ins = _inputs(S, k, V, 4)
    g = torch.Generator().manual_seed(1)
    T = 0.3 + torch.rand(S, generator=g)
    count = torch.randint(0, k + 1, (S,), generator=g, dtype=torch.int32)
    count[0], count[1] = 0, k
    acc, _ = _check(*ins, T, count)
    assert all(a <= int(c) for a, c in zip(acc, count))
    assert 0 < sum(acc) < int(count.sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k,V", [(4, 5003), (64, 130)])
def test_a_sequence_does_not_depend_on_the_others(k, V, dtype):
    """From one sequence to many (blocks of other sizes): the same decisions, and again when called again."""
    from littlebit_b200 import ops

    ins = [x.cuda() for x in _inputs(40, k, V, 7, dtype)]
    _check(*(x[:12].cpu() for x in ins), 1.0)
    acc, nxt = ops.accept_sampled(*ins, 1.0)
    for S in (1, 12, 13, 32, 33, 40):
        a, b = ops.accept_sampled(*(x[:S] for x in ins), 1.0)
        same = (a == acc[:S]) & (b == nxt[:S])  # (sums of other orders: an even call may fall either way)
        assert int(same.sum()) >= 0.9 * S, S
        a2, b2 = ops.accept_sampled(*(x[:S] for x in ins), 1.0)
        assert torch.equal(a, a2) and torch.equal(b, b2)


def test_greedy_temperature_takes_the_first_maximum():
    tok, t, d, u, e = _inputs(12, 4, 300, 6, T=0.0)
    t[:, :, 17] = t.amax(-1)  # ties with a later or an earlier index
    tok[:6] = t[:6, :4].argmax(-1)
    tok[0, 2] = (tok[0, 2] + 1) % 300
    acc, nxt = _check(tok, t, None, u, e, 0.0, clear=1.0)
    first = torch.from_numpy(np.argmax(t.numpy(), -1))
    assert acc[1:6] == [4] * 5 and acc[0] == 2
    assert nxt[1] == int(first[1, 4]) and nxt[0] == int(first[0, 2])
    # agrees with the greedy acceptance
    from littlebit_b200 import ops

    for s in range(12):
        want = ops.accept_greedy_chain(tok[s].cuda(), first[s].cuda()).tolist()
        assert [acc[s], nxt[s]] == want


def test_drafts_without_probabilities():
    tok, t, _, u, e = _inputs(40, 3, 50, 9, spread=1.0)
    acc, nxt = _check(tok, t, None, u, e, 1.0)
    for s in range(40):
        if acc[s] < 3:
            assert nxt[s] != int(tok[s, acc[s]])  # a refused draft is not drawn again


def test_masked_infinite_and_nan_logits():
    S, k, V = 6, 2, 700
    tok, t, d, u, e = _inputs(S, k, V, 12)
    t[:, :, ::3] = float("-inf")        # masked tokens
    t[1, :, 5] = float("nan")           # a NaN in a masked place
    t[2, 1] = float("-inf")             # a row with nothing
    d[2, 1] = float("-inf")
    t[3, 0, 10] = float("inf")          # a forced token
    d[4] = t[4, :k]                     # draft and target agree: nothing is left over
    u[4] = 0.999999
    e[5, 3], e[5, 4] = 1e-38, 1e30
    tok[0, 0] = 3                       # a masked draft
    tok[2, 0] = int(t[2, 0].argmax())
    u[2, 0] = 0.0
    acc, nxt = _check(tok, t, d, u, e, 1.0, clear=0.6)
    assert acc[0] == 0 and nxt[0] % 3 != 0
    assert acc[2] == 1 and nxt[2] == -1
    if (tok[4] % 3 != 0).all():         # (a draft that the masks took away is refused)
        assert acc[4] == 2
    if acc[3] == 0:
        assert nxt[3] == 10 or int(tok[3, 0]) == 10


def test_equal_rows_fall_back_to_the_target():
    """p == q everywhere but the draft is refused: the token comes from p, never -1."""
    from littlebit_b200 import ops

    V = 100
    t = torch.zeros(1, 2, V)
    d = torch.zeros(1, 1, V)
    t[0, 0, 7] = d[0, 0, 7] = float("-inf")
    e = torch.rand(1, V, generator=torch.Generator().manual_seed(1)) + 0.1
    acc, nxt = ops.accept_sampled(torch.tensor([[7]]).cuda(), t.cuda(), d.cuda(), torch.zeros(1, 1).cuda(), e.cuda())
    e[0, 7] = 9
    assert acc.item() == 0 and nxt.item() == int(e.argmin())


def test_strides_streams_and_views():
    from littlebit_b200 import ops

    S, k, V = 4, 3, 1001
    tok, t, d, u, e = _inputs(S, k, V, 21)
    want = ops.accept_sampled(tok.cuda(), t.cuda(), d.cuda(), u.cuda(), e.cuda())
    tb = torch.full((S, k + 2, V + 5), 50.0).cuda()
    tb[:, 1:, 3:V + 3] = t.cuda()
    db = torch.full((k, S, V + 2), 50.0).cuda()
    db[:, :, 1:V + 1] = d.transpose(0, 1).cuda()
    eb = torch.full((S, V + 1), 1e-30).cuda()
    eb[:, 1:] = e.cuda()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.accept_sampled(tok.cuda(), tb[:, 1:, 3:V + 3],
                                 db.transpose(0, 1)[:, :, 1:V + 1], u.cuda(), eb[:, 1:])
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one row of logits shared by every sequence
    one = ops.accept_sampled(None, t[:1, :1].cuda().expand(S, 1, V), None, None, e.cuda())
    each = ops.accept_sampled(None, t[:1, :1].cuda().expand(S, 1, V).contiguous(), None, None, e.cuda())
    assert torch.equal(one[1], each[1]) and (one[0] == 0).all()


def test_drawn_tokens_follow_the_target():
    """Drafts drawn from q and verified against p give tokens distributed as p: each
    frequency within 5 standard deviations (16 of them: a fair draw fails once in 100 000 runs;
    the seed is fixed)."""
    from littlebit_b200 import ops

    S, V = 40000, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    t = 1.5 * torch.randn(V, generator=g, device="cuda")
    d = 1.5 * torch.randn(V, generator=g, device="cuda")
    exp = lambda: torch.empty(S, V, device="cuda").exponential_(generator=g)  # noqa: E731
    _, tok = ops.accept_sampled(None, d.expand(S, 1, V), None, None, exp())
    u = torch.rand(S, 1, generator=g, device="cuda")
    acc, nxt = ops.accept_sampled(tok[:, None].contiguous(), t.expand(S, 2, V), d.expand(S, 1, V), u, exp())
    first = torch.where(acc > 0, tok, nxt)
    for got, logits in ((tok, d), (first, t)):
        p = torch.softmax(logits.double(), -1)
        f = torch.bincount(got, minlength=V).double() / S
        assert ((f - p).abs() <= 5 * (p * (1 - p) / S).sqrt()).all()
    q, p = torch.softmax(d.double(), -1), torch.softmax(t.double(), -1)
    rate = float(torch.minimum(p, q).sum())
    assert abs(acc.double().mean().item() - rate) <= 5 * (rate * (1 - rate) / S) ** 0.5


def test_tokens_out_of_range_are_told():
    from littlebit_b200 import ops

    tok, t, d, u, e = _inputs(2, 2, 40, 3)
    tok[0, 0], tok[1, 0] = -1, 40
    u[:] = 0
    ops.clear_device_error()
    acc, nxt = ops.accept_sampled(tok.cuda(), t.cuda(), d.cuda(), u.cuda(), e.cuda())
    assert ops.device_error() == 0x811 and acc.tolist() == [0, 0] and (nxt >= 0).all()
    ops.clear_device_error()
    ops.accept_sampled(tok.cuda().clamp(0, 39), t.cuda(), d.cuda(), u.cuda(), e.cuda(),
                       n_draft=torch.tensor([3, -1], dtype=torch.int32).cuda())
    assert ops.device_error() == 0x812
    ops.clear_device_error()


def test_refusals():
    from littlebit_b200 import ops

    tok, t, d, u, e = (x.cuda() for x in _inputs(2, 2, 40, 3))
    for bad in (lambda: ops.accept_sampled(tok, t.cpu(), d, u, e), lambda: ops.accept_sampled(tok, t.half(), d, u, e),
                lambda: ops.accept_sampled(tok, t, d.bfloat16(), u, e), lambda: ops.accept_sampled(tok, t, d, u, e[:, :39]),
                lambda: ops.accept_sampled(tok.int(), t, d, u, e), lambda: ops.accept_sampled(tok[:, :1], t, d, u, e),
                lambda: ops.accept_sampled(tok, t, d, u.double(), e), lambda: ops.accept_sampled(tok, t, d, u, e, -1.0),
                lambda: ops.accept_sampled(tok, t, d, u, e, float("nan")), lambda: ops.accept_sampled(tok, t[0], d, u, e),
                lambda: ops.accept_sampled(tok, t, d, u, e, 1.0, n_draft=torch.zeros(2, device="cuda")),
                lambda: ops.accept_sampled(None, t, d, u, e)):
        with pytest.raises(RuntimeError):
            bad()
    big = torch.zeros(1, 66, 8, device="cuda")
    with pytest.raises(RuntimeError, match="unsupported"):
        ops.accept_sampled(torch.zeros(1, 65, dtype=torch.int64, device="cuda"), big, big[:, :65], torch.zeros(1, 65, device="cuda"),
                           torch.ones(1, 8, device="cuda"))

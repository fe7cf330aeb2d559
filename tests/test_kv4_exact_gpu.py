"""Attention over the 4-bit cache against 64-bit sums, by what its arithmetic leaves: relative errors of whole heads.

Tolerance, of the norm of a sequence's results for one kv head.  float32 calls hold each factor of a product in two
fp16 terms, 22 bits: a score is off by about 2^-22 sigma, sigma = scale |q * k| (element by element, the root of the
sum of squares), a weight by as much of itself, a weighted value by 2^-22 more, and the tensor cores' sums of 64
dimensions or 32 slots by a few steps of 2^-23: 2^-20 (1 + sigma).  bfloat16 calls hold one fp16 term, 11 bits, and
round the result to 8: roundings to p bits have a root mean square of at most 2^-p / sqrt(3), which makes
(2^-8 + 2^-11 (1 + sigma)) / sqrt(3).  Losing one slot of n leaves about 1 / sqrt(n): 1e-2 at 8192 slots."""
import numpy as np
import pytest
import torch

from oracle import lowbit as olow

pytestmark = pytest.mark.gpu
THETA = 10000.0
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _filled(S, H, T, d, seed):
    from littlebit_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(seed)
    c = ops.Kv4Cache.empty(S, H, T, d)
    T = c.shape[2]
    loud = 1 + 3 * (torch.arange(H * d, device="cuda") % d % 29 == 3)
    for s0 in range(0, T, 1024):
        n = min(1024, T - s0)
        k, v = (torch.randn(S * n, H * d, generator=g, device="cuda") for _ in range(2))
        ops.kv4_append(k * loud, v, c, s0)
    return c


def _values(codes, par, value):
    """Values [H, t, d] (float64) of packed codes [H, t, d / 2] and (step, least) [H, t, d / 64, 2]."""
    H, t, half = codes.shape
    w = codes.contiguous().view(torch.int32)[..., torch.from_numpy(olow.kv4_words(2 * half, value)).cuda()]
    x = ((w[..., None] >> (4 * torch.arange(8, device="cuda", dtype=torch.int32))) & 15).double()
    p = par.double()
    return (p[..., 1:2] + p[..., 0:1] * x.reshape(H, t, -1, 64)).reshape(H, t, 2 * half)


def _check(out, q, c, s, prefix, n, heads, cs, masks, dtype):
    """Rows of sequence s: out, q [n, heads * d]."""
    S, H, T, d = c.shape
    rep, top, scale = heads // H, prefix + n, d ** -0.5
    k = _values(c.k_codes[s, :, :top], c.k_params[s, :, :top], False)
    v = _values(c.v_codes[s, :, :top], c.v_params[s, :, :top], True)
    x = q.double().reshape(n, heads, d)
    t = cs.double().reshape(n, 1, d // 2, 2)
    a, b = x[..., :d // 2], x[..., d // 2:]
    x = torch.cat([a * t[..., 0] - b * t[..., 1], b * t[..., 0] + a * t[..., 1]], -1).reshape(n, H, rep, d)
    see = torch.ones(n, top, dtype=torch.bool, device="cuda")
    if masks is None:
        see[:, prefix:] = torch.tril(torch.ones(n, n, dtype=torch.bool, device="cuda"))
    else:
        see[:, prefix:] = (masks[:, None] >> torch.arange(n, device="cuda")) & 1 == 1
    sc = torch.einsum("nhrd,htd->nhrt", x, k) * scale
    p = torch.softmax(sc.masked_fill(~see[:, None, None], -torch.inf), -1)
    ref = torch.einsum("nhrt,htd->nhrd", p.nan_to_num(0), v)  # (a row that sees nothing: 0)
    got = out.double().reshape(n, H, rep, d)
    for h in range(H):
        sigma = float(torch.einsum("nrd,td->", x[:, h] ** 2, k[h] ** 2) / (n * rep * top)) ** 0.5 * scale
        tol = 2.0 ** -20 * (1 + sigma) if dtype == "f32" else (2.0 ** -8 + 2.0 ** -11 * (1 + sigma)) / 3 ** 0.5
        err, size = float((got[:, h] - ref[:, h]).norm()), float(ref[:, h].norm())
        assert err <= tol * size, (s, h, prefix, err / max(size, 1e-300), tol)


def _run(S, n, heads, kvh, d, T, lengths, tree, dtype, look):
    """Every sequence in one call; those of ``look`` against 64 bits and, bit for bit, against calls of their own."""
    from littlebit_b200 import ops

    c = _filled(S, kvh, T, d, S + n + heads + T)
    for s in range(S):  # what lies past a sequence's own tokens is stale
        c.k_params[s, :, lengths[s] + n:] = float("nan")
        c.v_params[s, :, lengths[s] + n:, :, 0] = float("nan")
    g = torch.Generator().manual_seed(n + heads)
    q = torch.randn(S * n, heads * d, generator=g).to(DT[dtype]).cuda()
    pos = torch.tensor([p + i for p in lengths for i in range(n)], dtype=torch.int32).cuda()
    cs = ops.rope_table(pos, d, THETA)
    masks = None
    if tree:
        rng = np.random.default_rng(n)
        m = [int(rng.integers(0, 1 << min(n, 62))) & ((2 << i) - 1) | 1 << i for _ in range(S) for i in range(n)]
        m = [x - (1 << 64) if x >> 63 else x for x in m]
        masks = torch.tensor(m, dtype=torch.int64).cuda()
    out = ops.attention_kv4(q, c, torch.tensor(lengths, dtype=torch.int32).cuda(), max(lengths), heads, d ** -0.5,
                            rope_cs=cs, tree_mask=masks)
    assert not torch.isnan(out).any() and ops.device_error() == 0
    for s in look:
        r = slice(s * n, (s + 1) * n)
        ms = None if masks is None else masks[r]
        one = ops.Kv4Cache(*(t[s:s + 1] for t in (c.k_codes, c.k_params, c.v_codes, c.v_params)))
        alone = ops.attention_kv4(q[r], one, lengths[s], None, heads, d ** -0.5, rope_cs=cs[r], tree_mask=ms)
        assert torch.equal(alone, out[r]), s
        _check(out[r], q[r], c, s, lengths[s], n, heads, cs[r], ms, dtype)


# Many sequences: a warp takes several sub-chunks on end, and row tiles share a ring of copies (three of five
# and two, with one place idle; two, two runs a block; three; four; seven times four of a tree with idle places), beside
# one tile of rows with four runs a block.
MANY = [(64, 5, 64, 8, 128, 1024, False), (64, 2, 64, 8, 128, 2048, False), (64, 3, 64, 8, 64, 2048, False),
        (64, 4, 64, 8, 64, 2048, False), (64, 26, 32, 8, 64, 1024, True), (64, 1, 64, 8, 128, 8192, False),
        (64, 5, 64, 8, 128, 8192, False)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S,n,heads,kvh,d,T,tree", MANY)
def test_many_sequences(S, n, heads, kvh, d, T, tree, dtype):
    ck = 128 if T <= 4096 else 256
    rng = np.random.default_rng(T + n)
    lengths = [T - n, 0, ck - 1, ck, 2 * ck + 1, ck - n, T // 2] + rng.integers(0, T - n + 1, S - 7).tolist()
    _run(S, n, heads, kvh, d, T, lengths, tree, dtype, [0, 1, 2, 3, 4, 5, S - 1])


FEW = [(1, 1, 4, 4, 128, 64, 0, False), (1, 1, 32, 32, 128, 4096, 4000, False), (1, 5, 16, 2, 128, 4096, 2049, False),
       (1, 64, 16, 2, 128, 2048, 1000, False), (1, 33, 4, 1, 64, 512, 300, True), (1, 26, 32, 8, 64, 2048, 777, True),
       (1, 64, 6, 2, 64, 128, 0, True), (1, 1, 7, 1, 64, 16384, 16000, False), (1, 5, 16, 2, 128, 65536, 65001, False),
       (2, 100, 8, 2, 64, 256, 37, False)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S,n,heads,kvh,d,T,prefix,tree", FEW)
def test_few_sequences(S, n, heads, kvh, d, T, prefix, tree, dtype):
    _run(S, n, heads, kvh, d, T, [prefix] * S, tree, dtype, range(S))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("small", [0, 1])
@pytest.mark.parametrize("ratio", [2.0 ** -4, 2.0 ** -8, 2.0 ** -40])
def test_groups_of_other_magnitudes(ratio, small, dtype):
    """A weight times a group's step is held relative to the largest step that the row has seen: a group of values
    2^-8 of its neighbour keeps its own accuracy, and one far below is off by no more than the head's."""
    from littlebit_b200 import ops

    n, T, d, prefix = 3, 640, 128, 600
    c = _filled(1, 1, T, d, 5)
    size = c.v_params.float()
    size[:, :, :, small] *= ratio
    c.v_params.copy_(size)
    q = torch.randn(n, 4 * d, generator=torch.Generator().manual_seed(6)).to(DT[dtype]).cuda()
    out = ops.attention_kv4(q, c, prefix, None, 4, d ** -0.5).double().reshape(n, 4, 2, 64)
    k, v = (_values(x[0, :, :prefix + n], p[0, :, :prefix + n], val)[0]
            for x, p, val in ((c.k_codes, c.k_params, False), (c.v_codes, c.v_params, True)))
    x = q.double().reshape(n, 4, d)
    sc = torch.einsum("nhd,td->nht", x, k) * d ** -0.5
    sc[:, :, prefix:].masked_fill_(~torch.tril(torch.ones(n, n, dtype=torch.bool, device="cuda"))[:, None], -torch.inf)
    ref = torch.einsum("nht,td->nhd", torch.softmax(sc, -1), v).reshape(n, 4, 2, 64)
    sigma = float(torch.einsum("nhd,td->", x ** 2, k ** 2) / (4 * n * (prefix + n))) ** 0.5 * d ** -0.5
    tol = 2.0 ** -20 * (1 + sigma) if dtype == "f32" else (2.0 ** -8 + 2.0 ** -11 * (1 + sigma)) / 3 ** 0.5
    err, norm = ((out - ref) ** 2).sum((0, 1, 3)).sqrt(), (ref ** 2).sum((0, 1, 3)).sqrt()
    assert err[1 - small] <= tol * norm[1 - small]
    assert err[small] <= tol * (norm[small] if ratio >= 2.0 ** -8 else norm[1 - small])

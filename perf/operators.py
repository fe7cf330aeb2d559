"""The low-bit operators of the sampled decoding path: cases, inputs, and their plain forms.

Four operators, each reached through ``littlebit_b200.ops``:

* ``linear_int8``: y = s_t * w_n * sum_k c_tk W_nk (+ b_n), the tokens quantised to 8 bits in the call;
* ``kv4_append`` (with ``kv4_read``): rotate, quantise and store new keys and values in a 4-bit cache;
* ``attention_kv4``: attention of new tokens over that cache (decode, verify batch, tree, many sequences);
* ``accept_sampled``: verification of drafted tokens against the target's probabilities, from given
  random numbers.

The 4-bit cache holds, for each head and slot, head_dim codes in blocks of eight (one 32-bit word, dimension
8b + i in bits 4i..4i+3 of its block's word; ``_word_of_block`` says where a block's word lies) and, for each
group of 64 dimensions, the pair (step, least value) in bfloat16; a value is least + step * code.
"""
import math

import torch

own = False

DEV = "cuda"
GROUP = 64
TINY = 1.1754943508222875e-38  # the least normal float


def listed():
    return [
        # the lm_head of a 7B-shaped model for one token: the largest read of a drafting step
        {"name": "int8_head_1", "op": "int8", "m": 1, "k": 4096, "n": 32000, "dtype": "float32", "bias": False},
        # a few tokens through a small odd-sized layer: the smallest call, all latency
        {"name": "int8_odd_3", "op": "int8", "m": 3, "k": 2056, "n": 1030, "dtype": "float32", "bias": True},
        # the lm_head of a 70B-shaped model verifying 64 sequences of 5 tokens
        {"name": "int8_head_320", "op": "int8", "m": 320, "k": 8192, "n": 32000, "dtype": "float32", "bias": False},
        # a prompt of 4096 tokens through a 70B-shaped MLP projection: arithmetic bound
        {"name": "int8_prompt", "op": "int8", "m": 4096, "k": 8192, "n": 28672, "dtype": "bfloat16", "bias": False},
        # one decoded token's keys and values of a 7B-shaped layer
        {"name": "append_1", "op": "append", "s": 1, "n": 1, "kvh": 32, "d": 128, "prefix": 1023, "max_seq": 4096,
         "dtype": "float32"},
        # a prompt of 2048 tokens of a 70B-shaped layer
        {"name": "append_prompt", "op": "append", "s": 1, "n": 2048, "kvh": 8, "d": 128, "prefix": 0, "max_seq": 4096,
         "dtype": "float32"},
        # decoding one token of a 7B-shaped layer at 4K
        {"name": "attn_decode", "op": "attn", "s": 1, "n": 1, "heads": 32, "kvh": 32, "d": 128, "prefix": 4000,
         "max_seq": 4096, "tree": False, "dtype": "float32"},
        # verifying 5 tokens of a 70B-shaped layer over a long context
        {"name": "attn_verify_long", "op": "attn", "s": 1, "n": 5, "heads": 64, "kvh": 8, "d": 128, "prefix": 130001,
         "max_seq": 131072, "tree": False, "dtype": "float32"},
        # decoding one token of each of 64 sequences of different lengths, in bfloat16
        {"name": "attn_batch", "op": "attn", "s": 64, "n": 1, "heads": 64, "kvh": 8, "d": 128, "prefix": 8100,
         "max_seq": 8192, "tree": False, "dtype": "bfloat16"},
        # verifying a drafted tree of 26 nodes with heads of 64
        {"name": "attn_tree", "op": "attn", "s": 1, "n": 26, "heads": 32, "kvh": 8, "d": 64, "prefix": 777,
         "max_seq": 2048, "tree": True, "dtype": "float32"},
        # verifying 4 sampled drafts of one sequence
        {"name": "accept_1", "op": "accept", "s": 1, "k": 4, "v": 32000, "temperature": 1.0, "ragged": False,
         "dtype": "float32"},
        # verifying up to 8 sampled drafts of each of 64 sequences
        {"name": "accept_64", "op": "accept", "s": 64, "k": 8, "v": 32000, "temperature": 0.7, "ragged": True,
         "dtype": "float32"},
    ]


def _log_between(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["int8", "append", "attn", "accept"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "int8":
        m = _log_between(rng, 1, 4096)
        return {"op": op, "m": m, "k": _log_between(rng, 64, 8192), "n": _log_between(rng, 64, 28672), "dtype": dtype,
                "bias": rng.random() < 0.5}
    if op == "append":
        s = _log_between(rng, 1, 64)
        n = _log_between(rng, 1, max(1, 2048 // s))
        prefix = rng.randint(0, 2000)
        return {"op": op, "s": s, "n": n, "kvh": rng.choice([1, 2, 4, 8, 32]), "d": rng.choice([64, 128]),
                "prefix": prefix, "max_seq": -(-(prefix + n) // 64) * 64, "dtype": dtype}
    if op == "attn":
        s = rng.choice([1, 1, 1, _log_between(rng, 2, 64)])
        d = rng.choice([64, 128])
        kvh = rng.choice([1, 2, 4, 8, 32])
        rep = rng.choice([1, 2, 4, 7, 8])
        n = rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 64)])
        # no more cache, and no more products, than the largest listed cases hold
        top = min(130001, 64 * 8 * 8100 * 128 // (s * kvh * d), 5 * 64 * 130001 // (s * n * kvh * rep))
        prefix = _log_between(rng, 1, max(2, top)) - 1
        return {"op": op, "s": s, "n": n, "heads": kvh * rep, "kvh": kvh, "d": d, "prefix": prefix,
                "max_seq": -(-(prefix + n) // 64) * 64, "tree": n > 1 and rng.random() < 0.4, "dtype": dtype}
    s = _log_between(rng, 1, 64)
    return {"op": op, "s": s, "k": rng.randint(0, 8), "v": _log_between(rng, 1000, 64000),
            "temperature": rng.choice([0.5, 0.7, 1.0, 1.3]), "ragged": rng.random() < 0.5, "dtype": dtype}


# ---- inputs ---------------------------------------------------------------------------------------------


def _type(case):
    return getattr(torch, case["dtype"])


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _word_of_block(d, value):
    """Word index, within a slot's row, of each block of eight dimensions."""
    b = torch.arange(d // 8, device=DEV)
    g, r = b // 8, b % 8
    if value:
        return r * (d // 64) + g
    return (r % 4) * (d // 32) + 2 * g + r // 4


def _pack(codes, value):
    """Codes [..., d] of 0..15 (int32) -> bytes [..., d / 2] in the cache's order."""
    d = codes.shape[-1]
    shift = 4 * torch.arange(8, device=DEV, dtype=torch.int64)
    words = (codes.reshape(*codes.shape[:-1], d // 8, 8).to(torch.int64) << shift).sum(-1)
    out = torch.empty_like(words)
    out[..., _word_of_block(d, value)] = words
    byte = (out[..., None] >> (8 * torch.arange(4, device=DEV, dtype=torch.int64))) & 255
    return byte.reshape(*codes.shape[:-1], d // 2).to(torch.uint8)


def _unpack(packed, value):
    """Bytes [..., d / 2] -> codes [..., d] as float32."""
    d = packed.shape[-1] * 2
    byte = packed.reshape(*packed.shape[:-1], d // 8, 4)[..., _word_of_block(d, value), :]
    return torch.stack([byte & 15, byte >> 4], -1).reshape(*packed.shape[:-1], d).float()


def _random_cache(s, kvh, max_seq, d, g):
    """A cache as steps before this one left it: every slot holds the quantised rows of some token."""
    def half(value):
        codes = torch.empty(s, kvh, max_seq, d // 2, dtype=torch.uint8, device=DEV)
        par = torch.empty(s, kvh, max_seq, d // GROUP, 2, dtype=torch.bfloat16, device=DEV)
        step = max(1, (1 << 26) // (kvh * max_seq * d))
        for a in range(0, s, step):
            x = torch.randn(len(range(a, min(a + step, s))), kvh, max_seq, d, generator=g, device=DEV)
            x *= 1 + 2 * (torch.arange(d, device=DEV) % 37 == 5) if not value else 0.5
            c, p = _quantise(x)
            codes[a:a + step], par[a:a + step] = _pack(c.to(torch.int32), value), p
        return codes, par

    return (*half(False), *half(True))


def _quantise(x):
    """x [..., d] float32 -> codes [..., d] (float32) and (step, least) bfloat16 [..., d / 64, 2]."""
    y = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    lo, hi = y.amin(-1), y.amax(-1)
    fifteenth = torch.tensor(1 / 15, dtype=torch.float32, device=x.device)
    step = ((hi - lo) * fifteenth).to(torch.bfloat16)
    step = torch.where(step.float() < TINY, torch.zeros_like(step), step)
    least = lo.to(torch.bfloat16)
    inv = torch.where(step > 0, torch.ones_like(lo) / step.float(), torch.zeros_like(lo))
    codes = torch.clamp(torch.round((y - least.float()[..., None]) * inv[..., None]), 0, 15)
    return codes.reshape(x.shape), torch.stack([step, least], -1)


def _rope_table(pos, d):
    """(cos, sin) pairs [n, d] of each position: pos * 10000^(-2j/d) in 64 bits, rounded."""
    j = torch.arange(d // 2, device=DEV, dtype=torch.float64)
    a = pos.double()[:, None] * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=DEV), -2 * j / d)
    return torch.stack([a.cos(), a.sin()], -1).reshape(pos.numel(), d).float().contiguous()


def _tree_masks(n, g):
    """The masks of a random tree of n nodes: bit j of row i says that node j is i or one of its ancestors."""
    parent = (torch.rand(n, generator=g, device=DEV) * torch.arange(n, device=DEV)).long().tolist()
    masks = [1]
    for i in range(1, n):
        masks.append(masks[parent[i]] | 1 << i)
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device=DEV)


def _lengths(case, g):
    """Cached lengths of the sequences: the longest is the case's, the others a quarter of it or more."""
    p = case["prefix"]
    x = (p * (0.25 + 0.75 * torch.rand(case["s"], generator=g, device=DEV))).to(torch.int32)
    x[0] = p
    return x


def prepare(case, seed):
    g = _gen(seed)
    op, t = case["op"], _type(case)
    st = {"case": case}
    if op == "int8":
        m, k, n = case["m"], case["k"], case["n"]
        x = torch.randn(m, k, generator=g, device=DEV)
        st["x"] = (x * (1 + 9 * (torch.rand(k, generator=g, device=DEV) < 0.004))).to(t)  # a few loud channels
        # rows start on 16 bytes, as the weights' keeper lays them out
        w = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device=DEV)
        w[:, :k] = torch.randn(n, k, generator=g, device=DEV).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        st["w"] = w[:, :k]
        st["ws"] = (0.5 + torch.rand(n, generator=g, device=DEV)) / (32 * math.sqrt(k))
        st["bias"] = torch.randn(n, generator=g, device=DEV) if case["bias"] else None
    elif op == "append":
        s, n, kvh, d = case["s"], case["n"], case["kvh"], case["d"]
        kc, kp, vc, vp = _random_cache(s, kvh, case["max_seq"], d, g)
        st.update(kc=kc, kp=kp, vc=vc, vp=vp)
        st["k"] = torch.randn(s * n, kvh * d, generator=g, device=DEV).to(t)
        st["v"] = torch.randn(s * n, kvh * d, generator=g, device=DEV).to(t)
        st["start"] = _lengths(case, g)
        pos = (st["start"][:, None] + torch.arange(n, device=DEV)).reshape(-1)
        st["rope"] = _rope_table(pos, d)
    elif op == "attn":
        s, n, heads, kvh, d = case["s"], case["n"], case["heads"], case["kvh"], case["d"]
        kc, kp, vc, vp = _random_cache(s, kvh, case["max_seq"], d, g)
        st.update(kc=kc, kp=kp, vc=vc, vp=vp)
        st["q"] = torch.randn(s * n, heads * d, generator=g, device=DEV).to(t)
        st["prefix"] = _lengths(case, g)
        st["tree"] = torch.cat([_tree_masks(n, g) for _ in range(s)]) if case["tree"] else None
        pos = (st["prefix"][:, None] + torch.arange(n, device=DEV)).reshape(-1)
        st["rope"] = _rope_table(pos, d)
    else:
        s, k, v = case["s"], case["k"], case["v"]
        target = 3 * torch.randn(s, k + 1, v, generator=g, device=DEV)
        draft = target[:, :k] + 0.7 * torch.randn(s, k, v, generator=g, device=DEV)
        st["target"], st["draft"] = target.to(t), draft.to(t)
        noise = torch.empty(s, k, v, device=DEV).exponential_(generator=g).clamp_min_(TINY)
        st["tokens"] = (torch.exp(st["draft"].float() / case["temperature"]) / noise).argmax(-1) if k else \
            torch.empty(s, 0, dtype=torch.int64, device=DEV)
        st["u"] = torch.rand(s, k, generator=g, device=DEV)
        st["e"] = torch.empty(s, v, device=DEV).exponential_(generator=g).clamp_min_(TINY)
        st["count"] = torch.randint(0, k + 1, (s,), generator=g, device=DEV, dtype=torch.int32) if case["ragged"] \
            else None
    return st


# ---- one pass -------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    from littlebit_b200 import ops

    case, op = st["case"], st["case"]["op"]
    if op == "int8":
        return ops.linear_int8(st["x"], st["w"], st["ws"], bias=st["bias"])
    if op == "append":
        cache = ops.Kv4Cache(st["kc"], st["kp"], st["vc"], st["vp"])
        ops.kv4_append(st["k"], st["v"], cache, st["start"], case["prefix"], rope_cs=st["rope"])
        return ops.kv4_read(cache, st["start"], case["prefix"], case["n"])
    if op == "attn":
        cache = ops.Kv4Cache(st["kc"], st["kp"], st["vc"], st["vp"])
        return ops.attention_kv4(st["q"], cache, st["prefix"], case["prefix"], case["heads"], case["d"] ** -0.5,
                                 rope_cs=st["rope"], tree_mask=st["tree"])
    return ops.accept_sampled(st["tokens"], st["target"], st["draft"], st["u"], st["e"], case["temperature"],
                              n_draft=st["count"])


def _rotate(x, table):
    """Rotate-half embedding of x [rows, heads, d] with (cos, sin) pairs [rows, d]."""
    h = x.shape[-1] // 2
    cs = table.reshape(table.shape[0], 1, h, 2)
    c, s = cs[..., 0], cs[..., 1]
    x1, x2 = x[..., :h], x[..., h:]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def _values(codes, par, value):
    """The values [..., d] that packed codes and (step, least) pairs stand for."""
    c = _unpack(codes, value)
    y = c.reshape(*c.shape[:-1], c.shape[-1] // GROUP, GROUP)
    return (par[..., 1:2].float() + par[..., 0:1].float() * y).reshape(c.shape)


def _run_plain(st):
    case, op = st["case"], st["case"]["op"]
    if op == "int8":
        x = st["x"].float()
        a = x.abs().amax(-1, keepdim=True)
        inv = torch.where(a > 0, torch.full_like(a, 127) / a, torch.zeros_like(a))
        c = torch.round(x * inv)
        y = (c @ st["w"].float().T) * (a * (1 / 127)) * st["ws"]
        return (y if st["bias"] is None else y + st["bias"]).to(st["x"].dtype)
    if op == "append":
        s, n, kvh, d = case["s"], case["n"], case["kvh"], case["d"]
        slots = st["start"].long()[:, None] + torch.arange(n, device=DEV)
        seqs = torch.arange(s, device=DEV)[:, None]
        k = _rotate(st["k"].float().reshape(s * n, kvh, d), st["rope"]).reshape(s, n, kvh, d)
        v = st["v"].float().reshape(s, n, kvh, d)
        ck, pk = _quantise(k)
        cv, pv = _quantise(v)
        st["kc"][seqs, :, slots], st["kp"][seqs, :, slots] = _pack(ck.to(torch.int32), False), pk
        st["vc"][seqs, :, slots], st["vp"][seqs, :, slots] = _pack(cv.to(torch.int32), True), pv
        return (_values(st["kc"][seqs, :, slots], st["kp"][seqs, :, slots], False).transpose(1, 2).contiguous(),
                _values(st["vc"][seqs, :, slots], st["vp"][seqs, :, slots], True).transpose(1, 2).contiguous())
    if op == "attn":
        s, n, heads, kvh, d = case["s"], case["n"], case["heads"], case["kvh"], case["d"]
        top, rep = case["prefix"] + n, heads // kvh
        seen = _seen(st, top)  # [s, n, top]
        any_seen = seen.any(1)[:, None, :, None]
        k = _values(st["kc"][:, :, :top], st["kp"][:, :, :top], False)
        v = torch.where(any_seen, _values(st["vc"][:, :, :top], st["vp"][:, :, :top], True), 0)
        q = _rotate(st["q"].float().reshape(s * n, heads, d), st["rope"]).reshape(s, n, kvh, rep, d)
        q = q.permute(0, 2, 1, 3, 4).reshape(s, kvh, n * rep, d) * d ** -0.5
        score = (q @ k.transpose(-1, -2)).reshape(s, kvh, n, rep, top)
        score = torch.where(seen[:, None, :, None], score, -torch.inf)
        m = score.amax(-1, keepdim=True)
        p = torch.exp(score - torch.where(m == -torch.inf, 0, m))
        total = p.sum(-1, keepdim=True)
        o = (p.reshape(s, kvh, n * rep, top) @ v).reshape(s, kvh, n, rep, d)
        o = torch.where(total > 0, o / total, 0)
        return o.permute(0, 2, 1, 3, 4).reshape(s * n, heads * d).to(st["q"].dtype)
    return _accept(st, torch.float32)


def _seen(st, top):
    """Which slots each query sees, [s, n, top]: its sequence's cached ones, and the new ones its mask allows."""
    case = st["case"]
    s, n = case["s"], case["n"]
    prefix = st["prefix"].long()[:, None, None]
    j = torch.arange(top, device=DEV)[None, None] - prefix  # index among the new tokens
    if st["tree"] is None:
        new = j <= torch.arange(n, device=DEV)[None, :, None]
    else:
        new = (st["tree"].reshape(s, n, 1) >> j.clamp(0, 63)) & 1 == 1
    return (j < 0) | ((j < n) & new)


def _accept(st, t):
    case = st["case"]
    s, k, v = case["s"], case["k"], case["v"]
    target, draft = st["target"].to(t) / case["temperature"], st["draft"].to(t) / case["temperature"]
    p = torch.exp(target - target.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    count = torch.full((s,), k, device=DEV) if st["count"] is None else st["count"].long()
    rows = torch.arange(s, device=DEV)
    if k:
        q = torch.exp(draft - draft.amax(-1, keepdim=True))
        q = q / q.sum(-1, keepdim=True)
        at = st["tokens"][..., None]
        ratio = p[:, :k].gather(-1, at)[..., 0] / q.gather(-1, at)[..., 0].clamp_min(1e-10)
        ok = (st["u"] < ratio.clamp_max(1)) & (torch.arange(k, device=DEV) < count[:, None])
        a = torch.cumprod(ok.long(), 1).sum(1)
        rest = (p[rows, a] - q[rows, a.clamp_max(k - 1)]).clamp_min(0)
        rest = torch.where((a < count)[:, None] & (rest > 0).any(-1, keepdim=True), rest, p[rows, a])
    else:
        a = torch.zeros(s, dtype=torch.int64, device=DEV)
        rest = p[:, 0]
    return a, (rest / st["e"].to(t)).argmax(-1)


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------


def _exact_codes(x):
    """Dequantised values of x [..., d] (float64 holding float32 numbers), every rounding that the format names
    made where it names it: differences and products to float32, steps and least values to bfloat16."""
    y = x.unflatten(-1, (-1, GROUP))
    lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
    f32 = lambda v: v.float().double()  # noqa: E731
    bf16 = lambda v: v.float().bfloat16().double()  # noqa: E731
    step = bf16(f32(f32(hi - lo) * f32(torch.tensor(1 / 15, dtype=torch.float64, device=DEV))))
    step = step * (step >= TINY)
    least = bf16(lo)
    inv = f32(1 / step).masked_fill(step == 0, 0)
    code = torch.round(f32(f32(y - least) * inv)).clamp(0, 15)
    return (least + step * code).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "int8":
        x = st["x"].double()
        peak = x.abs().max(-1).values
        inv = (127 / peak).masked_fill(peak == 0, 0).float().double()
        c = (x * inv[:, None]).float().double().round()
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device=DEV)
        for a in range(0, case["n"], 4096):
            b = min(a + 4096, case["n"])
            out[:, a:b] = torch.einsum("mk,nk->mn", c, st["w"][a:b].double())
        out *= (peak / 127)[:, None]
        out *= st["ws"].double()
        return out if st["bias"] is None else out + st["bias"].double()
    if op == "append":
        s, n, kvh, d = case["s"], case["n"], case["kvh"], case["d"]
        k, v = (st[x].double().reshape(s, n, kvh, d) for x in "kv")
        cs = st["rope"].double().reshape(s, n, 1, d // 2, 2)
        f32 = lambda y: y.float().double()  # noqa: E731
        a, b = k.chunk(2, -1)
        turned = torch.cat([f32(f32(a * cs[..., 0]) - f32(b * cs[..., 1])), f32(f32(b * cs[..., 0]) + f32(a * cs[..., 1]))], -1)
        return _exact_codes(turned).movedim(1, 2), _exact_codes(v).movedim(1, 2)
    if op == "attn":
        s, n, heads, kvh, d = case["s"], case["n"], case["heads"], case["kvh"], case["d"]
        rep, out = heads // kvh, torch.zeros(s, n, heads, d, dtype=torch.float64, device=DEV)
        q = st["q"].double().reshape(s, n, heads, d)
        cs = st["rope"].double().reshape(s, n, 1, d // 2, 2)
        a, b = q.chunk(2, -1)
        q = torch.cat([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], -1)
        lengths = st["prefix"].tolist()
        masks = st["tree"].reshape(s, n).tolist() if st["tree"] is not None else None
        for i in range(s):
            top = lengths[i] + n
            new = [[bool(masks[i][t] >> j & 1) if masks else j <= t for j in range(n)] for t in range(n)]
            allow = torch.ones(n, top, dtype=torch.bool, device=DEV)
            allow[:, lengths[i]:] = torch.tensor(new, device=DEV)
            for h in range(kvh):
                kk = _exact_values(st["kc"][i, h, :top], st["kp"][i, h, :top], False)
                vv = _exact_values(st["vc"][i, h, :top], st["vp"][i, h, :top], True)
                w = torch.einsum("trd,jd->trj", q[i, :, h * rep:(h + 1) * rep], kk) / math.sqrt(d)
                w = torch.softmax(w.masked_fill(~allow[:, None], -torch.inf), -1)
                out[i, :, h * rep:(h + 1) * rep] = torch.einsum("trj,jd->trd", w, vv)
        return out.reshape(s * n, heads * d)
    return _exact_accept(st)


def _exact_values(codes, par, value):
    """The values of packed rows [t, d / 2], block by block, in float64."""
    t, d = codes.shape[0], codes.shape[1] * 2
    out = torch.empty(t, d, dtype=torch.float64, device=DEV)
    place = _word_of_block(d, value).tolist()
    for b in range(d // 8):
        for i in range(8):
            byte = codes[:, 4 * place[b] + i // 2]
            code = (byte >> 4 if i % 2 else byte & 15).double()
            out[:, 8 * b + i] = par[:, b // 8, 1].double() + par[:, b // 8, 0].double() * code
    return out


def _exact_accept(st):
    case = st["case"]
    kept, drawn = [], []
    for i in range(case["s"]):
        count = case["k"] if st["count"] is None else int(st["count"][i])
        a = 0
        while a < count:
            p = torch.softmax(st["target"][i, a].double() / case["temperature"], -1)
            q = torch.softmax(st["draft"][i, a].double() / case["temperature"], -1)
            tok = st["tokens"][i, a]
            if not float(st["u"][i, a]) < min(1.0, float(p[tok]) / max(float(q[tok]), 1e-10)):
                break
            a += 1
        rest = torch.softmax(st["target"][i, a].double() / case["temperature"], -1)
        if a < count:
            over = (rest - torch.softmax(st["draft"][i, a].double() / case["temperature"], -1)).clamp_min(0)
            rest = over if bool((over > 0).any()) else rest
        kept.append(a)
        drawn.append(int((rest / st["e"][i].double()).argmax()))
    return torch.tensor(kept, device=DEV), torch.tensor(drawn, device=DEV)


# ---- what a pass cannot do without ------------------------------------------------------------------------


def work(case):
    op, es = case["op"], 4 if case["dtype"] == "float32" else 2
    if op == "int8":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * es + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * es, "flops": 2 * m * k * n}
    if op == "append":
        rows, d = case["s"] * case["n"], case["d"]
        one = rows * case["kvh"] * d
        # keys and values in, the rotation's table, the stored rows, and the values read back
        return {"bytes": 2 * one * es + rows * d * 4 + 2 * one // 2 + 2 * one // GROUP * 4 + 2 * one * 4,
                "flops": 2 * one * 8}
    if op == "attn":
        s, n, heads, kvh, d = case["s"], case["n"], case["heads"], case["kvh"], case["d"]
        # sequences of different lengths: the mean of _lengths' distribution
        length = case["prefix"] * (1 + (s - 1) * 0.625) / s + n
        cached = s * length * kvh * (d + d // GROUP * 8)
        return {"bytes": int(cached + 2 * s * n * heads * d * es + s * n * d * 4),
                "flops": int(4 * s * n * heads * length * d)}
    s, k, v = case["s"], case["k"], case["v"]
    rows = s * (2 * (k / 2 if case["ragged"] else k) + 1)  # ragged: half the drafts on the mean
    return {"bytes": int(rows * v * es + s * v * 4), "flops": int(rows * v * 4)}

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


class _Stand:
    """A stand-in for a BatchDecoder on the CPU: the next token is a function of the sequence and of the last two
    tokens in its cache; ``off``: sequences whose tokens it gets wrong."""

    def __init__(self, S, max_seq, prompt, off=()):
        import types

        import torch

        self.S, self.max_seq, self.device = S, max_seq, torch.device("cpu")
        self.dec = types.SimpleNamespace(shape=types.SimpleNamespace(vocab_size=16))
        self.cache = torch.full((S, max_seq), -1, dtype=torch.int64)
        self.cache[:, :prompt.shape[1]] = prompt
        self.off = off

    @staticmethod
    def following(s, before, last):
        return (3 * before + 5 * last + s) % 16

    def logits(self, tokens, start_seq, max_start, n, head=None):
        import torch

        if max_start + n > self.max_seq:
            raise RuntimeError(f"KV cache full: {max_start}+{n} > {self.max_seq}")
        assert int(start_seq.min()) >= 0 and int(start_seq.max()) <= max_start
        out = torch.zeros(self.S, n, 16)
        for s in range(self.S):
            p = int(start_seq[s])
            self.cache[s, p:p + n] = tokens.view(self.S, n)[s]
            assert (self.cache[s, :p + n] >= 0).all()
            for i in range(n):
                if p + i:
                    t = self.following(s, int(self.cache[s, p + i - 1]), int(self.cache[s, p + i]))
                    out[s, i, (t + (s in self.off)) % 16] = 1.0
        return out.view(self.S * n, 16)


def _accept_on_the_cpu(tokens, target, draft, u, e, temperature, n_draft=None):
    import torch

    from oracle import lowbit as olow

    S, k1, _ = target.shape
    got = [olow.accept_sampled([] if tokens is None else tokens[s].numpy(), target[s].numpy(),
                               None if draft is None else draft[s].numpy(), [] if u is None else u[s].numpy(),
                               e[s].double().numpy(), temperature, k1 - 1)[:2] for s in range(S)]
    a, b = zip(*got)
    return torch.tensor(a), torch.tensor(b)


@pytest.mark.parametrize("gamma", [1, 3, 5])
@pytest.mark.parametrize("max_new", [0, 1, 12])
def test_sampled_loop_stays_within_the_cache_that_its_tokens_need(monkeypatch, gamma, max_new):
    """One sequence accepts every draft and another none: the fast one waits, and start + max_new + gamma slots do."""
    import torch

    from littlebit_b200 import batch_decode as bd

    monkeypatch.setattr(bd, "accept_sampled", _accept_on_the_cpu)
    S, start = 3, 5
    prompt = torch.randint(0, 16, (S, start + 1), generator=torch.Generator().manual_seed(gamma))
    tgt = _Stand(S, start + max_new + gamma, prompt[:, :start])
    drf = _Stand(S, start + max_new + gamma, prompt[:, :start], off=(1,))
    out, stats = bd.sampled_speculative_generate(drf, tgt, prompt[:, start - 1], prompt[:, start], start, max_new, gamma=gamma,
                                                 temperature=0.0)
    assert out.shape == (S, max_new)
    for s in range(S):
        a, b = prompt[s, start - 1:].tolist()
        for i in range(max_new):
            a, b = b, _Stand.following(s, a, b)
            assert int(out[s, i]) == b, (s, i)
    assert stats["num_steps"] == max_new  # (the sequence without accepted drafts: a token a step)
    fast = -(-max_new // (gamma + 1))
    assert stats["total_accepted_tokens"] == 2 * fast * gamma
    if max_new:
        assert stats["acceptance_rate"] == 2 * fast / (2 * fast + max_new)


def test_sampled_loop_refusals():
    import torch

    from littlebit_b200 import batch_decode as bd

    prompt = torch.zeros(1, 4, dtype=torch.int64)
    m = _Stand(1, 32, prompt)
    for kw in (dict(gamma=0), dict(max_new=-1), dict(start=0)):
        a = dict(start=4, max_new=3, gamma=2) | kw
        with pytest.raises(ValueError):
            bd.sampled_speculative_generate(m, m, prompt[:, 2], prompt[:, 3], a["start"], a["max_new"], gamma=a["gamma"])

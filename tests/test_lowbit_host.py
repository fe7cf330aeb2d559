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


def _scratch_on_the_cpu(monkeypatch):
    import torch

    from littlebit_b200 import ops

    plain = ops.Workspace.__init__
    monkeypatch.setattr(ops.Workspace, "__init__", lambda self, device: plain(self, torch.device("cpu")))
    monkeypatch.setattr(ops, "_SCRATCH", {})
    monkeypatch.setattr(ops, "_capturing", lambda: False)
    return ops


def test_threads_on_one_stream_take_turns_at_its_scratch(monkeypatch):
    """A call's launches stay together: while one thread has the scratch no other thread's call of the operator on
    that stream may enqueue; calls on other streams, and other operators', may."""
    import threading
    import time

    ops = _scratch_on_the_cpu(monkeypatch)
    inside, most, bufs = {}, {}, {}
    note = threading.Lock()

    def call(tag, stream, nbytes):
        for i in range(20):
            sc = ops._stream_ws(0, tag, stream)
            with sc.lock:
                assert sc.take(nbytes + i).numel() >= nbytes + i
                with note:
                    inside[tag, stream] = inside.get((tag, stream), 0) + 1
                    most[tag, stream] = max(most.get((tag, stream), 0), inside[tag, stream])
                    most["all"] = max(most.get("all", 0), sum(inside.values()))
                    bufs.setdefault((tag, stream), set()).add(id(sc))
                time.sleep(0.0005)  # (the C call: other threads run)
                with note:
                    inside[tag, stream] -= 1

    ts = [threading.Thread(target=call, args=a) for a in (("int8", 7, 64), ("int8", 7, 64), ("int8", 7, 640),
                                                          ("int8", 8, 64), ("kv4", 7, 64))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert most["int8", 7] == 1 and most["all"] > 1
    assert len(bufs["int8", 7]) == 1 and len(set.union(*bufs.values())) == 3
    assert all(v == 0 for v in inside.values())


class _Watch:
    """Stands in for the C library: notes calls that overlap in one scratch."""

    def __init__(self):
        import threading

        self.note, self.now, self.clash = threading.Lock(), {}, 0

    def lbx_linear_int8_workspace_size(self, m, n, k):
        return 8192

    def lbx_kv4_attn_workspace_size(self, a):
        return 8192

    def _call(self, ws):
        import time

        with self.note:
            self.clash += self.now.get(ws, 0) > 0
            self.now[ws] = self.now.get(ws, 0) + 1
        time.sleep(0.001)
        with self.note:
            self.now[ws] -= 1
        return 0

    def lbx_linear_int8(self, a, ws, nbytes, stream):
        return self._call(ws)

    def lbx_kv4_attn(self, a, ws, nbytes, stream):
        return self._call(ws)


@pytest.mark.parametrize("op", ["linear_int8", "attention_kv4"])
def test_calls_of_two_threads_do_not_overlap_in_their_scratch(monkeypatch, op):
    """The public entries, their library and device replaced, on tensors of the CPU that pass for the GPU's."""
    import threading
    import types

    import torch

    ops = _scratch_on_the_cpu(monkeypatch)
    watch = _Watch()
    monkeypatch.setattr(ops, "lib", lambda: watch)
    monkeypatch.setattr(ops, "_rows", lambda name, t, dtypes=None: t)
    scratch = ops._stream_ws
    monkeypatch.setattr(ops, "_stream_ws", lambda index, *a: scratch(0, *a))  # (a tensor of the CPU is on device -1)

    class On:
        def __init__(self, index):
            pass

        def __enter__(self):
            return 7

        def __exit__(self, *exc):
            pass

    monkeypatch.setattr(ops, "_on", On)
    cache = types.SimpleNamespace(struct=lambda: L.Kv4Cache(256, 256, 256, 256, 1, 1, 64, 64), index=-1)
    x, w, s = torch.zeros(2, 64), torch.zeros(16, 64, dtype=torch.int8), torch.ones(16)

    def work():
        for _ in range(20):
            if op == "linear_int8":
                ops.linear_int8(x, w, s)
            else:
                ops.attention_kv4(x, cache, 0, None, 1, 0.1)

    ts = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert watch.clash == 0 and sum(watch.now.values()) == 0 and len(watch.now) == 1


def test_scratch_is_given_up_after_an_error(monkeypatch):
    import threading

    ops = _scratch_on_the_cpu(monkeypatch)
    for _ in range(2):
        sc = ops._stream_ws(0, "int8", 1)
        with pytest.raises(RuntimeError, match="invalid argument"):
            with sc.lock:
                sc.take(64)
                L.check(L.load().lbx_linear_int8(None, None, 0, None), "linear_int8")
    got = []
    t = threading.Thread(target=lambda: got.append(sc.lock.acquire(blocking=False)))
    t.start()
    t.join()
    assert got == [True] and sc.get(64).numel() >= 64


def test_eight_bit_codes_of_rows_that_nearly_vanish():
    """127 / a is no float32 below a = 3.74e-37: codes 0, never another sign."""
    import numpy as np

    from oracle import lowbit as olow

    x = np.array([[1, -1, 0.5]], np.float32)
    for top, want in ((1e-45, 0), (1e-38, 0), (3.7e-37, 0), (3.8e-37, 127), (1e-30, 127)):
        q, s = olow.quantize_tokens((x * np.float32(top)).astype(np.float32))
        assert q[0, :2].tolist() == [want, -want] and 0 <= s[0] < 1e-32


def test_sizes_that_32_bits_do_not_hold_are_refused():
    """Indexes of the kernels are 32-bit within a row, a tile or a cache's slots: sizes so near 2^31 that a
    step past the end would wrap are refused by the host."""
    lib, top = L.load(), (1 << 31) - 1
    for m, n, k in ((top, 1, 16), (1, top, 16), (top - 300, 64, 64), (1, 64, top)):
        assert lib.lbx_linear_int8_workspace_size(m, n, k) == 0, (m, n, k)
        a = L.Int8Args(m, n, k, 0, 0, 0, 256, k, 256, -(-k // 16) * 16, 256, None, 256, n)
        assert lib.lbx_linear_int8(ctypes.byref(a), 256, 1 << 62, None) == L.LBX_EUNSUPPORTED
    assert lib.lbx_linear_int8_workspace_size((1 << 30), 1, 16) > 1 << 34
    assert lib.lbx_quant_tokens(256, 0, top, 1, top, 256, top, 256, None) == L.LBX_EUNSUPPORTED
    s = L.AcceptArgs(n_seq=1, k=0, vocab=top, temperature=1.0, target=256, target_seq=0, target_row=0, e=256, accepted=256,
                     next=256)
    assert lib.lbx_accept_sampled(ctypes.byref(s), None) == L.LBX_EUNSUPPORTED
    c = L.Kv4Cache(256, 256, 256, 256, 1, 1, (1 << 31) - 64, 64)
    t = L.Kv4AttnArgs(cache=c, n=1, heads=1, max_prefix=0, q=256, q_ld=64, out=256, scale=1.0)
    assert lib.lbx_kv4_attn_workspace_size(ctypes.byref(t)) == 0
    assert lib.lbx_kv4_attn(ctypes.byref(t), 256, 1 << 62, None) == L.LBX_EUNSUPPORTED

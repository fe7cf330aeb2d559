"""Multi-sequence decoding on one GPU: many independent requests per step.

The reference decodes one sequence per process (cpu_draft_model.py,
cpu_target_model.py); batching requests is how a GPU amortises the
packed-weight read of every projection over many tokens.  ``BatchDecoder``
runs S independent sequences through one decoder step per token
(lbx_forward_multi): the linear calls see S (or S x n) tokens, attention keeps
a KV cache per sequence, and every sequence's results are bit-identical to
decoding it alone (the kernels are batch-invariant), so

  * ``greedy_generate`` gives each sequence the tokens of its own
    target-only greedy run (speculative_decoding.py:401-451), and
  * ``speculative_generate`` (chain drafting, greedy acceptance of
    speculative_decoding.py:315-330 and the bonus token of :356-363, per
    sequence, on the device) gives the same tokens again.

Sequences advance in lockstep by steps, not by tokens: after a speculative
step each sequence has accepted its own number of drafts, and its next slot
is kept on the device (start_seq).

``sampled_speculative_generate`` is the sampling counterpart (drafts sampled from
the draft, accepted and continued by speculative_decoding.py:331-363's rule), with
what such a step still reads in wide types made narrow: the caches may be held in 4
bits (``kv_bits=4``), the lm_heads as 8-bit integers (``ops.Int8Linear``), and sampling
and verification are one kernel each.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence

import torch

from . import _lib as L
from .model import LittleBitDecoder, cache_slots
from .ops import Int8Linear, Kv4Cache, _p, _stream, accept_sampled, kv4_append, lib


class BatchDecoder:
    """S sequences over one LittleBitDecoder's weights, with their own KV caches
    ([S, kv_heads, max_seq, head_dim] bf16 per layer, or ops.Kv4Cache with ``kv_bits=4``:
    head_dim 64 or 128, max_seq rounded up to a multiple of 64)."""

    def __init__(self, dec: LittleBitDecoder, n_seq: int, max_seq: int, kv_bits: int = 16):
        if not 1 <= n_seq <= 64:
            raise ValueError("1..64 sequences per batch decoder")
        if kv_bits not in (4, 16):
            raise ValueError("kv_bits must be 4 or 16")
        self.dec, self.S, self.max_seq, self.kv_bits = dec, int(n_seq), cache_slots(max_seq, kv_bits), kv_bits
        s = dec.shape
        dev = dec.device
        self.device = dev
        kvs = (self.S, s.num_key_value_heads, self.max_seq, s.head_dim)
        self.k_cache, self.v_cache, self.kv4 = [], [], []
        if kv_bits == 4:
            self.kv4 = [Kv4Cache.empty(*kvs, dev) for _ in dec.layers]
        else:
            self.k_cache = [torch.zeros(kvs, dtype=torch.bfloat16, device=dev) for _ in dec.layers]
            self.v_cache = [torch.zeros(kvs, dtype=torch.bfloat16, device=dev) for _ in dec.layers]
        self.stride = s.num_key_value_heads * self.max_seq * s.head_dim
        # the decoder's descriptors with this batch's caches and length
        self._layer_arr = (L.Layer * len(dec.layers))()
        for i in range(len(dec.layers)):
            self._layer_arr[i] = dec._layer_arr[i]
            self._layer_arr[i].k_cache = None if self.kv4 else _p(self.k_cache[i])
            self._layer_arr[i].v_cache = None if self.kv4 else _p(self.v_cache[i])
        m = L.Model()
        ctypes.pointer(m)[0] = dec._model
        m.max_seq = self.max_seq
        m.exec_mode = L.LBX_EXEC_KERNELS
        m.layers = ctypes.cast(self._layer_arr, ctypes.POINTER(L.Layer))
        m.kv4 = None
        if self.kv4:
            self._kv4_arr = (L.Kv4Cache * len(self.kv4))(*[c.struct() for c in self.kv4])
            m.kv4 = ctypes.cast(self._kv4_arr, ctypes.POINTER(L.Kv4Cache))
        self._model = m
        self._ws = {}

    def workspace(self, n: int) -> torch.Tensor:
        if n not in self._ws:
            need = int(lib().lbx_forward_multi_workspace_size(ctypes.byref(self._model), self.S, n))
            if need == 0:
                raise RuntimeError(f"multi-sequence step of {self.S} x {n} tokens unsupported")
            self._ws[n] = torch.zeros(need, dtype=torch.uint8, device=self.device)
        return self._ws[n]

    def step(self, tokens: torch.Tensor, start_seq: torch.Tensor, max_start: int, n: int, *,
             argmax: Optional[torch.Tensor] = None, logits: Optional[torch.Tensor] = None,
             hidden: Optional[torch.Tensor] = None) -> None:
        """n tokens of every sequence (device int64 [S*n], sequence by sequence) at
        slots start_seq[s] .. start_seq[s]+n-1 (device int32 [S]; max_start bounds them).
        ``hidden`` [S*n, H] receives the final-RMSNorm output."""
        if max_start + n > self.max_seq:
            raise RuntimeError(f"KV cache full: {max_start}+{n} > {self.max_seq}")
        ws = self.workspace(n)
        L.check(lib().lbx_forward_multi(ctypes.byref(self._model), _p(tokens), self.S, n, int(max_start),
                                        _p(start_seq), self.stride, None, None, _p(hidden), _p(logits), _p(argmax),
                                        _p(ws), ws.numel(), _stream(self.device)), "lbx_forward_multi")

    def fill_synthetic_prefix(self, n_slots: int, seed: int, scale: float = 1.0) -> None:
        """Seeded random bf16 keys and values in slots [0, n_slots) of every
        sequence (a stand-in for a prompt prefill; the attention work per new
        token depends only on the cached length)."""
        g = torch.Generator(device=self.device).manual_seed(seed)
        for c in self.kv4:
            S, H, _, d = c.shape
            k, v = (scale * torch.randn(S * n_slots, H * d, generator=g, device=self.device) for _ in range(2))
            kv4_append(k, v, c, 0)
        for kc, vc in zip(self.k_cache, self.v_cache):
            for c in (kc, vc):
                c[:, :, :n_slots].copy_((scale * torch.randn(c[:, :, :n_slots].shape, generator=g,
                                                             device=self.device)).bfloat16())

    def copy_prefix_from(self, other: "BatchDecoder", n_slots: int) -> None:
        if self.kv_bits != other.kv_bits:
            raise ValueError("both caches must have the same kv_bits")
        mine, theirs = ([*d.k_cache, *d.v_cache, *(t for c in d.kv4 for t in (c.k_codes, c.k_params, c.v_codes, c.v_params))]
                        for d in (self, other))
        for a, b in zip(mine, theirs):
            a[:, :, :n_slots].copy_(b[:, :, :n_slots])

    def logits(self, tokens: torch.Tensor, start_seq: torch.Tensor, max_start: int, n: int,
               head: Optional[Int8Linear] = None) -> torch.Tensor:
        """Logits [S*n, vocab] float32 of a step, from the decoder's bf16 lm_head or from ``head``."""
        rows, s = self.S * n, self.dec.shape
        if head is None:
            out = torch.empty(rows, s.vocab_size, dtype=torch.float32, device=self.device)
            self.step(tokens, start_seq, max_start, n, logits=out)
            return out
        hid = torch.empty(rows, s.hidden_size, dtype=torch.float32, device=self.device)
        self.step(tokens, start_seq, max_start, n, hidden=hid)
        return head(hid)


def greedy_generate(tgt: BatchDecoder, last: torch.Tensor, start: int, max_new: int) -> torch.Tensor:
    """Target-only greedy decoding of S sequences whose caches hold slots
    [0, start) and whose next input token is last[s] (device int64 [S]).
    Returns the new tokens, device int64 [S, max_new]."""
    S, dev = tgt.S, tgt.device
    out = torch.empty(S, max_new, dtype=torch.int64, device=dev)
    tok = last.clone()
    st = torch.full((S,), start, dtype=torch.int32, device=dev)
    am = torch.empty(S, dtype=torch.int64, device=dev)
    for i in range(max_new):
        tgt.step(tok, st, start + i, 1, argmax=am)
        out[:, i] = am
        tok.copy_(am)
        st += 1
    return out


def speculative_generate(drf: BatchDecoder, tgt: BatchDecoder, prev: torch.Tensor, last: torch.Tensor,
                         start: int, max_new: int, gamma: int = 4):
    """Chain speculative decoding of S sequences in lockstep.

    Both models' caches hold slots [0, start) of every sequence; prev[s] is
    the token at slot start-1 and last[s] the next input token.  Each step:
    the draft re-feeds the previous token with the last one (a sequence whose
    drafts were all accepted has not fed its last draft; re-writing a slot
    with the same token writes the same bits) and greedy-drafts gamma tokens;
    the target verifies last + drafts (gamma + 1 tokens per sequence);
    acceptance and the bonus token are computed per sequence on the device.
    Returns (new tokens [S, max_new], stats)."""
    S, dev = tgt.S, tgt.device
    cap = max_new + gamma + 1
    out = torch.zeros(S, cap, dtype=torch.int64, device=dev)
    nacc = torch.zeros(S, dtype=torch.int64, device=dev)   # new tokens so far
    pos = torch.full((S,), start, dtype=torch.int32, device=dev)  # slot of `last`
    prev_t, last_t = prev.clone(), last.clone()
    ar = torch.arange(gamma + 1, device=dev)
    drafts = torch.empty(S, gamma + 1, dtype=torch.int64, device=dev)
    vtok = torch.empty(S, gamma + 1, dtype=torch.int64, device=dev)
    am = torch.empty(S * (gamma + 1), dtype=torch.int64, device=dev)
    two = torch.empty(S, 2, dtype=torch.int64, device=dev)
    am2 = torch.empty(S * 2, dtype=torch.int64, device=dev)
    dam = torch.empty(S, dtype=torch.int64, device=dev)
    steps, total_acc = 0, 0
    bound = start
    done = 0
    while done < max_new:
        # draft: [prev, last] at slots pos-1, pos, then gamma-1 single tokens
        two[:, 0], two[:, 1] = prev_t, last_t
        drf.step(two.reshape(-1), pos - 1, bound - 1, 2, argmax=am2)
        drafts[:, 0] = am2.view(S, 2)[:, 1]
        for i in range(1, gamma):
            drf.step(drafts[:, i - 1].contiguous(), pos + i, bound + i, 1, argmax=dam)
            drafts[:, i] = dam
        # verify: last + gamma drafts at slots pos .. pos+gamma
        vtok[:, 0] = last_t
        vtok[:, 1:] = drafts[:, :gamma]
        tgt.step(vtok.reshape(-1), pos, bound, gamma + 1, argmax=am)
        a = am.view(S, gamma + 1)
        match = (vtok[:, 1:] == a[:, :gamma]).to(torch.int64)
        m = torch.cumprod(match, dim=1).sum(dim=1)            # accepted drafts per sequence
        bonus = a.gather(1, m[:, None])[:, 0]
        # this step's tokens: the m accepted drafts, then the bonus; positions
        # past them are rewritten by later steps (or lie past max_new)
        cand = torch.cat([vtok[:, 1:], torch.zeros_like(vtok[:, :1])], dim=1)
        new = torch.where(ar[None, :] < m[:, None], cand, bonus[:, None])
        out.scatter_(1, (nacc[:, None] + ar[None, :]).clamp(max=cap - 1), new)
        # the new last token is the bonus; the token before it sits at slot pos + m
        prev_t = vtok.gather(1, m[:, None])[:, 0]
        last_t = bonus
        nacc += m + 1
        pos += (m + 1).to(torch.int32)
        steps += 1
        total_acc += int(m.sum())
        done = int(nacc.min())
        bound = start + int(nacc.max())
    stats = {"num_steps": steps, "total_accepted_tokens": total_acc,
             "acceptance_rate": total_acc / (steps * gamma * S),
             "mean_acceptance_length": total_acc / (steps * S) + 1.0}
    return out[:, :max_new], stats


def sampled_speculative_generate(drf: BatchDecoder, tgt: BatchDecoder, prev: torch.Tensor, last: torch.Tensor,
                                 start: int, max_new: int, gamma: int = 4, temperature: float = 1.0,
                                 generator: Optional[torch.Generator] = None, draft_head: Optional[Int8Linear] = None,
                                 target_head: Optional[Int8Linear] = None):
    """Sampled chain speculation of S sequences in lockstep (the arguments of
    :func:`speculative_generate`).

    Each step the draft samples gamma tokens d_i ~ q_i = softmax(draft / T), the target
    gives p_0 .. p_gamma in one batched step, and ``ops.accept_sampled`` keeps the drafts
    while u_i < min(1, p_i(d_i) / q_i(d_i)) and draws the token after them, so
    every sequence's tokens are distributed as the target's own samples.  At
    temperature 0 they are the target's greedy tokens.  ``draft_head`` /
    ``target_head``: 8-bit lm_heads used in place of the decoders' bf16 ones.
    A sequence that has its max_new tokens stands still until the others have theirs, so
    both caches need start + max_new + gamma slots.
    Returns (new tokens [S, max_new], stats over the steps that sequences needed)."""
    if gamma < 1 or max_new < 0 or start < 1:
        raise ValueError("gamma and start must be at least 1, max_new at least 0")
    S, dev, V = tgt.S, tgt.device, tgt.dec.shape.vocab_size
    cap = max_new + gamma + 1
    out = torch.zeros(S, cap, dtype=torch.int64, device=dev)
    nacc = torch.zeros(S, dtype=torch.int64, device=dev)
    pos = torch.full((S,), start, dtype=torch.int32, device=dev)  # slot of `last`
    prev_t, last_t = prev.clone(), last.clone()
    ar = torch.arange(gamma + 1, device=dev)
    vtok = torch.empty(S, gamma + 1, dtype=torch.int64, device=dev)
    dlog = torch.empty(S, gamma, V, dtype=torch.float32, device=dev)
    e = torch.empty(S, V, dtype=torch.float32, device=dev)
    tiny = torch.finfo(torch.float32).tiny

    def noise():  # exponentially distributed, never 0
        return e.exponential_(generator=generator).clamp_(min=tiny)

    counts = torch.zeros(2, dtype=torch.int64, device=dev)  # accepted drafts, steps of unfinished sequences
    steps = done = 0
    bound = start
    while done < max_new:
        # draft: [prev, last] at slots pos-1, pos (a sequence whose drafts were all accepted has
        # not fed its last one), then single tokens
        lg = drf.logits(torch.stack([prev_t, last_t], 1).reshape(-1), pos - 1, bound - 1, 2, draft_head)
        dlog[:, 0] = lg.view(S, 2, V)[:, 1]
        vtok[:, 0] = last_t
        for i in range(gamma):
            vtok[:, i + 1] = accept_sampled(None, dlog[:, i:i + 1], None, None, noise(), temperature)[1]
            if i + 1 < gamma:
                dlog[:, i + 1] = drf.logits(vtok[:, i + 1].contiguous(), pos + (i + 1), bound + i + 1, 1, draft_head)
        tlog = tgt.logits(vtok.reshape(-1), pos, bound, gamma + 1, target_head).view(S, gamma + 1, V)
        u = torch.rand(S, gamma, generator=generator, device=dev)
        m, nxt = accept_sampled(vtok[:, 1:], tlog, dlog, u, noise(), temperature)
        # this step's tokens: the m accepted drafts, then the drawn one; what lies
        # past them is rewritten by later steps (a finished sequence's lie past max_new)
        cand = torch.cat([vtok[:, 1:], nxt[:, None]], 1)
        new = torch.where(ar[None] < m[:, None], cand, nxt[:, None])
        out.scatter_(1, (nacc[:, None] + ar[None]).clamp(max=cap - 1), new)
        open_ = nacc < max_new
        counts += torch.stack([torch.where(open_, m, 0).sum(), open_.sum()])
        nacc = torch.where(open_, nacc + m + 1, nacc)
        # a sequence that is done feeds the same slots again: its place moves no further
        go = nacc < max_new
        prev_t = torch.where(go, vtok.gather(1, m[:, None])[:, 0], prev_t)
        last_t = torch.where(go, nxt, last_t)
        pos = torch.where(go, pos + (m + 1).to(torch.int32), pos)
        steps += 1
        done, most = torch.stack([nacc.min(), pos.max()]).tolist()
        bound = int(most)
    accepted, needed = counts.tolist()
    stats = {"num_steps": steps, "total_accepted_tokens": accepted,
             "acceptance_rate": accepted / max(1, needed * gamma),
             "mean_acceptance_length": accepted / max(1, needed) + 1.0}
    return out[:, :max_new], stats

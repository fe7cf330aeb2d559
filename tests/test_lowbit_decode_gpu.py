"""The low-bit operators in the decoding path: a decoder over a 4-bit cache is its own
operators one by one, bit for bit; batches and speculation over it keep the bits of
decoding alone; sampled speculation with 8-bit heads is greedy at temperature 0
and accepts every draft of a draft that is the target."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

TINY = dict(num_hidden_layers=2, hidden_size=256, intermediate_size=512, num_attention_heads=4,
            num_key_value_heads=2, vocab_size=512)
RANKS = {"q_proj": [64, 32], "k_proj": [32, 16], "v_proj": [32, 16], "o_proj": [64, 32],
         "gate_proj": [96, 40], "up_proj": [96, 40], "down_proj": [96, 40]}


def _state(seed=21):
    from littlebit_b200.model import DecoderShape, synthetic_runtime_state

    shape = DecoderShape(**TINY)
    st = synthetic_runtime_state(shape, RANKS, seed=seed, unit_gain=True)
    for k in list(st):
        if k.endswith(".u1_r"):
            st[k] = st[k] * 0.05
    return shape, st


@pytest.fixture(scope="module")
def dec():
    from littlebit_b200.model import LittleBitDecoder

    shape, st = _state()
    return LittleBitDecoder(shape, st, device=DEV, max_seq=150, kv_bits=4)


def _by_ops(dec, tokens, start, caches):
    """One step through the operators: final-RMSNorm output [n, H]."""
    from littlebit_b200 import _lib as L
    from littlebit_b200 import ops

    s, n = dec.shape, len(tokens)
    d, qd, kvd = s.head_dim, s.hidden_size, s.num_key_value_heads * s.head_dim
    x = ops.embedding_lookup(dec.embed, torch.tensor(tokens))
    cs = ops.rope_table(torch.arange(start, start + n, dtype=torch.int32, device=DEV), d, s.rope_theta)
    for ly, cache in zip(dec.layers, caches):
        q, k, v = (torch.empty(n, w, device=DEV) for w in (qd, kvd, kvd))
        ops.linear_group(ly["projs"][:3], x, [q, k, v], prologue=L.LBX_PRO_RMSNORM, norm_w=ly["ln1"], eps=s.rms_norm_eps)
        ops.kv4_append(k, v, cache, start, rope_cs=cs)
        att = ops.attention_kv4(q, cache, start, None, s.num_attention_heads, d ** -0.5, rope_cs=cs)
        ops.linear_group([ly["projs"][3]], att, [x], epilogue=L.LBX_EPI_ADD)
        g, u = (torch.empty(n, s.intermediate_size, device=DEV) for _ in range(2))
        ops.linear_group(ly["projs"][4:6], x, [g, u], prologue=L.LBX_PRO_RMSNORM, norm_w=ly["ln2"], eps=s.rms_norm_eps,
                         epilogue=L.LBX_EPI_SILU0)
        ops.linear_group([ly["projs"][6]], g, [x], prologue=L.LBX_PRO_MUL, x2=u, epilogue=L.LBX_EPI_ADD)
    return ops.rms_norm(x, dec.final_norm, s.rms_norm_eps)


def test_decoder_steps_are_their_operators(dec):
    from littlebit_b200 import ops

    s = dec.shape
    ids = torch.randint(0, s.vocab_size, (12,), generator=torch.Generator().manual_seed(1)).tolist()
    caches = [ops.Kv4Cache.empty(1, s.num_key_value_heads, 150, s.head_dim) for _ in dec.layers]
    assert caches[0].shape == (1, 2, 192, 64) and dec.max_seq == 192
    for a, b in ((0, 9), (9, 10), (10, 12)):
        got = dec.forward_tokens(ids[a:b], a, want_hidden=True)
        want = _by_ops(dec, ids[a:b], a, caches)
        assert torch.equal(got["hidden"], want), (a, b)
    for c, own in zip(caches, dec.kv4):
        assert torch.equal(c.k_codes[:, :, :12], own.k_codes[:, :, :12])
        assert torch.equal(c.v_codes[:, :, :12], own.v_codes[:, :, :12])


def test_long_prompt_equals_token_by_token(dec):
    ids = torch.randint(0, dec.shape.vocab_size, (100,), generator=torch.Generator().manual_seed(2)).tolist()
    run = dec.forward_tokens(ids, 0)["logits"]  # 64 + 36 tokens
    for i, t in enumerate(ids):
        one = dec.forward_tokens([t], i)["logits"]
        if i in (0, 1, 17, 63, 64, 99):
            assert torch.equal(one[0], run[i]), i


def test_four_bits_stay_near_sixteen(dec):
    """The cached values of one group are off by half a step at most, an eighth or so of a unit
    here, so the logits of 4-bit and bf16 caches agree to a few percent, and far better than chance."""
    from littlebit_b200.model import LittleBitDecoder

    shape, st = _state()
    full = LittleBitDecoder(shape, st, device=DEV, max_seq=150)
    ids = torch.randint(0, shape.vocab_size, (60,), generator=torch.Generator().manual_seed(3)).tolist()
    a, b = full.forward_tokens(ids, 0)["logits"], dec.forward_tokens(ids, 0)["logits"]
    rel = ((a - b).norm() / a.norm()).item()
    assert rel < 0.25 and rel > 0


def test_batched_sequences_keep_their_bits(dec):
    from littlebit_b200.batch_decode import BatchDecoder

    S, P, V = 3, 6, dec.shape.vocab_size
    prompts = torch.randint(0, V, (S, P + 2), generator=torch.Generator().manual_seed(5))
    bd = BatchDecoder(dec, S, max_seq=150, kv_bits=4)
    lg = bd.logits(prompts[:, :P].reshape(-1).to(DEV), torch.zeros(S, dtype=torch.int32, device=DEV), 0, P).view(S, P, V)
    st = torch.full((S,), P, dtype=torch.int32, device=DEV)
    l2 = bd.logits(prompts[:, P:].reshape(-1).to(DEV), st, P, 2).view(S, 2, V)
    for s in range(S):
        assert torch.equal(lg[s], dec.forward_tokens(prompts[s, :P].tolist(), 0)["logits"])
        assert torch.equal(l2[s], dec.forward_tokens(prompts[s, P:].tolist(), P)["logits"])


def _pair(dec, S, kv_bits, same=False):
    from littlebit_b200.batch_decode import BatchDecoder
    from littlebit_b200.cuda_models import _branch0_view

    draft = dec if same else _branch0_view(dec, 192)
    tgt = BatchDecoder(dec, S, max_seq=192, kv_bits=kv_bits)
    drf = BatchDecoder(draft, S, max_seq=192, kv_bits=kv_bits)
    ids = torch.randint(0, dec.shape.vocab_size, (S, 10), generator=torch.Generator().manual_seed(8)).to(DEV)
    z = torch.zeros(S, dtype=torch.int32, device=DEV)
    for b in (tgt, drf):
        b.logits(ids[:, :9].reshape(-1), z, 0, 9)
    return drf, tgt, ids


@pytest.mark.parametrize("kv_bits", [4, 16])
@pytest.mark.parametrize("S", [1, 5])
def test_sampled_speculation_at_temperature_zero_is_greedy(dec, S, kv_bits):
    from littlebit_b200 import ops
    from littlebit_b200.batch_decode import sampled_speculative_generate

    head = ops.Int8Linear.from_float(dec.lm_head)
    drf, tgt, ids = _pair(dec, S, kv_bits)
    toks, stats = sampled_speculative_generate(drf, tgt, ids[:, 8], ids[:, 9], 9, 20, gamma=3, temperature=0.0,
                                               draft_head=head, target_head=head)
    assert 0 < stats["acceptance_rate"] <= 1
    _, tgt, _ = _pair(dec, S, kv_bits)
    last, st = ids[:, 9].clone(), torch.full((S,), 9, dtype=torch.int32, device=DEV)
    for i in range(20):
        last = tgt.logits(last, st, 9 + i, 1, head).argmax(-1)
        assert torch.equal(toks[:, i], last), i
        st += 1


def test_a_draft_that_is_the_target_is_always_accepted(dec):
    from littlebit_b200 import ops
    from littlebit_b200.batch_decode import sampled_speculative_generate

    head = ops.Int8Linear.from_float(dec.lm_head)
    runs = []
    for _ in range(2):
        drf, tgt, ids = _pair(dec, 4, 4, same=True)
        g = torch.Generator(device=DEV).manual_seed(3)
        runs.append(sampled_speculative_generate(drf, tgt, ids[:, 8], ids[:, 9], 9, 24, gamma=4, temperature=0.8,
                                                 generator=g, draft_head=head, target_head=head))
    assert runs[0][1]["acceptance_rate"] == 1.0
    assert torch.equal(runs[0][0], runs[1][0])  # the same random numbers, the same tokens
    assert runs[0][0].unique().numel() > 8


def test_chain_speculation_over_four_bit_caches():
    from littlebit_b200.cuda_models import CudaDraftModel, CudaTargetModel
    from littlebit_b200.model import LittleBitDecoder
    from littlebit_b200.speculative_decoding import autoregressive_generate, speculative_decode

    shape, st = _state(7)
    d = LittleBitDecoder(shape, st, device=DEV, max_seq=512, kv_bits=4)
    tgt = CudaTargetModel.from_decoder(d)
    drf = CudaDraftModel.from_target(tgt)
    ids = torch.randint(0, shape.vocab_size, (1, 20), generator=torch.Generator().manual_seed(0)).to(DEV)
    ar, _ = autoregressive_generate(tgt, ids, None, max_new_tokens=32, eos_token_id=-1)
    sp, stats = speculative_decode(drf, tgt, ids, None, max_new_tokens=32, draft_length=4, eos_token_id=-1)
    assert sp.tolist() == ar.tolist() and stats["total_accepted_tokens"] > 0
    with pytest.raises(RuntimeError, match="bf16 cache"):
        tgt._units[0].kv_move(torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))


def test_refusals(dec):
    from littlebit_b200 import _lib as L
    from littlebit_b200.batch_decode import BatchDecoder
    from littlebit_b200.model import LittleBitDecoder

    shape, st = _state()
    with pytest.raises(ValueError):
        LittleBitDecoder(shape, st, device=DEV, kv_bits=8)
    with pytest.raises(ValueError):
        BatchDecoder(dec, 2, 64, kv_bits=2)
    p = LittleBitDecoder(shape, st, device=DEV, max_seq=64, kv_bits=4, exec_mode=L.LBX_EXEC_PROGRAM)
    with pytest.raises(RuntimeError, match="kernel path"):
        p.forward_tokens([1, 2], 0)
    bd = BatchDecoder(dec, 2, 64, kv_bits=4)
    with pytest.raises(RuntimeError, match="KV cache full"):
        bd.step(torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV), 64, 1)
    with pytest.raises(ValueError, match="kv_bits"):
        bd.copy_prefix_from(BatchDecoder(dec, 2, 64), 4)

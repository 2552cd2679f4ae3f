"""Rotary positions and packed causal attention: definitions, gradients and refusals on the CPU."""

import math

import pytest
import torch

from agentgarten_b200 import ops

import packed_oracle as oracle


def _offsets(lengths):
    return torch.tensor([0, *torch.tensor(lengths, dtype=torch.long).cumsum(0).tolist()], dtype=torch.int32)


# --------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotary_definition(interleaved, dtype):
    torch.manual_seed(0)
    q, k = torch.randn(11, 3, 10).to(dtype), torch.randn(11, 1, 10).to(dtype)
    positions = torch.tensor([0, 1, 2, 0, 5, 70000, 2 ** 24 + 1, 3, 3, 1, 9])
    f = ops.rotary_frequencies(6, 1e4)
    inverse = 1e4 ** (-torch.arange(3, dtype=torch.float64) / 3)
    torch.testing.assert_close(f.turns * 2 * math.pi, inverse, rtol=1e-14, atol=0)
    for got, x in zip(ops.rotary_embed(q, k, positions, f, interleaved=interleaved), (q, k)):
        oracle.assert_close(got, *oracle.rotary(x, positions, inverse, interleaved=interleaved))
        assert torch.equal(got[..., 6:], x[..., 6:])


def test_rotary_matches_the_towers_tables():
    """Half layout over a whole head with three axes: what the existing table + rotate-half gives."""
    from helpers import tiny_config
    from agentgarten_b200.networks.cosmos3.layers import Cosmos3RotaryEmbedding

    config = tiny_config()
    torch.manual_seed(1)
    positions = torch.rand(2, 9, 3) * 50
    q = torch.randn(2, 9, 4, 64)
    cos, sin = Cosmos3RotaryEmbedding(config)(positions, torch.float32)
    f = ops.rotary_frequencies(64, config.rope_theta, sections=config.mrope_section)
    got, none = ops.rotary_embed(q, None, positions, f)
    assert none is None
    # the tables hold FP32 angles up to 50: off by 50 * 2^-23 in the angle at most
    torch.testing.assert_close(got, ops.rotary(q, cos, sin), rtol=0, atol=50 * 2.0 ** -23 * 2 * q.abs().max().item())


def test_scaled_frequencies():
    plain = ops.rotary_frequencies(64, 5e6).turns
    assert torch.allclose(ops.rotary_frequencies(64, 5e6, scaling="linear", factor=4.0).turns, plain / 4)
    ntk = ops.rotary_frequencies(64, 5e6, scaling="ntk", factor=4.0).turns
    assert math.isclose(ntk[0], plain[0]) and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-12)
    yarn = ops.rotary_frequencies(64, 5e6, scaling="yarn", factor=4.0, trained_positions=4096)
    turns = plain * 4096
    assert torch.equal(yarn.turns[turns > 64], plain[turns > 64])
    assert torch.allclose(yarn.turns[turns < 0.25], plain[turns < 0.25] / 4)
    assert bool(((yarn.turns <= plain * (1 + 1e-12)) & (yarn.turns >= plain / 4 * (1 - 1e-12))).all())
    assert math.isclose(yarn.amplitude, 0.1 * math.log(4.0) + 1)
    assert torch.equal(ops.rotary_frequencies(64, 5e6, scaling="ntk", factor=1.0).turns, plain)


def test_rotary_gradient_is_the_turn_back():
    torch.manual_seed(2)
    q, k = (torch.randn(5, h, 8, dtype=torch.float64, requires_grad=True) for h in (2, 1))
    f = ops.rotary_frequencies(4, 100.0, scaling="yarn", factor=2.0, trained_positions=64)
    positions = torch.tensor([0.0, 0.5, 3.25, 7.0, 100.0])
    assert torch.autograd.gradcheck(lambda a, b: ops.rotary_embed(a, b, positions, f, interleaved=True), (q, k))


def test_rotary_refusals():
    f = ops.rotary_frequencies(8)
    q, k, at = torch.randn(4, 2, 8), torch.randn(4, 1, 8), torch.arange(4)
    with pytest.raises(ValueError, match="positions"):
        ops.rotary_embed(q, k, torch.arange(5), f)
    with pytest.raises(TypeError, match="int32"):
        ops.rotary_embed(q, k, at.to(torch.int16), f)
    with pytest.raises(ValueError, match="key"):
        ops.rotary_embed(q, k[:3], at, f)
    with pytest.raises(TypeError, match="key"):
        ops.rotary_embed(q, k.half(), at, f)
    with pytest.raises(ValueError, match="to turn"):
        ops.rotary_embed(q[..., :6], k[..., :6], at, f)
    with pytest.raises(ValueError, match="query"):
        ops.rotary_embed(q[0], None, at, f)
    with pytest.raises(ValueError, match="positions"):  # three axes wanted
        ops.rotary_embed(q, k, at, ops.rotary_frequencies(8, sections=(2, 1, 1)))
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="cubic"),
                dict(rotary_dim=8, scaling="yarn", factor=2.0), dict(rotary_dim=2, scaling="ntk", factor=2.0),
                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, theta=math.inf), dict(rotary_dim=8, sections=(1, 2))):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)


# ------------------------------------------------------------------------------------ attention
def _case(q_lengths, k_lengths, heads, kv_heads, dim, dtype, room=0, behind=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    rooms = [n + room for n in k_lengths]
    q = torch.randn(sum(q_lengths) + behind, heads, dim, generator=g).to(dtype)
    k, v = (torch.randn(sum(rooms) + behind, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    q_offsets, k_offsets = _offsets(q_lengths), _offsets(rooms)
    spans = list(zip(q_offsets.tolist(), q_lengths, k_offsets.tolist(), k_lengths))
    return q, k, v, q_offsets, k_offsets, torch.tensor(k_lengths, dtype=torch.int32), spans


@pytest.mark.parametrize("q_lengths,k_lengths", [([5], [5]), ([3, 0, 4], [3, 0, 4]), ([1, 1], [7, 1]), ([4, 2], [2, 0]),
                                                  ([0, 0], [3, 0])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_definition(q_lengths, k_lengths, dtype):
    q, k, v, qo, ko, kl, spans = _case(q_lengths, k_lengths, 4, 2, 16, dtype, room=2, behind=3)
    k[sum(k_lengths) + 2 * len(k_lengths):] = float("nan")   # rows of no sequence
    out = ops.packed_attention(q, k, v, qo, ko, k_lengths=kl)
    oracle.assert_close(out, *oracle.attention(q, k, v, spans, 0.25)["out"])
    assert not out[sum(q_lengths):].any()


def test_attention_gradients_on_the_cpu():
    q, k, v, qo, ko, kl, _ = _case([3, 2, 3], [3, 4, 1], 4, 2, 5, torch.float64, room=1, behind=1)
    for t in (q, k, v):
        t.requires_grad_()
    assert torch.autograd.gradcheck(lambda a, b, c: ops.packed_attention(a, b, c, qo, ko, k_lengths=kl, scale=0.7), (q, k, v))


def test_one_sequence_is_dense_causal_attention():
    torch.manual_seed(3)
    q, k, v = torch.randn(9, 4, 16), torch.randn(9, 2, 16), torch.randn(9, 2, 16)
    got = ops.packed_attention(q, k, v, _offsets([9]))
    want = ops.attention(q[None], k[None], v[None], causal=True)[0]
    torch.testing.assert_close(got, want, rtol=0, atol=1e-5)


def test_attention_refusals():
    q, k, v, qo, ko, kl, _ = _case([3, 2], [3, 4], 4, 2, 16, torch.float32)

    def call(**change):
        given = dict(query=q, key=k, value=v, q_offsets=qo, k_offsets=ko, k_lengths=kl, scale=None)
        given.update(change)
        return ops.packed_attention(**given)

    call()
    for change, error in ((dict(query=q[None]), ValueError), (dict(value=v[:-1]), ValueError),
                          (dict(key=k[:, :0], value=v[:, :0]), ValueError), (dict(query=q[:, :3]), ValueError),
                          (dict(key=k.double()), TypeError), (dict(query=q.long(), key=k.long(), value=v.long()), TypeError),
                          (dict(q_offsets=qo.long()), TypeError), (dict(q_offsets=qo[::2]), TypeError),
                          (dict(k_offsets=ko[:2]), ValueError), (dict(k_lengths=kl[:1]), ValueError),
                          (dict(q_offsets=qo[:0], k_offsets=ko[:0]), ValueError), (dict(scale=0.0), ValueError),
                          (dict(scale=math.nan), ValueError), (dict(k_offsets=None, k_lengths=None), ValueError)):
        with pytest.raises(error, match="packed_attention"):
            call(**change)
    for bad in ([1, 3, 5], [0, 4, 3], [0, 3, 6]):  # does not start at 0, falls, leaves the tensor
        with pytest.raises(ValueError, match="offsets"):
            call(q_offsets=torch.tensor(bad, dtype=torch.int32))
    with pytest.raises(ValueError, match="offsets"):
        call(k_lengths=torch.tensor([4, 4], dtype=torch.int32))


# ------------------------------------------------------------------------------- the text tower
def _prompts():
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(3, 128, (3, 12), generator=g)
    valid = torch.arange(12)[None] < torch.tensor([12, 3, 7])[:, None]
    return ids, valid


def test_packed_prompts_give_the_text_towers_context():
    from helpers import tiny_conditioner

    encoder = tiny_conditioner().text_encoder.double()
    ids, valid = _prompts()
    padded, packed = encoder(ids, valid), encoder.encode_packed(ids, valid)
    assert packed.lengths == padded.lengths and torch.equal(packed.valid_lengths, padded.valid_lengths)
    for mine, theirs in zip((*packed.keys, *packed.values), (*padded.keys, *padded.values)):
        assert mine.shape == theirs.shape
        for row, (a, b) in enumerate(zip(mine, theirs)):
            n = packed.lengths[row]
            # the padded tower's angles are FP32: off by 14 * 2^-24 at the last position, in values of
            # order 1 and through two layers
            torch.testing.assert_close(a[:n], b[:n], rtol=0, atol=14 * 2.0 ** -24 * 16)
            assert not a[n:].any()


def test_packed_prompts_train_the_text_tower():
    from helpers import tiny_conditioner

    encoder = tiny_conditioner().text_encoder.double()
    encoder.requires_grad_(True)
    ids, valid = _prompts()
    weights = [layer.self_attn.to_k.weight for layer in encoder.layers] + [encoder.embed_tokens.weight]

    def value():
        context = encoder.encode_packed(ids, valid, scaling="yarn", factor=2.0, trained_positions=64)
        return sum((t * t.detach().sign()).sum() for t in (*context.keys, *context.values))

    grads = torch.autograd.grad(value(), weights)
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        steps = [torch.randn(w.shape, generator=g, dtype=w.dtype) for w in weights]
        slope = sum((a * b).sum() for a, b in zip(grads, steps))
        h = 1e-7
        ends = []
        for sign in (1, -2):
            for w, s in zip(weights, steps):
                w += sign * h * s
            ends.append(value())
    # differences of a smooth function: h^2 terms and 2^-53 of its size over h
    assert abs((ends[0] - ends[1]) / (2 * h) - slope) < 1e-4 * abs(slope) + 1e-9 / h * 2.0 ** -20 * abs(ends[0])


def test_conditioner_packs_prompts_when_asked():
    from helpers import synthetic_batch, tiny_conditioner

    conditioner = tiny_conditioner()
    batch = conditioner.encode(synthetic_batch(batch=2), training=False)
    plain = conditioner.condition(batch).text
    conditioner.pack_prompts = True
    packed = conditioner.condition(batch).text
    assert packed.lengths == plain.lengths
    for a, b in zip(packed.keys, plain.keys):
        n = packed.lengths[0]
        torch.testing.assert_close(a[:, :n], b[:, :n], rtol=0, atol=1e-4)
    conditioner.cache_text_contexts = True
    again = conditioner.condition(batch).text
    assert conditioner.condition(batch).text is again
    conditioner.pack_prompts = False
    assert conditioner.condition(batch).text is not again

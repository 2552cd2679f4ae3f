"""Rotary positions and packed causal attention on the kernels, against 64-bit definitions."""

import math

import pytest
import torch

from agentgarten_b200 import ops
from agentgarten_b200.ops import native

import packed_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _status():
    torch.cuda.synchronize()
    return int(native.ext().status(torch.cuda.current_device()).item())


# --------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", [BF16, FP16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,turned", [
    (1, 32, 8, 128, 128), (3, 4, 2, 64, 32), (37, 3, 1, 80, 20), (130, 5, 5, 96, 96), (9, 2, 2, 6, 2),
    (1000, 32, 8, 128, 64), (5, 1, 1, 256, 128), (2, 3, 1, 7, 4)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(dtype, tokens, heads, kv_heads, dim, turned, interleaved):
    g = torch.Generator(device=DEV).manual_seed(tokens)
    q, k = (torch.randn(tokens, h, dim, device=DEV, generator=g).to(dtype) for h in (heads, kv_heads))
    positions = torch.randint(0, 1 << 20, (tokens,), device=DEV, generator=g)
    f = ops.rotary_frequencies(turned, 5e6, scaling="yarn", factor=8.0, trained_positions=4096, device=DEV)
    before = native.launches()
    got = ops.rotary_embed(q, k, positions, f, interleaved=interleaved)
    assert native.launches() == before + 1
    for out, x in zip(got, (q, k)):
        oracle.assert_close(out, *oracle.rotary(x, positions, f.turns * 2 * math.pi, f.amplitude, interleaved=interleaved))
        assert torch.equal(out[..., turned:], x[..., turned:])


def test_rotary_positions_of_every_type_and_axes():
    g = torch.Generator(device=DEV).manual_seed(5)
    q = torch.randn(2, 50, 4, 128, device=DEV, generator=g).bfloat16()
    k = torch.randn(2, 50, 2, 128, device=DEV, generator=g).bfloat16()
    inverse = ops.rotary_frequencies(128, 5e6, device=DEV).turns * 2 * math.pi
    whole = torch.randint(0, 1 << 30, (2, 50), device=DEV, generator=g)
    f = ops.rotary_frequencies(128, 5e6, device=DEV)
    for positions in (whole, whole.int(), -whole, whole + (1 << 40), whole.float() / 3):
        for out, x in zip(ops.rotary_embed(q, k, positions, f), (q, k)):
            # 2^40 positions are 2^38 turns: the fraction is exact to 2^-15 of a turn in 64 bits
            extra = 2 * math.pi * 2.0 ** -15 * 2 if int(positions.abs().max()) > 1 << 31 else 0.0
            value, bound = oracle.rotary(x, positions, inverse)
            oracle.assert_close(out, value, bound + extra * x.double().abs().amax())
    f = ops.rotary_frequencies(128, 5e6, sections=(24, 20, 20), device=DEV)
    positions = torch.rand(2, 50, 3, device=DEV, generator=g) * 20000
    for out, x in zip(ops.rotary_embed(q, k, positions, f), (q, k)):
        oracle.assert_close(out, *oracle.rotary(x, positions, inverse, axis=f.axis))


def test_rotary_strides():
    """Column slices of a joint projection, transposed heads, odd alignments: read in place or copied."""
    g = torch.Generator(device=DEV).manual_seed(6)
    joint = torch.randn(33, 6 * 64 + 4, device=DEV, generator=g).bfloat16()
    positions = torch.arange(33, device=DEV)
    f = ops.rotary_frequencies(64, 1e4, device=DEV)
    inverse = f.turns * 2 * math.pi
    for shift in (0, 1, 2, 4):
        q = joint[:, shift:shift + 256].unflatten(-1, (4, 64))
        k = joint[:, 256:384].unflatten(-1, (2, 64)).transpose(0, 1).contiguous().transpose(0, 1)
        for out, x in zip(ops.rotary_embed(q, k, positions, f), (q, k)):
            assert out.is_contiguous()
            oracle.assert_close(out, *oracle.rotary(x, positions, inverse))
    x = torch.randn(33, 1, 64, device=DEV, generator=g).expand(33, 3, 64)
    oracle.assert_close(ops.rotary_embed(x, None, positions, f)[0], *oracle.rotary(x, positions, inverse))
    x = torch.randn(4, 6, 2, 64, device=DEV, generator=g)[::2, ::3]
    at = torch.arange(4, device=DEV).view(2, 2)
    oracle.assert_close(ops.rotary_embed(x, None, at, f)[0], *oracle.rotary(x, at, inverse))
    x = torch.randn(4, 1, 2, 64, device=DEV, generator=g).expand(4, 3, 2, 64)
    at = torch.arange(12, device=DEV).view(4, 3)
    oracle.assert_close(ops.rotary_embed(x, None, at, f)[0], *oracle.rotary(x, at, inverse))
    empty = torch.randn(0, 4, 64, device=DEV)
    assert ops.rotary_embed(empty, empty, positions[:0], f)[1].shape == empty.shape


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradients(dtype, interleaved):
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, gq, gk = (torch.randn(21, h, 64, device=DEV, generator=g).to(dtype) for h in (4, 2, 4, 2))
    f = ops.rotary_frequencies(32, 1e4, scaling="yarn", factor=4.0, trained_positions=64, device=DEV)
    inverse, at = f.turns * 2 * math.pi, torch.arange(21, device=DEV)
    q.requires_grad_()
    k.requires_grad_()
    out = ops.rotary_embed(q, k, at, f, interleaved=interleaved)
    for got, x in zip(torch.autograd.grad(out, (q, k), (gq, gk), retain_graph=True), (gq, gk)):
        oracle.assert_close(got, *oracle.rotary(x, at, -inverse, f.amplitude, interleaved=interleaved))
    # only one output used, and a broadcast gradient
    (got,) = torch.autograd.grad(out[1].sum(), (k,))
    oracle.assert_close(got, *oracle.rotary(torch.ones_like(k), at, -inverse, f.amplitude, interleaved=interleaved))


def test_rotary_refusals():
    q, k, at = torch.randn(4, 2, 64, device=DEV), torch.randn(4, 1, 64, device=DEV), torch.arange(4, device=DEV)
    f = ops.rotary_frequencies(64, device=DEV)
    ops.rotary_embed(q, k, at, f)
    for args, error in (((q, k, at[:3], f), ValueError), ((q, k, at.short(), f), TypeError), ((q, k[:3], at, f), ValueError),
                        ((q, k.half(), at, f), TypeError), ((q[..., :32], k[..., :32], at, f), ValueError),
                        ((q[0], None, at, f), ValueError), ((q, k[:, :0], at, f), ValueError), ((q.int(), None, at, f), TypeError),
                        ((q, k, at, ops.rotary_frequencies(64, sections=(12, 10, 10), device=DEV)), ValueError)):
        with pytest.raises(error, match="rotary_embed"):
            ops.rotary_embed(*args)
    with pytest.raises(ValueError, match="one device"):
        ops.rotary_embed(q, None, torch.arange(4), f)
    with pytest.raises(ValueError, match="one device"):
        ops.rotary_embed(q, None, torch.arange(4, device=DEV), ops.rotary_frequencies(64))
    with pytest.raises(TypeError):
        ops.rotary_embed(q.to(torch.float8_e4m3fn), None, torch.arange(4, device=DEV), f)


# ------------------------------------------------------------------------------------ attention
def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def _case(q_lengths, k_lengths, heads, kv_heads, dim, dtype, room=0, behind=0, seed=0, stale=float("nan")):
    """Packed tensors; key rows that are no keys (room behind a sequence, rows behind the last) hold ``stale``."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rooms = [n + room for n in k_lengths]
    q = torch.randn(sum(q_lengths) + behind, heads, dim, device=DEV, generator=g).to(dtype)
    k, v = (torch.randn(sum(rooms) + behind, kv_heads, dim, device=DEV, generator=g).to(dtype) for _ in range(2))
    qo, ko = _offsets(q_lengths), _offsets(rooms)
    spans = list(zip(qo.tolist(), q_lengths, ko.tolist(), k_lengths))
    used = torch.zeros(k.shape[0], dtype=torch.bool, device=DEV)
    for _, _, k0, n in spans:
        used[k0:k0 + n] = True
    k[~used], v[~used] = stale, stale
    q[sum(q_lengths):] = stale
    return q, k, v, qo, ko, torch.tensor(k_lengths, dtype=torch.int32, device=DEV), spans


def _check_forward(q_lengths, k_lengths, heads, kv_heads, dim, dtype, **kw):
    q, k, v, qo, ko, kl, spans = _case(q_lengths, k_lengths, heads, kv_heads, dim, dtype, **kw)
    before = native.launches()
    out = ops.packed_attention(q, k, v, qo, ko, k_lengths=kl)
    assert native.launches() > before
    assert _status() == 0
    oracle.assert_close(out, *oracle.attention(q, k, v, spans, dim ** -0.5)["out"])
    assert not out[sum(q_lengths):].any()
    return q, k, v, qo, ko, kl, out


PROMPTS = [[1], [2, 1], [17], [127, 128, 129], [300, 0, 5, 514], [0], [256, 257, 1, 640]]


@pytest.mark.parametrize("lengths", PROMPTS)
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 3), (6, 2), (8, 1), (8, 2), (32, 1)])
def test_attention_of_prompts(lengths, heads, kv_heads):
    _check_forward(lengths, lengths, heads, kv_heads, 128, BF16, behind=7)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 80, 96, 120, 128])
def test_attention_head_sizes_and_types(dim, dtype):
    _check_forward([130, 3, 200], [130, 3, 200], 4, 2, dim, dtype, behind=1)


@pytest.mark.parametrize("q_lengths,k_lengths", [
    ([5, 100], [700, 333]), ([300], [301]), ([129, 1, 64], [129, 900, 70]), ([200], [1111]),
    ([50, 140, 10], [20, 100, 0]),        # more queries than keys: the first rows see nothing
    ([64, 3], [0, 0])])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (5, 5)])
def test_attention_of_continued_prompts(q_lengths, k_lengths, heads, kv_heads):
    _check_forward(q_lengths, k_lengths, heads, kv_heads, 128, BF16, room=13, behind=300)


@pytest.mark.parametrize("q_lengths,k_lengths", [([40, 200], [5001, 3000]), ([33], [20000]), ([100, 30, 70], [90, 8000, 1])])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 1), (16, 1)])
def test_attention_over_split_key_ranges(q_lengths, k_lengths, heads, kv_heads):
    """Few tiles against many keys: ranges of keys side by side, joined by a second launch."""
    _check_forward(q_lengths, k_lengths, heads, kv_heads, 72, BF16, room=3, behind=260)
    _check_gradients(q_lengths, k_lengths, heads, kv_heads, 72, FP16, room=3, behind=1)


@pytest.mark.parametrize("k_lengths", [[1], [15, 16, 17, 31], [100, 0, 1, 2049], [5000], [257] * 40])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (32, 1, 96), (40, 2, 80)])
def test_attention_of_single_tokens(k_lengths, heads, kv_heads, dim):
    _check_forward([1] * len(k_lengths), k_lengths, heads, kv_heads, dim, BF16, room=21, behind=2)


def test_attention_of_few_tokens_and_idle_sequences():
    _check_forward([3, 0, 9, 1, 0, 0, 1, 1, 1, 1, 0, 3], [5000, 7, 3000, 1, 0, 9, 40, 2, 1, 600, 1, 2], 16, 4, 128, BF16, room=3)
    _check_forward([2, 1, 1, 1], [4000, 900, 30, 1], 40, 1, 64, BF16, room=3)
    _check_forward([0, 1, 3, 0, 2], [40, 900, 33, 7, 2], 8, 2, 128, FP16, room=5, behind=1)
    _check_forward([1] * 30 + [40], [200] * 30 + [300], 8, 2, 128, BF16)


def test_attention_of_nothing():
    q = torch.randn(6, 4, 64, device=DEV).bfloat16()
    k = torch.randn(0, 2, 64, device=DEV).bfloat16()
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert not ops.packed_attention(q, k, k, none, none).any()
    assert not ops.packed_attention(q, k, k, torch.tensor([0, 6], dtype=torch.int32, device=DEV),
                                    torch.tensor([0, 0], dtype=torch.int32, device=DEV)).any()
    k = torch.randn(9, 2, 64, device=DEV).bfloat16()
    assert not ops.packed_attention(q, k, k, none, none).any()
    assert ops.packed_attention(q[:0], k, k, none, none).shape == (0, 4, 64)
    assert _status() == 0


def test_attention_strides():
    """Slices of a joint projection and head-major storage are read in place; others are copied."""
    g = torch.Generator(device=DEV).manual_seed(9)
    lengths = [70, 200]
    joint = torch.randn(270, (8 + 2 + 2) * 64 + 8, device=DEV, generator=g).bfloat16()
    spans = [(0, 70, 0, 70), (70, 200, 70, 200)]
    for shift in (0, 8, 3):
        q, k, v = (joint[:, shift + a:shift + b].unflatten(-1, (-1, 64)) for a, b in ((0, 512), (512, 640), (640, 768)))
        out = ops.packed_attention(q, k, v, _offsets(lengths))
        oracle.assert_close(out, *oracle.attention(q, k, v, spans, 0.125)["out"])
    q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    out = ops.packed_attention(q, k, v, _offsets(lengths))
    oracle.assert_close(out, *oracle.attention(q, k, v, spans, 0.125)["out"])
    k = k[:, :1].expand(270, 2, 64)
    out = ops.packed_attention(q, k, v, _offsets(lengths))
    oracle.assert_close(out, *oracle.attention(q, k, v, spans, 0.125)["out"])
    assert _status() == 0


def test_attention_scores_far_from_zero():
    """Large scores with a maximum that keeps growing along the keys: the running rescale."""
    q, k, v, qo, ko, kl, spans = _case([300, 1], [700, 700], 4, 2, 128, BF16)
    k *= torch.linspace(0.1, 12, k.shape[0], device=DEV)[:, None, None].to(BF16)
    q *= 4
    out = ops.packed_attention(q, k, v, qo, ko, k_lengths=kl)
    # scores up to some hundreds, each an FP32 sum: 2^-24 * |s| * log2(e) in the exponent
    value, bound = oracle.attention(q, k, v, spans, 128 ** -0.5)["out"]
    oracle.assert_close(out, value, bound + 2.0 ** -24 * 2048 * v.double().abs().amax())
    assert _status() == 0


def test_attention_results_do_not_depend_on_company():
    """A sequence gives bit for bit the same alone and among others (and on every run)."""
    q, k, v, qo, ko, kl, spans = _case([130, 300, 77], [130, 300, 77], 4, 2, 128, BF16)
    out = ops.packed_attention(q, k, v, qo)
    assert torch.equal(out, ops.packed_attention(q, k, v, qo))
    for q0, n, _, _ in spans:
        alone = ops.packed_attention(q[q0:q0 + n], k[q0:q0 + n], v[q0:q0 + n], _offsets([n]))
        assert torch.equal(alone, out[q0:q0 + n])


def test_attention_refusals():
    q, k, v, qo, ko, kl, _ = _case([3, 2], [3, 4], 4, 2, 16, BF16)

    def call(**change):
        given = dict(query=q, key=k, value=v, q_offsets=qo, k_offsets=ko, k_lengths=kl, scale=None)
        given.update(change)
        return ops.packed_attention(**given)

    call()
    for change, error in ((dict(query=q[None]), ValueError), (dict(value=v[:-1]), ValueError),
                          (dict(key=k[:, :0], value=v[:, :0]), ValueError), (dict(query=q[:, :3]), ValueError),
                          (dict(key=k.half()), TypeError), (dict(q_offsets=qo.long()), TypeError),
                          (dict(q_offsets=qo[::2]), TypeError), (dict(k_offsets=ko[:2]), ValueError),
                          (dict(k_lengths=kl[:1]), ValueError), (dict(q_offsets=qo[:0], k_offsets=ko[:0]), ValueError),
                          (dict(scale=0.0), ValueError), (dict(scale=math.nan), ValueError), (dict(scale=math.inf), ValueError),
                          (dict(k_offsets=None, k_lengths=None), ValueError), (dict(key=k.cpu()), ValueError),
                          (dict(k_offsets=ko.cpu()), ValueError)):
        with pytest.raises(error, match="packed_attention"):
            call(**change)


def test_uncovered_calls_take_the_definitions():
    """Types and head sizes without a kernel, and forward-mode tangents."""
    import torch.autograd.forward_ad as fwad

    q, k, v, qo, ko, kl, spans = _case([30, 2], [30, 7], 4, 2, 20, BF16, stale=0.0)
    for dtype in (BF16, torch.float32, torch.float64):
        x = [t.to(dtype) for t in (q, k, v)]
        oracle.assert_close(ops.packed_attention(*x, qo, ko, k_lengths=kl), *oracle.attention(*x, spans, 20 ** -0.5)["out"])
    q, k, v, qo, ko, kl, spans = _case([30], [30], 4, 2, 64, BF16)
    f = ops.rotary_frequencies(64, device=DEV)
    with fwad.dual_level():
        dual = fwad.make_dual(q, torch.ones_like(q))
        assert fwad.unpack_dual(ops.packed_attention(dual, k, v, qo)).tangent is not None
        tangent = fwad.unpack_dual(ops.rotary_embed(dual, k, torch.arange(30, device=DEV), f)[0]).tangent
    oracle.assert_close(tangent, *oracle.rotary(torch.ones_like(q), torch.arange(30, device=DEV), f.turns * 2 * math.pi))


@pytest.mark.parametrize("rows", [1, 140])
def test_attention_reports_bad_offsets(rows):
    """Offsets that leave the tensors are caught by the kernels' own checks: the sequence is skipped."""
    q, k, v, qo, ko, kl, spans = _case([rows, rows], [200, 200], 4, 2, 64, BF16)
    for bad in (dict(q_offsets=_offsets([rows, rows + 5])), dict(k_offsets=_offsets([200, 250])),
                dict(k_lengths=kl + 1), dict(k_lengths=-kl), dict(q_offsets=_offsets([rows, -1]))):
        given = dict(q_offsets=qo, k_offsets=ko, k_lengths=kl)
        given.update(bad)
        ops.packed_attention(q, k, v, given["q_offsets"], given["k_offsets"], k_lengths=given["k_lengths"])
        assert _status() == 7, bad
        native.ext().status(torch.cuda.current_device()).zero_()


def test_attention_reports_offsets_that_fall():
    """Sequences that overlap because the offsets fall: more work than the rows can have, refused in place."""
    q, k, v, qo, ko, kl, spans = _case([1] * 40, [700] * 40, 8, 2, 64, BF16)
    fall = qo.clone()
    fall[1::2] = 40
    ops.packed_attention(q, k, v, fall, ko)
    assert _status() == 7
    native.ext().status(torch.cuda.current_device()).zero_()
    fall = ko.clone()
    fall[1::2] = 28000
    ops.packed_attention(q, k, v, qo, fall)
    assert _status() == 7
    native.ext().status(torch.cuda.current_device()).zero_()
    out = ops.packed_attention(q, k, v, qo, ko)
    oracle.assert_close(out, *oracle.attention(q, k, v, spans, 0.125)["out"])
    assert _status() == 0


# ------------------------------------------------------------------------------------ gradients
def _check_gradients(q_lengths, k_lengths, heads, kv_heads, dim, dtype, **kw):
    q, k, v, qo, ko, kl, spans = _case(q_lengths, k_lengths, heads, kv_heads, dim, dtype, **kw)
    g = torch.Generator(device=DEV).manual_seed(77)
    grad = torch.randn(q.shape, device=DEV, generator=g).to(dtype)
    grad[sum(q_lengths):] = float("nan")  # rows of no sequence
    for t in (q, k, v):
        t.requires_grad_()
    before = native.launches()
    out = ops.packed_attention(q, k, v, qo, ko, k_lengths=kl)
    grads = torch.autograd.grad(out, (q, k, v), grad)
    assert native.launches() > before + 1
    assert _status() == 0
    want = oracle.attention(q.detach(), k.detach(), v.detach(), spans, dim ** -0.5, grad)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        oracle.assert_close(got, *want[name], name)
    for got, used in zip((out, *grads), (want["out"], want["dq"], want["dk"], want["dv"])):
        untouched = used[1].flatten(1).sum(-1) == 0  # rows of no sequence, room behind the keys
        assert not got[untouched].any()
    return q, k, v, qo, ko, kl, out, grad, grads


@pytest.mark.parametrize("lengths", PROMPTS)
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 3), (8, 1), (8, 2), (32, 1)])
def test_gradients_of_prompts(lengths, heads, kv_heads):
    _check_gradients(lengths, lengths, heads, kv_heads, 128, BF16, behind=150)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128])
def test_gradients_of_head_sizes_and_types(dim, dtype):
    _check_gradients([130, 3, 200], [130, 3, 200], 4, 2, dim, dtype)


@pytest.mark.parametrize("q_lengths,k_lengths", [([5, 100], [700, 333]), ([129, 1, 64], [129, 900, 70]),
                                                  ([50, 140, 10, 4], [20, 100, 0, 3]), ([64, 3], [0, 0]), ([260], [128])])
def test_gradients_of_continued_prompts(q_lengths, k_lengths):
    _check_gradients(q_lengths, k_lengths, 4, 2, 128, BF16, room=13, behind=2)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (8, 2, 64), (12, 2, 128), (6, 3, 80), (5, 5, 64)])
@pytest.mark.parametrize("lengths", [[700], [300, 129, 40], [3000, 2900]])
def test_gradients_with_shared_and_whole_groups(lengths, heads, kv_heads, dim):
    """Key tiles whose queries two CTAs share (few key tiles) or one CTA takes alone."""
    _check_gradients(lengths, lengths, heads, kv_heads, dim, BF16, behind=3)


def test_gradients_repeat_bit_for_bit_and_take_any_layout():
    q, k, v, qo, ko, kl, out, grad, grads = _check_gradients([130, 70], [130, 70], 4, 2, 64, BF16)
    again = ops.packed_attention(q, k, v, qo, ko, k_lengths=kl)
    head_major = grad.transpose(0, 1).contiguous().transpose(0, 1)
    for a, b in zip(grads, torch.autograd.grad(again, (q, k, v), head_major)):
        assert torch.equal(a, b)
    # a broadcast gradient, and only one leaf
    again = ops.packed_attention(q, k.detach(), v.detach(), qo, ko, k_lengths=kl)
    (got,) = torch.autograd.grad(again.sum(), (q,))
    want = oracle.attention(q.detach(), k.detach(), v.detach(), [(0, 130, 0, 130), (130, 70, 130, 70)], 0.125,
                            torch.ones_like(q))
    oracle.assert_close(got, *want["dq"])


def test_gradient_against_differences():
    """The directional derivative of a smooth function of the output, in a direction of all inputs."""
    q, k, v, qo, ko, kl, spans = _case([40, 90], [40, 90], 4, 2, 64, FP16, seed=3)
    g = torch.Generator(device=DEV).manual_seed(8)
    weight = torch.randn(q.shape, device=DEV, generator=g).to(FP16)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.packed_attention(*leaves, qo), leaves, weight)
    steps = [torch.randn(t.shape, device=DEV, generator=g).double() for t in (q, k, v)]
    slope = sum((a.double() * b).sum() for a, b in zip(grads, steps))
    h = 1e-5

    def value(sign):
        moved = [t.double() + sign * h * s for t, s in zip((q, k, v), steps)]
        return (oracle.attention(*moved, spans, 0.125)["out"][0] * weight.double()).sum()

    want = oracle.attention(q, k, v, spans, 0.125, weight)
    allowed = sum((want[n][1] * s.abs()).sum() for n, s in zip(("dq", "dk", "dv"), steps))
    assert abs(slope - (value(1) - value(-1)) / (2 * h)) <= allowed + 1e-6 * abs(slope) + 1e-3


def test_gradients_of_gradients_are_refused():
    q, k, v, qo, *_ = _case([20], [20], 4, 2, 64, BF16)
    f = ops.rotary_frequencies(64, device=DEV)
    q.requires_grad_()
    for out in (ops.packed_attention(q, k, v, qo), ops.rotary_embed(q, None, torch.arange(20, device=DEV), f)[0]):
        (grad,) = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            grad.sum().backward()


# ------------------------------------------------------------------------------ as they are used
@pytest.mark.parametrize("interleaved,turned,scaling", [(False, 128, None), (True, 64, "yarn")])
def test_prompt_then_tokens_against_a_cache(interleaved, turned, scaling):
    """Prompts turned and attended in one packed batch, then single tokens that are turned, written
    into a cache with room behind every prompt and attended against it: every row is the row of the
    whole sequence."""
    lengths, extra, room, heads, kv_heads, dim = [130, 5, 700], 3, 720, 8, 2, 128
    g = torch.Generator(device=DEV).manual_seed(12)
    whole = [n + extra for n in lengths]
    q, k, v = (torch.randn(sum(whole), h, dim, device=DEV, generator=g).bfloat16() for h in (heads, kv_heads, kv_heads))
    f = ops.rotary_frequencies(turned, 5e6, scaling=scaling, factor=4.0, trained_positions=512, device=DEV)
    starts = _offsets(whole).tolist()
    positions = torch.cat([torch.arange(n, device=DEV) for n in whole])
    qr, kr = ops.rotary_embed(q, k, positions, f, interleaved=interleaved)
    spans = [(a, n, a, n) for a, n in zip(starts, whole)]
    value, bound = oracle.attention(qr, kr, v, spans, dim ** -0.5)["out"]

    prompt = torch.cat([torch.arange(a, a + n, device=DEV) for a, n in zip(starts, lengths)])
    pq, pk = ops.rotary_embed(q[prompt], k[prompt], positions[prompt], f, interleaved=interleaved)
    assert torch.equal(pq, qr[prompt]) and torch.equal(pk, kr[prompt])
    out = ops.packed_attention(pq, pk, v[prompt], _offsets(lengths))
    oracle.assert_close(out, value[prompt], bound[prompt])

    cache = [torch.full((room * 3, kv_heads, dim), float("nan"), device=DEV, dtype=BF16) for _ in range(2)]
    rows = torch.cat([torch.arange(s * room, s * room + n, device=DEV) for s, n in enumerate(lengths)])
    cache[0][rows], cache[1][rows] = pk, v[prompt]
    at = torch.arange(0, 3 * room + 1, room, dtype=torch.int32, device=DEV)
    filled = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    one = _offsets([1, 1, 1])
    for step in range(extra):
        new = torch.tensor([a + n + step for a, n in zip(starts, lengths)], device=DEV)
        tq, tk = ops.rotary_embed(q[new], k[new], positions[new], f, interleaved=interleaved)
        slot = (at[:-1] + filled).long()
        cache[0][slot], cache[1][slot] = tk, v[new]
        filled += 1
        out = ops.packed_attention(tq, *cache, one, at, k_lengths=filled)
        oracle.assert_close(out, value[new], bound[new])
    assert _status() == 0


def _tower(dtype):
    from helpers import tiny_conditioner, tiny_config

    config = tiny_config(hidden_size=512, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                         mrope_section=(24, 20, 20), text_bucket_tokens=64)
    return tiny_conditioner(config, dtype=dtype).text_encoder


def test_text_tower_on_packed_prompts():
    """bf16 on the kernels against the same weights in 64 bits: no further off than the padded tower,
    whose roundings are the same or more, up to what a different draw of roundings gives."""
    encoder = _tower(BF16)
    ids = torch.randint(3, 128, (5, 50))
    valid = torch.arange(50)[None] < torch.tensor([50, 1, 33, 17, 49])[:, None]
    want = _tower(BF16).double().encode_packed(ids, valid)
    encoder.to(DEV)
    before = native.launches()
    packed = encoder.encode_packed(ids.to(DEV), valid.to(DEV))
    assert native.launches() > before
    padded = encoder(ids.to(DEV), valid.to(DEV))
    for mine, theirs, exact in zip((*packed.keys, *packed.values), (*padded.keys, *padded.values),
                                   (*want.keys, *want.values)):
        off = [0.0, 0.0]
        for row, n in enumerate(packed.lengths):
            for i, t in enumerate((mine, theirs)):
                off[i] += float((t[row, :n].double().cpu() - exact[row, :n]).square().sum())
            assert not mine[row, n:].any()
        assert off[0] ** 0.5 <= 1.5 * off[1] ** 0.5
    assert _status() == 0


def test_text_tower_trains_on_packed_prompts():
    """Gradients of all layers in bf16 on the kernels against 64 bits on the CPU."""
    ids = torch.randint(3, 128, (3, 40))
    valid = torch.arange(40)[None] < torch.tensor([40, 9, 26])[:, None]
    grads, yard = [], None
    for encoder, device in ((_tower(BF16).double(), "cpu"), (_tower(BF16).to(DEV), DEV)):
        encoder.requires_grad_(True)
        context = encoder.encode_packed(ids.to(device), valid.to(device))
        weights = [layer.self_attn.to_k.weight for layer in encoder.layers] + [encoder.embed_tokens.weight]
        loss = sum(t.double().square().sum() for t in (*context.keys, *context.values))
        grads.append([g.double().cpu() for g in torch.autograd.grad(loss, weights, retain_graph=True)])
        if yard is None:
            # The keys are normalised, so the sum of their squares is constant and its exact gradient next
            # to nothing: a rounding's size goes by the terms that cancel.  A rounding is a change of
            # 2^-8 of them in a direction of its own; what the sizes |2 t| of the loss's gradient come to
            # in random directions is the gradient of sum s |2 t| t with t of the factor held.
            g = torch.Generator().manual_seed(9)
            other = sum((t * (2 * t.detach().abs() * torch.randn(t.shape, generator=g, dtype=t.dtype).sign())).sum()
                        for t in (*context.keys, *context.values))
            yard = [x.norm() for x in torch.autograd.grad(other, weights)]
    # about 20 roundings of 2^-8 on the way through two layers and back, adding up as a random walk,
    # and bf16 weight gradients
    for a, b, size in zip(*grads, yard):
        assert (a - b).norm() <= 20 ** 0.5 * 2.0 ** -8 * 2 * max(size, a.norm())


# -------------------------------------------------------------------------------- graphs, streams
def test_calls_replay_in_graphs_with_other_lengths():
    """Captured calls read their lengths at replay: the same graph serves other lengths, also two graphs
    side by side on two streams."""
    def state(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        q = torch.randn(400, 8, 128, device=DEV, generator=g).bfloat16()
        k, v = (torch.randn(4000, 2, 128, device=DEV, generator=g).bfloat16() for _ in range(2))
        return q, k, v

    def spans(qo, ko, kl):
        qo, ko, kl = qo.tolist(), ko.tolist(), kl.tolist()
        return [(a, b - a, c, n) for a, b, c, n in zip(qo, qo[1:], ko, kl)]

    graphs = []
    for seed, lengths in ((1, [100, 300]), (2, [1] * 400)):
        q, k, v = state(seed)
        n = len(lengths)
        room = 4000 // n
        qo, ko = _offsets(lengths), _offsets([room] * n)
        kl = torch.full((n,), room, dtype=torch.int32, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.packed_attention(q, k, v, qo, ko, k_lengths=kl)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.packed_attention(q, k, v, qo, ko, k_lengths=kl)
        graphs.append((graph, q, k, v, qo, ko, kl, out))
    for shrink in (0, 7):
        for _, _, _, _, _, _, kl, _ in graphs:
            kl -= shrink
        torch.cuda.synchronize()
        for _ in range(3):
            streams = [torch.cuda.Stream() for _ in graphs]
            for stream, entry in zip(streams, graphs):
                with torch.cuda.stream(stream):
                    entry[0].replay()
            torch.cuda.synchronize()
        for _, q, k, v, qo, ko, kl, out in graphs:
            oracle.assert_close(out, *oracle.attention(q, k, v, spans(qo, ko, kl), 128 ** -0.5)["out"])
    assert _status() == 0


def test_training_step_replays_in_a_graph():
    q, k, v, qo, ko, kl, spans = _case([130, 70], [130, 70], 4, 2, 64, BF16, seed=6)
    f = ops.rotary_frequencies(64, 1e4, device=DEV)
    positions = torch.cat([torch.arange(n, device=DEV) for n in (130, 70)])
    grad = torch.randn_like(q)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        a, b = ops.rotary_embed(q, k, positions, f)
        out = ops.packed_attention(a, b, v, qo)
        return out.detach(), *torch.autograd.grad(out, leaves, grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        q.copy_(q.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in captured]
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    assert _status() == 0


def test_calls_on_another_stream_and_their_gradients():
    q, k, v, qo, ko, kl, spans = _case([300], [300], 4, 2, 128, BF16, seed=7)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grad = torch.randn_like(q)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out = ops.packed_attention(q, k, v, qo)
        grads = torch.autograd.grad(out, leaves, grad)
    stream.synchronize()
    want = oracle.attention(q.detach(), k.detach(), v.detach(), spans, 128 ** -0.5, grad)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        oracle.assert_close(got, *want[name], name)


def test_many_sequences():
    """More sequences than are ranked by length, and more than a step of the searches."""
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 40, (1500,), generator=g).tolist()
    _check_forward(lengths, lengths, 4, 2, 64, BF16, behind=9)
    _check_gradients(lengths[:300], lengths[:300], 4, 2, 64, BF16, behind=9)
    _check_forward([1] * 1500, [n + 1 for n in lengths], 8, 2, 64, FP16, room=2, behind=1)
    rows = torch.randint(0, 3, (1500,), generator=g).tolist()
    _check_forward(rows, [n + 2 for n in lengths], 8, 2, 64, FP16, room=2, behind=1)

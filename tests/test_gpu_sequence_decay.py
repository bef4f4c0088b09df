"""decay_attention and decay_attention_step on the device against the recurrence in 64 bits."""
import math

import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _make(dtype, b, h, kv, t, d, dv, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    q, k, v, go = (r(b, t, x, w).to(dtype).transpose(1, 2) for x, w in ((h, d), (kv, d), (kv, dv), (h, dv)))
    ld = -torch.exp2(-torch.linspace(0, 9, h, device="cuda"))
    return q, k, v, ld, r(b, h, d, dv), go, r(b, h, d, dv)


def _check(q, k, v, ld, state, lengths, go, gs, scale=None):
    from keops_amd.torch import decay_attention

    s = q.shape[-1] ** -0.5 if scale is None else scale
    want = ref.decay(q, k, v, ld, state, lengths, s, go, gs)
    leaves = [None if x is None else x.detach().requires_grad_(True) for x in (q, k, v, state)]
    out, last = decay_attention(*leaves[:3], ld, initial_state=leaves[3], lengths=lengths, scale=scale)
    assert out.dtype == q.dtype and last.dtype == FP32
    ref.assert_within(out.detach(), want["out"], want["tol_out"], "out")
    ref.assert_within(last.detach(), want["state"], want["tol_state"], "state")
    named = [(n, x) for n, x in zip(("q", "k", "v", "state"), leaves) if x is not None]
    outs, seeds = ([out], [go]) if gs is None else ([out, last], [go, gs])
    for (name, x), g in zip(named, torch.autograd.grad(outs, [x for _, x in named], seeds)):
        assert g.shape == x.shape and g.dtype == x.dtype
        ref.assert_within(g, want["grad_" + name], want["tol_grad_" + name], "grad_" + name)
    return out, last


# batch, heads, kv_heads, tokens, dim, dim_v, start state, lengths
CASES = [
    (2, 2, 2, 1, 64, 64, True, None),
    (1, 2, 1, 64, 64, 64, False, None),
    (2, 3, 3, 65, 32, 64, True, None),
    (2, 4, 2, 200, 128, 128, True, [200, 77]),
    (3, 2, 1, 130, 40, 72, True, [130, 0, 64]),   # a sequence without tokens
    (1, 1, 1, 300, 16, 128, False, None),
    (1, 2, 2, 127, 96, 24, True, [1]),
    (2, 6, 2, 70, 8, 8, False, [70, 69]),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("case", CASES)
def test_values_and_gradients(case, dtype):
    b, h, kv, t, d, dv, start, lengths = case
    q, k, v, ld, state, go, gs = _make(dtype, b, h, kv, t, d, dv)
    lengths = None if lengths is None else torch.tensor(lengths, device="cuda")
    _check(q, k, v, ld, state if start else None, lengths, go, gs if start else None)


def test_long_sequence_in_segments():
    """More chunks than one workgroup walks: states at the ends of segments, ragged within a segment."""
    q, k, v, ld, state, go, gs = _make(BF16, 2, 2, 1, 1500, 64, 64)
    _check(q, k, v, ld, state, torch.tensor([1500, 700], dtype=torch.int32, device="cuda"), go, gs)


@pytest.mark.parametrize("dtype,b,h,kv,t,d,dv", [(FP32, 8, 24, 8, 265, 40, 128), (BF16, 1, 4, 4, 2100, 128, 64), (FP16, 2, 3, 1, 1000, 16, 72)])
def test_training_in_segments_with_different_dims(dtype, b, h, kv, t, d, dv):
    q, k, v, ld, state, go, gs = _make(dtype, b, h, kv, t, d, dv)
    _check(q, k, v, ld, state, None, go, gs)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_dims_and_strides_that_are_copied_first(dtype):
    gen = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dtype)
    ld = torch.tensor([-0.3, -0.01], device="cuda")
    for d, dv in ((1, 3), (20, 33), (100, 7)):
        _check(r(2, 2, 70, d), r(2, 1, 70, d), r(2, 1, 70, dv), ld, r(2, 2, d, dv).float(), None, r(2, 2, 70, dv), r(2, 2, d, dv).float(), scale=0.5)
    k = r(2, 1, 16, 71)[..., 1:].transpose(2, 3)
    v = r(1, 1, 70, 16).expand(2, 1, 70, 16)
    _check(r(2, 2, 70, 16), k, v, ld, None, None, r(2, 2, 70, 1).expand(2, 2, 70, 16), None)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_gradients_of_shared_heads(dtype):
    """Joined over the heads that share, in the order of dimensions of the inputs; lengths behind which the gradient is zeros."""
    q, k, v, ld, state, go, gs = _make(dtype, 2, 12, 3, 150, 24, 40)
    lengths = torch.tensor([150, 31], device="cuda")
    _check(q, k, v, ld, state, lengths, go, gs)
    from keops_amd.torch import decay_attention

    k.requires_grad_(True)
    v.requires_grad_(True)
    dk, dv = torch.autograd.grad(decay_attention(q, k, v, ld, lengths=lengths)[0], (k, v), go)
    assert dk.stride() == k.stride() and dv.stride() == v.stride()
    assert (dk[1, :, 31:] == 0).all() and (dv[1, :, 31:] == 0).all()
    # no heads: nothing to add up
    none = decay_attention(q[:, :0], k, v, ld[:0])[0]
    dk, dv = torch.autograd.grad(none, (k, v), go[:, :0])
    assert (dk == 0).all() and (dv == 0).all()


def test_single_ones_may_have_any_stride_and_numbers_any_type():
    from keops_amd.torch import decay_attention, decay_attention_step

    gen = torch.Generator(device="cuda").manual_seed(9)
    base = torch.randn(2 * 130 * 64 + 6, device="cuda", generator=gen).bfloat16()
    q = base.as_strided((1, 1, 130, 64), (5, 3, 64, 1))
    k = base.as_strided((1, 1, 130, 64), (130 * 64 + 1, 7, 64, 1), 8)
    ld, state, go = torch.tensor([-0.2], device="cuda"), torch.zeros(1, 1, 64, 64, device="cuda"), torch.randn(1, 1, 130, 64, device="cuda").bfloat16()
    _check(q, k, k, ld, None, torch.tensor([2 ** 40], device="cuda"), go, None)
    # a scale that is a tensor counts by its value at the call
    scale = torch.tensor(0.5)
    a = decay_attention(q, k, k, ld, scale=scale)[0]
    step = decay_attention_step(q[:, :, 0], k[:, :, 0], k[:, :, 0], ld, state.clone(), scale=scale)
    scale.mul_(2)
    assert torch.equal(decay_attention(q, k, k, ld, scale=scale)[0], 2 * a)
    assert torch.equal(decay_attention_step(q[:, :, 0], k[:, :, 0], k[:, :, 0], ld, state.clone(), scale=scale), 2 * step)


def test_decays_at_the_ends_of_their_range():
    q, k, v, _, state, go, gs = _make(FP32, 1, 3, 1, 140, 32, 32)
    ld = torch.tensor([0.0, -math.inf, -60.0], device="cuda")
    out, last = _check(q, k, v, ld, state, None, go, gs)
    assert out.isfinite().all() and last.isfinite().all()


def test_what_lies_behind_the_lengths_is_not_read():
    q, k, v, ld, state, go, gs = _make(BF16, 2, 2, 2, 150, 64, 64)
    lengths = torch.tensor([90, 0], device="cuda")
    for i, n in enumerate((90, 0)):
        for x in (q, k, v):
            x[i, :, n:] = math.nan
    out, last = _check(q, k, v, ld, state, lengths, torch.where(torch.arange(150, device="cuda")[None, None, :, None] < lengths[:, None, None, None], go, go * 0), gs)
    assert (out[0, :, 90:] == 0).all() and (out[1] == 0).all() and torch.equal(last[1], state[1])


def test_prompt_then_tokens():
    """The state of a prompt carried on one token at a time is the whole sequence's, and so is a prompt in two pieces."""
    from keops_amd.torch import decay_attention, decay_attention_step

    for dtype, d, dv in ((BF16, 64, 128), (FP16, 128, 64), (FP32, 40, 72)):
        q, k, v, ld, state, _, _ = _make(dtype, 2, 4, 2, 100, d, dv, seed=2)
        want = ref.decay(q, k, v, ld, state, None, d ** -0.5)
        out, S = decay_attention(q[:, :, :70], k[:, :, :70], v[:, :, :70], ld, initial_state=state)
        rest, S2 = decay_attention(q[:, :, 70:], k[:, :, 70:], v[:, :, 70:], ld, initial_state=S)
        tokens = []
        S = S.clone()
        for t in range(70, 100):
            tokens.append(decay_attention_step(q[:, :, t], k[:, :, t], v[:, :, t], ld, S))
        for got in (rest, torch.stack(tokens, 2)):
            ref.assert_within(torch.cat([out, got], 2), want["out"], want["tol_out"] + 2 ** -22 * want["out"].abs(), "out")
        for got in (S, S2):
            ref.assert_within(got, want["state"], 2 * want["tol_state"], "state")


@pytest.mark.parametrize("b,h,kv,d,dv", [(1, 1, 1, 1, 4), (3, 4, 2, 40, 72), (64, 16, 16, 128, 128), (2, 8, 1, 128, 64), (300, 2, 2, 17, 12)])
def test_one_token(b, h, kv, d, dv):
    from keops_amd.torch import decay_attention_step

    for dtype in (BF16, FP16, FP32):
        q, k, v, ld, state, _, _ = _make(dtype, b, h, kv, 1, d, dv)
        want = ref.decay(q, k, v, ld, state, None, 0.3)
        S = state.clone()
        out = decay_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], ld, S, scale=0.3)
        ref.assert_within(out, want["out"][:, :, 0], want["tol_out"][:, :, 0], "out")
        ref.assert_within(S, want["state"], want["tol_state"], "state")


def test_gradients_against_differences():
    from keops_amd.torch import decay_attention

    q, k, v, ld, state, go, gs = _make(FP32, 1, 2, 1, 90, 24, 20, seed=7)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, state)]

    def f(ts):
        out, last = decay_attention(*ts[:3], ld, initial_state=ts[3])
        return (out.double() * go.double()).sum() + (last.double() * gs.double()).sum()

    grads = torch.autograd.grad(f(leaves), leaves)
    for i, g in enumerate(grads):
        w = torch.randn_like(leaves[i])
        eps = 1e-2
        moved = lambda e: [t.detach() + (e * w if j == i else 0) for j, t in enumerate(leaves)]
        diff = float(f(moved(eps)) - f(moved(-eps))) / (2 * eps)
        # linear in each input: the difference is exact up to the float32 values, 2 eps apart
        assert abs(diff - float((g * w).sum())) < 1e-3 * float((g.abs() * w.abs()).sum()), i


def test_graph_streams_and_repeats():
    from keops_amd.torch import decay_attention, decay_attention_step

    q, k, v, ld, state, go, gs = _make(BF16, 2, 4, 2, 700, 64, 64)
    one = [x[:, :, 0].contiguous() for x in (q, k, v)]

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, state)]
        out, last = decay_attention(*leaves[:3], ld, initial_state=leaves[3])
        grads = torch.autograd.grad([out, last], leaves, [go, gs])
        S = last.detach().clone()
        return (out.detach(), last.detach(), *grads, decay_attention_step(*one, ld, S), S)

    eager = run()
    assert all(torch.equal(a, b) for a, b in zip(eager, run()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    torch.cuda.synchronize()
    del eager, other
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for _ in range(3):
        for t in (q, k, v, state, go, gs, *one):
            t.copy_(torch.randn(t.shape, device="cuda"))
        want = run()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals_on_the_device():
    from keops_amd.torch import decay_attention, decay_attention_step

    q, k, v, ld, state, _, _ = _make(BF16, 2, 4, 2, 5, 16, 24)
    for change, match in [(dict(q=q.double()), "float32"), (dict(k=k.float()), "one type"), (dict(v=v[:, :, :4]), "do not fit"), (dict(q=q[:, :3]), "do not fit"),
                          (dict(log_decay=ld[:2]), "log_decay"), (dict(log_decay=ld.double()), "log_decay"), (dict(log_decay=ld.cpu()), "same device"),
                          (dict(log_decay=ld.clone().requires_grad_(True)), "constant"), (dict(initial_state=state[:1]), "state"),
                          (dict(initial_state=state.half()), "state"), (dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), "lengths")]:
        with pytest.raises(ValueError, match=match):
            decay_attention(**{**dict(q=q, k=k, v=v, log_decay=ld), **change})
    one = dict(q=q[:, :, 0], k=k[:, :, 0], v=v[:, :, 0], log_decay=ld, state=state)
    odd = torch.zeros(2, 2, 6, dtype=BF16, device="cuda")
    for change, match in [(dict(state=None), "state"), (dict(state=state.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
                          (dict(q=one["q"].detach().requires_grad_(True)), "no gradient"), (dict(q=q), "dimensions"),
                          (dict(v=odd, state=torch.zeros(2, 4, 16, 6, device="cuda")), "multiple of 4")]:
        with pytest.raises(ValueError, match=match):
            decay_attention_step(**{**one, **change})
    out, last = decay_attention(q[:, :, :0], k[:, :, :0], v[:, :, :0], ld, initial_state=state)  # no tokens: the state stays
    assert out.shape == (2, 4, 0, 24) and torch.equal(last, state)

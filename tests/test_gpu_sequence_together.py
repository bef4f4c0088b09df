"""The sequence operators as a model uses them: a layer of softmax attention with position buckets, a layer of linear attention with
decays, logits, log probabilities and entropies; trained on a padded batch, then generating one token at a time from its caches."""
import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu

B, T, H, KV, D, VOCAB, WIDTH = 2, 90, 4, 2, 32, 501, 128


def _weights(dtype, device):
    gen = torch.Generator().manual_seed(11)
    shapes = dict(embed=(VOCAB, WIDTH), qkv1=(WIDTH, (H + 2 * KV) * D), out1=(H * D, WIDTH), qkv2=(WIDTH, (H + 2 * KV) * D), out2=(H * D, WIDTH),
                  head=(WIDTH, VOCAB), bias=(H, 32))
    return {n: (torch.randn(*s, generator=gen) * (1.0 if n in ("embed", "bias") else s[0] ** -0.5)).to(dtype=dtype, device=device) for n, s in shapes.items()}


def _split(x):
    q, k, v = x.split((H * D, KV * D, KV * D), -1)
    return tuple(t.unflatten(-1, (-1, D)).transpose(1, 2) for t in (q, k, v))


def _merge(x):
    return x.transpose(1, 2).flatten(2)


def _model(w, tokens, lengths, attend, carry):
    x = w["embed"][tokens]
    x = x + _merge(attend(*_split(x @ w["qkv1"]))) @ w["out1"]
    x = x + _merge(carry(*_split(x @ w["qkv2"]))) @ w["out2"]
    return x @ w["head"]


def _data():
    gen = torch.Generator().manual_seed(12)
    tokens = torch.randint(0, VOCAB, (B, T + 1), generator=gen)
    lengths = torch.tensor([T, 61])
    targets = torch.where(torch.arange(T) < lengths[:, None], tokens[:, 1:], -100)
    return tokens[:, :-1], targets, lengths


LOG_DECAY = torch.tensor([-0.7, -0.2, -0.05, -0.01])


def test_training_step():
    from keops_amd.torch import PositionBuckets, bucket_attention, decay_attention, token_logprobs

    buckets = PositionBuckets(32, 64, bidirectional=False)
    tokens, targets, lengths = _data()
    w = {n: t.requires_grad_(True) for n, t in _weights(torch.float32, "cuda").items()}
    ld, lens = LOG_DECAY.cuda(), lengths.int().cuda()
    logits = _model(w, tokens.cuda(), lens, lambda q, k, v: bucket_attention(q, k, v, w["bias"], buckets, causal=True, key_lengths=lens),
                    lambda q, k, v: decay_attention(q, k, v, ld, lengths=lens)[0])
    r = token_logprobs(logits, targets.cuda(), top=3)
    live = (targets != -100).cuda()
    loss = -(r.logprob.sum() + 0.1 * (r.entropy * live).sum()) / live.sum()
    got = dict(zip(w, torch.autograd.grad(loss, list(w.values()))))

    w64 = {n: t.requires_grad_(True) for n, t in _weights(torch.float32, "cpu").items()}
    x64 = {n: t.double() for n, t in w64.items()}
    away = torch.arange(T) - torch.arange(T)[:, None]

    def attend(q, k, v):
        k, v = k.repeat_interleave(H // KV, 1), v.repeat_interleave(H // KV, 1)
        z = q @ k.transpose(-1, -2) * D ** -0.5 + x64["bias"][:, buckets(away)]
        return torch.softmax(z.masked_fill((away > 0) | (torch.arange(T) >= lengths[:, None, None])[:, None], -torch.inf), -1) @ v

    def carry(q, k, v):
        k, v = k.repeat_interleave(H // KV, 1), v.repeat_interleave(H // KV, 1)
        there = (torch.arange(T) < lengths[:, None])[:, None, :, None]
        g = torch.where(away <= 0, torch.exp(-away.clamp(max=0) * LOG_DECAY.double()[:, None, None]), 0.0)
        return torch.where(there, ((q @ k.transpose(-1, -2)) * D ** -0.5 * g) @ v, 0.0)

    lp = torch.log_softmax(_model(x64, tokens, lengths, attend, carry), -1)
    alive = targets != -100
    ent = -(lp.exp() * lp).sum(-1)
    loss64 = -((lp.gather(-1, targets.clamp(min=0)[..., None])[..., 0] * alive).sum() + 0.1 * (ent * alive).sum()) / alive.sum()
    want = dict(zip(w, torch.autograd.grad(loss64, list(w64.values()))))
    # float32: sums of at most 500 terms, 501 * 2^-24 = 3e-5 of their absolute sums at the worst, through ten products and reductions
    assert abs(loss.item() - loss64.item()) < 1e-4 * abs(loss64.item())
    for n in w:
        d = got[n].cpu().double() - want[n].double()
        assert float(d.norm()) < 3e-4 * float(want[n].norm()), n
    top = torch.sort(lp, dim=-1, descending=True).values[..., :3]
    assert (r.top_logprob.cpu().double() - top)[alive].abs().max() < 3e-4 * lp.abs().max().item()


def test_generation_from_caches_is_the_whole_sequence():
    from keops_amd.torch import PositionBuckets, bucket_attention, decay_attention, decay_attention_step, token_logprobs

    buckets = PositionBuckets(32, 64, bidirectional=False)
    tokens, targets, _ = _data()
    tokens, targets = tokens.cuda(), targets.clamp(min=0).cuda()
    for dtype, tol in ((torch.float32, 3e-4), (torch.bfloat16, 0.15)):
        # tol: of a log probability; float32 as above, bf16: logits of size 4 from products of 128 rounded terms, through seven roundings
        w, ld = _weights(dtype, "cuda"), LOG_DECAY.cuda()
        w["bias"] = w["bias"].float()
        kept = {}

        def attend(q, k, v):
            kept["k"], kept["v"] = k, v
            return bucket_attention(q, k, v, w["bias"], buckets, causal=True)

        def carry(q, k, v):
            out, kept["state"] = decay_attention(q, k, v, ld)
            return out

        with torch.no_grad():
            whole = token_logprobs(_model(w, tokens, None, attend, carry), targets, top=2)
            prompt = T - 12
            _model(w, tokens[:, :prompt], None, attend, carry)
            keys, values = (torch.zeros(B, KV, T, D, dtype=dtype, device="cuda") for _ in range(2))
            keys[:, :, :prompt], values[:, :, :prompt] = kept["k"], kept["v"]
            state = kept["state"]
            for t in range(prompt, T):
                lens = torch.full((B,), t + 1, dtype=torch.int32, device="cuda")

                def attend_one(q, k, v):
                    keys[:, :, t:t + 1], values[:, :, t:t + 1] = k, v
                    return bucket_attention(q, keys, values, w["bias"], buckets, causal=True, key_lengths=lens, query_start=lens - 1)

                def carry_one(q, k, v):
                    return decay_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], ld, state)[:, :, None]

                one = token_logprobs(_model(w, tokens[:, t:t + 1], None, attend_one, carry_one), targets[:, t:t + 1], top=2)
                for a, b in ((one.logprob, whole.logprob), (one.entropy, whole.entropy), (one.top_logprob, whole.top_logprob)):
                    assert (a[:, 0] - b[:, t]).abs().max() < tol * max(1.0, float(b.abs().max())), (dtype, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved_tensors_that_hooks_lay_out_anew(dtype):
    """Saved tensors that travel to the host and back come back contiguous, whatever the strides of the inputs were."""
    from keops_amd.torch import PositionBuckets, bucket_attention, decay_attention, token_logprobs

    gen = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dtype)
    q, k = r(2, 150, 4, 64)[..., :32].transpose(1, 2), r(2, 150, 2, 32).transpose(1, 2)  # rows of a wider tensor; another order
    v = r(1, 2, 150, 32).expand(2, 2, 150, 32)
    bias, b = torch.randn(4, 32, device="cuda", generator=gen), PositionBuckets()
    ld, x, tokens, go = -torch.rand(4, device="cuda", generator=gen), r(20, 600)[:, 40:], torch.arange(20, device="cuda"), r(2, 4, 150, 32)

    def gradients(offload):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, bias, x)]
        with torch.autograd.graph.save_on_cpu() if offload else contextlib.nullcontext():
            outs = (bucket_attention(*leaves[:4], b, causal=True), decay_attention(*leaves[:3], ld)[0], token_logprobs(leaves[4], tokens, top=3).logprob)
        return torch.autograd.grad(outs, leaves, (go, go, torch.ones(20, device="cuda")))

    for want, got in zip(gradients(False), gradients(True)):
        assert torch.equal(want, got)

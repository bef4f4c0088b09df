"""token_logprobs on the device against 64 bits."""
import math

import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _check(x, tokens, top, ignore_index=-100, seed=0):
    from keops_amd.torch import token_logprobs

    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    rows = x.shape[0]
    grads = (r(rows), r(rows), r(rows, top))
    want = ref.logprobs(x, tokens, top, ignore_index, grads)
    leaf = x.detach().requires_grad_(True)
    got = token_logprobs(leaf, tokens, top=top, ignore_index=ignore_index)
    assert torch.equal(got.top_index, want["top_index"])
    for name in ("logprob", "entropy", "top_logprob"):
        t = getattr(got, name).detach()
        assert t.dtype == FP32
        ref.assert_within(t, want[name], want["tol_" + name], name)
    (g,) = torch.autograd.grad([got.logprob, got.entropy, got.top_logprob], leaf, list(grads))
    assert g.dtype == x.dtype and g.shape == x.shape
    ref.assert_within(g, want["grad"], want["tol_grad"], "grad")
    with torch.no_grad():
        again = token_logprobs(x, tokens, top=top, ignore_index=ignore_index)
    assert all(torch.equal(a.detach(), b) for a, b in zip(got, again))
    return got, g


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 1, 0), (3, 5, 5), (7, 1000, 3), (2, 2048, 64), (5, 4099, 20), (1, 50021, 5), (600, 777, 2),
                                            (4, 32003, 64), (1100, 8193, 1), (2, 200000, 20), (1, 400003, 20),
                                            (2, 300000, 64), (3, 262145, 0), (700, 8192, 64)])
def test_values_and_gradients(rows, vocab, top, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows * vocab)
    x = (torch.randn(rows, vocab, device="cuda", generator=gen) * 3).to(dtype)  # 16 bits: many equal values
    _check(x, torch.randint(0, vocab, (rows,), device="cuda", generator=gen), top)


@pytest.mark.parametrize("vocab", [40, 3000, 70001, 280001])
def test_equal_ordered_and_masked_values(vocab):
    """All equal; increasing (every value is a new maximum); decreasing; few that are not -inf; the type's lowest value; none at all;
    zeros of both signs; the given token -inf."""
    a = torch.arange(vocab, device="cuda", dtype=FP32)
    rows = [torch.full_like(a, 2.5), a / 64, -a / 64, torch.where(a % 17 == 3, a * 0 + 1, -math.inf), torch.where(a > 5, torch.finfo(FP32).min, a),
            torch.full_like(a, -math.inf), torch.where(a % 2 == 0, -0.0, 0.0), torch.where(a == 1, -math.inf, a * 0), a * 0 + 3e4]
    x = torch.stack(rows)
    tokens = torch.full((len(rows),), 1, device="cuda")
    for dtype in (FP32, BF16):
        y = x.to(dtype)
        got, g = _check(y, tokens, min(24, vocab))
        assert got.logprob[5] == -math.inf and got.entropy[5] == 0 and (g[5] == 0).all()
        assert got.logprob[7] == -math.inf
        assert got.top_index[6].tolist() == list(range(min(24, vocab)))


def test_ignored_missing_and_not_finite():
    from keops_amd.torch import token_logprobs

    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(6, 9000, device="cuda", generator=gen)
    tokens = torch.tensor([5, -100, 8999, -100, 0, 17], device="cuda")
    got, g = _check(x, tokens, 4)
    assert got.logprob[1] == 0
    _check(x, torch.where(tokens < 0, 3, tokens).int(), 4, ignore_index=17)
    bad = tokens.clone()
    bad[0], bad[2] = 9000, -7
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, bad)
    assert r.logprob[[0, 2]].isnan().all() and r.logprob[[1, 3, 4, 5]].isfinite().all() and r.entropy.isfinite().all()
    (g,) = torch.autograd.grad(r.logprob.sum(), leaf)
    assert g[[0, 2]].isnan().any(1).all() and g[[1, 3, 4, 5]].isfinite().all()
    y = x.clone()
    y[0, 77], y[3, 8990] = math.nan, math.inf
    r = token_logprobs(y, tokens.clamp(min=0))
    assert r.logprob[[0, 3]].isnan().all() and r.entropy[[0, 3]].isnan().all()
    assert r.logprob[[1, 2, 4, 5]].isfinite().all() and r.entropy[[1, 2, 4, 5]].isfinite().all()


def test_shapes_and_strides():
    from keops_amd.torch import token_logprobs

    gen = torch.Generator(device="cuda").manual_seed(2)
    for dtype in (BF16, FP32):
        x = torch.randn(4, 3, 1003, device="cuda", generator=gen).to(dtype)
        tokens = torch.randint(0, 1001, (4, 3), device="cuda", generator=gen)
        flat = _check(x.view(12, -1)[:, 1:1002], tokens.view(-1), 3)[0]      # rows that begin anywhere
        leaf = x[:, :, 1:1002].detach().requires_grad_(True)
        r = token_logprobs(leaf, tokens, top=3)
        assert r.logprob.shape == (4, 3) and r.top_index.shape == (4, 3, 3)
        assert torch.equal(r.logprob.view(-1), flat.logprob) and torch.equal(r.top_logprob.view(12, 3), flat.top_logprob)
        torch.autograd.grad(r.entropy.sum(), leaf)
        t = x.view(12, -1).t().contiguous().t()                               # columns are not neighbours
        assert torch.equal(token_logprobs(t, tokens.view(-1)).entropy, token_logprobs(x.view(12, -1), tokens.view(-1)).entropy)
        one = token_logprobs(x[0, 0], tokens[0, 0], top=1)
        assert one.logprob.shape == () and one.top_index.shape == (1,)
        column = tokens.repeat(1, 5)[:, 3:4]                                  # tokens that are not neighbours
        assert torch.equal(token_logprobs(x[:, :1], column).logprob, token_logprobs(x[:, :1], column.contiguous()).logprob)
        none = token_logprobs(x[:0], tokens[:0], top=2)
        assert none.top_logprob.shape == (0, 3, 2)


def test_rows_beyond_32_bit_offsets():
    from keops_amd.torch import token_logprobs

    store = torch.zeros(3, 1 << 30, dtype=BF16, device="cuda")
    x = store[:, :5000]
    x.copy_(torch.randn(3, 5000, device="cuda"))
    tokens = torch.tensor([0, 17, 4999], device="cuda")
    got, want = token_logprobs(x, tokens, top=5), token_logprobs(x.contiguous(), tokens, top=5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradient_against_differences():
    from keops_amd.torch import token_logprobs

    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(5, 300, device="cuda", generator=gen)
    tokens = torch.randint(0, 300, (5,), device="cuda", generator=gen)

    def f(x):
        r = token_logprobs(x, tokens, top=3)
        return (r.logprob.double().sum() + 0.7 * r.entropy.double().sum() + 0.2 * r.top_logprob.double().sum())

    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(f(leaf), leaf)
    w = torch.randn(5, 300, device="cuda", generator=gen)
    diff = float(f(x + 1e-3 * w) - f(x - 1e-3 * w)) / 2e-3
    # 25 float32 values near 5, differenced over 2e-3
    assert abs(diff - float((g * w).sum())) < 25 * 5 * 2 ** -24 * 4 / 2e-3 + 1e-3 * float((g.abs() * w.abs()).sum())


def test_graph_and_streams():
    from keops_amd.torch import token_logprobs

    gen = torch.Generator(device="cuda").manual_seed(4)
    big = torch.randn(3, 60001, device="cuda", generator=gen).to(BF16)
    tokens = torch.randint(0, 60001, (3,), device="cuda", generator=gen)

    def run():
        leaf = big.detach().requires_grad_(True)
        r = token_logprobs(leaf, tokens, top=8)
        (g,) = torch.autograd.grad([r.logprob.sum(), r.entropy.sum()], leaf)
        return (*(t.detach() for t in r), g)

    eager = run()
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
        big.copy_(torch.randn(big.shape, device="cuda"))
        want = run()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_results_may_be_changed_in_place():
    """The log probabilities are a tensor of their own: masking them in place leaves what the gradient needs."""
    from keops_amd.torch import token_logprobs

    x = torch.randn(6, 500, device="cuda", requires_grad=True)
    tokens, mask = torch.arange(6, device="cuda"), torch.tensor([1.0, 0, 1, 1, 0, 1], device="cuda")
    r = token_logprobs(x, tokens)
    (want,) = torch.autograd.grad((r.logprob * mask).sum(), x)
    r = token_logprobs(x, tokens)
    r.logprob.mul_(mask)
    (got,) = torch.autograd.grad(r.logprob.sum(), x)
    assert torch.equal(got, want)


def test_refusals_on_the_device():
    from keops_amd.torch import token_logprobs

    x = torch.randn(3, 10, device="cuda")
    tok = torch.zeros(3, dtype=torch.int64, device="cuda")
    for args, kw, match in [((x.double(), tok), {}, "float32"), ((x, tok[:2]), {}, "tokens"), ((x, tok.cpu()), {}, "same device"), ((x, tok), dict(top=11), "top"),
                            ((x, tok), dict(top=-1), "top"), ((x, tok), dict(top=2.0), "top"), ((x[:, :0], tok), {}, "vocabulary")]:
        with pytest.raises(ValueError, match=match):
            token_logprobs(*args, **kw)
    with pytest.raises(TypeError, match="int64"):
        token_logprobs(x, tok.float())
    with pytest.raises(ValueError, match="top"):
        token_logprobs(torch.randn(2, 100, device="cuda"), tok[:2], top=65)

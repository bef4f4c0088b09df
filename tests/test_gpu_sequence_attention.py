"""bucket_attention on the device against 64 bits: values and gradients within bounds counted from the roundings
(sequence_reference.py), masks that leave rows empty, layouts, graphs, streams."""
import math

import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _make(dtype, b, h, kv, m, n, d, buckets=32, seed=0, by_token=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    if by_token:
        q, k, v = (r(b, t, x, d).to(dtype).transpose(1, 2) for t, x in ((m, h), (n, kv), (n, kv)))
    else:
        q, k, v = r(b, h, m, d).to(dtype), r(b, kv, n, d).to(dtype), r(b, kv, n, d).to(dtype)
    return q, k, v, r(h, buckets), r(b, h, m, d).to(dtype)


def _check(q, k, v, bias, go, buckets, causal, lengths, start, train, scale=None):
    from keops_amd.torch import bucket_attention

    s = q.shape[-1] ** -0.5 if scale is None else scale
    want = ref.attention(q, k, v, bias, buckets._host[0], causal, lengths, start, s, go if train else None)
    leaves = [t.detach().requires_grad_(train) for t in (q, k, v, bias)]
    out = bucket_attention(*leaves, buckets, causal=causal, key_lengths=lengths, query_start=start, scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype
    ref.assert_within(out.detach(), want["out"], want["tol_out"], "out")
    if train:
        grads = torch.autograd.grad(out, leaves, go)
        for name, g, leaf in zip(("q", "k", "v", "bias"), grads, leaves):
            assert g.shape == leaf.shape and g.dtype == leaf.dtype
            ref.assert_within(g, want["grad_" + name], want["tol_grad_" + name], "grad_" + name)
    return out


# batch, heads, kv_heads, queries, keys, dim, causal, both directions, lengths, start
CASES = [
    (2, 4, 2, 100, 130, 64, False, True, None, 0),
    (1, 2, 2, 1, 1, 64, True, False, None, 0),
    (2, 2, 1, 3, 70, 32, True, False, [70, 9], [67, 6]),            # few rows
    (2, 4, 4, 129, 129, 128, True, False, None, 0),
    (1, 3, 1, 65, 257, 96, True, False, None, 192),
    (3, 2, 2, 40, 300, 40, False, True, [300, 1, 0], 0),            # a sequence without keys
    (2, 2, 2, 70, 90, 72, True, True, [90, 50], [-30, 25]),         # rows before the first key
    (1, 2, 2, 200, 64, 16, False, True, None, -400),                # all keys beyond the reach, to the right
    (1, 2, 2, 64, 200, 24, False, True, None, 900),                 # and to the left
    (1, 1, 1, 400, 400, 80, False, False, None, 0),
    (2, 6, 3, 1, 700, 64, True, False, [700, 333], [699, 332]),     # one token against a cache
    (1, 8, 1, 4, 2500, 128, True, False, None, 2496),               # 32 rows, shares of a cache
    (1, 2, 1, 33, 0, 64, False, True, None, 0),                     # no keys at all
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("case", CASES)
def test_values_and_gradients(case, dtype):
    from keops_amd.torch import PositionBuckets

    b, h, kv, m, n, d, causal, both, lengths, start = case
    q, k, v, bias, go = _make(dtype, b, h, kv, m, n, d)
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    start = torch.tensor(start, device="cuda") if isinstance(start, list) else start
    _check(q, k, v, bias, go, PositionBuckets(32, 128, both), causal, lengths, start, True)


@pytest.mark.parametrize("num_buckets,max_distance,both", [(4, 2, True), (64, 512, False), (64, 1024, True)])
def test_reach_of_the_buckets(num_buckets, max_distance, both):
    from keops_amd.torch import PositionBuckets

    q, k, v, bias, go = _make(BF16, 1, 2, 2, 300, 700, 64, num_buckets)
    _check(q, k, v, bias, go, PositionBuckets(num_buckets, max_distance, both), False, None, 150, True)


def test_any_map_of_positions():
    from keops_amd.torch import PositionBuckets

    gen = torch.Generator().manual_seed(3)
    buckets = PositionBuckets.from_map(torch.randint(0, 7, (41,), generator=gen), num_buckets=9)  # buckets that no position has
    q, k, v, bias, go = _make(FP32, 2, 2, 2, 90, 75, 32, 9)
    _check(q, k, v, bias, go, buckets, False, None, 0, True, scale=0.4)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_dims_and_strides_that_are_copied_first(dtype):
    from keops_amd.torch import PositionBuckets

    gen = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dtype)
    buckets = PositionBuckets(32, 128, True)
    bias = torch.randn(3, 32, device="cuda", generator=gen)
    for d in (1, 7, 20, 100):
        _check(r(2, 3, 50, d), r(2, 1, 60, d), r(2, 1, 60, d), bias, r(2, 3, 50, d), buckets, True, None, 5, True)
    q = r(2, 3, 33, 50)[..., 1:].transpose(2, 3)                            # components are not neighbours, rows not aligned
    k = r(2, 1, 60, 33 + 8)[..., 3:36]
    v = r(1, 1, 60, 33).expand(2, 1, 60, 33)                                # one sequence's values for all
    go = r(2, 3, 49, 1).expand(2, 3, 49, 33)
    _check(q, k, v, bias, go, buckets, False, None, 0, True)


def test_bias_in_the_type_of_q_and_broadcast_inputs():
    from keops_amd.torch import PositionBuckets, bucket_attention

    buckets = PositionBuckets(16, 64, True)
    q, k, v, bias, go = _make(BF16, 2, 4, 2, 50, 60, 64, 16)
    half = bias.to(BF16).requires_grad_(True)
    one = v[:1].detach().clone().requires_grad_(True)
    out = bucket_attention(q, k, one.expand(2, -1, -1, -1), half, buckets)
    gb, gv = torch.autograd.grad(out, (half, one), go)
    want = ref.attention(q, k, v[:1].expand(2, -1, -1, -1), half.detach().float(), buckets._host[0], False, None, 0, 0.125, go)
    assert gb.dtype == BF16
    ref.assert_within(gb, want["grad_bias"], want["tol_grad_bias"] + ref.u(BF16) * want["grad_bias"].abs(), "grad_bias")
    # two gradients, each rounded, and their sum rounded
    tol = want["tol_grad_v"].sum(0, keepdim=True) * (1 + 2 * ref.u(BF16)) + ref.u(BF16) * want["grad_v"].sum(0, keepdim=True).abs()
    ref.assert_within(gv, want["grad_v"].sum(0, keepdim=True), tol, "grad_v")


def test_what_lies_behind_the_lengths_is_not_read():
    from keops_amd.torch import PositionBuckets

    buckets = PositionBuckets(32, 128, False)
    for m, d in ((1, 64), (90, 64), (90, 40)):
        q, k, v, bias, go = _make(BF16, 3, 4, 2, m, 200, d, by_token=False)
        lengths = torch.tensor([200, 77, 0], dtype=torch.int64, device="cuda")
        for i, n in enumerate(lengths.tolist()):
            k[i, :, n:], v[i, :, n:] = math.nan, math.inf
        out = _check(q, k, v, bias, go, buckets, False, lengths, 100, True)
        assert out.isfinite().all() and (out[2] == 0).all()


def test_values_that_are_not_finite_stay_in_their_rows():
    from keops_amd.torch import PositionBuckets, bucket_attention

    buckets = PositionBuckets(32, 128, True)
    q, k, v, bias, _ = _make(FP32, 1, 2, 2, 100, 100, 64)
    q[0, 0, 7] = math.nan
    out = bucket_attention(q, k, v, bias, buckets)
    assert out[0, 0, 7].isnan().all() and out.isnan().sum() == 64


def test_large_logits_and_lowest_biases():
    from keops_amd.torch import PositionBuckets

    buckets = PositionBuckets(8, 16, True)
    q, k, v, bias, go = _make(FP32, 1, 2, 2, 70, 90, 32, 8)
    bias[:, 3] = torch.finfo(FP32).min / 4     # a bucket that is as good as masked
    _check(q, k, v, bias.clamp(min=-1e4), go, buckets, False, None, 0, True)
    from keops_amd.torch import bucket_attention

    out = bucket_attention(q, k, v, bias, buckets)
    away = torch.arange(90, device="cuda") - torch.arange(70, device="cuda")[:, None]
    z = (q.double() @ k.double().transpose(-1, -2)) * 32 ** -0.5 + bias.double()[:, buckets(away)]
    assert (out.double() - torch.softmax(z, -1) @ v.double()).abs().max() < 1e-5
    _check(q * 8, k * 8, v, bias.clamp(min=-1e4), go, buckets, False, None, 0, False)  # logits of some hundreds
    out = bucket_attention(q, k, v, torch.full_like(bias, -math.inf), buckets)          # every pair masked by its bias
    assert (out == 0).all()


def test_rows_of_a_cache_beyond_32_bit_offsets():
    from keops_amd.torch import PositionBuckets

    step, n, d = 1 << 20, 2200, 64  # elements between rows: the last ones lie beyond 2^31
    store = torch.empty(n * step, dtype=BF16, device="cuda")
    k = store.as_strided((1, 1, n, d), (n * step, n * step, step, 1))
    v = store.as_strided((1, 1, n, d), (n * step, n * step, step, 1), 512)
    gen = torch.Generator(device="cuda").manual_seed(5)
    k.copy_(torch.randn(1, 1, n, d, device="cuda", generator=gen))
    v.copy_(torch.randn(1, 1, n, d, device="cuda", generator=gen))
    for m in (1, 40):
        q = torch.randn(1, 2, m, d, device="cuda", generator=gen).to(BF16)
        bias, go = torch.randn(2, 32, device="cuda", generator=gen), torch.randn(1, 2, m, d, device="cuda", generator=gen).to(BF16)
        _check(q, k, v, bias, go, PositionBuckets(32, 128, False), True, None, n - m, m > 1)


def test_gradients_against_differences():
    from keops_amd.torch import PositionBuckets, bucket_attention

    buckets = PositionBuckets(16, 64, True)
    q, k, v, bias, go = _make(FP32, 1, 2, 1, 45, 50, 32, 16, seed=9)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, bias)]
    f = lambda ts: (bucket_attention(*ts, buckets, causal=True, query_start=3).double() * go.double()).sum()
    grads = torch.autograd.grad(f(leaves), leaves)
    for i, g in enumerate(grads):
        w = torch.randn_like(leaves[i])
        eps = 1e-3 * float(leaves[i].detach().norm() / w.norm())
        moved = lambda e: [t.detach() + (e * w if j == i else 0) for j, t in enumerate(leaves)]
        diff = float(f(moved(eps)) - f(moved(-eps))) / (2 * eps)
        size = float((g.abs() * w.abs()).sum())
        # float32 values of a sum of 2880 terms, differenced over 2 eps, and the third-order term of the difference
        assert abs(diff - float((g * w).sum())) < 1e-3 * size, i


def test_graph_streams_and_repeats():
    from keops_amd.torch import PositionBuckets, bucket_attention

    buckets = PositionBuckets(32, 128, False)

    def step(q, k, v, bias, go):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, bias)]
        out = bucket_attention(*leaves, buckets, causal=True)
        return (out.detach(), *torch.autograd.grad(out, leaves, go))

    data = _make(BF16, 2, 4, 2, 150, 150, 64)
    token = _make(BF16, 2, 4, 2, 1, 3000, 64)
    run = lambda: step(*data) + (bucket_attention(*token[:4], buckets, causal=True, query_start=2999),)
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
    for i in range(3):
        for t in (*data, *token):
            t.copy_(torch.randn(t.shape, device="cuda"))
        want = run()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    # both graphs at once, on streams of their own
    for (g, _), s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n", [(64, 2), (1, 2), (70, 4000), (1, 4000), (33, 257)])
def test_what_the_rounding_of_the_output_leaves(m, n, dtype):
    """All logits equal, so outputs are means: a training call keeps a second term of them for the gradient's row sums.  Two terms are
    off by half a step of half a step, the sum of n values by a step of float32 for each, and by the underflow of the second term."""
    from keops_amd.torch import PositionBuckets, bucket_attention

    gen = torch.Generator(device="cuda").manual_seed(3)
    q = torch.zeros(2, 2, m, 48, device="cuda", dtype=dtype, requires_grad=True)
    k, v = (torch.randn(2, 2, n, 48, device="cuda", generator=gen).to(dtype) for _ in range(2))
    out = bucket_attention(q, k, v, torch.zeros(2, 32, device="cuda"), PositionBuckets())
    rest = out.grad_fn.saved_tensors[5]
    mean, size = v.double().mean(2, keepdim=True), v.double().abs().mean(2, keepdim=True)
    half = torch.finfo(dtype).eps / 2
    ref.assert_within(out.double() + rest.double(), mean.expand_as(out), (half ** 2 * mean.abs() + (n + 4) * 2.0 ** -23 * size + 2.0 ** -25).expand_as(out), "two terms")
    assert rest.stride() == out.stride() and bool((rest != 0).any())


def test_single_ones_may_have_any_stride_and_numbers_any_type():
    from keops_amd.torch import PositionBuckets, bucket_attention

    gen = torch.Generator(device="cuda").manual_seed(9)
    base = torch.randn(150 * 64 + 8, device="cuda", generator=gen).bfloat16()
    q, k = base.as_strided((1, 1, 70, 64), (5, 3, 64, 1)), base.as_strided((1, 1, 150, 64), (9, 1, 64, 1), 8)
    bias, b = torch.randn(1, 32, device="cuda", generator=gen), PositionBuckets()
    dense = bucket_attention(q.contiguous(), k.contiguous(), k.contiguous(), bias, b, scale=0.5)
    far = torch.tensor([2 ** 40], device="cuda")  # more keys than there are
    assert torch.equal(bucket_attention(q, k, k, bias, b, scale=0.5, key_lengths=far), dense)
    scale = torch.tensor(1.0)
    bucket_attention(q, k, k, bias, b, scale=scale)
    scale.mul_(0.5)
    assert torch.equal(bucket_attention(q, k, k, bias, b, scale=scale), dense)
    # no keys, cut out of others
    assert (bucket_attention(q, k[:, :, 3:3, :], k[:, :, 3:3, :], bias, b) == 0).all()


def test_refusals_on_the_device():
    from keops_amd.torch import PositionBuckets, bucket_attention

    b = PositionBuckets()
    q, k, v, bias, _ = _make(BF16, 2, 4, 2, 5, 6, 16)
    ok = dict(q=q, k=k, v=v, bias=bias, buckets=b)
    ints = torch.zeros(2, dtype=torch.int32, device="cuda")
    for change, match in [(dict(q=q.double()), "float32"), (dict(k=k.float()), "one type"), (dict(v=v[:, :, :5]), "kv_heads"), (dict(q=q[:, :3]), "do not fit"),
                          (dict(bias=bias[:, :31]), "bias"), (dict(bias=bias.half()), "bias"), (dict(bias=bias.cpu()), "HIP device"),
                          (dict(key_lengths=ints[:1]), "key_lengths"), (dict(key_lengths=ints.cpu()), "same device"),
                          (dict(query_start=2.5), "query_start"), (dict(query_start=1 << 30), "query_start"), (dict(q=q[0]), "must be"),
                          (dict(q=q[..., :0], k=k[..., :0], v=v[..., :0]), "dim")]:
        with pytest.raises(ValueError, match=match):
            bucket_attention(**{**ok, **change})
    for change, match in [(dict(buckets=32), "PositionBuckets"), (dict(key_lengths=[5, 6]), "int32"), (dict(key_lengths=ints.float()), "int32")]:
        with pytest.raises(TypeError, match=match):
            bucket_attention(**{**ok, **change})
    big = torch.zeros(1, 1, 2, 136, device="cuda")
    with pytest.raises(ValueError, match="dim must be"):
        bucket_attention(big, big, big, torch.zeros(1, 32, device="cuda"), b)
    out = bucket_attention(q.detach().requires_grad_(True), k, v, bias, b)
    (g,) = torch.autograd.grad(out.sum(), out, create_graph=True)
    with pytest.raises(RuntimeError):  # first order only
        x = q.detach().requires_grad_(True)
        (gx,) = torch.autograd.grad(bucket_attention(x, k, v, bias, b).float().square().sum(), x, create_graph=True)
        gx.float().sum().backward()
    empty = bucket_attention(q[:, :, :0].detach().requires_grad_(True), k, v, bias, b)
    assert empty.shape == (2, 4, 0, 16)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,n,causal,lengths", [(40, 1500, False, [1500, 700]), (1100, 1100, True, None), (1300, 90, False, [90, 0])])
def test_walks_shared_by_workgroups(m, n, causal, lengths, dtype):
    """Few blocks and long walks: shares of the keys (forward, gradient of q) and of the queries (gradients of k and v), joined."""
    from keops_amd.torch import PositionBuckets

    for d, h, kv in ((64, 2, 1), (96, 1, 1)):
        q, k, v, bias, go = _make(dtype, 2, h, kv, m, n, d, seed=m + d)
        lens = None if lengths is None else torch.tensor(lengths, device="cuda")
        _check(q, k, v, bias, go, PositionBuckets(32, 128, True), causal, lens, 0, True)

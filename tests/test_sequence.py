"""Sequence operators on the CPU: buckets of relative positions, what the entry points refuse, and the 64-bit references that the
device tests use (against torch's autograd and against differences)."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

import sequence_reference as ref
from keops_amd import binder
from keops_amd.torch import PositionBuckets, bucket_attention, decay_attention, decay_attention_step, token_logprobs


@pytest.mark.parametrize("num_buckets,max_distance,both", [(32, 128, True), (32, 128, False), (4, 2, True), (2, 2, False), (16, 64, True),
                                                           (64, 64, False), (64, 1024, True), (17, 100, False)])
def test_buckets_follow_their_definition(num_buckets, max_distance, both):
    b = PositionBuckets(num_buckets, max_distance, both)
    x = torch.arange(-2 * max_distance, 2 * max_distance + 1)
    got = b(x)
    assert got.tolist() == [ref.bucket(int(r), num_buckets, max_distance, both) for r in x]
    assert 0 <= int(got.min()) and int(got.max()) < num_buckets and b.reach <= max_distance
    assert bool((b(torch.tensor([-b.reach, -b.reach - 1, -10**6])) == b(torch.tensor([-b.reach]))).all())


def test_bucket_tables_of_the_device_code():
    b = PositionBuckets.from_map([2, 0, 0, 1, 2], num_buckets=4)
    of, order, begin = b._host
    assert of.tolist() == [2, 0, 0, 1, 2] and order.tolist() == [1, 2, 3, 0, 4] and begin.tolist() == [0, 2, 3, 5, 5]
    assert b.reach == 2 and b(torch.tensor([-9, -2, -1, 0, 1, 2, 9])).tolist() == [2, 2, 0, 0, 1, 2, 2]


@pytest.mark.parametrize("make", [
    lambda: PositionBuckets(31, 128, True), lambda: PositionBuckets(2, 128, True), lambda: PositionBuckets(1, 128, False),
    lambda: PositionBuckets(32, 8, True), lambda: PositionBuckets(62, 30, True), lambda: PositionBuckets(32, 4096, True), lambda: PositionBuckets.from_map([0, 1]),
    lambda: PositionBuckets.from_map([0]), lambda: PositionBuckets.from_map([0, -1, 0]), lambda: PositionBuckets.from_map([0, 1, 2], 2),
    lambda: PositionBuckets.from_map([0, 0, 0], 4), lambda: PositionBuckets.from_map([0] * 2051)])
def test_buckets_that_are_refused(make):
    with pytest.raises(ValueError, match="PositionBuckets"):
        make()


def test_host_tensors_and_types_are_refused():
    q = torch.zeros(1, 2, 3, 8)
    b = PositionBuckets()
    with pytest.raises(ValueError, match="HIP device"):
        bucket_attention(q, q, q, torch.zeros(2, 32), b)
    with pytest.raises(ValueError, match="HIP device"):
        decay_attention(q, q, q, torch.zeros(2))
    with pytest.raises(ValueError, match="HIP device"):
        decay_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], torch.zeros(2), torch.zeros(1, 2, 8, 8))
    with pytest.raises(ValueError, match="HIP device"):
        token_logprobs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError, match="torch tensor"):
        bucket_attention([1.0], q, q, torch.zeros(2, 32), b)


# The library's own checks come before anything touches a device, so they are tested here; the pointers below are never followed.
def _attention_args(**changes):
    a = binder.BucketAttention()
    a.dtype, a.batch, a.heads, a.kv_heads, a.dim, a.buckets, a.reach, a.queries, a.keys, a.scale = 0, 2, 4, 2, 64, 32, 91, 40, 50, 0.125
    for name in ("q", "k", "v", "out", "bias", "bucket_of", "bucket_order", "bucket_begin", "grad_out", "grad_k", "grad_v", "lse", "delta",
                 "grad_bias"):
        setattr(a, name, 1 << 12)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=3), "dtype"), (dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "kv_heads"), (dict(dim=12), "dim"),
    (dict(dim=136), "dim"), (dict(queries=0), "queries"), (dict(keys=-1), "keys"), (dict(keys=1 << 30), "keys"), (dict(reach=0), "reach"),
    (dict(reach=1025), "reach"), (dict(buckets=184), "buckets"), (dict(start=1 << 30), "query_start"), (dict(q=None), "null"),
    (dict(v=None), "null"), (dict(batch=1 << 20, heads=1 << 14, kv_heads=1), "workgroups")])
def test_attention_arguments_that_the_library_refuses(changes, message):
    a = _attention_args(**changes)
    for backward in (False, True):
        fn = binder.lib().keops_hip_bucket_attention_backward if backward else binder.lib().keops_hip_bucket_attention_forward
        assert fn(ctypes.byref(a), None, 0, 0, None) != 0
        assert message in binder.last_error() and "bucket attention" in binder.last_error()
    assert binder.lib().keops_hip_bucket_attention_forward_bytes(ctypes.byref(a)) == 0


def test_attention_workspaces():
    lib = binder.lib()
    a = _attention_args()
    need = lib.keops_hip_bucket_attention_backward_bytes(ctypes.byref(a))
    assert need == 2 * 1 * 4 * 32 * 4
    long = _attention_args(queries=3000, keys=3000)  # few blocks: shares of their walks are joined
    assert lib.keops_hip_bucket_attention_forward_bytes(ctypes.byref(long)) >= 2 * 4 * 3000 * 64 * 4
    assert lib.keops_hip_bucket_attention_backward_bytes(ctypes.byref(long)) > lib.keops_hip_bucket_attention_forward_bytes(ctypes.byref(long))
    assert lib.keops_hip_bucket_attention_backward(ctypes.byref(a), 1 << 12, need - 1, 0, None) != 0 and "workspace" in binder.last_error()
    assert lib.keops_hip_bucket_attention_forward_bytes(ctypes.byref(a)) == 0
    few = _attention_args(queries=1, keys=100000)
    need = lib.keops_hip_bucket_attention_forward_bytes(ctypes.byref(few))
    assert need > 0
    assert lib.keops_hip_bucket_attention_forward(ctypes.byref(few), None, 0, 0, None) != 0 and "workspace" in binder.last_error()
    assert lib.keops_hip_bucket_attention_backward(ctypes.byref(_attention_args(grad_k=None)), 1 << 12, 1 << 20, 0, None) != 0
    assert "null" in binder.last_error()
    assert lib.keops_hip_bucket_attention_forward(None, None, 0, 0, None) != 0


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=-1), "dtype"), (dict(q_heads=3), "multiple"), (dict(k_heads=0), "multiple"), (dict(dim=20), "dim"), (dict(dim_v=256), "dim"),
    (dict(tokens=-1), "tokens"), (dict(log_decay=None), "null"), (dict(out=None), "null"), (dict(batch=65536), "65535")])
def test_decay_arguments_that_the_library_refuses(changes, message):
    a = binder.DecayAttention()
    a.dtype, a.batch, a.heads, a.q_heads, a.k_heads, a.v_heads, a.dim, a.dim_v, a.tokens = 0, 2, 4, 4, 2, 2, 64, 64, 100
    for name in ("q", "k", "v", "out", "log_decay"):
        setattr(a, name, 1 << 12)
    for name, value in changes.items():
        setattr(a, name, value)
    lib = binder.lib()
    assert lib.keops_hip_decay_attention_run(ctypes.byref(a), 0, None) != 0
    assert message in binder.last_error() and "decay attention" in binder.last_error()
    assert lib.keops_hip_decay_attention_bytes(ctypes.byref(a)) == 0


def test_decay_workspaces():
    lib = binder.lib()
    a = binder.DecayAttention()
    a.dtype, a.batch, a.heads, a.q_heads, a.k_heads, a.v_heads, a.dim, a.dim_v, a.tokens = 0, 1, 2, 2, 2, 2, 64, 64, 64
    for name in ("q", "k", "v", "out", "log_decay"):
        setattr(a, name, 1 << 12)
    assert lib.keops_hip_decay_attention_bytes(ctypes.byref(a)) == 0  # one chunk: nothing to carry
    a.tokens = 6400
    need = lib.keops_hip_decay_attention_bytes(ctypes.byref(a))
    assert need > 0 and need % (2 * 64 * 64 * 4) == 0
    a.states, a.states_bytes = 1 << 12, need - 1
    assert lib.keops_hip_decay_attention_run(ctypes.byref(a), 0, None) != 0 and "workspace" in binder.last_error()
    a.states_bytes, a.states_given, a.state_out = need, 1, 1 << 12
    assert lib.keops_hip_decay_attention_run(ctypes.byref(a), 0, None) != 0 and "final state" in binder.last_error()


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_decay_states_serve_the_walks_with_exchanged_dims(dtype):
    """A training step's walks share the states before the segments, so both must cut the sequences alike."""
    lib = binder.lib()
    for units in (1, 2, 24, 192, 400):
        for tokens in (64, 65, 265, 1000, 9000):
            for d, dv in ((40, 128), (64, 72), (8, 64), (128, 128), (72, 8)):
                need = []
                for x, y in ((d, dv), (dv, d)):
                    a = binder.DecayAttention(dtype=dtype, batch=1, heads=units, q_heads=units, k_heads=units, v_heads=units, dim=x, dim_v=y, tokens=tokens)
                    for name in ("q", "k", "v", "out", "log_decay"):
                        setattr(a, name, 16)
                    need.append(lib.keops_hip_decay_attention_bytes(ctypes.byref(a)))
                assert need[0] == need[1], (units, tokens, d, dv)
    a.heads = a.q_heads = a.k_heads = a.v_heads = 24  # (few enough for segments)
    a.tokens, a.states, a.states_given = 9000, 16, 1
    need = lib.keops_hip_decay_attention_bytes(ctypes.byref(a))
    for size in (need + 16, need - 16):  # states of other segments
        a.states_bytes = size
        assert lib.keops_hip_decay_attention_run(ctypes.byref(a), 0, None) != 0
    assert "too small" in binder.last_error()
    a.states_bytes = need + 16
    assert lib.keops_hip_decay_attention_run(ctypes.byref(a), 0, None) != 0 and "segments" in binder.last_error()


def test_rows_off_16_bytes_are_refused_by_the_library():
    lib = binder.lib()
    for changes in (dict(q=24), dict(k_stride=(0, 0, 4)), dict(out_stride=(4, 0, 64)), dict(v_stride=(0, 2, 64)), dict(state_in=8)):
        a = binder.DecayAttention(dtype=0, batch=1, heads=1, q_heads=1, k_heads=1, v_heads=1, dim=64, dim_v=64, tokens=8)
        b = binder.BucketAttention(dtype=0, batch=1, heads=1, kv_heads=1, dim=64, queries=8, keys=8, buckets=3, reach=1)
        for x in (a, b):
            for name in ("q", "k", "v", "out", "log_decay", "bias", "bucket_of"):
                if hasattr(x, name):
                    setattr(x, name, 16)
            for name, value in changes.items():
                if not hasattr(x, name):
                    break
                setattr(x, name, (ctypes.c_int64 * 3)(*value) if isinstance(value, tuple) else value)
            else:
                rc = (lib.keops_hip_decay_attention_run(ctypes.byref(a), 0, None) if x is a
                      else lib.keops_hip_bucket_attention_forward(ctypes.byref(b), None, 0, 0, None))
                assert rc != 0 and "16 bytes" in binder.last_error(), changes


@pytest.mark.parametrize("changes", [dict(joined_heads=2), dict(joined_heads=3, out_float32=1, joined=16), dict(joined_heads=2, out_float32=1),
                                     dict(joined_heads=-1, out_float32=1, joined=16)])
def test_joined_outputs_that_the_library_refuses(changes):
    a = binder.DecayAttention(dtype=0, batch=1, heads=4, q_heads=4, k_heads=4, v_heads=4, dim=64, dim_v=64, tokens=8)
    for name in ("q", "k", "v", "out", "log_decay"):
        setattr(a, name, 16)
    for name, value in changes.items():
        setattr(a, name, value)
    assert binder.lib().keops_hip_decay_attention_run(ctypes.byref(a), 0, None) != 0 and "joined" in binder.last_error()


def test_copies_and_pickles_of_buckets_hold_the_map_alone():
    """A plan holds the addresses of the tables of the object that made it: no copy may take it along."""
    b = PositionBuckets(16, 40, False)
    b._plans["geometry"], b._device[torch.device("cpu")] = "plan", b._host
    for c in (copy.copy(b), copy.deepcopy(b), pickle.loads(pickle.dumps(b))):
        assert c is not b and not c._plans and not c._device
        assert (c.num_buckets, c.reach) == (b.num_buckets, b.reach) and all(map(torch.equal, c._host, b._host))


def test_first_use_of_buckets_inside_of_a_capture_is_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        PositionBuckets().on("cuda:0")


def test_step_and_logprob_arguments_that_the_library_refuses():
    lib = binder.lib()
    two = (ctypes.c_int64 * 2)(64, 64)
    data = (1 << 12, two, 1 << 12, two, 1 << 12, two, 1 << 12, 1 << 12, 1 << 12)
    for head, message in (((0, 0, 4, 2, 64, 64), "heads"), ((0, 1, 4, 3, 64, 64), "heads"), ((5, 1, 4, 2, 64, 64), "dtype"),
                          ((0, 1, 4, 2, 64, 66), "dim_v"), ((0, 1, 4, 2, 130, 64), "dim")):
        assert lib.keops_hip_decay_attention_step(*head, 1.0, *data, 0, None) != 0
        assert message in binder.last_error()
    assert lib.keops_hip_decay_attention_step(0, 1, 4, 2, 64, 64, 1.0, None, *data[1:], 0, None) != 0 and "null" in binder.last_error()

    def call(dtype, rows, vocab, top, logits=1 << 12):
        return lib.keops_hip_token_logprobs(dtype, rows, vocab, top, logits, vocab, 1 << 12, -100, *[1 << 12] * 5, None, 0, 0, None)

    for args, message in (((3, 2, 10, 0), "dtype"), ((0, -1, 10, 0), "rows"), ((0, 2, 0, 0), "vocabulary"), ((0, 2, 1 << 31, 0), "vocabulary"),
                          ((0, 2, 100, 65), "top"), ((0, 2, 10, 11), "top"), ((0, 2, 300000, 3), "workspace"), ((0, 2, 10, 1, None), "null")):
        assert call(*args) != 0, args
        assert message in binder.last_error(), (args, binder.last_error())
    assert call(0, 0, 10, 0) == 0  # no rows: nothing to do
    assert lib.keops_hip_token_logprobs_backward(0, 2, 10, 0, None, 10, None, -100, *[None] * 6, None, 10, 0, None) != 0
    assert "null" in binder.last_error()


def test_reference_attention_against_autograd_and_differences():
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    q, k, v, bias, go = r(2, 4, 5, 8), r(2, 2, 7, 8), r(2, 2, 7, 8), r(4, 6), r(2, 4, 5, 8)
    b = PositionBuckets.from_map([0, 1, 2, 3, 4, 5, 5])
    lengths, start = torch.tensor([7, 3]), torch.tensor([2, -1])

    def plain(q, k, v, bias):
        k, v = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        away = torch.arange(7) - (start[:, None, None] + torch.arange(5)[:, None])
        z = q @ k.transpose(-1, -2) * 0.3 + bias[:, b(away)].permute(1, 0, 2, 3)
        seen = ((away <= 0) & (torch.arange(7) < lengths[:, None, None]))[:, None]
        e = torch.where(seen, z.exp(), torch.zeros_like(z))
        return (e / e.sum(-1, keepdim=True).clamp(min=1e-300)) @ v

    leaves = [t.requires_grad_(True) for t in (q, k, v, bias)]
    grads = torch.autograd.grad((plain(*leaves) * go).sum(), leaves)
    got = ref.attention(*(t.detach() for t in leaves), b._host[0], True, lengths, start, 0.3, go)
    assert torch.allclose(got["out"], plain(*leaves).detach(), atol=1e-12)
    assert got["out"][1, :, 0].abs().max() == 0  # a row that sees nothing
    for name, g in zip(("q", "k", "v", "bias"), grads):
        assert torch.allclose(got["grad_" + name], g, atol=1e-11), name
    for t, name in zip(leaves, ("q", "k", "v", "bias")):  # directional differences
        w = torch.randn(t.shape, generator=gen, dtype=torch.float64)
        f = lambda e: (plain(*[(x + e * w if x is t else x).detach() for x in leaves]) * go).sum()
        assert math.isclose(float((f(1e-6) - f(-1e-6)) / 2e-6), float((got["grad_" + name] * w).sum()), rel_tol=1e-6, abs_tol=1e-7)


def test_reference_decay_against_autograd():
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    q, k, v, S, go, gs = r(2, 4, 9, 5), r(2, 2, 9, 5), r(2, 2, 9, 3), r(2, 4, 5, 3), r(2, 4, 9, 3), r(2, 4, 5, 3)
    ld, lengths = torch.tensor([-0.1, -0.5, -2.0, 0.0], dtype=torch.float64), torch.tensor([9, 4])
    leaves = [t.requires_grad_(True) for t in (q, k, v, S)]

    def plain(q, k, v, S):  # the quadratic form
        k, v = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        pos = torch.arange(9)
        there = (pos < lengths[:, None])[:, None, :, None].double()
        q, k, v = q * there, k * there, v * there
        away = pos[:, None] - pos
        w = torch.where(away >= 0, torch.exp(away.clamp(min=0) * ld[:, None, None]), torch.zeros((), dtype=torch.float64))
        out = ((q @ k.transpose(-1, -2)) * w) @ v + (q @ S) * torch.exp((pos + 1) * ld[:, None])[None, :, :, None]
        left = torch.exp((lengths[:, None, None] - 1 - pos).clamp(min=0) * ld[:, None])
        return out * 0.7, (k * left[..., None]).transpose(-1, -2) @ v + S * torch.exp(lengths[:, None] * ld)[..., None, None]

    out, last = plain(*leaves)
    grads = torch.autograd.grad((out * go).sum() + (last * gs).sum(), leaves)
    got = ref.decay(*(t.detach() for t in (q, k, v)), ld, S.detach(), lengths, 0.7, go, gs)
    assert torch.allclose(got["out"], out.detach(), atol=1e-12) and torch.allclose(got["state"], last.detach(), atol=1e-12)
    for name, g in zip(("q", "k", "v", "state"), grads):
        assert torch.allclose(got["grad_" + name], g, atol=1e-11), name


def test_reference_logprobs_against_autograd():
    gen = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    x, tok = r(4, 11).requires_grad_(True), torch.tensor([3, 0, -100, 10])
    a, c, gt = r(4), r(4), r(4, 3)
    lp = torch.log_softmax(x, -1)
    ent = -(lp.exp() * lp).sum(-1)
    got = ref.logprobs(x.detach(), tok, 3, grads=(a, c, gt))
    pick = torch.where(tok == -100, torch.zeros(4, dtype=torch.float64), lp.gather(-1, tok.clamp(min=0)[:, None])[:, 0])
    assert torch.allclose(got["logprob"], pick.detach()) and torch.allclose(got["entropy"], ent.detach())
    loss = (pick * a).sum() + (ent * c).sum() + (lp.gather(-1, got["top_index"]) * gt).sum()
    assert torch.allclose(got["grad"], torch.autograd.grad(loss, x)[0], atol=1e-12)

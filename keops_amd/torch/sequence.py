"""Sequence operators: three of the engine's reductions in the form in which models of token sequences use them, where no
formula can express them (a table looked up by position, a causal bound, shared heads, 16-bit types).

=========================  =====================================================  ==============================
:func:`bucket_attention`   softmax-weighted sum over keys (``SumSoftMaxWeight``)  learned bias by position bucket
:func:`decay_attention`    sum over past tokens (``Sum``) in linear time          decay for each head, carried state
:func:`token_logprobs`     ``LogSumExp`` and K largest values of rows of logits   log probability, entropy, alternatives
=========================  =====================================================  ==============================

Tensors live on one HIP device, in bfloat16, float16 or float32; sums, softmax statistics and states are float32.  Launches go to
the current stream of that device and can be captured in a HIP graph (for :class:`PositionBuckets`, after a first use on the
device outside the capture).  Results do not depend on the order in which workgroups run.  Gradients are of first order.
"""
import ctypes
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import binder

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_MAX_ROW_STRIDE = 1 << 23  # kMaxRowStride of csrc/sequence/keops_seq.h
_MAX_PLANS = 512
_raw_stream = torch._C._cuda_getCurrentRawStream  # hipStream_t of a device's current stream


def _check_data(what, **tensors):
    """All on one HIP device, all of one supported type."""
    device = dtype = None
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"[KeOps] {what}: {name} must be a torch tensor, got {type(t)}.")
        if not t.is_cuda:
            raise ValueError(f"[KeOps] {what}: {name} must be on a HIP device, it is on {t.device}.")
        if device is not None and t.device != device:
            raise ValueError("[KeOps] Input arrays must be all located on the same device.")
        if t.dtype not in _DTYPES:
            raise ValueError(f"[KeOps] {what}: {name} must be bfloat16, float16 or float32, it is {t.dtype}.")
        if dtype is not None and t.dtype != dtype:
            raise ValueError(f"[KeOps] {what}: {', '.join(tensors)} must be of one type, got {dtype} and {t.dtype}.")
        device, dtype = t.device, t.dtype
    return device, dtype


def _check_whole(what, name, t, shape, device):
    """An int32 / int64 tensor of this shape on this device, as int32."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"[KeOps] {what}: {name} must be an int32 or int64 tensor.")
    if t.device != device:
        raise ValueError("[KeOps] Input arrays must be all located on the same device.")
    if t.shape != shape:
        raise ValueError(f"[KeOps] {what}: {name} must be of shape {tuple(shape)}, got {tuple(t.shape)}.")
    if t.dtype is torch.int32 and t.is_contiguous():
        return t
    if t.dtype is torch.int64:  # (whole numbers that int32 does not hold mean the same as its ends)
        t = t.clamp(-2**31, 2**31 - 1)
    return t.to(torch.int32).contiguous()


def _strides_fit(x):
    """Rows as the kernels read them: neighbouring components, every row a multiple of 16 bytes from the first and not too far
    from the next."""
    size = x.element_size()
    shape, stride = x.shape, x.stride()
    return x.numel() == 0 or (
        (stride[-1] == 1 or shape[-1] == 1) and (shape[-2] == 1 or stride[-2] <= _MAX_ROW_STRIDE)
        and all(s * size % 16 == 0 for s, n in zip(stride[:-1], shape[:-1]) if n > 1)
    )


def _rows(x):
    """x with rows as the kernels read them, a copy if they are not."""
    return x if _strides_fit(x) and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def _dense_strides(x):
    """Strides of a new tensor of x's shape: x's own where x is dense and they fit, else those of the contiguous order."""
    y = torch.empty_like(x, device="meta")
    return y.stride() if _strides_fit(y) else torch.empty(x.shape, device="meta").stride()


def _pad(x, *multiples):
    """x with zeros behind its last dimensions, up to multiples (given from the last dimension on)."""
    pad = []
    for k, m in enumerate(multiples):
        pad += [0, -x.shape[-1 - k] % m]
    return torch.nn.functional.pad(x, pad) if any(pad) else x


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stride(shape, stride):
    """Strides of batch, head and row as the library takes them (a single one has none)."""
    return tuple(s if n > 1 else 0 for n, s in zip(shape[:3], stride)) if 0 not in shape else (0, 0, 0)


def _geometry(t):
    """What a plan depends on of a tensor: everything but where it is."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _keep(plans, key, plan):
    if len(plans) >= _MAX_PLANS:
        plans.clear()
    plans[key] = plan
    return plan


# --------------------------------------------------------------------------------------------------- position buckets
class PositionBuckets:
    """Buckets of relative positions ``key - query``, for :func:`bucket_attention`.

    One bucket for each of the first distances, then buckets in equal steps of the logarithm up to ``max_distance``; everything
    farther shares the last one.  With ``bidirectional`` half of the buckets are for keys after the query, otherwise those share
    the bucket of distance 0.  The borders are whole numbers found without rounding: with n buckets for a direction, m = n // 2
    and t > 0, bucket m + t begins at the smallest distance d with (d / m)^(n - m) >= (max_distance / m)^t.

    ``PositionBuckets.from_map`` takes any other map.  Objects are immutable; their device copies are made at first use on a
    device.
    """

    MAX_REACH = 1024  # KEOPS_HIP_MAX_REACH

    def __init__(self, num_buckets=32, max_distance=128, bidirectional=True):
        count = num_buckets // 2 if bidirectional else num_buckets
        near = count // 2
        if num_buckets < (4 if bidirectional else 2) or (bidirectional and num_buckets % 2):
            raise ValueError("[KeOps] PositionBuckets: num_buckets must be at least 2 (bidirectional: an even number, at least 4).")
        if not near < max_distance <= self.MAX_REACH:
            raise ValueError(f"[KeOps] PositionBuckets: max_distance must be above {near} (the distances with a bucket of their "
                             f"own) and at most {self.MAX_REACH}.")
        if num_buckets > 2 * max_distance + 1:
            raise ValueError("[KeOps] PositionBuckets: more buckets than positions within max_distance.")
        steps, t, by_distance = count - near, 0, []
        for d in range(max_distance + 1):
            while d >= near and t + 1 < steps and d ** steps >= near ** (steps - t - 1) * max_distance ** (t + 1):
                t += 1
            by_distance.append(d if d < near else near + t)
        reach = max(by_distance.index(by_distance[-1]), num_buckets // 2)  # the tables hold at least one entry a bucket
        before = [by_distance[d] for d in range(reach, -1, -1)]
        after = [count + by_distance[d] for d in range(1, reach + 1)] if bidirectional else [0] * reach
        self._set(before + after, num_buckets)

    @classmethod
    def from_map(cls, bucket_of, num_buckets=None):
        """Buckets from a sequence of 2 * reach + 1 whole numbers: the bucket of each relative position ``key - query`` from
        ``-reach`` to ``reach``; positions beyond take that of the nearer end."""
        bucket_of = [int(b) for b in (bucket_of.tolist() if isinstance(bucket_of, torch.Tensor) else bucket_of)]
        if len(bucket_of) % 2 == 0 or len(bucket_of) < 3 or len(bucket_of) // 2 > cls.MAX_REACH:
            raise ValueError(f"[KeOps] PositionBuckets: the map must have 2 * reach + 1 entries, with reach from 1 to {cls.MAX_REACH}.")
        count = max(bucket_of) + 1 if num_buckets is None else int(num_buckets)
        if min(bucket_of) < 0 or max(bucket_of) >= count or count > len(bucket_of):
            raise ValueError("[KeOps] PositionBuckets: the map's entries must be from 0 to num_buckets - 1, and num_buckets at most "
                             "the number of entries.")
        self = cls.__new__(cls)
        self._set(bucket_of, count)
        return self

    def _set(self, bucket_of, num_buckets):
        self.num_buckets, self.reach = num_buckets, len(bucket_of) // 2
        order = sorted(range(len(bucket_of)), key=lambda i: (bucket_of[i], i))
        begin = [sum(b < k for b in bucket_of) for k in range(num_buckets + 1)]
        self._host = tuple(torch.tensor(x, dtype=torch.int32) for x in (bucket_of, order, begin))
        self._device = {}
        self._plans = {}  # of bucket_attention with these buckets, by the geometry of the tensors

    def __reduce__(self):  # copies and pickles hold the map alone: device copies and plans (which hold their addresses) stay behind
        return PositionBuckets.from_map, (self._host[0].tolist(), self.num_buckets)

    def __call__(self, relative_position):
        """Bucket of each entry of an integer tensor of relative positions ``key - query``."""
        table = self._host[0].to(device=relative_position.device, dtype=torch.int64)
        return table[relative_position.clamp(-self.reach, self.reach).long() + self.reach]

    def on(self, device):
        """The tables on a device: bucket of each distance, distances by bucket, begin of each bucket."""
        device = torch.device(device)
        if device not in self._device:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("[KeOps] PositionBuckets: first use on a device inside of a graph capture; call .on(device) before it.")
            self._device[device] = tuple(t.to(device) for t in self._host)
        return self._device[device]


# --------------------------------------------------------------------------------------------------- bucket attention
class _BucketPlan:
    """Arguments of a call that depend on the geometry of its tensors alone, checked once."""

    def __init__(self, q, k, v, bias, buckets, causal, start, scale):
        self.tables, self.options = buckets.on(q.device), (buckets, causal, start, scale)
        self.out_strides, self.k_strides, self.v_strides = _dense_strides(q), _dense_strides(k), _dense_strides(v)
        self.index, self.saved_strides = q.device.index, (q.stride(), k.stride(), v.stride(), self.out_strides)
        a = binder.BucketAttention()
        a.dtype, a.batch, a.heads, a.kv_heads, a.dim = _DTYPES[q.dtype], q.shape[0], q.shape[1], k.shape[1], q.shape[3]
        a.queries, a.keys, a.causal, a.scale = q.shape[2], k.shape[2], int(causal), scale
        a.buckets, a.reach, a.start = buckets.num_buckets, buckets.reach, start
        a.q_stride[:], a.k_stride[:], a.v_stride[:] = (_stride(x.shape, x.stride()) for x in (q, k, v))
        a.out_stride[:] = a.grad_q_stride[:] = _stride(q.shape, self.out_strides)
        a.grad_k_stride[:], a.grad_v_stride[:] = _stride(k.shape, self.k_strides), _stride(v.shape, self.v_strides)
        a.bucket_of, a.bucket_order, a.bucket_begin = (t.data_ptr() for t in self.tables)
        self.empty = q.numel() == 0
        self.args, self.grad_args = bytes(a), {}
        if not self.empty:  # the library's own checks, on placeholders that it does not follow
            lib = binder.lib()
            a.q = a.k = a.v = a.out = a.bias = a.grad_bias = 16
            self.forward_bytes = lib.keops_hip_bucket_attention_forward_bytes(ctypes.byref(a))
            self.backward_bytes = lib.keops_hip_bucket_attention_backward_bytes(ctypes.byref(a))  # at most this much without grad_bias

    def fill(self, args, q, k, v, bias, key_lengths, query_start):
        a = binder.BucketAttention.from_buffer_copy(args)
        a.q, a.k, a.v, a.bias = q.data_ptr(), k.data_ptr(), v.data_ptr(), bias.data_ptr()
        if key_lengths is not None:
            a.key_lengths = key_lengths.data_ptr()
        if query_start is not None:
            a.query_start = query_start.data_ptr()
        return a

    def run(self, name, a, nbytes, device):
        work = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        rc = getattr(binder.lib(), name)(ctypes.byref(a), _ptr(work), nbytes, self.index, _raw_stream(self.index))
        if rc:
            binder.check(rc, name)

    def forward(self, q, k, v, bias, key_lengths, query_start, want_lse):
        out = torch.empty_strided(q.shape, self.out_strides, dtype=q.dtype, device=q.device)
        lse = rest = None
        if not self.empty:
            a = self.fill(self.args, q, k, v, bias, key_lengths, query_start)
            a.out = out.data_ptr()
            if want_lse:
                lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
                a.lse = lse.data_ptr()
                if q.dtype != torch.float32:
                    rest = torch.empty_strided(q.shape, self.out_strides, dtype=q.dtype, device=q.device)
                    a.out_rest = rest.data_ptr()
            self.run("keops_hip_bucket_attention_forward", a, self.forward_bytes, q.device)
        return out, rest, lse

    def backward(self, grad, q, k, v, bias, out, rest, lse, key_lengths, query_start, want_q, want_bias):
        args = self.grad_args.get(grad.stride())
        if args is None or grad.data_ptr() & 15:  # the first of these strides, or such that are copied
            grad = _rows(grad)
            a = binder.BucketAttention.from_buffer_copy(self.args)
            a.grad_out_stride[:] = _stride(grad.shape, grad.stride())
            args = _keep(self.grad_args, grad.stride(), bytes(a))
        new, delta = torch.empty_strided, torch.empty_like(lse)
        dk = new(k.shape, self.k_strides, dtype=k.dtype, device=k.device)
        dv = new(v.shape, self.v_strides, dtype=v.dtype, device=v.device)
        a = self.fill(args, q, k, v, bias, key_lengths, query_start)
        a.out, a.lse, a.delta, a.grad_out = out.data_ptr(), lse.data_ptr(), delta.data_ptr(), grad.data_ptr()
        a.grad_k, a.grad_v = dk.data_ptr(), dv.data_ptr()
        if rest is not None:
            a.out_rest = rest.data_ptr()
        dq = db = None
        if want_q:
            dq = new(q.shape, self.out_strides, dtype=q.dtype, device=q.device)
            a.grad_q = dq.data_ptr()
        if want_bias:
            db = torch.empty_like(bias)
            a.grad_bias = db.data_ptr()
        self.run("keops_hip_bucket_attention_backward", a, self.backward_bytes, q.device)
        return dq, dk, dv, db


class _BucketAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, plan, key_lengths, query_start):
        out, rest, lse = plan.forward(q, k, v, bias, key_lengths, query_start, True)
        ctx.plan = plan
        ctx.save_for_backward(q, k, v, bias, out, rest, lse, key_lengths, query_start)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, bias, out, rest, lse, key_lengths, query_start = ctx.saved_tensors
        plan = ctx.plan
        if plan.empty:
            return (*(torch.zeros_like(t) for t in (q, k, v, bias)), None, None, None)
        if (q.stride(), k.stride(), v.stride(), out.stride()) != plan.saved_strides or (rest is not None and rest.stride() != out.stride()):
            # hooks on saved tensors may lay them out anew
            q, k, v, out = (_rows(x.contiguous()) for x in (q, k, v, out))
            rest = None if rest is None else _rows(rest.contiguous())
            plan = _BucketPlan(q, k, v, bias, *plan.options)
        return (*plan.backward(grad, q, k, v, bias, out, rest, lse, key_lengths, query_start, ctx.needs_input_grad[0], ctx.needs_input_grad[3]),
                None, None, None)


def _check_bucket(q, k, v, bias, buckets, query_start):
    what = "bucket_attention"
    device, dtype = _check_data(what, q=q, k=k, v=v)
    if not isinstance(buckets, PositionBuckets):
        raise TypeError("[KeOps] bucket_attention: buckets must be a PositionBuckets.")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("[KeOps] bucket_attention: q must be (batch, heads, queries, dim), k and v (batch, kv_heads, keys, dim).")
    b, h, m, d = q.shape
    if k.shape[0] != b or k.shape[3] != d or k.shape[1] < 1 or h % k.shape[1]:
        raise ValueError(f"[KeOps] bucket_attention: q {tuple(q.shape)} and k {tuple(k.shape)} do not fit: same batch and dim, heads a "
                         "multiple of kv_heads.")
    if not 1 <= d <= 128:
        raise ValueError(f"[KeOps] bucket_attention: dim must be from 1 to 128, it is {d}.")
    if max(m, k.shape[2]) > 1 << 29:
        raise ValueError("[KeOps] bucket_attention: at most 2**29 queries and keys.")
    _check_data(what, bias=bias)
    if bias.device != device:
        raise ValueError("[KeOps] Input arrays must be all located on the same device.")
    if bias.dtype not in (torch.float32, dtype) or tuple(bias.shape) != (h, buckets.num_buckets):
        raise ValueError(f"[KeOps] bucket_attention: bias must be ({h}, {buckets.num_buckets}), float32 or {dtype}; got "
                         f"{tuple(bias.shape)}, {bias.dtype}.")
    if not isinstance(query_start, torch.Tensor) and (
            isinstance(query_start, bool) or not isinstance(query_start, int) or abs(query_start) > 1 << 29):
        raise ValueError("[KeOps] bucket_attention: query_start must be a whole number of absolute value at most 2**29, or a tensor.")


def bucket_attention(q, k, v, bias, buckets, *, causal=False, key_lengths=None, query_start=0, scale=None):
    r"""Softmax attention with a learned bias for each bucket of the relative position:

    ``out_i = sum_j softmax_j(scale * <q_i, k_j> + bias[h, buckets(j - query_start - i)]) v_j``

    Args:
        q: (batch, heads, queries, dim).
        k, v: (batch, kv_heads, keys, dim); ``heads`` is a multiple of ``kv_heads``, neighbouring heads share.  dim is at most
            128.  Any strides (rows that do not start at multiples of 16 bytes are copied first).
        bias: (heads, buckets.num_buckets), float32 or the type of q.
        buckets: a :class:`PositionBuckets`.
        causal: keys after the query's position do not count.
        key_lengths: (batch,) whole numbers: keys from there on do not exist; what is stored there is not read.
        query_start: position of the first query among the keys: a number, or (batch,) whole numbers, of absolute value at most
            2**29.  For one new token against a cache that already holds its key: ``key_lengths - 1``.
        scale: default ``dim ** -0.5``.

    A bias of -6e4 or less (``-inf``, the lowest value of a type) hides its pairs.  A query that sees no key has output 0 and gives
    no gradient.  Keys that are only hidden by ``causal`` are read with their tile: a value that is not finite there can reach
    earlier queries.

    Returns (batch, heads, queries, dim) in the type and order of dimensions of q.  Differentiable with respect to q, k, v and
    bias.  Up to 32 queries x shared heads use a form of their own that splits the keys over the chip (token generation).
    """
    start = query_start if type(query_start) is int else None
    if scale is not None and type(scale) is not float:
        scale = float(scale)  # (a tensor's value, not the tensor, is what a plan is for)
    plan = key = None
    try:
        key = (_geometry(q), _geometry(k), _geometry(v), _geometry(bias), bool(causal), start, scale)
        plan = buckets._plans.get(key)
    except (AttributeError, TypeError):  # not tensors, no PositionBuckets: said below
        pass
    if plan is None:
        _check_bucket(q, k, v, bias, buckets, query_start)
        d = q.shape[3]
        number = d ** -0.5 if scale is None else scale
        align = 16 // q.element_size()
        if d % align or not all(map(_strides_fit, (q, k, v))) or bias.dtype != torch.float32 or not bias.is_contiguous():
            out = bucket_attention(_rows(_pad(q, align)), _rows(_pad(k, align)), _rows(_pad(v, align)), bias.float().contiguous(), buckets,
                                   causal=causal, key_lengths=key_lengths, query_start=query_start, scale=number)
            return out if out.shape[3] == d else out[..., :d].contiguous()
        plan = _keep(buckets._plans, key, _BucketPlan(q, k, v, bias, buckets, causal, start or 0, number))
    if (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v = _rows(q), _rows(k), _rows(v)
        return bucket_attention(q, k, v, bias, buckets, causal=causal, key_lengths=key_lengths, query_start=query_start, scale=scale)
    batch, device = q.shape[:1], q.device
    if key_lengths is not None:
        key_lengths = _check_whole("bucket_attention", "key_lengths", key_lengths, batch, device)
    start = _check_whole("bucket_attention", "query_start", query_start, batch, device) if start is None else None
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or bias.requires_grad):
        return _BucketAttention.apply(q, k, v, bias, plan, key_lengths, start)
    return plan.forward(q, k, v, bias, key_lengths, start, False)[0]


# --------------------------------------------------------------------------------------------------- decay attention
class _DecayWalk:
    """One walk over the tokens (keops_hip_decay_attention of include/keops_hip.h): its arguments that depend on the geometry of
    the tensors alone.  q, k, v, out: (shape, strides)."""

    def __init__(self, dtype, device, heads, q, k, v, out, out_dtype, *, reverse=False, product_scale=1.0, query_scale=1.0,
                 update_scale=1.0, transposed=False, given=False, joined=None):
        (b, _, t, d), dv = q[0], v[0][3]
        self.device, self.index, self.out_dtype, self.given = device, device.index, out_dtype, given
        self.out, self.state_shape = out, (b, heads, d, dv)
        a = binder.DecayAttention()
        a.dtype, a.batch, a.heads, a.dim, a.dim_v, a.tokens = _DTYPES[dtype], b, heads, d, dv, t
        a.q_heads, a.k_heads, a.v_heads = q[0][1], k[0][1], v[0][1]
        a.reverse, a.out_float32 = int(reverse), int(out_dtype == torch.float32)
        a.product_scale, a.query_scale, a.update_scale = product_scale, query_scale, update_scale
        a.q_stride[:], a.k_stride[:], a.v_stride[:], a.out_stride[:] = (_stride(*x) for x in (q, k, v, out))
        a.state_in_stride[:] = (1, d) if transposed else (dv, 1)
        a.state_out_stride[:] = (dv, 1)
        a.states_stride[:] = (1, d) if transposed and given else (dv, 1)
        a.states_given = int(given)
        self.joined, self.dtype = joined, dtype
        if joined is not None:
            a.joined_heads, a.joined_stride[:], a.joined = joined[0][1], _stride(*joined), 16
        self.empty = b == 0 or heads == 0
        if not self.empty:
            a.q = a.k = a.v = a.out = a.log_decay = 16  # placeholders for the library's own checks
            self.states = binder.lib().keops_hip_decay_attention_bytes(ctypes.byref(a)) // 4
        self.args = bytes(a)

    def __call__(self, q, k, v, log_decay, lengths, state, want_state=False, states=None):
        """Outputs, the final state (or None) and the workspace; ``states``: the workspace of the walk that left the states."""
        if self.empty:
            out = torch.empty_strided(*(self.joined or self.out), dtype=self.dtype, device=self.device).zero_()
            return out, torch.empty(self.state_shape, dtype=torch.float32, device=self.device) if want_state else None, None
        out = torch.empty_strided(*self.out, dtype=self.out_dtype, device=self.device)
        last = torch.empty(self.state_shape, dtype=torch.float32, device=self.device) if want_state else None
        a = binder.DecayAttention.from_buffer_copy(self.args)
        if self.states:  # (sequences in one piece have none)
            if states is None:
                states = torch.empty(self.states, dtype=torch.float32, device=self.device)
            a.states, a.states_bytes = states.data_ptr(), states.nbytes
        a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        a.log_decay = log_decay.data_ptr()
        if lengths is not None:
            a.lengths = lengths.data_ptr()
        if state is not None:
            a.state_in = state.data_ptr()
        if want_state:
            a.state_out = last.data_ptr()
        if self.joined is not None:
            per_head, out = out, torch.empty_strided(*self.joined, dtype=self.dtype, device=self.device)
            a.joined = out.data_ptr()
        rc = binder.lib().keops_hip_decay_attention_run(ctypes.byref(a), self.index, _raw_stream(self.index))
        if rc:
            binder.check(rc, "keops_hip_decay_attention_run")
        return out, last, states


class _DecayPlan:
    """The walks of a call and of its gradients."""

    def __init__(self, q, k, v, scale):
        self.dtype, self.device, self.scale, self.heads, self.shared = q.dtype, q.device, scale, q.shape[1], k.shape[1]
        self.q, self.k, self.v = ((x.shape, x.stride()) for x in (q, k, v))
        self.saved_strides = (q.stride(), k.stride(), v.stride())
        shape = (*q.shape[:3], v.shape[3])
        if q.shape[3] == v.shape[3]:
            strides = _dense_strides(q)
        elif q.stride(1) < q.stride(2):  # (batch, tokens, heads, dim) in memory
            strides = torch.empty(shape[0], shape[2], shape[1], shape[3], device="meta").transpose(1, 2).stride()
        else:
            strides = torch.empty(shape, device="meta").stride()
        self.out = (torch.Size(shape), strides)
        self.like = {"q": (q.shape, _dense_strides(q)), "k": (k.shape, _dense_strides(k)), "v": (v.shape, _dense_strides(v))}
        self.forward = self.walk(self.q, self.k, self.v, self.out, self.dtype, query_scale=scale)
        self.gradients = {}

    def walk(self, q, k, v, out, out_dtype, **options):
        return _DecayWalk(self.dtype, self.device, self.heads, q, k, v, out, out_dtype, product_scale=self.scale, **options)

    def backward(self, grad_strides):
        """The walks that give the gradients of q, v and k.  A shared head's gradient is the sum over the heads that share it, rounded
        once: those walks leave float32 for each head."""
        walks = self.gradients.get(grad_strides)
        if walks is None:
            g = (self.out[0], grad_strides)

            def like(name):
                if self.heads == self.shared:
                    return {"out": self.like[name], "out_dtype": self.dtype}
                shape, _ = self.like[name]
                shape = torch.Size((shape[0], self.heads, *shape[2:]))
                return {"out": (shape, torch.empty(shape, device="meta").stride()), "out_dtype": torch.float32, "joined": self.like[name]}

            walks = _keep(self.gradients, grad_strides, (
                self.walk(g, self.v, self.k, self.like["q"], self.dtype, query_scale=self.scale, transposed=True, given=True),
                self.walk(self.k, self.q, g, **like("v"), reverse=True, update_scale=self.scale),
                self.walk(self.v, g, self.q, **like("k"), reverse=True, update_scale=self.scale, transposed=True),
                self.walk(self.v, g, self.q, **like("k"), reverse=True, update_scale=self.scale, transposed=True, given=True),
            ))
        return walks


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, log_decay, lengths, plan):
        ctx.set_materialize_grads(False)
        out, last, states = plan.forward(q, k, v, log_decay, lengths, state, True)
        ctx.plan = plan
        ctx.save_for_backward(q, k, v, state, log_decay, lengths, states)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_last):
        # gradients are walks of the same kind (csrc/sequence/keops_seq_decay.hip); that of q starts from the forward pass's states,
        # that of k from those of v's
        q, k, v, state, log_decay, lengths, states = ctx.saved_tensors
        plan = ctx.plan
        if (q.stride(), k.stride(), v.stride()) != plan.saved_strides:  # hooks on saved tensors may lay them out anew
            q, k, v = (_rows(x.contiguous()) for x in (q, k, v))
            plan = _DecayPlan(q, k, v, plan.scale)
        if grad is None:
            grad = torch.zeros(plan.out[0], dtype=q.dtype, device=q.device)
        elif grad.stride() not in plan.gradients or grad.data_ptr() & 15:  # (strides that have walks fit)
            grad = _rows(grad)
        if grad_last is not None:
            grad_last = grad_last.contiguous()
            grad_last = grad_last.clone() if grad_last.data_ptr() & 15 else grad_last
        to_q, to_v, to_k, to_k_given = plan.backward(grad.stride())
        want_q, want_k, want_v, want_state = ctx.needs_input_grad[:4]
        dq = dk = dv = ds = None
        if want_q:
            dq = to_q(grad, v, k, log_decay, lengths, state, states=states)[0]
        if want_v or want_state:
            dv, ds, back = to_v(k, q, grad, log_decay, lengths, grad_last, want_state)
        if want_k:
            if dv is None:
                dk = to_k(v, grad, q, log_decay, lengths, grad_last)[0]
            else:
                dk = to_k_given(v, grad, q, log_decay, lengths, grad_last, states=back)[0]
        return dq, dk, dv, ds, None, None, None


_decay_plans, _step_plans = {}, {}


_CONSTANT = "[KeOps] {}: log_decay is a constant of the layer, no gradient with respect to it is computed; detach it."


def _check_decay(what, q, k, v, log_decay, state, dims):
    device, dtype = _check_data(what, q=q, k=k, v=v)
    if any(x.dim() != dims for x in (q, k, v)):
        raise ValueError(f"[KeOps] {what}: q, k and v must have {dims} dimensions.")
    b, h, d, dv = q.shape[0], q.shape[1], q.shape[-1], v.shape[-1]
    if k.shape[:-1] != v.shape[:-1] or k.shape[0] != b or k.shape[-1] != d or k.shape[2:-1] != q.shape[2:-1] or k.shape[1] < 1 or h % k.shape[1]:
        raise ValueError(f"[KeOps] {what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit: same batch and tokens, k "
                         "as wide as q, heads a multiple of kv_heads.")
    if not (1 <= d <= 128 and 1 <= dv <= 128):
        raise ValueError(f"[KeOps] {what}: dim and dim_v must be from 1 to 128, they are {d} and {dv}.")
    if b * h > 65535:
        raise ValueError(f"[KeOps] {what}: at most 65535 sequences times heads.")
    for name, t, shape in (("log_decay", log_decay, (h,)), ("state", state, (b, h, d, dv))):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != shape:
            raise ValueError(f"[KeOps] {what}: {name} must be a float32 tensor of shape {shape}.")
        if t.device != device:
            raise ValueError("[KeOps] Input arrays must be all located on the same device.")
    if log_decay is None:
        raise ValueError(f"[KeOps] {what}: log_decay must be a float32 tensor of shape ({h},).")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(_CONSTANT.format(what))
    return device


def decay_attention(q, k, v, log_decay, *, initial_state=None, lengths=None, scale=None):
    r"""Linear attention with a decay for each head, over whole sequences.  With ``g = exp(log_decay[h])``:

    ``S_t = g * S_(t-1) + k_t v_t^T,   out_t = scale * q_t S_t,   S_(-1) = initial_state``

    Args:
        q: (batch, heads, tokens, dim).
        k: (batch, kv_heads, tokens, dim), v: (batch, kv_heads, tokens, dim_v); ``heads`` is a multiple of ``kv_heads``,
            neighbouring heads share.  dim and dim_v are at most 128.  Any strides.
        log_decay: (heads,), float32: logarithms of the decays, usually negative; ``-inf`` forgets everything but the token itself.
        initial_state: (batch, heads, dim, dim_v), float32, or None for zeros.
        lengths: (batch,) whole numbers: tokens from there on do not exist; they are not read, their outputs and gradients are
            zeros, and the state stops before them.
        scale: default ``dim ** -0.5``.

    Returns ``(out, state)``: (batch, heads, tokens, dim_v) in the type of q, and the state behind the last token, float32, from
    which :func:`decay_attention_step` or another call goes on.  Differentiable with respect to q, k, v and initial_state, through
    both results.  Tokens are worked on in chunks of 64; a value that is not finite can reach earlier tokens of its chunk.
    """
    if scale is not None and type(scale) is not float:
        scale = float(scale)  # (a tensor's value, not the tensor, is what a plan is for)
    plan = key = None
    try:
        key = (_geometry(q), _geometry(k), _geometry(v), _geometry(initial_state), _geometry(log_decay), scale)
        plan = _decay_plans.get(key)
    except (AttributeError, TypeError):  # not tensors: said below
        pass
    if plan is None:
        device = _check_decay("decay_attention", q, k, v, log_decay, initial_state, 4)
        if q.shape[2] > 1 << 29:
            raise ValueError("[KeOps] decay_attention: at most 2**29 tokens.")
        d, dv = q.shape[3], v.shape[3]
        number = d ** -0.5 if scale is None else scale
        align = 16 // q.element_size()
        if (d % align or dv % align or not all(map(_strides_fit, (q, k, v))) or not log_decay.is_contiguous()
                or (initial_state is not None and not initial_state.is_contiguous())):
            state = None if initial_state is None else _pad(initial_state, align, align).contiguous()
            out, last = decay_attention(_rows(_pad(q, align)), _rows(_pad(k, align)), _rows(_pad(v, align)), log_decay.contiguous(),
                                        initial_state=state, lengths=lengths, scale=number)
            return (out if out.shape[3] == dv else out[..., :dv].contiguous(),
                    last if last.shape[2:] == (d, dv) else last[:, :, :d, :dv].contiguous())
        plan = _keep(_decay_plans, key, _DecayPlan(q, k, v, number))
    if (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15 or (initial_state is not None and initial_state.data_ptr() & 15):
        state = None if initial_state is None else initial_state.clone()
        return decay_attention(_rows(q), _rows(k), _rows(v), log_decay, initial_state=state, lengths=lengths, scale=scale)
    if lengths is not None:
        lengths = _check_whole("decay_attention", "lengths", lengths, q.shape[:1], q.device)
    if torch.is_grad_enabled():
        if log_decay.requires_grad:
            raise ValueError(_CONSTANT.format("decay_attention"))
        if q.requires_grad or k.requires_grad or v.requires_grad or (initial_state is not None and initial_state.requires_grad):
            return _DecayAttention.apply(q, k, v, initial_state, log_decay, lengths, plan)
    return plan.forward(q, k, v, log_decay, lengths, initial_state, True)[:2]


def decay_attention_step(q, k, v, log_decay, state, *, scale=None):
    r"""One token of :func:`decay_attention` for every sequence: ``state`` becomes ``g * state + k v^T`` in place, the result is
    ``scale * q state``.

    Args:
        q: (batch, heads, dim), k: (batch, kv_heads, dim), v: (batch, kv_heads, dim_v), dim_v a multiple of 4.
        log_decay: (heads,), float32.
        state: (batch, heads, dim, dim_v), float32, contiguous; overwritten.
        scale: default ``dim ** -0.5``.

    Returns (batch, heads, dim_v) in the type of q.  No gradients.
    """
    if scale is not None and type(scale) is not float:
        scale = float(scale)  # (a tensor's value, not the tensor, is what a plan is for)
    key = plan = None
    try:
        key = (_geometry(q), _geometry(k), _geometry(v), _geometry(state), _geometry(log_decay), scale)
        plan = _step_plans.get(key)
    except (AttributeError, TypeError):  # not tensors: said below
        pass
    if plan is None:
        what = "decay_attention_step"
        if state is None:
            raise ValueError("[KeOps] decay_attention_step: state must be a float32 tensor of shape (batch, heads, dim, dim_v).")
        _check_decay(what, q, k, v, log_decay, state, 3)
        if v.shape[2] % 4:
            raise ValueError(f"[KeOps] decay_attention_step: dim_v must be a multiple of 4, it is {v.shape[2]}.")
        if not state.is_contiguous():
            raise ValueError("[KeOps] decay_attention_step: state must be contiguous, it is overwritten.")
        if not all(x.stride(2) == 1 or x.shape[2] == 1 for x in (q, k, v)) or not log_decay.is_contiguous():
            return decay_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), log_decay.contiguous(), state, scale=scale)
        b, h, d = q.shape
        pair = ctypes.c_int64 * 2
        plan = _keep(_step_plans, key, (
            (_DTYPES[q.dtype], b, h, k.shape[1], d, v.shape[2], d ** -0.5 if scale is None else scale),
            pair(*q.stride()[:2]), pair(*k.stride()[:2]), pair(*v.stride()[:2]), (b, h, v.shape[2]), q.device.index))
    if state.data_ptr() & 15:
        raise ValueError("[KeOps] decay_attention_step: state must be aligned to 16 bytes, it is overwritten.")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad or log_decay.requires_grad):
        raise ValueError("[KeOps] decay_attention_step overwrites the state and has no gradient: use decay_attention, or torch.no_grad().")
    head, q_stride, k_stride, v_stride, shape, index = plan
    out = torch.empty(shape, dtype=q.dtype, device=q.device)
    if shape[0] and shape[1]:
        rc = binder.lib().keops_hip_decay_attention_step(
            *head, q.data_ptr(), q_stride, k.data_ptr(), k_stride, v.data_ptr(), v_stride, log_decay.data_ptr(), state.data_ptr(),
            out.data_ptr(), index, _raw_stream(index))
        if rc:
            binder.check(rc, "keops_hip_decay_attention_step")
    return out


# --------------------------------------------------------------------------------------------------- log probabilities
class TokenLogprobs(NamedTuple):
    """Result of :func:`token_logprobs`."""

    logprob: torch.Tensor      # (...,) float32
    entropy: torch.Tensor      # (...,) float32
    top_logprob: torch.Tensor  # (..., top) float32
    top_index: torch.Tensor    # (..., top) int64


_logprob_bytes = {}  # workspace by type, rows, vocabulary and alternatives


def _logprobs_forward(logits, tokens, top, ignore_index):
    (rows, vocab), device = logits.shape, logits.device
    logprob, entropy, lse = (torch.empty(rows, dtype=torch.float32, device=device) for _ in range(3))
    top_logprob = torch.empty((rows, top), dtype=torch.float32, device=device)
    top_index = torch.empty((rows, top), dtype=torch.int64, device=device)
    if rows:
        lib, index = binder.lib(), device.index
        key = (_DTYPES[logits.dtype], rows, vocab, top)
        nbytes = _logprob_bytes.get(key)
        if nbytes is None:
            nbytes = _keep(_logprob_bytes, key, lib.keops_hip_token_logprobs_bytes(*key))
        work = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        rc = lib.keops_hip_token_logprobs(
            *key, logits.data_ptr(), logits.stride(0), tokens.data_ptr(), ignore_index, logprob.data_ptr(), entropy.data_ptr(),
            lse.data_ptr(), top_logprob.data_ptr(), top_index.data_ptr(), _ptr(work), nbytes, index, _raw_stream(index))
        if rc:
            binder.check(rc, "keops_hip_token_logprobs")
    return logprob, entropy, lse, top_logprob, top_index


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, ignore_index):
        ctx.set_materialize_grads(False)
        logprob, entropy, lse, top_logprob, top_index = _logprobs_forward(logits, tokens, top, ignore_index)
        ctx.save_for_backward(logits, tokens, entropy, lse, top_index)
        ctx.top, ctx.ignore_index = top, ignore_index
        ctx.mark_non_differentiable(top_index)
        return logprob, entropy, top_logprob, top_index

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_top, _):
        logits, tokens, entropy, lse, top_index = ctx.saved_tensors
        rows, vocab = logits.shape
        grad = torch.empty(rows, vocab, dtype=logits.dtype, device=logits.device)
        if rows:
            g_logprob, g_entropy, g_top = (None if g is None else g.contiguous() for g in (g_logprob, g_entropy, g_top))
            rc = binder.lib().keops_hip_token_logprobs_backward(
                _DTYPES[logits.dtype], rows, vocab, ctx.top, _ptr(logits), logits.stride(0), _ptr(tokens), ctx.ignore_index,
                _ptr(entropy), _ptr(lse), _ptr(top_index), _ptr(g_logprob), _ptr(g_entropy), _ptr(g_top), _ptr(grad), vocab,
                logits.device.index, _raw_stream(logits.device.index))
            if rc:
                binder.check(rc, "keops_hip_token_logprobs_backward")
        return grad, None, None, None


def token_logprobs(logits, tokens, *, top=0, ignore_index=-100):
    r"""Log probabilities of given tokens under ``softmax(logits)``, the entropies of the distributions and their ``top`` largest
    log probabilities, in one sweep over the logits.

    Args:
        logits: (..., vocab).
        tokens: (...), int64 or int32.
        top: number of alternatives, at most 64 and at most vocab; equal values: the lowest index first.
        ignore_index: rows with this token have log probability 0, without gradient; their entropy and alternatives are those of
            the row.  Any other token outside 0..vocab-1 gives NaN.

    Logits of ``-inf`` have probability 0; a row of nothing else has log probability and alternatives ``-inf`` and entropy 0, and
    gradient 0.  A NaN or ``+inf`` makes its row's results NaN.

    Returns a :class:`TokenLogprobs`, float32.  Differentiable with respect to the logits through ``logprob``, ``entropy`` and
    ``top_logprob``.
    """
    device, _ = _check_data("token_logprobs", logits=logits)
    if not isinstance(tokens, torch.Tensor) or tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError("[KeOps] token_logprobs: tokens must be an int64 or int32 tensor.")
    if tokens.device != device:
        raise ValueError("[KeOps] Input arrays must be all located on the same device.")
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"[KeOps] token_logprobs: logits must be (..., vocab) and tokens (...); got {tuple(logits.shape)} and {tuple(tokens.shape)}.")
    vocab = logits.shape[-1]
    if not 1 <= vocab <= 2**31 - 1:
        raise ValueError("[KeOps] token_logprobs: the vocabulary must have from 1 to 2**31 - 1 entries.")
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= min(64, vocab):
        raise ValueError(f"[KeOps] token_logprobs: top must be a whole number from 0 to {min(64, vocab)}, got {top}.")
    shape = tokens.shape
    flat = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    if flat.stride(1) != 1 and vocab > 1:
        flat = flat.contiguous()
    if tokens.dtype != torch.int64 or tokens.dim() != 1 or not tokens.is_contiguous():
        tokens = tokens.reshape(-1).long().contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        logprob, entropy, top_logprob, top_index = _TokenLogprobs.apply(flat, tokens, top, int(ignore_index))
    else:
        logprob, entropy, _, top_logprob, top_index = _logprobs_forward(flat, tokens, top, int(ignore_index))
    if len(shape) == 1:
        return TokenLogprobs(logprob, entropy, top_logprob, top_index)
    return TokenLogprobs(logprob.view(shape), entropy.view(shape), top_logprob.view(*shape, top), top_index.view(*shape, top))

"""64-bit references of the sequence operators on the CPU's or the device's plain operations, with the absolute sums that the
error bounds of the tests are made of.

Bounds.  A rounding is off by at most half a step: ``u(t) = finfo(t).eps / 2`` of the value.  ``e32`` collects the float32 part
of a sum of n terms whose terms have passed through k operations: (n + k) * 2^-24 of the sum of absolute values (the standard
bound of a sum in any order, to first order)."""
import math

import torch

U32 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


# exp2 gives 0 for results below 2^-126, the smallest normal float32.  Sums of fewer than 2^20 such terms times values below 2^6
# (every test here) miss less than 2^-100 by that.
VANISHED = 2.0 ** -100


def rounding(x, dtype):
    """What rounding x to dtype may be off by: half a step of x, or, below the normal range (fp16: 2^-14), half of the smallest
    subnormal number, smallest_normal * eps / 2 (fp16: 2^-25)."""
    return u(dtype) * x.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def bucket(rel, num_buckets, max_distance, bidirectional):
    """Bucket of one relative position, by the definition."""
    count = num_buckets // 2 if bidirectional else num_buckets
    base = count if bidirectional and rel > 0 else 0
    d = abs(rel) if bidirectional else max(-rel, 0)
    near = count // 2
    if d < near:
        return base + d
    t = 0
    while t + 1 < count - near and d ** (count - near) >= near ** (count - near - t - 1) * max_distance ** (t + 1):
        t += 1
    return base + near + t


def attention(q, k, v, bias, bucket_of, causal, lengths, start, scale, grad=None):
    """Everything about one call, in 64 bits: a dict with out, the gradients, and the bounds ``tol_*`` of what a kernel that rounds
    probabilities and score gradients to the inputs' type may be off by."""
    dtype = q.dtype
    reach = bucket_of.numel() // 2
    b, h, m, d = q.shape
    n, g = k.shape[2], h // k.shape[1]
    q, k, v, bias = q.double(), k.double(), v.double(), bias.double()
    lens = [n] * b if lengths is None else [min(max(int(x), 0), n) for x in lengths]
    starts = [int(x) for x in start] if isinstance(start, torch.Tensor) else [start] * b
    out = torch.zeros(b, h, m, d, dtype=torch.float64, device=q.device)
    res = {"out": out, "tol_out": torch.zeros_like(out)}
    if grad is not None:
        grad = grad.double()
        for name, x in (("q", q), ("k", k), ("v", v), ("bias", bias)):
            res["grad_" + name], res["tol_grad_" + name] = torch.zeros_like(x), torch.zeros_like(x)
    up = u(dtype)                                          # probabilities as operands
    us = u(dtype)                                          # score gradients as operands (fp16: scaled, so never subnormal)
    for i in range(b):
        end = lens[i]
        if end == 0 or m == 0:
            continue
        away = torch.arange(end, device=q.device)[None] - (starts[i] + torch.arange(m, device=q.device))[:, None]
        bk = bucket_of.to(q.device).long()[away.clamp(-reach, reach) + reach]
        for j in range(h):
            kk, vv = k[i, j // g, :end], v[i, j // g, :end]
            z = q[i, j] @ kk.t() * scale + bias[j][bk]
            zabs = (q[i, j].abs() @ kk.abs().t()) * abs(scale) + bias[j].abs()[bk]
            if causal:
                z = z.masked_fill(away > 0, -math.inf)
            p = torch.softmax(z, -1).nan_to_num(0.0)
            seen = torch.isfinite(z)
            # relative error of a probability: that of its logit (twice, with the normalisation), of exp2 and of the sum
            e32 = U32 * (2 * (d + 8) * float((zabs * seen).max()) + end + 32)
            o, oabs = p @ vv, p @ vv.abs()
            out[i, j] = o
            tol_o = (up + e32) * oabs * 1.01 + rounding(o, dtype) + VANISHED
            res["tol_out"][i, j] = tol_o
            if grad is None:
                continue
            go = grad[i, j]
            dp, dpabs = go @ vv.t(), go.abs() @ vv.abs().t()
            delta, dabs = (go * o).sum(-1, keepdim=True), (go.abs() * oabs).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            ds32 = (e32 + U32 * (d + 8)) * p * (dpabs + dabs)          # of a score gradient with the row's exact delta
            dsq = ds32 + p * (go.abs() * tol_o).sum(-1, keepdim=True)  # with delta from the rounded output
            res["grad_q"][i, j] = ds @ kk * scale
            res["tol_grad_q"][i, j] = ((dsq + us * (ds.abs() + dsq)) @ kk.abs()) * abs(scale) * 1.01
            res["grad_k"][i, j // g, :end] += ds.t() @ q[i, j] * scale
            res["tol_grad_k"][i, j // g, :end] += ((ds32 + us * (ds.abs() + ds32)).t() @ q[i, j].abs()) * abs(scale) * 1.01
            res["grad_v"][i, j // g, :end] += p.t() @ go
            res["tol_grad_v"][i, j // g, :end] += (us + e32 + U32 * m) * (p.t() @ go.abs()) * 1.01
            res["grad_bias"][j].index_add_(0, bk.reshape(-1), ds.reshape(-1))
            res["tol_grad_bias"][j].index_add_(0, bk.reshape(-1), (ds32 + U32 * (m + end) * ds.abs()).reshape(-1))
    if grad is not None:
        for name in ("q", "k", "v"):
            res["tol_grad_" + name] += rounding(res["grad_" + name], dtype) + VANISHED
        res["tol_grad_bias"] += U32 * res["grad_bias"].abs() + VANISHED
    return res


def decay(q, k, v, log_decay, state, lengths, scale, grad=None, grad_last=None):
    """The recurrence in 64 bits, token by token, and the same on absolute values for the bounds."""
    dtype = q.dtype
    b, h, t, d = q.shape
    dv, shared = v.shape[3], k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(h // shared, 1), v.double().repeat_interleave(h // shared, 1)
    g = torch.exp(log_decay.double())[None, :, None, None]
    size = (torch.full((b,), t) if lengths is None else lengths.cpu().clamp(0, t)).to(q.device).view(b, 1, 1, 1)
    # what is stored behind a sequence (NaN, for one) takes no part
    there = torch.arange(t, device=q.device)[None, None, :, None] < size
    q, k, v = (torch.where(there, x, torch.zeros_like(x)) for x in (q, k, v))
    grad = None if grad is None else torch.where(there, grad, torch.zeros_like(grad))
    zero = torch.zeros(b, h, d, dv, dtype=torch.float64, device=q.device)

    def walk(q, k, v, S, sq):
        out = torch.zeros_like(v)
        states = []
        for i in range(t):
            S = torch.where(i < size, g * S + k[:, :, i, :, None] * v[:, :, i, None, :], S)
            states.append(S)
            out[:, :, i] = (q[:, :, i, None] @ S)[:, :, 0] * sq * (i < size)[..., 0]
        return out, S, states

    def back(q, k, v, go, R, states, sq):
        dq, dk, dv_ = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        for i in reversed(range(t)):
            live = i < size
            dq[:, :, i] = (states[i] @ go[:, :, i, :, None])[..., 0] * sq * live[..., 0]
            R = torch.where(live, R + q[:, :, i, :, None] * go[:, :, i, None, :] * sq, R)
            dk[:, :, i] = (R @ v[:, :, i, :, None])[..., 0] * live[..., 0]
            dv_[:, :, i] = (k[:, :, i, None] @ R)[:, :, 0] * live[..., 0]
            R = torch.where(live, g * R, R)
        return dq, dk, dv_, R

    S0 = zero if state is None else state.double()
    out, last, states = walk(q, k, v, S0, scale)
    oabs, labs, sabs = walk(q.abs(), k.abs(), v.abs(), S0.abs(), abs(scale))
    # products of a chunk and the state are rounded to a bf16 operand, decayed values are two bf16 terms (2^-17, and 2^-16 with what
    # they add up to); fp16: products and state are two terms, the product of two terms leaves out 2^-18
    op = {torch.bfloat16: u(dtype) + 2.0 ** -16, torch.float16: 2.0 ** -15, torch.float32: 0.0, torch.float64: 0.0}[dtype]
    # sums over a row of the state (d), over tokens (t) and the decay's powers (a chunk's power is off by 2^-24, t / 64 times)
    e32 = U32 * (2 * t + d + dv + 64)
    res = {"out": out, "state": last, "tol_out": (op + e32) * oabs * 1.01 + rounding(out, dtype) + VANISHED,
           "tol_state": (e32 + 4 * U32) * labs + VANISHED}
    if grad is not None:
        R = zero if grad_last is None else grad_last.double()
        go = grad.double()
        exact = back(q, k, v, go, R, states, scale)
        bound = back(q.abs(), k.abs(), v.abs(), go.abs(), R.abs(), sabs, abs(scale))
        for name, x, a, heads in zip(("q", "k", "v", "state"), exact, bound, (h, shared, shared, h)):
            if heads != h:
                x, a = (y.view(b, shared, h // shared, t, -1).sum(2) for y in (x, a))
            last_round = rounding(x, dtype if name != "state" else torch.float32)
            res["grad_" + name] = x
            res["tol_grad_" + name] = ((op if name != "state" else 4 * U32) + e32) * a * 1.01 + last_round + VANISHED
    return res


def logprobs(x, tokens, top, ignore_index=-100, grads=None):
    """In 64 bits, rows that hold -inf included."""
    dtype = x.dtype
    vocab = x.shape[-1]
    z = x.double()
    nothing = (z == -math.inf).all(-1, keepdim=True)
    lse = torch.logsumexp(z, -1, keepdim=True)
    lp = torch.where(nothing, torch.full_like(z, -math.inf), z - lse)
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    ent = -plp.sum(-1)
    ign = tokens == ignore_index
    at = tokens.clamp(0, vocab - 1)[:, None]
    got = torch.where(ign, torch.zeros_like(ent), lp.gather(-1, at)[:, 0])
    best = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :top]
    # each exponential: its argument (x - m) * log2(e) twice rounded, exp2 off by 2 steps; then a sum over the row
    away = torch.where(p > 0, (z.amax(-1, keepdim=True) - z), torch.zeros_like(z))
    e = U32 * (vocab / 128 + 64 + 3 * (p * away).sum(-1))
    res = {"logprob": got, "entropy": ent, "top_logprob": lp.gather(-1, best), "top_index": best}
    res["tol_logprob"] = e + 4 * U32 * torch.where(got.isfinite(), got.abs(), torch.zeros_like(got))
    # entropy = log s - t / s: the weights' errors meet x - m there
    res["tol_entropy"] = e * (2 + (p * away).sum(-1)) + 3 * U32 * (p * away * (3 * away + 1)).sum(-1) + 8 * U32 * ent
    top_lp = res["top_logprob"]
    res["tol_top_logprob"] = e[:, None] + 4 * U32 * torch.where(top_lp.isfinite(), top_lp.abs(), torch.zeros_like(top_lp))
    if grads is not None:
        a, c, gt = (t.double() for t in grads)
        live = torch.where(ign, torch.zeros_like(a), a)[:, None]
        total, totabs = live + gt.sum(-1, keepdim=True), live.abs() + gt.abs().sum(-1, keepdim=True)
        c = c[:, None]
        safe = torch.where(p > 0, lp, torch.zeros_like(lp))
        dz = -p * (total + c * (safe + ent[:, None]))
        dz.scatter_add_(-1, at, live)
        dz.scatter_add_(-1, best, gt)
        dz = torch.where(nothing, torch.zeros_like(dz), dz)
        res["grad"] = dz
        ep = e[:, None] + U32 * (8 + 4 * (safe.abs() + lse.nan_to_num(0, 0, 0).abs()))
        mag = p * (totabs + c.abs() * (safe.abs() + ent[:, None] + 1))
        added = torch.zeros_like(p).scatter_add_(-1, at, live.abs()).scatter_add_(-1, best, gt.abs())
        res["tol_grad"] = (ep + U32 * (top + 8)) * (mag + added) + p * c.abs() * res["tol_entropy"][:, None] + rounding(dz, dtype) + 2.0 ** -126 * (totabs + c.abs() * ((lse - z).abs().nan_to_num(0, 0, 0) + ent[:, None] + 1))
    return res


def assert_within(got, ref, tol, name=""):
    got = got.double()
    bad = ~((got - ref).abs() <= tol) & ~((got == ref) | (got.isnan() & ref.isnan()))
    if bad.any():
        i = int(torch.argmax(torch.where(bad, (got - ref).abs() / tol, torch.zeros_like(ref))))
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off by more than their bound; worst {got.reshape(-1)[i]:.9g} "
                             f"for {ref.reshape(-1)[i]:.9g}, bound {tol.reshape(-1)[i]:.3g}")

"""Plain forms of the grouped-query operators (`dscuda_b200/flash.py`) for the tests: attention and rotations in 64 bits on whatever device
the tensors are, the 8-bit cache's rounding in the fp32 steps that define it, on the CPU.

Beside results, the attention functions return how far a correct kernel may be from them, element by element, from these roundings (half a
step is 2^-8 of a bf16 value, 2^-11 of an f16 one, 2^-24 of an fp32 one):
    scores   fp32 sums of 128 exact products: 128 * 2^-24 * scale * sum |q||k|, called `ds` below
    weights  rounded to bf16 or f16 before P V; exp2 and the factor in front of it add a few 2^-22, counted as 2^-19
    outputs  rounded to bf16
"""

from __future__ import annotations

import math

import torch

BF16, F16 = 2.0 ** -8, 2.0 ** -11
SUM = 128 * 2.0 ** -24
EXP = 2.0 ** -19
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def rope_axes(x, positions, sections, theta=10000.0, restart=False, inverse=False):
    """x [rows, heads, W], positions [axes, rows] -> the turned values and their largest error apart from the last rounding."""
    half = x.shape[-1] // 2
    out, slack = torch.empty(x.shape, dtype=torch.float64), torch.empty(x.shape, dtype=torch.float64)
    pair = 0
    for axis, count in enumerate(sections):
        for j in range(count):
            angle = positions[axis].double() * theta ** (-(j / count) if restart else -(pair / half))
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None] * (-1 if inverse else 1)
            a, b = x[..., pair].double(), x[..., pair + half].double()
            out[..., pair], out[..., pair + half] = a * c - b * s, a * s + b * c
            slack[..., pair] = slack[..., pair + half] = 2.0 ** -20 * (a.abs() + b.abs())       # of sine, cosine and the fp32 sums
            pair += 1
    return out, slack


def encode(x, scale, dtype):
    """Codes of fp32 values: one product with the rounded reciprocal, rounded half to even."""
    inverse = 1.0 / scale if scale > 0 else torch.tensor(0.0)
    scaled = torch.nan_to_num(x * inverse, nan=0.0, posinf=LARGEST[dtype], neginf=-LARGEST[dtype]).clamp(-LARGEST[dtype], LARGEST[dtype])
    return scaled.round().to(dtype) if dtype == torch.int8 else scaled.to(dtype)


def append(cache, scales, rows, table, starts, counts):
    """Writes rows [B, T, H, 128] (CPU) into cache [blocks, H, page, 128] and scales [blocks, H] in place, page by page.  Positions and
    pages outside the cache are left out."""
    blocks, heads, page, _ = cache.shape
    dtype = cache.dtype
    for b in range(rows.shape[0]):
        start, count = int(starts[b]), min(max(int(counts[b]), 0), rows.shape[1])
        for logical in range(max(start, 0) // page, -(-(start + count) // page)):
            begin, end = max(start, 0, logical * page), min(start + count, (logical + 1) * page)
            if begin >= end or logical >= table.shape[1] or not 0 <= int(table[b, logical]) < blocks:
                continue
            at, slot = int(table[b, logical]), begin - logical * page
            for h in range(heads):
                x = torch.nan_to_num(rows[b, begin - start:end - start, h].float(), nan=0.0, posinf=math.inf, neginf=-math.inf)
                amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax()
                need = amax * torch.tensor(1.0 / LARGEST[dtype]) if amax >= 2.0 ** -100 else torch.tensor(0.0)
                old = scales[at, h].clone() if slot > 0 else torch.tensor(0.0)
                new = torch.maximum(old, need)
                if new > old and slot > 0:
                    ratio = old * (1.0 / new)
                    moved = cache[at, h, :slot].float() * ratio
                    cache[at, h, :slot] = moved.round().to(dtype) if dtype == torch.int8 else moved.to(dtype)
                cache[at, h, slot:slot + end - begin] = encode(x, new, dtype)
                scales[at, h] = new


def cached(cache, scales, table, length):
    """The first `length` values of a sequence in 64 bits: [length, H, 128]."""
    page = cache.shape[2]
    at = table[: -(-length // page)].long()
    values = cache[at].to(torch.float64) * scales[at].double()[:, :, None, None]
    return values.transpose(1, 2).reshape(-1, cache.shape[1], 128)[:length]


def attention(query, keys, values, scale, limits, weight_step):
    """query [T, Hq, 128], keys and values [N, Hkv, 128], limits [T] keys that each token sees -> output [T, Hq, 128], lse [Hq, T] and the
    errors allowed for both."""
    t, hq, _ = query.shape
    group = hq // keys.shape[1]
    q, k, v = query.double(), keys.double().repeat_interleave(group, 1), values.double().repeat_interleave(group, 1)
    seen = torch.arange(k.shape[0], device=q.device)[None, None] < limits.to(q.device)[None, :, None]
    if not k.shape[0]:
        zero = torch.zeros(t, hq, 128, dtype=torch.float64, device=q.device)
        return zero, torch.full((hq, t), -math.inf, dtype=torch.float64, device=q.device), zero, torch.zeros(hq, t, dtype=torch.float64, device=q.device)
    scores = torch.einsum("thd,nhd->htn", q, k) * scale
    size = torch.einsum("thd,nhd->htn", q.abs(), k.abs()) * scale
    ds = SUM * torch.where(seen, size, 0.0).amax(-1)                                  # [h, t]
    lse = torch.logsumexp(torch.where(seen, scores, -math.inf), -1)
    p = torch.where(seen, torch.exp(scores - torch.where(torch.isfinite(lse), lse, 0.0)[..., None]), 0.0)
    out = torch.einsum("htn,nhd->thd", p, v)
    weighed = torch.einsum("htn,nhd->thd", p, v.abs())
    relative = (weight_step + EXP + 2 * ds).t()[..., None]
    # weights far below the largest one lose bits in f16: at most 2^-32 of it each
    out_slack = BF16 * out.abs() + (1 + BF16) * relative * weighed + k.shape[0] * 2.0 ** -32 * v.abs().amax()
    lse_slack = ds + EXP + 2.0 ** -22 * torch.where(torch.isfinite(lse), lse, 0.0).abs()
    return out, lse, out_slack, lse_slack


def cross(query, key, value, scale, lengths, weight_step=BF16):
    """Batched `attention` with one length for each entry."""
    t = query.shape[1]
    parts = [attention(query[b], key[b, :n], value[b, :n], scale, torch.full((t,), n), weight_step) for b, n in enumerate(lengths)]
    return [torch.stack(x) for x in zip(*parts)]


def cross_gradients(dout, query, key, value, scale, lengths):
    """dquery, dkey, dvalue in 64 bits and the errors allowed for them (delta comes from the rounded output, P and dS are rounded to bf16)."""
    grads = [torch.zeros(x.shape, dtype=torch.float64, device=x.device) for x in (query, key, value)]
    slacks = [torch.zeros_like(x) for x in grads]
    group = query.shape[2] // key.shape[2]
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        for h in range(query.shape[2]):
            g = h // group
            q, k, v, do = query[b, :, h].double(), key[b, :n, g].double(), value[b, :n, g].double(), dout[b, :, h].double()
            scores = q @ k.t() * scale
            ds_scores = SUM * (q.abs() @ k.abs().t() * scale).amax(-1, keepdim=True)
            p = torch.softmax(scores, -1)
            out = p @ v
            dp = do @ v.t()
            delta = (do * out).sum(-1, keepdim=True)
            ds = p * (dp - delta) * scale
            e = EXP + 3 * ds_scores                                                  # relative error of P from scores and lse
            p_err = (BF16 + e) * p
            # the output that delta is formed from: its own rounding and that of the weights
            out_err = BF16 * out.abs() + (BF16 + e) * (p @ v.abs())
            dp_err = SUM * (do.abs() @ v.abs().t()) + SUM * (do.abs() * out.abs()).sum(-1, keepdim=True) + (do.abs() * out_err).sum(-1, keepdim=True)
            ds_err = (BF16 + e) * ds.abs() + (1 + BF16) * p * dp_err * scale
            grads[0][b, :, h] = ds @ k
            slacks[0][b, :, h] = ds_err @ k.abs()
            grads[1][b, :n, g] += ds.t() @ q
            slacks[1][b, :n, g] += ds_err.t() @ q.abs()
            grads[2][b, :n, g] += p.t() @ do
            slacks[2][b, :n, g] += p_err.t() @ do.abs()
    # fp32 sums over rows and keys, and the last rounding
    return grads, [(1 + BF16) * s * (1 + 2.0 ** -10) + BF16 * g.abs() + 2.0 ** -40 for s, g in zip(slacks, grads)]


# ---- the same errors added as independent ones --------------------------------------------------------------------------
# The bounds above hold for any signs of the roundings and so grow with the number of terms, where the errors of a long sum grow with its root: a
# missing tile of a long loop stays below them.  A rounding's error is spread over +-half a step, at most `step` times the value, so
# its variance is at most (step value)^2 / 3; the sum of squared errors of a head's result is near the sum of their variances.

EXACT_DELTA = 128               # up to so many keys the gradients' delta is formed from P and dP, not from the rounded output


def _variance(values, step):
    return (step * values) ** 2 / 3


def attention_variances(query, keys, values, scale, limits, weight_step):
    """Output of `attention` [T, Hq, 128] and the variance of each element."""
    t, hq, _ = query.shape
    if not keys.shape[0]:
        return (torch.zeros(t, hq, 128, dtype=torch.float64, device=query.device),) * 2
    group = hq // keys.shape[1]
    out, variance = (torch.empty(t, hq, 128, dtype=torch.float64, device=query.device) for _ in range(2))
    seen = torch.arange(keys.shape[0], device=query.device)[None] < limits.to(query.device)[:, None]
    for h in range(hq):
        q, k, v = query[:, h].double(), keys[:, h // group].double(), values[:, h // group].double()
        scores = torch.where(seen, q @ k.t() * scale, -math.inf)
        p = torch.nan_to_num(torch.softmax(scores, -1))                                  # (zeros where nothing is seen)
        e = EXP + 2 * SUM * torch.where(seen, q.abs() @ k.abs().t() * scale, 0.0).amax(-1, keepdim=True)
        out[:, h] = p @ v
        tiny = keys.shape[0] * (2.0 ** -32 * v.abs().amax()) ** 2                         # weights far below the largest one in f16
        variance[:, h] = _variance(out[:, h], BF16) + (weight_step ** 2 / 3 + e ** 2) * (p ** 2 @ v ** 2) + (e * out[:, h]) ** 2 + tiny
    return out, variance


def cross_variances(dout, query, key, value, scale, lengths, exact_delta=EXACT_DELTA):
    """output, dquery, dkey, dvalue and the variance of each of their elements."""
    shapes = (query, query, key, value)
    results, variances = ([torch.zeros(x.shape, dtype=torch.float64, device=x.device) for x in shapes] for _ in range(2))
    group = query.shape[2] // key.shape[2]
    for b, n in enumerate(lengths):
        for h in range(query.shape[2] if n else 0):
            g = h // group
            q, k, v, do = query[b, :, h].double(), key[b, :n, g].double(), value[b, :n, g].double(), dout[b, :, h].double()
            p = torch.softmax(q @ k.t() * scale, -1)
            e = EXP + 3 * SUM * (q.abs() @ k.abs().t() * scale).amax(-1, keepdim=True)     # relative error of P
            weights = (BF16 ** 2 / 3 + e ** 2) * p ** 2
            out, dp = p @ v, do @ v.t()
            out_variance = _variance(out, BF16) + weights @ v ** 2
            delta = (do * out).sum(-1, keepdim=True)
            delta_variance = (e * delta) ** 2 + (SUM * (do * out).abs().sum(-1, keepdim=True)) ** 2
            if n > exact_delta:
                delta_variance = delta_variance + (do ** 2 * out_variance).sum(-1, keepdim=True)
            ds = p * (dp - delta) * scale
            ds_variance = (BF16 ** 2 / 3 + e ** 2) * ds ** 2 + (p * scale * SUM * (do.abs() @ v.abs().t())) ** 2
            shared = delta_variance * scale ** 2                                          # one error of delta for all of a row
            results[0][b, :, h], variances[0][b, :, h] = out, out_variance
            results[1][b, :, h] = ds @ k
            variances[1][b, :, h] = ds_variance @ k ** 2 + shared * (p @ k) ** 2 + (e * (ds @ k)) ** 2
            results[2][b, :n, g] += ds.t() @ q
            variances[2][b, :n, g] += ds_variance.t() @ q ** 2 + (shared * p ** 2).t() @ q ** 2
            results[3][b, :n, g] += p.t() @ do
            variances[3][b, :n, g] += weights.t() @ do ** 2
    for x, variance in zip(results[1:], variances[1:]):
        variance += _variance(x, BF16)
    return results, variances


def deviations(actual, expected, variance):
    """How many times the root of its summed variances the error of a head is, the largest over entries and heads of [B, T, H, 128]."""
    error, allowed = ((actual.double() - expected) ** 2).sum((1, 3)), variance.sum((1, 3))
    return float(torch.where(error > 0, (error / allowed).sqrt(), torch.zeros_like(error)).max())

"""The four-bit format of a KV cache and attention over it, plainly: the format in f32 and whole numbers as it is defined, the rest in
64 bits with loops over sequences."""
import math

import torch

GROUP = 64


def quantized(x):
    """Rows x [..., head_dim] of bfloat16 or float16 -> (codes uint8 [..., head_dim / 2], steps [..., groups, 2]), on the CPU."""
    x = x.cpu()
    dtype, width = x.dtype, x.shape[-1]
    codes = torch.zeros(x.shape, dtype=torch.uint8)
    steps = torch.zeros(*x.shape[:-1], -(-width // GROUP), 2, dtype=dtype)
    for g in range(steps.shape[-2]):
        at = slice(g * GROUP, min(width, (g + 1) * GROUP))
        part = x[..., at].float()
        low, high = part.amin(-1), part.amax(-1)
        span = high - low
        whole = torch.isfinite(part).all(-1) & torch.isfinite(span)
        wanted = torch.where(whole, span, torch.zeros_like(span)) / torch.full_like(span, 15.0)
        step = wanted.to(dtype)
        step = (step.view(torch.int16) + (step.float() < wanted).to(torch.int16)).view(dtype)
        beyond = low.double() + 15 * step.double() > torch.finfo(dtype).max                # rounded down where the type ends
        step = (step.view(torch.int16) - beyond.to(torch.int16)).view(dtype)
        ratio = (part - low[..., None]) / step.float()[..., None]
        code = torch.where((step.float() > 0)[..., None] & whole[..., None], ratio, torch.zeros_like(part)).round().clamp(0, 15)
        codes[..., at] = code.to(torch.uint8)
        nan = torch.full_like(step, float("nan"))
        steps[..., g, 0], steps[..., g, 1] = torch.where(whole, step, nan), torch.where(whole, low.to(dtype), nan)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), steps


def parts(codes, steps):
    """(code * step, low) of every element in float64, on the codes' device."""
    whole = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    spread = steps.double().repeat_interleave(GROUP, -2)[..., :whole.shape[-1], :]
    return whole * spread[..., 0], spread[..., 1]


def values(codes, steps):
    product, low = parts(codes, steps)
    return product + low


def attention(q, cache, batch, scale, causal=True, zero_fully_masked=False, kernel="chunk"):
    """(out, lse, bound_out, bound_lse) in float64 on q's device; rows of no sequence are NaN. K and V are low + code * step with
    m = |low| + code * step the size of what is added. Errors of an f32 kernel with the result rounded to q's type (half a step u):
      scores    scale (D + 16) 2^-24 sum_d |q_d| m_d    (sums over codes and lows apart, their scales, the last addition);
                "chunk": keys rounded to the type, scale u sum_d |q_d k_d| on top
      p         relative 2 |ds| + 2^-20 (exponential, its argument, the sums), and its rounding in front of the product with V:
                "general" none, "rows" 2^-11 (f16, whatever the type), "chunk" u
      V         "chunk": rounded to the type, u |v|
      out       u |out|
    """
    unit = torch.finfo(q.dtype).eps / 2
    rounded_p = {"general": 0.0, "rows": 2.0 ** -11, "chunk": unit}[kernel]
    rounded = unit if kernel == "chunk" else 0.0
    size, group, width = cache.shape[1], q.shape[1] // cache.shape[2], q.shape[2]
    nan = float("nan")
    out, bound = (torch.full(q.shape, nan, dtype=torch.float64, device=q.device) for _ in range(2))
    lse, bound_lse = (torch.full(q.shape[:2], nan, dtype=torch.float64, device=q.device) for _ in range(2))
    starts, lengths = batch.query_starts.tolist(), batch.key_lengths.tolist()
    for s, length in enumerate(lengths):
        n, rows = starts[s + 1] - starts[s], slice(starts[s], starts[s + 1])
        if n <= 0:
            continue
        if length == 0:
            out[rows] = 0.0 if zero_fully_masked else nan
            lse[rows], bound[rows], bound_lse[rows] = -math.inf, 0.0, 0.0
            continue
        at = torch.arange(length, device=q.device)
        pages, in_page = batch.page_table[s].long()[at // size], at % size
        kp, kl = (t.repeat_interleave(group, 1) for t in parts(cache.k_codes[pages, in_page], cache.k_steps[pages, in_page]))
        vp, vl = (t.repeat_interleave(group, 1) for t in parts(cache.v_codes[pages, in_page], cache.v_steps[pages, in_page]))
        x = q[rows].double()
        scores = torch.einsum("nhd,lhd->hnl", x, kp + kl) * scale
        slack = torch.einsum("nhd,lhd->hnl", x.abs(), kp + kl.abs()) * (scale * (width + 16) * 2.0 ** -24)
        slack += torch.einsum("nhd,lhd->hnl", x.abs(), (kp + kl).abs()) * (scale * rounded)
        if causal:
            hidden = at[None, :] > (torch.arange(n, device=q.device) + (length - n))[:, None]
            scores.masked_fill_(hidden, -math.inf)
            slack.masked_fill_(hidden, 0.0)
        top = torch.logsumexp(scores, -1)
        p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top)[..., None])
        error = 2 * slack.amax(-1) + 2.0 ** -20
        o = torch.einsum("hnl,lhd->nhd", p, vp + vl)
        empty = (top == -math.inf).T
        out[rows] = torch.where(empty[..., None], torch.full_like(o, 0.0 if zero_fully_masked else nan), o)
        lse[rows] = top.T
        spread = torch.einsum("hnl,lhd->nhd", p, vp + vl.abs()) * (rounded_p + error.T[..., None] + (width + 16) * 2.0 ** -24)
        spread += torch.einsum("hnl,lhd->nhd", p, (vp + vl).abs()) * rounded
        bound[rows] = spread * (1 + unit) + unit * o.abs()
        bound_lse[rows] = error.T + top.T.abs().nan_to_num(posinf=0.0) * 2.0 ** -22
    return out, lse, bound, bound_lse

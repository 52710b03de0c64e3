"""64-bit references of the 8-bit KV cache operators, written from their definitions (torch, float64, any device)."""
import math

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
DTYPES = [torch.float8_e4m3fn, torch.int8]


def heads_first(x, layout):
    return x.transpose(1, 2) if layout == 0 else x


def block_scale(amax, dtype):
    """The smallest 2^e, -60 <= e <= 60, with amax <= qmax * 2^e, by trying every e."""
    e = torch.arange(-60, 61, dtype=torch.float64, device=amax.device)
    fits = amax[..., None] <= QMAX[dtype] * torch.exp2(e)
    first = torch.where(fits.any(-1), fits.to(torch.uint8).argmax(-1), torch.full(amax.shape, 120, device=amax.device))
    return torch.exp2(first.double() - 60)


def to_code_values(x, dtype):
    """Values in units of the scale -> the nearest representable ones (ties to even), as doubles."""
    top = QMAX[dtype]
    if dtype == torch.int8:
        x = torch.where(torch.isnan(x), torch.zeros_like(x), x)
        return torch.round(x).clamp(-top, top)
    nan = torch.isnan(x)
    x = torch.where(nan, torch.zeros_like(x), x).clamp(-top, top)
    _, e = torch.frexp(x.abs())
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)  # smallest normal 2^-6, three mantissa bits
    return torch.where(nan, torch.full_like(x, math.nan), (torch.round(x / step) * step).clamp(-top, top))


def finite_amax(x, dims):
    return torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(dims)


def values(cache):
    """[B, Hkv, S, D] doubles the cache stands for."""
    x = heads_first(cache.k, cache.kv_layout).double(), heads_first(cache.v, cache.kv_layout).double()
    S = cache.capacity
    s = [t.double().repeat_interleave(cache.block_tokens, 2)[:, :, :S, None] for t in (cache.k_scale, cache.v_scale)]
    return x[0] * s[0], x[1] * s[1]


def append(codes, scales, rows, held, n, block, dtype):
    """One row of heads: codes [H,S,D] and scales [H,nb] (doubles, changed in place), rows [H,T,D], one sequence."""
    S = codes.shape[1]
    n = max(0, min(n, rows.shape[1], S - held))
    for blk in range(held // block, -(-(held + n) // block) if n else 0):
        lo, hi = max(held, blk * block), min(held + n, (blk + 1) * block)
        new = rows[:, lo - held:hi - held].double()
        s = block_scale(finite_amax(new, (1, 2)), dtype)
        if blk * block < held:
            old = codes[:, blk * block:held] * scales[:, blk, None, None]
            s = torch.maximum(s, scales[:, blk])
            codes[:, blk * block:held] = to_code_values(old / s[:, None, None], dtype)
        codes[:, lo:hi] = to_code_values(new / s[:, None, None], dtype)
        scales[:, blk] = s


def decode(q, cache, lens, scale):
    """(out, lse, p, sum p|v|, largest scale * sum |q k|, max_t (p vscale)_t * sum_t |v8|): p [B,Hq,S]."""
    k, v = values(cache)
    B, Hq, D = q.shape
    H = cache.num_kv_heads
    S = cache.capacity
    qd = q.double().view(B, H, Hq // H, D)
    seen = torch.arange(S, device=q.device) < lens.clamp(0, S)[:, None]
    k = torch.where(seen[:, None, :, None], k, torch.zeros_like(k))
    v = torch.where(seen[:, None, :, None], v, torch.zeros_like(v))
    s = (scale * qd) @ k.transpose(-1, -2)
    size = abs(scale) * (qd.abs() @ k.abs().transpose(-1, -2))
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
    vs = cache.v_scale.double().repeat_interleave(cache.block_tokens, 2)[:, :, None, :S]
    top = torch.where(seen[:, None, None], p * vs, torch.zeros_like(p)).amax(-1, keepdim=True)
    codes = torch.where(seen[:, None, :, None], heads_first(cache.v, cache.kv_layout).double().abs(), torch.zeros_like(v))
    return ((p @ v).reshape(B, Hq, D), lse.reshape(B, Hq), p.reshape(B, Hq, S), (p @ v.abs()).reshape(B, Hq, D),
            size.amax(-1).reshape(B, Hq), (top * codes.sum(2)[:, :, None]).reshape(B, Hq, D))


def weight_sums(q, k, lse, scale, causal, q_start=0, lens=None, window=None):
    """(sums, largest scale * sum |q k|, terms per sum)."""
    B, Hq, Sq, D = q.shape
    H, Skv = k.shape[1], k.shape[2]
    out = torch.zeros(B, H, Skv, dtype=torch.float64, device=q.device)
    big, terms = 0.0, 1
    t = torch.arange(Skv, device=q.device)
    pos = q_start + torch.arange(Sq, device=q.device)
    for b in range(B):
        n = Skv if lens is None else max(0, min(int(lens[b]), Skv))
        end = n if causal and lens is not None else q_start + Sq
        rows = pos < end
        if window is not None:
            rows &= pos >= end - window
        seen = rows[:, None] & (t < n)[None]
        if causal:
            seen &= t[None] <= pos[:, None]
        terms = max(terms, int(rows.sum()) * (Hq // H))
        for h in range(Hq):
            kd = k[b, h // (Hq // H)].double()
            s = scale * (q[b, h].double() @ kd.T)
            big = max(big, float(abs(scale) * (q[b, h].double().abs() @ kd.abs().T).max()))
            ok = seen & (lse[b, h] != -math.inf)[:, None]
            out[b, h // (Hq // H)] += torch.where(ok, torch.exp(s - lse[b, h].double()[:, None]), torch.zeros_like(s)).sum(0)
    return out, big, terms


def kept_positions(w, n, budget, sink, recent):
    """Positions kept of one row of n tokens with weights w (a list), in order."""
    if n <= budget:
        return list(range(n))
    middle = list(range(sink, n - recent))
    order = sorted(middle, key=lambda t: (0 if math.isnan(w[t]) else 1, 0.0 if math.isnan(w[t]) else -w[t], t))
    return sorted(list(range(sink)) + order[:budget - sink - recent] + list(range(n - recent, n)))

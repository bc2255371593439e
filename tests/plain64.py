"""Plain 64-bit definitions of the operators around attention with a cache, for the tests."""
import math

import torch


def turn(x, positions, inv_freq, interleaved, back=False):
    """Rotation of the first 2 * len(inv_freq) values of x [tokens, heads, d] (float64); `back`: its inverse."""
    half = inv_freq.numel()
    if half == 0:
        return x.clone()
    angle = (positions.double()[:, None] * inv_freq.double()[None, :])[:, None, :]
    c, s = angle.cos(), angle.sin() * (-1 if back else 1)
    first = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    y = x.clone()
    a, b = x[..., first], x[..., second]
    y[..., first] = a * c - b * s
    y[..., second] = a * s + b * c
    return y


def norm_rope(x, weight, positions, inv_freq, eps, interleaved):
    x = x.double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r if weight is None else x * r * weight.double()
    return turn(n, positions, inv_freq, interleaved)


def norm_rope_backward(x, weight, positions, inv_freq, eps, interleaved, grad):
    """(dx, dweight) of sum(norm_rope(x) * grad)."""
    x = x.double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = x * r
    g = turn(grad.double(), positions, inv_freq, interleaved, back=True)
    dweight = (g * u).sum((0, 1))
    if weight is not None:
        g = g * weight.double()
    return r * (g - u * (g * u).mean(-1, keepdim=True)), dweight


def paged_attention(q, k_cache, v_cache, table, q_start, kv_len, scale=None, causal=True, window=0):
    """(o, lse) in float64, sequence by sequence; rows that no sequence owns are NaN."""
    tokens, hq, d = q.shape
    page, hk = k_cache.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    o = torch.full((tokens, hq, d), math.nan, dtype=torch.float64, device=q.device)
    lse = torch.full((tokens, hq), math.nan, dtype=torch.float64, device=q.device)
    starts, lens = q_start.tolist(), kv_len.tolist()
    for b, kv in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        n = hi - lo
        if n == 0:
            continue
        pages = table[b, :-(-kv // page)].long()
        k = k_cache[pages].reshape(-1, hk, d)[:kv].double().repeat_interleave(hq // hk, 1)
        v = v_cache[pages].reshape(-1, hk, d)[:kv].double().repeat_interleave(hq // hk, 1)
        s = torch.einsum("thd,khd->htk", q[lo:hi].double(), k) * scale
        last = torch.arange(n, device=q.device) + kv - n
        key = torch.arange(kv, device=q.device)
        seen = torch.ones(n, kv, dtype=torch.bool, device=q.device)
        if causal:
            seen &= key[None] <= last[:, None]
        if window:
            seen &= key[None] > last[:, None] - window
        s = s.masked_fill(~seen[None], -math.inf)
        z = torch.logsumexp(s, -1) if kv else torch.full((hq, n), -math.inf, dtype=torch.float64, device=q.device)
        p = torch.where(seen[None], (s - torch.where(z == -math.inf, 0.0, z)[..., None]).exp(), 0.0)
        # a masked key counts for nothing, whatever its value row holds
        o[lo:hi] = torch.stack([p[:, t][:, seen[t]].unsqueeze(1).bmm(v[seen[t]].transpose(0, 1))[:, 0] for t in range(n)])
        lse[lo:hi] = z.T
    return o, lse

"""Measured cases of the serving and training operators around attention: the per-head RMS norms of
queries and keys with the position rotation (forward, backward, and the form that also appends to a
paged cache) and attention of new tokens over a paged cache.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits), or, with ``own``
set, through this package's entry points. ``exact`` is the operator's definition in 64 bits.

Definitions, for a row x of one head (head_dim values), weight w, rotary dimension R <= head_dim:
  n_i = x_i w_i / sqrt(mean(x^2) + eps)
  rotation of the first R values by the angles position * inv_freq_j (j < R / 2), on the pairs
  (n_j, n_{j + R/2}), or (n_{2j}, n_{2j+1}) when `interleaved`; the other values pass through.
Attention of sequence b with kv keys, the last `queries` of which are the new tokens: query t sees the keys
j <= kv - queries + t (j < kv without `causal`), and with a window W only those with
j > kv - queries + t - W. A query that sees no key gives zeros and a log-sum of -inf.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    """The listed cases. 32 query heads over 8 key/value heads of 128 values are a common layout of
    models served on one GPU; 16 heads of 64 values in fp32 are this package's own attention benchmark."""
    return [
        # one user, one new token: latency
        dict(name="decode_one", op="attention", dtype="bf16", q_heads=32, k_heads=8, head_dim=128, page=16, batch=1,
             q_max=1, kv_min=2000, kv_max=2000, window=0, idle=0, spread=1),
        # a full decoding batch, sequences of very different age, two idle slots
        dict(name="decode_ragged", op="attention", dtype="bf16", q_heads=32, k_heads=8, head_dim=128, page=16, batch=64,
             q_max=1, kv_min=30, kv_max=16384, window=0, idle=2, spread=2),
        # the package's fp32 attention layout, decoding
        dict(name="decode_fp32", op="attention", dtype="fp32", q_heads=16, k_heads=16, head_dim=64, page=64, batch=8,
             q_max=1, kv_min=200, kv_max=1024, window=0, idle=0, spread=3),
        # prompts in chunks, sliding window, half precision, small heads
        dict(name="chunk_window_fp16", op="attention", dtype="fp16", q_heads=32, k_heads=4, head_dim=64, page=32,
             batch=6, q_max=777, kv_min=300, kv_max=5001, window=1024, idle=0, spread=4),
        # decoding sequences and prompt chunks in one call
        dict(name="mixed", op="attention", dtype="bf16", q_heads=32, k_heads=8, head_dim=128, page=16, batch=13,
             q_max=1000, kv_min=100, kv_max=4096, window=0, idle=1, spread=5),
        # one long prompt, a late chunk of it
        dict(name="chunk_long", op="attention", dtype="bf16", q_heads=32, k_heads=8, head_dim=128, page=64, batch=1,
             q_max=2048, kv_min=34816, kv_max=34816, window=0, idle=0, spread=6),
        # one decoding step: norms, rotation and the cache's new rows, some slots of the batch idle
        dict(name="append_decode", op="append", dtype="bf16", q_heads=32, k_heads=8, head_dim=128, rotary=128,
             interleaved=False, tokens=16, page=16, idle=3),
        # the same for a batch of prompts
        dict(name="append_prompt", op="append", dtype="bf16", q_heads=32, k_heads=8, head_dim=128, rotary=128,
             interleaved=False, tokens=8192, page=16, idle=0),
        # training in fp32: 8 sequences of 1024, 16 heads of 64
        dict(name="rope_fp32", op="rope", dtype="fp32", q_heads=16, k_heads=16, head_dim=64, rotary=64,
             interleaved=True, tokens=8192),
        # training in bf16 on long sequences, half of each head rotated
        dict(name="rope_bf16", op="rope", dtype="bf16", q_heads=32, k_heads=8, head_dim=128, rotary=64,
             interleaved=False, tokens=32768),
        # their backward passes
        dict(name="rope_backward_fp32", op="rope_backward", dtype="fp32", q_heads=16, k_heads=16, head_dim=64,
             rotary=64, interleaved=True, tokens=8192),
        dict(name="rope_backward_bf16", op="rope_backward", dtype="bf16", q_heads=32, k_heads=8, head_dim=128,
             rotary=128, interleaved=False, tokens=16384),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "rope", "rope_backward"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    head_dim = rng.choice([64, 80, 96, 128, 128, 256])
    k_heads = rng.choice([1, 2, 4, 8])
    q_heads = k_heads * rng.choice([1, 2, 4, 5, 7, 8])
    if op != "attention":
        tokens = _log_uniform(rng, 1, 32768 * 40 * 128 // ((q_heads + 2 * k_heads) * head_dim * (2 if dtype == "fp32" else 1)))
        tokens = min(tokens, 32768 if op == "rope" else 16384)
        case = dict(op=op, dtype=dtype, q_heads=q_heads, k_heads=k_heads, head_dim=head_dim,
                    rotary=rng.choice([head_dim, head_dim, head_dim // 2]), interleaved=rng.random() < 0.4, tokens=tokens)
        if op == "append":
            case.update(page=rng.choice([8, 16, 32, 64, 128]), idle=rng.randrange(0, 1 + tokens // 4))
        return case
    q_max = 1 if rng.random() < 0.5 else _log_uniform(rng, 2, 2048)
    kv_max = max(q_max, _log_uniform(rng, 1, 32768))
    # at most the work and the scores (batch x q_heads x q_max x kv_max in the plain form) of the largest listed case
    heavy = 8 if dtype == "fp32" or head_dim > 128 else 1
    q_max = max(1, min(q_max, 32 * 2048 * 34816 * 128 // (heavy * q_heads * kv_max * head_dim)))
    room = 32 * 2048 * 34816 * 128 // (heavy * q_heads * q_max * kv_max * max(128, head_dim))
    rows = 64 * 16384 * 8 * 128 // (kv_max * k_heads * head_dim)
    batch = _log_uniform(rng, 1, max(1, min(256, room, rows)))
    return dict(op=op, dtype=dtype, q_heads=q_heads, k_heads=k_heads, head_dim=head_dim,
                page=rng.choice([8, 16, 32, 64, 128]), batch=batch, q_max=q_max, kv_min=max(1, kv_max // rng.choice([1, 4, 50])),
                kv_max=kv_max, window=rng.choice([0, 0, 0, 1 + kv_max // 3]), idle=rng.randrange(0, 1 + batch // 8),
                spread=rng.randrange(1 << 20))


def _lengths(case):
    """(new tokens, keys) of each sequence: part of the case, the same for every seed."""
    r = random.Random(case["spread"])
    out = []
    for b in range(case["batch"]):
        kv = case["kv_max"] if b == 0 else _log_uniform(r, case["kv_min"], case["kv_max"])
        if b == 0 or case["q_max"] == 1:
            q = case["q_max"]
        else:  # decoding sequences among the chunks
            q = 1 if r.random() < 0.4 else _log_uniform(r, 1, case["q_max"])
        if b >= case["batch"] - case["idle"]:  # an idle slot of the batch: a token, no keys
            q, kv = 1, 0
        out.append((q if kv == 0 else min(q, kv), kv))
    return out


def _inv_freq(rotary):
    j = torch.arange(0, rotary, 2, dtype=torch.float64)
    return (10000.0 ** (-j / rotary)).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d, hq, hk = DTYPES[case["dtype"]], case["head_dim"], case["q_heads"], case["k_heads"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    if case["op"] == "attention":
        lens = _lengths(case)
        page = case["page"]
        tokens = sum(q for q, _ in lens)
        width = max(1, max(-(-kv // page) for _, kv in lens))
        used = [-(-kv // page) for _, kv in lens]
        pages = sum(used) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        first = torch.tensor([sum(used[:b]) for b in range(len(used))], device="cuda")
        col = torch.arange(width, device="cuda")
        index = first[:, None] + col[None, :]
        table = torch.where(col[None, :] < torch.tensor(used, device="cuda")[:, None], order[index.clamp(max=pages - 1)], 0)
        starts = [0]
        for q, _ in lens:
            starts.append(starts[-1] + q)
        return dict(op="attention", q=normal(tokens, hq, d), k_cache=normal(pages, page, hk, d),
                    v_cache=normal(pages, page, hk, d), table=table.to(torch.int32).contiguous(),
                    q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                    kv_len=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda"),
                    q_max=max(q for q, _ in lens), kv_max=case["kv_max"], window=case["window"])

    tokens = case["tokens"]
    state = dict(op=case["op"], interleaved=case["interleaved"], rotary=case["rotary"],
                 q_weight=1.0 + 0.2 * torch.randn(d, generator=g, device="cuda"),
                 k_weight=1.0 + 0.2 * torch.randn(d, generator=g, device="cuda"),
                 inv_freq=_inv_freq(case["rotary"]).cuda())
    if case["op"] == "append":
        # queries, keys and values are the parts of one projection's output
        qkv = normal(tokens, (hq + 2 * hk) * d, scale=2.0)
        state.update(q=qkv[:, :hq * d].view(tokens, hq, d), k=qkv[:, hq * d:(hq + hk) * d].view(tokens, hk, d),
                     v=qkv[:, (hq + hk) * d:].view(tokens, hk, d))
        page, real = case["page"], tokens - case["idle"]
        pages = -(-tokens // page) + 5
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
        slots[real:] = -1  # padded tokens are not stored
        state.update(positions=torch.randint(0, 131072, (tokens,), generator=g, device="cuda"), slots=slots, real=real,
                     k_cache=normal(pages, page, hk, d), v_cache=normal(pages, page, hk, d))
        return state
    state.update(q=normal(tokens, hq, d, scale=2.0), k=normal(tokens, hk, d, scale=2.0),
                 positions=torch.arange(tokens, device="cuda") + int(torch.randint(0, 4096, (1,), generator=g, device="cuda")))
    if case["op"] == "rope_backward":
        state.update(dq_out=normal(tokens, hq, d), dk_out=normal(tokens, hk, d))
    return state


# ---- plain forms ---------------------------------------------------------------------------------

def _angles(state):
    a = state["positions"].double()[:, None] * state["inv_freq"].double()[None, :]
    return a.cos().float()[:, None, :], a.sin().float()[:, None, :]


def _rotate(x, cos, sin, rotary, interleaved):
    """The rotation of the first `rotary` values of every head; sin negated: its inverse."""
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((turned, x[..., rotary:]), dim=-1)


def _norm_rotate(x, weight, cos, sin, state):
    x = x.float()
    n = x * (x.square().mean(dim=-1, keepdim=True) + EPS).rsqrt() * weight
    return _rotate(n, cos, sin, state["rotary"], state["interleaved"])


def _norm_rotate_backward(x, weight, grad, cos, sin, state):
    x = x.float()
    r = (x.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
    dn = _rotate(grad.float(), cos, -sin, state["rotary"], state["interleaved"])
    unit = x * r
    dweight = (dn * unit).sum(dim=(0, 1), dtype=torch.float64).float()
    du = dn * weight
    return r * (du - unit * (du * unit).mean(dim=-1, keepdim=True)), dweight


def _plain_attention(s):
    q, page = s["q"].float(), s["k_cache"].shape[1]
    tokens, hq, d = q.shape
    hk = s["k_cache"].shape[2]
    batch, width = s["table"].shape
    keys = width * page
    k = s["k_cache"][s["table"].long()].float().view(batch, keys, hk, d)
    v = s["v_cache"][s["table"].long()].float().view(batch, keys, hk, d)
    start, count = s["q_start"][:-1].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    t = torch.arange(s["q_max"], device=q.device)
    rows = q[(start[:, None] + t).clamp(max=tokens - 1)].view(batch, s["q_max"], hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(rows.reshape(batch, hk, -1, d), k.permute(0, 2, 3, 1)) * d ** -0.5
    scores = scores.view(batch, hk, hq // hk, s["q_max"], keys)
    key, last = torch.arange(keys, device=q.device), s["kv_len"].long()[:, None] - count[:, None] + t
    seen = (key <= last[:, :, None]) & (key < s["kv_len"][:, None, None])
    if s["window"]:
        seen &= key > last[:, :, None] - s["window"]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    scores = scores.sub_(top).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.view(batch, hk, -1, keys), v.transpose(1, 2)).view(batch, hk, hq // hk, s["q_max"], d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(batch, s["q_max"], hq, d)
    lse = (top + total.log()).permute(0, 3, 1, 2, 4).reshape(batch, s["q_max"], hq)
    token = torch.arange(tokens, device=q.device)
    seq = (token[:, None] >= s["q_start"][None, 1:]).sum(dim=1)
    return out[seq, token - start[seq]].to(s["q"].dtype), lse[seq, token - start[seq]]


def _plain(s):
    if s["op"] == "attention":
        return _plain_attention(s)
    cos, sin = _angles(s)
    dtype = s["q"].dtype
    if s["op"] == "rope_backward":
        dq, dq_weight = _norm_rotate_backward(s["q"], s["q_weight"], s["dq_out"], cos, sin, s)
        dk, dk_weight = _norm_rotate_backward(s["k"], s["k_weight"], s["dk_out"], cos, sin, s)
        return dq.to(dtype), dk.to(dtype), dq_weight, dk_weight
    q = _norm_rotate(s["q"], s["q_weight"], cos, sin, s).to(dtype)
    k = _norm_rotate(s["k"], s["k_weight"], cos, sin, s).to(dtype)
    if s["op"] == "rope":
        return q, k
    slots = s["slots"][:s["real"]]
    s["k_cache"].view(-1, *k.shape[1:])[slots] = k[:s["real"]]
    s["v_cache"].view(-1, *k.shape[1:])[slots] = s["v"][:s["real"]]
    return q, s["k_cache"], s["v_cache"]


# ---- this package's operators --------------------------------------------------------------------

_context = None


def _own(s):
    global _context
    if _context is None:
        import kernelh_b200

        _context = kernelh_b200.Context(torch.cuda.current_device())
    ctx, stream = _context, torch.cuda.current_stream().cuda_stream
    q = s["q"]
    if s["op"] == "attention":
        if "workspace" not in s:
            s["workspace"] = torch.empty(ctx.paged_attention_workspace(q, s["k_cache"], s["kv_len"].numel(), s["q_max"], s["kv_max"]),
                                         dtype=torch.uint8, device="cuda")
        o = torch.empty_like(q)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        ctx.paged_attention(q, s["k_cache"], s["v_cache"], s["table"], s["q_start"], s["kv_len"], o, lse=lse,
                            max_q_len=s["q_max"], max_kv_len=s["kv_max"], causal=True, window=s["window"],
                            workspace=s["workspace"], stream=stream)
        return o, lse
    k = s["k"]
    if s["op"] == "rope":
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
        ctx.qk_norm_rope(q, k, s["q_weight"], s["k_weight"], s["inv_freq"], s["positions"], q_out, k_out, eps=EPS,
                         interleaved=s["interleaved"], stream=stream)
        return q_out, k_out
    if s["op"] == "append":
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ctx.qk_norm_rope_append(q, k, s["v"], s["q_weight"], s["k_weight"], s["inv_freq"], s["positions"], s["slots"], q_out,
                                s["k_cache"], s["v_cache"], eps=EPS, interleaved=s["interleaved"], stream=stream)
        return q_out, s["k_cache"], s["v_cache"]
    if "workspace" not in s:
        s["workspace"] = torch.empty(ctx.qk_norm_rope_backward_workspace(q, k), dtype=torch.uint8, device="cuda")
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    dq_weight, dk_weight = torch.empty_like(s["q_weight"]), torch.empty_like(s["k_weight"])
    ctx.qk_norm_rope_backward(q, k, s["q_weight"], s["k_weight"], s["inv_freq"], s["positions"], s["dq_out"], s["dk_out"],
                              dq, dk, dq_weight, dk_weight, eps=EPS, interleaved=s["interleaved"],
                              workspace=s["workspace"], stream=stream)
    return dq, dk, dq_weight, dk_weight


def run(state):
    return _own(state) if own else _plain(state)


# ---- the work and the definition in 64 bits -------------------------------------------------------

def _seen_pairs(q, kv, window):
    """(query, key) pairs that the mask leaves, and the keys that any query sees."""
    pairs = 0
    for t in range(q):
        last = kv - q + t
        pairs += max(0, min(last + 1, window or last + 1))
    lowest = max(0, kv - q - window + 1) if window else 0
    return pairs, kv - lowest


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    d, hq, hk = case["head_dim"], case["q_heads"], case["k_heads"]
    if case["op"] == "attention":
        flops = moved = 0
        for q, kv in _lengths(case):
            pairs, keys = _seen_pairs(q, kv, case["window"])
            flops += 4 * pairs * hq * d
            moved += size * d * (2 * q * hq + 2 * keys * hk) + 4 * q * hq + 4 * -(-keys // case["page"]) + 8
        return {"bytes": moved, "flops": flops}
    tokens = case["tokens"]
    rows = tokens * (hq + hk)
    small = 4 * (2 * d + case["rotary"] // 2) + 8 * tokens
    if case["op"] == "rope":
        return {"bytes": 2 * rows * d * size + small, "flops": 8 * rows * d}
    if case["op"] == "append":
        real = tokens - case["idle"]
        moved = 2 * (tokens * hq + 2 * real * hk) * d * size
        return {"bytes": moved + small + 8 * tokens, "flops": 8 * rows * d}
    return {"bytes": 3 * rows * d * size + small + 8 * d, "flops": 18 * rows * d}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    d, r, half = case["head_dim"], case["rotary"], case["rotary"] // 2
    angle = s["positions"].to(torch.float64).unsqueeze(1) * s["inv_freq"].to(torch.float64)
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)  # e^(i angle)
    first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)

    def rotated(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def forward(x, w):
        x = x.to(torch.float64)
        return rotated(w.to(torch.float64) * x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS), turn)

    def backward(x, w, grad):
        x, w = x.to(torch.float64), w.to(torch.float64)
        g = rotated(grad.to(torch.float64), turn.conj())
        m = torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS)
        dw = torch.einsum("thi,thi->i", g, x / m)
        gw = g * w
        return gw / m - x * (gw * x).sum(-1, keepdim=True) / (d * m ** 3), dw

    if case["op"] == "rope_backward":
        dq, dwq = backward(s["q"], s["q_weight"], s["dq_out"])
        dk, dwk = backward(s["k"], s["k_weight"], s["dk_out"])
        return dq, dk, dwq, dwk
    q, k = forward(s["q"], s["q_weight"]), forward(s["k"], s["k_weight"])
    if case["op"] == "rope":
        return q, k
    k_cache, v_cache = s["k_cache"].to(torch.float64), s["v_cache"].to(torch.float64)
    slots = s["slots"][:s["real"]]
    at, offset = slots // case["page"], slots % case["page"]
    k_cache[at, offset] = k[:s["real"]]
    v_cache[at, offset] = s["v"][:s["real"]].to(torch.float64)
    return q, k_cache, v_cache


def _exact_attention(case, s):
    tokens, hq, d = s["q"].shape
    group = hq // case["k_heads"]
    out = torch.zeros(tokens, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, hq), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for b, (count, kv) in enumerate(_lengths(case)):
        if kv:
            pages = s["table"][b, :-(-kv // case["page"])].long()
            k = s["k_cache"][pages].flatten(0, 1)[:kv].double()
            v = s["v_cache"][pages].flatten(0, 1)[:kv].double()
            position = torch.arange(kv - count, kv, device="cuda")
            hidden = torch.arange(kv, device="cuda") > position.unsqueeze(1)
            if case["window"]:
                hidden |= torch.arange(kv, device="cuda") <= position.unsqueeze(1) - case["window"]
            for h in range(hq):
                x = s["q"][at:at + count, h].double() @ k[:, h // group].T / math.sqrt(d)
                x[hidden] = -math.inf
                z = torch.logsumexp(x, dim=-1)
                lse[at:at + count, h] = z
                out[at:at + count, h] = torch.exp(x - z.unsqueeze(1)) @ v[:, h // group]
        at += count
    return out, lse

"""The per-head norm of queries and keys with rotation: forward, backward and the form that appends to a
paged cache, against the 64-bit definition, at the layouts and sizes where the kernels change their paths.

Tolerances. An output is rounded once to its type: eps/2 of its value. Before that everything is fp32: the
norm of a pair of values, N, carries a few roundings from the sum of squares (at most 16 terms in a lane, 5
additions across lanes: 21 * 2^-24 of the sum, half of that in its root), 1/sqrt (2 ulp), two products, and
the rotation two products, a sum and the errors of cos and sin (angle in [-pi, pi] rounded to fp32: 2^-24 of
a half turn = pi * 2^-25, plus 2 ulp): below 24 * 2^-24 of N, where N is the magnitude of the pair."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")
import kernelh_b200 as kh
from tests import plain64

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


# --------------------------------------------------------------------------- no device
def rope_call(**over):
    """A call whose arguments are all right except those in `over`; buffers are addresses that nothing reads."""
    a = dict(dtype=1, q_heads=4, k_heads=2, head_dim=64, rotary_dim=64, interleaved=0, eps=1e-6, tokens=8,
             q=(4096, 256, 64), k=(4096, 128, 64), q_weight=4096, k_weight=4096, inv_freq=4096, positions=4096,
             q_out=(4096, 256, 64), k_out=(4096, 128, 64))
    extra = {k: over.pop(k) for k in list(over) if k not in a}
    a.update(over)
    args = kh.QkNormRopeArgs(a["dtype"], a["q_heads"], a["k_heads"], a["head_dim"], a["rotary_dim"], a["interleaved"], a["eps"],
                             a["tokens"], kh.HeadRows(*a["q"]), kh.HeadRows(*a["k"]), a["q_weight"], a["k_weight"], a["inv_freq"],
                             a["positions"])
    return args, kh.HeadRows(*a["q_out"]), kh.HeadRows(*a["k_out"]), extra


def refusal(rc):
    assert rc == kh.USAGE_ERROR
    return kh.lib.kh_last_error().decode()


@pytest.mark.parametrize("over,words", [
    (dict(dtype=7), "dtype must be"), (dict(tokens=-1), "tokens must lie"), (dict(q_heads=0), "q_heads and k_heads"),
    (dict(head_dim=63), "head_dim must be even"), (dict(head_dim=258), "head_dim must be even"),
    (dict(rotary_dim=66), "rotary_dim must be even"), (dict(rotary_dim=31), "rotary_dim must be even"),
    (dict(interleaved=2), "interleaved"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"),
    (dict(q=(0, 256, 64)), "buffer 'q' is null"), (dict(k=(4097, 128, 64)), "buffer 'k' is not aligned"),
    (dict(q_out=(4096, 256, 32)), "rows of output 'q_out' overlap"), (dict(k_out=(4096, 0, 64)), "rows of output 'k_out' overlap"),
    (dict(positions=0), "'positions' is null"), (dict(positions=4100), "8-byte aligned"), (dict(inv_freq=0), "'inv_freq' is null"),
    (dict(q_weight=4098), "4-byte aligned")])
def test_forward_refusals(over, words):
    args, q_out, k_out, _ = rope_call(**over)
    assert words in refusal(kh.lib.kh_qk_norm_rope(None, args, q_out, k_out, None))


def test_good_arguments_get_as_far_as_the_context():
    args, q_out, k_out, _ = rope_call()
    assert "null kernelh_b200 context" in refusal(kh.lib.kh_qk_norm_rope(None, args, q_out, k_out, None))
    # strides of dimensions of size 1 are not read
    args, q_out, k_out, _ = rope_call(tokens=1, k_heads=1, q_out=(4096, 0, 64), k_out=(4096, 0, 0))
    assert "null kernelh_b200 context" in refusal(kh.lib.kh_qk_norm_rope(None, args, q_out, k_out, None))
    assert "null arguments" in refusal(kh.lib.kh_qk_norm_rope(None, None, q_out, k_out, None))


@pytest.mark.parametrize("over,words", [
    (dict(workspace=0), "the workspace must have"), (dict(workspace_bytes=100), "the workspace must have"),
    (dict(workspace=4098), "not 4-byte aligned"), (dict(dq_out=(0, 256, 64)), "buffer 'dq_out' is null"),
    (dict(dk_out=(4097, 128, 64)), "'dk_out' is not aligned"), (dict(dq_weight=4097), "4-byte aligned"),
    (dict(q_out=(4096, 256, 8)), "rows of output 'dq' overlap")])
def test_backward_refusals(over, words):
    args, dq, dk, e = rope_call(**over)
    e = dict(dict(workspace=4096, workspace_bytes=1 << 20, dq_out=(4096, 256, 64), dk_out=(4096, 128, 64), dq_weight=4096), **e)
    assert words in refusal(kh.lib.kh_qk_norm_rope_backward(None, args, kh.HeadRows(*e["dq_out"]), kh.HeadRows(*e["dk_out"]), dq, dk,
                                                            e["dq_weight"], None, e["workspace"], e["workspace_bytes"], None))


@pytest.mark.parametrize("over,words", [
    (dict(page_size=0), "page_size and num_pages"), (dict(num_pages=0), "page_size and num_pages"), (dict(slots=0), "'slots' is null"),
    (dict(slots=4100), "8-byte aligned"), (dict(v=(0, 128, 64)), "buffer 'v' is null"),
    (dict(k_cache=(4096, 2048, 100, 32)), "rows of output 'k_cache' overlap"),
    (dict(v_cache=(4096, 10, 128, 64)), "rows of output 'v_cache' overlap")])
def test_append_refusals(over, words):
    args, q_out, _, e = rope_call(**over)
    e = dict(dict(v=(4096, 128, 64), slots=4096, k_cache=(4096, 2048, 128, 64), v_cache=(4096, 2048, 128, 64), num_pages=4,
                  page_size=16), **e)
    assert words in refusal(kh.lib.kh_qk_norm_rope_append(None, args, kh.HeadRows(*e["v"]), e["slots"], q_out,
                                                          kh.PagedRows(*e["k_cache"]), kh.PagedRows(*e["v_cache"]), e["num_pages"],
                                                          e["page_size"], None))


def test_tensor_refusals():
    ctx = kh.Context.__new__(kh.Context)
    ctx._h, ctx._ordinal = None, 0
    q, k, w, p = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.ones(64), torch.arange(3)
    with pytest.raises(kh.KernelhError, match="must be on device 0"):
        ctx.qk_norm_rope(q, k, w, w, torch.ones(32), p, q, k)
    with pytest.raises(kh.KernelhError, match="'q' must be float32, bfloat16 or float16"):
        ctx.qk_norm_rope(q.double(), k, w, w, torch.ones(32), p, q, k)
    with pytest.raises(kh.KernelhError, match=r"must be \[tokens, heads, head_dim\]"):
        ctx.qk_norm_rope(q[0], k, w, w, torch.ones(32), p, q, k)


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_gradient_formula_agrees_with_differences(interleaved):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 2, 12, generator=g, dtype=torch.float64)
    w = torch.randn(12, generator=g, dtype=torch.float64)
    dy = torch.randn(3, 2, 12, generator=g, dtype=torch.float64)
    pos, freq = torch.tensor([0, 5, 70000]), torch.tensor([1.0, 0.1, 0.003], dtype=torch.float64)

    def loss(x, w):
        return (plain64.norm_rope(x, w, pos, freq, 1e-6, interleaved) * dy).sum()

    dx, dw = plain64.norm_rope_backward(x, w, pos, freq, 1e-6, interleaved, dy)
    h = 1e-6  # the third derivative of a norm is below 100 here: h^2 * 100 = 1e-10, cancellation 1e-15 / h = 1e-9
    for t, ref in ((x, dx), (w, dw)):
        flat = t.view(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + h
            up = loss(x, w)
            flat[i] = keep - h
            down = loss(x, w)
            flat[i] = keep
            assert abs((up - down).item() / (2 * h) - ref.reshape(-1)[i].item()) < 1e-7


# --------------------------------------------------------------------------- B200
@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    c = kh.Context(0)
    yield c
    c.close()


def stream():
    return torch.cuda.current_stream().cuda_stream


def inputs(dtype, tokens, hq, hk, d, rotary, layout="plain", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape):
        return (2 * torch.randn(*shape, generator=g, device="cuda")).to(dtype)

    if layout == "joint":  # parts of one projection's output
        joint = rnd(tokens, (hq + 2 * hk) * d)
        q, k, v = (x.unflatten(1, (-1, d)) for x in joint.split([hq * d, hk * d, hk * d], dim=1))
    elif layout == "heads_first":
        q, k, v = (rnd(h, tokens, d).transpose(0, 1) for h in (hq, hk, hk))
    elif layout == "odd":  # addresses and strides that only single values divide
        q, k, v = (rnd(tokens, h * d + 1)[:, 1:].unflatten(1, (h, d)) for h in (hq, hk, hk))
    else:
        q, k, v = rnd(tokens, hq, d), rnd(tokens, hk, d), rnd(tokens, hk, d)
    qw, kw = (1 + 0.3 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    freq = (10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))).float().cuda()
    pos = torch.randint(0, 200000, (tokens,), generator=g, device="cuda")
    return q, k, v, qw, kw, freq, pos, rnd


def pair_magnitude(ref, half, interleaved):
    """For every value the magnitude of the pair it was rotated in."""
    m = ref.abs()
    if half:
        r = ref[..., :2 * half]
        pairs = r.unflatten(-1, (half, 2)) if interleaved else r.unflatten(-1, (2, half)).transpose(-1, -2)
        n = pairs.norm(dim=-1, keepdim=True).expand_as(pairs)
        m[..., :2 * half] = n.flatten(-2) if interleaved else n.transpose(-1, -2).flatten(-2)
    return m


def check_forward(got, x, w, pos, freq, interleaved):
    ref = plain64.norm_rope(x, w, pos, freq, 1e-6, interleaved)
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + 24 * U * pair_magnitude(ref, freq.numel(), interleaved) + \
        torch.finfo(got.dtype).tiny
    assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() / tol).max()


CASES = [  # dtype, tokens, q heads, k heads, head_dim, rotary, interleaved, layout
    ("bf16", 1, 32, 8, 128, 128, False, "plain"), ("bf16", 1301, 8, 2, 128, 128, False, "joint"), ("bf16", 7, 5, 1, 64, 32, True, "joint"),
    ("bf16", 9, 3, 3, 80, 80, False, "plain"), ("bf16", 9, 3, 1, 80, 40, False, "plain"), ("bf16", 5, 2, 2, 96, 48, True, "heads_first"),
    ("bf16", 6, 4, 1, 256, 256, False, "plain"), ("bf16", 6, 4, 2, 128, 64, False, "odd"), ("bf16", 3, 2, 1, 6, 2, False, "plain"),
    ("f16", 1203, 4, 4, 64, 64, False, "heads_first"), ("f16", 11, 7, 1, 256, 128, True, "plain"), ("f16", 4, 1, 1, 2, 2, False, "plain"),
    ("f16", 3, 2, 1, 72, 72, True, "plain"), ("f32", 1, 1, 1, 64, 64, True, "plain"), ("f32", 1190, 16, 16, 64, 64, True, "plain"),
    ("f32", 5, 4, 2, 256, 256, False, "joint"), ("f32", 5, 4, 2, 256, 100, False, "plain"), ("f32", 5, 3, 1, 20, 12, False, "plain"),
    ("f32", 33, 9, 3, 128, 128, False, "odd"), ("f32", 4, 2, 1, 128, 0, False, "plain"), ("f32", 3, 2, 1, 254, 250, True, "plain")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens,hq,hk,d,rotary,interleaved,layout", CASES)
def test_forward(ctx, dtype, tokens, hq, hk, d, rotary, interleaved, layout):
    q, k, v, qw, kw, freq, pos, _ = inputs(TYPES[dtype], tokens, hq, hk, d, rotary, layout)
    qo, ko = torch.empty(q.shape, dtype=q.dtype, device="cuda"), torch.empty_like(k)
    ctx.qk_norm_rope(q, k, qw, kw, freq if rotary else None, pos, qo, ko, interleaved=interleaved, stream=stream())
    check_forward(qo, q, qw, pos, freq, interleaved)
    check_forward(ko, k, kw, pos, freq, interleaved)
    # without weights, in place: the same lanes read and write a row, so the inputs may be the outputs
    # (copies of one layout on both sides: the layout decides the vector width, and that the order of the norm's sum)
    q2, k2 = q.contiguous().clone(), k.contiguous().clone()
    want = torch.empty_like(q2), torch.empty_like(k2)
    ctx.qk_norm_rope(q2, k2, None, None, freq, pos, *want, interleaved=interleaved, stream=stream())
    ctx.qk_norm_rope(q2, k2, None, None, freq, pos, q2, k2, interleaved=interleaved, stream=stream())
    assert torch.equal(q2, want[0]) and torch.equal(k2, want[1])
    check_forward(q2, q, None, pos, freq, interleaved)


def check_backward(got, ref, x, w, grad, dtype):
    # dx = r (gw - u mean(gw u)): both terms are of the order of r |gw| and r |u| |gw| (rms); fp32 roundings as in
    # the forward pass for u and g, and the sum of at most 256 products, in lanes of at most 16 and 5 levels
    x, gw = x.double(), grad.double().abs().amax(-1, keepdim=True) * (1 if w is None else w.double().abs().max())
    r = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    scale = r * gw * 1.5 * (1 + (x * r).abs())
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + 64 * U * scale + torch.finfo(dtype).tiny
    assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens,hq,hk,d,rotary,interleaved,layout", CASES)
def test_backward(ctx, dtype, tokens, hq, hk, d, rotary, interleaved, layout):
    t = TYPES[dtype]
    q, k, _, qw, kw, freq, pos, rnd = inputs(t, tokens, hq, hk, d, rotary, layout, seed=1)
    gq, gk = rnd(tokens, hq, d), rnd(tokens, hk, d)
    dq, dk = torch.empty(q.shape, dtype=t, device="cuda"), torch.empty(k.shape, dtype=t, device="cuda")
    dqw, dkw = (torch.full((d,), math.nan, device="cuda") for _ in range(2))
    ws = torch.full((ctx.qk_norm_rope_backward_workspace(q, k),), 255, dtype=torch.uint8, device="cuda")
    call = lambda *out: ctx.qk_norm_rope_backward(q, k, qw, kw, freq if rotary else None, pos, gq, gk, *out, ws,  # noqa: E731
                                                  interleaved=interleaved, stream=stream())
    call(dq, dk, dqw, dkw)
    for x, w, g, dx, dw in ((q, qw, gq, dq, dqw), (k, kw, gk, dk, dkw)):
        ref, refw = plain64.norm_rope_backward(x, w, pos, freq, 1e-6, interleaved, g)
        check_backward(dx, ref, x, w, g, t)
        # sums of products that carry 32 roundings each at most, in chains of at most rows / 16 + 400 additions
        mags = (plain64.turn(g.double(), pos, freq, interleaved, back=True).abs() + g.double().abs().amax(-1, keepdim=True)) * \
            (x.double() * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()).abs()
        chain = x.shape[0] * x.shape[1] / 16 + 400
        assert ((dw.double() - refw).abs() <= (32 + chain) * U * mags.sum((0, 1))).all()
    # the same bits again, gradients written over their inputs, and weight gradients left out
    first = [x.clone() for x in (dq, dk, dqw, dkw)]
    gq2, gk2 = gq.clone(), gk.clone()
    ctx.qk_norm_rope_backward(q, k, qw, kw, freq, pos, gq2, gk2, gq2, gk2, None, dkw.zero_(), ws, interleaved=interleaved, stream=stream())
    assert torch.equal(gq2, first[0]) and torch.equal(gk2, first[1]) and torch.equal(dkw, first[3]) and torch.equal(dqw, first[2])


@pytest.mark.gpu
def test_no_tokens(ctx):
    q, k, _, qw, kw, freq, pos, _ = inputs(torch.bfloat16, 0, 4, 2, 64, 64)
    ctx.qk_norm_rope(q, k, qw, kw, freq, pos, q, k, stream=stream())
    dw = torch.full((2, 64), math.nan, device="cuda")
    ws = torch.empty(ctx.qk_norm_rope_backward_workspace(q, k), dtype=torch.uint8, device="cuda")
    ctx.qk_norm_rope_backward(q, k, qw, kw, freq, pos, q, k, q, k, dw[0], dw[1], ws, stream=stream())
    assert (dw == 0).all()  # sums over nothing


@pytest.mark.gpu
def test_far_positions_and_odd_rows(ctx):
    """Angles of far and negative positions keep their precision; a zero row stays zero; NaN and infinities
    stay in their own row."""
    q, k, _, qw, kw, freq, _, _ = inputs(torch.float32, 8, 2, 1, 64, 64, seed=3)
    pos = torch.tensor([0, 1, -1, 2 ** 20 + 1, 2 ** 31 + 7, -(2 ** 33) - 5, 10 ** 12 + 3, 4], device="cuda")
    q[2] = 0
    ko, qo = torch.empty_like(k), torch.empty_like(q)
    ctx.qk_norm_rope(q, k, qw, kw, freq, pos, qo, ko, stream=stream())
    # the angle's own rounding in 64 bits: |angle| * 2^-52 radians at most, on both sides
    ref = plain64.norm_rope(q, qw, pos, freq, 1e-6, False)
    extra = (pos.abs().double() * 2.0 ** -51)[:, None, None] * pair_magnitude(ref, 32, False)
    assert ((qo.double() - ref).abs() <= (U + 24 * U) * pair_magnitude(ref, 32, False) + extra + 1e-37).all()
    assert (qo[2] == 0).all()
    q[5, 1, 3], q[6, 0, 60] = math.nan, math.inf
    again = torch.empty_like(q)
    ctx.qk_norm_rope(q, k, qw, kw, freq, pos, again, ko, stream=stream())
    assert again[5, 1].isnan().all() and again[6, 0].isnan().any()
    again[5, 1], again[6, 0] = qo[5, 1], qo[6, 0]
    assert torch.equal(again, qo)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens,page,hq,hk,d,heads_first,layout", [
    ("bf16", 1, 16, 32, 8, 128, False, "joint"), ("bf16", 700, 16, 4, 2, 128, False, "joint"), ("f16", 45, 8, 3, 1, 64, True, "plain"),
    ("f32", 45, 1, 3, 3, 64, False, "plain"), ("f32", 1300, 32, 2, 1, 256, True, "joint"), ("bf16", 45, 64, 2, 2, 80, True, "odd")])
def test_append(ctx, dtype, tokens, page, hq, hk, d, heads_first, layout):
    t = TYPES[dtype]
    q, k, v, qw, kw, freq, pos, rnd = inputs(t, tokens, hq, hk, d, d, layout, seed=2)
    pages = -(-tokens // page) + 2
    caches = [rnd(pages, hk, page, d).transpose(1, 2) if heads_first else rnd(pages, page, hk, d) for _ in range(2)]
    before = [c.clone() for c in caches]
    slots = torch.randperm(pages * page, device="cuda")[:tokens]
    slots[tokens // 2::3] = -1
    qo, ko = torch.empty(q.shape, dtype=t, device="cuda"), torch.empty(k.shape, dtype=t, device="cuda")
    ctx.qk_norm_rope(q, k, qw, kw, freq, pos, qo.clone(), ko, stream=stream())
    ctx.qk_norm_rope_append(q, k, v, qw, kw, freq, pos, slots, qo, *caches, stream=stream())
    ctx.synchronize(stream())
    check_forward(qo, q, qw, pos, freq, False)
    check_forward(ko, k, kw, pos, freq, False)
    for cache, old, rows in zip(caches, before, (ko, v)):
        kept = slots >= 0
        old[slots[kept] // page, slots[kept] % page] = rows[kept]
        assert torch.equal(cache, old)  # the same bits as without the cache, and no other row touched


@pytest.mark.gpu
def test_a_slot_outside_the_cache_is_skipped_and_reported(ctx):
    q, k, v, qw, kw, freq, pos, rnd = inputs(torch.bfloat16, 4, 2, 1, 64, 64)
    kc, vc = rnd(3, 8, 1, 64), rnd(3, 8, 1, 64)
    before = kc.clone(), vc.clone()
    qo = torch.empty_like(q)
    for bad in (24, -2, 1 << 40):
        ctx.qk_norm_rope_append(q, k, v, qw, kw, freq, pos, torch.tensor([-1, -1, bad, -1], device="cuda"), qo, kc, vc, stream=stream())
        with pytest.raises(kh.KernelhError, match="token 2") as e:
            ctx.synchronize(stream())
        assert e.value.code == kh.BAD_DEVICE_INDEX
        assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    ctx.synchronize(stream())  # said once
    check_forward(qo, q, qw, pos, freq, False)


@pytest.mark.gpu
def test_captured_calls_and_other_streams(ctx):
    """Two captured backward passes with workspaces of their own, replayed at the same time on two streams, give
    what eager calls give."""
    sets, graphs, want = [], [], []
    for seed in (7, 8):
        q, k, _, qw, kw, freq, pos, rnd = inputs(torch.bfloat16, 2500, 8, 2, 128, 128, seed=seed)
        s = dict(q=q, k=k, w=(qw, kw, freq, pos), gq=rnd(*q.shape), gk=rnd(*k.shape), dq=torch.empty_like(q), dk=torch.empty_like(k),
                 dw=torch.zeros(2, 128, device="cuda"), ws=torch.empty(ctx.qk_norm_rope_backward_workspace(q, k), dtype=torch.uint8, device="cuda"))

        def call(st, s=s):
            ctx.qk_norm_rope_backward(s["q"], s["k"], *s["w"], s["gq"], s["gk"], s["dq"], s["dk"], s["dw"][0], s["dw"][1], s["ws"], stream=st)

        call(stream())
        torch.cuda.synchronize()
        want.append([s[n].clone() for n in ("dq", "dk", "dw")])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(stream())
        for n in ("dq", "dk", "dw"):
            s[n].zero_()
        sets.append(s)
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert all(torch.equal(s[n], x) for n, x in zip(("dq", "dk", "dw"), w))

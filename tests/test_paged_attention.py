"""Attention of new tokens over a paged cache, against the 64-bit definition, at the lengths, layouts and masks
where the kernels change their paths; and a run of the operators around it together.

Tolerance of one output value. Scores: products of 16-bit values are exact in fp32, products of fp32 values lose
2^-21 (two 11-bit parts each, the product of the low parts dropped, the low parts cut to 11 bits); a sum of
head_dim of them in fp32 loses at most head_dim * 2^-23 of sum |q||k| <= |q| |k|, with the scale and the exponent's
rounding: ds = (head_dim + 16) 2^-23 |q| max|k| scale, plus 2^-23 of the exponent's argument, below 2 ds again.
A probability is off by at most 2 (ds + 2^-22) of itself (its own and the sum's), plus eps/2 where it is rounded to
the values' type (16-bit types; 2^-21 in fp32). The weighted sum adds at most 2^-23 per addition in a chain of
kv / 8 + 64. All of these are relative to sum p |v|; the result is rounded once, eps/2 of its value. The
log-sum-exp is off by at most ds + 2^-22 (its sum) + 2^-23 of its value, twice."""
import math

import pytest

torch = pytest.importorskip("torch")
import kernelh_b200 as kh
from tests import plain64

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# --------------------------------------------------------------------------- no device
def call(**over):
    a = dict(dtype=1, q_heads=8, k_heads=2, head_dim=64, tokens=8, batch=2, max_q_len=4, max_kv_len=100, causal=1, window=0,
             scale=0.125, q=(4096, 512, 64), o=(8192, 512, 64), lse=4096, k_cache=(4096, 2048, 128, 64), v_cache=(4096, 2048, 128, 64),
             num_pages=10, page_size=16, table_width=7, page_table=4096, table_stride=7, q_start=4096, kv_len=4096, workspace=4096,
             workspace_bytes=1 << 30)
    assert set(over) <= set(a)
    a.update(over)
    rows, paged = ("q", "o"), ("k_cache", "v_cache")
    return kh.PagedAttentionArgs(**{k: kh.HeadRows(*v) if k in rows else kh.PagedRows(*v) if k in paged else v for k, v in a.items()})


@pytest.mark.parametrize("over,words", [
    (dict(dtype=3), "dtype must be"), (dict(q_heads=7), "multiple of k_heads"), (dict(k_heads=0), "multiple of k_heads"),
    (dict(head_dim=60), "head_dim must be a multiple of 8"), (dict(head_dim=264), "head_dim must be a multiple of 8"),
    (dict(tokens=-1), "tokens * q_heads"), (dict(tokens=1 << 30), "tokens * q_heads"), (dict(tokens=1 << 62), "tokens * q_heads"), (dict(batch=-1), "must not be negative"),
    (dict(causal=2), "causal"), (dict(window=-1), "window"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(num_pages=0), "num_pages"), (dict(page_size=0), "page_size"), (dict(table_width=1 << 28), "page table row"),
    (dict(table_stride=6), "rows of the page table overlap"), (dict(q=(0, 512, 64)), "buffer 'q' is null"),
    (dict(q=(4104, 512, 64)), "rows of 'q' do not start"), (dict(q=(4096, 516, 64)), "rows of 'q' do not start"),
    (dict(o=(8192, 512, 32)), "rows of output 'o' overlap"), (dict(o=(4096, 512, 64)), "o must not be q"),
    (dict(k_cache=(4096, 2048, 124, 64)), "rows of 'k_cache' do not start"), (dict(v_cache=(0, 1, 1, 1)), "buffer 'v_cache' is null"),
    (dict(page_table=0), "'page_table' is null"), (dict(q_start=0), "'q_start' is null"), (dict(kv_len=4098), "'kv_len' is not 4-byte"),
    (dict(lse=4097), "'lse' is not 4-byte"), (dict(workspace=0), "the workspace must have"), (dict(workspace_bytes=16), "the workspace must have"),
    (dict(workspace=4104), "workspace is not 16-byte aligned")])
def test_refusals(over, words):
    assert kh.lib.kh_paged_attention(None, call(**over), None) == kh.USAGE_ERROR
    assert words in kh.lib.kh_last_error().decode()


def test_good_arguments_get_as_far_as_the_context():
    for over in (dict(), dict(lse=0), dict(tokens=1, batch=1, table_stride=0, q=(4096, 1, 64), o=(8192, 3, 64)),
                 dict(tokens=0, q=(0, 0, 0)), dict(batch=0), dict(page_table=0, table_width=0, table_stride=0)):
        assert kh.lib.kh_paged_attention(None, call(**over), None) == kh.USAGE_ERROR
        assert "null kernelh_b200 context" in kh.lib.kh_last_error().decode()
    assert kh.lib.kh_paged_attention(None, None, None) == kh.USAGE_ERROR


def test_the_workspace_covers_the_call_and_is_bounded():
    for dtype in (0, 1, 2):
        for d in (8, 64, 80, 128, 256):
            small = kh.lib.kh_paged_attention_workspace(call(dtype=dtype, head_dim=d))
            large = kh.lib.kh_paged_attention_workspace(call(dtype=dtype, head_dim=d, tokens=1 << 20, batch=1 << 14, max_kv_len=1 << 30))
            assert 0 < small <= large <= 128 << 20  # it does not grow with the lengths
    # a larger call never needs less: the launch on a device with fewer SMs is a smaller one
    sizes = [kh.lib.kh_paged_attention_workspace(call(dtype=0, head_dim=128, tokens=n, max_kv_len=1)) for n in range(1, 1500, 7)]
    assert sizes == sorted(sizes)


def test_tensor_refusals():
    ctx = kh.Context.__new__(kh.Context)
    ctx._h, ctx._ordinal = None, 0
    q, c, n = torch.zeros(3, 4, 64), torch.zeros(2, 8, 2, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(kh.KernelhError, match="must be int32"):
        ctx.paged_attention(q, c, c, n, n, n, q, 1, 1, q)
    with pytest.raises(kh.KernelhError, match="must be on device 0"):
        ctx.paged_attention(q, c, c, n[None], n, n, q, 1, 1, q)
    with pytest.raises(kh.KernelhError, match="must be float32, bfloat16 or float16"):
        ctx.paged_attention(q.double(), c, c, n[None], n, n, q, 1, 1, q)


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


class Problem:
    """Sequences of (new tokens, keys) on shuffled pages. What no query sees - unused pages, slots past the last
    key, table entries past the last page - is NaN or nonsense. Two rows of q and o lie behind the last sequence."""

    def __init__(self, dtype, hq, hk, d, page, lens, heads_first=False, seed=0, spread=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = TYPES[dtype]

        def rnd(*shape):
            return (spread * torch.randn(*shape, generator=g, device="cuda")).to(t)

        used = [-(-kv // page) for _, kv in lens]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=g, device="cuda")
        width = max(used + [1]) + 1
        self.table = torch.full((len(lens), width + 1), 0x7fffffff, dtype=torch.int32, device="cuda")[:, :width]
        shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
        caches = [torch.full(shape, math.nan, dtype=t, device="cuda") for _ in range(2)]
        self.k, self.v = (c.transpose(1, 2) if heads_first else c for c in caches)
        at = 0
        for b, (_, kv) in enumerate(lens):
            mine = order[at:at + used[b]]
            at += used[b]
            self.table[b, :used[b]] = mine.to(torch.int32)
            for c in (self.k, self.v):
                rows = torch.full((used[b] * page, hk, d), math.nan, dtype=t, device="cuda")
                rows[:kv] = rnd(kv, hk, d)
                c[mine] = rows.view(-1, page, hk, d)
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.tokens = starts[-1]
        self.q = rnd(self.tokens + 2, hq, d)
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
        self.lens, self.dtype = lens, t
        self.o = torch.full_like(self.q, 7)
        self.lse = torch.full(self.q.shape[:2], 7.0, device="cuda")

    def hints(self):
        return dict(max_q_len=max(n for n, _ in self.lens), max_kv_len=max(kv for _, kv in self.lens))

    def run(self, ctx, workspace=None, stream_=None, hints=None, **kw):
        hints = hints or self.hints()
        ws = workspace
        if ws is None:
            ws = torch.full((ctx.paged_attention_workspace(self.q, self.k, len(self.lens), **hints),), 255, dtype=torch.uint8, device="cuda")
        ctx.paged_attention(self.q, self.k, self.v, self.table, self.q_start, self.kv_len, self.o, workspace=ws, lse=self.lse,
                            stream=stream() if stream_ is None else stream_, **hints, **kw)

    def check(self, **kw):
        d = self.q.shape[-1]
        scale = abs(kw.get("scale") or d ** -0.5)
        ref, lse = plain64.paged_attention(self.q, self.k, self.v, self.table, self.q_start, self.kv_len, **kw)
        mass, _ = plain64.paged_attention(self.q, self.k, self.v.abs(), self.table, self.q_start, self.kv_len, **kw)
        n = self.tokens
        ref, lse, mass = ref[:n], lse[:n], mass[:n]
        knorm = self.k.double().nan_to_num(0).norm(dim=-1).max()
        ds = 2 * (d + 16) * 2.0 ** -23 * scale * self.q[:n].double().norm(dim=-1) * knorm
        half = torch.finfo(self.dtype).eps / 2
        chain = max(kv for _, kv in self.lens) / 8 + 64
        tol = ((2 * ds + 2.0 ** -21 + chain * 2.0 ** -23)[..., None] + (2.0 ** -21 if half < 1e-6 else half)) * mass + half * ref.abs() + 1e-30
        if self.dtype == torch.float16:
            tol = tol + 2.0 ** -25  # half a step of its subnormal values, for probabilities too
        got = self.o[:n].double()
        assert not got.isnan().any()
        assert ((got - ref).abs() <= tol).all(), ((got - ref).abs() / tol).max()
        none = lse == -math.inf
        assert torch.equal(self.lse[:n] == -math.inf, none) and (got[none] == 0).all()
        err = (self.lse[:n].double() - lse)[~none].abs()
        assert (err <= (2 * (ds + 2.0 ** -22) + 2.0 ** -22 * lse.abs())[~none]).all()
        assert (self.o[n:] == 7).all() and (self.lse[n:] == 7).all()  # rows behind the last sequence


EDGES = [(1, 0), (1, 1), (0, 5), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 129), (0, 0), (1, 1000)]
CHUNKS = [(37, 37), (5, 1000), (1, 300), (64, 64), (16, 31), (130, 515), (0, 9), (1, 1), (33, 400)]
CASES = [  # dtype, q heads, k heads, head_dim, page, lengths, heads first, options
    ("bf16", 8, 2, 128, 16, EDGES, False, {}), ("f16", 4, 4, 64, 8, EDGES, True, {}), ("f32", 4, 4, 64, 64, EDGES, False, {}),
    ("f32", 7, 1, 128, 16, EDGES, False, {}), ("bf16", 5, 1, 80, 1, EDGES, False, {}), ("bf16", 40, 2, 96, 24, EDGES, True, {}),
    ("bf16", 2, 1, 256, 32, EDGES, False, {}), ("f32", 3, 1, 256, 5, EDGES, False, {}), ("f16", 2, 2, 8, 128, EDGES, False, {}),
    ("bf16", 8, 2, 128, 16, CHUNKS, False, {}), ("f16", 5, 1, 64, 8, CHUNKS, True, {}), ("f32", 6, 2, 80, 64, CHUNKS, False, {}),
    ("f32", 2, 1, 256, 16, CHUNKS, False, {}), ("bf16", 4, 1, 256, 128, CHUNKS, False, {}), ("bf16", 14, 2, 112, 40, CHUNKS, False, {}),
    ("bf16", 8, 2, 128, 16, CHUNKS, False, dict(causal=False)), ("f16", 4, 2, 64, 16, CHUNKS, False, dict(causal=False, window=70)),
    ("bf16", 8, 2, 128, 16, CHUNKS, False, dict(window=1)), ("f16", 8, 1, 96, 32, CHUNKS, False, dict(window=100)),
    ("f32", 2, 2, 64, 16, CHUNKS, False, dict(window=17)), ("bf16", 8, 1, 64, 16, EDGES, False, dict(window=40)),
    # the same lengths with a long one among them
    ("bf16", 8, 2, 128, 16, EDGES + [(1, 9001)], False, {}), ("f32", 4, 4, 64, 64, EDGES + [(1, 9001)], False, {}), ("f16", 4, 4, 64, 8, EDGES + [(2, 5000)], True, {}),
    ("bf16", 2, 1, 256, 32, EDGES + [(1, 9001)], False, {}), ("f32", 3, 1, 256, 5, EDGES + [(3, 2500)], False, dict(window=700)), ("bf16", 5, 1, 80, 1, EDGES + [(1, 4500)], False, {}),
    ("bf16", 2, 1, 256, 16, CHUNKS + [(7, 6000)], False, dict(window=3000)), ("f32", 4, 2, 128, 16, CHUNKS + [(7, 2200)], False, {}),
    # one item for every two, four or eight blocks of a cluster; rows that see nothing; one key
    ("bf16", 16, 16, 64, 16, [(1, 70 + b) for b in range(8)], False, {}), ("f16", 8, 8, 128, 32, [(1, 300), (1, 1), (2, 900)], False, dict(window=64)),
    ("f32", 8, 4, 128, 16, [(4, 2), (2, 500)], False, {}), ("bf16", 8, 2, 256, 8, [(1, 2000)], True, dict(causal=False)),
    # one row of fp32, split over blocks, over a cluster and whole
    ("f32", 2, 2, 256, 5, EDGES, False, {}), ("f32", 3, 3, 80, 16, EDGES + [(1, 9001)], True, dict(window=40)), ("f32", 2, 2, 128, 64, EDGES, False, dict(causal=False)),
    ("f32", 5, 5, 128, 24, [(1, 700)] * 3 + [(1, 0)], False, dict(scale=-0.2)), ("f32", 1, 1, 8, 16, [(1, 40), (3, 90)], False, {}),
    ("f32", 8, 1, 256, 16, EDGES + [(1, 5000)], False, {}), ("f32", 12, 2, 64, 8, EDGES, True, {}), ("f32", 10, 2, 112, 16, EDGES + [(1, 5000)], False, dict(window=500)), ("f32", 4, 2, 200, 16, [(1, 900), (2, 60), (4, 33)], False, {}), ("f32", 16, 16, 64, 16, [(1, 1 + 7 * b) for b in range(64)], False, {}),
    # more new tokens than keys: the first queries see nothing
    ("bf16", 4, 2, 128, 16, [(9, 4), (70, 3), (3, 0)], False, {}), ("f32", 4, 2, 64, 16, [(9, 4), (40, 20)], False, dict(causal=False)),
    # one long sequence over all workers; many short ones
    ("bf16", 8, 1, 128, 64, [(1, 40001)], False, {}), ("f32", 4, 1, 64, 16, [(2, 20011)], True, {}),
    ("f16", 32, 8, 64, 16, [(1, 1 + 37 * b % 230) for b in range(300)], False, {}),
    ("bf16", 8, 2, 128, 16, [(300, 2300), (1, 700), (1000, 1000), (17, 17)], False, {}),
    # more sequences than a block has threads, chunks and single tokens; pages larger than a tile; one head each
    ("bf16", 4, 4, 64, 16, [(1 + 29 * (b % 9 == 4), 40 + 31 * b % 190) for b in range(700)], False, {}),
    ("f16", 2, 1, 128, 256, [(300, 1000), (129, 129), (2, 600)], True, {}), ("bf16", 1, 1, 64, 128, [(1500, 1500), (700, 900)], False, {}),
    ("bf16", 3, 3, 72, 32, [(1400, 1500)], False, dict(window=333)), ("f32", 1, 1, 64, 16, [(900, 1000), (333, 300)], False, dict(window=90)),
    # a window that is larger than the sequence, with the first queries before the first key
    ("f16", 2, 2, 64, 8, [(700, 500), (40, 900)], False, dict(window=600)),
    ("bf16", 2, 2, 64, 16, [(1, 77), (4, 4)], False, dict(scale=-0.3)), ("bf16", 8, 2, 128, 16, [(40, 77), (40, 40)], False, dict(scale=0.0)), ("f16", 2, 1, 64, 16, [(3, 77)], False, dict(scale=1e-30)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(CASES)))
def test_against_the_definition(ctx, i):
    dtype, hq, hk, d, page, lens, heads_first, kw = CASES[i]
    p = Problem(dtype, hq, hk, d, page, lens, heads_first, seed=i)
    p.run(ctx, **kw)
    ctx.synchronize(stream())
    p.check(**kw)
    first, first_lse = p.o.clone(), p.lse.clone()
    p.run(ctx, **kw)  # the same bits again
    assert torch.equal(p.o, first) and torch.equal(p.lse, first_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 64), ("f16", 64)])
def test_large_scores(ctx, dtype, d):
    """Scores of several hundred: one key takes nearly all the weight, later tiles raise the maximum."""
    p = Problem(dtype, 8, 2, d, 16, [(1, 500), (20, 700), (150, 640)], spread=6.0, seed=5)
    p.run(ctx)
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,n", [("bf16", 128, 40), ("f32", 64, 40), ("f16", 256, 40), ("bf16", 64, 3)])
def test_a_nan_stays_with_those_who_see_it(ctx, dtype, d, n):
    """A NaN in one query row stays in it; one in a key reaches the queries that see the key and no other, nor any other
    sequence."""
    p = Problem(dtype, 2, 2, d, 16, [(n, 300), (n, 200)], seed=13)
    p.run(ctx)
    want, want_lse = p.o.clone(), p.lse.clone()
    p.q[1, 1, 5] = math.nan
    bad = 300 - n + 2  # seen by the queries 2 .. n - 1 of the first sequence
    p.k[p.table[0, bad // 16].item(), bad % 16, 0, 7] = math.nan
    p.run(ctx)
    ctx.synchronize(stream())
    hit = torch.zeros(p.q.shape[:2], dtype=torch.bool, device="cuda")
    hit[1, 1] = True
    hit[2:n, 0] = True
    assert p.o[hit].isnan().all() and p.lse[hit].isnan().all()
    assert torch.equal(p.o[~hit], want[~hit]) and torch.equal(p.lse[~hit], want_lse[~hit])


@pytest.mark.gpu
def test_lengths_beyond_the_hints(ctx):
    for dtype in ("bf16", "f32"):
        p = Problem(dtype, 8, 2, 128, 16, [(300, 900), (1, 1500)], seed=6)
        for keys in (1, 200, 5000):
            p.o[:p.tokens] = math.nan
            p.run(ctx, hints=dict(max_q_len=1, max_kv_len=keys))
            p.check()


@pytest.mark.gpu
def test_parts_of_a_joint_buffer_and_no_lse(ctx):
    p = Problem("bf16", 4, 2, 64, 16, [(30, 100), (1, 50)], seed=7)
    joint = torch.zeros(p.q.shape[0], 8 * 64, dtype=p.dtype, device="cuda")
    joint[:, 64:320] = p.q.flatten(1)
    p.q = joint[:, 64:320].unflatten(1, (4, 64))
    wide = torch.full((p.q.shape[0], 6, 64), 7, dtype=p.dtype, device="cuda")
    p.o = wide[:, 1:5]
    p.run(ctx)
    p.check()
    assert (wide[:, 0] == 7).all() and (wide[:, 5] == 7).all()
    want = p.o.clone()
    ws = torch.empty(ctx.paged_attention_workspace(p.q, p.k, 2, **p.hints()), dtype=torch.uint8, device="cuda")
    ctx.paged_attention(p.q, p.k, p.v, p.table, p.q_start, p.kv_len, p.o, workspace=ws, stream=stream(), **p.hints())
    assert torch.equal(p.o, want)


def laid_out(x, layout):
    """A cache with the values of `x` in another layout (with another layout's values where slots share memory)."""
    pages, page, heads, d = x.shape
    if layout == "heads outermost":
        return x.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    if layout == "slots outermost":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if layout == "padded":  # no stride a multiple of another
        strides = (page * (heads * (d + 8) + 16) + 8, heads * (d + 8) + 16, d + 8, 1)
        y = torch.full((pages * strides[0],), math.nan, dtype=x.dtype, device="cuda").as_strided(x.shape, strides)
        return y.copy_(x)
    if layout == "one head for all":
        return x[:, :, :1].expand(-1, -1, heads, -1)
    assert layout == "slots overlap"
    flat = x[:, :, :, 0].nan_to_num(1).flatten().repeat(d)
    return flat.as_strided(x.shape, (page * 8 + 16, 8, pages * (page * 8 + 16) + 8, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["heads outermost", "slots outermost", "padded", "one head for all", "slots overlap"])
@pytest.mark.parametrize("dtype,lens", [("bf16", [(70, 500), (1, 90), (300, 300)]), ("f32", [(9, 200), (1, 90)])])
def test_cache_layouts(ctx, layout, dtype, lens):
    p = Problem(dtype, 4, 2, 64, 16, lens, seed=14)
    p.k, p.v = laid_out(p.k, layout), laid_out(p.v, layout)
    p.run(ctx)
    ctx.synchronize(stream())
    p.check()
    joint = torch.stack([p.k, p.v], dim=1)  # keys and values of a page side by side
    p.k, p.v = joint[:, 0], joint[:, 1]
    p.o.fill_(7)
    p.run(ctx)
    p.check()  # (not the same bits: the layout may choose the kernel)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 100), (1, 40)], [(200, 700), (1, 40)]])
def test_bad_device_data_is_not_accessed_and_reported(ctx, lens):
    """Pages, lengths and offsets out of range: every one is checked on the device before it is used."""
    def spoil(p, what):
        if what == "page":
            p.table[0, 2] = p.k.shape[0]
        elif what == "negative page":
            p.table[0, 0] = -1
        elif what == "length":
            p.kv_len[0] = p.table.shape[1] * 16 + 1
        elif what == "negative length":
            p.kv_len[0] = -5
        elif what == "offset":
            p.q_start[1] = -1
        else:
            p.q_start[2] = p.q.shape[0] + 1

    for what in ("page", "negative page", "length", "negative length", "offset", "end"):
        p = Problem("bf16", 8, 2, 128, 16, lens, seed=8)
        spoil(p, what)
        p.run(ctx)
        with pytest.raises(kh.KernelhError) as e:
            ctx.synchronize(stream())
        assert e.value.code == kh.BAD_DEVICE_INDEX
        ctx.synchronize(stream())
    q = Problem("bf16", 8, 2, 128, 16, lens, seed=8)
    q.run(ctx)
    ctx.synchronize(stream())
    q.check()


@pytest.mark.gpu
def test_no_tokens_and_no_sequences(ctx):
    p = Problem("bf16", 4, 2, 64, 16, [(0, 5), (0, 0)], seed=9)
    p.run(ctx)
    ctx.synchronize(stream())
    assert (p.o == 7).all()
    p.q, p.o, p.lse = p.q[:0], p.o[:0], p.lse[:0]
    p.run(ctx)
    p = Problem("bf16", 4, 2, 64, 16, [(1, 5)], seed=9)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    ctx.paged_attention(p.q, p.k, p.v, p.table[:0], p.q_start[:1], p.kv_len[:0], p.o, 1, 1, ws, stream=stream())
    ctx.synchronize(stream())
    assert (p.o == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grown", [("bf16", [(1, 901), (1, 3), (1, 77)]), ("f32", [(1, 901), (1, 3), (1, 77)]),
                                         ("bf16", [(1, 30), (200, 900), (61, 400)]), ("bf16", [(1, 9001), (1, 3), (2, 4000)])])
def test_a_captured_call_follows_the_lengths(ctx, dtype, grown):
    """Captured with one set of lengths, replayed with others; two graphs at once on two streams, each with its
    own workspace."""
    base = [(n, max(n, kv // 3)) for n, kv in grown]
    a, b = Problem(dtype, 8, 2, 128, 16, grown, seed=10), Problem(dtype, 8, 2, 128, 16, grown, seed=11)
    graphs = []
    for p in (a, b):
        final = p.kv_len.clone()
        p.kv_len.copy_(torch.tensor([kv for _, kv in base], dtype=torch.int32))
        ws = torch.empty(ctx.paged_attention_workspace(p.q, p.k, len(grown), **p.hints()), dtype=torch.uint8, device="cuda")
        p.run(ctx, ws)  # loads the kernels outside the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p.run(ctx, ws, stream_=stream())
        p.o[:p.tokens] = math.nan
        p.kv_len.copy_(final)
        graphs.append((g, ws))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    a.check()
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_prompt_and_its_continuation(ctx, dtype):
    """The operators as a model uses them: a prompt in two chunks, then single tokens, each step norms, rotation
    and append, then attention over the cache - against the definition over the whole sequence at once; in fp32
    also against this package's own causal attention of whole sequences."""
    t, hq, hk, d, page, total = TYPES[dtype], 4, 4, 64, 16, 150
    g = torch.Generator(device="cuda").manual_seed(12)
    q, k, v = ((torch.randn(2, total, h, d, generator=g, device="cuda")).to(t) for h in (hq, hk, hk))
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    freq = (10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float().cuda()
    pages = 2 * -(-total // page) + 3
    kc, vc = (torch.full((pages, page, hk, d), math.nan, dtype=t, device="cuda") for _ in range(2))
    table = torch.randperm(pages, generator=g, device="cuda")[:2 * -(-total // page)].view(2, -1).to(torch.int32)
    out, turned = torch.empty(2, total, hq, d, dtype=t, device="cuda"), torch.empty(2, total, hq, d, dtype=t, device="cuda")
    ws = torch.empty(ctx.paged_attention_workspace(q[0], kc, 2, 100, total), dtype=torch.uint8, device="cuda")
    done = 0
    for n in [100, 37] + [1] * 13:
        at = torch.arange(done, done + n, device="cuda")
        slots = (table[:, at // page].long() * page + at % page).flatten()
        qn = torch.empty(2 * n, hq, d, dtype=t, device="cuda")
        ctx.qk_norm_rope_append(*(x[:, done:done + n].reshape(2 * n, -1, d) for x in (q, k, v)), qw, kw, freq, at.repeat(2), slots,
                                qn, kc, vc, stream=stream())
        o = torch.empty_like(qn)
        ctx.paged_attention(qn, kc, vc, table, torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda"),
                            torch.full((2,), done + n, dtype=torch.int32, device="cuda"), o, n, done + n, ws, stream=stream())
        out[:, done:done + n], turned[:, done:done + n] = o.view(2, n, hq, d), qn.view(2, n, hq, d)
        done += n
    ctx.synchronize(stream())
    p = Problem.__new__(Problem)
    p.q, p.k, p.v, p.table, p.dtype = turned.flatten(0, 1), kc, vc, table, t
    p.q_start = torch.tensor([0, total, 2 * total], dtype=torch.int32, device="cuda")
    p.kv_len = torch.full((2,), total, dtype=torch.int32, device="cuda")
    p.lens, p.tokens, p.o = [(total, total)] * 2, 2 * total, out.flatten(0, 1)
    _, lse = plain64.paged_attention(p.q, kc, vc, table, p.q_start, p.kv_len)
    p.lse = lse.float()
    p.check()
    pos = torch.arange(total, device="cuda")
    for b in range(2):
        ref = plain64.norm_rope(q[b], qw, pos, freq, 1e-6, False)
        assert ((turned[b].double() - ref).abs() <= (torch.finfo(t).eps / 2 + 2.0 ** -18) * ref.abs().amax(-1, keepdim=True)).all()
    if dtype == "f32":
        whole = torch.empty(2, hq, total, d, device="cuda")
        keys = kc[table.long()].view(2, -1, hk, d)[:, :total]
        values = vc[table.long()].view(2, -1, hk, d)[:, :total]
        ctx.launch("attention", f"batch=2,heads={hq},seq={total},head_dim={d},causal=1",
                   [x.transpose(1, 2).contiguous() for x in (turned, keys, values)] + [whole], stream())
        ctx.synchronize(stream())
        # both are held to about 1e-5 of sum p |v| by their own tests; values here are below 4.5 in magnitude
        assert (whole.transpose(1, 2) - out).abs().max() <= 1e-4

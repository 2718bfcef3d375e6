"""The paged operators on the GPU against plain 64-bit implementations: rotary positions, written rows, forks and compaction, attention
over pages. Needs a B200.

Tolerances follow from the roundings (a half step is eps / 2 of the value): see `attn_bound` and the comments beside each test."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from mechta_b200 import _lib, kv

pytestmark = pytest.mark.gpu
F16, F32 = kv.KvFormat.F16, kv.KvFormat.F32
FMTS = [F16, F32]
HALF_STEP = {torch.float16: 2.0**-11, torch.float32: 2.0**-24}


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "these tests need the GPU"
    torch.cuda.set_device(0)
    c = kv.KvContext(0, torch.cuda.current_stream())
    yield c
    c.close()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


# ---- rotary positions ----------------------------------------------------------------------------------------------

def rotate64(x, positions, f, m, layout, backward=False):
    rot = 2 * len(f)
    a = positions.double()[:, None, None] * torch.from_numpy(np.asarray(f)).cuda()
    c, s = m * torch.cos(a), m * torch.sin(a) * (-1 if backward else 1)
    y = x.double().clone()
    u, w = (x[..., :rot:2].double(), x[..., 1:rot:2].double()) if layout == "interleaved" else (x[..., : rot // 2].double(), x[..., rot // 2: rot].double())
    p, q = u * c - w * s, u * s + w * c
    if layout == "interleaved":
        y[..., :rot:2], y[..., 1:rot:2] = p, q
    else:
        y[..., : rot // 2], y[..., rot // 2: rot] = p, q
    return y


def rope_bound(x, rot, m, dtype, layout):
    """Cosine and sine are off by the f32 rounding of the angle's fraction of a turn (at most pi * 2^-24 * 2 radians) and a few half
    steps of sincospi and of the factor: under 2^-21 of each product in all with the two products' and the sum's own; then one
    rounding to the output's type (half a step of the subnormals at least)."""
    u, w = (x[..., :rot:2], x[..., 1:rot:2]) if layout == "interleaved" else (x[..., : rot // 2], x[..., rot // 2: rot])
    size = m * (u.double().abs() + w.double().abs())
    size = size.repeat_interleave(2, -1) if layout == "interleaved" else torch.cat((size, size), -1)
    size = torch.cat((size, x[..., rot:].double().abs()), -1)
    return size * (2.0**-21 + HALF_STEP[dtype]) + (2.0**-25 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("heads,dim,rot,layout", [(16, 256, 64, "half"), (3, 128, 128, "interleaved"), (5, 64, 30, "half"), (2, 80, 36, "interleaved"),
                                                  (1, 30, 2, "half"), (7, 33, 32, "half"), (2, 256, 256, "half"), (40, 1000, 256, "interleaved")])
@pytest.mark.parametrize("src,dst", [(torch.float32, torch.float16), (torch.float16, torch.float16), (torch.float32, torch.float32), (torch.float16, torch.float32)])
def test_rope(ctx, heads, dim, rot, layout, src, dst):
    g = gen(heads * 1000 + dim)
    for n, far, scaling in ((1, 5, "none"), (37, 1 << 20, "yarn"), (300, 2**31 - 1, "linear")):
        rope = kv.Rope(ctx, rot, layout=layout, scaling=scaling, factor=4.0, original=4096)
        f, m = rope.freqs()
        x = randn(g, n, heads, dim, dtype=src)
        pos = torch.randint(-3, far, (n,), device="cuda", generator=g, dtype=torch.int32)
        for backward in (False, True):
            out = torch.full((n, heads, dim), math.nan, device="cuda", dtype=dst)
            rope.apply(x, pos, out, backward=backward)
            want = rotate64(x, pos, f, m, layout, backward)
            assert ((out.double() - want).abs() <= rope_bound(x, rot, m, dst, layout)).all(), (n, scaling, backward)


def test_rope_in_place_strided_and_gradient(ctx):
    g = gen(3)
    rope = kv.Rope(ctx, 64, scaling="yarn", factor=4.0, original=4096)
    f, m = rope.freqs()
    qf = randn(g, 5, 16, 512)  # query and gate side by side, as the step's input
    pos = torch.arange(9000, 9005, device="cuda", dtype=torch.int32)
    want, gate = rotate64(qf[..., :256], pos, f, m, "half"), qf[..., 256:].clone()
    bound = rope_bound(qf[..., :256], 64, m, torch.float32, "half")
    view = qf[..., :256]
    rope.apply(view, pos, view)
    assert ((view.double() - want).abs() <= bound).all() and torch.equal(qf[..., 256:], gate)
    # heads outside tokens, odd addresses and strides: rows of a [heads][tokens][dims + 1] buffer
    buf = torch.zeros(16, 5, 257, device="cuda")
    x, y = randn(g, 16, 5, 257)[..., 1:].transpose(0, 1), buf[..., 1:].transpose(0, 1)
    for layout in ("half", "interleaved"):
        r = kv.Rope(ctx, 64, layout=layout)
        r.apply(x, pos, y)
        assert ((y.double() - rotate64(x, pos, r.freqs()[0], 1.0, layout)).abs() <= rope_bound(x, 64, 1.0, torch.float32, layout)).all()
    assert not buf[..., 0].any()
    # <R x, y> = <x, R^T y>, and against differences: the map is linear, so a step in x gives R of the step
    a, b = randn(g, 5, 4, 64), randn(g, 5, 4, 64)
    ra, rb = torch.empty_like(a), torch.empty_like(b)
    rope.apply(a, pos, ra)
    rope.apply(b, pos, rb, backward=True)
    lhs, rhs = (ra.double() * b.double()).sum(), (a.double() * rb.double()).sum()
    assert abs(lhs - rhs) <= 2 * (rope_bound(a, 64, m, torch.float32, "half") * b.double().abs()).sum()
    d = torch.zeros_like(a)
    d[2, 1, 40] = 1.0
    up, down = torch.empty_like(a), torch.empty_like(a)
    rope.apply(a + d, pos, up)
    rope.apply(a - d, pos, down)
    slope = ((up.double() - down.double()) / 2 * b.double()).sum()  # d<R x, b> / dx[2, 1, 40]
    slack = (2 * rope_bound(a.abs() + d, 64, m, torch.float32, "half") * b.double().abs())[2, 1].sum() + HALF_STEP[torch.float32] * 8
    assert abs(slope - rb[2, 1, 40].double()) <= slack
    rope.apply(torch.empty(0, 4, 64, device="cuda"), pos[:0], torch.empty(0, 4, 64, device="cuda"))
    for bad in ((a, pos[:4], ra), (a, pos.long(), ra), (a, pos, ra[:, :2]), (a.cpu(), pos, ra), (a[:, :1].expand(5, 4, 64), pos, ra), (a, pos, a[:, :, :].flip(0)[:, ::2]),
                (a.double(), pos, ra), (a, pos, ra[:, :, ::2])):
        with pytest.raises(_lib.MkvError):
            rope.apply(*bad)


# ---- a pool and its plain twin ---------------------------------------------------------------------------------------

def rows_of(pool, seq, layer=0, upto=None):
    """K and V rows of a sequence, in order."""
    pages = torch.from_numpy(pool.pages(seq).astype(np.int64)).cuda()
    n = pool.length(seq) if upto is None else upto
    return [t[pages].reshape(-1, pool.kv_heads, pool.head_dim)[:n] for t in pool.buffer_tensors(layer)]


def scattered(ctx, fmt, lens, page, seed, layers=1, spare=8, poison=None, heads=(16, 2, 256), longest=None):
    """A pool whose sequences have N(0, 1) rows on pages that lie among one another's; what no sequence has holds `poison`."""
    hq, hkv, dim = heads
    need = sum(-(-n // page) for n in lens) + spare
    pool = kv.KvPool(ctx, fmt, layers, need, page, len(lens) + 8, longest or max(max(lens), 1) + 600, hq, hkv, dim)
    g = gen(seed)
    ids = [pool.create() for _ in lens]
    for r in range(1, 6):
        for i, n in zip(ids, lens):
            pool.set_len(i, n * r // 5)
    for l in range(layers):
        for t in pool.buffer_tensors(l):
            if poison is None:
                t.normal_(generator=g)
            else:
                t.fill_(poison)
                for i, n in zip(ids, lens):
                    pages = torch.from_numpy(pool.pages(i).astype(np.int64)).cuda()
                    data = torch.full((len(pages) * page, hkv, dim), poison, device="cuda", dtype=t.dtype)
                    data[:n] = randn(g, n, hkv, dim, dtype=t.dtype)
                    t[pages] = data.view(len(pages), page, hkv, dim)
    return pool, ids, g


# ---- written rows ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,page,rot,layout,src", [((16, 2, 256), 16, 64, "half", torch.float32), ((32, 4, 128), 64, 128, "interleaved", torch.float16),
                                                       ((3, 3, 64), 128, 30, "half", torch.float32), ((8, 1, 64), 256, 0, "half", torch.float16),
                                                       ((16, 2, 256), 32, 54, "interleaved", torch.float32)])
def test_write(ctx, fmt, heads, page, rot, layout, src):
    lens = [0, 1, 15, 16, 17, 250, 256, 999]
    news = [1, 0, 3, 40, 1, 7, 300, 2]
    pool, ids, g = scattered(ctx, fmt, lens, page, 5, layers=2, spare=60, heads=heads)
    before = [rows_of(pool, i) for i in ids]
    other = [t.clone() for t in pool.buffer_tensors(1)]
    rope = kv.Rope(ctx, rot, layout=layout) if rot else None
    total = sum(news)
    wide = torch.zeros(total, 2 * heads[1] + 1, heads[2], device="cuda", dtype=src)  # k and v inside a wider buffer
    wide.normal_(generator=g)
    k, v = wide[:, :heads[1]], wide[:, heads[1]:2 * heads[1]]
    pool.write(0, [(i, 0, n, m) for i, n, m in zip(ids, lens, news)], k, v, rope)
    at = 0
    for i, n, m, (k0, v0) in zip(ids, lens, news, before):
        assert pool.length(i) == n + m
        k1, v1 = rows_of(pool, i)
        assert torch.equal(k1[:n], k0) and torch.equal(v1[:n], v0)
        kn, vn = k[at:at + m], v[at:at + m]
        assert torch.equal(v1[n:], vn.to(v1.dtype))
        if rope is None:
            assert torch.equal(k1[n:], kn.to(k1.dtype))
        elif m:
            pos = torch.arange(n, n + m, device="cuda")
            want, bound = rotate64(kn, pos, rope.freqs()[0], 1.0, layout), rope_bound(kn, rot, 1.0, k1.dtype, layout)
            assert ((k1[n:].double() - want).abs() <= bound).all()
        at += m
    for t, o in zip(pool.buffer_tensors(1), other):
        assert torch.equal(t, o)
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_steps_with_rollback_and_copy_on_write(ctx, fmt):
    """Layers written one after the other, refused drafts overwritten, forks that go their own ways: every sequence keeps its rows."""
    page, layers = 16, 3
    pool = kv.KvPool(ctx, fmt, layers, 60, page, 9, 1000)
    g = gen(8)
    truth = {}
    a = pool.create()
    truth[a] = [[torch.empty(0, 2, 256, device="cuda", dtype=pool.fmt.torch_dtype) for _ in range(2)] for _ in range(layers)]

    def step(plan):  # (sequence, pos, ntok)
        rows = sum(n for _, _, n in plan)
        for l in range(layers):
            k, v = randn(g, rows, 2, 256), randn(g, rows, 2, 256)
            pool.write(l, [(s, 0, p, n) for s, p, n in plan], k, v)
            at = 0
            for s, p, n in plan:
                for j, x in enumerate((k, v)):
                    truth[s][l][j] = torch.cat((truth[s][l][j][:p], x[at:at + n].to(pool.fmt.torch_dtype)))
                at += n
        verify()

    def verify():
        for s, t in truth.items():
            for l in range(layers):
                for got, want in zip(rows_of(pool, s, l), t[l]):
                    assert torch.equal(got, want)

    def fork(s, length, n, copy=False):
        kids = pool.fork(s, length, n, copy)
        for c in kids:
            truth[c] = [[x[:length].clone() for x in kv_] for kv_ in truth[s]]
        return kids

    step([(a, 0, 37)])
    step([(a, 37, 4)])
    step([(a, 39, 4)])          # two of the four were accepted
    b, c = fork(a, 41, 2)
    free = pool.free_pages
    step([(b, 41, 1), (a, 43, 4), (c, 41, 3)])  # c is the last on the page that all three had: two copies
    assert pool.free_pages == free - 2
    step([(b, 30, 2)])          # back into a page that is shared: rows 32.. of b are gone, 16..29 copied
    d = fork(c, 44, 1, copy=True)[0]
    step([(d, 44, 30), (c, 44, 1)])
    # with no free page a write that needs one is refused and changes nothing
    hold = pool.create()
    pool.set_len(hold, pool.free_pages * page)
    assert pool.free_pages == 0
    e = fork(d, 74, 1)[0]
    k = randn(g, 2, 2, 256)
    for plan in ([(e, 0, 74, 1), (c, 0, 45, 1)], [(c, 0, 45, 1), (e, 0, 74, 1)]):
        with pytest.raises(_lib.MkvError) as err:
            pool.write(0, plan, k, k)
        assert err.value.status == _lib.ERR_NOMEM
    verify()
    # d and e share every page: when both write, one needs a page; d gives its part up first
    pool.truncate(d, 64)
    truth[d] = [[x[:64] for x in kv_] for kv_ in truth[d]]
    step([(e, 74, 1)])
    pool.free([hold, a])
    del truth[a]
    moved = pool.compact()
    assert moved > 0
    verify()
    assert pool.compact() == 0
    step([(b, 32, 40), (e, 75, 1), (c, 45, 2)])
    pool.close()


@pytest.mark.parametrize("fmt,page,length,layers", [(F16, 16, 100, 3), (F32, 256, 700, 2), (F16, 64, 9001, 10), (F32, 32, 6000, 1)])
def test_copies_and_compaction(ctx, fmt, page, length, layers):
    """More pages than one launch lists, holes in between; rows behind the last page's stay as they were."""
    m = -(-length // page)
    pool, ids, g = scattered(ctx, fmt, [length, length // 3, 40], page, 11, layers=layers, spare=4 * m)
    want = [[t.clone() for t in rows_of(pool, ids[0], l)] for l in range(layers)]
    tails = [[t.clone() for t in pool.buffer_tensors(l)] for l in range(layers)]
    twin = pool.fork(ids[0], copy=True)[0]
    assert not set(pool.pages(twin)) & set(pool.pages(ids[0]))
    last = int(pool.pages(twin)[-1])
    for l in range(layers):
        for t, o in zip(pool.buffer_tensors(l), tails[l]):
            if length % page:
                assert torch.equal(t[last, length % page:], o[last, length % page:])
    kids = pool.fork(twin, length // 2, 2)
    pool.free([ids[0], ids[2]])
    assert pool.compact() > 0
    used = {int(p) for s in [twin, ids[1], *kids] for p in pool.pages(s)}
    assert used == set(range(len(used))) and pool.free_pages == pool.n_pages - len(used)
    for l in range(layers):
        for s, n in [(twin, length)] + [(c, length // 2) for c in kids]:
            for got, w in zip(rows_of(pool, s, l), want[l]):
                assert torch.equal(got, w[:n])
    pool.close()


# ---- attention -----------------------------------------------------------------------------------------------------------

def attn64(pool, items, q, window=0, sinks=None, scale=None, layer=0):
    """From the formula, in 64 bits: the outputs, and what their tolerance is made of: sum of weight * |v|, sum of |q k| * scale at its
    largest, the largest |v| among the keys seen, the number of keys."""
    group = pool.q_heads // pool.kv_heads
    scale = scale or pool.head_dim**-0.5
    outs, mags, qks, tops, at = [], [], [], [], 0
    for s, first, pos, n in items:
        if n == 0:
            continue
        k, v = rows_of(pool, s, layer, pos + n)
        k, v, x = k.double().transpose(0, 1), v.double().transpose(0, 1), q[at:at + n].double().transpose(0, 1)
        at += n
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        key, tok = torch.arange(pos + n, device="cuda")[None], torch.arange(pos, pos + n, device="cuda")[:, None]
        seen = (key <= tok) & (key >= first)
        if window:
            seen &= key > tok - window
        score = (x @ k.transpose(1, 2)) * scale
        score = torch.where(seen, score, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
        top = score.amax(-1, keepdim=True)
        if sinks is not None:
            top = torch.maximum(top, sinks.double()[:, None, None])
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        w = torch.exp(score - top)
        total = w.sum(-1, keepdim=True)
        if sinks is not None:
            total = total + torch.exp(sinks.double()[:, None, None] - top)
        w = torch.where(seen.any(-1)[None, :, None], w / total, torch.zeros_like(w))
        # (a masked row's infinities and NaN do not count)
        clean = torch.where(seen.any(0)[None, :, None], v, torch.zeros_like(v))
        outs.append((w @ clean).transpose(0, 1))
        mags.append((w @ clean.abs()).transpose(0, 1))
        qk = torch.where(seen, (x.abs() @ k.abs().transpose(1, 2)) * scale, torch.zeros_like(score))
        qks.append(qk.amax(-1, keepdim=True).transpose(0, 1))
        tops.append(torch.stack((clean.abs().amax((1, 2))[:, None, None].expand(-1, n, 1), torch.full((len(k), n, 1), float(pos + n), device="cuda",
                                                                                                      dtype=torch.float64))).transpose(1, 2))
    return torch.cat(outs), torch.cat(mags), torch.cat(qks), torch.cat(tops, 1)


def attn_bound(fmt, out, mag, qk, top):
    """f16: a weight is rounded to f16 (2^-11 of it, or half a subnormal step, 2^-25, against a largest weight of at least 1), the output
    once more; f32 sums and exponentials in between. A score is off by its f32 sums: at most 2^-20 of sum |q k| here (the tensor
    core's sums of 16 truncate: 16 steps of 2^-24 each), and a weight by as much, twice (sum and weight). f32: operands are
    split into two f16 parts (2^-23 of a value is left out, or half a subnormal step, 2^-25, where the largest of a tile of 64 keys is
    at least 2^8: 2^-33 of that largest), weights likewise; weights sum to at most 1."""
    top, keys = top
    exponent = 2 * qk * 2.0**-20 + 2.0**-20
    if fmt == F16:
        return mag * (2.0**-11 * 1.03 + exponent) + out.abs() * 2.0**-11 + top * keys * 2.0**-25 + 2.0**-25
    return mag * (2.0**-20 + exponent) + top * 2.0**-33 + 1e-30


def run_attn(pool, items, q, **kw):
    out = torch.full_like(q, math.nan)
    pool.attn(0, items, q, out, **kw)
    return out


def check_attn(pool, items, q, **kw):
    got = run_attn(pool, items, q, **kw)
    want, mag, qk, top = attn64(pool, items, q, **kw)
    off = (got.double() - want).abs()
    bound = attn_bound(pool.fmt, want, mag, qk, top)
    assert (off <= bound).all(), f"worst {float((off / bound).nan_to_num(1e9).max()):.3g} of the bound, {int((~(off <= bound)).sum())} values"
    return got


GEOMETRIES = [(16, 2, 256), (32, 4, 128), (4, 4, 64), (12, 4, 128), (5, 1, 256), (64, 1, 64), (40, 2, 64), (128, 2, 128)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads", GEOMETRIES)
def test_attention_layouts(ctx, fmt, heads):
    """Decode steps, drafts and blocks together, over every head layout; pages that end inside a tile."""
    lens = [1, 2, 16, 63, 64, 65, 127, 128, 129, 200, 513, 1000]
    news = [1, 2, 3, 1, 64, 4, 127, 1, 5, 33, 17, 300]
    for page in (16, 128):
        pool, ids, g = scattered(ctx, fmt, lens, page, sum(heads) + page, heads=heads)
        q = randn(g, sum(news), heads[0], heads[2], dtype=pool.fmt.torch_dtype)
        check_attn(pool, [(i, 0, n - m, m) for i, n, m in zip(ids, lens, news)], q)
        pool.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("length,ntok", [(1, 1), (5, 3), (128, 128), (129, 1), (384, 129), (2000, 1), (3001, 4), (2500, 700)])
def test_attention_lengths(ctx, fmt, page, length, ntok):
    pool, ids, g = scattered(ctx, fmt, [length], page, length + page)
    q = randn(g, ntok, 16, 256, dtype=pool.fmt.torch_dtype)
    check_attn(pool, [(ids[0], 0, length - ntok, ntok)], q)
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads", [(16, 2, 256), (32, 4, 128), (6, 2, 64)])
@pytest.mark.parametrize("window,first", [(1, 0), (7, 0), (100, 0), (513, 0), (129, 700), (0, 650), (2**32 - 1, 0), (0, 900), (300, 2**32 - 1)])
def test_attention_windows_sinks_and_empty_rows(ctx, fmt, heads, window, first):
    """first_pos behind the first tokens, or behind all: rows that see nothing are zero, whatever the sinks."""
    lens, news = [820, 33, 1400], [150, 33, 2]
    pool, ids, g = scattered(ctx, fmt, lens, 32, window % 1000 + first % 1000, heads=heads)
    q = randn(g, sum(news), heads[0], heads[2], dtype=pool.fmt.torch_dtype)
    items = [(i, first if j != 1 else 0, n - m, m) for j, (i, n, m) in enumerate(zip(ids, lens, news))]
    for sinks in (None, 3.0 * randn(g, heads[0]), torch.full((heads[0],), -math.inf, device="cuda")):
        got = check_attn(pool, items, q, window=window, sinks=sinks)
        if first >= 1400:
            assert not got[:150].any() and not got[183:].any()
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_attention_scales_and_extreme_scores(ctx, fmt):
    """Peaked and flat softmaxes, a maximum that keeps rising along the keys, scores whose exponentials would overflow."""
    pool, ids, g = scattered(ctx, fmt, [1500], 64, 77)
    q = randn(g, 9, 16, 256, dtype=pool.fmt.torch_dtype)
    items = [(ids[0], 0, 1491, 9)]
    for scale in (1e-6, 0.02, 1.0, 20.0):
        check_attn(pool, items, q, scale=scale)
    k, _ = pool.buffer_tensors(0)
    pages = torch.from_numpy(pool.pages(ids[0]).astype(np.int64)).cuda()
    ramp = torch.linspace(-8, 8, len(pages) * 64, device="cuda").view(len(pages), 64, 1, 1)
    k[pages] = (ramp * torch.ones_like(k[pages]) * 0.25).to(k.dtype)
    q.fill_(0.5)
    for sign in (1, -1):
        check_attn(pool, items, q * sign, scale=1.0)
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads", [(16, 2, 256), (12, 4, 128), (4, 4, 64)])
def test_what_no_row_sees_stays_out(ctx, fmt, poison, heads):
    """NaN and infinities in free pages, behind the last row, in front of first_pos and of the window, and in rows of later tokens."""
    lens, news = [1, 70, 300, 515], [1, 3, 40, 130]
    pool, ids, g = scattered(ctx, fmt, lens, 32, 5, poison=poison, heads=heads)
    q = randn(g, sum(news), heads[0], heads[2], dtype=pool.fmt.torch_dtype)
    items = [(i, 0, n - m, m) for i, n, m in zip(ids, lens, news)]
    check_attn(pool, items, q)
    k, v = pool.buffer_tensors(0)

    def place(s, p):
        return int(pool.pages(ids[s])[p // 32]), p % 32

    for p in (0, 3, 100):  # in front of first_pos = 101
        k[place(3, p)] = poison
        v[place(3, p)] = poison
    items[3] = (ids[3], 101, 385, 130)
    check_attn(pool, items, q)
    check_attn(pool, items, q, window=50)
    # the rows of token 7 of the third block and of token 60 of the fourth: earlier tokens do not see them
    clean = run_attn(pool, items, q)
    for s, p in ((2, 267), (3, 445)):
        k[place(s, p)] = poison
        v[place(s, p)] = poison
    got = run_attn(pool, items, q)
    assert torch.equal(got[:4 + 7], clean[:4 + 7]) and torch.equal(got[44:44 + 60], clean[44:44 + 60])
    assert not torch.isfinite(got[4 + 7:44]).any() and not torch.isfinite(got[44 + 60:]).any()
    # with a finite K row the one bad value of V reaches its dim alone, and only rows that see it
    k[place(3, 445)], v[place(3, 445)] = 0.25, 0.5
    v[place(3, 445)][0, 5] = poison
    k[place(2, 267)], v[place(2, 267)] = 0.25, 0.5
    got = run_attn(pool, items, q, window=30)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[44 + 60:44 + 90, : heads[0] // heads[1], 5] = True
    assert torch.equal(~torch.isfinite(got), bad)
    want, mag, qk, top = attn64(pool, items[:3], q[:44], window=30)
    assert ((got[:44].double() - want).abs() <= attn_bound(fmt, want, mag, qk, top)).all()
    v[place(3, 445)][0, 5] = 0.5
    want, mag, qk, top = attn64(pool, items, q, window=30)
    assert ((got.double() - want).abs() <= attn_bound(fmt, want, mag, qk, top))[~bad].all()
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_attention_strides_shared_prefix_and_many_items(ctx, fmt):
    """q inside a wider buffer; forks that share pages; more sequences than one launch takes; the rows around an output stay."""
    pool, ids, g = scattered(ctx, fmt, [777], 16, 9, spare=600, longest=1500)
    kids = [ids[0]]
    pool.close()
    pool = kv.KvPool(ctx, fmt, 1, 900, 16, 700, 1500)
    for t in pool.buffer_tensors(0):
        t.normal_(generator=g)
    a = pool.create()
    pool.set_len(a, 777)
    kids = pool.fork(a, n=600)
    k = randn(g, 600, 2, 256)
    for _ in range(2):  # (each child its own last page)
        pool.write(0, [(c, 0, 776, 1) for c in kids[:100]], k[:100], k[:100].flip(0))
    items = [(c, 0, 770 + i % 7, 1 + (i % 3 if i % 7 < 5 else 0)) for i, c in enumerate(kids)]
    total = sum(n for *_, n in items)
    dt = pool.fmt.torch_dtype
    wide = randn(g, total, 17, 256, dtype=dt)
    q = wide[:, 1:]
    room = torch.full((total + 2, 18, 256), 7.0, device="cuda", dtype=dt)
    pool.attn(0, items, q, room[1:-1, :16])
    want, mag, qk, top = attn64(pool, items, q)
    assert ((room[1:-1, :16].double() - want).abs() <= attn_bound(fmt, want, mag, qk, top)).all()
    assert (room[:, 16:] == 7.0).all() and (room[0] == 7.0).all() and (room[-1] == 7.0).all()
    out = torch.full((0, 16, 256), 1.0, device="cuda", dtype=dt)
    pool.attn(0, [], out, out)
    pool.attn(0, [(a, 0, 5, 0)], out, out)
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_the_same_call_gives_the_same_bits(ctx, fmt):
    pool, ids, g = scattered(ctx, fmt, [5000, 40, 900], 64, 21)
    q = randn(g, 40, 16, 256, dtype=pool.fmt.torch_dtype)
    items = [(ids[0], 0, 4998, 2), (ids[1], 0, 39, 1), (ids[2], 0, 863, 37)]
    first = run_attn(pool, items, q)
    for _ in range(20):
        assert torch.equal(run_attn(pool, items, q), first)
    pool.close()


# ---- the operators together ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FMTS)
def test_serving_run(ctx, fmt):
    """A prompt in blocks, samples forked from it, decode steps with rotated queries and rows, a session that ends, compaction: every
    output against the rows as a plain program would have kept them."""
    g, layers, page = gen(31), 2, 32
    dt = kv.KvFormat(fmt).torch_dtype
    pool = kv.KvPool(ctx, fmt, layers, 120, page, 8, 2000)
    rope = kv.Rope(ctx, 64, layout="half", scaling="yarn", factor=4.0, original=512)

    def step(plan):  # (sequence, pos, ntok)
        rows = sum(n for *_, n in plan)
        items = np.array([(s, 0, p, n) for s, p, n in plan], np.uint32)
        pos = torch.cat([torch.arange(p, p + n, device="cuda", dtype=torch.int32) for _, p, n in plan])
        for l in range(layers):
            x, k, v = randn(g, rows, 16, 512), randn(g, rows, 2, 256), randn(g, rows, 2, 256)
            q, out = torch.empty(rows, 16, 256, device="cuda", dtype=dt), torch.empty(rows, 16, 256, device="cuda", dtype=dt)
            rope.apply(x[..., :256], pos, q)
            pool.write(l, items, k, v, rope)
            pool.attn(l, items, q, out)
            want, mag, qk, top = attn64(pool, items.tolist(), q, layer=l)
            assert ((out.double() - want).abs() <= attn_bound(fmt, want, mag, qk, top)).all()

    a, z = pool.create(), pool.create()
    step([(a, 0, 300), (z, 0, 70)])
    step([(a, 300, 211), (z, 70, 1)])
    kids = pool.fork(a, n=3)
    step([(c, 511, 1) for c in kids] + [(z, 71, 4)])
    step([(z, 73, 4), (kids[1], 512, 4)])
    pool.free([a, kids[0]])
    assert pool.compact() > 0
    step([(kids[2], 512, 2), (z, 77, 1), (kids[1], 514, 3)])
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_captured_step_replays(ctx, fmt):
    """A captured rotation, write and attention, replayed with other inputs in the same memory; eager calls of the pool in between."""
    stream = torch.cuda.Stream()
    c2 = kv.KvContext(0, stream)
    with torch.cuda.stream(stream):
        pool, ids, g = scattered(c2, fmt, [3000, 100], 64, 41)
        dt = pool.fmt.torch_dtype
        rope = kv.Rope(c2)
        items = np.array([(ids[0], 0, 3000, 2), (ids[1], 0, 100, 2)], np.uint32)
        pos = torch.tensor([3000, 3001, 100, 101], device="cuda", dtype=torch.int32)
        x, k, v = randn(g, 4, 16, 256), randn(g, 4, 2, 256), randn(g, 4, 2, 256)
        q, out = torch.empty(4, 16, 256, device="cuda", dtype=dt), torch.empty(4, 16, 256, device="cuda", dtype=dt)

        def step():
            rope.apply(x, pos, q)
            pool.write(0, items, k, v, rope)
            pool.attn(0, items, q, out)

        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(3):
            for t in (x, k, v):
                t.normal_(generator=g)
            out.fill_(math.nan)
            graph.replay()
            replayed = out.clone()
            step()
            assert torch.equal(out, replayed)
            want, mag, qk, top = attn64(pool, items.tolist(), q)
            assert ((replayed.double() - want).abs() <= attn_bound(fmt, want, mag, qk, top)).all()
        stream.synchronize()
        del graph
        pool.close()
    c2.close()


def test_context_outlives_and_launches_count(ctx):
    c2 = kv.KvContext(0, torch.cuda.current_stream())
    pool = kv.KvPool(c2, F16, 1, 8, 16, 2, 100)
    a = pool.create()
    n0 = c2.launches
    pool.write(0, [(a, 0, 0, 20)], torch.ones(20, 2, 256, device="cuda"), torch.ones(20, 2, 256, device="cuda"))
    assert c2.launches == n0 + 2  # the page table, the rows
    view = pool.buffer_tensors(0)[0]
    c2.close()  # the pool keeps it alive
    q = torch.ones(20, 16, 256, device="cuda", dtype=torch.float16)
    out = torch.empty_like(q)
    pool.attn(0, [(a, 0, 0, 20)], q, out)
    assert (out == 1).all()
    del pool
    assert float(view[0].float().sum()) == 16 * 512
    with pytest.raises(_lib.MkvError) as e:
        kv.KvPool(ctx, F16, 256, 2**24, 64, 1, 1000)  # 256 TB
    assert e.value.status == _lib.ERR_NOMEM


@pytest.mark.parametrize("fmt", FMTS)
def test_slices_of_one_buffer(ctx, fmt):
    """q, its rotation and the output as slices of one [tokens][heads] buffer, beside rows that stay."""
    pool, ids, g = scattered(ctx, fmt, [300, 77], 32, 61)
    dt = pool.fmt.torch_dtype
    buf = randn(g, 40, 50, 256, dtype=dt)
    keep = buf.clone()
    items = [(ids[0], 0, 263, 37), (ids[1], 0, 74, 3)]
    pos = torch.tensor([*range(263, 300), 74, 75, 76], device="cuda", dtype=torch.int32)
    rope = kv.Rope(ctx, 128, layout="interleaved")
    rope.apply(buf[:, :16], pos, buf[:, 17:33])
    f, m = rope.freqs()
    assert ((buf[:, 17:33].double() - rotate64(keep[:, :16], pos, f, m, "interleaved")).abs() <= rope_bound(keep[:, :16], 128, m, dt, "interleaved")).all()
    want, mag, qk, top = attn64(pool, items, buf[:, 17:33])
    pool.attn(0, items, buf[:, 17:33], buf[:, 34:])
    assert ((buf[:, 34:].double() - want).abs() <= attn_bound(fmt, want, mag, qk, top)).all()
    for s in (slice(0, 17), slice(33, 34)):
        assert torch.equal(buf[:, s], keep[:, s])
    pool.close()


@pytest.mark.parametrize("fmt,page", [(F16, 256), (F32, 16)])
def test_rows_beyond_four_gigabytes(ctx, fmt, page):
    """Pages whose bytes, and f32 pages whose rows times their length, pass 32 bits: written, read, shared, copied and moved."""
    row = 2 * 256 * (2 if fmt == F16 else 4)
    low = 2**32 // row + 5 * page
    pool = kv.KvPool(ctx, fmt, 1, low // page + 150, page, 8, low + 1000)
    g = gen(71)
    front, a = pool.create(), pool.create()
    pool.set_len(front, low)
    k, v = randn(g, 700, 2, 256), randn(g, 700, 2, 256)
    pool.write(0, [(a, 0, 0, 700)], k, v)
    assert pool.pages(a).min() >= low // page
    dt = pool.fmt.torch_dtype
    for x, y in zip(rows_of(pool, a), (k, v)):
        assert torch.equal(x, y.to(dt))
    b, c = pool.fork(a, 693)[0], pool.fork(a, 690, copy=True)[0]
    pool.write(0, [(b, 0, 693, 2)], v[:2], k[:2])
    q = randn(g, 30, 16, 256, dtype=dt)
    items = [(a, 0, 680, 20), (b, 3, 688, 7), (c, 0, 687, 3)]
    first = check_attn(pool, items, q)
    pool.truncate(front, 100)
    assert pool.compact() > 0 and pool.pages(a).max() < 150
    assert torch.equal(check_attn(pool, items, q), first)
    pool.close()


def test_two_streams_at_once(ctx):
    """Pools of contexts on streams of their own, with calls of both in flight together and another stream current."""
    main = torch.cuda.current_stream()
    sides = []
    for i, fmt in enumerate((F16, F32, F16)):
        stream = torch.cuda.Stream()
        c = kv.KvContext(0, stream)
        with torch.cuda.stream(stream):
            pool, ids, g = scattered(c, fmt, [9000, 500, 64], 64, 80 + i)
            q = randn(g, 72, 16, 256, dtype=pool.fmt.torch_dtype)
        stream.synchronize()
        sides.append((stream, c, pool, [(ids[0], 0, 8999, 1), (ids[1], 0, 430, 70), (ids[2], 0, 63, 1)], q, kv.Rope(c)))
    main.synchronize()
    outs = [[torch.full_like(s[4], math.nan) for _ in range(20)] for s in sides]
    turned = [torch.empty_like(s[4]) for s in sides]
    pos = torch.arange(72, device="cuda", dtype=torch.int32)
    main.synchronize()
    for r in range(20):
        for (_, _, pool, items, q, rope), out, t in zip(sides, outs, turned):
            rope.apply(q, pos, t)
            pool.attn(0, items, t, out[r])
    for (stream, c, pool, items, q, rope), out, t in zip(sides, outs, turned):
        stream.synchronize()
        want, mag, qk, top = attn64(pool, items, t)
        bound = attn_bound(pool.fmt, want, mag, qk, top)
        for o in out:
            assert ((o.double() - want).abs() <= bound).all()
        pool.close()
        c.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,rot,layout", [((64, 64, 256), 6, "half"), ((64, 1, 256), 256, "interleaved"), ((64, 64, 64), 64, "half")])
def test_most_heads(ctx, fmt, heads, rot, layout):
    """The most KV heads and the most query heads of one, from rows at odd addresses."""
    hq, hkv, dim = heads
    pool, ids, g = scattered(ctx, fmt, [0, 130], 64, 90, heads=heads)
    rope = kv.Rope(ctx, rot, layout=layout)
    f, m = rope.freqs()
    k, v = (randn(g, 5, hkv * dim + 1)[:, 1:].unflatten(1, (hkv, dim)) for _ in range(2))
    pool.write(0, [(ids[0], 0, 0, 2), (ids[1], 0, 130, 3)], k, v, rope)
    pos = torch.tensor([0, 1, 130, 131, 132], device="cuda", dtype=torch.int32)
    want, bound = rotate64(k, pos, f, m, layout), rope_bound(k, rot, m, pool.fmt.torch_dtype, layout)
    for s, at in ((ids[0], slice(0, 2)), (ids[1], slice(2, 5))):
        gk, gv = rows_of(pool, s)
        n = at.stop - at.start
        assert ((gk[-n:].double() - want[at]).abs() <= bound[at]).all() and torch.equal(gv[-n:], v[at].to(gv.dtype))
    q = randn(g, 6, hq, dim, dtype=pool.fmt.torch_dtype)
    check_attn(pool, [(ids[0], 0, 1, 1), (ids[1], 0, 128, 5)], q)
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,front", [((16, 2, 256), 0.0), ((16, 2, 256), 2.0**-9), ((16, 2, 256), 2.0**9), ((32, 4, 128), 2.0**9), ((6, 2, 64), 1.0)])
@pytest.mark.parametrize("news", [(1, 2, 3), (70, 1, 33)])
def test_magnitudes_that_jump(ctx, fmt, heads, front, news):
    """Rows whose size changes from one stretch of keys to the next, the first 64 dims of another size than the rest: scales that are kept,
    left and found again, with few rows and with many."""
    hq, hkv, dim = heads
    lens = [500, 64, 333]
    pool, ids, g = scattered(ctx, fmt, lens, 16, 101, heads=heads)
    sizes = [1.0, 2.0**-8, 2.0**-8, 2.0**4, 0.0, 1.0] if fmt == F16 else [1.0, 2.0**-40, 2.0**-12, 2.0**6, 0.0, 2.0**-100, 1.0]
    for t, most in zip(pool.buffer_tensors(0), (1.0, 2.0**5 if fmt == F16 else 2.0**60)):
        for i, n in zip(ids, lens):
            pages = torch.from_numpy(pool.pages(i).astype(np.int64)).cuda()
            at = torch.arange(len(pages) * 16, device="cuda")
            size = torch.tensor(sizes, device="cuda")[(at // 83) % len(sizes)] * most
            rows = torch.randn(len(pages) * 16, hkv, dim, device="cuda", generator=g) * size[:, None, None]
            rows[..., :64] *= front
            t[pages] = rows.to(t.dtype).view(len(pages), 16, hkv, dim)
    q = randn(g, sum(news), hq, dim, dtype=pool.fmt.torch_dtype) * 2.0**-6
    items = [(i, 0, n - m, m) for i, n, m in zip(ids, lens, news)]
    got = run_attn(pool, items, q)
    want, mag, qk, top = attn64(pool, items, q)
    # The largest f16 rows are infinite: what the formula makes of those has to come out as well, or NaN in place of an infinity: scores are
    # hundreds apart here, a weight below 2^-149 (e^-104) is zero in 32 bits, and zero times an infinity is NaN.
    same = (got == want) | (got.isnan() & ~want.isfinite())
    assert (((got.double() - want).abs() <= attn_bound(fmt, want, mag, qk, top)) | same).all()
    pool.close()


@pytest.mark.parametrize("heads", [(6, 2, 64), (12, 4, 128), (6, 2, 256)])
def test_values_that_are_not_finite_on_both_sides_of_a_whole_tile(ctx, heads):
    """An item of three tiles of 128 keys: a window's lower edge, a tile that every token sees, the diagonal, with a V row that is not finite in
    both partly seen tiles. What the first one noted must not meet what the third one notes; many items at one time, several calls."""
    pos, ntok, window = 128 * 3 + 40, 42, 250        # keys 175 .. 465 in tiles 1, 2, 3; all tokens see 216 .. 424
    low, high = 178, 444                             # seen by tokens 0 .. 3, and by 20 ..
    n = 150
    pool, ids, g = scattered(ctx, F16, [pos + ntok] * n, 32, 7, heads=heads, spare=0)
    q = randn(g, n * ntok, heads[0], heads[2], dtype=torch.float16)
    items = [(i, 0, pos, ntok) for i in ids]
    k, v = pool.buffer_tensors(0)
    at = torch.from_numpy(np.array([pool.pages(i)[[low // 32, high // 32]] for i in ids], np.int64)).cuda()
    v[at[:, 0], low % 32], v[at[:, 1], high % 32] = 0.5, 0.5
    want, mag, qk, top = attn64(pool, items, q, window=window)
    bound = attn_bound(F16, want, mag, qk, top)
    v[at[:, 0], low % 32, :, 3], v[at[:, 1], high % 32, :, 5] = math.nan, math.inf
    bad = torch.zeros(n, ntok, heads[0], heads[2], device="cuda", dtype=torch.bool)
    bad[:, :4, :, 3] = True
    bad[:, 20:, :, 5] = True
    bad = bad.view_as(q)
    for _ in range(5):
        got = run_attn(pool, items, q, window=window)
        assert torch.equal(~torch.isfinite(got), bad)
        assert ((got.double() - want).abs() <= bound)[~bad].all()
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("length", [30, 5000])
def test_sinks_that_are_not_finite(ctx, fmt, length):
    """In an item that is whole and in one that is split: a sink of infinity (and one that is infinite in base-2 exponents) leaves nothing of the
    keys, one of NaN makes its head's rows NaN, those of minus infinity and of the lowest value are none."""
    pool, ids, g = scattered(ctx, fmt, [length], 64, 13)
    q = randn(g, 1, 16, 256, dtype=pool.fmt.torch_dtype)
    items = [(ids[0], 0, length - 1, 1)]
    sinks = torch.zeros(16, device="cuda")
    sinks[:5] = torch.tensor([math.inf, 3e38, math.nan, -math.inf, torch.finfo(torch.float32).min])
    got = run_attn(pool, items, q, sinks=sinks)
    assert (got[:, :2] == 0).all() and got[:, 2].isnan().all()
    plain = sinks.clone()
    plain[:3], plain[3:5] = 0.0, -1e4  # (as good as none, and finite in the formula)
    want, mag, qk, top = attn64(pool, items, q, sinks=plain)
    assert ((got.double() - want).abs() <= attn_bound(fmt, want, mag, qk, top))[:, 3:].all()
    pool.close()


@pytest.mark.parametrize("heads,n,times", [((8, 1, 64), 65536, 1), ((16, 2, 256), 65536, 1), ((8, 1, 64), 16384, 200), ((16, 2, 256), 16384, 100)])
@pytest.mark.parametrize("below", [12.0, 17.4, 19.0])
def test_a_key_above_a_long_flat_tail(ctx, heads, n, times, below):
    """One key, and all others `below` nats under it with values of one sign: what the tail adds up to comes out, in split and in whole items. Its
    weights are all rounded alike: by 2^-11 of themselves, or half a step of what f16 holds below 2^-14, 2^-25, of weights that are at least 2^7 times those
    against the row's largest; the output by 2^-11 once more."""
    pool, ids, g = scattered(ctx, F16, [n], 64, 3, heads=heads)
    k, v = pool.buffer_tensors(0)
    pages = torch.from_numpy(pool.pages(ids[0]).astype(np.int64)).cuda()
    k[pages], v[pages] = 0.0, 1.0
    k[pages[0], 0], v[pages[0], 0] = below / heads[2], 0.0
    q = torch.ones(1, heads[0], heads[2], device="cuda", dtype=torch.float16)
    items = [(ids[0], 0, n - 1, 1)] * times
    got = run_attn(pool, items, q.expand(len(items), -1, -1).contiguous(), scale=1.0)
    want, mag, qk, top = attn64(pool, items[:1], q, scale=1.0)
    off = (got.double() - want).abs()
    bound = want * (2.0**-10 + 2 * qk * 2.0**-20 + 2.0**-18) + n * 2.0**-32 + 2.0**-25
    assert (off <= bound).all(), f"{float(got.min())} to {float(got.max())} for {float(want.min())}"
    pool.close()


@pytest.mark.parametrize("heads", [(16, 2, 256), (12, 4, 128), (8, 1, 64)])
@pytest.mark.parametrize("value", [1.0, -0.0078125])
def test_equal_values_come_out_as_they_are(ctx, heads, value):
    """A mean of equal values is that value whatever the weights: the sums run over the weights as the products take them. (Both are f32 sums of
    the same f16 numbers, off by 2^-15 at most here, and the nearest other output is 2^-11 away.) Few keys, many, split rows, windows."""
    n = 3001
    pool, ids, g = scattered(ctx, F16, [n, 700], 64, 4, heads=heads)
    pool.buffer_tensors(0)[1].fill_(value)
    q = randn(g, 102, heads[0], heads[2], dtype=torch.float16)
    for scale in (0.3, 0.06, 1.0):
        for first, window in ((0, 0), (n - 100, 0), (n - 3, 0), (0, 130), (0, 3)):
            got = run_attn(pool, [(ids[0], first, n - 2, 2), (ids[1], max(first - n + 700, 0), 600, 100)], q, scale=scale, window=window)
            assert ((got == value) | ((got == 0).all(-1, keepdim=True))).all()
            assert (got[1] == value).all() and (got[-1] == value).all()
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads", [(16, 2, 256), (12, 4, 128), (4, 4, 64)])
@pytest.mark.parametrize("size", [2.0**7, 2.0**13, 2.0**15])
def test_scores_of_very_long_rows(ctx, fmt, heads, size):
    """Queries and keys of +size and -size: products and sums are exact, different scores are at least 2^10 apart, so a row is the mean of the
    values whose keys tie for its maximum (their weights are equal), rounded once, however large the scores are."""
    lens, news = [5, 700, 9000], [5, 40, 2]
    pool, ids, g = scattered(ctx, fmt, lens, 64, 17, heads=heads)
    k = pool.buffer_tensors(0)[0]
    k.copy_(k.sign() * size + (k == 0) * size)
    q = ((randn(g, sum(news), heads[0], heads[2]) > 0).float() * 2 - 1).mul_(size).to(k.dtype)
    items = [(i, 0, n - m, m) for i, n, m in zip(ids, lens, news)]
    for window in (0, 300):
        got = run_attn(pool, items, q, window=window)
        want, mag, *_ = attn64(pool, items, q, window=window)
        assert ((got.double() - want).abs() <= mag * 2.0**-18 + want.abs() * 2.0**-11 + 2.0**-25).all()
    pool.close()


@pytest.mark.parametrize("heads,n,ntok", [((64, 1, 64), 300000, 300), ((16, 2, 256), 200000, 600)])
def test_values_of_one_sign_over_a_long_history(ctx, heads, n, ntok):
    """Sums over hundreds of thousands of keys do not drift. The tensor core's sums truncate; a step of 16 keys loses up to 2^-23 of the
    sum in the end (an ulp of the present sum, twice, which is half the last one on average), 2^-15 + 2^-16 over the 384 steps that it adds up before
    they are put aside. What else an output is off by is a rounding each of weights, sums and output, which has no direction."""
    pool, ids, g = scattered(ctx, F16, [n], 256, 6, heads=heads, spare=0)
    v = pool.buffer_tensors(0)[1]
    v.uniform_(0.5, 1.5, generator=g)
    v.mul_(torch.linspace(1.0, 1.9, heads[2], device="cuda").half())
    q = randn(g, ntok, heads[0], heads[2], dtype=torch.float16)
    got = run_attn(pool, [(ids[0], 0, n - ntok, ntok)], q)
    last = 8192 // (heads[0] * heads[2])
    want = attn64(pool, [(ids[0], 0, n - last, last)], q[-last:])[0]
    drift = float(((got[-last:].double() - want) / want).mean())
    assert abs(drift) <= 2.0**-15 + 2.0**-16, drift
    pool.close()


@pytest.mark.parametrize("heads", [(16, 2, 256), (12, 4, 128), (4, 4, 64)])
@pytest.mark.parametrize("keys", ["flat", "rising", "falling", "jumping"])
def test_histories_of_many_tiles(ctx, heads, keys):
    """Segments of 130 to 500 tiles, whole and cut, with references that stay, rise tile by tile, fall behind or jump late; windows, sinks, values
    that are not finite in the last, partly seen tile, with which a new sum of outputs starts (144 and 192 whole tiles in front)."""
    hq, hkv, dim = heads
    ntok = min(16, 128 // (hq // hkv))
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for tiles, times in ((144, sms // hkv), (192, sms // hkv), (300, 5 + 2 * sms // hkv)):
        n = 128 * tiles + 100
        pool, ids, g = scattered(ctx, F16, [n], 128, tiles, heads=heads, spare=0)
        k, v = pool.buffer_tensors(0)
        pages = torch.from_numpy(pool.pages(ids[0]).astype(np.int64)).cuda()
        ramp = torch.linspace(0, 30, len(pages) * 128, device="cuda")
        along = {"flat": 0 * ramp, "rising": ramp, "falling": 30 - ramp, "jumping": torch.where(ramp > 29.9, 25.0, 0.0) + torch.where(ramp > 20, 9.0, 0.0)}[keys]
        k[pages, :, :, 0] = along.view(len(pages), 128, 1).half()
        q = randn(g, ntok, hq, dim, dtype=torch.float16)
        q[..., 0] = dim**0.5 if keys != "flat" else 0.5
        many = q.repeat(times, 1, 1)
        sinks = randn(g, hq)
        for window, first, s in ((0, 0, None), (n - 900, 0, sinks), (0, 5000, sinks)):
            items = [(ids[0], first, n - ntok, ntok)]
            got = run_attn(pool, items * times, many, window=window, sinks=s).view(times, ntok, hq, dim)
            want, mag, qk, top = attn64(pool, items, q, window=window, sinks=s)
            assert ((got.double() - want).abs() <= attn_bound(F16, want, mag, qk, top)).all(), (tiles, window, first)
        at = (int(pages[-1]), 100 - ntok + 3)  # the row of token 3
        items = [(ids[0], 0, n - ntok, ntok)]
        clean = run_attn(pool, items * times, many).view(times, ntok, hq, dim)
        want, mag, qk, top = attn64(pool, items, q)  # (the other dims and tokens stay as they are)
        v[at][:, 1], v[at][:, 2] = math.nan, math.inf
        got = run_attn(pool, items * times, many).view(times, ntok, hq, dim)
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[:, 3:, :, 1:3] = True
        assert torch.equal(~torch.isfinite(got), bad)
        assert torch.equal(got[:, :3], clean[:, :3])
        bound = attn_bound(F16, want, mag, qk, top) + 2.0**-11 * mag  # (that key's weight and the row's sum have roundings of their own)
        assert ((got.double() - want).abs() <= bound)[~bad].all()
        pool.close()


class failing_launches:
    """Launches on the stream return an error: the driver refuses a call that may not be captured and with it all that follows in that capture. Nothing
    reaches the GPU meanwhile."""

    def __init__(self, stream):
        self.cu, self.stream = C.CDLL("libcuda.so.1"), C.c_void_p(stream.cuda_stream)

    def __enter__(self):
        assert self.cu.cuStreamBeginCapture_v2(self.stream, 2) == 0  # 2: relaxed
        assert self.cu.cuStreamSynchronize(self.stream) == 900       # unsupported in a capture, which is invalid from now on

    def __exit__(self, *_):
        graph = C.c_void_p()
        assert self.cu.cuStreamEndCapture(self.stream, C.byref(graph)) == 901 and not graph


@pytest.mark.parametrize("fmt", FMTS)
def test_writes_and_forks_that_do_not_reach_the_device(ctx, fmt):
    """After an error of a launch the rows that it should have written are not there, forks are not made, and the call can be repeated."""
    stream = torch.cuda.Stream()
    c2 = kv.KvContext(0, stream)
    with torch.cuda.stream(stream):
        page = 16
        pool, ids, g = scattered(c2, fmt, [40, 20, 33], page, 19, layers=2, spare=30, longest=400)
        a, b, c = ids
        d = pool.fork(b)[0]
        dt = pool.fmt.torch_dtype
        k, v, q = randn(g, 50, 2, 256), randn(g, 50, 2, 256), randn(g, 50, 16, 256, dtype=dt)
        out = torch.empty_like(q)
        before = {s: [[t.clone() for t in rows_of(pool, s, l)] for l in range(2)] for s in (a, b, c, d)}
        free = pool.free_pages
        stream.synchronize()

        def fails(call, *args, **kw):
            with failing_launches(stream), pytest.raises(_lib.MkvError) as e:
                call(*args, **kw)
            assert e.value.status == _lib.ERR_CUDA

        def refused(items):
            with pytest.raises(_lib.MkvError) as e:
                pool.attn(1, items, q[:1], out[:1])
            assert e.value.status == _lib.ERR_STATE

        fails(pool.write, 1, [(a, 0, 40, 3)], k[:3], v[:3])                       # rows on a page that is there
        refused([(a, 0, 40, 1)])
        assert pool.length(a) == 40 and pool.free_pages == free
        fails(pool.write, 1, [(a, 0, 40, 30), (b, 0, 20, 4), (c, 0, 10, 2)], k[:36], v[:36])  # new pages, a copied page, rows in front of the end
        for s, n in ((a, 40), (b, 20), (c, 10)):
            refused([(s, 0, n, 1)])
            assert pool.length(s) == (12 if s == c else n)
        assert pool.free_pages == free + 2 - 1  # (c gave two pages back, b has one of its own now)
        for copy in (False, True):
            pool.set_len(a, 40)  # (what the failed call left for the device gets there)
            fails(pool.fork, a, 40, 3, copy)
            assert pool.free_pages == free + 1
        assert pool.create() == d + 1
        pool.free([d + 1])
        items = [(a, 0, 40, 30), (b, 0, 20, 4), (c, 0, 10, 2)]
        pool.write(1, items, k[:36], v[:36])
        pool.attn(1, items, q[:36], out[:36])
        want, mag, qk, top = attn64(pool, items, q[:36], layer=1)
        assert ((out[:36].double() - want).abs() <= attn_bound(fmt, want, mag, qk, top)).all()
        for (s, _, p, n), at in zip(items, (0, 30, 34)):
            for l in range(2):
                for got, old, new in zip(rows_of(pool, s, l), before[s][l], (k, v)):
                    assert torch.equal(got[:p], old[:p])
                    if l == 1:
                        assert torch.equal(got[p:], new[at:at + n].to(dt))
        for l in range(2):
            for got, old in zip(rows_of(pool, d, l), before[d][l]):
                assert torch.equal(got, old)
        stream.synchronize()
        pool.close()
    c2.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_tables_that_change_right_in_front_of_the_attention(ctx, fmt):
    """Tables of 2 entries, sixteen sequences in 128 bytes, copied from one another and read by the next launch, over and over: every row is the
    value of the pages that its sequence has now."""
    hq, hkv, dim, n = 4, 4, 64, 60
    pool = kv.KvPool(ctx, fmt, 1, 200, 16, n + 4, 32, hq, hkv, dim)
    k, v = pool.buffer_tensors(0)
    k.zero_()
    v.copy_(torch.arange(200, device="cuda").view(200, 1, 1, 1).expand_as(v))
    parents = [pool.create() for _ in range(4)]
    for p in parents:
        pool.set_len(p, 16)
    q = torch.ones(n, hq, dim, device="cuda", dtype=pool.fmt.torch_dtype)
    outs, wants = [], []
    for r in range(100):
        kids = [c for p in (parents[r % 4:] + parents[:r % 4]) for c in pool.fork(p, n=n // 4)]
        out = torch.full_like(q, math.nan)
        pool.attn(0, [(c, 0, 15, 1) for c in kids], q, out)
        outs.append(out)
        wants.append([float(pool.pages(c)[0]) for c in kids])
        pool.free(kids[::-1] if r % 3 else kids)
        if r % 5 == 0:  # the parents' pages change as well
            pool.free(parents)
            hold = pool.create()
            pool.set_len(hold, 16 + r % 17)
            parents = [pool.create() for _ in range(4)]
            for p in parents[::-1]:
                pool.set_len(p, 16)
            pool.free([hold])
    for out, want in zip(outs, wants):
        assert (out == torch.tensor(want, device="cuda")[:, None, None]).all()
    pool.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("runs", [0, 1])
def test_pages_that_change_in_a_capture(ctx, fmt, runs):
    """Pages are taken, shared, copied and moved in a capture whose graph then runs or is dropped; its writes are made again without a capture. Every
    sequence has the rows of a twin pool that did the same without captures, by the books and by the device's tables. A second capture before any
    other call is refused."""
    stream = torch.cuda.Stream()
    c2 = kv.KvContext(0, stream)
    dt = kv.KvFormat(fmt).torch_dtype
    with torch.cuda.stream(stream):
        (pool, ids, g), (twin, twin_ids, _) = (scattered(c2, fmt, [64, 48, 40, 64, 100], 16, 23, spare=30, longest=400) for _ in range(2))
        assert ids == twin_ids
        a, b, c, e, h = ids
        x = [randn(g, 9, 2, 256) for _ in range(2)]
        for p in (pool, twin):
            assert p.fork(c) == [5]  # (shares c's last page)

        def rows(p, s, pos, n, at):
            p.write(0, [(s, 0, pos, n)], x[0][at:at + n], x[1][at:at + n])

        def change(p, n):
            """In two parts, so that what the second one finds depends on the first."""
            if n == 0:
                p.write(0, [(a, 0, 64, 2), (b, 0, 48, 1), (5, 0, 40, 3)], x[0][:6], x[1][:6])  # two new pages, one copied
                rows(p, c, 37, 2, 1)                       # over rows that were copied just now
                kids = [*p.fork(a, 64), *p.fork(e), *p.fork(b, copy=True)]
                p.truncate(e, 48)
                rows(p, e, 48, 2, 3)                       # a new page in place of a shared one; the child keeps that
                rows(p, kids[0], 64, 1, 5)
            else:
                p.free([h])
                assert p.compact() > 0                     # pages that were copied to move on, others take their numbers
                more = p.create()
                rows(p, more, 0, 9, 0)

        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for n in range(2):
                change(pool, n)
        for n in range(2):
            change(twin, n)
        if runs:
            graph.replay()
        else:
            second, q = torch.cuda.CUDAGraph(), torch.zeros(1, 16, 256, device="cuda", dtype=dt)
            stream.synchronize()
            with torch.cuda.graph(second, stream=stream):
                free = pool.free_pages
                for call in (lambda: rows(pool, a, 66, 1, 0), lambda: pool.fork(a), lambda: pool.attn(0, [(a, 0, 0, 1)], q, q + 1), lambda: pool.compact()):
                    with pytest.raises(_lib.MkvError) as err:
                        call()
                    assert err.value.status == _lib.ERR_STATE
                assert pool.free_pages == free and pool.length(a) == 66
            stream.synchronize()
            del graph, second
        pool.compact()
        for p in (pool, twin):  # the writes of the capture once more
            p.write(0, [(a, 0, 64, 2), (b, 0, 48, 1), (5, 0, 40, 3)], x[0][:6], x[1][:6])
            p.write(0, [(c, 0, 37, 2)], x[0][1:3], x[1][1:3])
            rows(p, e, 48, 2, 3)
            rows(p, 6, 64, 1, 5)
            rows(p, 8, 48, 1, 2)  # (copied from b behind its write)
            rows(p, h, 0, 9, 0)  # (the number of the one that was freed)
        for s in range(9):
            n = pool.length(s)
            assert n == twin.length(s) and n > 0 and np.array_equal(pool.pages(s), twin.pages(s))
            for got, want in zip(rows_of(pool, s), rows_of(twin, s)):
                assert torch.equal(got, want), s
            # by the device's tables: attention to one key gives its value (f32: of two parts, 2^-23 of it, of sums of them, and 2^-33 of its tile's largest)
            seen, value = torch.empty(n, 16, 256, device="cuda", dtype=dt), rows_of(pool, s)[1].double()
            pool.attn(0, [(s, i, i, 1) for i in range(n)], torch.zeros_like(seen), seen)
            assert ((seen.view(n, 2, 8, 256)[:, :, 0].double() - value).abs() <= value.abs() * 2.0**-20 + 8 * 2.0**-33).all(), s
        stream.synchronize()
        third = torch.cuda.CUDAGraph()  # (all that was recorded is done: another capture may change pages)
        with torch.cuda.graph(third, stream=stream):
            rows(pool, c, 39, 9, 0)
        third.replay()
        third.replay()
        assert torch.equal(rows_of(pool, c)[0][39:], x[0].to(dt)) and torch.equal(rows_of(pool, 5)[0], rows_of(twin, 5)[0])
        stream.synchronize()
        if runs:
            del graph
        del third
        pool.close()
        twin.close()
    c2.close()

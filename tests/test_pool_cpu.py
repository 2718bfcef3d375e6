"""The pool's bookkeeping and the argument checks of the paged operators, without a device: pages, forks, copy on write, compaction
against a plain model; every refusal leaves the books as they were."""
import ctypes as C
import math
import random

import numpy as np
import pytest
import torch

from mechta_b200 import _lib, kv


def pool(n_pages=40, page=16, seqs=6, longest=400, layers=2, **kw):
    return kv.KvPool(None, kv.KvFormat.F16, layers, n_pages, page, seqs, longest, **kw)


def status(call, *a, **kw):
    with pytest.raises(_lib.MkvError) as e:
        call(*a, **kw)
    return e.value.status


class Model:
    """The header's rules in a few lines."""

    def __init__(self, n_pages, page, seqs, longest):
        self.n, self.page, self.max_seqs, self.longest = n_pages, page, seqs, longest
        self.seqs = {}  # id -> (length, pages)

    def used(self):
        return {p for _, t in self.seqs.values() for p in t}

    def take(self, k):
        free = sorted(set(range(self.n)) - self.used())
        return None if k > len(free) else free[:k]

    def name(self, k):
        free = [i for i in range(self.max_seqs) if i not in self.seqs]
        return None if k > len(free) else free[:k]

    def compact(self):
        used = sorted(self.used())
        high = [p for p in used if p >= len(used)]
        low = [p for p in range(len(used)) if p not in used]
        to = dict(zip(high, low))
        self.seqs = {i: (n, [to.get(p, p) for p in t]) for i, (n, t) in self.seqs.items()}
        return len(high)


def check(p, m):
    assert p.free_pages == m.n - len(m.used())
    for i in range(m.max_seqs):
        n, t = m.seqs.get(i, (0, None))
        assert p.length(i) == n
        if t is not None:
            assert p.pages(i).tolist() == t


@pytest.mark.parametrize("seed", range(12))
def test_books_follow_the_model(seed):
    rng = random.Random(seed)
    page = rng.choice([16, 32, 64])
    m = Model(rng.randint(5, 150), page, rng.randint(1, 70), page * rng.randint(1, 12) + rng.randint(0, 15))
    p = pool(m.n, page, m.max_seqs, m.longest)
    refused = 0
    for _ in range(400):
        op = rng.choice(["create", "fork", "fork", "free", "truncate", "set_len", "set_len", "compact"])
        live = sorted(m.seqs)
        if op == "create":
            k = m.name(1)
            if k is None:
                assert status(p.create) == _lib.ERR_NOMEM
                refused += 1
            else:
                assert p.create() == k[0]
                m.seqs[k[0]] = (0, [])
        elif op == "compact":
            assert p.compact() == m.compact()
            used = m.used()
            assert not used or max(used) == len(used) - 1
        elif not live:
            continue
        elif op == "fork":
            s, n, copy = rng.choice(live), rng.randint(1, 3), rng.random() < 0.4
            length = rng.randint(0, m.seqs[s][0])
            want = m.seqs[s][1][: -(-length // page)]
            ids, fresh = m.name(n), m.take(n * len(want)) if copy else []
            if ids is None or fresh is None:
                assert status(p.fork, s, length, n, copy) == _lib.ERR_NOMEM
                refused += 1
            else:
                assert p.fork(s, length, n, copy) == ids
                for j, i in enumerate(ids):
                    m.seqs[i] = (length, fresh[j * len(want): (j + 1) * len(want)] if copy else list(want))
        elif op == "free":
            k = rng.sample(live, rng.randint(1, min(3, len(live))))
            p.free(k)
            for i in k:
                del m.seqs[i]
        elif op == "truncate":
            s = rng.choice(live)
            length = rng.randint(0, m.seqs[s][0])
            p.truncate(s, length)
            m.seqs[s] = (length, m.seqs[s][1][: -(-length // page)])
        else:
            s = rng.choice(live)
            length = rng.randint(m.seqs[s][0], m.longest)
            fresh = m.take(-(-length // page) - len(m.seqs[s][1]))
            if fresh is None:
                assert status(p.set_len, s, length) == _lib.ERR_NOMEM
                refused += 1
            else:
                p.set_len(s, length)
                m.seqs[s] = (length, m.seqs[s][1] + fresh)
        check(p, m)
    p.close()


def test_pool_sizes_that_are_refused():
    for kw in (dict(n_pages=0), dict(page=8), dict(page=48), dict(page=512), dict(seqs=0), dict(seqs=65537), dict(longest=0),
               dict(longest=2**30 + 1), dict(layers=0), dict(layers=257), dict(kv_heads=0), dict(kv_heads=65, q_heads=65), dict(q_heads=3),
               dict(q_heads=130, kv_heads=2), dict(head_dim=96), dict(head_dim=512), dict(n_pages=2**27), dict(q_heads=0)):
        assert status(pool, **kw) == _lib.ERR_INVALID, kw
    with pytest.raises(_lib.MkvError):
        pool(n_pages=-1)
    # tables beyond 32-bit indexes
    assert status(pool, n_pages=2**26, seqs=65536, longest=2**30) == _lib.ERR_INVALID


def test_sequences_that_are_refused():
    p = pool()
    a = p.create()
    p.set_len(a, 100)
    before = p.pages(a).tolist()
    assert status(p.free, [a, a]) == _lib.ERR_INVALID       # the same one twice
    assert status(p.free, [a, 5]) == _lib.ERR_INVALID       # one that does not live: none is freed
    assert status(p.free, [77]) == _lib.ERR_INVALID
    assert status(p.set_len, a, 99) == _lib.ERR_STATE
    assert status(p.set_len, a, 401) == _lib.ERR_CAPACITY
    assert status(p.set_len, 3, 1) == _lib.ERR_INVALID
    assert status(p.truncate, a, 101) == _lib.ERR_STATE
    assert status(p.fork, a, 101) == _lib.ERR_STATE
    assert status(p.fork, a, 100, 6) == _lib.ERR_NOMEM      # five numbers are left
    assert status(p.fork, a, 100, 5, True) == _lib.ERR_NOMEM  # 35 pages, 33 are left
    assert status(p.fork, 4, 0) == _lib.ERR_INVALID
    assert status(p.pages, 4) == _lib.ERR_INVALID
    assert p.length(a) == 100 and p.pages(a).tolist() == before and p.free_pages == 33
    p.free([])
    p.free([a])
    assert p.free_pages == 40 and p.length(a) == 0
    assert status(p.buffers, 0) == _lib.ERR_UNSUPPORTED
    p.close()


def test_writes_and_attention_that_are_refused():
    p = pool()
    a, b = p.create(), p.create()
    p.set_len(a, 30)
    U, I, S, C_, N = _lib.ERR_UNSUPPORTED, _lib.ERR_INVALID, _lib.ERR_STATE, _lib.ERR_CAPACITY, _lib.ERR_NOMEM

    def rows(n, heads=2, dim=256, dtype=torch.float32):
        return torch.zeros(n, heads, dim, dtype=dtype)

    def write(items, n, layer=0, **kw):
        return status(p.write, layer, items, kw.get("k", rows(n)), kw.get("v", rows(n)), kw.get("rope"))

    assert write([(a, 0, 30, 4)], 4) == U                    # nothing wrong but the missing device
    assert write([], 0) == U
    assert write([(a, 0, 30, 0), (b, 0, 0, 3)], 3) == U
    assert write([(a, 0, 31, 4)], 4) == S                    # a gap
    assert write([(b, 0, 1, 1)], 1) == S
    assert write([(a, 0, 30, 2), (a, 0, 32, 2)], 4) == I     # one sequence twice
    assert write([(3, 0, 0, 1)], 1) == I
    assert write([(a, 0, 30, 371)], 371) == C_
    assert write([(a, 0, 2**32 - 1, 4)], 4) == C_
    assert write([(a, 0, 30, 4)], 4, layer=2) == I
    assert write([(a, 0, 30, 4)], 4, layer=-1) == I
    assert write([(a, 0, 30, 4)], 3) == I                    # fewer rows than the items have
    assert write([(a, 0, 30, 4)], 4, k=rows(4, dim=128), v=rows(4, dim=128)) == I
    assert write([(a, 0, 30, 4)], 4, v=rows(4, dtype=torch.float16)) == I
    assert write([(a, 0, 30, 4)], 4, k=rows(4).double(), v=rows(4).double()) == I
    assert write([(a, 0, 30, 4)], 4, k=rows(1).expand(4, 2, 256)) == I
    assert write([(a, 0, 30, 4)], 4, k=torch.zeros(4, 2, 512)[:, :, ::2]) == I
    small = pool(n_pages=3)
    c = small.create()
    assert status(small.write, 0, [(c, 0, 0, 49)], rows(49), rows(49)) == N
    half = pool(head_dim=64)
    d = half.create()
    assert status(half.write, 0, [(d, 0, 0, 1)], rows(1, dim=64), rows(1, dim=64), kv.Rope(None, 66)) == I
    assert status(half.write, 0, [(d, 0, 0, 1)], rows(1, dim=64), rows(1, dim=64), kv.Rope(None, 64)) == U

    def attn(items, n, layer=0, **kw):
        q, o = kw.pop("q", None), kw.pop("out", None)
        q = rows(n, 16, dtype=torch.float16) if q is None else q
        return status(p.attn, layer, items, q, torch.empty_like(q) if o is None else o, **kw)

    assert attn([(a, 0, 26, 4)], 4) == U
    assert attn([(a, 0, 26, 4), (a, 3, 0, 30), (b, 0, 0, 0)], 34) == U  # the same sequence twice is fine here
    assert attn([(a, 0, 27, 4)], 4) == S
    assert attn([(b, 0, 0, 1)], 1) == S
    assert attn([(a, 0, 2**32 - 1, 2)], 2) == S
    assert attn([(5, 0, 0, 1)], 1) == I
    assert attn([(a, 0, 26, 4)], 4, layer=2) == I
    assert attn([(a, 0, 26, 4)], 4, q=rows(4, 16)) == I                 # not the pool's type
    assert attn([(a, 0, 26, 4)], 4, q=rows(4, 8, dtype=torch.float16)) == I
    assert attn([(a, 0, 26, 4)], 4, scale=-1.0) == I
    assert attn([(a, 0, 26, 4)], 4, scale=math.inf) == I
    assert attn([(a, 0, 26, 4)], 4, scale=math.nan) == I
    assert attn([(a, 0, 26, 4)], 4, window=-1) == I
    assert attn([(a, 0, 26, 4)], 4, sinks=torch.zeros(2)) == I
    assert attn([(a, 0, 26, 4)], 4, sinks=torch.zeros(16).half()) == I
    assert attn([(a, 0, 26, 4)], 4, q=torch.zeros(4, 16 * 256 + 3, dtype=torch.float16)[:, :-3].view(4, 16, 256)) == I  # stride of 8,198 bytes
    assert attn([(a, 0, 26, 1)], 1, q=torch.zeros(4104, dtype=torch.float16)[1:4097].view(1, 16, 256)) == I              # address
    with pytest.raises((_lib.MkvError, OverflowError)):
        p.attn(0, [(a, 0, -1, 1)], rows(1, 16, dtype=torch.float16), rows(1, 16, dtype=torch.float16))
    assert p.length(a) == 30 and p.length(b) == 0 and p.free_pages == 38


def test_fork_of_the_layers_rows():
    """Rows that set_len declared count for all layers; truncation and forks take their share."""
    p = pool()
    a = p.create()
    p.set_len(a, 40)
    b = p.fork(a, 33)[0]
    q = torch.zeros(1, 16, 256, dtype=torch.float16)
    assert status(p.attn, 1, [(b, 0, 32, 1)], q, q.clone()) == _lib.ERR_UNSUPPORTED
    assert status(p.attn, 1, [(b, 0, 33, 1)], q, q.clone()) == _lib.ERR_STATE
    p.truncate(a, 0)
    assert status(p.attn, 1, [(a, 0, 0, 1)], q, q.clone()) == _lib.ERR_STATE
    assert p.pages(b).tolist() == [0, 1, 2] and p.free_pages == 37
    p.close()


# ---- rotary positions ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dims", [2, 30, 64, 128, 256])
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_frequencies(dims, scaling):
    s, base, original = (1.0 if scaling == "none" else 8.0), 1e6, 8192.0
    f, m = kv.Rope(None, dims, base, scaling=scaling, factor=s, original=original).freqs()
    i = np.arange(dims // 2)
    b = base * s ** (dims / (dims - 2)) if scaling == "ntk" and dims > 2 else base
    want = b ** (-2.0 * i / dims)
    if scaling == "linear":
        want = want / s
    if scaling == "yarn":
        turns = original * want / (2 * np.pi)
        want = np.where(turns >= 32, want, np.where(turns <= 1, want / s, want * ((turns - 1) / 31 + (32 - turns) / 31 / s)))
    np.testing.assert_allclose(f, want, rtol=1e-13)
    assert m == pytest.approx(0.1 * math.log(s) + 1 if scaling == "yarn" else 1.0, abs=1e-15)


def test_reference_frequencies():
    """The reference's own table (64 dims, base 1e7) is the same angles as far as its f32 steps go."""
    f, m = kv.Rope(None).freqs()
    t = kv.rope_table(3, 1)[0]
    assert m == 1.0
    np.testing.assert_allclose(np.cos(3 * f), t[:32], atol=2e-5)
    np.testing.assert_allclose(np.sin(3 * f), t[32:], atol=2e-5)


def test_ropes_that_are_refused():
    for kw in (dict(dims=0), dict(dims=3), dict(dims=258), dict(dims=-2), dict(base=1.0), dict(base=0.0), dict(base=math.nan), dict(base=math.inf),
               dict(layout="both"), dict(scaling="some"), dict(scaling="linear", factor=0.5), dict(scaling="ntk", factor=math.inf),
               dict(scaling="yarn", factor=2.0), dict(scaling="yarn", factor=2.0, original=-1.0),
               dict(scaling="yarn", factor=2.0, original=100.0, slow=3.0, fast=3.0), dict(scaling="yarn", factor=math.nan, original=100.0)):
        assert status(kv.Rope, None, **kw) == _lib.ERR_INVALID, kw
    L = _lib.lib()
    r = kv.Rope(None, 64)
    import ctypes as C
    x = np.zeros((4, 2, 64), np.float32)
    y = np.zeros_like(x)
    pos = np.zeros(4, np.int32)

    def apply(**kw):
        v = dict(x=x.ctypes.data, y=y.ctypes.data, xf=1, yf=1, n=4, heads=2, dim=64, xt=0, xh=0, yt=0, yh=0, pos=pos.ctypes.data, b=0) | kw
        rows = _lib.RopeRows(v["x"], v["y"], v["xf"], v["yf"], v["n"], v["heads"], v["dim"], v["xt"], v["xh"], v["yt"], v["yh"], v["pos"], v["b"])
        st = L.mkv_rope_apply(None, r._h, C.byref(rows))
        return st, L.mkv_last_error().decode()

    ok = (_lib.ERR_INVALID, "null ctx")  # nothing wrong but the missing context
    assert apply() == ok and apply(y=x.ctypes.data) == ok and apply(n=1, heads=1, xh=7) == ok
    assert apply(yt=64, yh=256) == ok  # heads outside tokens: fine as well
    for kw in (dict(x=0), dict(y=0), dict(pos=0), dict(xf=2), dict(yf=-1), dict(dim=62), dict(dim=1025), dict(heads=0), dict(heads=20000), dict(xt=-1),
               dict(yh=2**31), dict(yh=32), dict(yt=64), dict(yt=100, yh=64), dict(yt=32, yh=256), dict(x=x.ctypes.data + 2), dict(y=y.ctypes.data + 1),
               dict(y=x.ctypes.data + 16), dict(y=x.ctypes.data, yf=0), dict(y=x.ctypes.data, yt=256), dict(pos=y.ctypes.data), dict(n=2**31)):
        st, text = apply(**kw)
        assert st == _lib.ERR_INVALID and text != "null ctx", kw
    assert apply(n=0, x=0, y=0)[0] == _lib.OK
    with pytest.raises(_lib.MkvError):
        kv.Rope(None).apply(torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 64))


def test_blocks_that_overlap():
    """Slices of one buffer lie beside each other; anything else that shares bytes is refused."""
    import ctypes as C
    L = _lib.lib()
    r = kv.Rope(None, 64)
    buf = np.zeros((5, 6, 64), np.float32)  # [tokens][heads]
    pos = np.zeros(5, np.int32)

    def apply(x_head, y_head, heads, xt=384, yt=384, n=5, yf=1):
        rows = _lib.RopeRows(buf.ctypes.data + 256 * x_head, buf.ctypes.data + 256 * y_head, 1, yf, n, heads, 64, xt, 0, yt, 0, pos.ctypes.data, 0)
        assert L.mkv_rope_apply(None, r._h, C.byref(rows)) == _lib.ERR_INVALID
        return L.mkv_last_error().decode() == "null ctx"  # nothing wrong but the missing context

    assert apply(0, 0, 3) and apply(0, 3, 3) and apply(3, 0, 3) and apply(5, 0, 1) and apply(4, 2, 2, n=4) and apply(0, 0, 6)
    assert apply(8, 0, 2, n=3) and apply(9, 5, 1, n=3)            # a token further on, beside the rows
    assert not apply(0, 3, 2, yf=0)                               # (f16: the token strides in bytes differ)
    assert not apply(0, 2, 3) and not apply(2, 0, 3) and not apply(0, 6, 3, n=4) and not apply(7, 0, 2, n=3) and not apply(4, 0, 3)
    assert not apply(0, 3, 3, yt=448, n=4) and not apply(0, 3, 3, xt=192, n=3)
    p = pool()
    a = p.create()
    p.set_len(a, 30)
    wide = torch.zeros(4, 32, 256, dtype=torch.float16)

    def attn(q, out):
        return status(p.attn, 0, [(a, 0, 26, 4)], q, out)

    assert attn(wide[:, :16], wide[:, 16:]) == _lib.ERR_UNSUPPORTED and attn(wide[:, 16:], wide[:, :16]) == _lib.ERR_UNSUPPORTED
    assert attn(wide[:, :16], wide[:, :16]) == _lib.ERR_INVALID and attn(wide[:, :16], wide[:, 15:31]) == _lib.ERR_INVALID
    flat = torch.zeros(8, 16, 256, dtype=torch.float16)
    assert attn(flat[:4], flat[4:]) == _lib.ERR_UNSUPPORTED and attn(flat[:4], flat[1:5]) == _lib.ERR_INVALID
    with pytest.raises(_lib.MkvError):
        p.fork(a, n=2**31 - 1)


def test_a_closed_rope_is_not_taken_for_rotated_rows():
    p = pool()
    a = p.create()
    rope, k = kv.Rope(None, 64), torch.zeros(4, 2, 256)
    assert status(p.write, 0, [(a, 0, 0, 4)], k, k, rope) == _lib.ERR_UNSUPPORTED  # nothing wrong but the missing device
    rope.close()
    assert status(p.write, 0, [(a, 0, 0, 4)], k, k, rope) == _lib.ERR_INVALID
    assert status(rope.freqs) == _lib.ERR_INVALID
    p.close()


def test_a_closed_context_makes_no_pool():
    ctx = kv.KvContext.__new__(kv.KvContext)  # as close() leaves it
    ctx._h, ctx.device, ctx.stream = C.c_void_p(), 0, None
    assert status(kv.KvPool, ctx, kv.KvFormat.F16, 1, 4, 16, 2, 64) == _lib.ERR_INVALID


def test_numbers_beyond_32_bits_are_refused():
    """Sequences, lengths, layers, sizes and items, as Python numbers and as arrays of other types: none is cut to 32 bits or to a whole number."""
    p, I = pool(), _lib.ERR_INVALID
    a = p.create()
    p.set_len(a, 30)
    far = 2**32
    for seqs in ([far + a], [-1], (far + a,), np.array([far + a]), np.array([-far + a]), np.array([a + 0.0]), [a, far], [a + 0.5], [2**64 + a]):
        assert status(p.free, seqs) == I, seqs
    assert status(p.truncate, a, far) == I and status(p.truncate, far + a, 0) == I and status(p.truncate, a, -far) == I
    assert status(p.set_len, a, far + 40) == I and status(p.set_len, far + a, 40) == I
    assert status(p.fork, a, far + 7) == I and status(p.fork, far + a, 7) == I and status(p.fork, far + a) == I and status(p.fork, a, far + 7, 3) == I
    assert status(p.length, far + a) == I and status(p.pages, far + a) == I and status(p.buffers, far) == I
    k, q = torch.zeros(4, 2, 256), torch.zeros(4, 16, 256, dtype=torch.float16)
    good = [a, 0, 26, 4]
    for at in range(4):
        for off in (far, -far, 0.5, 2**64):
            row = list(good)
            row[at] += off
            for items in ([tuple(row)], np.array([row])):
                assert status(p.write, 0, items, k, k) == I, items
                assert status(p.attn, 0, items, q, q.clone()) == I, items
    for items in ([tuple(good)], np.array([good]), np.array([good], np.int32), np.array([good], np.uint32), np.array([good], np.uint64)):
        assert status(p.write, 0, items, k, k) == status(p.attn, 0, items, q, q.clone()) == _lib.ERR_UNSUPPORTED  # nothing wrong but the missing device
    assert status(p.write, far, [good], k, k) == I and status(p.attn, far, [good], q, q.clone()) == I
    for kw in (dict(layers=far + 2), dict(n_pages=far + 40), dict(kv_heads=far + 2), dict(q_heads=far + 16), dict(head_dim=far + 64), dict(longest=far + 400)):
        assert status(pool, **kw) == I, kw
    assert status(kv.Rope, None, far + 64) == I
    ctx = kv.KvContext.__new__(kv.KvContext)
    ctx._h, ctx.device, ctx.stream = C.c_void_p(), -1, None
    x = torch.empty(far + 5, 1, 64, device="meta")
    with pytest.raises(_lib.MkvError, match="at most 2"):
        kv.Rope(ctx, 64).apply(x, torch.empty(far + 5, dtype=torch.int32, device="meta"), x)
    assert p.length(a) == 30 and p.free_pages == 38
    p.free(np.array([a]))
    assert p.free_pages == 40
    p.close()


def test_slices_of_every_head_do_not_overlap():
    """x and y in one buffer, each a part of every head, in both orders of tokens and heads; parts that share a value are refused."""
    L = _lib.lib()
    r = kv.Rope(None, 64)
    buf = np.zeros((5, 6, 200), np.float32)
    pos = np.zeros(5, np.int32)

    def apply(x, y, dim=64, n=5, heads=6, xt=1200, yt=1200, xh=200, yh=200, yf=1):
        rows = _lib.RopeRows(buf.ctypes.data + 4 * x, buf.ctypes.data + 4 * y, 1, yf, n, heads, dim, xt, xh, yt, yh, pos.ctypes.data, 0)
        assert L.mkv_rope_apply(None, r._h, C.byref(rows)) == _lib.ERR_INVALID
        return L.mkv_last_error().decode() == "null ctx"  # nothing wrong but the missing context

    assert apply(0, 64) and apply(64, 0) and apply(0, 136) and apply(136, 0) and apply(0, 100, dim=100) and apply(0, 64, n=1)
    assert apply(0, 64, xt=200, yt=200, xh=1200, yh=1200, n=6, heads=5) and not apply(0, 63, xt=200, yt=200, xh=1200, yh=1200, n=6, heads=5)
    assert apply(0, 264, n=4) and apply(200, 64, n=4, heads=5)  # a head further on, another part of it
    assert not apply(0, 63) and not apply(63, 0) and not apply(0, 137, dim=64, n=4) and not apply(0, 100, dim=101)
    assert not apply(0, 64, yh=208, yt=1248, n=4) and not apply(0, 64, yf=0, n=2)
    assert not apply(0, 200) and not apply(0, 1200, n=4)

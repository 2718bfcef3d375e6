"""Cases of the operators on paged key/value rows, and their plain forms.

Rotary positions (`kv.Rope.apply`), rows written into the pages of many sequences (`kv.KvPool.write`), sequences forked, copied and
compacted (`kv.KvPool.fork`, `compact`, `free`) and the attention of new tokens over the pages (`kv.KvPool.attn`). With `own` false
`run()` computes them from their formulas with elementary torch operations; with `own` true it makes the calls that a host program
makes. `listed()` names the cases, `draw()` gives others from the same ranges, `exact()` gives the same results in 64 bits.
"""
from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

HALF, INTERLEAVED = "half", "interleaved"


def listed():
    return [
        # One short chat, decoded token by token: the smallest attention call, where latency counts.
        {"name": "decode_one", "kind": "attn", "fmt": "f16", "heads": 16, "kv_heads": 2, "dim": 256, "page": 64, "seqs": 1, "shortest": 4096,
         "longest": 4096, "least": 1, "most": 1, "window": 0, "sinks": False},
        # A server's decode step: 32 sessions of ragged lengths with one to four tokens each (drafts), small pages.
        {"name": "decode_32", "kind": "attn", "fmt": "f16", "heads": 16, "kv_heads": 2, "dim": 256, "page": 16, "seqs": 32, "shortest": 1001,
         "longest": 65536, "least": 1, "most": 4, "window": 0, "sinks": False},
        # A block of 2,048 new tokens over a 32,768-token prefix.
        {"name": "chunk_2k", "kind": "attn", "fmt": "f16", "heads": 16, "kv_heads": 2, "dim": 256, "page": 128, "seqs": 1, "shortest": 32768,
         "longest": 32768, "least": 2048, "most": 2048, "window": 0, "sinks": False},
        # Sliding-window layers with sinks, 32 heads of 128: follow-up messages of ragged sizes beside sessions that decode.
        {"name": "mixed_window", "kind": "attn", "fmt": "f16", "heads": 32, "kv_heads": 4, "dim": 128, "page": 32, "seqs": 12, "shortest": 77,
         "longest": 8100, "least": 1, "most": 389, "window": 513, "sinks": True},
        # Hosts that keep full precision: the decode step of a few sessions on f32 pages.
        {"name": "decode_f32", "kind": "attn", "fmt": "f32", "heads": 16, "kv_heads": 2, "dim": 256, "page": 64, "seqs": 8, "shortest": 500,
         "longest": 32000, "least": 1, "most": 3, "window": 0, "sinks": False},
        # A block on f32 pages.
        {"name": "chunk_f32", "kind": "attn", "fmt": "f32", "heads": 16, "kv_heads": 2, "dim": 256, "page": 16, "seqs": 2, "shortest": 1777,
         "longest": 4096, "least": 300, "most": 512, "window": 0, "sinks": False},
        # The queries of a 4-token verify step: 64 of 256 dims, read out of the rows that hold query and gate side by side.
        {"name": "rope_step", "kind": "rope", "src": "f32", "dst": "f16", "heads": 16, "dim": 256, "rot": 64, "layout": HALF, "scaling": "none",
         "factor": 1.0, "tokens": 4, "far": 65536, "gated": True, "backward": False},
        # Gradients of a long block's rotated heads, interleaved pairs, positions far beyond the original context.
        {"name": "rope_far_8k", "kind": "rope", "src": "f32", "dst": "f32", "heads": 32, "dim": 128, "rot": 128, "layout": INTERLEAVED,
         "scaling": "yarn", "factor": 16.0, "tokens": 8192, "far": 1000000, "gated": False, "backward": True},
        # The new rows of 32 sessions' verify steps: one launch however the pages lie.
        {"name": "write_32", "kind": "write", "fmt": "f16", "kv_heads": 2, "dim": 256, "page": 16, "seqs": 32, "shortest": 500, "longest": 4099,
         "least": 4, "most": 4, "rot": 64, "layout": HALF, "scaling": "none", "factor": 1.0},
        # The rows of three prefill blocks on f32 pages, positions scaled.
        {"name": "write_blocks", "kind": "write", "fmt": "f32", "kv_heads": 4, "dim": 128, "page": 64, "seqs": 3, "shortest": 0, "longest": 9001,
         "least": 1025, "most": 4096, "rot": 128, "layout": INTERLEAVED, "scaling": "ntk", "factor": 4.0},
        # 16 samples drawn from one prompt that ends inside a page: each gets its own last page when its first row is written.
        {"name": "fork_16", "kind": "fork", "fmt": "f16", "layers": 10, "kv_heads": 2, "dim": 256, "page": 64, "length": 9001, "forks": 16},
        # A session copied behind one that ends; then the pages in use are moved together.
        {"name": "compact", "kind": "compact", "fmt": "f16", "layers": 10, "kv_heads": 2, "dim": 256, "page": 64, "length": 30011},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _geometry(rng):
    return rng.choice([(16, 2, 256), (16, 2, 256), (32, 4, 128), (8, 8, 64), (12, 4, 128), (6, 1, 256), (20, 2, 64)])


def draw(rng):
    kind = rng.choice(["decode", "decode", "chunks", "chunks", "long", "rope", "rope", "write", "fork", "compact"])
    heads, kv_heads, dim = _geometry(rng)
    fmt = rng.choice(["f16", "f16", "f32"])
    page = rng.choice([16, 32, 64, 128])
    layout, scaling = rng.choice([HALF, INTERLEAVED]), rng.choice(["none", "linear", "ntk", "yarn"])
    factor = 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0])
    rot = 2 * rng.randint(4, dim // 2)
    if kind in ("decode", "chunks", "long"):
        case = {"kind": "attn", "fmt": fmt, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}
        if kind == "decode":
            shortest = _log(rng, 1, 4096)
            case |= {"seqs": _log(rng, 1, 32), "shortest": shortest, "longest": _log(rng, shortest, 32768), "least": 1, "most": rng.randint(1, 4)}
        elif kind == "chunks":
            shortest = _log(rng, 1, 1000) - 1
            case |= {"seqs": rng.randint(2, 8), "shortest": shortest, "longest": shortest + _log(rng, 1, 6000), "least": rng.randint(0, 40),
                     "most": _log(rng, 41, 400)}
        else:
            n = _log(rng, 0 + 1, 16384)
            t = _log(rng, 50, 1024)
            case |= {"seqs": 1, "shortest": n, "longest": n, "least": t, "most": t}
        return case | {"window": rng.choice([0, 0, _log(rng, 1, 4096)]), "sinks": rng.random() < 0.3}
    if kind == "rope":
        return {"kind": "rope", "src": rng.choice(["f32", "f16"]), "dst": rng.choice(["f32", "f16"]), "heads": heads, "dim": dim, "rot": rot,
                "layout": layout, "scaling": scaling, "factor": factor, "tokens": _log(rng, 1, 4096), "far": _log(rng, 1000, 1000000),
                "gated": rng.random() < 0.4, "backward": rng.random() < 0.4}
    if kind == "write":
        n, shortest = rng.randint(1, 32), rng.randint(0, 500)
        least = _log(rng, 1, 8)
        return {"kind": "write", "fmt": fmt, "kv_heads": kv_heads, "dim": dim, "page": page, "seqs": n, "shortest": shortest,
                "longest": shortest + _log(rng, 1, 4000), "least": least, "most": least + _log(rng, 1, 3000 // n + 1) - 1, "rot": rot,
                "layout": layout, "scaling": scaling, "factor": factor}
    case = {"kind": kind, "fmt": fmt, "layers": rng.randint(1, 10), "kv_heads": kv_heads, "dim": dim, "page": page, "length": _log(rng, 100, 16000)}
    return case | ({"forks": rng.randint(1, 32)} if kind == "fork" else {})


# ---- what a case's sizes are --------------------------------------------------------------------------------------

def _spread(lo, hi, n, stride):
    """n whole numbers from lo to hi, in a mixed order."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * stride + 1) % n) // (n - 1) for i in range(n)]


def _sequences(case):
    """(history, new tokens) of each sequence."""
    n = case["seqs"]
    return list(zip(_spread(case["shortest"], case["longest"], n, 1), _spread(case["least"], case["most"], n, 7 if n % 7 else 5)))


def _pages_of(tokens, page):
    return -(-tokens // page)


ROUNDS = 8  # the sequences grow in turn, so that their pages lie among one another's


def _tables(lens, page):
    """Each sequence's pages, as the pool hands them out: always the lowest free one."""
    tables, at = [[] for _ in lens], 0
    for r in range(1, ROUNDS + 1):
        for t, n in zip(tables, lens):
            while len(t) < _pages_of(n * r // ROUNDS, page):
                t.append(at)
                at += 1
    return tables, at


def _dtype(fmt):
    return torch.float16 if fmt == "f16" else torch.float32


def _frequencies(case):
    """Radians per position of each pair (64 bits), and the factor on cosine and sine."""
    rot, base, s, original = case["rot"], 1e7, case["factor"], 32768
    scaling = case["scaling"]
    if scaling == "ntk" and rot > 2:
        base = base * s ** (rot / (rot - 2))
    f = base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        return f / s, 1.0
    if scaling == "yarn":
        turns = original * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f / s * (1 - keep) + f * keep, 0.1 * math.log(s) + 1.0
    return f, 1.0


class _State:
    pass


@functools.lru_cache(maxsize=None)
def _context(device, stream):
    """A host program has one context for all its pools on a device and stream (which the context keeps, so that its handle stays its own)."""
    from mechta_b200 import kv
    return kv.KvContext(device, torch.cuda.current_stream())


def _rope(s, case):
    from mechta_b200 import kv
    return kv.Rope(s.ctx, case["rot"], base=1e7, layout=case["layout"], scaling=case["scaling"], factor=case["factor"], original=32768)


def _make_pool(s, case, g, layers, pages, seqs, longest, heads):
    """K and V pages of every layer, filled with N(0,1): the pool's own memory, or plain tensors of the same shape."""
    if own:
        from mechta_b200 import kv
        s.pool = kv.KvPool(s.ctx, kv.KvFormat.F16 if case["fmt"] == "f16" else kv.KvFormat.F32, layers, pages, case["page"], seqs, longest,
                           q_heads=heads, kv_heads=case["kv_heads"], head_dim=case["dim"])
        s.k, s.v = zip(*[s.pool.buffer_tensors(l) for l in range(layers)])
    else:
        shape = (pages, case["page"], case["kv_heads"], case["dim"])
        s.k, s.v = ([torch.empty(shape, device="cuda", dtype=_dtype(case["fmt"])) for _ in range(layers)] for _ in range(2))
    for t in (*s.k, *s.v):
        t.normal_(generator=g)


def _grow(s, lens, tables):
    """The sequences in the pool, grown in turn as _tables has it."""
    ids = [s.pool.create() for _ in lens]
    for r in range(1, ROUNDS + 1):
        for i, n in zip(ids, lens):
            s.pool.set_len(i, n * r // ROUNDS)
    assert all(s.pool.pages(i).tolist() == t for i, t in zip(ids, tables))
    return ids


def prepare(case, seed):
    s = _State()
    s.case, s.kind = case, case["kind"]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if own:
        s.ctx = _context(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    if s.kind == "rope":
        n, heads, dim = case["tokens"], case["heads"], case["dim"]
        x = normal(n, heads, 2 * dim if case["gated"] else dim).to(_dtype(case["src"]))
        s.x = x[:, :, :dim]
        s.positions = torch.randint(0, case["far"], (n,), device="cuda", generator=g, dtype=torch.int32)
        s.out = torch.empty(n, heads, dim, device="cuda", dtype=_dtype(case["dst"]))
        if own:
            s.rope = _rope(s, case)
        else:
            f, s.m = _frequencies(case)
            s.f = f.cuda()
    elif s.kind in ("attn", "write"):
        page, seqs = case["page"], _sequences(case)
        after = [h + n for h, n in seqs]
        lens = after if s.kind == "attn" else [h for h, _ in seqs]
        tables, used = _tables(lens, page)
        if s.kind == "write":  # the pages that the new rows take
            for t, n in zip(tables, after):
                while len(t) < _pages_of(n, page):
                    t.append(used)
                    used += 1
        _make_pool(s, case, g, 1, used + 3, len(seqs), max(max(after), 1), case.get("heads", case["kv_heads"]))
        total = sum(n for _, n in seqs)
        if s.kind == "attn":
            s.q = normal(total, case["heads"], case["dim"]).to(_dtype(case["fmt"]))
            s.out = torch.empty_like(s.q)
            s.sink = 2.0 * normal(case["heads"]) if case["sinks"] else None
        else:
            s.nk, s.nv = normal(total, case["kv_heads"], case["dim"]), normal(total, case["kv_heads"], case["dim"])
        if own:
            if s.kind == "write":
                s.rope = _rope(s, case)
            ids = _grow(s, lens, [t[:_pages_of(n, page)] for t, n in zip(tables, lens)])
            s.items = np.array([(i, 0, h, n) for i, (h, n) in zip(ids, seqs)], np.uint32)
        else:
            width = max(len(t) for t in tables)
            s.table = torch.tensor([t + [0] * (width - len(t)) for t in tables], device="cuda").reshape(len(seqs), width)
            s.before = torch.tensor([h for h, _ in seqs], device="cuda")
            s.new = torch.tensor([n for _, n in seqs], device="cuda")
            s.owner = torch.repeat_interleave(torch.arange(len(seqs), device="cuda"), s.new)  # packed row -> its sequence and token
            s.token = torch.arange(total, device="cuda") - (s.new.cumsum(0) - s.new)[s.owner]
            s.most = max(n for _, n in seqs)
            s.span = max(after)
            if s.kind == "write":
                f, s.m = _frequencies(case)
                s.f = f.cuda()
    else:
        page, n, layers = case["page"], case["length"], case["layers"]
        whole, m = _pages_of(n, page), _pages_of(n, page)
        forks = case.get("forks", 0)
        _make_pool(s, case, g, layers, whole + forks if s.kind == "fork" else 3 * whole, 3 + forks, n + 1 + page, case["kv_heads"])
        s.whole, s.part = m, n % page
        if s.kind == "fork":
            s.nk, s.nv = normal(forks, case["kv_heads"], case["dim"]), normal(forks, case["kv_heads"], case["dim"])
        if own:
            s.seq = s.pool.create()
            s.pool.set_len(s.seq, n)
            if s.kind == "fork":
                s.items = np.array([(0, 0, n, 1)] * forks, np.uint32)
        elif s.kind == "fork":
            s.dst = torch.arange(m, m + forks, device="cuda")
    torch.cuda.synchronize()
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def _rotated(x, positions, f, m, layout, rot, backward=False):
    """x [n][heads][dim], 32 bits: the first `rot` dims rotated by position * f, angles in 64 bits."""
    a = positions.double()[:, None] * f
    c, sn = (m * torch.cos(a)).float()[:, None], (m * torch.sin(a)).float()[:, None]
    if backward:
        sn = -sn
    r = x[..., :rot]
    u, w = (r[..., 0::2], r[..., 1::2]) if layout == INTERLEAVED else (r[..., : rot // 2], r[..., rot // 2:])
    p, q = u * c - w * sn, u * sn + w * c
    r = torch.stack((p, q), -1).flatten(-2) if layout == INTERLEAVED else torch.cat((p, q), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _plain_attn(s):
    case = s.case
    n_seq, kvh, dim, group = len(s.new), case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    q = torch.zeros(n_seq, s.most, kvh, group, dim, device="cuda")
    q[s.owner, s.token] = s.q.float().view(-1, kvh, group, dim)
    k = s.k[0][s.table].flatten(1, 2)[:, : s.span].float()
    v = s.v[0][s.table].flatten(1, 2)[:, : s.span].float()
    score = torch.einsum("bthgd,bkhd->bhgtk", q, k) / math.sqrt(dim)
    at = (s.before[:, None] + torch.arange(s.most, device="cuda"))[:, :, None]  # [sequence][token][1]: the token's position
    key = torch.arange(s.span, device="cuda")
    seen = key <= at
    if case["window"]:
        seen &= key > at - case["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s.sink is not None:
        top = torch.maximum(top, s.sink.view(1, kvh, group, 1, 1))
    score = torch.exp(score.sub_(top))
    total = score.sum(-1, keepdim=True)
    if s.sink is not None:
        total = total + torch.exp(s.sink.view(1, kvh, group, 1, 1) - top)
    o = torch.einsum("bhgtk,bkhd->bthgd", score, v) / total.permute(0, 3, 1, 2, 4)
    return o[s.owner, s.token].reshape(s.q.shape).to(s.q.dtype)


def run(s):
    case = s.case
    if s.kind == "rope":
        if own:
            s.rope.apply(s.x, s.positions, s.out, backward=case["backward"])
            return s.out
        return _rotated(s.x.float(), s.positions, s.f, s.m, case["layout"], case["rot"], case["backward"]).to(s.out.dtype)
    if s.kind == "attn":
        if own:
            s.pool.attn(0, s.items, s.q, s.out, window=case["window"], sinks=s.sink)
            return s.out
        return _plain_attn(s)
    if s.kind == "write":
        if own:
            s.pool.write(0, s.items, s.nk, s.nv, s.rope)
        else:
            at = s.before[s.owner] + s.token
            pages, rows = s.table[s.owner, at // case["page"]], at % case["page"]
            s.k[0][pages, rows] = _rotated(s.nk, at, s.f, s.m, case["layout"], case["rot"]).to(s.k[0].dtype)
            s.v[0][pages, rows] = s.nv.to(s.v[0].dtype)
        return [*s.k, *s.v]
    if s.kind == "fork":
        if own:
            kids = s.pool.fork(s.seq, n=case["forks"])
            s.items[:, 0] = kids
            s.pool.write(0, s.items, s.nk, s.nv)
            s.pool.free(kids)
        else:
            for t in (*s.k, *s.v):
                t[s.dst, : s.part] = t[s.whole - 1, : s.part]
            s.k[0][s.dst, s.part], s.v[0][s.dst, s.part] = s.nk.to(s.k[0].dtype), s.nv.to(s.v[0].dtype)
        return [*s.k, *s.v]
    m = s.whole
    if own:
        hold = s.pool.create()
        s.pool.set_len(hold, m * case["page"])  # a session's pages, which the copy lies behind
        twin = s.pool.fork(s.seq, copy=True)
        s.pool.free([hold])
        s.pool.compact()
        s.pool.free(twin)
    else:
        for t in (*s.k, *s.v):
            t[2 * m: 3 * m - 1] = t[: m - 1]
            last = s.part or case["page"]
            t[3 * m - 1, :last] = t[m - 1, :last]
            t[m: 2 * m] = t[2 * m:]
    return [*s.k, *s.v]


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    size = {"f16": 2, "f32": 4}
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": n * (size[case["src"]] + size[case["dst"]]) + 4 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    elem = size[case["fmt"]]
    row = 2 * case["kv_heads"] * case["dim"]  # K and V elements of one position
    if case["kind"] == "write":
        n = sum(n for _, n in _sequences(case))
        return {"bytes": n * row * (4 + elem), "flops": 3 * n * case["kv_heads"] * case["rot"]}
    if case["kind"] == "attn":
        rows = pairs = tokens = 0
        w = case["window"]
        for h, n in _sequences(case):
            if n:
                rows += h + n - (max(0, h + 1 - w) if w else 0)
                pairs += sum(min(h + t + 1, w) if w else h + t + 1 for t in range(n))
                tokens += n
        return {"bytes": rows * row * elem + 2 * tokens * case["heads"] * case["dim"] * elem, "flops": 4 * case["heads"] * case["dim"] * pairs}
    if case["kind"] == "fork":
        part = case["length"] % case["page"]
        return {"bytes": case["forks"] * row * (case["layers"] * part * 2 * elem + 4 + elem), "flops": 0}
    whole = _pages_of(case["length"], case["page"]) * case["page"]
    return {"bytes": case["layers"] * row * elem * 2 * (case["length"] + whole), "flops": 0}


# ---- the same in 64 bits ------------------------------------------------------------------------------------------

def _rotate64(x, positions, case, sign=1.0):
    """Each pair as a complex number, turned."""
    rot, s = case["rot"], case["factor"]
    i = np.arange(rot // 2, dtype=np.float64)
    base = 1e7 * (s ** (rot / (rot - 2)) if case["scaling"] == "ntk" and rot > 2 else 1.0)
    f, m = np.exp(-2.0 * i / rot * np.log(base)), 1.0
    if case["scaling"] == "linear":
        f = f / s
    elif case["scaling"] == "yarn":
        share = np.minimum(1.0, np.maximum(0.0, (32768 * f / (2 * np.pi) - 1.0) / 31.0))
        f, m = f * (share + (1.0 - share) / s), 1.0 + 0.1 * np.log(s)
    turn = torch.polar(torch.full((), m, dtype=torch.float64, device="cuda").expand(len(positions), rot // 2).contiguous(),
                       sign * positions.double()[:, None] * torch.from_numpy(f).cuda())
    y = x.double().clone()
    if case["layout"] == INTERLEAVED:
        z = torch.complex(y[..., 0:rot:2], y[..., 1:rot:2]) * turn[:, None]
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    else:
        z = torch.complex(y[..., : rot // 2], y[..., rot // 2: rot]) * turn[:, None]
        y[..., : rot // 2], y[..., rot // 2: rot] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "rope":
        return _rotate64(s.x, s.positions, case, -1.0 if case["backward"] else 1.0)
    page = case["page"]
    if s.kind == "attn":
        group, out, at = case["heads"] // case["kv_heads"], [], 0
        for i, (h, n) in enumerate(_sequences(case)):
            if n == 0:
                continue
            length = h + n
            pages = s.table[i, : _pages_of(length, page)]
            k = s.k[0][pages].reshape(-1, case["kv_heads"], case["dim"])[:length].double()
            v = s.v[0][pages].reshape(-1, case["kv_heads"], case["dim"])[:length].double()
            q = s.q[at: at + n].double()
            at += n
            delta = torch.arange(h, length, device="cuda")[:, None] - torch.arange(length, device="cuda")[None]
            hidden = (delta < 0) | (delta >= case["window"] if case["window"] else torch.zeros_like(delta, dtype=torch.bool))
            heads = []
            for j in range(case["heads"]):
                a = (q[:, j] @ k[:, j // group].T) * case["dim"] ** -0.5
                a[hidden] = -math.inf
                if s.sink is not None:
                    a = torch.cat((a, s.sink[j].double().expand(n, 1)), 1)
                heads.append(torch.softmax(a, 1)[:, :length] @ v[:, j // group])
            out.append(torch.stack(heads, 1))
        return torch.cat(out)
    k, v = [t.double() for t in s.k], [t.double() for t in s.v]
    if s.kind == "write":
        at = 0
        for i, (h, n) in enumerate(_sequences(case)):
            p = torch.arange(h, h + n, device="cuda")
            where = (s.table[i][p // page], p % page)
            k[0][where] = _rotate64(s.nk[at: at + n], p, case)
            v[0][where] = s.nv[at: at + n].double()
            at += n
        return [*k, *v]
    for t in (*k, *v):
        if s.kind == "fork":
            for j in range(case["forks"]):
                t[s.whole + j, : s.part] = t[s.whole - 1, : s.part]
        else:
            flat, n = t.view(3, s.whole * page, -1), case["length"]
            flat[2, :n] = flat[0, :n]
            flat[1] = flat[2]
    if s.kind == "fork":
        k[0][s.whole:, s.part], v[0][s.whole:, s.part] = s.nk.double(), s.nv.double()
    return [*k, *v]

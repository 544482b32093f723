"""page_plan, rope_pages, attention_pages and logits_pick on a B200 against plain numpy in 64 bits:
single tokens and long runs, odd sizes, pages that end inside a tile, spare rows left as they were,
not-a-numbers in what no row reads, words that point outside reported by the error word, and a step of
all four together, captured into a CUDA graph and replayed on another stream."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SPARE = 0xFFFFFFFF
HALF_STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # the most a rounding to the type moves a value


def put(pkg, ctx, a):
    a = np.ascontiguousarray(a)
    m = pkg.Memory(ctx, max(16, a.nbytes))
    if a.nbytes:
        m.write(a)
    return m


def typed(syn, a, dtype):
    """Values as the type stores them: (the stored array, its values in 64 bits)."""
    a = np.asarray(a, np.float32)
    if dtype == "f32":
        return a, a.astype(np.float64)
    bits = syn.bf16_bits(a)
    return bits, syn.bf16_to_f32(bits).astype(np.float64)


def read(syn, m, dtype, shape):
    n = int(np.prod(shape))
    if dtype == "f32":
        return m.read(np.float32, n).reshape(shape).astype(np.float64)
    return syn.bf16_to_f32(m.read(np.uint16, n)).reshape(shape).astype(np.float64)


def run(pkg, ctx, kernel, p, mems):
    pkg.dispatch_once(ctx, kernel, p, [(m, 0, m.nbytes) for m in mems])


# ---- page_plan ------------------------------------------------------------------------------------------


def plan_oracle(held, fresh, free, table, rows, page, pages, first):
    """The plan as its definition says it, request by request."""
    table, seqs = table.copy(), len(held)
    at, place = np.full(2 * rows, SPARE, np.uint32), np.full(rows, SPARE, np.uint32)
    starts, nxt = np.zeros(seqs + 1, np.uint32), held.copy()
    taken = placed = served = 0
    stop, bad = False, False
    for s in range(seqs):
        starts[s] = placed
        h, f = int(held[s]), int(fresh[s])
        old, new = -(-h // page), -(-(h + f) // page)
        stop = stop or (taken + new - old > len(free) or placed + f > rows or new > table.shape[1] or first + h + f >= SPARE)
        if stop:
            continue
        table[s, old:new] = free[taken:taken + new - old]
        for i in range(f):
            at[placed + i], at[rows + placed + i] = first + h + i, s
            to = int(table[s, (h + i) // page])
            if to < pages:
                place[placed + i] = to * page + (h + i) % page
            else:
                bad = True
        nxt[s], taken, placed, served = h + f, taken + new - old, placed + f, served + 1
    starts[seqs] = placed
    wanted = sum(-(-(int(h) + int(f)) // page) - -(-int(h) // page) for h, f in zip(held, fresh))
    return dict(table=table, at=at, place=place, starts=starts, next=nxt,
                counts=np.array([taken, placed, served, min(wanted, SPARE)], np.uint32)), bad


def plan_case(seqs, page, held_to, fresh_to, seed, spare_pages=3, width=None):
    rng = np.random.default_rng(seed)
    held = rng.integers(0, held_to + 1, seqs).astype(np.uint32)
    fresh = rng.integers(0, fresh_to + 1, seqs).astype(np.uint32)
    fresh[0] = max(fresh[0], 1)
    held[::5] = held[::5] // page * page  # at a page's end
    old = -(-held.astype(np.int64) // page)
    new = -(-(held.astype(np.int64) + fresh) // page)
    width = int(max(new.max(), 1)) if width is None else width
    perm = rng.permutation(int(old.sum() + (new - old).sum()) + spare_pages).astype(np.uint32)
    table = np.full((seqs, max(width, int(old.max()))), 0xABCDEF01, np.uint32)
    at = 0
    for s in range(seqs):
        table[s, :old[s]] = perm[at:at + old[s]]
        at += old[s]
    return held, fresh, perm[at:], table, len(perm)


def plan_run(pkg, ctx, held, fresh, free, table, rows, page, pages, first):
    seqs = len(held)
    p = pkg.TgParams(seqs=seqs, rows=rows, stride=table.shape[1], n=len(free), capacity=page, slots=pages, first=first)
    out = dict(table=put(pkg, ctx, table))
    for name, n in (("at", 2 * rows), ("place", rows), ("starts", seqs + 1), ("next", seqs), ("counts", 4)):
        out[name] = put(pkg, ctx, np.full(n, 0x77777777, np.uint32))
    sizes = dict(table=table.size, at=2 * rows, place=rows, starts=seqs + 1, next=seqs, counts=4)
    try:
        run(pkg, ctx, "page_plan", p, [put(pkg, ctx, held), put(pkg, ctx, fresh), put(pkg, ctx, free), *out.values()])
        bad = False
    except pkg.KernelError:
        bad = True
    return {n: m.read(np.uint32, sizes[n]) for n, m in out.items()}, bad


@pytest.mark.parametrize("seqs,page,held_to,fresh_to,slack", [
    (1, 16, 0, 1, 0), (1, 32, 100, 1, 5), (7, 48, 300, 1, 0), (33, 16, 50, 70, 9), (600, 128, 900, 3, 0),
    (3000, 32, 200, 5, 1000), (16384, 16, 40, 1, 7)])
def test_page_plan(pkg, ctx, seqs, page, held_to, fresh_to, slack):
    held, fresh, free, table, pages = plan_case(seqs, page, held_to, fresh_to, seed=seqs + page)
    rows, first = int(fresh.sum()) + slack, 1000 + page
    want, bad = plan_oracle(held, fresh, free, table, rows, page, pages, first)
    got, got_bad = plan_run(pkg, ctx, held, fresh, free, table, rows, page, pages, first)
    for name in want:
        assert np.array_equal(got[name], want[name].reshape(-1)), name
    assert not bad and not got_bad and want["counts"][2] == seqs


@pytest.mark.parametrize("what", ["pages", "rows", "width", "positions", "none", "empty", "no pages"])
def test_page_plan_serves_up_to_the_first_that_does_not_fit(pkg, ctx, what):
    held, fresh, free, table, pages = plan_case(50, 16, 60, 40, seed=3)
    rows, first = int(fresh.sum()), 7
    if what == "pages":
        free = free[:len(free) // 2]
    elif what == "rows":
        rows = rows * 2 // 3
    elif what == "width":
        held[20] = table.shape[1] * 16 - 1
        fresh[20] = 2
    elif what == "positions":
        first = SPARE - 64
    elif what == "none":
        held[0], fresh[0] = 0xFFFFFFF0, 0xFFFFFFF0
    elif what == "empty":
        fresh[:] = 0
    elif what == "no pages":
        free = free[:0]
    want, _ = plan_oracle(held, fresh, free, table, rows, 16, pages, first)
    got, bad = plan_run(pkg, ctx, held, fresh, free, table, rows, 16, pages, first)
    for name in want:
        assert np.array_equal(got[name], want[name].reshape(-1)), name
    assert not bad
    assert (want["counts"][2] < 50) == (what != "empty")


def test_page_plan_reports_pages_past_the_cache(pkg, ctx):
    held, fresh, free, table, pages = plan_case(20, 32, 100, 9, seed=5)
    free[1] = pages + 7
    table[4, int(held[4]) // 32] = SPARE
    held[4] |= 1  # its last page is not full
    fresh[4] = 3
    rows = int(fresh.sum())
    want, bad = plan_oracle(held, fresh, free, table, rows, 32, pages, 0)
    got, got_bad = plan_run(pkg, ctx, held, fresh, free, table, rows, 32, pages, 0)
    assert bad and got_bad
    for name in want:
        assert np.array_equal(got[name], want[name].reshape(-1)), name


# ---- rope_pages -------------------------------------------------------------------------------------------


def rope_case(syn, rows, heads, kv, hd, rot, page, positions, dtype, ctype, seed):
    rng = np.random.default_rng(seed)
    pages = -(-rows // page) + 2
    c, c64 = typed(syn, rng.standard_normal((rows, heads + 2 * kv, hd)), ctype)
    angle = rng.uniform(-4, 4, (positions, max(1, rot // 2)))
    cos, sin = np.cos(angle).astype(np.float32), (0.9 * np.sin(angle)).astype(np.float32)
    at = np.concatenate([rng.integers(0, positions, rows), np.zeros(rows)]).astype(np.uint32)
    place = rng.permutation(pages * page)[:rows].astype(np.uint32)
    old, old64 = typed(syn, rng.standard_normal((pages, kv, page, hd)), dtype)
    return pages, c, c64, cos, sin, at, place, old, old64


def rope_oracle(c64, cos, sin, at, place, old64, rot, inter, heads, kv, page, q64):
    k, v = old64.copy(), old64.copy()
    q = q64.copy()
    half = rot // 2
    for r in range(len(place)):
        if at[r] == SPARE:
            continue
        x = c64[r].copy()
        co, si = cos[at[r], :half].astype(np.float64), sin[at[r], :half].astype(np.float64)
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, half), slice(half, rot))
        t = x[:heads + kv]
        t[:, a], t[:, b] = t[:, a] * co - t[:, b] * si, t[:, b] * co + t[:, a] * si
        q[r] = x[:heads]
        if place[r] != SPARE:
            k[place[r] // page, :, place[r] % page] = x[heads:heads + kv]
            v[place[r] // page, :, place[r] % page] = x[heads + kv:]
    return q, k, v


@pytest.mark.parametrize("rows,heads,kv,hd,rot,inter,page,dtype,ctype", [
    (1, 16, 2, 64, 64, False, 32, "bf16", "f32"), (129, 4, 1, 64, 64, True, 16, "f32", "f32"),
    (37, 16, 2, 128, 128, False, 48, "bf16", "bf16"), (300, 20, 4, 128, 96, True, 64, "bf16", "bf16"),
    (5, 8, 8, 64, 2, False, 16, "f32", "f32"), (65, 8, 8, 64, 20, True, 128, "bf16", "f32"),
    (11, 4, 1, 64, 42, False, 16, "bf16", "bf16"), (70, 16, 2, 64, 8, False, 32, "f32", "f32"),
    (19, 32, 8, 128, 0, False, 32, "bf16", "f32"), (5000, 5, 1, 64, 50, False, 16, "bf16", "f32"),
    (5000, 7, 7, 64, 30, True, 16, "f32", "f32"), (1200, 32, 8, 128, 100, True, 48, "bf16", "bf16"),
    (1200, 20, 4, 128, 102, False, 32, "bf16", "f32")])
def test_rope_pages(pkg, ctx, syn, rows, heads, kv, hd, rot, inter, page, dtype, ctype):
    pages, c, c64, cos, sin, at, place, old, old64 = rope_case(syn, rows, heads, kv, hd, rot, page, 500, dtype, ctype, rows + rot)
    if rows > 4:
        at[2] = SPARE            # writes nothing, whatever its place
        place[3] = SPARE         # writes q alone
    q0, q064 = typed(syn, np.full((rows, heads, hd), 3.25), dtype)
    p = pkg.TgParams(dtype=pkg.DTYPES[dtype], heads=heads, kv_heads=kv, head_dim=hd, rows=rows, capacity=page, slots=pages,
                     rope=int(rot > 0), k=rot, n=500 if rot else 0, flags=int(inter) | (2 if ctype == "bf16" else 0))
    q, k, v = put(pkg, ctx, q0), put(pkg, ctx, old), put(pkg, ctx, old)
    run(pkg, ctx, "rope_pages", p, [put(pkg, ctx, a) for a in (at, place, c, cos, sin)] + [q, k, v])
    want = rope_oracle(c64, cos, sin, at, place, old64, rot, inter, heads, kv, page, q064)
    for got, w in zip((read(syn, q, dtype, q0.shape), read(syn, k, dtype, old.shape), read(syn, v, dtype, old.shape)), want):
        # One product and one fused multiply-add in f32 (each at most |c| (|cos| + |sin|) < 12 off by
        # 2^-24 of it), then the rounding to the type.
        assert np.all(np.abs(got - w) <= HALF_STEP[dtype] * np.abs(w) + 2 * 12 * 2.0 ** -24)
    # What no row writes is as it was, bit for bit.
    written = np.zeros((pages * page,), bool)
    written[[t for a, t in zip(at[:rows], place) if a != SPARE and t != SPARE]] = True
    for m in (k, v):
        keep = read(syn, m, dtype, old.shape).transpose(0, 2, 1, 3).reshape(pages * page, -1)[~written]
        assert np.array_equal(keep, old64.transpose(0, 2, 1, 3).reshape(pages * page, -1)[~written])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rope_pages_is_rope_rows_over_slots(pkg, ctx, syn, dtype):
    """A cache of slots is a cache of pages: the same bits as rope_rows for a page a slot."""
    rows, cap = 50, 64
    shape = pkg.Shape(hidden=1024, inner=4096, heads=16, kv_heads=2, head_dim=64, layers=1, capacity=cap)
    rng = np.random.default_rng(1)
    at = np.concatenate([rng.integers(0, cap, rows), np.arange(rows)]).astype(np.uint32)
    cos, sin = shape.rope_tables()
    c = put(pkg, ctx, rng.standard_normal((rows, 20 * 64), dtype=np.float32))
    es = 2 if dtype == "bf16" else 4
    outs = [[pkg.Memory(ctx, n * es) for n in (rows * 1024, rows * 2 * cap * 64, rows * 2 * cap * 64)] for _ in range(2)]
    tables = [put(pkg, ctx, cos), put(pkg, ctx, sin)]
    p = pkg.params(shape, dtype, rows=rows, slots=rows)
    run(pkg, ctx, "rope_rows", p, [put(pkg, ctx, at), c, *tables, *outs[0]])
    p = pkg.params(shape, dtype, rows=rows, slots=rows, k=64, n=cap)
    place = (at[rows:] * cap + at[:rows]).astype(np.uint32)
    run(pkg, ctx, "rope_pages", p, [put(pkg, ctx, at), put(pkg, ctx, place), c, *tables, *outs[1]])
    for a, b in zip(*outs):
        assert np.array_equal(a.read(np.uint8, a.nbytes), b.read(np.uint8, b.nbytes))


@pytest.mark.parametrize("hd,rot,dtype", [(64, 64, "bf16"), (128, 96, "f32"), (64, 42, "bf16")])
def test_rope_pages_rows_with_one_place_leave_values_of_theirs(pkg, ctx, syn, hd, rot, dtype):
    """Every value at a place that several rows have is one of these rows' (of any of them: the position may be a
    mixture); the rows' queries and the other places are as ever."""
    rows, heads, kv, page = 600, 16, 2, 32
    pages, c, c64, cos, sin, at, place, old, old64 = rope_case(syn, rows, heads, kv, hd, rot, page, 50, dtype, "f32", rot)
    place[1::3] = place[0::3]
    place[500:520] = place[40]
    p = pkg.TgParams(dtype=pkg.DTYPES[dtype], heads=heads, kv_heads=kv, head_dim=hd, rows=rows, capacity=page, slots=pages, rope=1, k=rot, n=50)
    q0, q064 = typed(syn, np.zeros((rows, heads, hd)), dtype)
    q, k, v = put(pkg, ctx, q0), put(pkg, ctx, old), put(pkg, ctx, old)
    run(pkg, ctx, "rope_pages", p, [put(pkg, ctx, a) for a in (at, place, c, cos, sin)] + [q, k, v])
    got_k, got_v = (read(syn, m, dtype, old.shape) for m in (k, v))
    fits = {}
    got_q = read(syn, q, dtype, q0.shape)
    for r in range(rows):  # a row at a time, so that each of a place's rows is compared with what is there
        wq, wk, wv = rope_oracle(c64[r:r + 1], cos, sin, at[r:r + 1], place[r:r + 1], old64, rot, False, heads, kv, page, q064[r:r + 1])
        t = int(place[r])
        for n, (got, w) in enumerate(((got_k, wk), (got_v, wv))):
            g, w = got[t // page, :, t % page], w[t // page, :, t % page]
            near = np.abs(g - w) <= HALF_STEP[dtype] * np.abs(w) + 2 * 12 * 2.0 ** -24  # as test_rope_pages's
            fits[t, n] = fits.get((t, n), False) | near
        assert np.all(np.abs(got_q[r] - wq[0]) <= HALF_STEP[dtype] * np.abs(wq[0]) + 2 * 12 * 2.0 ** -24)
    assert all(f.all() for f in fits.values())
    free = np.ones(pages * page, bool)
    free[place] = False
    for got in (got_k, got_v):
        flat = lambda a: a.transpose(0, 2, 1, 3).reshape(pages * page, -1)[free]  # noqa: E731
        assert np.array_equal(flat(got), flat(old64))


def test_rope_pages_skips_words_that_point_outside(pkg, ctx, syn):
    rows, heads, kv, hd, page = 9, 4, 1, 64, 16
    pages, c, c64, cos, sin, at, place, old, old64 = rope_case(syn, rows, heads, kv, hd, hd, page, 40, "f32", "f32", 2)
    p = pkg.TgParams(dtype=0, heads=heads, kv_heads=kv, head_dim=hd, rows=rows, capacity=page, slots=pages, rope=1, k=hd, n=40)
    q0 = np.zeros((rows, heads, hd))
    at[4], place[6] = 40, pages * page
    q, k, v = put(pkg, ctx, q0.astype(np.float32)), put(pkg, ctx, old), put(pkg, ctx, old)
    with pytest.raises(pkg.KernelError):
        run(pkg, ctx, "rope_pages", p, [put(pkg, ctx, a) for a in (at, place, c, cos, sin)] + [q, k, v])
    at[4] = at[6] = SPARE  # as if they were spare
    want = rope_oracle(c64, cos, sin, at, place, old64, hd, False, heads, kv, page, q0)
    for got, w in zip((read(syn, q, "f32", q0.shape), read(syn, k, "f32", old.shape), read(syn, v, "f32", old.shape)), want):
        assert np.all(np.abs(got - w) <= 2.0 ** -24 * np.abs(w) + 2 * 12 * 2.0 ** -24)


# ---- attention_pages ----------------------------------------------------------------------------------------


class Paged:
    """A random paged batch: request s has lengths[s] own positions, row r is the last but back[r] of
    request of[r]. Every value that no row reads is not a number; every unused table entry is past
    the cache."""

    def __init__(self, syn, dtype, heads, kv, hd, page, first, lengths, of, back, seed=0, scale=1.0):
        rng = np.random.default_rng(seed)
        self.dtype, self.heads, self.kv, self.hd, self.page, self.first = dtype, heads, kv, hd, page, first
        self.rows, self.seqs = len(of), len(lengths)
        own = [-(-n // page) for n in lengths]
        shared = -(-first // page)
        self.width = max(own) + 1
        self.pages = sum(own) + shared + 3
        perm = rng.permutation(self.pages).astype(np.uint32)
        self.shared = perm[:shared]
        self.table = np.full((self.seqs, self.width), 0xDEADBEEF, np.uint32)
        k = np.full((self.pages, kv, page, hd), np.nan, np.float32)
        v = k.copy()

        def fill(ids, n):
            for j, pg in enumerate(ids):
                m = min(page, n - j * page)
                k[pg, :, :m] = rng.standard_normal((kv, m, hd))
                v[pg, :, :m] = rng.standard_normal((kv, m, hd))

        fill(self.shared, first)
        at = shared
        for s, n in enumerate(own):
            self.table[s, :n] = perm[at:at + n]
            fill(self.table[s, :n], lengths[s])
            at += n
        (self.k, self.k64), (self.v, self.v64) = typed(syn, k, dtype), typed(syn, v, dtype)
        self.q, self.q64 = typed(syn, scale * rng.standard_normal((self.rows, heads, hd)), dtype)
        self.at = np.full(2 * self.rows, SPARE, np.uint32)
        for r, s in enumerate(of):
            if s is not None:
                self.at[r], self.at[self.rows + r] = first + lengths[s] - 1 - back[r], s

    def params(self, pkg, **kw):
        return pkg.TgParams(**{**dict(dtype=pkg.DTYPES[self.dtype], heads=self.heads, kv_heads=self.kv, head_dim=self.hd,
                                      rows=self.rows, capacity=self.page, slots=self.pages, first=self.first, seqs=self.seqs,
                                      stride=self.width), **kw})

    def run(self, pkg, ctx, rows=None, **kw):
        """The outputs' bytes of the batch, or of some of its rows run alone."""
        rows = np.arange(self.rows) if rows is None else np.asarray(rows)
        p = self.params(pkg, rows=len(rows), **kw)
        at = np.concatenate([self.at[rows], self.at[self.rows + rows]])
        out = put(pkg, ctx, np.full((len(rows),) + self.q.shape[1:], 0x4141 if self.dtype == "bf16" else 7, self.q.dtype))
        work = pkg.Memory(ctx, pkg.attention_pages_work(p))
        work.fill(0x7FC07FC0)  # not a number in every type
        run(pkg, ctx, "attention_pages", p, [put(pkg, ctx, a) for a in (self.q[rows], self.k, self.v, at, self.table, self.shared)] + [work, out])
        return out

    def expect(self):
        """(outputs, how far each may be off) in 64 bits; None for a spare row."""
        out, step = [], HALF_STEP[self.dtype]
        for r in range(self.rows):
            if self.at[r] == SPARE:
                out.append(None)
                continue
            n, s = int(self.at[r]) - self.first + 1, int(self.at[self.rows + r])
            i, j = np.arange(self.first), np.arange(n)
            spot = [(self.shared[i // self.page], i % self.page), (self.table[s][j // self.page], j % self.page)]
            k, v = (np.concatenate([c[pg, :, o] for pg, o in spot]) for c in (self.k64, self.v64))  # [n][kv][hd]
            q = self.q64[r].reshape(self.kv, -1, self.hd)
            score = np.einsum("kgd,nkd->kgn", q, k) / np.sqrt(self.hd)
            size = np.einsum("kgd,nkd->kgn", np.abs(q), np.abs(k)) / np.sqrt(self.hd)
            e = np.exp(score - score.max(-1, keepdims=True))
            prob = e / e.sum(-1, keepdims=True)
            o = np.einsum("kgn,nkd->kgd", prob, v).reshape(self.heads, self.hd)
            mass = np.einsum("kgn,nkd->kgd", prob, np.abs(v)).reshape(self.heads, self.hd)
            # A score is a sum of hd products in f32 (off by at most hd 2^-24 of the products' sizes), and
            # its exponential (within 2^-21) and place in the sums of n terms (n 2^-24) follow; a
            # probability is off by twice that, numerator and sum. For bf16 each probability is rounded
            # once more (half a step), and the output to the type.
            ds = ((self.hd + 2) * 2.0 ** -24 * size.max(-1) + 2.0 ** -21 + (self.first + n) * 2.0 ** -24).reshape(self.heads, 1)
            rounded = step if self.dtype == "bf16" else 0.0
            out.append((o, (2 * ds + rounded) * mass + step * np.abs(o) * (1 + 2 * ds) + 2.0 ** -24 * np.abs(o)))
        return out

    def check(self, syn, out, rows=None):
        rows = range(self.rows) if rows is None else rows
        got = read(syn, out, self.dtype, (len(rows), self.heads, self.hd))
        left = 12.0625 if self.dtype == "bf16" else 7.0  # 0x4141 as bf16
        want = self.expect()
        for i, r in enumerate(rows):
            if want[r] is None:
                assert np.all(got[i] == left), r
            else:
                o, tol = want[r]
                far = np.abs(got[i] - o) - tol
                assert np.all(far <= 0), (r, float(far.max()))


def batch(rng, rows, top, per=1):
    """rows over requests of random lengths up to top, `per` rows a request; some rows spare."""
    seqs = -(-rows // per)
    lengths = (per - 1 + rng.integers(1, top + 1, seqs)).tolist()
    of, back = [r // per for r in range(rows)], [per - 1 - r % per for r in range(rows)]
    return lengths, of, back


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,heads,kv,hd,page,first,top,per", [
    (1, 16, 2, 64, 32, 0, 1, 1), (1, 4, 1, 64, 16, 1, 1, 1), (3, 16, 2, 64, 48, 127, 40, 1), (2, 8, 8, 64, 16, 128, 300, 1),
    (9, 16, 2, 128, 32, 129, 17, 2), (17, 20, 4, 128, 64, 1000, 500, 3), (40, 16, 2, 64, 128, 2500, 700, 1),
    (33, 32, 8, 128, 16, 640, 130, 1), (70, 4, 1, 64, 16, 4097, 65, 5), (700, 32, 8, 128, 16, 130, 40, 1),
    (300, 8, 8, 64, 32, 0, 400, 1), (1300, 16, 2, 64, 48, 40, 20, 4), (40, 8, 8, 64, 32, 3001, 20, 1),
    (5, 32, 8, 128, 16, 9000, 30, 1)])
def test_attention_pages(pkg, ctx, syn, dtype, rows, heads, kv, hd, page, first, top, per):
    rng = np.random.default_rng(rows * 7 + first)
    lengths, of, back = batch(rng, rows, top, per)
    if rows > 2:
        of[1] = None
    b = Paged(syn, dtype, heads, kv, hd, page, first, lengths, of, back, seed=rows)
    b.check(syn, b.run(pkg, ctx))


@pytest.mark.parametrize("length", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513])
def test_attention_pages_lengths_at_the_pieces_edges(pkg, ctx, syn, length):
    for hd in (64, 128):
        b = Paged(syn, "bf16", 16, 2, hd, 16, 77, [length, 3], [0, 1], [0, 0], seed=length)
        b.check(syn, b.run(pkg, ctx))


@pytest.mark.parametrize("first", [1, 63, 64, 65, 127, 128, 129, 255, 257, 384, 2047, 2048, 2049, 2176, 4095])
def test_attention_pages_prefixes_at_the_pieces_edges(pkg, ctx, syn, first):
    for hd, page in ((64, 64), (128, 48)):
        b = Paged(syn, "bf16", 16, 2, hd, page, first, [5] * 20, list(range(20)), [0] * 20, seed=first)
        b.check(syn, b.run(pkg, ctx))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_pages_with_peaked_and_growing_scores(pkg, ctx, syn, dtype):
    """Large queries (one key takes nearly all), so that the running maximum moves late and far."""
    b = Paged(syn, dtype, 16, 2, 64, 32, 1500, [300, 1, 77], [0, 1, 2, 2], [0, 0, 0, 5], seed=4, scale=30.0)
    b.check(syn, b.run(pkg, ctx))


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_attention_pages_rows_are_the_same_bits_alone(pkg, ctx, syn, dtype, hd):
    rng = np.random.default_rng(8)
    lengths, of, back = batch(rng, 90, 400)
    b = Paged(syn, dtype, 16, 2, hd, 32, 1100, lengths, of, back, seed=8)
    whole = b.run(pkg, ctx)
    whole = whole.read(np.uint8, whole.nbytes).reshape(90, -1)
    for rows in ([0], [89], [5, 44], list(range(17, 60)), list(range(89, -1, -1))):
        some = b.run(pkg, ctx, rows)
        assert np.array_equal(some.read(np.uint8, some.nbytes).reshape(len(rows), -1), whole[rows])


def test_attention_pages_reports_words_that_point_outside(pkg, ctx, syn):
    for dtype in ("bf16", "f32"):
        for what in ("position", "length", "request", "page", "shared"):
            b = Paged(syn, dtype, 16, 2, 64, 32, 300, [40, 90, 10], [0, 1, 2], [0, 0, 0], seed=9)
            if what == "position":
                b.at[1] = 299
            elif what == "length":
                b.at[1] = 300 + b.width * 32
            elif what == "request":
                b.at[3 + 1] = 3
            elif what == "page":
                b.table[1, 0] = b.pages
            else:
                b.shared = b.shared.copy()
                b.shared[2] = SPARE
            p = b.params(pkg)
            out = put(pkg, ctx, np.full(b.q.shape, 0x4141 if dtype == "bf16" else 7, b.q.dtype))
            work = pkg.Memory(ctx, pkg.attention_pages_work(p))
            mems = [put(pkg, ctx, a) for a in (b.q, b.k, b.v, b.at, b.table, b.shared)] + [work, out]
            with pytest.raises(pkg.KernelError):
                run(pkg, ctx, "attention_pages", p, mems)
            ctx.synchronize()  # the word was taken: nothing is left for the next wait
            if what in ("position", "length", "request"):
                b.at[1] = b.at[3 + 1] = SPARE  # left as a spare row is
                b.check(syn, out)
            elif what == "page":
                got = read(syn, out, dtype, b.q.shape)
                b.at[1] = SPARE  # its output is meaningless, the others' are not
                for r in (0, 2):
                    o, tol = b.expect()[r]
                    assert np.all(np.abs(got[r] - o) <= tol)


# ---- logits_pick ----------------------------------------------------------------------------------------------


def pick_oracle(x64, seen, spans, pen, ids, bias, masks, vocab):
    out, size = x64.copy(), np.zeros_like(x64)
    for r, (begin, prompt, made, b0, nb, mask) in enumerate(spans.astype(np.int64)):
        x = x64[r, :vocab].copy()
        hist = seen[begin:begin + prompt + made].astype(np.int64)
        every = np.bincount(hist[hist < vocab], minlength=vocab)
        gen = hist[prompt:]
        c = np.bincount(gen[gen < vocab], minlength=vocab)
        rep, pres, freq = pen[r].astype(np.float64)
        with np.errstate(invalid="ignore"):
            y = np.where(every > 0, np.where(x > 0, x / rep, x * rep), x)
            s = np.abs(y) + c * abs(freq) + (c > 0) * abs(pres)
            y = y - c * freq - (c > 0) * pres
        last = {int(t): float(v) for t, v in zip(ids[b0:b0 + nb], bias[b0:b0 + nb])}
        for t, v in last.items():
            if t < vocab:
                y[t] += v
                s[t] += abs(v)
        if mask != SPARE:
            bits = np.unpackbits(masks[mask].view(np.uint8), bitorder="little")[:vocab]
            y[bits == 0] = -np.inf
            s[bits == 0] = 0
        out[r, :vocab], size[r, :vocab] = y, s
    return out, size


def pick_case(syn, rows, vocab, stride, hist, biases, masks, dtype, seed):
    rng = np.random.default_rng(seed)
    x, x64 = typed(syn, 4 * rng.standard_normal((rows, stride)), dtype)
    lengths = rng.integers(0, hist + 1, rows)
    seen = (vocab * rng.random(int(lengths.sum()) + 3) ** 4).astype(np.uint32)
    seen[::17] = vocab + rng.integers(0, 2 ** 31, len(seen[::17]))  # past the vocabulary
    ids = rng.integers(0, vocab + 3, rows * biases).astype(np.uint32)
    if biases > 1:
        ids[1::biases] = ids[0::biases]  # a token listed twice
    bias = (3 * rng.standard_normal(rows * biases)).astype(np.float32)
    bits = rng.integers(0, 2 ** 32, (max(1, masks), (vocab + 31) // 32), dtype=np.uint64).astype(np.uint32)
    spans = np.zeros((rows, 6), np.uint32)
    spans[:, 0] = np.cumsum(lengths) - lengths
    spans[:, 1] = lengths // 3
    spans[:, 2] = lengths - lengths // 3
    spans[:, 3], spans[:, 4], spans[:, 5] = np.arange(rows) * biases, biases, SPARE
    if masks:
        spans[::2, 5] = rng.integers(0, masks, len(spans[::2]))
    pen = np.stack([rng.uniform(0.8, 2, rows), rng.uniform(-1, 1, rows), rng.uniform(-1, 1, rows)], 1).astype(np.float32)
    return x, x64, seen, spans, pen, ids, bias, bits


def pick_run(pkg, ctx, x, seen, spans, pen, ids, bias, bits, vocab, masks, dtype, in_place=False):
    rows, stride = x.shape
    p = pkg.TgParams(dtype=pkg.DTYPES[dtype], rows=rows, n=vocab, stride=stride, k=len(seen), k1=len(ids), m=masks)
    mx = put(pkg, ctx, x)
    out = mx if in_place else put(pkg, ctx, np.full(x.shape, 0x4141 if dtype == "bf16" else 7, x.dtype))
    pick = put(pkg, ctx, np.full(rows, 0x55555555, np.uint32))
    bad = False
    try:
        run(pkg, ctx, "logits_pick", p, [mx] + [put(pkg, ctx, a) for a in (seen, spans, pen, ids, bias, bits)] + [out, pick])
    except pkg.KernelError:
        bad = True
    return out, pick.read(np.uint32, rows), bad


def pick_check(got, pick, want, size, vocab, dtype, rows):
    for r in rows:
        g, w = got[r, :vocab], want[r, :vocab]
        fine = np.isfinite(w)
        assert np.array_equal(g[~fine], w[~fine], equal_nan=True), r
        # Four f32 roundings of values no larger than the terms' sizes, then the type's.
        assert np.all(np.abs(g[fine] - w[fine]) <= 4 * 2.0 ** -24 * size[r, :vocab][fine] + HALF_STEP[dtype] * np.abs(w[fine]) * (1 + 2.0 ** -20)), r
        best = np.where(np.isnan(g), -np.inf, g)
        assert pick[r] == (SPARE if best.max() == -np.inf else int(np.argmax(best))), r


@pytest.mark.parametrize("rows,vocab,stride,hist,biases,masks,dtype", [
    (1, 32000, 32000, 700, 20, 1, "f32"), (3, 1, 1, 5, 2, 1, "f32"), (5, 33, 36, 50, 0, 0, "bf16"), (2, 4096, 4104, 3000, 7, 3, "bf16"),
    (7, 4097, 4097, 90, 3, 2, "f32"), (130, 50001, 50003, 300, 10, 5, "bf16"), (66, 70000, 70004, 2000, 64, 4, "f32"),
    (4, 131071, 131072, 9000, 500, 2, "bf16"), (9, 999, 1000, 0, 0, 0, "f32"), (6, 12000, 12000, 400, 5, 0, "f32")])
@pytest.mark.parametrize("in_place", [False, True])
def test_logits_pick(pkg, ctx, syn, rows, vocab, stride, hist, biases, masks, dtype, in_place):
    x, x64, seen, spans, pen, ids, bias, bits = pick_case(syn, rows, vocab, stride, hist, biases, masks, dtype, rows + vocab)
    out, pick, bad = pick_run(pkg, ctx, x, seen, spans, pen, ids, bias, bits, vocab, masks, dtype, in_place)
    assert not bad
    got = read(syn, out, dtype, x.shape)
    want, size = pick_oracle(x64, seen, spans, pen, ids, bias, bits, vocab)
    pick_check(got, pick, want, size, vocab, dtype, range(rows))
    left = x64[:, vocab:] if in_place else np.full((rows, stride - vocab), 12.0625 if dtype == "bf16" else 7.0)
    assert np.array_equal(got[:, vocab:], left)


def test_logits_pick_with_values_that_are_not_finite(pkg, ctx, syn):
    x, x64, seen, spans, pen, ids, bias, bits = pick_case(syn, 6, 5000, 5000, 40, 0, 6, "f32", 1)
    x[0, 10], x[0, 11] = np.nan, np.inf
    x[1] = -np.inf
    x[2] = np.nan
    x[3] = 2.5                      # all equal: the lowest token the mask allows
    x[4, ::2] = np.nan
    spans[:, 5] = SPARE
    spans[:, 1:3] = 0
    spans[3, 5], spans[5, 5] = 3, 5
    bits[5] = 0                     # a grammar that allows nothing
    out, pick, bad = pick_run(pkg, ctx, x, seen, spans, pen, ids, bias, bits, 5000, 6, "f32")
    want, size = pick_oracle(x.astype(np.float64), seen, spans, pen, ids, bias, bits, 5000)
    with np.errstate(invalid="ignore"):
        pick_check(read(syn, out, "f32", x.shape), pick, want, size, 5000, "f32", range(6))
    assert pick[0] == 11 and pick[1] == pick[2] == pick[5] == SPARE and not bad


def test_logits_pick_leaves_rows_whose_words_point_outside(pkg, ctx, syn):
    for column, value in ((0, 10 ** 6), (1, SPARE), (2, 2 ** 31), (3, 10 ** 6), (4, SPARE), (5, 2), (5, SPARE - 1)):
        x, x64, seen, spans, pen, ids, bias, bits = pick_case(syn, 5, 9000, 9000, 40, 3, 2, "f32", 2)
        spans[3, column] = value
        out, pick, bad = pick_run(pkg, ctx, x, seen, spans, pen, ids, bias, bits, 9000, 2, "f32")
        assert bad
        got = read(syn, out, "f32", x.shape)
        assert np.all(got[3] == 7) and pick[3] == 0x55555555
        spans[3] = (0, 0, 0, 0, 0, SPARE)
        want, size = pick_oracle(x64, seen, spans, pen, ids, bias, bits, 9000)
        pick_check(got, pick, want, size, 9000, "f32", (0, 1, 2, 4))


# ---- bindings, streams, and the four together ---------------------------------------------------------------


def test_bindings_that_overlap_or_are_too_small_are_refused(pkg, ctx):
    p = pkg.TgParams(rows=4, n=64, stride=64, dtype=0)
    big = pkg.Memory(ctx, 1 << 16)
    spans = np.zeros((4, 6), np.uint32)
    spans[:, 5] = SPARE
    big.write(spans, offset=2 * 4096)
    good = [(big, i * 4096, 4096) for i in range(9)]
    pkg.dispatch_once(ctx, "logits_pick", p, good)
    pkg.dispatch_once(ctx, "logits_pick", p, good[:7] + [good[0], good[8]])          # in place
    pkg.dispatch_once(ctx, "logits_pick", p, [good[0]] + [good[7]] + good[2:])       # an empty array is any 16 bytes
    for i, b, error in ((7, (big, 16, 4096), pkg.InvalidError), (8, good[0], pkg.InvalidError), (8, good[2], pkg.InvalidError),
                        (8, (big, 7 * 4096 + 512, 64), pkg.InvalidError), (8, (big, 8 * 4096 + 4, 64), pkg.InvalidError),
                        (8, (big, 8 * 4096, 12), pkg.ShapeError), (0, (big, 0, 1023), pkg.ShapeError),
                        (2, (big, 2 * 4096, 95), pkg.ShapeError), (0, (big, 1 << 16, 4096), pkg.ShapeError)):
        bad = list(good)
        bad[i] = b
        for call in (lambda: pkg.dispatch_once(ctx, "logits_pick", p, bad), lambda: pkg.Dispatch(ctx, "logits_pick", p, bad).enqueue(ctx.stream),
                     lambda: pkg.Program(ctx, [("logits_pick", p, bad, "")])):
            with pytest.raises(error):
                call()
    with pytest.raises(pkg.InvalidError):
        pkg.Dispatch(ctx, "logits_pick", p, good[:8]).enqueue(ctx.stream)
    with pytest.raises(pkg.ShapeError):
        pkg.Dispatch(ctx, "logits_pick", pkg.TgParams(rows=4, n=64, stride=60, dtype=0), good).enqueue(ctx.stream)
    d = pkg.Dispatch(ctx, "logits_pick", p, good)
    d.enqueue(ctx.stream)
    ctx.synchronize()
    d.close()
    with pytest.raises(pkg.InvalidError):
        d.enqueue(ctx.stream)


def test_wrap_takes_device_tensors_alone(pkg, ctx):
    import torch

    t = torch.arange(64, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    m = pkg.Memory.wrap(ctx, t)
    assert m.nbytes == 256 and m.device_ptr == t.data_ptr()
    assert np.array_equal(m.read(np.int32, 64), np.arange(64))
    m.free()  # leaves the tensor
    assert int(t.sum()) == 2016
    with pytest.raises(pkg.InvalidError):
        pkg.Memory.wrap(ctx, torch.zeros(8))
    with pytest.raises(pkg.InvalidError):
        pkg.Memory.wrap(ctx, torch.zeros(8).pin_memory())
    with pytest.raises(pkg.ShapeError):
        pkg.Memory.wrap(ctx, t.view(8, 8).t())


def step_program(pkg, ctx, syn, dtype):
    """A serving step over pages: the plan, then one layer's rotary append and attention, and the choice of
    a token from logits made of the outputs. Returns the buffers, the dispatches and the host's copy."""
    rng = np.random.default_rng(12)
    heads, kv, hd, page, first, seqs, rows, width = 16, 2, 64, 32, 90, 6, 9, 5
    pages = 40
    held = np.array([0, 31, 32, 100, 7, 0], np.uint32)
    fresh = np.array([1, 2, 1, 3, 0, 1], np.uint32)
    order = rng.permutation(pages).astype(np.uint32)
    shared, order = order[:3], order[3:]
    table = np.full((seqs, width), SPARE, np.uint32)
    for s in range(seqs):
        n = -(-int(held[s]) // page)
        table[s, :n], order = order[:n], order[n:]
    k, k64 = typed(syn, rng.standard_normal((pages, kv, page, hd)), dtype)
    v, v64 = typed(syn, rng.standard_normal((pages, kv, page, hd)), dtype)
    c = rng.standard_normal((rows, heads + 2 * kv, hd)).astype(np.float32)
    angle = np.arange(400)[:, None] * 10000.0 ** (-2 * np.arange(24) / 48)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    host = dict(held=held, fresh=fresh, free=order, table=table, k=k, v=v, c=c, cos=cos, sin=sin, shared=shared)
    m = {n: put(pkg, ctx, a) for n, a in host.items()}
    es = 2 if dtype == "bf16" else 4
    for n, size in (("at", 8 * rows), ("place", 4 * rows), ("starts", 4 * seqs + 4), ("next", 4 * seqs), ("counts", 16),
                    ("q", rows * heads * hd * es), ("out", rows * heads * hd * es), ("logits", rows * heads * hd * es), ("pick", 4 * rows)):
        m[n] = pkg.Memory(ctx, size)
    spans = np.zeros((rows, 6), np.uint32)
    spans[:, 5] = SPARE
    m["spans"], m["pen"] = put(pkg, ctx, spans), put(pkg, ctx, np.ones((rows, 3), np.float32))
    base = dict(dtype=pkg.DTYPES[dtype], heads=heads, kv_heads=kv, head_dim=hd, rows=rows, capacity=page, slots=pages, first=first, seqs=seqs, stride=width)
    p = [pkg.TgParams(**{**base, "n": len(order)}), pkg.TgParams(**{**base, "rope": 1, "k": 48, "n": 400, "flags": 1}), pkg.TgParams(**base),
         pkg.TgParams(dtype=pkg.DTYPES[dtype], rows=rows, n=heads * hd, stride=heads * hd)]
    m["work"] = pkg.Memory(ctx, pkg.attention_pages_work(p[2]))
    w = lambda names: [(m[n], 0, m[n].nbytes) for n in names.split()]  # noqa: E731
    steps = [("page_plan", p[0], w("held fresh free table at place starts next counts"), "plan"),
             ("rope_pages", p[1], w("at place c cos sin q k v"), "rope"),
             ("attention_pages", p[2], w("q k v at table shared work out"), "attend"),
             ("logits_pick", p[3], w("out spans spans pen spans spans spans logits pick"), "pick")]

    def expect():
        want, bad = plan_oracle(held, fresh, order, table, rows, page, pages, first)
        assert not bad
        q64, kk, vv = rope_oracle(c.astype(np.float64), cos, sin, want["at"], want["place"], k64, 48, True, heads, kv, page, np.zeros((rows, heads, hd)))
        vv = v64.copy()
        for r in range(rows):
            if want["at"][r] != SPARE:
                vv[want["place"][r] // page, :, want["place"][r] % page] = c[r, heads + kv:]
        b = Paged.__new__(Paged)
        b.dtype, b.heads, b.kv, b.hd, b.page, b.first, b.rows, b.seqs, b.width, b.pages = dtype, heads, kv, hd, page, first, rows, seqs, width, pages
        # The kernels' own stored q, k and v: the attention is held to what it read.
        b.q64 = read(syn, m["q"], dtype, (rows, heads, hd))
        b.k64, b.v64 = read(syn, m["k"], dtype, k.shape), read(syn, m["v"], dtype, v.shape)
        for got, w in ((b.q64, q64), (b.k64, kk), (b.v64, vv)):
            assert np.all(np.abs(got - w) <= HALF_STEP[dtype] * np.abs(w) + 2 * 12 * 2.0 ** -24)
        b.at, b.table, b.shared = want["at"], want["table"], shared
        return want, b

    return m, steps, expect


def step_check(pkg, syn, m, expect, dtype):
    want, b = expect()
    for n in ("table", "at", "place", "starts", "next", "counts"):
        assert np.array_equal(m[n].read(np.uint32, want[n].size), want[n].reshape(-1)), n
    got = read(syn, m["out"], dtype, (b.rows, b.heads, b.hd))
    for r, e in enumerate(b.expect()):
        if e is None:
            assert np.all(got[r] == 0)
        else:
            assert np.all(np.abs(got[r] - e[0]) <= e[1]), r
    flat = got.reshape(b.rows, -1)
    assert np.array_equal(read(syn, m["logits"], dtype, flat.shape), flat)
    assert np.array_equal(m["pick"].read(np.uint32, b.rows), flat.argmax(1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_step_of_all_four_as_a_program(pkg, ctx, syn, dtype):
    m, steps, expect = step_program(pkg, ctx, syn, dtype)
    prog = pkg.Program(ctx, steps, timed=True)
    for _ in range(3):
        prog.run()
        step_check(pkg, syn, m, expect, dtype)
    assert len(prog.timings()) == 4 and all(t > 0 for t in prog.timings())
    prog.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_step_of_all_four_enqueued_and_captured_on_other_streams(pkg, ctx, syn, dtype):
    import torch

    m, steps, expect = step_program(pkg, ctx, syn, dtype)
    calls = [pkg.Dispatch(ctx, k, p, b, label) for k, p, b, label in steps]
    side = torch.cuda.Stream()
    for stream in (0, side.cuda_stream, ctx.stream):
        for d in calls:
            d.enqueue(stream)
        torch.cuda.synchronize()
        ctx.synchronize()
        step_check(pkg, syn, m, expect, dtype)
        for n in ("out", "q", "pick", "logits", "place"):
            m[n].fill(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for d in calls:
            d.enqueue(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        step_check(pkg, syn, m, expect, dtype)
        for n in ("out", "q", "pick", "logits", "place"):
            m[n].fill(0)
    del graph


# ---- arrays of one to three entries, bound as those alone ------------------------------------------------


def exact(pkg, ctx, a, around=0x7FC00007):
    """The array as a binding of its own bytes, in a buffer whose other words are not what a kernel may use."""
    a = np.ascontiguousarray(a)
    words = np.full(64, around, np.uint32)
    words[4:4 + a.size] = a.reshape(-1).view(np.uint32)
    return put(pkg, ctx, words), 16, a.nbytes


def whole(m):
    return m, 0, m.nbytes


@pytest.mark.parametrize("count", [1, 2, 3])
def test_short_arrays_page_plan(pkg, ctx, count):
    held, fresh, free = np.zeros(4, np.uint32), np.full(4, 5, np.uint32), np.array([6, 2, 4], np.uint32)[:count]
    table = np.full((4, 2), SPARE, np.uint32)
    want, _ = plan_oracle(held, fresh, free, table, 20, 16, 8, 9)
    p = pkg.TgParams(seqs=4, rows=20, stride=2, n=count, capacity=16, slots=8, first=9)
    out = dict(table=put(pkg, ctx, table))
    for name in ("at", "place", "starts", "next", "counts"):
        out[name] = put(pkg, ctx, np.full(want[name].size, 0x77777777, np.uint32))
    pkg.dispatch_once(ctx, "page_plan", p, [whole(put(pkg, ctx, held)), whole(put(pkg, ctx, fresh)), exact(pkg, ctx, free),
                                            *map(whole, out.values())])
    assert want["counts"][2] == count
    for name in want:
        assert np.array_equal(out[name].read(np.uint32, want[name].size), want[name].reshape(-1)), name


@pytest.mark.parametrize("count", [1, 2, 3])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_short_arrays_rope_pages(pkg, ctx, syn, count, dtype):
    rows, heads, kv, hd, page = 6, 4, 1, 64, 16
    pages, c, c64, cos, sin, at, place, old, old64 = rope_case(syn, rows, heads, kv, hd, 2, page, count, dtype, "f32", count)
    p = pkg.TgParams(dtype=pkg.DTYPES[dtype], heads=heads, kv_heads=kv, head_dim=hd, rows=rows, capacity=page, slots=pages, rope=1, k=2, n=count)
    q0, q064 = typed(syn, np.zeros((rows, heads, hd)), dtype)
    q, k, v = put(pkg, ctx, q0), put(pkg, ctx, old), put(pkg, ctx, old)
    pkg.dispatch_once(ctx, "rope_pages", p, [*(whole(put(pkg, ctx, a)) for a in (at, place, c)), exact(pkg, ctx, cos), exact(pkg, ctx, sin),
                                             whole(q), whole(k), whole(v)])
    want = rope_oracle(c64, cos, sin, at, place, old64, 2, False, heads, kv, page, q064)
    for got, w in zip((read(syn, q, dtype, q0.shape), read(syn, k, dtype, old.shape), read(syn, v, dtype, old.shape)), want):
        # As test_rope_pages's.
        assert np.all(np.abs(got - w) <= HALF_STEP[dtype] * np.abs(w) + 2 * 12 * 2.0 ** -24)


@pytest.mark.parametrize("count", [1, 2, 3])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_short_arrays_attention_pages(pkg, ctx, syn, count, dtype):
    b = Paged(syn, dtype, 16, 2, 64, 32, 32 * count, [5, 40], [0, 1], [0, 0], seed=count)
    p = b.params(pkg)
    out, work = put(pkg, ctx, np.zeros(b.q.shape, b.q.dtype)), pkg.Memory(ctx, pkg.attention_pages_work(p))
    pkg.dispatch_once(ctx, "attention_pages", p, [*(whole(put(pkg, ctx, a)) for a in (b.q, b.k, b.v, b.at, b.table)), exact(pkg, ctx, b.shared),
                                                  whole(work), whole(out)])
    b.check(syn, out)


@pytest.mark.parametrize("count", [1, 2, 3])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_short_arrays_logits_pick(pkg, ctx, syn, count, dtype):
    rng = np.random.default_rng(count)
    vocab = 32 * count
    x, x64 = typed(syn, rng.standard_normal((2, vocab)), dtype)
    seen, ids = np.array([7, 3, 7], np.uint32)[:count], np.array([30, 3, 9], np.uint32)[:count]
    bias, bits = rng.standard_normal(count).astype(np.float32), rng.integers(0, 2 ** 32, (1, count), dtype=np.uint64).astype(np.uint32)
    spans = np.array([[0, 1, count - 1, 0, count, 0], [0, 0, count, 0, 0, SPARE]], np.uint32)
    pen = np.array([[1.5, 0.25, 0.5], [0.75, 1, 2]], np.float32)
    p = pkg.TgParams(dtype=pkg.DTYPES[dtype], rows=2, n=vocab, stride=vocab, k=count, k1=count, m=1)
    out, pick = put(pkg, ctx, np.zeros(x.shape, x.dtype)), put(pkg, ctx, np.zeros(2, np.uint32))
    pkg.dispatch_once(ctx, "logits_pick", p, [whole(put(pkg, ctx, x)), exact(pkg, ctx, seen, 5), whole(put(pkg, ctx, spans)),
                                              whole(put(pkg, ctx, pen)), exact(pkg, ctx, ids, 5), exact(pkg, ctx, bias), exact(pkg, ctx, bits),
                                              whole(out), whole(pick)])
    want, size = pick_oracle(x64, seen, spans, pen, ids, bias, bits, vocab)
    pick_check(read(syn, out, dtype, x.shape), pick.read(np.uint32, 2), want, size, vocab, dtype, range(2))


# ---- steps back to back, each from words that the one before stored ---------------------------------------


class Steps:
    """A run of serving steps whose words all come from the device: step i plans from the lengths that step i - 1 stored,
    appends its rows' keys and values to pages it has just handed out, and attends to them behind a shared prefix. Only
    the fresh counts, the free pages and the projections' outputs are given."""

    def __init__(self, pkg, ctx, syn, dtype, hd, first, steps, seed=0):
        rng = np.random.default_rng(seed)
        self.pkg, self.ctx, self.steps = pkg, ctx, steps
        heads, kv, page, seqs, rows, width, pages = 16, 2, 16, 48, 64, 24, 900
        es = 2 if dtype == "bf16" else 4
        order = rng.permutation(pages).astype(np.uint32)
        shared, order = order[:max(4, -(-first // page))], order[max(4, -(-first // page)):]
        held = rng.integers(0, 150, seqs).astype(np.uint32)
        table = np.full((seqs, width), SPARE, np.uint32)
        for s in range(seqs):
            n = -(-int(held[s]) // page)
            table[s, :n], order = order[:n], order[n:]
        kv0 = [typed(syn, rng.standard_normal((pages, kv, page, hd)), dtype)[0] for _ in range(2)]
        angle = np.arange(first + 400)[:, None] * 10000.0 ** (-2 * np.arange(hd // 2) / hd)
        m = {"shared": shared, "k": kv0[0], "v": kv0[1], "cos": np.cos(angle).astype(np.float32), "sin": np.sin(angle).astype(np.float32),
             "held0": held, "table": table}
        self.start = {n: m[n] for n in ("k", "v", "held0", "table")}
        for i in range(steps):
            m[f"fresh{i}"] = rng.integers(0, 2, seqs).astype(np.uint32)
            # As if held pages were many steps' apart: each step hands out pages of its own.
            m[f"free{i}"], order = order[:seqs], order[int(seqs // 8):]
            m[f"c{i}"] = rng.standard_normal((rows, (heads + 2 * kv) * hd)).astype(np.float32)
        self.m = m = {n: put(pkg, ctx, a) for n, a in m.items()}
        base = dict(dtype=pkg.DTYPES[dtype], heads=heads, kv_heads=kv, head_dim=hd, rows=rows, capacity=page, slots=pages, first=first,
                    seqs=seqs, stride=width)
        attend = pkg.TgParams(**base)
        for n, size in (("at", 8 * rows), ("place", 4 * rows), ("starts", 4 * seqs + 4), ("held1", 4 * seqs), ("counts", 16),
                        ("q", rows * heads * hd * es), ("work", pkg.attention_pages_work(attend))):
            m[n] = pkg.Memory(ctx, size)
        self.list = []
        for i in range(steps):
            m[f"out{i}"] = pkg.Memory(ctx, rows * heads * hd * es)
            for kernel, p, names in (
                    ("page_plan", pkg.TgParams(**{**base, "n": seqs}), f"held{i % 2} fresh{i} free{i} table at place starts held{1 - i % 2} counts"),
                    ("rope_pages", pkg.TgParams(**{**base, "rope": 1, "k": hd, "n": first + 400}), f"at place c{i} cos sin q k v"),
                    ("attention_pages", attend, f"q k v at table shared work out{i}")):
                self.list.append((kernel, p, [whole(m[n]) for n in names.split()]))

    def reset(self):
        for n, a in self.start.items():
            self.m[n].write(a)
        for n in ("held1", "at", "place", "q", "work", *(f"out{i}" for i in range(self.steps))):
            self.m[n].fill(0)
        self.ctx.synchronize()

    def results(self):
        return {n: self.m[n].read(np.uint8, self.m[n].nbytes) for n in ("k", "v", "table", "held0", "held1", *(f"out{i}" for i in range(self.steps)))}


@pytest.mark.parametrize("dtype,hd,first", [("bf16", 64, 700), ("bf16", 128, 1500), ("f32", 64, 300), ("bf16", 64, 0), ("bf16", 128, 1)])
def test_steps_back_to_back_are_the_same_bits_as_steps_waited_for(pkg, ctx, syn, dtype, hd, first):
    import torch

    run_ = Steps(pkg, ctx, syn, dtype, hd, first, steps=8, seed=first)
    run_.reset()
    for kernel, p, bindings in run_.list:
        pkg.dispatch_once(ctx, kernel, p, bindings)
    want = run_.results()
    counts = run_.m["counts"].read(np.uint32, 4)
    assert counts[1] > 0 and counts[2] == 48  # rows were placed, and no request was left out
    calls = [pkg.Dispatch(ctx, *step) for step in run_.list]
    side = torch.cuda.Stream()

    def enqueue(stream):
        for d in calls:
            d.enqueue(stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        enqueue(torch.cuda.current_stream().cuda_stream)
    for go in (lambda: enqueue(side.cuda_stream), lambda: enqueue(0), graph.replay, graph.replay):
        run_.reset()
        go()
        torch.cuda.synchronize()
        ctx.synchronize()  # no error word
        got = run_.results()
        for n in want:
            assert np.array_equal(got[n], want[n]), n
    del graph


# ---- calls of different sizes at the same time -------------------------------------------------------------


def plan_call(pkg, ctx, seqs):
    """A plan of one fresh position a request, as a call, with what it makes and how that is read."""
    held, fresh, free, table, pages = plan_case(seqs, 16, 40, 1, seed=seqs)
    fresh[:] = 1
    old = -(-held.astype(np.int64) // 16)
    new = -(-(held.astype(np.int64) + 1) // 16)
    width = int(new.max())
    table = np.full((seqs, width), SPARE, np.uint32)
    ids = np.arange(int(new.sum()), dtype=np.uint32)
    for s, at in enumerate(np.cumsum(old) - old):
        table[s, :old[s]] = ids[at:at + old[s]]
    free = ids[int(old.sum()):]
    want, bad = plan_oracle(held, fresh, free, table, seqs, 16, len(ids), 3)
    assert not bad
    p = pkg.TgParams(seqs=seqs, rows=seqs, stride=width, n=len(free), capacity=16, slots=len(ids), first=3)
    out = dict(table=put(pkg, ctx, table))
    for name in ("at", "place", "starts", "next", "counts"):
        out[name] = put(pkg, ctx, np.zeros(want[name].size, np.uint32))
    call = pkg.Dispatch(ctx, "page_plan", p, [whole(put(pkg, ctx, a)) for a in (held, fresh, free)] + [whole(m) for m in out.values()])
    return call, out, want


def plan_call_check(out, want):
    for name in want:
        assert np.array_equal(out[name].read(np.uint32, want[name].size), want[name].reshape(-1)), name


def linear_call(pkg, ctx, k):
    """A projection of one row over k inputs, as a call; its shared memory grows with k."""
    rng = np.random.default_rng(k)
    x, w = rng.standard_normal(k).astype(np.float32), rng.standard_normal((8, k)).astype(np.float32)
    out = dict(y=put(pkg, ctx, np.zeros(8, np.float32)))
    mems = [put(pkg, ctx, a) for a in (x, x, w, np.zeros(8, np.float32))] + [out["y"]]
    call = pkg.Dispatch(ctx, "gemv_linear", pkg.TgParams(dtype=pkg.F32, rows=1, slots=1, n=8, k=k, stride=8), [whole(m) for m in mems])
    return call, out, (w.astype(np.float64) @ x, np.abs(w.astype(np.float64)) @ np.abs(x), k)


def linear_call_check(out, want):
    y, size, k = want
    # A sum of k products in f32.
    assert np.all(np.abs(out["y"].read(np.float32, 8) - y) <= (k + 1) * 2.0 ** -24 * size)


@pytest.mark.parametrize("make,check,sizes", [(plan_call, plan_call_check, (16384, 3000)), (plan_call, plan_call_check, (5000, 16384, 4000, 9)),
                                              (linear_call, linear_call_check, (6000, 2000, 1200, 4096))])
def test_calls_of_different_sizes_enqueued_from_several_threads(pkg, ctx, make, check, sizes):
    import threading

    import torch

    made = [make(pkg, ctx, n) for n in sizes]
    ctx.synchronize()
    streams, failed = [torch.cuda.Stream() for _ in sizes], []
    start = threading.Barrier(len(sizes))

    def work(call, stream):
        start.wait()
        for i in range(1500):
            try:
                call.enqueue(stream.cuda_stream)
            except pkg.Error as e:
                failed.append(f"{i}: {e}")
                return
            if i % 100 == 99:
                stream.synchronize()

    threads = [threading.Thread(target=work, args=(made[i][0], streams[i])) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ctx.synchronize()
    assert not failed, failed
    for _, out, want in made:
        check(out, want)


def test_a_captured_call_replays_after_smaller_and_larger_ones(pkg, ctx):
    import torch

    big, out, want = plan_call(pkg, ctx, 12000)
    others = [plan_call(pkg, ctx, n) for n in (4000, 16384, 8)]
    ctx.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        big.enqueue(torch.cuda.current_stream().cuda_stream)
    for other, *_ in others:
        out["place"].fill(0)
        out["at"].fill(0)
        other.enqueue(ctx.stream)
        ctx.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        plan_call_check(out, want)
    for _, o, w in others:
        plan_call_check(o, w)
    del graph


# ---- one key among thousands --------------------------------------------------------------------------------


NEEDLE = 1.0 + np.arange(128) * 5 % 16  # the values at a needle, other ones at its neighbours


def needles(syn, b, spots, strength=20.0):
    """Row r's queries all point along dimension r % len(spots), as the key at spots[r % len(spots)] alone does (a position
    of the prefix, or from `first` on the row's own): the row's output is that position's values, up to e^-20 or so."""
    rng = np.random.default_rng(1)
    k, v, q = b.k64.copy(), b.v64.copy(), np.zeros_like(b.q64)
    for r in range(b.rows):
        j = r % len(spots)
        q[r] = 0.05 * rng.standard_normal(q[r].shape)
        q[r, :, j] = strength
        if b.at[r] == SPARE:
            continue
        t, s = spots[j], int(b.at[b.rows + r])
        pg = b.shared[t // b.page] if t < b.first else b.table[s, (t - b.first) // b.page]
        off = (t if t < b.first else t - b.first) % b.page
        k[pg, :, off] = 0.0
        k[pg, :, off, j] = strength
        v[pg, :, off] = NEEDLE[j]
    (b.k, b.k64), (b.v, b.v64), (b.q, b.q64) = (typed(syn, a, b.dtype) for a in (k, v, q))


def edges(steps, end):
    """Positions beside multiples of the steps, the first and the last, below `end`."""
    out = {0, end - 1}
    for s in steps:
        for t in range(s, end + 1, s):
            out |= {t - 1, t}
    return sorted(t for t in out if t < end)


@pytest.mark.parametrize("dtype,heads,kv,hd,page,first", [
    ("bf16", 16, 2, 64, 16, 1000), ("bf16", 16, 2, 64, 64, 8191), ("bf16", 32, 8, 128, 16, 1500), ("bf16", 8, 4, 128, 48, 6001),
    ("bf16", 4, 1, 128, 128, 2049), ("bf16", 20, 4, 64, 32, 4100), ("bf16", 12, 4, 128, 32, 700), ("f32", 16, 2, 64, 32, 1000),
    ("f32", 8, 8, 128, 16, 400)])
def test_attention_pages_finds_one_key_of_the_prefix(pkg, ctx, syn, dtype, heads, kv, hd, page, first):
    """Keys beside the edges of pages, of copies' boxes, of tiles and of pieces, in the first and second half of a tile;
    the queries of a tile move their references at different tiles."""
    spots = edges((128, page), first) + [t + 64 for t in edges((128,), first - 64)] + [t + 16 for t in edges((128,), first - 16)]
    spots = [int(spots[i]) for i in np.linspace(0, len(spots) - 1, min(len(spots), hd)).astype(int)]
    spots = sorted(set(spots) | {0, first - 1})[:hd]
    spots[-1] = first - 1
    rows = 2 * len(spots) + 3
    b = Paged(syn, dtype, heads, kv, hd, page, first, [3] * rows, list(range(rows)), [0] * rows, seed=first)
    needles(syn, b, spots)
    out = b.run(pkg, ctx)
    b.check(syn, out)
    got = read(syn, out, dtype, b.q.shape)
    assert np.all(np.abs(got - NEEDLE[np.arange(rows) % len(spots)][:, None, None]) < 0.5)


@pytest.mark.parametrize("dtype,heads,kv,hd,page,first", [
    ("bf16", 16, 2, 64, 16, 0), ("bf16", 32, 8, 128, 16, 0), ("bf16", 16, 2, 128, 48, 300), ("bf16", 5, 1, 64, 128, 77),
    ("f32", 16, 2, 64, 32, 0), ("f32", 4, 1, 128, 16, 30)])
def test_attention_pages_finds_one_key_of_its_own(pkg, ctx, syn, dtype, heads, kv, hd, page, first):
    """Keys beside the edges of pages, chunks and pieces of a request's own positions."""
    spots = [first + t for t in edges((16, 128), 395)]
    spots = [spots[i] for i in np.linspace(0, len(spots) - 1, min(len(spots), hd)).astype(int)]
    rows = len(spots)
    b = Paged(syn, dtype, heads, kv, hd, page, first, [395] * rows, list(range(rows)), [0] * rows, seed=page)
    needles(syn, b, spots)
    out = b.run(pkg, ctx)
    b.check(syn, out)
    got = read(syn, out, dtype, b.q.shape)
    assert np.all(np.abs(got - NEEDLE[:rows][:, None, None]) < 0.5)


@pytest.mark.parametrize("hd,first", [(64, 3000), (128, 1500), (128, 5000)])
@pytest.mark.parametrize("scale", [8.0, 30.0])
def test_attention_pages_with_peaked_scores_over_several_tiles_of_queries(pkg, ctx, syn, hd, first, scale):
    rows = 70
    lengths = [int(n) for n in np.random.default_rng(hd).integers(1, 500, rows)]
    b = Paged(syn, "bf16", 16, 2, hd, 32, first, lengths, list(range(rows)), [0] * rows, seed=hd, scale=scale)
    b.check(syn, b.run(pkg, ctx))


# ---- large vocabularies and long histories -------------------------------------------------------------------


def wide_case(syn, rows, vocab, stride, hist, dtype, seed, flat=False):
    """Rows over a large vocabulary with histories of as many different tokens as `hist` even draws give. `flat`: whole
    logits with many equal largest ones and controls that change nothing."""
    rng = np.random.default_rng(seed)
    base = rng.integers(-3, 3, stride) if flat else 4 * rng.standard_normal(stride)
    x = np.stack([np.roll(base, 977 * r) for r in range(rows)])
    if flat:
        for r in range(rows):  # equal largest values beside the ends of runs, tiles and blocks' shares
            t = np.concatenate([rng.integers(0, vocab, 4)] + [np.arange(e - 2, e + 2) for e in range(4096, vocab, 4096 * (1 + r % 5))])
            x[r, rng.choice(t[t < vocab], min(6, len(t)), replace=False)] = 5
    x, x64 = typed(syn, x, dtype)
    seen = rng.integers(0, vocab, max(1, hist)).astype(np.uint32)
    spans = np.zeros((rows, 6), np.uint32)
    spans[:, 5] = SPARE
    if hist:
        spans[:, 0] = rng.integers(0, hist // 8, rows)
        spans[:, 1] = hist // 4
        spans[:, 2] = hist - hist // 4 - spans[:, 0]
    if not flat:
        spans[::3, 5] = 0
    pen = np.tile(np.array([[1, 0, 0]], np.float32), (rows, 1)) if flat else np.stack(
        [rng.uniform(0.8, 2, rows), rng.uniform(-1, 1, rows), rng.uniform(-1, 1, rows)], 1).astype(np.float32)
    ids, bias = rng.integers(0, vocab, 40).astype(np.uint32), (3 * rng.standard_normal(40)).astype(np.float32)
    if not flat:
        spans[1::2, 4] = 40
    bits = rng.integers(0, 2 ** 32, (1, (vocab + 31) // 32), dtype=np.uint64).astype(np.uint32)
    return x, x64, seen, spans, pen, ids, bias, bits


@pytest.mark.parametrize("rows,vocab,stride,hist,dtype,in_place,flat", [
    # Two runs of a block's bit map (past 65,536 of its tokens): without controls, with them, with ties, odd ends.
    (66, 150001, 150016, 0, "f32", False, False), (66, 150001, 150016, 0, "bf16", True, True), (66, 150001, 150008, 500, "f32", True, False),
    (66, 150001, 150016, 500, "bf16", False, False), (66, 150001, 150001, 400, "bf16", True, False), (66, 140001, 140004, 300, "f32", False, True),
    (3, 530003, 530003, 900, "f32", False, False),
    # More than 4096, and than 8192, different touched tokens in a block's share: runs cut shorter.
    (2, 131000, 131072, 60000, "f32", False, False), (2, 131000, 131072, 60000, "bf16", True, True), (66, 40001, 40008, 60000, "bf16", False, False),
    (66, 40001, 40004, 60000, "f32", True, True), (1, 20000, 20000, 200000, "f32", False, True), (66, 150001, 150004, 90000, "f32", False, False)])
def test_logits_pick_over_several_runs(pkg, ctx, syn, rows, vocab, stride, hist, dtype, in_place, flat):
    x, x64, seen, spans, pen, ids, bias, bits = wide_case(syn, rows, vocab, stride, hist, dtype, rows + vocab, flat)
    out, pick, bad = pick_run(pkg, ctx, x, seen, spans, pen, ids, bias, bits, vocab, 1, dtype, in_place)
    assert not bad
    got = read(syn, out, dtype, x.shape)
    want, size = pick_oracle(x64, seen, spans, pen, ids, bias, bits, vocab)
    pick_check(got, pick, want, size, vocab, dtype, range(rows))
    left = x64[:, vocab:] if in_place else np.full((rows, stride - vocab), 12.0625 if dtype == "bf16" else 7.0)
    assert np.array_equal(got[:, vocab:], left)

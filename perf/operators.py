"""Cases of the paged serving operators (page_plan, rope_pages, attention_pages, logits_pick), their
plain forms in elementary torch operations, and the same results in 64 bits."""

import math

import torch

own = False
SPARE = -1  # TG_SPARE's bits in an int32 tensor
DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_context = None


def _library():
    """The package and one context on the current device, as a program keeps them."""
    global _context
    import __graft_entry__

    pkg = __graft_entry__.load_package()
    if _context is None:
        _context = pkg.Context(torch.cuda.current_device())
    return pkg, _context


def listed():
    plan, rope, att, pick = "page_plan", "rope_pages", "attention_pages", "logits_pick"
    return [
        # A decode step's bookkeeping for a handful of requests: one new position each.
        dict(name="plan_decode_8", op=plan, seqs=8, chunk=1, page=32, held=2048, first=512, pad=0, short=False),
        # A large mixed step: prefill chunks beside decode rows, some requests idle, padding rows behind.
        dict(name="plan_mixed_2048", op=plan, seqs=2048, chunk=40, page=16, held=1500, first=777, pad=300, short=False),
        # One decode row of the 0.5B-shaped backbone: launch latency.
        dict(name="rope_row", op=rope, rows=1, heads=16, kv_heads=2, head_dim=64, rot=64, inter=False, page=32, positions=2048,
             pad=0, type="bf16", c="f32"),
        # A prefill launch of that backbone (16 prompts of 2048 positions).
        dict(name="rope_prefill_32768", op=rope, rows=32768, heads=16, kv_heads=2, head_dim=64, rot=64, inter=False, page=64,
             positions=4096, pad=0, type="bf16", c="f32"),
        # A chunk with wide heads, part of each rotated in the interleaved layout, from a bf16 projection.
        dict(name="rope_part_2047", op=rope, rows=2047, heads=32, kv_heads=8, head_dim=128, rot=96, inter=True, page=48,
             positions=32768, pad=9, type="bf16", c="bf16"),
        # One request behind a short shared prompt: the step's latency.
        dict(name="attend_row", op=att, rows=1, chunk=1, heads=16, kv_heads=2, head_dim=64, first=512, ownlen=100, page=32, pad=0,
             type="bf16"),
        # 64 requests of ragged lengths behind a 1024-position voice prompt.
        dict(name="attend_64_1024", op=att, rows=64, chunk=1, heads=16, kv_heads=2, head_dim=64, first=1024, ownlen=2048, page=32,
             pad=0, type="bf16"),
        # A full batch behind a long shared prefix that ends inside a page.
        dict(name="attend_128_8191", op=att, rows=128, chunk=1, heads=16, kv_heads=2, head_dim=64, first=8191, ownlen=768, page=64,
             pad=3, type="bf16"),
        # Wide heads, a very long prefix, small pages.
        dict(name="attend_64_16384", op=att, rows=64, chunk=1, heads=32, kv_heads=8, head_dim=128, first=16384, ownlen=1024,
             page=16, pad=0, type="bf16"),
        # The tiny f32 stack, several new positions a request.
        dict(name="attend_f32", op=att, rows=10, chunk=3, heads=4, kv_heads=1, head_dim=64, first=333, ownlen=77, page=48, pad=2,
             type="f32"),
        # Greedy choice for one request: vocabulary of the optional head.
        dict(name="pick_row", op=pick, rows=1, vocab=32000, gap=0, seen=700, biases=20, masks=1, type="f32"),
        # A full batch over a large vocabulary with long histories, half the rows under a grammar.
        dict(name="pick_128_128000", op=pick, rows=128, vocab=128000, gap=0, seen=4096, biases=64, masks=16, type="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((4, 1, 64), (16, 2, 64), (16, 2, 128), (8, 8, 64), (20, 4, 128), (32, 8, 128))


def draw(rng):
    op = rng.choice(("page_plan", "rope_pages", "attention_pages", "attention_pages", "logits_pick"))
    page = rng.choice((16, 32, 48, 64, 128))
    if op == "page_plan":
        return dict(op=op, seqs=_log(rng, 1, 2000), chunk=_log(rng, 1, 40), page=page, held=_log(rng, 1, 1500),
                    first=rng.choice((0, rng.randint(1, 9000))), pad=rng.randint(0, 300), short=rng.random() < 0.3)
    h, kv, hd = rng.choice(_HEADS)
    if op == "rope_pages":
        most = 32768 * 1280 // ((h + 2 * kv) * hd)
        rows = _log(rng, 1, most)
        rot = rng.choice((hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)))
        t = rng.choice(("bf16", "bf16", "f32"))
        return dict(op=op, rows=rows, heads=h, kv_heads=kv, head_dim=hd, rot=rot, inter=rng.random() < 0.5, page=page,
                    positions=_log(rng, 64, 32768), pad=rng.randint(0, min(9, rows - 1)), type=t,
                    c="f32" if t == "f32" else rng.choice(("f32", "bf16")))
    if op == "attention_pages":
        t = rng.choice(("bf16", "bf16", "bf16", "f32"))
        rows = _log(rng, 1, 128 if h * hd <= 2048 else 64)
        first = 0 if rng.random() < 0.15 else _log(rng, 1, 16384 if t == "bf16" else 4096)
        return dict(op=op, rows=rows, chunk=rng.choice((1, 1, 1, rng.randint(2, 5))), heads=h, kv_heads=kv, head_dim=hd, first=first,
                    ownlen=_log(rng, 1, 1024), page=page, pad=rng.randint(0, min(5, rows - 1)), type=t)
    rows = _log(rng, 1, 128)
    return dict(op=op, rows=rows, vocab=_log(rng, 1000, 126000), gap=rng.choice((0, 0, rng.randint(1, 63))), seen=_log(rng, 1, 4096),
                biases=rng.choice((0, rng.randint(1, 64))), masks=rng.choice((0, 1, 16)), type=rng.choice(("f32", "f32", "bf16")))


# ---- inputs -------------------------------------------------------------------------------------------


def _rand(g, n, hi):
    """n whole numbers in [0, hi), int64."""
    return torch.randint(0, max(1, hi), (n,), generator=g, device=DEV)


def _pages_of(counts, perm, width):
    """A block table: request s holds counts[s] pages, handed out of `perm` in order; the rest as nothing left them."""
    before = torch.cumsum(counts, 0) - counts
    j = torch.arange(width, device=DEV)
    ids = perm[(before[:, None] + j).clamp(max=perm.numel() - 1)]
    return torch.where(j < counts[:, None], ids, SPARE).to(torch.int32)


def _plan_inputs(c, g):
    n, page = c["seqs"], c["page"]
    held = _rand(g, n, c["held"] + 1)
    fresh = _rand(g, n, c["chunk"] + 1) if c["chunk"] > 1 else torch.ones(n, dtype=torch.int64, device=DEV)
    old = (held + page - 1) // page
    new = (held + fresh + page - 1) // page - old
    total, want = int(old.sum()), int(new.sum())
    perm = torch.randperm(total + want + 5, generator=g, device=DEV)
    width = (c["held"] + c["chunk"] + page - 1) // page + 1
    return dict(held=held.to(torch.int32), fresh=fresh.to(torch.int32), free=perm[total:].to(torch.int32),
                n_free=want * 2 // 3 if c["short"] else want + 5, table=_pages_of(old, perm, width),
                rows=n * c["chunk"] + c["pad"], width=width, pages=perm.numel())


def _rope_inputs(c, g):
    rows, page, hd = c["rows"], c["page"], c["head_dim"]
    real = rows - c["pad"]
    pages = (rows + page - 1) // page + 1
    at = torch.full((2 * rows,), SPARE, dtype=torch.int32, device=DEV)
    at[:real] = _rand(g, real, c["positions"]).to(torch.int32)
    at[rows:rows + real] = 0
    place = torch.full((rows,), SPARE, dtype=torch.int32, device=DEV)
    place[:real] = torch.randperm(pages * page, generator=g, device=DEV)[:real].to(torch.int32)
    x = torch.randn(rows, (c["heads"] + 2 * c["kv_heads"]) * hd, generator=g, device=DEV).to(_TYPES[c["c"]])
    half = c["rot"] // 2
    # Divisors that grow along the head, as long-context scalings have them, and a magnitude.
    i = torch.arange(half, device=DEV, dtype=torch.float64)
    freq = 10000.0 ** (-2 * i / c["rot"]) / (1 + 7 * i / half)
    angle = torch.arange(c["positions"], device=DEV, dtype=torch.float64)[:, None] * freq
    t = _TYPES[c["type"]]
    return dict(at=at, place=place, c=x, cos=(1.05 * angle.cos()).float(), sin=(1.05 * angle.sin()).float(), real=real, pages=pages,
                q=torch.zeros(rows, c["heads"], hd, dtype=t, device=DEV),
                k=torch.zeros(pages, c["kv_heads"], page, hd, dtype=t, device=DEV),
                v=torch.zeros(pages, c["kv_heads"], page, hd, dtype=t, device=DEV))


def _attention_inputs(c, g):
    rows, page, hd, first = c["rows"], c["page"], c["head_dim"], c["first"]
    real = rows - c["pad"]
    seqs = (real + c["chunk"] - 1) // c["chunk"]
    row = torch.arange(real, device=DEV)
    request, step = row // c["chunk"], row % c["chunk"]
    top = c["ownlen"] + c["chunk"]
    length = (_rand(g, seqs, c["ownlen"]) + 1)[request] + step  # own positions a row attends to
    most = torch.zeros(seqs, dtype=torch.int64, device=DEV).scatter_reduce(0, request, length, "amax")
    counts, shared = (most + page - 1) // page, (first + page - 1) // page
    width = (top + page - 1) // page
    pages = int(counts.sum()) + shared
    perm = torch.randperm(pages, generator=g, device=DEV)
    at = torch.full((2 * rows,), SPARE, dtype=torch.int32, device=DEV)
    at[:real] = (first + length - 1).to(torch.int32)
    at[rows:rows + real] = request.to(torch.int32)
    t = _TYPES[c["type"]]
    cache = (pages, c["kv_heads"], page, hd)
    return dict(q=torch.randn(rows, c["heads"], hd, generator=g, device=DEV).to(t), k=torch.randn(cache, generator=g, device=DEV).to(t),
                v=torch.randn(cache, generator=g, device=DEV).to(t), at=at, table=_pages_of(counts, perm[shared:], width),
                shared=torch.cat([perm[:shared], perm.new_zeros(4)])[:max(4, shared)].to(torch.int32), real=real, seqs=seqs, width=width,
                pages=pages, out=torch.zeros(rows, c["heads"], hd, dtype=t, device=DEV))


def _pick_inputs(c, g):
    rows, vocab = c["rows"], c["vocab"]
    stride = vocab + c["gap"]
    logits = (3 * torch.randn(rows, stride, generator=g, device=DEV)).to(_TYPES[c["type"]])
    length = _rand(g, rows, c["seen"]) + 1
    prompt = (torch.rand(rows, generator=g, device=DEV) * length).long()
    begin = torch.cumsum(length, 0) - length
    total = int(length.sum())
    # Histories repeat a few tokens often, as text does.
    seen = (vocab * torch.rand(total, generator=g, device=DEV) ** 3).long().clamp(max=vocab - 1)
    b = c["biases"]
    ids = torch.rand(rows, vocab, generator=g, device=DEV).topk(b, 1).indices.reshape(-1) if b else seen[:0]
    mask = torch.full((rows,), SPARE, dtype=torch.int64, device=DEV)
    if c["masks"]:
        mask[::2] = _rand(g, (rows + 1) // 2, c["masks"])
    words = (vocab + 31) // 32
    bits = torch.randint(-2 ** 31, 2 ** 31, (max(1, c["masks"]), words), generator=g, device=DEV).to(torch.int32)
    ones = torch.ones_like(length)
    spans = torch.stack([begin, prompt, length - prompt, torch.arange(rows, device=DEV) * b, b * ones, mask], 1)
    u = torch.rand(rows, 3, generator=g, device=DEV)
    return dict(logits=logits, seen=seen.to(torch.int32), spans=spans.to(torch.int32).contiguous(),
                penalties=torch.stack([1 + 0.5 * u[:, 0], u[:, 1], u[:, 2]], 1).contiguous(), bits=bits,
                ids=torch.cat([ids, ids.new_zeros(4)]).to(torch.int32),
                bias=5 * torch.randn(rows * b + 4, generator=g, device=DEV), n_bias=rows * b, stride=stride,
                out=torch.zeros(rows, stride, dtype=_TYPES[c["type"]], device=DEV),
                pick=torch.zeros(rows, dtype=torch.int32, device=DEV))


_INPUTS = {"page_plan": _plan_inputs, "rope_pages": _rope_inputs, "attention_pages": _attention_inputs, "logits_pick": _pick_inputs}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(_INPUTS[case["op"]](case, g), case=case)
    if own:
        s["call"] = _dispatch(case, s)
    return s


def _dispatch(c, s):
    """The dispatch a program makes once over its buffers and enqueues every step."""
    pkg, ctx = _library()
    op, z = c["op"], lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)  # noqa: E731
    w = lambda *names: [pkg.Memory.wrap(ctx, s[n]) for n in names]  # noqa: E731
    if op == "page_plan":
        s.update(at=z(2 * s["rows"]), place=z(s["rows"]), starts=z(c["seqs"] + 1), next=z(c["seqs"]), counts=z(4))
        p = pkg.TgParams(rows=s["rows"], seqs=c["seqs"], stride=s["width"], n=s["n_free"], capacity=c["page"], slots=s["pages"],
                         first=c["first"])
        return pkg.Dispatch(ctx, op, p, w("held", "fresh", "free", "table", "at", "place", "starts", "next", "counts"))
    if op == "logits_pick":
        p = pkg.TgParams(dtype=pkg.DTYPES[c["type"]], rows=c["rows"], n=c["vocab"], stride=s["stride"], k=s["seen"].numel(),
                         k1=s["n_bias"], m=c["masks"])
        return pkg.Dispatch(ctx, op, p, w("logits", "seen", "spans", "penalties", "ids", "bias", "bits", "out", "pick"))
    p = pkg.TgParams(dtype=pkg.DTYPES[c["type"]], heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["head_dim"], rows=c["rows"],
                     capacity=c["page"], slots=s["pages"])
    if op == "rope_pages":
        p.rope, p.k, p.n, p.flags = 1, c["rot"], c["positions"], (1 if c["inter"] else 0) | (2 if c["c"] == "bf16" else 0)
        return pkg.Dispatch(ctx, op, p, w("at", "place", "c", "cos", "sin", "q", "k", "v"))
    p.first, p.seqs, p.stride = c["first"], s["seqs"], s["width"]
    s["work"] = torch.empty(max(16, pkg.attention_pages_work(p)), dtype=torch.uint8, device=DEV)
    return pkg.Dispatch(ctx, op, p, w("q", "k", "v", "at", "table", "shared", "work", "out"))


# ---- one pass -----------------------------------------------------------------------------------------


def run(s):
    c = s["case"]
    if own:
        s["call"].enqueue(torch.cuda.current_stream().cuda_stream)
        if c["op"] == "page_plan":
            return {n: s[n] for n in ("table", "at", "place", "starts", "next", "counts")}
        if c["op"] == "rope_pages":
            return {n: s[n] for n in ("q", "k", "v")}
        if c["op"] == "logits_pick":
            return {"out": s["out"][:, :c["vocab"]], "pick": s["pick"]}
        return {"out": s["out"]}
    return {"page_plan": _plan_plain, "rope_pages": _rope_plain, "attention_pages": _attention_plain, "logits_pick": _pick_plain}[c["op"]](c, s)


def _plan_plain(c, s):
    page, rows, width = c["page"], s["rows"], s["width"]
    held, fresh = s["held"].long(), s["fresh"].long()
    old = (held + page - 1) // page
    after = (held + fresh + page - 1) // page
    need = after - old
    pages, tokens = torch.cumsum(need, 0), torch.cumsum(fresh, 0)
    bad = (pages > s["n_free"]) | (tokens > rows) | (after > width)
    served = torch.cumsum(bad, 0) == 0
    fresh, need = fresh * served, need * served
    tokens, taken = torch.cumsum(fresh, 0), torch.cumsum(need, 0)
    j = torch.arange(width, device=DEV)
    source = (taken - need)[:, None] + j - old[:, None]
    new = (j >= old[:, None]) & (j < (old + need)[:, None])
    table = torch.where(new, s["free"][source.clamp(0, s["free"].numel() - 1)], s["table"])
    r = torch.arange(rows, device=DEV)
    request = torch.searchsorted(tokens, r, right=True)
    real = request < c["seqs"]
    request = request.clamp(max=c["seqs"] - 1)
    index = held[request] + r - (tokens - fresh)[request]
    place = table[request, (index // page).clamp(0, width - 1)].long() * page + index % page
    at = torch.cat([torch.where(real, c["first"] + index, SPARE), torch.where(real, request, SPARE)])
    counts = torch.stack([taken[-1], tokens[-1], served.sum(), pages[-1]])
    starts = torch.cat([tokens.new_zeros(1), tokens])
    out = dict(table=table, at=at, place=torch.where(real, place, SPARE), starts=starts, next=held + fresh, counts=counts)
    return {n: x.to(torch.int32) for n, x in out.items()}


def _rope_plain(c, s):
    n, h, kv, hd, rot, page = s["real"], c["heads"], c["kv_heads"], c["head_dim"], c["rot"], c["page"]
    x = s["c"][:n].float().view(n, h + 2 * kv, hd)
    cos, sin = (s[t][s["at"][:n].long()][:, None] for t in ("cos", "sin"))
    qk = x[:, :h + kv]
    if c["inter"]:
        a, b = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    qk = torch.cat([turned, qk[..., rot:]], -1).to(s["q"].dtype)
    place = s["place"][:n].long()
    s["q"][:n] = qk[:, :h]
    s["k"][place // page, :, place % page] = qk[:, h:]
    s["v"][place // page, :, place % page] = x[:, h + kv:].to(s["v"].dtype)
    return {t: s[t] for t in ("q", "k", "v")}


def _attention_plain(c, s):
    n, h, kv, hd, page, first = s["real"], c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["first"]
    q = s["q"][:n].float().view(n, kv, h // kv, hd) / math.sqrt(hd)
    shared = s["shared"][:(first + page - 1) // page].long()
    ks, vs = (s[t][shared].float().transpose(0, 1).reshape(kv, len(shared) * page, hd)[:, :first] for t in "kv")
    ids = s["table"][s["at"][c["rows"]:c["rows"] + n].long()].clamp(min=0).long()
    ko, vo = (s[t][ids].float().transpose(1, 2).reshape(n, kv, -1, hd) for t in "kv")
    length = s["at"][:n].long() - first + 1
    masked = torch.arange(s["width"] * page, device=DEV) >= length[:, None]
    score = torch.cat([torch.matmul(q.permute(1, 0, 2, 3).reshape(kv, n * (h // kv), hd), ks.transpose(1, 2)).view(kv, n, h // kv, first).transpose(0, 1),
                       torch.matmul(q, ko.transpose(2, 3)).masked_fill(masked[:, None, None], -math.inf)], -1)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    far = torch.matmul(p[..., :first].transpose(0, 1).reshape(kv, n * (h // kv), first), vs).view(kv, n, h // kv, hd).transpose(0, 1)
    o = far + torch.matmul(p[..., first:], vo.masked_fill(masked[:, None, :, None], 0.0))
    s["out"][:n] = o.reshape(n, h, hd).to(s["out"].dtype)
    return {"out": s["out"]}


def _pick_plain(c, s):
    rows, vocab = c["rows"], c["vocab"]
    x = s["logits"][:, :vocab].float()
    begin, prompt, made, bias0, biases, mask = s["spans"].long().unbind(1)
    i = torch.arange(s["seen"].numel(), device=DEV)
    row = torch.searchsorted(begin + prompt + made, i, right=True)
    at = row * vocab + s["seen"].long()
    zero = torch.zeros(rows * vocab, device=DEV)
    made_of = (i >= (begin + prompt)[row]).float()
    every, counts = (zero.index_add(0, at, v).view(rows, vocab) for v in (torch.ones_like(made_of), made_of))
    r, presence, frequency = (s["penalties"][:, j:j + 1] for j in range(3))
    x = torch.where(every > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - counts * frequency - (counts > 0) * presence
    if s["n_bias"]:
        j = torch.arange(s["n_bias"], device=DEV)
        at = j // c["biases"] * vocab + s["ids"][:s["n_bias"]].long()
        x = x + zero.index_put((at,), s["bias"][:s["n_bias"]]).view(rows, vocab)
    t = torch.arange(vocab, device=DEV)
    allowed = (s["bits"][mask.clamp(min=0)][:, t // 32] >> (t % 32)) & 1
    x = torch.where((allowed == 0) & (mask >= 0)[:, None], -math.inf, x).to(s["logits"].dtype)
    best = x.amax(1, keepdim=True)
    pick = torch.where(x == best, t, vocab).amin(1)
    return {"out": x, "pick": torch.where(best[:, 0] == -math.inf, SPARE, pick).to(torch.int32)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"page_plan": lambda c, s: None, "rope_pages": _rope_exact, "attention_pages": _attention_exact,
            "logits_pick": _pick_exact}[case["op"]](case, s)


def _rope_exact(c, s):
    h, kv, hd, rot, page = c["heads"], c["kv_heads"], c["head_dim"], c["rot"], c["page"]
    n, half = s["real"], c["rot"] // 2
    out = {t: torch.zeros(s[t].shape, dtype=torch.float64, device=DEV) for t in "qkv"}
    pos, place = s["at"][:n].long(), s["place"][:n].long()
    turn = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])
    for head in range(h + 2 * kv):
        x = s["c"][:n, head * hd:(head + 1) * hd].double()
        if head < h + kv:
            first, second = (slice(0, rot, 2), slice(1, rot, 2)) if c["inter"] else (slice(0, half), slice(half, rot))
            z = torch.complex(x[:, first], x[:, second]) * turn
            x[:, first], x[:, second] = z.real, z.imag
        if head < h:
            out["q"][:n, head] = x
        else:
            out["k" if head < h + kv else "v"][place // page, (head - h) % kv, place % page] = x
    return out


def _attention_exact(c, s):
    h, kv, hd, page, first, rows = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["first"], c["rows"]
    group, out = h // kv, torch.zeros(rows, h, hd, dtype=torch.float64, device=DEV)
    i = torch.arange(first, device=DEV)
    at, table, shared = s["at"].tolist(), s["table"].long(), s["shared"].long()
    common = [s[t][shared[i // page], :, i % page].double() for t in "kv"]  # [first][kv][hd]
    for r in range(s["real"]):
        j = torch.arange(at[r] - first + 1, device=DEV)
        pages = table[at[rows + r]][j // page]
        k, v = (torch.cat([f, s[t][pages, :, j % page].double()]).transpose(0, 1) for f, t in zip(common, "kv"))
        q = s["q"][r].double().view(kv, group, hd)
        out[r] = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(hd), -1).matmul(v).view(h, hd)
    return {"out": out}


def _pick_exact(c, s):
    vocab, out = c["vocab"], []
    for r, (begin, prompt, made, bias0, biases, mask) in enumerate(s["spans"].tolist()):
        x = s["logits"][r, :vocab].double()
        repetition, presence, frequency = s["penalties"][r].double().unbind()
        seen = s["seen"][begin:begin + prompt + made].long()
        every, counts = torch.bincount(seen, minlength=vocab), torch.bincount(seen[prompt:], minlength=vocab)
        x = torch.where(every > 0, x * torch.where(x > 0, 1 / repetition, repetition), x) - frequency * counts
        x[counts > 0] -= presence
        x[s["ids"][bias0:bias0 + biases].long()] += s["bias"][bias0:bias0 + biases].double()
        if mask >= 0:
            bits = (s["bits"][mask].long()[:, None] >> torch.arange(32, device=DEV)) & 1
            x[bits.view(-1)[:vocab] == 0] = -math.inf
        out.append(x)
    return {"out": torch.stack(out), "pick": None}


# ---- what a pass cannot do without -------------------------------------------------------------------------


def work(case):
    c, size = case, {"f32": 4, "bf16": 2}
    if c["op"] == "page_plan":
        new = c["seqs"] * (c["chunk"] / 2 if c["chunk"] > 1 else 1)
        return {"bytes": 16 * c["seqs"] + 12 * (c["seqs"] * c["chunk"] + c["pad"]) + 8 * new / c["page"], "flops": 0}
    if c["op"] == "logits_pick":
        return {"bytes": c["rows"] * (2 * c["vocab"] * size[c["type"]] + 2 * c["seen"] + 8 * c["biases"]) + c["masks"] * c["vocab"] / 8,
                "flops": 4 * c["rows"] * c["vocab"]}
    h, kv, hd, t = c["heads"], c["kv_heads"], c["head_dim"], size[c["type"]]
    real = c["rows"] - c["pad"]
    if c["op"] == "rope_pages":
        values = real * (h + 2 * kv) * hd
        return {"bytes": values * (size[c["c"]] + t) + 4 * real * min(1, c["positions"] / real) * c["rot"], "flops": 3 * values}
    length = c["ownlen"] / 2 + 1
    return {"bytes": t * (2 * real * h * hd + 2 * kv * hd * (c["first"] + real / c["chunk"] * length)),
            "flops": 4 * hd * h * real * (c["first"] + length)}

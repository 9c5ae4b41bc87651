"""What is measured of the paged 8-bit key/value cache and of beam search: cases, inputs, plain forms.

Four operators, as one step of a decode loop uses them:

* ``append``: rotary embedding of new query / key heads, and the keys and values written to a paged
  cache as e4m3 codes with one power-of-two scale for each page and head;
* ``attend``: causal attention of the newest tokens of every sequence over that cache;
* ``reorder`` / ``compact``: sequences that continue other sequences (shared pages, a copy of the
  page that is still being filled, pages nobody holds any more), and the pool's live pages moved to
  its front;
* ``select``: the best continuations over beams and vocabulary.

``own`` picks the framework's kernels or the plain torch forms below.
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
EXP_MIN, EXP_MAX = -24, 60          # scales are 2**EXP_MIN .. 2**EXP_MAX


# ---- cases ----------------------------------------------------------------------------------------
def _append(name, dtype, n, nh, nkv, hd, page, past, t):
    return dict(name=name, op="append", dtype=dtype, n=n, nh=nh, nkv=nkv, hd=hd, page=page,
                past_lo=past[0], past_hi=past[1], t_lo=t[0], t_hi=t[1])


def _attend(name, dtype, n, nh, nkv, hd, page, past, t):
    return dict(_append(name, dtype, n, nh, nkv, hd, page, past, t), op="attend")


def listed():
    return [
        # one decode step of a batch of eight, 7B-class heads, in the middle of the answers
        _append("append 8x1 f16", "float16", 8, 32, 8, 128, 64, (511, 1535), (1, 1)),
        # the same for many short sequences of a small float32 model with small pages
        _append("append 64x1 f32 d64", "float32", 64, 12, 12, 64, 16, (9, 4000), (1, 1)),
        # four prompts of uneven length enter an empty cache
        _append("append prompts bf16", "bfloat16", 4, 32, 32, 128, 64, (0, 0), (700, 4096)),
        # one answer, a key head for every query head: the smallest call, latency counts
        _attend("attend 1x1 f16 mha", "float16", 1, 32, 32, 128, 64, (639, 639), (1, 1)),
        # a decode step of a batch of eight with four query heads to a key head
        _attend("attend 8x1 f16", "float16", 8, 32, 8, 128, 64, (511, 1535), (1, 1)),
        # a serving batch of uneven, long sequences, eight query heads to a key head
        _attend("attend 32x1 bf16 long", "bfloat16", 32, 64, 8, 128, 64, (1000, 32000), (1, 1)),
        # a piece of a prompt after a long cached beginning
        _attend("attend 2x256 bf16", "bfloat16", 2, 32, 8, 128, 64, (2000, 6000), (200, 256)),
        # 4 prompts x 4 beams after a step: some beams end, others are continued twice
        dict(name="reorder 4x4", op="reorder", layers=32, nkv=8, hd=128, page=64, groups=4, beams=4,
             len_lo=700, len_hi=1100),
        # a pool that many requests came to and left: the live pages go to the front
        dict(name="compact 1024", op="compact", layers=8, nkv=8, hd=128, page=64, pages=1024,
             live=620, seqs=40),
        # one prompt with four beams
        dict(name="select 1x4 f16", op="select", dtype="float16", n=1, beams=4, vocab=32000),
        # four prompts with four beams, float32 logits
        dict(name="select 4x4 f32", op="select", dtype="float32", n=4, beams=4, vocab=32000),
        # a large batch over a large vocabulary of odd size
        dict(name="select 32x8 bf16", op="select", dtype="bfloat16", n=32, beams=8, vocab=129283),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "reorder", "compact", "select"])
    if op in ("append", "attend"):
        while True:
            nkv = rng.choice([1, 2, 4, 5, 8, 12, 32])
            group = 1 if nkv > 8 else rng.choice([1, 2, 3, 4, 7, 8])
            n, hd, page = _log(rng, 1, 64), rng.choice([32, 64, 96, 128, 128]), rng.choice([16, 32, 64, 128])
            past = sorted(_log(rng, 1, 30000) - 1 for _ in range(2))
            t = [1, 1] if rng.random() < 0.55 else sorted(_log(rng, 1, 300) for _ in range(2))
            c = dict(op=op, dtype=rng.choice(list(TYPES)), n=n, nh=nkv * group, nkv=nkv, hd=hd, page=page,
                     past_lo=past[0], past_hi=past[1], t_lo=t[0], t_hi=t[1])
            padded = n * (past[1] + t[1])
            if padded * nkv * hd <= 5e8 and padded * c["nh"] * t[1] <= 5e8 and work(c)["flops"] <= 2e10 * (1 + 3 * (t[1] > 1)):
                return c
    if op == "reorder":
        lo = _log(rng, 20, 3000)
        return dict(op=op, layers=rng.randint(1, 32), nkv=rng.choice([1, 2, 4, 8]), hd=rng.choice([32, 64, 96, 128]),
                    page=rng.choice([16, 32, 64, 128]), groups=rng.randint(1, 8), beams=rng.randint(2, 8),
                    len_lo=lo, len_hi=min(3000, lo + rng.randint(0, 500)))
    if op == "compact":
        pages = _log(rng, 20, 1000)
        live = rng.randint(pages // 4 + 1, pages - pages // 8 - 1)
        return dict(op=op, layers=rng.randint(1, 8), nkv=rng.choice([1, 2, 4, 8]), hd=rng.choice([64, 96, 128]),
                    page=rng.choice([16, 32, 64]), pages=pages, live=live, seqs=rng.randint(1, min(live, 100)))
    n, beams = _log(rng, 1, 32), rng.randint(1, 8)
    return dict(op=op, dtype=rng.choice(list(TYPES)), n=n, beams=beams,
                vocab=_log(rng, 500, 129283))


# ---- shapes of a case, the same for every seed --------------------------------------------------------
def _spread(n, lo, hi, salt):
    """n whole numbers from lo to hi, evenly over their logarithm, in a mixed order."""
    v = [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / max(1, n - 1)))) - 1 for i in range(n)]
    random.Random(salt).shuffle(v)
    return v


def _lengths(c):
    return _spread(c["n"], c["past_lo"], c["past_hi"], 1), _spread(c["n"], c["t_lo"], c["t_hi"], 2)


def _beams(c):
    """(lengths of the groups, parents): in each group the survivors keep their slot and the others
    continue one of them, so that the same call again finds the same state."""
    r = random.Random(3)
    parents = []
    for g in range(c["groups"]):
        keep = r.sample(range(c["beams"]), max(1, c["beams"] // 2))
        parents += [g * c["beams"] + (b if b in keep else r.choice(keep)) for b in range(c["beams"])]
    return _spread(c["groups"], c["len_lo"], c["len_hi"], 4), parents


def _copies(c):
    """Rows that a reorder has to copy, for each beam that needs a page of its own."""
    lens, parents = _beams(c)
    return [lens[i // c["beams"]] % c["page"] for i, p in enumerate(parents)
            if p != i and lens[i // c["beams"]] % c["page"]]


def _live(c):
    """(ids of the live pages, how many of them have to move)."""
    ids = random.Random(5).sample(range(c["pages"]), c["live"])
    return ids, sum(i >= c["live"] for i in ids)


def work(c):
    if c["op"] in ("append", "attend"):
        past, t = _lengths(c)
        es = 4 if c["dtype"] == "float32" else 2
        tokens, row = sum(t), c["nkv"] * c["hd"]
        if c["op"] == "append":      # q, k, v and cos, sin in; q and the codes out
            return {"bytes": tokens * ((2 * c["nh"] + 2 * c["nkv"]) * c["hd"] * es + 2 * c["hd"] * es + 2 * row),
                    "flops": 3 * tokens * (c["nh"] + c["nkv"]) * c["hd"]}
        keys = sum(p + n for p, n in zip(past, t))
        seen = sum(p * n + n * (n + 1) // 2 for p, n in zip(past, t))
        return {"bytes": 2 * keys * row + 2 * tokens * c["nh"] * c["hd"] * es, "flops": 4 * seen * c["nh"] * c["hd"]}
    if c["op"] == "reorder":
        row = c["layers"] * 2 * c["nkv"] * c["hd"]
        return {"bytes": 2 * row * sum(_copies(c)) + 8 * c["groups"] * c["beams"] * (c["len_hi"] // c["page"] + 1), "flops": 0}
    if c["op"] == "compact":
        return {"bytes": 2 * _live(c)[1] * c["layers"] * 2 * c["nkv"] * c["page"] * c["hd"] + 8 * c["pages"], "flops": 0}
    es = 4 if c["dtype"] == "float32" else 2
    values = c["n"] * c["beams"] * c["vocab"]
    return {"bytes": values * es, "flops": 3 * values}


# ---- inputs -------------------------------------------------------------------------------------------
def _power(e):
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _exponent(amax):
    """The least e in EXP_MIN..EXP_MAX with amax <= 448 * 2**e (448 is e4m3's largest value)."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).to(torch.int32)
    return torch.where(amax == 0, EXP_MIN, e.clamp(EXP_MIN, EXP_MAX)).to(torch.int32)


def _filled(shape, g):
    """Codes and scales of a pool of pages [layers, pages, 2, heads, page, head_dim]: heads and
    channels of uneven size, as keys and values have them."""
    L, P, _, H, S, D = shape
    codes = torch.empty(shape, dtype=E4M3, device="cuda")
    scales = torch.empty(shape[:4], dtype=torch.float32, device="cuda")
    size = torch.exp(torch.randn((2, H, 1, D), generator=g, device="cuda") * 0.5)
    for layer in range(L):
        for p in range(0, P, 4096):
            v = torch.randn((min(4096, P - p), 2, H, S, D), generator=g, device="cuda") * size
            e = _exponent(v.abs().amax((-1, -2)))
            scales[layer, p:p + 4096] = _power(e)
            codes[layer, p:p + 4096] = (v * _power(-e)[..., None, None]).to(E4M3)
    return codes, scales


def _tables(lens, page, pages, max_pages, g):
    """Page table and reference counts of sequences that lie scattered over the pool."""
    at = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    held = [-(-n // page) for n in lens]
    table = torch.full((len(lens), max_pages), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at, k = at.cpu(), 0
    for i, h in enumerate(held):
        table[i, :h] = at[k:k + h]
        k += h
    refs[at[:k].long()] = 1
    return table.cuda(), refs.cuda()


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = SimpleNamespace(case=c, cache=None)
    if c["op"] == "select":
        shape = (c["n"], c["beams"], c["vocab"])
        s.logits = (torch.randn(shape, generator=g, device="cuda") * 2.5).to(TYPES[c["dtype"]])
        s.scores = -20 * torch.rand(shape[:2], generator=g, device="cuda")
        s.done = torch.rand(shape[:2], generator=g, device="cuda") < 0.15      # beams that have ended
        s.eos = 2
        if own:
            from cats_b200 import ops
            s.ops = ops
        return s
    if c["op"] in ("append", "attend"):
        past, t = _lengths(c)
        lens, layers = [p + n for p, n in zip(past, t)], 1
        s.page, s.past, s.t = c["page"], past, t
        max_pages = -(-max(lens) // c["page"]) + 1
        pages = sum(-(-n // c["page"]) for n in lens) + 3
    elif c["op"] == "reorder":
        group_lens, parents = _beams(c)
        layers, lens = c["layers"], [n for n in group_lens for _ in range(c["beams"])]
        max_pages = -(-max(lens) // c["page"]) + 1
        pages = sum(-(-n // c["page"]) + c["beams"] for n in group_lens) + c["beams"] * c["groups"]
        s.parents = torch.tensor(parents, dtype=torch.int32, device="cuda")
        s.n_copies = len(_copies(c))
    else:
        ids, s.n_moves = _live(c)
        layers, pages = c["layers"], c["pages"]
        cut = sorted(random.Random(6).sample(range(1, c["live"]), c["seqs"] - 1)) if c["seqs"] > 1 else []
        held = [b - a for a, b in zip([0] + cut, cut + [c["live"]])]
        lens = [h * c["page"] - 5 for h in held]
        max_pages = max(held) + 1
    s.codes, s.scales = _filled((layers, pages, 2, c["nkv"], c["page"], c["hd"]), g)
    if c["op"] == "reorder":     # the beams of a group share their full pages
        at, k = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu(), 0
        table = torch.full((len(lens), max_pages), -1, dtype=torch.int32)
        for i, n in enumerate(lens):
            full = n // c["page"]
            if i % c["beams"] == 0:
                table[i, :full] = at[k:k + full]
                k += full
            else:
                table[i, :full] = table[i - 1, :full]
            if n % c["page"]:
                table[i, full] = at[k]
                k += 1
        s.refs = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32).cuda()
        s.table = table.cuda()
    elif c["op"] == "compact":
        shuffle = torch.randperm(c["live"], generator=g, device="cuda").cpu()
        at, k = torch.tensor(ids, dtype=torch.int32)[shuffle], 0
        table = torch.full((len(lens), max_pages), -1, dtype=torch.int32)
        for i, h in enumerate(held):
            table[i, :h] = at[k:k + h]
            k += h
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[at.long()] = 1
        s.table, s.refs = table.cuda(), refs.cuda()
        s.table0, s.refs0 = s.table.clone(), s.refs.clone()
    else:
        s.table, s.refs = _tables(lens, c["page"], pages, max_pages, g)
        dt = TYPES[c["dtype"]]
        s.cu = torch.tensor([0] + torch.tensor(t).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        if c["t_lo"] == c["t_hi"] == 1:
            s.cu = None                  # one token of every sequence
        s.tokens, s.t_max, s.len_max = sum(t), max(t), max(lens)
        if c["op"] == "append":
            s.qkv = torch.randn((s.tokens, (c["nh"] + 2 * c["nkv"]) * c["hd"]), generator=g, device="cuda").to(dt)
            ang = torch.outer(torch.arange(max_pages * c["page"], device="cuda", dtype=torch.float64),
                              10000.0 ** (-torch.arange(0, c["hd"], 2, device="cuda", dtype=torch.float64) / c["hd"]))
            s.cos, s.sin = (torch.cat((f(ang), f(ang)), -1).to(dt).contiguous() for f in (torch.cos, torch.sin))
        else:
            s.q = torch.randn((s.tokens, c["nh"], c["hd"]), generator=g, device="cuda").to(dt)
    s.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if own:
        from cats_b200.kv8 import KVCache8
        s.cache = KVCache8.from_tensors(s.codes, s.scales, s.table, s.lens, s.refs)
    return s


# ---- plain forms -----------------------------------------------------------------------------------------
def _tokens(s):
    """(sequence, position) of every new token, and each sequence's count of them and first token."""
    n = s.lens.numel()
    cu = s.cu if s.cu is not None else torch.arange(n + 1, device="cuda", dtype=torch.int32)
    count = (cu[1:] - cu[:-1]).long()
    i = torch.arange(s.tokens, device="cuda")
    seq = torch.searchsorted(cu.long(), i, right=True) - 1
    return seq, s.lens.long()[seq] - count[seq] + i - cu.long()[seq], count, cu.long()[:-1]


def _plain_append(s):
    c = s.case
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    seq, pos, count, first = _tokens(s)
    x = s.qkv.float().view(s.tokens, nh + 2 * nkv, hd)
    qk, v = x[:, :nh + nkv], x[:, nh + nkv:]
    turned = torch.cat((-qk[..., hd // 2:], qk[..., :hd // 2]), -1)
    qk = qk * s.cos.float()[pos][:, None] + turned * s.sin.float()[pos][:, None]
    q = qk[:, :nh].to(s.qkv.dtype)
    kv = torch.stack((qk[:, nh:], v), 1)                                       # [tokens, 2, nkv, hd]
    # pages that get new rows: up to `most` of a sequence, the last one again where it has fewer
    most = (s.t_max - 1) // page + 2
    lens = s.lens.long()
    start = lens - count
    p0 = start // page
    j = torch.minimum(torch.arange(most, device="cuda")[None], ((lens - 1) // page - p0)[:, None])
    place = seq * most + pos // page - p0[seq]
    amax = torch.where(kv.isfinite(), kv.abs(), 0.0).amax(-1)
    top = torch.zeros((lens.numel() * most, 2, nkv), device="cuda")
    top.scatter_reduce_(0, place[:, None, None].expand_as(amax), amax, "amax")
    top = top.view(-1, most, 2, nkv).gather(1, j[:, :, None, None].expand(-1, -1, 2, nkv))
    ids = s.table.long().gather(1, p0[:, None] + j)
    base = (p0[:, None] + j) * page
    old = (start[:, None] - base).clamp(0, page)                               # rows that were there
    held = torch.where(old[..., None, None] > 0, s.scales[0][ids], _power(torch.tensor(EXP_MIN, device="cuda")))
    scale = torch.maximum(held, _power(_exponent(top)))
    r = torch.arange(page, device="cuda")
    token = (first[:, None, None] + base[..., None] + r - start[:, None, None]).clamp(0, s.tokens - 1)
    fresh = kv[token].permute(0, 1, 3, 4, 2, 5) / scale[..., None, None]       # [n, most, 2, nkv, page, hd]
    was = s.codes[0][ids]
    moved = was.float() * (held / scale)[..., None, None]
    r = r[None, None, None, None, :, None]
    row = lambda t: t[:, :, None, None, None, None]  # noqa: E731
    now = torch.where(r < row(old), moved, torch.where(r < row(lens[:, None] - base), fresh, was.float()))
    s.codes[0][ids] = now.to(E4M3)
    s.scales[0][ids] = scale
    return {"q": q, "codes": s.codes, "scales": s.scales}


def _plain_attend(s):
    c = s.case
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    n, group, pages = s.lens.numel(), c["nh"] // c["nkv"], -(-s.len_max // c["page"])
    seq, pos, count, first = _tokens(s)
    place = torch.arange(s.tokens, device="cuda") - first[seq]
    q = torch.zeros((n, s.t_max, nh, hd), device="cuda")
    q[seq, place] = s.q.float()
    q = q.view(n, s.t_max, nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, group * s.t_max, hd)
    ids = s.table[:, :pages].long().clamp(min=0)
    kv = s.codes[0][ids].float() * s.scales[0][ids][..., None, None]           # [n, pages, 2, nkv, page, hd]
    k, v = (kv[:, :, i].transpose(1, 2).reshape(n, nkv, pages * page, hd) for i in (0, 1))
    lens = s.lens.long()[:, None, None]
    at = lens - count[:, None, None] + torch.arange(s.t_max, device="cuda")[None, :, None]
    key = torch.arange(pages * page, device="cuda")[None, None]
    seen = ((key <= at) & (key < lens))[:, None, None]                         # [n, 1, 1, t, keys]
    x = (q @ k.transpose(2, 3)).view(n, nkv, group, s.t_max, -1) * hd ** -0.5
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, nkv, group * s.t_max, -1) @ v).view(n, nkv, group, s.t_max, hd) / total.clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(n, s.t_max, nh, hd)[seq, place].to(s.q.dtype)


def _plain_reorder(s):
    page, n = s.case["page"], s.lens.numel()
    i = torch.arange(n, device="cuda")
    p = s.parents.long()
    lens = s.lens.long()
    full, held = lens // page, (lens + page - 1) // page
    children = torch.zeros(n, dtype=torch.int32, device="cuda").index_add_(0, p, torch.ones_like(s.parents))
    j = torch.arange(s.table.shape[1], device="cuda")[None]
    change = torch.where(j < full[:, None], children[:, None] - 1,
                         torch.where((j < held[:, None]) & (children[:, None] == 0), -1, 0)).to(torch.int32)
    s.refs.index_add_(0, s.table.long().clamp(min=0).view(-1), change.view(-1))
    eldest = torch.full((n,), n, device="cuda").scatter_reduce_(0, p, i, "amin")
    more = (eldest[p] != i) & (held > full)[p]                       # needs a page of its own
    free = torch.argsort((s.refs > 0).to(torch.int32), stable=True)[:n]
    fresh = free[(more.long().cumsum(0) - 1).clamp(min=0)]
    table = s.table[p]
    last = full[p].clamp(max=table.shape[1] - 1)[:, None]
    source = table.long().gather(1, last)[:, 0]
    table.scatter_(1, last, torch.where(more, fresh, source).to(torch.int32)[:, None])
    s.refs.index_add_(0, fresh, more.to(torch.int32))
    which = torch.argsort((~more).to(torch.int32), stable=True)[:s.n_copies]
    a, b, fill = source[which], fresh[which], (lens % page)[p][which]
    rows = (torch.arange(page, device="cuda")[None] < fill[:, None])[None, :, None, None, :, None]
    s.codes.view(torch.uint8)[:, b] = torch.where(rows, s.codes.view(torch.uint8)[:, a], s.codes.view(torch.uint8)[:, b])
    s.scales[:, b] = s.scales[:, a]
    s.table.copy_(table)
    s.lens.copy_(lens[p])
    return {"codes": s.codes, "scales": s.scales, "table": s.table, "refs": s.refs, "lens": s.lens}


def _plain_compact(s):
    alive = s.refs > 0
    ids = torch.arange(alive.numel(), device="cuda")
    n = alive.sum()
    to = torch.argsort((alive | (ids >= n)).to(torch.int32), stable=True)[:s.n_moves]
    of = torch.argsort((~(alive & (ids >= n))).to(torch.int32), stable=True)[:s.n_moves]
    s.codes.view(torch.uint8)[:, to] = s.codes.view(torch.uint8)[:, of]
    s.scales[:, to] = s.scales[:, of]
    ids[of] = to
    s.table.copy_(torch.where(s.table >= 0, ids[s.table.long().clamp(min=0)].to(torch.int32), -1))
    s.refs[to] = s.refs[of]
    s.refs[of] = 0
    return n.to(torch.int32)


def _plain_select(s):
    n, beams, vocab = s.logits.shape
    x = s.logits.double()
    x = x - x.amax(-1, keepdim=True)
    x = s.scores.double()[..., None] + x - torch.log(torch.exp(x).sum(-1, keepdim=True))
    ended = torch.full((vocab,), -math.inf, dtype=torch.float64, device="cuda")
    ended[s.eos] = 0
    x = torch.where(s.done[..., None], s.scores.double()[..., None] + ended, x).view(n, -1)
    best, flat = torch.sort(x, dim=-1, descending=True, stable=True)
    best, flat = best[:, :beams], flat[:, :beams]
    rows = (flat // vocab + torch.arange(n, device="cuda")[:, None] * beams).to(torch.int32)
    token = flat % vocab
    done = s.done.view(-1)[rows.long()] | (token == s.eos)
    return {"scores": best.float(), "rows": rows, "tokens": token, "done": done}


def run(s):
    op = s.case["op"]
    if op == "append":
        if own:
            q = s.cache.append(0, s.qkv, s.case["nh"], s.cos, s.sin, cu=s.cu)
            return {"q": q, "codes": s.codes, "scales": s.scales}
        return _plain_append(s)
    if op == "attend":
        if own:
            return s.cache.attend(0, s.q, cu=s.cu)
        return _plain_attend(s)
    if op == "reorder":
        if own:
            s.cache.reorder(s.parents)
            return {"codes": s.codes, "scales": s.scales, "table": s.table, "refs": s.refs, "lens": s.lens}
        return _plain_reorder(s)
    if op == "compact":
        # a pool that was compacted is not fragmented any more: table and counts as they were
        s.table.copy_(s.table0)
        s.refs.copy_(s.refs0)
        if own:
            n = s.cache.compact()
        else:
            n = _plain_compact(s)
        return {"n": n, "codes": s.codes, "scales": s.scales, "table": s.table, "refs": s.refs}
    if own:
        scores, rows, tokens, done = s.ops.beam_select(s.logits, s.scores, s.case["beams"], done=s.done, eos=s.eos)
        return {"scores": scores, "rows": rows, "tokens": tokens, "done": done}
    return _plain_select(s)


# ---- in 64 bits ------------------------------------------------------------------------------------------
def _exact_append(s):
    c, page, hd = s.case, s.case["page"], s.case["hd"]
    codes, scales = s.codes.double(), s.scales.double()
    x = s.qkv.double().view(s.tokens, -1, hd)
    cos, sin = s.cos.double(), s.sin.double()
    q_all, k0 = [], 0
    for b, (past, t) in enumerate(zip(s.past, s.t)):
        cs, sn = cos[past:past + t, None], sin[past:past + t, None]
        mine = x[k0:k0 + t]
        k0 += t
        lo, hi = mine[..., :hd // 2], mine[..., hd // 2:]
        rot = torch.cat((lo * cs[..., :hd // 2] - hi * sn[..., :hd // 2], hi * cs[..., hd // 2:] + lo * sn[..., hd // 2:]), -1)
        q_all.append(rot[:, :c["nh"]])
        new = torch.stack((rot[:, c["nh"]:c["nh"] + c["nkv"]], mine[:, c["nh"] + c["nkv"]:]), 0).transpose(1, 2)
        for p in range(past // page, (past + t - 1) // page + 1):
            a, z = max(past, p * page), min(past + t, (p + 1) * page)
            pid, rows = int(s.table[b, p]), new[:, :, a - past:z - past]
            need = torch.ceil(torch.log2(rows.abs().amax((-1, -2)) / 448)).clamp(EXP_MIN, EXP_MAX)
            had = scales[0, pid].log2() if a > p * page else torch.full_like(need, EXP_MIN)
            e = torch.maximum(need, had)
            grown = codes[0, pid, :, :, :a - p * page] * torch.exp2(had - e)[..., None, None]
            codes[0, pid, :, :, :a - p * page] = grown.to(E4M3).double()
            codes[0, pid, :, :, a - p * page:z - p * page] = (rows * torch.exp2(-e)[..., None, None]).to(E4M3).double()
            scales[0, pid] = torch.exp2(e)
    return {"q": torch.cat(q_all), "codes": codes, "scales": scales}


def _exact_attend(s):
    c, k0, outs = s.case, 0, []
    group = c["nh"] // c["nkv"]
    for b, (past, t) in enumerate(zip(s.past, s.t)):
        n = past + t
        ids = s.table[b, :-(-n // c["page"])].long()
        kv = s.codes[0, ids].double() * s.scales[0, ids].double()[..., None, None]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(2, c["nkv"], -1, c["hd"])[:, :, :n]
        kv = kv.repeat_interleave(group, 1)
        q = s.q[k0:k0 + t].double().transpose(0, 1)
        k0 += t
        x = torch.einsum("htd,hkd->htk", q, kv[0]) / math.sqrt(c["hd"])
        hide = torch.ones((t, n), dtype=torch.bool, device="cuda").triu(past + 1)
        outs.append(torch.softmax(x.masked_fill(hide, -math.inf), -1).matmul(kv[1]).transpose(0, 1))
    return torch.cat(outs)


def exact(c, seed):
    if c["op"] in ("reorder", "compact"):
        return None                      # bytes moved and whole numbers: nothing is computed
    s = prepare(c, seed)
    if c["op"] == "append":
        return _exact_append(s)
    if c["op"] == "attend":
        return _exact_attend(s)
    scores = []
    for x, sc, done in zip(s.logits, s.scores.double(), s.done):
        logp = sc[:, None] + torch.log_softmax(x.double(), -1)
        only = torch.full_like(logp, -math.inf)
        only[:, s.eos] = sc
        scores.append(torch.topk(torch.where(done[:, None], only, logp).flatten(), c["beams"]).values)
    return {"scores": torch.stack(scores), "rows": None, "tokens": None, "done": None}

"""Cases of the paged 8-bit KV cache operators: attention over the cache, appending to it and reading it back, and the
page operations (reserve, fork, free, compact), each as one call of a user's program.

The cache (every case): codes int8 [n_pages][n_layers][2: K, V][n_kv][page_tokens * head_dim], the K tile of a page stored
[head_dim / 16][page_tokens][16 dims] and its V tile [page_tokens / 16][head_dim][16 tokens]; scales f32
[n_pages][n_layers][2][n_kv][page_tokens / 16], one for each block of 16 tokens and head; refs int32 [n_pages]; table int32
[max_seqs][max_pages] (-1: no page); lens int32 [max_seqs].

`own` false: the plain forms, elementary torch operations in 32 bits.  `own` true: quanta.cpp_b200's PagedKV.
"""
import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 16  # tokens that share a scale
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one chat session soon after its start: latency only
        dict(name="decode 1x130 f32", op="attention", dtype="f32", n=1, lo=130, hi=130, q_lo=1, q_hi=1, heads=14, kv=2,
             hd=64, page=64, window=0),
        # one step of the batched job: 256 sequences past their 512-token prompts
        dict(name="decode 256x640 f32", op="attention", dtype="f32", n=256, lo=512, hi=640, q_lo=1, q_hi=1, heads=14, kv=2,
             hd=64, page=64, window=0),
        # a serving batch of very different lengths, wide heads
        dict(name="decode ragged 192x8191 bf16", op="attention", dtype="bf16", n=192, lo=1, hi=8191, q_lo=1, q_hi=1, heads=32,
             kv=8, hd=128, page=64, window=0),
        # one very long document
        dict(name="decode 1x131071 f16", op="attention", dtype="f16", n=1, lo=131071, hi=131071, q_lo=1, q_hi=1, heads=14,
             kv=2, hd=64, page=64, window=0),
        # the first chunk of a prompt: 512 queries over themselves
        dict(name="chunk 512 f32", op="attention", dtype="f32", n=1, lo=512, hi=512, q_lo=512, q_hi=512, heads=14, kv=2,
             hd=64, page=64, window=0),
        # chunks of several long prompts and drafts to verify, with a sliding window
        dict(name="chunk ragged 6x8191 f16", op="attention", dtype="f16", n=6, lo=2111, hi=8191, q_lo=5, q_hi=509, heads=32,
             kv=8, hd=128, page=32, window=4096),
        # the new token of each of 256 sequences enters a block whose other tokens are there already
        dict(name="append 256x1 f32", op="append", dtype="f32", n=256, lo=512, hi=640, new_lo=1, new_hi=1, kv=2, hd=64,
             page=64),
        # whole prompts enter the cache
        dict(name="append ragged 32 prompts bf16", op="append", dtype="bf16", n=32, lo=97, hi=4093, new_lo=97, new_hi=4093,
             kv=8, hd=128, page=64),
        # 16 samples of each of 4 prompts: every child gets its own copy of the part-filled last page, in all layers
        dict(name="fork 4 to 64", op="fork", n=4, children=16, lo=77, hi=2019, layers=24, kv=2, hd=64, page=64,
             pages=512),
        # sequences ended here and there in a large pool: its live pages move together
        dict(name="compact 2048 pages", op="compact", n=128, live=1229, layers=24, kv=2, hd=64, page=64, pages=2048),
        # bookkeeping between two steps: some sequences end, others get room for their next tokens
        dict(name="recycle 64 of 256", op="recycle", n=256, ended=64, lo=300, hi=1500, extra_lo=1, extra_hi=97, kv=2,
             hd=64, page=16, pages=32768),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: any kind, sizes over the logarithm of their range."""
    op = rng.choice(["attention", "attention", "chunk", "append", "append", "fork", "compact", "recycle"])
    kv, group, hd = rng.choice([(2, 7, 64), (8, 4, 128), (1, 8, 64), (4, 1, 128), (2, 16, 64), (3, 3, 64)])
    dtype, page = rng.choice(list(TYPES)), rng.choice([16, 32, 64, 128])
    if op in ("attention", "chunk"):
        hi = _log(rng, 2, 65536)
        most = 180_000_000 // (kv * hd * hi)  # at most the tokens of the largest listed cases
        n = _log(rng, 1, max(1, min(256, most)))
        lo = rng.choice([hi, max(1, hi // 2), max(1, hi // 100)])
        q_hi = 1
        if op == "chunk":
            hi = min(hi, 8192)
            q_hi = _log(rng, 2, 512)
            lo, n = min(lo, hi), min(n, max(1, 4_000_000 // (q_hi * hi)))
        window = rng.choice([0, 0, _log(rng, 16, 4096)])
        return dict(op="attention", dtype=dtype, n=n, lo=lo, hi=hi, q_lo=max(1, q_hi // rng.choice([1, 7])), q_hi=q_hi,
                    heads=kv * group, kv=kv, hd=hd, page=page, window=window)
    if op == "append":
        if rng.random() < 0.5:
            hi = _log(rng, 20, 4096)
            new = _log(rng, 1, 4)
            return dict(op=op, dtype=dtype, n=_log(rng, 1, 256), lo=max(new, hi // 3), hi=hi, new_lo=1, new_hi=new, kv=kv,
                        hd=hd, page=page)
        hi = _log(rng, 16, 4096)
        lo = max(1, hi // rng.choice([1, 3, 40]))
        return dict(op=op, dtype=dtype, n=_log(rng, 1, 32), lo=lo, hi=hi, new_lo=lo, new_hi=hi, kv=kv, hd=hd, page=page)
    if op == "fork":
        n, children = _log(rng, 1, 8), _log(rng, 1, 16)
        hi = _log(rng, 16, 2048)
        return dict(op=op, n=n, children=children, lo=max(1, hi // 5), hi=hi, layers=rng.choice([2, 12, 24]), kv=2, hd=64,
                    page=rng.choice([32, 64]), pages=n * (hi // 32 + 1) + n * children + _log(rng, 1, 100))
    if op == "compact":
        pages = _log(rng, 64, 2048)
        return dict(op=op, n=_log(rng, 2, 128), live=max(2, int(pages * rng.uniform(0.2, 0.95))),
                    layers=rng.choice([2, 12, 24]), kv=2, hd=64, page=rng.choice([32, 64]), pages=pages)
    n = _log(rng, 4, 256)
    hi = _log(rng, 32, 1500)
    return dict(op="recycle", n=n, ended=max(1, n // rng.choice([2, 4])), lo=max(1, hi // 4), hi=hi, extra_lo=1,
                extra_hi=_log(rng, 1, 97), kv=2, hd=64, page=16, pages=n * (hi // 16 + 10) + _log(rng, 1, 4000))


def _spread(n, lo, hi, turn=0.6180339887498949):
    """n sizes over [lo, hi], spread over their logarithm, in no order; the same for every seed."""
    if n == 1:
        return [hi]
    return [max(lo, min(hi, int(round(lo * (hi / lo) ** ((i + 1) * turn % 1.0))))) for i in range(n)]


def _lens(case):
    lens = _spread(case["n"], case["lo"], case["hi"])
    if case["op"] == "attention":
        news = [min(a, b) for a, b in zip(_spread(case["n"], case["q_lo"], case["q_hi"], 0.7548776662466927), lens)]
    elif case["op"] == "append":
        whole = case["new_lo"] == case["lo"] and case["new_hi"] == case["hi"]
        news = lens if whole else [min(a, b) for a, b in zip(_spread(case["n"], case["new_lo"], case["new_hi"]), lens)]
    else:
        news = None
    return lens, news


def _visible(case):
    """Visible (query, key) pairs, and the keys that some query sees, summed over the sequences."""
    pairs = keys = 0
    lens, news = _lens(case)
    for n, m in zip(lens, news):
        w = case["window"] or n
        pairs += sum(min(p + 1, w) for p in range(n - m, n))
        keys += min(n, m + w - 1)
    return pairs, keys


def work(case):
    kv, hd = case["kv"], case["hd"]
    if case["op"] == "attention":
        pairs, keys = _visible(case)
        item, n_tok = TYPES[case["dtype"]].itemsize, sum(_lens(case)[1])
        return {"bytes": keys * 2 * kv * (hd + 4 / BLOCK) + n_tok * case["heads"] * (2 * hd * item + 4),
                "flops": 4.0 * pairs * case["heads"] * hd}
    if case["op"] == "append":
        lens, news = _lens(case)
        kept = sum((n - m) % BLOCK for n, m in zip(lens, news))
        item, n_tok = TYPES[case["dtype"]].itemsize, sum(news)
        # the new rows in, their codes out; the touched blocks' values read back
        return {"bytes": 2 * kv * hd * (n_tok * (item + 1) + kept * 2 + (n_tok + kept) * (1 + 4)), "flops": 0}
    page = case.get("layers", 1) * 2 * kv * case["page"] * (hd + 4 / BLOCK)
    if case["op"] == "fork":
        lens = _spread(case["n"], case["lo"], case["hi"])
        copied = sum(case["children"] for n in lens if n % case["page"])
        shared = sum(case["children"] * (n // case["page"]) for n in lens)
        return {"bytes": copied * page * 2 + shared * 8 + case["pages"] * 4, "flops": 0}
    if case["op"] == "compact":
        moved = case["live"] * (case["pages"] - case["live"]) / case["pages"]
        return {"bytes": moved * page * 2 + case["pages"] * 8 + case["live"] * 8, "flops": 0}
    return {"bytes": case["pages"] * 4 + case["n"] * (case["hi"] + case["lo"]) / 2 / case["page"] * 4, "flops": 0}


# ---------------------------------------------------------------- inputs

def _cache(case, lens, gen, pages=None, layers=1, max_seqs=None, extra=0):
    """A cache that holds sequences of these lengths in pages of random order, with its integers in one buffer."""
    dev, pt, hd, kv = "cuda", case["page"], case["hd"], case["kv"]
    need = [-(-n // pt) for n in lens]
    max_pages = max(need) + -(-extra // pt)
    pages = pages or sum(need) + 3
    max_seqs = max_seqs or len(lens)
    ints = torch.empty(pages + max_seqs * max_pages + max_seqs, dtype=torch.int32, device=dev)
    refs, table, lens_t = _views(ints, pages, max_seqs, max_pages)
    order = torch.randperm(pages, generator=gen, device=dev)[: sum(need)].to(torch.int32)
    refs.zero_()
    refs[order.long()] = 1
    table.fill_(-1)
    have = torch.zeros(max_seqs, dtype=torch.int64, device=dev)
    have[: len(need)] = torch.tensor(need, device=dev)
    table[torch.arange(max_pages, device=dev)[None] < have[:, None]] = order
    lens_t.zero_()
    lens_t[: len(lens)] = torch.tensor(lens, dtype=torch.int32, device=dev)
    # a block's largest value has code 127 or -127: about 3.3 deviations for values of a normal distribution
    shape = (pages, layers, 2, kv, pt * hd)
    codes = torch.empty(shape, dtype=torch.int8, device=dev)
    for p in range(0, pages, 256):  # in pieces: the normal numbers are four times the codes
        part = torch.randn((min(256, pages - p),) + shape[1:], generator=gen, device=dev)
        codes[p: p + 256] = (part * 38.0).round_().clamp_(-127, 127).to(torch.int8)
    scales = torch.exp(torch.randn(pages, layers, 2, kv, pt // BLOCK, generator=gen, device=dev) * 0.4) / 38.0
    return dict(codes=codes, scales=scales, ints=ints, refs=refs, table=table, lens=lens_t)


def _views(ints, pages, max_seqs, max_pages):
    return (ints[:pages], ints[pages: pages + max_seqs * max_pages].view(max_seqs, max_pages),
            ints[pages + max_seqs * max_pages:])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    op, state = case["op"], dict(case=case)
    if op in ("attention", "append"):
        lens, news = _lens(case)
        state |= _cache(case, lens, gen)
        dtype, n_tok = TYPES[case["dtype"]], sum(news)
        starts = [0]
        for m in news:
            starts.append(starts[-1] + m)
        perm = torch.randperm(case["n"], generator=gen, device="cuda")  # the call names the sequences in its own order
        starts_of = torch.tensor([0] + [news[i] for i in perm.tolist()], device="cuda").cumsum(0)
        state |= dict(seqs=perm.to(torch.int32), starts=starts_of.to(torch.int32), max_q=max(news), max_len=max(lens))
        if op == "attention":
            # sharper than the unit normal's scores, as trained heads are
            state["q"] = (torch.randn(n_tok, case["heads"], case["hd"], generator=gen, device="cuda") * 1.5).to(dtype)
        else:
            # k and v lie in the rows of one projection's output
            rows = torch.randn(n_tok, 2, case["kv"], case["hd"], generator=gen, device="cuda")
            rows = (rows * torch.exp(torch.randn(n_tok, 2, case["kv"], 1, generator=gen, device="cuda") * 0.3)).to(dtype)
            state["k"], state["v"] = rows[:, 0], rows[:, 1]
            # what is read back: from the start of the first touched block
            first = [(lens[i] - news[i]) // BLOCK * BLOCK for i in perm.tolist()]
            back = [0]
            for i, f in zip(perm.tolist(), first):
                back.append(back[-1] + lens[i] - f)
            state |= dict(first=_ints(first), back=_ints(back), n_back=back[-1])
    elif op == "fork":
        lens, n, c = _spread(case["n"], case["lo"], case["hi"]), case["n"], case["children"]
        state |= _cache(case, lens, gen, case["pages"], case["layers"], n + n * c)
        order = torch.randperm(n * c, generator=gen, device="cuda")
        state |= dict(src=(torch.arange(n * c, device="cuda") // c)[order].to(torch.int32), dst=(order + n).to(torch.int32))
    elif op == "compact":
        pt, n = case["page"], min(case["n"], case["live"])
        per = [case["live"] // n + (i < case["live"] % n) for i in range(n)]
        state |= _cache(case, [p * pt - (i * 7) % pt for i, p in enumerate(per)], gen, case["pages"], case["layers"])
    else:
        lens, n = _spread(case["n"], case["lo"], case["hi"]), case["n"]
        state |= _cache(case, lens, gen, case["pages"], extra=case["extra_hi"])
        order = torch.randperm(n, generator=gen, device="cuda").to(torch.int32)
        state |= dict(ended=order[: case["ended"]].contiguous(), grown=order[case["ended"]:].contiguous(),
                      extra=_ints(_spread(n - case["ended"], case["extra_lo"], case["extra_hi"])))
    state["scale"] = case["hd"] ** -0.5
    if "refs" in state and op in ("fork", "compact", "recycle"):
        state["before"] = state["ints"].clone()
    if own:  # the cache object that a program keeps
        state["kv"] = _package().PagedKV(state["codes"], state["scales"], state["refs"], state["table"], state["lens"])
    return state


def _package():
    at = str(Path(__file__).resolve().parent.parent / "quanta.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import quanta_b200
    return quanta_b200


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)(state, case, case["op"])


def _run_own(s, case, op):
    kv = s["kv"]
    if op == "attention":
        out, lse = kv.attention(0, s["q"], s["seqs"], s["starts"], s["max_q"], s["max_len"], scale=s["scale"],
                                window=case["window"], lse=True)
        return dict(out=out, lse=lse)
    if op == "append":
        kv.append(0, s["k"], s["v"], s["seqs"], s["starts"], s["max_q"])
        k, v = kv.read(0, s["seqs"], s["first"], s["back"], s["n_back"])
        return dict(k=k, v=v)
    s["ints"].copy_(s["before"])  # each pass starts from the same tables
    if op == "fork":
        kv.fork(s["src"], s["dst"])
        return dict(ints=s["ints"], codes=s["codes"], scales=s["scales"])
    if op == "compact":
        kv.compact()
        return dict(ints=s["ints"], codes=s["codes"], scales=s["scales"])
    kv.free(s["ended"])
    kv.reserve(s["grown"], s["extra"])
    return dict(ints=s["ints"])


def _run_plain(s, case, op):
    if op == "attention":
        return _plain_attention(s, case)
    if op == "append":
        return _plain_append(s, case)
    s["ints"].copy_(s["before"])
    if op == "fork":
        _plain_fork(s, case)
        return dict(ints=s["ints"], codes=s["codes"], scales=s["scales"])
    if op == "compact":
        _plain_compact(s, case)
        return dict(ints=s["ints"], codes=s["codes"], scales=s["scales"])
    _plain_free(s, case)
    _plain_reserve(s, case)
    return dict(ints=s["ints"])


# ---------------------------------------------------------------- plain forms

def _plain_values(s, case):
    """K and V of the called sequences in f32, [n][kv][max_pages * page][hd] (what lies past a sequence's end is not
    meaningful)."""
    pt, hd, kv = case["page"], case["hd"], case["kv"]
    pages = s["table"][s["seqs"].long()].clamp(min=0).long()
    n, mp = pages.shape
    codes, scales = s["codes"][pages, 0], s["scales"][pages, 0]  # [n][mp][2][kv][...]
    scales = scales.repeat_interleave(BLOCK, -1).movedim(1, 3).reshape(n, 2, kv, mp * pt, 1)
    k = codes[:, :, 0].view(n, mp, kv, hd // 16, pt, 16).permute(0, 2, 1, 4, 3, 5).reshape(n, kv, mp * pt, hd)
    v = codes[:, :, 1].view(n, mp, kv, pt // 16, hd, 16).permute(0, 2, 1, 3, 5, 4).reshape(n, kv, mp * pt, hd)
    return k.float() * scales[:, 0], v.float() * scales[:, 1]


def _plain_rows(s, n_tok):
    """Of each token of the call: its sequence's place in the call, its place among the sequence's tokens, its position."""
    starts = s["starts"].long()
    tok = torch.arange(n_tok, device="cuda")
    at = (tok[:, None] >= starts[None, 1:]).sum(1)
    i = tok - starts[at]
    return at, i, s["lens"][s["seqs"].long()].long()[at] - (starts[at + 1] - starts[at]) + i


def _plain_attention(s, case):
    q, kv, hd = s["q"], case["kv"], case["hd"]
    n_tok, heads, g = q.shape[0], q.shape[1], q.shape[1] // kv
    k, v = _plain_values(s, case)
    at, i, pos = _plain_rows(s, n_tok)
    n, m = k.shape[0], s["max_q"]
    rows = torch.zeros(n, m, heads, hd, device="cuda")
    rows[at, i] = q.float()
    where = torch.full((n, m), -1, dtype=torch.int64, device="cuda")
    where[at, i] = pos
    rows = rows.view(n, m, kv, g, hd).transpose(1, 2).reshape(n, kv, m * g, hd)
    sc = torch.matmul(rows, k.transpose(2, 3)).mul_(s["scale"]).view(n, kv, m, g, -1)
    j = torch.arange(k.shape[2], device="cuda")
    seen = j[None, None] <= where[:, :, None]
    if case["window"]:
        seen &= j[None, None] > where[:, :, None] - case["window"]
    sc.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(top.clamp(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((j[None] < s["lens"][s["seqs"].long()][:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(p.view(n, kv, m * g, -1), v).view(n, kv, m, g, hd) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    o = o.permute(0, 2, 1, 3, 4).reshape(n, m, heads, hd)[at, i]
    return dict(out=o.to(q.dtype), lse=lse.permute(0, 2, 1, 3).reshape(n, m, heads)[at, i])


def _plain_append(s, case):
    pt, hd, kv = case["page"], case["hd"], case["kv"]
    at, i, pos = _plain_rows(s, s["k"].shape[0])
    seqs = s["seqs"].long()
    x = torch.stack([s["k"], s["v"]], 1).float()  # [n_tok][2][kv][hd]
    page, off = s["table"][seqs[at], pos // pt].long(), pos % pt
    block = page * (pt // BLOCK) + off // BLOCK  # a number of its own for each block of the pool
    n_blocks = s["codes"].shape[0] * (pt // BLOCK)
    top = torch.zeros(n_blocks, 2, kv, device="cuda")
    top.scatter_reduce_(0, block[:, None, None].expand(-1, 2, kv), x.abs().amax(-1), "amax")
    touched = torch.zeros(n_blocks, dtype=torch.bool, device="cuda")
    touched[block] = True
    # tokens of a touched block that were there before: those below the call's first position
    p0 = pos - i
    kept = torch.zeros(n_blocks, dtype=torch.int64, device="cuda")
    kept[block] = (p0 - (pos - pos % BLOCK)).clamp(min=0)
    scales = s["scales"][:, 0].permute(0, 3, 1, 2).reshape(n_blocks, 2, kv)
    old = torch.where(kept[:, None, None] > 0, scales, 0.0)
    new = torch.where(touched[:, None, None], torch.maximum(old, top / 127.0), scales)
    s["scales"][:, 0] = new.view(-1, pt // BLOCK, 2, kv).permute(0, 2, 3, 1)
    # codes as [block][16 tokens][2][kv][hd]
    codes = s["codes"][:, 0]
    pages = codes.shape[0]
    k = codes[:, 0].view(pages, kv, hd // 16, pt, 16).permute(0, 3, 1, 2, 4).reshape(n_blocks, BLOCK, kv, hd)
    v = codes[:, 1].view(pages, kv, pt // 16, hd, 16).permute(0, 2, 4, 1, 3).reshape(n_blocks, BLOCK, kv, hd)
    b = touched.nonzero()[:, 0]
    both = torch.stack([k[b], v[b]], 2).float()  # [touched][16][2][kv][hd]
    ratio = old[b] / torch.where(new[b] > 0, new[b], 1.0)
    both = torch.where((torch.arange(BLOCK, device="cuda")[None] < kept[b][:, None])[:, :, None, None, None],
                       (both * ratio[:, None, :, :, None]).round(), both)
    place = torch.zeros(n_blocks, dtype=torch.int64, device="cuda")
    place[b] = torch.arange(b.numel(), device="cuda")
    inv = torch.where(new > 0, 1.0 / new, 0.0)[block]
    both[place[block], off % BLOCK] = (x * inv[..., None]).round().clamp(-127, 127)
    both = both.to(torch.int8)
    k[b], v[b] = both[:, :, 0], both[:, :, 1]
    codes[:, 0] = k.view(pages, pt, kv, hd // 16, 16).permute(0, 2, 3, 1, 4).reshape(pages, kv, pt * hd)
    codes[:, 1] = v.view(pages, pt // 16, 16, kv, hd).permute(0, 3, 1, 4, 2).reshape(pages, kv, pt * hd)
    # the touched blocks' values, from the first touched block of each sequence to its end
    row = torch.arange(s["n_back"], device="cuda")
    back = s["back"].long()
    a = (row[:, None] >= back[None, 1:]).sum(1)
    p = s["first"].long()[a] + row - back[a]
    blk = s["table"][seqs[a], p // pt].long() * (pt // BLOCK) + p % pt // BLOCK
    d = new[blk]
    return dict(k=k[blk, p % BLOCK].float() * d[:, 0, :, None], v=v[blk, p % BLOCK].float() * d[:, 1, :, None])


def _free_pages(refs):
    """Page numbers, the free ones first and ascending."""
    return torch.argsort((refs > 0).to(torch.int32), stable=True)


def _plain_fork(s, case):
    pt = case["page"]
    src, dst = s["src"].long(), s["dst"].long()
    lens, row = s["lens"][src].long(), s["table"][src].clone()
    part = lens % pt > 0
    at = lens // pt
    fresh = _free_pages(s["refs"])[(part.long().cumsum(0) - 1).clamp(min=0)]
    one = part.nonzero()[:, 0]
    old = row[one, at[one]].long()
    row[one, at[one]] = fresh[one].to(torch.int32)
    s["table"][dst], s["lens"][dst] = row, lens.to(torch.int32)
    used = row[row >= 0].long()
    s["refs"].index_add_(0, used, torch.ones_like(used, dtype=torch.int32))
    s["codes"][fresh[one]], s["scales"][fresh[one]] = s["codes"][old], s["scales"][old]


def _plain_compact(s, case):
    refs = s["refs"]
    n = refs.numel()
    idx = torch.arange(n, device="cuda")
    live = refs > 0
    n_live = int(live.sum())
    src, dst = (live & (idx >= n_live)).nonzero()[:, 0], (~live & (idx < n_live)).nonzero()[:, 0]
    to = idx.clone()
    to[src] = dst
    s["codes"][dst], s["scales"][dst] = s["codes"][src], s["scales"][src]
    refs[dst], refs[src] = refs[src], 0
    t = s["table"]
    t.copy_(torch.where(t >= 0, to[t.clamp(min=0).long()].to(torch.int32), t))


def _plain_free(s, case):
    e = s["ended"].long()
    row = s["table"][e]
    used = row[row >= 0].long()
    s["refs"].index_add_(0, used, torch.full_like(used, -1, dtype=torch.int32))
    s["table"][e], s["lens"][e] = -1, 0


def _plain_reserve(s, case):
    pt, g = case["page"], s["grown"].long()
    lens = s["lens"][g].long()
    have, want = -(-lens // pt), -(-(lens + s["extra"].long()) // pt)
    need = want - have
    base = need.cumsum(0) - need
    k = torch.arange(s["table"].shape[1], device="cuda")[None] - have[:, None]  # which of the row's new pages
    new = (k >= 0) & (k < need[:, None])
    order = _free_pages(s["refs"])
    row = s["table"][g]
    page = order[torch.where(new, base[:, None] + k, 0)]
    s["table"][g] = torch.where(new, page.to(torch.int32), row)
    s["refs"][page[new]] = 1
    s["lens"][g] = (lens + s["extra"].long()).to(torch.int32)


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    if case["op"] not in ("attention", "append"):
        return None  # whole numbers and moved bytes only
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return (_exact_attention if case["op"] == "attention" else _exact_append)(s, case)


def _exact_sequence(s, case, seq):
    """K and V of one sequence as [kv][len][hd] in f64, token by token of the layout."""
    pt, hd, kv = case["page"], case["hd"], case["kv"]
    p = torch.arange(int(s["lens"][seq]), device="cuda")
    page, t = s["table"][seq].long()[p // pt], p % pt
    d = torch.arange(hd, device="cuda")
    k_at = (d // 16)[None] * (pt * 16) + t[:, None] * 16 + (d % 16)[None]
    v_at = (t // 16)[:, None] * (hd * 16) + d[None] * 16 + (t % 16)[:, None]
    got = []
    for w, idx in ((0, k_at), (1, v_at)):
        tile = s["codes"][:, 0, w][page]  # [len][kv][pt * hd]
        c = torch.gather(tile, 2, idx[:, None].expand(-1, kv, -1)).double()
        got.append((c * s["scales"][:, 0, w][page, :, t // BLOCK].double()[..., None]).transpose(0, 1))
    return got


def _exact_attention(s, case):
    kv, g = case["kv"], case["heads"] // case["kv"]
    starts, outs, lses = s["starts"].tolist(), [], []
    for a, seq in enumerate(s["seqs"].tolist()):
        n = int(s["lens"][seq])
        q = s["q"][starts[a]: starts[a + 1]].double()
        m = q.shape[0]
        k, v = _exact_long(s, case, seq, 1 << 14)
        sc = torch.einsum("mhgd,hjd->hmgj", q.view(m, kv, g, -1), k) * s["scale"]
        pos, j = torch.arange(n - m, n, device="cuda"), torch.arange(n, device="cuda")
        seen = j[None] <= pos[:, None]
        if case["window"]:
            seen &= j[None] > pos[:, None] - case["window"]
        sc = sc.masked_fill(~seen[None, :, None], -math.inf)
        lses.append(torch.logsumexp(sc, -1).transpose(0, 1).reshape(m, -1))
        outs.append(torch.einsum("hmgj,hjd->mhgd", torch.softmax(sc, -1), v).reshape(m, kv * g, -1))
    return dict(out=torch.cat(outs), lse=torch.cat(lses))


def _exact_long(s, case, seq, step):
    """_exact_sequence in stretches, so that the gathered tiles stay small."""
    pt, n = case["page"], int(s["lens"][seq])
    ks, vs = [], []
    for b in range(0, n, step):  # step is a multiple of every page size
        row = s["table"][seq][b // pt: -(-min(n, b + step) // pt)]
        one = dict(s, table=row[None], lens=torch.tensor([min(n, b + step) - b]))
        k, v = _exact_sequence(one, case, 0)
        ks.append(k)
        vs.append(v)
    return torch.cat(ks, 1), torch.cat(vs, 1)


def _exact_append(s, case):
    kv, hd = case["kv"], case["hd"]
    starts, first = s["starts"].tolist(), s["first"].tolist()
    lens = s["lens"].tolist()
    out = {"k": [], "v": []}
    for a, seq in enumerate(s["seqs"].tolist()):
        n, m, f = lens[seq], starts[a + 1] - starts[a], first[a]
        kept = n - m - f
        old_k, old_v = _exact_tail(s, case, seq, f, n - m)
        for name, x, before, w in (("k", s["k"], old_k, 0), ("v", s["v"], old_v, 1)):
            new = x[starts[a]: starts[a + 1]].double()  # [m][kv][hd]
            pad = (-(kept + m)) % BLOCK
            rows = torch.cat([torch.zeros(kept, kv, hd, dtype=torch.float64, device="cuda"), new,
                              torch.zeros(pad, kv, hd, dtype=torch.float64, device="cuda")]).view(-1, BLOCK, kv, hd)
            d = rows.abs().amax((1, 3)) / 127  # [blocks][kv]
            vals = torch.zeros_like(rows)
            if kept:
                scale0, codes0 = before
                d[0] = torch.maximum(d[0], scale0)
                vals[0, :kept] = torch.round(codes0 * (scale0 / d[0])[None, :, None]) * d[0][None, :, None]
            q = torch.round(rows / torch.where(d > 0, d, 1.0)[:, None, :, None]) * d[:, None, :, None]
            vals = vals.view(-1, kv, hd)
            vals[kept: kept + m] = q.view(-1, kv, hd)[kept: kept + m]
            out[name].append(vals[: kept + m])
    return dict(k=torch.cat(out["k"]), v=torch.cat(out["v"]))


def _exact_tail(s, case, seq, f, end):
    """(scale [kv], codes [end - f][kv][hd]) of the block that starts at f, for K and V, before the call; None if empty."""
    if end == f:
        return None, None
    pt, hd, kv = case["page"], case["hd"], case["kv"]
    page, t0 = int(s["table"][seq][f // pt]), f % pt
    tile, sc = s["codes"][page, 0].double(), s["scales"][page, 0].double()
    k = tile[0].view(kv, hd // 16, pt, 16)[:, :, t0: t0 + end - f].permute(2, 0, 1, 3).reshape(end - f, kv, hd)
    v = tile[1].view(kv, pt // 16, hd, 16)[:, t0 // 16, :, : end - f].permute(2, 0, 1)
    return (sc[0, :, t0 // BLOCK], k), (sc[1, :, t0 // BLOCK], v)

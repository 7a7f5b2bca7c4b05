"""Cases of the operators around a decoder layer and around a beam search: RMS norm with the residual's addition and 8-bit rows
out, rotary positions, the selection of a beam search's next step, and the reordering of the paged cache's sequences.

8-bit rows (every norm case): codes int8 [tokens, n] and a f32 scale for each 32 consecutive values, value = code * scale, the
operand of the quantized matrix products.  The cache (reorder cases): codes int8 [n_pages][n_layers][2: K, V][n_kv]
[page_tokens * head_dim], the K tile of a page stored [head_dim / 16][page_tokens][16 dims] and its V tile [page_tokens / 16]
[head_dim][16 tokens]; scales f32 [n_pages][n_layers][2][n_kv][page_tokens / 16]; refs int32 [n_pages]; table int32 [max_seqs]
[max_pages] (-1: no page); lens int32 [max_seqs].

`own` false: the plain forms, elementary torch operations in 32 bits (angles and candidates' scores in 64: far positions and
candidates next to each other need them).  `own` true: quanta.cpp_b200's operators.
"""
import functools
import math
import sys
from pathlib import Path

import torch

own = False

QK = 32     # values that share a scale in 8-bit rows
BLOCK = 16  # tokens that share a scale in the cache
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a layer's norm for the one new token of a chat session: latency only
        dict(name="norm 1x896 f32", op="norm", dtype="f32", tokens=1, n=896, residual="f32", pad=0),
        # the same for one step of 256 sequences
        dict(name="norm 256x896 f32", op="norm", dtype="f32", tokens=256, n=896, residual="f32", pad=0),
        # a chunk of a long prompt in a wide model, 16-bit residual stream
        dict(name="norm 8192x4096 bf16", op="norm", dtype="bf16", tokens=8192, n=4096, residual="same", pad=0),
        # rows inside a wider buffer, no residual (a norm before the head), an odd number of them
        dict(name="norm 1021x4864 f16 in rows", op="norm", dtype="f16", tokens=1021, n=4864, residual="none", pad=40),
        # the new token's query and key heads
        dict(name="rope 1 f32", op="rope", dtype="f32", tokens=1, heads=14, kv=2, hd=64, rot=64, far=4096, layout="half",
             scaling="none"),
        # prompts packed one behind the other, wide heads, a context stretched 8 times
        dict(name="rope 8192 bf16 stretched", op="rope", dtype="bf16", tokens=8192, heads=32, kv=8, hd=128, rot=128,
             far=32768, layout="half", scaling="yarn"),
        # pairs side by side, a quarter of the head rotated, far positions
        dict(name="rope 3001 f16 interleaved part", op="rope", dtype="f16", tokens=3001, heads=16, kv=4, hd=128, rot=32,
             far=1000000, layout="interleaved", scaling="none"),
        # one request's four beams: the head's logits of the tokenizer's ids within the padded vocabulary
        dict(name="beams 1x4x151665 f32", op="beams", dtype="f32", groups=1, beams=4, vocab=151665, pad=271, k=4, ended=0.0,
             banned=0.0),
        # 64 requests, twice as many candidates as beams (some of them will be ends)
        dict(name="beams 64x4x151936 bf16", op="beams", dtype="bf16", groups=64, beams=4, vocab=151936, pad=0, k=8, ended=0.0,
             banned=0.0),
        # an odd vocabulary in rows of its own length, beams that have ended, tokens that a grammar forbids
        dict(name="beams 13x10x50257 f16", op="beams", dtype="f16", groups=13, beams=10, vocab=50257, pad=0, k=20, ended=0.3,
             banned=0.5),
        # one request: 4 beams behind a prompt of 500 tokens
        dict(name="reorder 1x4", op="reorder", groups=1, beams=4, lo=530, hi=530, prompt=500, layers=24, kv=2, hd=64, page=64),
        # 64 requests of very different prompts
        dict(name="reorder 64x4 ragged", op="reorder", groups=64, beams=4, lo=77, hi=2019, prompt=0, layers=24, kv=2, hd=64,
             page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: any operator, sizes over the logarithm of their range."""
    op, dtype = rng.choice(["norm", "rope", "beams", "reorder"]), rng.choice(list(TYPES))
    if op == "norm":
        n = 32 * _log(rng, 1, 512)
        return dict(op=op, dtype=dtype, tokens=_log(rng, 1, min(16384, 16_000_000 // n)), n=n,
                    residual=rng.choice(["none", "same", "f32"]), pad=rng.choice([0, 0, 32, 5]))
    if op == "rope":
        kv, group, hd = rng.choice([(2, 7, 64), (8, 4, 128), (1, 8, 64), (4, 1, 96), (3, 3, 80), (1, 16, 256)])
        return dict(op=op, dtype=dtype, tokens=_log(rng, 1, 20_000_000 // (kv * (group + 1) * hd)), heads=kv * group, kv=kv, hd=hd,
                    rot=rng.choice([hd, hd, hd // 2, hd // 4]), far=_log(rng, 100, 1_000_000),
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]))
    if op == "beams":
        beams, vocab = _log(rng, 1, 16), _log(rng, 100, 200_000)
        groups = _log(rng, 1, max(1, min(64, 16_000_000 // (beams * vocab))))
        return dict(op=op, dtype=dtype, groups=groups, beams=beams, vocab=vocab, pad=rng.choice([0, 0, 1, 64]),
                    k=min(vocab, rng.choice([beams, 2 * beams, _log(rng, 1, 64)])), ended=rng.choice([0.0, 0.0, 0.4]),
                    banned=rng.choice([0.0, 0.0, 0.5, 0.99]))
    groups, beams, hi = _log(rng, 1, 48), _log(rng, 2, 8), _log(rng, 16, 2019)
    return dict(op=op, groups=groups, beams=min(beams, max(2, 192 // groups)), lo=max(2, hi // rng.choice([1, 5, 25])), hi=hi,
                prompt=0, layers=rng.choice([2, 12, 24]), kv=2, hd=64, page=rng.choice([16, 32, 64]))


def _spread(n, lo, hi, turn=0.6180339887498949):
    """n sizes over [lo, hi], spread over their logarithm, in no order; the same for every seed."""
    if n == 1:
        return [hi]
    return [max(lo, min(hi, int(round(lo * (hi / lo) ** ((i + 1) * turn % 1.0))))) for i in range(n)]


def _beam_lens(case):
    """Length of each group's beams, and of the prompt that they share (half of it where the case says nothing)."""
    lens = _spread(case["groups"], case["lo"], case["hi"])
    return lens, [min(case["prompt"] or n // 2 + 1, n) for n in lens]


def work(case):
    op = case["op"]
    if op == "norm":
        item, m = TYPES[case["dtype"]].itemsize, case["tokens"] * case["n"]
        res = {"none": 0, "same": item, "f32": 4}[case["residual"]]
        # x and the residual in, the residual, codes and scales out; codes and scales in, their values out
        return {"bytes": m * (item + 2 * res + 2 * (1 + 4 / QK) + 2) + 4 * case["n"], "flops": 6 * m}
    if op == "rope":
        rows = case["tokens"] * (case["heads"] + case["kv"])
        return {"bytes": rows * case["hd"] * 2 * TYPES[case["dtype"]].itemsize + case["tokens"] * 4, "flops": 3 * rows * case["rot"]}
    if op == "beams":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * TYPES[case["dtype"]].itemsize + 5) + case["groups"] * case["k"] * 12,
                "flops": 4 * rows * case["vocab"]}
    # filled blocks of the part-filled pages, for the beams but one of each parent (about half of uniformly drawn ones share)
    lens, _ = _beam_lens(case)
    block = case["layers"] * 2 * case["kv"] * (BLOCK * case["hd"] + 4)
    copies = case["beams"] - case["beams"] * (1 - (1 - 1 / case["beams"]) ** case["beams"])
    blocks = sum(-(-(n % case["page"]) // BLOCK) for n in lens)
    rows = case["beams"] * sum(-(-n // case["page"]) for n in lens)
    return {"bytes": copies * blocks * block * 2 + rows * 8 + _pages(case) * 4, "flops": 0}


def _pages(case):
    lens, prompts = _beam_lens(case)
    pt = case["page"]
    return sum(p // pt + case["beams"] * (-(-n // pt) - p // pt) for n, p in zip(lens, prompts)) + case["groups"] * case["beams"] + 5


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 29)
    return {"norm": _norm_inputs, "rope": _rope_inputs, "beams": _beam_inputs, "reorder": _cache_inputs}[case["op"]](case, gen)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _norm_inputs(case, gen):
    m, n, dtype = case["tokens"], case["n"], TYPES[case["dtype"]]
    s = dict(case=case, eps=1e-6, weight=1 + 0.3 * _normal(gen, n))
    s["x"] = _normal(gen, m, n + case["pad"]).to(dtype)[:, :n]
    if case["residual"] != "none":  # a residual stream has a few dimensions much larger than the others
        r = _normal(gen, m, n) * torch.exp(_normal(gen, n)) * 2
        s["residual"] = r.to(dtype if case["residual"] == "same" else torch.float32)
    s["values"] = torch.float16 if case["dtype"] == "f16" else torch.bfloat16
    return s


SCALINGS = {
    "none": None,
    "linear": dict(kind="linear", factor=4.0),
    "ntk": dict(kind="ntk", factor=8.0),
    "yarn": dict(kind="yarn", factor=8.0, original=4096, beta_fast=32.0, beta_slow=1.0),
    "bands": dict(kind="bands", factor=8.0, original=8192, low=1.0, high=4.0),
}
BASE = 1e6


def _rope_inputs(case, gen):
    m, hd, dtype = case["tokens"], case["hd"], TYPES[case["dtype"]]
    heads, kv = case["heads"], case["kv"]
    # query, key and value heads lie in the rows of one projection's output
    rows = _normal(gen, m, heads + 2 * kv, hd).to(dtype)
    # packed sequences: each of them a stretch of consecutive positions that starts anywhere
    n = max(1, m // 700)
    first = torch.randint(0, max(1, case["far"] - m // n), (n,), generator=gen, device="cuda")
    tok = torch.arange(m, device="cuda")
    pos = (first[tok * n // m] + tok - (tok * n // m * m + n - 1) // n).to(torch.int32)
    s = dict(case=case, q=rows[:, :heads], k=rows[:, heads: heads + kv], positions=pos)
    # the table of frequencies that a program keeps
    f, scale = _frequencies(case)
    s["plain_table"] = (torch.tensor(f, dtype=torch.float64, device="cuda"), scale)
    if own:
        s["rope"] = _package().Rope(case["rot"], base=BASE, interleaved=case["layout"] == "interleaved",
                                    scaling=SCALINGS[case["scaling"]])
    return s


def _frequencies(case):
    """Radians a position of each pair, and the factor on rotated values, in 64 bits."""
    rot, sc = case["rot"], SCALINGS[case["scaling"]] or dict(kind="none")
    base, factor = BASE, sc.get("factor", 1.0)
    if sc["kind"] == "ntk" and rot > 2:
        base *= factor ** (rot / (rot - 2))
    f = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if sc["kind"] == "linear":
        return [x / factor for x in f], 1.0
    if sc["kind"] == "yarn":  # pairs that turn often stay, pairs that hardly turn are stretched, a ramp between them
        at = [rot * math.log(sc["original"] / (2 * math.pi * b)) / (2 * math.log(base)) for b in (sc["beta_fast"], sc["beta_slow"])]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        keep = [1 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(rot // 2)]
        return [x * k + x / factor * (1 - k) for x, k in zip(f, keep)], 0.1 * math.log(factor) + 1
    if sc["kind"] == "bands":  # by how often a pair turns within the original context
        turns = [sc["original"] * x / (2 * math.pi) for x in f]
        keep = [min(1.0, max(0.0, (t - sc["low"]) / (sc["high"] - sc["low"]))) for t in turns]
        return [x * k + x / factor * (1 - k) for x, k in zip(f, keep)], 1.0
    return f, 1.0


def _beam_inputs(case, gen):
    g, b, v, dtype = case["groups"], case["beams"], case["vocab"], TYPES[case["dtype"]]
    x = _normal(gen, g, b, v + case["pad"]) * 2.0
    # some tokens that the beams of a request favour together, by amounts of their own
    n = min(v, 40)
    at = torch.randint(0, v, (g, 1, n), generator=gen, device="cuda").expand(g, b, n)
    x.scatter_add_(2, at, 4.0 - 2.5 * torch.log(torch.rand(g, b, n, generator=gen, device="cuda")))
    x = x.to(dtype)
    if case["banned"]:
        x.masked_fill_(torch.rand(g, 1, v + case["pad"], generator=gen, device="cuda") < case["banned"], -math.inf)
    s = dict(case=case, logits=x[:, :, :v], scores=-(torch.rand(g, b, generator=gen, device="cuda") * 4 + 9))
    s["ended"] = (torch.rand(g, b, generator=gen, device="cuda") < case["ended"]).to(torch.uint8) if case["ended"] else None
    s["end_id"] = v // 3
    if own:
        s["select"] = _package().BeamSelector(case["k"], end_id=s["end_id"])
    return s


def _views(ints, pages, max_seqs, max_pages):
    return (ints[:pages], ints[pages: pages + max_seqs * max_pages].view(max_seqs, max_pages),
            ints[pages + max_seqs * max_pages:])


def _cache_inputs(case, gen):
    """Groups of beams whose rows of the page table share their prompt's full pages; the others are each beam's own."""
    dev, pt, g, b = "cuda", case["page"], case["groups"], case["beams"]
    lens, prompts = _beam_lens(case)
    pages, max_pages = _pages(case), -(-max(lens) // pt) + 1
    ints = torch.empty(pages + g * b * max_pages + g * b, dtype=torch.int32, device=dev)
    refs, table, lens_t = _views(ints, pages, g * b, max_pages)
    order = torch.randperm(pages, generator=gen, device=dev).tolist()
    rows, counts, at = [], [0] * pages, 0
    for n, p in zip(lens, prompts):
        shared = order[at: at + p // pt]
        at += p // pt
        for _ in range(b):
            mine = order[at: at + -(-n // pt) - p // pt]
            at += len(mine)
            rows.append(shared + mine + [-1] * (max_pages - len(shared) - len(mine)))
            for page in shared + mine:
                counts[page] += 1
    refs.copy_(torch.tensor(counts, dtype=torch.int32))
    seqs = torch.randperm(g * b, generator=gen, device=dev)  # which rows of the table the beams have
    table[seqs] = torch.tensor(rows, dtype=torch.int32, device=dev)
    lens_t[seqs] = torch.tensor([n for n in lens for _ in range(b)], dtype=torch.int32, device=dev)
    shape = (pages, case["layers"], 2, case["kv"], pt * case["hd"])
    codes = torch.randint(-127, 128, shape, generator=gen, device=dev, dtype=torch.int8)
    scales = torch.exp(_normal(gen, *shape[:4], pt // BLOCK) * 0.4) / 38.0
    # better beams have more children
    parents = (torch.rand(g, b, generator=gen, device=dev) ** 1.5 * b).to(torch.int32).clamp_(max=b - 1)
    s = dict(case=case, codes=codes, scales=scales, ints=ints, refs=refs, table=table, lens=lens_t, before=ints.clone(),
             seqs=seqs.to(torch.int32), parents=parents)
    if own:  # the cache object that a program keeps
        s["kv"] = _package().PagedKV(codes, scales, refs, table, lens_t)
    return s


@functools.cache
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
    if op == "norm":
        qb = _package()
        q, d = qb.rms_norm_q8(s["x"], s["weight"], s["eps"], residual=s.get("residual"))
        return dict(values=qb.dequantize_q8(q, d, s["values"]), scales=d, residual=s.get("residual"))
    if op == "rope":
        q, k = s["rope"](s["q"], s["k"], s["positions"])
        return dict(q=q, k=k)
    if op == "beams":
        scores, tokens, parents = s["select"](s["logits"], s["scores"], s["ended"])
        return dict(scores=scores, tokens=tokens, parents=parents)
    s["ints"].copy_(s["before"])  # each pass starts from the same tables
    s["kv"].reorder(s["seqs"], s["parents"], case["beams"])
    return dict(ints=s["ints"], codes=s["codes"], scales=s["scales"])


def _run_plain(s, case, op):
    if op == "reorder":
        s["ints"].copy_(s["before"])
    return {"norm": _plain_norm, "rope": _plain_rope, "beams": _plain_beams, "reorder": _plain_reorder}[op](s, case)


# ---------------------------------------------------------------- plain forms

def _plain_norm(s, case):
    h = s["x"].float()
    r = s.get("residual")
    if r is not None:
        h = h + r.float()
        r.copy_(h)
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + s["eps"]) * s["weight"]
    y = y.view(y.shape[0], -1, QK)
    d = y.abs().amax(-1) / 127
    t = y * torch.where(d > 0, 1 / d, 0.0)[..., None]
    q = torch.copysign((t.abs() + 0.5).floor(), t).to(torch.int8)  # halves away from zero
    return dict(values=(q.float() * d[..., None]).to(s["values"]).view(s["x"].shape), scales=d, residual=r)


def _plain_rope(s, case):
    f, scale = s["plain_table"]
    angle = s["positions"].double()[:, None] * f
    cos, sin = (angle.cos() * scale).float()[:, None], (angle.sin() * scale).float()[:, None]
    return dict(q=_plain_rotate(s["q"], cos, sin, case), k=_plain_rotate(s["k"], cos, sin, case))


def _plain_rotate(x, cos, sin, case):
    rot = case["rot"]
    y = x.float()
    if case["layout"] == "half":
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _plain_beams(s, case):
    x = s["logits"].double()
    g, b, v = x.shape
    top = x.amax(-1, keepdim=True)
    cand = x - (top + (x - top).exp().sum(-1, keepdim=True).log()) + s["scores"].double()[..., None]
    cand = torch.where(cand.isnan(), -math.inf, cand)
    if s["ended"] is not None:  # one candidate: itself
        itself = torch.full((v,), -math.inf, dtype=torch.float64, device="cuda")
        itself[s["end_id"]] = 0.0
        cand = torch.where(s["ended"][..., None] > 0, itself + s["scores"].double()[..., None], cand)
    cand = cand.view(g, b * v)
    k = case["k"]
    least = cand.topk(k).values[:, -1:]
    over, even = cand > least, cand == least
    keep = over | (even & (even.cumsum(-1) <= k - over.sum(-1, keepdim=True)))  # of even ones those of the lowest index
    at = keep.nonzero()[:, 1].view(g, k)
    best, order = cand.gather(1, at).sort(dim=-1, descending=True, stable=True)
    at = at.gather(1, order)
    return dict(scores=best.float(), tokens=(at % v).to(torch.int32), parents=(at // v).to(torch.int32))


def _plain_reorder(s, case):
    pt, b, hd, kv = case["page"], case["beams"], case["hd"], case["kv"]
    seqs, parents = s["seqs"].long(), s["parents"].long().view(-1)
    n = seqs.numel()
    i = torch.arange(n, device="cuda")
    parent = i - i % b + parents  # its place in the list
    rows, lens, old = s["table"][seqs][parent], s["lens"][seqs].long()[parent], s["table"][seqs]
    # one child takes over its parent's part-filled page (the parent itself if it goes on, else the first), the others get copies
    first = torch.full((n,), n, device="cuda").scatter_reduce_(0, parent, i, "amin")
    heir = torch.where(parent == i, i, first)
    copy = ((lens % pt > 0) & (heir[parent] != i)).nonzero()[:, 0]
    at = lens // pt
    src = rows[copy, at[copy]].long()
    rows[copy, at[copy]] = -1
    refs = s["refs"]
    for t, by in ((old, -1), (rows, 1)):
        used = t[t >= 0].long()
        refs.index_add_(0, used, torch.full_like(used, by, dtype=torch.int32))
    dst = torch.argsort((refs > 0).to(torch.int32), stable=True)[: copy.numel()]  # free pages, the lowest first
    refs[dst] = 1
    rows[copy, at[copy]] = dst.to(torch.int32)
    s["table"][seqs], s["lens"][seqs] = rows, lens.to(torch.int32)
    # the filled blocks of the copied pages, in all layers
    m, layers = copy.numel(), case["layers"]
    fill = torch.arange(pt // BLOCK, device="cuda")[None] * BLOCK < (lens[copy] % pt)[:, None]  # [copies][blocks]
    both = torch.stack([s["codes"][src], s["codes"][dst]])
    k = both[:, :, :, 0].view(2, m, layers, kv, hd // 16, pt // BLOCK, BLOCK * 16)
    v = both[:, :, :, 1].view(2, m, layers, kv, pt // BLOCK, hd * BLOCK)
    k = torch.where(fill[:, None, None, None, :, None], k[0], k[1]).view(m, layers, kv, pt * hd)
    v = torch.where(fill[:, None, None, :, None], v[0], v[1]).view(m, layers, kv, pt * hd)
    s["codes"][dst] = torch.stack([k, v], 2)
    s["scales"][dst] = torch.where(fill[:, None, None, None], s["scales"][src], s["scales"][dst])
    return dict(ints=s["ints"], codes=s["codes"], scales=s["scales"])


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    if case["op"] == "reorder":
        return None  # whole numbers and moved bytes only
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "beams": _exact_beams}[case["op"]](s, case)


def _exact_norm(s, case):
    values, scales, sums = [], [], []
    for at in range(0, case["tokens"], 1024):  # in pieces: 64-bit rows are large
        x = s["x"][at: at + 1024].double()
        if "residual" in s:
            x += s["residual"][at: at + 1024].double()
            sums.append(x.clone())
        x /= (x.square().sum(1) / x.shape[1] + s["eps"]).sqrt()[:, None]
        x *= s["weight"].double()
        blocks = x.unflatten(1, (-1, QK))
        peak = blocks.abs().max(-1).values
        step = torch.where(peak > 0, peak, 1.0)[..., None] / 127
        t = blocks / step
        codes = torch.where(t < 0, (t - 0.5).ceil(), (t + 0.5).floor())
        values.append((codes * step * (peak > 0)[..., None]).flatten(1))
        scales.append(peak / 127)
    return dict(values=torch.cat(values), scales=torch.cat(scales), residual=torch.cat(sums) if sums else None)


def _exact_rope(s, case):
    # complex numbers: a pair is a + ib, and it is multiplied by m * exp(i p f)
    f, scale = _frequencies(case)
    turn = torch.polar(torch.full((case["tokens"], len(f)), scale, dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda"))
    out = {}
    for name in ("q", "k"):
        x, h = s[name].double().clone(), case["rot"] // 2
        lo, hi = (slice(0, h), slice(h, 2 * h)) if case["layout"] == "half" else (slice(0, 2 * h, 2), slice(1, 2 * h, 2))
        z = torch.complex(x[..., lo], x[..., hi]) * turn[:, None]
        x[..., lo], x[..., hi] = z.real, z.imag
        out[name] = x
    return out


def _exact_beams(s, case):
    """Beam by beam: the k best of each (stable sort of its logits), then the k best of a group's."""
    g, b, v = s["logits"].shape
    k, rows = case["k"], []
    for j in range(g):
        found = []
        for i in range(b):
            score = s["scores"][j, i].double()
            if s["ended"] is not None and bool(s["ended"][j, i]):
                found.append(score[None])
                continue
            x = s["logits"][j, i].double()
            best = x.sort(descending=True).values[:k]
            found.append(score + best - torch.logsumexp(x, 0))
        best = torch.cat(found).nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).sort(descending=True).values[:k]
        rows.append(torch.cat([best, torch.full((k - best.numel(),), -math.inf, dtype=torch.float64, device="cuda")]))
    return dict(scores=torch.stack(rows), tokens=None, parents=None)

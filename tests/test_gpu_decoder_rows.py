"""RMS norm to 8-bit rows, values of 8-bit rows and rotary positions on the GPU, against their definitions in 64 bits.

Bounds, with u = 2^-24 (half a step of f32):
  norm: h is rounded once; a row's sum of squares passes at most 8 R + 12 additions (R chunks of 8 a thread, R <= 4; then 5 steps in
  a warp and 5 over warps), its root halves that error; the root, two products and the division by 127 add 4 u.  A scale is off by
  at most (44 / 2 + 1 + 4) u < 32 u.  A code is round(y / d) with y / d off by at most 127 * 32 u < 3e-4, so a value is within
  (0.5 + 3e-4) d of y, and the code of the block's largest value is 127.
  rope: the fraction of a revolution is rounded to f32 (an angle off by 2 pi 2^-26), sincospif by 2 u, so cos and sin are within
  6e-7 of theirs (positions to 2^20; at 2^31 the f64 count adds 2 pi 2^31 2^-52 / 6.3 < 5e-7); the products and the sum add 3 u.
  |out - exact| <= 1.2e-6 (|a| + |b|) scale + r |exact|, r = eps / 2 of the type, + 2^-25 for f16 (subnormal results).
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def rows(m, n, name, seed=0, pad=0, lead=0, std=1.0):
    """Rows [m, n] inside wider ones, starting `lead` elements into the buffer."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(m * (n + pad) + lead, generator=g, device="cuda") * std).to(TYPES[name])
    return x[lead:].view(m, n + pad)[:, :n]


def check_norm(qb, x, w, eps, r):
    before = None if r is None else r.clone()
    around = None if r is None or r.is_contiguous() else r._base.clone()
    q, d = qb.rms_norm_q8(x, w, eps, residual=r)
    h = x.double() + (0 if r is None else before.double())
    if r is not None:
        assert torch.equal(r, (x.float() + before.float()).to(r.dtype))
        if around is not None:  # what lies between the rows stays
            mask = torch.ones_like(around, dtype=torch.bool)
            mask.as_strided(r.shape, r.stride(), r.storage_offset())[:] = False
            assert torch.equal(r._base[mask], around[mask])
    y = h / (h.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
    top = y.unflatten(1, (-1, 32)).abs().amax(-1)
    assert bool(((d.double() - top / 127).abs() <= 32 * U * top / 127).all())
    codes = q.unflatten(1, (-1, 32)).int()
    assert int(codes.abs().max()) <= 127
    assert bool((codes.abs().amax(-1) == torch.where(top > 1e-30, 127, 0)).all())
    got = codes.double() * d.double()[..., None]
    assert bool(((got - y.unflatten(1, (-1, 32))).abs() <= (0.5 + 3e-4) * d.double()[..., None]).all())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("residual", [None, "same", "f32"])
@pytest.mark.parametrize("m, n", [(1, 32), (1, 896), (3, 64), (2, 2048), (5, 2080), (7, 4864), (2, 8192), (3, 8224), (257, 896), (1, 32768)])
def test_norm(qb, name, residual, m, n):
    x = rows(m, n, name, seed=n)
    w = 1 + 0.3 * rows(1, n, "f32", seed=1)[0]
    r = None if residual is None else rows(m, n, name if residual == "same" else "f32", seed=2, std=3.0)
    check_norm(qb, x, w, 1e-6, r)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("residual, pad, lead", [(None, 0, 0), ("same", 0, 0), ("f32", 0, 0), (None, 3, 1), ("same", 5, 3), ("f32", 1, 1)])
@pytest.mark.parametrize("m, n", [(5000, 256), (4700, 288), (3900, 352), (2000, 896), (1201, 1024), (651, 2048)])
def test_norm_of_many_short_rows(qb, name, residual, pad, lead, m, n):
    x = rows(m, n, name, seed=n, pad=pad, lead=lead)
    w = 1 + 0.3 * rows(1, n, "f32", seed=1, lead=lead)[0]
    r = None if residual is None else rows(m, n, name if residual == "same" else "f32", seed=2, pad=pad, lead=lead, std=3.0)
    check_norm(qb, x, w, 1e-6, r)


def test_norm_of_the_smallest_numbers(qb):
    """Scales below the normal numbers: a block reads as zeros, which is within 128 of 2^-126; above, as ever."""
    x, w = rows(2, 160, "f32", seed=12), torch.full((160,), 1e-36, device="cuda")
    w[32:64], w[64:96], w[96:128] = 1e-38, 3e-37, 1e-35
    q, d = qb.rms_norm_q8(x, w)
    v = qb.dequantize_q8(q, d, torch.float32).double().unflatten(1, (-1, 32))
    y = (x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()).unflatten(1, (-1, 32))
    top = y.abs().amax(-1, keepdim=True)
    assert bool(((v - y).abs() <= torch.where(top > 127.5 * 2.0 ** -126, (0.5 + 3e-4) * top / 127, 128 * 2.0 ** -126)).all())
    assert bool((q.unflatten(1, (-1, 32))[:, 3] != 0).any()) and not q.unflatten(1, (-1, 32))[:, 1].any()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("pad, lead", [(8, 0), (8, 8), (1, 0), (0, 1), (3, 5)])
def test_norm_of_rows_in_wider_ones(qb, name, pad, lead):
    w = rows(1, 896, "f32", seed=3, lead=lead)[0]
    check_norm(qb, rows(9, 896, name, seed=4, pad=pad, lead=lead), w, 1e-5, rows(9, 896, name, seed=5, pad=pad, lead=lead))
    check_norm(qb, rows(9, 896, name, seed=4), w, 1e-5, rows(9, 896, "f32", seed=5, pad=pad, lead=lead))
    check_norm(qb, rows(9, 8224, name, seed=4, pad=pad, lead=lead), rows(1, 8224, "f32", seed=3)[0], 1e-5, None)


@pytest.mark.parametrize("std", [1e-3, 1e3])
def test_norm_of_small_and_large_rows(qb, std):
    check_norm(qb, rows(4, 896, "f32", seed=6, std=std), rows(1, 896, "f32", seed=7)[0], 1e-6, rows(4, 896, "f32", seed=8, std=std))


def test_norm_of_zeros_and_of_no_rows(qb):
    w = torch.ones(64, device="cuda")
    q, d = qb.rms_norm_q8(torch.zeros(2, 64, device="cuda"), w)
    assert not q.any() and not d.any()
    q, d = qb.rms_norm_q8(torch.zeros(0, 64, device="cuda"), w)
    assert q.shape == (0, 64) and d.shape == (0, 2)
    x = rows(2, 96, "f32", seed=9)
    w = torch.ones(96, device="cuda")
    w[32:64] = 0  # a block of zeros among others
    q, d = qb.rms_norm_q8(x, w)
    assert not q[:, 32:64].any() and not d[:, 1].any() and bool((d[:, [0, 2]] > 0).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_norm_of_values_that_are_not_finite(qb, bad):
    x = rows(3, 128, "f32", seed=10)
    x[1, 40] = bad
    q, d = qb.rms_norm_q8(x, torch.ones(128, device="cuda"))
    v = qb.dequantize_q8(q, d, torch.float32)
    assert bool(v[1, 32:64].isnan().all()) and not v[[0, 2]].isnan().any()
    w = torch.ones(128, device="cuda")
    w[70] = bad  # one block of every row
    v = qb.dequantize_q8(*qb.rms_norm_q8(rows(3, 128, "f32", seed=11), w), torch.float32)
    assert bool(v[:, 64:96].isnan().all()) and not v[:, :64].isnan().any() and not v[:, 96:].isnan().any()


def test_norm_halves_go_away_from_zero(qb):
    """A block whose y / d is exact: with w = 1 and a mean square of 1, values k / 2 of a largest one of 127."""
    x = torch.zeros(1, 64, device="cuda")
    x[0, :8] = torch.tensor([127, 0.5, -0.5, 1.5, -1.5, 2.5, 63.5, -126.5], device="cuda")
    q, _ = qb.rms_norm_q8(x, torch.ones(64, device="cuda"), eps=0.0)
    codes = q[0, :8].tolist()
    y = x.double() / x.double().square().mean().sqrt()
    t = (y / (y.abs().max() / 127))[0, :8]
    assert codes[0] == 127
    for c, v in zip(codes, t.tolist()):  # (rounded in f32 on the way: the half itself may fall to either side)
        assert abs(c - v) <= 0.5 + 3e-4


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m, n", [(1, 32), (5, 96), (3, 4864), (1021, 896)])
def test_dequantize(qb, name, m, n):
    g = torch.Generator(device="cuda").manual_seed(m)
    q = torch.randint(-128, 128, (m, n), generator=g, device="cuda", dtype=torch.int8)
    d = torch.exp(torch.randn(m, n // 32, generator=g, device="cuda"))
    d[0, 0] = -2.0
    want = (q.float().unflatten(1, (-1, 32)) * d[..., None]).flatten(1).to(TYPES[name])
    assert torch.equal(qb.dequantize_q8(q, d, TYPES[name]), want)
    assert torch.equal(qb.dequantize_q8(q, d), (q.float().unflatten(1, (-1, 32)) * d[..., None]).flatten(1).to(torch.bfloat16))


def test_norm_agrees_with_quantize(qb):
    """Rows whose norm is 1 and weights of 1: the codes are quantize_q8's of the normed row, where no rounding decides."""
    x = rows(1, 4864, "f32", seed=12)
    q, d = qb.rms_norm_q8(x, torch.ones(4864, device="cuda"), eps=0.0)
    y = (x.double() / x.double().square().mean().sqrt()).float()
    q2, d2 = qb.quantize_q8(y[0].cpu().numpy())
    assert bool(((d[0].cpu().double() - torch.from_numpy(d2).double()).abs() <= 40 * U * d2.max()).all())
    assert int((q[0].cpu().int() - torch.from_numpy(q2).int()).abs().max()) <= 1


def turned(x, pos, freqs, scale, rot, interleaved):
    """The definition in 64 bits, and |a| + |b| of each pair."""
    y, mag = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    angle = pos.double()[:, None] * torch.tensor(freqs, dtype=torch.float64, device="cuda")
    c, s = (angle.cos() * scale)[:, None], (angle.sin() * scale)[:, None]
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., lo].double(), x[..., hi].double()
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    mag[..., lo] = mag[..., hi] = (a.abs() + b.abs()) * scale
    return y, mag


def check_rope(qb, rope, q, k, pos, name, rot, interleaved, freqs, scale=1.0, **more):
    r = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]
    before = [None if x is None else x.clone() for x in (q, k)]
    got = rope(q, k, pos, **more)
    for x, y in zip(before, got):
        if x is None:
            assert y is None
            continue
        want, mag = turned(x, pos, freqs, scale, rot, interleaved)
        tol = 1.2e-6 * mag + r * want.abs() + (2.0 ** -25 if name == "f16" else 0)
        assert y.dtype == x.dtype and y.shape == x.shape
        assert bool(((y.double() - want).abs() <= tol).all()), float(((y.double() - want).abs() / (tol + 1e-300)).max())
        assert torch.equal(y[..., rot:], x[..., rot:])
    return got


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("m, heads, kv, hd, rot", [(1, 14, 2, 64, 64), (300, 14, 2, 64, 64), (5, 32, 8, 128, 32), (1300, 3, 3, 80, 20),
                                                   (17, 1, 1, 96, 2), (2, 5, 1, 256, 192), (9, 2, 1, 6, 6), (2500, 8, 2, 128, 128),
                                                   (3, 2, 2, 10, 4), (1, 300, 40, 1024, 1024)])
def test_rope(qb, name, interleaved, m, heads, kv, hd, rot):
    g = torch.Generator(device="cuda").manual_seed(m)
    rope = qb.Rope(rot, base=1e6, interleaved=interleaved)
    freqs = [1e6 ** (-2 * i / rot) for i in range(rot // 2)]
    both = torch.randn(m, heads + 2 * kv, hd, generator=g, device="cuda").to(TYPES[name])  # rows of one projection
    pos = torch.randint(0, 1 << 20, (m,), generator=g, device="cuda", dtype=torch.int32)
    q, k = check_rope(qb, rope, both[:, :heads], both[:, heads: heads + kv], pos, name, rot, interleaved, freqs)
    assert q.is_contiguous() and k.is_contiguous()
    check_rope(qb, rope, both[:, :heads], None, pos, name, rot, interleaved, freqs)
    # in place: the same bits, and the value heads behind stay
    tail = both[:, heads + kv:].clone()
    got = check_rope(qb, rope, both[:, :heads], both[:, heads: heads + kv], pos, name, rot, interleaved, freqs, inplace=True)
    assert got[0].data_ptr() == both.data_ptr() and torch.equal(got[0], q) and torch.equal(got[1], k)
    assert torch.equal(both[:, heads + kv:], tail)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("lead", [1, 2, 4])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_of_rows_at_any_address(qb, name, lead, interleaved):
    x = rows(33, 4 * 64, name, seed=20, pad=lead, lead=lead)
    q = x.unflatten(1, (4, 64))
    assert q.stride() == (256 + lead, 64, 1)
    check_rope(qb, qb.Rope(64, interleaved=interleaved), q[:, :3], q[:, 3:], torch.arange(33, device="cuda", dtype=torch.int32), name, 64,
               interleaved, [10000.0 ** (-i / 32) for i in range(32)])


def test_rope_positions_far_and_negative(qb):
    pos = torch.tensor([0, 1, -1, 2 ** 20, -(2 ** 20), 2 ** 31 - 1, -(2 ** 31)], device="cuda", dtype=torch.int32)
    q = rows(7, 128, "f32", seed=21).unflatten(1, (2, 64))
    q0, _ = check_rope(qb, qb.Rope(64, base=1e6), q, None, pos, "f32", 64, False, [1e6 ** (-i / 32) for i in range(32)])
    assert torch.equal(q0[0], q[0])


SCALINGS = [dict(kind="linear", factor=4.0), dict(kind="ntk", factor=8.0), dict(kind="yarn", factor=8.0, original=4096),
            dict(kind="yarn", factor=4.0, original=2048, beta_fast=16, beta_slow=2, attention=1.25),
            dict(kind="bands", factor=8.0, original=8192), dict(kind="bands", factor=32.0, original=4096, low=0.5, high=8)]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["kind"])
@pytest.mark.parametrize("rot", [2, 64, 128])
def test_rope_scaled_for_long_contexts(qb, scaling, rot):
    """Each scaling's property: which pairs keep their frequency, which have it divided, and the factor on the values."""
    rope, base = qb.Rope(rot, base=1e5, scaling=scaling), [1e5 ** (-2 * i / rot) for i in range(rot // 2)]
    f, scale = qb.Rope.frequencies(rot, 1e5, scaling)
    factor, kind = scaling["factor"], scaling["kind"]
    assert len(f) == rot // 2 and all(b / factor * (1 - 1e-12) <= x <= b * (1 + 1e-12) for x, b in zip(f, base))
    if kind == "linear":
        assert f == [b / factor for b in base]
    if kind == "ntk" and rot > 2:
        assert f[0] == 1.0 and math.isclose(f[-1], base[-1] / factor, rel_tol=1e-12)  # the slowest pair is stretched by the factor
    if kind == "bands":
        turns = [scaling["original"] * b / (2 * math.pi) for b in base]
        lo, hi = scaling.get("low", 1), scaling.get("high", 4)
        assert all(math.isclose(x, b, rel_tol=1e-12) for x, b, t in zip(f, base, turns) if t >= hi)
        assert all(math.isclose(x, b / factor, rel_tol=1e-12) for x, b, t in zip(f, base, turns) if t <= lo)
    if kind == "yarn":
        assert math.isclose(scale, scaling.get("attention", 0.1 * math.log(factor) + 1))
        turns = [scaling["original"] * b / (2 * math.pi) for b in base]
        # (the ramp's ends are whole pairs: one pair of slack)
        step = base[0] / base[1] if rot > 2 else 1
        assert all(math.isclose(x, b, rel_tol=1e-12) for x, b, t in zip(f, base, turns) if t >= scaling.get("beta_fast", 32) * step ** 2)
        if rot > 2:
            assert all(math.isclose(x, b / factor, rel_tol=1e-12) for x, b, t in zip(f, base, turns) if t * step ** 2 <= scaling.get("beta_slow", 1))
    else:
        assert scale == 1.0
    pos = torch.arange(0, 40000, 997, device="cuda", dtype=torch.int32)
    x = rows(pos.numel(), 3 * 128, "f32", seed=22).unflatten(1, (3, 128))
    check_rope(qb, rope, x[:, :2], x[:, 2:], pos, "f32", rot, False, f, scale)
    check_rope(qb, qb.Rope(rot, frequencies=f), x[:, :2], x[:, 2:], pos, "f32", rot, False, f)


def test_streams_and_graphs(qb):
    """On a stream that is not the current one, and captured: the same bits, with new inputs at each replay."""
    x, r, w = rows(40, 896, "bf16", seed=30), rows(40, 896, "f32", seed=31), rows(1, 896, "f32", seed=32)[0]
    pos = torch.arange(40, device="cuda", dtype=torch.int32)
    rope = qb.Rope(64)

    def all_of(x, r, stream=None):
        q, d = qb.rms_norm_q8(x, w, residual=r, stream=stream)
        v = qb.dequantize_q8(q, d, stream=stream)
        a, b = rope(x.view(40, 14, 64), x.view(40, 14, 64)[:, :2], pos, stream=stream)
        return q, d, v, a, b

    want = [t.clone() for t in all_of(x, r.clone())]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream, 0):
        mine = r.clone()
        torch.cuda.synchronize()
        got = all_of(x, mine, stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs, rs = x.clone(), r.clone()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = all_of(xs, rs)
    for seed in (33, 34):
        x2, r2 = rows(40, 896, "bf16", seed=seed), rows(40, 896, "f32", seed=seed + 10)
        xs.copy_(x2)
        rs.copy_(r2)
        g.replay()
        want = all_of(x2, r2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(rs, r2)


def test_what_is_refused(qb):
    x, w = torch.zeros(2, 64, device="cuda"), torch.ones(64, device="cuda")
    for bad in (dict(x=x.double()), dict(x=x.cpu()), dict(x=x[0]), dict(x=x.t()), dict(weight=w.half()), dict(weight=w[:32]),
                dict(weight=w.cpu()), dict(residual=x.half()), dict(residual=x[:1]), dict(residual=x.cpu())):
        with pytest.raises(TypeError):
            qb.rms_norm_q8(**(dict(x=x, weight=w) | bad))
    with pytest.raises(qb.QntError, match="multiple of 32"):
        qb.rms_norm_q8(x[:, :40], w[:40])
    with pytest.raises(qb.QntError, match="not be x"):
        qb.rms_norm_q8(x, w, residual=x)
    with pytest.raises(qb.QntError, match="eps"):
        qb.rms_norm_q8(x, w, eps=-1.0)
    with pytest.raises(qb.QntError, match="stride"):
        qb.rms_norm_q8(w.expand(2, 64), w)
    q, d = qb.rms_norm_q8(x, w)
    for bad in (dict(q=q.int()), dict(q=q[:, :32]), dict(d=d[:1]), dict(d=d.half()), dict(d=d.cpu()), dict(dtype=torch.int8)):
        with pytest.raises(TypeError):
            qb.dequantize_q8(**(dict(q=q, d=d) | bad))
    rope, heads, pos = qb.Rope(64), torch.zeros(2, 3, 64, device="cuda"), torch.zeros(2, device="cuda", dtype=torch.int32)
    for a in ((heads.double(), None, pos), (heads, heads.half(), pos), (heads, heads[..., :32], pos), (heads[:, :, ::2], None, pos),
              (heads, heads[:1], pos), (heads, None, pos.long()), (heads, None, pos[:1]), (heads, None, pos.cpu()), (heads.cpu(), None, pos),
              (heads[0], None, pos), (heads.transpose(0, 1), None, torch.zeros(3, device="cuda", dtype=torch.int32))):
        with pytest.raises(TypeError):
            rope(*a)
    with pytest.raises(qb.QntError, match="rotary_dim"):
        rope(heads[..., :32].contiguous(), None, pos)

"""Token operators on the GPU against their definitions in float64.

Bounds are worked out per element from the roundings that the kernels make, u = half a step of the storage type
(2^-8 bf16, 2^-24 float32) and e = 2^-24 for float32 arithmetic, before the first run:

attention   a score is a sum of D products: |ds| <= D e scale |q||k|^T =: es;  a probability is exp of it (argument and
            result rounded in float32) and, in bf16, rounded once:  |dp| <= p (u + ep), ep = 4 max(es) + 2^-22 (2 + max|s|)
            + Sk e.  So |do| <= (u + 2 ep) p|v| + u |o|, and for the gradients with delta = sum do o:
              dv: (u + 2 ep) p^T|do| + u |dv|
              dsc = p (dp - delta): |d dsc| <= p (D e |do||v|^T + |do| |bound of o|) + (2 ep + u) |dsc|
              dq: scale (bound of dsc) |k| + u |dq|;  dk: scale (bound of dsc)^T |q| + u |dk|
            each plus (number of terms) e of the sum of magnitudes for the float32 accumulation.
LayerNorm   a row sum passes at most 40 + N / 1024 additions: c = (80 + N / 512) e;  the mean is off by c mean|s|, so
            xhat by c (mean|s| rstd + 4 |xhat| + 1);  gradients by the same through their formulas.
linear      K products and additions: |da| <= (K + 4) e |x||w|^T;  activations have slopes up to 1.13.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cycle_gan_rna_amd import _lib, tokens  # noqa: E402

BF, F32 = torch.bfloat16, torch.float32
E = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def rand(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def within(got, ref, bound, what):
    got, ref = got.detach().cpu().double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    over = ((got - ref).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 0, "%s: %.3g over its bound (largest error %.3g)" % (what, over, (got - ref).abs().max())


# --------------------------------------------------------------------------- #
# attention                                                                    #
# --------------------------------------------------------------------------- #
def attention_reference(q, k, v, do, causal, mask, scale):
    """o, dq, dk, dv and their bounds, all (B, S, heads, D) float64, from the formulas."""
    dt = q.dtype
    u = half_step(dt)
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, do))
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1:3]
    G = H // Hkv
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    seen = torch.ones(B, 1, Sq, Sk, dtype=torch.bool)
    if mask is not None:
        seen = seen & mask[:, None, None, :].bool()
        hide = ~mask.bool()
        kk, vv = (torch.where(hide[:, None, :, None], 0.0, t) for t in (kk, vv))     # hidden keys may hold anything
    if causal:
        seen = seen & torch.ones(Sq, Sk, dtype=torch.bool).tril(Sk - Sq)
    s = scale * q @ kk.transpose(2, 3)
    es = D * E * scale * (q.abs() @ kk.abs().transpose(2, 3))
    top = torch.where(seen, s, -math.inf).amax(-1, keepdim=True) if Sk else torch.full((B, H, Sq, 1), -math.inf)
    p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    mag = float(torch.where(seen, s, 0.0).abs().max()) if s.numel() else 0.0
    ep = 4 * (float(es.max()) if es.numel() else 0.0) + 2 ** -22 * (2 + mag) + Sk * E
    pu = u if dt == BF else 0.0
    o = p @ vv
    bo = (pu + 2 * ep + Sk * E) * (p @ vv.abs()) + u * o.abs() + 1e-30
    delta = (do * o).sum(-1, keepdim=True)
    dp = do @ vv.transpose(2, 3)
    ds = p * (dp - delta)
    bds = p * (D * E * (do.abs() @ vv.abs().transpose(2, 3)) + (do.abs() * (bo + D * E * o.abs())).sum(-1, keepdim=True)) + \
        (2 * ep + pu + 4 * E) * ds.abs() + 2 * ep * p * (dp.abs() + delta.abs())
    dv = p.transpose(2, 3) @ do
    bdv = (pu + 2 * ep + Sq * G * E) * (p.transpose(2, 3) @ do.abs())
    dq = scale * ds @ kk
    bdq = scale * (bds + Sk * E * ds.abs()) @ kk.abs() + u * dq.abs() + 1e-30
    dk = scale * ds.transpose(2, 3) @ q
    bdk = scale * (bds + Sq * G * E * ds.abs()).transpose(2, 3) @ q.abs()
    fold = lambda t: t.reshape(B, Hkv, G, Sk, D).sum(2)  # noqa: E731
    dk, dv, bdk, bdv = fold(dk), fold(dv), fold(bdk), fold(bdv)
    bdk, bdv = bdk + u * dk.abs() + 1e-30, bdv + u * dv.abs() + 1e-30
    return [t.transpose(1, 2) for t in (o, dq, dk, dv)], [t.transpose(1, 2) for t in (bo, bdq, bdk, bdv)]


def make_qkv(gen, dt, B, H, Hkv, Sq, Sk, D, layout):
    """q, k, v on the GPU in a layout and their values on the CPU."""
    q, k, v = rand(gen, B, Sq, H, D, dtype=dt), rand(gen, B, Sk, Hkv, D, dtype=dt), rand(gen, B, Sk, Hkv, D, dtype=dt)
    if layout == "dense":
        g = [t.cuda() for t in (q, k, v)]
    elif layout == "heads first":            # (B, H, S, D) in memory
        g = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (q, k, v)]
    elif layout == "packed":                 # views of one (B, S, H + 2 Hkv, D) projection
        assert Sq == Sk
        w = torch.cat([q, k, v], 2).cuda()
        g = [w[:, :, :H], w[:, :, H:H + Hkv], w[:, :, H + Hkv:]]
    elif layout == "odd":                    # rows that start 2 or 4 bytes off, with a gap: copied by the wrapper
        g = []
        for t in (q, k, v):
            w = torch.zeros(*t.shape[:3], D + 3, dtype=dt, device="cuda")
            w[..., 1:D + 1] = t.cuda()
            g.append(w[..., 1:D + 1])
    elif layout == "batch last":             # (S, H, B, D) in memory: token stride largest
        g = [t.permute(1, 2, 0, 3).contiguous().cuda().permute(2, 0, 1, 3) for t in (q, k, v)]
    return (q, k, v), g


CASES = [
    # B, H, Hkv, Sq, Sk, D, causal, mask, layout
    (1, 1, 1, 1, 1, 8, False, None, "dense"),
    (2, 3, 3, 1, 63, 16, False, "ragged", "dense"),
    (2, 4, 2, 2, 64, 64, False, None, "heads first"),
    (1, 2, 2, 33, 65, 40, False, "scatter", "odd"),
    (2, 2, 1, 31, 129, 128, True, None, "dense"),
    (2, 4, 4, 128, 128, 64, True, "scatter", "packed"),
    (3, 2, 2, 200, 333, 32, False, "ragged", "batch last"),
    (1, 4, 4, 257, 64, 72, True, None, "heads first"),      # more rows than keys: the first 193 see nothing
    (2, 8, 2, 5, 1000, 64, False, "ragged", "dense"),       # few rows, many keys: four heads share a tile, keys split
    (1, 8, 1, 1, 4097, 128, False, None, "dense"),          # one query
    (2, 6, 3, 130, 130, 104, True, None, "packed"),
    (4, 1, 1, 7, 70, 24, False, "empty", "dense"),          # cells without any key
    (1, 2, 1, 300, 20, 128, False, None, "dense"),          # few keys, many rows: rows split for dk, dv
    (1, 1, 1, 129, 4100, 8, True, None, "dense"),
]


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D,causal,mask,layout", CASES)
def test_attention(dt, B, H, Hkv, Sq, Sk, D, causal, mask, layout):
    gen = torch.Generator().manual_seed(Sq * 7 + Sk)
    cpu, gpu = make_qkv(gen, dt, B, H, Hkv, Sq, Sk, D, layout)
    do = rand(gen, B, Sq, H, D, dtype=dt)
    m = None
    if mask == "ragged":
        m = torch.arange(Sk)[None] < torch.tensor([Sk - (b * Sk) // (B + 1) for b in range(B)])[:, None]
    elif mask == "scatter":
        m = torch.rand(B, Sk, generator=gen) < 0.6
    elif mask == "empty":
        m = torch.rand(B, Sk, generator=gen) < 0.5
        m[::2] = False
    (o, dq, dk, dv), bounds = attention_reference(*cpu, do, causal, m, D ** -0.5)
    leaves = [t.detach().requires_grad_() for t in gpu]
    gm = m.cuda() if m is not None else None
    out = tokens.attention(*leaves, causal=causal, key_mask=gm)
    grads = torch.autograd.grad(out, leaves, do.cuda())
    for what, got, ref, b in zip(("o", "dq", "dk", "dv"), (out, *grads), (o, dq, dk, dv), bounds):
        within(got, ref, b, what)
    with torch.no_grad():
        assert torch.equal(tokens.attention(*gpu, causal=causal, key_mask=gm), out)
    again = torch.autograd.grad(tokens.attention(*leaves, causal=causal, key_mask=gm), leaves, do.cuda())
    assert all(torch.equal(a, b) for a, b in zip(again, grads))           # no order of atomics in it


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
def test_attention_gradient_against_differences(dt):
    """<gradient, direction> against central differences of the definition in float64."""
    gen = torch.Generator().manual_seed(3)
    B, H, Hkv, Sq, Sk, D = 2, 4, 2, 40, 50, 32
    cpu, gpu = make_qkv(gen, dt, B, H, Hkv, Sq, Sk, D, "dense")
    do = rand(gen, B, Sq, H, D, dtype=dt)
    m = torch.rand(B, Sk, generator=gen) < 0.7
    _, bounds = attention_reference(*cpu, do, True, m, 0.3)
    leaves = [t.detach().requires_grad_() for t in gpu]
    grads = torch.autograd.grad(tokens.attention(*leaves, causal=True, key_mask=m.cuda(), scale=0.3), leaves, do.cuda())

    def value(x):
        q, k, v = (t.transpose(1, 2) for t in x)
        k, v = k.repeat_interleave(H // Hkv, 1), v.repeat_interleave(H // Hkv, 1)
        seen = m[:, None, None] & torch.ones(Sq, Sk, dtype=torch.bool).tril(Sk - Sq)
        s = torch.where(seen, 0.3 * q @ k.transpose(2, 3), torch.finfo(torch.float64).min)
        return ((torch.softmax(s, -1) * seen.any(-1, keepdim=True) @ v).transpose(1, 2) * do.double()).sum()
    x0 = [t.double() for t in cpu]
    for i in range(3):
        d = torch.randn(x0[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-4
        up, down = ([t + (h * s * d if j == i else 0) for j, t in enumerate(x0)] for s in (1, -1))
        slope = (value(up) - value(down)) / (2 * h)
        got = (grads[i].cpu().double() * d).sum()
        # the bounds of every element at once, and the third derivative's share of the difference, h^2 times O(10^3)
        limit = (bounds[i + 1] * d.abs()).sum() + 1e-4 * abs(slope) + 1e-4
        assert abs(got - slope) <= limit, (i, got, slope, limit)


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("Sq,Sk", [(70, 150), (1, 600)])
def test_what_masked_keys_hold_reaches_nothing(dt, Sq, Sk):
    gen = torch.Generator().manual_seed(5)
    B, H, D = 2, 2, 64
    (q, k, v), gpu = make_qkv(gen, dt, B, H, H, Sq, Sk, D, "dense")
    do = rand(gen, B, Sq, H, D, dtype=dt).cuda()
    m = (torch.rand(B, Sk, generator=gen) < 0.5).cuda()
    m[0] = torch.arange(Sk, device="cuda") < Sk // 3

    def run(k, v):
        leaves = [t.detach().requires_grad_() for t in (gpu[0], k, v)]
        o = tokens.attention(*leaves, key_mask=m)
        return [o, *torch.autograd.grad(o, leaves, do)]
    want = run(gpu[1], gpu[2])
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(dt).min):
        k, v = (torch.where(m[:, :, None, None], t, torch.full_like(t, bad)) for t in gpu[1:])
        for a, b in zip(run(k, v), want):
            assert torch.equal(a, b)
    assert not want[2][~m].any() and not want[3][~m].any()


def test_rows_that_see_nothing():
    """They give 0 and 0 gradient, whatever their do holds, and leave the others alone; their own k and v too."""
    gen = torch.Generator().manual_seed(6)
    for dt in (F32, BF):
        Sq, Sk, B = 100, 30, 2                       # causal: rows 0 .. 69 see nothing
        _, gpu = make_qkv(gen, dt, B, 2, 2, Sq, Sk, 32, "dense")
        do = rand(gen, B, Sq, 2, 32, dtype=dt).cuda()
        m = torch.ones(B, Sk, dtype=torch.bool, device="cuda")
        m[1] = False
        bad = do.clone()
        bad[:, :70] = float("nan")
        outs = []
        for g in (do, bad):
            leaves = [t.detach().requires_grad_() for t in gpu]
            o = tokens.attention(*leaves, causal=True, key_mask=m)
            outs.append([o, *torch.autograd.grad(o, leaves, g)])
        for a, b in zip(*outs):
            assert torch.equal(a, b) and torch.isfinite(a).all()
        o, dq, dk, dv = outs[0]
        assert not o[:, :70].any() and not o[1].any() and not dq[:, :70].any() and not dq[1].any()
        assert not dk[1].any() and not dv[1].any() and o[0, 70:].abs().min(-1).values.max() > 0


def test_not_a_number_shows():
    """A NaN at a visible key or query is not swallowed by the running maximum."""
    gen = torch.Generator().manual_seed(7)
    for dt in (F32, BF):
        for which in range(3):
            _, gpu = make_qkv(gen, dt, 1, 1, 1, 40, 200, 32, "dense")
            gpu[which][0, 7, 0, 3] = float("nan")
            o = tokens.attention(*gpu)
            rows = torch.isnan(o[0, :, 0]).any(-1)
            assert rows.all() if which else (rows[7] and rows.sum() == 1)
            assert which != 2 or torch.isnan(o[0, :, 0, 3]).all() and not torch.isnan(o[0, :, 0, 4:]).any()


def test_large_scores_and_late_maxima():
    """Scores that grow along the keys by more than the lazily raised maximum tolerates, and ones that differ by
    thousands: against float64 with the bounds of the module."""
    gen = torch.Generator().manual_seed(8)
    for dt, scale in ((F32, 1.0), (BF, 1.0), (F32, 30.0)):
        B, H, Sq, Sk, D = 1, 2, 50, 400, 32
        q, k = rand(gen, B, Sq, H, D, dtype=dt), rand(gen, B, Sk, H, D, dtype=dt)
        k = (k * torch.linspace(0.01, 6, Sk)[None, :, None, None]).to(dt)
        v, do = rand(gen, B, Sk, H, D, dtype=dt), rand(gen, B, Sq, H, D, dtype=dt)
        refs, bounds = attention_reference(q, k, v, do, False, None, scale)
        leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
        o = tokens.attention(*leaves, scale=scale)
        for what, got, ref, b in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do.cuda())), refs, bounds):
            within(got, ref, b, what)


def test_attention_lengths_of_zero():
    for dt in (F32, BF):
        def z(*s):
            return torch.ones(*s, dtype=dt, device="cuda", requires_grad=True)
        q, k, v = z(2, 5, 4, 16), z(2, 0, 2, 16), z(2, 0, 2, 16)
        o = tokens.attention(q, k, v, causal=True)
        g = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
        assert o.shape == (2, 5, 4, 16) and not o.any() and not g[0].any() and g[1].shape == k.shape
        q, k, v = z(2, 0, 4, 16), z(2, 7, 2, 16), z(2, 7, 2, 16)
        o = tokens.attention(q, k, v)
        g = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
        assert o.shape == (2, 0, 4, 16) and not g[1].any() and not g[2].any()
        q, k, v = z(0, 3, 4, 16), z(0, 7, 2, 16), z(0, 7, 2, 16)
        assert tokens.attention(q, k, v, key_mask=torch.ones(0, 7, dtype=torch.bool, device="cuda")).shape == (0, 3, 4, 16)


def test_attention_mask_layouts():
    """bool and uint8, rows of a wider tensor, one row for all cells, every other column."""
    gen = torch.Generator().manual_seed(9)
    _, gpu = make_qkv(gen, BF, 3, 2, 2, 20, 130, 32, "dense")
    wide = torch.rand(3, 400, generator=gen).cuda() < 0.5
    for m in (wide[:, 7:137], wide[:, 0:260:2], wide[:1, :130].expand(3, 130), wide.t()[:130].t()):
        want = tokens.attention(*gpu, key_mask=m.contiguous())
        assert torch.equal(tokens.attention(*gpu, key_mask=m), want)
        assert torch.equal(tokens.attention(*gpu, key_mask=m.to(torch.uint8) * 2), want)


def test_cache_behind_its_length_is_left_alone_and_offsets_pass_32_bits():
    """One query against a stored context whose keys lie further than 2^32 bytes behind the first: the first length rows
    are read through 64-bit offsets, against the same keys in a dense copy."""
    n, step = 4200, 1 << 19                     # 2^20 bytes between tokens, 4.4 GB for all of them
    store = torch.zeros(n * step + 4096, dtype=BF, device="cuda")
    kv = torch.as_strided(store, (1, n, 2, 64), (n * step, step, 64, 1))
    gen = torch.Generator().manual_seed(10)
    vals = rand(gen, 1, n, 2, 64, dtype=BF).cuda()
    kv.copy_(vals)
    q = rand(gen, 1, 1, 2, 64, dtype=BF).cuda()
    assert torch.equal(tokens.attention(q, kv, kv), tokens.attention(q, vals, vals))
    assert torch.equal(tokens.attention(q, kv[:, :4100], kv[:, :4100]), tokens.attention(q, vals[:, :4100], vals[:, :4100]))
    assert torch.equal(kv, vals)


MORE = [
    # B, H, Hkv, Sq, Sk, D, causal, mask
    (1, 2, 2, 32, 513, 128, False, None),        # few rows: as many as a wave holds
    (2, 4, 2, 16, 5000, 64, False, "ragged"),    # two heads in one tile, keys split
    (1, 4, 1, 8, 700, 32, True, "scatter"),
    (2, 2, 2, 20, 9, 64, True, None),            # more rows than keys
    (1, 2, 1, 3, 20000, 64, False, "ragged"),
    (1, 3, 3, 31, 33, 120, True, "scatter"),
    (2, 2, 2, 1, 31, 40, False, None),           # one row
    (3, 2, 2, 1, 513, 64, False, "scatter"),
    (1, 1, 1, 1, 9000, 100, True, "ragged"),
    (2, 1, 1, 1, 257, 8, False, "empty"),
    (1, 4, 2, 700, 700, 128, True, None),        # several blocks of keys, the first with the most rows
    (1, 2, 1, 2500, 300, 128, True, "scatter"),  # rows split for dk, dv; the first 2200 see nothing
    (1, 1, 1, 5000, 130, 64, False, "scatter"),
    (1, 1, 1, 1500, 257, 32, True, None),
    (12, 1, 1, 1, 12053, 32, False, "ragged"),   # one row, splits of an odd number of 32-key tiles
    (5, 1, 1, 1, 7003, 16, False, "scatter"),
    (7, 2, 2, 1, 3301, 64, False, "scatter"),
    (2, 1, 1, 1, 12053, 128, False, "scatter"),
]


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D,causal,mask", MORE)
def test_attention_row_and_key_divisions(dt, B, H, Hkv, Sq, Sk, D, causal, mask):
    if D % (8 if dt == BF else 4):                # head dimensions go in whole 16 bytes
        with pytest.raises(ValueError, match="head dimensions"):
            test_attention(dt, B, H, Hkv, Sq, Sk, D, causal, mask, "dense")
    else:
        test_attention(dt, B, H, Hkv, Sq, Sk, D, causal, mask, "dense")


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("Sq,Sk,D", [(300, 300, 32), (300, 300, 64), (300, 300, 128), (20, 300, 64), (20, 20, 32)])
def test_rows_before_the_first_visible_key(dt, Sq, Sk, D):
    """Causal order and a mask of the first keys leave rows empty in the middle of a block: their do reaches nothing."""
    gen = torch.Generator().manual_seed(11)
    _, gpu = make_qkv(gen, dt, 1, 2, 2, Sq, Sk, D, "dense")
    hidden = Sk - Sq + Sq // 2
    m = torch.arange(Sk, device="cuda")[None] >= hidden
    do = rand(gen, 1, Sq, 2, D, dtype=dt).cuda()
    bad = do.clone()
    bad[:, :Sq // 2] = float("nan")
    outs = []
    for g in (do, bad):
        leaves = [t.detach().requires_grad_() for t in gpu]
        o = tokens.attention(*leaves, causal=True, key_mask=m)
        outs.append([o, *torch.autograd.grad(o, leaves, g)])
    for a, b in zip(*outs):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert not outs[0][0][:, :Sq // 2].any() and not outs[0][1][:, :Sq // 2].any()
    assert outs[0][2][:, hidden:].any() and not outs[0][2][:, :hidden].any()


# --------------------------------------------------------------------------- #
# LayerNorm                                                                    #
# --------------------------------------------------------------------------- #
def layer_norm_reference(x, w, b, r, dy, ds, eps):
    dt, N = x.dtype, x.shape[-1]
    u, c = half_step(dt), (80 + N / 512) * E
    s = x.double() + (r.double() if r is not None else 0)
    wd = w.double() if w is not None else torch.ones(N, dtype=torch.float64)
    bd = b.double() if b is not None else torch.zeros(N, dtype=torch.float64)
    mean = s.mean(-1, keepdim=True)
    rstd = 1 / ((s - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (s - mean) * rstd
    bx = c * ((s.abs().mean(-1, keepdim=True) + s.abs()) * rstd + 4 * xh.abs() + 1)
    y = xh * wd + bd
    by = bx * wd.abs() + 4 * E * (xh * wd).abs() + u * y.abs() + 1e-30
    g = dy.double() * wd
    m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    add = ds.double() if ds is not None else 0.0
    dx = rstd * (g - m1 - xh * m2) + add
    ga = g.abs().mean(-1, keepdim=True)
    bm2 = (g.abs() * (bx + c * xh.abs())).mean(-1, keepdim=True)
    bdx = rstd * (c * (4 * g.abs() + 8 * ga + (xh * m2).abs()) + bx * m2.abs() + xh.abs() * (bm2 + c * m2.abs())) + \
        u * dx.abs() + 4 * E * (abs(add) if r is not None else 0.0) + 1e-30
    pu = half_step(w.dtype) if w is not None else 0.0
    M = s.shape[0]
    dw, db = (dy.double() * xh).sum(0), dy.double().sum(0)
    bdw = (dy.double().abs() * (bx + (M + 4) * E * xh.abs())).sum(0) + pu * dw.abs() + 1e-30
    bdb = (M + 4) * E * dy.double().abs().sum(0) + pu * db.abs() + 1e-30
    return (y, s, dx, dw, db), (by, u * s.abs() + E * s.abs(), bdx, bdw, bdb)


# the row lengths on both sides of every change of layout: 512 / 1024 / 4096 ... elements a group holds, and odd ones
LENGTHS = [1, 2, 7, 64, 65, 255, 513, 1000, 1025, 2049, 4097, 8192, 8193, 12289, 20000, 24577, 32769]


@pytest.mark.parametrize("residual", [False, True], ids=["alone", "residual"])
@pytest.mark.parametrize("dt,wt", [(F32, F32), (BF, BF), (BF, F32)], ids=["float32", "bf16", "bf16 rows"])
@pytest.mark.parametrize("N", LENGTHS)
def test_layer_norm(N, dt, wt, residual):
    gen = torch.Generator().manual_seed(N)
    M = 5 if N > 2000 else 131
    x = rand(gen, M, N, dtype=dt) + torch.randn(M, 1, generator=gen).to(dt)
    r = rand(gen, M, N, dtype=dt, scale=2.0) if residual else None
    w, b = (1 + rand(gen, N, scale=0.3)).to(wt), rand(gen, N, dtype=wt)
    dy, ds = rand(gen, M, N, dtype=dt), rand(gen, M, N, dtype=dt) if residual else None
    eps = 1e-3 if N == 1 else 1e-5
    refs, bounds = layer_norm_reference(x, w, b, r, dy, ds, eps)
    gx, gw, gb = (t.cuda().requires_grad_() for t in (x, w, b))
    gr = r.cuda().requires_grad_() if residual else None
    out = tokens.layer_norm(gx, gw, gb, residual=gr, eps=eps)
    if residual:
        y, s = out
        grads = torch.autograd.grad(out, (gx, gw, gb, gr), (dy.cuda(), ds.cuda()))
        assert torch.equal(grads[0], grads[3])
        within(s, refs[1], bounds[1], "s")
    else:
        y = out
        grads = torch.autograd.grad(out, (gx, gw, gb), dy.cuda())
    for what, got, i in (("y", y, 0), ("dx", grads[0], 2), ("dw", grads[1], 3), ("db", grads[2], 4)):
        within(got, refs[i], bounds[i], what)
    with torch.no_grad():
        plain = tokens.layer_norm(gx, gw, gb, residual=gr, eps=eps)
    assert torch.equal(plain[0] if residual else plain, y)


@pytest.mark.parametrize("M", [0, 1, 3, 4, 1023, 5000])
def test_layer_norm_row_counts(M):
    gen = torch.Generator().manual_seed(M)
    N = 72
    for dt in (F32, BF):
        x, w, b, dy = rand(gen, M, N, dtype=dt), rand(gen, N, dtype=dt), rand(gen, N, dtype=dt), rand(gen, M, N, dtype=dt)
        refs, bounds = layer_norm_reference(x, w, b, None, dy, None, 1e-5)
        leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
        y = tokens.layer_norm(*leaves)
        grads = torch.autograd.grad(y, leaves, dy.cuda())
        for what, got, i in (("y", y, 0), ("dx", grads[0], 2), ("dw", grads[1], 3), ("db", grads[2], 4)):
            within(got, refs[i], bounds[i], what)


def test_layer_norm_layouts_and_partial_gradients():
    """Strided rows, rows that start off a 16-byte address, more axes, no parameters, one parameter, a gradient for
    one output alone; what is not asked for is None."""
    gen = torch.Generator().manual_seed(1)
    for dt in (F32, BF):
        wide = rand(gen, 6, 11, 205, dtype=dt).cuda()
        x = wide[:, 2:9, 3:104]
        w = rand(gen, 101, dtype=dt).cuda()
        want = tokens.layer_norm(x.contiguous(), w)
        assert torch.equal(tokens.layer_norm(x, w), want)
        assert torch.equal(tokens.layer_norm(x.transpose(0, 1), w), want.transpose(0, 1))
        assert torch.equal(tokens.layer_norm(x[3, 4], w), want[3, 4])
        first = wide[:1, :1, :101].expand(4, 5, 101)
        assert torch.equal(tokens.layer_norm(first, w), tokens.layer_norm(first.contiguous(), w))
        y = tokens.layer_norm(x, None, w)
        refs, bounds = layer_norm_reference(x.reshape(-1, 101).cpu(), None, w.cpu(), None, torch.zeros(42, 101), None, 1e-5)
        within(y.reshape(-1, 101), refs[0], bounds[0], "y without weight")
        xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
        r = rand(gen, 6, 7, 101, dtype=dt).cuda()
        y, s = tokens.layer_norm(xg, wg, residual=r)
        (gs,) = torch.autograd.grad(s, xg, torch.ones_like(s), retain_graph=True)
        assert torch.equal(gs, torch.ones_like(gs))                       # the stream alone: its gradient passes through
        gx, = torch.autograd.grad(y, xg, torch.ones_like(y), retain_graph=True)
        gw, = torch.autograd.grad(y, wg, torch.ones_like(y).sum(-1, keepdim=True).expand_as(y) / 101)
        refs, bounds = layer_norm_reference(x.reshape(-1, 101).cpu(), w.cpu(), None, r.reshape(-1, 101).cpu(), torch.ones(42, 101), None, 1e-5)
        within(gx.reshape(-1, 101), refs[2], bounds[2], "dx of y alone")
        within(gw, refs[3], bounds[3], "dw alone")


def test_layer_norm_constant_and_far_rows():
    """A constant row has variance 0 (y = bias); rows whose mean is 10^4 times their spread keep their digits: the
    deviation from the mean is taken before it is squared."""
    for dt in (F32,):
        x = torch.full((3, 1000), 7.0, device="cuda")
        b = torch.randn(1000, device="cuda")
        assert torch.equal(tokens.layer_norm(x, None, b), b.expand(3, 1000))
        gen = torch.Generator().manual_seed(2)
        far = (rand(gen, 9, 1000) + 1e4).cuda()
        refs, bounds = layer_norm_reference(far.cpu(), None, None, None, torch.zeros(9, 1000), None, 1e-5)
        within(tokens.layer_norm(far), refs[0], bounds[0], "far rows")


# --------------------------------------------------------------------------- #
# dense layer                                                                  #
# --------------------------------------------------------------------------- #
def act_and_slope(a, act, slope):
    if act == "leaky":
        return torch.where(a > 0, a, slope * a), torch.where(a > 0, 1.0, slope).double()
    if act == "gelu":
        c = torch.special.ndtr(a)
        return a * c, c + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    if act == "silu":
        g = torch.sigmoid(a)
        return a * g, g * (1 + a * (1 - g))
    return a, torch.ones_like(a)


def linear_reference(x, w, b, r, dy, act, slope):
    """y, dx, dw, db and their bounds.  Activations: slope up to 1.13, second derivative up to 0.8 (leaky: data whose
    sums are exact); their float32 evaluation within 2^-19 of a."""
    u, K, (M, N) = half_step(x.dtype), x.shape[1], dy.shape
    xd, wd, dyd = x.double(), w.double(), dy.double()
    a = xd @ wd.T + (b.double() if b is not None else 0)
    ba = (K + 4) * E * (xd.abs() @ wd.abs().T + (b.double().abs() if b is not None else 0))
    if act == "leaky":
        ba = 0 * ba
    y, sl = act_and_slope(a, act, slope)
    y = y + (r.double() if r is not None else 0)
    fine = 0.0 if act == "none" else 2.0 ** -19
    by = 1.13 * ba + fine * a.abs() + 4 * E * (r.double().abs() if r is not None else 0) + u * y.abs() + 1e-30
    da = dyd * sl
    bda = dyd.abs() * (0.0 if act in ("none", "leaky") else 1.0) * (0.8 * (ba + u * a.abs()) + 2.0 ** -19) + 4 * E * da.abs()
    ru = 0.0 if act == "none" else u
    dx, dw, db = da @ wd, da.T @ xd, da.sum(0)
    bdx = (bda + (ru + (N + 4) * E) * da.abs()) @ wd.abs() + u * dx.abs() + 1e-30
    bdw = (bda + (ru + (M + 4) * E) * da.abs()).T @ xd.abs() + u * dw.abs() + 1e-30
    bdb = (bda + (M + 4) * E * da.abs()).sum(0) + u * db.abs() + 1e-30
    return (y, dx, dw, db), (by, bdx, bdw, bdb)


LINEAR = [
    # M, N, K
    (1, 1, 1), (1, 1000, 4096), (3, 77, 129), (4, 64, 64), (5, 33, 40), (17, 130, 65), (64, 64, 64), (100, 5000, 31),
    (129, 257, 513), (300, 8, 1030), (513, 384, 128), (2048, 40, 24), (1000, 600, 200),
    (2100, 2050, 72),        # the 256-row tiles
    (70, 90, 9000),          # a long sum over few tiles: split
]


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear(dt, M, N, K):
    gen = torch.Generator().manual_seed(M + N + K)
    i = LINEAR.index((M, N, K))
    act = ("none", "gelu", "silu")[i % 3]
    with_b, with_r = i % 2 == 0, i % 4 < 2
    x, w = rand(gen, M, K, dtype=dt), rand(gen, N, K, dtype=dt, scale=K ** -0.5)
    b = rand(gen, N, dtype=dt) if with_b else None
    r = rand(gen, M, N, dtype=dt) if with_r else None
    dy = rand(gen, M, N, dtype=dt)
    refs, bounds = linear_reference(x, w, b, r, dy, act, 0.0)
    gx, gw, gb, gr = (t.cuda().requires_grad_() if t is not None else None for t in (x, w, b, r))
    y = tokens.linear(gx, gw, gb, activation=act, residual=gr)
    leaves = [t for t in (gx, gw, gb, gr) if t is not None]
    grads = list(torch.autograd.grad(y, leaves, dy.cuda()))
    within(y, refs[0], bounds[0], "y")
    within(grads[0], refs[1], bounds[1], "dx")
    within(grads[1], refs[2], bounds[2], "dw")
    if with_b:
        within(grads[2], refs[3], bounds[3], "db")
    if with_r:
        assert torch.equal(grads[-1], dy.cuda())
    again = torch.autograd.grad(tokens.linear(gx, gw, gb, activation=act, residual=gr), leaves, dy.cuda())
    assert all(torch.equal(a, c) for a, c in zip(again, grads))
    with torch.no_grad():
        assert torch.equal(tokens.linear(gx, gw, gb, activation=act, residual=gr), y)


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 40, 64), (3, 40, 63), (200, 130, 72), (600, 520, 40)])
@pytest.mark.parametrize("slope", [0.0, 0.25])
def test_linear_leaky_on_exact_sums(dt, M, N, K, slope):
    """Small integers: every sum is exact in float32, so a value of 0 is 0, and the lane, row and column maps of the three
    products show as whole differences.  The operands are not symmetric."""
    gen = torch.Generator().manual_seed(M + K)
    x = torch.randint(-2, 3, (M, K), generator=gen).to(dt)
    w = (torch.arange(N * K).reshape(N, K) % 5 - 2).to(dt)
    b = (torch.arange(N) % 7 - 3).to(dt)
    dy = torch.randint(-2, 3, (M, N), generator=gen).to(dt)
    a = x.double() @ w.double().T + b.double()
    da = dy.double() * torch.where(a > 0, 1.0, slope)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = tokens.linear(*leaves, activation="leaky", slope=slope)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    for got, ref in ((y, torch.where(a > 0, a, slope * a)), (grads[0], da @ w.double()), (grads[1], da.T @ x.double()),
                     (grads[2], da.sum(0))):
        assert torch.equal(got.cpu(), ref.to(dt))


def test_linear_layouts_and_partial_gradients():
    gen = torch.Generator().manual_seed(11)
    for dt in (F32, BF):
        wide = rand(gen, 9, 30, 150, dtype=dt).cuda()
        x = wide[:, 3:20, 5:101]                                  # (9, 17, 96), rows 2 or 4 bytes off
        w = rand(gen, 96, 200, dtype=dt).cuda()[:, 7:157].t()     # (150, 96) along its rows
        want = tokens.linear(x.contiguous(), w.contiguous())
        got = tokens.linear(x, w)
        assert torch.equal(got, want) and got.shape == (9, 17, 150)
        assert torch.equal(tokens.linear(x[0, 0], w), tokens.linear(x[0, 0].contiguous(), w.contiguous()))
        xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
        xc, wc = x.contiguous().requires_grad_(), w.contiguous().requires_grad_()
        full = torch.autograd.grad(tokens.linear(xc, wc, activation="silu").sum(), (xc, wc))
        assert torch.equal(torch.autograd.grad(tokens.linear(xg, w, activation="silu").sum(), xg)[0], full[0])
        assert torch.equal(torch.autograd.grad(tokens.linear(x, wg, activation="silu").sum(), wg)[0], full[1])
        b = rand(gen, 150, dtype=dt).cuda().requires_grad_()
        (db,) = torch.autograd.grad(tokens.linear(x, w, b).sum(), b)
        assert torch.equal(db, torch.full_like(db, 9 * 17))
        e = tokens.linear(torch.zeros(0, 96, dtype=dt, device="cuda"), wg, b)
        assert e.shape == (0, 150) and not torch.autograd.grad(e.sum(), wg)[0].any()


# --------------------------------------------------------------------------- #
# together                                                                     #
# --------------------------------------------------------------------------- #
def layer(x, P, heads, mask, linear, attention, layer_norm):
    """A pre-norm transformer layer over (B, S, E) tokens."""
    B, S, D = x.shape
    h = layer_norm(x, P["g1"], P["b1"])
    qkv = linear(h, P["wqkv"], P["bqkv"]).view(B, S, 3, heads, D // heads)
    o = attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], key_mask=mask)
    a = linear(o.reshape(B, S, D), P["wo"], P["bo"])
    h, x = layer_norm(a, P["g2"], P["b2"], residual=x)
    return linear(linear(h, P["w1"], P["c1"], activation="gelu"), P["w2"], P["c2"], residual=x)


def reference_ops():
    def linear(x, w, b, activation="none", residual=None):
        a = x @ w.T + b
        a = a * torch.special.ndtr(a) if activation == "gelu" else a
        return a if residual is None else a + residual

    def attention(q, k, v, key_mask):
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        s = q @ k.transpose(2, 3) / math.sqrt(q.shape[-1])
        return (torch.softmax(s.masked_fill(~key_mask[:, None, None], -math.inf), -1) @ v).transpose(1, 2)

    def layer_norm(x, w, b, residual=None):
        s = x if residual is None else x + residual
        y = torch.nn.functional.layer_norm(s, (s.shape[-1],), w, b)
        return y if residual is None else (y, s)
    return linear, attention, layer_norm


def layer_parameters(gen, D, F):
    P = {"g1": 1 + rand(gen, D, scale=0.1), "b1": rand(gen, D, scale=0.1), "g2": 1 + rand(gen, D, scale=0.1), "b2": rand(gen, D, scale=0.1),
         "wqkv": rand(gen, 3 * D, D, scale=D ** -0.5), "bqkv": rand(gen, 3 * D, scale=0.1), "wo": rand(gen, D, D, scale=D ** -0.5),
         "bo": rand(gen, D, scale=0.1), "w1": rand(gen, F, D, scale=D ** -0.5), "c1": rand(gen, F, scale=0.1),
         "w2": rand(gen, D, F, scale=F ** -0.5), "c2": rand(gen, D, scale=0.1)}
    return P


@pytest.mark.parametrize("dt,tol", [(F32, 2e-5), (BF, 6e-2)], ids=["float32", "bf16"])
def test_transformer_layer(dt, tol):
    """Eight operators in a row, forward and backward, against the same layer in float64.  float32: the framework's bar
    for float32 chains, 2e-5 of the largest value.  bf16: every tensor between two operators is rounded (2^-8 of its
    largest value at most each, 8 forward and 8 backward: 16 x 2^-8)."""
    gen = torch.Generator().manual_seed(12)
    B, S, D, heads = 3, 77, 96, 4
    P = {k: v.to(dt) for k, v in layer_parameters(gen, D, 200).items()}
    x, dy = rand(gen, B, S, D, dtype=dt), rand(gen, B, S, D, dtype=dt)
    mask = torch.arange(S)[None] < torch.tensor([77, 50, 3])[:, None]
    ref_x = x.double().requires_grad_()
    ref_p = {k: v.double().requires_grad_() for k, v in P.items()}
    ref = layer(ref_x, ref_p, heads, mask, *reference_ops())
    ref_g = torch.autograd.grad(ref, [ref_x, *ref_p.values()], dy.double())
    gx = x.cuda().requires_grad_()
    gp = {k: v.cuda().requires_grad_() for k, v in P.items()}
    got = layer(gx, gp, heads, mask.cuda(), tokens.linear, tokens.attention, tokens.layer_norm)
    grads = torch.autograd.grad(got, [gx, *gp.values()], dy.cuda())
    for what, a, b in zip(["y", "x", *P], (got, *grads), (ref, *ref_g)):
        err = float((a.detach().cpu().double() - b).abs().max() / b.abs().max())
        assert err <= tol, (what, err)


def test_self_attention_module_takes_any_tokens():
    """GeneSelfAttention on token sets that the fused kernel is not built for, with a mask, against torch.nn in float64."""
    from cycle_gan_rna_amd import GAN_functions as F
    for (B, S, Em, heads) in ((3, 50, 64, 4), (2, 16, 48, 2), (2, 300, 16, 4)):
        torch.manual_seed(S)
        at = F.GeneSelfAttention(Em, heads, dropout_rate=0.0).cuda()
        x = torch.randn(B, S, Em)
        mask = torch.rand(B, S) < 0.8
        mask[:, 0] = True
        xa = x.cuda().requires_grad_()
        ya = at(xa, key_mask=mask.cuda())
        ya.square().sum().backward()
        ref = torch.nn.MultiheadAttention(Em, heads, batch_first=True).double()
        ref.load_state_dict({k: v.cpu().double() for k, v in at.attention.state_dict().items()})
        xb = x.double().requires_grad_()
        yb = torch.nn.functional.layer_norm(xb + ref(xb, xb, xb, key_padding_mask=~mask)[0], (Em,))
        yb.square().sum().backward()
        for a, b in ((ya, yb), (xa.grad, xb.grad), (at.attention.in_proj_weight.grad, ref.in_proj_weight.grad),
                     (at.attention.out_proj.weight.grad, ref.out_proj.weight.grad)):
            assert float((a.detach().cpu().double() - b.detach()).abs().max()) <= 2e-5 * max(float(b.abs().max()), 1.0)
        with pytest.raises(RuntimeError, match="no attention dropout"):
            F.GeneSelfAttention(Em, heads).cuda().train()(x.cuda()[:, :S], key_mask=mask.cuda())


def test_backward_twice_through_is_refused():
    q = torch.ones(1, 4, 1, 8, device="cuda", requires_grad=True)
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    for y, t in ((tokens.attention(q, q, q), q), (tokens.layer_norm(x), x), (tokens.linear(x, x), x)):
        with pytest.raises(RuntimeError, match="first-order only"):
            torch.autograd.grad(y.sum(), t, create_graph=True)


def test_on_another_stream_and_two_at_once():
    """Work on a side stream (its inputs made there), and two streams running the same operators at the same time with
    different data: the same bits as one after the other on the default stream."""
    gen = torch.Generator().manual_seed(13)
    P = {k: v.to(BF).cuda() for k, v in layer_parameters(gen, 128, 256).items()}
    xs = [rand(gen, 4, 200, 128, dtype=BF).cuda() for _ in range(2)]
    mask = torch.ones(4, 200, dtype=torch.bool, device="cuda")

    def run(x):
        x = x.detach().requires_grad_()
        y = layer(x, P, 4, mask, tokens.linear, tokens.attention, tokens.layer_norm)
        return [y.detach(), *torch.autograd.grad(y, x, torch.ones_like(y))]
    want = [run(x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_captured_and_replayed():
    """Forward and backward of a layer, and one query over split keys, in one HIP graph: replayed several times on new
    data with eager work in between, while an eager graph of the same parameters lives."""
    gen = torch.Generator().manual_seed(14)
    P = {k: v.cuda().requires_grad_() for k, v in layer_parameters(gen, 64, 128).items()}
    mask = torch.rand(2, 150, generator=gen).cuda() < 0.8
    mask[:, 0] = True
    x = torch.zeros(2, 150, 64, device="cuda", requires_grad=True)
    q, kv = torch.zeros(1, 1, 4, 64, dtype=BF, device="cuda"), torch.zeros(1, 3000, 2, 64, dtype=BF, device="cuda")

    def run(x, q, kv, P):
        y = layer(x, P, 4, mask, tokens.linear, tokens.attention, tokens.layer_norm)
        g = torch.autograd.grad(y, [x, *P.values()], torch.ones_like(y))
        with torch.no_grad():
            o = tokens.attention(q, kv, kv)
        return [y.detach(), *g, o]

    held = layer(x.detach(), P, 4, mask, tokens.linear, tokens.attention, tokens.layer_norm)      # alive during the capture
    own = {k: v.detach().requires_grad_() for k, v in P.items()}      # the captured pass's leaves
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, q, kv, own)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, q, kv, own)
    for k in range(4):
        nx, nq, nkv = torch.randn(2, 150, 64, generator=gen), rand(gen, 1, 1, 4, 64, dtype=BF), rand(gen, 1, 3000, 2, 64, dtype=BF)
        with torch.no_grad():
            x.copy_(nx), q.copy_(nq), kv.copy_(nkv)
        graph.replay()
        torch.cuda.synchronize()
        want = run(nx.cuda().requires_grad_(), nq.cuda(), nkv.cuda(), P)
        for a, b in zip(out, want):
            assert torch.equal(a, b), k
        torch.cuda.synchronize()
    assert torch.isfinite(torch.autograd.grad(held.sum(), P["wo"])[0]).all()


# --------------------------------------------------------------------------- #
# sizes                                                                        #
# --------------------------------------------------------------------------- #
def test_more_rows_than_one_launch():
    """2^26 + 3 short rows: the same bits as the last of them on their own, forward and backward."""
    M, N = (1 << 26) + 3, 8
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(M, N, generator=gen, device="cuda", dtype=BF)
    w = torch.randn(N, generator=gen, device="cuda", dtype=BF)
    y = tokens.layer_norm(x, w)
    part = x[-1000:].clone()
    assert torch.equal(y[-1000:], tokens.layer_norm(part, w))
    assert torch.equal(y[:1000], tokens.layer_norm(x[:1000].clone(), w))
    del y
    a, b = x.requires_grad_(), part.requires_grad_()
    g, = torch.autograd.grad(tokens.layer_norm(a, w), a, a.detach())
    h, = torch.autograd.grad(tokens.layer_norm(b, w), b, b.detach())
    assert torch.equal(g[-1000:], h)


def test_more_cells_than_a_grid_dimension():
    """70 001 cells of 9 tokens, masked: as their last ones on their own."""
    B, S, H, D = 70001, 9, 2, 8
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v, do = (torch.randn(B, S, H, D, generator=gen, device="cuda", dtype=BF) for _ in range(4))
    m = torch.rand(B, S, generator=gen, device="cuda") < 0.7

    def run(n):
        leaves = [t[-n:].clone().requires_grad_() for t in (q, k, v)]
        o = tokens.attention(*leaves, key_mask=m[-n:].clone())
        return [o, *torch.autograd.grad(o, leaves, do[-n:].clone())]
    for a, b in zip(run(B), run(500)):
        assert torch.equal(a[-500:], b)


@pytest.mark.parametrize("M", [2, 70])
def test_linear_rows_far_apart(M):
    """Rows further apart than the kernels' offsets inside a tile reach."""
    N, K, pitch = 24, 40, (1 << 21) + 8
    gen = torch.Generator(device="cuda").manual_seed(3)
    base = torch.zeros((M - 1) * pitch + K, device="cuda", dtype=BF)
    x = torch.as_strided(base, (M, K), (pitch, 1))
    x.copy_(torch.randn(M, K, generator=gen, device="cuda", dtype=BF))
    w = torch.randn(N, K, generator=gen, device="cuda", dtype=BF)
    r = torch.as_strided(base, (M, N), (pitch, 1))
    want = tokens.linear(x.contiguous(), w, residual=r.contiguous())
    assert torch.equal(tokens.linear(x, w, residual=r), want)
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    c, d = x.contiguous().detach().requires_grad_(), w.detach().requires_grad_()
    one = torch.autograd.grad(tokens.linear(a, b), (a, b), want)
    two = torch.autograd.grad(tokens.linear(c, d), (c, d), want)
    assert all(torch.equal(s, t) for s, t in zip(one, two))


def test_few_rows_over_a_context_of_2_to_26_keys():
    """32 query heads over one key head and 2^26 + 64 keys: rows times keys pass 2^31.  Causal order hides nothing from a
    single query, so its gradients have the bits of the call without it."""
    Sk, H, D = (1 << 26) + 64, 32, 8
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, do = (torch.randn(1, 1, H, D, generator=gen, device="cuda", dtype=BF) for _ in range(2))
    k, v = (torch.randn(1, Sk, 1, D, generator=gen, device="cuda", dtype=BF) for _ in range(2))

    def run(causal):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(tokens.attention(*leaves, causal=causal), leaves, do)
    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b) and b[:, :64].any()


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("Sq,Sk,D,causal", [(40, 200, 32, False), (300, 300, 64, True), (150, 200, 128, False), (2500, 300, 128, True),
                                             (16, 200, 64, False), (1, 200, 32, False), (20, 9, 64, True)])
def test_rows_that_do_not_exist_meet_no_infinity(dt, Sq, Sk, D, causal):
    """A key of -inf whose scores are all -inf has no weight: its dk and dv are 0, whatever the rows of a tile that lie behind
    the last query, or see nothing, would make of it; the other keys' are finite."""
    gen = torch.Generator().manual_seed(22)
    q, k, v = rand(gen, 1, Sq, 2, D, dtype=dt), rand(gen, 1, Sk, 2, D, dtype=dt), rand(gen, 1, Sk, 2, D, dtype=dt)
    do = rand(gen, 1, Sq, 2, D, dtype=dt)
    q[..., 3] = q[..., 3].abs() + 0.5
    low = torch.rand(Sk, generator=gen) < 0.5
    low[0] = False                                           # every row that sees a key sees this one
    k[0, low, :, 3] = -float("inf")
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    _, dk, dv = torch.autograd.grad(tokens.attention(*leaves, causal=causal), leaves, do.cuda())
    assert torch.isfinite(dk).all() and torch.isfinite(dv).all()
    assert not dk[:, low].any() and not dv[:, low].any() and dv[:, ~low].any()


# --------------------------------------------------------------------------- #
# infinities and NaN at visible keys                                           #
# --------------------------------------------------------------------------- #
KINDS = [
    # B, H, Hkv, Sq, Sk, D: one for each way the rows and keys are divided
    (1, 1, 1, 1, 200, 32),        # one row
    (1, 1, 1, 1, 9000, 64),       # one row, keys split
    (1, 2, 1, 1, 200, 32),        # few rows: heads packed
    (2, 4, 2, 16, 5000, 64),      # few rows, keys split
    (1, 2, 2, 20, 300, 128),
    (1, 2, 2, 40, 200, 32),       # many rows
    (1, 1, 1, 200, 3001, 64),     # many rows, keys split
    (1, 2, 1, 150, 700, 128),
]
HOLDS = ["+inf", "-inf", "all -inf", "all but one -inf", "visible -inf", "late half -inf", "nan"]


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("holds", HOLDS)
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D", KINDS)
def test_infinite_scores(dt, holds, B, H, Hkv, Sq, Sk, D):
    """As the definition has it, in every kernel: a row with a score of +inf or NaN, or whose visible scores are all -inf,
    is NaN, and so are the gradients that it takes part in; a score of -inf beside finite ones has no weight; a row that
    sees no key stays 0.  Finite rows against float64, with the bounds at the top of this file."""
    gen = torch.Generator().manual_seed(15)
    q, k, v, do = (rand(gen, B, s, h, D, dtype=dt) for s, h in ((Sq, H), (Sk, Hkv), (Sk, Hkv), (Sq, H)))
    m = torch.rand(B, Sk, generator=gen) < 0.7
    if B > 1:
        m[1] = False                                         # a cell without keys
    at = int(m[0].nonzero()[m[0].sum() // 2])
    low = holds not in ("+inf", "-inf", "nan")
    if low:                                                  # the sign of a row's score is that of the infinity
        q[..., 3] = q[..., 3].abs() + 0.5
    if holds in ("+inf", "-inf", "nan"):
        k[0, at, 0, 3] = float(holds)
    else:
        hit = torch.zeros(Sk, dtype=torch.bool)
        hit[:] = True
        if holds == "all but one -inf":
            hit[at] = False
        elif holds == "visible -inf":
            hit = m[0].clone()
        elif holds == "late half -inf":
            hit[:Sk // 2] = False
        k[0, hit, 0, 3] = -float("inf")

    G, scale = H // Hkv, D ** -0.5
    Q, K, V, DO = (t.double().transpose(1, 2) for t in (q, k, v, do))
    hide = ~m[:, None, :, None]
    K, V = torch.where(hide, 0.0, K).repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    seen = m[:, None, None, :].expand(B, H, Sq, Sk)
    s = torch.where(seen, scale * Q @ K.transpose(2, 3), -math.inf)
    some = seen.any(-1, keepdim=True)
    p = torch.where(seen, torch.softmax(s, -1), 0.0)
    o = p @ V
    dp = DO @ V.transpose(2, 3)
    ds = torch.where(seen, p * (dp - (DO * o).sum(-1, keepdim=True)), 0.0)
    dq, dk, dv = scale * ds @ K, scale * ds.transpose(2, 3) @ Q, p.transpose(2, 3) @ DO
    dk, dv = (t.reshape(B, Hkv, G, Sk, D).sum(2) for t in (dk, dv))
    finite = torch.where(torch.isfinite(K), K, 0.0)
    es = float((D * E * scale * (Q.abs() @ finite.abs().transpose(2, 3))).max())
    mag = float(torch.where(torch.isfinite(s), s, 0.0).abs().max())
    ep = 4 * es + 2 ** -22 * (2 + mag) + Sk * E
    bound = ((half_step(dt) if dt == BF else 0.0) + 2 * ep + Sk * E) * (p @ V.abs()) + half_step(dt) * o.abs() + 1e-30

    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    got = tokens.attention(*leaves, key_mask=m.cuda())
    grads = torch.autograd.grad(got, leaves, do.cuda())
    got = got.detach().cpu().double().transpose(1, 2)
    nan = torch.isnan(o)
    assert nan.any() or holds not in ("all -inf", "visible -inf", "nan")
    assert torch.equal(torch.isnan(got), nan)
    assert ((got - o).abs() <= bound)[~nan].all()
    assert not got[~some.expand_as(got)].any()
    for what, a, b in zip(("dq", "dk", "dv"), grads, (dq, dk, dv)):
        assert torch.equal(torch.isnan(a.cpu()), torch.isnan(b).transpose(1, 2)), what


# --------------------------------------------------------------------------- #
# activations                                                                  #
# --------------------------------------------------------------------------- #
def tail(a):
    """Distribution function of the normal distribution (torch.special.ndtr takes it from 1 + erf: 2^-53 off at any size)."""
    return 0.5 * torch.erfc(-a / math.sqrt(2))


def act_bounds(a, act, dt):
    """What a value of `act` at a and its slope may be off by, before they are rounded to dt.

    gelu = a c, c the tail of the normal distribution or 1 minus it.  The tail is bell(a) t Q(t): in units of 2^-24 of its
    value the fit of Q is off by 1.6, t = 1 / (1 + c |a|) by 4.5 (reciprocal 2, its argument 1, and it enters Q to a power of
    up to 1.5), the eight steps of Q by 3, two products by 2, exp2 by 2, the corrected exponent by 1.5; with the product by a
    15.6: 2^-20.  bf16 leaves the exponent a^2 / 2 log2(e) as it was rounded: half a^2 and three more units.  The slope is
    c + a phi(a), each by the same share of its size.
    silu = a g, g = 1 / (1 + exp(-a)): the exponent's rounding |a| units, 8 for exp2, sum, reciprocal and product, doubled;
    slope g (1 + a (1 - g)), whose 1 - g is off by a unit of 1."""
    u = 2.0 ** -24
    if act == "gelu":
        c = tail(a)
        rel = 16 * u + (0.0 if dt == F32 else (a * a / 2 + 3) * u)
        bell = torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
        return rel * (a * c).abs(), rel * (c + a.abs() * bell)
    g = torch.sigmoid(a)
    rel = 2 * (a.abs() + 8) * u
    return rel * (a * g).abs(), rel * (g + a.abs() * g * torch.sigmoid(-a)) + 2 * a.abs() * g * u


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_activation_values_and_slopes(act, dt):
    """From -10 to 10, in the product's epilogue and (four rows) beside the dot product: the error is a share of the value,
    however small that is, not of the argument."""
    gen = torch.Generator().manual_seed(16)
    a = torch.cat([torch.linspace(-10, 10, 20001), torch.randn(4000, generator=gen), -torch.logspace(-6, 1, 999)]).to(dt)
    one = torch.ones(1, 1, dtype=dt, device="cuda")
    x = a[:, None].cuda().requires_grad_()
    y = tokens.linear(x, one, activation=act)
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    rows = torch.cat([tokens.linear(t.detach(), one, activation=act) for t in x[:2000:20].split(4)])
    ad, u = a.double(), half_step(dt)
    v, s = act_and_slope(ad, act, 0.0)
    if act == "gelu":
        v, s = ad * tail(ad), tail(ad) + ad * torch.exp(-0.5 * ad * ad) / math.sqrt(2 * math.pi)
    bv, bs = act_bounds(ad, act, dt)
    within(y[:, 0], v, bv + u * (v.abs() + bv) + 1e-37, "value")
    within(rows[:, 0], v[:2000:20], (bv + u * (v.abs() + bv) + 1e-37)[:2000:20], "value of few rows")
    within(g[:, 0], s, bs + u * (s.abs() + bs) + 1e-37, "slope")


def test_activations_of_infinities():
    for dt in (F32, BF):
        x = torch.tensor([[float("inf")], [1e30], [-1e30], [-300.0], [300.0], [0.0]], dtype=dt, device="cuda")
        one = torch.ones(1, 1, dtype=dt, device="cuda")
        for act in ("gelu", "silu"):
            y = tokens.linear(x, one, activation=act)[:, 0].cpu()
            assert torch.equal(y[[0, 1, 4, 5]], x.cpu()[[0, 1, 4, 5], 0]) and not y[[2, 3]].any()
        n = torch.full((6, 1), float("nan"), dtype=dt, device="cuda")
        assert all(torch.isnan(tokens.linear(n, one, activation=act)).all() for act in ("gelu", "silu"))


def test_linear_copies_more_than_one_launch_of_rows():
    """2^23 rows of 2049 float32 values, whose padded copy has 2^32 16-byte pieces and more: the first rows, the last and
    some between against float64."""
    M, N, K = 1 << 23, 8, 2049
    gen = torch.Generator().manual_seed(21)
    at = torch.tensor([0, 1, 2, M // 2 - 1, M // 2, M - 130, M - 129, M - 2, M - 1])
    rows, w = rand(gen, len(at), K), rand(gen, N, K)
    x = torch.zeros(M, K, device="cuda")
    x[at.cuda()] = rows.cuda()
    y = tokens.linear(x, w.cuda())
    del x
    ref = rows.double() @ w.double().T
    within(y[at.cuda()], ref, (K + 4) * E * (rows.double().abs() @ w.double().abs().T) + E * ref.abs(), "y")
    y[at.cuda()] = 0
    assert not y.any()
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
def test_attention_gradient_along_itself(dt):
    """<gradient, direction> against central differences of the definition in float64, along the gradient that the formulas
    give: there the slope adds up as the bounds of the elements do, which have to stay well below it."""
    gen = torch.Generator().manual_seed(17)
    B, H, Hkv, Sq, Sk, D = 2, 4, 2, 40, 50, 32
    cpu, gpu = make_qkv(gen, dt, B, H, Hkv, Sq, Sk, D, "dense")
    do = rand(gen, B, Sq, H, D, dtype=dt)
    m = torch.rand(B, Sk, generator=gen) < 0.7
    refs, bounds = attention_reference(*cpu, do, True, m, 0.3)
    leaves = [t.detach().requires_grad_() for t in gpu]
    grads = torch.autograd.grad(tokens.attention(*leaves, causal=True, key_mask=m.cuda(), scale=0.3), leaves, do.cuda())

    def value(x):
        q, k, v = (t.transpose(1, 2) for t in x)
        k, v = k.repeat_interleave(H // Hkv, 1), v.repeat_interleave(H // Hkv, 1)
        seen = m[:, None, None] & torch.ones(Sq, Sk, dtype=torch.bool).tril(Sk - Sq)
        s = torch.where(seen, 0.3 * q @ k.transpose(2, 3), torch.finfo(torch.float64).min)
        return ((torch.softmax(s, -1) * seen.any(-1, keepdim=True) @ v).transpose(1, 2) * do.double()).sum()
    x0 = [t.double() for t in cpu]
    for i in range(3):
        d = refs[i + 1] / refs[i + 1].square().mean().sqrt()
        h = 1e-4
        up, down = ([t + (h * s * d if j == i else 0) for j, t in enumerate(x0)] for s in (1, -1))
        slope = float((value(up) - value(down)) / (2 * h))
        got = float((grads[i].cpu().double() * d).sum())
        limit = float((bounds[i + 1] * d.abs()).sum()) + 1e-4 * abs(slope)
        assert limit <= 0.25 * slope, (i, limit, slope)
        assert abs(got - slope) <= limit, (i, got, slope, limit)


# --------------------------------------------------------------------------- #
# workspaces                                                                   #
# --------------------------------------------------------------------------- #
def guarded(need, behind=1 << 20):
    """`need` bytes and `behind` more that hold a pattern; the check that the pattern is whole."""
    buf = torch.full((need + behind,), 0xA5, dtype=torch.uint8, device="cuda")
    return buf.data_ptr() if need else None, lambda: bool((buf[need:] == 0xA5).all())


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D", [(1, 8, 2, 1, 5000, 64), (2, 4, 4, 1, 5003, 128), (2, 4, 2, 16, 5000, 64), (1, 2, 2, 200, 3001, 64),
                                              (1, 4, 2, 2500, 300, 128), (1, 1, 1, 33, 2000, 8)])
def test_attention_stays_inside_its_workspace(dt, B, H, Hkv, Sq, Sk, D):
    """Through the C entry points, with exactly the bytes that they ask for: nothing behind them is written, and the results
    are those of the public function.  With and without a mask and causal order, for which the splits differ."""
    lib, code = _lib.load_ctypes(), 1 if dt == BF else 0
    gen = torch.Generator().manual_seed(18)
    _, (q, k, v) = make_qkv(gen, dt, B, H, Hkv, Sq, Sk, D, "dense")
    do, m = rand(gen, B, Sq, H, D, dtype=dt).cuda(), (torch.rand(B, Sk, generator=gen) < 0.8).cuda()
    words = torch.empty(B, (Sk + 63) // 64, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    st = torch.cuda.current_stream().cuda_stream
    assert lib.cg_attention_mask_words(words.data_ptr(), m.data_ptr(), Sk, B, Sk, st) == 0
    at = lambda t: (t.data_ptr(), *t.stride()[:3])  # noqa: E731
    for masked in (False, True):
        for causal in (0, 1):
            args = (words.data_ptr() if masked else None, B, H, Hkv, Sq, Sk, D, D ** -0.5, causal, code)
            o, low, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(B, H, Sq, device="cuda")
            rest = low.data_ptr() if dt == BF else None
            need = lib.cg_attention_fwd_workspace_bytes(B, H, Hkv, Sq, Sk, D, code)
            ws, whole = guarded(need)
            assert lib.cg_attention_fwd_low(o.data_ptr(), rest, lse.data_ptr(), *at(q), *at(k), *at(v), *args, ws, need, st) == 0
            assert whole()
            dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
            need = lib.cg_attention_bwd_workspace_bytes(B, H, Hkv, Sq, Sk, D, code)
            ws, whole = guarded(need)
            assert lib.cg_attention_bwd_low(dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *at(do), o.data_ptr(), rest, lse.data_ptr(),
                                            *at(q), *at(k), *at(v), *args, ws, need, st) == 0
            assert whole()
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            want = tokens.attention(*leaves, causal=bool(causal), key_mask=m if masked else None)
            for a, b in zip((o, dq, dk, dv), (want, *torch.autograd.grad(want, leaves, do))):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(5, 33, 41), (70, 90, 9001), (300, 1000, 1000), (129, 257, 513), (2, 77, 129), (2100, 2050, 72)])
def test_linear_stays_inside_its_workspace(dt, M, N, K):
    lib, code = _lib.load_ctypes(), 1 if dt == BF else 0
    gen = torch.Generator().manual_seed(19)
    x, w, b, dy = (rand(gen, *s, dtype=dt).cuda() for s in ((M, K), (N, K), (N,), (M, N)))
    torch.cuda.synchronize()
    st = torch.cuda.current_stream().cuda_stream
    for act, name in ((0, "none"), (2, "gelu")):
        y, z = torch.empty_like(dy), torch.empty_like(dy)
        need = lib.cg_linear_fwd_workspace_bytes(M, N, K, code)
        ws, whole = guarded(need)
        assert lib.cg_linear_fwd(y.data_ptr(), N, z.data_ptr(), N, x.data_ptr(), K, w.data_ptr(), K, b.data_ptr(), None, 0, M, N, K, act,
                                 0.0, code, ws, need, st) == 0
        assert whole()
        dx, dw, db = (torch.empty_like(t) for t in (x, w, b))
        need = lib.cg_linear_bwd_workspace_bytes(M, N, K, code)
        ws, whole = guarded(need)
        assert lib.cg_linear_bwd(dx.data_ptr(), K, dw.data_ptr(), db.data_ptr(), dy.data_ptr(), N, z.data_ptr(), N, x.data_ptr(), K,
                                 w.data_ptr(), K, M, N, K, act, 0.0, code, ws, need, st) == 0
        assert whole()
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        want = tokens.linear(*leaves, activation=name)
        for a, c in zip((y, dx, dw, db), (want, *torch.autograd.grad(want, leaves, dy))):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("M,N", [(3, 7), (5000, 72), (1100, 2049), (300, 12289), (70, 32769)])
def test_layer_norm_stays_inside_its_workspace(dt, M, N):
    lib, code = _lib.load_ctypes(), 1 if dt == BF else 0
    gen = torch.Generator().manual_seed(20)
    x, w, b, dy = (rand(gen, *s, dtype=dt).cuda() for s in ((M, N), (N,), (N,), (M, N)))
    y, dx, dw, db = (torch.empty_like(t) for t in (x, x, w, b))
    mean, rstd = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    torch.cuda.synchronize()
    st = torch.cuda.current_stream().cuda_stream
    assert lib.cg_ln_fwd(y.data_ptr(), N, None, 0, x.data_ptr(), N, None, 0, w.data_ptr(), b.data_ptr(), 1e-5, mean.data_ptr(),
                         rstd.data_ptr(), M, N, code, code, st) == 0
    need = lib.cg_ln_bwd_workspace_bytes(M, N, code)
    ws, whole = guarded(need)
    assert lib.cg_ln_bwd(dx.data_ptr(), N, dy.data_ptr(), N, None, 0, x.data_ptr(), N, None, 0, w.data_ptr(), mean.data_ptr(),
                         rstd.data_ptr(), dw.data_ptr(), db.data_ptr(), M, N, code, code, ws, need, st) == 0
    assert whole()
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    want = tokens.layer_norm(*leaves)
    for a, c in zip((y, dx, dw, db), (want, *torch.autograd.grad(want, leaves, dy))):
        assert torch.equal(a, c)


@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D,gain", [(4, 4, 2, 17, 2, 128, 3.0), (4, 8, 8, 2, 2, 64, 1.0), (2, 4, 4, 40, 300, 64, 6.0), (2, 2, 2, 300, 300, 128, 8.0),
                                                   (4, 4, 4, 1, 3, 64, 2.0), (2, 4, 1, 4, 2000, 32, 6.0)])
def test_gradients_where_one_key_has_the_weight(B, H, Hkv, Sq, Sk, D, gain):
    """bf16.  There dp - delta is a small difference of large sums: with delta from o as it was rounded, the root of the mean
    square error of dq was 4.8 to 6 thousandths of dq's own in four of these six.  With what the rounding left of o it is that
    of ds and dq alone, whose relative errors are spread evenly over a step (2^-8 to 2^-7 of the value): 2^-7 / sqrt(12) each
    at most, sqrt(2) of that together; the scores' own float32 errors and the rounded p in o come on top, a quarter of it."""
    gen = torch.Generator().manual_seed(23)
    q, k, v, do = (rand(gen, B, s, h, D, dtype=BF, scale=g) for s, h, g in ((Sq, H, gain), (Sk, Hkv, 1), (Sk, Hkv, 1), (Sq, H, 1)))
    refs, _ = attention_reference(q, k, v, do, False, None, D ** -0.5)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    for what, got, ref in zip(("dq", "dk"), torch.autograd.grad(tokens.attention(*leaves), leaves, do.cuda()), refs[1:]):
        err = float((got.cpu().double() - ref).norm() / ref.norm())
        assert err <= 1.25 * 2 ** 0.5 * 2 ** -7 / 12 ** 0.5, (what, err)


@pytest.mark.parametrize("dt", [F32, BF], ids=["float32", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D", [(2, 4, 2, 1, 700, 64), (2, 4, 2, 16, 300, 64), (1, 2, 2, 150, 200, 128), (1, 1, 1, 1, 90, 32)])
def test_attention_entry_points_without_the_rest_of_o(dt, B, H, Hkv, Sq, Sk, D):
    """cg_attention_fwd and cg_attention_bwd: the same results, and gradients within the bounds that count o's rounding in
    delta; in float32, where there is no rest, the same gradients."""
    lib, code = _lib.load_ctypes(), 1 if dt == BF else 0
    gen = torch.Generator().manual_seed(24)
    cpu, (q, k, v) = make_qkv(gen, dt, B, H, Hkv, Sq, Sk, D, "dense")
    do = rand(gen, B, Sq, H, D, dtype=dt)
    refs, bounds = attention_reference(*cpu, do, False, None, D ** -0.5)
    leaves, do = [t.detach().requires_grad_() for t in (q, k, v)], do.cuda()
    want = tokens.attention(*leaves)
    grads = torch.autograd.grad(want, leaves, do)
    st = torch.cuda.current_stream().cuda_stream
    at = lambda t: (t.data_ptr(), *t.stride()[:3])  # noqa: E731
    args = (None, B, H, Hkv, Sq, Sk, D, D ** -0.5, 0, code)
    o, lse = torch.empty_like(q), torch.empty(B, H, Sq, device="cuda")
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    n = max(lib.cg_attention_fwd_workspace_bytes(B, H, Hkv, Sq, Sk, D, code), lib.cg_attention_bwd_workspace_bytes(B, H, Hkv, Sq, Sk, D, code))
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert lib.cg_attention_fwd(o.data_ptr(), lse.data_ptr(), *at(q), *at(k), *at(v), *args, ws.data_ptr(), n, st) == 0
    assert lib.cg_attention_bwd(dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *at(do), o.data_ptr(), lse.data_ptr(), *at(q), *at(k), *at(v),
                                *args, ws.data_ptr(), n, st) == 0
    assert torch.equal(o, want)
    for what, got, ref, b, g in zip(("dq", "dk", "dv"), (dq, dk, dv), refs[1:], bounds[1:], grads):
        within(got, ref, b, what)
        assert torch.equal(got, g) or dt == BF and what != "dv"

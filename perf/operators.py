"""The token operators' measured cases: self- and cross-attention over any number of tokens, LayerNorm with an
optional residual sum, and the dense layer with bias, activation and residual, forward alone and forward with backward.

A case is a dict of plain values; prepare() makes its inputs on the GPU, run() is one pass of the operator - in plain
torch where `own` is false, through the package's public functions where it is true -, exact() the same outputs in 64
bits from the definition, work() the bytes and operations that no implementation can do without.

Attention (op "attn"):  q (B, Sq, H, D), k and v (B, Sk, Hkv, D); query head h reads key head h // (H / Hkv);
  s = scale q k^T; key j is hidden from row i where the cell's key mask is false, or (causal) where j > i + Sk - Sq;
  o = softmax(s) v over the visible keys, 0 where there is none.
LayerNorm (op "ln"):  s = x + residual;  y = (s - mean) / sqrt(var + eps) * weight + bias over the last axis.
Dense layer (op "linear"):  y = act(x weight^T + bias) + residual, x (M, K), weight (N, K);  act is the identity, leaky
  (a < 0 multiplied by 0.2), gelu (a times the normal distribution function at a) or silu (a / (1 + exp(-a))).
"""
import math

import torch

own = False

BF16, F32 = "bfloat16", "float32"


def _attn(name, dtype, train, B, H, Hkv, Sq, Sk, D, causal=False, mask="none", packed=False):
    c = dict(op="attn", dtype=dtype, train=train, B=B, H=H, Hkv=Hkv, Sq=Sq, Sk=Sk, D=D, causal=causal, mask=mask,
             packed=packed)
    return dict(c, name=name) if name else c


def _ln(name, dtype, train, M, N, residual, affine=True):
    c = dict(op="ln", dtype=dtype, train=train, M=M, N=N, residual=residual, affine=affine)
    return dict(c, name=name) if name else c


def _linear(name, dtype, train, M, N, K, act="none", residual=False, bias=True):
    c = dict(op="linear", dtype=dtype, train=train, M=M, N=N, K=K, act=act, residual=residual, bias=bias)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one pooling query over the tokens of one cell: answering for a single cell, latency counts
        _attn("pool one cell", F32, False, 1, 8, 8, 1, 513, 64),
        # one new token against a long stored context, keys and values shared by four heads
        _attn("one query, 65537 keys", BF16, False, 4, 32, 8, 1, 65537, 128),
        # embedding a batch of cells: each has its own number of expressed genes, the rest of its tokens is padding
        _attn("embed padded cells", BF16, False, 16, 8, 8, 2000, 2000, 64, mask="ragged", packed=True),
        # sixteen latent tokens of a cell read its expressed genes among 5000 gene tokens, training
        _attn("16 latents read 5000 genes", BF16, True, 32, 8, 8, 16, 5000, 64, mask="ragged"),
        # training of a token encoder in float32, an odd number of genes
        _attn("train 1000 genes float32", F32, True, 8, 8, 8, 1000, 1000, 64, packed=True),
        # training of a causal model over long token sequences with shared key heads: the largest
        _attn("train causal 8192", BF16, True, 1, 32, 8, 8192, 8192, 128, causal=True),
        # the sixteen latent tokens of one cell
        _ln("one cell's 16 tokens", F32, False, 16, 128, True),
        # whole expression rows of a batch of cells, 20 000 genes
        _ln("train 512 x 20000 float32", F32, True, 512, 20000, False),
        # pre-norm residual stream in bfloat16, training
        _ln("train 32768 x 1024", BF16, True, 32768, 1024, True),
        # the layer that ends a feed-forward block, on one token
        _linear("one token 4096 to 1024", BF16, False, 1, 1024, 4096, residual=True),
        # first encoder layer of a batch of cells, 5000 genes to 2048, training
        _linear("train 512 x 5000 to 2048", F32, True, 512, 2048, 5000, act="leaky"),
        # the layer that opens a feed-forward block, on a batch's tokens, training
        _linear("train 8192 x 1024 to 4096", BF16, True, 8192, 4096, 1024, act="gelu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice([BF16, BF16, F32])
    train = rng.random() < 0.6
    op = rng.choice(["attn", "attn", "ln", "linear"])
    if op == "linear":
        N, K = _log(rng, 16, 5000), _log(rng, 16, 5000)
        top = (1 << 35) // (1 if dtype == BF16 else 8)
        return _linear(None, dtype, train, _log(rng, 1, max(2, min(32768, top // (N * K)))), N, K,
                       rng.choice(["none", "leaky", "gelu", "silu"]), rng.random() < 0.5, rng.random() < 0.8)
    if op == "ln":
        N = _log(rng, 16, 20000)
        top = (1 << 28) // (1 if dtype == BF16 else 4)
        return _ln(None, dtype, train, _log(rng, 1, max(2, min(65536, top // N))), N, rng.random() < 0.5, rng.random() < 0.9)
    D = rng.choice([16, 32, 40, 64, 64, 64, 80, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([1, 1, 1, 2, 4])
    B = _log(rng, 1, 16)
    form = rng.choice(["self", "self", "self", "cross", "one"])
    if form == "one":
        return _attn(None, dtype, False, B, H, Hkv, 1, _log(rng, 1, 32768), D, mask=rng.choice(["none", "ragged"]))
    # no more score entries than the largest listed case has at the matrix rate of the type
    most = (1 << 30) if dtype == BF16 else (1 << 27)
    Sk = _log(rng, 16, min(8192, math.sqrt(most / (B * H))))
    Sq = Sk if form == "self" else _log(rng, 2, max(3, min(8192, most // (B * H * Sk))))
    causal = rng.random() < 0.4
    mask = "none" if causal else rng.choice(["none", "ragged", "scatter"])
    return _attn(None, dtype, train, B, H, Hkv, Sq, Sk, D, causal, mask, form == "self" and rng.random() < 0.5)


def _lengths(case):
    """Visible keys of each cell under a "ragged" mask, before the seed puts them in order: half of them to all."""
    B, Sk = case["B"], case["Sk"]
    return [max(1, Sk - (Sk // 2) * b // max(1, B - 1)) for b in range(B)]


def prepare(case, seed):
    dev, dt = torch.device("cuda"), getattr(torch, case["dtype"])
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dt)
    st = dict(case)
    if case["op"] == "ln":
        M, N = case["M"], case["N"]
        # a token row with a level of its own, as the sums of a residual stream have
        st["x"] = (torch.randn(M, N, generator=gen, device=dev) + 0.5 * torch.randn(M, 1, generator=gen, device=dev)).to(dt)
        st["residual"] = rand(M, N, scale=2.0) if case["residual"] else None
        st["weight"] = (1 + 0.2 * torch.randn(N, generator=gen, device=dev)).to(dt) if case["affine"] else None
        st["bias"] = rand(N, scale=0.2) if case["affine"] else None
        names = ("x", "residual", "weight", "bias")
        if case["train"]:
            st["dy"] = rand(M, N)
            st["ds"] = rand(M, N) if case["residual"] else None
    elif case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        st["x"], st["weight"] = rand(M, K), rand(N, K, scale=K ** -0.5)
        st["bias"] = rand(N, scale=0.5) if case["bias"] else None
        st["residual"] = rand(M, N) if case["residual"] else None
        names = ("x", "weight", "bias", "residual")
        if case["train"]:
            st["dy"] = rand(M, N)
    else:
        B, Sq, Sk, H, Hkv, D = (case[n] for n in ("B", "Sq", "Sk", "H", "Hkv", "D"))
        if case["packed"]:      # views of one projection's output, as a fused q, k, v product leaves them
            qkv = rand(B, Sk, H + 2 * Hkv, D)
            st["q"], st["k"], st["v"] = qkv[:, :, :H].detach(), qkv[:, :, H:H + Hkv].detach(), qkv[:, :, H + Hkv:].detach()
        else:
            st["q"], st["k"], st["v"] = rand(B, Sq, H, D), rand(B, Sk, Hkv, D), rand(B, Sk, Hkv, D)
        st["key_mask"] = None
        if case["mask"] == "ragged":
            lengths = torch.tensor(_lengths(case), device=dev)[torch.randperm(B, generator=gen, device=dev)]
            st["key_mask"] = torch.arange(Sk, device=dev)[None] < lengths[:, None]
        elif case["mask"] == "scatter":     # genes hidden at random; one cell of several may have none left
            m = torch.rand(B, Sk, generator=gen, device=dev) < 0.7
            if B > 2:
                m[int(torch.randint(B, (1,), generator=gen, device=dev))] = False
            st["key_mask"] = m
        names = ("q", "k", "v")
        if case["train"]:
            st["do"] = rand(B, Sq, H, D)
    if case["train"]:
        st["leaves"] = [st[n].requires_grad_() for n in names if st[n] is not None]
    return st


def _visible(st):
    """(B or 1, 1, Sq or 1, Sk) truth values: which keys a row sees; None: all."""
    Sq, Sk, seen = st["Sq"], st["Sk"], None
    if st["key_mask"] is not None:
        seen = st["key_mask"][:, None, None, :]
    if st["causal"]:
        i = torch.arange(Sq, device=st["q"].device)
        j = torch.arange(Sk, device=st["q"].device)
        below = (j[None, :] <= i[:, None] + (Sk - Sq))[None, None]
        seen = below if seen is None else seen & below
    return seen


def _plain_attn(st):
    dt, G = st["q"].dtype, st["H"] // st["Hkv"]
    q = st["q"].float().transpose(1, 2).contiguous()
    k = st["k"].float().transpose(1, 2).repeat_interleave(G, 1)
    v = st["v"].float().transpose(1, 2).repeat_interleave(G, 1)
    scale = st["D"] ** -0.5
    s = torch.matmul(q * scale, k.transpose(2, 3).contiguous())
    seen = _visible(st)
    if seen is not None:
        s = torch.where(seen, s, float("-inf"))
    top = s.max(-1, keepdim=True).values
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p, v)
    out = o.transpose(1, 2).to(dt).contiguous()
    if not st["train"]:
        return out
    do = st["do"].float().transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    B, Sk, Hkv, D = st["B"], st["Sk"], st["Hkv"], st["D"]
    dk, dv = (t.view(B, Hkv, G, Sk, D).sum(2) for t in (dk, dv))
    return [out] + [t.transpose(1, 2).to(dt).contiguous() for t in (dq, dk, dv)]


def _plain_ln(st, eps=1e-5):
    dt = st["x"].dtype
    s = st["x"].float()
    if st["residual"] is not None:
        s = s + st["residual"].float()
    c = s - s.mean(-1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
    xhat = c * rstd
    y = xhat
    if st["affine"]:
        y = y * st["weight"].float() + st["bias"].float()
    outs = [y.to(dt)] + ([s.to(dt)] if st["residual"] is not None else [])
    if not st["train"]:
        return outs
    dy = st["dy"].float()
    g = dy * st["weight"].float() if st["affine"] else dy
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    if st["residual"] is not None:
        dx = dx + st["ds"].float()
        outs += [dx.to(dt), dx.to(dt)]
    else:
        outs += [dx.to(dt)]
    if st["affine"]:
        outs += [(dy * xhat).sum(0).to(dt), dy.sum(0).to(dt)]
    return outs


def _plain_linear(st):
    dt, act = st["x"].dtype, st["act"]
    x, w = st["x"].float(), st["weight"].float()
    a = torch.matmul(x, w.t())
    if st["bias"] is not None:
        a = a + st["bias"].float()
    if act == "leaky":
        slope = torch.where(a > 0, 1.0, 0.2)
        y = a * slope
    elif act == "gelu":
        below = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        y = a * below
        slope = below + a * torch.exp(-0.5 * a * a) * (1 / math.sqrt(2 * math.pi))
    elif act == "silu":
        gate = 1 / (1 + torch.exp(-a))
        y = a * gate
        slope = gate * (1 + a * (1 - gate))
    else:
        y, slope = a, None
    if st["residual"] is not None:
        y = y + st["residual"].float()
    if not st["train"]:
        return y.to(dt)
    da = st["dy"].float() if slope is None else st["dy"].float() * slope
    outs = [y.to(dt), torch.matmul(da, w).to(dt), torch.matmul(da.t(), x).to(dt)]
    if st["bias"] is not None:
        outs.append(da.sum(0).to(dt))
    if st["residual"] is not None:
        outs.append(st["dy"].clone())
    return outs


def _own_linear(st):
    from cycle_gan_rna_amd.tokens import linear
    if not st["train"]:
        with torch.no_grad():
            return linear(st["x"], st["weight"], st["bias"], activation=st["act"], slope=0.2, residual=st["residual"])
    y = linear(st["x"], st["weight"], st["bias"], activation=st["act"], slope=0.2, residual=st["residual"])
    return [y.detach(), *torch.autograd.grad(y, st["leaves"], st["dy"])]


def _own_attn(st):
    from cycle_gan_rna_amd.tokens import attention
    if not st["train"]:
        with torch.no_grad():
            return attention(st["q"], st["k"], st["v"], causal=st["causal"], key_mask=st["key_mask"])
    o = attention(st["q"], st["k"], st["v"], causal=st["causal"], key_mask=st["key_mask"])
    return [o.detach(), *torch.autograd.grad(o, st["leaves"], st["do"])]


def _own_ln(st):
    from cycle_gan_rna_amd.tokens import layer_norm
    if not st["train"]:
        with torch.no_grad():
            out = layer_norm(st["x"], st["weight"], st["bias"], residual=st["residual"])
        return list(out) if st["residual"] is not None else [out]
    out = layer_norm(st["x"], st["weight"], st["bias"], residual=st["residual"])
    if st["residual"] is not None:
        return [t.detach() for t in out] + list(torch.autograd.grad(out, st["leaves"], (st["dy"], st["ds"])))
    return [out.detach(), *torch.autograd.grad(out, st["leaves"], st["dy"])]


def run(state):
    if own:
        return {"attn": _own_attn, "ln": _own_ln, "linear": _own_linear}[state["op"]](state)
    with torch.no_grad():
        return {"attn": _plain_attn, "ln": _plain_ln, "linear": _plain_linear}[state["op"]](state)


def exact(case, seed):
    """One head at a time in float64, gradients by differentiation of the definition."""
    st = prepare(case, seed)
    if case["op"] == "ln":
        keep = dict(zip(("x", "residual", "weight", "bias"),
                        (None if st[n] is None else st[n].detach().double().requires_grad_(case["train"])
                         for n in ("x", "residual", "weight", "bias"))))
        s = keep["x"] if keep["residual"] is None else keep["x"] + keep["residual"]
        var, mean = torch.var_mean(s, -1, unbiased=False, keepdim=True)
        y = (s - mean) / (var + 1e-5).sqrt()
        if case["affine"]:
            y = y * keep["weight"] + keep["bias"]
        outs = [y] if keep["residual"] is None else [y, s]
        if not case["train"]:
            return outs
        leaves = [t for t in keep.values() if t is not None]
        cot = [st["dy"].double()] + ([st["ds"].double()] if keep["residual"] is not None else [])
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, cot))
    if case["op"] == "linear":
        names = [n for n in ("x", "weight", "bias", "residual") if st[n] is not None]
        keep = {n: st[n].detach().double().requires_grad_(case["train"]) for n in names}
        y = keep["x"] @ keep["weight"].T
        if "bias" in keep:
            y = y + keep["bias"]
        if case["act"] == "leaky":
            y = torch.maximum(y, torch.zeros_like(y)) + 0.2 * torch.minimum(y, torch.zeros_like(y))
        elif case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        elif case["act"] == "silu":
            y = y * torch.special.expit(y)
        if "residual" in keep:
            y = y + keep["residual"]
        if not case["train"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, list(keep.values()), st["dy"].double())]
    B, Sq, Sk, H, Hkv, D = (case[n] for n in ("B", "Sq", "Sk", "H", "Hkv", "D"))
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    reach = None
    if case["causal"]:
        reach = torch.ones(Sq, Sk, dtype=torch.bool, device=q.device).tril(Sk - Sq)
    for b in range(B):
        seen = reach
        if st["key_mask"] is not None:
            row = st["key_mask"][b].expand(Sq, Sk)
            seen = row if seen is None else seen & row
        some = None if seen is None else seen.any(-1, keepdim=True)
        for h in range(H):
            kv = h // (H // Hkv)
            a, c, e = (t.clone().requires_grad_(case["train"]) for t in (q[b, :, h], k[b, :, kv], v[b, :, kv]))
            s = a @ c.T / math.sqrt(D)
            if seen is None:
                p = torch.softmax(s, -1)
            else:       # a row that sees nothing: scores of one value, then weights of zero
                p = torch.softmax(s.masked_fill(~seen & some, float("-inf")), -1) * some
            o = p @ e
            out[b, :, h] = o.detach()
            if case["train"]:
                ga, gc, ge = torch.autograd.grad(o, (a, c, e), st["do"][b, :, h].double())
                dq[b, :, h] = ga
                dk[b, :, kv] += gc
                dv[b, :, kv] += ge
    return [out, dq, dk, dv] if case["train"] else out


def work(case):
    size = 2 if case["dtype"] == BF16 else 4
    if case["op"] == "ln":
        M, N = case["M"], case["N"]
        tensors = 2 + (2 if case["residual"] else 0)        # x, y and residual, s
        flops = 8 * M * N
        if case["train"]:
            tensors += 2 + (1 if case["residual"] else 0)   # dy, dx and ds; x is read once
            flops += 14 * M * N
        small = (2 + (2 if case["train"] else 0)) * N if case["affine"] else 0
        return {"bytes": size * (tensors * M * N + small), "flops": flops}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        edge = M * N * (2 if case["residual"] else 1) + (N if case["bias"] else 0)     # y, residual, bias
        if not case["train"]:
            return {"bytes": size * (M * K + N * K + edge), "flops": 2 * M * N * K}
        # dy, dx, the weight's and the bias's gradient (the residual's is dy)
        return {"bytes": size * (2 * M * K + 2 * N * K + edge + M * N + (N if case["bias"] else 0)), "flops": 6 * M * N * K}
    B, Sq, Sk, H, Hkv, D = (case[n] for n in ("B", "Sq", "Sk", "H", "Hkv", "D"))
    pairs = Sq * Sk
    if case["causal"]:
        n = min(Sq, Sk)
        pairs = n * (n + 1) // 2 + max(Sk - Sq, 0) * Sq
    share = {"none": 1.0, "ragged": sum(_lengths(case)) / (B * Sk),
             "scatter": 0.7 * ((B - 1) / B if B > 2 else 1.0)}[case["mask"]]
    pairs = share * pairs * B * H
    rows = 2 * B * Sq * H * D                               # q and o
    keys = 2 * B * Sk * Hkv * D * share                     # k and v, as far as they are seen
    mask = 0 if case["mask"] == "none" else B * Sk
    if not case["train"]:
        return {"bytes": int(size * (rows + keys) + mask), "flops": int(4 * pairs * D)}
    # do and dq beside q and o; dk and dv whole
    return {"bytes": int(size * (2 * rows + keys + 2 * B * Sk * Hkv * D) + mask), "flops": int(14 * pairs * D)}

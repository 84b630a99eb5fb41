"""Token operators without a GPU: what the public functions and the C entry points refuse.  Nothing is launched: every
call here ends in the host's argument checks."""
import ctypes as C

import pytest
import torch

from cycle_gan_rna_amd import _lib, tokens

BF, F32 = torch.bfloat16, torch.float32


def z(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("q,k,v,kw,match", [
    (z(2, 3, 4, 8), z(2, 5, 4, 8), z(2, 5, 4, 8, dtype=BF), {}, "v is torch.bfloat16"),
    (z(2, 3, 4, 8).double(), z(2, 5, 4, 8).double(), z(2, 5, 4, 8).double(), {}, "float32 or bfloat16"),
    (z(3, 4, 8), z(2, 5, 4, 8), z(2, 5, 4, 8), {}, r"\(B, Sq, H, D\)"),
    (z(2, 3, 4, 8), z(2, 5, 3, 8), z(2, 5, 3, 8), {}, "does not go with"),          # 4 heads over 3
    (z(2, 3, 4, 8), z(2, 5, 0, 8), z(2, 5, 0, 8), {}, "does not go with"),
    (z(2, 3, 4, 8), z(1, 5, 4, 8), z(1, 5, 4, 8), {}, "does not go with"),
    (z(2, 3, 4, 8), z(2, 5, 4, 8), z(2, 6, 4, 8), {}, "does not go with"),
    (z(2, 3, 4, 8), z(2, 5, 4, 16), z(2, 5, 4, 16), {}, "does not go with"),
    (z(1, 3, 1, 6), z(1, 5, 1, 6), z(1, 5, 1, 6), {}, "head dimensions"),
    (z(1, 3, 1, 12, dtype=BF), z(1, 5, 1, 12, dtype=BF), z(1, 5, 1, 12, dtype=BF), {}, "head dimensions"),
    (z(1, 3, 1, 136), z(1, 5, 1, 136), z(1, 5, 1, 136), {}, "head dimensions"),
    (z(1, 3, 1, 8), z(1, 5, 1, 8), z(1, 5, 1, 8), {"scale": 0.0}, "positive"),
    (z(1, 3, 1, 8), z(1, 5, 1, 8), z(1, 5, 1, 8), {"scale": -1.0}, "positive"),
    (z(1, 3, 1, 8), z(1, 5, 1, 8), z(1, 5, 1, 8), {"scale": float("nan")}, "positive"),
    (z(2, 3, 1, 8), z(2, 5, 1, 8), z(2, 5, 1, 8), {"key_mask": torch.ones(2, 6, dtype=torch.bool)}, "key_mask"),
    (z(2, 3, 1, 8), z(2, 5, 1, 8), z(2, 5, 1, 8), {"key_mask": torch.ones(2, 5)}, "key_mask"),
])
def test_attention_refuses(q, k, v, kw, match):
    with pytest.raises(ValueError, match=match):
        tokens.attention(q, k, v, **kw)


@pytest.mark.parametrize("x,w,b,kw,match", [
    (z(4, 0), None, None, {}, "last axis"),
    (z(4, 8).double(), None, None, {}, "float32 or bfloat16"),
    (z(4, 8), z(7), None, {}, "weight"),
    (z(4, 8), z(8, dtype=BF), None, {}, "weight is torch.bfloat16"),        # float32 rows take float32 parameters
    (z(4, 8, dtype=BF), z(8), z(8, dtype=BF), {}, "weight is torch.float32, bias"),
    (z(4, 8), None, None, {"residual": z(4, 7)}, "residual"),
    (z(4, 8), None, None, {"residual": z(4, 8, dtype=BF)}, "residual"),
    (z(4, 8), None, None, {"eps": -1e-5}, "eps"),
    (z(4, 8), None, None, {"eps": float("inf")}, "eps"),
])
def test_layer_norm_refuses(x, w, b, kw, match):
    with pytest.raises(ValueError, match=match):
        tokens.layer_norm(x, w, b, **kw)


@pytest.mark.parametrize("x,w,b,kw,match", [
    (z(4, 8), z(3, 7), None, {}, "does not go with"),
    (z(4, 8), z(0, 8), None, {}, "does not go with"),
    (z(4, 8), z(3, 8, dtype=BF), None, {}, "weight is torch.bfloat16"),
    (z(4, 8), z(3, 8), z(4), {}, "bias"),
    (z(4, 8), z(3, 8), None, {"residual": z(4, 8)}, "residual"),
    (z(4, 8), z(3, 8), None, {"activation": "tanh"}, "activation"),
    (z(4, 8), z(3, 8), None, {"activation": "leaky", "slope": float("nan")}, "slope"),
])
def test_linear_refuses(x, w, b, kw, match):
    with pytest.raises(ValueError, match=match):
        tokens.linear(x, w, b, **kw)


def test_cpu_tensors_are_refused():
    q = z(1, 2, 1, 8)
    for call in (lambda: tokens.attention(q, q, q), lambda: tokens.layer_norm(q), lambda: tokens.linear(z(2, 8), z(3, 8))):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


P = C.c_void_p(1 << 20)          # a device address that nothing may touch: the checks come first


def attn(lib, D=64, H=4, Hkv=2, Sq=8, Sk=8, scale=0.1, dtype=1, q=P, strides=None, words=None, ws=None, nws=0, B=2):
    st = strides or (Sk * H * D, H * D, D)
    return lib.cg_attention_fwd(P, None, q, *st, P, *st, P, *st, words, B, H, Hkv, Sq, Sk, D, scale, 0, dtype, ws, nws, None)


def test_attention_entry_point_refuses():
    lib = _lib.load_ctypes()
    assert attn(lib, H=3) == -1                              # query heads are not whole groups
    assert attn(lib, dtype=2) == -1
    assert attn(lib, scale=0.0) == -1 and attn(lib, scale=float("nan")) == -1
    assert attn(lib, q=None) == -1
    assert attn(lib, D=136) == -2 and attn(lib, D=12) == -2 and attn(lib, D=6, dtype=0) == -2
    assert attn(lib, q=C.c_void_p((1 << 20) + 8)) == -2      # address not a multiple of 16
    assert attn(lib, strides=(4096, 260, 64)) == -2          # a token stride that is not whole pieces
    assert attn(lib, strides=(1 << 33, 1 << 24, 64)) == -2   # 64 rows further apart than 2^31 bytes
    need = lib.cg_attention_fwd_workspace_bytes(1, 4, 2, 1, 8192, 64, 1)
    assert need > 0 and attn(lib, B=1, Sq=1, Sk=8192, ws=P, nws=need - 1) == -3
    assert attn(lib, B=1, Sq=1, Sk=8192) == -3
    assert attn(lib, B=0) == 0 and attn(lib, Sq=0) == 0      # nothing to do
    assert lib.cg_attention_mask_words(None, P, 8, 2, 8, None) == -1
    assert lib.cg_attention_mask_words(P, P, 8, 7, (1 << 30) + 1, None) == -1
    st = (8 * 4 * 64, 4 * 64, 64)
    def bwd(ws, n, scale=0.1):
        return lib.cg_attention_bwd(P, P, P, P, *st, P, P, P, *st, P, *st, P, *st, None, 2, 4, 2, 8, 8, 64, scale, 0, 1, ws, n, None)
    need = lib.cg_attention_bwd_workspace_bytes(2, 4, 2, 8, 8, 64, 1)
    assert need >= 2 * 4 * 8 * 8
    assert bwd(P, need - 1) == -3 and bwd(C.c_void_p((1 << 20) + 4), need) == -3 and bwd(P, need, 0.0) == -1


def test_layer_norm_entry_point_refuses():
    lib = _lib.load_ctypes()
    def fwd(M=4, N=8, ld=8, dtype=0, wdtype=0, y=P, mean=None, rstd=None):
        return lib.cg_ln_fwd(y, ld, None, 0, P, ld, None, 0, P, P, 1e-5, mean, rstd, M, N, dtype, wdtype, None)
    assert fwd(N=0) == -1 and fwd(M=-1) == -1 and fwd(ld=7) == -1 and fwd(y=None) == -1
    assert fwd(dtype=0, wdtype=1) == -1 and fwd(dtype=3) == -1
    assert fwd(mean=P) == -1                                  # both statistics or neither
    assert fwd(M=0) == 0
    def bwd(dx=P, dw=P, db=P, ws=P, n=1 << 30, M=4, N=8, ld=8):
        return lib.cg_ln_bwd(dx, ld, P, ld, None, 0, P, ld, None, 0, P, P, P, dw, db, M, N, 0, 0, ws, n, None)
    need = lib.cg_ln_bwd_workspace_bytes(4, 8, 0)
    assert need >= 2 * 8 * 4
    assert bwd(n=need - 1) == -3 and bwd(ws=None) == -3 and bwd(ld=7) == -1 and bwd(None, None, None) == -1
    assert bwd(dw=None, db=None, M=0) == 0


def test_linear_entry_point_refuses():
    lib = _lib.load_ctypes()
    def fwd(M=8, N=16, K=32, act=0, slope=0.0, dtype=1, ldx=None, ws=P, n=1 << 40, y=P):
        return lib.cg_linear_fwd(y, N, None, 0, P, K if ldx is None else ldx, P, K, None, None, 0, M, N, K, act, slope, dtype, ws, n, None)
    assert fwd(N=0) == -1 and fwd(K=0) == -1 and fwd(act=4) == -1 and fwd(dtype=2) == -1 and fwd(slope=float("nan")) == -1
    assert fwd(ldx=31) == -1 and fwd(y=None) == -1 and fwd(M=0) == 0
    assert fwd(K=(1 << 21) + 8) == -2
    need = lib.cg_linear_fwd_workspace_bytes(8, 16, 32, 1)
    assert need > 0 and fwd(n=need - 1) == -3 and fwd(ws=None) == -3
    def bwd(dx=P, dw=P, db=P, act=0, z=None, ws=P, n=1 << 40):
        return lib.cg_linear_bwd(dx, 32, dw, db, P, 16, z, 16, P, 32, P, 32, 8, 16, 32, act, 0.0, 1, ws, n, None)
    need = lib.cg_linear_bwd_workspace_bytes(8, 16, 32, 1)
    assert bwd(None, None, None) == -1 and bwd(act=2) == -1 and bwd(n=need - 1) == -3 and bwd(ws=None) == -3


@pytest.mark.parametrize("dtype", [0, 1])
def test_workspaces_grow_with_what_they_hold(dtype):
    """The sizes are those of the plans the launches use: a monotone sample over the shapes (never negative, never a
    wrapped product)."""
    lib = _lib.load_ctypes()
    for M in (0, 1, 5, 64, 513, 8192, 100000):
        for N in (1, 7, 64, 1000, 20000):
            assert 2 * N * 4 <= lib.cg_ln_bwd_workspace_bytes(M, N, dtype) <= 1024 * 2 * N * 4
            for K in (1, 33, 4096):
                f, b = lib.cg_linear_fwd_workspace_bytes(M, N, K, dtype), lib.cg_linear_bwd_workspace_bytes(M, N, K, dtype)
                assert 0 <= f < 1 << 40 and N * 4 <= b < 1 << 40
    assert lib.cg_attention_fwd_workspace_bytes(64, 16, 16, 4096, 4096, 64, dtype) == 0       # enough rows: no splits
    assert lib.cg_attention_bwd_workspace_bytes(64, 16, 16, 4096, 4096, 64, dtype) == 64 * 16 * 4096 * 8


def each(x):
    """The three operators on (2, 8) values."""
    q = x.view(1, 2, 1, 8)
    return (lambda: tokens.attention(q, q, q), lambda: tokens.layer_norm(x), lambda: tokens.linear(x, z(3, 8)),
            lambda: tokens.attention(z(1, 2, 1, 8), q, z(1, 2, 1, 8)), lambda: tokens.layer_norm(z(2, 8), residual=x),
            lambda: tokens.linear(z(2, 8), z(3, 8), residual=x[:, :3]), lambda: tokens.linear(z(2, 4), z(8, 4), x[0]))


def test_forward_mode_derivatives_are_refused():
    """A result without its tangent would be one whose derivative is silently 0."""
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        for x in (z(2, 8), z(2, 8).requires_grad_()):
            for call in each(fwd.make_dual(x, torch.ones(2, 8))):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()


def test_traces_are_refused():
    """A trace would hold the allocation of the result and not what fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    for i in range(7):
        with pytest.raises(RuntimeError, match="trac"):
            torch.jit.trace(lambda x: each(x)[i](), z(2, 8))
        with pytest.raises(RuntimeError, match="trac"):
            make_fx(lambda x: each(x)[i]())(z(2, 8))


def test_rows_longer_than_2_to_30_are_refused():
    """The kernels count columns in 32 bits and step past the last of them."""
    lib = _lib.load_ctypes()
    for N in ((1 << 30) + 1, (1 << 31) - 8, (1 << 31) - 1):
        assert lib.cg_ln_fwd(P, N, None, 0, P, N, None, 0, None, None, 1e-5, None, None, 1, N, 0, 0, None) == -2
        assert lib.cg_ln_bwd_workspace_bytes(1, N, 1) == 0
        assert lib.cg_ln_bwd(P, N, P, N, None, 0, P, N, None, 0, None, P, P, P, P, 1, N, 1, 1, P, 1 << 50, None) == -2
    with pytest.raises(ValueError, match="columns"):
        tokens.layer_norm(z(1).expand((1 << 30) + 1))
    assert lib.cg_ln_bwd_workspace_bytes(1, 1 << 30, 1) == 2 * 4 << 30


@pytest.mark.parametrize("dtype", [0, 1])
def test_workspaces_hold_what_goes_through_them(dtype):
    """Lower bounds from what a call lays down: padded copies of rows that are not whole 16-byte pieces, the activation's
    gradient and column sums of the dense layer; two partial results at least where attention's keys are split, and two
    float32 values a row of its backward pass."""
    lib, e, size = _lib.load_ctypes(), (4, 8)[dtype], (4, 2)[dtype]
    up = lambda n: -(-n // e) * e  # noqa: E731
    for M in (5, 64, 513, 8192):
        for N in (1, 7, 64, 1000):
            for K in (1, 33, 4096):
                assert lib.cg_linear_fwd_workspace_bytes(M, N, K, dtype) >= (M + N) * up(K) * size
                assert lib.cg_linear_bwd_workspace_bytes(M, N, K, dtype) >= ((M + N) * up(K) + M * up(N)) * size + 4 * N
    split = 0
    for B, H, Hkv, Sq, Sk, D in ((1, 8, 2, 1, 5000, 64), (2, 4, 4, 16, 5000, 64), (1, 2, 2, 200, 3001, 64), (1, 4, 2, 2500, 300, 128),
                                 (64, 16, 16, 512, 512, 32), (1, 1, 1, 1, 1, 8)):
        f = lib.cg_attention_fwd_workspace_bytes(B, H, Hkv, Sq, Sk, D, dtype)
        assert f == 0 or f >= 2 * B * Sq * H * (D + 1) * 4
        b = lib.cg_attention_bwd_workspace_bytes(B, H, Hkv, Sq, Sk, D, dtype)
        assert b >= B * H * Sq * 8
        split += (f > 0) + (b > B * H * Sq * 8 + 16)
    assert split >= 5


def test_attention_entry_points_with_the_rest_of_o_refuse():
    lib = _lib.load_ctypes()
    st = (8 * 4 * 64, 4 * 64, 64)
    off = C.c_void_p((1 << 20) + 8)

    def fwd(low, dtype=1):
        return lib.cg_attention_fwd_low(P, low, None, P, *st, P, *st, P, *st, None, 2, 4, 4, 8, 8, 64, 0.1, 0, dtype, None, 0, None)

    def bwd(low, dtype=1):
        return lib.cg_attention_bwd_low(P, P, P, P, *st, P, low, P, P, *st, P, *st, P, *st, None, 2, 4, 4, 8, 8, 64, 0.1, 0, dtype, None, 0, None)
    assert fwd(P, 0) == -1 and bwd(P, 0) == -1               # float32 has no rest
    assert fwd(off) == -2 and bwd(off) == -2
    assert bwd(None) == -3 and bwd(P) == -3

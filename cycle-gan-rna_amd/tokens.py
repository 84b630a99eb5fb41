"""Token operators for any number of tokens and any width, forward and backward, on MI355X.

The reference's token path has 16 tokens of latent_dim / 16 features (GAN_functions.py:28-56, :81, :138-140), and the
fused kernels behind GeneSelfAttention are built for those.  These are its pieces on their own - the product inside
nn.MultiheadAttention, nn.LayerNorm after a residual sum, nn.Linear with what follows it - for token sets of other
sizes: thousands of genes as tokens, padded batches of cells, a single query that pools a cell, wide features, bf16
storage.

  attention(q, k, v, causal=False, key_mask=None, scale=None)
  layer_norm(x, weight=None, bias=None, residual=None, eps=1e-5)
  linear(x, weight, bias=None, activation="none", slope=0.0, residual=None)

Tensors are float32 or bfloat16 on a HIP device; sums, statistics and the softmax are float32 in either case.  Calls are
enqueued on the device's current stream, allocate through torch's caching allocator (so they can be captured into a HIP
graph after one eager call) and have first-order gradients; forward-mode derivatives and tracing raise RuntimeError.
There is no CPU or eager-PyTorch fallback.  Arguments that do not go together raise ValueError.  A backward pass is
captured on leaves of its own (detach().requires_grad_()): with an eager graph of the same leaves alive, ending the
capture has ended the process.

The arithmetic is in csrc/sdpa.hip, ln.hip and linear.hip behind the C ABI (cg_attention_*, cg_ln_*, cg_linear_*), checks,
memory and autograd in csrc/tokens.cpp.
"""
from __future__ import annotations

from . import _lib


def attention(q, k, v, *, causal=False, key_mask=None, scale=None):
    """softmax(scale q k^T) v per cell and head: the product inside nn.MultiheadAttention (GAN_functions.py:34,53-55).

    q: (B, Sq, H, D);  k, v: (B, Sk, Hkv, D), H a multiple of Hkv: query head h reads key head h // (H / Hkv).
    D: up to 128, a multiple of 8 (bfloat16) or 4 (float32).  Any strides (views of a packed projection are read where
    they are; a layout that breaks 16-byte pieces is copied first).
    causal: key j is visible to row i where j <= i + Sk - Sq.
    key_mask: (B, Sk) bool (or uint8), true where a key of the cell is visible.  Whatever k and v hold at a hidden
        key, NaN included, reaches no result, and its gradients are 0.  (At a key that only `causal` hides from some
        rows, a NaN or infinity may reach those rows.)
    scale: a positive number, default D ** -0.5.
    Returns (B, Sq, H, D) of q's type.  A row that sees no key gives 0, and 0 gradient to q.  A row with a score of +inf or
    NaN, or whose visible scores are all -inf, gives NaN, and NaN to the gradients that it takes part in.  bfloat16: the
    probabilities and the scores' gradients are rounded to bfloat16 for the products with v, q, k and the output's
    gradient.  One query (Sq = 1) or few rows over many keys are split over the keys.  Lengths of 0 are allowed.
    """
    return _lib.load_tokens().attention(q, k, v, causal, key_mask, scale)


def layer_norm(x, weight=None, bias=None, *, residual=None, eps=1e-5):
    """LayerNorm over the last axis, optionally of a residual sum: norm(x + attn) of GAN_functions.py:35,54.

    x: (..., N), any strides, N up to 2^30;  weight, bias: (N,) of x's type or float32, either may be None;  residual: like x.
    Returns y of x's type; with a residual (y, s), where s = x + residual is the residual stream for the next layer (y and
    the gradients are those of the unrounded sum).  eps: not negative.
    """
    return _lib.load_tokens().layer_norm(x, weight, bias, residual, eps)


def linear(x, weight, bias=None, *, activation="none", slope=0.0, residual=None):
    """act(x weight^T + bias) + residual in one product: nn.Linear and what follows it (GAN_functions.py:53-54,59-61,89-98).

    x: (..., K);  weight: (N, K);  bias: (N,) or None;  residual: (..., N) or None; all of one type.
    activation: "none", "leaky" (values a <= 0 times `slope`; 0 is ReLU), "gelu" (a times the normal distribution
        function at a) or "silu" (a / (1 + exp(-a))).
    Returns (..., N).  Products are exact float32 or bf16 with float32 sums; bias, activation and residual are applied in
    float32 and the result is rounded once.  For the backward pass bfloat16 keeps a = x weight^T + bias as rounded to
    bfloat16, and the gradient of a is rounded to bfloat16 for its products with x and weight (the bias's is summed
    before).  Values of gelu are right to a share of themselves however small they are (float32: 2^-20).  Rows of K (and
    for the backward pass N) that are not whole 16-byte pieces cost a padded copy.
    """
    return _lib.load_tokens().linear(x, weight, bias, activation, slope, residual)

"""Python wrappers over ``torch.ops.cuda_transformer`` with fake (meta)
implementations -- the same ten functions, names and argument meaning as the
reference's ``cuda_transformer/ops.py:4-139``, plus this implementation's
LayerNorm and precision-explicit variants, the token-generation operators
(paged key/value cache, one-token attention, logits processing) and those of
speculative decoding (attention of drafted tokens, their verification, moving
and copying what the cache holds).

``precision`` (the ``*_ex`` functions): 0 = 3xTF32 (FP32-accurate, the default
of the plain functions), 1 = TF32, 2 = FP32 on the CUDA cores.  The plain
functions follow the ``CUDA_TRANSFORMER_PRECISION`` environment variable.
"""
import torch
from torch import Tensor

__all__ = [
    "cuda_fma", "db_calculation",
    "cuda_softmax", "cuda_softmax_bwd",
    "gelu_activation", "gelu_activation_bwd",
    "causal_self_attention_fwd", "causal_self_attention_bwd",
    "flash_attention_fwd", "flash_attention_bwd",
    "flash_attention_fwd_ex", "flash_attention_bwd_ex", "cuda_fma_ex",
    "layernorm_fwd", "layernorm_bwd",
    "linear_fused", "linear_accumulate_", "cross_entropy_fwd_bwd_",
    "kv_append_", "rotary_tables", "paged_attention", "paged_attention_workspace",
    "logits_process",
    "tree_attention", "verify_drafts", "kv_compact_", "kv_copy_pages_",
]

PRECISION_3XTF32 = 0
PRECISION_TF32 = 1
PRECISION_FP32 = 2
EPILOGUE_NONE = 0
EPILOGUE_GELU = 1
EPILOGUE_GELU_GRAD = 2


def _f32(*ts):
    for t in ts:
        torch._check(t.dtype == torch.float32)


def _same_device(*ts):
    torch._check(all(t.device == ts[0].device for t in ts))


# ---------------------------------------------------------------- linear layer
def cuda_fma(x: Tensor, weights: Tensor, bias: Tensor) -> Tensor:
    """out[b] = x[b] @ weights[b or 0] + bias (weights pre-transposed, (k, n))."""
    return torch.ops.cuda_transformer.cuda_fma.default(x, weights, bias)


def cuda_fma_ex(x: Tensor, weights: Tensor, bias: Tensor, precision: int) -> Tensor:
    """cuda_fma with an explicit precision mode."""
    return torch.ops.cuda_transformer.cuda_fma_ex.default(x, weights, bias, precision)


def _fma_meta(x, weights, bias):
    _f32(x, weights, bias)
    _same_device(x, weights, bias)
    w = weights if weights.dim() == 3 else weights.unsqueeze(0)
    return torch.empty(x.size(0), x.size(1), w.size(2), dtype=x.dtype, device=x.device)


@torch.library.register_fake("cuda_transformer::cuda_fma")
def _(x, weights, bias):
    return _fma_meta(x, weights, bias)


@torch.library.register_fake("cuda_transformer::cuda_fma_ex")
def _(x, weights, bias, precision):
    return _fma_meta(x, weights, bias)


def db_calculation(dy: Tensor) -> Tensor:
    """Bias gradient: column sum of dy over (batch, m)."""
    return torch.ops.cuda_transformer.db_calculation.default(dy)


@torch.library.register_fake("cuda_transformer::db_calculation")
def _(dy):
    _f32(dy)
    return torch.empty(dy.size(-1), dtype=dy.dtype, device=dy.device)


# --------------------------------------------------------------------- softmax
def cuda_softmax(x: Tensor) -> Tensor:
    """Row softmax over the last dimension of a contiguous 3-D tensor."""
    return torch.ops.cuda_transformer.cuda_softmax.default(x)


@torch.library.register_fake("cuda_transformer::cuda_softmax")
def _(x):
    _f32(x)
    return torch.empty_like(x)


def cuda_softmax_bwd(probs: Tensor, dp: Tensor) -> Tensor:
    """Softmax backward: probs * (dp - sum(probs * dp))."""
    return torch.ops.cuda_transformer.cuda_softmax_bwd.default(probs, dp)


@torch.library.register_fake("cuda_transformer::cuda_softmax_bwd")
def _(probs, dp):
    _f32(probs, dp)
    _same_device(probs, dp)
    return torch.empty_like(probs)


# ------------------------------------------------------------------------ GELU
def gelu_activation(x: Tensor) -> Tensor:
    """Exact (erf) GELU."""
    return torch.ops.cuda_transformer.gelu_activation.default(x)


@torch.library.register_fake("cuda_transformer::gelu_activation")
def _(x):
    _f32(x)
    return torch.empty_like(x)


def gelu_activation_bwd(x: Tensor, dy: Tensor) -> Tensor:
    """GELU backward."""
    return torch.ops.cuda_transformer.gelu_activation_bwd.default(x, dy)


@torch.library.register_fake("cuda_transformer::gelu_activation_bwd")
def _(x, dy):
    _f32(x, dy)
    _same_device(x, dy)
    return torch.empty_like(x)


# ------------------------------------------------- materialised attention
def causal_self_attention_fwd(qkv: Tensor, nh: int, causal: bool) -> tuple[Tensor, Tensor]:
    """Attention with the full probability matrix (not the hot path)."""
    return torch.ops.cuda_transformer.causal_self_attention_fwd.default(qkv, nh, causal)


@torch.library.register_fake("cuda_transformer::causal_self_attention_fwd")
def _(qkv, nh, causal):
    _f32(qkv)
    b, t, three_c = qkv.shape
    c = three_c // 3
    out = torch.empty((b, t, c), dtype=qkv.dtype, device=qkv.device)
    probs = torch.empty((b, nh, t, t), dtype=qkv.dtype, device=qkv.device)
    return out, probs


def causal_self_attention_bwd(Q: Tensor, K: Tensor, V: Tensor, probs: Tensor,
                              dO: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """Backward of causal_self_attention_fwd (dq, dk returned times sqrt(hs))."""
    return torch.ops.cuda_transformer.causal_self_attention_bwd.default(Q, K, V, probs, dO)


@torch.library.register_fake("cuda_transformer::causal_self_attention_bwd")
def _(Q, K, V, probs, dO):
    _f32(Q, K, V, probs, dO)
    _same_device(Q, K, V, probs, dO)
    return torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)


# ------------------------------------------------------------ FlashAttention-2
def flash_attention_fwd(Q: Tensor, K: Tensor, V: Tensor, causal: bool) -> tuple[Tensor, Tensor]:
    """FlashAttention-2 forward: returns O [B,nh,T,hs] and L = logsumexp [B,nh,T]."""
    return torch.ops.cuda_transformer.flash_attention_fwd.default(Q, K, V, causal)


def flash_attention_fwd_ex(Q: Tensor, K: Tensor, V: Tensor, causal: bool,
                           precision: int) -> tuple[Tensor, Tensor]:
    """flash_attention_fwd with an explicit precision mode."""
    return torch.ops.cuda_transformer.flash_attention_fwd_ex.default(Q, K, V, causal, precision)


def _fa_fwd_meta(Q, K, V):
    _f32(Q, K, V)
    _same_device(Q, K, V)
    O = torch.empty((Q.size(0), Q.size(1), Q.size(2), Q.size(3)), dtype=Q.dtype, device=Q.device)
    L = torch.empty((Q.size(0), Q.size(1), Q.size(2)), dtype=Q.dtype, device=Q.device)
    return O, L


@torch.library.register_fake("cuda_transformer::flash_attention_fwd")
def _(Q, K, V, causal):
    return _fa_fwd_meta(Q, K, V)


@torch.library.register_fake("cuda_transformer::flash_attention_fwd_ex")
def _(Q, K, V, causal, precision):
    return _fa_fwd_meta(Q, K, V)


def flash_attention_bwd(Q: Tensor, K: Tensor, V: Tensor, O: Tensor, dO: Tensor, L: Tensor,
                        causal: bool):
    """FlashAttention-2 backward: returns dQ, dK, dV."""
    return torch.ops.cuda_transformer.flash_attention_bwd.default(Q, K, V, O, dO, L, causal)


def flash_attention_bwd_ex(Q: Tensor, K: Tensor, V: Tensor, O: Tensor, dO: Tensor, L: Tensor,
                           causal: bool, precision: int):
    """flash_attention_bwd with an explicit precision mode."""
    return torch.ops.cuda_transformer.flash_attention_bwd_ex.default(Q, K, V, O, dO, L, causal,
                                                                     precision)


def _fa_bwd_meta(Q, K, V, O, dO, L):
    _f32(Q, K, V, O, dO, L)
    _same_device(Q, K, V, O, dO, L)
    return (torch.empty(Q.shape, dtype=Q.dtype, device=Q.device),
            torch.empty(K.shape, dtype=K.dtype, device=K.device),
            torch.empty(V.shape, dtype=V.dtype, device=V.device))


@torch.library.register_fake("cuda_transformer::flash_attention_bwd")
def _(Q, K, V, O, dO, L, causal):
    return _fa_bwd_meta(Q, K, V, O, dO, L)


@torch.library.register_fake("cuda_transformer::flash_attention_bwd_ex")
def _(Q, K, V, O, dO, L, causal, precision):
    return _fa_bwd_meta(Q, K, V, O, dO, L)


# ------------------------------------------------------------------- LayerNorm
def layernorm_fwd(x: Tensor, gamma: Tensor, beta: Tensor, eps: float = 1e-5):
    """LayerNorm over the last dim (biased variance); returns y, mean, rstd."""
    return torch.ops.cuda_transformer.layernorm_fwd.default(x, gamma, beta, eps)


@torch.library.register_fake("cuda_transformer::layernorm_fwd")
def _(x, gamma, beta, eps):
    _f32(x, gamma, beta)
    rows = x.numel() // x.size(-1)
    return (torch.empty_like(x), torch.empty(rows, dtype=x.dtype, device=x.device),
            torch.empty(rows, dtype=x.dtype, device=x.device))


def layernorm_bwd(x: Tensor, gamma: Tensor, mean: Tensor, rstd: Tensor, dy: Tensor):
    """LayerNorm backward; returns dx, dgamma, dbeta."""
    return torch.ops.cuda_transformer.layernorm_bwd.default(x, gamma, mean, rstd, dy)


@torch.library.register_fake("cuda_transformer::layernorm_bwd")
def _(x, gamma, mean, rstd, dy):
    _f32(x, gamma, mean, rstd, dy)
    return torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)


# ------------------------------------------------- linear layer, fused options
def linear_fused(x: Tensor, weights: Tensor, bias: Tensor, precision: int = PRECISION_3XTF32,
                 epilogue: int = EPILOGUE_NONE, act_in: Tensor | None = None,
                 want_colsum: bool = False):
    """out = x @ weights + bias with GELU (EPILOGUE_GELU: also returns
    gelu(out)) or the GELU gradient (EPILOGUE_GELU_GRAD: out * gelu'(act_in))
    applied in the GEMM's epilogue, and optionally the column sums of
    `weights` over its reduction index (the bias gradient when weights is dY,
    batch 1).  Returns (out, act, colsum); unused ones are empty."""
    return torch.ops.cuda_transformer.linear_fused.default(x, weights, bias, precision, epilogue,
                                                           act_in, want_colsum)


@torch.library.register_fake("cuda_transformer::linear_fused")
def _(x, weights, bias, precision, epilogue, act_in, want_colsum):
    out = _fma_meta(x, weights, bias)
    act = torch.empty_like(out) if epilogue == EPILOGUE_GELU else out.new_empty(0)
    cs = out.new_empty(out.size(2)) if want_colsum else out.new_empty(0)
    return out, act, cs


def linear_accumulate_(out: Tensor, colsum: Tensor | None, x: Tensor, weights: Tensor,
                       bias: Tensor, precision: int = PRECISION_3XTF32) -> None:
    """out += x @ weights + bias, and colsum += the column sums of weights."""
    torch.ops.cuda_transformer.linear_accumulate_.default(out, colsum, x, weights, bias, precision)


@torch.library.register_fake("cuda_transformer::linear_accumulate_")
def _(out, colsum, x, weights, bias, precision):
    return None


def cross_entropy_fwd_bwd_(logits: Tensor, targets: Tensor, ignore_index: int = -100) -> Tensor:
    """Per-row cross entropy of (rows, vocab) logits; the logits are
    overwritten with softmax - onehot(targets) (unscaled gradient)."""
    return torch.ops.cuda_transformer.cross_entropy_fwd_bwd_.default(logits, targets, ignore_index)


@torch.library.register_fake("cuda_transformer::cross_entropy_fwd_bwd_")
def _(logits, targets, ignore_index):
    return logits.new_empty(logits.size(0))


# ------------------------------------------------------------ token generation
# (looked up once: a decoding step is made of calls that take longer on the host
# than on the device, and the look-up is 0.4 of their 9 us)
_kv_append = torch.ops.cuda_transformer.kv_append_.default
_paged_attention = torch.ops.cuda_transformer.paged_attention.default
_logits_process = torch.ops.cuda_transformer.logits_process.default


def rotary_tables(positions: int, rot: int, base: float = 10000.0, device=None):
    """cos and sin of position * base^(-2i/rot), i < rot/2, for kv_append_:
    FP32 [positions, rot/2], formed in FP64 (an FP32 angle loses its low bits
    as the position grows)."""
    torch._check(rot >= 0 and rot % 2 == 0, lambda: f"rot must be even, not {rot}")
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def kv_append_(k_cache: Tensor, v_cache: Tensor, k: Tensor, v: Tensor, block_table: Tensor,
               positions: Tensor, seq_ids: Tensor | None = None, q: Tensor | None = None,
               cos: Tensor | None = None, sin: Tensor | None = None, interleaved: bool = False,
               want_k: bool = False,
               rotary_positions: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Appends k, v [tokens, kv_heads, hs] to a paged cache, turning k (and q
    [tokens, nh, hs]) by the rotary angles of their positions on the way.

    k_cache, v_cache: [pages, kv_heads, page_size, hs], any order of the first
    three in memory, float32, bfloat16 or float16 (k, v, q: float32 or the
    cache's type).  block_table: int32 [batch, max_pages], the pages of each
    sequence in order.  Token t goes to position positions[t] (int32) of
    sequence seq_ids[t] (int32; default: sequence t).  cos, sin: float32
    [positions, rot/2] (rotary_tables); element i pairs with i + rot/2, or 2i
    with 2i + 1 when interleaved; None: no rotation.  A negative position is
    padding (nothing appended, zero outputs); a token that has no place in the
    cache gives NaN outputs.  rotary_positions (int32 [tokens]): the positions
    that the angles are taken of, where they are not the slots' (a drafted
    token's depth in its tree).  Returns (turned q, turned k if want_k); unused
    ones are empty."""
    return _kv_append(k_cache, v_cache, k, v, block_table, positions, seq_ids, q, cos, sin,
                      interleaved, want_k, rotary_positions)


@torch.library.register_fake("cuda_transformer::kv_append_")
def _(k_cache, v_cache, k, v, block_table, positions, seq_ids, q, cos, sin, interleaved, want_k,
      rotary_positions=None):
    _same_device(k, v, k_cache, v_cache, block_table, positions)
    torch._check(k.dtype == v.dtype and k_cache.dtype == v_cache.dtype)
    q_out = q.new_empty(q.shape) if q is not None else k.new_empty(0)
    return q_out, k.new_empty(k.shape) if want_k else k.new_empty(0)


def paged_attention_workspace(nh: int, kv_heads: int, hs: int, device=None) -> Tensor:
    """The workspace of paged_attention for these heads, whatever the batch and
    lengths: cleared once here, it serves any number of calls, but not two that
    can run at the same time on different streams."""
    size = torch.ops.cuda_transformer.paged_attention_workspace_size.default(nh, kv_heads, hs)
    return torch.zeros(size, dtype=torch.uint8, device="cuda" if device is None else device)


def paged_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor,
                    seq_lens: Tensor, scale: float | None = None,
                    workspace: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Attention of one new token per sequence, q [batch, nh, hs], over the
    first seq_lens[b] (int32) tokens of a paged cache (kv_append_'s layout; nh
    a multiple of kv_heads; cache rows 16-byte aligned).  Returns O
    [batch, nh, hs] and L = logsumexp [batch, nh]; a length of 0 gives O = 0,
    L = -inf, one that the table cannot hold gives NaN.  scale: hs^-0.5 by
    default.  workspace: paged_attention_workspace's; a temporary one is
    cleared for the call when it is not given."""
    s = q.shape[-1] ** -0.5 if scale is None else scale
    return _paged_attention(q, k_cache, v_cache, block_table, seq_lens, s, workspace)


@torch.library.register_fake("cuda_transformer::paged_attention")
def _(q, k_cache, v_cache, block_table, seq_lens, scale, workspace):
    _same_device(q, k_cache, v_cache, block_table, seq_lens)
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


def logits_process(logits: Tensor, tokens: Tensor | None = None, lens: Tensor | None = None,
                   prompt_lens: Tensor | None = None, repetition: Tensor | None = None,
                   frequency: Tensor | None = None, presence: Tensor | None = None,
                   bias_ids: Tensor | None = None, bias_values: Tensor | None = None,
                   mask: Tensor | None = None) -> Tensor:
    """Sampling penalties, biases and a grammar mask on logits [rows, vocab]
    (float32, bfloat16 or float16); returns new float32 logits.

    tokens: int64 [rows, max_len] histories, lens (int32 [rows]) their lengths
    (default: all of max_len), prompt_lens (int32 [rows]) how many of them are
    the prompt (default: none).  repetition (float32 [rows]): x / r for x > 0,
    else x * r, for every token of the history; frequency, presence (float32
    [rows]): subtracted once per occurrence, and once, for tokens of the part
    after the prompt.  bias_ids, bias_values (int64, float32 [rows, n]): added.
    mask (int32 [rows, ceil(vocab/32)]): -inf where bit i % 32 of word i / 32
    is 0.  Ids outside [0, vocab) are ignored."""
    return _logits_process(logits, tokens, lens, prompt_lens, repetition, frequency, presence,
                           bias_ids, bias_values, mask)


@torch.library.register_fake("cuda_transformer::logits_process")
def _(logits, tokens, lens, prompt_lens, repetition, frequency, presence, bias_ids, bias_values,
      mask):
    return logits.new_empty(logits.shape, dtype=torch.float32)


# -------------------------------------------------------- speculative decoding
_tree_attention = torch.ops.cuda_transformer.tree_attention.default
_verify_drafts = torch.ops.cuda_transformer.verify_drafts.default
_kv_compact = torch.ops.cuda_transformer.kv_compact_.default
_kv_copy_pages = torch.ops.cuda_transformer.kv_copy_pages_.default


def tree_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor,
                   context_lens: Tensor, draft_lens: Tensor | None = None,
                   mask: Tensor | None = None,
                   scale: float | None = None) -> tuple[Tensor, Tensor]:
    """Attention of several new tokens per sequence, q [batch, drafts, nh, hs],
    over a paged cache (kv_append_'s layout; nh a multiple of kv_heads; cache
    rows 16-byte aligned).

    context_lens (int32 [batch]): tokens before the new ones; new token i is in
    the cache at position context_lens[b] + i.  draft_lens (int32 [batch]): how
    many there are (default: all).  mask (int32 [batch, drafts, ceil(drafts /
    32)]): new token i sees new token j where bit j % 32 of word j / 32 of its
    row is set, as a tree's node sees its ancestors and itself; default: all
    up to itself (a chain, or a piece of a prompt).  The tokens before the new
    ones are seen by all.  Returns O [batch, drafts, nh, hs] and L = logsumexp
    [batch, drafts, nh]; rows that are not there or see nothing, and sequences
    with a negative context_lens, give O = 0, L = -inf; lengths that the table
    cannot hold give NaN.  scale: hs^-0.5 by default."""
    s = q.shape[-1] ** -0.5 if scale is None else scale
    return _tree_attention(q, k_cache, v_cache, block_table, context_lens, draft_lens, mask, s)


@torch.library.register_fake("cuda_transformer::tree_attention")
def _(q, k_cache, v_cache, block_table, context_lens, draft_lens, mask, scale):
    _same_device(q, k_cache, v_cache, block_table, context_lens)
    return q.new_empty(q.shape), q.new_empty(q.shape[:3], dtype=torch.float32)


def verify_drafts(target: Tensor, tokens: Tensor, parents: Tensor | None = None,
                  draft_lens: Tensor | None = None, draft_probs: Tensor | None = None,
                  uniform: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """Which drafted tokens are kept, and the token after them, so that the
    result is distributed as the target's own tokens.

    A sequence's draft is a tree: node 0 is its last certain token, node i > 0
    proposes tokens[b, i] (int64 [batch, drafts]) after node parents[b, i] < i
    (int32 [batch, drafts]; default: i - 1).  draft_lens (int32 [batch]): its
    nodes (default: all; 0: it takes no part).  target [batch, drafts, vocab]
    (float32, bfloat16 or float16): the target's probabilities after each node.
    draft_probs (target's type and shape): the drafter's, which the proposals
    were drawn from one by one; None: proposals that were certain to be made
    (looked up, or the drafter's best).  uniform (float32 [batch, drafts]):
    numbers in [0, 1); those of the nodes decide over them, the one of node 0
    draws the token after the path.  uniform None: target holds scores (logits)
    and the best token is kept at each place.

    Returns (new_tokens int64 [batch, drafts], path int32 [batch, drafts],
    counts int32 [batch]): the path's nodes from node 0 on, counts[b] of them,
    and the token after each; -1 behind them, and where there is no next token
    (a row without probabilities, of -inf, with a NaN).  kv_compact_ takes path
    and counts."""
    return _verify_drafts(target, tokens, parents, draft_lens, draft_probs, uniform)


@torch.library.register_fake("cuda_transformer::verify_drafts")
def _(target, tokens, parents, draft_lens, draft_probs, uniform):
    _same_device(target, tokens)
    return (tokens.new_empty(tokens.shape), tokens.new_empty(tokens.shape, dtype=torch.int32),
            tokens.new_empty(tokens.shape[:1], dtype=torch.int32))


def kv_compact_(caches: list[Tensor], block_table: Tensor, context_lens: Tensor, keep: Tensor,
                counts: Tensor) -> None:
    """Moves the kept ones of the last tokens up, in all of `caches` (keys and
    values of any layers, of one shape and type, kv_append_'s layout): what is
    at position context_lens[b] + keep[b, j] goes to context_lens[b] + j, for
    j < counts[b].  keep (int32 [batch, n]) ascends along a row; context_lens,
    counts: int32 [batch].  verify_drafts gives path and counts to pass here;
    any other choice of tokens to keep is made the same way.  A move without a
    place in the cache is left out.  No cache may be in the list twice or
    overlap another, and sequences must not share the pages that are written
    (kv_copy_pages_ gives a fork its own)."""
    _kv_compact(caches, block_table, context_lens, keep, counts)


@torch.library.register_fake("cuda_transformer::kv_compact_")
def _(caches, block_table, context_lens, keep, counts):
    return None


def kv_copy_pages_(caches: list[Tensor], src: Tensor, dst: Tensor) -> None:
    """Copies page src[i] to page dst[i] (int32 [n]) in all of `caches` (of one
    shape and type, kv_append_'s layout).  No dst may be among src or twice.  A
    pair with a page out of range is left out."""
    _kv_copy_pages(caches, src, dst)


@torch.library.register_fake("cuda_transformer::kv_copy_pages_")
def _(caches, src, dst):
    return None

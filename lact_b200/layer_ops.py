"""Row-wise stages of the LaCT layer around the chunk recurrence (the layer's own code,
lact_llm/lact_model/layer_lact_swiglu.py, is outside this package; these are the passes over
[b, s, n_h * d] that sit directly on the recurrence's inputs and output).

Forward: one fused CUDA pass each.  Backward (training): one fused pass each that recomputes from the saved inputs (the
forward's bf16 roundings are treated as identities).  Registered operators, csrc/native/layer.cpp and attention.cpp.

Attention half of the hybrid layers (tcgen05 kernels, forward and backward, head dimension 64 or 128):
`sliding_window_attention` (causal band; packed sequences by `cu_seqlens`, padded batches by `attention_mask`),
`block_attention` (not causal, own key count) and, under the reference's names, the autoregressive-video layer's
`batched_sliding_window_attention`, `batched_sliding_window_attention_with_repeated_chunks` and
`sliding_window_attention_inference`.

Linear attention with a decay per head (`linear_attention` for prompts and training, `linear_attention_step` for single tokens): the
recurrence with a linear memory, beside the fast weights.  `group_norm`: channels last, with an activation; with one spot a sample
the norm of every head of every token behind such a mixer.  Neither has a counterpart in the reference.

Generation: `rotary_axes` (rotary positions of the attention's q and k, one axis or several; also for training), `PagedCache` with
`paged_cache_write` / `paged_cache_read` (keys and values in pages, bf16 or 8 bits) and `paged_attention_step` (one new token of every
sequence over its pages, with the layer's window)."""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib as L
from .ops import _op

BF16 = torch.bfloat16


def _seq_start(cu_seqlens: torch.Tensor, n_tokens: int, device) -> torch.Tensor:
    """int32 [n_tokens]: for every token of a packed batch entry, the first token of its sequence (no host
    synchronisation: the output size is known)."""
    if cu_seqlens.is_cuda and cu_seqlens.device == torch.device(device):
        return L.call(_op("seq_start"), cu_seqlens, n_tokens)
    cu = cu_seqlens.to(device=device, dtype=torch.int64)
    return torch.repeat_interleave(cu[:-1], cu[1:] - cu[:-1], output_size=n_tokens).to(torch.int32).contiguous()


def rotary_tables(head_dim: int, n_positions: int, base: float = 500000.0, device=None, dtype=BF16):
    """cos / sin tables [n_positions, head_dim / 2] as fla.modules.RotaryEmbedding(dim=head_dim, base=rope_theta)
    caches them (fp32 inverse frequencies and positions, result cast to the activations' dtype)."""
    inv_freq = 1.0 / (base ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim))
    freqs = torch.outer(torch.arange(n_positions, dtype=torch.float32, device=device), inv_freq)
    return torch.cos(freqs).to(dtype), torch.sin(freqs).to(dtype)


def qkv_prologue(xq: torch.Tensor, xk: torch.Tensor, xv: torch.Tensor, num_heads: int, qkv_silu: bool = True,
                 no_v_silu: bool = False, rotary: Optional[Tuple[torch.Tensor, torch.Tensor, int]] = None,
                 seqlen_offset: int = 0, cu_seqlens: Optional[torch.Tensor] = None):
    """fast_q, fast_k, fast_v of layer_lact_swiglu.py:399-446 in one pass: `[b, s, (n_h d)] -> [(b n_h), s, d]`, SiLU
    on q, k (and v unless `no_v_silu`), per-head l2_norm of q and k (ttt_operation.py:19-26) and, when `rotary` =
    (cos, sin, attention_head_dim) is given (`ttt_nope` off), the rotary embedding of q and k over attention heads of
    that size (tables as `rotary_tables` / fla.modules.RotaryEmbedding build them, bf16 [positions, head_dim / 2]).
    Inputs may be views of a fused projection.  Differentiable (see the module docstring).  `cu_seqlens` (with
    `rotary`, batch of one): sequences packed back to back, positions restart at every sequence start (:434)."""
    if not (xq.is_cuda and xk.is_cuda and xv.is_cuda):
        raise ValueError("qkv_prologue needs CUDA tensors (there is no CPU implementation)")
    assert xq.shape == xk.shape == xv.shape and xq.dim() == 3 and xq.shape[2] % num_heads == 0
    assert xq.dtype == xk.dtype == xv.dtype == BF16, "expected [b, s, n_heads * d] bf16 tensors"
    cos = sin = None
    rope_hd = 0
    if rotary is not None:
        cos, sin, rope_hd = rotary
        assert cos.dtype == BF16 and sin.dtype == BF16 and cos.shape == sin.shape and cos.shape[1] * 2 == rope_hd
        cos, sin = cos.contiguous(), sin.contiguous()
    seq_start = None
    if cu_seqlens is not None and rotary is not None:
        if xq.shape[0] != 1:
            raise ValueError("packed sequences (cu_seqlens) need a batch of one")
        seq_start = _seq_start(cu_seqlens, xq.shape[1], xq.device)
    q, k, v = L.call(_op("qkv_prologue"), xq, xk, xv, num_heads, bool(qkv_silu), not no_v_silu, cos, sin, int(rope_hd),
                     int(seqlen_offset), seq_start)
    return q, k, v


def lr_prologue(lr_proj: torch.Tensor, num_heads: int, base_lr: float, momentum_logits: torch.Tensor = None):
    """fw_lr1, fw_lr2, fw_lr3 (and momentum) of layer_lact_swiglu.py:463-480: softplus(lr_proj.float() +
    inv_softplus(base_lr)) split per head into three fp32 [(b n_h), s, 1] tensors; `momentum_logits` is the output of
    the momentum Linear BEFORE its Sigmoid ([b, s, n_h]); the result is sigmoid(.) in the logits' dtype, as float.
    Differentiable with respect to the projections."""
    if not lr_proj.is_cuda:
        raise ValueError("lr_prologue needs CUDA tensors (there is no CPU implementation)")
    assert lr_proj.dim() == 3 and lr_proj.shape[2] == 3 * num_heads
    if momentum_logits is not None:
        assert momentum_logits.shape == (*lr_proj.shape[:2], num_heads)
    base_lr_inv = base_lr + math.log(-math.expm1(-base_lr))
    outs = L.call(_op("lr_prologue"), lr_proj, momentum_logits, num_heads, base_lr_inv)
    return outs[0], outs[1], outs[2], outs[3] if len(outs) == 4 else None


def out_epilogue(fw_x: torch.Tensor, norm_weight: torch.Tensor, num_heads: int, scale_proj: torch.Tensor = None,
                 o: torch.Tensor = None, eps: float = 1e-5) -> torch.Tensor:
    """`o + merge_heads(ttt_norm(fw_x) * silu(scale_proj))` of layer_lact_swiglu.py:556-568 in one pass.
    fw_x: [(b n_h), s, d] bf16 (output of the recurrence); norm_weight: [d]; scale_proj (the output of
    `ttt_scale_proj`, before its SiLU) and o (attention output): [b, s, n_h * d] bf16 or None.
    Differentiable with respect to fw_x, the norm weight, scale_proj and o."""
    if not fw_x.is_cuda:
        raise ValueError("out_epilogue needs CUDA tensors (there is no CPU implementation)")
    assert fw_x.dim() == 3 and fw_x.dtype == BF16 and fw_x.shape[0] % num_heads == 0
    B, s, d = fw_x.shape
    assert norm_weight.shape == (d,)
    for t, name in ((scale_proj, "scale_proj"), (o, "o")):
        assert t is None or (t.shape == (B // num_heads, s, num_heads * d) and t.dtype == BF16), \
            f"{name}: expected a [b, s, n_heads * d] bf16 tensor"
    return L.call(_op("out_epilogue"), fw_x, norm_weight, scale_proj, o, num_heads, float(eps))


# ------------------------------------------------------------------------------------------ group norm
def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, activation: Optional[str] = None) -> torch.Tensor:
    """Group norm with an activation, channels last: `act((x - mean) / sqrt(var + eps) * weight + bias)`, x [n, ..., C] bf16 or
    float32, mean and var over all spots of a sample and the C / num_groups adjacent channels of a group, activation None or
    "silu"; weight, bias [C] float32 or bf16, or None.  Behind a token mixer, x [tokens, heads * d] with num_groups = heads is
    the norm of every head of every token (one spot a sample); maps and frames are [n, h, w, C] or [n, frames, h, w, C].
    Result: x's shape and type, contiguous.  Differentiable with respect to x, weight and bias."""
    if activation not in (None, "silu"):
        raise ValueError("activation: None or 'silu'")
    if x.dim() < 2:
        raise ValueError("x: [n, ..., channels]")
    if x.dtype not in (BF16, torch.float32):
        raise TypeError("x: bf16 or float32")
    C = x.shape[-1]
    if num_groups < 1 or C == 0 or C % num_groups:
        raise ValueError("num_groups must divide the channels")
    if not 0.0 <= eps < math.inf:
        raise ValueError("eps must be finite and not negative")
    for t in (weight, bias):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != C or t.get_device() != x.get_device():
            raise ValueError("weight, bias: [channels] on the device of x")
        if t.dtype not in (BF16, torch.float32):
            raise TypeError("weight, bias: bf16 or float32")
    if not x.is_cuda:
        raise ValueError("group_norm needs CUDA tensors (there is no CPU implementation)")
    return L.call(_op("group_norm_fwd"), x, weight, bias, num_groups, eps, activation == "silu")[0]


# ------------------------------------------------------------------------------------------ linear attention
def _linear_heads(what, q, k, v, log_decay, dims):
    """Checks shared by the prompt and the token form (`dims` axes, heads and features last); returns heads, dk, dv."""
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != dims or len(ks) != dims or len(vs) != dims:
        raise ValueError(f"q, k, v must have {dims} axes")
    if q.dtype != BF16 or k.dtype != BF16 or v.dtype != BF16:
        raise TypeError("q, k, v: bf16 activations")
    h, dk, dv = qs[-2], qs[-1], vs[-1]
    if qs[:-2] != ks[:-2] or ks[:-1] != vs[:-1] or ks[-1] != dk:
        raise ValueError("q [..., h, dk], k [..., h_kv, dk], v [..., h_kv, dv] of the same batch and tokens")
    if dk not in (64, 128) or dv not in (64, 128):
        raise ValueError("dk and dv must be 64 or 128")
    if h == 0 or ks[-2] == 0 or h % ks[-2]:
        raise ValueError("the heads of k and v must divide those of q")
    if log_decay.dtype != torch.float32 or log_decay.dim() != 1 or log_decay.shape[0] != h:
        raise ValueError("log_decay: [heads] in float32")
    at = q.get_device()
    if k.get_device() != at or v.get_device() != at or log_decay.get_device() != at:
        raise ValueError("all tensors must be on the same device")
    if not q.is_cuda:
        raise ValueError(f"{what} needs CUDA tensors (there is no CPU implementation)")
    return h, dk, dv


def _linear_scale(scale, dk):
    if scale is None:
        return dk ** -0.5
    scale = float(scale)
    if not 1e-18 <= abs(scale) <= 1e18:
        raise ValueError("scale must be of a size between 1e-18 and 1e18")
    return scale


def _linear_state(name, state, shape, device):
    if state.shape != shape or state.dtype != torch.float32 or state.get_device() != device:
        raise ValueError(f"{name}: a float32 {list(shape)} tensor on the device of q")


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: Optional[float] = None,
                     initial_state: Optional[torch.Tensor] = None, output_final_state: bool = False,
                     cu_seqlens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Causal linear attention with a decay per head, the recurrence with a linear memory beside this package's fast weights:
    `S_t = exp(log_decay[h]) S_(t-1) + k_t v_t^T`, `o_t = scale q_t^T S_t` with S [dk, dv] in float32.

    q [b, l, h, dk], k [b, l, h_kv, dk], v [b, l, h_kv, dv] bf16 (dk, dv 64 or 128; h a multiple of h_kv: consecutive heads share a
    key and value head; views of a fused projection are read where they lie, whatever strides axes of one entry have), log_decay [h] float32, not above 0 (-inf: a head
    without memory); it gets no gradient.  `scale`: dk ** -0.5 by default.  initial_state [b, h, dk, dv] float32 or None (zeros).
    `cu_seqlens` (int32 [n + 1] on the device, b must be 1): n sequences packed back to back, empty ones allowed, each with its
    own state ([n, h, dk, dv]); tokens outside of them have zero outputs (bounds that fall or pass the end stay inside the arrays, with
    numbers that mean nothing).  Returns o [b, l, h, dv] bf16 and the state behind the
    last token (None without `output_final_state`).  Differentiable with respect to q, k, v and initial_state, through both.
    Products take q, k, v as they are and round the weights of a tile's tokens and its incoming state to bf16; sums and the state
    itself are kept in float32.  A NaN or an infinity in k, v reaches the outputs of its whole tile of 128 tokens (counted from
    the start of its sequence) and later ones, for as long at least as its weight has not decayed below the smallest float32: the rows
    that pad a batch hold finite numbers, or its sequences are packed (what lies behind those is not looked at)."""
    h, dk, dv = _linear_heads("linear_attention", q, k, v, log_decay, 4)
    n = q.shape[0]
    if cu_seqlens is not None:
        if q.shape[0] != 1:
            raise ValueError("packed sequences (cu_seqlens) need a batch of one")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise ValueError("cu_seqlens: whole numbers [n + 1]")
        cu_seqlens = cu_seqlens.to(device=q.device, dtype=torch.int32).contiguous()
        n = cu_seqlens.numel() - 1
    if initial_state is not None:
        _linear_state("initial_state", initial_state, (n, h, dk, dv), q.get_device())
    r = L.call(_op("linear_attention_fwd"), q, k, v, log_decay, _linear_scale(scale, dk), initial_state, cu_seqlens,
               bool(output_final_state))
    return r[0], r[1] if output_final_state else None


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                          scale: Optional[float] = None, new_state: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token of every sequence (generation): `linear_attention` in its recurrent form.  q [b, h, dk], k [b, h_kv, dk],
    v [b, h_kv, dv] bf16, state [b, h, dk, dv] float32, contiguous: read, and written in place, or to `new_state` (an array apart
    from it).  Returns o [b, h, dv] bf16.  No backward: a call with gradients raises.  To autograd the array that is written has
    changed in place: a backward that has saved it (as `linear_attention` saves its `initial_state`) raises."""
    h, dk, dv = _linear_heads("linear_attention_step", q, k, v, log_decay, 3)
    shape, at = (q.shape[0], h, dk, dv), q.get_device()
    if new_state is None:
        new_state = state
    for t in (state,) if new_state is state else (state, new_state):
        _linear_state("state, new_state", t, shape, at)
        if not t.is_contiguous():
            raise ValueError("state and new_state must be contiguous: they are read and written where they lie")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad or state.requires_grad or
                                    new_state.requires_grad):
        raise NotImplementedError("linear_attention_step has no backward: use linear_attention")
    return L.call(_op("linear_attention_step"), q, k, v, log_decay, _linear_scale(scale, dk), state, new_state)


# ------------------------------------------------------------------------------------------ rotary positions
def rotary_frequencies(sections: Sequence[int], base: float = 10000.0, shared: bool = False, device=None) -> torch.Tensor:
    """Frequencies of `rotary_axes`, float64 [sum(sections)]: every axis its own `base ** (-j / n)`, j < n pairs of its section (the video
    layer's three axes; with one axis of half a head the usual table), or with `shared` one table over all pairs."""
    sections = [sum(sections)] if shared else sections
    return torch.cat([base ** (-torch.arange(n, dtype=torch.float64, device=device) / max(n, 1)) for n in sections])


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, sections: Sequence[int],
                interleaved: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions with several axes (text: one; images: rows and columns; video: time, height, width) of the attention's q
    [b, l, h, d] and k [b, l, h_kv, d] (or None), or of new tokens [n, h, d]; bf16 or float32, d even, 512 at most, any strides.
    positions (int32 or int64) [l, axes], or [b, l, axes].  The first 2 P features of a head are P = sum(sections) pairs, (j, j + P) or, with
    `interleaved`, (2j, 2j + 1); pairs go to the axes in sections (at most 8), and pair j turns by `positions[axis] * frequencies[j]`
    (float64 [P], `rotary_frequencies`): (x, y) -> (x cos - y sin, y cos + x sin).  Features from 2 P on are copied.  Returns the turned q
    and k, contiguous.  Differentiable with respect to q and k, any number of times.  Angles are whole numbers of 2^-64 turns, from the
    float64 frequencies, in which full turns drop out by themselves (what float64 leaves of a position of 2^31 is 2^-24 of a turn at a frequency of
    1); of a turn they keep 32 bits and then float32 (2^-26 of a turn) for their cosines and sines, which bf16 results take from the
    hardware's approximations (2^-20.9).  The results are rounded once."""
    r = L.call(_op("rotary_axes"), q, k, positions, frequencies, sections, interleaved)
    return r[0], r[1] if k is not None else None


# ------------------------------------------------------------------------------------------ paged cache
class PagedCache(NamedTuple):
    """Keys and values in pages.  k, v [pages, kv_heads, page_size, head_dim]: bf16, or float8_e4m3fn with k_exponent, v_exponent (uint8
    [pages, kv_heads, page_size]): a row of a head stands for its values times 2 ** (byte - 127) (byte 255: NaN).  Pages are contiguous in
    themselves; page_size 16, 32, 64, 128 or 256, head_dim 64 or 128.  Which pages a sequence has says its row of a page table (int32
    [sequences, pages of the longest]): position p lies in page `page_table[i, p // page_size]`, row `p % page_size`; entries of pages without
    a position that a call needs (past a sequence's length; in front of its window) are not looked at.  k and v begin on 32 bytes, exponents on 16, and page strides are multiples of as much.  An entry
    that the cache does not have, or a length past the table's end, is left out, and a later call raises LactError (of a window with no
    page at all, attention is NaN).  Page tables and lengths are read on the device: a captured call follows what they hold at its replay."""
    k: torch.Tensor
    v: torch.Tensor
    k_exponent: Optional[torch.Tensor] = None
    v_exponent: Optional[torch.Tensor] = None


def paged_cache(num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = BF16, device=None) -> PagedCache:
    """An empty (zero) cache of bf16, or of 8 bits with `dtype=torch.float8_e4m3fn`."""
    if dtype not in (BF16, torch.float8_e4m3fn):
        raise TypeError("dtype: bf16 or float8_e4m3fn")
    shape = (num_pages, kv_heads, page_size, head_dim)
    zeros = lambda s, dt: torch.zeros(s, dtype=dt, device=device)
    if dtype == BF16:
        return PagedCache(zeros(shape, BF16), zeros(shape, BF16))
    return PagedCache(*(zeros(shape, torch.uint8).view(dtype) for _ in range(2)), *(zeros(shape[:3], torch.uint8) for _ in range(2)))


def paged_cache_write(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                      cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """New keys and values into the cache, in place: k, v [sequences, l, kv_heads, head_dim] bf16 (views of a fused projection are read where
    they lie) become the last l tokens of sequences that then have lengths[i] (int32) tokens: row j goes to position `lengths[i] - l + j`,
    and nowhere where that is negative (rows that pad a batch in front; a sequence of length 0 is not touched).  `cu_seqlens` (int32
    [sequences + 1] on the device, b = 1): the rows of all sequences packed back to back, empty ones allowed; rows outside of them are not
    written.  A cache of 8 bits gets e4m3 values of the row divided by a power of two, the smallest (from 2^-126 to 2^119) that leaves none
    above 448; a row of a head with a NaN or an infinity is NaN when it is read.  Two rows of one call must not have the same place: what is
    there then is not defined.  To autograd the cache has changed in place.  No backward: a call with gradients raises."""
    L.call(_op("paged_cache_write"), *cache, k, v, page_table, lengths, cu_seqlens)


def paged_cache_read(cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, num_tokens: int,
                     cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The last `num_tokens` tokens of every sequence out of the cache: bf16 [2 sequences, num_tokens, kv_heads, head_dim], the keys of all
    sequences and then their values (what `sliding_window_attention_inference` takes as `kv_cache`).  Row j is position
    `lengths[i] - num_tokens + j`, zeros where that is negative.  `cu_seqlens` (int32 [sequences + 1]): [2, num_tokens, kv_heads, head_dim], of
    sequence i the last cu_seqlens[i + 1] - cu_seqlens[i] tokens; rows outside of them are zeros.  8 bits become the bf16 values that
    they stand for: exactly, as `paged_cache_write` leaves them (bytes of 0 to 2 and above 246 can stand for values that bf16 does not have; those of a
    cache that others filled are rounded).  No backward."""
    return L.call(_op("paged_cache_read"), *cache, page_table, lengths, num_tokens, cu_seqlens)


def paged_attention_step(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, window_size: Optional[int] = None,
                         softmax_scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one new token of every sequence over its cache (generation): q [sequences, heads, head_dim] bf16, keys and values those
    of positions `max(0, lengths[i] - window_size)` to `lengths[i] - 1` (`window_size` None: all; the new token's own are written before,
    and lengths count them).  The heads of the cache divide those of q (consecutive heads share).  softmax_scale: head_dim ** -0.5 by
    default.  Returns o [sequences, heads, head_dim] bf16; a sequence without tokens has zeros.  Scores, maxima and sums are float32; weights
    are rounded to two bf16 pieces (bf16 cache) or to fp16 (8 bits) for their product with the values.  Pages that hold nothing of the
    window may have been given back (their entries are not looked at), and whatever other rows outside of it hold counts for nothing.  Within
    it a NaN among the keys makes its heads' outputs NaN, one among the values their outputs of that feature; an infinite value makes these
    infinite or NaN (both pieces of its weight meet it, and the second may be 0 or negative).  How the work is split is chosen on the host, by the
    page table's width (lengths are on the device): short texts under a wide table take longer (one of 777 tokens, 12 heads of 128: 6.4 us with the
    13 columns that it needs, 11.6 with 2048), so that a caller who knows a bound of the lengths passes `page_table[:, :columns]`.  No backward: a
    call with gradients raises."""
    return L.call(_op("paged_attention_step"), q, *cache, page_table, lengths, int(window_size) if window_size else 0,
                  float(softmax_scale) if softmax_scale is not None else cache[0].shape[-1] ** -0.5)


# ------------------------------------------------------------------------------------------ sliding-window attention
def sliding_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window_size: Optional[int] = None,
                             softmax_scale: Optional[float] = None,
                             cu_seqlens: Optional[torch.Tensor] = None,
                             attention_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over the last `window_size` keys (the query's own position included), q, k, v and the
    result [b, l, n_heads, head_dim] bf16: what `flash_attn_func(q, k, v, causal=True, window_size=(window_size - 1,
    0))` computes at lact_llm/lact_model/layer_lact_swiglu.py:386-394 and
    minimal_implementations/causal_lact_with_sliding_window_attn.py:380-384 (`window_size=None`: all earlier keys).
    head_dim 64 or 128.  Differentiable (dq, dk, dv by `lact_swa_bwd`).  `cu_seqlens` (int32 [n + 1], device): the batch
    entry (b must be 1) is n sequences packed back to back, as for `flash_attn_varlen_func` (:371-385): no query sees
    a key of an earlier sequence.  `attention_mask` ([b, l], nonzero = token, zero = padding, any padding side): the
    padded-batch branch (:351-370): the real tokens of all entries are gathered into one packed entry, attended per
    sequence and scattered back, padding positions of the result are zero (`unpad_input` / `pad_input`).  Like the
    reference's, this branch reads the number of real tokens on the host."""
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise ValueError("sliding_window_attention needs CUDA tensors (there is no CPU implementation)")
    assert q.dim() == 4 and q.shape == k.shape == v.shape, "q, k, v: [b, l, n_heads, head_dim], equal head counts"
    assert q.dtype == k.dtype == v.dtype == BF16, "bf16 activations"
    if q.shape[3] not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    scale = float(softmax_scale) if softmax_scale is not None else q.shape[3] ** -0.5
    window = int(window_size) if window_size else 0
    if attention_mask is not None:
        if cu_seqlens is not None:
            raise ValueError("give attention_mask or cu_seqlens, not both")
        b, l, h, d = q.shape
        assert attention_mask.shape == (b, l), "attention_mask: [b, l]"
        mask = attention_mask.to(device=q.device) != 0
        idx = torch.nonzero(mask.reshape(-1)).reshape(-1)   # (host synchronisation: data-dependent size)
        if idx.numel() == 0:
            return torch.zeros_like(q)
        cu = torch.nn.functional.pad(torch.cumsum(mask.sum(dim=1), 0), (1, 0)).to(torch.int32)
        packed = [t.reshape(b * l, h, d).index_select(0, idx).unsqueeze(0) for t in (q, k, v)]
        o = L.call(_op("swa_fwd"), *packed, window, scale, _seq_start(cu, idx.numel(), q.device))[0]
        return torch.zeros(b * l, h, d, dtype=q.dtype, device=q.device).index_copy(0, idx, o[0]).reshape(b, l, h, d)
    seq_start = None
    if cu_seqlens is not None:
        if q.shape[0] != 1:
            raise ValueError("packed sequences (cu_seqlens) need a batch of one")
        seq_start = _seq_start(cu_seqlens, q.shape[1], q.device)
    return L.call(_op("swa_fwd"), q, k, v, window, scale, seq_start)[0]


def block_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    softmax_scale: Optional[float] = None) -> torch.Tensor:
    """Full (not causal) attention of every query of a batch entry over all keys of that entry: q [b, lq, h, d],
    k, v [b, lk, h, d] bf16, result [b, lq, h, d].  What `flash_attention(q, k, v, k_lens=<all keys>, window_size=(-1,
    -1))` computes for the frame blocks of the autoregressive-video layer
    (lact_ar_video/minVid/models/blocks/ar_lact_swa_repeat.py:313-318, 344-364).  The same tcgen05 kernels as
    `sliding_window_attention`, band and sequence masks off.  head_dim 64 or 128.  Differentiable."""
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise ValueError("block_attention needs CUDA tensors (there is no CPU implementation)")
    assert q.dim() == 4 and k.shape == v.shape and k.dim() == 4, "q [b, lq, h, d]; k, v [b, lk, h, d]"
    assert q.shape[0] == k.shape[0] and q.shape[2:] == k.shape[2:], "q and k, v differ in the token count only"
    assert q.dtype == k.dtype == v.dtype == BF16, "bf16 activations"
    if q.shape[3] not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    if q.shape[1] == 0 or k.shape[1] == 0:
        return torch.zeros_like(q)
    scale = float(softmax_scale) if softmax_scale is not None else q.shape[3] ** -0.5
    return L.call(_op("swa_fwd"), q, k, v, -1, scale, None)[0]


def batched_sliding_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mini_batch_size: int,
                                     update_every: int, num_chunks: int, kv_cache_size: int) -> torch.Tensor:
    """The block attention of the autoregressive-video layer, same name and arguments as
    ar_lact_swa_repeat.py:299-365.  q, k, v: [b, l, h, d] with l = update_every - mini_batch_size + update_every *
    (num_chunks - 1).  The first update_every - mini_batch_size tokens attend among themselves; every later block of
    update_every tokens is a clean part (the first mini_batch_size tokens, attending among themselves) followed by a
    noisy part that attends over the last kv_cache_size clean keys and the keys after them (mini_batch_size +
    kv_cache_size keys, as the reference's k_lens says)."""
    b, l = q.shape[:2]
    first, n_c, mb = update_every - mini_batch_size, num_chunks - 1, mini_batch_size
    assert l == first + update_every * n_c, "l = update_every - mini_batch_size + update_every * (num_chunks - 1)"
    assert 0 <= kv_cache_size <= mb
    parts = [block_attention(q[:, :first], k[:, :first], v[:, :first])] if first > 0 else []
    if n_c > 0:
        q_r, k_r, v_r = (t[:, first:].reshape(b * n_c, update_every, *t.shape[2:]) for t in (q, k, v))
        o_clean = block_attention(q_r[:, :mb], k_r[:, :mb], v_r[:, :mb])
        k_end = min(update_every, 2 * mb)   # keys [mb - kv_cache_size, mb - kv_cache_size + (mb + kv_cache_size))
        o_noise = block_attention(q_r[:, mb:], k_r[:, mb - kv_cache_size:k_end], v_r[:, mb - kv_cache_size:k_end])
        parts.append(torch.cat([o_clean, o_noise], dim=1).reshape(b, n_c * update_every, *q.shape[2:]))
    return torch.cat(parts, dim=1) if len(parts) > 1 else parts[0]


def batched_sliding_window_attention_with_repeated_chunks(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                                                          mini_batch_size: int, update_every: int, num_chunks: int,
                                                          kv_cache_size: int) -> torch.Tensor:
    """ar_lact_swa_repeat.py:368-463, same name and arguments: update_every = (num_repeat + 1) * mini_batch_size.  The
    first update_every - mini_batch_size tokens are num_repeat blocks of mini_batch_size tokens, each attending within
    itself; every later block of update_every tokens is a clean part (mini_batch_size tokens, attending within itself)
    and num_repeat noisy parts, each attending over the last kv_cache_size clean keys and its own keys."""
    b, l = q.shape[:2]
    first, n_c, mb = update_every - mini_batch_size, num_chunks - 1, mini_batch_size
    nr = update_every // mb - 1
    assert update_every == (nr + 1) * mb and nr >= 1, "update_every must be a multiple (>= 2) of mini_batch_size"
    assert l == first + update_every * n_c and 0 <= kv_cache_size <= mb
    tail = q.shape[2:]
    blocks = lambda t: t[:, :first].reshape(b * nr, mb, *tail)
    parts = [block_attention(blocks(q), blocks(k), blocks(v)).reshape(b, first, *tail)]
    if n_c > 0:
        q_r, k_r, v_r = (t[:, first:].reshape(b * n_c, update_every, *tail) for t in (q, k, v))
        o_clean = block_attention(q_r[:, :mb], k_r[:, :mb], v_r[:, :mb])
        noisy = lambda t: t[:, mb:].reshape(b * n_c * nr, mb, *tail)
        cached = lambda t: t[:, mb - kv_cache_size:mb].repeat_interleave(nr, dim=0)
        o_noise = block_attention(noisy(q_r), torch.cat([cached(k_r), noisy(k_r)], dim=1),
                                  torch.cat([cached(v_r), noisy(v_r)], dim=1)).reshape(b * n_c, nr * mb, *tail)
        parts.append(torch.cat([o_clean, o_noise], dim=1).reshape(b, n_c * update_every, *tail))
    return torch.cat(parts, dim=1) if len(parts) > 1 else parts[0]


def sliding_window_attention_inference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mini_batch_size: int,
                                       kv_cache: Optional[torch.Tensor] = None, interleave: bool = False,
                                       kv_cache_size: int = 1560) -> torch.Tensor:
    """ar_lact_swa_repeat.py:464-531, same name and arguments: the attention of one generation step of the
    autoregressive-video layer.  (1) no cache, not interleaved: full attention; (2) interleaved: the first
    mini_batch_size (clean) tokens attend among themselves, the rest over the last kv_cache_size clean keys and their
    own; (3) with a cache ([2 b, l_c, h, d]: keys of all entries, then values): full attention over cache + k."""
    if kv_cache is None and not interleave:
        return block_attention(q, k, v)
    if interleave:
        mb = mini_batch_size
        o_clean = block_attention(q[:, :mb], k[:, :mb], v[:, :mb])
        o_rest = block_attention(q[:, mb:], k[:, mb - kv_cache_size:], v[:, mb - kv_cache_size:])
        return torch.cat([o_clean, o_rest], dim=1)
    k_cache, v_cache = kv_cache.chunk(2, dim=0)
    every = (q, k_cache, v_cache, k, v)
    if (all(t.is_cuda and t.dtype == BF16 and t.dim() == 4 and t.device == q.device for t in every) and k.shape == v.shape
            and k_cache.shape == v_cache.shape and all(t.shape[0] == q.shape[0] and t.shape[2:] == q.shape[2:] for t in every)
            and q.shape[3] in (64, 128) and min(t.shape[1] for t in every) > 0):
        return L.call(_op("swa_fwd_cache"), *every, q.shape[3] ** -0.5)   # (the keys are read where they lie)
    return block_attention(q, torch.cat([k_cache, k], dim=1), torch.cat([v_cache, v], dim=1))

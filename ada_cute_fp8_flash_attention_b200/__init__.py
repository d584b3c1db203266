"""B200-native (sm_100a) FP8 flash-attention forward.

Drop-in for the module ``ada_cute_fp8_flash_attention`` of
Lemon7-UP/ada_cute_fp8_flash_attention, whose only export is
``flash_attn_fp8_forward(q, k, v)`` (csrc/attention_api.cpp:6-9):

* ``q``, ``k``: ``torch.float8_e4m3fn`` of shape (B, H, S, D), D in {64, 128};
* ``v``: ``torch.float8_e4m3fn`` pre-transposed to (B, H, D, S) (test.py:51-52);
* causal attention with scale 1/sqrt(D) (csrc/flash_attention.cu:524);
* returns fp16 O of shape (B, H, S, D).

The computation runs in the native library ``libfa8.so`` (C ABI,
``include/fa8.h``) through the PyTorch extension ``_fa8_torch``. There is no
CPU or eager-PyTorch fallback: importing this package raises ImportError when
the native extension has not been built (``python
ada_cute_fp8_flash_attention_b200/_build.py``).
"""
from __future__ import annotations

import importlib.util
import sys
from typing import Any, NamedTuple

from . import _build

__all__ = [
    "flash_attn_fp8_forward",
    "flash_attn_fp8_forward_ex",
    "flash_attn_fp8_varlen_forward",
    "flash_attn_fp8_backward",
    "lse_merge",
    "quantize_e4m3",
    "KVCacheFP8",
    "kv_cache_alloc",
    "kv_cache_write",
    "kv_cache_read",
    "flash_attn_fp8_decode",
    "flash_attn_fp8_shared_prefix",
    "launch_count",
]


def _load_ext():
    path = _build.ext_path()
    if not path.exists():
        raise ImportError(
            f"native extension {path.name} is not built; run "
            "`python ada_cute_fp8_flash_attention_b200/_build.py` (no CPU fallback exists)")
    import torch  # noqa: F401  (loads libc10 / libtorch for the extension)

    name = f"{__name__}.{_build.EXT_NAME}"
    spec = importlib.util.spec_from_file_location(name, str(path))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    sys.modules[name] = mod
    return mod


_C = _load_ext()


def flash_attn_fp8_forward(q, k, v):
    """Reference-compatible entry point: causal FP8 attention, V in (B,H,D,S), fp16 out."""
    return _C.flash_attn_fp8_forward(q, k, v)


def flash_attn_fp8_forward_ex(q, k, v, causal=True, softmax_scale=None, v_layout="bhds",
                              return_lse=False, out_dtype="fp16", q_offset=0, kv_offset=0,
                              split_keys=-1, out=None, lse=None, descale_q=1.0, descale_k=1.0,
                              descale_v=1.0, sm_budget=0):
    """FP8 attention forward with options.

    Returns ``out`` or ``(out, lse)`` when ``return_lse`` is set. ``lse`` is the
    natural-log log-sum-exp of the scaled scores per query row (fp32, (B,H,S)),
    ``-inf`` for rows with no visible key. ``q_offset``/``kv_offset`` are global
    positions used by the causal mask (context-parallel chunks). ``split_keys``:
    query tiles whose first row sees fewer keys than this use a two-term (hi +
    lo) e4m3 P; -1 = default (1024), 0 = never. ``descale_q/k/v``: dequantisation
    factors of scaled e4m3 inputs (real value = code x factor), each a float
    (per tensor) or a device tensor that broadcasts to (B, H) for Q and to
    (B, H_kv) for K and V (per batch and head). ``sm_budget`` > 0 runs the kernel
    on at most that many SMs (a multiple of 8) of a green-context partition,
    leaving the rest to concurrent work such as NCCL transfers; 0 = whole GPU.
    """
    import torch

    def split(d):
        return (1.0, d) if isinstance(d, torch.Tensor) else (float(d), None)
    (sq, tq), (sk, tk), (sv, tv) = split(descale_q), split(descale_k), split(descale_v)
    res = _C.flash_attn_fp8_forward_ex(q, k, v, causal, softmax_scale, v_layout, return_lse,
                                       out_dtype, q_offset, kv_offset, split_keys, out, lse,
                                       sq, sk, sv, tq, tk, tv, int(sm_budget))
    return (res[0], res[1]) if return_lse else res[0]


def flash_attn_fp8_varlen_forward(q, k, v, cu_seqlens_q, cu_seqlens_kv, max_seqlen_q,
                                  causal=True, softmax_scale=None, v_layout="thd",
                                  return_lse=False, out_dtype="fp16", status=None):
    """FP8 attention over packed variable-length sequences.

    q: (total_q, H, D), k: (total_kv, H_kv, D), v: (total_kv, H_kv, D) ("thd", read
    in place) or (H_kv, D, total_kv) ("hdt"), all e4m3; cu_seqlens_*: int32 prefix
    sums (batch+1) on q's device. Every cu_seqlens_kv entry must be a multiple of 16.
    The offsets are never read on the host (no device synchronisation): the kernel
    refuses a sequence that breaks the rules, leaves it unwritten and ORs a bit into
    ``status`` (optional int32 device tensor): 2 = unaligned K/V start, 4 = offsets
    outside the packed tensors or a sequence longer than ``max_seqlen_q``.
    Returns out (total_q, H, D) or (out, lse (H, total_q)).
    """
    res = _C.flash_attn_fp8_varlen_forward(q, k, v, cu_seqlens_q, cu_seqlens_kv,
                                           int(max_seqlen_q), causal, softmax_scale, v_layout,
                                           return_lse, out_dtype, status)
    return (res[0], res[1]) if return_lse else res[0]


def flash_attn_fp8_backward(q, k, v, out, grad_out, lse, causal=True, softmax_scale=None,
                            v_layout="bhds"):
    """Gradients of the FP8 attention with respect to its e4m3 inputs.

    q (B,H,S_q,D), k (B,H_kv,S_kv,D), v (B,H_kv,D,S_kv) for "bhds" or (B,H_kv,S_kv,D)
    for "bhsd", all e4m3; ``out`` (fp16) and ``lse`` (fp32 (B,H,S_q)) as the forward
    returned them (``return_lse=True``); ``grad_out`` fp16 like ``out``. P is
    recomputed exactly in fp32. Returns (dq, dk, dv) in fp32; dk and dv are
    (B, H_kv, S_kv, D) with the query heads of each K/V head summed. The
    reference has no backward; this is the gradient of the same forward.
    """
    dq, dk, dv = _C.flash_attn_fp8_backward(q, k, v, out, grad_out, lse, causal, softmax_scale,
                                            v_layout)
    return dq, dk, dv


def lse_merge(outs, lses):
    """Merge partial outputs of the same rows: returns (fp16 out, fp32 lse)."""
    o, l = _C.lse_merge(list(outs), list(lses))
    return o, l


def quantize_e4m3(x, scale=1.0, transpose_last2=False):
    """fp16/bf16 -> e4m3 (RNE, saturating at +-448), optionally transposing the last 2 dims."""
    return _C.quantize_e4m3(x, scale, transpose_last2)


class KVCacheFP8(NamedTuple):
    """A paged e4m3 key/value cache: the tensors and nothing else.

    ``k``, ``v``: float8_e4m3fn (pages, H_kv, page_size, D), unit last stride, the
    other strides multiples of 16 (a (pages, page_size, H_kv, D) tensor is passed as
    its ``transpose(1, 2)``); ``k_exp``, ``v_exp``: uint8 (pages, H_kv, page_size),
    unit last stride, the others multiples of 16. The row of a token and head has the values
    ``code * 2**(exp - 127)``; 255 marks a row that held an infinity or a NaN and
    reads as NaN. Codes are finite (``kv_cache_write`` stores no others); any other byte
    may be given, and rows of any size stand beside each other (attention over V rows
    with bytes outside 80..160 takes several times as long). page_size is 16, 32, 64 or a
    multiple of 128, D 64 or 128.
    """
    k: Any
    v: Any
    k_exp: Any
    v_exp: Any


def kv_cache_alloc(num_pages, heads_kv, page_size, head_dim, device="cuda"):
    """A new ``KVCacheFP8`` on ``device``: zero codes, unit exponents."""
    import torch
    shape = (num_pages, heads_kv, page_size)

    def codes():
        return torch.zeros(*shape, head_dim, dtype=torch.uint8, device=device).view(
            torch.float8_e4m3fn)

    def exps():
        return torch.full(shape, 127, dtype=torch.uint8, device=device)
    return KVCacheFP8(codes(), codes(), exps(), exps())


def kv_cache_write(cache, k, v, page_table, seqlens, cu_seqlens=None, status=None):
    """Quantise new tokens' K and V into a paged e4m3 cache (in place).

    ``page_table`` int32 (batch, max_pages): token t of sequence b lies in slot
    t % page_size of page ``page_table[b, t // page_size]``. ``seqlens`` int32
    (batch): tokens each sequence holds with the new ones, as
    ``flash_attn_fp8_decode`` takes it; the new tokens are its last. ``k``, ``v``
    (fp16 or bf16): (batch, H_kv, S_new, D), or packed (tokens, H_kv, D) with
    ``cu_seqlens`` int32 (batch + 1); rows outside cu_seqlens[0]..cu_seqlens[-1]
    are ignored. Every row gets the least power of two that brings its largest
    magnitude to 448 or less (2**-63 at least) and e4m3 codes rounded once to
    nearest even.

    Tables and lengths are never read on the host. What does not fit is not
    written and ORs a bit into ``status`` (optional int32 device tensor): 4 = a
    sequence longer than its table row, or shorter than its new tokens; 8 = a page
    id outside the cache. No two tokens of a call may share a slot.
    """
    _C.kv_cache_write(cache[0], cache[1], cache[2], cache[3], k, v, page_table, seqlens,
                      cu_seqlens, status)


def kv_cache_read(cache, page_table, seqlens, cu_seqlens, total, dtype="fp16", out=None,
                  status=None):
    """Each sequence's last tokens read back from a paged e4m3 cache: (k, v).

    With ``cu_seqlens`` int32 (batch + 1) the last cu_seqlens[b + 1] - cu_seqlens[b]
    tokens of sequence b, packed (total, H_kv, D); with ``cu_seqlens=None`` the last
    ``total`` tokens of each, (batch, H_kv, total, D). ``dtype`` "fp16" or "bf16":
    ``code * 2**(exp - 127)`` rounded once, saturating. ``out``: (k, v) tensors to
    write to; rows outside cu_seqlens[0]..cu_seqlens[-1] and refused sequences
    (``status`` bit 4) are left as they were there (and undefined without ``out``),
    tokens on a page id outside the cache (bit 8) are NaN. ``total`` is a host
    number: nothing is read from the device.
    """
    ok, ov = (None, None) if out is None else out
    k, v = _C.kv_cache_read(cache[0], cache[1], cache[2], cache[3], page_table, seqlens,
                            cu_seqlens, total, dtype, ok, ov, status)
    return k, v


def flash_attn_fp8_decode(q, cache, page_table, seqlens, softmax_scale=None, return_lse=False,
                          out=None, status=None):
    """Attention of each sequence's last tokens over a paged e4m3 cache.

    ``q`` fp16 or bf16 (B, H, S_q, D), S_q = 1 for a decoding step, more for drafted
    tokens or a chunk of a prompt; ``cache``, ``page_table`` (B, max_pages) and
    ``seqlens`` (B) as ``kv_cache_write`` left them, the S_q tokens included: query i
    of sequence b has position seqlens[b] - S_q + i and sees the keys up to it. H is a
    multiple of the cache's H_kv. Returns ``out`` (q's shape and dtype) or
    ``(out, lse)``, lse fp32 (B, H, S_q), natural log; queries that see no key give 0
    and -inf. Lengths stay on the device and any mixture of them shares the GPU
    evenly. ``status`` (optional int32 device tensor) bits: 4 = a sequence whose
    length does not fit its table row, left unwritten; 8 = a page id outside the
    cache, its sequence's queries that see it are NaN; 1 = a wait inside the kernel
    gave up. For serving: nothing is recorded for a backward pass.
    """
    res = _C.flash_attn_fp8_decode(q, cache[0], cache[1], cache[2], cache[3], page_table, seqlens,
                                   0, softmax_scale, return_lse, out, status)
    return (res[0], res[1]) if return_lse else res[0]


def flash_attn_fp8_shared_prefix(q, cache, page_table, seqlens, prefix_len, softmax_scale=None,
                                 return_lse=False, out=None, status=None):
    """``flash_attn_fp8_decode`` for a batch whose sequences begin with the same tokens.

    Of the first ``prefix_len`` tokens (a host number, any value a table row can hold)
    those in whole pages, the first ``prefix_len // page_size`` columns, are taken from
    ``page_table``'s row 0 for all sequences: row 0 lists these pages whatever
    ``seqlens[0]`` is, and the other rows' entries for them are not read. Tokens behind
    them, the page that the prefix ends in among them, come from each sequence's own
    row. All the batch's queries meet the shared pages together; a prefix too short for
    that to pay is met by each sequence for itself, from the same pages. The result is
    that of ``flash_attn_fp8_decode`` up to the order of its sums, given that every
    row's first prefix_len tokens hold what row 0's hold. Sequences shorter than the
    prefix, the first one too, see their own length of it.
    """
    res = _C.flash_attn_fp8_decode(q, cache[0], cache[1], cache[2], cache[3], page_table, seqlens,
                                   int(prefix_len), softmax_scale, return_lse, out, status)
    return (res[0], res[1]) if return_lse else res[0]


def launch_count():
    """Kernel launches issued through the C ABI by this process."""
    return _C.launch_count()

"""Operators that read the passages a search found: the embedding lookup of gathered tokens and the
attention of a question to the states of its passages, each with its gradient.

``DeviceTokenStore.gather`` (``art_amd.token_store``) leaves padded token rows and their lengths on the
GPU; what follows in the reference is the model that reads them (``megatron/model/art_model.py``): an
embedding lookup (``megatron/mpu/layers.py``, VocabParallelEmbedding), an encoder, and a decoder whose
cross attention reads the encoder's states (``megatron/model/transformer.py``, AttnType.cross_attn).
Both operators here take the gather's lengths and never touch what lies behind them.

All work runs in libartread.so (include/artread.h) on the current stream of the tensors' device.  A
call allocates its outputs and workspace from torch's allocator on that stream, keeps nothing for the
next call and never waits for the host, so it may be captured into a graph.  To capture gradients, use
``cross_attention_grad`` and ``embed_tokens_grad``: autograd's own bookkeeping of leaves that are
shared with an eager graph does not survive a capture.

Derivatives are reverse-mode only: tensors with a forward-mode tangent are refused, since the call would drop it.
So are calls under ``torch.jit.trace`` and ``make_fx``, which would record the outputs and not what fills them.
"""
import ctypes
import math
import os
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from .engine import _on_device

_HERE = os.path.dirname(os.path.abspath(__file__))
READ_LIB_PATH = os.path.join(_HERE, "lib", "libartread.so")
READ_SYMBOLS = ("artread_embed", "artread_embed_grad_workspace", "artread_embed_grad",
                "artread_attend_workspace", "artread_attend", "artread_attend_grad_workspace",
                "artread_attend_grad", "artread_last_error")
MAX_HEAD_DIM = 128
MAX_ROW = 1 << 20   # elements of an embedding
_ABI = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # ARTREAD_F16, ARTREAD_BF16, ARTREAD_F32
_lib = None

_vp, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class AttendArgs(ctypes.Structure):
    """artread_attend_t"""
    _fields_ = ([(n, _vp) for n in ("q", "k", "v", "lengths", "out", "lse", "rest")]
                + [(n, _i64) for n in ("batch", "rows", "passages", "len", "heads", "kv_heads", "dim",
                                       "q_batch", "q_row", "q_head",
                                       "k_batch", "k_passage", "k_row", "k_head",
                                       "v_batch", "v_passage", "v_row", "v_head")]
                + [("dtype", _i32), ("scale", ctypes.c_float)])


class AttendGrads(ctypes.Structure):
    """artread_attend_grads_t"""
    _fields_ = [("grad_out", _vp), ("g_batch", _i64), ("g_row", _i64), ("g_head", _i64),
                ("grad_q", _vp), ("grad_k", _vp), ("grad_v", _vp)]


class ArtreadError(RuntimeError):
    def __init__(self, code, message):
        super().__init__("artread error %d: %s" % (code, message))
        self.code = code


def _read():
    """Load libartread.so on first use; there is no fallback (fails loudly if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(READ_LIB_PATH):
            raise ImportError("%s is missing: run art_amd/csrc/build.sh (or __graft_entry__.build())"
                              % READ_LIB_PATH)
        lib = ctypes.CDLL(READ_LIB_PATH)
        f32, args, grads = ctypes.c_float, _vp, _vp   # the two structures, as their bytes or by reference
        lib.artread_embed.argtypes = [_i32, _vp, _i32, _i64, _i64, _i64, _vp, _i32, _vp, _i64, _i64, _i64, f32,
                                      _vp, _i32, _vp]
        lib.artread_embed.restype = _i32
        lib.artread_embed_grad_workspace.argtypes = [_i64, _i64, _i64, _i64]
        lib.artread_embed_grad_workspace.restype = _i64
        lib.artread_embed_grad.argtypes = [_i32, _vp, _i32, _vp, _i32, _vp, _i64, _i64, _i64, _i64, _i64, f32,
                                           _vp, _i32, _vp, _i64, _vp]
        lib.artread_embed_grad.restype = _i32
        lib.artread_attend_workspace.argtypes = [args]
        lib.artread_attend_workspace.restype = _i64
        lib.artread_attend.argtypes = [_i32, args, _vp, _i64, _vp]
        lib.artread_attend.restype = _i32
        lib.artread_attend_grad_workspace.argtypes = [args]
        lib.artread_attend_grad_workspace.restype = _i64
        lib.artread_attend_grad.argtypes = [_i32, args, grads, _vp, _i64, _vp]
        lib.artread_attend_grad.restype = _i32
        lib.artread_last_error.argtypes = []
        lib.artread_last_error.restype = ctypes.c_char_p
        _lib = lib
    return _lib


def _rcheck(rc):
    if rc != 0:
        raise ArtreadError(rc, _read().artread_last_error().decode("utf-8", "replace"))


_tracing_state, _dispatch_modes = torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack


def _refuse_tangents(*tensors):
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("forward-mode derivatives are not implemented: a tensor has a tangent")


def _one_device(first, *others):
    """Every tensor of a call lives on one GPU: the kernels read them all by address.  What torch would keep
    beside a tensor's values, and a call by address would lose, is refused first."""
    if forward_ad._current_level >= 0:   # inside a dual level
        _refuse_tangents(first, *others)
    if _tracing_state() is not None or _dispatch_modes() and get_proxy_mode() is not None:
        raise NotImplementedError("a traced graph would hold the outputs' allocation but not the call that fills them")
    if not first.is_cuda:
        raise ValueError("tensors must be on a GPU, got %s" % first.device)
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError("all tensors of a call must be on one device, got %s and %s" % (first.device, t.device))
    return first.device


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def _scale_value(scale):
    scale = float(scale)
    if not abs(scale) < 3.4e38:   # of a 32-bit float
        raise ValueError("scale must be finite, got %r" % scale)
    return scale


def _base_value(base):
    base = int(base)
    if not -(1 << 63) <= base < 1 << 63:
        raise ValueError("vocab_base must fit 64 bits, got %d" % base)
    return base


# ---- embedding lookup -----------------------------------------------------------------------------
def _check_tokens(tokens, lengths):
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.dim() < 1:
        raise ValueError("tokens must be an int32 or int64 tensor [..., len]")
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != tokens.shape[:-1]):
        raise ValueError("lengths must be an int32 tensor %s, one per row of tokens"
                         % (tuple(tokens.shape[:-1]),))
    if tokens.numel() >= 1 << 31:
        raise ValueError("tokens holds %d positions, the limit is 2**31 - 1" % tokens.numel())


def _check_row(dim):
    if dim > MAX_ROW:
        raise ValueError("an embedding holds at most %d elements, got %d" % (MAX_ROW, dim))


def _embed(tokens, table, lengths, scale, vocab_base, out_dtype):
    dev, shape = table.device, tokens.shape
    vocab, dim = table.shape
    out = torch.empty((*shape, dim), dtype=out_dtype, device=dev)
    positions, length = tokens.numel(), shape[-1]
    if positions * dim == 0:
        return out
    tokens = tokens.contiguous()
    lengths = lengths.contiguous() if lengths is not None else None
    with _on_device(dev):
        _rcheck(_read().artread_embed(
            dev.index, table.data_ptr(), _ABI[table.dtype], vocab, dim, table.stride(0), tokens.data_ptr(),
            tokens.element_size(), lengths.data_ptr() if lengths is not None else None, positions // length, length,
            vocab_base, scale, out.data_ptr(), _ABI[out_dtype], _stream(dev)))
    return out


def _embed_grad(grad_out, tokens, lengths, vocab, scale, vocab_base, dtype):
    dev, dim, length, positions = grad_out.device, grad_out.shape[-1], tokens.shape[-1], tokens.numel()
    if positions * dim == 0:
        return torch.zeros((vocab, dim), dtype=dtype, device=dev)
    out = torch.empty((vocab, dim), dtype=dtype, device=dev)
    grad_out, tokens = grad_out.contiguous(), tokens.contiguous()
    lengths = lengths.contiguous() if lengths is not None else None
    n, lib = positions // length, _read()
    size = lib.artread_embed_grad_workspace(vocab, dim, n, length)
    with _on_device(dev):
        ws = torch.empty((size,), dtype=torch.uint8, device=dev)
        _rcheck(lib.artread_embed_grad(
            dev.index, grad_out.data_ptr(), _ABI[grad_out.dtype], tokens.data_ptr(), tokens.element_size(),
            lengths.data_ptr() if lengths is not None else None, n, length, vocab, dim, vocab_base, scale,
            out.data_ptr(), _ABI[dtype], ws.data_ptr(), size, _stream(dev)))
    return out


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, lengths, scale, vocab_base, out_dtype):
        ctx.save_for_backward(tokens, lengths)
        ctx.of = (table.shape[0], scale, vocab_base, table.dtype)
        return _embed(tokens, table, lengths, scale, vocab_base, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        tokens, lengths = ctx.saved_tensors
        vocab, scale, vocab_base, dtype = ctx.of
        if forward_ad._current_level >= 0:
            _refuse_tangents(grad_out)
        return _embed_grad(grad_out, tokens, lengths, vocab, scale, vocab_base, dtype), None, None, None, None, None


def embed_tokens(tokens, table, lengths=None, scale=1.0, vocab_base=0, out_dtype=None):
    """``scale * table[tokens - vocab_base]`` for the valid positions of padded token rows, zeros elsewhere.

    tokens: CUDA int32 or int64 [..., len], lengths: int32 [...] (None: every position is valid), both as
    ``DeviceTokenStore.gather`` returns them.  table: [vocab, dim], float16, bfloat16 or float32 with
    contiguous rows.  A token outside [vocab_base, vocab_base + vocab) gives zeros, so the lookups of a
    vocabulary split over ranks add up.  Returns [..., len, dim] of the table's type, or of ``out_dtype``
    (float16 or bfloat16 from a float32 table); the product is formed in 32 bits and rounded once.
    Differentiable in ``table``."""
    _check_tokens(tokens, lengths)
    if table.dim() != 2 or table.dtype not in _ABI or table.shape[0] < 1 or table.shape[0] >= 1 << 31:
        raise ValueError("table must be a float16, bfloat16 or float32 tensor [vocab, dim]")
    if table.shape[1] > 1 and table.stride(1) != 1 or table.stride(0) < table.shape[1] and table.shape[0] > 1:
        raise ValueError("the rows of table must be contiguous and must not overlap")
    _check_row(table.shape[1])
    out_dtype = table.dtype if out_dtype is None else out_dtype
    if out_dtype != table.dtype and (table.dtype != torch.float32 or out_dtype not in _ABI):
        raise ValueError("out_dtype must be the table's type, or float16 / bfloat16 of a float32 table")
    scale, vocab_base = _scale_value(scale), _base_value(vocab_base)
    _one_device(table, tokens, lengths)
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbedTokens.apply(table, tokens, lengths, scale, vocab_base, out_dtype)
    return _embed(tokens, table, lengths, scale, vocab_base, out_dtype)


def embed_tokens_grad(grad_out, tokens, vocab, lengths=None, scale=1.0, vocab_base=0, dtype=None):
    """Gradient of ``embed_tokens`` in its table: [vocab, dim], every row written (zeros where no valid
    position holds the token).  The tokens are sorted and each row is the 32-bit sum of its positions in a
    fixed order, rounded once: equal inputs give equal bits.  ``dtype`` is grad_out's type (default) or
    float32.  Not differentiable itself."""
    _check_tokens(tokens, lengths)
    if grad_out.dtype not in _ABI or grad_out.dim() < 2 or grad_out.shape[:-1] != tokens.shape:
        raise ValueError("grad_out must be a float16, bfloat16 or float32 tensor %s"
                         % (tuple(tokens.shape) + ("dim",),))
    _check_row(grad_out.shape[-1])
    vocab = int(vocab)
    if not 1 <= vocab < 1 << 31:
        raise ValueError("vocab must be in [1, 2**31), got %d" % vocab)
    dtype = grad_out.dtype if dtype is None else dtype
    if dtype != grad_out.dtype and dtype != torch.float32:
        raise ValueError("dtype must be grad_out's type or float32")
    scale, vocab_base = _scale_value(scale), _base_value(vocab_base)
    _one_device(grad_out, tokens, lengths)
    return _embed_grad(grad_out, tokens, lengths, vocab, scale, vocab_base, dtype)


# ---- cross attention ------------------------------------------------------------------------------
# artread_attend_t as bytes: filling a ctypes structure field by field costs more than the smallest launch
_pack_args = struct.Struct("=7Q18qif").pack
_pack_grads = struct.Struct("=Q3q3Q").pack


def _plan(query, key, value, lengths, scale):
    """Checks a call and returns (sizes, scale): sizes are batch, rows, passages, len, heads, kv_heads, dim."""
    q_shape, k_shape = query.shape, key.shape
    if len(q_shape) != 4 or len(k_shape) not in (4, 5) or value.shape != k_shape:
        raise ValueError("query must be [batch, rows, heads, dim], key and value [batch, len, kv_heads, dim] or "
                         "[batch, passages, len, kv_heads, dim]")
    dtype = query.dtype
    if dtype not in (torch.float16, torch.bfloat16) or key.dtype != dtype or value.dtype != dtype:
        raise ValueError("query, key and value must share a type, float16 or bfloat16")
    batch, rows, heads, dim = q_shape
    passages, (length, kv_heads) = (k_shape[1] if len(k_shape) == 5 else 1), k_shape[-3:-1]
    if k_shape[0] != batch or k_shape[-1] != dim:
        raise ValueError("key %s does not fit query %s" % (tuple(k_shape), tuple(q_shape)))
    if dim < 8 or dim > MAX_HEAD_DIM or dim % 8:
        raise ValueError("the head size must be a multiple of 8 up to %d, got %d" % (MAX_HEAD_DIM, dim))
    if kv_heads < 1 or heads % kv_heads:
        raise ValueError("%d query heads cannot share %d key heads" % (heads, kv_heads))
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != k_shape[:-3]):
        raise ValueError("lengths must be an int32 tensor %s, one per passage" % (tuple(k_shape[:-3]),))
    if max(batch * rows * heads, batch * passages * length * kv_heads) >= 1 << 31 or passages * length > (1 << 31) - (1 << 20):
        raise ValueError("query and key hold at most 2**31 - 1 rows each, a batch entry at most 2**31 - 2**20 states")
    return (batch, rows, passages, length, heads, kv_heads, dim), _scale_value(dim ** -0.5 if scale is None else scale)


def _layout(t, share=1):
    """`t` [batch, (passages,) rows, heads, dim] and the strides of all its dimensions but the last, in the layout
    the kernels address: innermost stride 1, the others multiples of 8 elements, rows less than 2**24 apart, the
    `share` query heads of a key head within 2**29, 16-byte aligned.  Anything else is copied."""
    strides = t.stride()
    *outer, row, head, one = strides
    if one != 1 or t.data_ptr() & 15 or (row | head) & 7 or any(x & 7 for x in outer) or row >= 1 << 24 or share * head >= 1 << 29:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = t.stride()
    return t, (strides if len(strides) == 5 else (strides[0], 0) + strides[1:])


def _args(query, key, value, lengths, out, lse, rest, sizes, scale):
    """artread_attend_t of a call, and the tensors it points into."""
    share = sizes[4] // sizes[5]
    query, (q_batch, _, q_row, q_head, _) = _layout(query, share)
    key, k_strides = _layout(key)
    value, v_strides = _layout(value)
    if lengths is not None:
        lengths = lengths.contiguous()
    return (_pack_args(query.data_ptr(), key.data_ptr(), value.data_ptr(),
                       lengths.data_ptr() if lengths is not None else 0, out.data_ptr(),
                       lse.data_ptr() if lse is not None else 0, rest.data_ptr() if rest is not None else 0, *sizes,
                       q_batch, q_row, q_head, *k_strides[:4], *v_strides[:4], _ABI[query.dtype], scale),
            (query, key, value, lengths))


def _attend(query, key, value, lengths, sizes, scale, want_lse, want_rest):
    dev = query.device
    batch, rows, passages, length, heads, kv_heads, dim = sizes
    out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    lse = torch.empty((batch, heads, rows), dtype=torch.float32, device=dev) if want_lse else None
    rest = torch.empty_like(out) if want_rest else None
    if not (batch and rows and heads and passages and length):
        out.zero_()
        return out, lse.fill_(-math.inf) if want_lse else None, rest.zero_() if want_rest else None
    args, _held = _args(query, key, value, lengths, out, lse, rest, sizes, scale)
    lib = _read()
    size = lib.artread_attend_workspace(args)
    with _on_device(dev):
        ws = torch.empty((size,), dtype=torch.uint8, device=dev) if size > 0 else None
        _rcheck(lib.artread_attend(dev.index, args, ws.data_ptr() if ws is not None else None, size, _stream(dev)))
    return out, lse, rest


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, lengths, sizes, scale, want_saved):
        out, lse, rest = _attend(query, key, value, lengths, sizes, scale, True, True)
        ctx.save_for_backward(query, key, value, lengths, out, lse, rest)
        ctx.of = sizes, scale
        if not want_saved:   # each further result costs the call some microseconds
            return out
        ctx.mark_non_differentiable(lse, rest)
        ctx.set_materialize_grads(False)   # no zeros for lse and rest
        return out, lse, rest

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, *_):
        if grad_out is None:
            return (None,) * 7
        query, key, value, lengths, out, lse, rest = ctx.saved_tensors
        _one_device(query, grad_out)
        return _attend_grad(grad_out, query, key, value, lengths, out, lse, rest, *ctx.of) + (None, None, None, None)


def cross_attention(query, key, value, lengths=None, scale=None, return_lse=False, return_saved=False):
    """Attention of ``query`` [batch, rows, heads, dim] to the states of each batch entry's passages:
    ``key`` and ``value`` [batch, passages, len, kv_heads, dim] with ``lengths`` int32 [batch, passages]
    (``DeviceTokenStore.gather``'s), or [batch, len, kv_heads, dim] with [batch]; None: all of len.

    One softmax of ``scale * query . key`` (default scale: dim ** -0.5) runs over the valid entries of all
    passages of a batch entry.  A row without any gives zeros and an lse of -inf.  Padding is neither read
    into the result nor worked on.  ``heads`` is a multiple of ``kv_heads``; head h reads key head
    ``h // (heads // kv_heads)``.  float16 or bfloat16, dim a multiple of 8 up to 128; any strides (rows
    that are not 16-byte aligned are copied first).  ``rows`` of 1 is the single-token form.  Several
    answers read from the same passages (beams, samples) are further rows.

    Returns [batch, rows, heads, dim], with ``return_lse`` also the float32 [batch, heads, rows] log of the
    softmax's sum (not differentiable), with ``return_saved`` instead what ``cross_attention_grad`` takes: that
    log and what rounding took from the result.  Differentiable in query, key and value.

    Statistics and sums are 32 bits, the weights are rounded once to the inputs' type.  Equal inputs give equal
    bits; the last ones may depend on whether passages lie one behind the other in memory or with gaps."""
    sizes, scale = _plan(query, key, value, lengths, scale)
    _one_device(query, key, value, lengths)
    if (query.requires_grad or key.requires_grad or value.requires_grad) and torch.is_grad_enabled():
        if not (return_lse or return_saved):
            return _CrossAttention.apply(query, key, value, lengths, sizes, scale, False)
        out, lse, rest = _CrossAttention.apply(query, key, value, lengths, sizes, scale, True)
    else:
        out, lse, rest = _attend(query, key, value, lengths, sizes, scale, return_lse or return_saved, return_saved)
    if return_saved:
        return out, (lse, rest)
    return (out, lse) if return_lse else out


def _attend_grad(grad_out, query, key, value, lengths, out, lse, rest, sizes, scale):
    dev = query.device
    batch, rows, passages, length, heads, kv_heads, dim = sizes
    grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (query, key, value)]
    if not (batch and rows and heads and passages and length):
        return tuple(t.zero_() for t in grads)
    args, _held = _args(query, key, value, lengths, out, lse, rest, sizes, scale)
    grad_out, (g_batch, _, g_row, g_head, _) = _layout(grad_out, heads // kv_heads)
    more = _pack_grads(grad_out.data_ptr(), g_batch, g_row, g_head, *[t.data_ptr() for t in grads])
    lib = _read()
    size = lib.artread_attend_grad_workspace(args)
    with _on_device(dev):
        ws = torch.empty((size,), dtype=torch.uint8, device=dev) if size > 0 else None
        _rcheck(lib.artread_attend_grad(dev.index, args, more, ws.data_ptr() if ws is not None else None, size,
                                        _stream(dev)))
    return tuple(grads)


def cross_attention_grad(grad_out, query, key, value, out, saved, lengths=None, scale=None):
    """Gradients (query, key, value) of ``cross_attention`` from its result ``out`` and what it ``saved``.
    Written whole, zeros behind each passage's length; equal inputs in equal layouts give equal bits.  Not
    differentiable itself."""
    sizes, scale = _plan(query, key, value, lengths, scale)
    if grad_out.shape != query.shape or grad_out.dtype != query.dtype:
        raise ValueError("grad_out must have query's shape and type")
    lse, rest = saved
    for t in (out, rest):
        if t.shape != query.shape or t.dtype != query.dtype or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError("out and saved must be what cross_attention returned")
    batch, rows, heads, _ = query.shape
    if lse.shape != (batch, heads, rows) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError("out and saved must be what cross_attention returned")
    _one_device(query, key, value, lengths, grad_out, out, lse, rest)
    return _attend_grad(grad_out, query, key, value, lengths, out, lse, rest, sizes, scale)


__all__ = ["embed_tokens", "embed_tokens_grad", "cross_attention", "cross_attention_grad", "ArtreadError"]

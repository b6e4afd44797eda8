"""Op-level entry points over device buffers (torch CUDA tensors as plumbing).

``mesh_forward`` / ``mesh_backward`` wrap ``mb_op_mesh_forward`` /
``mb_op_mesh_backward``: one two-parent mesh stack, the per-op boundary of
the reference's ``gpt_mesh`` and ``gpt_mesh_gradient`` kernels
(src/gpt/gpu.rs:103-146, :1087-1149).  The other wrappers follow the
remaining ``mb_op_*`` entry points: RMSNorm (:65-94, :1035-1077), RoPE
(:175-208), causal attention (:381-779), XSA (:781-897), the tied head and
cross-entropy (:927-1021) and AdamW (:1369-1391).  Operands are [rows][width]
row-major float32 CUDA tensors; each call runs on torch's current stream.

The serving operators (no reference counterpart) take float32, bfloat16 or
float16 rows of any row and head stride: ``cache_write`` and ``cache_read``
of an 8-bit paged key/value cache (``KvCache``), ``cache_attention`` over it,
and ``token_logprobs`` with its gradient.  They do not synchronise; pass a
``new_status`` tensor to collect what only the device can see, and look at it
with ``check_status`` when convenient.
"""

import ctypes
import functools
import math
import struct
from typing import NamedTuple

from . import _lib
from ._lib import check


def _dev(t, name):
    if not (t.is_cuda and t.is_contiguous() and str(t.dtype) == "torch.float32"):
        raise ValueError(f"{name} must be a contiguous float32 CUDA tensor")
    return ctypes.c_void_p(t.data_ptr())


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def mesh_forward(x, weights, connectivity: int = 0):
    """y = stack(x); x [rows][width], weights [depth][width][2]."""
    import torch
    rows, width = x.shape
    depth = weights.shape[0]
    y = torch.empty_like(x)
    check(_lib.load().mb_op_mesh_forward(_dev(x, "x"), _dev(y, "y"), rows, width, depth, connectivity,
                                         _dev(weights, "weights"), _stream()))
    return y


def mesh_backward(x, dy, weights, connectivity: int = 0):
    """(dx, dweights) of a stack from its input x and output gradient dy."""
    import torch
    rows, width = x.shape
    depth = weights.shape[0]
    dx = torch.empty_like(x)
    dw = torch.empty_like(weights)
    check(_lib.load().mb_op_mesh_backward(_dev(x, "x"), _dev(dy, "dy"), _dev(dx, "dx"), _dev(dw, "dweights"), rows,
                                          width, depth, connectivity, _dev(weights, "weights"), _stream()))
    return dx, dw


def gemm_tf32x3(a, b, layout: int = 0):
    """FP32 GEMM via tcgen05 3xTF32, C [m][n] = A . B^T over k.  Layout bits:
    1 = b given [k][n] (else [n][k]); 2 = accepted, the same as 0 (A is always
    staged through tensor memory);
    4 = a given [k][m] (else [m][k]; not with 2)."""
    import torch
    m, k = (a.shape[1], a.shape[0]) if layout & 4 else a.shape
    n, k2 = (b.shape[1], b.shape[0]) if layout & 1 else b.shape
    if k != k2:
        raise ValueError("inner dimensions differ")
    c = torch.empty((m, n), dtype=torch.float32, device=a.device)
    status = torch.zeros(1, dtype=torch.int32, device=a.device)
    check(_lib.load().mb_op_gemm_tf32x3(_dev(a, "a"), _dev(b, "b"), _dev(c, "c"), m, n, k, layout,
                                        ctypes.c_void_p(status.data_ptr()), _stream()))
    if int(status.item()) != 0:
        raise RuntimeError("tensor-core completion wait timed out")
    return c


def _u32(t, name):
    if not (t.is_cuda and t.is_contiguous() and str(t.dtype) in ("torch.int32", "torch.uint32")):
        raise ValueError(f"{name} must be a contiguous 32-bit integer CUDA tensor")
    return ctypes.c_void_p(t.data_ptr())


def _status(device):
    import torch
    return torch.zeros(1, dtype=torch.int32, device=device)


def _raise_status(status, what):
    code = int(status.item())
    if code:
        raise RuntimeError(f"{what}: device status {code}")


def rmsnorm_forward(x, heads: int = 1):
    """(y, inv): per-(row, head) RMSNorm and 1/rms [rows][heads]."""
    import torch
    rows, width = x.shape
    y = torch.empty_like(x)
    inv = torch.empty((rows, heads), dtype=torch.float32, device=x.device)
    check(_lib.load().mb_op_rmsnorm_forward(_dev(x, "x"), _dev(y, "y"), _dev(inv, "inv"), rows, width, heads,
                                            _stream()))
    return y, inv


def rmsnorm_backward(x, dy, heads: int = 1):
    import torch
    rows, width = x.shape
    dx = torch.empty_like(x)
    check(_lib.load().mb_op_rmsnorm_backward(_dev(x, "x"), _dev(dy, "dy"), _dev(dx, "dx"), rows, width, heads,
                                             _stream()))
    return dx


def rope(x, sequence: int, heads: int, inverse: bool = False):
    import torch
    rows, width = x.shape
    y = torch.empty_like(x)
    check(_lib.load().mb_op_rope(_dev(x, "x"), _dev(y, "y"), rows, sequence, width, heads, int(inverse), _stream()))
    return y


def attention_forward(q, k, v, sequence: int, heads: int):
    """(o, lse2): causal attention per head; lse2 [heads][rows] is the
    base-2 log-sum-exp of each row's scores scaled by log2(e) / sqrt(hd)."""
    import torch
    rows, width = q.shape
    o = torch.empty_like(q)
    lse = torch.empty((heads, rows), dtype=torch.float32, device=q.device)
    status = _status(q.device)
    check(_lib.load().mb_op_attn_forward(_dev(q, "q"), _dev(k, "k"), _dev(v, "v"), _dev(o, "o"), _dev(lse, "lse"),
                                         rows, sequence, width, heads, ctypes.c_void_p(status.data_ptr()), _stream()))
    _raise_status(status, "attention forward")
    return o, lse


def attention_backward(q, k, v, o, dout, lse, sequence: int, heads: int):
    import torch
    rows, width = q.shape
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    status = _status(q.device)
    check(_lib.load().mb_op_attn_backward(_dev(q, "q"), _dev(k, "k"), _dev(v, "v"), _dev(o, "o"),
                                          _dev(dout, "dout"), _dev(lse, "lse"), _dev(dq, "dq"), _dev(dk, "dk"),
                                          _dev(dv, "dv"), rows, sequence, width, heads,
                                          ctypes.c_void_p(status.data_ptr()), _stream()))
    _raise_status(status, "attention backward")
    return dq, dk, dv


def xsa_forward(y, v, heads: int):
    import torch
    rows, width = y.shape
    z = torch.empty_like(y)
    check(_lib.load().mb_op_xsa_forward(_dev(y, "y"), _dev(v, "v"), _dev(z, "z"), rows, width, heads, _stream()))
    return z


def xsa_backward(y, v, dz, heads: int):
    import torch
    rows, width = y.shape
    dy, dv = torch.empty_like(y), torch.empty_like(v)
    check(_lib.load().mb_op_xsa_backward(_dev(y, "y"), _dev(v, "v"), _dev(dz, "dz"), _dev(dy, "dy"), _dev(dv, "dv"),
                                         rows, width, heads, _stream()))
    return dy, dv


def head_ce(h, embeddings, targets, backward: bool = True):
    """(logits, loss, dh, dembeddings) of the tied head and mean
    cross-entropy; dh and dembeddings are None without ``backward``."""
    import torch
    rows, width = h.shape
    vocab = embeddings.shape[0]
    logits = torch.empty((rows, vocab), dtype=torch.float32, device=h.device)
    loss = torch.empty(1, dtype=torch.float64, device=h.device)
    dh = torch.empty_like(h) if backward else None
    de = torch.empty_like(embeddings) if backward else None
    status = _status(h.device)
    check(_lib.load().mb_op_head_ce(_dev(h, "h"), _dev(embeddings, "embeddings"), _u32(targets, "targets"), rows,
                                    width, vocab, _dev(logits, "logits"), ctypes.c_void_p(loss.data_ptr()),
                                    _dev(dh, "dh") if backward else None,
                                    _dev(de, "dembeddings") if backward else None,
                                    ctypes.c_void_p(status.data_ptr()), _stream()))
    _raise_status(status, "head cross-entropy")
    return logits, float(loss.item()), dh, de


def adamw(weights, m, v, gradient, options, step: int):
    """One AdamW update of float32 CUDA tensors in place (update number ``step``)."""
    o = options.to_c()
    check(_lib.load().mb_op_adamw(_dev(weights, "weights"), _dev(m, "m"), _dev(v, "v"), _dev(gradient, "gradient"),
                                  weights.numel(), ctypes.byref(o), step, _stream()))


# ------------------------------------------------------------------ serving
class KvCache(NamedTuple):
    """An 8-bit paged key/value cache: int8 codes ``k`` and ``v``
    [pages][heads][page_tokens][width] and one float32 scale for each page and
    head, ``k_scale`` and ``v_scale`` [pages][heads]; a stored value is
    code * scale.  page_tokens is 16, 32, 64 or 128; width is the head width
    (1..128) rounded up to 32."""
    k: "torch.Tensor"
    v: "torch.Tensor"
    k_scale: "torch.Tensor"
    v_scale: "torch.Tensor"


class TokenLogprobs(NamedTuple):
    logprob: "torch.Tensor"      # [rows]
    entropy: "torch.Tensor"      # [rows], nats
    lse: "torch.Tensor"          # [rows], natural log
    top_logprob: "torch.Tensor"  # [rows][top]
    top_index: "torch.Tensor"    # [rows][top] int32


@functools.cache
def _torch():
    import torch
    return torch


@functools.cache
def _dtypes():
    torch = _torch()
    return {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # MB_F32, MB_BF16, MB_F16


def _dtype(dtype, name):
    code = _dtypes().get(dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16")
    return code


# The C argument structures (include/meshb200.h); every one begins with a
# cache and the rows' places where the operator has them.
_CACHE_WHERE = "4P4I3P2N2I"
_WRITE = struct.Struct(_CACHE_WHERE + "2P4NP4I")
_READ = struct.Struct(_CACHE_WHERE + "4P4I")
_ATTENTION = struct.Struct(_CACHE_WHERE + "6P3N5If")
_LOGPROBS = struct.Struct("8P2N4I")
_LOGPROBS_BACKWARD = struct.Struct("8P2N2I")


def new_kv_cache(pages: int, heads: int, head_dim: int, page_tokens: int = 32, device="cuda") -> KvCache:
    """An empty cache of ``pages`` pages."""
    import torch
    shape = (pages, heads, page_tokens, -(-head_dim // 32) * 32)
    return KvCache(torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape[:2], dtype=torch.float32, device=device),
                   torch.zeros(shape[:2], dtype=torch.float32, device=device))


def new_status(device="cuda"):
    """A zeroed device status word for the serving operators' ``status``."""
    return _status(device)


_STATUS_BITS = ((1, "a copy's wait gave up"), (2, "a page or token out of range"),
                (4, "a length below its new rows or past the table"),
                (8, "offsets outside the rows, or more new rows than announced"))


def check_status(status) -> None:
    """Waits for the status word and raises if an operator reported anything."""
    code = int(status.item())
    if code:
        raise RuntimeError("; ".join(text for bit, text in _STATUS_BITS if code & bit) or f"device status {code}")


def _cache_where(cache, table, lengths, offsets, rows):
    """(fields of the cache and of the rows' places, device index)."""
    torch = _torch()
    k, v, ks, vs = cache
    shape, device = k.shape, k.get_device()
    i8, f32, i32 = torch.int8, torch.float32, torch.int32
    if len(shape) != 4 or v.shape != shape or not (
            k.dtype is i8 and v.dtype is i8 and k.is_contiguous() and v.is_contiguous()):
        raise ValueError("cache.k and cache.v must be contiguous int8 tensors [pages][heads][page_tokens][width]")
    pages, heads, tokens, width = shape
    scales = shape[:2]
    if not (ks.shape == scales and vs.shape == scales and ks.dtype is f32 and vs.dtype is f32
            and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache.k_scale and cache.v_scale must be contiguous float32 tensors [pages][heads]")
    if table.dtype is not i32 or table.ndim != 2:
        raise ValueError("table must be an int32 tensor [batch][pages]")
    batch, per = table.shape
    stride, step = table.stride()
    if step != 1 and per > 1:
        raise ValueError("table must have adjacent page numbers")
    if batch <= 1:
        stride = per
    if lengths.dtype is not i32 or lengths.shape != (batch,) or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 tensor [batch]")
    if offsets is None:
        at = 0
    elif offsets.dtype is not i32 or offsets.shape != (batch + 1,) or not offsets.is_contiguous():
        raise ValueError("offsets must be a contiguous int32 tensor [batch + 1]")
    else:
        at = offsets.data_ptr()
        if offsets.get_device() != device:
            raise ValueError("the operands must be on one CUDA device")
    if device < 0 or not (v.get_device() == ks.get_device() == vs.get_device() == table.get_device()
                          == lengths.get_device() == device):
        raise ValueError("the operands must be on one CUDA device")
    return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, tokens, width,
            table.data_ptr(), lengths.data_ptr(), at, stride, rows, per, batch), device


def _int32(t, name, shape, device):
    """The address of an optional int32 tensor."""
    if t is None:
        return 0
    if not (t.dtype is _torch().int32 and t.get_device() == device and t.shape == shape and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor {list(shape)} on the operands' device")
    return t.data_ptr()


def _rows3(t, name, device):
    """(address, row stride, head stride) of [rows][heads][head_dim] rows."""
    row, head, channel = t.stride()
    if channel != 1 and t.shape[2] > 1:
        raise ValueError(f"{name} must have adjacent channels")
    if row < 0 or head < 0:
        raise ValueError(f"{name} must not have negative strides")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the cache's device")
    return t.data_ptr(), row, head


def _sizes(*values):
    for v in values:
        if not 0 <= v < 1 << 32:
            raise ValueError("sizes must be in 0..2^32-1")


def _current(device):
    """The current stream's handle; the operands must be on the current device."""
    torch = _torch()
    if device != torch.cuda.current_device():
        raise ValueError("operands must be on the current CUDA device")
    return torch._C._cuda_getCurrentRawStream(device)


@functools.lru_cache(maxsize=4096)
def _attention_workspace(device, *sizes):
    """Bytes that an attention of these sizes needs on this device."""
    n = ctypes.c_size_t()
    check(_lib.load().mb_op_cache_attention_workspace(*sizes, ctypes.byref(n)))
    return n.value


def cache_write(cache: KvCache, k, v, table, lengths, offsets=None, *, max_new: int = None, status=None) -> None:
    """Quantises the new rows k, v [rows][heads][head_dim] into their pages.

    ``table`` [batch][pages] int32 names each sequence's pages in order,
    ``lengths`` [batch] int32 its tokens with the new ones; rows
    offsets[b] .. offsets[b+1] are sequence b's newest (``offsets`` None: row b
    is).  ``max_new``: at least the largest number of new rows of a sequence
    (default: 1 without offsets, else all rows)."""
    if k.ndim != 3 or v.shape != k.shape or v.dtype is not k.dtype:
        raise ValueError("k and v must be [rows][heads][head_dim] of one shape and type")
    rows, heads, head_dim = k.shape
    if heads != cache[0].shape[1]:
        raise ValueError("k and v must have the cache's heads")
    if max_new is None:
        max_new = rows if offsets is not None else 1
    fields, device = _cache_where(cache, table, lengths, offsets, rows)
    at_k, k_row, k_head = _rows3(k, "k", device)
    at_v, v_row, v_head = _rows3(v, "v", device)
    _sizes(max_new)
    args = _WRITE.pack(*fields, at_k, at_v, k_row, k_head, v_row, v_head, _int32(status, "status", (1,), device),
                       head_dim, _dtype(k.dtype, "k"), max_new, 0)
    check(_lib.load().mb_op_cache_write(args, _current(device)))


def cache_read(cache: KvCache, table, lengths, tokens: int, *, first=None, head_dim: int = None, dtype=None,
               status=None):
    """(k, v) [batch][tokens][heads][head_dim]: positions first[b] ..
    first[b] + tokens - 1 (``first`` None: from 0) of each sequence, zeros
    past its length.  ``head_dim`` defaults to the cache's width, ``dtype`` to
    float32."""
    torch = _torch()
    batch = table.shape[0]
    fields, device = _cache_where(cache, table, lengths, None, batch)
    heads, width = fields[5], fields[7]
    head_dim = width if head_dim is None else head_dim
    dtype = torch.float32 if dtype is None else dtype
    code = _dtype(dtype, "dtype")
    _sizes(tokens, head_dim)
    at = _int32(first, "first", (batch,), device)
    stream = _current(device)
    shape = (batch, tokens, heads, head_dim)
    k = torch.empty(shape, dtype=dtype, device=cache[0].device)
    v = torch.empty_like(k)
    args = _READ.pack(*fields, at, k.data_ptr(), v.data_ptr(), _int32(status, "status", (1,), device), head_dim, code,
                      tokens, 0)
    check(_lib.load().mb_op_cache_read(args, stream))
    return k, v


def cache_attention(q, cache: KvCache, table, lengths, offsets=None, *, first=None, scale: float = None,
                    max_new: int = None, max_tokens: int = None, status=None):
    """(out, lse2): attention of the new rows q [rows][q_heads][head_dim] over
    their sequences' cached tokens, the new ones among them (write them
    first).  Row i of the n new ones of sequence b sees positions first[b]
    (``first`` None: 0) .. lengths[b] - n + i; query head a reads key head
    a // (q_heads // heads).  out has q's shape and type; lse2
    [q_heads][rows] is the base-2 log-sum-exp of the scaled scores times
    log2(e).  A row that sees nothing gives 0 and -inf.

    table, lengths, offsets, max_new as in ``cache_write``; ``scale`` defaults
    to 1 / sqrt(head_dim); ``max_tokens``, about the largest length, is how
    long sequences are cut over the GPU (default: what the table can hold)."""
    torch = _torch()
    if q.ndim != 3:
        raise ValueError("q must be [rows][q_heads][head_dim]")
    rows, heads, head_dim = q.shape
    fields, device = _cache_where(cache, table, lengths, offsets, rows)
    at_q, row, head = _rows3(q, "q", device)
    code = _dtype(q.dtype, "q")
    kv_heads, batch = fields[5], fields[14]
    if max_new is None:
        max_new = rows if offsets is not None else 1
    if max_tokens is None:
        max_tokens = min(fields[13] * fields[6], (1 << 31) - 1)
    _sizes(max_new, max_tokens)
    at = _int32(first, "first", (batch,), device)
    stream = _current(device)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((heads, rows), dtype=torch.float32, device=q.device)
    size = _attention_workspace(device, batch, rows, heads, kv_heads, head_dim, code, max_new, max_tokens)
    work = torch.empty(size, dtype=torch.uint8, device=q.device).data_ptr() if size else 0
    args = _ATTENTION.pack(*fields, at, at_q, out.data_ptr(), lse.data_ptr(), work,
                           _int32(status, "status", (1,), device), row, head, size, heads, head_dim, code, max_new,
                           max_tokens, 1.0 / math.sqrt(head_dim) if scale is None else scale)
    check(_lib.load().mb_op_cache_attention(args, stream))
    return out, lse


def _logit_rows(logits):
    """(address, row stride, rows, vocab, type, device) of logits."""
    if logits.ndim != 2:
        raise ValueError("logits must be [rows][vocab]")
    rows, vocab = logits.shape
    row, column = logits.stride()
    device = logits.get_device()
    if device < 0 or (column != 1 and vocab > 1) or row < 0:
        raise ValueError("logits must be a CUDA tensor [rows][vocab] with adjacent columns")
    return logits.data_ptr(), row if rows > 1 else vocab, rows, vocab, _dtype(logits.dtype, "logits"), device


def token_logprobs(logits, tokens, top: int = 0, *, status=None) -> TokenLogprobs:
    """Log-probabilities of the given ``tokens`` [rows] (int32; -1, the bits
    of IGNORE_TARGET, gives 0), entropies, and the ``top`` (0..32) most likely
    tokens of each row of ``logits`` [rows][vocab], ties to the lowest index.
    -inf masks a token; a row of masked tokens gives -inf and entropy 0."""
    torch = _torch()
    at, stride, rows, vocab, code, device = _logit_rows(logits)
    _sizes(vocab, top)
    at_tokens = _int32(tokens, "tokens", (rows,), device)
    word = _int32(status, "status", (1,), device)
    stream = _current(device)
    # one allocation: logprob, entropy, lse, then the top log-probabilities and their indices
    room = torch.empty(rows * (3 + 2 * top), dtype=torch.float32, device=logits.device)
    logprob, entropy, lse, best, index = room.split((rows, rows, rows, rows * top, rows * top))
    if rows:
        to = room.data_ptr()
        args = _LOGPROBS.pack(at, at_tokens, to, to + 4 * rows, to + 8 * rows, to + 12 * rows,
                              to + (12 + 4 * top) * rows, word, stride, rows, vocab, code, top, 0)
        check(_lib.load().mb_op_token_logprobs(args, stream))
    return TokenLogprobs(logprob, entropy, lse, best.view(rows, top), index.view(torch.int32).view(rows, top))


def token_logprobs_backward(logits, tokens, lse, entropy, dlogprob=None, dentropy=None, *, status=None):
    """dlogits of sum(dlogprob * logprob + dentropy * entropy), in the type of
    the logits, from the forward's ``lse`` and ``entropy``; dlogprob or
    dentropy None: zeros."""
    torch = _torch()
    at, stride, rows, vocab, code, device = _logit_rows(logits)
    _sizes(vocab)
    at_tokens = _int32(tokens, "tokens", (rows,), device)
    given = []
    for t, name in ((lse, "lse"), (entropy, "entropy"), (dlogprob, "dlogprob"), (dentropy, "dentropy")):
        if t is None:
            given.append(0)
        elif t.dtype is torch.float32 and t.shape == (rows,) and t.get_device() == device and t.is_contiguous():
            given.append(t.data_ptr())
        else:
            raise ValueError(f"{name} must be a contiguous float32 tensor [rows] on the logits' device")
    word = _int32(status, "status", (1,), device)
    stream = _current(device)
    d = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
    if rows:
        args = _LOGPROBS_BACKWARD.pack(at, at_tokens, *given, d.data_ptr(), word, stride, rows, vocab, code)
        check(_lib.load().mb_op_token_logprobs_backward(args, stream))
    return d

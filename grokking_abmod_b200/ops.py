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
import math
from typing import NamedTuple

from . import _lib
from ._lib import KvCacheC, CacheRowsC, check


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


_DTYPES = {}  # torch dtype -> MB_F32, MB_BF16, MB_F16


def _dtype(dtype, name):
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16")
    return code


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


def _cache(cache):
    import torch
    k, v, ks, vs = cache
    if k.ndim != 4:
        raise ValueError("cache.k must be [pages][heads][page_tokens][width]")
    pages, heads, tokens, width = shape = k.shape
    for t, name in ((k, "cache.k"), (v, "cache.v")):
        if not (t.dtype is torch.int8 and t.is_cuda and t.is_contiguous() and t.shape == shape
                and t.get_device() == k.get_device()):
            raise ValueError(f"{name} must be a contiguous int8 CUDA tensor [pages][heads][page_tokens][width]")
    for t, name in ((ks, "cache.k_scale"), (vs, "cache.v_scale")):
        if t.shape != (pages, heads) or t.get_device() != k.get_device():
            raise ValueError(f"{name} must be [pages][heads] on the cache's device")
        _dev(t, name)
    return KvCacheC(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, tokens, width)


def _int32(t, name, shape, device):
    import torch
    if not (t.dtype is torch.int32 and t.get_device() == device and t.shape == shape and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor {list(shape)} on the operands' device")
    return t.data_ptr()


def _where(table, lengths, offsets, rows, device):
    import torch
    if not (table.ndim == 2 and table.dtype is torch.int32 and table.get_device() == device
            and (table.stride(1) == 1 or table.shape[1] == 1)):
        raise ValueError("table must be an int32 tensor [batch][pages] on the operands' device")
    batch, pages = table.shape
    stride = table.stride(0) if batch > 1 else pages
    return CacheRowsC(table.data_ptr(), _int32(lengths, "lengths", (batch,), device),
                      _int32(offsets, "offsets", (batch + 1,), device) if offsets is not None else None,
                      stride, rows, pages, batch)


def _rows3(t, name):
    if not (t.is_cuda and t.ndim == 3 and (t.stride(2) == 1 or t.shape[2] == 1)):
        raise ValueError(f"{name} must be a CUDA tensor [rows][heads][head_dim] with adjacent channels")
    if min(t.stride()) < 0:
        raise ValueError(f"{name} must not have negative strides")
    return t.data_ptr()


def _word(status, device):
    return _int32(status, "status", (1,), device) if status is not None else None


def _on(t):
    """The tensor's device as the current one, and its current stream."""
    import torch
    if t.get_device() != torch.cuda.current_device():
        raise ValueError("operands must be on the current CUDA device")
    return torch.cuda.current_stream().cuda_stream


def cache_write(cache: KvCache, k, v, table, lengths, offsets=None, *, max_new: int = None, status=None) -> None:
    """Quantises the new rows k, v [rows][heads][head_dim] into their pages.

    ``table`` [batch][pages] int32 names each sequence's pages in order,
    ``lengths`` [batch] int32 its tokens with the new ones; rows
    offsets[b] .. offsets[b+1] are sequence b's newest (``offsets`` None: row b
    is).  ``max_new``: at least the largest number of new rows of a sequence
    (default: 1 without offsets, else all rows)."""
    c = _cache(cache)
    rows, heads, head_dim = k.shape
    device = cache.k.get_device()
    if v.shape != k.shape or v.dtype != k.dtype or heads != c.heads or not (k.get_device() == v.get_device() == device):
        raise ValueError("k and v must have one shape and type, the cache's heads and its device")
    if max_new is None:
        max_new = rows if offsets is not None else 1
    w = _where(table, lengths, offsets, rows, device)
    check(_lib.load().mb_op_cache_write(
        ctypes.byref(c), ctypes.byref(w), head_dim, _rows3(k, "k"), k.stride(0), k.stride(1), _rows3(v, "v"),
        v.stride(0), v.stride(1), _dtype(k.dtype, "k"), max_new, _word(status, device), _on(k)))


def cache_read(cache: KvCache, table, lengths, tokens: int, *, first=None, head_dim: int = None, dtype=None,
               status=None):
    """(k, v) [batch][tokens][heads][head_dim]: positions first[b] ..
    first[b] + tokens - 1 (``first`` None: from 0) of each sequence, zeros
    past its length.  ``head_dim`` defaults to the cache's width, ``dtype`` to
    float32."""
    import torch
    c = _cache(cache)
    device = cache.k.get_device()
    head_dim = c.width if head_dim is None else head_dim
    dtype = torch.float32 if dtype is None else dtype
    code = _dtype(dtype, "dtype")
    if tokens < 0 or head_dim < 1:
        raise ValueError("tokens must not be negative, head_dim must be positive")
    w = _where(table, lengths, None, table.shape[0], device)
    at = _int32(first, "first", lengths.shape, device) if first is not None else None
    stream = _on(cache.k)
    shape = (table.shape[0], tokens, c.heads, head_dim)
    k = torch.empty(shape, dtype=dtype, device=cache.k.device)
    v = torch.empty(shape, dtype=dtype, device=cache.k.device)
    check(_lib.load().mb_op_cache_read(ctypes.byref(c), ctypes.byref(w), head_dim, at, tokens, k.data_ptr(),
                                       v.data_ptr(), code, _word(status, device), stream))
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
    import torch
    c = _cache(cache)
    rows, heads, head_dim = q.shape
    device = cache.k.get_device()
    if q.get_device() != device:
        raise ValueError("q must be on the cache's device")
    at_q, code = _rows3(q, "q"), _dtype(q.dtype, "q")
    if max_new is None:
        max_new = rows if offsets is not None else 1
    if max_tokens is None:
        max_tokens = table.shape[1] * c.page_tokens
    w = _where(table, lengths, offsets, rows, device)
    at = _int32(first, "first", lengths.shape, device) if first is not None else None
    stream = _on(q)
    lib = _lib.load()
    out = torch.empty((rows, heads, head_dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((heads, rows), dtype=torch.float32, device=q.device)
    size = ctypes.c_size_t()
    check(lib.mb_op_cache_attention_workspace(w.batch, rows, heads, c.heads, head_dim, max_new, max_tokens,
                                              ctypes.byref(size)))
    work = torch.empty(size.value, dtype=torch.uint8, device=q.device) if size.value else None
    check(lib.mb_op_cache_attention(
        ctypes.byref(c), ctypes.byref(w), at, at_q, q.stride(0), q.stride(1), heads, head_dim, code,
        1.0 / math.sqrt(head_dim) if scale is None else scale, max_new, max_tokens, out.data_ptr(), lse.data_ptr(),
        work.data_ptr() if work is not None else None, size.value, _word(status, device), stream))
    return out, lse


def _logit_rows(logits):
    if not (logits.is_cuda and logits.ndim == 2 and (logits.stride(1) == 1 or logits.shape[1] == 1)):
        raise ValueError("logits must be a CUDA tensor [rows][vocab] with adjacent columns")
    rows, vocab = logits.shape
    return rows, vocab, logits.stride(0) if rows > 1 else vocab


def token_logprobs(logits, tokens, top: int = 0, *, status=None) -> TokenLogprobs:
    """Log-probabilities of the given ``tokens`` [rows] (int32; -1, the bits
    of IGNORE_TARGET, gives 0), entropies, and the ``top`` (0..32) most likely
    tokens of each row of ``logits`` [rows][vocab], ties to the lowest index.
    -inf masks a token; a row of masked tokens gives -inf and entropy 0."""
    import torch
    rows, vocab, stride = _logit_rows(logits)
    code, device = _dtype(logits.dtype, "logits"), logits.get_device()
    at_t = _int32(tokens, "tokens", (rows,), device)
    stream = _on(logits)
    dev = logits.device
    stats = torch.empty((3, rows), dtype=torch.float32, device=dev)
    top_lp = torch.empty((rows, top), dtype=torch.float32, device=dev)
    top_ix = torch.empty((rows, top), dtype=torch.int32, device=dev)
    at = stats.data_ptr()
    if rows:
        check(_lib.load().mb_op_token_logprobs(
            logits.data_ptr(), code, stride, rows, vocab, at_t, top, at, at + 4 * rows, at + 8 * rows,
            top_lp.data_ptr(), top_ix.data_ptr(), _word(status, device), stream))
    return TokenLogprobs(stats[0], stats[1], stats[2], top_lp, top_ix)


def token_logprobs_backward(logits, tokens, lse, entropy, dlogprob=None, dentropy=None, *, status=None):
    """dlogits of sum(dlogprob * logprob + dentropy * entropy), in the type of
    the logits, from the forward's ``lse`` and ``entropy``; dlogprob or
    dentropy None: zeros."""
    import torch
    rows, vocab, stride = _logit_rows(logits)
    code, device = _dtype(logits.dtype, "logits"), logits.get_device()
    at_t = _int32(tokens, "tokens", (rows,), device)
    at = []
    for t, name in ((lse, "lse"), (entropy, "entropy"), (dlogprob, "dlogprob"), (dentropy, "dentropy")):
        if t is None:
            at.append(None)
            continue
        if t.shape != (rows,) or t.get_device() != device:
            raise ValueError(f"{name} must be [rows] on the logits' device")
        at.append(_dev(t, name))
    stream = _on(logits)
    d = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
    if rows:
        check(_lib.load().mb_op_token_logprobs_backward(logits.data_ptr(), code, stride, rows, vocab, at_t, *at,
                                                        d.data_ptr(), _word(status, device), stream))
    return d

"""The operators of a decoder pass around its projections: rotary positions
and head norms (``rope``, ``qk_norm_rope``; the reference's attention_prepare,
attention.metal:15), low-rank adapters beside a projection (``lora``,
``linear_lora``), attention over a paged key/value cache and what a server does
with its pages (``attention``, ``cache_write``, ``cache_assign``,
``cache_compact``; the reference's attention_scan and attention_reduce,
attention.metal:104-216, over its sparse pages, device.cpp:147-198) and
penalties, biases and grammar masks on logits (``process_logits``).

All work is done by libq4k.so through its C ABI.  Tensors are torch tensors on
one GPU; every call launches on ``stream`` (default: the current stream of that
GPU) and returns without waiting.  What describes a batch on the device
(positions, adapter ids, page tables, texts, biases, masks) is read when the call runs, so
a captured call follows it from replay to replay.
"""
import ctypes
import struct

import torch

from ._lib import DTYPE_F16, DTYPE_F32, POST_ADD, POST_GATE, POST_STORE, check, lib

ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}

_DTYPES = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16}
# The C ABI's parameter structures (include/q4k.h), packed: cheaper per call
# than ctypes structures or twenty scalar arguments.
_HEADS = struct.Struct("=3Q4qI4x").pack
_ROTATION = struct.Struct("=2Q2If4x").pack
_ADAPTERS = struct.Struct("=5Q2I").pack
_LOGITS = struct.Struct("=12Q5I4x").pack
_CACHE = struct.Struct("=2Q3q2Q6I").pack
_ATTENTION = struct.Struct("=2fQI4x").pack
_POOL = struct.Struct("=Q4I").pack
_COUNTS = [struct.Struct(f"={n}I").pack for n in range(65)]

try:
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:
    def _raw_stream(device):
        return torch.cuda.current_stream(device).cuda_stream


def _stream_of(stream):
    return stream.cuda_stream if isinstance(stream, torch.cuda.Stream) else stream


_rope, _qk_norm_rope, _lora, _linear_lora, _process_logits = (lib.q4k_rope, lib.q4k_qk_norm_rope, lib.q4k_lora, lib.q4k_linear_lora,
                                                              lib.q4k_process_logits)
_attention, _cache_write, _cache_assign, _cache_compact = lib.q4k_attention, lib.q4k_cache_write, lib.q4k_cache_assign, lib.q4k_cache_compact


def _cut(*sizes):
    """The C ABI's sizes have 32 bits, to which ctypes would cut what it is given."""
    return ValueError(f"sizes must be 0 to 2^32 - 1, got {', '.join(map(str, sizes))}")


def _activations(t, what):
    """(dtype code, device index) of an activation tensor."""
    code = _DTYPES.get(t.dtype)
    device = t.get_device()
    if code is None:
        raise TypeError(f"{what} must be float32 or float16, got {t.dtype}")
    if device < 0:
        raise ValueError(f"{what} must be a GPU tensor")
    return code, device


def _address(t, dtype, numel, device, what):
    """The address of a contiguous tensor of ``dtype`` on ``device`` that holds
    at least ``numel`` elements (0 for None): the C ABI takes raw pointers, so
    what does not fit is refused here."""
    if t is None:
        return 0
    if t.dtype is dtype and t.get_device() == device and t.numel() >= numel and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{what} must be on cuda:{device}, is on {t.device}")
    if t.numel() < numel:
        raise ValueError(f"{what} holds {t.numel()} elements, needs {numel}")
    raise ValueError(f"{what} must be contiguous")


def rope_frequencies(rot_dim, base=10000.0, scaling="none", factor=1.0, original_context=0, beta_slow=1.0, beta_fast=32.0, device="cuda"):
    """(inv_freq, scale) for ``rope`` and ``qk_norm_rope``: the rot_dim / 2
    angles per position in 64 bits on ``device``, and the factor of the rotated
    values.  ``scaling``: "none"; "linear" (positions divided by ``factor``);
    "ntk" (base * factor^(rot_dim / (rot_dim - 2))); "yarn" (frequencies of
    fewer than ``beta_slow`` turns in ``original_context`` divided by
    ``factor``, those of more than ``beta_fast`` kept, a ramp between that is
    linear in the turns, as the method's paper writes it).  Models whose code
    ramps over the pair index instead differ in the middle pairs, by up to twice a
    frequency and more: pass theirs as ``inv_freq``, a float64 tensor of any
    frequencies."""
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"scaling must be one of {', '.join(ROPE_SCALINGS)}, got {scaling!r}")
    if (rot_dim | original_context) >> 32:
        raise _cut(rot_dim, original_context)
    values = (ctypes.c_double * min(max(1, rot_dim // 2), 1 << 16))()
    scale = ctypes.c_float()
    check(lib.q4k_rope_frequencies(rot_dim, float(base), ROPE_SCALINGS[scaling], float(factor), original_context, float(beta_slow),
                                   float(beta_fast), values, ctypes.byref(scale)))
    return torch.tensor(list(values), dtype=torch.float64).to(device), scale.value


def _heads(t, out, weight, what):
    """A q4k_heads of ``t`` and ``out`` [rows, heads, head_dim]."""
    shape = t.shape
    if len(shape) != 3 or out.shape != shape:
        raise ValueError(f"{what} and its output must be [rows, heads, head_dim] alike, got {tuple(shape)} and {tuple(out.shape)}")
    if out.dtype is not t.dtype:
        raise TypeError(f"{what} and its output must share a dtype")
    if out.get_device() != t.get_device():
        raise ValueError(f"{what} and its output must be on one GPU")
    ir, ih, ie = t.stride()
    orow, oh, oe = out.stride()
    if (ie != 1 or oe != 1) and shape[2] > 1:
        raise ValueError(f"the elements of a head of {what} and its output must be contiguous")
    return _HEADS(t.data_ptr(), out.data_ptr(), weight, ir, ih, orow, oh, shape[1])


def _rotation(inv_freq, positions, rows, device, interleaved, scale):
    n = inv_freq.numel()
    return _ROTATION(_address(inv_freq, torch.float64, n, device, "inv_freq"), _address(positions, torch.int32, rows, device, "positions"),
                     2 * n, 1 if interleaved else 0, scale)


def rope(x, inv_freq, positions, y, interleaved=False, scale=1.0, stream=None):
    """Rotary positions: pair i of every head of row r of ``x`` [rows, heads,
    head_dim] turned by positions[r] * inv_freq[i] (and scaled) into ``y``,
    elements behind the pairs copied.  Pairs are (i, i + n) of the n
    frequencies, or (2i, 2i + 1) with ``interleaved``.  ``x`` and ``y`` may be
    strided over rows and heads (parts of a joined projection's output); ``y``
    may be ``x``.  ``positions``: int32, ``inv_freq``: float64
    (rope_frequencies)."""
    code, device = _activations(x, "x")
    heads = _heads(x, y, 0, "x")
    rows, _, dim = x.shape
    if (rows | dim) >> 32:
        raise _cut(rows, dim)
    rc = _rope(_raw_stream(device) if stream is None else _stream_of(stream), device, heads,
               _rotation(inv_freq, positions, rows, device, interleaved, scale), rows, dim, code)
    if rc:
        check(rc)
    return y


def qk_norm_rope(q, k, q_weight, k_weight, inv_freq, positions, q_out, k_out, interleaved=False, scale=1.0, eps=1e-6, stream=None):
    """RMS norm of every head of ``q`` [rows, heads, head_dim] and ``k`` [rows,
    kv heads, head_dim] with the float32 weights [head_dim], then rope's
    rotation, into ``q_out`` and ``k_out`` (which may be ``q`` and ``k``).  An
    empty ``inv_freq`` norms only."""
    code, device = _activations(q, "q")
    rows, _, dim = q.shape
    if (rows | dim) >> 32:
        raise _cut(rows, dim)
    if k.dtype is not q.dtype or k.get_device() != device or k.shape[0] != rows or k.shape[-1] != dim:
        raise ValueError("q and k must share dtype, GPU, rows and head_dim")
    heads = _heads(q, q_out, _address(q_weight, torch.float32, dim, device, "q_weight"), "q")
    kv_heads = _heads(k, k_out, _address(k_weight, torch.float32, dim, device, "k_weight"), "k")
    rc = _qk_norm_rope(_raw_stream(device) if stream is None else _stream_of(stream), device, heads, kv_heads,
                       _rotation(inv_freq, positions, rows, device, interleaved, scale), rows, dim, eps, code)
    if rc:
        check(rc)
    return q_out, k_out


def _adapters(a, b, ids, ranks, scales, sequences, k, n, device):
    """A q4k_adapters of stacks a [slots, rank, k] and b [slots, n, rank]."""
    slots, rank, ak = a.shape
    if ak != k or b.shape != (slots, n, rank):
        raise ValueError(f"adapters must be a [slots, rank, {k}] and b [slots, {n}, rank], got {tuple(a.shape)} and {tuple(b.shape)}")
    return _ADAPTERS(_address(a, torch.float16, 0, device, "a"), _address(b, torch.float16, 0, device, "b"),
                     _address(ids, torch.int32, sequences, device, "adapter_ids"), _address(ranks, torch.int32, slots, device, "ranks"),
                     _address(scales, torch.float32, slots, device, "scales"), slots, rank)


def _counts(query_counts, count):
    if query_counts is None:
        return _COUNTS[1](count), 1
    n = len(query_counts)
    return (_COUNTS[n] if n < len(_COUNTS) else struct.Struct(f"={n}I").pack)(*query_counts), n


def lora(x, a, b, adapter_ids, count, output, auxiliary=None, query_counts=None, ranks=None, scales=None, stream=None):
    """output[count, n] = auxiliary + scale * (x[count, k] A^T) B^T, with the
    adapter adapter_ids[q] (int32; outside [0, slots): none) of each sequence q
    of ``query_counts`` (default: one sequence).  ``a`` [slots, rank, k] and
    ``b`` [slots, n, rank] are the float16 stacks, ``ranks`` (int32) the ranks in
    use (default: all) and ``scales`` (float32; default 1) of the slots.
    ``auxiliary`` may be ``output``; without it the sum starts at zero."""
    code, device = _activations(x, "x")
    if a.dim() != 3 or b.dim() != 3:
        raise ValueError("adapters must be a [slots, rank, k] and b [slots, n, rank]")
    k, n = a.shape[2], b.shape[1]
    if (count | k | n) >> 32:
        raise _cut(count, k, n)
    counts, sequences = _counts(query_counts, count)
    ad = _adapters(a, b, adapter_ids, ranks, scales, sequences, k, n, device)
    dtype = x.dtype
    rc = _lora(_raw_stream(device) if stream is None else _stream_of(stream), device, ad, _address(x, dtype, count * k, device, "x"),
               _address(output, dtype, count * n, device, "output"), _address(auxiliary, dtype, count * n, device, "auxiliary"), count, k, n,
               counts, sequences, code)
    if rc:
        check(rc)
    return output


def linear_lora(x, w, a, b, adapter_ids, count, output, auxiliary=None, gated=False, query_counts=None, ranks=None, scales=None, stream=None):
    """linear(x, w, ...) with the sequences' adapters added to the projection
    before its epilogue (arguments as linear's and lora's, but ``auxiliary`` is a
    tensor: the fused gate/up pair takes no adapters).  In float16 the adapters'
    part is rounded before the projection is added, and the sum before the gate."""
    if auxiliary is not None and not isinstance(auxiliary, torch.Tensor):
        raise TypeError(f"auxiliary must be a tensor, got {type(auxiliary).__name__}: the fused gate/up pair takes no adapters")
    code, device = _activations(x, "x")
    if a.dim() != 3 or b.dim() != 3:
        raise ValueError("adapters must be a [slots, rank, k] and b [slots, n, rank]")
    if device != w.device:
        raise ValueError(f"x is on cuda:{device}, the weights on cuda:{w.device}")
    if count >> 32:
        raise _cut(count)
    counts, sequences = _counts(query_counts, count)
    ad = _adapters(a, b, adapter_ids, ranks, scales, sequences, w.k, w.n, device)
    post = POST_GATE if gated else POST_ADD if auxiliary is not None else POST_STORE
    dtype = x.dtype
    rc = _linear_lora(_raw_stream(device) if stream is None else _stream_of(stream), w.handle, ad, _address(x, dtype, count * w.k, device, "x"),
                      _address(output, dtype, count * w.n, device, "output"), _address(auxiliary, dtype, count * w.n, device, "auxiliary"),
                      count, counts, sequences, post, code)
    if rc:
        check(rc)
    return output


def _sequences(query_counts, rows):
    """(packed counts, sequences, rows that they cover) of up to ``rows`` rows."""
    if query_counts is None:
        return _COUNTS[1](rows), 1, rows
    n = len(query_counts)
    covered = sum(query_counts)
    if covered > rows:
        raise ValueError(f"query_counts cover {covered} rows, there are {rows}")
    return (_COUNTS[n] if n < len(_COUNTS) else struct.Struct(f"={n}I").pack)(*query_counts), n, covered


def _cache(k_cache, v_cache, shape, tables, slots, positions, sequences, device):
    """A q4k_cache of caches of ``shape``, and the address of the positions."""
    pages, heads, size, dim = shape
    strides = k_cache.stride()
    if k_cache.dtype is not torch.float16 or v_cache.dtype is not torch.float16:
        raise TypeError(f"k_cache and v_cache must be float16, got {k_cache.dtype} and {v_cache.dtype}")
    if k_cache.get_device() != device or v_cache.get_device() != device:
        raise ValueError(f"k_cache and v_cache must be on cuda:{device}")
    if strides != v_cache.stride() or (strides[3] != 1 and dim > 1):
        raise ValueError("k_cache and v_cache must have the same strides and contiguous tokens")
    table = tables.shape
    if len(table) != 2:
        raise ValueError("tables must be [table rows, width]")
    rows, width = table
    if (pages | heads | size | dim | rows | width) >> 32:
        raise _cut(pages, heads, size, dim, rows, width)
    return (_CACHE(k_cache.data_ptr(), v_cache.data_ptr(), strides[0], strides[1], strides[2], _address(tables, torch.int32, 0, device, "tables"),
                   _address(slots, torch.int32, sequences, device, "slots"), pages, size, heads, dim, rows, width),
            _address(positions, torch.int32, sequences, device, "positions"))


def _cache_shape(k_cache, v_cache):
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"k_cache and v_cache must be [pages, heads, page_size, head_dim] alike, got {tuple(shape)} and {tuple(v_cache.shape)}")
    return shape


def _rows_of(t, heads, what):
    """A q4k_heads of ``t``, read only."""
    row, head, element = t.stride()
    if element != 1 and t.shape[2] > 1:
        raise ValueError(f"the elements of a head of {what} must be contiguous")
    return _HEADS(t.data_ptr(), 0, 0, row, head, 0, 0, heads)


def cache_write(k, v, k_cache, v_cache, tables, positions, query_counts=None, slots=None, stream=None):
    """Keys and values of new tokens into their pages: row t of sequence q of
    ``k`` and ``v`` [rows, heads, head_dim] (float32 or float16, any row and head
    strides; ``query_counts`` as linear's, up to 64 sequences, default one) goes to
    position positions[q] + t, rounded to float16.  ``k_cache`` and ``v_cache`` are
    [pages, heads, page_size, head_dim], views of any page, head and token strides
    (multiples of 8; page_size a power of two from 16, head_dim a multiple of 8 up to 256).
    ``tables`` (int32 [table rows, width]) lists the pages of a sequence's tokens 0,
    1, ... in row ``slots``[q] (int32, default: q); numbers outside the cache are
    pages that are not there.  Rows behind the last sequence, and rows whose place
    is not there, are not written."""
    code, device = _activations(k, "k")
    shape, of = k.shape, _cache_shape(k_cache, v_cache)
    if len(shape) != 3 or v.shape != shape or shape[1] != of[1] or shape[2] != of[3]:
        raise ValueError(f"k and v must be [rows, heads, head_dim] of the cache's heads, got {tuple(shape)} and {tuple(v.shape)} for a cache of "
                         f"{tuple(of)}")
    if v.dtype is not k.dtype or v.get_device() != device:
        raise ValueError("k and v must share dtype and GPU")
    counts, sequences, rows = _sequences(query_counts, shape[0])
    if rows >> 32:
        raise _cut(rows)
    cache, at = _cache(k_cache, v_cache, of, tables, slots, positions, sequences, device)
    heads = of[1]
    rc = _cache_write(_raw_stream(device) if stream is None else _stream_of(stream), device, cache, _rows_of(k, heads, "k"), _rows_of(v, heads, "v"),
                      at, counts, sequences, rows, code)
    if rc:
        check(rc)
    return k_cache, v_cache


def attention(q, k_cache, v_cache, tables, positions, out, query_counts=None, slots=None, scale=None, softcap=0.0, window=0, slopes=None,
              stream=None):
    """Causal attention of new tokens over their sequences' pages (cache_write's,
    the new tokens' own keys and values among them): row t of sequence q of ``q``
    [rows, heads, head_dim] stands at positions[q] + t and sees the keys up to
    there, head h those of cache head h // (heads / cache heads).  Scores are
    ``scale`` (default 1 / sqrt(head_dim)) times the products; ``softcap`` (2^-64
    to 2^64; 0: none) bounds them (softcap * tanh(score / softcap)); ``window``,
    above 0, is the number of keys that a row sees, its own the last; ``slopes`` (float32 [heads])
    times the (negative) distance to the key is added.  ``out`` is like ``q``, of
    any row and head strides, and must not overlap it.  A row that sees no key
    becomes zero (one whose scores are all -inf NaN); rows behind the last sequence
    are left as they were."""
    code, device = _activations(q, "q")
    heads = _heads(q, out, 0, "q")
    shape, of = q.shape, _cache_shape(k_cache, v_cache)
    if shape[2] != of[3]:
        raise ValueError(f"q must have the cache's head_dim, got {tuple(shape)} for a cache of {tuple(of)}")
    counts, sequences, rows = _sequences(query_counts, shape[0])
    if rows >> 32 or window >> 32:
        raise _cut(rows, window)
    cache, at = _cache(k_cache, v_cache, of, tables, slots, positions, sequences, device)
    params = _ATTENTION(shape[2] ** -0.5 if scale is None else scale, softcap, _address(slopes, torch.float32, shape[1], device, "slopes"), window)
    rc = _attention(_raw_stream(device) if stream is None else _stream_of(stream), device, heads, cache, params, at, counts, sequences, rows, code)
    if rc:
        check(rc)
    return out


def _pool(pool, tables, lengths, new_tables):
    """(q4k_pool, device, slots, width) of a pool [pages, ..., page_size, token]."""
    device = pool.get_device()
    if device < 0:
        raise ValueError("pool must be a GPU tensor")
    if pool.dim() < 3 or not pool.is_contiguous():
        raise ValueError("pool must be contiguous, [pages, ..., page_size, elements of a token]")
    pages, size = pool.shape[0], pool.shape[-2]
    token = pool.shape[-1] * pool.element_size()
    blocks = pool.numel() // max(1, pages * size * pool.shape[-1])
    if tables.dim() != 2 or new_tables.shape != tables.shape:
        raise ValueError(f"tables and new_tables must be [slots, width] alike, got {tuple(tables.shape)} and {tuple(new_tables.shape)}")
    slots, width = tables.shape
    if (pages | blocks | size | token | slots | width) >> 32:
        raise _cut(pages, blocks, size, token, slots, width)
    i32 = torch.int32
    return (_POOL(pool.data_ptr(), pages, blocks, size, token), device, slots, width, _address(tables, i32, 0, device, "tables"),
            _address(lengths, i32, slots, device, "lengths"), _address(new_tables, i32, 0, device, "new_tables"))


def cache_assign(pool, tables, lengths, parents, new_tables, new_lengths, counts=None, missing=None, stream=None):
    """The slots take over the states of their parents, all at once: slot s holds
    the ``lengths``[p] tokens of p = ``parents``[s] (outside the slots: none, it is
    free; None: p = s) and has pages for ``counts``[s] more (default: none).  Forks,
    beams in a new order, sequences that end and pages for the next tokens are all
    this call.

    ``pool`` [pages, ..., page_size, elements of a token] holds the pages, of all
    layers, keys and values, say; its parts are what cache_write and attention take
    (pool[:, layer, 0] of a pool [pages, layers, 2, heads, page_size, head_dim]).
    Full pages are shared.  A last page that is not full stays with the lowest slot
    that holds it, the others get a page with a copy of its tokens.  New pages are
    the lowest that no slot's new tokens lie in, in the order of the slots; entries
    of ``new_tables`` [slots, width] without a page are -1, and ``missing`` (int32
    [1]) becomes the number of pages asked for and not given.  A page counts as held
    where it lies below a slot's length: add the tokens that were written to the
    lengths before the next call.  Whole numbers are int32; tables and lengths are
    read, the new ones must not overlap them."""
    p, device, slots, width, old, held, new = _pool(pool, tables, lengths, new_tables)
    i32 = torch.int32
    rc = _cache_assign(_raw_stream(device) if stream is None else _stream_of(stream), device, p, old, held, slots, width,
                       _address(parents, i32, slots, device, "parents"), _address(counts, i32, slots, device, "counts"), new,
                       _address(new_lengths, i32, slots, device, "new_lengths"), _address(missing, i32, 1, device, "missing"))
    if rc:
        check(rc)
    return new_tables, new_lengths


def cache_compact(pool, tables, lengths, new_tables, used=None, stream=None):
    """Moves the n pages that slots hold tokens in to the front of ``pool``: the
    i-th held one, by number, behind page n - 1 to the i-th free one before page n.
    ``new_tables`` lists them (entries behind a slot's length are -1), ``used`` (int32
    [1]) becomes n.  Arguments as cache_assign's."""
    p, device, slots, width, old, held, new = _pool(pool, tables, lengths, new_tables)
    rc = _cache_compact(_raw_stream(device) if stream is None else _stream_of(stream), device, p, old, held, slots, width, new,
                        _address(used, torch.int32, 1, device, "used"))
    if rc:
        check(rc)
    return new_tables


def process_logits(logits, out, tokens=None, slots=None, lengths=None, prompts=None, repetition=None, frequency=None, presence=None,
                   bias_offsets=None, bias_tokens=None, bias_values=None, mask=None, mask_rows=None, stream=None):
    """``logits`` [rows, vocab] into ``out`` (which may be ``logits``), row r

    * with the tokens of its text divided (positive logits) or multiplied by
      ``repetition``[r], and the generated ones lowered by ``frequency``[r] per
      occurrence and ``presence``[r].  The text is the first ``lengths``[r]
      tokens of row ``slots``[r] (default: r) of ``tokens`` (int32 [slots,
      capacity], the request token buffer of embedding_batch); its first
      ``prompts``[r] tokens (default: none) were given, not generated;
    * with entries bias_offsets[r] .. bias_offsets[r + 1] - 1 of ``bias_tokens``
      (int32) and ``bias_values`` (float32) added, of a token's entries the last;
    * with -inf for the tokens that bit mask ``mask_rows``[r] (int32, default: r,
      negative: none) of ``mask`` (int32 [masks, words], bit v % 32 of word
      v / 32 allows token v) forbids.

    Arguments left out leave their step out."""
    code, device = _activations(logits, "logits")
    if logits.dim() != 2 or out.shape != logits.shape or out.dtype is not logits.dtype or out.get_device() != device:
        raise ValueError("logits and out must be [rows, vocab] of one dtype on one GPU")
    rows, vocab = logits.shape
    if (rows | vocab) >> 32:
        raise _cut(rows, vocab)
    in_stride, ie = logits.stride()
    out_stride, oe = out.stride()
    if vocab > 1 and (ie != 1 or oe != 1):
        raise ValueError("the rows of logits and out must be contiguous")
    if rows == 0:
        return out
    nslots = capacity = nbias = nmasks = words = 0
    i32, f32 = torch.int32, torch.float32
    if tokens is not None:
        if tokens.dim() != 2:
            raise ValueError("tokens must be [slots, capacity]")
        nslots, capacity = tokens.shape
        if nslots < rows and slots is None:
            raise ValueError(f"without slots every row needs a text ({rows} rows, {nslots} texts)")
        if tokens.numel() == 0:  # a buffer of no tokens: every text is empty
            tokens = slots = lengths = prompts = repetition = frequency = presence = None
    if bias_tokens is not None and bias_values is not None:
        nbias = bias_tokens.numel()
        if nbias == 0 and bias_values.numel() == 0:  # no row has a bias
            bias_offsets = bias_tokens = bias_values = None
    if mask is not None:
        if mask.dim() != 2:
            raise ValueError("mask must be [masks, words]")
        nmasks, words = mask.shape
        if words < (vocab + 31) // 32 or (nmasks < rows and mask_rows is None):
            raise ValueError(f"a mask of {vocab} tokens needs {(vocab + 31) // 32} words a row, and without mask_rows every row a mask "
                             f"(got {nmasks} masks of {words} for {rows} rows)")
        if nmasks == 0:  # no mask to take
            mask = mask_rows = None
    text = bias = (0, 0, 0)
    given = (0, 0, 0, 0)
    if tokens is not None or slots is not None or lengths is not None or prompts is not None:
        given = (_address(tokens, i32, 0, device, "tokens"), _address(slots, i32, rows, device, "slots"),
                 _address(lengths, i32, rows, device, "lengths"), _address(prompts, i32, rows, device, "prompts"))
    if repetition is not None or frequency is not None or presence is not None:
        text = (_address(repetition, f32, rows, device, "repetition"), _address(frequency, f32, rows, device, "frequency"),
                _address(presence, f32, rows, device, "presence"))
    if bias_offsets is not None or bias_tokens is not None or bias_values is not None:
        bias = (_address(bias_offsets, i32, rows + 1, device, "bias_offsets"), _address(bias_tokens, i32, nbias, device, "bias_tokens"),
                _address(bias_values, f32, nbias, device, "bias_values"))
    params = _LOGITS(*given, *text, *bias, _address(mask, i32, 0, device, "mask"), _address(mask_rows, i32, rows, device, "mask_rows"), nslots,
                     capacity, nbias, nmasks, words)
    rc = _process_logits(_raw_stream(device) if stream is None else _stream_of(stream), device, logits.data_ptr(), out.data_ptr(), rows, vocab,
                         in_stride, out_stride, params, code)
    if rc:
        check(rc)
    return out


__all__ = ["rope", "qk_norm_rope", "rope_frequencies", "lora", "linear_lora", "attention", "cache_write", "cache_assign", "cache_compact",
           "process_logits", "ROPE_SCALINGS"]

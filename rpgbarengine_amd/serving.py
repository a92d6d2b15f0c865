"""The serving operators of include/rpg_hip.h on torch tensors: one paged
key-value cache for many sequences, the attention that reads it and a sampler
of many rows, for hosts that schedule sessions themselves.

    cache = serving.PagedCache.zeros(n_pages, 16, n_kv, 128, torch.bfloat16)
    serving.append(cache, table, lens, starts, k, v, q=q, q_norm=..., k_norm=..., rope=...)
    out = serving.prompt_attention(q, cache, table, lens, starts)   # prompts, packed
    out = serving.decode_attention(q, cache, table, lens)           # one token each
    out = serving.shared_attention(q, cache, table, lens, groups, shared)  # with prefixes in common
    logits = serving.edit_logits(logits, history, history_lens, repetition=..., mask=...)
    tokens, logprobs = serving.sample(logits, u, temperature, top_k, top_p, min_p)

A QuantCache in the cache's place holds its rows in 8 bits.

`table` is int32 [sequences, pages]: position p of a sequence lies in page
table[s, p // page_size]; `lens` int32 [sequences] counts a sequence's
positions, the new tokens among them; `starts` int32 [sequences + 1] are the
packed rows at which each sequence's new tokens start (and the last ones end).

The work is enqueued on the current torch stream of the tensors' GPU; work
memory comes from torch's allocator on that stream. Lengths, pages, starts and
sampling parameters are read on the GPU, so a call captured into a graph takes
the values of each replay. There is no backward pass and no forward-mode one:
tensors that require gradients are refused while gradients are recorded, and
those that carry a tangent always.
"""

from __future__ import annotations

import ctypes
import functools
import struct

import torch
from torch.autograd import forward_ad

from . import EngineError, lib

_P, _I32, _I64, _F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}  # ggml ids
# rpg_hip_paged_cache, rpg_hip_sequences, rpg_hip_rows, packed as C lays them out
_CACHE, _SEQS, _ROWS = struct.Struct("PPqqqiiiii"), struct.Struct("PqPPiii"), struct.Struct("Pqq")
# rpg_hip_quant_cache, rpg_hip_edits, rpg_hip_groups
_QUANT, _EDITS, _GROUPS = struct.Struct("PPPPqqqqqiiiii"), struct.Struct("PqPPPPPPqPqPqPiii"), struct.Struct("PPi")
_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}

_SIGS = {
    "rpg_hip_paged_append": ([_P, _P, _P, _P, _P, _P, _I32, _P, _P, _F, _P, _I64, _P], _I32),
    "rpg_hip_paged_decode": ([_P, _P, _P, _P, _I32, _F, _P, _I64, _P], _I32),
    "rpg_hip_paged_prompt": ([_P, _P, _P, _P, _I32, _F, _P, _I64, _P], _I32),
    "rpg_hip_paged_work": ([_P, _P, _I32, _I32], _I64),
    "rpg_hip_quant_append": ([_P, _P, _I32, _P, _P, _P, _P, _I32, _P, _P, _F, _P, _I64, _P], _I32),
    "rpg_hip_quant_read": ([_P, _P, _I32, _P, _P, _P], _I32),
    "rpg_hip_quant_decode": ([_P, _P, _I32, _P, _P, _I32, _F, _P, _I64, _P], _I32),
    "rpg_hip_quant_prompt": ([_P, _P, _I32, _P, _P, _I32, _F, _P, _I64, _P], _I32),
    "rpg_hip_quant_work": ([_P, _P, _I32, _I32, _I32], _I64),
    "rpg_hip_paged_shared": ([_P, _P, _P, _P, _P, _I32, _F, _P, _I64, _P], _I32),
    "rpg_hip_paged_shared_work": ([_P, _P, _I32, _I32], _I64),
    "rpg_hip_quant_shared": ([_P, _P, _P, _I32, _P, _P, _I32, _F, _P, _I64, _P], _I32),
    "rpg_hip_quant_shared_work": ([_P, _P, _I32, _I32, _I32], _I64),
    "rpg_hip_edit_logits": ([_I32, _P, _I64, _I64, _I64, _P, _P, _I64, _P], _I32),
    "rpg_hip_sample_rows": ([_I32, _P, _I64, _I64, _I64, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _P], _I32),
    "rpg_hip_sample_rows_work": ([_I64, _I64], _I64),
}
_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = lib()
        for name, (args, res) in _SIGS.items():
            f = getattr(L, name)
            f.argtypes, f.restype = args, res
        _bound = L
    return _bound


def _ok(rc):
    if rc < 0:
        raise EngineError(_lib().rpg_hip_last_error().decode())
    return rc


def _need(cond, what):
    if not cond:
        raise EngineError(what)


def _plain(x, name):
    """No derivative is asked of x. (Called where it may be: a call's seven tensors
    otherwise cost 0.5 us.)"""
    if x.requires_grad and torch.is_grad_enabled():
        raise EngineError(f"{name} requires gradients: there is no backward pass")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise EngineError(f"{name} carries a tangent: there are no forward-mode gradients")


class PagedCache:
    """A pool of key and value pages, [pages, key heads, page size, head dim] each
    (f32, f16 or bf16; views of a larger pool are fine). A larger pool is a new
    PagedCache; one whose tensors were given other memory since is refused."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _need(k.dim() == 4 and v.shape == k.shape, "k and v are [pages, key heads, page size, head dim]")
        _need(k.dtype in _TYPES and v.dtype == k.dtype, "k and v are both float32, float16 or bfloat16")
        _need(k.is_cuda and v.device == k.device, "k and v lie on one GPU")
        _plain(k, "the cache's k")
        _plain(v, "the cache's v")
        _need(k.stride(3) == 1 and k.stride() == v.stride(), "k and v have the same strides, 1 in the last dimension")
        self._k, self._v = k, v
        self.device, self.dtype = k.device, k.dtype
        n_pages, n_kv, page, dim = k.shape
        self.n_kv, self.head_dim, self.page_size = n_kv, dim, page
        strides = [s if n > 1 else page * dim * 16 for n, s in zip(k.shape, k.stride())]
        self._at = k.data_ptr(), v.data_ptr()
        self._c = _CACHE.pack(*self._at, *strides[:3], n_pages, page, n_kv, dim, _TYPES[k.dtype])

    k = property(lambda self: self._k, doc="the pool of keys")
    v = property(lambda self: self._v, doc="the pool of values")

    def _packed(self):
        if (self._k.data_ptr(), self._v.data_ptr()) != self._at:
            raise EngineError("the cache's tensors lie elsewhere than when it was made: make a new PagedCache")
        return self._c

    @classmethod
    def zeros(cls, n_pages: int, page_size: int, n_kv: int, head_dim: int, dtype=torch.float32,
              device="cuda") -> "PagedCache":
        shape = (n_pages, n_kv, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))


class QuantCache:
    """A pool of pages held in 8 bits: k and v [pages, key heads, page size, head dim]
    of codes (torch.int8 or torch.float8_e4m3fn) and k_scale and v_scale [pages, key
    heads, page size] float32; an element is its code times its row's scale. Views of
    larger pools are fine, rows at multiples of 16 bytes. What goes in and comes out is
    float32, float16 or bfloat16."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        _need(k.dim() == 4 and v.shape == k.shape, "k and v are [pages, key heads, page size, head dim]")
        _need(k.dtype in _CODES and v.dtype == k.dtype, "k and v are both int8 or float8_e4m3fn")
        _need(k_scale.shape == k.shape[:3] and v_scale.shape == k.shape[:3]
              and k_scale.dtype == torch.float32 and v_scale.dtype == torch.float32,
              "k_scale and v_scale are float32 [pages, key heads, page size]")
        _need(k.is_cuda and all(x.device == k.device for x in (v, k_scale, v_scale)),
              "k, v, k_scale and v_scale lie on one GPU")
        for x, name in ((k, "k"), (v, "v"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            _plain(x, "the cache's " + name)
        _need(k.stride(3) == 1 and k.stride() == v.stride(), "k and v have the same strides, 1 in the last dimension")
        _need(k_scale.stride(2) == 1 and k_scale.stride() == v_scale.stride(),
              "k_scale and v_scale have the same strides, 1 in the last dimension")
        self._held = k, v, k_scale, v_scale
        self.device, self.codes = k.device, k.dtype
        n_pages, n_kv, page, dim = k.shape
        self.n_kv, self.head_dim, self.page_size = n_kv, dim, page
        strides = [s if n > 1 else page * dim * 16 for n, s in zip(k.shape, k.stride())]
        scales = [s if n > 1 else page for n, s in zip(k_scale.shape, k_scale.stride())]
        self._at = [x.data_ptr() for x in self._held]
        self._c = _QUANT.pack(*self._at, *strides[:3], *scales[:2], n_pages, page, n_kv, dim, _CODES[k.dtype])

    k = property(lambda self: self._held[0], doc="the pool of the keys' codes")
    v = property(lambda self: self._held[1], doc="the pool of the values' codes")
    k_scale = property(lambda self: self._held[2], doc="the keys' scales")
    v_scale = property(lambda self: self._held[3], doc="the values' scales")

    def _packed(self):
        if [x.data_ptr() for x in self._held] != self._at:
            raise EngineError("the cache's tensors lie elsewhere than when it was made: make a new QuantCache")
        return self._c

    @classmethod
    def zeros(cls, n_pages: int, page_size: int, n_kv: int, head_dim: int, codes=torch.float8_e4m3fn,
              device="cuda") -> "QuantCache":
        shape = (n_pages, n_kv, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(codes) for _ in "kv")
        return cls(k, v, *(torch.zeros(shape[:3], device=device) for _ in "kv"))


def _ints(x, name, dims, device):
    shape = x.shape
    if x.dtype is not torch.int32 or len(shape) != dims or x.device != device or (shape[-1] > 1 and x.stride(-1) != 1):
        raise EngineError(f"{name} is int32, of {dims} dimension(s), contiguous in the last, on the cache's GPU")
    return shape


def _seqs(cache, table, lens, starts, n_tokens):
    dev = cache.device
    n, pages = _ints(table, "table", 2, dev)
    if _ints(lens, "lens", 1, dev)[0] != n:
        raise EngineError("lens and table are of one number of sequences")
    at = 0
    if starts is not None:
        if _ints(starts, "starts", 1, dev)[0] != n + 1:
            raise EngineError("starts has one value more than there are sequences")
        at = starts.data_ptr()
    return _SEQS.pack(table.data_ptr(), table.stride(0), lens.data_ptr(), at, pages, n, n_tokens), n, pages


def _rows(x, name, cache, dtype=None):
    """dtype: of the call's rows, where the cache is a QuantCache."""
    shape, strides = x.shape, x.stride()
    if (len(shape) != 3 or x.dtype is not (dtype or cache.dtype) or x.device != cache.device
            or shape[2] != cache.head_dim or strides[2] != 1):
        raise EngineError(f"{name} is [tokens, heads, head dim] of the cache's type and GPU, contiguous in the last dimension"
                          if dtype is None else
                          f"{name} is [tokens, heads, head dim] of {dtype} on the cache's GPU, contiguous in the last dimension")
    if x.requires_grad or forward_ad._current_level >= 0:
        _plain(x, name)
    n, heads, dim = shape
    return _ROWS.pack(x.data_ptr(), strides[0] if n > 1 else heads * dim, strides[1] if heads > 1 else dim)


def _vector(x, name, n, dtype, device):
    """The address of a contiguous vector; None stays None."""
    if x is None:
        return None
    if x.requires_grad or forward_ad._current_level >= 0:
        _plain(x, name)
    if x.dtype is not dtype or x.shape != (n,) or x.device != device or (n > 1 and x.stride(0) != 1):
        raise EngineError(f"{name} is {dtype} [{n}], contiguous, on the same GPU")
    return x.data_ptr()


def _enqueue(device, f, *args):
    """f(*args, stream) on the current stream of the tensors' GPU, that GPU current."""
    if _current() == device.index:
        rc = f(*args, _stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = f(*args, _stream(device.index))
    if rc < 0:
        _ok(rc)


def _row_type(x, name):
    """The type of a call's rows on a QuantCache."""
    if x.dtype not in _TYPES:
        raise EngineError(f"{name} is float32, float16 or bfloat16")
    return x.dtype


# What a call writes in place is a new version of the tensor to autograd: a
# backward pass that saved the old one refuses.
_written = torch.autograd.graph.increment_version


def _stream(index):
    return torch.cuda.current_stream(index).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):  # the same without a Stream object for each call
    _stream = torch._C._cuda_getCurrentRawStream
_current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def append(cache, table, lens, starts, k, v, q=None, q_out=None, q_norm=None, k_norm=None,
           eps: float = 1e-6, rope=None):
    """Stores the packed new tokens' keys and values, k and v [tokens, key heads,
    dim], in their pages; q [tokens, heads, dim] goes to q_out (made when not
    given; may be q). Keys and queries are RMS-normed per head with the gains
    k_norm and q_norm (float32 [dim]) and rotated by rope (float32 [positions,
    dim]: cos | sin) where those are given. A QuantCache holds each row as codes and
    a scale; k, v and q are of one type. Returns q_out."""
    quant = isinstance(cache, QuantCache)
    kind = _row_type(k, "k") if quant else None
    kr, vr = _rows(k, "k", cache, kind), _rows(v, "v", cache, kind)
    n = k.shape[0]
    seqs = _seqs(cache, table, lens, starts, n)[0]
    if v.shape != k.shape or k.shape[1] != cache.n_kv:
        raise EngineError("k and v are [tokens, key heads of the cache, head dim]")
    heads, qr, qo = 0, None, None
    if q is not None:
        qr = _rows(q, "q", cache, kind)
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if q.shape[0] != n or q_out.shape != q.shape:
            raise EngineError("q, q_out and k are of one number of tokens")
        qo = _rows(q_out, "q_out", cache, kind)
    dev, dim = cache.device, cache.head_dim
    rp, rope_rows = None, 0
    if rope is not None:
        if (rope.dtype is not torch.float32 or rope.dim() != 2 or rope.shape[1] != dim or not rope.is_contiguous()
                or rope.device != dev):
            raise EngineError("rope is float32 [positions, head dim], contiguous, on the same GPU")
        if rope.requires_grad or forward_ad._current_level >= 0:
            _plain(rope, "rope")
        rp, rope_rows = rope.data_ptr(), rope.shape[0]
    rest = (kr, vr, qr, qo, heads, _vector(q_norm, "q_norm", dim, torch.float32, dev),
            _vector(k_norm, "k_norm", dim, torch.float32, dev), eps, rp, rope_rows)
    if quant:
        _enqueue(dev, _lib().rpg_hip_quant_append, cache._packed(), seqs, _TYPES[kind], *rest)
        _written(cache._held if qo is None else (*cache._held, q_out))
    else:
        _enqueue(dev, _lib().rpg_hip_paged_append, cache._packed(), seqs, *rest)
        _written((cache._k, cache._v) if qo is None else (cache._k, cache._v, q_out))
    return q_out


def read_rows(cache: QuantCache, table, lens, starts, k_out, v_out):
    """The last positions of each sequence out of a QuantCache: those of sequence s
    go to rows starts[s] .. starts[s + 1] of k_out and v_out [tokens, key heads, dim],
    both of one type. Rows of no sequence are left as they are; positions whose pages
    the table does not name read as zeros. Returns (k_out, v_out)."""
    if not isinstance(cache, QuantCache):
        raise EngineError("cache is a QuantCache")
    kind = _row_type(k_out, "k_out")
    kr, vr = _rows(k_out, "k_out", cache, kind), _rows(v_out, "v_out", cache, kind)
    if v_out.shape != k_out.shape or k_out.shape[1] != cache.n_kv:
        raise EngineError("k_out and v_out are [tokens, key heads of the cache, head dim]")
    if starts is None:
        raise EngineError("starts is needed")
    seqs = _seqs(cache, table, lens, starts, k_out.shape[0])[0]
    _enqueue(cache.device, _lib().rpg_hip_quant_read, cache._packed(), seqs, _TYPES[kind], kr, vr)
    _written((k_out, v_out))
    return k_out, v_out


@functools.lru_cache(maxsize=4096)
def _work_bytes(n_kv, page_size, head_dim, kind, pages, n_seqs, n_tokens, heads, prompt):
    """rpg_hip_paged_work of these sizes."""
    wide = page_size * head_dim
    c = _CACHE.pack(0, 0, n_kv * wide, wide, head_dim, 1, page_size, n_kv, head_dim, kind)
    return _ok(_lib().rpg_hip_paged_work(c, _SEQS.pack(0, pages, 0, 0, pages, n_seqs, n_tokens), heads, prompt))


@functools.lru_cache(maxsize=4096)
def _quant_work_bytes(n_kv, page_size, head_dim, kind, pages, n_seqs, n_tokens, heads, prompt):
    """rpg_hip_quant_work of these sizes."""
    wide = page_size * head_dim
    c = _QUANT.pack(0, 0, 0, 0, n_kv * wide, wide, head_dim, n_kv * page_size, page_size, 1, page_size, n_kv, head_dim, 0)
    return _ok(_lib().rpg_hip_quant_work(c, _SEQS.pack(0, pages, 0, 0, pages, n_seqs, n_tokens), kind, heads, prompt))


def _attention(q, cache, table, lens, starts, scale, out, prompt):
    quant = isinstance(cache, QuantCache)
    kind = _row_type(q, "q") if quant else None
    qr = _rows(q, "q", cache, kind)
    n_tokens = q.shape[0] if prompt else 0
    seqs, n_seqs, pages = _seqs(cache, table, lens, starts, n_tokens)
    if not prompt and q.shape[0] != n_seqs:
        raise EngineError("q has a row for each sequence")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise EngineError("out has the shape of q")
    heads, dim = q.shape[1], cache.head_dim
    size = (_quant_work_bytes if quant else _work_bytes)(
        cache.n_kv, cache.page_size, dim, _TYPES[q.dtype], pages, n_seqs, n_tokens, heads, prompt)
    work = torch.empty(size, dtype=torch.uint8, device=cache.device) if size else None
    rest = (qr, _rows(out, "out", cache, kind), heads, dim ** -0.5 if scale is None else scale,
            work.data_ptr() if size else None, size)
    if quant:
        f = _lib().rpg_hip_quant_prompt if prompt else _lib().rpg_hip_quant_decode
        _enqueue(cache.device, f, cache._packed(), seqs, _TYPES[kind], *rest)
    else:
        f = _lib().rpg_hip_paged_prompt if prompt else _lib().rpg_hip_paged_decode
        _enqueue(cache.device, f, cache._packed(), seqs, *rest)
    _written(out)
    return out


def decode_attention(q, cache, table, lens, scale=None, out=None):
    """Attention of one token per sequence, q [sequences, heads, dim], over all of
    its sequence's positions. scale: 1 / sqrt(dim) when not given. out (may be q)
    is made when not given."""
    return _attention(q, cache, table, lens, None, scale, out, 0)


def prompt_attention(q, cache, table, lens, starts, scale=None, out=None):
    """Causal attention of the packed new tokens, q [tokens, heads, dim]: the token
    at position p of its sequence over positions 0 .. p, whose keys and values
    lie in the cache (the new tokens' own too). out (may be q) is made when not
    given; rows of no sequence are not written."""
    if starts is None:
        raise EngineError("starts is needed")
    return _attention(q, cache, table, lens, starts, scale, out, 1)


@functools.lru_cache(maxsize=4096)
def _shared_bytes(quant, n_kv, page_size, head_dim, kind, pages, n_seqs, n_groups, heads):
    """rpg_hip_paged_shared_work or rpg_hip_quant_shared_work of these sizes."""
    wide = page_size * head_dim
    s = _SEQS.pack(0, pages, 0, 0, pages, n_seqs, 0)
    if quant:
        c = _QUANT.pack(0, 0, 0, 0, n_kv * wide, wide, head_dim, n_kv * page_size, page_size, 1, page_size, n_kv, head_dim, 0)
        return _ok(_lib().rpg_hip_quant_shared_work(c, s, n_groups, kind, heads))
    c = _CACHE.pack(0, 0, n_kv * wide, wide, head_dim, 1, page_size, n_kv, head_dim, kind)
    return _ok(_lib().rpg_hip_paged_shared_work(c, s, n_groups, heads))


def shared_attention(q, cache, table, lens, groups, shared, scale=None, out=None):
    """decode_attention where the first positions of a group's sequences lie in the
    same pages, which are read once for the group: group g is sequences groups[g] ..
    groups[g + 1] (int32 [groups + 1]), and the tables of those that have positions
    name the same pages for the first shared[g] (int32 [groups]) positions (a larger
    count gives some of them another's keys and values). out (may be q) is made when not
    given."""
    quant = isinstance(cache, QuantCache)
    kind = _row_type(q, "q") if quant else None
    qr = _rows(q, "q", cache, kind)
    seqs, n_seqs, pages = _seqs(cache, table, lens, None, 0)
    if q.shape[0] != n_seqs:
        raise EngineError("q has a row for each sequence")
    dev, heads, dim = cache.device, q.shape[1], cache.head_dim
    n_groups = _ints(shared, "shared", 1, dev)[0]
    if _ints(groups, "groups", 1, dev)[0] != n_groups + 1:
        raise EngineError("groups has one value more than shared")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise EngineError("out has the shape of q")
    size = _shared_bytes(quant, cache.n_kv, cache.page_size, dim, _TYPES[q.dtype], pages, n_seqs, n_groups, heads)
    work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    of = _GROUPS.pack(groups.data_ptr(), shared.data_ptr(), n_groups)
    rest = (qr, _rows(out, "out", cache, kind), heads, dim ** -0.5 if scale is None else scale,
            work.data_ptr() if size else None, size)
    if quant:
        _enqueue(dev, _lib().rpg_hip_quant_shared, cache._packed(), seqs, of, _TYPES[kind], *rest)
    else:
        _enqueue(dev, _lib().rpg_hip_paged_shared, cache._packed(), seqs, of, *rest)
    _written(out)
    return out


@functools.lru_cache(maxsize=4096)
def _sample_bytes(rows, vocab):
    return _ok(_lib().rpg_hip_sample_rows_work(rows, vocab))


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits [rows, vocab], for given numbers u in [0, 1).
    temperature, top_p and min_p (float32), top_k (int32) and u are [rows] on the
    logits' GPU; None sets no limit (temperature 1). Returns (tokens int32, log
    of each token's probability among those kept, float32)."""
    if (logits.dim() != 2 or logits.dtype not in _TYPES or not logits.is_cuda
            or (logits.shape[1] > 1 and logits.stride(1) != 1)):
        raise EngineError("logits are [rows, vocab] float32, float16 or bfloat16 on a GPU, contiguous in the last dimension")
    if logits.requires_grad or forward_ad._current_level >= 0:
        _plain(logits, "logits")
    if u is None:
        raise EngineError("u is needed")
    rows, vocab = logits.shape
    dev, f32 = logits.device, torch.float32
    size = _sample_bytes(rows, vocab)
    tokens = torch.empty(rows, dtype=torch.int32, device=dev)
    logprobs = torch.empty(rows, dtype=f32, device=dev)
    work = torch.empty(size, dtype=torch.uint8, device=dev)
    _enqueue(dev, _lib().rpg_hip_sample_rows, _TYPES[logits.dtype], logits.data_ptr(), rows, vocab, logits.stride(0),
             _vector(temperature, "temperature", rows, f32, dev), _vector(top_k, "top_k", rows, torch.int32, dev),
             _vector(top_p, "top_p", rows, f32, dev), _vector(min_p, "min_p", rows, f32, dev), _vector(u, "u", rows, f32, dev),
             tokens.data_ptr(), logprobs.data_ptr(), work.data_ptr(), size)
    return tokens, logprobs


def _list(x, name, rows, dtype, device):
    """(address, elements between rows, row length) of a [rows, n] matrix whose rows
    are contiguous; rows may be one and the same (an expanded view)."""
    if (x.dim() != 2 or x.dtype is not dtype or x.device != device or (rows is not None and x.shape[0] != rows)
            or (x.shape[1] > 1 and x.stride(1) != 1) or x.stride(0) < 0):
        raise EngineError(f"{name} is {dtype} [{'masks' if rows is None else 'rows'}, n], contiguous in the last dimension, on the logits' GPU")
    if x.requires_grad or forward_ad._current_level >= 0:
        _plain(x, name)
    return x.data_ptr(), x.stride(0), x.shape[1]


def edit_logits(logits, history=None, history_lens=None, prompts=None, repetition=None, presence=None, frequency=None,
                bias_ids=None, bias=None, mask=None, mask_rows=None, out=None):
    """logits [rows, vocab] with penalties, biases and masks, into out (made when not
    given; may be logits, and else lies apart from them). In this order, where c counts how often a row's history
    holds a token behind the row's prompt:

        x = x / repetition if x > 0 else x * repetition   tokens of the history
        x = x - frequency * c - presence                  tokens with c > 0
        x = x + bias                                      tokens of bias_ids
        x = -inf                                          tokens whose mask bit is 0

    history int32 [rows, n], of which the first history_lens [rows] tokens are there,
    the first prompts [rows] of those the prompt; repetition, presence and frequency
    float32 [rows]; bias_ids int32 and bias float32 [rows, m] (numbers outside the
    vocabulary are no entries, of several for a token the last counts); mask int32
    [masks, ceil(vocab / 32)], token t at bit t % 32 of word t / 32; row r goes by mask
    mask_rows[r] (int32 [rows]; r when not given), by none where that names no mask.
    None leaves an edit out. Returns out."""
    if (logits.dim() != 2 or logits.dtype not in _TYPES or not logits.is_cuda
            or (logits.shape[1] > 1 and logits.stride(1) != 1)):
        raise EngineError("logits are [rows, vocab] float32, float16 or bfloat16 on a GPU, contiguous in the last dimension")
    if logits.requires_grad or forward_ad._current_level >= 0:
        _plain(logits, "logits")
    rows, vocab = logits.shape
    dev, f32, i32 = logits.device, torch.float32, torch.int32
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=dev)
    elif (out.shape != logits.shape or out.dtype is not logits.dtype or out.device != dev
          or (vocab > 1 and out.stride(1) != 1)):
        raise EngineError("out is of the logits' shape, type and GPU, contiguous in the last dimension")
    elif out.requires_grad or forward_ad._current_level >= 0:
        _plain(out, "out")
    if history is None and not (history_lens is prompts is repetition is presence is frequency is None):
        raise EngineError("history_lens, prompts and penalties go with a history")
    if (bias_ids is None) != (bias is None):
        raise EngineError("bias_ids and bias go together")
    if mask is None and mask_rows is not None:
        raise EngineError("mask_rows goes with a mask")
    h = b = w = m = (None, 0, 0)
    if history is not None:
        h = _list(history, "history", rows, i32, dev)
    if bias is not None:
        b, w = _list(bias_ids, "bias_ids", rows, i32, dev), _list(bias, "bias", rows, f32, dev)
        if b[2] != w[2]:
            raise EngineError("bias_ids and bias are of one shape")
    masks = 0
    if mask is not None:
        m, masks = _list(mask, "mask", None, i32, dev), mask.shape[0]
        if m[2] != (vocab + 31) // 32:
            raise EngineError("mask has a bit for each token: ceil(vocab / 32) words a row")
        if mask_rows is None and masks < rows:
            raise EngineError("mask has a row for each row of logits, or mask_rows says which")
    row = [_vector(x, name, rows, t, dev) or 0 for x, name, t in (
        (history_lens, "history_lens", i32), (prompts, "prompts", i32), (repetition, "repetition", f32),
        (presence, "presence", f32), (frequency, "frequency", f32), (mask_rows, "mask_rows", i32))]
    if not h[2]:  # no token: no penalty
        h, row[:5] = (0, 0, 0), [0] * 5
    if not b[2]:
        b = w = (0, 0, 0)
    if not masks:  # no mask that a row could go by
        m, row[5] = (0, 0, 0), 0
    edits = _EDITS.pack(h[0], h[1], *row[:5], b[0], b[1], w[0], w[1], m[0] or 0, m[1], row[5], h[2], b[2], masks)
    _enqueue(dev, _lib().rpg_hip_edit_logits, _TYPES[logits.dtype], logits.data_ptr(), rows, vocab, logits.stride(0), edits,
             out.data_ptr(), out.stride(0))
    _written(out)
    return out

"""The serving operators of include/rpg_hip.h on torch tensors: one paged
key-value cache for many sequences, the attention that reads it and a sampler
of many rows, for hosts that schedule sessions themselves.

    cache = serving.PagedCache.zeros(n_pages, 16, n_kv, 128, torch.bfloat16)
    serving.append(cache, table, lens, starts, k, v, q=q, q_norm=..., k_norm=..., rope=...)
    out = serving.prompt_attention(q, cache, table, lens, starts)   # prompts, packed
    out = serving.decode_attention(q, cache, table, lens)           # one token each
    tokens, logprobs = serving.sample(logits, u, temperature, top_k, top_p, min_p)

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

_SIGS = {
    "rpg_hip_paged_append": ([_P, _P, _P, _P, _P, _P, _I32, _P, _P, _F, _P, _I64, _P], _I32),
    "rpg_hip_paged_decode": ([_P, _P, _P, _P, _I32, _F, _P, _I64, _P], _I32),
    "rpg_hip_paged_prompt": ([_P, _P, _P, _P, _I32, _F, _P, _I64, _P], _I32),
    "rpg_hip_paged_work": ([_P, _P, _I32, _I32], _I64),
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


def _rows(x, name, cache):
    shape, strides = x.shape, x.stride()
    if (len(shape) != 3 or x.dtype is not cache.dtype or x.device != cache.device or shape[2] != cache.head_dim
            or strides[2] != 1):
        raise EngineError(f"{name} is [tokens, heads, head dim] of the cache's type and GPU, contiguous in the last dimension")
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
    if torch.cuda.current_device() == device.index:
        rc = f(*args, _stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = f(*args, _stream(device.index))
    if rc < 0:
        _ok(rc)


# What a call writes in place is a new version of the tensor to autograd: a
# backward pass that saved the old one refuses.
_written = torch.autograd.graph.increment_version


def _stream(index):
    return torch.cuda.current_stream(index).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):  # the same without a Stream object for each call
    _stream = torch._C._cuda_getCurrentRawStream


def append(cache: PagedCache, table, lens, starts, k, v, q=None, q_out=None, q_norm=None, k_norm=None,
           eps: float = 1e-6, rope=None):
    """Stores the packed new tokens' keys and values, k and v [tokens, key heads,
    dim], in their pages; q [tokens, heads, dim] goes to q_out (made when not
    given; may be q). Keys and queries are RMS-normed per head with the gains
    k_norm and q_norm (float32 [dim]) and rotated by rope (float32 [positions,
    dim]: cos | sin) where those are given. Returns q_out."""
    kr, vr = _rows(k, "k", cache), _rows(v, "v", cache)
    n = k.shape[0]
    seqs = _seqs(cache, table, lens, starts, n)[0]
    if v.shape != k.shape or k.shape[1] != cache.n_kv:
        raise EngineError("k and v are [tokens, key heads of the cache, head dim]")
    heads, qr, qo = 0, None, None
    if q is not None:
        qr = _rows(q, "q", cache)
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if q.shape[0] != n or q_out.shape != q.shape:
            raise EngineError("q, q_out and k are of one number of tokens")
        qo = _rows(q_out, "q_out", cache)
    dev, dim = cache.device, cache.head_dim
    rp, rope_rows = None, 0
    if rope is not None:
        if (rope.dtype is not torch.float32 or rope.dim() != 2 or rope.shape[1] != dim or not rope.is_contiguous()
                or rope.device != dev):
            raise EngineError("rope is float32 [positions, head dim], contiguous, on the same GPU")
        if rope.requires_grad or forward_ad._current_level >= 0:
            _plain(rope, "rope")
        rp, rope_rows = rope.data_ptr(), rope.shape[0]
    _enqueue(dev, _lib().rpg_hip_paged_append, cache._packed(), seqs, kr, vr, qr, qo, heads,
             _vector(q_norm, "q_norm", dim, torch.float32, dev), _vector(k_norm, "k_norm", dim, torch.float32, dev), eps,
             rp, rope_rows)
    _written((cache._k, cache._v) if qo is None else (cache._k, cache._v, q_out))
    return q_out


@functools.lru_cache(maxsize=4096)
def _work_bytes(n_kv, page_size, head_dim, kind, pages, n_seqs, n_tokens, heads, prompt):
    """rpg_hip_paged_work of these sizes."""
    wide = page_size * head_dim
    c = _CACHE.pack(0, 0, n_kv * wide, wide, head_dim, 1, page_size, n_kv, head_dim, kind)
    return _ok(_lib().rpg_hip_paged_work(c, _SEQS.pack(0, pages, 0, 0, pages, n_seqs, n_tokens), heads, prompt))


def _attention(f, q, qr, cache, seqs, n_seqs, pages, n_tokens, scale, out, prompt):
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise EngineError("out has the shape of q")
    heads, dim = q.shape[1], cache.head_dim
    size = _work_bytes(cache.n_kv, cache.page_size, dim, _TYPES[cache.dtype], pages, n_seqs, n_tokens, heads, prompt)
    work = torch.empty(size, dtype=torch.uint8, device=cache.device) if size else None
    _enqueue(cache.device, f, cache._packed(), seqs, qr, _rows(out, "out", cache), heads, dim ** -0.5 if scale is None else scale,
             work.data_ptr() if size else None, size)
    _written(out)
    return out


def decode_attention(q, cache: PagedCache, table, lens, scale=None, out=None):
    """Attention of one token per sequence, q [sequences, heads, dim], over all of
    its sequence's positions. scale: 1 / sqrt(dim) when not given. out (may be q)
    is made when not given."""
    qr = _rows(q, "q", cache)
    seqs, n, pages = _seqs(cache, table, lens, None, 0)
    if q.shape[0] != n:
        raise EngineError("q has a row for each sequence")
    return _attention(_lib().rpg_hip_paged_decode, q, qr, cache, seqs, n, pages, 0, scale, out, 0)


def prompt_attention(q, cache: PagedCache, table, lens, starts, scale=None, out=None):
    """Causal attention of the packed new tokens, q [tokens, heads, dim]: the token
    at position p of its sequence over positions 0 .. p, whose keys and values
    lie in the cache (the new tokens' own too). out (may be q) is made when not
    given; rows of no sequence are not written."""
    qr = _rows(q, "q", cache)
    tokens = q.shape[0]
    if starts is None:
        raise EngineError("starts is needed")
    seqs, n, pages = _seqs(cache, table, lens, starts, tokens)
    return _attention(_lib().rpg_hip_paged_prompt, q, qr, cache, seqs, n, pages, tokens, scale, out, 1)


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

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
the values of each replay. There is no backward pass: tensors that require
gradients are refused while gradients are recorded.
"""

from __future__ import annotations

import ctypes

import torch

from . import EngineError, lib

_P, _I32, _I64, _F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}  # ggml ids


class _Cache(ctypes.Structure):
    _fields_ = [("k", _P), ("v", _P), ("page_stride", _I64), ("head_stride", _I64), ("row_stride", _I64),
                ("n_pages", _I32), ("page_size", _I32), ("n_kv", _I32), ("head_dim", _I32), ("type", _I32)]


class _Seqs(ctypes.Structure):
    _fields_ = [("table", _P), ("table_stride", _I64), ("lens", _P), ("starts", _P), ("pages", _I32),
                ("n_seqs", _I32), ("n_tokens", _I32)]


class _Rows(ctypes.Structure):
    _fields_ = [("data", _P), ("token_stride", _I64), ("head_stride", _I64)]


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


def _check(cond, what):
    if not cond:
        raise EngineError(what)


class PagedCache:
    """A pool of key and value pages, [pages, key heads, page size, head dim] each
    (f32, f16 or bf16; views of a larger pool are fine)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _check(k.dim() == 4 and v.shape == k.shape, "k and v are [pages, key heads, page size, head dim]")
        _check(k.dtype in _TYPES and v.dtype == k.dtype, "k and v are both float32, float16 or bfloat16")
        _check(k.is_cuda and v.device == k.device, "k and v lie on one GPU")
        _check(k.stride(3) == 1 and k.stride() == v.stride(), "k and v have the same strides, 1 in the last dimension")
        self.k, self.v = k, v
        self.device, self.dtype = k.device, k.dtype
        n_pages, n_kv, page, dim = k.shape
        self.n_kv, self.head_dim, self.page_size = n_kv, dim, page
        strides = [s if n > 1 else page * dim * 16 for n, s in zip(k.shape, k.stride())]
        self._c = _Cache(k.data_ptr(), v.data_ptr(), strides[0], strides[1], strides[2], n_pages, page, n_kv, dim,
                         _TYPES[k.dtype])
        self._p = ctypes.byref(self._c)

    @classmethod
    def zeros(cls, n_pages: int, page_size: int, n_kv: int, head_dim: int, dtype=torch.float32,
              device="cuda") -> "PagedCache":
        shape = (n_pages, n_kv, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))


def _ints(x, name, dims, device):
    _check(x.dtype == torch.int32 and x.dim() == dims and x.device == device and (x.shape[-1] <= 1 or x.stride(-1) == 1),
           f"{name} is int32, of {dims} dimension(s), contiguous in the last, on the cache's GPU")
    return x.data_ptr()


def _seqs(cache, table, lens, starts, n_tokens):
    dev = cache.device
    n, pages = table.shape if table.dim() == 2 else (-1, 0)
    t, le = _ints(table, "table", 2, dev), _ints(lens, "lens", 1, dev)
    _check(lens.shape[0] == n, "lens and table are of one number of sequences")
    st = None
    if starts is not None:
        st = _ints(starts, "starts", 1, dev)
        _check(starts.shape[0] == n + 1, "starts has one value more than there are sequences")
    return _Seqs(t, table.stride(0), le, st, pages, n, n_tokens)


def _rows(x, name, cache, heads=None):
    _check(x.dim() == 3 and x.dtype == cache.dtype and x.device == cache.device and x.shape[2] == cache.head_dim
           and x.stride(2) == 1 and (heads is None or x.shape[1] == heads),
           f"{name} is [tokens, heads, head dim] of the cache's type and GPU, contiguous in the last dimension")
    _check(not (x.requires_grad and torch.is_grad_enabled()), f"{name} requires gradients: there is no backward pass")
    t, h = x.stride(0), x.stride(1)
    if x.shape[0] == 1:
        t = x.shape[1] * x.shape[2]
    if x.shape[1] == 1:
        h = x.shape[2]
    return _Rows(x.data_ptr(), t, h)


def _vector(x, name, n, dtype, device):
    """The address of a contiguous vector; None stays None."""
    if x is None:
        return None
    _check(x.dtype == dtype and x.shape == (n,) and x.device == device and (n <= 1 or x.stride(0) == 1),
           f"{name} is {dtype} [{n}], contiguous, on the same GPU")
    return x.data_ptr()


def _enqueue(device, call):
    """call(stream) with the tensors' GPU current."""
    if torch.cuda.current_device() == device.index:
        return _ok(call(torch.cuda.current_stream().cuda_stream))
    with torch.cuda.device(device):
        return _ok(call(torch.cuda.current_stream().cuda_stream))


def append(cache: PagedCache, table, lens, starts, k, v, q=None, q_out=None, q_norm=None, k_norm=None,
           eps: float = 1e-6, rope=None):
    """Stores the packed new tokens' keys and values, k and v [tokens, key heads,
    dim], in their pages; q [tokens, heads, dim] goes to q_out (made when not
    given; may be q). Keys and queries are RMS-normed per head with the gains
    k_norm and q_norm (float32 [dim]) and rotated by rope (float32 [positions,
    dim]: cos | sin) where those are given. Returns q_out."""
    L = _lib()
    seqs = _seqs(cache, table, lens, starts, k.shape[0])
    kr, vr = _rows(k, "k", cache, cache.n_kv), _rows(v, "v", cache, cache.n_kv)
    _check(v.shape == k.shape, "k and v are of one number of tokens")
    heads, qr, qo = 0, None, None
    if q is not None:
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _check(q.shape[0] == k.shape[0] and q_out.shape == q.shape, "q, q_out and k are of one number of tokens")
        qr, qo = ctypes.byref(_rows(q, "q", cache)), ctypes.byref(_rows(q_out, "q_out", cache))
    dev, dim = cache.device, cache.head_dim
    qn, kn = _vector(q_norm, "q_norm", dim, torch.float32, dev), _vector(k_norm, "k_norm", dim, torch.float32, dev)
    rp, rope_rows = None, 0
    if rope is not None:
        _check(rope.dtype == torch.float32 and rope.dim() == 2 and rope.shape[1] == dim and rope.is_contiguous()
               and rope.device == dev, "rope is float32 [positions, head dim], contiguous, on the same GPU")
        rp, rope_rows = rope.data_ptr(), rope.shape[0]
    _enqueue(dev, lambda s: L.rpg_hip_paged_append(cache._p, ctypes.byref(seqs), ctypes.byref(kr), ctypes.byref(vr), qr,
                                                   qo, heads, qn, kn, eps, rp, rope_rows, s))
    return q_out


def _attention(q, cache, seqs, scale, out, prompt):
    L = _lib()
    qr = _rows(q, "q", cache)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check(out.shape == q.shape, "out has the shape of q")
    o = _rows(out, "out", cache)
    heads = q.shape[1]
    if scale is None:
        scale = cache.head_dim ** -0.5
    sp = ctypes.byref(seqs)
    size = _ok(L.rpg_hip_paged_work(cache._p, sp, heads, prompt))
    work = torch.empty(size, dtype=torch.uint8, device=cache.device) if size else None
    f = L.rpg_hip_paged_prompt if prompt else L.rpg_hip_paged_decode
    _enqueue(cache.device, lambda s: f(cache._p, sp, ctypes.byref(qr), ctypes.byref(o), heads, scale,
                                       work.data_ptr() if size else None, size, s))
    return out


def decode_attention(q, cache: PagedCache, table, lens, scale=None, out=None):
    """Attention of one token per sequence, q [sequences, heads, dim], over all of
    its sequence's positions. scale: 1 / sqrt(dim) when not given. out (may be q)
    is made when not given."""
    _check(q.dim() == 3 and q.shape[0] == lens.shape[0], "q has a row for each sequence")
    return _attention(q, cache, _seqs(cache, table, lens, None, 0), scale, out, 0)


def prompt_attention(q, cache: PagedCache, table, lens, starts, scale=None, out=None):
    """Causal attention of the packed new tokens, q [tokens, heads, dim]: the token
    at position p of its sequence over positions 0 .. p, whose keys and values
    lie in the cache (the new tokens' own too)."""
    _check(q.dim() == 3, "q is [tokens, heads, head dim]")
    return _attention(q, cache, _seqs(cache, table, lens, starts, q.shape[0]), scale, out, 1)


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits [rows, vocab], for given numbers u in [0, 1).
    temperature, top_p and min_p (float32), top_k (int32) and u are [rows] on the
    logits' GPU; None sets no limit (temperature 1). Returns (tokens int32, log
    of each token's probability among those kept, float32)."""
    L = _lib()
    _check(logits.dim() == 2 and logits.dtype in _TYPES and logits.is_cuda
           and (logits.shape[1] <= 1 or logits.stride(1) == 1),
           "logits are [rows, vocab] float32, float16 or bfloat16 on a GPU, contiguous in the last dimension")
    _check(not (logits.requires_grad and torch.is_grad_enabled()), "logits require gradients: there is no backward pass")
    rows, vocab = logits.shape
    dev, f32 = logits.device, torch.float32
    _check(u is not None, "u is needed")
    up, t, p = _vector(u, "u", rows, f32, dev), _vector(temperature, "temperature", rows, f32, dev), _vector(
        top_p, "top_p", rows, f32, dev)
    m, k = _vector(min_p, "min_p", rows, f32, dev), _vector(top_k, "top_k", rows, torch.int32, dev)
    size = _ok(L.rpg_hip_sample_rows_work(rows, vocab))
    tokens = torch.empty(rows, dtype=torch.int32, device=dev)
    logprobs = torch.empty(rows, dtype=f32, device=dev)
    work = torch.empty(size, dtype=torch.uint8, device=dev)
    _enqueue(dev, lambda s: L.rpg_hip_sample_rows(_TYPES[logits.dtype], logits.data_ptr(), rows, vocab, logits.stride(0),
                                                  t, k, p, m, up, tokens.data_ptr(), logprobs.data_ptr(),
                                                  work.data_ptr(), size, s))
    return tokens, logprobs

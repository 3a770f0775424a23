"""Language-model serving operators: Python mirror of include/parakeet_lm.h.

What a decoder-only model that answers a decoded turn needs beside its matrix
products, over sessions that share one paged cache held in 4 bits:

    plan    = lm.kv_plan(...)       which page each session's new tokens go to
    lm.kv4_store(k, v, ...)         a layer's key and value rows into the cache
    lm.kv4_attend(q, ...)           attention over it: single tokens, a few, whole prompts
    lm.sample(logits, u, ...)       the next token of every session
    lm.kv4_load(...)                rows back out of the cache

Arrays are ``torch`` tensors on the GPU or ``hipmem.Tensor``s, inputs and
outputs alike: outputs are given by the caller and written in place.  Calls are
enqueued on ``stream`` (a hipStream_t as an integer; by default torch's current
stream for torch tensors, the default stream for others), allocate nothing but
the workspaces below, wait for nothing and can be captured into a graph.
Arguments are checked here and in the library; ``pk.PkError`` carries the
library's status.

Workspaces (``kv4_attend``, ``sample``) are kept per operator, device and stream and only
ever grow; one that has been handed out is never freed, since a captured graph
may hold it.  For torch tensors a graph's capture has its own, which the graph zeroes, so that
graphs may be replayed in any order and beside each other.  Other graphs share their
stream's: one that is to run beside calls on that stream, or beside another of its
graphs, is given a ``workspace=`` (zeroed uint8) of its own.

torch tensors are read by an extension of their own (csrc/lm_torch.cpp), others
here, through ctypes.  The operators have no backward pass: a tensor that requires a
gradient is refused unless gradients are off (``torch.no_grad()``).  Tensors given with a
``stream`` other than torch's current one have to stay until it has passed the call
(``Tensor.record_stream``).  torch and this library have to share one HIP runtime:
where torch tensors are used, import torch before the library is first loaded.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import os
import struct
import sys

from . import hipmem, pk

F32, F16, BF16 = 0, 1, 2                 # parakeet_lm.h PK_DTYPE_*
PAGES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)
MAX_REQUESTS, MAX_VOCAB = 4096, 1048576

EXPORTED = ["pk_kv_plan", "pk_kv4_store", "pk_kv4_load", "pk_kv4_attend", "pk_kv4_attend_workspace", "pk_sample",
            "pk_sample_workspace"]
TORCH_PATH = os.path.join(pk.HERE, "_lm_torch.so")

_FLOATS = {"f32": F32, "f16": F16, "bf16": BF16}
_calls: dict = {}
_workspaces: dict = {}


class _NoTorch:
    """Stands for torch.Tensor until a torch tensor is met."""


_Tensor = _NoTorch
_torch_calls = None

# the descriptors of parakeet_lm.h, in their order (native alignment)
_PLAN = struct.Struct("11Pq5i0P")
_ROWS = struct.Struct("4P5q6i0P")
_ATTEND = struct.Struct("8P7q12if0P")
_SAMPLE = struct.Struct("10P2q4i0P")


def _load():
    L = pk.lib()
    for name in EXPORTED:
        f = getattr(L, name)
        f.argtypes = [C.c_char_p, C.c_void_p]
        _calls[name] = f


def _new_torch(t):
    """Whether t is a torch tensor, the first one to come: loads the extension that reads them."""
    global _Tensor, _torch_calls
    torch = sys.modules.get("torch")
    if _Tensor is not _NoTorch or torch is None or not isinstance(t, torch.Tensor):
        return False
    pk.lib()
    runtimes = set()
    with open("/proc/self/maps") as f:
        for line in f:
            if "libamdhip64" in line:
                runtimes.add(line.split(None, 5)[5].strip())
    if len(runtimes) > 1:
        raise RuntimeError(f"two HIP runtimes are loaded ({', '.join(sorted(runtimes))}): import torch before the parakeet library")
    if not os.path.exists(TORCH_PATH):
        raise RuntimeError(f"{TORCH_PATH} is not built: run __graft_entry__.build()")
    spec = importlib.util.spec_from_file_location("_lm_torch", TORCH_PATH)
    _torch_calls = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(_torch_calls)
    _Tensor = torch.Tensor
    return True


def _call(name, packed, stream):
    if not _calls:
        _load()
    rc = _calls[name](packed, stream)
    if rc:
        pk.check(rc)


def _dtype(t, what):
    d = _FLOATS.get(t.dtype)
    if d is None:
        raise TypeError(f"{what}: {t.dtype} (f32, f16 or bf16)")
    return d


def _i32(t, shape, what):
    """Pointer of a contiguous int32 array of this shape."""
    if t.dtype != "i32":
        raise TypeError(f"{what}: {t.dtype} (int32)")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: not contiguous")
    return t.data_ptr()


def _f32(t, shape, what):
    if _dtype(t, what) != F32:
        raise TypeError(f"{what}: {t.dtype} (f32)")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: not contiguous")
    return t.data_ptr()


def _rows(t, what):
    """(pointer, row stride) of a 2-d array whose last axis is adjacent."""
    s = t.stride()
    if s[1] != 1 and t.shape[1] > 1:
        raise ValueError(f"{what}: the last axis is not adjacent (strides {tuple(s)})")
    return t.data_ptr(), s[0]


def _heads(t, what):
    """(pointer, row stride, head stride) of an array [rows, heads, head_dim] whose channels are adjacent."""
    if len(t.shape) != 3:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected [rows, heads, head_dim]")
    s = t.stride()
    if s[2] != 1:
        raise ValueError(f"{what}: channels are not adjacent (strides {tuple(s)})")
    return t.data_ptr(), s[0], s[1]


def _cache(cache, page, what):
    """(pointer, page stride, pages, heads, head_dim) of cache [n_pages, kv_heads, page (D + D/16)] bytes."""
    if cache.dtype != "u8":
        raise TypeError(f"{what}: cache of {cache.dtype} (uint8)")
    n, heads, size = cache.shape
    s = cache.stride()
    dim, odd = divmod(size * 16, page * 17)
    if odd or s[2] != 1 or (heads > 1 and s[1] != size):
        raise ValueError(f"{what}: cache of shape {tuple(cache.shape)}, strides {tuple(s)}: expected kv4_shape(...) "
                         f"for pages of {page} tokens, the records of a page adjacent")
    return cache.data_ptr(), s[0] if n > 1 else heads * size, n, heads, dim


def kv4_shape(n_pages: int, kv_heads: int, head_dim: int, page: int):
    """Shape of a cache (uint8) of n_pages pages of `page` tokens: 17 bytes per 32 values of K and of V."""
    if page not in PAGES or head_dim not in HEAD_DIMS:
        raise ValueError(f"pages of {page} tokens (one of {PAGES}), head_dim {head_dim} (one of {HEAD_DIMS})")
    return n_pages, kv_heads, page * (head_dim + head_dim // 16)


def _workspace(kind, stream, wanted, given):
    """(pointer, bytes) of at least `wanted` bytes, zeroed before the first use; each kind of call has its own on each device
    and stream."""
    if given is not None:
        if given.dtype != "u8" or not given.is_contiguous():
            raise TypeError("workspace: not contiguous uint8")
        return given.data_ptr(), given.numel()
    if wanted == 0:
        return 0, 0
    kept = _workspaces.setdefault((kind, hipmem.device(), stream), [])
    if not kept or kept[-1].numel() < wanted:
        if hipmem.capturing(stream):
            raise RuntimeError(f"{kind}: a workspace of {wanted} bytes cannot be made during a capture: give workspace=, "
                               "or make one call of these sizes on the stream before")
        t = hipmem.Tensor((max(1 << 20, 1 << (wanted - 1).bit_length()),), "u8")
        t.zero()
        hipmem.synchronize()
        kept.append(t)
    return kept[-1].data_ptr(), kept[-1].numel()


def kv_plan(old_len, new_len, table, ring, state, page: int, *, state_out, lens, ok, first, slots, pos=None, stream=None):
    """pk_kv_plan: request b holds old_len[b] tokens and is to hold new_len[b].

    table [requests, width] page ids (new ones are entered), ring [n_pages] the
    free page ids, state [2] its {head, count}.  Written: state_out [2], lens and
    ok [requests], first [requests + 1], slots and pos [n_tokens].
    """
    if isinstance(table, _Tensor) or _new_torch(table):
        rc = _torch_calls.kv_plan(old_len, new_len, table, ring, state, page, state_out, lens, ok, first, slots, pos, stream)
        if rc:
            pk.check(rc)
        return
    B, width = table.shape
    if table.dtype != "i32":
        raise TypeError(f"table: {table.dtype} (int32)")
    tp, ts = _rows(table, "table")
    n, cap = ring.shape[0], slots.shape[0]
    packed = _PLAN.pack(_i32(old_len, (B,), "old_len"), _i32(new_len, (B,), "new_len"), tp, _i32(ring, (n,), "ring"),
                        _i32(state, (2,), "state"), _i32(state_out, (2,), "state_out"), _i32(lens, (B,), "lens"),
                        _i32(ok, (B,), "ok"), _i32(first, (B + 1,), "first"), _i32(slots, (cap,), "slots"),
                        0 if pos is None else _i32(pos, (cap,), "pos"), ts, B, width, n, page, cap)
    _call("pk_kv_plan", packed, stream)


def _kv4_rows(name, k, v, slots, cache, page, stream):
    dt = _dtype(k, "k")
    if v.dtype != k.dtype or tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"k {k.dtype} {tuple(k.shape)}, v {v.dtype} {tuple(v.shape)}")
    kp, kr, kh = _heads(k, "k")
    vp, vr, vh = _heads(v, "v")
    cp, ps, n_pages, heads, dim = _cache(cache, page, name)
    n = k.shape[0]
    if k.shape[1] != heads or k.shape[2] != dim:
        raise ValueError(f"rows of {k.shape[1]} heads of {k.shape[2]}, a cache of {heads} heads of {dim}")
    packed = _ROWS.pack(kp, vp, _i32(slots, (n,), "slots"), cp, kr, kh, vr, vh, ps, n, heads, dim, dt, page, n_pages)
    _call(name, packed, stream)


def kv4_store(k, v, slots, cache, page: int, stream=None):
    """pk_kv4_store: rows k, v [n, kv_heads, head_dim] into cache at slots [n]; rows with a slot outside it (-1) are
    skipped."""
    if isinstance(cache, _Tensor) or _new_torch(cache):
        rc = _torch_calls.kv4_store(k, v, slots, cache, page, stream)
        if rc:
            pk.check(rc)
        return
    _kv4_rows("pk_kv4_store", k, v, slots, cache, page, stream)


def kv4_load(cache, slots, k, v, page: int, stream=None):
    """pk_kv4_load: what the cache holds at slots [n], into k, v [n, kv_heads, head_dim]; rows with a slot outside it
    are left as they are."""
    if isinstance(cache, _Tensor) or _new_torch(cache):
        rc = _torch_calls.kv4_load(cache, slots, k, v, page, stream)
        if rc:
            pk.check(rc)
        return
    _kv4_rows("pk_kv4_load", k, v, slots, cache, page, stream)


def kv4_attend(q, cache, table, lens, out, page: int, *, first=None, max_new: int = 1, max_len: int | None = None,
               scale: float | None = None, window: int = 0, lse=None, workspace=None, stream=None):
    """pk_kv4_attend: out = softmax(scale q K^T) V, causal.

    q, out [n_rows, heads, head_dim]; table [requests, width]; lens [requests]
    tokens held, q's included; first [requests + 1] where each request's queries
    begin (None: one query each); max_new and max_len bound the queries and the
    tokens of any request (max_len defaults to what the table can name); window
    > 0 limits every query to its last `window` keys; lse [n_rows, heads] f32.
    """
    if isinstance(q, _Tensor) or _new_torch(q):
        rc = _torch_calls.kv4_attend(q, cache, table, lens, out, page, first, max_new, max_len, scale, window, lse, workspace, stream)
        if rc:
            pk.check(rc)
        return
    dt = _dtype(q, "q")
    if out.dtype != q.dtype or tuple(out.shape) != tuple(q.shape):
        raise ValueError(f"q {q.dtype} {tuple(q.shape)}, out {out.dtype} {tuple(out.shape)}")
    qp, qr, qh = _heads(q, "q")
    op, our, oh = _heads(out, "out")
    cp, ps, n_pages, kv_heads, dim = _cache(cache, page, "kv4_attend")
    n, heads, d = q.shape
    B, width = table.shape
    if d != dim or heads % kv_heads:
        raise ValueError(f"{heads} query heads of {d}, a cache of {kv_heads} heads of {dim}")
    if (heads > 1 and oh < dim) or (n > 1 and our < dim):
        raise ValueError(f"out: rows overlap (strides {our}, {oh})")
    if table.dtype != "i32":
        raise TypeError(f"table: {table.dtype} (int32)")
    tp, ts = _rows(table, "table")
    if max_len is None:
        max_len = min(width * page, 2 ** 31 - 4097)
    head = (qp, op, 0 if lse is None else _f32(lse, (n, heads), "lse"), cp, tp, _i32(lens, (B,), "lens"),
            0 if first is None else _i32(first, (B + 1,), "first"))
    tail = (qr, qh, our, oh, ps, ts, n, B, heads, kv_heads, dim, dt, page, n_pages, width, max_new, max_len, window,
            dim ** -0.5 if scale is None else scale)
    wanted = C.c_int64()
    _call("pk_kv4_attend_workspace", _ATTEND.pack(*head, 0, 0, *tail), C.addressof(wanted))
    wp, wb = _workspace("attend", stream, wanted.value, workspace)
    _call("pk_kv4_attend", _ATTEND.pack(*head, wp, wb, *tail), stream)


def sample(logits, u, token, *, temperature=None, top_k=None, top_p=None, min_p=None, prob=None, kept=None, workspace=None,
           stream=None):
    """pk_sample: one token per row of logits [rows, vocab], from the uniform numbers u [rows].

    temperature, top_p, min_p [rows] f32 and top_k [rows] int32, each nullable;
    token [rows] int32, prob [rows] f32 (its share of the kept weight) and kept
    [rows] int32 (how many tokens were kept) are written.
    """
    if isinstance(logits, _Tensor) or _new_torch(logits):
        rc = _torch_calls.sample(logits, u, token, temperature, top_k, top_p, min_p, prob, kept, workspace, stream)
        if rc:
            pk.check(rc)
        return
    dt = _dtype(logits, "logits")
    B, V = logits.shape
    lp, lr = _rows(logits, "logits")
    shape = (B,)
    opt = lambda f, t, what: 0 if t is None else f(t, shape, what)  # noqa: E731
    head = (lp, _f32(u, shape, "u"), opt(_f32, temperature, "temperature"), opt(_i32, top_k, "top_k"),
            opt(_f32, top_p, "top_p"), opt(_f32, min_p, "min_p"), _i32(token, shape, "token"), opt(_f32, prob, "prob"),
            opt(_i32, kept, "kept"))
    wanted = C.c_int64()
    _call("pk_sample_workspace", _SAMPLE.pack(*head, 0, 0, lr, B, V, dt, 0), C.addressof(wanted))
    wp, wb = _workspace("sample", stream, wanted.value, workspace)
    _call("pk_sample", _SAMPLE.pack(*head, wp, wb, lr, B, V, dt, 0), stream)

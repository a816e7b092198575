"""A paged cache of keys and values held in 4 bits, and causal attention over it: the serving side of a token decoder.

Host side of `b200_kv4_append`, `b200_kv4_read` and `b200_kv4_attention` (include/b200_decoder.h, which states the layout). The cache
is a plain tensor, pages are handed out by the caller: `page_table` `[batch, columns]` int32 holds the pages of each sequence in order,
`lengths` `[batch]` int32 its tokens, those of the current call among them. A decoding step is

    q = kv4_append_(cache, k, v, page_table, lengths, table=table, q=q)     # q and k turned, k and v written
    o = kv4_attention(q, cache, page_table, lengths)
"""

from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib
from .rotary import refuse_tangent

BLOCK = 16  # tokens
HEAD_DIMS = (64, 128)
_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}

# Partial results and counters of attention by (device, stream), as attention() keeps its own.
_WORKSPACES: dict[tuple[int, int], tuple[torch.Tensor, torch.Tensor]] = {}
_WORKSPACES_LOCK = threading.Lock()


def kv4_cache(pages: int, kv_heads: int, head_dim: int, *, page: int = 64, device: torch.device | str = "cuda") -> torch.Tensor:
    """An empty cache, uint8 `[pages, kv_heads, page / 16, 16 (head_dim + 8)]`: 4 bits a value and a step and a least value (bfloat16)
    for K and for V of each head and token.

    Raises:
        ValueError: A head dim other than 64 or 128, or a page that is no multiple of 16 tokens.
    """
    if head_dim not in HEAD_DIMS or page < BLOCK or page % BLOCK or pages < 1 or kv_heads < 1:
        msg = f"kv4_cache: head_dim {head_dim} must be one of {HEAD_DIMS}, page {page} a multiple of {BLOCK}, pages {pages} and kv_heads {kv_heads} positive"
        raise ValueError(msg)
    return torch.zeros(pages, kv_heads, page // BLOCK, BLOCK * (head_dim + 8), dtype=torch.uint8, device=device)


def reserve_kv4_workspace(device: torch.device | int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Scratch of the current stream of `device` for `kv4_attention`, allocated on first use: partial results (39.4 MB on a B200) and zeroed
    counters. `kv4_attention` calls this itself; called by hand on the stream of a capture, before it, it keeps the scratch out of the
    graph's own memory."""
    index = device if isinstance(device, int) else None if device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    stream = torch._C._cuda_getCurrentRawStream(index)  # noqa: SLF001
    ws = _WORKSPACES.get((index, stream))
    if ws is not None:
        return ws
    size, words = ctypes.c_int64(0), ctypes.c_int64(0)
    with torch.cuda.device(index):
        _lib.raise_for_code(_lib.library().b200_kv4_workspace(ctypes.byref(size), ctypes.byref(words)), "kv4 workspace")
        capturing = torch.cuda.is_current_stream_capturing()
        at = torch.device("cuda", index)
        ws = (torch.empty(size.value, dtype=torch.uint8, device=at), torch.zeros(words.value, dtype=torch.int32, device=at))
    if not capturing:
        with _WORKSPACES_LOCK:
            ws = _WORKSPACES.setdefault((index, stream), ws)
    return ws


def reset_counters(index: int) -> None:
    """Zero the counters of a device's workspaces again, which a launch that gave up may have left raised."""
    for (dev, _), (_, counters) in list(_WORKSPACES.items()):
        if dev == index:
            counters.zero_()


def _batch(what: str, name: str, t: torch.Tensor) -> int:
    if t.dim() == 0:
        msg = f"{what}: {name} has no batch dimension"
        raise ValueError(msg)
    return t.shape[0]


def _check_cache(what: str, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, batch: int) -> int:
    """The cache's head dim."""
    if cache.dim() != 4 or cache.dtype != torch.uint8 or not cache.is_cuda or not cache.is_contiguous():  # noqa: PLR2004
        msg = f"{what}: cache must be a contiguous uint8 CUDA tensor of kv4_cache, got {tuple(cache.shape)} {cache.dtype} on {cache.device}"
        raise ValueError(msg)
    dim, rest = divmod(cache.shape[3], BLOCK)
    if rest or dim - 8 not in HEAD_DIMS or cache.numel() == 0:
        msg = f"{what}: a cache of {tuple(cache.shape)} has no head dim of {HEAD_DIMS}"
        raise ValueError(msg)
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != cache.device or page_table.shape[0] != batch or page_table.shape[1] < 1 or page_table.stride(1) != 1:  # noqa: PLR2004
        msg = f"{what}: page_table must be int32 [{batch}, columns] with unit last stride on {cache.device}, got {tuple(page_table.shape)} {page_table.dtype} on {page_table.device}"
        raise ValueError(msg)
    if lengths.shape != (batch,) or lengths.dtype != torch.int32 or lengths.device != cache.device or not lengths.is_contiguous():
        msg = f"{what}: lengths must be contiguous int32 [{batch}] on {cache.device}, got {tuple(lengths.shape)} {lengths.dtype} on {lengths.device}"
        raise ValueError(msg)
    return dim - 8


def _check_heads(what: str, name: str, t: torch.Tensor, cache: torch.Tensor, dim: int, *, like: torch.Tensor | None = None, heads: int | None = None) -> None:
    if t.dim() != 4 or t.dtype not in _DTYPES or t.device != cache.device or t.shape[3] != dim or t.stride(3) != 1:  # noqa: PLR2004
        msg = f"{what}: {name} must be float16 / bfloat16 [batch, tokens, heads, {dim}] with unit last stride on {cache.device}, got {tuple(t.shape)} {t.dtype} on {t.device}"
        raise ValueError(msg)
    if like is not None and (t.dtype != like.dtype or t.shape[:2] != like.shape[:2]):
        msg = f"{what}: {name} {tuple(t.shape)} {t.dtype} does not go with {tuple(like.shape)} {like.dtype}"
        raise ValueError(msg)
    if heads is not None and t.shape[2] != heads:
        msg = f"{what}: {name} has {t.shape[2]} heads, expected {heads}"
        raise ValueError(msg)
    if t.requires_grad and torch.is_grad_enabled():
        msg = f"{what}: {name} requires grad; the 4-bit cache is for inference (use torch.no_grad())"
        raise ValueError(msg)
    refuse_tangent(what, name, t)


def _fill_cache(a: _lib.B200Kv4Args | _lib.B200Kv4AttnArgs, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, dim: int) -> None:
    a.struct_size = ctypes.sizeof(a)
    a.pages, a.kv_heads, blocks, _ = cache.shape
    a.page, a.head_dim, a.table_pages, a.table_stride = blocks * BLOCK, dim, page_table.shape[1], page_table.stride(0)
    a.cache, a.page_table, a.lengths = cache.data_ptr(), page_table.data_ptr(), lengths.data_ptr()


def _set(a: ctypes.Structure, name: str, t: torch.Tensor) -> None:
    setattr(a, name, t.data_ptr())
    getattr(a, f"{name}_stride")[:] = (t.stride(0), t.stride(1), t.stride(2))


def _call(what: str, function: str, a: ctypes.Structure, device: torch.device) -> None:
    with torch.cuda.device(device):
        code = getattr(_lib.library(), function)(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(device.index))  # noqa: SLF001
    _lib.raise_for_code(code, what)
    _lib.use_fast()


def kv4_append_(  # noqa: PLR0913
    cache: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    table: torch.Tensor | None = None,
    interleaved: bool = False,
    q: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Write the last `k.shape[1]` tokens of each sequence into the cache, with k (and q) turned by their positions on the way.

    Token i of `tokens` is at position `lengths[b] - tokens + i`; negative ones are padding on the left and are not written. A head's
    vector of one token is held as 16 levels between its least and its largest value. Sequences must not share the pages that are
    written.

    Args:
        cache: `kv4_cache`, changed in place.
        k: fp16 / bf16 `[batch, tokens, kv_heads, dim]`, unit last stride, other strides multiples of 8, 16-byte aligned (a view of a packed
            qkv tensor).
        v: The same.
        page_table: int32 `[batch, columns]`.
        lengths: int32 `[batch]`, the new tokens included.
        table: `rotary_table` of at least the longest sequence, or None: nothing is turned. A position past it is not turned, and
            `device_status()` reports it, as it does a page outside the cache or the page table (nothing is written for it).
        interleaved: Pairs of neighbouring dimensions instead of halves (`rotary`).
        q: Queries of the same tokens `[batch, tokens, q_heads, dim]`, to be turned in the same launch.
        out: Gets the turned q, may be `q` itself; else a new tensor.

    Returns:
        The turned q, or None without `q`.

    Raises:
        ValueError: Operands outside the contract (checked before the launch).
        KernelUnavailableError: The CUDA library is not built or does not load.
    """
    if out is None and _lib.fast is not None:
        done = _lib.fast.kv4_append_(cache, k, v, page_table, lengths, table, interleaved, q)
        if done is not None:
            return done if q is not None else None
    what = "kv4_append_"
    dim = _check_cache(what, cache, page_table, lengths, _batch(what, "k", k))
    _check_heads(what, "k", k, cache, dim, heads=cache.shape[1])
    _check_heads(what, "v", v, cache, dim, like=k, heads=cache.shape[1])
    if q is not None:
        _check_heads(what, "q", q, cache, dim, like=k)
        if out is not None:
            _check_heads(what, "out", out, cache, dim, like=q, heads=q.shape[2])
    elif out is not None:
        msg = f"{what}: out without q"
        raise ValueError(msg)
    if table is not None and (table.dim() != 3 or table.shape[1] != 2 or 2 * table.shape[2] > dim or table.dtype != torch.float32 or table.device != k.device or table.shape[0] < 1):  # noqa: PLR2004
        msg = f"{what}: table must be float32 [rows, 2, <= {dim // 2}] on {k.device}, got {tuple(table.shape)} {table.dtype} on {table.device}"
        raise ValueError(msg)
    if q is not None and out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k.numel() == 0:
        return out
    a = _lib.B200Kv4Args()
    _fill_cache(a, cache, page_table, lengths, dim)
    a.dtype, a.batch, a.tokens, a.interleaved = _DTYPES[k.dtype], k.shape[0], k.shape[1], interleaved
    if table is not None:
        table = table.contiguous()
        a.rot, a.cs, a.table_rows = 2 * table.shape[2], table.data_ptr(), table.shape[0]
    _set(a, "k", k)
    _set(a, "v", v)
    if q is not None:
        a.q_heads = q.shape[2]
        _set(a, "q", q)
        _set(a, "q_out", out)
    _call(what, "b200_kv4_append", a, k.device)
    return out


def kv4_read(cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, tokens: int, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of the last `tokens` tokens of each sequence as the cache holds them, `[batch, tokens, kv_heads, dim]` of `dtype` each, zeros
    in front of a sequence's start.

    Raises:
        ValueError: Operands outside the contract (checked before the launch).
        KernelUnavailableError: The CUDA library is not built or does not load.
    """
    if _lib.fast is not None:
        done = _lib.fast.kv4_read(cache, page_table, lengths, tokens, dtype is torch.float16 if dtype in _DTYPES else None)
        if done is not None:
            return done
    what = "kv4_read"
    dim = _check_cache(what, cache, page_table, lengths, _batch(what, "lengths", lengths))
    if dtype not in _DTYPES or tokens < 0:
        msg = f"{what}: {tokens} tokens of {dtype}: expected float16 or bfloat16, and no negative count"
        raise ValueError(msg)
    k, v = (torch.empty(lengths.shape[0], tokens, cache.shape[1], dim, dtype=dtype, device=cache.device) for _ in range(2))
    if k.numel() == 0:
        return k, v
    a = _lib.B200Kv4Args()
    _fill_cache(a, cache, page_table, lengths, dim)
    a.dtype, a.batch, a.tokens = _DTYPES[dtype], lengths.shape[0], tokens
    _set(a, "k_out", k)
    _set(a, "v_out", v)
    _call(what, "b200_kv4_read", a, cache.device)
    return k, v


def kv4_attention(  # noqa: PLR0913
    q: torch.Tensor,
    cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    scale: float | None = None,
    *,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of the last `q.shape[1]` tokens of each sequence over the cache: `[batch, queries, q_heads, dim]`.

    Query i is at position `lengths[b] - queries + i` and sees the keys up to its own; a query in front of the sequence's start sees none
    and gets zeros, one that sees a key on a page outside the cache gets NaN (and `device_status()` reports it). The lengths are read on the device: work is dealt by them in equal runs of steps, and a captured graph
    follows them. (Steps that a tile of rows does not see count in a run too: a prompt whose queries are its whole sequence is dealt unevenly, the
    busiest part of the GPU has about twice the mean.) Accumulation and softmax are fp32.

    Args:
        q: fp16 / bf16 `[batch, queries, q_heads, dim]`, already turned; q_heads a multiple of the cache's kv heads, consecutive ones
            sharing a kv head; unit last stride, other strides multiples of 8, 16-byte aligned.
        cache: `kv4_cache`, with the queries' own tokens in it.
        page_table: int32 `[batch, columns]`.
        lengths: int32 `[batch]`.
        scale: Factor of the logits, positive, default `dim ** -0.5`.
        out: Gets the result; else a new tensor.

    Raises:
        ValueError: Operands outside the contract (checked before the launch).
        KernelUnavailableError: The CUDA library is not built or does not load.
    """
    if out is None and _lib.fast is not None:
        done = _lib.fast.kv4_attention(q, cache, page_table, lengths, scale)
        if done is not None:
            return done
    what = "kv4_attention"
    dim = _check_cache(what, cache, page_table, lengths, _batch(what, "q", q))
    _check_heads(what, "q", q, cache, dim)
    if q.shape[2] == 0 or q.shape[2] % cache.shape[1]:
        msg = f"{what}: {q.shape[2]} q heads are no multiple of {cache.shape[1]} kv heads"
        raise ValueError(msg)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_heads(what, "out", out, cache, dim, like=q, heads=q.shape[2])
    if q.numel() == 0:
        return out
    a = _lib.B200Kv4AttnArgs()
    _fill_cache(a, cache, page_table, lengths, dim)
    a.dtype, a.batch, a.queries, a.q_heads = _DTYPES[q.dtype], q.shape[0], q.shape[1], q.shape[2]
    a.scale = dim**-0.5 if scale is None else scale
    _set(a, "q", q)
    _set(a, "o", out)
    work, counters = reserve_kv4_workspace(q.device.index)
    a.workspace, a.workspace_bytes, a.counters, a.counter_words = work.data_ptr(), work.numel(), counters.data_ptr(), counters.numel()
    _call(what, "b200_kv4_attention", a, q.device)
    if _lib.fast is not None and (q.device.index, stream := torch._C._cuda_getCurrentRawStream(q.device.index)) in _WORKSPACES:  # noqa: SLF001
        _lib.fast.register_kv4_workspace(q.device.index, stream, work.data_ptr(), work.numel(), counters.data_ptr(), counters.numel())
    return out

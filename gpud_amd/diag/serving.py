"""Operators of one token step of a served language model, on MI355X.

The diagnostics in ``_diag`` drive the matrix units, LDS and HBM with regular
streams. These operators drive the card as a serving job does: 4- and 8-bit
decoding, bytes gathered by page tables, exp and log units, wave reductions
and joins of split work. ``accelerator-amd-diag-serving`` runs them as one
step against a host oracle; here they take a program's own tensors.

* :func:`w4_matmul` - product with 4-bit weights and group scales
* :func:`cache_append` - new keys and values into an 8-bit paged cache
* :func:`cache_attention` - attention over that cache
* :func:`token_logprobs` - log probabilities of given tokens, with entropy,
  rank and the top alternatives

All work is enqueued on the current stream of the tensors' device; these four
never wait for the GPU, and results do not depend on timing. Each may be
captured into a graph: workspaces are allocated per call from torch's
allocator, so two graphs share none. (:func:`pack_w4` waits for its checks.) Arguments that do not fit raise
``TypeError`` or ``ValueError`` before anything is enqueued. Page numbers,
lengths and tokens that live on the GPU are bounded there: see each function.
Tensors that have a shape but no memory (freed storages, fake tensors, wrapper
subclasses) are among those. The operators have no backward pass and no forward
mode: they refuse inputs that require a gradient while gradients are recorded,
and inputs with a tangent.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _serving

__all__ = [
    "TokenLogprobs",
    "cache_append",
    "cache_attention",
    "cache_scale",
    "new_cache",
    "pack_w4",
    "token_logprobs",
    "unpack_w4",
    "w4_matmul",
]

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_HALVES = {torch.bfloat16: 0, torch.float16: 1}
F8 = torch.float8_e4m3fn
_CODES = (F8, torch.uint8)
_INT_MAX = 2**31 - 1
_MOST = 2**30  # positions of a sequence
# A launch has fewer than 2^32 threads in all; these sizes stay under it.
_MOST_FEATURES = 2**26
_MOST_PRODUCTS = 2**33
_MOST_HEADS = 2**22  # heads of all sequences
_MOST_HEAD_ROWS = 2**26  # (row, head) pairs
_MOST_LOGIT_ROWS = 2**24 - 1
_MOST_SCALE = torch.finfo(torch.float32).max

GROUPS = (32, 64, 128)
MAX_COLUMNS = _serving.MAX_COLUMNS
MAX_TOKENS = _serving.MAX_TOKENS
MAX_TOP = _serving.MAX_TOP
MAX_VOCAB = _serving.MAX_VOCAB
MAX_HEAD_DIM = 256


_stream = torch._C._cuda_getCurrentRawStream  # of a device number


def _fits(t, device: int, dtype, shape) -> bool:
    """Whether a contiguous tensor is what a call needs; the checks below say why not."""
    return (
        type(t) is torch.Tensor
        and t.dtype is dtype
        and t.get_device() == device
        and t.shape == shape
        and t.is_contiguous()
        and not t.requires_grad
    )


def _primary(name: str, t, dim: int, dtypes) -> int:
    """The native number of the type of a call's first tensor, which has to be in `dtypes`."""
    if type(t) is not torch.Tensor or t.dtype not in dtypes or t.dim() != dim or t.requires_grad:
        _check_input(name, t, None, tuple(dtypes), dim)
    return dtypes[t.dtype]


def _check_input(name: str, t: torch.Tensor, device: Optional[torch.device], dtypes, dim: int) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, not {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}; expected one of {', '.join(str(d) for d in dtypes)}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, not {t.dim()}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and the operator has no backward pass")


def _check_gpu(device: torch.device) -> None:
    if device.type != "cuda":
        raise ValueError(f"the tensors must be on a GPU, not on {device}")


def _refuse_tangents(**tensors) -> None:
    """Forward mode marks a tensor by its tangent alone; it would be dropped without a word."""
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} has a tangent, and the operator has no forward mode")


def _memory(name: str, t: torch.Tensor) -> int:
    """The address of a tensor that may be missing: 0 has to mean that it is."""
    at = t.data_ptr()
    if not at:
        raise ValueError(f"{name} has no memory")
    return at


def _check_shape(name: str, t: torch.Tensor, shape: Tuple[int, ...]) -> None:
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}; expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


# ---------------------------------------------------------------------------
# product with 4-bit weights
# ---------------------------------------------------------------------------


def pack_w4(
    codes: torch.Tensor,
    scales: torch.Tensor,
    zeros: Optional[torch.Tensor] = None,
    *,
    group_size: int = 128,
) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Lays 4-bit weights out for :func:`w4_matmul`, once.

    ``codes`` is [N, K] with values 0..15, ``scales`` (bf16 or fp16) and
    ``zeros`` (whole numbers 0..15) are [N, ceil(K / group_size)]. Returns the
    packed codes uint8 [ceil(N/16), ceil(K/128), 64, 16], and scales and zeros
    as [ceil(N/16), groups, 16].

    A tile holds rows 16n..16n+15 and columns 128b..128b+127. Lane 16g+r has
    row r; its dword j has the columns 32j + 8g + e, with e = 2 (i mod 4) +
    i // 4 in nibble i.
    """
    if group_size not in GROUPS:
        raise ValueError(f"group_size must be one of {GROUPS}, not {group_size}")
    if codes.dim() != 2 or codes.is_floating_point():
        raise ValueError("codes must be whole numbers of shape [N, K]")
    n, k = codes.shape
    if n < 1 or k < 1:
        raise ValueError("codes must not be empty")
    groups = -(-k // group_size)
    if tuple(scales.shape) != (n, groups):
        raise ValueError(f"scales has shape {tuple(scales.shape)}; expected {(n, groups)}")
    if zeros is not None and tuple(zeros.shape) != (n, groups):
        raise ValueError(f"zeros has shape {tuple(zeros.shape)}; expected {(n, groups)}")
    if zeros is not None and not torch.equal(zeros, zeros.round() if zeros.is_floating_point() else zeros):
        raise ValueError("zeros must be whole numbers")
    for name, t in (("codes", codes), ("zeros", zeros)):
        if t is not None and (int(t.min()) < 0 or int(t.max()) > 15):
            raise ValueError(f"{name} must be in 0..15")
    tiles, blocks = -(-n // 16), -(-k // 128)
    full = torch.zeros(tiles * 16, blocks * 128, dtype=torch.uint8, device=codes.device)
    full[:n, :k] = codes.to(torch.uint8)
    # tile, row, block, j, g, i mod 4, i // 4
    full = full.view(tiles, 16, blocks, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5)
    full = full.reshape(tiles, blocks, 64, 16, 2)
    packed = full[..., 0] | full[..., 1] << 4

    def tile(t: torch.Tensor) -> torch.Tensor:
        pad = torch.zeros(tiles * 16, groups, dtype=t.dtype, device=t.device)
        pad[:n] = t
        return pad.view(tiles, 16, groups).transpose(1, 2).contiguous()

    return packed, tile(scales), None if zeros is None else tile(zeros.to(torch.uint8))


def unpack_w4(packed: torch.Tensor, out_features: int, in_features: int) -> torch.Tensor:
    """The codes [N, K] (uint8) that :func:`pack_w4` laid out."""
    _check_input("packed", packed, None, (torch.uint8,), 4)
    tiles, blocks = -(-out_features // 16), -(-in_features // 128)
    _check_shape("packed", packed, (tiles, blocks, 64, 16))
    nibbles = torch.stack((packed & 15, packed >> 4), -1).view(tiles, blocks, 4, 16, 4, 2, 4)
    full = nibbles.permute(0, 3, 1, 4, 2, 6, 5).reshape(tiles * 16, blocks * 128)
    return full[:out_features, :in_features].contiguous()


def w4_matmul(
    x: torch.Tensor,
    codes: torch.Tensor,
    scales: torch.Tensor,
    zeros: Optional[torch.Tensor] = None,
    *,
    out_features: int,
    group_size: int = 128,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """y[m, n] = sum_k x[m, k] (q[n, k] - z[n, k // G]) s[n, k // G].

    ``x`` is [M, K] in bf16 or fp16, its rows at any stride; ``codes``,
    ``scales`` (x's type) and ``zeros`` are as :func:`pack_w4` lays them out
    (no zeros: every zero point is 8). Meant for the tokens of a decode batch,
    M up to 64; larger M, up to ``MAX_TOKENS``, are taken 64 rows at a time.
    K is at most ``MAX_COLUMNS``, N 2^26 and M N 2^33. ``out`` may not share
    memory with the other arguments.
    Sums are fp32, rounded once to x's type. ``x`` has to be finite, and under
    2^115 (4e34) in magnitude: a group's sum is formed from x times whole numbers
    up to 31 and comes to 2^12 times the largest x on its way.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents(x=x, scales=scales, out=out)
    dtype = _primary("x", x, 2, _HALVES)
    m, k = x.shape
    n = int(out_features)
    if group_size not in GROUPS:
        raise ValueError(f"group_size must be one of {GROUPS}, not {group_size}")
    if k < 1 or n < 1 or k > MAX_COLUMNS or n > _MOST_FEATURES or m > MAX_TOKENS or m * n > _MOST_PRODUCTS:
        raise ValueError(f"no product of {m} rows with weights [{n}, {k}]")
    tiles, groups = -(-n // 16), -(-k // group_size)
    at, device = x.get_device(), x.device
    if not _fits(codes, at, torch.uint8, (tiles, -(-k // 128), 64, 16)):
        _check_input("codes", codes, device, (torch.uint8,), 4)
        _check_shape("codes", codes, (tiles, -(-k // 128), 64, 16))
    if not _fits(scales, at, x.dtype, (tiles, groups, 16)):
        _check_input("scales", scales, device, (x.dtype,), 3)
        _check_shape("scales", scales, (tiles, groups, 16))
    if zeros is not None and not _fits(zeros, at, torch.uint8, (tiles, groups, 16)):
        _check_input("zeros", zeros, device, (torch.uint8,), 3)
        _check_shape("zeros", zeros, (tiles, groups, 16))
    zp = 0 if zeros is None else _memory("zeros", zeros)
    if codes.data_ptr() % 16 or scales.data_ptr() % 8 or zp % 4:
        raise ValueError("codes, scales and zeros must be aligned to 16, 8 and 4 bytes")
    if out is None:
        _check_gpu(device)
        out = x.new_empty((m, n))
    else:
        _check_input("out", out, device, (x.dtype,), 2)
        if tuple(out.shape) != (m, n) or (out.stride(1) != 1 and n > 1):
            raise ValueError(f"out must be [{m}, {n}] with dense rows")
        if m > 1 and out.stride(0) < n:
            raise ValueError("rows of out overlap")
        _check_gpu(device)
    if x.stride(1) != 1 and k > 1:
        x = x.contiguous()
    if m:
        args = (x.data_ptr(), x.stride(0), m, n, k, group_size, dtype)
        size = _serving.w4_workspace(*args)
        work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _serving.w4_matmul(
            *args, codes.data_ptr(), scales.data_ptr(), zp,
            out.data_ptr(), out.stride(0), work.data_ptr() if size else 0, at, _stream(at),
        )
    return out


# ---------------------------------------------------------------------------
# 8-bit paged cache
# ---------------------------------------------------------------------------


def cache_scale(amax: torch.Tensor) -> torch.Tensor:
    """The scale of a page whose largest magnitude is ``amax`` (float32).

    The smallest power of two that brings it within 448, at least 2^-64.
    """
    bits = amax.float().contiguous().view(torch.int32)
    return torch.exp2(((bits + 0x1FFFFF >> 23) - 135).clamp_min(-64).float())


def new_cache(
    pages: int, heads: int, head_dim: int, page_size: int = 64, *, device="cuda"
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """An empty cache: (keys, values, key scales, value scales).

    Keys are float8_e4m3fn [pages, heads, page_size, head_dim], values
    [pages, heads, head_dim, page_size] (a token's values are a column, as the
    attention takes them), scales float32 [pages, heads].
    """
    _check_cache_sizes(pages, heads, page_size, head_dim)

    def codes(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)

    k, v = codes(pages, heads, page_size, head_dim), codes(pages, heads, head_dim, page_size)
    scales = [torch.full((pages, heads), 2.0**-64, device=device) for _ in range(2)]
    return k, v, scales[0], scales[1]


def _check_cache_sizes(pages: int, heads: int, page: int, dim: int) -> None:
    if pages < 1 or heads < 1 or pages > _INT_MAX or heads > 65535:
        raise ValueError(f"no cache of {pages} pages and {heads} heads")
    if page < 16 or page > 4096 or page & (page - 1):
        raise ValueError(f"page size must be a power of two in 16..4096, not {page}")
    if dim < 16 or dim % 16 or dim > MAX_HEAD_DIM:
        raise ValueError(f"head dimension must be a multiple of 16 up to {MAX_HEAD_DIM}, not {dim}")


def _cache_args(k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start, device, at, rows):
    if type(k_cache) is not torch.Tensor or k_cache.dim() != 4 or not _fits(k_cache, at, F8, k_cache.shape):
        _check_input("k_cache", k_cache, device, _CODES, 4)
        if not k_cache.is_contiguous():
            raise ValueError("k_cache must be contiguous")
    pages, heads, page, dim = k_cache.shape
    _check_cache_sizes(pages, heads, page, dim)
    if not _fits(v_cache, at, k_cache.dtype, (pages, heads, dim, page)):
        _check_input("v_cache", v_cache, device, _CODES, 4)
        _check_shape("v_cache", v_cache, (pages, heads, dim, page))
    if not _fits(k_scale, at, torch.float32, (pages, heads)):
        _check_input("k_scale", k_scale, device, (torch.float32,), 2)
        _check_shape("k_scale", k_scale, (pages, heads))
    if not _fits(v_scale, at, torch.float32, (pages, heads)):
        _check_input("v_scale", v_scale, device, (torch.float32,), 2)
        _check_shape("v_scale", v_scale, (pages, heads))
    if type(block_table) is not torch.Tensor or block_table.dim() != 2 or not _fits(block_table, at, torch.int32, block_table.shape):
        _check_input("block_table", block_table, device, (torch.int32,), 2)
        if block_table.shape[1] > 1 and block_table.stride(1) != 1:
            raise ValueError("rows of block_table must be dense")
    batch, blocks = block_table.shape
    if not _fits(seq_lens, at, torch.int32, (batch,)):
        _check_input("seq_lens", seq_lens, device, (torch.int32,), 1)
        _check_shape("seq_lens", seq_lens, (batch,))
    if blocks * page > _MOST or batch * heads > _MOST_HEADS:
        raise ValueError("block_table covers more than 2^30 positions, or more than 2^22 heads of sequences")
    starts = 0
    if query_start is None:
        if rows != batch:
            raise ValueError(f"{rows} rows for {batch} sequences: give query_start, or one row for each sequence")
    else:
        if not _fits(query_start, at, torch.int32, (batch + 1,)):
            _check_input("query_start", query_start, device, (torch.int32,), 1)
            _check_shape("query_start", query_start, (batch + 1,))
        starts = _memory("query_start", query_start)
    kp, vp = k_cache.data_ptr(), v_cache.data_ptr()
    if kp % 16 or vp % 16:
        raise ValueError("k_cache and v_cache must be aligned to 16 bytes")
    return (
        kp, vp, k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), starts,
        block_table.stride(0), pages, heads, page, dim, batch, blocks, rows,
    )


def cache_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start: Optional[torch.Tensor] = None,
) -> None:
    """Writes new keys and values [T, heads, dim] (bf16 or fp16) into the cache.

    Sequence b's new tokens are rows ``query_start[b] .. query_start[b+1]``
    (int32 [B+1], from 0 and never falling), or row b alone without
    ``query_start``; they become its last ones, and ``seq_lens`` (int32 [B])
    counts them in. ``block_table``
    (int32 [B, blocks]) names the page of each ``page_size`` positions. Rows
    may lie at any row and head stride.

    A page's scale is :func:`cache_scale` of what it holds; where tokens go
    behind ones that it holds already it only grows, and those are rounded
    again to it. A page whose first position is written starts afresh.
    Infinities are held as the largest code, NaN as NaN. Tokens whose page is
    out of range, or whose position is negative, are left out. A page that gets
    tokens may stand in the table once only.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents(k=k, v=v, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale)
    dtype = _primary("k", k, 3, _HALVES)
    device, at = k.device, k.get_device()
    _check_input("v", v, device, (k.dtype,), 3)
    rows = k.shape[0]
    cache = _cache_args(k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start, device, at, rows)
    heads, dim, batch = cache[9], cache[11], cache[12]
    if k.shape != (rows, heads, dim) or v.shape != (rows, heads, dim):
        raise ValueError(f"k and v must be [T, {heads}, {dim}], not {tuple(k.shape)} and {tuple(v.shape)}")
    if rows * heads > _MOST_HEAD_ROWS:
        raise ValueError("more than 2^26 new keys")
    _check_gpu(device)
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    if rows and batch:
        _serving.cache_append(
            *cache, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
            dtype, at, _stream(at),
        )


def cache_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start: Optional[torch.Tensor] = None,
    *,
    max_seq_len: Optional[int] = None,
    scale: Optional[float] = None,
    window: Optional[int] = None,
    out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of ``q`` [T, q_heads, dim] (bf16 or fp16) over the cache.

    The arguments of :func:`cache_append` name the sequences; a sequence's
    rows are its last tokens, whose keys and values the cache holds already.
    A row at position p sees the positions up to p, with ``window`` only the
    last ``window`` of them. ``q_heads`` is a multiple of the cache's heads.
    ``scale``, over 0 and finite in float32, is dim ** -0.5 unless given.
    ``max_seq_len``, the longest length as far as the program knows it, only
    steers how work is split.

    Returns (out [T, q_heads, dim] in q's type, lse float32 [T, q_heads]), lse
    the logarithm of the sum of the exponentials of a row's scores. The scales
    of pages that a row sees have to be positive and finite; others may hold
    anything. The value scales of a sequence's head may differ by a factor of
    2^100, which values under 2^44 (1e13) never pass, beside zeros either; queries
    are under 2^110 (1e33) in magnitude. Beyond that fp32 does not hold a row's
    sums. A row that sees nothing gets 0 and -inf. A sequence whose pages are out
    of range, or that is longer than its row of ``block_table``, gets NaN. Rows behind the
    last sequence are left as they were in ``out`` if that is given, and else
    0; their lse is -inf. ``out`` may not share memory with the other arguments.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents(q=q, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, out=out)
    dtype = _primary("q", q, 3, _HALVES)
    device, at = q.device, q.get_device()
    rows, q_heads, dim = q.shape
    cache = _cache_args(k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start, device, at, rows)
    heads, batch = cache[9], cache[12]
    if dim != cache[11]:
        raise ValueError(f"q has head dimension {dim}, the cache {cache[11]}")
    if q_heads < 1 or q_heads % heads or q_heads > 65535:
        raise ValueError(f"{q_heads} query heads do not share {heads} cached ones evenly")
    if rows * q_heads > _MOST_HEAD_ROWS or batch * q_heads > _MOST_HEAD_ROWS:
        raise ValueError("more than 2^26 query rows")
    if scale is None:
        scale = dim**-0.5
    elif not 0 < scale <= _MOST_SCALE:
        raise ValueError(f"scale must be positive, and finite in float32, not {scale}")
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, not {window}")
    room = cache[13] * cache[10]
    max_seq_len = room if max_seq_len is None else min(max_seq_len, room)
    fill = out is None
    if not fill:
        _check_input("out", out, device, (q.dtype,), 3)
        _check_shape("out", out, (rows, q_heads, dim))
        if out.data_ptr() % 8:
            raise ValueError("out must be aligned to 8 bytes")
    _check_gpu(device)
    # 16-byte loads of the queries
    row, head, one = q.stride()
    if one != 1 or row % 8 or head % 8 or q.data_ptr() % 16:
        row, head = q_heads * dim, dim
        q = q.clone(memory_format=torch.contiguous_format)
    if fill:
        out = q.new_empty((rows, q_heads, dim))
    lse = torch.empty(rows, q_heads, dtype=torch.float32, device=device)
    if not rows:
        return out, lse
    if not batch:
        if fill:
            out.zero_()
        lse.fill_(-math.inf)
        return out, lse
    window = min(window, _MOST) if window else 0
    floats = _serving.attention_workspace(
        rows, batch, heads, q_heads, dim, query_start is not None, window, max_seq_len
    )
    work = torch.empty(floats, dtype=torch.float32, device=device) if floats else None
    _serving.cache_attention(
        *cache, q.data_ptr(), row, head, out.data_ptr(), q_heads * dim, dim, lse.data_ptr(),
        work.data_ptr() if floats else 0,
        q_heads, window, max_seq_len, fill, scale, dtype, at, _stream(at),
    )
    return out, lse


# ---------------------------------------------------------------------------
# log probabilities of given tokens
# ---------------------------------------------------------------------------


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor  # float32 [R]
    entropy: torch.Tensor  # float32 [R], in nats
    rank: torch.Tensor  # int64 [R]: tokens whose logit is larger
    top_ids: Optional[torch.Tensor]  # int64 [R, k]
    top_logprobs: Optional[torch.Tensor]  # float32 [R, k]


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Of each row of ``logits`` [R, V]: its given token's log probability, the
    distribution's entropy, the given token's rank, and the ``top_k`` likeliest
    tokens with theirs, ties by the lower index.

    ``logits`` is bf16, fp16 or fp32, its rows at any stride; ``targets`` is
    int64 [R]. A negative target is padding: log probability 0, rank -1. One of
    V or more gets NaN and rank -1. Logits of -inf are tokens that are not
    allowed; a row that allows none has entropy 0 and log probabilities -inf. A
    row with NaN or +inf has NaN as its log probability and entropy; NaN comes
    first among its alternatives.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents(logits=logits)
    dtype = _primary("logits", logits, 2, _DTYPES)
    device, at = logits.device, logits.get_device()
    rows, vocab = logits.shape
    if rows > _MOST_LOGIT_ROWS:
        raise ValueError("more than 2^24 - 1 rows")
    if not _fits(targets, at, torch.int64, (rows,)):
        _check_input("targets", targets, device, (torch.int64,), 1)
        if targets.shape[0] != rows:
            raise ValueError(f"{targets.shape[0]} targets for {rows} rows")
        targets = targets.contiguous()
    if vocab < 1 or vocab > MAX_VOCAB:
        raise ValueError(f"vocabulary must have 1..{MAX_VOCAB} tokens, not {vocab}")
    if top_k < 0 or top_k > min(MAX_TOP, vocab):
        raise ValueError(f"top_k must be in 0..{min(MAX_TOP, vocab)}, not {top_k}")
    _check_gpu(device)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    logprob = torch.empty(rows, dtype=torch.float32, device=device)
    entropy = logprob.new_empty(rows)
    rank = targets.new_empty(rows)
    top_ids = top_logprobs = None
    if top_k:
        top_ids, top_logprobs = rank.new_empty((rows, top_k)), logprob.new_empty((rows, top_k))
    if rows:
        floats = _serving.logprob_workspace(rows, vocab, dtype)
        work = logprob.new_empty(floats) if floats else None
        _serving.token_logprobs(
            logits.data_ptr(), logits.stride(0), targets.data_ptr(), logprob.data_ptr(), entropy.data_ptr(),
            rank.data_ptr(), top_ids.data_ptr() if top_k else 0, top_logprobs.data_ptr() if top_k else 0,
            work.data_ptr() if floats else 0, rows, vocab, top_k, dtype, at, _stream(at),
        )
    return TokenLogprobs(logprob, entropy, rank, top_ids, top_logprobs)

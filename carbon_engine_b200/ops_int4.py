"""Operators of a model held in 4 bits: keys and values quantised into the pages of a cache and read back, attention over
such a cache, and products of a few tokens with 4-bit weights.

The format (``csrc/kernels/int4.cuh`` has its layout): ``group`` neighbouring values share a minimum z and a step s, both float16; a
value is c s + z with a code c of 0 .. 15, z = float16(min x), s = float16((max x - z) / 15) (as a product with the float32 next to 1/15), c = (x - z) / s rounded to the nearest.
A group that holds a value beyond 60,000 in magnitude, or one that is not finite, reads back as NaN.

Like :mod:`carbon_engine_b200.ops`, every function takes tensors on the GPU, checks them, and launches on the current stream of the
tensors' device, which has to be the current one; scratch memory comes from torch's allocator at each call, so calls on several streams and captured graphs share none.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import ops
from .csrc import kernel_lib
from .csrc.kernel_lib import KernelError, kernels

_i, _f, _ll, _p = ctypes.c_int, ctypes.c_float, ctypes.c_longlong, ctypes.c_void_p
kernel_lib.declare("ce_int4_cache_tile_bytes", _i, [_i, _i])
kernel_lib.declare("ce_int4_weight_tile_bytes", _i, [_i])
# dtype, k, v, strides of k and v (token, head), pages, positions, seq_of_token, seq_slot, block_table, status,
# T, nkv, d, group, page_size, max_pages, num_pages, stream
_kv = [_i, _p, _p] + [_ll] * 4 + [_p] * 6 + [_i] * 7 + [_p]
kernel_lib.declare("ce_int4_kv_write", _i, _kv)
kernel_lib.declare("ce_int4_kv_read", _i, _kv)
# dtype, w, ld, tiles, rows, part, width, group, stream
kernel_lib.declare("ce_int4_quantise_weight", _i, [_i, _p, _ll, _p, _i, _i, _i, _i, _p])
kernel_lib.declare("ce_int4_dequantise_weight", _i, [_i, _p, _ll, _p, _i, _i, _i, _i, _p])
# each, d, tile
kernel_lib.declare("ce_int4_attention_rows", _i, [_i] * 3)
kernel_lib.declare("ce_int4_attention_blocks", _i, [_i] * 3)
# dtype, q, q_stride, pages, out, seq_slot, q_start, ctx_len, block_table, tiles, status, part_o, part_ml, count, nh, nkv, d, group,
# page_size, max_pages, num_pages, window, splits, scale, stream
kernel_lib.declare("ce_int4_attention", _i, [_i, _p, _ll] + [_p] * 10 + [_i] * 10 + [_f, _p])
# dtype, M, K, group
kernel_lib.declare("ce_int4_gemm_scratch", _ll, [_i] * 4)
# dtype, x, ldx, w, out, ldo, M, N, K, group, mode, scratch, stream
kernel_lib.declare("ce_int4_gemm", _i, [_i, _p, _ll, _p, _p] + [_i] * 6 + [_p, _p])

HEAD_SIZES = (64, 128, 192, 256)
CACHE_GROUPS = (32, 64)
WEIGHT_GROUPS = (32, 64, 128)
#: tokens a product with a 4-bit weight takes
MAX_TOKENS = 64
#: keys of a tile of the cache: page sizes are multiples of it
TILE_TOKENS = 16


def _same_device(first: torch.Tensor, *others) -> None:
    if first.device.index != torch.cuda.current_device():
        raise KernelError(f"the tensors are on {first.device}, but the current device is cuda:{torch.cuda.current_device()}")
    for t in others:
        if t is not None and t.device != first.device:
            raise KernelError(f"tensors on {first.device} and {t.device} in one call")


def cache_problem(head_dim: int, group: int, page_size: int) -> Optional[str]:
    """Why a 4-bit cache cannot have these sizes, or None."""
    if head_dim not in HEAD_SIZES:
        return f"head size {head_dim} (a 4-bit cache takes {', '.join(map(str, HEAD_SIZES))})"
    if group not in CACHE_GROUPS:
        return f"group {group} (a 4-bit cache takes {' or '.join(map(str, CACHE_GROUPS))})"
    if page_size < TILE_TOKENS or page_size % TILE_TOKENS:
        return f"page size {page_size} (a 4-bit cache takes multiples of {TILE_TOKENS})"
    return None


def cache_bytes_per_token(kv_heads: int, head_dim: int, group: int) -> int:
    """Bytes a token's keys and values take."""
    return kv_heads * (head_dim + 8 * (head_dim // group))


class Int4Pages:
    """Pages of keys and values in 4 bits: what ``k_pool`` and ``v_pool`` are to a 16-bit cache.  ``data`` [num_pages, kv_heads,
    page_size / 16, bytes of a tile]; a page's bytes are those of its tokens alone, so pages can be handed on and copied."""

    def __init__(self, num_pages: int, kv_heads: int, page_size: int, head_dim: int, group: int = 64, device="cuda",
                 poison: bool = False):
        """``poison``: pages start as NaN instead of zeros, so that what was never written shows when it is read."""
        problem = cache_problem(head_dim, group, page_size)
        if problem:
            raise KernelError(problem)
        if num_pages < 1 or kv_heads < 1:
            raise KernelError(f"{num_pages} pages of {kv_heads} heads")
        self.num_pages, self.kv_heads, self.page_size = int(num_pages), int(kv_heads), int(page_size)
        self.head_dim, self.group = int(head_dim), int(group)
        tile = (16 * head_dim + 128 * (head_dim // group))
        self.data = torch.empty((num_pages, kv_heads, page_size // TILE_TOKENS, tile), dtype=torch.uint8, device=device)
        self.data.fill_(255 if poison else 0)           # (two bytes of 255 are a float16 NaN)

    def element_size(self) -> float:
        """Bytes a key or value takes, steps and minima included."""
        return 0.5 + 4.0 / self.group


def _rows(t: torch.Tensor, name: str, pages: Int4Pages, tokens: int, dtype=None) -> None:
    if not t.is_cuda:
        raise KernelError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dim() != 3 or t.shape != (tokens, pages.kv_heads, pages.head_dim):
        raise KernelError(f"{name} is {tuple(t.shape)}, not {(tokens, pages.kv_heads, pages.head_dim)}")
    if t.numel() and t.stride(2) != 1:
        raise KernelError(f"{name}: the channels of a head must lie together")
    if dtype is not None and t.dtype != dtype:
        raise KernelError(f"{name} must be {dtype}, got {t.dtype}")


def _kv_call(fn, k, v, pages, positions, seq_of_token, seq_slot, block_table, status) -> None:
    T = positions.numel()
    _rows(k, "k", pages, T)
    _rows(v, "v", pages, T, k.dtype)
    for name, t in (("positions", positions), ("seq_of_token", seq_of_token), ("seq_slot", seq_slot), ("block_table", block_table),
                    ("status", status)):
        ops._need(t, name, torch.int32)
    if seq_of_token.numel() != T or block_table.dim() != 2:
        raise KernelError("one position and one sequence a token, and a table of [slots, pages]")
    code = ops.dtype_code(k.dtype)
    _same_device(k, v, pages.data, positions, seq_of_token, seq_slot, block_table, status)
    if T == 0:
        return
    prof = ops.profiling()
    if prof is not None:
        n = 2 * T * pages.kv_heads * pages.head_dim
        prof.note_work(int(n * (k.element_size() + pages.element_size())), 0)
    ops._ok(fn(code, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), pages.data.data_ptr(),
               positions.data_ptr(), seq_of_token.data_ptr(), seq_slot.data_ptr(), block_table.data_ptr(), status.data_ptr(), T,
               pages.kv_heads, pages.head_dim, pages.group, pages.page_size, block_table.shape[1], pages.num_pages, ops._stream()))


def kv_write(pages: Int4Pages, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, seq_of_token: torch.Tensor,
             seq_slot: torch.Tensor, block_table: torch.Tensor, status: torch.Tensor) -> None:
    """Quantise the keys and values of T tokens into the pages: token t of sequence ``seq_of_token[t]`` (its table row
    ``seq_slot`` of that) goes to position ``positions[t]``.  ``k``, ``v`` [T, kv_heads, head_dim] bfloat16 or float32, tokens and heads at any stride (the columns of a step's
    projection, for instance).  No two tokens of a call may have the same place.  ``status`` becomes 2 where a token's page is not held; its row is dropped then."""
    _kv_call(kernels().ce_int4_kv_write, k, v, pages, positions, seq_of_token, seq_slot, block_table, status)


def kv_read(pages: Int4Pages, k_out: torch.Tensor, v_out: torch.Tensor, positions: torch.Tensor, seq_of_token: torch.Tensor,
            seq_slot: torch.Tensor, block_table: torch.Tensor, status: torch.Tensor) -> None:
    """Read back what T places hold, as :func:`kv_write` names them, rounded once to the outputs' type.  ``status`` becomes 4 where a
    place's page is not held; its rows stay as they were."""
    _kv_call(kernels().ce_int4_kv_read, k_out, v_out, pages, positions, seq_of_token, seq_slot, block_table, status)


def _splits(jobs: int, max_ctx: int, window: int, tokens: int) -> int:
    """Blocks that share a sequence's keys: enough to fill the chip twice, but two tiles of 16 keys a warp at least."""
    keys = min(max_ctx, window + tokens) if window > 0 else max_ctx
    most = max(1, (keys + 255) // 256)
    return max(1, min(most, 64, (2 * 148 + jobs - 1) // jobs))


def _attend(q, pages, out, seq_slot, q_start, ctx_len, block_table, status, tiles, count, max_ctx, window, scale) -> None:
    k = kernels()
    heads = q.shape[1]
    each = heads // pages.kv_heads
    tile = 0 if tiles is None else 1
    jobs = count * pages.kv_heads * k.ce_int4_attention_blocks(each, pages.head_dim, tile)
    splits = _splits(jobs, max_ctx, window, 64 if tile else 1)
    part_o = part_ml = None
    if splits > 1:
        rows = jobs * splits * k.ce_int4_attention_rows(each, pages.head_dim, tile)
        part_o = torch.empty(rows * pages.head_dim, dtype=torch.float32, device=q.device)
        part_ml = torch.empty(rows * 2, dtype=torch.float32, device=q.device)
    ops._ok(k.ce_int4_attention(
        ops.dtype_code(q.dtype), q.data_ptr(), q.stride(0), pages.data.data_ptr(), out.data_ptr(), seq_slot.data_ptr(), q_start.data_ptr(),
        ctx_len.data_ptr(), block_table.data_ptr(), ops._ptr(tiles), status.data_ptr(), ops._ptr(part_o), ops._ptr(part_ml), count, heads,
        pages.kv_heads, pages.head_dim, pages.group, pages.page_size, block_table.shape[1], pages.num_pages, window, splits, scale,
        ops._stream()), 2 if splits > 1 else 1)


def attention(q: torch.Tensor, pages: Int4Pages, out: torch.Tensor, seq_slot: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor,
              block_table: torch.Tensor, status: torch.Tensor, *, n_decode: int, max_ctx: int, tiles: Optional[torch.Tensor] = None,
              n_tiles: Optional[int] = None, window: int = 0, scale: float = 1.0) -> None:
    """Causal attention of a step's queries over the pages, which hold the step's own keys and values already.

    ``q`` [T, heads, head_dim] (tokens at any stride, the heads of a token together), ``out`` [T, heads, head_dim] contiguous; sequence b has
    the rows ``q_start[b]`` .. ``q_start[b + 1]`` and ``ctx_len[b]`` keys with them, and its pages in row ``seq_slot[b]`` of ``block_table``.  The first ``n_decode`` sequences bring one
    token each; the others are listed in ``tiles`` (int32 [n_tiles, 2]: sequence, first of up to 64 of its tokens).  ``max_ctx``: at least the longest
    ``ctx_len`` (it only shapes the launch: a smaller number is slower, not wrong).  ``window`` > 0: a query sees that many keys, itself the last of them.  A row that sees no key becomes zeros; rows of ``out`` that
    belong to no sequence stay as they were.  ``status`` becomes 4 where a page is not held, 7 where a wait gave up."""
    if q.dim() != 3 or not q.is_cuda:
        raise KernelError("q must be [tokens, heads, head_dim] on the GPU")
    T, heads, d = q.shape
    if d != pages.head_dim or heads % pages.kv_heads or heads == 0:
        raise KernelError(f"{heads} heads of {d} do not fit a cache of {pages.kv_heads} heads of {pages.head_dim}")
    if T and (q.stride(2) != 1 or (heads > 1 and q.stride(1) != d)):
        raise KernelError("the heads of a token of q must lie together")
    ops._need(out, "out", q.dtype)
    if out.shape != q.shape:
        raise KernelError(f"out is {tuple(out.shape)}, not {tuple(q.shape)}")
    for name, t in (("seq_slot", seq_slot), ("q_start", q_start), ("ctx_len", ctx_len), ("block_table", block_table), ("status", status)):
        ops._need(t, name, torch.int32)
    if block_table.dim() != 2 or window < 0 or n_decode < 0 or max_ctx < 0:
        raise KernelError("attention: a table of [slots, pages], no negative numbers")
    if n_decode > seq_slot.numel() or q_start.numel() < seq_slot.numel() + 1 or ctx_len.numel() < seq_slot.numel():
        raise KernelError("attention: one slot and one length a sequence, one start more")
    if tiles is not None:
        ops._need(tiles, "tiles", torch.int32)
        n_tiles = tiles.numel() // 2 if n_tiles is None else int(n_tiles)
        if n_tiles < 0 or 2 * n_tiles > tiles.numel():
            raise KernelError(f"{n_tiles} tiles in a list of {tiles.numel() // 2}")
    ops.dtype_code(q.dtype)
    _same_device(q, out, pages.data, seq_slot, q_start, ctx_len, block_table, status, tiles)
    args = (q, pages, out, seq_slot, q_start, ctx_len, block_table, status)
    if T and n_decode:
        _attend(*args, None, n_decode, int(max_ctx), int(window), float(scale))
    if T and tiles is not None and n_tiles:
        _attend(*args, tiles, n_tiles, int(max_ctx), int(window), float(scale))


class Int4Weight:
    """A weight [rows, width] in 4 bits, laid out for :func:`matmul`.  ``gated``: the first half of the rows are gate rows, the
    second half the up rows that belong to them (for the gated epilogues, and only for them)."""

    def __init__(self, rows: int, width: int, group: int = 64, gated: bool = False, device="cuda"):
        if group not in WEIGHT_GROUPS:
            raise KernelError(f"group {group} (a 4-bit weight takes {', '.join(map(str, WEIGHT_GROUPS))})")
        if rows < 1 or width < 1 or width % group or (gated and rows % 2):
            raise KernelError(f"a 4-bit weight of {rows} rows of {width}: the width must be a multiple of the group ({group})"
                              + (", the rows of two" if gated else ""))
        self.rows, self.width, self.group, self.gated = int(rows), int(width), int(group), bool(gated)
        kept = min(group, 64)
        tiles = (self.part + 15) // 16 * (2 if gated else 1)
        self.data = torch.empty((tiles, (width + 63) // 64, 512 + 64 * (64 // kept)), dtype=torch.uint8, device=device)

    @property
    def part(self) -> int:
        """Columns of the result."""
        return self.rows // 2 if self.gated else self.rows

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 64, gated: bool = False) -> "Int4Weight":
        """``weight`` [rows, width] bfloat16 or float32 on the GPU."""
        if weight.dim() != 2 or not weight.is_cuda or weight.stride(1) != 1:
            raise KernelError("a weight is [rows, width] on the GPU, the columns of a row together")
        self = cls(weight.shape[0], weight.shape[1], group, gated, weight.device)
        _same_device(weight)
        ld = weight.stride(0) if self.rows > 1 else self.width
        ops._ok(kernels().ce_int4_quantise_weight(ops.dtype_code(weight.dtype), weight.data_ptr(), ld, self.data.data_ptr(),
                                                  self.rows, self.part, self.width, self.group, ops._stream()))
        return self

    def dequantize(self, out: torch.Tensor) -> torch.Tensor:
        """The values held, rounded once to the type of ``out`` [rows, width]."""
        if out.shape != (self.rows, self.width) or not out.is_cuda or out.stride(1) != 1:
            raise KernelError(f"out is {tuple(out.shape)}, not {(self.rows, self.width)} on the GPU")
        _same_device(out, self.data)
        ld = out.stride(0) if self.rows > 1 else self.width
        ops._ok(kernels().ce_int4_dequantise_weight(ops.dtype_code(out.dtype), out.data_ptr(), ld, self.data.data_ptr(),
                                                    self.rows, self.part, self.width, self.group, ops._stream()))
        return out


_MODES = (ops.GEMM_STORE, ops.GEMM_STORE_F32, ops.GEMM_ACCUM_F32, ops.GEMM_SWIGLU, ops.GEMM_RELUGLU, ops.GEMM_RELU2)


def matmul(x: torch.Tensor, w: Int4Weight, out: torch.Tensor, mode: int = ops.GEMM_STORE) -> None:
    """out (op)= x @ w.T with the epilogue ``mode`` (``ops.GEMM_*``), for up to :data:`MAX_TOKENS` tokens.  ``x`` [M, width]
    bfloat16 or float32; ``out`` [M, rows] (half the rows with a gated epilogue) in the type of x, float32 with ``GEMM_STORE_F32`` and
    ``GEMM_ACCUM_F32``; rows of both at any stride.  A token of x with a value that is not finite gives a row of NaN."""
    if mode not in _MODES:
        raise KernelError(f"a product with a 4-bit weight has no epilogue {mode}")
    gated = mode in (ops.GEMM_SWIGLU, ops.GEMM_RELUGLU)
    if gated != w.gated:
        raise KernelError("a gated epilogue and a gated weight go together")
    if x.dim() != 2 or not x.is_cuda or x.shape[1] != w.width or (x.shape[0] and x.stride(1) != 1):
        raise KernelError(f"x is {tuple(x.shape)}, not [tokens, {w.width}] on the GPU with the columns of a row together")
    M = x.shape[0]
    if M > MAX_TOKENS:
        raise KernelError(f"{M} tokens: a product with a 4-bit weight takes {MAX_TOKENS}")
    want = torch.float32 if mode in (ops.GEMM_STORE_F32, ops.GEMM_ACCUM_F32) else x.dtype
    if out.shape != (M, w.part) or out.dtype != want or not out.is_cuda or (M and out.stride(1) != 1):
        raise KernelError(f"out is {tuple(out.shape)} {out.dtype}, not {(M, w.part)} {want} with the columns of a row together")
    code = ops.dtype_code(x.dtype)
    _same_device(x, w.data, out)
    if M == 0:
        return
    k = kernels()
    scratch = torch.empty(k.ce_int4_gemm_scratch(code, M, w.width, w.group), dtype=torch.float32, device=x.device)
    prof = ops.profiling()
    if prof is not None:
        prof.note_work(w.data.numel() + M * w.width * x.element_size() + out.numel() * out.element_size(), 2 * M * w.rows * w.width)
    ldx, ldo = (x.stride(0), out.stride(0)) if M > 1 else (w.width, w.part)           # (a single row's stride says nothing)
    ops._ok(k.ce_int4_gemm(code, x.data_ptr(), ldx, w.data.data_ptr(), out.data_ptr(), ldo, M, w.part, w.width, w.group,
                           mode, scratch.data_ptr(), ops._stream()), 2)

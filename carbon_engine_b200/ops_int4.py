"""Operators of a model held in 4 bits: keys and values quantised into the pages of a cache and read back, attention over
such a cache, and products of a few tokens with 4-bit weights.

The format (``csrc/kernels/int4.cuh`` has its layout): ``group`` neighbouring values share a minimum z and a step s, both float16; a
value is c s + z with a code c of 0 .. 15, z = float16(min x), s = float16(max(max x - z, 0) / 15) (as a product with the float32 next to 1/15), c = (x - z) / s rounded to the nearest.
A group that holds a value beyond 60,000 in magnitude, or one that is not finite, reads back as NaN.

Like :mod:`carbon_engine_b200.ops`, every function takes tensors on the GPU, checks them, and launches on the current stream of the
tensors' device, which has to be the current one; scratch memory comes from torch's allocator at each call, so calls on several streams and captured graphs share none.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional

import torch

from . import ops, ops_tensor
from .csrc import kernel_lib
from .csrc.kernel_lib import KernelError, kernels

_i, _ll, _p = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p
# These take one pointer to their arguments, 8 bytes each (ctypes takes 0.2 us for every argument of its own):
# dtype, k, v, strides of k and v (token, head), pages, positions, seq_of_token, seq_slot, block_table, status,
# T, nkv, d, group, page_size, max_pages, num_pages, stream
kernel_lib.declare("ce_int4_kv_write", _i, [ctypes.c_char_p])
kernel_lib.declare("ce_int4_kv_read", _i, [ctypes.c_char_p])
_KV = struct.Struct("=21q").pack
# dtype, q, q_stride, pages, out, seq_slot, q_start, ctx_len, block_table, status, tiles, count, nh, nkv, d, group, page_size, max_pages,
# num_pages, window, splits, share, part_o, part_ml, scale, stream
kernel_lib.declare("ce_int4_attention", _i, [ctypes.c_char_p])
_ATTENTION = struct.Struct("=24qdq").pack
# dtype, x, ldx, w, out, ldo, M, N, K, group, mode, scratch, status, stream
kernel_lib.declare("ce_int4_gemm", _i, [ctypes.c_char_p])
_GEMM = struct.Struct("=14q").pack
# dtype, w, ld, tiles, rows, gated, width, group, stream
kernel_lib.declare("ce_int4_quantise_weight", _i, [_i, _p, _ll, _p, _i, _i, _i, _i, _p])
kernel_lib.declare("ce_int4_dequantise_weight", _i, [_i, _p, _ll, _p, _i, _i, _i, _i, _p])
# each, d, tile
kernel_lib.declare("ce_int4_attention_rows", _i, [_i] * 3)
kernel_lib.declare("ce_int4_attention_blocks", _i, [_i] * 3)
# each, d
kernel_lib.declare("ce_int4_attention_tc_blocks", _i, [_i] * 2)
# dtype, M, K, group
kernel_lib.declare("ce_int4_gemm_scratch", _ll, [_i] * 4)

HEAD_SIZES = (64, 128, 192, 256)
CACHE_GROUPS = (32, 64)
WEIGHT_GROUPS = (32, 64, 128)
#: tokens a product with a 4-bit weight takes
MAX_TOKENS = 64
#: keys of a tile of the cache: page sizes are multiples of it
TILE_TOKENS = 16


_CODES = {torch.float32: ops.F32, torch.bfloat16: ops.BF16}
_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


_entries = {}


def _entry(name: str):
    """An entry point of the kernels' library, looked up (behind that library's lock) once."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(kernels(), name)
    return fn


def _code(t: torch.Tensor, name: str) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise KernelError(f"{name} is {t.dtype} (float32 or bfloat16)")
    return code


_I32 = torch.int32


def _ints(device: int, names: str, *tensors) -> None:
    """Contiguous int32 tensors on the given device.  (A call's checks are most of its time where the kernel is short: they ask for what is cheap
    to answer, and for the words of an error only when there is one.)"""
    for t in tensors:
        if t.dtype is not _I32 or t.get_device() != device or not t.is_contiguous():
            name = names.split()[[u is t for u in tensors].index(True)]
            ops._need(t, name, _I32)
            raise KernelError(f"{name} is on {t.device}, the call's other tensors on cuda:{device}")


def _current(t: torch.Tensor, name: str) -> int:
    """The device of the call's first tensor, which has to be the current one."""
    device = t.get_device()
    if device < 0:
        raise KernelError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if device != _device():
        raise KernelError(f"{name} is on cuda:{device}, but the current device is cuda:{_device()}")
    return device


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

    def bytes_per_token(self) -> int:
        """Bytes a token's keys and values take."""
        return cache_bytes_per_token(self.kv_heads, self.head_dim, self.group)


def _kv_call(fn, k, v, pages, positions, seq_of_token, seq_slot, block_table, status) -> None:
    device = _current(k, "k")
    code = _code(k, "k")
    shape = (positions.numel(), pages.kv_heads, pages.head_dim)
    T = shape[0]
    if k.shape != shape or v.shape != shape or v.dtype is not k.dtype or v.get_device() != device or pages.data.get_device() != device:
        raise KernelError(f"k is {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} on {v.device}: not both {shape} of one type where the pages "
                          f"are ({pages.data.device})")
    k_token, k_head, k_channel = k.stride()
    v_token, v_head, v_channel = v.stride()
    if T and (k_channel != 1 or v_channel != 1):
        raise KernelError("the channels of a head of k and v must lie together")
    _ints(device, "positions seq_of_token seq_slot block_table status", positions, seq_of_token, seq_slot, block_table, status)
    if seq_of_token.numel() != T or block_table.dim() != 2:
        raise KernelError("one position and one sequence a token, and a table of [slots, pages]")
    if T == 0:
        return
    if ops._profile is not None:
        n = 2 * T * pages.kv_heads * pages.head_dim
        ops._profile.note_work(int(n * (k.element_size() + pages.element_size())), 0)
    ops._ok(fn(_KV(code, k.data_ptr(), v.data_ptr(), k_token, k_head, v_token, v_head, pages.data.data_ptr(), positions.data_ptr(),
                   seq_of_token.data_ptr(), seq_slot.data_ptr(), block_table.data_ptr(), status.data_ptr(), T, pages.kv_heads, pages.head_dim,
                   pages.group, pages.page_size, block_table.shape[1], pages.num_pages, _stream(device))))


def kv_write(pages: Int4Pages, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, seq_of_token: torch.Tensor,
             seq_slot: torch.Tensor, block_table: torch.Tensor, status: torch.Tensor) -> None:
    """Quantise the keys and values of T tokens into the pages: token t of sequence ``seq_of_token[t]`` (its table row
    ``seq_slot`` of that) goes to position ``positions[t]``.  ``k``, ``v`` [T, kv_heads, head_dim] bfloat16 or float32, tokens and heads at any stride (the columns of a step's
    projection, for instance).  No two tokens of a call may have the same place.  ``status`` becomes 2 where a token's page is not held; its row is dropped then."""
    _kv_call(_entry("ce_int4_kv_write"), k, v, pages, positions, seq_of_token, seq_slot, block_table, status)


def kv_read(pages: Int4Pages, k_out: torch.Tensor, v_out: torch.Tensor, positions: torch.Tensor, seq_of_token: torch.Tensor,
            seq_slot: torch.Tensor, block_table: torch.Tensor, status: torch.Tensor) -> None:
    """Read back what T places hold, as :func:`kv_write` names them, rounded once to the outputs' type.  ``status`` becomes 4 where a
    place's page is not held; its rows stay as they were."""
    _kv_call(_entry("ce_int4_kv_read"), k_out, v_out, pages, positions, seq_of_token, seq_slot, block_table, status)


@functools.lru_cache(maxsize=4096)
def _splits(jobs: int, tiles: int):
    """(blocks that share a row block's keys, tiles of 16 keys a block) for ``jobs`` row blocks of up to ``tiles`` tiles: what is least by the time
    that blocks take.  Blocks of 8 warps, two an SM, or of 4, four an SM, where there are more than 296; a block takes 1.03 us for each tile of a
    warp (0.65 with an SM to itself) and 4.5 to begin and end.  Of more than the chip holds at once, the mean of what it is for requests of one
    length and for those of half the longest on the average, whose long ones end alone; and what a second kernel takes that joins them.  The model
    lies within a tenth of the best: 64 sequences of 8,192 keys, 8 KV heads of 128, in 1, 2, 3, 4 and 8 blocks a row block take 138, 138, 135, 130 and
    144 us, and it takes 3; 21 of 450 to 9,000 keys, groups of 32, in 1 to 6 take 74, 76, 65, 56, 49 and 50 us, and it takes 6.  (Its numbers are the
    B200's: 148 SMs, 296 blocks of 8 warps or 592 of 4 at once.)"""
    best = (float("inf"), 1, tiles)
    for splits in (1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 20, 24, 32, 48, 64):
        share = -(-tiles // splits)
        if splits > 1 and (share < 8 or -(-tiles // share) < splits):
            continue
        blocks = jobs * splits
        rounds, turns = (blocks / 296, -(-share // 8)) if blocks <= 296 else (blocks / 592, -(-share // 4))
        cost = turns * (0.65 if blocks <= 96 else 0.85 if blocks <= 148 else 1.03) + 4.5
        if rounds > 1:
            cost *= ((rounds + 0.12) + (max(1.0, 0.55 * rounds) + 0.25)) / 2
        if _joined(jobs, splits):
            cost += 2.0 + blocks / 500
        best = min(best, (cost, splits, share))
    return best[1:]


def _shares(jobs: int, max_ctx: int, window: int, tokens: int):
    """:func:`_splits` for the keys that ``tokens`` tokens side by side may see.  ``max_ctx`` may be any bound: positions are int32."""
    keys = min(max_ctx, (1 << 31) - 1)
    if window > 0:
        keys = min(keys, window + tokens + 15)
    return _splits(jobs, max(1, (keys + 15) // 16))


def _joined(jobs: int, splits: int) -> bool:
    """Whether a second kernel joins the splits; up to 8 of few row blocks are a cluster and join through shared memory."""
    return splits > 8 or (splits > 1 and jobs * splits > 296)


#: Query rows (tokens by heads) for each round of its blocks from which portions of bfloat16 go to the tcgen05 kernel, whose blocks take up to 256
#: rows of a KV head and all of their keys: its time is the rounds' and the keys', that of the kernel on mma.sync the rows' and the keys'.  (8 KV
#: heads of 128, 2,048 keys: 52 us, against 32 for 2,048 rows, 42 for 4,096, 83 for 8,192; 16,000 keys: 330 us, against 139 for 2,048 rows
#: and 426 for 8,192.)
TENSOR_ROWS = 6000


@functools.lru_cache(maxsize=256)
def _row_blocks(each: int, d: int, tile: int):
    """Blocks a KV head takes of a sequence's token (tile 0) or of a tile of 64 tokens (1), their rows, and blocks
    of the tcgen05 kernel (0: not such heads)."""
    k = kernels()
    return k.ce_int4_attention_blocks(each, d, tile), k.ce_int4_attention_rows(each, d, tile), k.ce_int4_attention_tc_blocks(each, d) if tile else 0


def _attend(device, code, q, q_stride, heads, pages, out, seq_slot, q_start, ctx_len, block_table, status, tiles, count, max_ctx, window, scale) -> None:
    each = heads // pages.kv_heads
    tile = 0 if tiles is None else 1
    blocks, block_rows, tensor_blocks = _row_blocks(each, pages.head_dim, tile)
    jobs, tensor_blocks = count * pages.kv_heads * blocks, count * pages.kv_heads * tensor_blocks
    if (code == ops.BF16 and tensor_blocks and min(64 * count, q.shape[0]) * heads >= TENSOR_ROWS * max(1.0, tensor_blocks / 148) and count <= 65535 and q_stride % 8 == 0
            and (q.data_ptr() | out.data_ptr()) % 16 == 0):
        splits = share = 0
    else:
        splits, share = _shares(jobs, max_ctx, window, 64 if tile else 1)
    part_o = part_ml = None
    if _joined(jobs, splits):
        rows = jobs * splits * block_rows
        part_o = torch.empty(rows * (pages.head_dim + 2), dtype=torch.float32, device=q.device)
        part_ml = part_o.data_ptr() + 4 * rows * pages.head_dim
    ops._ok(_entry("ce_int4_attention")(_ATTENTION(
        code, q.data_ptr(), q_stride, pages.data.data_ptr(), out.data_ptr(), seq_slot.data_ptr(), q_start.data_ptr(), ctx_len.data_ptr(),
        block_table.data_ptr(), status.data_ptr(), 0 if tiles is None else tiles.data_ptr(), count, heads, pages.kv_heads, pages.head_dim,
        pages.group, pages.page_size, block_table.shape[1], pages.num_pages, window, splits, share,
        0 if part_o is None else part_o.data_ptr(), part_ml or 0, scale, _stream(device))), 1 if part_o is None else 2)


def attention(q: torch.Tensor, pages: Int4Pages, out: torch.Tensor, seq_slot: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor,
              block_table: torch.Tensor, status: torch.Tensor, *, n_decode: int, max_ctx: int, tiles: Optional[torch.Tensor] = None,
              n_tiles: Optional[int] = None, window: int = 0, scale: float = 1.0) -> None:
    """Causal attention of a step's queries over the pages, which hold the step's own keys and values already.

    ``q`` [T, heads, head_dim] (tokens at any stride, the heads of a token together), ``out`` [T, heads, head_dim] contiguous; sequence b has
    the rows ``q_start[b]`` .. ``q_start[b + 1]`` and ``ctx_len[b]`` keys with them, and its pages in row ``seq_slot[b]`` of ``block_table``.  The first ``n_decode`` sequences bring one
    token each, or none; the others are listed in ``tiles`` (int32 [n_tiles, 2]: sequence, first of up to 64 of its tokens).  ``max_ctx``: at least the longest
    ``ctx_len`` (it only shapes the launch: a smaller number is slower, not wrong).  ``window`` > 0: a query sees that many keys, itself the last of them.  A row that sees no key becomes zeros; rows of ``out`` that
    belong to no sequence stay as they were.  ``status`` becomes 4 where a page is not held, 7 or 61 to 69 where a wait gave up (61 on: portions on
    tcgen05).  Scores may have any size that float32 holds; those within a few of its steps of a row's largest may count alike."""
    device = _current(q, "q")
    code = _code(q, "q")
    if q.dim() != 3:
        raise KernelError("q must be [tokens, heads, head_dim]")
    T, heads, d = q.shape
    if d != pages.head_dim or heads % pages.kv_heads or heads == 0:
        raise KernelError(f"{heads} heads of {d} do not fit a cache of {pages.kv_heads} heads of {pages.head_dim}")
    q_token, q_head, q_channel = q.stride()
    if T and (q_channel != 1 or (heads > 1 and q_head != d)):
        raise KernelError("the heads of a token of q must lie together")
    if out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != device or not out.is_contiguous():
        raise KernelError(f"out is {tuple(out.shape)} {out.dtype} on {out.device}, not {tuple(q.shape)} {q.dtype}, contiguous, where q is")
    if pages.data.get_device() != device:
        raise KernelError(f"the pages are on {pages.data.device}, q on {q.device}")
    _ints(device, "seq_slot q_start ctx_len block_table status", seq_slot, q_start, ctx_len, block_table, status)
    if block_table.dim() != 2 or window < 0 or n_decode < 0 or max_ctx < 0:
        raise KernelError("attention: a table of [slots, pages], no negative numbers")
    if not 2.0 ** -149 <= scale < 2.0 ** 127:
        raise KernelError(f"attention: a scale of {scale} (it must be positive, and a number of float32 below 2^127)")
    seqs = seq_slot.numel()
    if n_decode > seqs or q_start.numel() <= seqs or ctx_len.numel() < seqs:
        raise KernelError("attention: one slot and one length a sequence, one start more")
    if tiles is not None:
        _ints(device, "tiles", tiles)
        n_tiles = tiles.numel() // 2 if n_tiles is None else int(n_tiles)
        if n_tiles < 0 or 2 * n_tiles > tiles.numel():
            raise KernelError(f"{n_tiles} tiles in a list of {tiles.numel() // 2}")
    window = min(int(window), (1 << 31) - 1)           # (positions are int32: such a window hides nothing)
    args = (device, code, q, q_token, heads, pages, out, seq_slot, q_start, ctx_len, block_table, status)
    if T and n_decode:
        _attend(*args, None, n_decode, int(max_ctx), window, float(scale))
    if T and tiles is not None and n_tiles:
        _attend(*args, tiles, n_tiles, int(max_ctx), window, float(scale))


class Int4Weight:
    """A weight [rows, width] in 4 bits, laid out for :func:`matmul`, which reads it ahead of the kernels in front: :meth:`quantize` is what writes
    it (whoever writes ``data`` otherwise synchronises before the next product).  ``gated``: the first half of the rows are gate rows, the
    second half the up rows that belong to them (for the gated epilogues, and only for them)."""

    def __init__(self, rows: int, width: int, group: int = 64, gated: bool = False, device="cuda"):
        if group not in WEIGHT_GROUPS:
            raise KernelError(f"group {group} (a 4-bit weight takes {', '.join(map(str, WEIGHT_GROUPS))})")
        if not 0 < rows < 1 << 30 or not 0 < width < 1 << 30 or width % group or (gated and rows % 2):
            raise KernelError(f"a 4-bit weight of {rows} rows of {width}: the width must be a multiple of the group ({group})"
                              + (", the rows of two" if gated else "") + ", both less than 2^30")
        self.rows, self.width, self.group, self.gated = int(rows), int(width), int(group), bool(gated)
        #: columns of the result
        self.part = self.rows // 2 if self.gated else self.rows
        kept = min(group, 64)
        tiles = (self.part + 7) // 8 if gated else (self.part + 15) // 16
        self.kblocks = (self.width + 63) // 64
        self.data = torch.empty((tiles, self.kblocks, 512 + 64 * (64 // kept)), dtype=torch.uint8, device=device)
        #: the word that kernels of products report to (``ops_tensor.gemm_status``)
        self.status = ops_tensor.gemm_workspace(self.data.device).status

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 64, gated: bool = False) -> "Int4Weight":
        """``weight`` [rows, width] bfloat16 or float32 on the GPU."""
        device = _current(weight, "weight")
        if weight.dim() != 2 or weight.stride(1) != 1:
            raise KernelError("a weight is [rows, width], the columns of a row together")
        self = cls(weight.shape[0], weight.shape[1], group, gated, weight.device)
        ld = weight.stride(0) if self.rows > 1 else self.width
        if ops._profile is not None:
            ops._profile.note_work(weight.numel() * weight.element_size() + self.data.numel(), 0)
        ops._ok(kernels().ce_int4_quantise_weight(_code(weight, "weight"), weight.data_ptr(), ld, self.data.data_ptr(),
                                                  self.rows, int(self.gated), self.width, self.group, _stream(device)), 2)
        return self

    def dequantize(self, out: torch.Tensor) -> torch.Tensor:
        """The values held, rounded once to the type of ``out`` [rows, width]."""
        device = _current(out, "out")
        if out.shape != (self.rows, self.width) or out.stride(1) != 1 or self.data.get_device() != device:
            raise KernelError(f"out is {tuple(out.shape)} on {out.device}, not {(self.rows, self.width)} where the weight is ({self.data.device})")
        ld = out.stride(0) if self.rows > 1 else self.width
        if ops._profile is not None:
            ops._profile.note_work(self.data.numel() + out.numel() * out.element_size(), 0)
        ops._ok(kernels().ce_int4_dequantise_weight(_code(out, "out"), out.data_ptr(), ld, self.data.data_ptr(),
                                                    self.rows, int(self.gated), self.width, self.group, _stream(device)), 2)
        return out


_MODES = (ops.GEMM_STORE, ops.GEMM_STORE_F32, ops.GEMM_ACCUM_F32, ops.GEMM_SWIGLU, ops.GEMM_RELUGLU, ops.GEMM_RELU2)
_GATED_MODES = (ops.GEMM_SWIGLU, ops.GEMM_RELUGLU)
_F32_MODES = (ops.GEMM_STORE_F32, ops.GEMM_ACCUM_F32)


def matmul(x: torch.Tensor, w: Int4Weight, out: torch.Tensor, mode: int = ops.GEMM_STORE) -> None:
    """out (op)= x @ w.T with the epilogue ``mode`` (``ops.GEMM_*``), for up to :data:`MAX_TOKENS` tokens (faster than the 16-bit product for up to
    some 16 of them).  Waits that gave up are reported as 51 to 59 in the weight's ``status``.  ``x`` [M, width]
    bfloat16 or float32; ``out`` [M, rows] (half the rows with a gated epilogue) in the type of x, float32 with ``GEMM_STORE_F32`` and
    ``GEMM_ACCUM_F32``; rows of both at any stride.  A token of x with a value that is not finite gives a row of NaN, a group of the weight
    that reads back as NaN its column."""
    if mode not in _MODES:
        raise KernelError(f"a product with a 4-bit weight has no epilogue {mode}")
    if (mode in _GATED_MODES) != w.gated:
        raise KernelError("a gated epilogue and a gated weight go together")
    device = _current(x, "x")
    code = _code(x, "x")
    if x.dim() != 2 or x.shape[1] != w.width:
        raise KernelError(f"x is {tuple(x.shape)}, not [tokens, {w.width}]")
    M, N = x.shape[0], w.part
    if M > MAX_TOKENS:
        raise KernelError(f"{M} tokens: a product with a 4-bit weight takes {MAX_TOKENS}")
    want = torch.float32 if mode in _F32_MODES else x.dtype
    if out.shape != (M, N) or out.dtype is not want or out.get_device() != device or w.data.get_device() != device:
        raise KernelError(f"out is {tuple(out.shape)} {out.dtype} on {out.device}, not {(M, N)} {want} where x and the weight are ({w.data.device})")
    if M == 0:
        return
    (ldx, x_step), (ldo, out_step) = x.stride(), out.stride()
    if x_step != 1 or (out_step != 1 and N > 1):
        raise KernelError("the columns of a row of x and out must lie together")
    if M == 1:
        ldx, ldo = w.width, N               # (a single row's stride says nothing)
    # up to 16 tokens that fit the registers of 8 blocks: no scratch memory, one launch (the launcher checks it too)
    scratch = None
    if (M + 7) // 8 * (1 if code else 2) * w.kblocks > 512 or M > 16:
        scratch = torch.empty(_entry("ce_int4_gemm_scratch")(code, M, w.width, w.group), dtype=torch.float32, device=x.device)
    if ops._profile is not None:
        ops._profile.note_work(w.data.numel() + M * w.width * x.element_size() + out.numel() * out.element_size(), 2 * M * w.rows * w.width)
    ops._ok(_entry("ce_int4_gemm")(_GEMM(code, x.data_ptr(), ldx, w.data.data_ptr(), out.data_ptr(), ldo, M, N, w.width, w.group, mode,
                                 0 if scratch is None else scratch.data_ptr(), w.status.data_ptr(), _stream(device))), 1 if scratch is None else 2)

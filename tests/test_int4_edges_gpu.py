"""Operators of a 4-bit model at the edges of their range: groups whose minimum rounds up, scores and tokens of any size, values that are not
numbers in every epilogue, strides and windows beyond 32 bits.  Beside test_int4_gpu.py, whose helpers it uses."""
import math

import pytest
import torch

import int4_cases as plain
from test_int4_gpu import Cache, attend, check_product, filled, gpu, normal, product_case

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def place_of_steps(pages):
    """(step, minimum) of all tokens of all pages: float16 [..., 2]."""
    return pages.data[..., 16 * pages.head_dim:].contiguous().view(torch.float16).unflatten(-1, (-1, 2))


# ---- groups whose float16 minimum lies above all their values
@pytest.mark.parametrize("value", [0.7, -0.3, 1000.3, 2049.3])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_that_are_all_alike(monkeypatch, value, dtype):
    """Their code is 0 and their step nothing: attention returns the value held, for one key and for many, whoever shares the keys."""
    from carbon_engine_b200 import ops_int4
    for d, heads, group, lengths in ((64, 4, 32, [1, 37]), (128, 8, 64, [300, 16]), (192, 3, 64, [40, 5]), (256, 2, 32, [129, 2])):
        c = Cache(lengths, 1, d, group, 16)
        n = sum(lengths)
        k, v = normal((n, 1, d), 1, F32), torch.full((n, 1, d), value, device="cuda")
        c.write(k, v)
        assert bool((place_of_steps(c.pages)[..., 0].nan_to_num(0.0) >= 0).all())
        for splits in (1, 3, 11):
            monkeypatch.setattr(ops_int4, "_splits", lambda jobs, tiles: (splits, -(-19 // splits)))
            out = attend(c, normal((2, heads, d), 9, dtype), k, v, [1, 1], lengths, group, 0, dtype)
            held = plain.held(v, group)[0, 0, 0]
            assert float((out.double() - held).abs().max()) <= abs(float(held)) * (torch.finfo(dtype).eps / 2 + 2.0 ** -20)
        # keys that are all alike; such values beside ordinary ones, group by group and key by key
        c.write(v, k)
        attend(c, normal((2, heads, d), 10, dtype), v, k, [1, 1], lengths, group, 0, dtype)
        mixed = torch.where((torch.arange(d, device="cuda") // group % 2 == 0) ^ (torch.arange(n, device="cuda")[:, None, None] % 3 == 0), v, k)
        c.write(k, mixed)
        attend(c, normal((2, heads, d), 11, dtype), k, mixed, [1, 1], lengths, group, 0, dtype)


@pytest.mark.parametrize("value", [0.7, -0.3, 2049.3])
@pytest.mark.parametrize("rows", [1, 10 ** 9])
def test_values_that_are_all_alike_in_portions(monkeypatch, value, rows):
    """On both kernels of portions."""
    from carbon_engine_b200 import ops_int4
    monkeypatch.setattr(ops_int4, "TENSOR_ROWS", rows)
    for dtype in (BF16, F32):
        c = Cache([200], 2, 128, 32, 16)
        k, v = normal((200, 2, 128), 1, F32), torch.full((200, 2, 128), value, device="cuda")
        c.write(k, v)
        attend(c, normal((90, 8, 128), 9, dtype), k, v, [90], [200], 32, 0, dtype, n_decode=0)


def test_pages_with_steps_below_zero():
    """Such pages are not written, but may be copied in: the codes beside them are zeros, and the result is the minimum's."""
    c = Cache([40], 1, 128, 64, 16)
    k, v = normal((40, 1, 128), 1, F32), torch.full((40, 1, 128), 0.75, device="cuda")
    c.write(k, v)
    steps = place_of_steps(c.pages)
    steps[..., 0] = torch.where(steps[..., 0] == 0, torch.full_like(steps[..., 0], -1.3e-5), steps[..., 0])
    c.pages.data[..., 16 * 128:] = steps.flatten(-2).view(torch.uint8).reshape(c.pages.data[..., 16 * 128:].shape)
    for dtype in (BF16, F32):
        attend(c, normal((1, 4, 128), 9, dtype), k, v, [1], [40], 64, 0, dtype)


# ---- scores of any size
def decided(q, k, v, new, lengths, off):
    """The least and the most that attention may return where scores are far apart: the values, channel by channel, of the keys whose scores
    lie by no more below a row's largest than both may err - ``off`` of the sums of their products' magnitudes each - and 100 (the others' weights,
    exp(-100) and less, are nothing).  Mostly that is one key."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    each, scale, low, high = q.shape[1] // k.shape[1], 1.0 / math.sqrt(q.shape[2]), torch.zeros_like(q), torch.zeros_like(q)
    row = first = 0
    for n, h in zip(new, lengths):
        for i in range(n):
            kk, vv = (t[first:first + h - n + i + 1].repeat_interleave(each, dim=1) for t in (k, v))
            s = (kk * q[row + i]).sum(-1) * scale
            reach = ((kk * q[row + i]).abs().sum(-1) * scale).max(0).values
            near = (s >= s.max(0).values - 100.0 - 2.0 * off * reach)[..., None]
            low[row + i] = torch.where(near, vv, math.inf).amin(0)
            high[row + i] = torch.where(near, vv, -math.inf).amax(0)
        row, first = row + n, first + h
    return low, high


def check_decided(c, q, k, v, new, lengths, group, dtype):
    heads, d = q.shape[1:]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    decoding = len(new) if max(new) == 1 else 0
    tiles = [(b, at) for b, n in enumerate(new) if b >= decoding for at in range(0, n, 64)]
    out = torch.empty_like(q)
    c.ops.attention(q, c.pages, out, c.slots, gpu(starts), gpu(lengths), c.table, c.status, n_decode=decoding, max_ctx=max(lengths),
                    tiles=gpu(tiles) if tiles else None, scale=1.0 / math.sqrt(d))
    # keys are met as they are held (scores err by float32's sums, and by the queries' 22 bits), on tcgen05 rounded to float16 (2^-11 of themselves)
    on_tcgen05 = c.ops.TENSOR_ROWS == 1 and tiles and dtype == BF16
    low, high = decided(q, plain.held(k, group), plain.held(v, group), new, lengths, 2.0 ** -10 if on_tcgen05 else 2.0 ** -20)
    # one weight of 1: its product with the step, or (on tcgen05) the value, is rounded to float16, by 2^-11 of itself at most, of twice the
    # largest value; float32: two pieces
    largest = float(plain.held(v, group).abs().max())
    slack = 2.0 * largest * (2.0 ** -11 if dtype == BF16 else 2.0 ** -22) + largest * 2.0 ** -18
    got = out.double().cpu()
    assert int(c.status) == 0
    assert bool((got >= low - low.abs() * torch.finfo(dtype).eps / 2 - slack).all()) and bool((got <= high + high.abs() * torch.finfo(dtype).eps / 2 + slack).all())
    return float((low == high).all(-1).double().mean())


SIZES = [(1e4, 2e4), (1e8, 2e4), (1e20, 1.0)]          # of queries and keys: scores of 2e8, 2e12 and 1e20


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_size,k_size", SIZES)
def test_single_tokens_with_scores_of_any_size(monkeypatch, dtype, q_size, k_size):
    """One key decides, and the result is its value: neither infinite nor nothing, though float32's own steps between such scores are large."""
    from carbon_engine_b200 import ops_int4
    for d, heads, group in ((128, 8, 64), (64, 4, 32), (256, 4, 32)):
        lengths = [400, 33, 1, 16]
        c = Cache(lengths, 1, d, group, 16)
        k = (normal((450, 1, d), 1, F32) * k_size).clamp(-6e4, 6e4)
        for v in (normal((450, 1, d), 2, F32), torch.full((450, 1, d), 0.75, device="cuda"), normal((450, 1, d), 2, F32, 1000.0)):
            c.write(k, v)
            q = normal((4, heads, d), 3, dtype, q_size)
            for splits in (1, 3, 11):
                monkeypatch.setattr(ops_int4, "_splits", lambda jobs, tiles: (splits, -(-25 // splits)))
                assert check_decided(c, q, k, v, [1] * 4, lengths, group, dtype) > 0.9          # nearly all rows of one key


@pytest.mark.parametrize("rows", [1, 10 ** 9])
@pytest.mark.parametrize("q_size,k_size", SIZES)
def test_portions_with_scores_of_any_size(monkeypatch, rows, q_size, k_size):
    from carbon_engine_b200 import ops_int4
    monkeypatch.setattr(ops_int4, "TENSOR_ROWS", rows)
    c = Cache([300], 1, 128, 64, 16)
    k, v = (normal((300, 1, 128), 1, F32) * k_size).clamp(-6e4, 6e4), normal((300, 1, 128), 2, F32)
    c.write(k, v)
    check_decided(c, normal((70, 4, 128), 3, BF16, q_size), k, v, [70], [300], 64, BF16)


@pytest.mark.parametrize("q_size", [1e4, 1e8])
def test_equal_keys_share_a_score_of_any_size(q_size):
    """The same key everywhere: the mean of the values."""
    c = Cache([16], 1, 128, 64, 16)
    k, v = normal((1, 1, 128), 1, F32, 2e4).clamp(-6e4, 6e4).expand(16, 1, 128).contiguous(), normal((16, 1, 128), 2, F32)
    c.write(k, v)
    for dtype in (BF16, F32):
        q, out = normal((1, 8, 128), 3, dtype, q_size), torch.empty((1, 8, 128), dtype=dtype, device="cuda")
        c.ops.attention(q, c.pages, out, c.slots, gpu([0, 1]), gpu([16]), c.table, c.status, n_decode=1, max_ctx=16, scale=0.09)
        held = plain.held(v, 64)
        want, largest = held.mean(0).expand(8, 128), float(held.abs().max())
        slack = 2.0 * largest * (2.0 ** -11 if dtype == BF16 else 2.0 ** -22) + largest * 2.0 ** -18
        assert bool(((out[0].double() - want).abs() <= want.abs() * torch.finfo(dtype).eps / 2 + slack).all())


# ---- numbers that are none, through every epilogue
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("mode", ["STORE", "STORE_F32", "ACCUM_F32", "SWIGLU", "RELUGLU", "RELU2"])
@pytest.mark.parametrize("M", [3, 12, 20, 64])
def test_tokens_and_weights_that_are_no_numbers(dtype, mode, M):
    """A token with a value that is not finite gives a row of NaN; a group of a weight that is not a number gives its column."""
    from carbon_engine_b200 import ops, ops_int4
    mode = getattr(ops, "GEMM_" + mode)
    gated = mode in (ops.GEMM_SWIGLU, ops.GEMM_RELUGLU)
    x, w, w4, _ = product_case(dtype, mode, M, 40, 256, 64)
    kind = F32 if mode in (ops.GEMM_STORE_F32, ops.GEMM_ACCUM_F32) else dtype

    def result(x, w4):
        out = torch.ones((M, 40), dtype=kind, device="cuda")
        ops_int4.matmul(x, w4, out, mode)
        return out

    fine = result(x, w4)
    assert not bool(fine.isnan().any())
    bad = x.clone()
    bad[0, 17], bad[2, 255] = math.nan, -math.inf
    out = result(bad, w4)
    assert bool(out[[0, 2]].isnan().all()) and not bool(out[[t for t in range(M) if t not in (0, 2)]].isnan().any())
    w = w.clone()
    w[5, 70] = math.inf                                   # (a gate row of gated weights)
    if gated:
        w[40 + 9, 3] = math.nan                           # an up row
    out = result(x, ops_int4.Int4Weight.quantize(w, 64, gated))
    columns = [5, 9] if gated else [5]
    others = [n for n in range(40) if n not in columns]
    assert bool(out[:, columns].isnan().all()) and torch.equal(out[:, others], fine[:, others])


# ---- tokens and queries as large and as small as their type holds
@pytest.mark.parametrize("M", [3, 12, 20])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_as_large_as_their_type_holds(dtype, M):
    from carbon_engine_b200 import ops, ops_int4
    x, w, w4, _ = product_case(dtype, ops.GEMM_STORE_F32, M, 40, 256, 64)
    for size in (2e35, 4e37, 1e-36):
        y = x * size                                       # results of up to 1e38: float32 holds them
        out = torch.empty((M, 40), device="cuda")
        ops_int4.matmul(y, w4, out, ops.GEMM_STORE_F32)
        assert bool(out.isfinite().all())
        if size > 1:
            check_product(y, w, 64, w4, ops.GEMM_STORE_F32, out)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_queries_as_large_as_their_type_holds(monkeypatch, dtype):
    c = Cache([300, 20], 1, 128, 64, 16)
    k, v = normal((320, 1, 128), 1, F32, 0.01), normal((320, 1, 128), 2, F32)
    c.write(k, v)
    for size in (1e35, 4e37):
        check_decided(c, normal((2, 8, 128), 3, dtype, size), k, v, [1, 1], [300, 20], 64, dtype)
    if dtype == BF16:
        from carbon_engine_b200 import ops_int4
        monkeypatch.setattr(ops_int4, "TENSOR_ROWS", 1)
        check_decided(c, normal((20 + 7, 8, 128), 3, dtype, 4e37), k, v, [20, 7], [300, 20], 64, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales_as_small_as_float32_holds(monkeypatch, dtype):
    """Every key counts the same, and what is masked counts nothing."""
    from carbon_engine_b200 import ops_int4
    c, k, v = filled([30], 1, 64, 32, 16, dtype)
    for rows in (1, 10 ** 9):
        monkeypatch.setattr(ops_int4, "TENSOR_ROWS", rows)
        for n in (1, 5):
            q = normal((n, 4, 64), 9, dtype, 1e-30)
            out = torch.empty_like(q)
            c.ops.attention(q, c.pages, out, c.slots, gpu([0, n]), gpu([30]), c.table, c.status, n_decode=int(n == 1), max_ctx=30,
                            tiles=gpu([[0, 0]]) if n > 1 else None, scale=1e-37)
            held = plain.held(v, 32)
            want = torch.stack([held[:30 - n + i + 1].mean(0).expand(4, 64) for i in range(n)])
            slack = float(held.abs().max()) * (2.0 ** -10 if dtype == BF16 else 2.0 ** -18)
            assert bool(((out.double() - want).abs() <= want.abs() * torch.finfo(dtype).eps / 2 + slack).all())


@pytest.mark.parametrize("scale", [0.0, -1.0, 1e-300, math.inf, math.nan, 1e300])
def test_scales_that_float32_does_not_hold_are_refused(scale):
    from carbon_engine_b200.csrc.kernel_lib import KernelError
    c, k, v = filled([30], 1, 64, 32, 16, BF16)
    q = normal((1, 4, 64), 9, BF16)
    with pytest.raises(KernelError, match="scale"):
        c.ops.attention(q, c.pages, torch.empty_like(q), c.slots, gpu([0, 1]), gpu([30]), c.table, c.status, n_decode=1, max_ctx=30, scale=scale)


# ---- sizes beyond 32 bits
@pytest.mark.parametrize("max_ctx", [1 << 31, 1 << 36, 1 << 40, (1 << 63) - 1])
def test_any_bound_on_the_keys(max_ctx):
    c, k, v = filled([90, 400], 2, 64, 32, 16, BF16)
    attend(c, normal((2, 4, 64), 9, BF16), k, v, [1, 1], [90, 400], 32, 0, BF16, max_ctx=max_ctx)
    attend(c, normal((20, 4, 64), 9, BF16), k, v, [12, 8], [90, 400], 32, 0, BF16, n_decode=0, max_ctx=max_ctx)


@pytest.mark.parametrize("dtype,K", [(BF16, 128), (BF16, 70016), (F32, 16448)])       # on each of the three kernels
@pytest.mark.parametrize("stride", [(1 << 31) + 8, (1 << 32) + 40])
def test_rows_of_a_result_at_strides_beyond_32_bits(dtype, K, stride):
    from carbon_engine_b200 import ops, ops_int4
    x, w, w4, _ = product_case(dtype, ops.GEMM_STORE, 2, 40, K, 64)
    whole = torch.empty(stride + 256, dtype=dtype, device="cuda")
    out = torch.as_strided(whole, (2, 40), (stride, 1))
    whole[:256] = 3.0
    out.fill_(3.0)
    ops_int4.matmul(x, w4, out, ops.GEMM_STORE)
    check_product(x, w, 64, w4, ops.GEMM_STORE, out)
    assert bool((whole[40:256] == 3).all())


@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 31, (1 << 32) + 5])
def test_windows_beyond_32_bits_hide_nothing(window):
    c, k, v = filled([90], 1, 64, 32, 16, BF16)
    q = normal((1, 4, 64), 9, BF16)
    outs = []
    for w in (0, window):
        out = torch.empty_like(q)
        c.ops.attention(q, c.pages, out, c.slots, gpu([0, 1]), gpu([90]), c.table, c.status, n_decode=1, max_ctx=90, window=w, scale=0.1)
        outs.append(out)
    assert torch.equal(*outs)


# ---- float32 tokens on either side of what the stream's registers hold
@pytest.mark.parametrize("M,K,streamed", [(8, 16384, True), (5, 16448, False), (16, 8192, True), (12, 8256, False), (1, 16448, False)])
def test_float32_products_beyond_the_streams_registers(M, K, streamed):
    from carbon_engine_b200 import ops, ops_int4
    for group, mode in ((64, ops.GEMM_STORE_F32), (32, ops.GEMM_SWIGLU)):
        x, w, w4, _ = product_case(F32, mode, M, 33, K, group)
        out = torch.empty((M, 33), device="cuda")
        before = ops.kernel_counts().get("int4_gemm_kernel", 0)
        ops_int4.matmul(x, w4, out, mode)
        check_product(x, w, group, w4, mode, out)
        assert ops.kernel_counts().get("int4_gemm_kernel", 0) - before == (0 if streamed else 1)


# ---- groups of very different steps side by side
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("spread", [1.0, 8.0])
def test_small_groups_beside_large_ones(dtype, spread):
    """Each group with a tolerance of its own.  A weight's product with its step is rounded by 2^-11 of itself (2^-22 for float32's two pieces), and
    below 2^-14 by float16's fixed half step of 2^-25.  The row's largest weight is 2^10 over a power of two that is less than twice the largest
    step s met, so in units of that weight 2^-25 is at most 2^-34 s; a key's codes are at most 15, and n keys err by n 15 2^-34 s together."""
    n, d, group = 800, 128, 32
    c = Cache([n], 1, d, group, 16)
    sizes = torch.tensor([1000.0, 1e-2, 1.0, 0.1], device="cuda").repeat_interleave(group)
    k, v = normal((n, 1, d), 1, F32, spread / 11.3), normal((n, 1, d), 2, F32) * sizes
    c.write(k, v)
    q, scale = normal((1, 8, d), 3, dtype), 1.0 / math.sqrt(d)
    out = torch.empty_like(q)
    c.ops.attention(q, c.pages, out, c.slots, gpu([0, 1]), gpu([n]), c.table, c.status, n_decode=1, max_ctx=n, scale=scale)
    held = plain.held(v, group).cpu()
    want, reach, _ = plain.attend(q.cpu(), plain.held(k, group).cpu(), held, [1], [n], scale, 0)
    largest_step = float((held.unflatten(-1, (-1, group)).amax(-1) - held.unflatten(-1, (-1, group)).amin(-1)).max()) / 15
    for g in range(d // group):
        part = slice(g * group, (g + 1) * group)
        largest = float(held[..., part].abs().max())
        tolerance = want[..., part].abs() * torch.finfo(dtype).eps / 2 + 2.0 * largest * (reach + 4.0) * 2.0 ** -21 \
            + 2.0 * largest * (2.0 ** -11 if dtype == BF16 else 2.0 ** -22) + n * 15 * 2.0 ** -34 * largest_step + largest * (n / 128 + 32) * 2.0 ** -23
        off = (out[..., part].double().cpu() - want[..., part]).abs()
        assert bool((off <= tolerance).all()), (g, float(off.max()), float(tolerance.max()))


# ---- as they are used: the tcgen05 forms
def test_graphs_and_streams_of_portions_and_of_many_tokens():
    """Two captured steps (write, attend, a product of many tokens) replayed on two streams at once, and eager calls beside them."""
    from carbon_engine_b200 import ops, ops_int4
    jobs = []
    for seed, d, heads, kv_heads in ((0, 128, 32, 8), (100, 64, 48, 4)):
        c, k, v = filled([900], kv_heads, d, 64, 16, BF16, seed=seed)
        q = normal((500, heads, d), seed + 9, BF16)
        out, y = torch.empty_like(q), torch.empty((40, 700), dtype=BF16, device="cuda")
        w4 = ops_int4.Int4Weight.quantize(normal((700, heads * d), seed + 3, BF16, 0.05), 64)
        starts, held, tiles = gpu([0, 500]), gpu([900]), gpu([(0, at) for at in range(0, 500, 64)])

        def step(c=c, k=k, v=v, q=q, out=out, y=y, w4=w4, starts=starts, held=held, tiles=tiles):
            c.write(k, v)
            c.ops.attention(q, c.pages, out, c.slots, starts, held, c.table, c.status, n_decode=0, max_ctx=900, tiles=tiles, scale=0.09)
            ops_int4.matmul(out.flatten(1)[:40], w4, y, ops.GEMM_STORE)

        before = [ops.kernel_counts().get(n, 0) for n in ("int4_attention_tc_kernel", "int4_gemm_tc_kernel")]
        step()
        torch.cuda.synchronize()
        assert [ops.kernel_counts().get(n, 0) for n in ("int4_attention_tc_kernel", "int4_gemm_tc_kernel")] == [n + 1 for n in before]
        want = out.clone(), y.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        jobs.append((graph, step, out, y, want, c, w4))
    streams = [torch.cuda.Stream() for _ in jobs]
    for run in (lambda job: job[0].replay(), lambda job: job[1]()):
        for _ in range(5):
            for s, job in zip(streams, jobs):
                with torch.cuda.stream(s):
                    job[2].zero_(); job[3].zero_()
                    run(job)
        torch.cuda.synchronize()
        for _, _, out, y, want, c, w4 in jobs:
            assert torch.equal(out, want[0]) and torch.equal(y, want[1]) and int(c.status) == 0 and int(w4.status) == 0

"""Operators of a 4-bit model against plain float64 (int4_cases.py)."""
import math

import pytest
import torch

import int4_cases as plain

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def gpu(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def normal(shape, seed, dtype, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


class Cache:
    """Pages (NaN until written) with a table, and the places of all tokens of sequences of the given lengths."""

    def __init__(self, lengths, kv_heads, d, group, page, seed=0, slots=None):
        from carbon_engine_b200 import ops_int4
        self.ops = ops_int4
        table, pages = plain.block_table(lengths, page, torch.Generator().manual_seed(seed), slots)
        self.table = table.cuda()
        self.pages = ops_int4.Int4Pages(pages, kv_heads, page, d, group, device="cuda", poison=True)
        self.slots = gpu(list(range(len(lengths))) if slots is None else slots)
        self.status = gpu([0])
        pos, seq = plain.places([0] * len(lengths), [max(n, 0) for n in lengths])
        self.pos, self.seq = gpu(pos), gpu(seq)

    def where(self, pick=None):
        pos, seq = (self.pos, self.seq) if pick is None else (self.pos[pick].contiguous(), self.seq[pick].contiguous())
        return pos, seq, self.slots, self.table, self.status

    def write(self, k, v, pick=None):
        self.ops.kv_write(self.pages, k, v, *self.where(pick))

    def read(self, like, pick=None):
        k, v = torch.full_like(like, 7.0), torch.full_like(like, 7.0)
        self.ops.kv_read(self.pages, k, v, *self.where(pick))
        return k, v


# ---- quantising and reading back: equal, bit for bit (c s + z is exact in float64, and rounded once to float32, then to the output's type)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,kv_heads,group,page,lengths", [
    (64, 1, 32, 16, [1]), (64, 3, 64, 16, [17, 1, 33]), (128, 8, 64, 16, [8, 40]), (128, 2, 32, 32, [50]), (192, 2, 32, 48, [5, 70]),
    (192, 1, 64, 64, [65]), (256, 4, 64, 64, [3, 1]), (256, 1, 32, 16, [31])])
def test_written_values_come_back(dtype, d, kv_heads, group, page, lengths):
    c = Cache(lengths, kv_heads, d, group, page)
    n = sum(lengths)
    k, v = normal((n, kv_heads, d), 1, dtype, 3.0), normal((n, kv_heads, d), 2, dtype, 0.01)
    c.write(k, v)
    assert int(c.status) == 0
    for got_type in (F32, BF16):
        kb, vb = c.read(torch.empty((n, kv_heads, d), dtype=got_type, device="cuda"))
        for got, x in ((kb, k), (vb, v)):
            assert torch.equal(got, plain.held(x, group).float().to(got_type))


def test_rows_at_any_stride_and_alignment():
    c = Cache([23], 2, 64, 32, 16)
    row = normal((23, 2 * 2 * 64 + 3), 3, F32)
    for off, dtype in ((0, F32), (1, F32), (3, BF16), (2, BF16)):
        part = row.to(dtype)[:, off:]
        k, v = part[:, :128].unflatten(1, (2, 64)), part[:, 128:256].unflatten(1, (2, 64))
        c.write(k, v)
        kb, vb = c.read(torch.empty((23, 2, 64), device="cuda"))
        assert torch.equal(kb, plain.held(k, 32).float()) and torch.equal(vb, plain.held(v, 32).float())
        wide = torch.full((23, 2 * 2 * 64 + 3), 9.0, dtype=dtype, device="cuda")
        ko, vo = wide[:, off:off + 128].unflatten(1, (2, 64)), wide[:, off + 128:off + 256].unflatten(1, (2, 64))
        c.ops.kv_read(c.pages, ko, vo, *c.where())
        assert torch.equal(ko, kb.to(dtype)) and torch.equal(vo, vb.to(dtype))
        assert bool((wide[:, :off] == 9).all()) and bool((wide[:, off + 256:] == 9).all())


def test_one_token_at_a_time_and_the_neighbours_stay():
    c = Cache([40], 2, 128, 64, 16)
    k, v = normal((40, 2, 128), 4, BF16), normal((40, 2, 128), 5, BF16)
    for t in torch.randperm(40, generator=torch.Generator().manual_seed(0)).tolist():
        c.write(k[t:t + 1], v[t:t + 1], slice(t, t + 1))
    kb, vb = c.read(k)
    assert torch.equal(kb, plain.held(k, 64).float().bfloat16()) and torch.equal(vb, plain.held(v, 64).float().bfloat16())
    # a place is written again: only it changes
    c.write(v[7:8], k[7:8], slice(7, 8))
    k2, v2 = c.read(k)
    others = [t for t in range(40) if t != 7]
    assert torch.equal(k2[others], kb[others]) and torch.equal(k2[7], plain.held(v[7], 64).float().bfloat16())


def test_borders_between_codes():
    """Steps of 1 and of 0.1: values on the border between two codes (ties to even) and one float32 step beside it."""
    rows = []
    for step in (1.0, 0.1, 3.3e-5, 250.0):
        s = float(torch.tensor(step).half())
        base = torch.tensor([0.0, 15 * s] + [(i + 0.5) * s for i in range(15)])
        for side in (0, 1, -1):
            near = base.clone()
            if side:
                near[2:] = torch.nextafter(base[2:], torch.full((15,), math.copysign(math.inf, side)))
            rows.append(torch.cat([near, torch.zeros(64 - 17)]))
    x = torch.stack(rows).reshape(-1, 1, 64).cuda()
    c = Cache([len(rows)], 1, 64, 64, 16)
    c.write(x, -x)
    kb, vb = c.read(x)
    assert torch.equal(kb, plain.held(x, 64).float()) and torch.equal(vb, plain.held(-x, 64).float())


def test_groups_that_are_constant_tiny_large_or_no_numbers():
    x = normal((12, 1, 128), 6, F32)
    x[0] = 0.0
    x[1] = -3.25
    x[2] = 1e-9                      # below float16's smallest step: held as 0
    x[3] *= 1e-7
    x[4] *= 1e4
    x[4, 0, 5] = 60000.0
    x[5, 0, 40] = math.inf
    x[6, 0, 70] = math.nan
    x[7, 0, 3] = -60001.0
    x[8, 0, 127] = -math.inf
    x[9, 0, :32] = -0.0
    x[10, 0, 1] = 3e38
    c = Cache([12], 1, 128, 32, 16)
    c.write(x, x)
    want = plain.held(x, 32).float()
    for got in c.read(x):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert int(want.isnan().sum()) == 5 * 32


def test_pages_not_held_set_the_status():
    c = Cache([40], 1, 64, 64, 16)
    k = normal((1, 1, 64), 7, BF16)
    before = c.pages.data.clone()
    for pos, table in ((-1, None), (16 * c.table.shape[1], None), (40 + 16, None), (3, c.pages.num_pages)):
        t = c.table.clone()
        if table is not None:
            t[0, 0] = table
        c.status.zero_()
        c.ops.kv_write(c.pages, k, k, gpu([pos]), gpu([0]), c.slots, t, c.status)
        assert int(c.status) == 2 and torch.equal(c.pages.data, before)
        c.status.zero_()
        out = torch.full_like(k, 5.0)
        c.ops.kv_read(c.pages, out, out, gpu([pos]), gpu([0]), c.slots, t, c.status)
        assert int(c.status) == 4 and bool((out == 5).all())


# ---- attention
def attend(c, q, k, v, new, lengths, group, window, dtype, *, n_decode=None, stride=0, max_ctx=None):
    heads, d = q.shape[1], q.shape[2]
    T = q.shape[0]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    n_decode = sum(1 for n in new if n == 1) if n_decode is None else n_decode
    tiles = [(b, at) for b, n in enumerate(new) if b >= n_decode for at in range(0, n, 64)]
    if stride:
        wide = torch.full((T, heads * d + stride), 3.0, dtype=dtype, device="cuda")
        wide[:, :heads * d] = q.flatten(1)
        q = wide[:, :heads * d].unflatten(1, (heads, d))
    out = torch.full((T + 3, heads, d), 11.0, dtype=dtype, device="cuda")
    whole = torch.cat([q, q[:1].expand(3, -1, -1)]) if not stride else torch.cat([wide, wide[:1].expand(3, -1)])[:, :heads * d].unflatten(1, (heads, d))
    scale = 1.0 / math.sqrt(d)
    c.ops.attention(whole, c.pages, out, c.slots, gpu(starts), gpu(lengths), c.table, c.status, n_decode=n_decode,
                    max_ctx=max(lengths) if max_ctx is None else max_ctx, tiles=gpu(tiles) if tiles else None, window=window, scale=scale)
    assert int(c.status) == 0
    assert bool((out[T:] == 11).all())                     # rows of no sequence stay as they were
    want, reach, largest = plain.attend(q.cpu(), plain.held(k, group).cpu(), plain.held(v, group).cpu(), new, lengths, scale, window)
    got = out[:T].double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    off = (got - want).abs() - plain.attend_tolerance(want, dtype, reach, largest, max(lengths))
    assert float(off.nan_to_num(-1.0).max()) <= 0.0, float((got - want).abs().nan_to_num().max())
    return out[:T]


def filled(lengths, kv_heads, d, group, page, dtype, seed=0, slots=None):
    c = Cache(lengths, kv_heads, d, group, page, seed, slots)
    n = sum(max(x, 0) for x in lengths)
    k, v = normal((n, kv_heads, d), seed + 1, dtype, 1.5), normal((n, kv_heads, d), seed + 2, dtype, 0.7)
    c.write(k, v)
    return c, k, v


DECODE = [
    # d, heads, kv heads, group, page, keys of each sequence, window
    (64, 1, 1, 32, 16, [1], 0), (64, 4, 2, 64, 16, [2, 15, 16, 17], 0), (128, 32, 8, 64, 16, [300, 1, 47], 0), (128, 40, 8, 32, 64, [129, 700], 0),
    (128, 7, 1, 64, 32, [1000], 0), (128, 12, 1, 32, 16, [33, 260], 0), (128, 17, 1, 64, 16, [90], 0), (192, 6, 2, 32, 48, [77, 5], 0),
    (192, 9, 1, 64, 16, [200], 0), (256, 8, 1, 32, 64, [513], 0), (256, 10, 1, 64, 16, [31, 64], 0), (64, 16, 4, 32, 16, [350, 90, 200, 7], 100),
    (128, 8, 2, 64, 16, [500, 20], 1), (128, 8, 2, 64, 32, [500, 65], 64), (128, 8, 8, 64, 16, [4500], 0), (64, 24, 1, 32, 16, [100], 17)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,heads,kv_heads,group,page,lengths,window", DECODE)
def test_attention_of_single_tokens(dtype, d, heads, kv_heads, group, page, lengths, window):
    c, k, v = filled(lengths, kv_heads, d, group, page, dtype)
    attend(c, normal((len(lengths), heads, d), 9, dtype), k, v, [1] * len(lengths), lengths, group, window, dtype)


PORTIONS = [
    # d, heads, kv heads, group, page, tokens brought, keys with them, window
    (64, 4, 2, 32, 16, [2], [2], 0), (64, 2, 2, 64, 16, [65], [65], 0), (128, 8, 2, 64, 16, [1, 70, 3], [40, 200, 3], 0), (128, 10, 2, 32, 32, [130], [131], 0),
    (128, 3, 1, 64, 16, [5, 64], [300, 64], 33), (192, 4, 1, 64, 48, [17], [90], 0), (256, 4, 2, 32, 16, [9, 33], [9, 100], 20), (64, 7, 1, 32, 64, [128], [700], 0),
    (128, 16, 1, 64, 16, [66], [1200], 0)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,heads,kv_heads,group,page,new,lengths,window", PORTIONS)
def test_attention_of_portions(dtype, d, heads, kv_heads, group, page, new, lengths, window):
    c, k, v = filled(lengths, kv_heads, d, group, page, dtype)
    attend(c, normal((sum(new), heads, d), 9, dtype), k, v, new, lengths, group, window, dtype)


@pytest.mark.parametrize("d,heads,kv_heads,group,page,new,lengths,window", [c for c in PORTIONS if c[0] <= 128] + [
    (128, 4, 1, 32, 16, [64, 1, 200], [64, 700, 260], 0), (64, 4, 4, 64, 32, [129, 70], [129, 1000], 0), (128, 32, 8, 64, 64, [100], [1500], 0),
    (128, 8, 2, 32, 16, [90], [600], 100), (128, 8, 2, 64, 16, [70], [71], 1), (64, 12, 1, 32, 16, [200], [333], 64), (128, 5, 1, 64, 16, [3], [64], 0)])
def test_attention_of_portions_on_tcgen05(monkeypatch, d, heads, kv_heads, group, page, new, lengths, window):
    """The kernel that takes portions of many row blocks, at any number of them."""
    from carbon_engine_b200 import ops, ops_int4
    monkeypatch.setattr(ops_int4, "TENSOR_ROWS", 1)
    c, k, v = filled(lengths, kv_heads, d, group, page, BF16)
    q = normal((sum(new), heads, d), 9, BF16)
    before = ops.kernel_counts().get("int4_attention_tc_kernel", 0)
    attend(c, q, k, v, new, lengths, group, window, BF16, n_decode=0)
    assert ops.kernel_counts()["int4_attention_tc_kernel"] == before + 1


def test_portions_on_tcgen05_with_numbers_that_are_none(monkeypatch):
    from carbon_engine_b200 import ops_int4
    monkeypatch.setattr(ops_int4, "TENSOR_ROWS", 1)
    for which in ("k", "v", "window"):
        lengths, new = [150], [140]
        c = Cache(lengths, 1, 128, 32, 16)
        k, v = normal((150, 1, 128), 1, BF16), normal((150, 1, 128), 2, BF16)
        (k if which == "k" else v)[80, 0, 40] = math.nan
        c.write(k, v)
        window = 30 if which == "window" else 0
        out = attend(c, normal((140, 4, 128), 9, BF16), k, v, new, lengths, 32, window, BF16, n_decode=0)
        seen = out.isnan()
        last = 80 + 29 - 10 if window else 139
        assert not bool(seen[:70].any()) and not bool(seen[last + 1:].any())
        assert bool(seen[70:last + 1].all()) if which == "k" else bool(seen[70:last + 1, :, 32:64].all()) and int(seen.sum()) == (last - 69) * 4 * 32
    c, k, v = filled([100], 1, 64, 32, 16, BF16)
    q, out = normal((80, 4, 64), 9, BF16), torch.empty((80, 4, 64), dtype=BF16, device="cuda")
    q[17, 2, 5], q[40, 0, 0] = math.inf, math.nan
    c.ops.attention(q, c.pages, out, c.slots, gpu([0, 80]), gpu([100]), c.table, c.status, n_decode=0, max_ctx=100, tiles=gpu([[0, 0], [0, 64]]), scale=0.1)
    assert bool(out[17, 2].isnan().all()) and bool(out[40, 0].isnan().all()) and int(out.isnan().sum()) == 128
    # a sequence whose length says that its tokens are not there: rows that see nothing are zeros
    c.ops.attention(q, c.pages, out, c.slots, gpu([0, 80]), gpu([0]), c.table, c.status, n_decode=0, max_ctx=100, tiles=gpu([[0, 0], [0, 64]]), scale=0.1)
    assert bool((out == 0).all()) and int(c.status) == 0


def test_portions_on_tcgen05_with_scores_far_apart(monkeypatch):
    from carbon_engine_b200 import ops_int4
    monkeypatch.setattr(ops_int4, "TENSOR_ROWS", 1)
    for spread in (3.0, 30.0):
        c = Cache([400], 1, 128, 32, 16)
        k = normal((400, 1, 128), 1, F32, spread / 11.3)
        v = normal((400, 1, 128), 2, F32) * torch.logspace(-2, 2, 400, device="cuda")[:, None, None]
        c.write(k, v)
        for size in (1.0, 1e-4):
            attend(c, normal((100, 4, 128), 20, BF16, size), k, v, [100], [400], 32, 0, BF16, n_decode=0)


def test_one_token_as_a_portion_is_that_token():
    c, k, v = filled([100, 37], 2, 128, 64, 16, BF16)
    q = normal((2, 8, 128), 9, BF16)
    attend(c, q, k, v, [1, 1], [100, 37], 64, 0, BF16, n_decode=0)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_places_of_a_batch_that_nobody_took(monkeypatch, dtype):
    """Among single tokens, at the end too, whether keys are shared among blocks or not."""
    from carbon_engine_b200 import ops_int4
    new, lengths = [1, 0, 1, 0, 0], [40, 33, 300, 0, 17]
    c, k, v = filled(lengths, 2, 64, 32, 16, dtype)
    for splits in (1, 2, 9):
        monkeypatch.setattr(ops_int4, "_splits", lambda jobs, n: (splits, -(-19 // splits)))
        attend(c, normal((2, 4, 64), 9, dtype), k, v, new, lengths, 32, 0, dtype, n_decode=5)


def test_slots_strides_and_a_launch_shaped_for_less():
    lengths = [260, 90, 33]
    c, k, v = filled(lengths, 2, 128, 64, 16, BF16, slots=[4, 0, 2])
    q = normal((3, 8, 128), 9, BF16)
    a = attend(c, q, k, v, [1] * 3, lengths, 64, 0, BF16, stride=256)
    b = attend(c, q, k, v, [1] * 3, lengths, 64, 0, BF16, stride=3)           # rows between 16-byte boundaries
    attend(c, q, k, v, [1] * 3, lengths, 64, 0, BF16, max_ctx=5)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,heads,kv_heads,group,lengths,window", [
    (64, 4, 2, 32, [3000, 40, 1, 0], 0), (128, 8, 2, 64, [2500, 17], 0), (128, 12, 1, 32, [2100, 900], 0), (192, 2, 1, 64, [1700, 33], 0),
    (256, 6, 2, 32, [1600, 5], 0), (128, 5, 1, 32, [3100], 2500)])
def test_keys_shared_among_blocks(monkeypatch, dtype, d, heads, kv_heads, group, lengths, window):
    """Blocks that join as a cluster (up to 8 of few row blocks), and by a second kernel."""
    from carbon_engine_b200 import ops, ops_int4
    c, k, v = filled(lengths, kv_heads, d, group, 16, dtype)
    q = normal((len(lengths), heads, d), 9, dtype)
    tiles = -(-(min(max(lengths), window + 16) if window else max(lengths)) // 16)
    for splits in (1, 2, 5, 8, 11, 24, 40):
        monkeypatch.setattr(ops_int4, "_splits", lambda jobs, n: (splits, -(-tiles // splits)))
        before = ops.kernel_counts().get("int4_attention_merge_kernel", 0)
        attend(c, q, k, v, [1] * len(lengths), lengths, group, window, dtype)
        assert ops.kernel_counts().get("int4_attention_merge_kernel", 0) - before == (1 if splits > 8 else 0)


@pytest.mark.parametrize("d,heads,kv_heads,group", [(128, 16, 8, 64), (64, 8, 8, 32), (128, 20, 4, 32), (256, 8, 8, 64)])
def test_more_blocks_than_run_at_once(monkeypatch, d, heads, kv_heads, group):
    """... which have fewer warps each; alone and with a second kernel that joins them."""
    from carbon_engine_b200 import ops_int4
    lengths = [1 + (i * 37) % 230 for i in range(320 // kv_heads)]
    for splits in (1, 3):
        monkeypatch.setattr(ops_int4, "_splits", lambda jobs, n: (splits, -(-15 // splits)))
        for dtype in (BF16, F32):
            c, k, v = filled(lengths, kv_heads, d, group, 16, dtype)
            attend(c, normal((len(lengths), heads, d), 9, dtype), k, v, [1] * len(lengths), lengths, group, 0, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_see_nothing_are_zeros(dtype):
    c, k, v = filled([20, 0, 33], 2, 64, 32, 16, dtype)
    out = attend(c, normal((3, 4, 64), 9, dtype), k, v, [1, 1, 1], [20, 0, 33], 32, 0, dtype)
    assert bool((out[1] == 0).all())


@pytest.mark.parametrize("spread", [30.0, 300.0])
def test_scores_far_apart_and_steps_of_every_size(spread):
    """A few keys carry everything, the largest at any place; steps of values from 1e-4 to 1e3, the largest late."""
    lengths = [800]
    c = Cache(lengths, 1, 128, 32, 16)
    k = normal((800, 1, 128), 1, F32, spread / 11.3)
    v = normal((800, 1, 128), 2, F32) * torch.logspace(-4, 3, 800, device="cuda")[:, None, None]
    c.write(k, v)
    for seed in range(3):
        attend(c, normal((1, 4, 128), 20 + seed, F32), k, v, [1], lengths, 32, 0, F32)
        attend(c, normal((1, 4, 128), 20 + seed, BF16), k, v, [1], lengths, 32, 0, BF16)


def test_queries_of_any_size():
    c, k, v = filled([70], 1, 64, 64, 16, F32)
    for size in (1e-30, 1e-4, 1e5):
        q = normal((1, 4, 64), 9, F32, size)
        q[0, 1] = 0.0
        attend(c, q, k, v, [1], [70], 64, 0, F32)
        attend(c, q.bfloat16(), k, v, [1], [70], 64, 0, BF16)


def test_a_value_that_is_no_number_reaches_the_rows_that_see_it():
    """... and its own group's channels only; a key that is none makes those rows NaN."""
    lengths, new = [50], [40]
    for which in ("k", "v"):
        c = Cache(lengths, 1, 128, 32, 16)
        k, v = normal((50, 1, 128), 1, BF16), normal((50, 1, 128), 2, BF16)
        (k if which == "k" else v)[30, 0, 40] = math.nan
        c.write(k, v)
        out = attend(c, normal((40, 4, 128), 9, BF16), k, v, new, lengths, 32, 0, BF16, n_decode=0)
        seen = out.isnan()
        assert not bool(seen[:20].any())
        assert bool(seen[20:].all()) if which == "k" else bool(seen[20:, :, 32:64].all()) and int(seen.sum()) == 20 * 4 * 32


def test_a_query_that_is_no_number_stays_alone():
    c, k, v = filled([50, 60], 1, 64, 32, 16, BF16)
    q = normal((2, 4, 64), 9, BF16)
    q[0, 2, 5], q[1, 0, 0] = math.inf, math.nan
    out = torch.empty_like(q)
    c.ops.attention(q, c.pages, out, c.slots, gpu([0, 1, 2]), gpu([50, 60]), c.table, c.status, n_decode=2, max_ctx=60, scale=0.1)
    bad = out.isnan()
    assert bool(bad[0, 2].all()) and bool(bad[1, 0].all()) and int(bad.sum()) == 128


def test_a_page_that_is_not_held_sets_the_status():
    c, k, v = filled([100], 1, 64, 32, 16, BF16)
    q, out = normal((1, 4, 64), 9, BF16), torch.empty((1, 4, 64), dtype=BF16, device="cuda")
    for bad in (-1, c.pages.num_pages):
        t = c.table.clone()
        t[0, 3] = bad
        c.status.zero_()
        c.ops.attention(q, c.pages, out, c.slots, gpu([0, 1]), gpu([100]), t, c.status, n_decode=1, max_ctx=100, scale=0.1)
        assert int(c.status) == 4


def test_offsets_beyond_32_bits():
    """The last page of a cache of more than 4 GB."""
    from carbon_engine_b200 import ops_int4
    tile = ops_int4.Int4Pages(1, 8, 64, 256, 32).data[0].numel()
    pages = ops_int4.Int4Pages((1 << 32) // tile + 2, 8, 64, 256, 32)
    status, last = gpu([0]), pages.num_pages - 1
    k, v = normal((64, 8, 256), 1, BF16), normal((64, 8, 256), 2, BF16)
    where = (gpu(list(range(64))), gpu([0] * 64), gpu([0]), gpu([[last]]), status)
    ops_int4.kv_write(pages, k, v, *where)
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    ops_int4.kv_read(pages, kb, vb, *where)
    assert torch.equal(kb, plain.held(k, 32).float().bfloat16()) and torch.equal(vb, plain.held(v, 32).float().bfloat16())
    q, out = normal((1, 8, 256), 3, BF16), torch.empty((1, 8, 256), dtype=BF16, device="cuda")
    ops_int4.attention(q, pages, out, gpu([0]), gpu([0, 1]), gpu([64]), gpu([[last]]), status, n_decode=1, max_ctx=64, scale=1 / 16)
    want, reach, largest = plain.attend(q.cpu(), plain.held(k, 32).cpu(), plain.held(v, 32).cpu(), [1], [64], 1 / 16, 0)
    assert bool(((out.double().cpu() - want).abs() <= plain.attend_tolerance(want, BF16, reach, largest, 64)).all()) and int(status) == 0


# ---- products
def product_case(dtype, mode, M, N, K, group, seed=0, x_scale=1.0):
    from carbon_engine_b200 import ops, ops_int4
    gated = mode in (ops.GEMM_SWIGLU, ops.GEMM_RELUGLU)
    w = normal((N * (2 if gated else 1), K), seed + 1, BF16, 0.05)
    x = normal((M, K), seed + 2, dtype, x_scale)
    return x, w, ops_int4.Int4Weight.quantize(w, group, gated), gated


def product(x, w, group, mode, before=None):
    """The product in float64, and how far float32 sums may take it: every product x c s and x z is off by 2^-22 (x of float32 as 22 bits), sums of
    them in runs by less than 2^-20 of their magnitudes."""
    from carbon_engine_b200 import ops
    v = plain.held(w, group).cpu()
    x = x.double().cpu()
    parts = v.unflatten(-1, (-1, group))
    spread = (parts.amax(-1, keepdim=True) - parts.amin(-1, keepdim=True)).abs() + parts.abs()         # at least |s c| + |z|, per value
    y, reach = x @ v.T, x.abs() @ (2 * spread.flatten(-2)).T * 2.0 ** -20
    if mode in (ops.GEMM_SWIGLU, ops.GEMM_RELUGLU):
        n = y.shape[1] // 2
        (g, u), (eg, eu) = (y[:, :n], y[:, n:]), (reach[:, :n], reach[:, n:])
        act = g * torch.sigmoid(g) if mode == ops.GEMM_SWIGLU else g.clamp(min=0)
        # the gates' slopes are at most 1.1
        return act * u, 1.1 * eg * u.abs() + act.abs() * eu + 1.1 * eg * eu + (act * u).abs() * 2.0 ** -20
    if mode == ops.GEMM_RELU2:
        p = y.clamp(min=0)
        return p * p, 2 * p * reach + reach * reach
    if mode == ops.GEMM_ACCUM_F32:
        return y + before.double().cpu(), reach + (y.abs() + before.double().cpu().abs()) * 2.0 ** -23
    return y, reach


def check_product(x, w, group, w4, mode, out, before=None):
    want, slack = product(x, w, group, mode, before)
    off = (out.double().cpu() - want).abs() - slack - (want.abs() + slack) * torch.finfo(out.dtype).eps / 2
    assert float(off.max()) <= 0.0, float((out.double().cpu() - want).abs().max())


MODES = ["STORE", "STORE_F32", "ACCUM_F32", "SWIGLU", "RELUGLU", "RELU2"]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("M,N,K,group", [(1, 16, 64, 64), (3, 40, 96, 32), (8, 100, 1024, 64), (9, 33, 128, 128), (17, 200, 640, 32), (64, 130, 512, 64)])
def test_product_with_a_4_bit_weight(dtype, mode, M, N, K, group):
    from carbon_engine_b200 import ops, ops_int4
    mode = getattr(ops, "GEMM_" + mode)
    x, w, w4, gated = product_case(dtype, mode, M, N, K, group)
    kind = F32 if mode in (ops.GEMM_STORE_F32, ops.GEMM_ACCUM_F32) else dtype
    out = normal((M, N), 5, kind)
    before = out.clone()
    ops_int4.matmul(x, w4, out, mode)
    check_product(x, w, group, w4, mode, out, before)



@pytest.mark.parametrize("M,N,K,group", [(20, 24, 16448, 32), (64, 16, 24576, 64), (33, 300, 8192 + 32, 32), (17, 2000, 64, 64), (40, 129, 192, 64), (3, 20, 70016, 64)])
def test_products_of_wide_narrow_and_odd_weights(M, N, K, group):
    """Tokens wider than what a thread of their preparation keeps, slices of K of one block of columns and of odd numbers of them."""
    from carbon_engine_b200 import ops, ops_int4
    x, w, w4, _ = product_case(BF16, ops.GEMM_STORE_F32, M, N, K, group)
    out = normal((M, N), 5, F32)
    ops_int4.matmul(x, w4, out, ops.GEMM_STORE_F32)
    check_product(x, w, group, w4, ops.GEMM_STORE_F32, out)
    assert int(w4.status) == 0


@pytest.mark.parametrize("M", list(range(1, 65, 3)))
def test_product_of_every_number_of_tokens(M):
    from carbon_engine_b200 import ops, ops_int4
    x, w, w4, _ = product_case(BF16, ops.GEMM_STORE, M, 48, 320, 64)
    out = torch.full((M + 2, 50), 3.0, dtype=BF16, device="cuda")
    ops_int4.matmul(x, w4, out[:M, 1:49], ops.GEMM_STORE)
    check_product(x, w, 64, w4, ops.GEMM_STORE, out[:M, 1:49])
    assert bool((out[M:] == 3).all()) and bool((out[:, 0] == 3).all()) and bool((out[:, 49] == 3).all())


def test_product_of_wide_and_of_tall_weights():
    from carbon_engine_b200 import ops, ops_int4
    for dtype, M, N, K, group in ((BF16, 1, 5000, 64, 32), (BF16, 2, 17, 12288, 64), (F32, 5, 1003, 2048, 32), (BF16, 31, 4096, 1024, 64), (F32, 64, 64, 8192, 128)):
        x, w, w4, _ = product_case(dtype, ops.GEMM_STORE_F32, M, N, K, group)
        out = torch.empty((M, N), device="cuda")
        ops_int4.matmul(x, w4, out, ops.GEMM_STORE_F32)
        check_product(x, w, group, w4, ops.GEMM_STORE_F32, out)


def test_product_of_tokens_of_any_size_stride_and_alignment():
    from carbon_engine_b200 import ops, ops_int4
    x, w, w4, _ = product_case(F32, ops.GEMM_STORE_F32, 6, 64, 256, 64)
    x = x * torch.tensor([1e-30, 1e-5, 1.0, 1e4, 1e20, 0.0], device="cuda")[:, None]
    for dtype in (F32, BF16):
        wide = torch.zeros((6, 261), dtype=dtype, device="cuda")
        for off in (0, 1, 4):
            wide[:, off:off + 256] = x
            out = torch.empty((6, 64), device="cuda")
            ops_int4.matmul(wide[:, off:off + 256], w4, out, ops.GEMM_STORE_F32)
            check_product(wide[:, off:off + 256], w, 64, w4, ops.GEMM_STORE_F32, out)
    x[2, 17], x[4, 255] = math.nan, math.inf
    out = torch.empty((6, 64), device="cuda")
    ops_int4.matmul(x, w4, out, ops.GEMM_STORE_F32)
    assert bool(out[[2, 4]].isnan().all()) and not bool(out[[0, 1, 3, 5]].isnan().any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,width,group,gated", [(1, 32, 32, False), (50, 96, 32, False), (34, 64, 64, True), (48, 384, 128, False), (20, 640, 64, True)])
def test_weight_comes_back(dtype, rows, width, group, gated):
    from carbon_engine_b200 import ops_int4
    w = normal((rows, width), 3, dtype, 0.02)
    w4 = ops_int4.Int4Weight.quantize(w, group, gated)
    for kind in (F32, BF16):
        got = w4.dequantize(torch.empty((rows, width), dtype=kind, device="cuda"))
        assert torch.equal(got, plain.held(w, group).float().to(kind))
    wide = torch.zeros((rows, width + 5), dtype=dtype, device="cuda")
    wide[:, 3:3 + width] = w
    assert torch.equal(ops_int4.Int4Weight.quantize(wide[:, 3:3 + width], group, gated).dequantize(torch.empty_like(w)), plain.held(w, group).float().to(dtype))


# ---- as they are used
def test_graphs_and_streams_share_nothing():
    """Two captured steps (write, attend, product) replayed on two streams at once, and eager calls beside them."""
    from carbon_engine_b200 import ops, ops_int4
    jobs = []
    for seed in (0, 100):
        lengths = [700, 300]
        c, k, v = filled(lengths, 2, 128, 64, 16, BF16, seed=seed)
        q = normal((2, 8, 128), seed + 9, BF16)
        out, y = torch.empty_like(q), torch.empty((2, 96), dtype=BF16, device="cuda")
        w4 = ops_int4.Int4Weight.quantize(normal((96, 1024), seed + 3, BF16, 0.05), 64)
        starts, held = gpu([0, 1, 2]), gpu(lengths)

        def step(c=c, k=k, v=v, q=q, out=out, y=y, w4=w4, starts=starts, held=held):
            c.write(k, v)
            c.ops.attention(q, c.pages, out, c.slots, starts, held, c.table, c.status, n_decode=2, max_ctx=700, scale=0.09)
            ops_int4.matmul(out.flatten(1), w4, y, ops.GEMM_STORE)

        step()
        torch.cuda.synchronize()
        want = out.clone(), y.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        jobs.append((graph, step, out, y, want))
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        for s, (graph, step, out, y, _) in zip(streams, jobs):
            with torch.cuda.stream(s):
                out.zero_(); y.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, y, want in jobs:
        assert torch.equal(out, want[0]) and torch.equal(y, want[1])
    for s, (graph, step, out, y, _) in zip(streams, jobs):
        with torch.cuda.stream(s):
            out.zero_(); y.zero_()
            step()
    torch.cuda.synchronize()
    for _, _, out, y, want in jobs:
        assert torch.equal(out, want[0]) and torch.equal(y, want[1])


def test_refusals():
    from carbon_engine_b200 import ops, ops_int4
    from carbon_engine_b200.csrc.kernel_lib import KernelError
    c, k, v = filled([20], 2, 64, 32, 16, BF16)
    q = normal((1, 4, 64), 9, BF16)
    out = torch.empty_like(q)
    args = (c.slots, gpu([0, 1]), gpu([20]), c.table, c.status)
    ok = dict(n_decode=1, max_ctx=20)
    w4 = ops_int4.Int4Weight.quantize(normal((32, 64), 1, BF16), 64)
    x, y = normal((2, 64), 2, BF16), torch.empty((2, 32), dtype=BF16, device="cuda")
    other = c.where()[1:]
    for call in (
            lambda: ops_int4.Int4Pages(2, 1, 16, 96, 32), lambda: ops_int4.Int4Pages(2, 1, 8, 64, 32), lambda: ops_int4.Int4Pages(2, 1, 16, 64, 16),
            lambda: ops_int4.Int4Pages(0, 1, 16, 64, 32),
            lambda: ops_int4.kv_write(c.pages, k.half(), v.half(), *c.where()), lambda: ops_int4.kv_write(c.pages, k, v.float(), *c.where()),
            lambda: ops_int4.kv_write(c.pages, k[:3], v[:3], *c.where()), lambda: ops_int4.kv_write(c.pages, k.cpu(), v.cpu(), *c.where()),
            lambda: ops_int4.kv_write(c.pages, k, v, c.pos.long(), *other), lambda: ops_int4.kv_read(c.pages, k.transpose(1, 2), v, *c.where()),
            lambda: ops_int4.attention(q[:, :3], c.pages, out[:, :3].contiguous(), *args, **ok), lambda: ops_int4.attention(q.float(), c.pages, out, *args, **ok),
            lambda: ops_int4.attention(q, c.pages, out, *args, n_decode=2, max_ctx=20), lambda: ops_int4.attention(q, c.pages, out, *args, n_decode=1, max_ctx=20, window=-1),
            lambda: ops_int4.attention(q.half(), c.pages, out.half(), *args, **ok),
            lambda: ops_int4.attention(q, c.pages, out, *args, n_decode=0, max_ctx=20, tiles=gpu([[0, 0]]), n_tiles=2),
            lambda: ops_int4.Int4Weight.quantize(normal((4, 60), 1, BF16), 32), lambda: ops_int4.Int4Weight.quantize(normal((3, 64), 1, BF16), 64, gated=True),
            lambda: ops_int4.Int4Weight.quantize(normal((4, 64), 1, BF16), 16), lambda: ops_int4.Int4Weight.quantize(normal((4, 64), 1, BF16).cpu(), 64),
            lambda: ops_int4.matmul(normal((65, 64), 1, BF16), w4, torch.empty((65, 32), dtype=BF16, device="cuda")),
            lambda: ops_int4.matmul(x, w4, y, ops.GEMM_SWIGLU), lambda: ops_int4.matmul(x, w4, y, ops.GEMM_CLAMPGLU), lambda: ops_int4.matmul(x, w4, y, ops.GEMM_STORE_F32),
            lambda: ops_int4.matmul(x.float(), w4, y), lambda: ops_int4.matmul(x[:, :32], w4, y), lambda: ops_int4.matmul(x, w4, y[:, :16]),
            lambda: w4.dequantize(torch.empty((32, 32), device="cuda"))):
        with pytest.raises(KernelError):
            call()
    # nothing to do is no error
    empty = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    none = gpu([])
    ops_int4.kv_write(c.pages, empty, empty, none, none, c.slots, c.table, c.status)
    ops_int4.attention(q[:0], c.pages, out[:0], *args, n_decode=0, max_ctx=0)
    ops_int4.matmul(x[:0], w4, y[:0])
    assert int(c.status) == 0

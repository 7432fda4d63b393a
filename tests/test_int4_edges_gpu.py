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

"""The 4-bit format and its operators in float64, in plain torch: what the kernels are compared with."""
import math

import torch

LIMIT = 60000.0


def held(x, group):
    """Values that 4 bits hold for x (groups along the last axis), float64; NaN for a group with a value beyond the limit or not finite."""
    y = x.float().unflatten(-1, (-1, group))
    fine = (y.abs() <= LIMIT).all(-1, keepdim=True)
    y = torch.where(fine, y, torch.zeros_like(y))
    z = y.amin(-1, keepdim=True).half()
    s = ((y.amax(-1, keepdim=True) - z.float()) * torch.tensor(1 / 15, dtype=torch.float32, device=y.device)).half().double()
    c = torch.where(s > 0, ((y.double() - z.double()) / s).round().clamp(0, 15), torch.zeros_like(y, dtype=torch.float64))
    v = torch.where(fine, c * s + z.double(), torch.full_like(c, math.nan))
    return v.flatten(-2)


def places(first, counts):
    seq = [b for b, n in enumerate(counts) for _ in range(n)]
    pos = [first[b] + i for b, n in enumerate(counts) for i in range(n)]
    return pos, seq


def block_table(lengths, page, generator, slots=None):
    """Pages in random order for sequences of these lengths, in the table rows ``slots``."""
    per = [max(1, -(-n // page)) for n in lengths]
    slots = list(range(len(lengths))) if slots is None else slots
    order = torch.randperm(sum(per) + 2, generator=generator)[:sum(per)]
    table = torch.full((max(slots) + 1, max(per) + 1), -1, dtype=torch.int32)
    at = 0
    for slot, n in zip(slots, per):
        table[slot, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table, sum(per) + 2


def attend(q, k, v, new, held_tokens, scale, window):
    """Causal attention in float64 over the keys and values [tokens, kv_heads, d] of all sequences one after another.  Returns the result, the
    largest sum of |q_c k_c| scale of a row (by which scores err) and the largest |v| (by which the result errs)."""
    q, k, v = q.double(), k.double(), v.double()
    each = q.shape[1] // k.shape[1]
    out = torch.zeros_like(q)
    reach, row, first = 0.0, 0, 0
    for n, h in zip(new, held_tokens):
        for i in range(n):
            p = h - n + i
            lo = max(0, p - window + 1) if window else 0
            if p >= 0:
                kk, vv = (t[first + lo:first + p + 1].repeat_interleave(each, dim=1) for t in (k, v))
                score = (kk * q[row + i][None]).sum(-1) * scale
                reach = max(reach, float(((kk.abs() * q[row + i].abs()[None]).sum(-1) * scale).nan_to_num().max()))
                w = torch.softmax(score, dim=0)
                out[row + i] = (w[..., None] * vv).sum(0)
        row, first = row + n, first + max(h, 0)
    return out, reach, float(v.abs().nan_to_num().max())


def attend_tolerance(want, dtype, reach, largest, keys):
    """How far the kernel may be off.  Its scores err by 2^-22 of the products' magnitudes (queries as 22 bits, float32 sums of 64 channels at a
    time), a probability by that and by 2^-21 (the exponential); its product with the step is rounded to float16 (2^-12 of itself, 2^-23 for
    float32's two pieces), where the steps' part of a value is at most twice the largest value; sums over n keys err by n 2^-24 at most, in
    runs; the result is rounded once, by half a step."""
    scores = 2.0 * largest * (reach + 4.0) * 2.0 ** -21
    weights = 2.0 * largest * (2.0 ** -12 if dtype == torch.bfloat16 else 2.0 ** -22)
    sums = largest * (keys / 128 + 32) * 2.0 ** -23
    return want.abs() * torch.finfo(dtype).eps / 2 + scores + weights + sums

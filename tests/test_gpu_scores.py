"""Attention over scores of all sizes, chosen so that they are exact in 32 bits: what is left to round is small beside a result."""
import pytest
import torch

from attn_util import Paged, check, cumulated, packed_reference, rows
from tiny_vllm_b200.attention import decode_attention, prefill_attention

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def exact_scores(shape, n, m, dtype, dim, heads, kv, gen):
    """q, k, v whose scores are exact in 32 bits and differ by small numbers beside large ones: heads see a course of up to 256, which
    `shape` gives, times 1, 2, 4, 8, and another component of a few units.  Values are 1 or more."""
    q, k = torch.zeros(n, heads, dim, device="cuda"), torch.zeros(m, kv, dim, device="cuda")
    j = torch.arange(m, device="cuda", dtype=torch.float64)
    course = {"rising": j * 512 / m - 256, "falling": 256 - j * 512 / m, "steps": 40 * ((j // 16) % 13) - 256,
              "waves": 256 * torch.sin(j / 23), "late": torch.where(j % 128 >= 100, 250 - j / 50 % 250, -200.0 + j % 7)}[shape]
    q[:, :, 0] = 2.0 ** (torch.arange(heads, device="cuda") % 4)
    q[:, :, dim - 3] = torch.randint(-2, 3, (n, heads), device="cuda", generator=gen).float()
    k[:, :, 0] = course.round()[:, None].float()
    k[:, :, dim - 3] = torch.randint(-2, 3, (m, kv), device="cuda", generator=gen).float()
    v = 1 + torch.randn(m, kv, dim, device="cuda", generator=gen).abs()
    return q.to(dtype), k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("shape", ["rising", "falling", "steps", "waves", "late"])
@pytest.mark.parametrize("dtype,dim,n,m", [(BF, 128, 400, 400), (HF, 64, 300, 400), (BF, 64, 3, 6000), (HF, 128, 70, 2500)])
def test_maxima_that_move_by_far_more_than_a_weights_range(dtype, dim, n, m, shape):
    heads, kv = 4, 2
    gen = generator(2)
    q, k, v = exact_scores(shape, n, m, dtype, dim, heads, kv, gen)
    want, _ = packed_reference(q, k, v, [n], [m], 1.0)
    # Scores are exact: products of whole numbers under 2^12.  Left, with values that are positive (A = o, see attn_util): the result's
    # and the weights' rounding, u each; 2 (ds + 2^-16), ds = 2^-22 of the largest score; 32-bit sums over m keys; weights below
    # fp16's smallest normal.
    u, ds = torch.finfo(dtype).eps / 2, (8 * 256 + 4) * 2.0 ** -22
    tol = (2 * u + 2 * (ds + 2.0 ** -16) + m * 2.0 ** -23) * 1.01 * want
    if dtype == HF:
        tol = tol + 2.0 ** -25 * (m + 1) * float(v.max())
    assert float((tol / want).max()) < 0.02
    check(prefill_attention(q, k, v, cumulated([n]), cumulated([m]), n, m, scale=1.0), want, tol)
    paged = Paged(gen, k, v, [m], 64)
    check(prefill_attention(q, paged.k, paged.v, cumulated([n]), cumulated([m]), n, m, scale=1.0, block_tables=paged.tables), want, tol)
    lengths = torch.tensor([m], dtype=torch.int32, device="cuda")
    check(decode_attention(q[-1:], paged.k, paged.v, lengths, paged.tables, scale=1.0), want[-1:], tol[-1:])

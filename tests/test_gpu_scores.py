"""Attention over scores of all sizes, chosen so that they are exact in 32 bits: what is left to round is small beside a result."""
import pytest
import torch

from attn_util import Paged, check, cumulated, packed_reference, rows
from gpu_util import device_status_ok
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


@pytest.mark.parametrize("n,m", [(300, 300), (3, 6000)], ids=["whole", "cut"])
@pytest.mark.parametrize("dtype,power", [(BF, 24), (BF, 31), (BF, 60), (BF, 120), (HF, 22), (HF, 24), (HF, 28)])
def test_scores_of_any_size(dtype, power, n, m):
    # Scores are whole multiples of 2^power, zero among them, of either sign and exact: a row is the mean of the values of its
    # largest ones, all other weights being 2^-(2^22) or less.  Courses rise, fall, do both, and rise in a tile's last columns.
    dim, heads, kv = 64, 4, 2
    gen = generator(power)
    j = torch.arange(m, device="cuda")
    q, unit = torch.zeros(n, heads, dim, device="cuda"), torch.zeros(dim, device="cuda")
    if dtype == BF:
        q[:, :, 5], unit[5] = 2.0 ** (power - power // 2), 2.0 ** (power // 2)
    else:      # as many components as it takes: 2^14 2^8 each
        q[:, :, :2 ** (power - 22)], unit[:2 ** (power - 22)] = 2.0 ** 14, 2.0 ** 8
    lengths = torch.tensor([m], dtype=torch.int32, device="cuda")
    for course in (j // 50 - 3, -(j // 50), torch.full_like(j, -1), torch.full_like(j, 77), (j * 7) % 53 - 60,
                   20 - (j - m // 2).abs() // 40, (j % 128 >= 100).int() - 3, j % 97 - j // 31):
        course = course.clamp(-127, 127)
        k = course[:, None, None] * unit.expand(m, kv, dim)
        v = rows(gen, m, kv, dim, dtype)
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda").tril(m - n)
        top = torch.where(seen, course, -1000).amax(1, keepdim=True)
        p = (seen & (course == top)).double()
        p = p / p.sum(1, keepdim=True)
        want = torch.einsum("nm,mhd->nhd", p, v.double()).repeat_interleave(2, 1)
        a = torch.einsum("nm,mhd->nhd", p, v.double().abs()).repeat_interleave(2, 1)
        # weights are 1, up to the exponential's 2^-16 and a factor that a row's sums share; then sums over m keys in 32 bits, the rounding
        tol = torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -15 + m * 2.0 ** -23) * 1.01 * a + 2.0 ** -25
        kk = k.to(dtype)
        assert torch.equal(kk.float(), k)
        check(prefill_attention(q.to(dtype), kk, v, cumulated([n]), cumulated([m]), n, m, scale=1.0), want, tol)
        paged = Paged(gen, kk, v, [m], 64)
        check(prefill_attention(q.to(dtype), paged.k, paged.v, cumulated([n]), cumulated([m]), n, m, scale=1.0,
                                block_tables=paged.tables), want, tol)
        check(decode_attention(q[-1:].to(dtype), paged.k, paged.v, lengths, paged.tables, scale=1.0), want[-1:], tol[-1:])
    assert device_status_ok()


def test_queries_that_are_overwritten_by_their_results():
    # scores far from zero and near it: rows of the first kind are worked on twice
    queries, keys = [300, 70], [300, 4000]
    gen = generator(3)
    q, k, v = rows(gen, 370, 8, 64, BF, 2.0), rows(gen, 4300, 2, 64, BF), rows(gen, 4300, 2, 64, BF)
    q[100:200, :, 3] = 2.0 ** 20
    q[340:350, 3, 3] = -2.0 ** 20
    want = prefill_attention(q, k, v, cumulated(queries), cumulated(keys), 300, 4000)
    assert not torch.equal(want[100:200], want[:100])
    out = q.clone()
    got = prefill_attention(out, k, v, cumulated(queries), cumulated(keys), 300, 4000, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    parts = torch.cat([q, q], 1)      # strided queries over which a dense result is laid
    over = parts.view(-1)[:q.numel()].view_as(q)
    got = prefill_attention(parts[:, 8:], k, v, cumulated(queries), cumulated(keys), 300, 4000, out=over)
    assert torch.equal(got, want)
    last = torch.tensor(keys, dtype=torch.int32, device="cuda")
    paged = Paged(gen, k, v, keys, 16)
    one = q[[299, 369]].clone()
    want = decode_attention(one, paged.k, paged.v, last, paged.tables)
    parts = torch.cat([one, one], 1)
    got = decode_attention(one, paged.k, paged.v, last, paged.tables, out=one)
    assert torch.equal(got, want)
    got = decode_attention(parts[:, 8:], paged.k, paged.v, last, paged.tables, out=parts.view(-1)[:one.numel()].view_as(one))
    assert torch.equal(got, want)

"""Attention where results are easily lost on the way: pieces of a cut item that hold no finite score, values that are not finite
in places that the mask hides."""
import pytest
import torch

from attn_util import Paged, check, cumulated, packed_reference, rows
from gpu_util import device_status_ok
from tiny_vllm_b200.attention import decode_attention, prefill_attention

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("dtype,dim,m", [(BF, 128, 8192), (HF, 64, 8190), (BF, 128, 5000)])
def test_nan_keys_reach_their_rows_from_every_piece_of_a_cut_prompt(dtype, dim, m, page):
    # Few queries over a long prefix: the keys are divided over the GPU.  From `first` on, at every border of a tile of 128, keys are
    # NaN: a piece may then hold nothing but NaN and what the mask hides, and the rows are NaN all the same.
    n, heads, kv = 3, 4, 2
    gen = generator(1)
    q, k, v = rows(gen, n, heads, dim, dtype, 2.0), rows(gen, m, kv, dim, dtype), rows(gen, m, kv, dim, dtype)
    q[:, :, 0] = q[:, :, 0].abs() + 1
    for first in range((m - 1) // 128 * 128, m - 2600, -128):
        for kind in ("nan", "-inf"):
            kk = k.clone()
            kk[first:] = float("nan")
            if kind == "-inf":      # scores of -inf: the rest of the keys decide
                kk[first:] = 0
                kk[first:, :, 0] = -torch.inf
                want, tol = packed_reference(q, k[:first], v[:first], [n], [first], dim ** -0.5, causal=False)
            vv, tables = v, None
            if page:
                paged = Paged(gen, kk, v, [m], page)
                kk, vv, tables = paged.k, paged.v, paged.tables
            got = prefill_attention(q, kk, vv, cumulated([n]), cumulated([m]), n, m, block_tables=tables)
            if kind == "nan":
                assert bool(got.isnan().all()), f"finite rows, keys of NaN from {first} on"
            else:
                check(got, want, tol)
            if page:
                lengths = torch.tensor([m], dtype=torch.int32, device="cuda")
                dec = decode_attention(q[-1:], kk, vv, lengths, tables)
                if kind == "nan":
                    assert bool(dec.isnan().all()), first
                else:
                    check(dec, want[-1:], tol[-1:])
    assert device_status_ok()


@pytest.mark.parametrize("kind", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("dtype,heads,kv,dim,n,m,page", [(BF, 2, 1, 64, 160, 160, 0), (HF, 8, 2, 128, 129, 300, 16), (BF, 7, 1, 80, 40, 400, 0),
                                                         (BF, 4, 2, 128, 130, 7000, 64)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them_alone(dtype, heads, kv, dim, n, m, page, kind):
    # In sequence b the value at one position of the last n, of the prefix or of neither is not finite in one dimension.
    where = list(range(m - n, m, 7 if m < 1000 else 41)) + [0, m - n - 1, m // 2, m - 1]
    where = sorted({w for w in where if w >= 0})
    count = len(where)
    gen = generator(4)
    q, k, v = rows(gen, n, heads, dim, dtype, 2.0), rows(gen, m, kv, dim, dtype), rows(gen, m, kv, dim, dtype)
    want, tol = packed_reference(q, k, v, [n], [m], dim ** -0.5)
    big_q, big_k, big_v = (torch.cat([t] * count) for t in (q, k, v))
    for b, w in enumerate(where):
        big_v[b * m + w, kv - 1, 9] = float(kind) if kind != "nan" else float("nan")
    tables, kk, vv = None, big_k, big_v
    if page:
        paged = Paged(gen, big_k, big_v, [m] * count, page)
        kk, vv, tables = paged.k, paged.v, paged.tables
    for group in (slice(0, count), slice(0, 1), slice(count - 1, count)):      # many sequences, and one alone, whose keys are cut
        some = range(count)[group]
        cu_q, cu_k = cumulated([n] * len(some)), cumulated([m] * len(some))
        first, last = some[0], some[-1] + 1
        args = (kk, vv) if page else (kk[first * m:last * m], vv[first * m:last * m])
        got = prefill_attention(big_q[first * n:last * n], *args, cu_q, cu_k, n, m, block_tables=tables[group] if page else None)
        for b, o in zip(some, got.unflatten(0, (-1, n))):
            w, mine = where[b], slice(heads - heads // kv, heads)
            seen = max(0, w - (m - n))      # rows from here on see it
            part = o[seen:, mine, 9]
            assert bool(part.isnan().all() if kind == "nan" else (part == float(kind)).all()), w
            rest = o.clone()
            rest[seen:, mine, 9] = want[seen:, mine, 9].to(dtype)
            check(rest, want, tol)
    assert device_status_ok()

"""Attention where results are easily lost on the way: pieces of a cut item that hold no finite score, scores whose sums have to
be rescaled often."""
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

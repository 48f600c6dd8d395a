"""Attention over packed and paged keys against the formula in 64 bits (attn_util has the tolerance's derivation)."""
import pytest
import torch

from attn_util import Paged, check, cumulated, packed_reference, reference, rows
from gpu_util import device_status_ok
from tiny_vllm_b200 import _lib
from tiny_vllm_b200.attention import copy_pages, decode_attention, prefill_attention, store_kv

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prefill_case(seed, dtype, heads, kv, dim, queries, keys, gain=2.0, wide=0):
    gen = generator(seed)
    q = rows(gen, sum(queries), heads, dim, dtype, gain, wide)
    k = rows(gen, sum(keys), kv, dim, dtype, 1.0, wide)
    v = rows(gen, sum(keys), kv, dim, dtype, 1.0, wide)
    return gen, q, k, v


PREFILL = [  # dtype, heads, kv heads, dim, queries, prefixes
    (BF, 16, 8, 128, [1], [0]),
    (BF, 16, 8, 128, [23], [0]),
    (HF, 16, 8, 128, [64, 65, 63], [0, 0, 0]),
    (BF, 4, 1, 128, [1, 2, 3, 130, 257, 31], [0] * 6),
    (BF, 8, 8, 128, [127, 128, 129, 256, 1], [0] * 5),             # a head for itself
    (HF, 7, 1, 128, [300, 19], [0, 0]),                             # a group that divides no tile
    (BF, 24, 2, 128, [100, 50], [0, 0]),
    (BF, 128, 1, 64, [5, 3], [0, 0]),                               # the largest group
    (BF, 40, 8, 128, [77, 1, 260], [0, 500, 3]),
    (HF, 8, 2, 64, [513, 1, 511], [0, 0, 0]),
    (BF, 6, 2, 80, [200, 90], [0, 11]),
    (HF, 4, 4, 96, [129, 64], [0, 0]),
    (BF, 2, 2, 8, [70, 200], [0, 0]),
    (BF, 2, 1, 120, [70, 200], [9, 0]),
    (BF, 32, 8, 128, [1500], [0]),
    (HF, 32, 8, 128, [33, 1, 256], [2000, 777, 128]),
    (BF, 4, 2, 128, [3], [9000]),                                   # few rows over a long prefix
]


def ids(c):
    return "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c)


@pytest.mark.parametrize("case", PREFILL, ids=ids)
@pytest.mark.parametrize("page", [0, 16, 48, 256])
def test_prefill(case, page):
    dtype, heads, kv, dim, queries, prefixes = case
    keys = [n + m for n, m in zip(queries, prefixes)]
    gen, q, k, v = prefill_case(1, dtype, heads, kv, dim, queries, keys)
    want, tol = packed_reference(q, k, v, queries, keys, dim ** -0.5)
    tables = None
    if page:
        paged = Paged(gen, k, v, keys, page)
        k, v, tables = paged.k, paged.v, paged.tables
    got = prefill_attention(q, k, v, cumulated(queries), cumulated(keys), max(queries), max(keys), block_tables=tables)
    check(got, want, tol)
    assert device_status_ok()


@pytest.mark.parametrize("page", [0, 32])
def test_prefill_without_causal_mask(page):
    queries, keys = [40, 3, 130, 9], [300, 1, 128, 0]
    gen, q, k, v = prefill_case(2, BF, 8, 2, 128, queries, keys)
    want, tol = packed_reference(q, k, v, queries, keys, 0.3, causal=False)
    tables = None
    if page:
        paged = Paged(gen, k, v, keys, page)
        k, v, tables = paged.k, paged.v, paged.tables
    got = prefill_attention(q, k, v, cumulated(queries), cumulated(keys), 130, 300, scale=0.3, causal=False,
                            block_tables=tables)
    check(got, want, tol)


@pytest.mark.parametrize("page", [0, 16])
def test_rows_that_see_nothing_and_empty_sequences(page):
    # more queries than keys: the first rows see no key; sequences without queries, without keys, without both
    queries, keys = [200, 0, 5, 0, 300], [60, 40, 0, 0, 300]
    gen, q, k, v = prefill_case(3, BF, 4, 2, 128, queries, keys)
    want, tol = packed_reference(q, k, v, queries, keys, 128 ** -0.5)
    tables = None
    if page:
        paged = Paged(gen, k, v, keys, page)
        k, v, tables = paged.k, paged.v, paged.tables
    got = prefill_attention(q, k, v, cumulated(queries), cumulated(keys), 300, 300, block_tables=tables)
    check(got, want, tol)
    assert torch.equal(got[:140], torch.zeros_like(got[:140])) and torch.equal(got[200:205], torch.zeros_like(got[:5]))


@pytest.mark.parametrize("dim,kv", [(128, 8), (64, 2)])
def test_many_short_sequences(dim, kv):
    # items of one tile of keys, whose end is cleared, follow one another as fast as their copies come from memory
    n, m = 4096, 100
    gen = generator(22)
    q, k, v = rows(gen, n, 4 * kv, dim, BF), rows(gen, n * m, kv, dim, BF), rows(gen, n * m, kv, dim, BF)
    queries, keys = cumulated([1] * n), cumulated([m] * n)
    got = [prefill_attention(q, k, v, queries, keys, 1, m) for _ in range(10)]
    qd, kd, vd = (t.double().unflatten(0, (n, -1)) for t in (q, k, v))
    p = torch.einsum("nxhgd,nmhd->nhgm", qd.unflatten(2, (kv, 4)), kd).mul(dim ** -0.5).softmax(-1)
    want = torch.einsum("nhgm,nmhd->nhgd", p, vd).flatten(1, 2)
    # u |o| + (u + 2 (ds + 2^-16) + m 2^-23) A with |o| <= A = sum p |v|, scores under 8: ds < 2^-13
    tol = (2 * 2.0 ** -8 + 2.0 ** -11) * torch.einsum("nhgm,nmhd->nhgd", p, vd.abs()).flatten(1, 2) + 2.0 ** -26
    check(got[0], want, tol)
    for other in got[1:]:
        assert torch.equal(got[0], other)
    assert device_status_ok()


def test_no_keys_at_all():
    q = torch.ones(7, 4, 128, dtype=BF, device="cuda")
    k = torch.empty(0, 2, 128, dtype=BF, device="cuda")
    got = prefill_attention(q, k, k, cumulated([7]), cumulated([0]), 7, 0)
    assert torch.equal(got, torch.zeros_like(q))
    assert prefill_attention(q[:0], k, k, cumulated([0]), cumulated([0]), 0, 0).shape == (0, 4, 128)


def test_rows_behind_the_last_sequence_stay():
    queries = [30, 100]
    gen, q, k, v = prefill_case(4, BF, 4, 2, 128, [30, 100, 50], [180])
    out = torch.full_like(q, 7.0)
    got = prefill_attention(q, k, v, cumulated(queries), cumulated(queries), 100, 100, out=out)
    assert got.data_ptr() == out.data_ptr()
    want, tol = packed_reference(q[:130], k[:130], v[:130], queries, queries, 128 ** -0.5)
    check(got[:130], want, tol)
    assert torch.equal(got[130:], torch.full_like(got[130:], 7.0))


def test_neighbours_nan_stays_with_them():
    # the sequence behind (packed in the same tile of keys) is all NaN and infinite; so are the rows behind the last one
    queries = [70, 90, 20]
    gen, q, k, v = prefill_case(5, BF, 4, 2, 128, queries, queries)
    want, tol = packed_reference(q, k, v, queries, queries, 128 ** -0.5)
    for t in (k, v):
        t[70:160] = float("nan")
        t[75:100] = float("inf")
    got = prefill_attention(q, k, v, cumulated(queries), cumulated(queries), 90, 90)
    check(got[:70], want[:70], tol[:70])
    check(got[160:], want[160:], tol[160:])
    assert got[71:160].isnan().all()


def test_hints_of_the_lengths_do_not_change_the_result():
    queries, keys = [5, 40], [3000, 700]
    gen, q, k, v = prefill_case(6, HF, 8, 2, 128, queries, keys)
    want, tol = packed_reference(q, k, v, queries, keys, 128 ** -0.5)
    for hint_q, hint_k in ((40, 3000), (1, 1), (0, 0), (100000, 1 << 20)):
        check(prefill_attention(q, k, v, cumulated(queries), cumulated(keys), hint_q, hint_k), want, tol)


@pytest.mark.parametrize("layout", ["thd", "htd"])
def test_strides(layout):
    queries, keys = [90, 200], [130, 200]
    gen, q, k, v = prefill_case(7, BF, 6, 2, 64, queries, keys, wide=40)      # parts of longer rows
    assert not q.is_contiguous()
    want, tol = packed_reference(q, k, v, queries, keys, 0.125)
    check(prefill_attention(q, k, v, cumulated(queries), cumulated(keys), 200, 200), want, tol)
    odd = prefill_case(7, BF, 6, 2, 64, queries, keys, wide=3)               # not on 16-byte boundaries
    want_odd, tol_odd = packed_reference(*odd[1:], queries, keys, 0.125)
    check(prefill_attention(*odd[1:], cumulated(queries), cumulated(keys), 200, 200), want_odd, tol_odd)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]   # heads outermost
    check(prefill_attention(*turned, cumulated(queries), cumulated(keys), 200, 200), want, tol)
    paged = Paged(gen, k, v, keys, 32, layout=layout)
    wide = torch.full((2, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, :paged.tables.shape[1]] = paged.tables
    got = prefill_attention(q, paged.k, paged.v, cumulated(queries), cumulated(keys), 200, 200,
                            block_tables=wide[:, :paged.tables.shape[1] + 2])
    check(got, want, tol)
    last = q[torch.tensor([89, 289], device="cuda")]
    got = decode_attention(last, paged.k, paged.v, torch.tensor(keys, dtype=torch.int32, device="cuda"), wide[:, :9])
    check(got, want[[89, 289]], tol[[89, 289]])


def test_large_scores():
    # scores of thousands: weights of one key, sums that rise by far more than a type's range on the way
    queries = [400]
    gen, q, k, v = prefill_case(8, BF, 4, 2, 128, queries, queries, gain=60.0)
    ramp = torch.linspace(0.1, 6, 400, device="cuda")[:, None, None]
    for kk in ((k * ramp).to(BF), (k * ramp.flip(0)).to(BF)):
        want, tol = packed_reference(q, kk, v, queries, queries, 1.0)
        got = prefill_attention(q, kk, v, cumulated(queries), cumulated(queries), 400, 400, scale=1.0)
        check(got, want, tol)
        paged = Paged(gen, kk, v, queries, 64)
        got = decode_attention(q[-1:], paged.k, paged.v, torch.tensor([400], dtype=torch.int32, device="cuda"),
                               paged.tables, scale=1.0)
        check(got, want[-1:], tol[-1:])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("gap", [9.0, 90.0, 128.0, 200.0, 1000.0])
def test_one_key_far_ahead_wherever_it_stands(gap, dim):
    # 256 sequences of 300 keys: in sequence j key j has a score that is `gap` (of the exponent of 2) above all others
    n, m = 256, 300
    q = torch.zeros(n, 2, dim, dtype=BF, device="cuda")
    q[:, :, 0] = 8.0
    gen = generator(9)
    k, v = rows(gen, n * m, 1, dim, BF), rows(gen, n * m, 1, dim, BF)
    k[:, :, 0] = 0
    j = torch.arange(n, device="cuda")
    k[j * m + j, :, 0] = gap / 8
    keys = [m] * n
    scale = 0.6931471805599453
    want, tol = packed_reference(q, k, v, [1] * n, keys, scale)
    check(prefill_attention(q, k, v, cumulated([1] * n), cumulated(keys), 1, m, scale=scale), want, tol)
    paged = Paged(gen, k, v, keys, 16)
    check(decode_attention(q, paged.k, paged.v, torch.tensor(keys, dtype=torch.int32, device="cuda"), paged.tables, scale=scale),
          want, tol)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_the_largest_scores(dtype):
    # q . k = 2^24 for one key of each row's, at most 2^23 for the others: a row is that key's value
    n, dim = 300, 64
    one = torch.zeros(n, 1, dim, dtype=dtype, device="cuda")
    one[:, 0, 0] = 4096
    k = one / torch.arange(2, n + 2, device="cuda", dtype=torch.float32)[:, None, None].to(dtype)
    for best in (0, 7, 150, 299):
        kk = k.clone()
        kk[best] = one[best]
        v = rows(generator(best), n, 1, dim, dtype)
        got = prefill_attention(one, kk, v, cumulated([n]), cumulated([n]), n, n, scale=1.0)
        # the weight, whose 32-bit argument may be off by one, is rounded to the type; its sum is not; then the result is
        want = v[best:best + 1].double().expand(n - best, 1, dim)
        check(got[best:], want, (torch.finfo(dtype).eps + 2.0 ** -15) * want.abs() + 2.0 ** -24)
        paged = Paged(generator(1), kk, v, [n], 16)
        got = decode_attention(one[-1:], paged.k, paged.v, torch.tensor([n], dtype=torch.int32, device="cuda"), paged.tables,
                               scale=1.0)
        assert torch.equal(got, v[best:best + 1])


def test_infinite_and_lowest_scores():
    # a key at the type's lowest value (its scores are -inf or of the order of the largest float), one of zeros
    q = torch.ones(3, 2, 64, dtype=BF, device="cuda")
    k = torch.zeros(3, 2, 64, dtype=BF, device="cuda")
    k[1] = torch.finfo(BF).min
    v = torch.arange(3, device="cuda", dtype=BF)[:, None, None].expand(3, 2, 64).contiguous()
    got = prefill_attention(q, k, v, cumulated([3]), cumulated([3]), 3, 3)
    assert torch.equal(got[:, 0, 0].float().cpu(), torch.tensor([0.0, 0.0, 1.0]))


DECODE = [  # dtype, heads, kv heads, dim, lengths
    (BF, 16, 8, 128, [1]),
    (BF, 16, 8, 128, [300]),
    (HF, 32, 8, 128, [63, 64, 65, 0, 1, 500]),
    (BF, 4, 4, 128, [1000, 17]),
    (BF, 7, 1, 128, [129, 2048]),
    (HF, 24, 2, 128, [333, 64]),                    # 12 heads of a group
    (BF, 64, 2, 64, [200, 31, 90]),                  # 32
    (HF, 100, 1, 64, [70, 200]),
    (BF, 6, 2, 80, [77, 400]),
    (HF, 4, 2, 8, [77, 400]),
    (BF, 10, 5, 96, [300] * 20),
    (BF, 32, 8, 128, [20000]),
    (BF, 4, 1, 128, [30000, 3, 200]),
    (HF, 16, 8, 128, [5 + 13 * i for i in range(100)]),
    (BF, 2, 1, 64, [0, 0, 0]),
    (BF, 2, 1, 64, [i % 3 for i in range(700)]),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: ids(c)[:60])
@pytest.mark.parametrize("page", [16, 48, 256])
def test_decode(case, page):
    dtype, heads, kv, dim, keys = case
    n = len(keys)
    gen, q, k, v = prefill_case(11, dtype, heads, kv, dim, [1] * n, keys)
    paged = Paged(gen, k, v, keys, page)
    lengths = torch.tensor(keys, dtype=torch.int32, device="cuda")
    want, tol = packed_reference(q, k, v, [1] * n, keys, dim ** -0.5)
    got = decode_attention(q, paged.k, paged.v, lengths, paged.tables)
    check(got, want, tol)
    again = decode_attention(q, paged.k, paged.v, lengths, paged.tables)
    assert torch.equal(got, again)                              # the same bits
    # tables wider than the longest sequence, as a captured batch has them
    wide = torch.full((n, paged.tables.shape[1] + 500), -1, dtype=torch.int32, device="cuda")
    wide[:, :paged.tables.shape[1]] = paged.tables
    out = torch.empty_like(q)
    check(decode_attention(q, paged.k, paged.v, lengths, wide, out=out), want, tol)
    assert device_status_ok()


def test_lengths_are_cut_to_the_tables():
    gen, q, k, v = prefill_case(12, BF, 4, 2, 128, [1, 1], [64, 128])
    paged = Paged(gen, k, v, [64, 128], 64)
    lengths = torch.tensor([-5, 100000], dtype=torch.int32, device="cuda")
    got = decode_attention(q, paged.k, paged.v, lengths, paged.tables)
    want, tol = packed_reference(q, k, v, [1, 1], [64, 128], 128 ** -0.5)
    check(got[1:], want[1:], tol[1:])
    assert torch.equal(got[:1], torch.zeros_like(got[:1]))
    assert device_status_ok()


@pytest.mark.parametrize("bad", [-1, 6, 1 << 30])
def test_pages_outside_of_the_cache_count_as_zeros_and_are_told(bad):
    keys, page = [100, 150], 48
    gen, q, k, v = prefill_case(13, BF, 4, 2, 128, [1, 1], keys)
    paged = Paged(gen, k, v, keys, page, spare=0)
    assert paged.k.shape[0] == 7
    bad = 7 if bad == 6 else bad
    paged.tables[0, 1] = bad
    lengths = torch.tensor(keys, dtype=torch.int32, device="cuda")
    k, v = k.clone(), v.clone()
    k[48:96] = 0
    v[48:96] = 0
    want, tol = packed_reference(q, k, v, [1, 1], keys, 128 ** -0.5)
    check(decode_attention(q, paged.k, paged.v, lengths, paged.tables), want, tol)
    torch.cuda.synchronize()
    with pytest.raises(_lib.B200QError, match="0xa01"):
        _lib.check_device()
    got = prefill_attention(q, paged.k, paged.v, cumulated([1, 1]), cumulated(keys), 1, 150, block_tables=paged.tables)
    check(got, want, tol)
    torch.cuda.synchronize()
    with pytest.raises(_lib.B200QError, match="0xa01"):
        _lib.check_device()


def test_a_captured_step_follows_lengths_tables_and_slots():
    keys = [500, 3, 70]
    gen, q, k, v = prefill_case(14, BF, 16, 8, 128, [1] * 3, keys)
    paged = Paged(gen, k, v, keys, 16, spare=20)
    kc, vc = paged.k.clone(), paged.v.clone()
    new_k, new_v = rows(gen, 3, 8, 128, BF), rows(gen, 3, 8, 128, BF)
    tables = torch.full((3, 64), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")
    slots = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def step():
        store_kv(new_k, new_v, kc, vc, slots)
        decode_attention(q, kc, vc, lengths, tables, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    second = torch.cuda.CUDAGraph()      # shares nothing with the first but the tensors
    with torch.cuda.graph(second):
        step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, torch.zeros_like(out))
    tables[:, :paged.tables.shape[1]] = paged.tables
    lengths.copy_(torch.tensor(keys))
    last = [paged.slots[sum(keys[:i + 1]) - 1].item() for i in range(3)]
    slots.copy_(torch.tensor(last))
    for i in range(3):
        k[sum(keys[:i + 1]) - 1], v[sum(keys[:i + 1]) - 1] = new_k[i], new_v[i]
    want, tol = packed_reference(q, k, v, [1] * 3, keys, 128 ** -0.5)
    for g in (graph, second):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        check(out, want, tol)


def test_two_streams_at_once():
    keys = [20000, 40]
    gen, q, k, v = prefill_case(15, BF, 8, 2, 128, [1, 1], keys)
    paged = Paged(gen, k, v, keys, 64)
    lengths = torch.tensor(keys, dtype=torch.int32, device="cuda")
    want, tol = packed_reference(q, k, v, [1, 1], keys, 128 ** -0.5)
    want2, tol2 = packed_reference(q * 0.5, k, v, [1, 1], keys, 128 ** -0.5)
    half = q * 0.5
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(decode_attention((q, half)[i], paged.k, paged.v, lengths, paged.tables))
                got[i].append(prefill_attention((q, half)[i], k, v, cumulated([1, 1]), cumulated(keys), 1, 20000))
    torch.cuda.synchronize()
    for x in got[0]:
        check(x, want, tol)
    for x in got[1]:
        check(x, want2, tol2)


@pytest.mark.parametrize("dtype,heads,dim,page,tokens", [(BF, 8, 128, 256, 64), (HF, 8, 128, 16, 1000), (BF, 1, 8, 16, 1),
                                                          (HF, 5, 80, 48, 77), (BF, 2, 264, 32, 30), (BF, 64, 128, 16, 9)])
@pytest.mark.parametrize("wide", [0, 24])
def test_store(dtype, heads, dim, page, tokens, wide):
    gen = generator(21)
    pages = tokens // page + 3
    cache = torch.randn(2, pages, page, heads, dim, generator=gen, device="cuda").to(dtype)
    k, v = rows(gen, tokens, heads, dim, dtype, wide=wide), rows(gen, tokens, heads, dim, dtype, wide=2 * wide)
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].to(torch.int32)
    slots[::5] = -1
    want = cache.clone()
    kept = slots >= 0
    want[0].flatten(0, 1)[slots[kept].long()] = k[kept]
    want[1].flatten(0, 1)[slots[kept].long()] = v[kept]
    store_kv(k, v, cache[0], cache[1], slots)
    assert torch.equal(cache, want)
    # heads outside of positions
    turned = torch.zeros(2, pages, heads, page, dim, dtype=dtype, device="cuda").transpose(2, 3)
    store_kv(k, v, turned[0], turned[1], slots)
    assert torch.equal(turned[0].flatten(0, 1)[slots[kept].long()], k[kept]) and int((turned != 0).sum()) <= 2 * k[kept].numel()
    store_kv(k[:0], v[:0], cache[0], cache[1], slots[:0])
    assert torch.equal(cache, want) and device_status_ok()


def test_store_outside_of_the_cache_is_skipped_and_told():
    cache = torch.zeros(2, 2, 16, 2, 64, dtype=BF, device="cuda")
    guarded = cache[:, :1]
    k = torch.ones(3, 2, 64, dtype=BF, device="cuda")
    store_kv(k, k, guarded[0], guarded[1], torch.tensor([16, 3, -7], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(_lib.B200QError, match="0xa02"):
        _lib.check_device()
    assert int(cache.sum()) == 2 * 2 * 64 and int(cache[:, 0, 3].sum()) == 2 * 2 * 64


def test_offsets_beyond_32_bits():
    # 2^31 elements lie between the first and the last page of a cache of 4.4 GB
    pages, page, kv, dim = 4200, 256, 16, 128
    cache = torch.empty(1, pages, page, kv, dim, dtype=BF, device="cuda")
    assert (pages - 1) * page * kv * dim > 1 << 31
    kc = cache[0]
    gen, q, k, v = prefill_case(16, BF, 16, 16, 128, [1], [300])
    tables = torch.tensor([[pages - 1, 1]], dtype=torch.int32, device="cuda")
    slots = torch.cat([torch.arange(256) + (pages - 1) * page, torch.arange(44) + page]).to(torch.int32).cuda()
    kc[pages - 1], kc[1], kc[2] = 0, 0, 0
    store_kv(k, k, kc, kc, slots)          # keys are the values as well
    lengths = torch.tensor([300], dtype=torch.int32, device="cuda")
    want, tol = packed_reference(q, k, k, [1], [300], 128 ** -0.5)
    check(decode_attention(q, kc, kc, lengths, tables), want, tol)
    check(prefill_attention(q, kc, kc, cumulated([1]), cumulated([300]), 1, 300, block_tables=tables), want, tol)
    copy_pages(kc, [pages - 1], [2])
    assert torch.equal(kc[2], kc[pages - 1]) and torch.equal(kc[2, :, :, :], k[:256])


@pytest.mark.parametrize("dtype,lead,page,heads,dim", [(BF, (2, 3), 16, 2, 64), (HF, (), 256, 1, 8), (torch.int8, (2, 5), 16, 1, 48),
                                                       (BF, (4,), 128, 8, 128)])
@pytest.mark.parametrize("count", [1, 5, 700])
def test_copy_pages(dtype, lead, page, heads, dim, count):
    pages = 2 * count + 3
    cache = torch.randint(-100, 100, (*lead, pages, page, heads, dim), device="cuda").to(dtype)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(count)).tolist()
    src, dst = order[:count], order[count:2 * count]
    src[-1] = src[0]                                     # one page to two places
    want = cache.clone()
    want[..., dst, :, :, :] = cache[..., src, :, :, :]
    copy_pages(cache, src, dst)
    assert torch.equal(cache, want)
    copy_pages(cache, [], [])
    if lead:                                              # one layer's part
        part = cache[:, -1] if len(lead) > 1 else cache[-1]
        want_part = part.clone()
        want_part[..., dst[:1], :, :, :] = part[..., src[:1], :, :, :]
        rest = cache.clone()
        copy_pages(part, src[:1], dst[:1])
        assert torch.equal(part, want_part)
        (rest[:, -1] if len(lead) > 1 else rest[-1]).copy_(want_part)
        assert torch.equal(cache, rest)


def test_a_captured_copy_keeps_its_pairs():
    cache = torch.randn(2, 2, 6, 16, 2, 64, device="cuda").to(BF)
    src, dst = [0, 1], [4, 5]
    copy_pages(cache, [2], [3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy_pages(cache, src, dst)
    src[:], dst[:] = [2, 2], [0, 1]
    cache[:, :, 0] += 1
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(cache[:, :, [0, 1]], cache[:, :, [4, 5]])

"""The attention operators as an engine uses them together, and what a user may do with single calls."""
import pytest
import torch

from attn_util import Paged, check, cumulated, packed_reference, reference, rows
from gpu_util import device_status_ok
from tiny_vllm_b200 import _lib
from tiny_vllm_b200.attention import copy_pages, decode_attention, prefill_attention, store_kv
from tiny_vllm_b200.layers.attention import Attention
from tiny_vllm_b200.utils.context import reset_context, set_context

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Engine:
    """Pages, tables and slots of a few sequences over a cache of several layers, as a block manager keeps them."""

    def __init__(self, layers, pages, page, kv, dim, dtype):
        self.cache = torch.full((2, layers, pages, page, kv, dim), float("nan"), dtype=dtype, device="cuda")
        self.page, self.free, self.tables, self.lengths = page, list(range(pages))[::-1], {}, {}

    def extend(self, name, n):
        """Slots of n more positions."""
        table, m = self.tables.setdefault(name, []), self.lengths.get(name, 0)
        while len(table) * self.page < m + n:
            table.append(self.free.pop())
        self.lengths[name] = m + n
        return [table[j // self.page] * self.page + j % self.page for j in range(m, m + n)]

    def table_tensor(self, names, width=None):
        width = width or max(len(self.tables[n]) for n in names)
        return ints([self.tables[n] + [-1] * (width - len(self.tables[n])) for n in names])


@pytest.mark.parametrize("dtype,heads,kv,dim,page", [(BF, 16, 8, 128, 16), (HF, 8, 2, 64, 32), (BF, 4, 4, 128, 256)])
def test_prompts_chunks_decoding_forks_and_compaction(dtype, heads, kv, dim, page):
    gen, layers, scale = generator(1), 2, dim ** -0.5
    e = Engine(layers, 80 if page < 256 else 24, page, kv, dim, dtype)
    stack = [Attention(heads, dim, scale, kv) for _ in range(layers)]
    for i, layer in enumerate(stack):
        layer.k_cache, layer.v_cache = e.cache[0, i], e.cache[1, i]
    seen = {}      # name -> per layer (k, v) so far

    def new(n):
        return [tuple(rows(gen, n, h, dim, dtype, g) for h, g in ((heads, 2.0), (kv, 1.0), (kv, 1.0))) for _ in range(layers)]

    def remember(name, parts):
        old = seen.get(name)
        seen[name] = [(k, v) if old is None else (torch.cat([old[i][0], k]), torch.cat([old[i][1], v]))
                      for i, (_, k, v) in enumerate(parts)]

    def step(names, counts, is_prefill):
        parts = {n: new(c) for n, c in zip(names, counts)}
        slots = sum((e.extend(n, c) for n, c in zip(names, counts)), [])
        for n in names:
            remember(n, parts[n])
        lengths = [e.lengths[n] for n in names]
        cached = any(m > c for m, c in zip(lengths, counts))
        if is_prefill:
            set_context(True, cumulated(counts), cumulated(lengths), max(counts), max(lengths), ints(slots),
                        block_tables=e.table_tensor(names) if cached else None)
        else:
            set_context(False, slot_mapping=ints(slots + [-1] * 2), context_lens=ints(lengths + [0] * 2),
                        block_tables=torch.cat([e.table_tensor(names, 40), torch.full_like(e.table_tensor(names, 40)[:1], -1).expand(2, -1)]))
        for i, layer in enumerate(stack):
            q, k, v = (torch.cat([parts[n][i][x] for n in names]) for x in range(3))
            if not is_prefill:      # a captured batch's padding
                q, k, v = (torch.cat([t, torch.full_like(t[:1], float("nan")).expand(2, -1, -1)]) for t in (q, k, v))
            got = layer(q.flatten(1), k.flatten(1), v.flatten(1)).view(-1, heads, dim)
            want, tol, at = [], [], 0
            for n, c in zip(names, counts):
                x, y = reference(parts[n][i][0], *seen[n][i], scale)
                want.append(x), tol.append(y)
            check(got[:sum(counts)], torch.cat(want), torch.cat(tol))
            if not is_prefill:
                assert torch.equal(got[sum(counts):], torch.zeros_like(got[sum(counts):]))
        reset_context()

    step(["a", "b", "c"], [70, 1, 300], True)                     # prompts
    step(["a", "b"], [40, 130], True)                              # chunks behind what is cached
    for _ in range(3):
        step(["a", "c", "b"], [1, 1, 1], False)
    # fork: full pages are shared, the last one is copied
    old = e.tables["c"]
    if e.lengths["c"] % page:
        fresh = e.free.pop()
        copy_pages(e.cache, [old[-1]], [fresh])
        e.tables["d"] = old[:-1] + [fresh]
    else:
        e.tables["d"] = list(old)
    e.lengths["d"], seen["d"] = e.lengths["c"], list(seen["c"])
    step(["c", "d", "a"], [1, 1, 1], False)
    step(["d", "c"], [5, 9], True)
    # compaction: pages from the end of the cache go to free ones at its beginning
    used = sorted({p for t in e.tables.values() for p in t}, reverse=True)
    holes = sorted(set(range(e.cache.shape[2])) - set(used))
    moves = [(s, d) for s, d in zip(used, holes) if d < s]
    copy_pages(e.cache, [s for s, _ in moves], [d for _, d in moves])
    place = dict(moves)
    e.tables = {n: [place.get(p, p) for p in t] for n, t in e.tables.items()}
    e.free = sorted(set(range(e.cache.shape[2])) - {p for t in e.tables.values() for p in t}, reverse=True)
    for s, _ in moves:
        e.cache[:, :, s] = float("nan")
    step(["a", "b", "c", "d"], [1, 1, 1, 1], False)
    step(["b", "e"], [200, 33], True)
    assert device_status_ok()


@pytest.mark.parametrize("queries,prefixes", [([50, 3], [0, 0]), ([900, 1100, 700, 30], [0] * 4), ([20], [6000])],
                         ids=["direct", "listed", "cut"])
def test_a_captured_prefill_follows_its_lengths(queries, prefixes):
    keys = [n + m for n, m in zip(queries, prefixes)]
    gen = generator(2)
    q, k, v = rows(gen, sum(queries), 8, 128, BF, 2.0), rows(gen, sum(keys), 2, 128, BF), rows(gen, sum(keys), 2, 128, BF)
    cu_q, cu_k, out = cumulated(queries), cumulated(keys), torch.empty_like(q)

    def run():
        prefill_attention(q, k, v, cu_q, cu_k, max(queries), max(keys), out=out)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    out.zero_()
    graph.replay()
    want, tol = packed_reference(q, k, v, queries, keys, 128 ** -0.5)
    check(out, want, tol)
    first = out.clone()
    graph.replay()
    assert torch.equal(first, out)               # the same bits
    # other lengths in the same buffers
    queries = [max(1, n // 3) for n in queries]
    keys = [n + m // 2 for n, m in zip(queries, prefixes)]
    cu_q.copy_(cumulated(queries))
    cu_k.copy_(cumulated(keys))
    out.fill_(3.0)
    graph.replay()
    want, tol = packed_reference(q[:sum(queries)], k[:sum(keys)], v[:sum(keys)], queries, keys, 128 ** -0.5)
    check(out[:sum(queries)], want, tol)
    assert torch.equal(out[sum(queries):], torch.full_like(out[sum(queries):], 3.0))
    assert device_status_ok()


@pytest.mark.parametrize("kind", ["nan", "inf", "-inf"])
def test_a_key_that_is_not_finite_reaches_the_rows_that_see_it(kind):
    # every column of a tile of keys, whichever way its exponential is taken
    n = 160
    gen = generator(3)
    q, k, v = rows(gen, n, 2, 64, BF), rows(gen, n, 1, 64, BF), rows(gen, n, 1, 64, BF)
    queries = [n] * 130
    big_q = torch.cat([q] * 130)
    big_k, big_v = torch.cat([k] * 130), torch.cat([v] * 130)
    where = torch.arange(130, device="cuda")
    big_k[where * n + where, 0, :] = 0
    big_k[where * n + where, 0, 5] = float(kind)
    got = prefill_attention(big_q, big_k, big_v, cumulated(queries), cumulated(queries), n, n).unflatten(0, (130, n))
    want, tol = reference(q, k, v, 64 ** -0.5)
    for i in range(130):
        check(got[i, :i], want[:i], tol[:i])
        s = q[i:, :, 5].float() * float(kind)        # the score of the key at i, up to a positive factor
        bad = s.isnan() | (s == float("inf"))
        rest = got[i, i:]
        assert rest[bad].isnan().all(), i
        assert rest[~bad].isfinite().all(), i
    lengths = torch.full((130,), n, dtype=torch.int32, device="cuda")
    paged = Paged(gen, big_k, big_v, queries, 32)
    last = torch.arange(130, device="cuda") * n + n - 1
    dec = decode_attention(big_q[last], paged.k, paged.v, lengths, paged.tables)
    s = q[-1, :, 5].float() * float(kind)
    bad = s.isnan() | (s == float("inf"))
    assert dec[:, bad].isnan().all() and dec[:, ~bad].isfinite().all()


def test_thousands_of_sequences():
    queries = [i % 4 for i in range(5000)]
    gen = generator(4)
    q, k, v = rows(gen, sum(queries), 4, 64, BF, 2.0), rows(gen, sum(queries), 2, 64, BF), rows(gen, sum(queries), 2, 64, BF)
    got = prefill_attention(q, k, v, cumulated(queries), cumulated(queries), 3, 3)
    # padded to three rows, in 64 bits
    pick = [i for i in range(0, 5000, 37)]
    starts = torch.tensor([0] + queries).cumsum(0)
    for b in pick:
        a, n = int(starts[b]), queries[b]
        want, tol = reference(q[a:a + n], k[a:a + n], v[a:a + n], 64 ** -0.5)
        check(got[a:a + n], want, tol)
    assert got.isfinite().all() and device_status_ok()


def test_lengths_that_do_not_rise_are_told_and_stay_in_bounds():
    # far more work than rows: the list ends where its memory does
    n = 400
    gen = generator(5)
    q, k, v = rows(gen, n, 16, 64, BF), rows(gen, n, 1, 64, BF), rows(gen, n, 1, 64, BF)
    cu = ints([0, n] * 300 + [0])
    out = torch.full((n + 8, 16, 64), 5.0, dtype=BF, device="cuda")
    prefill_attention(q, k, v, cu, cu, n, n, out=out[:n])
    torch.cuda.synchronize()
    with pytest.raises(_lib.B200QError, match="0xa03"):
        _lib.check_device()
    assert torch.equal(out[n:], torch.full_like(out[n:], 5.0))
    # beyond the tensors
    cu = ints([-7, 200, 900])
    prefill_attention(q, k, v, cu, cu, n, n, out=out[:n])
    torch.cuda.synchronize()
    _lib.lib().b200q_device_status()
    assert torch.equal(out[n:], torch.full_like(out[n:], 5.0))


@pytest.mark.parametrize("heads,kv", [(32, 8), (16, 16)])
def test_a_long_prompt_and_its_last_token(heads, kv):
    n = 5000
    gen = generator(6)
    q, k, v = rows(gen, n, heads, 128, BF, 2.0), rows(gen, n, kv, 128, BF), rows(gen, n, kv, 128, BF)
    got = prefill_attention(q, k, v, cumulated([n]), cumulated([n]), n, n)
    again = prefill_attention(q, k, v, cumulated([n]), cumulated([n]), n, n)
    assert torch.equal(got, again)
    for a, b in ((0, 300), (2400, 2600), (4800, 5000)):      # each against its own prefix
        want, tol = reference(q[a:b], k[:b], v[:b], 128 ** -0.5)
        check(got[a:b], want, tol)
    paged = Paged(gen, k, v, [n], 16)
    dec = decode_attention(q[-1:], paged.k, paged.v, ints([n]), paged.tables)
    check(dec, want[-1:], tol[-1:])


def test_results_on_a_side_stream_and_a_given_output():
    gen = generator(7)
    q, k, v = rows(gen, 300, 8, 128, HF), rows(gen, 300, 8, 128, HF), rows(gen, 300, 8, 128, HF)
    want, tol = reference(q, k, v, 128 ** -0.5)
    side, out = torch.cuda.Stream(), torch.zeros(2, 300, 8, 128, dtype=HF, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = prefill_attention(q, k, v, cumulated([300]), cumulated([300]), 300, 300, out=out[1])
    torch.cuda.current_stream().wait_stream(side)
    assert r.data_ptr() == out[1].data_ptr()
    check(out[1], want, tol)
    assert torch.equal(out[0], torch.zeros_like(out[0]))
    with torch.inference_mode():
        check(prefill_attention(q, k, v, cumulated([300]), cumulated([300]), 300, 300), want, tol)

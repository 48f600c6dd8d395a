"""Performance cases of the attention operators over a paged key-value cache.

A serving engine runs them in every decoder layer, between the qkv projection and the output
projection, and between steps:

* ``prefill``   attention over whole prompts: sequences of different lengths packed one after another,
  grouped heads, causal.  With ``pages`` the keys and values of a sequence stand in cache pages and begin
  with a cached prefix (prefix caching, chunked prefill);
* ``decode``    attention of one new token per sequence over its cache pages;
* ``store``     the new tokens' keys and values go to their slots of the cache;
* ``copy``      pages of all layers are copied (a fork's last page, compaction).

With T the element type, per sequence with n queries and m >= n keys (bottom right aligned):

    o[i, h] = T(sum_j p[i, h, j] v[j, h / G]),   p = softmax over j <= i + m - n of scale q[i, h] . k[j, h / G]

A row that sees no key gives zeros.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

# heads of the benchmark's two models and of one rank of the larger one at TP = 8
HEADS_0_6B = {"heads": 16, "kv_heads": 8, "dim": 128}
HEADS_8B = {"heads": 32, "kv_heads": 8, "dim": 128}

# Cost limits of a drawn case, those of the largest listed ones: scores (queries x keys x heads, padded to the longest
# sequence), values of keys and values read, values stored or copied.
MAX_SCORES = 32 * 8192 * 8192
MAX_CACHE_VALUES = 2 * 131071 * 8 * 128
MAX_STORED = 2 * 16384 * 8 * 128
MAX_COPIED = 40 * 28 * 2 * 256 * 8 * 128


def listed():
    return [
        # a short prompt arrives alone: the smallest prefill, where latency counts
        {"name": "prefill 0.6b 23 tokens", "op": "prefill", **HEADS_0_6B, "dtype": "bf16", "pages": 0,
         "queries": "23", "prefixes": "0"},
        # a prefill batch of prompts of all lengths, one token among them
        {"name": "prefill 0.6b 8 prompts", "op": "prefill", **HEADS_0_6B, "dtype": "bf16", "pages": 0,
         "queries": "1999,512,77,1024,1,300,2048,130", "prefixes": "0,0,0,0,0,0,0,0"},
        # one long prompt of the larger model
        {"name": "prefill 8b 8192 tokens", "op": "prefill", **HEADS_8B, "dtype": "bf16", "pages": 0,
         "queries": "8192", "prefixes": "0"},
        # prompts whose beginning is cached already, and chunks of longer ones, out of the engine's 256-token pages
        {"name": "prefill 8b cached prefixes", "op": "prefill", **HEADS_8B, "dtype": "fp16", "pages": 256,
         "queries": "256,33,512,1,700", "prefixes": "4096,7936,0,1500,300"},
        # one user at the beginning of an answer: the smallest decode step
        {"name": "decode 0.6b 1 x 300", "op": "decode", **HEADS_0_6B, "dtype": "bf16", "pages": 256,
         "sequences": 1, "shortest": 300, "longest": 300},
        # a batch of very different lengths in small pages
        {"name": "decode 8b 64 ragged fp16", "op": "decode", **HEADS_8B, "dtype": "fp16", "pages": 16,
         "sequences": 64, "shortest": 40, "longest": 8000},
        # the engine's full decode batch
        {"name": "decode 0.6b 512", "op": "decode", **HEADS_0_6B, "dtype": "bf16", "pages": 256,
         "sequences": 512, "shortest": 100, "longest": 2048},
        # one long document: the work of one sequence has to be spread over the GPU
        {"name": "decode 8b 1 x 131071", "op": "decode", **HEADS_8B, "dtype": "bf16", "pages": 256,
         "sequences": 1, "shortest": 131071, "longest": 131071},
        # a decode step's tokens, and a full prefill batch
        {"name": "store 64 tokens", "op": "store", **HEADS_0_6B, "dtype": "bf16", "pages": 256, "tokens": 64,
         "padded": 5},
        {"name": "store 16384 tokens", "op": "store", **HEADS_8B, "dtype": "fp16", "pages": 256,
         "tokens": 16384, "padded": 0},
        # two sequences fork: their last pages are copied in every layer; and a cache is compacted
        {"name": "copy 2 pages", "op": "copy", "kv_heads": 8, "dim": 128, "dtype": "bf16", "pages": 256,
         "layers": 28, "held": 16, "copied": 2},
        {"name": "copy 40 pages", "op": "copy", "kv_heads": 8, "dim": 128, "dtype": "fp16", "pages": 256,
         "layers": 28, "held": 96, "copied": 40},
    ]


def _log_int(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    op = rng.choice(("prefill", "prefill", "decode", "decode", "store", "copy"))
    case = {"op": op, "dtype": rng.choice(("bf16", "bf16", "fp16")), "dim": rng.choice((64, 80, 96, 128, 128, 128)),
            "kv_heads": rng.choice((1, 2, 4, 5, 8, 8)), "pages": rng.choice((16, 32, 48, 64, 128, 256, 256))}
    if op in ("prefill", "decode"):
        case["heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4, 4, 6, 7, 8))
    width = case["kv_heads"] * case["dim"]
    if op == "prefill":
        if rng.random() < 0.5:
            case["pages"] = 0
        n = _log_int(rng, 1, 32)
        top = _log_int(rng, 16, 8192)
        queries = [max(1, min(8192, _log_int(rng, 1, top))) for _ in range(n)]
        prefixes = [_log_int(rng, 1, 8192) - 1 if rng.random() < 0.5 else 0 for _ in range(n)]
        if rng.random() < 0.5:
            prefixes = [0] * n
        # fewer sequences until the padded scores fit
        while len(queries) * max(queries) * max(a + b for a, b in zip(queries, prefixes)) * case["heads"] > MAX_SCORES:
            if len(queries) > 1:
                queries.pop(), prefixes.pop()
            elif prefixes[0]:
                prefixes[0] //= 2
            else:
                queries[0] //= 2
        case |= {"queries": ",".join(map(str, queries)), "prefixes": ",".join(map(str, prefixes))}
    elif op == "decode":
        n = _log_int(rng, 1, 512)
        longest = max(1, min(_log_int(rng, 1, 131071), MAX_CACHE_VALUES // (2 * width * n)))
        case |= {"sequences": n, "longest": longest, "shortest": max(1, round(longest * rng.choice((0.01, 0.1, 1.0))))}
    elif op == "store":
        tokens = max(1, min(_log_int(rng, 1, 16384), MAX_STORED // (2 * width)))
        case |= {"tokens": tokens, "padded": rng.randrange(tokens // 4 + 1)}
    else:
        case["layers"] = rng.randint(1, 36)
        page = case["layers"] * 2 * case["pages"] * width
        copied = max(1, min(_log_int(rng, 1, 64), MAX_COPIED // page))
        case |= {"copied": copied, "held": 2 * copied + rng.randrange(copied + 1)}
    return case


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _context_lengths(case):
    """The contexts' lengths of a decode case: spread over their logarithm, the longest one among them."""
    rng = random.Random(case["sequences"])
    lengths = [_log_int(rng, case["shortest"], case["longest"]) for _ in range(case["sequences"])]
    lengths[rng.randrange(len(lengths))] = case["longest"]
    return lengths


def _lengths(case):
    """(queries, keys) of every sequence of a prefill or decode case."""
    if case["op"] == "decode":
        return [1] * case["sequences"], _context_lengths(case)
    queries = _numbers(case["queries"])
    return queries, [n + m for n, m in zip(queries, _numbers(case["prefixes"]))]


class _State:
    pass


def _cumulated(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def _random(gen, dtype, *shape):
    return torch.randn(shape, device="cuda", generator=gen, dtype=dtype)


def _paged(s, case, gen, keys):
    """A cache with a few pages more than the sequences take, and tables of pages in no order."""
    size = case["pages"]
    need = [-(-n // size) for n in keys]
    held = sum(need) + 3
    order = torch.randperm(held, device="cuda", generator=gen).to(torch.int32)
    s.cache = _random(gen, s.dtype, 2, held, size, case["kv_heads"], case["dim"])
    s.k, s.v = s.cache[0], s.cache[1]
    # a sequence's pages first, -1 behind them
    row = torch.repeat_interleave(torch.arange(len(keys)), torch.tensor(need)).cuda()
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    column = torch.arange(sum(need), device="cuda") - first[row]
    s.tables = torch.full((len(keys), max(need)), -1, dtype=torch.int32, device="cuda")
    s.tables[row, column] = order[: sum(need)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = _State()
    s.op, s.dtype, s.tables = case["op"], DTYPES[case["dtype"]], None
    if s.op in ("prefill", "decode"):
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        queries, keys = _lengths(case)
        s.scale = dim ** -0.5
        # queries and keys are normalised per head with a learnt gain, so that some heads look at few tokens
        gain = 1 + 1.5 * torch.rand(heads, 1, device="cuda", generator=gen)
        total = sum(queries)
        # q is what norm and rotation wrote; v is a part of the qkv projection's rows
        s.q = (torch.randn(total, heads, dim, device="cuda", generator=gen) * gain).to(s.dtype)
        if case["pages"]:
            _paged(s, case, gen, keys)
        else:
            s.k = _random(gen, s.dtype, sum(keys), kv, dim)
            s.v = _random(gen, s.dtype, sum(keys), (heads + 2 * kv) * dim)[:, (heads + kv) * dim:].unflatten(1, (kv, dim))
        s.max_q, s.max_k = max(queries), max(keys)
        if s.op == "prefill":
            s.cu_q, s.cu_k = _cumulated(queries), _cumulated(keys)
        else:
            s.lengths = torch.tensor(keys, dtype=torch.int32, device="cuda")
    elif s.op == "store":
        tokens, kv, dim = case["tokens"], case["kv_heads"], case["dim"]
        blocks = -(-tokens // case["pages"]) + 4
        s.cache = _random(gen, s.dtype, 2, blocks, case["pages"], kv, dim)
        s.new_k = _random(gen, s.dtype, tokens, kv, dim)
        s.new_v = _random(gen, s.dtype, tokens, 4 * kv * dim)[:, 3 * kv * dim:].unflatten(1, (kv, dim))
        # a decode batch has one slot in each of many pages, a prefill batch runs of them; padding comes last
        slots = torch.randperm(blocks * case["pages"], device="cuda", generator=gen)[:tokens].to(torch.int32)
        if tokens > 512:
            slots = slots.sort().values
        s.slots = slots
        if case["padded"]:
            s.slots[-case["padded"]:] = -1
    else:
        s.cache = _random(gen, s.dtype, 2, case["layers"], case["held"], case["pages"], case["kv_heads"], case["dim"])
        order = torch.randperm(case["held"], device="cuda", generator=gen).tolist()
        s.src, s.dst = order[: case["copied"]], order[case["copied"]: 2 * case["copied"]]
    return s


def _padded(rows, starts, lengths, longest):
    """Packed rows [T, ...] -> ([B, longest, ...] in 32 bits, truth of the places that hold one)."""
    place = torch.arange(longest, device="cuda")
    held = place < lengths[:, None]
    at = (starts[:, None] + place).clamp_(max=max(rows.shape[0] - 1, 0))
    return rows[at].float(), held


def _keys(s, lengths, starts, cache):
    """The keys or values of all sequences [B, Hkv, longest, D], zeros behind a sequence's end."""
    if s.tables is None:
        x, held = _padded(cache, starts, lengths, s.max_k)
    else:
        x = cache[s.tables.clamp(min=0).long()].flatten(1, 2)[:, : s.max_k].float()
        held = torch.arange(x.shape[1], device="cuda") < lengths[:, None]
    x.masked_fill_(~held[:, :, None, None], 0.0)
    return x.transpose(1, 2), held


def _attention(s):
    """Softmax attention of all sequences, padded to the longest one, in 32 bits."""
    kv = s.k.shape[-2]
    heads, dim = s.q.shape[1:]
    if s.op == "prefill":
        starts_q, starts_k = s.cu_q[:-1].long(), s.cu_k[:-1].long()
        lengths_q, lengths_k = (s.cu_q[1:] - s.cu_q[:-1]).long(), (s.cu_k[1:] - s.cu_k[:-1]).long()
        q, held_q = _padded(s.q, starts_q, lengths_q, s.max_q)
    else:
        starts_k, lengths_k = None, s.lengths.long()
        lengths_q = torch.ones_like(lengths_k)
        q, held_q = s.q[:, None].float(), None
    k, held_k = _keys(s, lengths_k, starts_k, s.k)
    v, _ = _keys(s, lengths_k, starts_k, s.v)
    n = q.shape[1]
    q = q.unflatten(2, (kv, heads // kv)).permute(0, 2, 3, 1, 4).flatten(2, 3)           # [B, Hkv, G n, D]
    p = torch.matmul(q, k.transpose(2, 3)).mul_(s.scale).unflatten(2, (heads // kv, n))
    last = torch.arange(n, device="cuda") + (lengths_k - lengths_q)[:, None]            # [B, n]
    hidden = (torch.arange(k.shape[2], device="cuda") > last[:, :, None]) | ~held_k[:, None]
    p.masked_fill_(hidden[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (heads // kv, n)).div_(torch.where(total > 0, total, 1.0))
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                                            # [B, n, H, D]
    return (o[held_q] if held_q is not None else o[:, 0]).to(s.dtype)


def _plain(s):
    if s.op in ("prefill", "decode"):
        return _attention(s)
    if s.op == "store":
        kept = s.slots >= 0
        slots = s.slots[kept].long()
        s.cache[0].flatten(0, 1)[slots] = s.new_k[kept]
        s.cache[1].flatten(0, 1)[slots] = s.new_v[kept]
    else:
        s.cache[:, :, s.dst] = s.cache[:, :, s.src]
    return s.cache


def _own(s):
    from tiny_vllm_b200.attention import copy_pages, decode_attention, prefill_attention, store_kv
    if s.op == "prefill":
        return prefill_attention(s.q, s.k, s.v, s.cu_q, s.cu_k, s.max_q, s.max_k, scale=s.scale, block_tables=s.tables)
    if s.op == "decode":
        return decode_attention(s.q, s.k, s.v, s.lengths, s.tables, scale=s.scale)
    if s.op == "store":
        store_kv(s.new_k, s.new_v, s.cache[0], s.cache[1], s.slots)
    else:
        copy_pages(s.cache, s.src, s.dst)
    return s.cache


def run(state):
    with torch.inference_mode():
        return _own(state) if own else _plain(state)


def work(case):
    if case["op"] in ("store", "copy"):
        width = case["kv_heads"] * case["dim"]
        if case["op"] == "store":
            tokens = case["tokens"] - case["padded"]
            return {"bytes": tokens * (2 * 2 * 2 * width) + 4 * case["tokens"], "flops": 0}
        return {"bytes": 2 * 2 * case["copied"] * case["layers"] * 2 * case["pages"] * width, "flops": 0}
    queries, keys = _lengths(case)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    # the pairs of a causal triangle at the bottom right of queries x keys
    pairs = sum(n * m - n * (n - 1) // 2 for n, m in zip(queries, keys))
    return {"bytes": 2 * 2 * sum(queries) * heads * dim + 2 * 2 * sum(keys) * kv * dim, "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    """Head by head and sequence by sequence, in 64 bits."""
    if case["op"] in ("store", "copy"):
        return None     # nothing is computed
    s = prepare(case, seed)
    queries, keys = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    at_q = at_k = 0
    for b, (n, m) in enumerate(zip(queries, keys)):
        if s.tables is None:
            k, v = s.k[at_k: at_k + m].double(), s.v[at_k: at_k + m].double()
        else:
            pages = s.tables[b, : -(-m // case["pages"])].tolist()
            k = torch.cat([s.k[p] for p in pages])[:m].double()
            v = torch.cat([s.v[p] for p in pages])[:m].double()
        for h in range(case["kv_heads"]):
            for i in range(0, n, 2048):      # blocks of queries
                q = s.q[at_q + i: at_q + min(n, i + 2048), h * group: (h + 1) * group].double()
                z = torch.einsum("igd,jd->gij", q, k[:, h]) / math.sqrt(case["dim"])
                seen = torch.ones(z.shape[1:], dtype=torch.bool, device="cuda").tril(m - n + i)
                z = z.masked_fill(~seen, -math.inf)
                out[at_q + i: at_q + i + q.shape[0], h * group: (h + 1) * group] = torch.einsum(
                    "gij,jd->igd", torch.softmax(z, dim=-1), v[:, h])
        at_q, at_k = at_q + n, at_k + m
    return out

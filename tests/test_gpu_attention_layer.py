"""A decoder layer's attention block as an engine's model file writes it, over the modules that
``install_under_nanovllm(replace_attention=True)`` puts under the engine's names: quantized qkv projection, norms and rotation of
queries and keys, the attention layer with a runner's cache and step context, output projection."""
import sys
import types

import pytest
import torch
from torch import nn

from attn_util import check, cumulated, reference
from gpu_util import device_status_ok
from oracle import quant_linear_oracle as O
from tiny_vllm_b200.integration import install_under_nanovllm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HIDDEN, HEADS, KV, DIM, PAGE = 512, 8, 2, 64, 16


@pytest.fixture
def installed():
    """The engine's package with nothing in it but the aliases."""
    def ours():
        return [name for name in sys.modules if name.split(".")[0] == "nanovllm"]
    before = {name: sys.modules.pop(name) for name in ours()}
    for name in ("nanovllm", "nanovllm.layers", "nanovllm.utils"):
        sys.modules[name] = types.ModuleType(name)
        sys.modules[name].__path__ = []
    install_under_nanovllm(replace_attention=True)
    yield
    for name in ours():
        del sys.modules[name]
    sys.modules.update(before)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def block(quant, flat):
    from nanovllm.layers.attention import Attention
    from nanovllm.layers.linear import QKVParallelLinear, RowParallelLinear

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.qkv_proj = QKVParallelLinear(HIDDEN, DIM, HEADS, KV, quantization=quant)
            self.o_proj = RowParallelLinear(HEADS * DIM, HIDDEN, quantization=quant)
            self.attn = Attention(HEADS, DIM, DIM ** -0.5, KV)

        def forward(self, positions, x):
            q, k, v = self.qkv_proj(x).split([HEADS * DIM, KV * DIM, KV * DIM], dim=-1)
            angle = positions[:, None] * 1e4 ** (-torch.arange(0, DIM, 2, device="cuda") / DIM)
            cos, sin = angle.cos()[:, None], angle.sin()[:, None]

            def norm_and_rotate(t, heads):
                t = t.unflatten(-1, (heads, DIM)).float()
                a, b = (t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)).chunk(2, -1)
                return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(BF)
            q, k = norm_and_rotate(q, HEADS), norm_and_rotate(k, KV)
            o = self.attn(q.flatten(1), k.flatten(1), v) if flat else self.attn(q, k, v.unflatten(-1, (KV, DIM)))
            assert o.shape == (q.flatten(1) if flat else q).shape
            self.seen = q, k, v.unflatten(-1, (KV, DIM)), o.view(-1, HEADS, DIM)
            return self.o_proj(o.flatten(1, -1))

    torch.set_default_dtype(BF)
    try:
        with torch.device("cuda"):
            model = Block()
    finally:
        torch.set_default_dtype(torch.float32)
    for layer in (model.qkv_proj, model.o_proj):
        if quant is None:
            layer.weight.data.normal_(0, 0.05, generator=torch.Generator("cuda").manual_seed(1))
        else:
            q, s = O.make_weight(*layer.qweight.shape, seed=layer.qweight.shape[0])
            layer.qweight.data.copy_(q)
            getattr(layer, "scales" if quant == "int8" else "w_scales").data.copy_(s)
    return model


@pytest.mark.parametrize("flat", [True, False], ids=["2d", "3d"])
@pytest.mark.parametrize("quant", [None, "int8", "w8a8"])
def test_prompts_cached_prefixes_and_captured_steps(installed, quant, flat):
    from nanovllm.utils.context import get_context, reset_context, set_context
    model, gen = block(quant, flat), torch.Generator("cuda").manual_seed(2)
    tables = [[9, 4, 0], [7, 2, 11, 1]]
    stored, lengths = [[], []], [0, 0]

    def slots(b, n):
        return [tables[b][p // PAGE] * PAGE + p % PAGE for p in range(lengths[b], lengths[b] + n)]

    def x(n):
        return torch.randn(n, HIDDEN, device="cuda", generator=gen).to(BF)

    def verify(counts, y):
        """The outputs of the tokens that were just worked on, against everything that their sequences have stored."""
        q, k, v, o = model.seen
        at = 0
        for b, n in enumerate(counts):
            stored[b].append((k[at:at + n].clone(), v[at:at + n].clone()))
            keys, values = (torch.cat(t) for t in zip(*stored[b]))
            want, tol = reference(q[at:at + n], keys, values, DIM ** -0.5)
            check(o[at:at + n], want, tol)
            lengths[b] += n
            at += n
        assert y.shape[1] == HIDDEN and bool(y[:at].isfinite().all())
        assert torch.equal(y, model.o_proj(o.flatten(1)))

    with torch.inference_mode():
        # a runner's warm-up: no cache yet
        set_context(True, cumulated([40]), cumulated([40]), 40, 40, ints([]), None, None)
        model(torch.arange(40, device="cuda"), x(40))
        reset_context()
        cache = torch.full((2, 12, PAGE, KV, DIM), float("nan"), dtype=BF, device="cuda")
        for module in model.modules():
            if hasattr(module, "k_cache") and hasattr(module, "v_cache"):
                module.k_cache, module.v_cache = cache[0], cache[1]
        for counts in ([21, 33], [5, 1]):      # prompts; then chunks behind what is cached
            after = [a + n for a, n in zip(lengths, counts)]
            positions = torch.cat([torch.arange(a, b) for a, b in zip(lengths, after)]).cuda()
            new = sum((slots(b, n) for b, n in enumerate(counts)), [])
            set_context(True, cumulated(counts), cumulated(after), max(counts), max(after), ints(new), None,
                        ints([t + [-1] * (4 - len(t)) for t in tables]) if lengths[0] else None)
            y = model(positions, x(sum(counts)))
            reset_context()
            verify(counts, y)
        # decode steps of two sequences in a captured batch of four
        inputs, positions = torch.zeros(4, HIDDEN, dtype=BF, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
        slot_mapping, context_lens, block_tables = ints([-1] * 4), ints([0] * 4), ints([[0] * 6] * 4)
        set_context(False, slot_mapping=slot_mapping, context_lens=context_lens, block_tables=block_tables)
        assert not get_context().is_prefill
        model(positions, inputs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model(positions, inputs)
        reset_context()
        for _ in range(3):
            inputs[:2].copy_(x(2))
            positions[:2].copy_(torch.tensor(lengths))
            slot_mapping[:2].copy_(ints(slots(0, 1) + slots(1, 1)))
            context_lens[:2].copy_(ints([n + 1 for n in lengths]))
            for b, t in enumerate(tables):
                block_tables[b, :len(t)] = ints(t)
            graph.replay()
            assert torch.equal(model.seen[3][2:], torch.zeros_like(model.seen[3][2:]))
            verify([1, 1], y)
    assert device_status_ok()

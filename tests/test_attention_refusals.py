"""What the attention entry points refuse, and what they share with the C header (no GPU: a stand-in that takes nothing, the
check for CUDA tensors off, host addresses that are never dereferenced)."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import tiny_vllm_b200  # noqa: F401
from tiny_vllm_b200 import _lib, build as b200_build
from tiny_vllm_b200.attention import cuda as A
from tiny_vllm_b200.utils import context

ROOT = Path(__file__).resolve().parent.parent
BF = torch.bfloat16


class TakesNothing:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture
def no_gpu(monkeypatch):
    monkeypatch.setattr(A, "_native", TakesNothing)
    monkeypatch.setattr(A, "_require_cuda", lambda *tensors: None)


def tensors(**other):
    t = {"q": torch.zeros(6, 4, 64, dtype=BF), "k": torch.zeros(9, 2, 64, dtype=BF), "v": torch.zeros(9, 2, 64, dtype=BF),
         "cu_q": torch.tensor([0, 2, 6], dtype=torch.int32), "cu_k": torch.tensor([0, 4, 9], dtype=torch.int32),
         "kc": torch.zeros(5, 16, 2, 64, dtype=BF), "vc": torch.zeros(5, 16, 2, 64, dtype=BF),
         "lens": torch.ones(6, dtype=torch.int32), "tables": torch.zeros(6, 2, dtype=torch.int32),
         "slots": torch.zeros(9, dtype=torch.int32), "out": None}
    t.update(other)
    return t


def prefill(t):
    return A.prefill_attention(t["q"], t["k"], t["v"], t["cu_q"], t["cu_k"], t.get("max_q", 4), 5, out=t["out"])


def paged(t):
    return A.prefill_attention(t["q"], t["kc"], t["vc"], t["cu_q"], t["cu_k"], 4, 5, block_tables=t["tables"][:2])


def decode(t):
    return A.decode_attention(t["q"], t["kc"], t["vc"], t["lens"], t["tables"], out=t["out"])


def store(t):
    return A.store_kv(t["k"], t["v"], t["kc"], t["vc"], t["slots"])


REFUSED = [
    (prefill, {"q": torch.zeros(6, 256, dtype=BF)}, "queries"),
    (prefill, {"q": torch.zeros(6, 4, 64)}, "expects"),
    (prefill, {"q": torch.zeros(6, 3, 64, dtype=BF)}, "3 query heads are not a multiple of 2"),
    (prefill, {"k": torch.zeros(9, 2, 64, dtype=torch.float16)}, "of the queries' type"),
    (prefill, {"v": torch.zeros(8, 2, 64, dtype=BF)}, "expects k and v"),
    (prefill, {"cu_q": torch.tensor([0, 2, 6])}, "cu_seqlens_q must be a 1-D int32"),
    (prefill, {"cu_k": torch.tensor([0, 9], dtype=torch.int32)}, "one entry per sequence"),
    (prefill, {"max_q": -1}, "must not be negative"),
    (prefill, {"out": torch.zeros(6, 4, 32, dtype=BF)}, "out must be a contiguous"),
    (prefill, {"out": torch.zeros(6, 64, 4, dtype=BF).transpose(1, 2)}, "out must be a contiguous"),
    (paged, {"vc": torch.zeros(5, 16, 2, 32, dtype=BF)}, "caches"),
    (paged, {"kc": torch.zeros(5, 16, 2, 64), "vc": torch.zeros(5, 16, 2, 64)}, "caches"),
    (paged, {"tables": torch.zeros(1, 2, dtype=torch.int32)}, "row of pages for each of the 2"),
    (paged, {"tables": torch.zeros(2, 0, dtype=torch.int32)}, "row of pages for each of the 2"),
    (paged, {"kc": torch.zeros(5, 16, 2, 67, dtype=BF)[..., :64], "vc": torch.zeros(5, 16, 2, 67, dtype=BF)[..., :64]}, "16-byte"),
    (paged, {"kc": torch.zeros(1, 16, 2, 64, dtype=BF).expand(5, -1, -1, -1)}, "16-byte"),
    (decode, {"q": torch.zeros(6, 4, 32, dtype=BF)}, "do not fit"),
    (decode, {"lens": torch.ones(5, dtype=torch.int32)}, "an entry for each of the 6"),
    (decode, {"lens": torch.ones(6)}, "context_lens must be a 1-D int32"),
    (decode, {"tables": torch.zeros(6, dtype=torch.int32)}, "block_tables must be a 2-D int32"),
    (decode, {"kc": torch.zeros(0, 16, 2, 64, dtype=BF), "vc": torch.zeros(0, 16, 2, 64, dtype=BF)}, "no page"),
    (store, {"k": torch.zeros(9, 128, dtype=BF)}, "expects"),
    (store, {"v": torch.zeros(9, 2, 64, dtype=torch.float16)}, "expects"),
    (store, {"slots": torch.zeros(8, dtype=torch.int32)}, "one entry per token"),
    (store, {"slots": torch.zeros(9, dtype=torch.int64)}, "int32"),
    (store, {"kc": torch.zeros(5, 16, 4, 64, dtype=BF), "vc": torch.zeros(5, 16, 4, 64, dtype=BF)}, "do not fit"),
]


@pytest.mark.parametrize("call,other,message", REFUSED, ids=[f"{c.__name__}-{m[:25]}" for c, _, m in REFUSED])
def test_what_is_wrong_is_named(no_gpu, call, other, message):
    with pytest.raises(RuntimeError, match=message):
        call(tensors(**other))


@pytest.mark.parametrize("dim", [4, 63, 136, 256])
def test_dims_that_no_kernel_takes(no_gpu, dim):
    t = tensors(q=torch.zeros(6, 4, dim, dtype=BF), k=torch.zeros(9, 2, dim, dtype=BF), v=torch.zeros(9, 2, dim, dtype=BF))
    with pytest.raises(_lib.B200QError) as e:
        prefill(t)
    assert e.value.code == _lib.ERR_UNSUPPORTED_SHAPE


@pytest.mark.parametrize("call", [prefill, paged, decode, store])
def test_tensors_on_two_devices_are_named(no_gpu, call):
    name = "q" if call is not store else "slots"
    t = tensors()
    t[name] = t[name].to("meta")
    with pytest.raises(RuntimeError, match="must be on one GPU"):
        call(t)


@pytest.mark.parametrize("call", [prefill, paged, decode, store, lambda t: A.copy_pages(t["kc"], [0], [1])])
def test_cpu_tensors_are_refused(monkeypatch, call):
    monkeypatch.setattr(A, "_native", TakesNothing)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        call(tensors())


@pytest.mark.parametrize("src,dst,message", [
    ([0, 1], [2], "2 sources and 1"), ([0], [5], "not one of the cache's 5"), ([-1], [2], "not one of"),
    ([0, 1], [2, 2], "stands twice"), ([0, 1], [2, 0], "a source as well"), ([3], [3], "a source as well"),
    (torch.tensor([0]), [1], "lists of page numbers"), ([0.0], [1], "lists of page numbers")])
def test_page_copies_that_are_refused(no_gpu, src, dst, message):
    with pytest.raises(ValueError, match=message):
        A.copy_pages(torch.zeros(2, 5, 16, 2, 64, dtype=BF), src, dst)


def test_a_cache_whose_layers_are_not_evenly_spaced_is_refused(no_gpu):
    with pytest.raises(RuntimeError, match="evenly spaced"):
        A.copy_pages(torch.zeros(2, 3, 5, 16, 2, 64, dtype=BF).transpose(0, 1)[:2], [0], [1])


def test_nothing_to_do(no_gpu):
    t = tensors()
    assert prefill(dict(t, q=t["q"][:0], cu_q=torch.zeros(3, dtype=torch.int32))).shape == (0, 4, 64)
    assert decode(dict(t, q=t["q"][:0], lens=t["lens"][:0], tables=t["tables"][:0])).shape == (0, 4, 64)
    assert store(dict(t, k=t["k"][:0], v=t["v"][:0], slots=t["slots"][:0])) is None
    assert A.copy_pages(t["kc"], [], []) is None


# ------------------------------------------------------------------------------- C interface
@pytest.fixture(scope="module")
def L():
    b200_build.build()
    return _lib.lib()


def address():
    buf = ctypes.create_string_buffer(4096 + 64)
    p = (ctypes.addressof(buf) + 63) & ~63
    address.keep = buf
    return p


def arguments(**other):
    p = address()
    a = _lib.Attention()
    a.q, a.k, a.v = _lib.View(p, 0, 256, 64), _lib.View(p, 2048, 128, 64), _lib.View(p, 2048, 128, 64)
    a.out = a.cu_q = a.cu_k = a.lengths = a.tables = p
    a.table_stride = 4
    a.tokens, a.key_tokens, a.sequences, a.heads, a.kv_heads, a.dim = 6, 9, 6, 4, 2, 64
    a.pages, a.page_size, a.table_width, a.max_q, a.max_k, a.causal, a.dtype, a.scale = 5, 16, 4, 4, 5, 1, 1, 0.125
    for name, value in other.items():
        view, _, field = name.partition("_of_")
        if field:
            setattr(getattr(a, field), view, value)
        else:
            setattr(a, name, value)
    return a


ARGUMENTS = [
    ({"out": None}, _lib.ERR_NULL_POINTER), ({"data_of_k": None}, _lib.ERR_NULL_POINTER), ({"tables": None}, _lib.ERR_NULL_POINTER),
    ({"dtype": 7}, _lib.ERR_BAD_ARGUMENT), ({"scale": float("nan")}, _lib.ERR_BAD_ARGUMENT), ({"scale": 0.0}, _lib.ERR_BAD_ARGUMENT),
    ({"scale": float("inf")}, _lib.ERR_BAD_ARGUMENT), ({"scale": -1.0}, _lib.ERR_BAD_ARGUMENT),
    ({"tokens": 0}, _lib.ERR_BAD_SHAPE), ({"tokens": 2 ** 31 - 1}, _lib.ERR_BAD_SHAPE),
    ({"page_size": 0, "key_tokens": 2 ** 31 - 1}, _lib.ERR_BAD_SHAPE), ({"sequences": 0}, _lib.ERR_BAD_SHAPE), ({"heads": 3}, _lib.ERR_BAD_SHAPE),
    ({"kv_heads": 0}, _lib.ERR_BAD_SHAPE), ({"pages": 0}, _lib.ERR_BAD_SHAPE), ({"table_width": 0}, _lib.ERR_BAD_SHAPE),
    ({"page_size": -16}, _lib.ERR_BAD_SHAPE), ({"max_k": -1}, _lib.ERR_BAD_SHAPE), ({"heads": 1 << 16}, _lib.ERR_BAD_SHAPE),
    ({"dim": 60}, _lib.ERR_UNSUPPORTED_SHAPE), ({"dim": 136}, _lib.ERR_UNSUPPORTED_SHAPE), ({"heads": 258}, _lib.ERR_UNSUPPORTED_SHAPE),
    ({"page_size": 24}, _lib.ERR_UNSUPPORTED_SHAPE), ({"token_of_q": 260}, _lib.ERR_UNSUPPORTED_SHAPE),
    ({"head_of_v": -64}, _lib.ERR_UNSUPPORTED_SHAPE), ({"page_of_k": 1 << 39}, _lib.ERR_UNSUPPORTED_SHAPE),
    ({"head_of_q": 0}, _lib.ERR_UNSUPPORTED_SHAPE), ({"token_of_k": 0}, _lib.ERR_UNSUPPORTED_SHAPE),
    ({"page_of_v": 0}, _lib.ERR_UNSUPPORTED_SHAPE),
]


@pytest.mark.parametrize("other,code", ARGUMENTS, ids=lambda x: str(x)[:40])
@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_arguments_are_checked_before_a_device_is_touched(L, entry, other, code):
    a = arguments(**other)
    p = address()
    assert getattr(L, f"b200q_attn_{entry}")(ctypes.byref(a), p, 1 << 30, None) == code
    assert getattr(L, f"b200q_attn_{entry}_workspace_bytes")(ctypes.byref(a)) == 0


def test_addresses_and_workspace_are_checked(L):
    p = address()
    for entry in ("prefill", "decode"):
        f = getattr(L, f"b200q_attn_{entry}")
        assert f(None, None, 0, None) == _lib.ERR_NULL_POINTER
        assert f(ctypes.byref(arguments(out=p + 8)), p, 1 << 30, None) == _lib.ERR_MISALIGNED
        assert f(ctypes.byref(arguments(data_of_q=p + 2)), p, 1 << 30, None) == _lib.ERR_MISALIGNED
        assert f(ctypes.byref(arguments(tables=p + 2)), p, 1 << 30, None) == _lib.ERR_MISALIGNED
        a = arguments(table_width=4000, max_k=60000)      # a context that may be divided
        need = getattr(L, f"b200q_attn_{entry}_workspace_bytes")(ctypes.byref(a))
        assert need > 0
        assert f(ctypes.byref(a), None, 0, None) == _lib.ERR_WORKSPACE
        assert f(ctypes.byref(a), p, need - 1, None) == _lib.ERR_WORKSPACE
        assert f(ctypes.byref(a), p + 8, need, None) == _lib.ERR_MISALIGNED
    assert L.b200q_attn_prefill(ctypes.byref(arguments(cu_k=None)), p, 1 << 30, None) == _lib.ERR_NULL_POINTER
    assert L.b200q_attn_decode(ctypes.byref(arguments(lengths=None)), p, 1 << 30, None) == _lib.ERR_NULL_POINTER
    assert L.b200q_attn_decode(ctypes.byref(arguments(page_size=0)), p, 1 << 30, None) == _lib.ERR_BAD_SHAPE
    assert L.b200q_attn_decode(ctypes.byref(arguments(sequences=5)), p, 1 << 30, None) == _lib.ERR_BAD_SHAPE


def test_store_and_copy_check_their_arguments(L):
    p = address()
    view, cache = _lib.View(p, 0, 128, 64), _lib.View(p, 2048, 128, 64)

    def stored(k=view, c=cache, slots=p, tokens=3, heads=2, dim=64, pages=5, size=16):
        return L.b200q_kv_store(ctypes.byref(k), ctypes.byref(view), ctypes.byref(c), ctypes.byref(cache), slots, tokens,
                                heads, dim, pages, size, None)

    assert stored(slots=None) == _lib.ERR_NULL_POINTER
    assert stored(c=_lib.View(None, 0, 0, 0)) == _lib.ERR_NULL_POINTER
    assert stored(tokens=0) == stored(tokens=2 ** 31 - 1) == stored(pages=0) == stored(size=0) == _lib.ERR_BAD_SHAPE
    assert stored(dim=60) == stored(k=_lib.View(p, 0, 100, 64)) == _lib.ERR_UNSUPPORTED_SHAPE
    assert stored(k=_lib.View(p + 8, 0, 128, 64)) == stored(slots=p + 2) == _lib.ERR_MISALIGNED

    def copied(src=(0,), dst=(1,), cache=p, outer=2, outer_stride=1 << 20, page_stride=4096, page_bytes=4096, pages=5):
        a, b = ((ctypes.c_int32 * len(x))(*x) for x in (src, dst))
        return L.b200q_kv_copy_pages(cache, outer, outer_stride, page_stride, page_bytes, pages, a, b, len(src), None)

    assert copied(cache=None) == _lib.ERR_NULL_POINTER
    assert copied(outer=0) == copied(pages=0) == copied(page_bytes=0) == _lib.ERR_BAD_SHAPE
    assert copied(page_bytes=4100) == copied(page_stride=-16) == copied(outer_stride=8) == _lib.ERR_UNSUPPORTED_SHAPE
    assert copied(cache=p + 8) == _lib.ERR_MISALIGNED
    for src, dst in (((0,), (5,)), ((-1,), (1,)), ((0, 1), (2, 2)), ((0, 1), (2, 0)), ((4,), (4,))):
        assert copied(src, dst) == _lib.ERR_BAD_ARGUMENT
    # pages or layers that overlap
    assert copied(page_stride=0) == copied(page_stride=4080) == copied(outer_stride=0) == _lib.ERR_UNSUPPORTED_SHAPE


def test_structures_are_the_headers(tmp_path):
    fields = [n for n, _ in _lib.Attention._fields_]
    source = tmp_path / "layout.c"
    lines = "\n".join(f'  printf("%zu\\n", offsetof(b200q_attention, {n}));' for n in fields)
    source.write_text(f'#include <stdio.h>\n#include "b200q.h"\nint main(void) {{\n{lines}\n'
                      '  printf("%zu\\n%zu\\n", sizeof(b200q_attention), sizeof(b200q_view));\n  return 0;\n}\n')
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(source), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    want = [getattr(_lib.Attention, n).offset for n in fields] + [ctypes.sizeof(_lib.Attention), ctypes.sizeof(_lib.View)]
    assert got == want


# ------------------------------------------------------------------------------ layer, context
def test_context():
    context.set_context(True, 1, 2, 3, 4, 5, block_tables=6)
    c = context.get_context()
    assert (c.is_prefill, c.cu_seqlens_q, c.cu_seqlens_k, c.max_seqlen_q, c.max_seqlen_k, c.slot_mapping, c.context_lens,
            c.block_tables) == (True, 1, 2, 3, 4, 5, None, 6)
    context.reset_context()
    assert context.get_context() == context.Context()


def test_the_layer_and_its_context_stand_under_the_references_names():
    code = ("import sys; sys.path.insert(0, %r)\n"
            "from tiny_vllm_b200.integration import install_under_nanovllm\n"
            "names = install_under_nanovllm(replace_attention=True)\n"
            "assert {'nanovllm.layers.attention', 'nanovllm.utils.context'} <= set(names), names\n"
            "import importlib\n"
            "layer = sys.modules['nanovllm.layers.attention'].Attention(8, 128, 0.1, 2)\n"
            "assert layer.k_cache.numel() == 0 and layer.v_cache.numel() == 0\n"
            "sys.modules['nanovllm.utils.context'].set_context(False)\n"
            "assert not sys.modules['nanovllm.layers.attention'].get_context().is_prefill\n" % str(ROOT))
    subprocess.run([sys.executable, "-c", code], check=True)

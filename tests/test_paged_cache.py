"""The paged cache's operators without a GPU: index guards and the split over
CTAs (a C++ check of the kernels' own headers), the C-ABI's argument checks,
and the torch ops' Meta kernels with their refusals."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import operatorlib

REPO = Path(__file__).resolve().parents[1]
CSRC = REPO / "orin-cuda-operator-library_b200" / "csrc"
INVALID = 1
FAKE = 0x1000  # never dereferenced: validation rejects before any launch


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_index_guards_and_split(tmp_path):
    exe = tmp_path / "paged_index_check"
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{CSRC}",
                    str(REPO / "tests" / "cpp" / "paged_index_check.cpp"), "-o", str(exe)],
                   check=True, capture_output=True, timeout=120)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120).stdout
    assert out.strip() == "PASS", out


# ------------------------------------------------------------ C-ABI refusals

def rope_spec(**kw):
    spec = operatorlib.RopeSpec(FAKE, FAKE, 64, 1)
    spec.sections[0] = 32
    for name, value in kw.items():
        if name == "sections":
            for i, n in enumerate(value):
                spec.sections[i] = n
        else:
            setattr(spec, name, value)
    return ctypes.byref(spec)


def cache(**kw):
    c = operatorlib.KvCache(FAKE, FAKE + 65536, 4, 16, 2, 64, 2048, 128, 64, 2048, 128, 64)
    for name, value in kw.items():
        setattr(c, name, value)
    return ctypes.byref(c)


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("change", [
    dict(x=None), dict(out=None), dict(tokens=0), dict(heads=-1), dict(head_dim=0),
    dict(head_dim=257), dict(spec=None), dict(spec=dict(rot_dim=66)), dict(spec=dict(rot_dim=-2)),
    dict(spec=dict(rot_dim=31)), dict(spec=dict(axes=0)), dict(spec=dict(axes=5)),
    dict(spec=dict(positions=None)), dict(spec=dict(inv_freq=None)),
    dict(spec=dict(sections=[31])), dict(spec=dict(axes=2, sections=[40, -8])),
    dict(spec=dict(axes=2, sections=[32, 1])),
])
def test_rope_refusals(suffix, change):
    a = dict(x=FAKE, out=FAKE, tokens=3, heads=2, head_dim=64, spec={})
    a.update(change)
    spec = None if a["spec"] is None else rope_spec(**a["spec"])
    fn = getattr(operatorlib.capi(), f"opl_rope_{suffix}")
    assert fn(a["x"], a["out"], a["tokens"], a["heads"], a["head_dim"], 128, 64, 128, 64, spec,
              None) == INVALID


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("change", [
    dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(slots=None),
    dict(tokens=0), dict(heads=0), dict(cache=None), dict(cache=dict(k=None)),
    dict(cache=dict(v=None)), dict(cache=dict(pages=0)), dict(cache=dict(page_size=0)),
    dict(cache=dict(kv_heads=0)), dict(cache=dict(head_dim=0)), dict(cache=dict(head_dim=260)),
    dict(cache=dict(head_dim=62)), dict(cache=dict(v=FAKE)), dict(spec=dict(sections=[30])),
])
def test_kv_append_refusals(suffix, change):
    a = dict(q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, slots=FAKE, tokens=3, heads=4, cache={}, spec={})
    a.update(change)
    c = None if a["cache"] is None else cache(**a["cache"])
    fn = getattr(operatorlib.capi(), f"opl_kv_append_{suffix}")
    assert fn(a["q"], 256, 64, a["k"], 128, 64, a["v"], 128, 64, a["q_out"], 256, 64, c,
              a["slots"], a["tokens"], a["heads"], rope_spec(**a["spec"]), None) == INVALID


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("change", [
    dict(q=None), dict(out=None), dict(table=None), dict(lens=None), dict(workspace=None),
    dict(workspace=FAKE + 8), dict(bytes=16), dict(batch=0), dict(heads=0), dict(heads=5),
    dict(max_pages=0), dict(max_pages=2 ** 26 + 1), dict(max_pages=2 ** 25, batch=33),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(cache=None),
    dict(cache=dict(k=None)), dict(cache=dict(v=None)), dict(cache=dict(pages=0)),
    dict(cache=dict(page_size=-1)), dict(cache=dict(kv_heads=0)), dict(cache=dict(head_dim=0)),
    dict(cache=dict(head_dim=257)),
])
def test_paged_attention_refusals(suffix, change):
    a = dict(q=FAKE, out=FAKE, table=FAKE, lens=FAKE, workspace=FAKE, bytes=1 << 30, batch=3,
             heads=4, max_pages=2, scale=0.125, cache={})
    a.update(change)
    c = None if a["cache"] is None else cache(**a["cache"])
    fn = getattr(operatorlib.capi(), f"opl_paged_attention_{suffix}")
    assert fn(a["q"], 256, 64, c, a["table"], 2, a["max_pages"], a["lens"], a["out"], a["batch"],
              a["heads"], a["scale"], a["workspace"], a["bytes"], None) == INVALID


@pytest.mark.parametrize("args", [(0, 1, 64), (4, 0, 64), (5, 2, 64), (4, 2, 0), (4, 2, 257)])
def test_workspace_refusals(args):
    size = ctypes.c_size_t()
    assert operatorlib.capi().opl_paged_attention_workspace(*args, ctypes.byref(size)) == INVALID
    assert operatorlib.capi().opl_paged_attention_workspace(4, 2, 64, None) == INVALID


def test_raw_helper_refuses_five_axes():
    with pytest.raises(ValueError, match="at most 4"):
        operatorlib.rope_into(torch.zeros(1, 1, 8), torch.zeros(1, 1, 8),
                              torch.zeros(5, 1, dtype=torch.int64), torch.zeros(4), [1] * 5)


# ---------------------------------------------------------------- torch ops

@pytest.fixture(scope="module")
def ops():
    operatorlib.load_operatorlib()
    return torch.ops.operatorlib


def meta(*shape, dtype=torch.float16):
    return torch.empty(*shape, device="meta", dtype=dtype)


def rope_args(**kw):
    a = dict(x=meta(5, 3, 64), positions=meta(5, dtype=torch.int64),
             inv_freq=meta(32, dtype=torch.float32), sections=[], adjacent=False, inverse=False)
    a.update(kw)
    return a.values()


def append_args(**kw):
    a = dict(q=meta(5, 4, 64), k=meta(5, 2, 64), v=meta(5, 2, 64), k_cache=meta(3, 16, 2, 64),
             v_cache=meta(3, 16, 2, 64), slots=meta(5, dtype=torch.int64),
             positions=meta(5, dtype=torch.int64), inv_freq=meta(32, dtype=torch.float32),
             sections=[], adjacent=False)
    a.update(kw)
    return a.values()


def attention_args(**kw):
    a = dict(q=meta(5, 4, 64), k_cache=meta(3, 16, 2, 64), v_cache=meta(3, 16, 2, 64),
             block_table=meta(5, 2, dtype=torch.int32), seq_lens=meta(5, dtype=torch.int32),
             scale=None)
    a.update(kw)
    return a.values()


def test_schemas(ops):
    assert str(ops.rope.default._schema) == (
        "operatorlib::rope(Tensor x, Tensor positions, Tensor inv_freq, int[] sections=[], "
        "bool adjacent=False, bool inverse=False) -> Tensor")
    assert str(ops.kv_append.default._schema) == (
        "operatorlib::kv_append(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, "
        "Tensor(b!) v_cache, Tensor slots, Tensor positions, Tensor inv_freq, int[] sections=[], "
        "bool adjacent=False) -> Tensor")
    assert str(ops.paged_attention.default._schema) == (
        "operatorlib::paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, "
        "Tensor block_table, Tensor seq_lens, float? scale=None) -> Tensor")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_shapes_and_dtypes(ops, dtype):
    packed = meta(5, 8, 64, dtype=dtype)
    q, k, v = packed.split([4, 2, 2], dim=1)
    caches = dict(k_cache=meta(3, 2, 16, 64, dtype=dtype).transpose(1, 2),
                  v_cache=meta(3, 16, 2, 64, dtype=dtype))
    for out in (ops.rope(*rope_args(x=q)), ops.kv_append(*append_args(q=q, k=k, v=v, **caches)),
                ops.paged_attention(*attention_args(q=q, **caches))):
        assert out.shape == (5, 4, 64) and out.dtype == dtype and out.is_contiguous()
    three = dict(positions=meta(3, 5, dtype=torch.int64), sections=[16, 8, 8])
    assert ops.rope(*rope_args(**three)).shape == (5, 3, 64)
    assert ops.kv_append(*append_args(**three)).shape == (5, 4, 64)


@pytest.mark.parametrize("change,text", [
    (dict(x=meta(5, 192)), "3 dimensions"),
    (dict(x=meta(5, 64, 3).transpose(1, 2)), "contiguous in its last"),
    (dict(x=meta(5, 3, 64, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (dict(x=meta(0, 3, 64)), "positive int32"),
    (dict(x=meta(5, 3, 260)), "at most 256"),
    (dict(positions=meta(5, dtype=torch.int32)), "positions must be int64"),
    (dict(positions=meta(6, dtype=torch.int64)), "one column for each token"),
    (dict(positions=meta(2, 5, dtype=torch.int64)), "an axis for each section"),
    (dict(positions=meta(5, 2, dtype=torch.int64).t(), sections=[16, 16]), "contiguous"),
    (dict(inv_freq=meta(33, dtype=torch.float32)), "head_dim / 2"),
    (dict(inv_freq=meta(32, dtype=torch.float64)), "inv_freq must be float32"),
    (dict(sections=[16, 8]), "add up"),
    (dict(sections=[40, -8]), "pairs of inv_freq"),
    (dict(sections=[8, 8, 8, 4, 4]), "at most 4"),
])
def test_rope_op_refusals(ops, change, text):
    with pytest.raises(RuntimeError, match=text):
        ops.rope(*rope_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(k=meta(5, 2, 64, dtype=torch.bfloat16)), "same dtype"),
    (dict(v=meta(5, 1, 64)), "identical shapes"),
    (dict(k=meta(4, 2, 64), v=meta(4, 2, 64)), "q's tokens"),
    (dict(k=meta(5, 3, 64), v=meta(5, 3, 64)), "key-value heads"),
    (dict(k_cache=meta(3, 16, 2, 32)), "identical shapes"),
    (dict(k_cache=meta(3, 16, 2, 32), v_cache=meta(3, 16, 2, 32)), "q's head_dim"),
    (dict(k_cache=meta(1, 16, 2, 64).expand(3, -1, -1, -1)), "must not be expanded"),
    (dict(slots=meta(5, dtype=torch.int32)), "slots must be int64"),
    (dict(slots=meta(4, dtype=torch.int64)), "one element a token"),
    (dict(sections=[32, 0]), "an axis for each section"),
])
def test_kv_append_op_refusals(ops, change, text):
    with pytest.raises(RuntimeError, match=text):
        ops.kv_append(*append_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(q=meta(5, 3, 64)), "multiple of the key-value heads"),
    (dict(q=meta(5, 4, 64, dtype=torch.float32)), "same dtype"),
    (dict(q=meta(0, 4, 64)), "positive int32"),
    (dict(k_cache=meta(3, 16, 2, 64, dtype=torch.float32)), "same dtype"),
    (dict(v_cache=meta(3, 16, 64)), "4 dimensions"),
    (dict(block_table=meta(5, 2, dtype=torch.int64)), "block_table must be int32"),
    (dict(block_table=meta(4, 2, dtype=torch.int32)), "one row a sequence"),
    (dict(block_table=meta(5, 0, dtype=torch.int32)), "positive int32"),
    (dict(seq_lens=meta(5, dtype=torch.int64)), "seq_lens must be int32"),
    (dict(seq_lens=meta(4, dtype=torch.int32)), "one element a sequence"),
    (dict(block_table=meta(5, 2 ** 26 + 1, dtype=torch.int32)), "2\\^30 keys a sequence"),
    (dict(scale=float("inf")), "scale must be finite"),
    (dict(scale=1e39), "scale must be finite"),
])
def test_paged_attention_op_refusals(ops, change, text):
    with pytest.raises(RuntimeError, match=text):
        ops.paged_attention(*attention_args(**change))


def test_no_cpu_kernel(ops):
    with pytest.raises(NotImplementedError):
        ops.rope(torch.ones(2, 1, 8), torch.zeros(2, dtype=torch.int64), torch.ones(4))

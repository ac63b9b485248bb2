"""The raw helpers of the paged cache refuse operands that do not go together:
the C entries see pointers only.  Without a GPU: every call is refused before
a pointer is used."""
from __future__ import annotations

import ctypes

import pytest
import torch

import operatorlib

I32, I64 = torch.int32, torch.int64


def t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def rope_args(**kw):
    a = dict(x=t(5, 3, 64), out=t(5, 3, 64), positions=t(5, dtype=I64),
             inv_freq=t(32, dtype=torch.float32), sections=None)
    a.update(kw)
    return a


def append_args(**kw):
    a = dict(q=t(5, 4, 64), k=t(5, 2, 64), v=t(5, 2, 64), q_out=t(5, 4, 64),
             k_cache=t(3, 16, 2, 64), v_cache=t(3, 16, 2, 64), slots=t(5, dtype=I64),
             positions=t(5, dtype=I64), inv_freq=t(32, dtype=torch.float32), sections=None)
    a.update(kw)
    return a


def attention_args(**kw):
    a = dict(q=t(5, 4, 64), k_cache=t(3, 16, 2, 64), v_cache=t(3, 16, 2, 64),
             block_table=t(5, 2, dtype=I32), seq_lens=t(5, dtype=I32), out=t(5, 4, 64),
             workspace=t(1 << 20, dtype=torch.uint8))
    a.update(kw)
    return a


ROPE = [
    (dict(positions=t(4, dtype=I64)), "positions must be contiguous with at least 5"),
    (dict(positions=t(3, 6, dtype=I64), sections=[16, 8, 8]), "positions must be .* with 15 elem"),
    (dict(positions=t(5, dtype=I32)), "positions must be int64"),
    (dict(positions=t(5, dtype=I64), sections=[16, 8, 8]), "positions must be contiguous"),
    (dict(positions=t(2, 5, dtype=I64), sections=[16, 8, 8]), "positions must be contiguous"),
    (dict(positions=t(5, 3, dtype=I64).t(), sections=[16, 8, 8]), "positions must be contiguous"),
    (dict(positions=t(10, dtype=I64)[::2]), "positions must be contiguous"),
    (dict(inv_freq=t(32, dtype=torch.float64)), "inv_freq must be float32"),
    (dict(inv_freq=t(64, dtype=torch.float32)[::2]), "inv_freq must be contiguous"),
]


@pytest.mark.parametrize("change,text", ROPE + [
    (dict(x=t(5, 192)), "x must have 3 dimensions"),
    (dict(x=t(5, 64, 3).transpose(1, 2)), "x must be contiguous in its last"),
    (dict(out=t(4, 3, 64)), "out must have the shape"),
    (dict(out=t(5, 3, 64, dtype=torch.bfloat16)), "out must have the other tensors' dtype"),
    (dict(out=t(5, 3, 64).to("meta")), "out must have the other tensors' dtype and device"),
    (dict(out=t(5, 1, 64).expand(5, 3, 64)), "out is written and must not be expanded"),
])
def test_rope_into(change, text):
    with pytest.raises(ValueError, match=text):
        operatorlib.rope_into(**rope_args(**change))


@pytest.mark.parametrize("change,text", ROPE + [
    (dict(k=t(4, 2, 64)), "k must have the shape"),
    (dict(v=t(5, 1, 64)), "v must have the shape"),
    (dict(v=t(5, 2, 64, dtype=torch.float32)), "v must have the other tensors' dtype"),
    (dict(q_out=t(5, 3, 64)), "q_out must have the shape"),
    (dict(q_out=t(1, 4, 64).expand(5, 4, 64)), "q_out is written"),
    (dict(k_cache=t(3, 32, 64)), "k_cache must have 4 dimensions"),
    (dict(v_cache=t(3, 8, 2, 64)), "v_cache must have the shape"),
    (dict(v_cache=t(2, 16, 2, 64)), "v_cache must have the shape"),
    (dict(v_cache=t(3, 16, 2, 64, dtype=torch.bfloat16)), "v_cache must have the other tensors'"),
    (dict(k_cache=t(1, 16, 2, 64).expand(3, 16, 2, 64)), "k_cache is written"),
    (dict(k_cache=t(3, 16, 2, 32), v_cache=t(3, 16, 2, 32)), "with q's head_dim"),
    (dict(slots=t(5, dtype=I32)), "slots must be int64"),
    (dict(slots=t(4, dtype=I64)), "slots must be contiguous with at least 5"),
    (dict(slots=t(10, dtype=I64)[::2]), "slots must be contiguous"),
])
def test_kv_append_into(change, text):
    with pytest.raises(ValueError, match=text):
        operatorlib.kv_append_into(**append_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(q=t(5, 256)), "q must have 3 dimensions"),
    (dict(out=t(4, 4, 64)), "out must be contiguous with at least 1280"),
    (dict(out=t(5, 4, 128)[..., :64]), "out must be contiguous"),
    (dict(out=t(5, 4, 64, dtype=torch.float32)), "out must be float16"),
    (dict(v_cache=t(2, 16, 2, 64)), "v_cache must have the shape"),
    (dict(k_cache=t(3, 16, 2, 64, dtype=torch.float32)), "k_cache must have the other tensors'"),
    (dict(k_cache=t(3, 16, 2, 32), v_cache=t(3, 16, 2, 32)), "with q's head_dim"),
    (dict(block_table=t(5, 2, dtype=I64)), "block_table must be int32"),
    (dict(block_table=t(4, 2, dtype=I32)), "block_table must be int32 .batch, pages"),
    (dict(block_table=t(2, 5, dtype=I32).t()), "contiguous in its last"),
    (dict(block_table=t(10, dtype=I32)), "block_table must have 2 dimensions"),
    (dict(seq_lens=t(5, dtype=I64)), "seq_lens must be int32"),
    (dict(seq_lens=t(4, dtype=I32)), "seq_lens must be contiguous with at least 5"),
    (dict(workspace=t(1 << 20, dtype=torch.uint8)[::2]), "workspace must be contiguous"),
    (dict(workspace=t(1 << 20, dtype=torch.uint8).to("meta")), "workspace must be"),
])
def test_paged_attention_into(change, text):
    with pytest.raises(ValueError, match=text):
        operatorlib.paged_attention_into(**attention_args(**change))


def test_operands_that_go_together_are_not_refused():
    """Past the checks, a CPU tensor is refused by the device guard.  Buffers for
    more tokens or sequences than the call has may be passed whole."""
    for call, args in ((operatorlib.rope_into, rope_args()),
                       (operatorlib.rope_into, rope_args(positions=t(1, 5, dtype=I64))),
                       (operatorlib.rope_into, rope_args(positions=t(3, 5, dtype=I64),
                                                         sections=[16, 8, 8])),
                       (operatorlib.rope_into, rope_args(positions=t(9, dtype=I64),
                                                         out=t(8, 3, 64))),
                       (operatorlib.rope_into, rope_args(
                           x=t(5, 9, 64)[:, 2:5], out=t(3, 5, 64).transpose(0, 1))),
                       (operatorlib.kv_append_into, append_args(
                           k_cache=t(3, 2, 16, 64).transpose(1, 2), k=t(5, 1, 64).expand(5, 2, 64))),
                       (operatorlib.paged_attention_into, attention_args(
                           block_table=t(5, 9, dtype=I32)[:, 2:4])),
                       (operatorlib.paged_attention_into, attention_args(
                           block_table=t(7, 2, dtype=I32), seq_lens=t(7, dtype=I32),
                           out=t(5, 256)))):
        with pytest.raises(ValueError, match="Expected a cuda device"):
            call(**args)


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(2 ** 31 - 1, 1), (2 ** 31 - 1, 2 ** 31 - 1),
                                            (2 ** 30, 2 ** 30), (2 ** 27, 1)])
def test_too_many_heads(suffix, heads, kv_heads):
    """More than 2^30 vectors a token, counted in 64 bits: invalid argument."""
    fake = 0x1000  # never dereferenced
    spec = operatorlib.RopeSpec(fake, fake, 64, 1)
    spec.sections[0] = 32
    cache = operatorlib.KvCache(fake, fake + 65536, 4, 16, kv_heads, 64, 2048, 128, 64, 2048, 128,
                                64)
    fn = getattr(operatorlib.capi(), f"opl_kv_append_{suffix}")
    assert fn(fake, 256, 1, fake, 128, 64, fake, 128, 64, fake, 256, 64, ctypes.byref(cache), fake,
              3, heads, ctypes.byref(spec), None) == 1

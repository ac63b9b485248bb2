"""The serving step around a paged key-value cache: its cases, its plain forms
and the library's calls for them.

Three operators, in the order in which a decoder layer runs them:

* ``rope``       rotary position embedding with one or several position axes,
                 and its inverse (the gradient of the rotation);
* ``append``     rotates the new tokens' queries and keys and writes keys and
                 values into the pages of the cache;
* ``attention``  one new token per sequence against its pages.

``run`` computes the plain form with elementary torch operations while ``own``
is false, and makes the library's calls while it is true.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_DEVICE = "cuda"


# --------------------------------------------------------------------- cases

def _rope(name, **kw):
    case = dict(name=name, op="rope", dtype="bf16", tokens=1, heads=12, dim=128, rot=128,
                axes=1, adjacent=False, inverse=False, packed=False, far=0)
    case.update(kw)
    return case


def _append(name, **kw):
    case = dict(name=name, op="append", dtype="bf16", tokens=1, heads=32, kv_heads=8, dim=128,
                rot=128, axes=1, adjacent=False, packed=True, page=16, pages=64,
                heads_first=False, scattered=False, far=0)
    case.update(kw)
    return case


def _attention(name, **kw):
    case = dict(name=name, op="attention", dtype="bf16", batch=1, heads=32, kv_heads=8, dim=128,
                page=16, shortest=1024, longest=1024, empty=0, heads_first=False)
    case.update(kw)
    return case


def listed():
    return [
        # One decode step of a small batch: the launch is all there is.
        _rope("rope_decode_f16", dtype="f16", tokens=16, heads=12),
        # Frames of a video, time/height/width axes, a whole prompt at once.
        _rope("rope_video_bf16", tokens=32768, heads=32, axes=3),
        # Gradient of a training batch's rotation in FP32: adjacent pairs, an
        # odd token count, the gradient a slice of the packed projection's.
        _rope("rope_grad_f32", dtype="f32", tokens=4097, heads=12, dim=64, rot=64,
              adjacent=True, inverse=True, packed=True, far=1 << 20),
        # One new token for each of 64 running sequences.
        _append("append_decode_bf16", tokens=64, pages=512, scattered=True, far=100_000),
        # A prompt of images written into the cache in one call.
        _append("append_prompt_f16", dtype="f16", tokens=16384, axes=3, page=64, pages=320,
                heads_first=True),
        # FP32, part of the head rotated, a head size that fills no tile.
        _append("append_partial_f32", dtype="f32", tokens=1023, heads=12, kv_heads=12, dim=80,
                rot=32, packed=False, pages=96, scattered=True),
        # One sequence at a short context: latency.
        _attention("attention_single_f16", dtype="f16", heads=12, kv_heads=12),
        # One sequence at a very long context: all SMs on eight heads.
        _attention("attention_long_bf16", page=64, shortest=131071, longest=131071),
        # A full serving batch, lengths all over the range, some rows padding.
        _attention("attention_batch_bf16", batch=128, shortest=16, longest=8191, empty=4),
        # Many short sequences (the beginning of many answers).
        _attention("attention_short_f16", dtype="f16", batch=256, shortest=1, longest=160),
        # One key-value head shared by sixteen query heads of 256.
        _attention("attention_shared_bf16", batch=16, heads=16, kv_heads=1, dim=256, page=32,
                   shortest=700, longest=9000, heads_first=True),
        # FP32 cache, a head size of 64, every query head with its own keys.
        _attention("attention_f32", dtype="f32", batch=8, heads=12, kv_heads=12, dim=64,
                   page=32, shortest=333, longest=4096),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention"])
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    axes = rng.choice([1, 1, 2, 3])
    rot = rng.choice([dim, dim, dim, dim // 2])
    far = rng.choice([0, 4096, 1 << 20])
    if op == "rope":
        heads = rng.choice([1, 4, 8, 12, 16, 32])
        most = min(32768, 32768 * 32 * 128 // (heads * dim * (2 if dtype == "f32" else 1)))
        case = _rope("", dtype=dtype, tokens=_log_uniform(rng, 1, most), heads=heads, dim=dim,
                     rot=rot, axes=axes, adjacent=rng.random() < 0.3,
                     inverse=rng.random() < 0.4, packed=rng.random() < 0.4, far=far)
    elif op == "append":
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 2, 4])
        page = rng.choice([1, 8, 16, 16, 32, 64, 128])
        tokens = _log_uniform(rng, 1, 16384 * 128 * 48 // (dim * (heads + 2 * kv_heads) * 4))
        pages = -(-tokens // page) + _log_uniform(rng, 1, 256)
        case = _append("", dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                       rot=rot, axes=axes, adjacent=rng.random() < 0.3,
                       packed=rng.random() < 0.7, page=page, pages=pages,
                       heads_first=rng.random() < 0.4, scattered=rng.random() < 0.5, far=far)
    else:
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8, 16])
        batch = _log_uniform(rng, 1, 256)
        token = kv_heads * dim * 2 * _BYTES[dtype]
        longest = _log_uniform(rng, 1, max(64, min(131072, 1_500_000_000 // (batch * token))))
        shortest = rng.choice([longest, _log_uniform(rng, 1, longest)])
        case = _attention("", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim,
                          page=rng.choice([1, 8, 16, 16, 24, 32, 64, 128]), shortest=shortest,
                          longest=longest, empty=rng.choice([0, 0, batch // 8]),
                          heads_first=rng.random() < 0.4)
    del case["name"]
    return case


def _lengths(case):
    """The sequence lengths of an attention case, evenly over its range (their
    order is the seed's)."""
    filled = case["batch"] - case["empty"]
    low, high = case["shortest"], case["longest"]
    steps = max(1, filled - 1)
    return [low + (high - low) * (steps - i) // steps for i in range(filled)] + \
        [0] * case["empty"]


def _sections(pairs, axes):
    """How many of the rotated pairs belong to each position axis: the first
    axis takes what is left after equal parts for the others."""
    part = pairs * 3 // 8 if axes == 3 else pairs // axes
    return [pairs - part * (axes - 1)] + [part] * (axes - 1)


# -------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device=_DEVICE).manual_seed(seed)


def _frequencies(rot):
    exponent = torch.arange(0, rot, 2, device=_DEVICE, dtype=torch.float64) / rot
    return (10000.0 ** -exponent).float()


def _positions(case, gen):
    """[axes, tokens] (or [tokens] for one axis) of int64."""
    tokens, axes = case["tokens"], case["axes"]
    index = torch.arange(tokens, device=_DEVICE)
    start = int(torch.randint(0, case["far"] + 1, (1,), generator=gen, device=_DEVICE)) \
        if case["far"] else 0
    if case.get("scattered"):  # tokens of unrelated sequences
        index = torch.randint(0, 4096, (tokens,), generator=gen, device=_DEVICE)
    if axes == 1:
        return index + start
    width = 32
    grid = [index // (width * width), index // width % width, index % width]
    return torch.stack([g + start for g in grid[3 - axes:]]).contiguous()


def _heads(parts, tokens, dim, dtype, packed, gen):
    """Tensors [tokens, heads, dim], one for each number of heads: slices of
    one packed projection, or tensors of their own."""
    if packed:
        whole = torch.randn(tokens, sum(parts), dim, generator=gen, device=_DEVICE).to(dtype)
        return list(whole.split(parts, dim=1))
    return [torch.randn(tokens, h, dim, generator=gen, device=_DEVICE).to(dtype) for h in parts]


def _cache(pages, page, heads, dim, dtype, heads_first, gen):
    """Keys and values [pages, page, heads, dim], N(0, 1); heads_first keeps a
    head's tokens next to one another in memory."""
    shape = (pages, heads, page, dim) if heads_first else (pages, page, heads, dim)
    out = []
    for _ in range(2):
        t = torch.empty(shape, dtype=dtype, device=_DEVICE)
        flat = t.view(-1)
        for part in flat.split(1 << 27):
            part.copy_(torch.randn(part.numel(), generator=gen, device=_DEVICE))
        out.append(t.transpose(1, 2) if heads_first else t)
    return out


def prepare(case, seed):
    gen = _generator(seed)
    dtype = _DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] in ("rope", "append"):
        state["positions"] = _positions(case, gen)
        state["inv_freq"] = _frequencies(case["rot"])
        state["sections"] = _sections(case["rot"] // 2, case["axes"])
    if case["op"] == "rope":
        parts = [case["heads"]] * (3 if case["packed"] else 1)
        state["x"] = _heads(parts, case["tokens"], case["dim"], dtype, case["packed"], gen)[0]
    elif case["op"] == "append":
        parts = [case["heads"], case["kv_heads"], case["kv_heads"]]
        state["q"], state["k"], state["v"] = _heads(parts, case["tokens"], case["dim"], dtype,
                                                    case["packed"], gen)
        state["k_cache"], state["v_cache"] = _cache(case["pages"], case["page"],
                                                    case["kv_heads"], case["dim"], dtype,
                                                    case["heads_first"], gen)
        page, pages = case["page"], case["pages"]
        if case["scattered"]:
            order = torch.randperm(pages * page, generator=gen, device=_DEVICE)
            state["slots"] = order[:case["tokens"]].contiguous()
        else:  # a prompt: consecutive tokens in pages of any order
            order = torch.randperm(pages, generator=gen, device=_DEVICE)
            index = torch.arange(case["tokens"], device=_DEVICE)
            state["slots"] = order[index // page] * page + index % page
    else:
        lengths = torch.tensor(_lengths(case), device=_DEVICE)
        lengths = lengths[torch.randperm(case["batch"], generator=gen, device=_DEVICE)]
        page = case["page"]
        used = (lengths + page - 1) // page
        total = int(used.sum())
        width = max(1, int(used.max()))
        state["k_cache"], state["v_cache"] = _cache(total + 1, page, case["kv_heads"],
                                                    case["dim"], dtype, case["heads_first"], gen)
        order = torch.randperm(total + 1, generator=gen, device=_DEVICE)
        first = used.cumsum(0) - used
        column = torch.arange(width, device=_DEVICE)
        index = first[:, None] + column[None, :]
        table = order[index.clamp(max=total)]
        state["block_table"] = torch.where(column[None, :] < used[:, None], table,
                                           torch.zeros_like(table)).int().contiguous()
        state["seq_lens"] = lengths.int().contiguous()
        # Peaked attention, as trained models have it.
        state["q"] = (2 * torch.randn(case["batch"], case["heads"], case["dim"], generator=gen,
                                      device=_DEVICE)).to(dtype)
    return state


# --------------------------------------------------------------- plain forms

def _plain_angles(state):
    """cos and sin [tokens, 1, pairs]; the angle in 64 bits, where a far
    position times a frequency would lose its fraction in 32."""
    positions = state["positions"]
    if positions.dim() == 1:
        positions = positions[None]
    frequencies = state["inv_freq"].double().split(state["sections"])
    angle = torch.cat([p.double()[:, None] * f[None, :]
                       for p, f in zip(positions, frequencies)], dim=1)
    return torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]


def _plain_rotate(x, cos, sin, adjacent, inverse=False):
    y = x.float().clone()
    rot = 2 * cos.shape[-1]
    if inverse:
        sin = -sin
    if adjacent:
        first, second = slice(0, rot, 2), slice(1, rot, 2)
    else:
        first, second = slice(0, rot // 2), slice(rot // 2, rot)
    a, b = x[..., first].float(), x[..., second].float()
    y[..., first] = a * cos - b * sin
    y[..., second] = a * sin + b * cos
    return y.to(x.dtype)


def _plain_attention(state):
    q, table, lengths = state["q"], state["block_table"], state["seq_lens"]
    keys, values = state["k_cache"], state["v_cache"]
    batch, heads, dim = q.shape
    page, kv_heads = keys.shape[1], keys.shape[2]
    rows = table.long()

    def gather(cache):  # [batch, kv_heads, positions, dim] in 32 bits
        return cache[rows].reshape(batch, -1, kv_heads, dim).transpose(1, 2).float()

    queries = q.float().reshape(batch, kv_heads, heads // kv_heads, dim) / math.sqrt(dim)
    scores = queries @ gather(keys).transpose(-1, -2)
    seen = torch.arange(table.shape[1] * page, device=q.device)[None, :] < lengths[:, None]
    seen = seen[:, None, None, :]
    scores = torch.where(seen, scores, torch.full_like(scores, -1e30))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = torch.where(seen, weights, torch.zeros_like(weights))
    total = weights.sum(-1, keepdim=True)
    out = (weights @ gather(values)) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(batch, heads, dim).to(q.dtype)


def _plain(state):
    case = state["case"]
    if case["op"] == "attention":
        return _plain_attention(state)
    cos, sin = _plain_angles(state)
    if case["op"] == "rope":
        return _plain_rotate(state["x"], cos, sin, case["adjacent"], case["inverse"])
    slots = state["slots"]
    page = state["k_cache"].shape[1]
    k = _plain_rotate(state["k"], cos, sin, case["adjacent"])
    state["k_cache"][slots // page, slots % page] = k
    state["v_cache"][slots // page, slots % page] = state["v"]
    q = _plain_rotate(state["q"], cos, sin, case["adjacent"])
    return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


# ------------------------------------------------------------ library's calls

_ops = None


def _library():
    global _ops
    if _ops is None:
        package = Path(__file__).resolve().parents[1] / "orin-cuda-operator-library_b200"
        if str(package) not in sys.path:
            sys.path.insert(0, str(package))
        import operatorlib

        operatorlib.load_operatorlib()
        _ops = torch.ops.operatorlib
    return _ops


def _library_run(state):
    ops = _library()
    case = state["case"]
    if case["op"] == "attention":
        return ops.paged_attention(state["q"], state["k_cache"], state["v_cache"],
                                   state["block_table"], state["seq_lens"])
    if case["op"] == "rope":
        return ops.rope(state["x"], state["positions"], state["inv_freq"], state["sections"],
                        case["adjacent"], case["inverse"])
    q = ops.kv_append(state["q"], state["k"], state["v"], state["k_cache"], state["v_cache"],
                      state["slots"], state["positions"], state["inv_freq"], state["sections"],
                      case["adjacent"])
    return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def run(state):
    return _library_run(state) if own else _plain(state)


# ---------------------------------------------------------------------- work

def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "attention":
        keys = sum(_lengths(case))
        table = sum(-(-n // case["page"]) for n in _lengths(case))
        rows = case["batch"] * case["heads"] * case["dim"]
        return {"bytes": size * (2 * keys * case["kv_heads"] * case["dim"] + 2 * rows)
                + 4 * (table + case["batch"]),
                "flops": 4 * keys * case["heads"] * case["dim"]}
    tokens, pairs = case["tokens"], case["rot"] // 2
    small = 8 * case["axes"] * tokens + 4 * pairs
    if case["op"] == "rope":
        return {"bytes": 2 * size * tokens * case["heads"] * case["dim"] + small,
                "flops": 6 * tokens * case["heads"] * pairs}
    rows = case["heads"] + 2 * case["kv_heads"]
    return {"bytes": 2 * size * tokens * rows * case["dim"] + small + 8 * tokens,
            "flops": 6 * tokens * (case["heads"] + case["kv_heads"]) * pairs}


# --------------------------------------------------------------------- exact

def _exact_rotate(state, x, sign):
    """The rotation as a product of complex numbers of 64 bits each."""
    case = state["case"]
    positions = state["positions"].reshape(case["axes"], -1)
    axis = torch.tensor(np.repeat(np.arange(case["axes"]), state["sections"]), device=x.device)
    angle = positions[axis].t().double() * state["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), sign * angle)[:, None, :]
    half = case["rot"] // 2
    wide = x.double()
    pairs = wide[..., :2 * half]
    if case["adjacent"]:
        pairs = pairs.unflatten(-1, (half, 2))
    else:
        pairs = pairs.unflatten(-1, (2, half)).transpose(-1, -2)
    turned = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
    if not case["adjacent"]:
        turned = turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), wide[..., 2 * half:]], dim=-1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rotate(state, state["x"], -1 if case["inverse"] else 1)
    if case["op"] == "append":
        out = {"q": _exact_rotate(state, state["q"], 1)}
        slots, page = state["slots"], case["page"]
        for name, rows in (("k_cache", _exact_rotate(state, state["k"], 1)),
                           ("v_cache", state["v"].double())):
            flat = state[name].double().reshape(-1, case["kv_heads"], case["dim"])
            flat.index_copy_(0, slots, rows)
            out[name] = flat.unflatten(0, (-1, page))
        return out
    q = state["q"].double()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    for b, length in enumerate(state["seq_lens"].tolist()):
        if length == 0:
            continue
        where = torch.arange(length, device=q.device)
        pages = state["block_table"][b].long()[where // case["page"]]
        inside = where % case["page"]
        keys, values = (state[n][pages, inside].double() for n in ("k_cache", "v_cache"))
        for h in range(case["heads"]):
            score = keys[:, h // group] @ q[b, h] / math.sqrt(case["dim"])
            weight = torch.softmax(score, dim=0)
            out[b, h] = weight @ values[:, h // group]
    return out

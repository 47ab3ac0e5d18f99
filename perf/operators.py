"""Performance cases of the quantized key / value cache: what a decoder that serves text asks of it.

Three kinds of work, each through the package's public entry points and on data that is already on the device:

  store   keys and values of new tokens are quantized into their slots of the paged cache and read back as the values
          that they now stand for (what a chunk's own attention sees)
  load    rows that the cache has held for a while are read back as floats, by slot (a prefix that moves to another
          program, or that is attended to densely)
  attend  attention of new tokens, one or many per sequence, over the pages of their sequences

Where ``own`` is false ``run`` computes the same in elementary torch operations.  ``listed()`` gives named cases,
``draw(rng)`` one more of the same ranges; ``prepare`` makes the inputs and what a program keeps between calls, ``run`` is
one pass, ``exact`` the result from the definition in 64 bits.

The cache: pages of ``page`` tokens, per page and key / value head ``page`` rows of ``dim`` codes.  A row x has the grid
[qmin, qmax] of its bits: lo = min(x, 0), hi = max(x, 0), scale = max(|lo|, |hi|) / ((qmax - qmin) / 2) and zero point 0
(symmetric), or (hi - lo) / (qmax - qmin) and clip(qmin - rint(lo / scale)) (affine), scale at least 1e-8;
c = clip(rint(x / scale) + zero, qmin, qmax), all in float32.  It stands for (c - zero) * scale; what is stored is c - qmin,
two 4-bit codes in a byte, the first in the low half.
"""

from __future__ import annotations

import math

import torch

own = False


# ---------------------------------------------------------------- cases
def listed():
    heads = dict(kv_heads=8, dim=128)
    return [
        # one decoding step of 64 sequences: a token each
        dict(name="store_64_i8", kind="store", tokens=64, page=16, bits=8, symmetric=True, dtype="float16", padded=False, **heads),
        # a ragged prompt, twelve heads of 64, its batch padded to a fixed size, 4-bit codes
        dict(name="store_1111_i4", kind="store", tokens=1111, page=32, kv_heads=12, dim=64, bits=4, symmetric=False, dtype="float32",
             padded=True),
        # prompts of a large batch
        dict(name="store_65536_i8", kind="store", tokens=65536, page=64, bits=8, symmetric=True, dtype="float16", padded=False, **heads),
        # one short sequence, float32
        dict(name="load_333_i8", kind="load", tokens=333, page=16, kv_heads=12, dim=64, bits=8, symmetric=True, dtype="float32",
             padded=True),
        # a long document, 4-bit
        dict(name="load_131072_i4", kind="load", tokens=131072, page=64, bits=4, symmetric=False, dtype="float16", padded=False, **heads),
        # one token of one short sequence: latency
        dict(name="attend_1_197_f32", kind="attend", batch=1, chunk=1, context=197, ragged=False, heads=12, kv_heads=12, dim=64, page=16,
             bits=8, symmetric=True, dtype="float32", window=0),
        # a decoding step of 64 sequences of all lengths up to 8192, four query heads to a key head
        dict(name="attend_64x1_8192_i8", kind="attend", batch=64, chunk=1, context=8192, ragged=True, heads=32, page=16, bits=8,
             symmetric=True, dtype="float16", window=0, **heads),
        # a decoding step over one long document, 4-bit codes
        dict(name="attend_1_131072_i4", kind="attend", batch=1, chunk=1, context=131072, ragged=False, heads=32, page=64, bits=4,
             symmetric=False, dtype="float16", window=0, **heads),
        # sixteen sequences, five drafted tokens each, float32
        dict(name="attend_16x5_4096_f32", kind="attend", batch=16, chunk=5, context=4096, ragged=True, heads=32, page=32, bits=8,
             symmetric=True, dtype="float32", window=0, **heads),
        # chunks of ragged prompts, a window of 1024, odd head size, float32
        dict(name="attend_3x333_2048_f32", kind="attend", batch=3, chunk=333, context=2048, ragged=True, heads=10, kv_heads=5, dim=80,
             page=16, bits=8, symmetric=False, dtype="float32", window=1024),
        # a chunk of 512 tokens of each of four prompts
        dict(name="attend_4x512_8192_i4", kind="attend", batch=4, chunk=512, context=8192, ragged=True, heads=32, page=64, bits=4,
             symmetric=False, dtype="float16", window=0, **heads),
        # the second half of a long prompt
        dict(name="attend_8192_16384_i8", kind="attend", batch=1, chunk=8192, context=16384, ragged=False, heads=32, page=64, bits=8,
             symmetric=True, dtype="float16", window=0, **heads),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["store", "load", "attend", "attend", "attend"])
    bits = rng.choice([8, 8, 4])
    kv_heads, dim = rng.choice([1, 2, 4, 5, 8, 8, 12]), rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 256] + [16, 48, 80, 112] * (bits == 8))
    case = dict(kind=kind, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 16, 32, 48, 64, 128]), bits=bits, symmetric=rng.random() < 0.5,
                dtype=rng.choice(["float16", "float16", "float32"]))
    if kind != "attend":
        most = 131072 * 8 * 128 // (2 * kv_heads * dim) if kind == "store" else 131072 * 8 * 128 // (kv_heads * dim)
        return dict(case, tokens=_log_int(rng, 1, min(131072, most)), padded=rng.random() < 0.5)
    group = rng.choice([1, 1, 2, 4, 4, 7, 8, 16])
    while True:
        batch, chunk = _log_int(rng, 1, 128), rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 4096)])
        context = _log_int(rng, max(chunk, 16), 131072)
        rows = batch * chunk * kv_heads * group
        if rows * context <= 1.2e9 and batch * context * kv_heads * dim <= 0.8e9 and rows * dim <= 1 << 26:
            break
    return dict(case, batch=batch, chunk=chunk, context=context, ragged=rng.random() < 0.6, heads=kv_heads * group,
                window=_log_int(rng, 1, context) if rng.random() < 0.2 else 0)


def _lengths(case):
    """New tokens and cached tokens (the new ones included) of each sequence.  Ragged: spread over the range by the golden ratio."""
    b, chunk, context = case["batch"], case["chunk"], case["context"]
    if not case["ragged"]:
        return [chunk] * b, [context] * b
    part = [(i * 0.6180339887498949 + 1.0) % 1.0 or 1.0 for i in range(b)]
    q = [max(1, round(chunk * (0.5 + p / 2))) for p in part]
    return q, [max(n, round(context * p)) for n, p in zip(q, part)]


# ---------------------------------------------------------------- the format, in elementary operations
def _grid(case):
    half = 1 << (case["bits"] - 1)
    return -half, half - 1


def _ratio(a, b):
    """The float32 next to a / b (by way of 64 bits, whose own rounding changes nothing: torch multiplies by the inverse of a
    number, and a row's largest value lies on the border between two codes)."""
    return (a.double() / b).float()


def _quantize(case, x):
    """Codes less qmin as integers, scales and zero points of rows of float32."""
    qmin, qmax = _grid(case)
    lo, hi = x.amin(-1).clamp(max=0.0), x.amax(-1).clamp(min=0.0)
    if case["symmetric"]:
        scale = _ratio(torch.maximum(-lo, hi), (qmax - qmin) / 2).clamp(min=1e-8)
        zero = torch.zeros_like(scale)
    else:
        scale = _ratio(hi - lo, qmax - qmin).clamp(min=1e-8)
        zero = (qmin - torch.round(_ratio(lo, scale))).clamp(qmin, qmax)
    c = (torch.round(_ratio(x, scale[..., None])) + zero[..., None]).clamp(qmin, qmax)
    return (c - qmin).to(torch.uint8), scale, zero


def _pack(case, u):
    return u if case["bits"] == 8 else u[..., 0::2] | u[..., 1::2] << 4


def _unpack(case, u):
    return u if case["bits"] == 8 else torch.stack((u & 15, u >> 4), -1).flatten(-2)


def _values(case, codes, scale, zero):
    """Float32 values of rows of the cache."""
    return (_unpack(case, codes).float() + (_grid(case)[0] - zero)[..., None]) * scale[..., None]


def _places(slots, page):
    """Page, place in the page, and whether there is one at all."""
    there = slots >= 0
    s = torch.where(there, slots, 0).long()
    return s // page, s % page, there


# ---------------------------------------------------------------- a case's state
_DTYPES = {"float16": torch.float16, "float32": torch.float32}


def _rows(gen, case, *shape):
    """Keys or values: a few channels of each head are larger than the rest, as in trained models."""
    gain = 1 + 3 * (torch.rand(case["kv_heads"], case["dim"], generator=gen, device="cuda") < 0.06).float()
    return torch.randn(*shape, case["kv_heads"], case["dim"], generator=gen, device="cuda") * gain


def _empty_cache(case, pages):
    shape = (pages, case["kv_heads"], case["page"])
    codes = lambda: torch.zeros(*shape, case["dim"] * case["bits"] // 8, dtype=torch.uint8, device="cuda")
    number = lambda: torch.zeros(shape, device="cuda")
    return {"k_codes": codes(), "v_codes": codes(), "k_scale": number(), "v_scale": number(), "k_zero": number(), "v_zero": number()}


def _fill(case, cache, gen):
    """A cache in which every slot is taken, page by page so that no large float tensor is needed."""
    pages = cache["k_scale"].shape[0]
    step = max(1, (1 << 25) // (case["page"] * case["kv_heads"] * case["dim"]))
    gain = torch.randint(1, 1 << 30, (1,), generator=gen, device="cuda").item()
    for name in ("k", "v"):
        sub = torch.Generator(device="cuda").manual_seed(gain + (name == "v"))
        for lo in range(0, pages, step):
            n = min(step, pages - lo)
            codes, scale, zero = _quantize(case, _rows(sub, case, n, case["page"]).transpose(1, 2))
            cache[name + "_codes"][lo:lo + n], cache[name + "_scale"][lo:lo + n], cache[name + "_zero"][lo:lo + n] = _pack(case, codes), scale, zero


def _slots(case, gen):
    """Slots of consecutive tokens in pages that lie anywhere; a few tokens of a padded batch have none."""
    n, page = case["tokens"], case["page"]
    need = -(-n // page)
    pages = need + need // 4 + 1
    order = torch.randperm(pages, generator=gen, device="cuda")[:need]
    slots = (order[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n].to(torch.int32)
    if case["padded"]:
        slots[n - n // 8:] = -1
    return pages, slots


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case), "kind": case["kind"]}
    dtype = _DTYPES[case["dtype"]]
    if case["kind"] in ("store", "load"):
        pages, s["slots"] = _slots(case, gen)
        s["cache"] = _empty_cache(case, pages)
        if case["kind"] == "store":
            s["k"], s["v"] = (_rows(gen, case, case["tokens"]).to(dtype) for _ in range(2))
        else:
            _fill(case, s["cache"], gen)
        s["k_out"], s["v_out"] = (torch.empty(case["tokens"], case["kv_heads"], case["dim"], dtype=dtype, device="cuda") for _ in range(2))
    else:
        q_lens, kv_lens = _lengths(case)
        wide = -(-max(kv_lens) // case["page"])
        used = [-(-n // case["page"]) for n in kv_lens]
        pages = sum(used) + 3
        s["cache"] = _empty_cache(case, pages)
        _fill(case, s["cache"], gen)
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
        table, at = torch.full((case["batch"], wide), -1, dtype=torch.int32), 0
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n]
            at += n
        s["table"] = table.cuda()
        s["q_starts"] = torch.tensor([sum(q_lens[:b]) for b in range(case["batch"] + 1)], dtype=torch.int32).cuda()
        s["kv_lens"] = torch.tensor(kv_lens, dtype=torch.int32).cuda()
        s["q"] = (1.5 * torch.randn(sum(q_lens), case["heads"], case["dim"], generator=gen, device="cuda")).to(dtype)
        s["out"] = torch.empty_like(s["q"])
        s["most"] = max(q_lens)  # what a program knows of its batch on the host
    if own:
        _in_package(s)  # the same data as the package's tensors: what its programs hold
    return s


# ---------------------------------------------------------------- the package's tensors
class _Memory:
    """A package tensor's device memory as torch sees it; keeps the tensor alive."""

    def __init__(self, t):
        import numpy as np
        self.t = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": np.dtype(t.dtype.np).str, "strides": None, "data": (t.data_ptr, False),
                                         "version": 2}


def _view(t):
    return torch.as_tensor(_Memory(t), device="cuda")


def _in_package(s):
    import lucid_amd as L
    import lucid_amd.quantization as Q

    case = s["case"]

    def put(name):
        t = L.Tensor.empty(tuple(s[name].shape), str(s[name].dtype).removeprefix("torch."), "hip")
        _view(t).copy_(s[name])
        s[name] = _view(t)
        return t

    cache = Q.PagedKVCache(s["cache"]["k_scale"].shape[0], case["page"], case["kv_heads"], case["dim"],
                           Q.per_channel_symmetric if case["symmetric"] else Q.per_channel_affine, Q.qint8 if case["bits"] == 8 else Q.qint4)
    for name, t in s["cache"].items():
        if getattr(cache, name) is not None:  # (a symmetric cache has no zero points)
            _view(getattr(cache, name)).copy_(t.view(torch.int8) if t.dtype == torch.uint8 else t)
    s["cache"] = cache
    s["own"] = {name: put(name) for name in ("slots", "k", "v", "k_out", "v_out", "table", "q_starts", "kv_lens", "q", "out") if name in s}


# ---------------------------------------------------------------- one pass
def run(s):
    if own:
        import lucid_amd.nn.functional as F
        import lucid_amd.quantization as Q

        t = s["own"]
        if s["kind"] == "attend":
            F.paged_attention(t["q"], s["cache"], t["table"], t["q_starts"], t["kv_lens"], window=s["case"]["window"] or None,
                              max_chunk=s["most"], out=t["out"])
            return s["out"]
        if s["kind"] == "store":
            Q.kv_cache_write(s["cache"], t["k"], t["v"], t["slots"])
        Q.kv_cache_read(s["cache"], t["slots"], out=(t["k_out"], t["v_out"]))
        return s["k_out"], s["v_out"]
    return _attend(s) if s["kind"] == "attend" else _store_or_load(s)


def _store_or_load(s):
    case, cache = s["case"], s["cache"]
    page, at, there = _places(s["slots"], case["page"])
    out = []
    for name in ("k", "v"):
        if s["kind"] == "store":
            codes, scale, zero = _quantize(case, s[name].float())
            keep = slice(case["tokens"] - case["tokens"] // 8 if case["padded"] else None)  # (the others have no slot)
            cache[name + "_codes"][page[keep], :, at[keep]] = _pack(case, codes)[keep]
            cache[name + "_scale"][page[keep], :, at[keep]] = scale[keep]
            cache[name + "_zero"][page[keep], :, at[keep]] = zero[keep]
        x = _values(case, *(cache[name + part][page, :, at] for part in ("_codes", "_scale", "_zero")))
        out.append((x * there[:, None, None]).to(_DTYPES[case["dtype"]]))
    return tuple(out)


def _attend(s):
    case, cache, starts, kv_lens = s["case"], s["cache"], s["q_starts"].long(), s["kv_lens"].long()
    b, h, hk, d, most = case["batch"], case["heads"], case["kv_heads"], case["dim"], s["most"]
    long = s["table"].shape[1] * case["page"]
    # keys and values of every sequence, [sequence, head, key, dim]
    pages = s["table"].long().clamp(min=0)
    k, v = (_values(case, *(cache[name + part][pages] for part in ("_codes", "_scale", "_zero"))).transpose(1, 2).reshape(b, hk, long, d)
            for name in ("k", "v"))
    # the queries, padded to the longest chunk
    q_lens = starts[1:] - starts[:-1]
    i, j = torch.arange(most, device="cuda"), torch.arange(long, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].reshape(b, most, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    score = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(d)).view(b, hk, h // hk, most, long)
    place = (kv_lens - q_lens)[:, None] + i
    seen = (j <= place[..., None]) & (j < kv_lens[:, None, None])
    if case["window"]:
        seen &= j > place[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = score.sum(-1, keepdim=True)
    o = score.view(b, hk, -1, long) @ v / torch.where(total > 0, total, 1.0).view(b, hk, -1, 1)
    o = o.view(b, hk, h // hk, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, h, d)
    out = torch.zeros(s["q"].shape, device="cuda")
    used = i < q_lens[:, None]
    out[row[used]] = o[used]
    return out.to(s["q"].dtype)


# ---------------------------------------------------------------- the definition, in 64 bits
def _exact_row(case, x):
    """What rows of float64 stand for in the cache.  The format rounds to float32 at the scale, at lo / scale and at x / scale: so here."""
    f32 = lambda t: t.float().double()
    half = 2 ** (case["bits"] - 1)
    lo, hi = x.min(-1).values.clamp(max=0), x.max(-1).values.clamp(min=0)
    if case["symmetric"]:
        scale = f32(torch.maximum(lo.abs(), hi.abs()) / (half - 0.5))
        scale, zero = scale.clamp(min=float(torch.tensor(1e-8))), torch.zeros_like(scale)
    else:
        scale = f32(f32(hi - lo) / (2 * half - 1)).clamp(min=float(torch.tensor(1e-8)))
        zero = (-half - f32(lo / scale).round()).clamp(-half, half - 1)
    code = (f32(x / scale[..., None]).round() + zero[..., None]).clamp(-half, half - 1)
    return (code - zero[..., None]) * scale[..., None]


def _exact_held(case, cache, name, page, at):
    """Float64 values of cached rows, [row, head, dim]."""
    u = cache[name + "_codes"][page, :, at].long()
    if case["bits"] == 4:
        u = torch.stack([u % 16, u // 16], dim=-1).reshape(*u.shape[:-1], -1)
    scale, zero = (cache[name + part][page, :, at].double() for part in ("_scale", "_zero"))
    return (u - 2 ** (case["bits"] - 1) - zero[..., None]) * scale[..., None]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    page = case["page"]
    if case["kind"] == "store":
        there = (s["slots"] >= 0).double()[:, None, None]
        return tuple(_exact_row(case, s[name].double()) * there for name in ("k", "v"))
    if case["kind"] == "load":
        slots = s["slots"].long()
        there, slots = (slots >= 0).double()[:, None, None], slots.clamp(min=0)
        return tuple(_exact_held(case, s["cache"], name, slots // page, slots % page) * there for name in ("k", "v"))
    q_lens, kv_lens = _lengths(case)
    group, at, out = case["heads"] // case["kv_heads"], 0, torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, length) in enumerate(zip(q_lens, kv_lens)):
        j = torch.arange(length, device="cuda")
        k, v = (_exact_held(case, s["cache"], name, s["table"][b].long()[j // page], j % page) for name in ("k", "v"))
        place = length - n + torch.arange(n, device="cuda")[:, None]
        hidden = (j > place) | ((j <= place - case["window"]) if case["window"] else (j < 0))
        for g in range(case["kv_heads"]):
            q = s["q"][at:at + n, g * group:(g + 1) * group].double()
            for lo in range(0, n, 1024):  # (a slice of the queries at a time: float64 scores of a long chunk fill the memory)
                part = q[lo:lo + 1024]
                score = torch.tensordot(part, k[:, g], ([2], [1])) / math.sqrt(case["dim"])
                p = torch.softmax(score.masked_fill(hidden[lo:lo + 1024, None], -math.inf), -1)
                out[at + lo:at + lo + part.shape[0], g * group:(g + 1) * group] = torch.tensordot(p, v[:, g], ([2], [0]))
        at += n
    return out


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    item = 2 if case["dtype"] == "float16" else 4
    held = case["dim"] * case["bits"] // 8 + (4 if case["symmetric"] else 8)  # bytes of a row in the cache
    if case["kind"] != "attend":
        tokens, heads = case["tokens"], case["kv_heads"]
        rows = 2 * (tokens - tokens // 8 if case["padded"] else tokens) * heads
        whole = 2 * tokens * heads * case["dim"] * item
        store = case["kind"] == "store"
        return {"bytes": 4 * tokens + whole + rows * held + store * (rows * case["dim"] * item), "flops": 0}
    q_lens, kv_lens = _lengths(case)
    keys = pairs = 0
    for n, length in zip(q_lens, kv_lens):
        window = case["window"] or length
        first = length - n  # of its first new token
        keys += length - max(0, first - window + 1)
        short = max(0, min(n, window - first))  # rows that see all keys up to their own
        pairs += short * first + short * (short + 1) // 2 + (n - short) * window
    return {"bytes": 2 * keys * case["kv_heads"] * held + 2 * sum(q_lens) * case["heads"] * case["dim"] * item + 4 * -(-keys // case["page"]),
            "flops": 4 * case["dim"] * case["heads"] * pairs}

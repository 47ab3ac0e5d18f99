"""Performance cases of what stands around a decoder's attention: the block's other half, and what a step with drafted tokens does at its end.

Five kinds of work, each through the package's public entry points and on data that is already on the device:

  gated    both projections of a gated feed-forward block on group-wise 4- or 8-bit weights, h = act(x Wg' + bg) * (x Wu' + bu)
  norm     the residual connection between two blocks: a norm of a block's result, its gate and its scale, the sum with the residual, and the
           norm in front of the next block
  verify   drafted tokens against the target's probabilities, from given random numbers: what is accepted and the token that follows
  copy     pages of a quantized key / value cache copied into other pages (the last page of a sequence that is forked)
  compact  the rows that a sequence keeps of the cache moved together to its beginning (what it evicts leaves whole pages free)

Where ``own`` is false ``run`` computes the same in elementary torch operations.  ``listed()`` gives named cases, ``draw(rng)`` one more of
the same ranges; ``prepare`` makes the inputs and what a program keeps between calls, ``run`` is one pass, ``exact`` the result from the
definition in 64 bits.

Weights: per row and group of ``group`` consecutive elements scale s = max((max - min) / (2^bits - 1), 1e-7), bias b = min, code
c = clip(rint((w - b) / s), 0, 2^bits - 1); the codes stand little-endian in 32-bit words, and w is c s + b.

Norms, over the last axis: rms x / sqrt(mean(x^2) + eps) * weight, layer (x - mean) / sqrt(var + eps) * weight + bias.  The residual
r' = r + gate * scale * post(x), the result pre(r').

Drafts: a sequence has rows starts[b] .. starts[b + 1] - 1 of a step, its last token and after it the drafted ones; row i of the target holds
the probabilities p of the token behind it, row i of the draft those, q, that the next row's token was drawn from (q = 1 at that token where
there are none).  In order, token x of row i + 1 is accepted if u[i] q(x) < p(x).  Behind the last accepted one comes a token drawn with the sequence's
own number w: from max(p - q, 0) of the row that refused, from p where none did (or where nothing of p - q is positive), the lowest token whose
running sum of weights passes w times their sum.
"""

from __future__ import annotations

import math

import torch

own = False


# ---------------------------------------------------------------- cases
def listed():
    wide = dict(k=4096, n=11008)
    cache = dict(kv_heads=8, dim=128)
    return [
        # one sequence decoding: bound by the weights
        dict(name="gated_1_i4_f16", kind="gated", m=1, bits=4, group=64, act="silu", bias=False, dtype="float16", **wide),
        # sixteen sequences decoding, 8-bit weights, float32 activations
        dict(name="gated_16_i8_f32", kind="gated", m=16, bits=8, group=64, act="gelu", bias=False, dtype="float32", **wide),
        # a ragged prompt in float32, with biases
        dict(name="gated_333_i4_f32", kind="gated", m=333, bits=4, group=128, act="silu", bias=True, dtype="float32", **wide),
        # a prefill of 2048 tokens
        dict(name="gated_2048_i4_f16", kind="gated", m=2048, bits=4, group=128, act="silu", bias=False, dtype="float16", **wide),
        # one token between two blocks: latency
        dict(name="norm_1_4096_f16", kind="norm", rows=1, cols=4096, norm="rms", post=False, gate=0, scale=False, dtype="float16", residual="float16"),
        # 64 sequences of 197 tokens, a gate for each sequence, a scale for each channel, norms on both sides
        dict(name="norm_12608_768_f32", kind="norm", rows=12608, cols=768, norm="layer", post=True, gate=64, scale=True, dtype="float32",
             residual="float32"),
        # sixteen sequences with up to five drafted tokens
        dict(name="verify_16x5_32000_f32", kind="verify", batch=16, drafts=5, vocab=32000, ragged=True, given=True, dtype="float32"),
        # a large batch over a large vocabulary, float16 probabilities, drafts that were looked up
        dict(name="verify_128x3_131072_f16", kind="verify", batch=128, drafts=3, vocab=131072, ragged=False, given=False, dtype="float16"),
        # eight sequences forked: the last page of each
        dict(name="copy_8x16_i8", kind="copy", pages=8, page=16, bits=8, symmetric=True, padded=False, **cache),
        # long documents copied whole, 4-bit, the list padded to a fixed size
        dict(name="copy_2500x64_i4", kind="copy", pages=2500, page=64, bits=4, symmetric=False, padded=True, **cache),
        # sixteen sequences of all lengths up to 4096 keep half of their rows, twelve heads of 64
        dict(name="compact_16x4096_i8", kind="compact", batch=16, context=4096, ragged=True, part=0.5, page=16, kv_heads=12, dim=64, bits=8,
             symmetric=False),
        # a long document keeps three quarters of its rows
        dict(name="compact_1x131072_i8", kind="compact", batch=1, context=131072, ragged=False, part=0.75, page=64, bits=8, symmetric=True, **cache),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _cache_of(rng):
    bits = rng.choice([8, 8, 4])
    return dict(kv_heads=rng.choice([1, 2, 4, 5, 8, 8, 12]), dim=rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 256] + [16, 48, 80, 112] * (bits == 8)),
                bits=bits, symmetric=rng.random() < 0.5, page=rng.choice([16, 16, 32, 48, 64, 128]))


def draw(rng):
    kind = rng.choice(["gated", "gated", "norm", "verify", "copy", "compact"])
    dtype = rng.choice(["float16", "float32"])
    if kind == "gated":
        group = rng.choice([32, 64, 128])
        while True:
            m, k, n = _log_int(rng, 1, 4096), group * _log_int(rng, 2, 14336 // group), _log_int(rng, 48, 14336)
            if m * k * n <= 2048 * 4096 * 11008 * (1 if dtype == "float16" else 0.5) and k * n <= 1 << 27:
                break
        return dict(kind=kind, m=m, k=k, n=n, bits=rng.choice([4, 8]), group=group, act=rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]),
                    bias=rng.random() < 0.4, dtype=dtype)
    if kind == "norm":
        while True:
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 16, 16384)
            if rng.random() < 0.7:
                cols = max(16, cols // 16 * 16)
            if rows * cols <= 1 << 25:
                break
        gate = rng.choice([0, 0, 1, rows])
        for per in (7, 5, 4, 3, 2):
            if gate == rows and rows % per == 0 and rng.random() < 0.3:
                gate = rows // per
        return dict(kind=kind, rows=rows, cols=cols, norm=rng.choice(["rms", "layer"]), post=rng.random() < 0.5, gate=gate, scale=rng.random() < 0.4,
                    dtype=dtype, residual=rng.choice([dtype, "float32"]))
    if kind == "verify":
        while True:
            batch, drafts, vocab = _log_int(rng, 1, 128), rng.choice([0, 1, 2, 3, 4, 5, 8, 16, 70]), _log_int(rng, 250, 262144)
            if batch * (drafts + 1) * vocab <= 1 << 26:
                break
        return dict(kind=kind, batch=batch, drafts=drafts, vocab=vocab, ragged=rng.random() < 0.5, given=rng.random() < 0.7, dtype=dtype)
    case = dict(kind=kind, **_cache_of(rng))
    row = case["kv_heads"] * case["dim"]
    if kind == "copy":
        most = (1 << 27) // (row * case["page"])
        return dict(case, pages=_log_int(rng, 1, min(8192, most)), padded=rng.random() < 0.4)
    while True:
        batch, context = _log_int(rng, 1, 128), _log_int(rng, 16, 131072)
        if batch * context * row <= 1 << 27:
            break
    return dict(case, batch=batch, context=context, ragged=rng.random() < 0.6, part=rng.choice([0.1, 0.5, 0.75, 0.9, 0.99]))


_DTYPES = {"float16": torch.float16, "float32": torch.float32}
_EPS = 1e-6


def _spread(case, most, least):
    """Sizes of the sequences of a batch; ragged: spread over the range by the golden ratio."""
    b = case["batch"]
    if not case["ragged"]:
        return [most] * b
    return [least + round((most - least) * ((i * 0.6180339887498949 + 1.0) % 1.0 or 1.0)) for i in range(b)]


# ---------------------------------------------------------------- a case's state
def _weight(gen, case):
    """Packed codes, scales and biases of a weight with the spread of a trained one."""
    n, k, bits, group = case["n"], case["k"], case["bits"], case["group"]
    w = (torch.randn(n, k, generator=gen, device="cuda") * 0.02).view(n, k // group, group)
    low = w.amin(-1)
    scale = ((w.amax(-1) - low) / (2 ** bits - 1)).clamp(min=1e-7)
    code = torch.round((w - low[..., None]) / scale[..., None]).clamp(0, 2 ** bits - 1).to(torch.uint8).view(n, k)
    if bits == 4:
        code = code[:, 0::2] | code[:, 1::2] << 4
    return code.contiguous().view(torch.int32), scale, low


def _channels(gen, *shape):
    """Activations: a few channels are larger than the rest, as in trained models."""
    return torch.randn(*shape, generator=gen, device="cuda") * (1 + 7 * (torch.rand(shape[-1], generator=gen, device="cuda") < 0.02).float())


def _prepare_gated(case, gen):
    s = {"x": _channels(gen, case["m"], case["k"]).to(_DTYPES[case["dtype"]])}
    for name in ("gate", "up"):
        s[name + "_packed"], s[name + "_scales"], s[name + "_biases"] = _weight(gen, case)
        if case["bias"]:
            s[name + "_bias"] = 0.1 * torch.randn(case["n"], generator=gen, device="cuda")
    s["out"] = torch.empty(case["m"], case["n"], dtype=s["x"].dtype, device="cuda")
    return s


def _prepare_norm(case, gen):
    rows, cols = case["rows"], case["cols"]
    s = {"x": _channels(gen, rows, cols).to(_DTYPES[case["dtype"]]), "r": (2 * _channels(gen, rows, cols)).to(_DTYPES[case["residual"]])}
    near_one = lambda: 1 + 0.2 * torch.randn(cols, generator=gen, device="cuda")
    s["weight"] = near_one()
    if case["post"]:
        s["post_weight"] = near_one()
    if case["norm"] == "layer":
        s["bias"] = 0.2 * torch.randn(cols, generator=gen, device="cuda")
        if case["post"]:
            s["post_bias"] = 0.2 * torch.randn(cols, generator=gen, device="cuda")
    if case["gate"]:
        s["gate"] = torch.randn(case["gate"], cols, generator=gen, device="cuda").to(s["x"].dtype)
    if case["scale"]:
        s["scale"] = 0.3 * torch.rand(cols, generator=gen, device="cuda")
    s["y_out"], s["r_out"] = torch.empty_like(s["x"]), torch.empty_like(s["r"])
    return s


def _prepare_verify(case, gen):
    dtype, vocab = _DTYPES[case["dtype"]], case["vocab"]
    counts = [n + 1 for n in _spread(case, case["drafts"], 0)]
    rows = sum(counts)
    s = {"starts": torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32).cuda()}
    s["target"] = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    s["draft"] = torch.empty(rows, vocab, dtype=dtype, device="cuda") if case["given"] else None
    s["tokens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    step = max(1, (1 << 24) // vocab)
    for lo in range(0, rows, step):
        hi = min(rows, lo + step)
        logits = 4 * torch.randn(hi - lo, vocab, generator=gen, device="cuda")
        s["target"][lo:hi] = torch.softmax(logits, -1)
        drawn = torch.softmax(logits + 0.6 * torch.randn(hi - lo, vocab, generator=gen, device="cuda"), -1)
        if s["draft"] is not None:
            s["draft"][lo:hi] = drawn
            drawn = s["draft"][lo:hi].float()
        # the token that follows each row, as the draft had it (a looked-up one: the likeliest)
        token = torch.multinomial(drawn, 1, generator=gen)[:, 0] if s["draft"] is not None else drawn.argmax(-1)
        s["tokens"][lo + 1:hi + 1] = token[:max(0, min(hi, rows - 1) - lo)].to(torch.int32)
    s["uniforms"], s["last"] = (torch.rand(n, generator=gen, device="cuda") for n in (rows, len(counts)))
    s["new"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    s["count"] = torch.empty(len(counts), dtype=torch.int32, device="cuda")
    return s


_BUFFERS = ("k_codes", "v_codes", "k_scale", "v_scale", "k_zero", "v_zero")


def _cache(case, pages, gen):
    """A cache whose every slot is taken (by codes and scales of any kind: nothing here computes with them)."""
    shape = (pages, case["kv_heads"], case["page"])
    make = lambda name: (torch.randint(0, 256, (*shape, case["dim"] * case["bits"] // 8), generator=gen, device="cuda", dtype=torch.uint8)
                         if name.endswith("codes") else torch.rand(shape, generator=gen, device="cuda"))
    return {name: make(name) for name in _BUFFERS[:4 if case["symmetric"] else 6]}


def _prepare_copy(case, gen):
    n = case["pages"]
    pages = 2 * n + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    s = {"cache": _cache(case, pages, gen), "src": order[:n].clone(), "dst": order[n:2 * n].clone()}
    if case["padded"]:
        s["src"][n - n // 8:] = -1
        s["dst"][n - n // 8:] = -1
    return s


def _prepare_compact(case, gen):
    lengths = _spread(case, case["context"], 1)
    page = case["page"]
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + 3
    s = {"cache": _cache(case, pages, gen)}
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((case["batch"], max(used)), -1, dtype=torch.int32), 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    s["table"] = table.cuda()
    kept = [_kept(case, n) for n in lengths]
    # the rows with the highest of random weights, in their order; the first few stay (the beginning of a text does)
    keep = []
    for n, m in zip(lengths, kept):
        weight = torch.rand(n, generator=gen, device="cuda")
        weight[:4] = 2
        keep.append(weight.topk(m).indices.sort().values)
    s["keep"] = torch.cat(keep).to(torch.int32)
    s["starts"] = torch.tensor([sum(kept[:b]) for b in range(len(kept) + 1)], dtype=torch.int32).cuda()
    return s


def _kept(case, length):
    return max(1, round(case["part"] * length))


_PREPARE = {"gated": _prepare_gated, "norm": _prepare_norm, "verify": _prepare_verify, "copy": _prepare_copy, "compact": _prepare_compact}


def prepare(case, seed):
    s = _PREPARE[case["kind"]](case, torch.Generator(device="cuda").manual_seed(seed))
    s["case"] = dict(case)
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

    def put(name):
        t = L.Tensor.empty(tuple(s[name].shape), str(s[name].dtype).removeprefix("torch."), "hip")
        _view(t).copy_(s[name])
        s[name] = _view(t)
        return t

    case = s["case"]
    s["own"] = {name: put(name) for name, v in list(s.items()) if isinstance(v, torch.Tensor)}
    if "cache" in s:
        cache = Q.PagedKVCache(s["cache"]["k_scale"].shape[0], case["page"], case["kv_heads"], case["dim"],
                               Q.per_channel_symmetric if case["symmetric"] else Q.per_channel_affine, Q.qint8 if case["bits"] == 8 else Q.qint4)
        for name, t in s["cache"].items():
            held = _view(getattr(cache, name)).view(t.dtype)
            held.copy_(t)
            s["cache"][name] = held
        s["own"]["cache"] = cache


# ---------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if own:
        return _OWN[case["kind"]](s, s["own"], case)
    return _PLAIN[case["kind"]](s, case)


def _own_gated(s, t, case):
    from lucid_amd.quantization import _qgemm

    _qgemm.quantized_gated_matmul(t["x"], (t["gate_packed"], t["gate_scales"], t["gate_biases"]), (t["up_packed"], t["up_scales"], t["up_biases"]),
                                  activation=case["act"], group_size=case["group"], bits=case["bits"], gate_bias=t.get("gate_bias"),
                                  up_bias=t.get("up_bias"), out=t["out"])
    return s["out"]


def _own_norm(s, t, case):
    import lucid_amd.nn.functional as F

    F.residual_norm(t["x"], t["r"], t["weight"], t.get("bias"), norm=case["norm"], eps=_EPS, post=case["post"], post_weight=t.get("post_weight"),
                    post_bias=t.get("post_bias"), gate=t.get("gate"), scale=t.get("scale"), out=t["y_out"], residual_out=t["r_out"])
    return s["y_out"], s["r_out"]


def _own_verify(s, t, case):
    import lucid_amd.nn.functional as F

    F.verify_drafts(t["target"], t["tokens"], t["starts"], t["uniforms"], t["last"], draft=t.get("draft"), out=(t["new"], t["count"]))
    return s["new"], s["count"]


def _own_copy(s, t, case):
    import lucid_amd.quantization as Q

    Q.kv_cache_copy(t["cache"], t["src"], t["dst"])
    return s["cache"]


def _own_compact(s, t, case):
    import lucid_amd.quantization as Q

    Q.kv_cache_compact(t["cache"], t["table"], t["keep"], t["starts"])
    return s["cache"]


_OWN = {"gated": _own_gated, "norm": _own_norm, "verify": _own_verify, "copy": _own_copy, "compact": _own_compact}


def _decoded(case, packed, scales, biases):
    """Float32 weight of packed codes."""
    code = packed.view(torch.uint8)
    if case["bits"] == 4:
        code = torch.stack((code & 15, code >> 4), -1).flatten(1)
    group = code.view(case["n"], -1, case["group"]).float()
    return (group * scales[..., None] + biases[..., None]).view(case["n"], case["k"])


def _act(case, v):
    if case["act"] == "silu":
        return v / (1 + torch.exp(-v))
    if case["act"] == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    if case["act"] == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v.clamp(min=0)


def _plain_gated(s, case):
    x = s["x"].float()
    gate, up = (x @ _decoded(case, s[n + "_packed"], s[n + "_scales"], s[n + "_biases"]).t() for n in ("gate", "up"))
    if case["bias"]:
        gate, up = gate + s["gate_bias"], up + s["up_bias"]
    return (_act(case, gate) * up).to(s["x"].dtype)


def _normed(case, v, weight, bias):
    if case["norm"] == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + _EPS) * weight
    return v if bias is None else v + bias


def _plain_norm(s, case):
    v = s["x"].float()
    if case["post"]:
        v = _normed(case, v, s["post_weight"], s.get("post_bias"))
    if case["scale"]:
        v = v * s["scale"]
    if case["gate"]:
        v = (v.view(case["gate"], -1, case["cols"]) * s["gate"].float()[:, None]).view(case["rows"], case["cols"])
    r = s["r"].float() + v
    return _normed(case, r, s["weight"], s.get("bias")).to(s["x"].dtype), r.to(s["r"].dtype)


def _plain_verify(s, case):
    starts, tokens = s["starts"].long(), s["tokens"].long()
    rows, most = tokens.numel(), case["drafts"]
    first, count = starts[:-1], starts[1:] - starts[:-1]
    # which drafts would be accepted, [sequence, place]; u q(x) < p(x) in 64 bits: exact
    place = torch.arange(most, device="cuda")
    row = (first[:, None] + place).clamp(max=rows - 1)
    x = tokens[(row + 1).clamp(max=rows - 1)]
    p = s["target"][row, x].double()
    q = s["draft"][row, x].double() if case["given"] else torch.ones_like(p)
    accept = (s["uniforms"][row].double() * q < p) & (place < (count - 1)[:, None])
    accepted = accept.long().cumprod(1).sum(1)
    # the row that decides, and what it leaves
    at = first + accepted
    weight = s["target"][at].double()
    refused = accepted < count - 1
    drafted = tokens[(at + 1).clamp(max=rows - 1)]
    if case["given"]:
        rest = (weight - s["draft"][at].double()).clamp(min=0)
    else:
        rest = weight.scatter(1, drafted[:, None], 0.0)
    rest = rest * refused[:, None]
    some = rest.sum(1) > 0
    weight = torch.where(some[:, None], rest, weight)
    total = weight.cumsum(1)
    over = (total > (s["last"].double() * total[:, -1])[:, None]) & (weight > 0)
    following = over.long().argmax(1)
    # the new tokens in their sequence's rows, -1 behind them
    i = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts, i, right=True) - 1
    step = i - first[seq]
    new = torch.where(step < accepted[seq], tokens[(i + 1).clamp(max=rows - 1)], torch.where(step == accepted[seq], following[seq], -1))
    return new.to(torch.int32), (accepted + 1).to(torch.int32)


def _plain_copy(s, case):
    n = case["pages"] - case["pages"] // 8 if case["padded"] else case["pages"]  # (the others have no page)
    src, dst = s["src"][:n].long(), s["dst"][:n].long()
    for t in s["cache"].values():
        t[dst] = t[src]
    return s["cache"]


def _plain_compact(s, case):
    starts, keep, page = s["starts"].long(), s["keep"].long(), case["page"]
    i = torch.arange(keep.numel(), device="cuda")
    seq = torch.searchsorted(starts, i, right=True) - 1
    to = i - starts[seq]
    table = s["table"].long()
    src, dst = table[seq, keep // page], table[seq, to // page]
    for t in s["cache"].values():
        t[dst, :, to % page] = t[src, :, keep % page]
    return s["cache"]


_PLAIN = {"gated": _plain_gated, "norm": _plain_norm, "verify": _plain_verify, "copy": _plain_copy, "compact": _plain_compact}


# ---------------------------------------------------------------- the definition, in 64 bits
def _exact_weight(case, s, name):
    """Rows of float64 from the words' bits."""
    bits = case["bits"]
    shift = torch.arange(0, 32, bits, device="cuda", dtype=torch.int32)
    code = (s[name + "_packed"][..., None] >> shift) & (2 ** bits - 1)
    of_group = torch.arange(case["k"], device="cuda") // case["group"]
    return code.reshape(case["n"], case["k"]).double() * s[name + "_scales"].double()[:, of_group] + s[name + "_biases"].double()[:, of_group]


def _exact_gated(s, case):
    x, half = s["x"].double(), []
    for name in ("gate", "up"):
        v = torch.nn.functional.linear(x, _exact_weight(case, s, name))
        half.append(v + s[name + "_bias"].double() if case["bias"] else v)
    g, u = half
    if case["act"] == "gelu":
        return g * torch.special.ndtr(g) * u
    return (g.relu() if case["act"] == "relu" else torch.sigmoid(g) * (g if case["act"] == "silu" else 1.0)) * u


def _exact_norm(s, case):
    d = {n: t.double() for n, t in s.items() if isinstance(t, torch.Tensor)}

    def norm(v, weight, bias):
        if case["norm"] == "layer":
            return torch.nn.functional.layer_norm(v, (case["cols"],), weight, bias, _EPS)
        return weight * v * (v.square().sum(-1, keepdim=True) / case["cols"] + _EPS) ** -0.5

    block = norm(d["x"], d["post_weight"], d.get("post_bias")) if case["post"] else d["x"]
    if case["gate"]:
        block = block * d["gate"].repeat_interleave(case["rows"] // case["gate"], 0)
    r = torch.addcmul(d["r"], block, d["scale"]) if case["scale"] else d["r"] + block
    return norm(r, d["weight"], d.get("bias")), r


def exact(case, seed):
    """Of norms and gated projections; what is verified or moved are whole numbers and bits, which are compared as such."""
    if case["kind"] not in ("gated", "norm"):
        return None
    s = _PREPARE[case["kind"]](case, torch.Generator(device="cuda").manual_seed(seed))
    return (_exact_gated if case["kind"] == "gated" else _exact_norm)(s, case)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    size = lambda name: 2 if case[name] == "float16" else 4
    if kind == "gated":
        m, k, n = case["m"], case["k"], case["n"]
        weights = 2 * n * (k * case["bits"] // 8 + 8 * (k // case["group"]) + 4 * case["bias"])
        return {"bytes": weights + m * (k + n) * size("dtype"), "flops": 4 * m * n * k}
    if kind == "norm":
        vectors = (1 + case["post"]) * (2 if case["norm"] == "layer" else 1) + case["scale"]
        return {"bytes": case["rows"] * case["cols"] * 2 * (size("dtype") + size("residual")) + case["cols"] * (4 * vectors + case["gate"] * size("dtype")),
                "flops": 0}
    if kind == "verify":
        # of each sequence the row that decides (of a refused draft the draft's too: counted for half of them), and what its drafts have
        counts = [n + 1 for n in _spread(case, case["drafts"], 0)]
        rows = len(counts) * (1.5 if case["given"] and case["drafts"] else 1.0)
        return {"bytes": rows * case["vocab"] * size("dtype") + sum(counts) * (12 + 2 * size("dtype")) + 12 * len(counts), "flops": 0}
    row = 2 * case["kv_heads"] * (case["dim"] * case["bits"] // 8 + (4 if case["symmetric"] else 8))  # a token's keys and values in the cache
    if kind == "copy":
        n = case["pages"] - case["pages"] // 8 if case["padded"] else case["pages"]
        return {"bytes": 2 * n * case["page"] * row + 8 * case["pages"], "flops": 0}
    kept = sum(_kept(case, n) for n in _spread(case, case["context"], 1))
    return {"bytes": 2 * kept * row + 4 * kept, "flops": 0}

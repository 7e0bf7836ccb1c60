"""What is measured of the 4-bit key / value cache: appending tokens and reading them back, attention over the cache
(with the attention weight each slot has received), and eviction by that weight.

run() computes a case with elementary torch operations, or, where `own` is true, with the calls a program makes of the
framework's cache (we.py). A slot of the cache holds, per kv head, a K row and a V row of `dim` values in groups of 64: a
4-bit code each (two to a byte, the first in the low bits) and per group an f16 scale and an f16 minimum, value = minimum
+ scale * code. The cache is one buffer of four regions: K codes, K scales, V codes, V scales, each [batch, kv head, slot].
Which code a value gets is part of the format, roundings included: with every step rounded to f32, minimum = f16(lo),
scale = f16((hi - lo) / 15) and code = round((x - minimum) / scale), ties to even, within 0 .. 15 (0 where scale is 0).
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
GROUP = 64
F16_MAX = 65504.0


def listed():
    return [
        # one token after a short prompt, a single sequence: latency
        {"name": "decode_short", "kind": "attention", "batch": 1, "heads": 28, "kv_heads": 4, "dim": 128, "tokens": 1,
         "len": 131, "ragged": False, "causal": True, "weight": False, "dtype": "f16"},
        # a decode step of a batch whose sequences differ in length, with the weights an eviction will go by
        {"name": "decode_batch", "kind": "attention", "batch": 16, "heads": 28, "kv_heads": 4, "dim": 128, "tokens": 1,
         "len": 4093, "ragged": True, "causal": True, "weight": True, "dtype": "bf16"},
        # a decode step over long documents: the cache's bandwidth
        {"name": "decode_long", "kind": "attention", "batch": 4, "heads": 32, "kv_heads": 8, "dim": 128, "tokens": 1,
         "len": 65521, "ragged": True, "causal": True, "weight": False, "dtype": "f16"},
        # a few drafted tokens checked at once, no shared kv heads, in f32
        {"name": "verify_f32", "kind": "attention", "batch": 3, "heads": 24, "kv_heads": 24, "dim": 64, "tokens": 5,
         "len": 1031, "ragged": True, "causal": True, "weight": False, "dtype": "f32"},
        # the next piece of a prompt, with the weights
        {"name": "chunk", "kind": "attention", "batch": 2, "heads": 28, "kv_heads": 4, "dim": 128, "tokens": 509,
         "len": 4099, "ragged": True, "causal": True, "weight": True, "dtype": "bf16"},
        # a long prompt in one call
        {"name": "prompt", "kind": "attention", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "tokens": 2048,
         "len": 8192, "ragged": False, "causal": True, "weight": False, "dtype": "f16"},
        # one new token of every sequence of a batch, written and read back
        {"name": "append_step", "kind": "append", "batch": 16, "kv_heads": 4, "dim": 128, "tokens": 1, "len": 1000,
         "ragged": True, "dtype": "bf16"},
        # a padded batch of prompts, in the framework's default type
        {"name": "append_prompt", "kind": "append", "batch": 4, "kv_heads": 8, "dim": 128, "tokens": 2039, "len": 0,
         "ragged": True, "dtype": "f32"},
        # one slot given up per sequence and head, as after each decode step of a full cache
        {"name": "evict_step", "kind": "evict", "batch": 16, "kv_heads": 4, "dim": 128, "len": 4097, "ragged": False,
         "keep": 4096, "sinks": 4, "recent": 512},
        # a long prompt cut down to a budget
        {"name": "evict_prompt", "kind": "evict", "batch": 4, "kv_heads": 8, "dim": 128, "len": 32749, "ragged": True,
         "keep": 8192, "sinks": 4, "recent": 1024},
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "append", "evict"])
    dim = rng.choice([64, 128, 128, 128, 192, 256])
    kv = rng.choice([1, 2, 4, 8])
    if kind == "attention":
        group = rng.choice([1, 2, 4, 5, 7, 8])
        decode = rng.random() < 0.6
        tokens = rng.choice([1, 1, 1, 1, 2, 3, 8]) if decode else _log(rng, 16, 1024)
        batch = _log(rng, 1, 24) if decode else rng.randint(1, 2)
        # at most the bytes of the longest decode step and the products of the longest prompt
        longest = min(65536, 200_000_000 // (batch * kv * dim)) if decode else 8192
        longest = max(tokens, min(longest, 60_000_000_000 // (batch * tokens * kv * group * dim)))
        return {"kind": kind, "batch": batch, "heads": kv * group, "kv_heads": kv, "dim": dim, "tokens": tokens,
                "len": _log(rng, tokens, longest), "ragged": rng.random() < 0.7, "causal": rng.random() < 0.8,
                "weight": rng.random() < 0.4, "dtype": rng.choice(["bf16", "bf16", "f16", "f16", "f32"])}
    batch = _log(rng, 1, 24)
    if kind == "append":
        return {"kind": kind, "batch": batch, "kv_heads": kv, "dim": dim,
                "tokens": _log(rng, 1, min(4096, 6_000_000 // (batch * kv * dim))), "len": _log(rng, 1, 4096),
                "ragged": rng.random() < 0.6, "dtype": rng.choice(["bf16", "f16", "f32"])}
    length = _log(rng, 2, min(65536, 60_000_000 // (batch * kv * dim)))
    keep = rng.choice([length - 1, max(1, length - length // 5), max(1, length // 3), max(1, length // 8)])
    return {"kind": kind, "batch": batch, "kv_heads": kv, "dim": dim, "len": length, "ragged": rng.random() < 0.6,
            "keep": keep, "sinks": rng.choice([0, 4]), "recent": rng.choice([0, keep // 8, keep // 2])}


def _lens(case):
    """the slots in use of each sequence before the call: all `len`, or (ragged) from there down to about half of it"""
    n, b = case["len"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    low = case["tokens"] if case["kind"] == "attention" else 1
    return [max(min(low, n), n - i * n // (2 * b)) for i in range(b)]


def _counts(case):
    """the new tokens of each sequence: all of them, or (an append of a padded batch) fewer"""
    t, b = case["tokens"], case["batch"]
    return [t - i * t // (2 * b) if case["ragged"] and case["kind"] == "append" else t for i in range(b)]


def _capacity(case):
    return -(-(case["len"] + case.get("tokens", 0)) // 64) * 64


# ------------------------------------------------------------------------------------------------- the cache's format

def _regions(flat, batch, kv_heads, dim, capacity):
    """K codes, K scales, V codes, V scales (codes as bytes, scales as pairs of f16) as views of the cache's bytes"""
    rows = batch * kv_heads * capacity
    sizes = [rows * dim // 2, rows * dim // GROUP * 4] * 2
    kc, ks, vc, vs = torch.split(flat, sizes)
    shape = (batch, kv_heads, capacity)
    return (kc.view(*shape, dim // 2), ks.view(torch.float16).view(*shape, dim // GROUP, 2),
            vc.view(*shape, dim // 2), vs.view(torch.float16).view(*shape, dim // GROUP, 2))


def _quantize(x):
    """codes (two to a byte) and (scale, minimum) of x [..., dim], in f32"""
    g = x.float().clamp(-F16_MAX, F16_MAX).unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    mn, s = lo.half(), ((hi - lo) / torch.full_like(hi, 15)).half()  # by a tensor: a number's reciprocal would be rounded first
    u = torch.where(s > 0, ((g - mn.float()) / s.float()).round().clamp(0, 15), 0.0).to(torch.uint8).flatten(-2)
    return u[..., 0::2] | (u[..., 1::2] << 4), torch.cat([s, mn], -1)


def _dequantize(codes, scales):
    """[..., dim] in f32 of codes [..., dim / 2] and scales [..., dim / 64, 2]"""
    u = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return (scales[..., 1:].float() + scales[..., :1].float() * u).flatten(-2)


# ------------------------------------------------------------------------------------------------------------ inputs

def _data(case, seed, device="cuda"):
    """the tensors a program holds before the call"""
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    b, kv, d, cap = case["batch"], case["kv_heads"], case["dim"], _capacity(case)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    def heads_of(*shape):
        """K or V rows as a model makes them: every channel with an offset and a spread of its own"""
        return normal(*shape, d) * (0.5 + normal(kv, d).abs()) + normal(kv, d) * 0.5

    flat = torch.zeros(b * kv * cap * (d + d // 8), dtype=torch.uint8, device=device)
    s = {"cache": flat, "lens": torch.tensor(_lens(case), dtype=torch.int32, device=device)}
    if case["kind"] != "append":
        kc, ks, vc, vs = _regions(flat, b, kv, d, cap)
        for codes, scales in ((kc, ks), (vc, vs)):
            for i in range(b):  # one sequence at a time: the f32 rows of a long cache are eight times its size
                c, sc = _quantize(heads_of(case["len"], kv).transpose(0, 1))
                codes[i, :, :case["len"]] = c
                scales[i, :, :case["len"]] = sc
    if case["kind"] == "attention":
        s["q"] = normal(b, case["tokens"], case["heads"], d).to(TORCH[case["dtype"]])
        if case["weight"]:
            s["weight"] = normal(b, kv, cap).abs()
    elif case["kind"] == "append":
        dt = TORCH[case["dtype"]]
        s["k"], s["v"] = (heads_of(b, case["tokens"], kv).to(dt) for _ in range(2))
        s["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=device)
        s["seen"] = s["lens"] + 7  # an earlier eviction gave up seven slots
        s["pos"] = torch.zeros(b, kv, cap, dtype=torch.int32, device=device)
        s["weight"] = normal(b, kv, cap).abs()
    else:
        # attention received so far: heavy-tailed; the newest slots have little yet, some exactly none
        s["weight"] = torch.exp(2 * normal(b, kv, cap)) * (torch.rand(b, kv, cap, generator=gen, device=device) > 0.02)
        # slots hold tokens in another order than they came in once an eviction has filled holes
        slot = torch.arange(cap, device=device)
        old = slot < (s["lens"] - case["recent"]).view(b, 1, 1)
        key = torch.where(old, torch.rand(b, kv, cap, generator=gen, device=device, dtype=torch.float64), 1.0 + slot)
        s["pos"] = key.argsort(-1).int()
        s["seen"] = s["lens"].clone()
    return s


_graph = None


def _the_graph():
    """The context that serves every case of a process."""
    global _graph
    if _graph is None:
        import pathlib
        import sys
        sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "web-engine_amd"))
        import we
        _graph = we.Graph(0)
    return _graph


class _Device:
    """A buffer of the graph seen by torch; the torch view keeps it alive."""

    def __init__(self, graph, nbytes):
        self.graph, self.buf = graph, graph.buffer(nbytes)
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (self.buf.ptr, False), "version": 2}

    def __del__(self):
        if self.graph.ctx is not None:
            self.graph.free(self.buf)


def _empty(shape, dtype):
    """zeros: in a buffer of the framework's graph where `own` is true, as its calls take them"""
    if not own:
        return torch.zeros(shape, dtype=dtype, device="cuda")
    n = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
    return torch.as_tensor(_Device(_the_graph(), n), device="cuda").view(dtype).reshape(shape)


def prepare(case, seed):
    s = _data(case, seed)
    if own:  # the same values in the graph's buffers
        held = {k: _empty(tuple(t.shape), t.dtype) for k, t in s.items()}
        _the_graph().sync()  # a fresh buffer is zeroed on the graph's stream
        for k, t in s.items():
            held[k].copy_(t)
        s = held
    b, kv, d, cap = case["batch"], case["kv_heads"], case["dim"], _capacity(case)
    if case["kind"] == "attention":
        s["out"] = _empty(tuple(s["q"].shape), s["q"].dtype)
        if case["weight"]:
            s["weight_out"] = _empty((b, kv, cap), torch.float32)
    elif case["kind"] == "append":
        s["lens_out"], s["seen_out"] = _empty((b,), torch.int32), _empty((b,), torch.int32)
        s["k_out"], s["v_out"] = (_empty(tuple(s["k"].shape), s["k"].dtype) for _ in range(2))
    else:
        s["lens_out"] = _empty((b,), torch.int32)
        s["weight_out"], s["pos_out"] = _empty((b, kv, cap), torch.float32), _empty((b, kv, cap), torch.int32)
    s["case"] = case
    if own:
        import we
        s["handle"] = we.Cache4(_the_graph(), b, kv, d, cap, data=s["cache"].data_ptr())
        _the_graph().sync()
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------------------------------- the plain forms

def _attention(s):
    case = s["case"]
    b, kv, d, n, length = case["batch"], case["kv_heads"], case["dim"], case["tokens"], case["len"]
    kc, ks, vc, vs = (t[:, :, :length] for t in _regions(s["cache"], b, kv, d, _capacity(case)))
    group = case["heads"] // kv
    q = s["q"].float().view(b, n, kv, group, d).permute(0, 2, 1, 3, 4).reshape(b, kv, n * group, d)
    scores = q @ _dequantize(kc, ks).transpose(-1, -2) / math.sqrt(d)
    visible = s["lens"].view(b, 1, 1, 1) - torch.zeros(n, 1, dtype=torch.int32, device=q.device)
    if case["causal"]:
        visible = visible - torch.arange(n - 1, -1, -1, device=q.device).view(n, 1)
    visible = visible.expand(b, 1, n, group).reshape(b, 1, n * group, 1)
    hidden = torch.arange(length, device=q.device) >= visible
    scores.masked_fill_(hidden, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-37)
    o = (p @ _dequantize(vc, vs)).view(b, kv, n, group, d).permute(0, 2, 1, 3, 4)
    s["out"].copy_(o.reshape(b, n, kv * group, d))
    if not case["weight"]:
        return s["out"]
    used = torch.arange(length, device=q.device) < s["lens"].view(b, 1, 1)
    s["weight_out"][:, :, :length] = torch.where(used, s["weight"][:, :, :length] + p.sum(-2), s["weight_out"][:, :, :length])
    return {"out": s["out"], "weight": s["weight_out"]}


def _append(s):
    case = s["case"]
    b, kv, d, n, cap = case["batch"], case["kv_heads"], case["dim"], case["tokens"], _capacity(case)
    regions = _regions(s["cache"], b, kv, d, cap)
    step = torch.arange(n, device=s["k"].device)
    slot = s["lens"].view(b, 1).long() + step
    live = (step < s["counts"].view(b, 1)) & (slot < cap)
    seq, at = live.nonzero(as_tuple=True)
    to = slot[seq, at]
    for x, codes, scales in ((s["k"], *regions[:2]), (s["v"], *regions[2:])):
        c, sc = _quantize(x)
        codes[seq, :, to] = c[seq, at]
        scales[seq, :, to] = sc[seq, at]
    s["pos"][seq, :, to] = (s["seen"].view(b, 1) + step)[seq, at].int().unsqueeze(-1)
    s["weight"][seq, :, to] = 0.0
    torch.minimum(s["lens"] + s["counts"], torch.tensor(cap, device=to.device), out=s["lens_out"])
    torch.add(s["seen"], s["counts"], out=s["seen_out"])
    for out, codes, scales in ((s["k_out"], *regions[:2]), (s["v_out"], *regions[2:])):
        out[seq, at] = _dequantize(codes[seq, :, to], scales[seq, :, to]).to(out.dtype)
    return {name: s[name] for name in ("k_out", "v_out", "lens_out", "seen_out", "pos", "weight")}


def _evict(s):
    case = s["case"]
    b, kv, d, length = case["batch"], case["kv_heads"], case["dim"], case["len"]
    regions = _regions(s["cache"], b, kv, d, _capacity(case))
    lens = s["lens"].view(b, 1, 1).long()
    left = lens.clamp(max=case["keep"])
    slot = torch.arange(length, device=lens.device).expand(b, kv, length)
    weight, pos = s["weight"][:, :, :length], s["pos"][:, :, :length]
    kept = (pos < case["sinks"]) | (pos >= s["seen"].view(b, 1, 1) - case["recent"])
    rank = torch.where(slot < lens, kept.long(), 2)
    order = weight.argsort(dim=-1, stable=True)
    order = order.gather(-1, rank.gather(-1, order).argsort(dim=-1, stable=True))
    gone = torch.empty_like(kept).scatter_(-1, order, slot < lens - left)
    hole = gone & (slot < left)
    move = ~gone & (slot >= left) & (slot < lens)
    source = torch.zeros(b, kv, length + 1, dtype=torch.long, device=lens.device)
    source.scatter_(-1, torch.where(move, move.long().cumsum(-1) - 1, length), slot)
    come = torch.where(hole, source.gather(-1, (hole.long().cumsum(-1) - 1).clamp(min=0)), slot)
    top = min(case["keep"], length)
    come, live = come[..., :top], slot[..., :top] < left
    for r in regions:
        flat = r.flatten(3)
        flat[:, :, :top] = flat.gather(2, come.unsqueeze(-1).expand(*come.shape, flat.shape[-1]))
    for out, held in ((s["weight_out"], weight), (s["pos_out"], pos)):
        out[:, :, :top] = torch.where(live, held.gather(-1, come), out[:, :, :top])
    s["lens_out"].copy_(left.view(b))
    return _evicted(s)


def _evicted(s):
    """An eviction moves slots and computes nothing, so the cache's words are returned as they are: they have to be equal."""
    return {"cache": s["cache"].view(torch.int32), "lens": s["lens_out"], "weight": s["weight_out"], "pos": s["pos_out"]}


# -------------------------------------------------------------------------------------------------- the framework's

def _ptr(s, name):
    return s[name].data_ptr() if name in s else None


def _own(s):
    import we
    g, case, cache = _the_graph(), s["case"], s["handle"]
    if case["kind"] == "attention":
        g.cache4_attention(cache, case["tokens"], case["heads"], case["causal"], we.DTYPES[case["dtype"]], _ptr(s, "q"),
                           _ptr(s, "lens"), _ptr(s, "out"), max_len=case["len"], weight=_ptr(s, "weight"),
                           weight_out=_ptr(s, "weight_out"))
        return {"out": s["out"], "weight": s["weight_out"]} if case["weight"] else s["out"]
    if case["kind"] == "append":
        dt = we.DTYPES[case["dtype"]]
        g.cache4_append(cache, case["tokens"], dt, _ptr(s, "k"), _ptr(s, "v"), _ptr(s, "lens"), _ptr(s, "lens_out"),
                        counts=_ptr(s, "counts"), seen=_ptr(s, "seen"), seen_out=_ptr(s, "seen_out"), pos=_ptr(s, "pos"),
                        weight=_ptr(s, "weight"))
        g.cache4_load(cache, case["tokens"], dt, _ptr(s, "k_out"), _ptr(s, "v_out"), first=_ptr(s, "lens"),
                      lens=_ptr(s, "lens_out"))
        return {name: s[name] for name in ("k_out", "v_out", "lens_out", "seen_out", "pos", "weight")}
    g.cache4_evict(cache, case["keep"], _ptr(s, "lens"), _ptr(s, "lens_out"), _ptr(s, "weight"), _ptr(s, "weight_out"),
                   _ptr(s, "pos"), _ptr(s, "pos_out"), seen=_ptr(s, "seen"), sinks=case["sinks"], recent=case["recent"],
                   max_len=case["len"])
    return _evicted(s)


def run(state):
    if own:
        return _own(state)
    return {"attention": _attention, "append": _append, "evict": _evict}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------- what it takes

def work(case):
    kv, d = case["kv_heads"], case["dim"]
    slot = kv * (d + d // 8)  # bytes of K and V, codes and scales
    lens = _lens(case)
    if case["kind"] == "attention":
        n = case["tokens"]
        pairs = sum(sum(max(0, x - i) for i in range(n)) if case["causal"] else n * x for x in lens)
        return {"bytes": sum(lens) * (slot + (8 * kv if case["weight"] else 0)) +
                2 * len(lens) * n * case["heads"] * d * BYTES[case["dtype"]], "flops": 4 * d * case["heads"] * pairs}
    if case["kind"] == "append":
        n = sum(_counts(case))
        return {"bytes": n * (2 * slot + 4 * kv * d * BYTES[case["dtype"]] + 8 * kv), "flops": 10 * n * kv * d}
    total = 0
    for x in lens:
        left = min(x, case["keep"])
        free = max(0, x - case["sinks"] - case["recent"])  # unprotected: evicted slots are spread over these
        moves = min(x - left, left * min(1.0, (x - left) / free) if free else x - left)
        total += kv * 8 * (x + left) + moves * 2 * slot
    return {"bytes": int(total), "flops": 0}


# ------------------------------------------------------------------------------------------ the results in 64 bits

def _values(codes, scales):
    """the stored values in f64, from the definition: minimum + scale * code"""
    lo, hi = codes.to(torch.int16) % 16, torch.div(codes.to(torch.int16), 16, rounding_mode="floor")
    d = 2 * codes.shape[-1]
    u = torch.empty(*codes.shape[:-1], d, dtype=torch.float64, device=codes.device)
    u[..., 0::2], u[..., 1::2] = lo.double(), hi.double()
    s = scales.double().repeat_interleave(GROUP, dim=-2)
    return u * s[..., 0] + s[..., 1]


def _exact_attention(case, s):
    b, kv, d, n, cap = case["batch"], case["kv_heads"], case["dim"], case["tokens"], _capacity(case)
    kc, ks, vc, vs = _regions(s["cache"], b, kv, d, cap)
    group = case["heads"] // kv
    out = torch.zeros(b, n, case["heads"], d, dtype=torch.float64, device=kc.device)
    received = torch.zeros(b, kv, cap, dtype=torch.float64, device=kc.device)
    for i, length in enumerate(_lens(case)):
        for g in range(kv):
            k, v = _values(kc[i, g, :length], ks[i, g, :length]), _values(vc[i, g, :length], vs[i, g, :length])
            kt = k.t().contiguous()
            total = torch.zeros(length, dtype=torch.float64, device=kc.device)
            for h in range(g * group, (g + 1) * group):
                scores = s["q"][i, :, h].double() @ kt / d ** 0.5
                if case["causal"]:
                    last = length - n + torch.arange(n, device=kc.device)
                    scores[torch.arange(length, device=kc.device)[None] > last[:, None]] = -math.inf
                p = torch.softmax(scores, -1)
                out[i, :, h] = p @ v
                total += p.sum(0)
            if case["weight"]:
                received[i, g, :length] = s["weight"][i, g, :length].double() + total
    return {"out": out, "weight": received} if case["weight"] else out


def _exact_append(case, s):
    b, kv, n, cap = case["batch"], case["kv_heads"], case["tokens"], _capacity(case)
    pos, weight = s["pos"].clone(), s["weight"].double()
    outs = []

    def f32(v):  # the format's roundings: of a sum, a difference or a quotient in 64 bits they are those of 32-bit arithmetic
        return v.float().double()

    for x in (s["k"], s["v"]):
        g = x.double().clamp(-F16_MAX, F16_MAX).unflatten(-1, (-1, GROUP))
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        mn, sc = lo.half().double(), f32(f32(hi - lo) / 15).half().double()
        code = torch.where(sc > 0, torch.round(f32(f32(g - mn) / sc)), 0.0).clamp(0, 15)
        outs.append((mn + sc * code).flatten(-2))
    for i, (at, count) in enumerate(zip(_lens(case), _counts(case))):
        for y in outs:
            y[i, count:] = 0
        pos[i, :, at:at + count] = (int(s["seen"][i]) + torch.arange(count, device=pos.device)).int()
        weight[i, :, at:at + count] = 0
    return {"k_out": outs[0], "v_out": outs[1], "lens_out": s["lens"] + s["counts"], "seen_out": s["seen"] + s["counts"],
            "pos": pos, "weight": weight}


def _exact_evict(case, s):
    import numpy as np
    b, kv = case["batch"], case["kv_heads"]
    regions = [r.flatten(3) for r in _regions(s["cache"], b, kv, case["dim"], _capacity(case))]
    weights, where = torch.zeros_like(s["weight"]), torch.zeros_like(s["pos"])
    lens = []
    for i, length in enumerate(_lens(case)):
        left = min(length, case["keep"])
        lens.append(left)
        for g in range(kv):
            w, p = s["weight"][i, g, :length].cpu().numpy(), s["pos"][i, g, :length].cpu().numpy()
            safe = (p < case["sinks"]) | (p >= int(s["seen"][i]) - case["recent"])
            out = np.lexsort((np.arange(length), w, safe))[:length - left]
            stays = np.ones(length, bool)
            stays[out] = False
            come = np.arange(left)
            come[~stays[:left]] = left + np.flatnonzero(stays[left:])
            at = torch.from_numpy(come).to(weights.device)
            weights[i, g, :left], where[i, g, :left] = s["weight"][i, g][at], s["pos"][i, g][at]
            for r in regions:
                r[i, g, :left] = r[i, g][at]
    return {"cache": s["cache"].view(torch.int32), "lens": torch.tensor(lens, dtype=torch.int32), "weight": weights, "pos": where}


def exact(case, seed):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    if case["kind"] == "attention" and work(case)["flops"] > 1e13:
        return None  # over the time an exact result may take
    with torch.no_grad():
        return {"attention": _exact_attention, "append": _exact_append, "evict": _exact_evict}[case["kind"]](case, _data(case, seed, device))

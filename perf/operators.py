"""The serving operators in 8 and 4 bits, as a program that decodes with irontensor_amd calls them: the
quantised key/value cache, the attention that reads it, and the linear layer in 8-bit integers.

`listed()` names the fixed cases, `draw(rng)` gives another one of the same ranges. A case's `kind`:

  store   kv_cache_write of `n` new tokens of every sequence, then kv_cache_read of the part of the
          cache that they went to
  attend  cached_attention of `n` queries of every sequence over its cached tokens
  linear  linear_i8: the activations quantised per token, times a weight that was quantised per output
          channel when the model was loaded, with the scales and an optional bias

The cache holds a token's key in groups of 32 channels and its value whole, each with one scale
s = bf16(max|x| / L), L = 7 in 4 bits and 127 in 8, and the codes rne(x / s). Activations and upstream
values are N(0, 1), with some channels of the keys eight times as large, as keys have them; weights
N(0, 0.02).
"""
import math

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_GROUP = 32          # channels of a key that share a scale
_TINY = 2.0 ** -126  # a smaller scale is stored as zero


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One token of the 256-wide model through its Q|K|V projection: the smallest product.
        {"name": "linear_token_f32", "kind": "linear", "m": 1, "n": 768, "k": 256, "dtype": "f32", "bias": False},
        # A few tokens against a large weight: decoding, bound by reading the weight.
        {"name": "linear_decode_bf16", "kind": "linear", "m": 4, "n": 11008, "k": 4096, "dtype": "bf16", "bias": False},
        # Sizes no tile divides, with a bias: a user's own model over a prompt.
        {"name": "linear_ragged_f32", "kind": "linear", "m": 1999, "n": 3001, "k": 1237, "dtype": "f32", "bias": True},
        # A prompt of a batch through a large feed-forward projection.
        {"name": "linear_prompt_bf16", "kind": "linear", "m": 8192, "n": 11008, "k": 4096, "dtype": "bf16",
         "bias": False},
        # One decoding step of a batch of 16 into the small model's cache.
        {"name": "store_token_f32", "kind": "store", "bits": 4, "batch": 16, "kv_heads": 4, "dim": 64, "n": 1,
         "start": 255, "dtype": "f32"},
        # The medium model's prompts, 8 sequences of 1024 tokens.
        {"name": "store_prompt_bf16", "kind": "store", "bits": 8, "batch": 8, "kv_heads": 16, "dim": 64, "n": 1024,
         "start": 0, "dtype": "bf16"},
        # Long prompts of a batch, grouped 128-wide heads.
        {"name": "store_long_bf16", "kind": "store", "bits": 4, "batch": 16, "kv_heads": 8, "dim": 128, "n": 4096,
         "start": 17, "dtype": "bf16"},
        # One token of the small model over 256 cached ones: the smallest attention.
        {"name": "attend_token_f32", "kind": "attend", "bits": 4, "batch": 1, "kv_heads": 4, "share": 1, "dim": 64,
         "n": 1, "context": 256, "dtype": "f32", "ragged": False},
        # A few proposed tokens of every sequence checked at once, ragged, with odd sizes.
        {"name": "attend_verify_f32", "kind": "attend", "bits": 8, "batch": 8, "kv_heads": 2, "share": 7, "dim": 64,
         "n": 5, "context": 777, "dtype": "f32", "ragged": True},
        # One token over a very long context: one user, latency.
        {"name": "attend_long_bf16", "kind": "attend", "bits": 4, "batch": 1, "kv_heads": 8, "share": 4, "dim": 128,
         "n": 1, "context": 131072, "dtype": "bf16", "ragged": False},
        # One decoding step of a large batch with contexts of different lengths.
        {"name": "attend_batch_bf16", "kind": "attend", "bits": 4, "batch": 64, "kv_heads": 8, "share": 8, "dim": 128,
         "n": 1, "context": 4096, "dtype": "bf16", "ragged": True},
        # A piece of a long prompt over what is cached before it.
        {"name": "attend_prompt_bf16", "kind": "attend", "bits": 4, "batch": 1, "kv_heads": 8, "share": 4, "dim": 128,
         "n": 2048, "context": 8192, "dtype": "bf16", "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Log-uniform; half of them multiples of 16 (model widths), half anything."""
    v = _log(rng, lo, hi)
    return max(16, v // 16 * 16) if rng.random() < 0.5 and v >= 16 else v


def draw(rng):
    while True:
        kind = rng.choice(["linear", "store", "attend", "attend"])
        dtype = rng.choice(["f32", "bf16"])
        if kind == "linear":
            m = _log(rng, 1, 16) if rng.random() < 0.4 else _size(rng, 1, 8192)
            c = {"kind": kind, "m": m, "n": _size(rng, 16, 16384), "k": _size(rng, 16, 11008), "dtype": dtype,
                 "bias": rng.random() < 0.4}
            if c["m"] * c["n"] * c["k"] <= 3.6e11:
                return c
            continue
        c = {"kind": kind, "bits": rng.choice([4, 8]), "batch": _log(rng, 1, 64), "kv_heads": _log(rng, 1, 16),
             "dim": rng.choice([64, 128, 128, 256]), "dtype": dtype}
        if kind == "store":
            c.update(n=1 if rng.random() < 0.3 else _log(rng, 1, 4096), start=_log(rng, 1, 4096) - 1)
            tokens = c["batch"] * c["kv_heads"] * (c["n"] + c["start"] + 16)
            if tokens * c["dim"] <= 6.7e7:
                return c
            continue
        c.update(share=rng.choice([1, 1, 2, 3, 4, 6, 7, 8, 16]), n=1 if rng.random() < 0.5 else _log(rng, 1, 2048),
                 ragged=rng.random() < 0.5)
        c["context"] = max(c["n"], _log(rng, 1, 131072))
        heads = c["batch"] * c["kv_heads"]
        if heads * c["context"] * c["dim"] <= 2.6e8 and _pairs(c) * c["dim"] * 4 <= 2.3e11 and \
                heads * c["share"] * c["n"] * c["context"] <= 5e8:
            return c


# ---------------------------------------------------------------- inputs

class _Inputs:
    """Seeded values on the GPU, the same ones in the same order for one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, shape, std=1.0, dtype="f32"):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(_TORCH[dtype])

    def integers(self, lo, hi, shape):
        return torch.randint(lo, hi + 1, shape, generator=self.g, device="cuda").to(torch.int32)

    def keys(self, shape, dtype):
        """Keys of which every 37th channel is eight times as large."""
        k = torch.randn(shape, generator=self.g, device="cuda")
        k[..., 5::37] *= 8
        return k.to(_TORCH[dtype])


def _linear_inputs(c, seed):
    r = _Inputs(seed)
    x, w = r.normal([c["m"], c["k"]], 1.0, c["dtype"]), r.normal([c["n"], c["k"]], 0.02)
    return x, w, r.normal([c["n"]], 0.02) if c["bias"] else None


def _capacity(c):
    return c["start"] + c["n"] + 15 if c["kind"] == "store" else c["context"]


def _store_inputs(c, seed):
    """(history of K, of V, new K, new V, start): the sequences stand at most 15 tokens apart."""
    r = _Inputs(seed)
    whole, new = ([c["batch"], t, c["kv_heads"], c["dim"]] for t in (_capacity(c), c["n"]))
    start = c["start"] + r.integers(0, 15, [c["batch"]])
    return (r.keys(whole, c["dtype"]), r.normal(whole, 1.0, c["dtype"]), r.keys(new, c["dtype"]),
            r.normal(new, 1.0, c["dtype"]), start)


def _attend_inputs(c, seed):
    """(K, V, q, start, count): with `ragged`, sequences of any length, one in eight with fewer queries than n."""
    r = _Inputs(seed)
    shape = [c["batch"], c["context"], c["kv_heads"], c["dim"]]
    k, v = r.keys(shape, c["dtype"]), r.normal(shape, 1.0, c["dtype"])
    q = r.normal([c["batch"], c["n"], c["kv_heads"] * c["share"], c["dim"]], 1.0, c["dtype"])
    room = c["context"] - c["n"]
    if c["ragged"]:
        fewer = r.integers(1, 3, [c["batch"]]) * (r.integers(0, 7, [c["batch"]]) == 0)
        return k, v, q, r.integers(0, room, [c["batch"]]), (c["n"] - fewer).clamp_min(0).to(torch.int32)
    whole = torch.zeros(c["batch"], dtype=torch.int32, device="cuda")
    return k, v, q, whole + room, whole + c["n"]


# ---------------------------------------------------------------- the plain forms

def _levels(bits):
    return 7 if bits == 4 else 127


def _codes(x, scale, levels):
    """rne(x / scale) as int8, decided in 64 bits (a quotient next to a half); zero where the scale is."""
    q = torch.round(x.double() / scale.double()).clamp(-levels, levels)
    return torch.where(scale > 0, q, torch.zeros_like(q)).to(torch.int8)


def _quantise(x, group, bits):
    """[.., D] -> (codes int8 [.., D], scales bf16 [.., D / group])."""
    x = x.float().unflatten(-1, (-1, group))
    most = x.abs().amax(-1, keepdim=True)
    scale = (most / _levels(bits)).to(torch.bfloat16)
    scale = torch.where(scale.float() < _TINY, torch.zeros_like(scale), scale)
    return _codes(x, scale.float(), _levels(bits)).flatten(-2), scale.squeeze(-1)


def _pack(codes, bits):
    if bits == 8:
        return codes
    u = (codes + 8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _values(packed, scales, bits):
    """The FP32 values that codes and scales stand for."""
    if bits == 4:
        packed = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).to(torch.float32) - 8
    x = packed.to(torch.float32).unflatten(-1, (scales.shape[-1], -1))
    return (x * scales.float().unsqueeze(-1)).flatten(-2)


def _plain_cache(k, v, bits):
    """Packed codes and scales of [B, T, H, D] keys and values."""
    kc, ks = _quantise(k, _GROUP, bits)
    vc, vs = _quantise(v, v.shape[-1], bits)
    return [_pack(kc, bits), ks, _pack(vc, bits), vs]


def _plain_store(s):
    new = _plain_cache(s["k"], s["v"], s["bits"])
    at = s["start"].long()[:, None] + torch.arange(s["k"].shape[1], device="cuda")
    rows = torch.arange(at.shape[0], device="cuda")[:, None]
    for whole, part in zip(s["cache"], new):
        whole[rows, at] = part
    kc, ks, vc, vs = (t[:, s["begin"]:] for t in s["cache"])
    return {"k": _values(kc, ks, s["bits"]).to(s["k"].dtype), "v": _values(vc, vs, s["bits"]).to(s["k"].dtype)}


def _plain_attend(s):
    kc, ks, vc, vs = s["cache"]
    k = _values(kc, ks, s["bits"]).transpose(1, 2)  # [B, Hkv, T, D]
    v = _values(vc, vs, s["bits"]).transpose(1, 2)
    b, n, h, d = s["q"].shape
    hkv, t = k.shape[1], k.shape[2]
    q = s["q"].float().view(b, n, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    x = torch.matmul(q, k.transpose(-1, -2)).view(b, hkv, h // hkv, n, t) / math.sqrt(d)
    i = torch.arange(n, device="cuda")
    last = torch.where(i < s["count"][:, None], s["start"][:, None] + i, -1)  # [B, n]
    seen = (torch.arange(t, device="cuda") <= last[..., None])[:, None, None]
    x = torch.where(seen, x, -math.inf)
    most = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(most == -math.inf, torch.zeros_like(most), most))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p.view(b, hkv, -1, t), v).view(b, hkv, h // hkv, n, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(s["q"].dtype)


def _quantise_rows(x):
    x = x.float()
    scale = x.abs().amax(-1, keepdim=True) / 127
    scale = torch.where(scale < _TINY, torch.zeros_like(scale), scale)
    return _codes(x, scale, 127), scale


def _plain_linear(s):
    codes, scale = _quantise_rows(s["x"])
    y = torch.matmul(codes.float(), s["w"].float().T) * scale * s["ws"].T
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------- the framework's calls

class _Shared:
    """A device tensor's memory for torch (shares the buffer and keeps it alive)."""

    def __init__(self, t):
        self.tensor = t
        self.__cuda_array_interface__ = {"shape": tuple(t.shape()), "typestr": "<i2" if t.is_bf16() else "<f4",
                                         "data": (t.ptr, False), "strides": None, "version": 2}


def _view(t):
    v = torch.as_tensor(_Shared(t), device="cuda")
    return v.view(torch.bfloat16) if t.is_bf16() else v


def _empty(shape, dtype):
    import irontensor_amd as it
    return it.Tensor.empty(list(shape), it.Precision.BF16 if dtype is torch.bfloat16 else it.Precision.FP32)


def _filled(values):
    t = _empty(values.shape, values.dtype)
    _view(t).copy_(values)
    return t


def _positions(values):
    import irontensor_amd as it
    return it.upload_positions(values.cpu().numpy())


def _own_cache(k, v, bits):
    """A KvCache that holds [B, T, H, D] keys and values from position 0 on."""
    import irontensor_amd as it
    b, t, h, d = k.shape
    cache = it.KvCache(b, h, t, d, bits)
    k, v = _filled(k), _filled(v)
    torch.cuda.synchronize()
    it.kv_cache_write(cache, k, v, it.upload_positions([0] * b))
    return cache


def _own_prepare(c, seed):
    import irontensor_amd as it
    if c["kind"] == "linear":
        x, w, bias = _linear_inputs(c, seed)
        w = _filled(w)
        torch.cuda.synchronize()
        s = {"x": _filled(x), "w": it.quantize_i8(w), "bias": None if bias is None else _filled(bias)}
        s["out"] = _empty([c["m"], c["n"]], x.dtype)
        s["result"] = _view(s["out"])
    elif c["kind"] == "store":
        hk, hv, k, v, start = _store_inputs(c, seed)
        s = {"cache": _own_cache(hk, hv, c["bits"]), "k": _filled(k), "v": _filled(v), "start": _positions(start),
             "begin": c["start"], "read": c["n"] + 15}
        s["out"] = [_empty([c["batch"], s["read"], c["kv_heads"], c["dim"]], k.dtype) for _ in range(2)]
        s["result"] = dict(zip("kv", map(_view, s["out"])))
    else:
        k, v, q, start, count = _attend_inputs(c, seed)
        s = {"cache": _own_cache(k, v, c["bits"]), "q": _filled(q), "start": _positions(start),
             "count": _positions(count), "out": _empty(q.shape, q.dtype)}
        s["result"] = _view(s["out"])
    it.Context.global_().sync()
    return s


def _own_run(s):
    import irontensor_amd as it
    if s["kind"] == "linear":
        it.linear_i8(s["x"], s["w"], s["bias"], out=s["out"])
    elif s["kind"] == "store":
        it.kv_cache_write(s["cache"], s["k"], s["v"], s["start"])
        it.kv_cache_read(s["cache"], s["begin"], s["read"], out=s["out"])
    else:
        it.cached_attention(s["q"], s["cache"], s["start"], s["count"], out=s["out"])
    return s["result"]


# ---------------------------------------------------------------- prepare and run

def prepare(case, seed):
    c = case
    torch.cuda.synchronize()  # torch fills memory that the library's stream may have used before
    if own:
        s = _own_prepare(c, seed)
    elif c["kind"] == "linear":
        x, w, bias = _linear_inputs(c, seed)
        codes, scale = _quantise_rows(w)
        s = {"x": x, "w": codes, "ws": scale, "bias": bias}
    elif c["kind"] == "store":
        hk, hv, k, v, start = _store_inputs(c, seed)
        s = {"cache": _plain_cache(hk, hv, c["bits"]), "k": k, "v": v, "start": start, "begin": c["start"]}
    else:
        k, v, q, start, count = _attend_inputs(c, seed)
        s = {"cache": _plain_cache(k, v, c["bits"]), "q": q, "start": start, "count": count}
    s.update(kind=c["kind"], bits=c.get("bits"))
    torch.cuda.synchronize()
    return s


def run(state):
    if own:
        return _own_run(state)
    return {"linear": _plain_linear, "store": _plain_store, "attend": _plain_attend}[state["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def _pairs(c):
    """Query-key pairs of an attention call (ragged: the mean length)."""
    n, room = c["n"], c["context"] - c["n"]
    before = room / 2 if c["ragged"] else room
    return c["batch"] * c["kv_heads"] * c["share"] * (n * before + n * (n + 1) / 2)


def _token_bytes(c):
    """A cached token of one head: the codes of its key and value, and their scales."""
    return c["dim"] * c["bits"] / 4 + 2 * (c["dim"] / _GROUP + 1)


def work(case):
    c = case
    e = 2 if c["dtype"] == "bf16" else 4
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": float(e * m * (k + n) + n * (k + 4) + (4 * n if c["bias"] else 0)), "flops": 2.0 * m * n * k}
    rows = c["batch"] * c["kv_heads"]
    if c["kind"] == "store":
        new, read = rows * c["n"], rows * (c["n"] + 15)
        return {"bytes": float((new + read) * (2 * c["dim"] * e + _token_bytes(c))), "flops": 0.0}
    live = c["n"] + (c["context"] - c["n"]) / (2 if c["ragged"] else 1)
    q = rows * c["share"] * c["n"] * c["dim"]
    return {"bytes": float(rows * live * _token_bytes(c) + 2 * q * e), "flops": float(4 * _pairs(c) * c["dim"])}


# ---------------------------------------------------------------- the same in 64 bits

def _stands_for(x, channels, most, scale_type):
    """What a value reads back as: its group's step times the nearest whole number of steps, in float64."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // channels, channels)
    step = (g.abs().max(-1, keepdim=True).values / most).float().to(scale_type).double()
    step[step < _TINY] = 0
    whole = torch.where(step > 0, g / step, torch.zeros_like(g)).round_()
    return (whole.clamp_(-most, most) * step).reshape(x.shape)


def exact(case, seed):
    c = case
    if c["kind"] == "linear":
        x, w, bias = _linear_inputs(c, seed)
        y = _stands_for(x, c["k"], 127, torch.float32) @ _stands_for(w, c["k"], 127, torch.float32).T
        return y if bias is None else y + bias.double()
    most = 2 ** (c["bits"] - 1) - 1
    kept = lambda k, v: (_stands_for(k, _GROUP, most, torch.bfloat16),  # noqa: E731
                         _stands_for(v, c["dim"], most, torch.bfloat16))
    if c["kind"] == "store":
        hk, hv, k, v, start = _store_inputs(c, seed)
        for b, at in enumerate(start.tolist()):
            hk[b, at:at + c["n"]], hv[b, at:at + c["n"]] = k[b], v[b]
        return dict(zip("kv", kept(hk[:, c["start"]:], hv[:, c["start"]:])))
    k, v, q, start, count = _attend_inputs(c, seed)
    k, v = kept(k, v)
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    j = torch.arange(c["context"], device="cuda")
    for b in range(c["batch"]):
        m, at = int(count[b]), int(start[b])
        if m == 0:
            continue
        hidden = j[None, :] > at + torch.arange(m, device="cuda")[:, None]
        for g in range(c["kv_heads"]):
            own_heads = slice(g * c["share"], (g + 1) * c["share"])
            x = torch.tensordot(q[b, :m, own_heads].double(), k[b, :, g], ([-1], [-1])) * c["dim"] ** -0.5
            p = torch.softmax(x.masked_fill_(hidden[:, None], -math.inf), -1)
            o[b, :m, own_heads] = torch.tensordot(p, v[b, :, g], ([-1], [0]))
    return o

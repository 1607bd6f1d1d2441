"""Attention beside the block-sparse core, as cases that can be timed and checked.

* ``cross``  cross attention: queries over the keys of another sequence (an encoder's states), each batch entry
  with its own number of valid keys. ``train`` is forward + backward, ``infer`` the forward over many queries,
  ``token`` one to four queries per sequence, as a decoder's step makes them.
* ``step``   a serving step of the rolling cache held in 8 bits: the new keys and values are quantised as they are
  written, then the queries attend.
* ``store``  a prompt written into such a cache, and what the cache holds read back.
* ``prefix`` a decode step of a batch whose sequences share a long prefix, kept once for all of them, in front of
  each sequence's own rolling cache (16 or 8 bits).

``listed()`` gives the fixed cases, ``draw(rng)`` another one of the same ranges. A row of the 8-bit cache is D
e4m3 codes and one power of two: 2^e with the smallest e for which the row's largest magnitude is at most 448 * 2^e.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_F8 = torch.float8_e4m3fn
_MIN_EXPONENT = -117
_MAX_QUERY = 4


def _cross(name, mode, dtype, batch, heads, kv_heads, n_q, n_kv, head_dim, ragged=True):
    case = dict(kind="cross", mode=mode, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, n_q=n_q,
                n_kv=n_kv, head_dim=head_dim, ragged=ragged)
    return dict(case, name=name) if name else case


def _cache(name, kind, dtype, batch, heads, kv_heads, n_q, past, head_dim, sink, window, prefix=0, bits=8):
    case = dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, n_q=n_q, past=past,
                head_dim=head_dim, sink=sink, window=window, prefix=prefix, bits=bits)
    return dict(case, name=name) if name else case


def listed():
    return [
        # a training batch of target sequences over encoded sources, narrow heads
        _cross("cross_train_bf16_b8h16_q448_kv1500_d64", "train", "bf16", 8, 16, 16, 448, 1500, 64),
        # a small full-precision model with odd lengths
        _cross("cross_train_fp32_b2h4_q333_kv777_d64", "train", "fp32", 2, 4, 4, 333, 777, 64),
        # training over long sources with grouped-query heads, the widest head
        _cross("cross_train_bf16_b4h16kv4_q2048_kv4096_d128", "train", "bf16", 4, 16, 4, 2048, 4096, 128),
        # a long document encoded once, read by many positions; every key valid
        _cross("cross_infer_fp16_b2h32kv8_q4096_kv8192_d128", "infer", "fp16", 2, 32, 8, 4096, 8192, 128, False),
        # a decoder's step over a batch of encoded sources
        _cross("cross_token_fp16_b16h16_q1_kv2000_d64", "token", "fp16", 16, 16, 16, 1, 2000, 64),
        # the smallest cache call: one sequence's step, where latency counts
        _cache("step_fp16_b1h8_w2048_d64", "step", "fp16", 1, 8, 8, 1, 2100, 64, 4, 2048),
        # a batched serving step of grouped-query sequences
        _cache("step_bf16_b8h32kv8_w2048_d128", "step", "bf16", 8, 32, 8, 1, 2100, 128, 4, 2048),
        # a large batch with a long window, every head its own keys
        _cache("step_bf16_b16h32_w8192_d128", "step", "bf16", 16, 32, 32, 1, 8300, 128, 4, 8192),
        # a long prompt written into a cache that keeps its end, and read back
        _cache("store_bf16_b4h8_n10000_w4096_d128", "store", "bf16", 4, 8, 8, 10000, 0, 128, 4, 4096),
        # short continuations of one system prompt, grouped-query heads
        _cache("prefix_bf16_b32h32kv8_p8192_own300_d128", "prefix", "bf16", 32, 32, 8, 1, 300, 128, 4, 2048,
               prefix=8192, bits=16),
        # two positions per sequence behind a prefix of odd length, every head its own keys
        _cache("prefix_fp16_b8h12_q2_p1777_d64", "prefix", "fp16", 8, 12, 12, 2, 700, 64, 4, 512,
               prefix=1777, bits=16),
        # a large batch behind a long document, its own part in 8 bits
        _cache("prefix_bf16_b64h32kv8_p32768_w2048_d128", "prefix", "bf16", 64, 32, 8, 1, 2100, 128, 4, 2048,
               prefix=32768, bits=8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["train", "train", "infer", "token", "step", "step", "store", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = min(32, kv * rng.choice([1, 1, 2, 4, 8]))
    heads -= heads % kv
    batch = rng.choice([1, 2, 4, 8, 16])
    if kind == "train":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        n_q, n_kv = _log_int(rng, 5, 2048), _log_int(rng, 60, 4096)
        batch = max(1, min(batch, (1 << (28 if dtype != "fp32" else 26)) // (heads * n_q * n_kv)))
        return _cross(None, kind, dtype, batch, heads, kv, n_q, n_kv, rng.choice([16, 32, 64, 64, 128]))
    if kind == "infer":
        n_q, n_kv = _log_int(rng, 40, 4096), _log_int(rng, 60, 8192)
        batch = max(1, min(batch, (1 << 28) // (heads * n_q * n_kv)))
        return _cross(None, kind, dtype, batch, heads, kv, n_q, n_kv, rng.choice([32, 64, 128]),
                      rng.random() < 0.7)
    if kind == "token":
        return _cross(None, kind, dtype, batch, heads, kv, rng.choice([1, 1, 1, 2, 4]), _log_int(rng, 60, 8192), d)
    sink = rng.choice([0, 1, 4, 4, 16])
    window = _log_int(rng, 128, 8192)
    n_q = rng.choice([1, 1, 1, 2, 4])
    if kind == "step":
        return _cache(None, kind, rng.choice(["bf16", "fp16"]), batch, heads, kv, n_q,
                      window + sink + rng.randint(8, 99), d, sink, window)
    if kind == "store":
        return _cache(None, kind, rng.choice(["bf16", "fp16", "fp32"]), min(batch, 4), kv, kv,
                      _log_int(rng, 30, 20000), 0, d, sink, window)
    batch = rng.choice([2, 4, 8, 16, 32])
    return _cache(None, kind, dtype, batch, heads, kv, n_q, _log_int(rng, 4, 3000), d, sink, min(window, 2048),
                  prefix=_log_int(rng, 100, 20000), bits=rng.choice([16, 8]))


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    dt, b, h, hkv, d = (_DTYPES[case["dtype"]], case["batch"], case["heads"], case["kv_heads"], case["head_dim"])
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(heads, n, batch=b):
        return torch.randn((batch, heads, n, d), generator=gen, device="cuda", dtype=dt)

    if case["kind"] == "cross":
        x = {"q": normal(h, case["n_q"]), "k": normal(hkv, case["n_kv"]), "v": normal(hkv, case["n_kv"])}
        n = case["n_kv"]
        lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
        if case["ragged"]:       # a padded batch: one entry fills it, the others end somewhere in its last three quarters
            lengths = torch.randint(max(1, n // 4), n + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
            lengths[0] = n
        x["lengths"] = lengths
        if case["mode"] == "train":
            x["do"] = normal(h, case["n_q"])
        return x
    # keys carry a few strong channels, as rotary and outlier channels make them
    gain = torch.ones(d, device="cuda", dtype=dt)
    gain[:: max(1, d // 4)] = 4.0
    x = {"k": normal(hkv, case["n_q"]) * gain, "v": normal(hkv, case["n_q"])}
    if case["kind"] != "store":
        x["q"] = normal(h, case["n_q"]) * 0.5
    if case["past"]:
        x["past_k"], x["past_v"] = normal(hkv, case["past"]) * gain, normal(hkv, case["past"])
    if case["prefix"]:
        x["prefix_k"], x["prefix_v"] = normal(hkv, case["prefix"], 1) * gain, normal(hkv, case["prefix"], 1)
    return x


# ---- plain forms ---------------------------------------------------------------------------------------------------


def _quantise(x):
    """Rows as e4m3 codes and their exponents (biased by 127, as a byte)."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp_(min=_MIN_EXPONENT)
    inverse = ((127 - e) << 23).view(torch.float32)
    return (x * inverse[..., None]).to(_F8), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(codes, scale):
    return codes.float() * scale.float()[..., None]


class _PlainCache:
    """Sink slots, then a ring: position p < sink in slot p, any other in slot sink + (p - sink) % ring."""

    def __init__(self, case):
        self.sink, self.window = case["sink"], case["window"]
        self.ring = max(1, self.window + _MAX_QUERY - 1)
        self.bits, self.dtype = case["bits"], _DTYPES[case["dtype"]]
        shape = (case["batch"], case["kv_heads"], self.sink + self.ring, case["head_dim"])
        held = _F8 if self.bits == 8 else self.dtype
        self.k, self.v = (torch.zeros(shape, dtype=held, device="cuda") for _ in range(2))
        if self.bits == 8:
            self.k_scale, self.v_scale = (
                torch.zeros(shape[:3], dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
        self.length = 0

    def held(self):
        """Positions in the cache, ascending, and their slots."""
        a = torch.arange(min(self.length, self.sink), device="cuda")
        b = torch.arange(max(self.sink, self.length - self.ring), max(self.sink, self.length), device="cuda")
        return torch.cat([a, b]), torch.cat([a, self.sink + (b - self.sink) % self.ring])

    def append(self, k, v):
        start, self.length = self.length, self.length + k.shape[2]
        positions, slots = self.held()
        first = min(start, self.sink) + max(0, start - max(self.sink, self.length - self.ring))
        positions, slots = positions[first:], slots[first:]
        k, v = k[:, :, positions - start], v[:, :, positions - start]
        if self.bits == 8:
            self.k[:, :, slots], self.k_scale[:, :, slots] = _quantise(k)
            self.v[:, :, slots], self.v_scale[:, :, slots] = _quantise(v)
        else:
            self.k[:, :, slots], self.v[:, :, slots] = k, v

    def rows(self, slots):
        if self.bits == 8:
            return (_values(self.k[:, :, slots], self.k_scale[:, :, slots]),
                    _values(self.v[:, :, slots], self.v_scale[:, :, slots]))
        return self.k[:, :, slots].float(), self.v[:, :, slots].float()

    def attend(self, q, prefix_k=None, prefix_v=None):
        b, h, n_q, d = q.shape
        hkv = self.k.shape[1]
        group = h // hkv
        positions, slots = self.held()
        at = torch.arange(self.length - n_q, self.length, device="cuda")[:, None]
        seen = (positions <= at) & ((positions < self.sink) | (positions > at - self.window))
        k, v = self.rows(slots)
        qf = q.float().reshape(b, hkv, group * n_q, d)
        s = torch.matmul(qf, k.transpose(2, 3)) / math.sqrt(d)
        s = s.masked_fill(~seen.repeat(group, 1), -math.inf)
        if prefix_k is not None:
            rows = qf.transpose(0, 1).reshape(hkv, b * group * n_q, d)
            sp = torch.matmul(rows, prefix_k[0].float().transpose(1, 2)) / math.sqrt(d)
            s = torch.cat([sp.reshape(hkv, b, group * n_q, -1).transpose(0, 1), s], -1)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        n_p = 0 if prefix_k is None else prefix_k.shape[2]
        o = torch.matmul(p[..., n_p:], v)
        if prefix_k is not None:
            pp = p[..., :n_p].transpose(0, 1).reshape(hkv, b * group * n_q, n_p)
            o = o + torch.matmul(pp, prefix_v[0].float()).reshape(hkv, b, group * n_q, d).transpose(0, 1)
        return o.reshape(b, h, n_q, d).to(q.dtype)


def _plain_cross(x, train):
    q, k, v = (x[n].detach().float() for n in ("q", "k", "v"))
    b, h, n_q, d = q.shape
    hkv, n_kv = k.shape[1:3]
    q = q.reshape(b, hkv, -1, d)
    gone = (torch.arange(n_kv, device="cuda") >= x["lengths"][:, None])[:, None, None]
    s = (torch.matmul(q, k.transpose(2, 3)) / math.sqrt(d)).masked_fill_(gone, -math.inf)
    p = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
    p = p.div_(p.sum(-1, keepdim=True))
    dt = x["q"].dtype
    out = {"o": torch.matmul(p, v).reshape(b, h, n_q, d).to(dt)}
    if train:
        do = x["do"].float().reshape(b, hkv, -1, d)
        ds = torch.matmul(do, v.transpose(2, 3))
        ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).div_(math.sqrt(d))
        out["dq"] = torch.matmul(ds, k).reshape(b, h, n_q, d).to(dt)
        out["dk"] = torch.matmul(ds.transpose(2, 3), q).to(dt)
        out["dv"] = torch.matmul(p.transpose(2, 3), do).to(dt)
    return out


# ---- the calls -----------------------------------------------------------------------------------------------------


def _gki():
    root = str(Path(__file__).resolve().parents[1] / "graph-kernel-injection_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gki

    return gki


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case}
    if case["kind"] == "cross":
        if case["mode"] == "train":
            for name in ("q", "k", "v"):
                x[name].requires_grad_(True)
        return dict(state, **x)
    if own:
        gki = _gki()
        cache = gki.StreamingKVCache(
            case["batch"], case["kv_heads"], case["head_dim"], gki.StreamingMaskSpec(case["sink"], case["window"]),
            dtype=_DTYPES[case["dtype"]], device="cuda", max_query=_MAX_QUERY,
            storage_dtype=_F8 if case["bits"] == 8 else None)
        if case["prefix"]:
            cache.set_prefix(x["prefix_k"], x["prefix_v"])
    else:
        cache = _PlainCache(case)
    if case["past"]:
        cache.append(x.pop("past_k"), x.pop("past_v"))
    return dict(state, cache=cache, **x)


def run(state):
    case = state["case"]
    k, v = state["k"], state["v"]
    if case["kind"] == "cross":
        train = case["mode"] == "train"
        if not own:
            return _plain_cross(state, train)
        q = state["q"]
        out = _gki().cross_attention(q, k, v, state["lengths"] if case["ragged"] else None,
                                     enable_gqa=case["heads"] != case["kv_heads"])
        if not train:
            return {"o": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["do"])
        return {"o": out, "dq": dq, "dk": dk, "dv": dv}
    cache = state["cache"]
    if case["kind"] == "store":
        if own:
            cache.reset()
            cache.append(k, v)
            positions, kr, vr = cache.read()
        else:
            cache.length = 0
            cache.append(k, v)
            positions, slots = cache.held()
            kr, vr = (t.to(cache.dtype) for t in cache.rows(slots))
        return {"positions": positions, "k": kr, "v": vr}
    if own:
        o = cache.step(state["q"], k, v)
        got = {"o": o, "k": cache.k_cache, "v": cache.v_cache}
        return dict(got, k_scale=cache.k_scale, v_scale=cache.v_scale) if case["bits"] == 8 else got
    cache.append(k, v)
    o = cache.attend(state["q"], state.get("prefix_k"), state.get("prefix_v"))
    got = {"o": o, "k": cache.k, "v": cache.v}
    return dict(got, k_scale=cache.k_scale, v_scale=cache.v_scale) if case["bits"] == 8 else got


def work(case):
    el = _DTYPES[case["dtype"]].itemsize
    b, h, hkv, n_q, d = case["batch"], case["heads"], case["kv_heads"], case["n_q"], case["head_dim"]
    q_bytes = b * h * n_q * d * el
    if case["kind"] == "cross":
        # a ragged entry holds five eighths of the keys on average, the first all of them
        keys = case["n_kv"] * (1 + 0.625 * (b - 1) if case["ragged"] else b)
        kv_bytes = hkv * keys * d * el
        if case["mode"] == "train":      # in: q, k, v, do; out: o, dq and the whole dk, dv
            return {"bytes": 4 * q_bytes + 2 * kv_bytes + 2 * b * hkv * case["n_kv"] * d * el,
                    "flops": 14 * h * n_q * keys * d}
        return {"bytes": 2 * q_bytes + 2 * kv_bytes, "flops": 4 * h * n_q * keys * d}
    row = d + 1 if case["bits"] == 8 else d * el     # what the cache keeps of a key or a value
    if case["kind"] == "store":
        held = min(n_q, case["sink"] + max(1, case["window"] + _MAX_QUERY - 1))
        return {"bytes": 2 * b * hkv * held * (2 * d * el + 2 * row), "flops": 8 * b * hkv * held * d}
    length = case["past"] + n_q
    keys = min(length, case["sink"] + case["window"] + n_q - 1)
    pairs = n_q * min(length, case["sink"] + case["window"])
    return {"bytes": 2 * q_bytes + 2 * b * hkv * (keys * row + n_q * (d * el + row)) + 2 * hkv * case["prefix"] * d * el,
            "flops": 4 * b * h * d * (pairs + n_q * case["prefix"])}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------


def _e4m3_rows(x):
    """(codes, 2^e) of rows, rounded by arithmetic: steps of 2^(exponent - 3), 2^-9 below the normal numbers."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448.0)).clamp(min=_MIN_EXPONENT)
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where((top <= 448.0 * torch.exp2(e - 1)) & (e > _MIN_EXPONENT), e - 1, e)
    unit = torch.exp2(e)
    y = x / unit
    place = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    place = torch.where(y.abs() >= torch.exp2(place + 1), place + 1, place)
    place = torch.where((y.abs() < torch.exp2(place)) & (place > -6), place - 1, place)
    step = torch.exp2(place - 3)
    return torch.round(y / step) * step, unit[..., 0]


def _softmax64(s):
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _exact_cross(case, x):
    b, h, hkv, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    group = h // hkv
    names = ("q", "k", "v", "do") if case["mode"] == "train" else ("q", "k", "v")
    q, k, v, *do = (x[n].double() for n in names)
    out = {"o": torch.zeros_like(q)}
    if do:
        out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    for i, n in enumerate(x["lengths"].tolist()):
        for j in range(hkv):
            heads = slice(j * group, (j + 1) * group)
            kk, vv, qq = k[i, j, :n], v[i, j, :n], q[i, heads].reshape(-1, d)
            p = _softmax64((qq @ kk.T) * d ** -0.5)
            out["o"][i, heads] = (p @ vv).view(group, -1, d)
            if do:
                g = do[0][i, heads].reshape(-1, d)
                dp = g @ vv.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * d ** -0.5
                out["dq"][i, heads] = (ds @ kk).view(group, -1, d)
                out["dk"][i, j, :n] = ds.T @ qq
                out["dv"][i, j, :n] = p.T @ g
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "cross":
        return _exact_cross(case, x)
    b, h, hkv, n_q, d = case["batch"], case["heads"], case["kv_heads"], case["n_q"], case["head_dim"]
    sink, window = case["sink"], case["window"]
    ring = max(1, window + _MAX_QUERY - 1)
    k, v = ((torch.cat([x["past_" + n], x[n]], 2) if case["past"] else x[n]) for n in ("k", "v"))
    length = k.shape[2]
    first = max(sink, length - ring)       # older ones behind the sinks have left the cache
    kept = [p for p in range(length) if p < sink or p >= first]
    at = torch.tensor(kept, device="cuda")
    slots = torch.tensor([p if p < sink else sink + (p - sink) % ring for p in kept], device="cuda")
    state, rows = {}, {}
    for name, t in (("k", k[:, :, at]), ("v", v[:, :, at])):
        if case["bits"] == 8:
            codes, unit = _e4m3_rows(t)
            rows[name] = codes * unit[..., None]
            scale = torch.full((b, hkv, sink + ring), 2.0 ** -127, dtype=torch.float64, device="cuda")
            scale[:, :, slots] = unit
            state[name + "_scale"] = scale
        else:
            codes = rows[name] = t.double()
        state[name] = torch.zeros((b, hkv, sink + ring, d), dtype=torch.float64, device="cuda")
        state[name][:, :, slots] = codes
    if case["kind"] == "store":
        return {"positions": at, "k": rows["k"], "v": rows["v"]}
    o = torch.empty((b, h, n_q, d), dtype=torch.float64, device="cuda")
    for i in range(n_q):
        pos = length - n_q + i
        seen = [n for n, p in enumerate(kept) if p <= pos and (p < sink or p > pos - window)]
        seen = torch.tensor(seen, device="cuda")
        for head in range(h):
            j = head // (h // hkv)
            kk, vv = rows["k"][:, j, seen], rows["v"][:, j, seen]
            q = x["q"][:, head, i].double() * d ** -0.5
            s = (kk * q[:, None]).sum(-1)
            if case["prefix"]:
                s = torch.cat([s, q @ x["prefix_k"][0, j].double().T], 1)
            p = _softmax64(s)
            got = (p[:, : len(seen), None] * vv).sum(1)
            if case["prefix"]:
                got = got + p[:, len(seen):] @ x["prefix_v"][0, j].double()
            o[:, head, i] = got
    return dict(state, o=o)

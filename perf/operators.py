"""Performance cases of the long-context operators: the 4-bit KV cache with the attention that reads it, its eviction by attention
weight, and the 8-bit integer product with a scale for each token and each output channel.

Where `own` is false, run() computes an operator from elementary torch operations in 32 bits; where it is true, it makes the
library's calls on the same state. The sizes are those of the models that this repository's tests and benchmark use (Mistral-7B
and TinyLlama shapes: 32 heads over 8 of 128, 32 over 4 of 64) and generic ones beside them.
"""
import math

import torch

own = False

GROUP = 32                                        # values that share a scale in the 4-bit cache
_shared = {}


# ── cases ──────────────────────────────────────────────────────────────────────────────────────────────────────────
def _decode(heads, kv, hd, rows, B, weights=False):
    return {"kind": "decode", "heads": heads, "kv": kv, "hd": hd, "rows": rows, "B": B, "weights": weights}


def _attention(heads, kv, hd, rows, B, weights):
    return {"kind": "attention", "heads": heads, "kv": kv, "hd": hd, "rows": rows, "B": B, "weights": weights}


def _append(kv, hd, rows, B, theta):
    return {"kind": "append", "kv": kv, "hd": hd, "rows": rows, "B": B, "theta": theta}


def _evict(kv, hd, rows, keep, sink, recent):
    return {"kind": "evict", "kv": kv, "hd": hd, "rows": rows, "keep": keep, "sink": sink, "recent": recent}


def _w8a8(M, n, N, B):
    return {"kind": "w8a8", "M": M, "tensors": n, "N": N, "B": B}


def listed():
    return [
        # the next token of a 7B model after 512 positions: key rotation, the cache row, attention
        {"name": "decode after 512", **_decode(32, 8, 128, 512, 1)},
        # the same at the end of a long context, where the cache is most of what a step reads
        {"name": "decode after 32767", **_decode(32, 8, 128, 32767, 1)},
        # six drafted tokens checked at once by a TinyLlama-shaped model whose cache is kept to a budget: weights are tracked
        {"name": "draft of 6 with weights", **_decode(32, 4, 64, 3001, 6, True)},
        # a prompt of 2048 tokens attending to itself, with the weights that the eviction after it goes by
        {"name": "prompt 2048 with weights", **_attention(32, 8, 128, 0, 2048, True)},
        # a few tokens, and the keys and values of a prompt, into the cache, and back as the values that it holds
        {"name": "append 7", **_append(4, 64, 3001, 7, 10000.0)},
        {"name": "append 2048", **_append(8, 128, 37, 2048, 1000000.0)},
        # a cache of one layer cut to a quarter, and a long one to a budget of 8192 rows
        {"name": "evict 4096 to 1024", **_evict(8, 128, 4096, 1024, 4, 256)},
        {"name": "evict 65529 to 8192", **_evict(8, 128, 65529, 8192, 4, 1000)},
        # one token through a projection; an odd small product; the gate and up projections of a prompt; the down projection of a ragged one
        {"name": "w8a8 one token", **_w8a8(4096, 1, 4096, 1)},
        {"name": "w8a8 odd 37 tokens", **_w8a8(1003, 1, 2056, 37)},
        {"name": "w8a8 gate up 2048", **_w8a8(14336, 2, 4096, 2048)},
        {"name": "w8a8 down 511", **_w8a8(4096, 1, 14336, 511)},
    ]


def _between(rng, lo, hi, step=1):
    """a multiple of step, spread over the logarithm of [lo, hi]"""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


_LAYOUTS = [(32, 8, 128), (32, 4, 64), (32, 32, 128), (8, 1, 256), (16, 2, 96), (12, 12, 64), (10, 2, 192), (6, 3, 32), (16, 16, 64)]


def draw(rng):
    kind = rng.choice(["decode", "decode", "attention", "append", "evict", "w8a8", "w8a8"])
    heads, kv, hd = rng.choice(_LAYOUTS)
    if kind == "decode":
        return _decode(heads, kv, hd, _between(rng, 1, 32768 * 8 // max(8, kv)), rng.choice([1, 1, _between(rng, 2, 12)]), rng.random() < 0.3)
    if kind == "attention":
        B = _between(rng, 13, 2048)
        return _attention(heads, kv, hd, rng.choice([0, _between(rng, 1, 1024)]) if B < 1024 else 0, B if heads * hd <= 4096 else B // 2, rng.random() < 0.5)
    if kind == "append":
        return _append(kv, hd, _between(rng, 1, 4096) - 1, _between(rng, 1, 2048), rng.choice([10000.0, 500000.0, 0.0]))
    if kind == "evict":
        rows = _between(rng, 16, 65536 * 8 // max(8, kv))
        keep = min(rows, _between(rng, 8, max(8, rows // 2)))
        recent = rng.randint(0, keep // 2)
        return _evict(kv, hd, rows, keep, min(4, keep - recent), recent)
    return _w8a8(_between(rng, 200, 14336), rng.choice([1, 1, 2, 3]), _between(rng, 256, 14336, rng.choice([1, 8, 64, 64])), _between(rng, 1, 1024))


# ── inputs ─────────────────────────────────────────────────────────────────────────────────────────────────────────
class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _keys(g, B, kv, hd):
    """keys as models have them: a few channels of each head several times larger than the others"""
    loud = torch.ones(kv, hd, device="cuda")
    loud[:, :: max(8, hd // 4)] = 3.0
    return (_normal(g, B, kv, hd) * loud).reshape(B, kv * hd)


def _quantise(x):
    """codes 1..15 and fp16 scales of groups of 32: [..., hd] -> [..., hd], [..., hd / 32]"""
    y = x.reshape(*x.shape[:-1], -1, GROUP)
    s = (y.abs().amax(-1) / 7).to(torch.float16)
    inv = torch.where(s > 0, 1 / s.float(), torch.zeros((), device=x.device))
    c = (y * inv[..., None]).round().clamp(-7, 7) + 8
    return c.reshape(x.shape).to(torch.uint8), s


def _bytes(c):
    c = c.reshape(*c.shape[:-1], -1, 2)
    return c[..., 0] | (c[..., 1] << 4)


def _pack_k(c):
    """order of a key row: piece t of four holds values 8t..8t+7 of every group of 32"""
    s = c.shape
    return _bytes(c.reshape(*s[:-1], -1, 4, 8).transpose(-3, -2).reshape(s))


def _pack_v(c):
    """order of a value row: piece g of eight holds values 4g..4g+3 of every group of 32"""
    s = c.shape
    return _bytes(c.reshape(*s[:-1], -1, 8, 4).transpose(-3, -2).reshape(s))


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


def _unpack(b, pieces, s):
    """values [..., hd] of packed rows and their scales"""
    c = _nibbles(b)
    ng = s.shape[-1]
    c = c.reshape(*c.shape[:-1], pieces, ng, GROUP // pieces).transpose(-3, -2).reshape(*c.shape[:-1], ng, GROUP)
    return ((c.float() - 8) * s.float()[..., None]).reshape(*b.shape[:-1], ng * GROUP)


def _cache(g, kv, hd, rows, max_rows):
    """a cache of `rows` rows as the library holds it: planes per KV head"""
    ng = hd // GROUP
    k = torch.zeros(kv, max_rows, hd // 2, device="cuda", dtype=torch.uint8)
    v = torch.zeros_like(k)
    scale = torch.zeros(kv, max_rows, 2 * ng, device="cuda", dtype=torch.float16)
    if rows:
        kc, ks = _quantise(_keys(g, rows, kv, hd).reshape(rows, kv, hd).transpose(0, 1))
        vc, vs = _quantise(_normal(g, kv, rows, hd))
        k[:, :rows], v[:, :rows] = _pack_k(kc), _pack_v(vc)
        scale[:, :rows, :ng], scale[:, :rows, ng:] = ks, vs
    return k, v, scale


def _weights(g, kv, rows):
    """accumulated attention as it looks: a few rows draw most of it, many little; coarse values, so that equal ones occur"""
    return torch.exp(2 * _normal(g, kv, rows)).to(torch.bfloat16).float()


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = _State(case=dict(case), kind=kind, calls=None)
    if kind in ("decode", "attention"):
        heads, kv, hd, rows, B = (case[n] for n in ("heads", "kv", "hd", "rows", "B"))
        s.max_rows = (rows + B + 7) // 8 * 8
        s.k, s.v, s.scale = _cache(g, kv, hd, rows + (B if kind == "attention" else 0), s.max_rows)
        s.weight = torch.zeros(kv, s.max_rows, device="cuda")
        s.q, s.out = _normal(g, B, heads * hd), torch.zeros(B, heads * hd, device="cuda")
        if kind == "decode":
            s.k_new, s.v_new = _keys(g, B, kv, hd), _normal(g, B, kv * hd)
    elif kind == "append":
        kv, hd, rows, B = (case[n] for n in ("kv", "hd", "rows", "B"))
        s.max_rows = (rows + B + 7) // 8 * 8
        s.k, s.v, s.scale = _cache(g, kv, hd, 0, s.max_rows)
        s.k_new, s.v_new = _keys(g, B, kv, hd), _normal(g, B, kv * hd)
        s.k_out, s.v_out = torch.zeros(B, kv * hd, device="cuda"), torch.zeros(B, kv * hd, device="cuda")
    elif kind == "evict":
        kv, hd, rows, keep = (case[n] for n in ("kv", "hd", "rows", "keep"))
        s.max_rows, s.dst_rows = (rows + 7) // 8 * 8, (keep + 7) // 8 * 8
        s.k, s.v, s.scale = _cache(g, kv, hd, 0, s.max_rows)
        s.k.random_(0, 256, generator=g)
        s.v.random_(0, 256, generator=g)
        s.scale.uniform_(0.01, 0.5, generator=g)
        s.weight = torch.zeros(kv, s.max_rows, device="cuda")
        s.weight[:, :rows] = _weights(g, kv, rows)
        s.dk, s.dv = (torch.zeros(kv, s.dst_rows, hd // 2, device="cuda", dtype=torch.uint8) for _ in range(2))
        s.dscale = torch.zeros(kv, s.dst_rows, s.scale.shape[2], device="cuda", dtype=torch.float16)
        s.dweight = torch.zeros(kv, s.dst_rows, device="cuda")
        s.kept = torch.zeros(kv, keep, device="cuda", dtype=torch.int32)
    else:
        M, n, N, B = (case[x] for x in ("M", "tensors", "N", "B"))
        s.w = torch.randint(-127, 128, (n, M, N), generator=g, device="cuda", dtype=torch.int8)
        s.sw = (torch.rand(n, M, generator=g, device="cuda") * 0.009 + 0.001).to(torch.float16)
        s.x = _normal(g, B, N) * torch.exp(_normal(g, B, 1))
        s.out = torch.zeros(n, B, M, device="cuda")
    torch.cuda.synchronize()                      # the library's stream does not wait for torch's
    return s


# ── the library's calls ────────────────────────────────────────────────────────────────────────────────────────────
def _calls(s):
    import ctypes as C
    from libinferbit_b200 import Backend, LinearT
    from libinferbit_b200._ffi import Kv4T
    if "be" not in _shared:
        _shared["be"] = Backend(0)
    be, c = _shared["be"], s.case
    lib, ctx = be.lib, be.ctx

    def cache(k, v, scale, weight, max_rows):
        t = Kv4T(k.data_ptr(), v.data_ptr(), scale.data_ptr(), weight.data_ptr() if weight is not None else None, 0.0, c["kv"], c["hd"], max_rows)
        return C.pointer(t)
    if s.kind == "decode":
        t = cache(s.k, s.v, s.scale, s.weight if c["weights"] else None, s.max_rows)
        return [(lib.ibcu_attention_decode_kv4, (ctx, t, s.q.data_ptr(), s.k_new.data_ptr(), s.v_new.data_ptr(), s.out.data_ptr(), c["heads"], c["rows"], c["rows"],
                                                 c["B"], 10000.0))]
    if s.kind == "attention":
        t = cache(s.k, s.v, s.scale, s.weight if c["weights"] else None, s.max_rows)
        return [(lib.ibcu_attention_kv4, (ctx, t, s.q.data_ptr(), s.out.data_ptr(), c["heads"], c["rows"], c["B"]))]
    if s.kind == "append":
        t = cache(s.k, s.v, s.scale, None, s.max_rows)
        return [(lib.ibcu_kv4_write, (ctx, t, s.k_new.data_ptr(), s.v_new.data_ptr(), c["rows"], c["rows"], c["B"], c["theta"])),
                (lib.ibcu_kv4_read, (ctx, t, s.k_out.data_ptr(), s.v_out.data_ptr(), c["rows"], c["B"]))]
    if s.kind == "evict":
        src, dst = cache(s.k, s.v, s.scale, s.weight, s.max_rows), cache(s.dk, s.dv, s.dscale, s.dweight, s.dst_rows)
        return [(lib.ibcu_kv4_evict, (ctx, src, dst, c["rows"], c["keep"], c["sink"], c["recent"], s.kept.data_ptr()))]
    n, M = c["tensors"], c["M"]
    ts = (LinearT * n)(*[LinearT(s.w[i].data_ptr(), s.sw[i].data_ptr(), s.out[i].data_ptr(), M, M, 0, 0) for i in range(n)])
    return [(lib.ibcu_linear_w8a8_fp32, (ctx, ts, n, s.x.data_ptr(), c["N"], c["B"]))]


# ── the plain form ─────────────────────────────────────────────────────────────────────────────────────────────────
def _rotate(x, heads, pos0, theta):
    """adjacent pairs by pos * theta^(-2m / hd), in 64 bits (far positions), rounded once"""
    B, hd = x.shape[0], x.shape[1] // heads
    if not theta:
        return x
    m = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    ang = torch.arange(pos0, pos0 + B, device="cuda", dtype=torch.float64)[:, None] * torch.exp2(m * (-2.0 / hd * math.log2(theta)))
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    y = x.double().reshape(B, heads, hd // 2, 2)
    return torch.stack([y[..., 0] * c - y[..., 1] * s, y[..., 0] * s + y[..., 1] * c], -1).reshape(B, heads * hd).float()


def _attend(q, k, v, heads, rows):
    """q [B, heads * hd], k and v [kv, rows + B, hd] -> out, probabilities [kv, B, group, rows + B]"""
    kv, R, hd = k.shape
    B, group = q.shape[0], heads // kv
    qh = q.reshape(B, kv, group, hd).transpose(0, 1).reshape(kv, B * group, hd)
    s = (qh @ k.transpose(1, 2) * hd ** -0.5).reshape(kv, B, group, R)
    hidden = torch.arange(R, device="cuda")[None, :] > rows + torch.arange(B, device="cuda")[:, None]
    s = s.masked_fill(hidden[None, :, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    out = (p.reshape(kv, B * group, R) @ v).reshape(kv, B, group, hd).transpose(0, 1).reshape(B, heads * hd)
    return out, p


def _plain(s):
    c = s.case
    if s.kind in ("decode", "attention"):
        heads, kv, hd, rows, B = (c[n] for n in ("heads", "kv", "hd", "rows", "B"))
        ng, R, q, new = hd // GROUP, rows + B, s.q, {}
        if s.kind == "decode":
            q, kr = _rotate(s.q, heads, rows, 10000.0), _rotate(s.k_new, kv, rows, 10000.0)
            kc, ks = _quantise(kr.reshape(B, kv, hd).transpose(0, 1))
            vc, vs = _quantise(s.v_new.reshape(B, kv, hd).transpose(0, 1))
            s.k[:, rows:R], s.v[:, rows:R] = _pack_k(kc), _pack_v(vc)
            s.scale[:, rows:R, :ng], s.scale[:, rows:R, ng:] = ks, vs
            new = {"k": s.k[:, rows:R], "v": s.v[:, rows:R], "scale": s.scale[:, rows:R]}
        k, v = _unpack(s.k[:, :R], 4, s.scale[:, :R, :ng]), _unpack(s.v[:, :R], 8, s.scale[:, :R, ng:])
        out, p = _attend(q, k, v, heads, rows)
        return {"out": out, **new, **({"weight": p.sum((1, 2))} if c["weights"] else {})}
    if s.kind == "append":
        kv, hd, rows, B = (c[n] for n in ("kv", "hd", "rows", "B"))
        ng = hd // GROUP
        kc, ks = _quantise(_rotate(s.k_new, kv, rows, c["theta"]).reshape(B, kv, hd))
        vc, vs = _quantise(s.v_new.reshape(B, kv, hd))
        s.k[:, rows:rows + B], s.v[:, rows:rows + B] = _pack_k(kc).transpose(0, 1), _pack_v(vc).transpose(0, 1)
        s.scale[:, rows:rows + B, :ng], s.scale[:, rows:rows + B, ng:] = ks.transpose(0, 1), vs.transpose(0, 1)
        k = _unpack(s.k[:, rows:rows + B], 4, s.scale[:, rows:rows + B, :ng])
        v = _unpack(s.v[:, rows:rows + B], 8, s.scale[:, rows:rows + B, ng:])
        return {"k": k.transpose(0, 1).reshape(B, kv * hd), "v": v.transpose(0, 1).reshape(B, kv * hd)}
    if s.kind == "evict":
        rows, keep, sink, recent = (c[n] for n in ("rows", "keep", "sink", "recent"))
        w = s.weight[:, :rows].clone()
        w[:, :sink] = math.inf
        w[:, rows - recent:] = math.inf
        kept = w.sort(dim=1, descending=True, stable=True).indices[:, :keep].sort(dim=1).values
        at = kept[..., None]
        take = lambda plane: plane.gather(1, at.expand(-1, -1, plane.shape[2]))  # noqa: E731
        return {"kept": kept.int(), "k": take(s.k), "v": take(s.v), "scale": take(s.scale), "weight": s.weight.gather(1, kept)}
    amax = s.x.abs().amax(1, keepdim=True)
    sx = amax / 127
    xq = (s.x * (1 / sx)).round()
    acc = xq @ s.w.float().transpose(1, 2)                    # whole numbers: the sums lose what FP32 products of this length lose
    return {"out": acc * (s.sw.float()[:, None, :] * sx)}


def run(state):
    if not own:
        return _plain(state)
    s, c = state, state.case
    if s.calls is None:
        s.calls = _calls(s)
    for fn, args in s.calls:
        rc = fn(*args)
        if rc != 0:
            _shared["be"]._check(rc)
    if s.kind in ("decode", "attention"):
        rows, R = c["rows"], c["rows"] + c["B"]
        # the new rows as they lie in the cache: their bytes are compared, which asks for more than their values would
        new = {"k": s.k[:, rows:R], "v": s.v[:, rows:R], "scale": s.scale[:, rows:R]} if s.kind == "decode" else {}
        return {"out": s.out, **new, **({"weight": s.weight[:, :R]} if c["weights"] else {})}
    if s.kind == "append":
        return {"k": s.k_out, "v": s.v_out}
    if s.kind == "evict":
        keep = c["keep"]
        return {"kept": s.kept, "k": s.dk[:, :keep], "v": s.dv[:, :keep], "scale": s.dscale[:, :keep], "weight": s.dweight[:, :keep]}
    return {"out": s.out}


# ── what the formulas say, in 64 bits ──────────────────────────────────────────────────────────────────────────────
def _exact_turn(x, pos, theta):
    """[heads, hd] of one position, turned by complex multiplication"""
    if not theta:
        return x.double()
    hd = x.shape[-1]
    ang = pos * theta ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    z = torch.view_as_complex(x.double().reshape(x.shape[0], hd // 2, 2).contiguous()) * torch.polar(torch.ones_like(ang), ang)
    return torch.view_as_real(z).reshape(x.shape)


def _exact_held(x):
    """the values that the cache holds for x [..., hd]: the rows are FP32 and the scales fp16 by definition, the rest is in 64 bits"""
    y = x.float().double().unflatten(-1, (-1, GROUP))
    s = (y.abs().amax(-1).float() / 7).half()
    inv = (1 / s.float()).double()
    held = torch.clamp(torch.round((y * inv[..., None]).float().double()), -7, 7) * s.double()[..., None]
    return torch.where(s[..., None] == 0, torch.zeros_like(held), held).flatten(-2)


def _exact_rows(plane, scale, key):
    """64-bit values of a head's packed rows, value by value in the order of the row"""
    R, hd = plane.shape[0], plane.shape[1] * 2
    ng = hd // GROUP
    i = torch.arange(hd, device="cuda")
    j, r = i // GROUP, i % GROUP
    at = (r // 8 * ng + j) * 8 + r % 8 if key else (r // 4 * ng + j) * 4 + r % 4
    code = (plane[:, at // 2].int() >> (4 * (at % 2)).int()) & 15
    return (code - 8).double() * scale.double()[:, j]


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("decode", "attention"):
        heads, kv, hd, rows, B = (case[n] for n in ("heads", "kv", "hd", "rows", "B"))
        ng, R, group = hd // GROUP, rows + B, heads // kv
        old = rows if kind == "decode" else R
        out = torch.zeros(B, heads, hd, device="cuda", dtype=torch.float64)
        weight = torch.zeros(kv, R, device="cuda", dtype=torch.float64)
        q = s.q.reshape(B, heads, hd).double()
        if kind == "decode":
            q = torch.stack([_exact_turn(s.q[b].reshape(heads, hd), rows + b, 10000.0) for b in range(B)])
            kn = _exact_held(torch.stack([_exact_turn(s.k_new[b].reshape(kv, hd), rows + b, 10000.0) for b in range(B)]))
            vn = _exact_held(s.v_new.reshape(B, kv, hd))
        seen = torch.arange(R, device="cuda")[None] <= rows + torch.arange(B, device="cuda")[:, None]
        for h in range(heads):
            n = h // group
            k, v = _exact_rows(s.k[n, :old], s.scale[n, :old, :ng], True), _exact_rows(s.v[n, :old], s.scale[n, :old, ng:], False)
            if kind == "decode":
                k, v = torch.cat([k, kn[:, n]]), torch.cat([v, vn[:, n]])
            p = torch.softmax(torch.where(seen, q[:, h] @ k.T / math.sqrt(hd), torch.tensor(-math.inf, device="cuda", dtype=torch.float64)), -1)
            out[:, h] = p @ v
            weight[n] += p.sum(0)
        new = {"k": None, "v": None, "scale": None} if kind == "decode" else {}
        return {"out": out.reshape(B, heads * hd), **new, **({"weight": weight} if case["weights"] else {})}
    if kind == "append":
        kv, hd, rows, B = (case[n] for n in ("kv", "hd", "rows", "B"))
        k = torch.stack([_exact_turn(s.k_new[b].reshape(kv, hd), rows + b, case["theta"]) for b in range(B)])
        return {"k": _exact_held(k).reshape(B, kv * hd), "v": _exact_held(s.v_new.reshape(B, kv, hd)).reshape(B, kv * hd)}
    if kind == "evict":
        return None                               # rows are moved as they are
    sx = (s.x.abs().amax(1) / 127).double()
    q = torch.round((s.x * (1 / sx.float())[:, None]).double())
    return {"out": torch.stack([(q @ s.w[i].double().T) * s.sw[i].double() * sx[:, None] for i in range(case["tensors"])])}


# ── what a pass cannot do without ──────────────────────────────────────────────────────────────────────────────────
def work(case):
    """bytes: each input read once and each output written once; flops: multiplications and additions of the products"""
    kind = case["kind"]
    if kind in ("decode", "attention"):
        heads, kv, hd, rows, B = (case[n] for n in ("heads", "kv", "hd", "rows", "B"))
        R, row = rows + B, case["hd"] + 4 * case["hd"] // GROUP          # bytes of a row: two planes of half bytes, two scales a group
        new = B * kv * (8 * hd + row) if kind == "decode" else 0         # FP32 keys and values read, their rows written
        held = (rows if kind == "decode" else R) * kv * row
        return {"bytes": held + new + 8 * B * heads * hd + (4 * kv * R if case["weights"] else 0), "flops": 4 * hd * heads * (B * rows + B * (B + 1) // 2)}
    if kind == "append":
        kv, hd, B = case["kv"], case["hd"], case["B"]
        return {"bytes": B * kv * (16 * hd + 2 * (hd + 4 * hd // GROUP)), "flops": 8 * B * kv * hd}
    if kind == "evict":
        kv, hd, rows, keep = (case[n] for n in ("kv", "hd", "rows", "keep"))
        return {"bytes": kv * (4 * rows + keep * (2 * (hd + 4 * hd // GROUP) + 12)), "flops": 0}
    M, n, N, B = (case[x] for x in ("M", "tensors", "N", "B"))
    return {"bytes": n * M * (N + 2) + 4 * B * (N + n * M), "flops": 2 * n * M * N * B}

"""Timed cases of soft correspondence: the softmax match of feature maps, its gradient, and the 8-bit template store.

`run` computes a case either in plain torch operations in 32 bits (`own` false) or through this repository's entry points
(`own` true); `exact` computes the same outputs in 64 bits from the definition.

kind "match": soft_match(query, ref, value) -> out, lse          kind "train": the same with the gradients of its inputs
kind "bank":  write views into a template store and read others   kind "recall": soft_match against stored views
"""
import math

import torch

own = False

INT8, FP8 = "int8", "fp8"


# ------------------------------------------------------------------------------------------------ cases
def _match(name, dtype, batch, h, w, channels, heads=1, queries=0, value=0, scale=20.0, cap=0.0, falloff=0.0, masked=False,
           ragged=False, kind="match"):
    """queries = 0: every cell of a query map of the same size; value = 0: the reference map is its own value."""
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "h": h, "w": w, "channels": channels, "heads": heads,
            "queries": queries, "value": value, "scale": scale, "cap": cap, "falloff": falloff, "masked": masked,
            "ragged": ragged}


def _bank(name, dtype, store, stored, count, h, w, channels):
    return {"name": name, "kind": "bank", "dtype": dtype, "store": store, "stored": stored, "count": count, "h": h, "w": w,
            "channels": channels}


def _recall(name, dtype, store, stored, batch, views, queries, h, w, channels, heads=1, scale=20.0, cap=0.0):
    return {"name": name, "kind": "recall", "dtype": dtype, "store": store, "stored": stored, "batch": batch, "views": views,
            "queries": queries, "h": h, "w": w, "channels": channels, "heads": heads, "scale": scale, "cap": cap}


def listed():
    return [
        # ten annotated keypoints of one image against one template on the correlation layers' 28 x 28 grid: latency
        _match("keypoints-f32-28", "f32", 1, 28, 28, 128, queries=10, masked=True),
        # one pair of 64 x 64 x 128 maps in float32
        _match("pair-f32-64", "f32", 1, 64, 64, 128),
        # ground-truth correspondences of a batch (up to 1000 each, ragged) on an odd grid, two heads of 50 channels
        _match("ragged-f32-57x43", "f32", 5, 57, 43, 100, heads=2, queries=1000, masked=True, ragged=True),
        # a batch of pairs in bfloat16 with a locality prior, and the value map apart
        _match("batch-bf16-64", "bf16", 64, 64, 64, 128, value=128, falloff=0.002),
        # three template views at 128 x 128 x 256, capped scores, background masked
        _match("views-bf16-128", "bf16", 3, 128, 128, 256, heads=2, cap=15.0, masked=True),
        # a training step of the 28 x 28 grid in float32, batch 8
        _match("train-f32-28", "f32", 8, 28, 28, 128, cap=15.0, kind="train"),
        # a training step of 64 x 64 maps in bfloat16
        _match("train-bf16-64", "bf16", 16, 64, 64, 128, falloff=0.002, masked=True, kind="train"),
        # a training step on odd maps, three heads, a narrower value map, ragged queries
        _match("train-bf16-45x61", "bf16", 6, 45, 61, 192, heads=3, value=96, cap=15.0, ragged=True, kind="train"),
        # two dozen views of a class at the networks' 56 x 56 x 128, stored and read back
        _bank("bank-int8-56", "f32", INT8, 64, 24, 56, 56, 128),
        _bank("bank-fp8-31x47", "bf16", FP8, 40, 17, 31, 47, 200),
        # ten keypoints per image against its three stored views, batch 8
        _recall("recall-int8-56", "bf16", INT8, 64, 8, 3, 10, 56, 56, 128),
        # one query cell against 24 stored views of 128 x 128 x 256
        _recall("recall-fp8-128", "f32", FP8, 32, 1, 24, 1, 128, 128, 256, heads=2, cap=15.0),
    ]


_MOST = 8.2e11          # flops of the largest listed case


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["match", "match", "train", "bank", "recall"])
    dtype = rng.choice(["f32", "bf16"])
    h, w = _log(rng, 5, 100), _log(rng, 5, 100)
    if kind == "bank":
        count = _log(rng, 1, 24)
        return _bank(None, dtype, rng.choice([INT8, FP8]), count + rng.randrange(40), count, h, w, _log(rng, 3, 256)) | {"name": ""}
    heads = rng.choice([1, 1, 2, 3])
    channels = heads * _log(rng, 4, 256 // heads)
    scale, cap = rng.choice([1.0, 10.0, 30.0]), rng.choice([0.0, 0.0, 12.0, 30.0])
    if kind == "recall":
        views = _log(rng, 1, 12)
        return _recall("", dtype, rng.choice([INT8, FP8]), views + rng.randrange(12), _log(rng, 1, 8), views, _log(rng, 1, 600),
                       h, w, channels, heads, scale, cap)
    queries = rng.choice([0, 0, _log(rng, 1, 1000)])
    value = heads * _log(rng, 2, 256 // heads) if rng.random() < 0.5 else 0
    c = _match("", dtype, 1, h, w, channels, heads, queries, value, scale, cap, rng.choice([0.0, 0.001, 0.05]), rng.random() < 0.5,
               rng.random() < 0.4, kind)
    if queries:
        c["falloff"] = 0.0
    most = min(48, int(0.25 * _MOST / (work(c)["flops"] * (8 if dtype == "f32" else 1))))
    c["batch"] = _log(rng, 1, max(1, most))
    return c


# ------------------------------------------------------------------------------------------------ inputs
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _unit(x):
    return x / x.square().sum(1, keepdim=True).sqrt()


def _features(g, shape):
    return _unit(torch.randn(shape, generator=g, device="cuda"))


def _blobs(g, n, h, w):
    """Silhouettes: a filled ellipse per map, as a rendered object's alpha channel gives."""
    cy, cx, ry, rx = (torch.rand((n, 1, 1), generator=g, device="cuda") for _ in range(4))
    y = torch.arange(h, device="cuda").view(1, -1, 1) / h - (0.3 + 0.4 * cy)
    x = torch.arange(w, device="cuda").view(1, 1, -1) / w - (0.3 + 0.4 * cx)
    return (y / (0.2 + 0.3 * ry)).square() + (x / (0.2 + 0.3 * rx)).square() < 1


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]
    h, w, c = case["h"], case["w"], case["channels"]
    s = {"case": case}
    if case["kind"] in ("bank", "recall"):
        n = case["stored"]
        kind = torch.int8 if case["store"] == INT8 else torch.float8_e4m3fn
        s["codes"] = torch.zeros((n, c, h * w), dtype=torch.uint8, device="cuda").view(kind)
        s["scales"] = torch.zeros((n, h * w), device="cuda")
        s["mask"] = torch.zeros((n, h * w), dtype=torch.uint8, device="cuda")
        order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    if case["kind"] == "bank":
        # trunk features before the norm layer: cells of very different size
        gain = torch.exp(torch.randn((case["count"], 1, h, w), generator=g, device="cuda"))
        s["features"] = (torch.randn((case["count"], c, h, w), generator=g, device="cuda") * gain).to(t)
        s["object"] = _blobs(g, case["count"], h, w)
        s["write"] = order[:case["count"]].contiguous()
        s["read"] = s["write"].flip(0).contiguous()
        return s
    if case["kind"] == "recall":
        b, v, q = case["batch"], case["views"], case["queries"]
        for i in range(0, n, 4):
            m = min(4, n - i)
            f = _features(g, (m, c, h * w))
            s["codes"][i:i + m], s["scales"][i:i + m], _ = _quantise(f, case["store"])
            s["mask"][i:i + m] = _blobs(g, m, h, w).view(m, -1)
        s["views"] = torch.stack([order.roll(3 * i)[:v] for i in range(b)]).contiguous()
        s["query"] = _features(g, (b, c, q)).to(t)
        return s
    b, n = case["batch"], case["queries"]
    ref = _features(g, (b, c, h, w))
    if n:       # cells of the reference map seen again, a little off
        at = torch.randint(h * w, (b, 1, n), generator=g, device="cuda").expand(b, c, n)
        seen = ref.view(b, c, -1).gather(2, at)
    else:
        seen = ref.roll((h // 7, -(w // 5)), (2, 3))
    s["query"] = _unit(seen + 0.08 * torch.randn(seen.shape, generator=g, device="cuda")).to(t)
    s["ref"] = ref.to(t)
    s["value"] = torch.randn((b, case["value"], h, w), generator=g, device="cuda").to(t) if case["value"] else None
    s["object"] = _blobs(g, b, h, w) if case["masked"] else None
    s["falloff"] = case["falloff"] * torch.arange(1, case["heads"] + 1, device="cuda") if case["falloff"] else None
    nq = n or h * w
    s["count"] = torch.randint(nq // 3, nq + 1, (b,), generator=g, device="cuda").to(torch.int32) if case["ragged"] else None
    if case["kind"] == "train":
        # both uses of the match are trained: the transferred features and the confidence
        s["d_out"] = torch.randn((b, case["value"] or c) + tuple(s["query"].shape[2:]), generator=g, device="cuda").to(t)
        s["d_lse"] = torch.randn((b, case["heads"], nq), generator=g, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(x, store):
    """x (n,C,cells) float32 -> codes, scales (n,cells), finite (n,cells)."""
    finite = torch.isfinite(x).all(1)
    x = torch.where(finite[:, None], x, torch.zeros_like(x))
    top = 127.0 if store == INT8 else 448.0
    scale = x.abs().amax(1) / top
    # 64 bits: a quotient that 32 bits round onto the border between two codes takes the wrong one now and then
    y = torch.where(scale[:, None] > 0, x.double() / scale[:, None].double(), torch.zeros_like(x, dtype=torch.float64))
    y = y.clamp(-top, top)
    if store == INT8:
        return y.round().to(torch.int8), scale, finite
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent.clamp_min(-5) - 4)
    return ((y / step).round() * step).float().to(torch.float8_e4m3fn), scale, finite


def _grid(h, w):
    j = torch.arange(h * w, device="cuda")
    return j % w, j // w


def _plain_match(q, k, v, heads, scale, cap, penalty, allowed, count):
    """q (b,C,n), k (b,C,m), v (b,Cv,m) in one type, penalty (heads,n,m) or None, allowed (b,m) or None, count (b,) or None."""
    b, n, m = q.shape[0], q.shape[2], k.shape[2]
    split = lambda x: x.reshape(b, heads, -1, x.shape[2])
    z = torch.matmul(split(q).transpose(2, 3) * scale, split(k))
    if cap:
        z = torch.tanh(z / cap) * cap
    if penalty is not None:
        z = z - penalty
    if allowed is not None:
        z = z.masked_fill(~allowed[:, None, None, :], -math.inf)
    if count is not None:
        z = z.masked_fill((torch.arange(n, device=z.device) >= count[:, None])[:, None, :, None], -math.inf)
    top = z.amax(3, keepdim=True).detach()
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = torch.exp(z - top)
    total = e.sum(3, keepdim=True)
    some = total > 0
    p = e / torch.where(some, total, torch.ones_like(total))
    lse = torch.where(some, torch.log(torch.where(some, total, torch.ones_like(total))) + top, torch.full_like(total, -math.inf))
    out = torch.matmul(split(v), p.transpose(2, 3).contiguous())
    return out.reshape(b, -1, n), lse[..., 0]


def _penalty(s, dtype):
    if s["falloff"] is None:
        return None
    x, y = (t.to(dtype) for t in _grid(s["case"]["h"], s["case"]["w"]))
    d2 = (x[:, None] - x[None]).square() + (y[:, None] - y[None]).square()
    return s["falloff"].to(dtype)[:, None, None] * d2


def _plain_inputs(s, dtype):
    c = s["case"]
    flat = lambda x: x.to(dtype).flatten(2)
    allowed = s["object"].flatten(1) if s["object"] is not None else None
    q, k = flat(s["query"]), flat(s["ref"])
    if s["count"] is not None:
        q = torch.where(torch.arange(q.shape[2], device="cuda") < s["count"][:, None, None], q, torch.zeros_like(q))
    return q, k, (flat(s["value"]) if s["value"] is not None else None), allowed


def _plain(s):
    c = s["case"]
    t = _TYPES[c["dtype"]]
    if c["kind"] == "bank":
        f = s["features"].float().flatten(2)
        codes, scales, finite = _quantise(f, c["store"])
        at, of = s["write"].long(), s["read"].long()
        s["codes"].view(torch.uint8)[at] = codes.view(torch.uint8)
        s["scales"][at] = scales
        s["mask"][at] = (finite & s["object"].flatten(1)).to(torch.uint8)
        values = s["codes"].view(torch.uint8)[of].view(s["codes"].dtype).float() * s["scales"][of][:, None]
        return values.view(-1, c["channels"], c["h"], c["w"]).to(t), s["mask"][of].view(-1, c["h"], c["w"])
    if c["kind"] == "recall":
        k = s["codes"].view(torch.uint8)[s["views"].long()].view(s["codes"].dtype).float() * s["scales"][s["views"].long()][:, :, None]
        k = k.transpose(1, 2).flatten(2)                                       # (b, C, V * cells)
        allowed = s["mask"][s["views"].long()].flatten(1) > 0
        out, lse = _plain_match(s["query"].float(), k, k, c["heads"], c["scale"], c["cap"], None, allowed, None)
        return out.to(t), lse
    q, k, v, allowed = _plain_inputs(s, torch.float32)
    penalty = _penalty(s, torch.float32)
    if c["kind"] == "match":
        out, lse = _plain_match(q, k, k if v is None else v, c["heads"], c["scale"], c["cap"], penalty, allowed, s["count"])
        return out.to(t).view(out.shape[:2] + s["query"].shape[2:]), lse
    leaves = [x.requires_grad_() for x in (q.detach(), k, v) if x is not None]
    out, lse = _plain_match(leaves[0], leaves[1], leaves[-1], c["heads"], c["scale"], c["cap"], penalty, allowed, s["count"])
    d_lse = torch.where(torch.isfinite(lse.detach()), s["d_lse"], torch.zeros_like(s["d_lse"]))
    grads = torch.autograd.grad([out, torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))], leaves,
                                [s["d_out"].float().flatten(2), d_lse])
    shapes = [s[n].shape for n in ("query", "ref", "value") if s[n] is not None]
    return [out.detach().to(t).view(s["d_out"].shape), lse.detach()] + [g.to(t).view(z) for g, z in zip(grads, shapes)]


# ------------------------------------------------------------------------------------------------ one pass
def _own(s):
    from pose_estimation_amd import soft_correspondence as sc
    c = s["case"]
    if c["kind"] in ("bank", "recall"):
        store = sc.TemplateStore.from_tensors(s["codes"], s["scales"], s["mask"], (c["h"], c["w"]))
    if c["kind"] == "bank":
        store.write(s["write"], s["features"], mask=s["object"])
        return store.read(s["read"], dtype=_TYPES[c["dtype"]]), store.read_mask(s["read"])
    if c["kind"] == "recall":
        return store.soft_match(s["query"], s["views"], heads=c["heads"], scale=c["scale"], cap=c["cap"], return_lse=True)
    options = dict(heads=c["heads"], scale=c["scale"], cap=c["cap"], falloff=s["falloff"], mask=s["object"],
                   num_query=s["count"], return_lse=True)
    if c["kind"] == "match":
        return sc.soft_match(s["query"], s["ref"], s["value"], **options)
    leaves = [x.detach().requires_grad_() for x in (s["query"], s["ref"], s["value"]) if x is not None]
    out, lse = sc.soft_match(*leaves, **options)
    grads = torch.autograd.grad([out, lse], leaves, [s["d_out"], s["d_lse"]])
    return [out.detach(), lse.detach(), *grads]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    cells = c["h"] * c["w"]
    if c["kind"] == "bank":
        stored = c["count"] * cells * (c["channels"] + 4 + 1)
        return {"bytes": c["count"] * cells * (2 * size * c["channels"] + 2) + 2 * stored, "flops": 4 * c["count"] * cells * c["channels"]}
    if c["kind"] == "recall":
        m, n = c["views"] * cells, c["queries"]
        read = min(c["stored"], c["batch"] * c["views"]) * cells * (c["channels"] + 5)
        return {"bytes": read + c["batch"] * n * (2 * size * c["channels"] + 4 * c["heads"]),
                "flops": 4 * c["batch"] * n * m * c["channels"]}
    b, n, q, v = c["batch"], c["queries"] or cells, c["channels"], c["value"] or c["channels"]
    maps = b * size * (n * (q + v) + cells * (q + (c["value"] and v))) + 4 * b * c["heads"] * n + (b * cells if c["masked"] else 0)
    if c["kind"] == "match":
        return {"bytes": maps, "flops": 2 * b * n * cells * (q + v)}
    grads = b * size * (n * (q + v) + cells * (q + (c["value"] and v))) + 4 * b * c["heads"] * n
    return {"bytes": maps + grads, "flops": 2 * b * n * cells * (q + v) + 2 * b * n * cells * (3 * q + 2 * v)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _e4m3(y):
    """Round to the nearest e4m3 value, ties to the even one, in 64 bits."""
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    return (y / step).round() * step


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    h, w = c["h"], c["w"]
    if c["kind"] == "bank":
        x = s["features"].double()
        top = 127.0 if c["store"] == INT8 else 448.0
        scale = (x.abs().amax(1, keepdim=True).float() / top).double()        # scales are held in 32 bits
        y = torch.where(scale > 0, x / scale, torch.zeros_like(x))
        y = y.round() if c["store"] == INT8 else _e4m3(y)
        return (y * scale).flip(0), s["object"].to(torch.uint8).flip(0)
    d = torch.float64
    heads = c["heads"]
    if c["kind"] == "recall":
        outs, lses = [], []
        for b in range(c["batch"]):
            at = s["views"][b].tolist()
            k = torch.cat([s["codes"][i].float().to(d) * s["scales"][i].to(d) for i in at], 1)
            ok = torch.cat([s["mask"][i] for i in at]) > 0
            o, l, _ = _item64(s["query"][b].to(d), k, k, c, None, ok, s["query"].shape[2])
            outs.append(o)
            lses.append(l)
        return torch.stack(outs), torch.stack(lses)
    q, k, v = (s[x].flatten(2).to(d) if s[x] is not None else None for x in ("query", "ref", "value"))
    shared = v is None
    v = k if shared else v
    outs = []
    for b in range(c["batch"]):
        ok = s["object"][b].flatten() if s["object"] is not None else None
        live = int(s["count"][b]) if s["count"] is not None else q.shape[2]
        d_out = (s["d_out"][b].flatten(1).to(d), s["d_lse"][b].to(d)) if c["kind"] == "train" else None
        outs.append(_item64(q[b], k[b], v[b], c, s["falloff"], ok, live, d_out))
    out = torch.stack([o[0] for o in outs]).view((c["batch"], -1) + s["query"].shape[2:])
    lse = torch.stack([o[1] for o in outs])
    if c["kind"] == "match":
        return out, lse
    dq, dk, dv = (torch.stack([o[2][i] for o in outs]) for i in range(3))
    if shared:
        return [out, lse, dq.view(s["query"].shape), (dk + dv).view(s["ref"].shape)]
    return [out, lse, dq.view(s["query"].shape), dk.view(s["ref"].shape), dv.view(s["value"].shape)]


def _item64(q, k, v, c, falloff, ok, live, d_out=None):
    """One item head by head, `live` queries of it: out, lse and, with d_out, the three gradients by their formulas."""
    n, m = q.shape[1], k.shape[1]
    dim, vdim = q.shape[0] // c["heads"], v.shape[0] // c["heads"]
    out, lse = q.new_zeros((v.shape[0], n)), q.new_full((c["heads"], n), -math.inf)
    grads = [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    some = live > 0 and (ok is None or bool(ok.any()))
    for i in range(c["heads"] if some else 0):
        a, e = slice(i * dim, (i + 1) * dim), slice(i * vdim, (i + 1) * vdim)
        for j in range(0, live, 4096):
            r = slice(j, min(live, j + 4096))
            x = c["scale"] * (q[a, r].t() @ k[a])
            t = torch.tanh(x / c["cap"]) if c["cap"] else None
            z = c["cap"] * t if c["cap"] else x
            if falloff is not None:
                y0, x0 = torch.div(torch.arange(m, device="cuda"), c["w"], rounding_mode="floor"), torch.arange(m, device="cuda") % c["w"]
                z = z - falloff[i].double() * ((x0[r, None] - x0) ** 2 + (y0[r, None] - y0) ** 2)
            if ok is not None:
                z = torch.where(ok, z, -math.inf)
            l = torch.logsumexp(z, 1)
            p = torch.exp(z - l[:, None])
            out[e, r] = v[e] @ p.t()
            lse[i, r] = l
            if d_out is not None:
                do = d_out[0][e, r]
                dp = do.t() @ v[e]
                dx = p * (dp - (p * dp).sum(1, keepdim=True) + d_out[1][i, r, None])
                dx = c["scale"] * (dx * (1 - t * t) if c["cap"] else dx)
                grads[0][a, r] = k[a] @ dx.t()
                grads[1][a] += q[a, r] @ dx
                grads[2][e] += do @ p
    return out, lse, grads

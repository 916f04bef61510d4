"""The workloads of the packed-sequence operators (VAESNe.PackedLayers): what is measured, and on which sizes.

Four operators of a transformer that trains on sequences of different lengths without padding them:

attn   softmax attention over packed sequences, grouped key / value heads, causal or not: a whole prompt, a few
       last queries over long keys, a training step
bias   the same with a learned relative position bias by buckets, and the bias table's gradient
norm   the norm after a block, its gate, the scaled residual and the norm before the next block, in one
act8   an activation kept in 8 bits for the backward pass: GELU with its gradient, and the plain store and read

`own` False: the plain form, elementary torch operations in 32 bits.  `own` True: the framework's operators.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 32          # values that share one exponent in the 8-bit form


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a batch of 16 light curves (20 to 60 observations each, 4 heads of 8, the models' own width): latency
        dict(name="attn_photometry_f32", op="attn", mode="prompt", type="float32", seqs=16, shortest=20, longest=60,
             lens=1, queries=0, heads=4, kv_heads=4, dim=8, causal=False),
        # one training step of a causal block over ragged documents of up to 4096 tokens, 4 query heads a key head
        dict(name="attn_train_bf16", op="attn", mode="train", type="bfloat16", seqs=4, shortest=1000, longest=4096,
             lens=2, queries=0, heads=16, kv_heads=4, dim=128, causal=True),
        # a prompt batch as a server packs it: long, odd lengths, 32 heads over 8 key heads
        dict(name="attn_prompt_bf16", op="attn", mode="prompt", type="bfloat16", seqs=3, shortest=2000, longest=8001,
             lens=3, queries=0, heads=32, kv_heads=8, dim=128, causal=True),
        # one new token for each of 32 sequences over caches of very different length
        dict(name="attn_last_token_bf16", op="attn", mode="prompt", type="bfloat16", seqs=32, shortest=100,
             longest=16384, lens=4, queries=1, heads=32, kv_heads=8, dim=128, causal=True),
        # light curves again, with a bias by distance in the sequence, trained: latency of forward and backward
        dict(name="bias_photometry_train_f32", op="bias", mode="train", type="float32", seqs=16, shortest=20,
             longest=60, lens=5, queries=0, heads=4, kv_heads=4, dim=8, causal=False, buckets=32, distance=128),
        # spectra of up to 982 wavelengths read in both directions: an encoder's forward pass
        dict(name="bias_spectra_bf16", op="bias", mode="prompt", type="bfloat16", seqs=32, shortest=300, longest=982,
             lens=6, queries=0, heads=16, kv_heads=16, dim=64, causal=False, buckets=32, distance=128),
        # a causal training step with the bias table's gradient over odd lengths
        dict(name="bias_train_f16", op="bias", mode="train", type="float16", seqs=6, shortest=500, longest=2047,
             lens=7, queries=0, heads=12, kv_heads=12, dim=64, causal=True, buckets=32, distance=128),
        # the residual joins of the models' own width, 16 x 60 observations: latency
        dict(name="norm_photometry_f32", op="norm", mode="train", type="float32", rows=960, width=32, kind="layer",
             gate="channel", scale=1.0),
        # a serving pass over a prompt: forward only, no gradient
        dict(name="norm_prompt_bf16", op="norm", mode="prompt", type="bfloat16", rows=4099, width=4096, kind="rms",
             gate="none", scale=1.0),
        # a training step's join with a learned gate for each token and channel
        dict(name="norm_train_bf16", op="norm", mode="train", type="bfloat16", rows=16384, width=4096, kind="rms",
             gate="token", scale=0.5),
        # the feed-forward activations of a training step, kept in 8 bits
        dict(name="act8_gelu_train_bf16", op="act8", mode="gelu", type="bfloat16", rows=8192, width=16384),
        # one light-curve batch's activations put away and read back: latency
        dict(name="act8_store_f32", op="act8", mode="store", type="float32", rows=960, width=33),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges; at most as costly as the largest listed one."""
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["attn", "attn", "bias", "bias", "norm", "act8"])
        kind = rng.choice(sorted(TYPES))
        if op in ("attn", "bias"):
            groups = rng.choice([1, 1, 2, 3, 4, 8]) if op == "attn" else rng.choice([1, 1, 2])
            kv = rng.choice([1, 2, 4, 8, 12])
            longest = _log_int(rng, 16, 8192)
            few = op == "attn" and rng.random() < 0.25
            case = dict(op=op, mode=rng.choice(["prompt", "train"]), type=kind, seqs=_log_int(rng, 1, 64),
                        shortest=rng.choice([1, max(1, longest // 8), longest]), longest=longest,
                        lens=rng.randrange(1 << 20), queries=rng.choice([1, 1, 5, 8]) if few else 0,
                        heads=kv * groups, kv_heads=kv, dim=rng.choice([8, 16, 24, 32, 64, 64, 80, 96, 128, 128]),
                        causal=rng.random() < 0.5)
            if op == "bias":
                case.update(buckets=rng.choice([8, 16, 32, 64]), distance=rng.choice([64, 100, 128, 512]))
        elif op == "norm":
            case = dict(op=op, mode=rng.choice(["prompt", "train"]), type=kind, rows=_log_int(rng, 1, 32768),
                        width=rng.choice([8 * _log_int(rng, 1, 1024), _log_int(rng, 8, 4096)]),
                        kind=rng.choice(["rms", "layer"]), gate=rng.choice(["none", "channel", "token"]),
                        scale=rng.choice([1.0, 0.5]))
        else:
            case = dict(op=op, mode=rng.choice(["gelu", "store"]), type=kind, rows=_log_int(rng, 1, 32768),
                        width=_log_int(rng, 1, 16384))
        if _cost(case) <= most and _plain_scores(case) <= 6.5e9:
            return case


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / (1e14 if case["type"] == "float32" else 1e15)


def _lengths(case):
    """(queries, keys) of each sequence."""
    r = random.Random(case["lens"])
    low, high = math.log(case["shortest"]), math.log(case["longest"])
    keys = [case["longest"]] + [int(round(math.exp(r.uniform(low, high)))) for _ in range(case["seqs"] - 1)]
    r.shuffle(keys)
    return [min(k, case["queries"]) if case["queries"] else k for k in keys], keys


def _plain_scores(case):
    """Scores that the padded plain form holds at once."""
    if case["op"] not in ("attn", "bias"):
        return 0
    return case["seqs"] * case["heads"] * max(_lengths(case)[0]) * case["longest"]


def work(case):
    size = torch.empty(0, dtype=TYPES[case["type"]]).element_size()
    train = case["mode"] in ("train", "gelu")
    if case["op"] in ("attn", "bias"):
        nq, nk = _lengths(case)
        pairs = sum(a * b - a * (a - 1) // 2 if case["causal"] else a * b for a, b in zip(nq, nk))
        q = sum(nq) * case["heads"] * case["dim"]
        kv = 2 * sum(nk) * case["kv_heads"] * case["dim"]
        table = case.get("buckets", 0) * case["heads"]
        # forward: two products of each pair; training: five more (scores again, dP, dV, dK, dQ)
        return {"bytes": size * ((4 * q + 2 * kv + 2 * table) if train else (2 * q + kv + table)),
                "flops": pairs * case["heads"] * case["dim"] * 2 * (7 if train else 2)}
    n = case["rows"] * case["width"]
    if case["op"] == "norm":
        gate = {"none": 0, "channel": case["width"], "token": n}[case["gate"]]
        params = case["width"] * (4 if case["kind"] == "layer" else 2)
        # forward: x, branch in, y, n out; training: dy, dn in, dx, dbranch out besides
        return {"bytes": size * ((8 * n + 2 * gate + 2 * params) if train else (4 * n + gate + params)),
                "flops": n * (40 if train else 12)}
    # x in, y out, dy in, dx out; or x in, the values out; the 8-bit form is written and read once besides
    kept = 2 * (n + (n + BLOCK - 1) // BLOCK)
    return {"bytes": (4 if train else 2) * n * size + kept, "flops": n * (40 if train else 6)}


# --------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(t)

    s = {"case": case}
    if case["op"] in ("attn", "bias"):
        nq, nk = _lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        s["q"], s["k"], s["v"] = normal(sum(nq), h, d), normal(sum(nk), hk, d), normal(sum(nk), hk, d)
        if case["op"] == "bias":
            s["table"] = normal(case["buckets"], h, scale=0.5)
        if case["mode"] == "train":
            s["dout"] = normal(sum(nq), h, d, scale=0.05)
        if own:
            P = _layers()
            s["plan"] = P.PackedSequences(nq, nk, device="cuda")
            if case["op"] == "bias":
                s["buckets"] = P.RelativeBuckets(case["buckets"], case["distance"], bidirectional=not case["causal"])
        else:
            s["plan"] = _plain_plan(nq, nk)
    elif case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # a residual stream: some channels much larger than the others
        channel = torch.exp(torch.randn(width, generator=g, device="cuda"))
        s["x"] = (torch.randn(rows, width, generator=g, device="cuda") * channel).to(t)
        s["branch"] = normal(rows, width, scale=0.3, mean=0.05)
        s["pre_weight"], s["post_weight"] = normal(width, scale=0.1, mean=1.0), normal(width, scale=0.1, mean=1.0)
        layer = case["kind"] == "layer"
        s["pre_bias"] = normal(width, scale=0.1) if layer else None
        s["post_bias"] = normal(width, scale=0.1) if layer else None
        s["gate"] = {"none": lambda: None, "channel": lambda: normal(width, scale=0.3, mean=0.5),
                     "token": lambda: normal(rows, width, scale=0.3, mean=0.5)}[case["gate"]]()
        if case["mode"] == "train":
            s["dy"], s["dn"] = normal(rows, width), normal(rows, width)
    else:
        # pre-activations: mostly small, a few rows far out, some exact zeros
        x = torch.randn(case["rows"], case["width"], generator=g, device="cuda") * 1.2
        x *= torch.exp(0.5 * torch.randn(case["rows"], 1, generator=g, device="cuda"))
        x *= torch.rand(case["rows"], case["width"], generator=g, device="cuda") > 0.01
        s["x"] = x.to(t)
        if case["mode"] == "gelu":
            s["dy"] = normal(case["rows"], case["width"], scale=0.1)
    if own and case["mode"] in ("train", "gelu"):
        for name in ("q", "k", "v", "table", "x", "branch", "pre_weight", "post_weight", "pre_bias", "post_bias",
                     "gate"):
            if s.get(name) is not None:
                s[name].requires_grad_()
    return s


def _layers():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vaesne-dev_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from VAESNe import PackedLayers
    return PackedLayers


def _plain_plan(nq, nk):
    """Where each padded place's row lies, and each packed row's padded place."""
    plan = {}
    for side, n in (("q", nq), ("k", nk)):
        n = torch.tensor(n)
        start = torch.cumsum(n, 0) - n
        place = torch.arange(int(n.max()))
        inside = place < n[:, None]
        plan[side] = {"row": torch.where(inside, start[:, None] + place, 0).cuda(), "inside": inside.cuda(),
                      "back": torch.nonzero(inside.reshape(-1)).reshape(-1).cuda(), "n": n.cuda()}
    return plan


# ------------------------------------------------------------------------------------------------------ run
def run(state):
    op, mode = state["case"]["op"], state["case"]["mode"]
    if own:
        return _own_attention(state) if op in ("attn", "bias") else _own_norm(state) if op == "norm" else _own_act8(state)
    if op in ("attn", "bias"):
        return _plain_attention(state)
    if op == "norm":
        return _plain_norm(state)
    return _plain_act8(state, mode)


def _own_attention(s):
    c, P = s["case"], _layers()
    more = {"bias": s["table"], "buckets": s["buckets"]} if c["op"] == "bias" else {}
    if c["mode"] != "train":
        with torch.no_grad():
            return {"o": P.packed_attention(s["q"], s["k"], s["v"], s["plan"], causal=c["causal"], **more)}
    leaves = [s["q"], s["k"], s["v"]] + ([s["table"]] if c["op"] == "bias" else [])
    o = P.packed_attention(s["q"], s["k"], s["v"], s["plan"], causal=c["causal"], **more)
    grads = torch.autograd.grad(o, leaves, s["dout"])
    return {"o": o.detach(), **dict(zip(("dq", "dk", "dv", "dtable"), grads))}


def _own_norm(s):
    c, P = s["case"], _layers()
    names = [n for n in ("x", "branch", "pre_weight", "post_weight", "pre_bias", "post_bias", "gate")
             if s[n] is not None]

    def call():
        return P.gated_norm(s["x"], s["branch"], s["pre_weight"], s["post_weight"], pre_bias=s["pre_bias"],
                            post_bias=s["post_bias"], gate=s["gate"], residual_scale=c["scale"], kind=c["kind"])

    if c["mode"] != "train":
        with torch.no_grad():
            y, n = call()
        return {"y": y, "n": n}
    y, n = call()
    grads = torch.autograd.grad([y, n], [s[k] for k in names], [s["dy"], s["dn"]])
    return {"y": y.detach(), "n": n.detach(), **{"d" + k: v for k, v in zip(names, grads)}}


def _own_act8(s):
    P = _layers()
    if s["case"]["mode"] == "store":
        return {"values": P.unpack8(P.pack8(s["x"]))}
    y = P.gelu8(s["x"])
    return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


# -------------------------------------------------------------------------------------------- the plain form
def _pad(x, side):
    """[rows, heads, dim] packed -> [sequence, head, place, dim] in 32 bits, zeros behind each sequence."""
    x = x.float()[side["row"]] * side["inside"][..., None, None]
    return x.permute(0, 2, 1, 3).contiguous()


def _packed(x, side):
    return x.permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[side["back"]]


def _plain_buckets(rel, count, distance, both):
    """Bucket of each key position minus query position: exact up close, by the logarithm further out."""
    if both:
        count //= 2
        base, far = torch.where(rel > 0, count, 0), rel.abs()
    else:
        base, far = torch.zeros_like(rel), (-rel).clamp(min=0)
    near = count // 2
    # 64 bits and a hair upwards: a distance that lies on a border belongs to the bucket above it
    step = torch.log(far.clamp(min=near).double() / near) / math.log(distance / near) * (count - near)
    return base + torch.where(far < near, far, (near + (step + 1e-9).floor().long()).clamp(max=count - 1))


def _plain_attention(s):
    c, side = s["case"], s["plan"]
    scale = 1.0 / math.sqrt(c["dim"])
    group = c["heads"] // c["kv_heads"]
    q = _pad(s["q"], side["q"])
    k = _pad(s["k"], side["k"]).repeat_interleave(group, 1)
    v = _pad(s["v"], side["k"]).repeat_interleave(group, 1)
    nq, nk = side["q"]["n"], side["k"]["n"]
    at = torch.arange(q.shape[2], device="cuda")[None, :] + (nk - nq)[:, None]          # the queries are the last ones
    rel = torch.arange(k.shape[2], device="cuda")[None, None, :] - at[:, :, None]
    seen = side["k"]["inside"][:, None, :] & side["q"]["inside"][:, :, None]
    seen = seen & (rel <= 0) if c["causal"] else seen
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    if c["op"] == "bias":
        bucket = _plain_buckets(rel, c["buckets"], c["distance"], not c["causal"])
        p += s["table"].float()[bucket].permute(0, 3, 1, 2)
    p.masked_fill_(~seen[:, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    o = torch.matmul(p, v)
    t = s["q"].dtype
    out = {"o": _packed(o, side["q"]).to(t)}
    if c["mode"] != "train":
        return out
    do = _pad(s["dout"], side["q"])
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous()).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    del p
    if c["op"] == "bias":
        # as many queries as keys here: shifting each row by its place puts one distance in one column
        n = q.shape[2]
        skewed = torch.nn.functional.pad(ds.double().sum(0).flip(1), (0, n)).reshape(c["heads"], -1)
        by_distance = skewed[:, :n * (2 * n - 1)].reshape(c["heads"], n, 2 * n - 1).sum(1)
        bucket = _plain_buckets(torch.arange(1 - n, n, device="cuda"), c["buckets"], c["distance"], not c["causal"])
        flat = torch.zeros(c["buckets"], c["heads"], dtype=torch.float64, device="cuda")
        flat.index_add_(0, bucket, by_distance.T.contiguous())
        out["dtable"] = flat.to(t)
    dq = torch.matmul(ds, k).mul_(scale)
    dk = torch.matmul(ds.transpose(2, 3), q).mul_(scale)

    def shared(x):
        return x.reshape(x.shape[0], c["kv_heads"], group, *x.shape[2:]).sum(2)

    out.update(dq=_packed(dq, side["q"]).to(t), dk=_packed(shared(dk), side["k"]).to(t),
               dv=_packed(shared(dv), side["k"]).to(t))
    return out


EPS = 1e-5


def _plain_normed(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _plain_norm_back(d, hat, r, kind):
    d = d - hat * (d * hat).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if kind == "layer" else 0.0)
    return d * r


def _plain_norm(s):
    c, t = s["case"], s["x"].dtype
    f = {n: None if s[n] is None else s[n].float()
         for n in ("x", "branch", "pre_weight", "post_weight", "pre_bias", "post_bias", "gate")}
    fhat, fr = _plain_normed(f["branch"], c["kind"])
    u = fhat * f["post_weight"]
    u = u if f["post_bias"] is None else u + f["post_bias"]
    y = f["x"] * c["scale"] + (u if f["gate"] is None else u * f["gate"])
    yhat, yr = _plain_normed(y, c["kind"])
    n = yhat * f["pre_weight"]
    n = n if f["pre_bias"] is None else n + f["pre_bias"]
    out = {"y": y.to(t), "n": n.to(t)}
    if c["mode"] != "train":
        return out
    dy, dn = s["dy"].float(), s["dn"].float()
    dy = dy + _plain_norm_back(dn * f["pre_weight"], yhat, yr, c["kind"])
    du = dy if f["gate"] is None else dy * f["gate"]
    out.update(dx=(dy * c["scale"]).to(t), dbranch=_plain_norm_back(du * f["post_weight"], fhat, fr, c["kind"]).to(t),
               dpre_weight=(dn * yhat).sum(0).to(t), dpost_weight=(du * fhat).sum(0).to(t))
    if f["pre_bias"] is not None:
        out.update(dpre_bias=dn.sum(0).to(t), dpost_bias=du.sum(0).to(t))
    if f["gate"] is not None:
        dgate = dy * u
        out["dgate"] = (dgate.sum(0) if f["gate"].dim() == 1 else dgate).to(t)
    return out


def _plain_eight_bits(x):
    """The values that x's 8-bit form stands for: blocks of 32 share a power of two, 7 bits and a sign each."""
    flat = x.float().reshape(-1)
    blocks = torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).reshape(-1, BLOCK)
    step = (torch.frexp(blocks.abs().amax(1, keepdim=True))[1] - 1).clamp(min=-126) - 6
    codes = torch.ldexp(blocks, -step).round().clamp(-127, 127)
    return torch.ldexp(codes, step).reshape(-1)[:flat.numel()].reshape(x.shape)


def _plain_act8(s, mode):
    x = s["x"]
    kept = _plain_eight_bits(x)
    if mode == "store":
        return {"values": kept.to(x.dtype)}
    y = x.float()
    y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    slope = 0.5 * (1.0 + torch.erf(kept * math.sqrt(0.5))) + kept * torch.exp(-0.5 * kept * kept) / math.sqrt(2 * math.pi)
    return {"y": y.to(x.dtype), "dx": (s["dy"].float() * slope).to(x.dtype)}


# -------------------------------------------------------------------------------------------- the definition
def exact(case, seed):
    """The operators' definitions in 64 bits, one sequence and key head at a time."""
    if work(case)["flops"] > 4e12:
        return None
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    if case["op"] in ("attn", "bias"):
        return _exact_attention(case, s)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    return _exact_act8(case, s)


def _exact_table(count, distance, both, low, high):
    """Buckets of the relative positions low .. high by whole-number comparisons: the k-th far bucket starts at the
    first n with n^m >= near^(m-k) distance^k."""
    m = count // 2 if both else count
    near = m // 2
    wide = m - near
    first = []
    for k in range(wide):
        n = near
        while n ** wide < near ** (wide - k) * distance ** k:
            n += 1
        first.append(n)
    got = []
    for rel in range(low, high + 1):
        n = abs(rel) if both else max(-rel, 0)
        n = min(n, distance)
        b = n if n < near else near - 1 + sum(f <= n for f in first)
        got.append(b + (m if both and rel > 0 else 0))
    return torch.tensor(got, device="cuda")


def _exact_attention(c, s):
    nq, nk = _lengths(c)
    d, group = c["dim"], c["heads"] // c["kv_heads"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    train = c["mode"] == "train"
    out = {"o": torch.zeros_like(q)}
    if train:
        do = s["dout"].double()
        out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    if c["op"] == "bias":
        table = s["table"].double()
        far = max(nk)
        of = _exact_table(c["buckets"], c["distance"], not c["causal"], -far, far)
        if train:
            out["dtable"] = torch.zeros_like(table)
    a = b = 0
    for m, n in zip(nq, nk):
        rel = torch.arange(n, device="cuda")[None, :] - (torch.arange(m, device="cuda")[:, None] + n - m)
        for h in range(c["kv_heads"]):
            kk, vv = k[b:b + n, h], v[b:b + n, h]
            heads = slice(h * group, (h + 1) * group)
            qq = q[a:a + m, heads].transpose(0, 1).reshape(group * m, d)
            z = (qq @ kk.T / math.sqrt(d)).reshape(group, m, n)
            if c["op"] == "bias":
                z = z + table[of[rel + far]][:, :, heads].permute(2, 0, 1)
            if c["causal"]:
                z = torch.where(rel > 0, float("-inf"), z)
            w = torch.softmax(z, -1)
            w = torch.where(torch.isnan(w), 0.0, w).reshape(group * m, n)
            o = w @ vv
            out["o"][a:a + m, heads] = o.reshape(group, m, d).transpose(0, 1)
            if train:
                g = do[a:a + m, heads].transpose(0, 1).reshape(group * m, d)
                dz = w * (g @ vv.T - (g * o).sum(1, keepdim=True))
                out["dv"][b:b + n, h] = w.T @ g
                out["dk"][b:b + n, h] = dz.T @ qq / math.sqrt(d)
                out["dq"][a:a + m, heads] = (dz @ kk / math.sqrt(d)).reshape(group, m, d).transpose(0, 1)
                if c["op"] == "bias":
                    out["dtable"][:, heads].index_add_(0, of[rel + far].reshape(-1),
                                                       dz.reshape(group, -1).T.contiguous())
        a, b = a + m, b + n
    return out


def _exact_norm(c, s):
    width = c["width"]
    p = {n: None if s.get(n) is None else s[n].double()
         for n in ("x", "branch", "pre_weight", "post_weight", "pre_bias", "post_bias", "gate", "dy", "dn")}
    zero, one = torch.zeros((), dtype=torch.float64, device="cuda"), torch.ones((), dtype=torch.float64, device="cuda")
    layer = c["kind"] == "layer"
    mean = (lambda z: z.sum(1, keepdim=True) / width) if layer else (lambda z: zero)
    f = p["branch"] - mean(p["branch"])
    fs = torch.sqrt((f ** 2).sum(1, keepdim=True) / width + EPS)
    gate = one if p["gate"] is None else p["gate"]
    u = f / fs * p["post_weight"] + (p["post_bias"] if layer else zero)
    y = c["scale"] * p["x"] + gate * u
    z = y - mean(y)
    zs = torch.sqrt((z ** 2).sum(1, keepdim=True) / width + EPS)
    out = {"y": y, "n": z / zs * p["pre_weight"] + (p["pre_bias"] if layer else zero)}
    if c["mode"] != "train":
        return out
    g = p["dn"] * p["pre_weight"]
    g = g / zs - z * (g * z).sum(1, keepdim=True) / (width * zs ** 3)
    g = p["dy"] + g - mean(g)
    out["dx"] = c["scale"] * g
    out["dpre_weight"] = (p["dn"] * z / zs).sum(0)
    e = g * gate
    out["dpost_weight"] = (e * f / fs).sum(0)
    if layer:
        out["dpre_bias"], out["dpost_bias"] = p["dn"].sum(0), e.sum(0)
    if p["gate"] is not None:
        out["dgate"] = (g * u).sum(0) if p["gate"].dim() == 1 else g * u
    e = e * p["post_weight"]
    e = e / fs - f * (e * f).sum(1, keepdim=True) / (width * fs ** 3)
    out["dbranch"] = e - mean(e)
    return out


def _exact_act8(c, s):
    x = s["x"].double()
    flat = x.reshape(-1)
    blocks = torch.cat([flat, flat.new_zeros(-flat.numel() % BLOCK)]).reshape(-1, BLOCK)
    top = blocks.abs().amax(1, keepdim=True)
    power = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))       # then put right where the logarithm rounds
    power = power + (torch.exp2(power + 1) <= top).double() - ((torch.exp2(power) > top) & (top > 0)).double()
    step = torch.exp2(power.clamp(min=-126) - 6)
    kept = (torch.round(blocks / step).clamp(-127, 127) * step).reshape(-1)[:flat.numel()].reshape(x.shape)
    if c["mode"] == "store":
        return {"values": kept}
    density = torch.exp(-kept ** 2 / 2) / math.sqrt(2 * math.pi)
    return {"y": x * torch.special.ndtr(x), "dx": s["dy"].double() * (torch.special.ndtr(kept) + kept * density)}

"""Cases of the training and serving operators that stand beside the fused score head: attention over a sorted edge list with a learned bias by
length buckets and counter-based dropout, the norms around a block fused with its gate and residual, and dropout of whole irreps channels.

``run`` computes a case in plain torch operations, or, with ``own`` set, through the package.  Sizes are the score head's and the feature
extractors' (irreps of lmax 1 to 3, 4 heads, 20 or 1 000 poses, 16 384-point scenes) or generic."""
import math

import torch

own = False

IRREPS = {1: "64x0e+32x1e", 2: "64x0e+32x1e+16x2e", 3: "64x0e+32x1e+16x2e+8x3e"}
HEAD_DIM = {1: 40, 2: 60, 3: 74}              # channels of one of four heads: 16x0e+8x1e(+4x2e(+2x3e))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST_EDGES = 1_970_000                        # the score head's edges of one step: 1 000 poses x 103 query points
MOST_ROWS = 103_000
SLOPE, ACT_NORM = 0.2, 1.531320475574866      # smooth leaky ReLU and its second-moment constant
EPS = 1e-5
LONGEST = 20.0                                # the largest finite radius of the score head's graphs


# ---- cases ----------------------------------------------------------------------------------------------------------------------------------

def _attention(name, dtype, nodes, edges, lmax=2, train=True, buckets=32, drop=0.1, spread="even", masked=0.0, heads=4, k=16, d=None):
    return {"name": name, "op": "attention", "dtype": dtype, "nodes": nodes, "edges": edges, "heads": heads, "k": k, "d": d or HEAD_DIM[lmax],
            "train": train, "buckets": buckets, "drop": drop if train else 0.0, "spread": spread, "masked": masked}


def _norm(name, dtype, rows, irreps, train=True, groups=1, drop=0.1, post=True, nxt=True):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "irreps": irreps, "train": train, "groups": groups,
            "drop": drop if train else 0.0, "post": post, "next": nxt}


def _dropout(name, dtype, rows, irreps, drop=0.1):
    return {"name": name, "op": "dropout", "dtype": dtype, "rows": rows, "irreps": irreps, "train": True, "drop": drop}


def listed():
    return [
        # 20 poses x 2 static key points of a picking head, one evaluation: latency
        _attention("attn_serve_pick", "f32", 40, 797, train=False),
        # a placing head in half precision, all 1 000 poses x 103 query points of one evaluation
        _attention("attn_serve_poses_f16", "f16", MOST_ROWS, MOST_EDGES, train=False),
        # a training step on one demonstration: 20 noised poses x 103 query points
        _attention("attn_train_demo", "f32", 2_060, 39_411),
        # a training step over as many poses as the sampler carries
        _attention("attn_train_poses", "f32", MOST_ROWS, MOST_EDGES),
        # a feature extractor's finest level at lmax 3: crowded and empty neighbourhoods side by side, masked edges
        _attention("attn_train_scene_bf16", "bf16", 16_384, 499_979, lmax=3, spread="skewed", masked=0.05),
        # a handful of points that see a whole scene (the all-pairs scale): few rows, long ones
        _attention("attn_train_long_f16", "f16", 7, 300_007, lmax=1, buckets=16),
        # between two blocks of a picking head, one evaluation: latency
        _norm("norm_serve_pick", "f32", 40, IRREPS[2], train=False),
        # between two blocks in training, a gate for each pose's time
        _norm("norm_train_poses", "f32", MOST_ROWS, IRREPS[2], groups=1_000),
        # a scene's finest level at lmax 3 with a learned scale for each channel
        _norm("norm_train_scene_f16", "f16", 16_384, IRREPS[3], groups=1),
        # the width of the feed-forward network, a gate for each node, on the pooled scene
        _norm("norm_train_wide_bf16", "bf16", 3_277, "192x0e+96x1e+48x2e", groups=3_277),
        # dropout behind the projection of the attention, forward and backward
        _dropout("drop_train_poses", "f32", MOST_ROWS, IRREPS[2]),
        # the same on a pooled scene at lmax 1
        _dropout("drop_train_pooled_bf16", "bf16", 3_277, IRREPS[1]),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _some_irreps(rng):
    kind = rng.random()
    if kind < 0.6:
        return IRREPS[rng.choice((1, 2, 3))]
    if kind < 0.8:
        return "192x0e+96x1e+48x2e"
    return "+".join("%dx%de" % (_between(rng, 2, 70), l) for l in range(rng.randint(1, 4)))


def _width(irreps):
    return sum(m * (2 * l + 1) for m, l in _blocks(irreps))


def draw(rng):
    dtype = rng.choice(("f32", "f32", "f16", "bf16"))
    op = rng.choice(("attention", "attention", "attention", "norm", "norm", "dropout"))
    if op == "attention":
        nodes = _between(rng, 1, MOST_ROWS)
        generic = rng.random() < 0.3
        heads, k, d = (rng.choice((1, 2, 3, 8)), rng.randint(1, 32), rng.randint(1, 80)) if generic else (4, 16, HEAD_DIM[rng.choice((1, 2, 3))])
        most = MOST_EDGES * 4 * 76 // (heads * (k + d))          # no more bytes than the largest listed case
        edges = min(MOST_EDGES, most, max(16, int(nodes * math.exp(rng.uniform(math.log(2.0), math.log(60.0))))), 400_000 if dtype != "f32" and generic else MOST_EDGES)
        if nodes < 64 and rng.random() < 0.5:
            edges = _between(rng, 64, 300_000)
        edges = min(edges, most)
        return _attention(None, dtype, nodes, edges, d=d, train=rng.random() < 0.7, buckets=rng.choice((0, 2, 16, 32, 50)), drop=rng.choice((0.0, 0.1, 0.35)),
                          spread=rng.choice(("even", "skewed")), masked=rng.choice((0.0, 0.0, 0.1)), heads=heads, k=k) | {"name": "drawn"}
    irreps = _some_irreps(rng)
    rows = _between(rng, 1, MOST_ROWS * 240 // max(240, _width(irreps)))
    if op == "dropout":
        return _dropout("drawn", dtype, rows, irreps, drop=rng.choice((0.05, 0.1, 0.5)))
    groups = rng.choice((0, 1, rows, max(1, rows // 103)))
    rows = rows if groups in (0, 1, rows) else 103 * groups
    return _norm("drawn", dtype, rows, irreps, train=rng.random() < 0.7, groups=groups, drop=rng.choice((0.0, 0.1)), post=rng.random() < 0.7, nxt=rng.random() < 0.8)


def _blocks(irreps):
    return [(int(t.split("x")[0]), int(t.split("x")[1][:-1])) for t in irreps.split("+")]


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, dtype=t, mean=0.0, std=1.0, grad=case["train"]):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype if dtype != torch.bfloat16 else torch.float32).mul_(std).add_(mean).to(dtype).requires_grad_(grad)

    s = {"case": dict(case), "rng": torch.tensor([seed * 1_000_003 + 17, seed % 97], device=dev)}
    if case["op"] == "attention":
        E, N, H = case["edges"], case["nodes"], case["heads"]
        u = torch.rand(E, generator=g, device=dev, dtype=torch.float64)
        s["edge_dst"] = ((u ** 3 if case["spread"] == "skewed" else u) * N).long().clamp_(max=N - 1).sort().values
        s["alpha"], s["value"] = normal(E, H, case["k"]), normal(E, H, case["d"])
        s["alpha_dot"] = normal(H, case["k"], dtype=torch.float32, std=(6.0 / (case["k"] + 1)) ** 0.5 / 3 ** 0.5)
        # soft cut-offs: most edges far inside the radius (logit 0), the outer fifth falling off to log 1e-12
        r = torch.rand(E, generator=g, device=dev) ** (1 / 3)
        s["edge_length"] = r * LONGEST
        logits = torch.where(r < 0.8, torch.zeros_like(r), (1 - (r - 0.8) / 0.2).clamp(min=0).pow(2).clamp(min=1e-12).log())
        if case["masked"]:
            logits = torch.where(torch.rand(E, generator=g, device=dev) < case["masked"], torch.full_like(r, -math.inf), logits)
        s["edge_logits"] = logits.requires_grad_(case["train"])
        if case["buckets"]:
            s["boundaries"] = torch.linspace(0.0, LONGEST, case["buckets"] + 1, device=dev)[1:-1].contiguous()
            s["table"] = normal(case["buckets"], H, dtype=torch.float32, std=0.5)
        if case["train"]:
            s["grad"] = normal(N, H, case["d"], grad=False)
        if own:
            from diffusion_edf_amd.edge_attention import EdgeSegments
            s["segments"] = EdgeSegments(s["edge_dst"], N)
        return s
    blocks = _blocks(case["irreps"])
    R, W, C = case["rows"], _width(case["irreps"]), sum(m for m, _ in blocks)
    scalars = blocks[0][0] if blocks[0][1] == 0 else 0
    s["x"] = normal(R, W, mean=0.3)
    if case["train"]:
        s["grad_h"] = normal(R, W, grad=False)
    if case["op"] == "dropout":
        return s
    s["y"] = normal(R, W, mean=-0.2, std=2.0)
    if case["groups"]:
        s["gate"] = normal(case["groups"], C, mean=0.5, std=0.3, dtype=torch.float32 if case["groups"] == 1 else t)
    for which in ("post", "next"):
        if case[which]:
            s[which + "_weight"] = normal(C, dtype=torch.float32, mean=1.0, std=0.2)
            s[which + "_bias"] = normal(scalars, dtype=torch.float32, std=0.2)
    if case["train"] and case["next"]:
        s["grad_z"] = normal(R, W, grad=False)
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------------------------------

def _philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10: counters and keys are int64 tensors (or numbers) that hold 32-bit words; products wrap at 64 bits, which keeps every bit."""
    word = 0xFFFFFFFF
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & word) ^ c1 ^ k0, b & word, ((a >> 32) & word) ^ c3 ^ k1, a & word
        k0, k1 = (k0 + 0x9E3779B9) & word, (k1 + 0xBB67AE85) & word
    return torch.stack([c0, c1, c2, c3], -1)


def _keep(rows, columns, p, rng, first):
    """(rows, columns) factors 0 or 1/(1-p): word column % 4 of the counter (row, first + column // 4, offset)"""
    at = torch.arange(rows, device=rng.device)[:, None]
    group = first + torch.arange(-(-columns // 4), device=rng.device)[None, :]
    at, group = torch.broadcast_tensors(at, group)
    word = 0xFFFFFFFF
    drawn = _philox(at, group, rng[1] & word, (rng[1] >> 32) & word, rng[0] & word, (rng[0] >> 32) & word)
    return (drawn.flatten(1)[:, :columns] >= int(p * 2.0 ** 32)).float() / (1.0 - p)


def _slots(dst, rows):
    """each row stands several times where rows are few, and its edges take turns, so that additions into a row do not queue up"""
    ways = max(1, min(256, 262_144 // rows))
    return ways, dst * ways + torch.arange(len(dst), device=dst.device) % ways if ways > 1 else dst


def _row_sums(x, dst, rows):
    ways, at = _slots(dst, rows)
    return torch.zeros(rows * ways, *x.shape[1:], dtype=x.dtype, device=x.device).index_add(0, at, x).view(rows, ways, *x.shape[1:]).sum(1)


def _to_edges(x, dst):
    ways, at = _slots(dst, len(x))
    return x[:, None].expand(len(x), ways, x.shape[1]).reshape(-1, x.shape[1]).index_select(0, at)


def _plain_attention(s):
    c = s["case"]
    a, v, w, dst = s["alpha"].float(), s["value"].float(), s["alpha_dot"], s["edge_dst"]
    E, N, H = c["edges"], c["nodes"], c["heads"]
    act = ((1 + SLOPE) / 2 * a + (1 - SLOPE) / 2 * a * (2 * torch.sigmoid(a) - 1)) * ACT_NORM
    logit = (act * w).sum(-1).double() + s["edge_logits"].double()[:, None]
    if c["buckets"]:
        bucket = torch.bucketize(s["edge_length"], s["boundaries"], right=True)
        logit = logit + _to_edges(s["table"].double(), bucket)
    live = logit > -math.inf
    ways, at = _slots(dst, N)
    top = torch.full((N * ways, H), -math.inf, dtype=torch.float64, device=dst.device).scatter_reduce(0, at[:, None].expand(E, H), logit.detach(), "amax")
    e = torch.where(live, torch.where(live, logit - _to_edges(top.view(N, ways, H).amax(1), dst), 0.0).exp(), 0.0)
    total = _row_sums(e, dst, N)
    p = (e / _to_edges(torch.where(total > 0, total, 1.0), dst)).float()
    if c["drop"]:
        p = p * _keep(E, H, c["drop"], s["rng"], 0)
    wide = torch.float64 if E > 256 * N else torch.float32          # long rows are summed in 64 bits
    return _row_sums((p[..., None] * v).to(wide), dst, N).to(s["value"].dtype)


def _per_channel(values, blocks):
    """(..., channels) -> (..., width): each channel's value on its 2l+1 components"""
    parts, at = [], 0
    for m, l in blocks:
        part = values[..., at:at + m]
        parts.append(part[..., None].expand(*part.shape, 2 * l + 1).flatten(-2))
        at += m
    return torch.cat(parts, -1)


def _plain_layer_norm(x, blocks, weight, bias):
    parts, at = [], 0
    for m, l in blocks:
        f = x[:, at:at + m * (2 * l + 1)]
        at += m * (2 * l + 1)
        if l == 0:
            f = f - f.mean(-1, keepdim=True)
        parts.append(f * (f.square().mean(-1, keepdim=True) + EPS).rsqrt())
    z = torch.cat(parts, -1) * _per_channel(weight, blocks)
    return torch.cat([z[:, :len(bias)] + bias, z[:, len(bias):]], -1) if len(bias) else z


def _plain_norm(s):
    c, blocks = s["case"], _blocks(s["case"]["irreps"])
    t, R, C = s["x"].dtype, s["case"]["rows"], sum(m for m, _ in blocks)
    u = s["y"].float()
    if c["post"]:
        u = _plain_layer_norm(u, blocks, s["post_weight"], s["post_bias"])
    if c["drop"]:
        u = u * _per_channel(_keep(R, C, c["drop"], s["rng"], 1 << 16), blocks)
    if c["groups"]:
        G = c["groups"]
        u = (u.view(G, R // G, -1) * _per_channel(s["gate"].float(), blocks)[:, None]).view(R, -1)
    h = s["x"].float() + 0.5 * u
    z = _plain_layer_norm(h, blocks, s["next_weight"], s["next_bias"]).to(t) if c["next"] else None
    return h.to(t), z


def _plain_dropout(s):
    c, blocks = s["case"], _blocks(s["case"]["irreps"])
    keep = _keep(c["rows"], sum(m for m, _ in blocks), c["drop"], s["rng"], 1 << 16)
    return (s["x"].float() * _per_channel(keep, blocks)).to(s["x"].dtype)


# ---- one pass -------------------------------------------------------------------------------------------------------------------------------

def _own_attention(s):
    from diffusion_edf_amd.edge_attention import edge_attention
    c = s["case"]
    bias = {"edge_length": s["edge_length"], "bias_boundaries": s["boundaries"], "bias_table": s["table"]} if c["buckets"] else {}
    return edge_attention(s["alpha"], s["value"], s["alpha_dot"], s["segments"], edge_logits=s["edge_logits"], dropout=c["drop"], rng=s["rng"], **bias)


def _own_norm(s):
    from diffusion_edf_amd.layer_norm import norm_gate_residual
    c = s["case"]
    return norm_gate_residual(s["x"], s["y"], c["irreps"], scale=0.5, gate=s.get("gate"), post_weight=s.get("post_weight"), post_bias=s.get("post_bias"),
                              dropout=c["drop"], rng=s["rng"], next_weight=s.get("next_weight"), next_bias=s.get("next_bias"), eps=EPS)


def _own_dropout(s):
    from diffusion_edf_amd.drop import equivariant_dropout
    return equivariant_dropout(s["x"], s["case"]["irreps"], s["case"]["drop"], s["rng"])


LEAVES = {"attention": ("alpha", "value", "alpha_dot", "edge_logits", "table"),
          "norm": ("x", "y", "gate", "post_weight", "post_bias", "next_weight", "next_bias"), "dropout": ("x",)}


def run(state):
    c = state["case"]
    forward = {"attention": (_plain_attention, _own_attention), "norm": (_plain_norm, _own_norm), "dropout": (_plain_dropout, _own_dropout)}[c["op"]][bool(own)]
    if not c["train"]:
        with torch.no_grad():
            out = forward(state)
        return {"out": out} if c["op"] != "norm" else {"h": out[0], "z": out[1]}
    out = forward(state)
    leaves = [k for k in LEAVES[c["op"]] if k in state and state[k].numel()]
    if c["op"] == "norm":
        outs = {"h": out[0], "z": out[1]} if c["next"] else {"h": out[0]}
        cotangents = [state["grad_h"]] + ([state["grad_z"]] if c["next"] else [])
    else:
        outs = {"out": out}
        cotangents = [state["grad"] if c["op"] == "attention" else state["grad_h"]]
    grads = torch.autograd.grad(list(outs.values()), [state[k] for k in leaves], cotangents)
    return {k: v.detach() for k, v in outs.items()} | {"d_" + k: v for k, v in zip(leaves, grads)}


# ---- the least that a pass reads, writes and computes ------------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "attention":
        E, N, H, K, D = (case[k] for k in ("edges", "nodes", "heads", "k", "d"))
        row, B = H * (K + D) * size, case["buckets"]
        read = E * (row + 4 + 4 + (4 if B else 0)) + (H * K + B * H) * 4
        written = N * H * D * size
        flops = E * H * (2 * D + 12 * K)
        if case["train"]:
            read += N * H * D * size
            written += E * (row + 4) + (H * K + B * H) * 4
            flops += E * H * (4 * D + 24 * K)
        return {"bytes": read + written, "flops": flops}
    R, W = case["rows"], _width(case["irreps"])
    C = sum(m for m, _ in _blocks(case["irreps"]))
    if case["op"] == "dropout":
        return {"bytes": 4 * R * W * size, "flops": 2 * R * W}
    rows = 2 + 1 + (1 if case["next"] else 0)
    params = case["groups"] * C * size + (case["post"] + case["next"]) * C * 4
    if case["train"]:
        rows += 2 + 1 + (1 if case["next"] else 0)
        params *= 2
    return {"bytes": rows * R * W * size + params, "flops": R * W * (40 if case["train"] else 15)}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------------------

def _exact_words(rows, columns, rng, first):
    """Philox4x32-10 again, with the 32 x 32 bit products put together from 16-bit halves"""
    def product(x, m):
        low, high = x * (m & 0xFFFF), x * (m >> 16)
        return (high + (low >> 16)) >> 16, (low + ((high & 0xFFFF) << 16)) & 0xFFFFFFFF

    seed, offset = (int(v) for v in rng.tolist())
    quads = (columns + 3) // 4
    flat = torch.arange(rows * quads, device=rng.device)
    x = [flat // quads, first + flat % quads, torch.full_like(flat, offset & 0xFFFFFFFF), torch.full_like(flat, (offset >> 32) & 0xFFFFFFFF)]
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for i in range(10):
        h0, l0 = product(x[0], 0xD2511F53)
        h1, l1 = product(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ ((key[0] + i * 0x9E3779B9) & 0xFFFFFFFF), l1, h0 ^ x[3] ^ ((key[1] + i * 0xBB67AE85) & 0xFFFFFFFF), l0]
    return torch.stack(x, 1).view(rows, 4 * quads)[:, :columns]


def _exact_attention(s):
    c = s["case"]
    dst, H = s["edge_dst"], c["heads"]
    a, v, w = (s[k].detach().double() for k in ("alpha", "value", "alpha_dot"))
    sig = 1 / (1 + torch.exp(-a))
    act = ACT_NORM * (0.6 * a + 0.4 * a * (2 * sig - 1))
    slope = ACT_NORM * (0.6 + 0.4 * (2 * sig - 1) + 0.8 * a * sig * (1 - sig))
    logit = torch.einsum("ehk,hk->eh", act, w) + s["edge_logits"].detach().double()[:, None]
    if c["buckets"]:
        bucket = (s["edge_length"][:, None] >= s["boundaries"][None, :]).sum(1) if c["buckets"] > 1 else torch.zeros_like(dst)
        logit = logit + s["table"].detach().double()[bucket]
    ends = torch.searchsorted(dst, torch.arange(c["nodes"], device=dst.device), right=True)
    first = torch.cat([ends.new_zeros(1), ends[:-1]])

    def per_row(x):                       # sums over the edges of a row: differences of running sums
        run = torch.cat([x.new_zeros(1, *x.shape[1:]), x.cumsum(0)])
        return run[ends] - run[first]

    raw = torch.exp(logit - logit.amax())          # (the logits of a case span a few dozen: nothing underflows in 64 bits)
    total = torch.zeros(c["nodes"], H, dtype=torch.float64, device=dst.device).index_add_(0, dst, raw)
    p = raw / total.clamp(min=1e-300)[dst]
    m = (_exact_words(c["edges"], H, s["rng"], 0) >= int(c["drop"] * 2.0 ** 32)).double() / (1 - c["drop"]) if c["drop"] else torch.ones_like(p)
    found = {"out": per_row((p * m)[..., None] * v)}
    if c["train"]:
        up = s["grad"].double()[dst]
        found["d_value"] = (p * m)[..., None] * up
        dp = m * (up * v).sum(-1)
        del up
        ds = p * (dp - torch.zeros(c["nodes"], H, dtype=torch.float64, device=dst.device).index_add_(0, dst, p * dp)[dst])
        found |= {"d_alpha": ds[..., None] * w * slope, "d_alpha_dot": (ds[..., None] * act).sum(0), "d_edge_logits": ds.sum(1)}
        if c["buckets"]:
            found["d_table"] = torch.zeros(c["buckets"], H, dtype=torch.float64, device=dst.device).index_add_(0, bucket, ds)
    return found


def _exact_rows(case, s):
    """norm and dropout: values and gradients of each block, written out"""
    blocks = _blocks(case["irreps"])
    of_element = torch.cat([torch.full((m * (2 * l + 1),), i) for i, (m, l) in enumerate(blocks)]).to(s["x"].device)
    channel, base = [], 0
    for m, l in blocks:
        channel.append(base + torch.arange(m * (2 * l + 1)) // (2 * l + 1))
        base += m
    channel = torch.cat(channel).to(s["x"].device)
    R, C = case["rows"], base
    keep = (_exact_words(R, C, s["rng"], 1 << 16) >= int(case["drop"] * 2.0 ** 32)).double()[:, channel] / (1 - case["drop"]) if case["drop"] else 1.0
    x = s["x"].detach().double()
    if case["op"] == "dropout":
        return {"out": x * keep, "d_x": s["grad_h"].double() * keep}
    scalar = torch.tensor([l == 0 for _, l in blocks], device=x.device)[of_element].double()
    member = torch.nn.functional.one_hot(of_element, len(blocks)).double()
    mean_of = lambda f: (f @ (member / member.sum(0))) @ member.T          # noqa: E731  a block's mean, on each of its elements
    to_channel = torch.nn.functional.one_hot(channel, C).double()

    def unit(f):
        f = f - scalar * mean_of(f)
        r = (mean_of(f * f) + EPS) ** -0.5
        return f * r, r

    def unit_back(g, n, r):
        g = r * (g - n * mean_of(g * n))
        return g - scalar * mean_of(g)

    def get(name):
        return s[name].detach().double() if name in s else None

    scalars = int(scalar.sum())
    y, gate = get("y"), get("gate")
    G = case["groups"]
    gain = 0.5 * keep * (gate[:, channel].repeat_interleave(R // G, 0) if G else 1.0)
    if case["post"]:
        n1, r1 = unit(y)
        u = n1 * get("post_weight")[channel]
        u[:, :scalars] += get("post_bias")
    else:
        u = y
    h = x + gain * u
    found = {"h": h, "z": None}
    if case["next"]:
        n2, r2 = unit(h)
        z = n2 * get("next_weight")[channel]
        z[:, :scalars] += get("next_bias")
        found["z"] = z
    if not case["train"]:
        return found
    up = s["grad_h"].double()
    if case["next"]:
        gz = s["grad_z"].double()
        found |= {"d_next_weight": (gz * n2).sum(0) @ to_channel}
        if scalars:
            found["d_next_bias"] = gz[:, :scalars].sum(0)
        up = up + unit_back(gz * get("next_weight")[channel], n2, r2)
    found["d_x"] = up
    if G:
        found["d_gate"] = (up * 0.5 * keep * u @ to_channel).view(G, R // G, C).sum(1)
    du = gain * up
    if case["post"]:
        found["d_post_weight"] = (du * n1).sum(0) @ to_channel
        if scalars:
            found["d_post_bias"] = du[:, :scalars].sum(0)
        du = unit_back(du * get("post_weight")[channel], n1, r1)
    found["d_y"] = du
    if not case["next"]:
        found.pop("z")
    return found


def exact(case, seed):
    global own
    was, own = own, False          # the inputs alone, without the package's plan
    try:
        s = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        return _exact_attention(s) if case["op"] == "attention" else _exact_rows(case, s)

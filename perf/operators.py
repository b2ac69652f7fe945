"""The mixture-of-experts operators of libfm_b200 as measured work: 4-bit projections, routing, experts' products.

Every case is one call of fm_proj_forward, fm_moe_route or fm_moe_experts.  With `own` false, run() computes the same
numbers with elementary torch operations; with `own` true it makes the library's call on the same tensors.
"""
import math
import sys
from pathlib import Path

import torch

own = False

GROUP = 64            # inputs that share a scale and a bias in the 4-bit affine format
SOFTMAX, SIGMOID = 0, 1


def listed():
    return [
        # -- projections that share their input (y_i = W_i x) --
        # decode, one token: q | gate, k and v of a full-attention layer
        {"name": "proj 1 token q+k+v", "op": "proj", "n": 1, "k": 4096, "outs": "16384,512,512"},
        # a small router with its shared-expert gate for a handful of sequences; odd sizes
        {"name": "proj 7 tokens small odd", "op": "proj", "n": 7, "k": 1088, "outs": "100,1"},
        # a ragged prompt through the four input projections of a GatedDeltaNet layer
        {"name": "proj 300 tokens qkv+z+b+a", "op": "proj", "n": 300, "k": 4096, "outs": "12288,8192,64,64"},
        # a long prompt through an output projection
        {"name": "proj 4096 tokens", "op": "proj", "n": 4096, "k": 8192, "outs": "4096"},
        # -- routing --
        # decode, one token, many experts, with the shared expert's gate in the last column
        {"name": "route 1 of 512", "op": "route", "n": 1, "experts": 512, "top": 10, "score": SOFTMAX, "bias": False, "groups": 1,
         "top_groups": 1, "group_best": 1, "renorm": True, "scale": 1.0, "shared": True, "masked": 0.0},
        # a ragged prompt with some experts switched off
        {"name": "route 333 of 100 masked", "op": "route", "n": 333, "experts": 100, "top": 6, "score": SOFTMAX, "bias": False, "groups": 5,
         "top_groups": 2, "group_best": 1, "renorm": False, "scale": 16.0, "shared": False, "masked": 0.3},
        # a long prompt: sigmoid scores, a bias for balance, groups of experts
        {"name": "route 8192 of 256 groups", "op": "route", "n": 8192, "experts": 256, "top": 8, "score": SIGMOID, "bias": True, "groups": 8,
         "top_groups": 4, "group_best": 2, "renorm": True, "scale": 2.5, "shared": False, "masked": 0.0},
        # -- experts --
        # decode, one token
        {"name": "experts 1 token of 512", "op": "experts", "n": 1, "hidden": 4096, "inter": 1024, "experts": 512, "held": 512, "first": 0,
         "top": 10},
        # a few tokens of a tiny model
        {"name": "experts 3 tokens tiny", "op": "experts", "n": 3, "hidden": 256, "inter": 192, "experts": 8, "held": 8, "first": 0, "top": 2},
        # batched decode: nearly every expert is used, by one or two tokens each
        {"name": "experts 48 tokens of 512", "op": "experts", "n": 48, "hidden": 4096, "inter": 1024, "experts": 512, "held": 512, "first": 0,
         "top": 10},
        # a ragged prompt on a rank that holds half of the experts
        {"name": "experts 501 tokens half held", "op": "experts", "n": 501, "hidden": 2048, "inter": 704, "experts": 60, "held": 30, "first": 15,
         "top": 4},
        # a long prompt
        {"name": "experts 4096 tokens of 512", "op": "experts", "n": 4096, "hidden": 4096, "inter": 1024, "experts": 512, "held": 512,
         "first": 0, "top": 10},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["proj", "proj", "route", "experts", "experts"])
    if op == "proj":
        k = GROUP * _spread(rng, 1, 128)
        outs = [_spread(rng, 1, 16384) for _ in range(rng.randint(1, 4))]
        while sum(outs) * k > 4096 * 20480:  # a matrix set of a layer, at most
            outs = [max(1, o // 2) for o in outs]
        most = max(1, min(4096, int(4096 * 8192 * 4096 / (sum(outs) * k))))
        return {"op": "proj", "n": _spread(rng, 1, most), "k": k, "outs": ",".join(str(o) for o in outs)}
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 5, 8])
        experts = groups * _spread(rng, 4, 512 // groups)
        top_groups = rng.randint(1, groups)
        return {"op": "route", "n": _spread(rng, 1, 8192), "experts": experts, "top": min(_spread(rng, 1, 16), experts // groups * top_groups),
                "score": rng.choice([SOFTMAX, SIGMOID]), "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                "group_best": rng.choice([1, 2]), "renorm": rng.random() < 0.5, "scale": rng.choice([1.0, 2.5]),
                "shared": rng.random() < 0.5, "masked": rng.choice([0.0, 0.0, 0.2])}
    hidden, inter, experts = GROUP * _spread(rng, 2, 64), GROUP * _spread(rng, 1, 16), _spread(rng, 4, 512)
    top = min(_spread(rng, 1, 12), experts)
    held = experts if rng.random() < 0.6 else max(1, experts // 2)
    return {"op": "experts", "n": _spread(rng, 1, 4096 * 10 // max(10, top)), "hidden": hidden, "inter": inter, "experts": experts, "held": held,
            "first": rng.randint(0, experts - held), "top": top}


# ---- inputs -------------------------------------------------------------------------------------
def _matrix(gen, *shape, fan):
    """A 4-bit affine matrix [..., out, in]: words (eight nibbles each, lowest first), scales and biases of bf16.  The
    weights come out about N(0, 1 / fan), as trained ones of that fan-in are."""
    *lead, out, k = shape
    w = torch.randint(-2 ** 31, 2 ** 31, (*lead, out, k // 8), generator=gen, device="cuda", dtype=torch.int32)
    step = (0.5 + torch.rand((*lead, out, k // GROUP), generator=gen, device="cuda")) * (0.217 / math.sqrt(fan))
    scales = step.bfloat16()
    offset = 0.5 * torch.randn(step.shape, generator=gen, device="cuda")
    return w, scales, (-(7.5 + offset) * scales.float()).bfloat16()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    n, s = case["n"], {"case": case}
    if case["op"] == "proj":
        k, outs = case["k"], [int(o) for o in case["outs"].split(",")]
        s["x"] = rnd(n, k)
        s["w"] = [_matrix(gen, o, k, fan=k) for o in outs]
        s["y"] = [torch.empty((n, o), device="cuda") for o in outs]
    elif case["op"] == "route":
        e, slots = case["experts"], case["top"] + int(case["shared"])
        logits = 1.5 * rnd(n, e + int(case["shared"]))
        if case["masked"]:
            off = torch.rand((n, e), generator=gen, device="cuda") < case["masked"]
            logits[:, :e].masked_fill_(off, -math.inf)
        s["logits"] = logits
        s["bias"] = 0.05 * rnd(e) if case["bias"] else None
        s["ids"] = torch.empty((n, slots), device="cuda", dtype=torch.int32)
        s["weights"] = torch.empty((n, slots), device="cuda")
    else:
        h, i, held, top = case["hidden"], case["inter"], case["held"], case["top"]
        # some experts are more popular than others, as in a trained router
        logits = rnd(n, case["experts"]) + 0.4 * rnd(case["experts"])
        best = torch.sort(logits, dim=1, descending=True, stable=True)
        s["ids"] = best.indices[:, :top].to(torch.int32).contiguous()
        s["weights"] = torch.softmax(best.values[:, :top], dim=1).contiguous()
        s["x"], s["residual"] = rnd(n, h), rnd(n, h)
        s["norm_w"] = (1.0 + 0.1 * rnd(h)).bfloat16()
        s["gate"], s["up"], s["down"] = (_matrix(gen, held, *d, fan=d[1]) for d in ((i, h), (i, h), (h, i)))
        s["h_out"], s["h_norm"] = torch.empty((n, h), device="cuda"), torch.empty((n, h), device="cuda")
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _weights(w, scales, biases):
    """The matrix that words, scales and biases stand for, in 32 bits."""
    shifts = torch.arange(0, 32, 4, device=w.device, dtype=torch.int32)
    q = ((w.unsqueeze(-1) >> shifts) & 15).reshape(*scales.shape, GROUP).float()
    return (q * scales.float().unsqueeze(-1) + biases.float().unsqueeze(-1)).flatten(-2)


def _route(s):
    c = s["case"]
    e, top, groups = c["experts"], c["top"], c["groups"]
    x = s["logits"][:, :e].double()  # selection compares values next to each other: in 64 bits
    there = x > -math.inf
    score = torch.softmax(x, dim=1).nan_to_num(0.0) if c["score"] == SOFTMAX else torch.sigmoid(x)
    choice = score if s["bias"] is None else score + s["bias"].double()
    if groups > 1:
        best = choice.masked_fill(~there, -math.inf).view(-1, groups, e // groups).sort(dim=2, descending=True).values[:, :, : c["group_best"]]
        total = best.masked_fill(best == -math.inf, 0.0).sum(dim=2).masked_fill(best[:, :, 0] == -math.inf, -math.inf)
        kept = torch.zeros_like(total, dtype=torch.bool).scatter_(1, total.sort(dim=1, descending=True, stable=True).indices[:, : c["top_groups"]], True)
        there = there & kept.repeat_interleave(e // groups, dim=1)
    order = choice.masked_fill(~there, -math.inf).sort(dim=1, descending=True, stable=True).indices[:, :top]
    some = there.gather(1, order)
    w = torch.where(some, score.gather(1, order), 0.0)
    if c["renorm"]:
        w = w / w.sum(dim=1, keepdim=True).clamp_min(torch.finfo(torch.float64).tiny)
    ids, w = torch.where(some, order, -1), w * c["scale"]
    if c["shared"]:
        ids = torch.cat([ids, torch.full_like(ids[:, :1], e)], dim=1)
        w = torch.cat([w, torch.sigmoid(s["logits"][:, e:].double())], dim=1)
    return ids.to(torch.int32), w.float()


def _experts(s):
    c = s["case"]
    x, ids = s["x"], s["ids"] - c["first"]
    y = torch.zeros((*ids.shape, c["hidden"]), device="cuda")
    here = ids[(ids >= 0) & (ids < c["held"])]
    for e in torch.unique(here).tolist():
        token, slot = (ids == e).nonzero(as_tuple=True)
        gate, up, down = (_weights(*(t[e] for t in s[m])) for m in ("gate", "up", "down"))
        g = x[token] @ gate.T
        y[token, slot] = (g / (1 + torch.exp(-g)) * (x[token] @ up.T)) @ down.T
    h = s["residual"] + (s["weights"].unsqueeze(-1) * y).sum(dim=1)
    return h, h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + 1e-6) * s["norm_w"].float()


def run(s):
    if own:
        if "call" not in s:
            s["call"] = _call(s)
        return s["call"]()
    op = s["case"]["op"]
    if op == "proj":
        return [s["x"] @ _weights(*w).T for w in s["w"]]
    return _route(s) if op == "route" else _experts(s)


# ---- the library's calls ------------------------------------------------------------------------
_contexts = {}


def _context():
    """The one context that a program keeps: 8192 tokens a call, on the current stream."""
    if "ctx" not in _contexts:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
        from __graft_entry__ import load_package
        pkg = load_package()
        cfg = pkg.default_config(num_attn_heads=1, num_kv_heads=1, num_full_layers=0, num_linear_layers=0, linear_num_v_heads=1,
                                 linear_num_k_heads=1, max_batch_tokens=8192)
        ctx = pkg.Context(cfg)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        _contexts["ctx"], _contexts["pkg"] = ctx, pkg
    return _contexts["pkg"], _contexts["ctx"]


def _call(s):
    """The library's call for this state, its arguments converted once, as a program that steps layers holds it."""
    pkg, ctx = _context()
    c, n = s["case"], s["case"]["n"]
    if c["op"] == "proj":
        call, out = ctx.prepared_proj_forward([pkg.proj_weights(*w) for w in s["w"]], n, s["x"], s["y"]), s["y"]
    elif c["op"] == "route":
        rc = pkg.route_config(num_experts=c["experts"], top_k=c["top"], score=c["score"], num_groups=c["groups"], top_groups=c["top_groups"],
                              group_best=c["group_best"], renormalize=int(c["renorm"]), scale=c["scale"], shared_expert=int(c["shared"]))
        call, out = ctx.prepared_moe_route(rc, n, s["logits"], s["bias"], s["ids"], s["weights"]), (s["ids"], s["weights"])
    else:
        w = pkg.expert_weights(s["gate"], s["up"], s["down"], first_expert=c["first"], total_experts=c["experts"])
        call = ctx.prepared_moe_experts(w, n, c["top"], s["x"], s["ids"], s["weights"], s["residual"], s["norm_w"], s["h_out"], s["h_norm"])
        out = (s["h_out"], s["h_norm"])

    def whole():
        call()
        return out
    return whole


# ---- what a pass cannot do without --------------------------------------------------------------
def work(case):
    n = case["n"]
    if case["op"] == "proj":
        k, out = case["k"], sum(int(o) for o in case["outs"].split(","))
        return {"bytes": out * k * 0.5625 + 4 * n * (k + out), "flops": 2 * n * k * out}
    if case["op"] == "route":
        e, slots = case["experts"] + int(case["shared"]), case["top"] + int(case["shared"])
        return {"bytes": 4 * n * e + 4 * case["experts"] * int(case["bias"]) + 8 * n * slots, "flops": n * e * 4}
    h, i, share = case["hidden"], case["inter"], case["held"] / case["experts"]
    pairs = n * case["top"] * share
    # experts that a pass reaches, were all of them equally popular
    used = case["held"] * (1 - (1 - case["top"] / case["experts"]) ** n)
    return {"bytes": used * 3 * h * i * 0.5625 + n * h * 16 + 8 * n * case["top"], "flops": pairs * 6 * h * i}


# ---- 64 bits ------------------------------------------------------------------------------------
def _exact_matrix(w, scales, biases):
    b = w.contiguous().view(torch.uint8)
    q = torch.stack((b & 15, b >> 4), dim=-1).flatten(-2).double()
    return q * scales.double().repeat_interleave(GROUP, dim=-1) + biases.double().repeat_interleave(GROUP, dim=-1)


def _exact_route(s):
    c = s["case"]
    n, e, size = c["n"], c["experts"], c["experts"] // c["groups"]
    x = s["logits"][:, :e].double()
    m = x.max(dim=1, keepdim=True).values
    p = torch.where(x == -math.inf, 0.0, torch.exp(x - torch.where(m == -math.inf, 0.0, m)))
    score = p / p.sum(dim=1, keepdim=True).clamp_min(1e-300) if c["score"] == SOFTMAX else 1 / (1 + torch.exp(-x))
    choice = torch.where(x == -math.inf, -math.inf, score + (s["bias"].double() if s["bias"] is not None else 0.0))

    def rank(v):  # how many come before each: larger ones, and equal ones of a lower index
        a, b = v.unsqueeze(2), v.unsqueeze(1)
        low = torch.ones((v.shape[1], v.shape[1]), device=v.device, dtype=torch.bool).tril(-1)
        return ((b > a) | ((b == a) & low)).sum(dim=2)

    ids, weights = [], []
    for part in range(0, n, 256):
        ch, sc = choice[part:part + 256], score[part:part + 256]
        if c["groups"] > 1:
            g = ch.reshape(-1, size)
            lead = (rank(g) < c["group_best"]) & (g > -math.inf)
            total = torch.where(lead, g, 0.0).sum(dim=1)
            total = torch.where((g > -math.inf).any(dim=1), total, -math.inf).view(-1, c["groups"])
            keep = rank(total) < c["top_groups"]
            ch = torch.where(keep.repeat_interleave(size, dim=1), ch, -math.inf)
        r = torch.where(ch > -math.inf, rank(ch), e)
        at = torch.full((ch.shape[0], e + 1), -1, device="cuda", dtype=torch.int64)
        at.scatter_(1, r, torch.arange(e, device="cuda").expand_as(r))
        at = torch.where(torch.arange(c["top"], device="cuda") < (r < e).sum(dim=1, keepdim=True), at[:, : c["top"]], -1)
        w = torch.where(at >= 0, sc.gather(1, at.clamp_min(0)), 0.0)
        ids.append(at)
        weights.append(w / w.sum(dim=1, keepdim=True).clamp_min(1e-300) * c["scale"] if c["renorm"] else w * c["scale"])
    ids, weights = torch.cat(ids), torch.cat(weights)
    if c["shared"]:
        last = s["logits"][:, e].double()
        ids = torch.cat([ids, torch.full((n, 1), e, device="cuda")], dim=1)
        weights = torch.cat([weights, (1 / (1 + torch.exp(-last))).unsqueeze(1)], dim=1)
    return ids, weights


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "proj":
        return [s["x"].double().matmul(_exact_matrix(*w).t()) for w in s["w"]]
    if case["op"] == "route":
        return _exact_route(s)
    x, h = s["x"].double(), s["residual"].double()
    for e in range(case["held"]):
        share = torch.where(s["ids"] == e + case["first"], s["weights"].double(), 0.0).sum(dim=1)
        rows = (s["ids"] == e + case["first"]).any(dim=1).nonzero().flatten()
        if rows.numel() == 0:
            continue
        g = x[rows].matmul(_exact_matrix(*(t[e] for t in s["gate"])).t())
        a = g * torch.sigmoid(g) * x[rows].matmul(_exact_matrix(*(t[e] for t in s["up"])).t())
        h[rows] += share[rows].unsqueeze(1) * a.matmul(_exact_matrix(*(t[e] for t in s["down"])).t())
    return h, h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-6) * s["norm_w"].double()

"""Operators of layers of experts, and the clipping before the optimizer's step, as timing cases.

CRESSO5 steps the stacked weights [experts, outputs, inputs] of a layer of
experts as one tensor.  The operators here are what such a layer computes and
what happens to its gradients before the step:

  route    the router: from logits [tokens, experts] the `top` experts of each
           token, their weights, and the order that brings the token's copies
           together by expert.  Chosen by logit plus bias (in fp32), ties to the
           lowest expert; -inf is never chosen, and where fewer are left the
           rest are absent (expert -1, weight 0).  Weights: softmax or sigmoid
           of the logits, divided by the chosen ones' sum or not, times a scale.
           Its gradient goes to the logits.
  move     the rows on their way to the experts and back: a copy of a token's
           row for each of its experts, sorted by expert; and the sum of the
           experts' answers times the weights.  With the gradients of both.
  product  rows times the weight of the expert that they belong to, groups of
           any size one after another; rows behind the last group give zeros.
           Gradients of the rows and of all weights.
  clip     the norm over all gradients, and the gradients times
           grad_scale * min(1, max_norm / norm), in place or to other tensors.

`own` chooses between plain torch operations in 32 bits and the framework's
operators; inputs are the same for both.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
DEVICE = "cuda"


def listed():
    return [
        # decoding: eight tokens choose among 64 experts
        dict(name="route_token", op="route", train=False, dtype="bf16", tokens=8, experts=64, top=8, score="softmax",
             normalize=True, bias=False, hidden=0.0),
        # training: eight sequences of 2048 tokens, the router in fp32 as most hold it
        dict(name="route_train", op="route", train=True, dtype="fp32", tokens=16384, experts=64, top=8, score="softmax",
             normalize=False, bias=False, hidden=0.0),
        # sigmoid scores, a bias that balances the load, experts that tokens may not use
        dict(name="route_train_odd", op="route", train=True, dtype="bf16", tokens=2777, experts=37, top=3, score="sigmoid",
             normalize=True, bias=True, hidden=0.2),
        # training: 16384 tokens of width 2048 to two experts each and back
        dict(name="move_train", op="move", dtype="bf16", tokens=16384, width=2048, experts=8, top=2, absent=0.0),
        # a short fp32 batch of an odd width, some of whose copies have no expert
        dict(name="move_train_odd", op="move", dtype="fp32", tokens=333, width=1001, experts=13, top=3, absent=0.1),
        # decoding: eight tokens, two experts each, through up projections of the 2048-wide transformer's size
        dict(name="product_token", op="product", train=False, dtype="bf16", rows=16, experts=16, inner=2048, outer=5632,
             idle=0.0, behind=0.0),
        # a prompt of 500 tokens, four small experts each
        dict(name="product_prompt", op="product", train=False, dtype="fp16", rows=2000, experts=32, inner=2048, outer=1024,
             idle=0.0, behind=0.0),
        # training: 16384 tokens, two experts each, forward and both gradients
        dict(name="product_train", op="product", train=True, dtype="bf16", rows=32768, experts=8, inner=2048, outer=5632,
             idle=0.0, behind=0.0),
        # fp32 sizes that are no multiples of anything, experts without a row, rows without an expert
        dict(name="product_train_odd", op="product", train=True, dtype="fp32", rows=777, experts=9, inner=1001, outer=1500,
             idle=0.3, behind=0.1),
        # 840 adapter factors whose norm stays below the limit, in place: most steps of a training run
        dict(name="clip_adapters", op="clip", form="below", kind="adapters", dtype="fp32", tensors=840, most=65536, seed=0,
             norm="2", grad_scale=1.0),
        # the 1.2 B-parameter transformer: bf16 gradients to the fp32 ones that the optimizer steps from, clipped
        dict(name="clip_model", op="clip", form="out", kind="model", dtype="bf16", tensors=199, most=65536000, seed=0, norm="2",
             grad_scale=1.0),
        # a few gradients of odd sizes under a loss scale, packed without gaps
        dict(name="clip_odd", op="clip", form="out", kind="odd", dtype="fp16", tensors=23, most=300001, seed=5, norm="2",
             grad_scale=1.0 / 1024),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high):
    """As _spread; half of them multiples of 64, as most programs have them, and the others odd."""
    n = _spread(rng, low, high)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else (n - 1) | 1


def draw(rng):
    op = rng.choice(("route", "move", "product", "product", "clip"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "route":
        experts = _spread(rng, 2, 256)
        return dict(op=op, train=rng.random() < 0.7, dtype=dtype, tokens=_spread(rng, 1, 16384), experts=experts,
                    top=rng.randint(1, min(8, experts)), score=rng.choice(("softmax", "sigmoid")), normalize=rng.random() < 0.6,
                    bias=rng.random() < 0.4, hidden=rng.choice((0.0, 0.0, 0.3)))
    if op == "move":
        top = rng.randint(1, 8)
        return dict(op=op, dtype=dtype, tokens=_spread(rng, 1, 32768 // top), width=_size(rng, 64, 2048),
                    experts=_spread(rng, top, 128), top=top, absent=rng.choice((0.0, 0.0, 0.2)))
    if op == "product":
        inner, outer = _size(rng, 64, 4096), _size(rng, 64, 5632)
        return dict(op=op, train=rng.random() < 0.7, dtype=dtype, rows=_spread(rng, 1, 16384 if dtype != "fp32" else 2048),
                    experts=_spread(rng, 1, min(64, (1 << 28) // (inner * outer))), inner=inner, outer=outer,
                    idle=rng.choice((0.0, 0.0, 0.4)), behind=rng.choice((0.0, 0.0, 0.2)))
    tensors, most = _spread(rng, 1, 400), _spread(rng, 100, 1 << 22)
    most = min(most, (1 << 28) // tensors)
    return dict(op=op, form=rng.choice(("below", "out")), kind="odd", dtype=rng.choice(("fp32", "bf16", "fp16", "mixed")),
                tensors=tensors, most=most, seed=rng.randint(0, 10 ** 6), norm=rng.choice(("2", "2", "inf")),
                grad_scale=1.0)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32) * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed) * 7919 + 29)
    return globals()["_prepare_" + case["op"]](case, gen)


def _prepare_route(c, gen):
    tokens, experts, dtype = c["tokens"], c["experts"], DTYPES[c["dtype"]]
    # some experts are liked more than others
    z = 1.5 * torch.randn((tokens, experts), generator=gen, device=DEVICE) + 0.5 * torch.randn(experts, generator=gen, device=DEVICE)
    if c["hidden"]:
        z[torch.rand((tokens, experts), generator=gen, device=DEVICE) < c["hidden"]] = -math.inf
        z[torch.rand(tokens, generator=gen, device=DEVICE) < 0.05] = -math.inf   # padding
    s = dict(case=c, logits=z.to(dtype), bias=_randn(gen, (experts,), torch.float32, 0.3) if c["bias"] else None)
    if c["train"]:
        s["logits"].requires_grad_(True)
        s["grad"] = _randn(gen, (tokens, c["top"]), torch.float32, 0.1)
    return s


SCALE = 2.0   # of the router's weights


def _prepare_move(c, gen):
    tokens, width, experts, top, dtype = c["tokens"], c["width"], c["experts"], c["top"], DTYPES[c["dtype"]]
    chosen = (torch.randn((tokens, experts), generator=gen, device=DEVICE)
              + 0.5 * torch.randn(experts, generator=gen, device=DEVICE)).topk(top, dim=1).indices
    if c["absent"]:
        chosen[torch.rand((tokens, top), generator=gen, device=DEVICE) < c["absent"]] = experts
    flat = chosen.flatten()
    order = torch.sort(flat, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(tokens * top, device=DEVICE)
    counts = torch.bincount(flat, minlength=experts + 1)[:experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    chosen = torch.where(chosen == experts, -1, chosen)
    weights = torch.rand((tokens, top), generator=gen, device=DEVICE) + 0.1
    weights = torch.where(chosen < 0, 0.0, weights / weights.sum(1, keepdim=True))
    s = dict(case=c, experts=chosen.int(), order=order.int(), places=places.view(tokens, top).int(), offsets=offsets.int(),
             weights=weights, x=_randn(gen, (tokens, width), dtype), rows=_randn(gen, (tokens * top, width), dtype),
             d_rows=_randn(gen, (tokens * top, width), dtype, 1e-2), d_out=_randn(gen, (tokens, width), dtype, 1e-2))
    for k in ("x", "rows", "weights"):
        s[k].requires_grad_(True)
    return s


def _prepare_product(c, gen):
    rows, experts, inner, outer, dtype = c["rows"], c["experts"], c["inner"], c["outer"], DTYPES[c["dtype"]]
    liked = torch.exp(0.3 * torch.randn(experts, generator=gen, device=DEVICE))
    off = torch.rand(experts, generator=gen, device=DEVICE) < c["idle"]
    off[0] = False
    liked[off] = 0.0
    taken = rows - int(rows * c["behind"])
    group = torch.multinomial(liked, taken, replacement=True, generator=gen)
    counts = torch.bincount(group, minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    s = dict(case=c, x=_randn(gen, (rows, inner), dtype), weight=_randn(gen, (experts, outer, inner), dtype, inner ** -0.5),
             offsets=offsets)
    if c["train"]:
        s["x"].requires_grad_(True)
        s["weight"].requires_grad_(True)
        s["grad"] = _randn(gen, (rows, outer), dtype, 1e-2)
    return s


def _shapes(c):
    """The elements of each gradient, and its type."""
    if c["kind"] == "adapters":
        return [65536] * c["tensors"], [c["dtype"]] * c["tensors"]
    if c["kind"] == "model":
        layer = [2048 * 2048] * 4 + [5632 * 2048] * 3 + [2048] * 2
        return ([32000 * 2048] + layer * 22)[:c["tensors"]], [c["dtype"]] * c["tensors"]
    rng = random.Random(c["seed"])
    numels = [_spread(rng, 1, c["most"]) for _ in range(c["tensors"])]
    types = [c["dtype"] if c["dtype"] != "mixed" else ("fp32", "bf16", "fp16")[i * 3 // c["tensors"]] for i in range(c["tensors"])]
    return numels, types


BUCKETS = 24   # gradients lie one behind another in buckets, as a program that exchanges them holds them


def _prepare_clip(c, gen):
    numels, types = _shapes(c)
    per = -(-len(numels) // BUCKETS)
    grads, buckets, outs, out_buckets = [], [], [], []
    at = 0
    while at < len(numels):
        end = at + 1
        while end < len(numels) and end - at < per and types[end] == types[at]:
            end += 1
        bucket = torch.empty(sum(numels[at:end]), dtype=DTYPES[types[at]], device=DEVICE)
        parts = bucket.split(numels[at:end])
        for g in parts:
            std = 10.0 ** random.Random(len(grads)).uniform(-4, -2)
            g.copy_(torch.randn(g.shape, generator=gen, device=DEVICE) * std)
            grads.append(g)
        buckets.append(bucket)
        if c["form"] == "out":
            out_buckets.append(torch.empty(bucket.shape, dtype=torch.float32, device=DEVICE))
            outs.extend(out_buckets[-1].split(numels[at:end]))
        at = end
    return dict(case=c, grads=grads, buckets=buckets, outs=outs, out_buckets=out_buckets)


def _max_norm(c):
    """Far above what the gradients reach, or far below."""
    return 1e6 if c["form"] == "below" else 1e-2 * c["grad_scale"]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


def _own_route(s):
    import cresso_amd

    c = s["case"]
    weights, r = cresso_amd.route_experts(s["logits"], c["top"], score=c["score"], normalize=c["normalize"], scale=SCALE,
                                          bias=s["bias"])
    out = dict(weights=weights.detach(), experts=r.experts, order=r.order, places=r.places, offsets=r.offsets)
    if c["train"]:
        out["d_logits"] = torch.autograd.grad(weights, s["logits"], s["grad"])[0]
    return out


@torch.no_grad()
def _plain_route(s):
    c, top = s["case"], s["case"]["top"]
    z = s["logits"].float()
    key = z if s["bias"] is None else z + s["bias"]
    best = torch.sort(key, dim=1, descending=True, stable=True)
    chosen = best.indices[:, :top]
    there = best.values[:, :top] > -math.inf
    zc = z.gather(1, chosen)
    if c["score"] == "softmax":
        m = zc.amax(1, keepdim=True) if c["normalize"] else z.amax(1, keepdim=True)
        m = torch.where(m > -math.inf, m, 0.0)
        q = torch.exp(zc - m) * there
        total = q.sum(1, keepdim=True) if c["normalize"] else torch.exp(z - m).sum(1, keepdim=True)
        p = q / torch.where(total > 0, total, 1.0)
    else:
        # sigmoid(z) = e^min(z,0) / (1 + e^-|z|), of which the chosen ones' largest factor e^m is taken out
        m = torch.where(there, zc, -math.inf).amax(1, keepdim=True).clamp(max=0.0) if c["normalize"] else torch.zeros_like(zc[:, :1])
        m = torch.where(m > -math.inf, m, 0.0)
        q = torch.exp(zc.clamp(max=0.0) - m) / (1.0 + torch.exp(-zc.abs())) * there
        total = q.sum(1, keepdim=True)
        p = q / torch.where(total > 0, total, 1.0) if c["normalize"] else q
    experts = torch.where(there, chosen, c["experts"]).flatten()
    ordered = torch.sort(experts, stable=True)
    places = torch.empty_like(ordered.indices)
    places[ordered.indices] = torch.arange(places.numel(), device=places.device)
    offsets = torch.searchsorted(ordered.values, torch.arange(c["experts"] + 1, device=places.device))
    out = dict(weights=SCALE * p, experts=torch.where(there, chosen, -1).int(), order=ordered.indices.int(),
               places=places.view(-1, top).int(), offsets=offsets.int())
    if c["train"]:
        d = s["grad"]
        if c["score"] == "softmax":
            mean = (p * d).sum(1, keepdim=True)
            if c["normalize"]:
                grad = torch.zeros_like(z).scatter_(1, chosen, SCALE * p * (d - mean))
            else:
                grad = -SCALE * mean * torch.exp(z - m) / torch.where(total > 0, total, 1.0)
                grad.scatter_add_(1, chosen, SCALE * p * d)
        else:
            rest = torch.exp(-zc.clamp(min=0.0)) / (1.0 + torch.exp(-zc.abs()))   # 1 - sigmoid(z)
            inner = d - (p * d).sum(1, keepdim=True) if c["normalize"] else d
            grad = torch.zeros_like(z).scatter_(1, chosen, SCALE * p * inner * torch.where(there, rest, 0.0))
        out["d_logits"] = grad.to(s["logits"].dtype)
    return out


def _own_move(s):
    import cresso_amd

    routing = cresso_amd.Routing(s["experts"], s["order"], s["places"], s["offsets"])
    sent = cresso_amd.dispatch_rows(s["x"], routing)
    out = cresso_amd.combine_rows(s["rows"], routing, s["weights"])
    d_x, d_rows, d_weights = torch.autograd.grad((sent, out), (s["x"], s["rows"], s["weights"]), (s["d_rows"], s["d_out"]))
    return dict(sent=sent.detach(), out=out.detach(), d_x=d_x, d_rows=d_rows, d_weights=d_weights)


@torch.no_grad()
def _plain_move(s):
    x, rows, dtype = s["x"], s["rows"], s["x"].dtype
    tokens, top = s["experts"].shape
    places, order = s["places"].long(), s["order"].long()
    there = (s["experts"] >= 0).unsqueeze(2)
    used = there.flatten()[order].unsqueeze(1)
    weights = (s["weights"] * (s["experts"] >= 0)).unsqueeze(2)
    sent = x[order // top] * used
    of = rows[places].float()
    out = (weights * of).sum(1)
    d_x = (s["d_rows"][places].float() * there).sum(1)
    d_out = s["d_out"].float()
    d_rows = (d_out.unsqueeze(1) * weights).view(tokens * top, -1)[order]
    d_weights = (d_out.unsqueeze(1) * of).sum(2) * there.squeeze(2)
    return dict(sent=sent, out=out.to(dtype), d_x=d_x.to(dtype), d_rows=d_rows.to(dtype), d_weights=d_weights)


def _own_product(s):
    import cresso_amd

    y = cresso_amd.expert_product(s["x"], s["weight"], s["offsets"])
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["grad"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


@torch.no_grad()
def _plain_product(s):
    x, weight, offsets, dtype = s["x"], s["weight"].float(), s["offsets"].long(), s["x"].dtype
    rows = x.shape[0]
    # every group in as many rows as the largest has; the places beyond a group show a row of zeros
    counts = offsets.diff().unsqueeze(1)
    slot = torch.arange(max(1, int(counts.max())), device=x.device)
    at = torch.where(slot < counts, offsets[:-1].unsqueeze(1) + slot, rows)
    padded = lambda t: torch.cat([t.float(), torch.zeros((1, t.shape[1]), device=t.device)])[at]   # noqa: E731

    def back(groups):
        out = torch.zeros((rows + 1, groups.shape[2]), device=x.device)
        out[at] = groups
        return out[:rows].to(dtype)

    groups = padded(x)
    out = {"y": back(torch.bmm(groups, weight.transpose(1, 2)))}
    if s["case"]["train"]:
        d = padded(s["grad"])
        out["dx"] = back(torch.bmm(d, weight))
        out["dw"] = torch.bmm(d.transpose(1, 2), groups).to(dtype)
    return out


def _own_clip(s):
    import cresso_amd

    c = s["case"]
    norm = cresso_amd.clip_gradients(s["grads"], _max_norm(c), norm_type=float(c["norm"]), grad_scale=c["grad_scale"],
                                     out=s["outs"] if c["form"] == "out" else None)
    return {"norm": norm, "grads": s["out_buckets"] if c["form"] == "out" else s["buckets"]}


@torch.no_grad()
def _plain_clip(s):
    c = s["case"]
    norms = torch.stack(torch._foreach_norm(s["grads"], float(c["norm"]), dtype=torch.float32)).double()
    norm = c["grad_scale"] * (norms.square().sum().sqrt() if c["norm"] == "2" else norms.max())
    factor = (c["grad_scale"] * (_max_norm(c) / norm).clamp(max=1.0)).float()
    if c["form"] == "out":
        torch._foreach_copy_(s["outs"], s["grads"])
        torch._foreach_mul_(s["outs"], factor)
    else:
        torch._foreach_mul_(s["grads"], factor)
    return {"norm": norm.float(), "grads": s["out_buckets"] if c["form"] == "out" else s["buckets"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    return globals()["_work_" + case["op"]](case)


def _work_route(c):
    table, slots = c["tokens"] * c["experts"], c["tokens"] * c["top"]
    n, flops = table * SIZES[c["dtype"]] + slots * 16 + c["experts"] * 4, 4 * table
    if c["train"]:   # the gradient that arrives, the logits once more, and their gradient
        n += slots * 4 + 2 * table * SIZES[c["dtype"]]
        flops += 4 * table
    return {"bytes": n, "flops": flops}


def _work_move(c):
    size, row = SIZES[c["dtype"]], c["width"] * SIZES[c["dtype"]]
    slots = c["tokens"] * c["top"]
    used = slots * (1 - c["absent"])
    # dispatch: x read, the copies written; its gradient: the copies' read, x's written; combine: the answers read, the
    # sum written; its gradient: the sum's and the answers read, the answers' written
    n = (4 * c["tokens"] + 4 * used + (slots - used)) * row + slots * 20
    return {"bytes": n, "flops": 6 * slots * row / size}


def _work_product(c):
    size, rows = SIZES[c["dtype"]], c["rows"] - int(c["rows"] * c["behind"])
    busy = max(1.0, c["experts"] * (1 - c["idle"]))
    hit = busy * (1 - (1 - 1 / busy) ** rows)   # experts with a row
    matrix, flops = c["inner"] * c["outer"] * size, 2 * rows * c["inner"] * c["outer"]
    n = hit * matrix + rows * c["inner"] * size + c["rows"] * c["outer"] * size
    if c["train"]:
        n += hit * matrix + rows * (c["inner"] + 2 * c["outer"]) * size + c["rows"] * c["inner"] * size
        n += c["experts"] * matrix
        flops *= 3
    return {"bytes": n, "flops": flops}


def _work_clip(c):
    numels, types = _shapes(c)
    n = sum(k * SIZES[t] for k, t in zip(numels, types))
    total = sum(numels)
    return {"bytes": n + 4 * total * (c["form"] == "out"), "flops": 2 * total + total * (c["form"] == "out")}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    return globals()["_exact_" + case["op"]](case, prepare(case, seed))


def _exact_route(c, s):
    tokens, experts, top = c["tokens"], c["experts"], c["top"]
    z32 = s["logits"].detach().float().cpu().numpy()
    key = z32 if s["bias"] is None else z32 + s["bias"].cpu().numpy()   # in fp32, as the choice is defined
    chosen = np.argsort(-key, axis=1, kind="stable")[:, :top]
    there = np.take_along_axis(key, chosen, 1) > -np.inf
    z = torch.tensor(z32.astype(np.float64), requires_grad=bool(c["train"]))
    mask, at = torch.from_numpy(there), torch.from_numpy(chosen)
    zc = z.gather(1, at)
    if c["score"] == "softmax":
        logs = torch.log_softmax(zc.masked_fill(~mask, -math.inf), 1) if c["normalize"] else torch.log_softmax(z, 1).gather(1, at)
        w = torch.where(mask, logs, -math.inf).exp()
    else:
        w = torch.where(mask, torch.sigmoid(zc), 0.0)
        if c["normalize"]:
            w = w / w.sum(1, keepdim=True)
    w = SCALE * torch.where(mask, w, 0.0)
    flat = np.where(there, chosen, experts).ravel()
    order = np.lexsort((np.arange(flat.size), flat))
    places = np.argsort(order)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=experts + 1)[:experts])])
    whole = lambda a: torch.from_numpy(a.astype(np.int32))   # noqa: E731
    out = dict(weights=w.detach(), experts=whole(np.where(there, chosen, -1)), order=whole(order),
               places=whole(places.reshape(tokens, top)), offsets=whole(offsets))
    if c["train"]:
        # rows whose experts are all absent have no weights that depend on anything
        some = mask.any(1)
        g = torch.autograd.grad(w[some].mul(s["grad"].double().cpu()[some]).sum(), z)[0] if bool(some.any()) else torch.zeros_like(z)
        out["d_logits"] = torch.nan_to_num(g, nan=0.0)
    return out


@torch.no_grad()
def _exact_move(c, s):
    tokens, top, width = c["tokens"], c["top"], c["width"]
    experts, places = s["experts"].long(), s["places"].long()
    x, rows, weights = s["x"].double(), s["rows"].double(), s["weights"].double()
    d_sent, d_out = s["d_rows"].double(), s["d_out"].double()
    zeros = lambda n: torch.zeros((n, width), dtype=torch.float64, device=DEVICE)   # noqa: E731
    sent, out, d_x, d_rows = zeros(tokens * top), zeros(tokens), zeros(tokens), zeros(tokens * top)
    d_weights = torch.zeros((tokens, top), dtype=torch.float64, device=DEVICE)
    for k in range(top):
        t = (experts[:, k] >= 0).nonzero().squeeze(1)
        to = places[t, k]
        sent[to] = x[t]
        out[t] += weights[t, k, None] * rows[to]
        d_x[t] += d_sent[to]
        d_rows[to] = weights[t, k, None] * d_out[t]
        d_weights[t, k] = (d_out[t] * rows[to]).sum(1)
    return dict(sent=sent, out=out, d_x=d_x, d_rows=d_rows, d_weights=d_weights)


@torch.no_grad()
def _exact_product(c, s):
    at = s["offsets"].tolist()
    y = torch.zeros((c["rows"], c["outer"]), dtype=torch.float64, device=DEVICE)
    dx = torch.zeros((c["rows"], c["inner"]), dtype=torch.float64, device=DEVICE)
    dw = torch.zeros(s["weight"].shape, dtype=torch.float64, device=DEVICE)
    for e in range(c["experts"]):
        a, b = at[e], at[e + 1]
        if a == b:
            continue
        x, w = s["x"][a:b].double(), s["weight"][e].double()
        y[a:b] = x @ w.t()
        if c["train"]:
            g = s["grad"][a:b].double()
            dx[a:b] = g @ w
            dw[e] = g.t() @ x
    return {"y": y, "dx": dx, "dw": dw} if c["train"] else {"y": y}


@torch.no_grad()
def _exact_clip(c, s):
    if c["norm"] == "2":
        norm = math.sqrt(sum(float(b.double().pow(2).sum()) for b in s["buckets"]))
    else:
        norm = max(float(b.double().abs().max()) for b in s["buckets"])
    norm *= c["grad_scale"]
    limit = _max_norm(c)
    factor = c["grad_scale"] * (limit / norm if norm > limit else 1.0)
    return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [b.double() * factor for b in s["buckets"]]}

"""Operators of a language model's training step around CRESSO5, as timing cases.

The optimizer steps what a model trains: adapters and norm gains on a frozen
base, embedding tables, heads.  The operators here make the gradients that it
takes, in the order in which a step meets them:

  embed    rows of an embedding table times a scale; ids outside the table
           (padding) give rows of zeros and take no gradient.  Its gradient is
           the dense table that the optimizer steps.
  norm     the seam between two blocks: the norm after a block, its gate, the
           scaled residual and the norm before the next block in one operator.
             H = s*h + act(g)*(y*rms(y)*w1),   n = H*rms(H)*w2,   rms(x) = 1/sqrt(mean(x*x)+eps)
           The gate is given per channel, per sequence or per element.
  product  a frozen linear layer whose weight is held in 8-bit floating point
           (e4m3) with one 32-bit scale for each block of 128 x 128.  The
           other operand is rounded to e4m3 in the call, with one power of two
           for each row and 128 of its elements: the smallest 2^e with
           max|x| <= 448 * 2^e.  Forward y = x W^T; backward dx = dy W.
  distill  the loss against a teacher's top logits, at a temperature, mixed
           with the hard label's cross entropy, and its gradient:
             w_r * (a*t^2*KL(p || softmax(z/t)) + (1-a)*CE(z, label))
           p is the softmax of the teacher's entries that are present; a row
           without any, without a label or without weight gives nothing.

`own` chooses between plain torch operations in 32 bits and the framework's
operators; inputs are the same for both.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"
EPS = 1e-6
BLOCK = 128
IGNORE = -100


def listed():
    return [
        # eight sequences decode one token each with the table of the 22-layer, 2048-wide transformer
        dict(name="embed_token", op="embed", train=False, dtype="bf16", tokens=8, vocab=32000, width=2048, wide_ids=True,
             padded=0.0),
        # eight sequences of 2048 tokens and the gradient of a 4096-wide table; a few words make up most of the text
        dict(name="embed_train", op="embed", train=True, dtype="bf16", tokens=16384, vocab=32000, width=4096, wide_ids=True,
             padded=0.0),
        # an fp32 table whose vocabulary is not a round number, a padded batch
        dict(name="embed_train_odd", op="embed", train=True, dtype="fp32", tokens=2777, vocab=50257, width=768,
             wide_ids=False, padded=0.2),
        # decoding: the seam of eight tokens
        dict(name="norm_token", op="norm", train=False, dtype="bf16", rows=8, width=2048, groups=1, act="none"),
        # training: eight sequences of 2048 tokens, a gate and a residual scale per channel
        dict(name="norm_train", op="norm", train=True, dtype="bf16", rows=16384, width=4096, groups=1, act="none"),
        # a gate per sequence, as a condition gives it, at an odd width in fp32
        dict(name="norm_train_odd", op="norm", train=True, dtype="fp32", rows=1533, width=1001, groups=7, act="sigmoid"),
        # scoring of 512 positions against a stored teacher: the loss alone
        dict(name="distill_score", op="distill", form="loss", dtype="bf16", rows=512, vocab=32000, top=32, temperature=1.0,
             mix=1.0, labels=False, absent=0.0),
        # a training batch of 4096 tokens with a large vocabulary, loss and gradient in one call
        dict(name="distill_train", op="distill", form="loss_and_grad", dtype="bf16", rows=4096, vocab=131072, top=64,
             temperature=2.0, mix=0.7, labels=True, absent=0.05),
        # a small fp32 batch through autograd, with teachers of different lengths and masked rows
        dict(name="distill_train_odd", op="distill", form="backward", dtype="fp32", rows=301, vocab=50257, top=17,
             temperature=3.0, mix=0.5, labels=True, absent=0.3),
        # decoding: eight tokens through the transformer's up projection
        dict(name="product_token", op="product", train=False, dtype="bf16", rows=8, inner=2048, outer=5632),
        # training: eight sequences of 2048 tokens, forward and the gradient that goes on to the layers below
        dict(name="product_train", op="product", train=True, dtype="bf16", rows=16384, inner=2048, outer=5632),
        # a short prompt through a layer whose sizes are no multiples of anything
        dict(name="product_train_odd", op="product", train=True, dtype="fp16", rows=333, inner=1001, outer=1500),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    n = max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))
    return n - (n == 3 << 10)


def _size(rng, low, high):
    """As _spread; half of them multiples of 64, as most programs have them, and the others odd."""
    n = _spread(rng, low, high)
    n = max(64, n // 64 * 64) if rng.random() < 0.5 else (n - 1) | 1
    return n - (n == 3 << 10)


def draw(rng):
    op = rng.choice(("embed", "norm", "distill", "product"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    train = rng.random() < 0.7
    if op == "embed":
        width = _size(rng, 64, 4096)
        return dict(op=op, train=train, dtype=dtype, tokens=_spread(rng, 1, 16384), vocab=_size(rng, 100, 32000), width=width,
                    wide_ids=rng.random() < 0.5, padded=rng.choice((0.0, 0.0, 0.3)))
    if op == "norm":
        rows = _spread(rng, 1, 8192)
        divisors = [g for g in range(1, min(rows, 64) + 1) if rows % g == 0]
        return dict(op=op, train=train, dtype=dtype, rows=rows, width=_size(rng, 64, 4096), groups=rng.choice(divisors + [1, rows]),
                    act=rng.choice(("none", "sigmoid", "tanh")))
    if op == "distill":
        vocab = _size(rng, 100, 131072)
        return dict(op=op, form=rng.choice(("loss", "loss_and_grad", "backward")), dtype=dtype, rows=_spread(rng, 1, 1024),
                    vocab=vocab, top=_spread(rng, 1, min(vocab, 128)), temperature=rng.choice((1.0, 1.5, 2.0, 4.0)),
                    mix=rng.choice((1.0, 0.5, 0.9)), labels=rng.random() < 0.6, absent=rng.choice((0.0, 0.25)))
    return dict(op=op, train=train, dtype=dtype, rows=_spread(rng, 1, 8192), inner=_size(rng, 64, 4096),
                outer=_size(rng, 64, 5632))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32) * std + mean).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed) * 7919 + 17)
    dtype = DTYPES[case["dtype"]]
    return globals()["_prepare_" + case["op"]](case, gen, dtype)


def _prepare_embed(c, gen, dtype):
    tokens, vocab, width = c["tokens"], c["vocab"], c["width"]
    # word frequencies fall off steeply: half of the text is the first eighth of the words, one word is a tenth
    u = torch.rand(tokens, generator=gen, device=DEVICE)
    ids = (vocab * u ** 3).long().clamp_(max=vocab - 1)
    ids = (ids * 7919) % vocab   # spread over the table, as a tokenizer's numbers are
    ids[torch.rand(tokens, generator=gen, device=DEVICE) < 0.1] = vocab // 3
    if c["padded"]:
        ids[torch.rand(tokens, generator=gen, device=DEVICE) < c["padded"]] = -1
    s = dict(case=c, ids=ids if c["wide_ids"] else ids.int(), weight=_randn(gen, (vocab, width), dtype, 0.02),
             scale=math.sqrt(width))
    if c["train"]:
        s["weight"].requires_grad_(True)
        s["grad"] = _randn(gen, (tokens, width), dtype, 1e-3)
    return s


def _prepare_norm(c, gen, dtype):
    rows, width, groups = c["rows"], c["width"], c["groups"]
    # sequences x tokens x width; a gate per sequence is (sequences, 1, width)
    full = (groups, rows // groups, width)
    s = dict(case=c, residual=_randn(gen, full, dtype, 2.0), update=_randn(gen, full, dtype, 0.5),
             gate=_randn(gen, (width,) if groups == 1 else (groups, 1, width), dtype, 0.5, 0.3), post=_randn(gen, (width,), dtype, 0.1, 1.0),
             pre=_randn(gen, (width,), dtype, 0.1, 1.0), scale=_randn(gen, (width,), dtype, 0.05, 0.9))
    if c["train"]:
        for k in ("residual", "update", "gate", "post", "pre", "scale"):
            s[k].requires_grad_(True)
        s["grads"] = (_randn(gen, full, dtype, 1e-2), _randn(gen, full, dtype, 1e-2))
    return s


def _prepare_distill(c, gen, dtype):
    rows, vocab, top = c["rows"], c["vocab"], c["top"]
    z = torch.randn((rows, vocab), generator=gen, device=DEVICE)
    z.mul_(2.0)
    # distinct words for each row, in no order, with the teacher's logits falling from the first to the last
    step = vocab // top
    index = torch.arange(top, device=DEVICE)[torch.randperm(top, generator=gen, device=DEVICE)] * step
    index = index + torch.randint(0, step, (rows, top), generator=gen, device=DEVICE)
    teacher = _randn(gen, (rows, top), torch.float32, 1.5).sort(dim=1, descending=True).values + 12.0
    z.scatter_add_(1, index, 0.5 * teacher)   # the student agrees in part
    if c["absent"]:
        kept = torch.rand((rows, top), generator=gen, device=DEVICE)
        index[kept < c["absent"]] = -1
        index[torch.rand(rows, generator=gen, device=DEVICE) < 0.3 * c["absent"]] = -1
    s = dict(case=c, logits=z.to(dtype), index=index.int(), teacher=teacher.to(dtype), labels=None)
    if c["labels"]:
        s["labels"] = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE)
        s["labels"][torch.rand(rows, generator=gen, device=DEVICE) < 0.2 * c["absent"]] = IGNORE
    s["weights"] = torch.full((rows,), 1.0 / rows, device=DEVICE)
    if c["absent"]:
        s["weights"][torch.rand(rows, generator=gen, device=DEVICE) < 0.5 * c["absent"]] = 0.0
    if c["form"] == "backward":
        s["logits"].requires_grad_(True)
    return s


def _prepare_product(c, gen, dtype):
    rows, inner, outer = c["rows"], c["inner"], c["outer"]
    w = torch.randn((outer, inner), generator=gen, device=DEVICE) * 0.02
    w *= torch.exp(0.5 * torch.randn((outer, 1), generator=gen, device=DEVICE))
    nb, kb = -(-outer // BLOCK), -(-inner // BLOCK)
    wide = torch.zeros((nb * BLOCK, kb * BLOCK), device=DEVICE)
    wide[:outer, :inner] = w
    tiles = wide.view(nb, BLOCK, kb, BLOCK)
    scales = (tiles.abs().amax(dim=(1, 3)) / 448.0).clamp_(min=1e-12)
    values = (tiles / scales[:, None, :, None]).clamp_(-448.0, 448.0).view(nb * BLOCK, kb * BLOCK)[:outer, :inner]
    x = torch.randn((rows, inner), generator=gen, device=DEVICE)
    x *= torch.exp(torch.randn((1, inner), generator=gen, device=DEVICE))   # some channels are large, as activations are
    s = dict(case=c, x=x.to(dtype), values=values.contiguous().to(torch.float8_e4m3fn), scales=scales)
    if c["train"]:
        s["x"].requires_grad_(True)
        s["grad"] = _randn(gen, (rows, outer), dtype, 1e-3)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


def _own_embed(s):
    import cresso_amd

    out = cresso_amd.embedding(s["ids"], s["weight"], scale=s["scale"])
    if not s["case"]["train"]:
        return {"out": out}
    return {"out": out, "grad": torch.autograd.grad(out, s["weight"], s["grad"])[0]}


@torch.no_grad()
def _plain_embed(s):
    ids, weight = s["ids"].long(), s["weight"]
    there = ((ids >= 0) & (ids < weight.shape[0])).unsqueeze(1)
    at = ids.clamp(0, weight.shape[0] - 1)
    out = {"out": (weight[at].float() * s["scale"] * there).to(weight.dtype)}
    if s["case"]["train"]:
        total = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device)
        total.index_add_(0, at, s["grad"].float() * there)
        out["grad"] = (total * s["scale"]).to(weight.dtype)
    return out


NORM_INPUTS = ("residual", "update", "gate", "post", "pre", "scale")


def _own_norm(s):
    import cresso_amd

    out, normed = cresso_amd.residual_norm(s["residual"], s["update"], gate=s["gate"], gate_act=s["case"]["act"],
                                           post_weight=s["post"], pre_weight=s["pre"], residual_scale=s["scale"], eps=EPS)
    if not s["case"]["train"]:
        return {"out": out, "normed": normed}
    grads = torch.autograd.grad((out, normed), [s[k] for k in NORM_INPUTS], s["grads"])
    return {"out": out, "normed": normed, **{"d_" + k: g for k, g in zip(NORM_INPUTS, grads)}}


@torch.no_grad()
def _plain_norm(s):
    dtype, act, groups = s["residual"].dtype, s["case"]["act"], s["case"]["groups"]
    h, y, g, w1, w2, r = (s[k].float() for k in NORM_INPUTS)
    a = torch.sigmoid(g) if act == "sigmoid" else torch.tanh(g) if act == "tanh" else g
    ry = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    yn = y * ry
    u = yn * w1
    total = r * h + a * u
    rh = torch.rsqrt((total * total).mean(-1, keepdim=True) + EPS)
    hn = total * rh
    out = {"out": total.to(dtype), "normed": (hn * w2).to(dtype)}
    if not s["case"]["train"]:
        return out
    d_out, d_normed = (d.float() for d in s["grads"])
    e = d_normed * w2
    d = d_out + rh * (e - hn * (e * hn).mean(-1, keepdim=True))
    d_a = (d * u).sum((0, 1)) if groups == 1 else (d * u).sum(1, keepdim=True)
    d_g = d_a * a * (1 - a) if act == "sigmoid" else d_a * (1 - a * a) if act == "tanh" else d_a
    d_u = d * a
    f = d_u * w1
    grads = dict(residual=r * d, update=ry * (f - yn * (f * yn).mean(-1, keepdim=True)), gate=d_g,
                 post=(d_u * yn).sum((0, 1)), pre=(d_normed * hn).sum((0, 1)), scale=(d * h).sum((0, 1)))
    return {**out, **{"d_" + k: grads[k].to(dtype) for k in NORM_INPUTS}}


def _own_distill(s):
    import cresso_amd

    c = s["case"]
    kw = dict(labels=s["labels"], row_weights=s["weights"], temperature=c["temperature"], mix=c["mix"], ignore_index=IGNORE)
    if c["form"] == "loss":
        return {"loss": cresso_amd.distill_loss(s["logits"], s["index"], s["teacher"], reduction="none", **kw)}
    if c["form"] == "loss_and_grad":
        loss, grad = cresso_amd.distill_loss_and_grad(s["logits"], s["index"], s["teacher"], **kw)
        return {"loss": loss, "grad": grad}
    loss = cresso_amd.distill_loss(s["logits"], s["index"], s["teacher"], **kw)
    return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, s["logits"])[0]}


@torch.no_grad()
def _plain_distill(s):
    c, logits, vocab = s["case"], s["logits"], s["case"]["vocab"]
    t, mix, w = c["temperature"], c["mix"], s["weights"]
    z = logits.float()
    z = z - z.amax(1, keepdim=True)
    there = (s["index"] >= 0) & (s["index"] < vocab)
    index = s["index"].long().clamp(0, vocab - 1)
    a = torch.where(there, s["teacher"].float() / t, -math.inf)
    some = there.any(1, keepdim=True)
    top = torch.where(some, a.amax(1, keepdim=True), 0.0)
    p = torch.exp(a - top)
    p = torch.where(some, p / p.sum(1, keepdim=True), 0.0)
    log_p = torch.where(p > 0, torch.log(p), 0.0)
    zt = z / t
    log_zt = torch.log(torch.exp(zt).sum(1, keepdim=True))
    log_q = zt.gather(1, index) - log_zt
    loss = mix * t * t * torch.where(p > 0, p * (log_p - log_q), 0.0).sum(1)
    if c["form"] != "loss":
        grad = torch.exp(zt - log_zt) * some
        grad.scatter_add_(1, index, -p)
        grad *= mix * t
    if s["labels"] is not None:
        has = (s["labels"] != IGNORE).unsqueeze(1)
        label = s["labels"].clamp(0, vocab - 1).unsqueeze(1)
        log_z = torch.log(torch.exp(z).sum(1, keepdim=True))
        loss = loss + (1 - mix) * ((log_z - z.gather(1, label)) * has).squeeze(1)
        if c["form"] != "loss":
            hard = torch.exp(z - log_z)
            hard.scatter_add_(1, label, torch.full_like(log_z, -1.0))
            grad += (1 - mix) * hard * has
    loss = loss * w
    if c["form"] == "loss":
        return {"loss": loss}
    return {"loss": loss.sum(), "grad": (grad * w.unsqueeze(1)).to(logits.dtype)}


def _own_product(s):
    import cresso_amd

    y = cresso_amd.block_product(s["x"], s["values"], s["scales"])
    if not s["case"]["train"]:
        return {"y": y}
    return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["grad"])[0]}


def _rounded(x):
    """x in 32 bits as its e4m3 values times their powers of two, one for each row and 128 elements."""
    rows, n = x.shape
    wide = torch.zeros((rows, -(-n // BLOCK) * BLOCK), device=x.device)
    wide[:, :n] = x.float()
    tiles = wide.view(rows, -1, BLOCK)
    m, e = torch.frexp(tiles.abs().amax(2, keepdim=True))
    scale = torch.exp2((e - 9 + (m > 0.875).int()).clamp(-127, 127).float())
    return ((tiles / scale).to(torch.float8_e4m3fn).float() * scale).view(rows, -1)[:, :n]


@torch.no_grad()
def _plain_product(s):
    values = s["values"].float()
    outer, inner = values.shape
    scales = s["scales"].repeat_interleave(BLOCK, 0)[:outer].repeat_interleave(BLOCK, 1)[:, :inner]
    w = values * scales
    out = {"y": (_rounded(s["x"]) @ w.t()).to(s["x"].dtype)}
    if s["case"]["train"]:
        out["dx"] = (_rounded(s["grad"]) @ w).to(s["x"].dtype)
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    return globals()["_work_" + case["op"]](case, torch.finfo(DTYPES[case["dtype"]]).bits // 8)


def _work_embed(c, size):
    tokens, vocab = c["tokens"] * (1 - c["padded"]), c["vocab"]
    row = c["width"] * size
    # how many of the table's rows the tokens name, by the frequencies that the ids are made with
    edges = np.cbrt(np.arange(vocab + 1) / vocab)
    named = float((1 - np.exp(-0.9 * tokens * np.diff(edges))).sum())
    n = (named + c["tokens"]) * row + c["tokens"] * (8 if c["wide_ids"] else 4)
    flops = c["tokens"] * c["width"]
    if c["train"]:   # the tokens' gradients are read and the table's is written whole
        n += (c["tokens"] + vocab) * row
        flops *= 2
    return {"bytes": n, "flops": flops}


def _work_norm(c, size):
    rows, width = c["rows"], c["width"]
    small = (c["groups"] + 3) * width * size
    n, flops = 4 * rows * width * size + small, 10 * rows * width
    if c["train"]:   # both inputs and both gradients are read, two gradients are written
        n += 6 * rows * width * size + 2 * small
        flops += 26 * rows * width
    return {"bytes": n, "flops": flops}


def _work_distill(c, size):
    rows, vocab, top = c["rows"], c["vocab"], c["top"]
    # "backward" reads the logits in each of its two calls, as no call knows of the next
    passes = {"loss": 1, "loss_and_grad": 2, "backward": 3}[c["form"]]
    once = rows * top * (4 + size) + rows * 8
    return {"bytes": passes * rows * vocab * size + once, "flops": (4 + 6 * (passes > 1)) * rows * vocab}


def _work_product(c, size):
    rows, inner, outer = c["rows"], c["inner"], c["outer"]
    once = inner * outer + 4 * (-(-inner // BLOCK)) * (-(-outer // BLOCK)) + rows * (inner + outer) * size
    return {"bytes": once * (1 + c["train"]), "flops": 2 * rows * inner * outer * (1 + c["train"])}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    return globals()["_exact_" + case["op"]](case, prepare(case, seed))


@torch.no_grad()
def _exact_embed(c, s):
    table = torch.cat([s["weight"].double(), torch.zeros((1, c["width"]), dtype=torch.float64, device=DEVICE)])
    ids = torch.where(s["ids"] < 0, c["vocab"], s["ids"]).long()   # the zeros beyond the last row
    out = {"out": table.index_select(0, ids) * s["scale"]}
    if c["train"]:
        grad = torch.zeros_like(table)
        grad.scatter_add_(0, ids.unsqueeze(1).expand(-1, c["width"]), s["grad"].double() * s["scale"])
        out["grad"] = grad[:-1]
    return out


def _exact_norm(c, s):
    given = [s[k].detach().double().requires_grad_(c["train"]) for k in NORM_INPUTS]
    h, y, g, w1, w2, r = given
    act = {"none": lambda v: v, "sigmoid": lambda v: 1 / (1 + torch.exp(-v)), "tanh": torch.tanh}[c["act"]]
    total = r * h + act(g) * (y / (y.pow(2).sum(2, keepdim=True) / c["width"] + EPS).sqrt() * w1)
    normed = total / (total.pow(2).sum(2, keepdim=True) / c["width"] + EPS).sqrt() * w2
    out = {"out": total.detach(), "normed": normed.detach()}
    if c["train"]:
        grads = torch.autograd.grad((total, normed), given, tuple(d.double() for d in s["grads"]))
        out.update({"d_" + k: d for k, d in zip(NORM_INPUTS, grads)})
    return out


def _exact_distill(c, s):
    losses, grads = [], []
    t = c["temperature"]
    for r in range(0, c["rows"], 512):
        z = s["logits"][r:r + 512].detach().double().requires_grad_(c["form"] != "loss")
        index, a = s["index"][r:r + 512].long(), s["teacher"][r:r + 512].double() / t
        w = s["weights"][r:r + 512].double()
        there = index >= 0
        a = a.masked_fill(~there, -math.inf)
        p = torch.softmax(a, 1).nan_to_num(0.0)   # a row without a teacher has no entries at all
        soft = torch.log_softmax(z / t, 1).gather(1, index.clamp(min=0))
        entropy = torch.special.entr(p).sum(1)
        loss = c["mix"] * t * t * (-entropy - (p * soft).sum(1))
        if s["labels"] is not None:
            label = s["labels"][r:r + 512]
            hard = -torch.log_softmax(z, 1).gather(1, label.clamp(min=0).unsqueeze(1)).squeeze(1)
            loss = loss + (1 - c["mix"]) * torch.where(label >= 0, hard, torch.zeros_like(hard))
        loss = loss * w
        losses.append(loss.detach())
        if c["form"] != "loss":
            grads.append(torch.autograd.grad(loss.sum(), z)[0])
    loss = torch.cat(losses)
    return {"loss": loss} if c["form"] == "loss" else {"loss": loss.sum(), "grad": torch.cat(grads)}


def _exact_rounded(x):
    """Rows of x rounded to a sign, four significant bits and a power of two per 128, halves to even."""
    x = x.detach().double()
    for k in range(0, x.shape[1], BLOCK):
        part = x[:, k:k + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        unit = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top / 448.0))), 1.0)
        unit = torch.where(top > 448.0 * unit, unit * 2, torch.where(top <= 224.0 * unit, unit / 2, unit))
        q = part / unit
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)   # subnormal below 2^-6
        x[:, k:k + BLOCK] = torch.round(q / step) * step * unit
    return x


@torch.no_grad()
def _exact_product(c, s):
    w = s["values"].float().double()
    for n in range(s["scales"].shape[0]):
        for k in range(s["scales"].shape[1]):
            w[n * BLOCK:(n + 1) * BLOCK, k * BLOCK:(k + 1) * BLOCK] *= s["scales"][n, k].double()
    out = {"y": _exact_rounded(s["x"]) @ w.t()}
    if c["train"]:
        out["dx"] = _exact_rounded(s["grad"]) @ w
    return out

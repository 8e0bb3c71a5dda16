"""A layer of experts as it is used: router, rows to the experts and back, two
grouped products, backward pass, clipping and the optimizer's step; in graphs, on
other streams, with padded tokens, past 2^31 elements."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.nn.functional import silu

from gpu_util import announce, needs_gpu
from operator_util import EPS32, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

WIDTH, HIDDEN, EXPERTS, TOP = 64, 96, 7, 2


def layer(x, gate, up, down, top=TOP, bias=None):
    logits = x.float() @ gate.float().t()
    if bias is not None:
        logits = logits + bias   # masks: -inf for tokens that are padding
    weights, routing = cresso_amd.route_experts(logits, top, scale=1.5)
    rows = cresso_amd.dispatch_rows(x, routing)
    rows = cresso_amd.expert_product(rows, up, routing.offsets)
    rows = cresso_amd.expert_product(silu(rows), down, routing.offsets)
    return cresso_amd.combine_rows(rows, routing, weights), routing


def layer64(x, gate, up, down, experts, bias=None):
    """The same in 64 bits, with the experts that were chosen ([tokens, top], -1 for none)."""
    logits = x @ gate.t() if bias is None else x @ gate.t() + bias
    there = experts >= 0
    z = torch.where(there, logits.gather(1, experts.clamp(min=0)), -math.inf)
    z = torch.where(there.any(1, keepdim=True), z, 0.0)
    w = torch.where(there, 1.5 * torch.softmax(z, 1), 0.0)
    out = torch.zeros_like(x)
    for k in range(experts.shape[1]):
        for e in range(up.shape[0]):
            t = (experts[:, k] == e).nonzero().squeeze(1)
            if t.numel():
                out = out.index_add(0, t, w[t, k, None] * (silu(x[t] @ up[e].t()) @ down[e].t()))
    return out


def make(dtype=torch.float32, tokens=90, seed=0, width=WIDTH, hidden=HIDDEN, experts=EXPERTS):
    return [rand((tokens, width), dtype, seed), rand((experts, width), dtype, seed + 1, width ** -0.5),
            rand((experts, hidden, width), dtype, seed + 2, width ** -0.5), rand((experts, width, hidden), dtype, seed + 3, hidden ** -0.5)]


def near(got, want, dtype, what):
    """2-norm of the error.  In fp32 an element passes through WIDTH + HIDDEN additions and some 32 operations more, each off by
    2^-24 of magnitudes whose sums are up to sqrt(WIDTH * HIDDEN) times those of the results; 16-bit types round five times on the way."""
    got, want = got.detach().double().cpu(), want.detach().cpu()
    room = (WIDTH + HIDDEN + 32) * EPS32 * math.sqrt(WIDTH * HIDDEN)
    if dtype != torch.float32:
        room += 8 * torch.finfo(dtype).eps / 2
    assert float((got - want).norm()) <= room * float(want.norm()) + 1e-30, what


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_layer_and_gradients(dtype):
    announce(f"layer of experts {dtype}")
    given = make(dtype)
    leaves = [t.detach().requires_grad_(True) for t in given]
    out, routing = layer(*leaves)
    d = rand(tuple(out.shape), dtype, 9)
    got = torch.autograd.grad(out, leaves, d)
    exact = [t.detach().double().cpu().requires_grad_(True) for t in given]
    experts = routing.experts.cpu().long()
    want = layer64(*exact, experts)
    near(out, want, dtype, "layer")
    for g, w, name in zip(got, torch.autograd.grad(want, exact, d.double().cpu()), ("x", "gate", "up", "down")):
        near(g, w, dtype, f"gradient of {name}")


def test_padded_tokens():
    """Tokens whose logits are all -inf go to no expert: zeros, gradients of zero, and nothing of theirs in the others'."""
    announce("layer of experts, padded")
    x, gate, up, down = make()
    pad = torch.zeros(90, EXPERTS).cuda()
    pad[::4] = -math.inf
    pad[:, 3] = -math.inf      # an expert that nobody may take
    keep = torch.arange(90) % 4 != 0
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, up, down)]
    out, routing = layer(*leaves, bias=pad)
    assert not out[~keep.cuda()].any() and int(routing.offsets[-1]) == 2 * int(keep.sum())
    grads = torch.autograd.grad(out, leaves[2:], torch.ones_like(out))
    assert all(torch.isfinite(g).all() for g in grads) and not grads[0][3].any() and not grads[1][3].any()
    short = [t.detach().requires_grad_(True) for t in (x[keep.cuda()], gate, up, down)]
    same, _ = layer(*short, bias=pad[keep.cuda()])
    assert torch.equal(out[keep.cuda()], same)
    for a, b in zip(grads, torch.autograd.grad(same, short[2:], torch.ones_like(same))):
        assert torch.equal(a, b)


def test_more_experts_than_are_left():
    announce("layer of experts, few left")
    x, gate, up, down = make()
    pad = torch.full((90, EXPERTS), -math.inf).cuda()
    pad[:, 2] = 0.0
    pad[::3, 5] = 0.0
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, up, down)]
    out, routing = layer(*leaves, top=4, bias=pad)
    exact = [t.detach().double().cpu().requires_grad_(True) for t in (x, gate, up, down)]
    want = layer64(*exact, routing.experts.cpu().long(), pad.double().cpu())
    near(out, want, torch.float32, "layer")
    d = rand(tuple(out.shape), torch.float32, 9)
    for g, w in zip(torch.autograd.grad(out, leaves[2:], d), torch.autograd.grad(want, exact[2:], d.double().cpu())):
        near(g, w, torch.float32, "gradient")


def train(steps, dtype=torch.float32):
    x, *weights = make(dtype, seed=3)
    params = [torch.nn.Parameter(w) for w in weights]
    target = rand((90, WIDTH), torch.float32, 8)
    opt = cresso_amd.CRESSO5(params, lr=2e-3, rank=4, hash_bins=64, cuda_ops="required")
    norms = []
    for step in range(steps):
        out, _ = layer(x, *params)
        opt.zero_grad()
        ((out.float() - target) ** 2).sum().backward()
        norms.append(opt.clip_gradients(1.0))
        total = torch.linalg.vector_norm(torch.cat([p.grad.double().flatten() for p in params]))
        assert float(total) <= 1.0 + torch.finfo(dtype).eps   # each rounding is off by half of that at most
        opt.step()
    return params, torch.stack(norms)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_steps_repeat(dtype):
    """Stacked weights are stepped by the spectral route; every kernel on the way sums in a fixed order."""
    announce(f"training steps of a layer of experts {dtype}")
    params, norms = train(4, dtype)
    assert torch.isfinite(norms).all() and (norms > 1.0).all()
    again, same = train(4, dtype)
    assert torch.equal(norms, same) and all(torch.equal(a, b) for a, b in zip(params, again))


def whole_step(x, gate, up, down, d):
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, up, down)]
    out, routing = layer(*leaves)
    grads = torch.autograd.grad(out, leaves, d)
    clipped = [torch.empty_like(g) for g in grads]
    norm = cresso_amd.clip_gradients(grads, 0.5, out=clipped)
    return [out, norm, *clipped, *routing]


@pytest.mark.parametrize("tokens", [40, 300])
def test_graph(tokens):
    """One launch for few tokens, three for more; replays on new inputs, eager work between them."""
    announce(f"layer of experts in a graph, {tokens} tokens")
    inputs = [*make(torch.bfloat16, tokens), rand((tokens, WIDTH), torch.bfloat16, 9)]
    whole_step(*inputs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        whole_step(*inputs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = whole_step(*inputs)
    for k in range(4):
        for j, t in enumerate(inputs):
            t.copy_(rand(tuple(t.shape), t.dtype, 30 + 5 * k + j, 0.2 + 0.1 * j))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, whole_step(*inputs)):
            assert torch.equal(a, b)


def test_graph_of_odd_rows():
    """Operands that are laid out anew, in the graph's own memory, while eager calls of the same go on beside it."""
    announce("products of odd rows in a graph")
    offsets = torch.tensor([0, 9000, 9000, 9300, 16600], dtype=torch.int32).cuda()
    x, w, d = rand((16600, 333), torch.bfloat16, 1), rand((4, 1283, 333), torch.bfloat16, 2, 0.5), rand((16600, 1283), torch.bfloat16, 3)

    def step():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = cresso_amd.expert_product(a, b, offsets)
        return [y, *torch.autograd.grad(y, (a, b), d)]

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        for j, t in enumerate((x, w, d)):
            t.copy_(rand(tuple(t.shape), t.dtype, 40 + 3 * k + j))
        graph.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_two_streams_at_once():
    announce("layers of experts on two streams")
    sets = [[*make(torch.bfloat16, 200, seed=s), rand((200, WIDTH), torch.bfloat16, s + 9)] for s in (0, 20)]
    want = [whole_step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = whole_step(*sets[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_past_32_bits():
    announce("rows of experts past 2^31 elements")
    tokens, top, width = 40000, 8, 8192   # 2.6e9 elements of rows
    experts = torch.arange(top).expand(tokens, top).int().contiguous()
    slots = torch.arange(tokens * top).view(tokens, top)
    places = (torch.arange(top) * tokens + torch.arange(tokens).unsqueeze(1)).int()
    r = cresso_amd.Routing(experts.cuda(), slots.t().flatten().int().cuda(), places.cuda(), (torch.arange(top + 1) * tokens).int().cuda())
    x = torch.zeros(tokens, width, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 17, 32769, 39999]).cuda()
    x[at] = rand((4, width), torch.bfloat16, 3)
    rows = cresso_amd.dispatch_rows(x, r)
    for k in (0, 6, 7):
        assert torch.equal(rows[k * tokens + at], x[at])
    w = torch.full((tokens, top), 0.125).cuda()
    assert torch.equal(cresso_amd.combine_rows(rows, r, w), x)
    offsets = torch.tensor([0, 262143, 262145, tokens * top], dtype=torch.int32).cuda()
    weight = rand((3, 64, width), torch.bfloat16, 4, 2.0 ** -6)
    y = cresso_amd.expert_product(rows, weight, offsets)
    last = tokens * 7 + at
    torch.testing.assert_close(y[last].float(), (rows[last].double() @ weight[2].double().t()).float(), rtol=2.0 ** -7, atol=1e-3)
    assert not y[tokens * 7 + 1:tokens * 7 + 17].any()
    rows.requires_grad_(True)   # the gradient of the rows is as large again
    d = torch.zeros_like(y)
    d[last] = rand((4, 64), torch.bfloat16, 5)
    dx = torch.autograd.grad(cresso_amd.expert_product(rows, weight, offsets), rows, d)[0]
    torch.testing.assert_close(dx[last].float(), (d[last].double() @ weight[2].double()).float(), rtol=2.0 ** -7, atol=1e-3)
    assert not dx[:tokens * 7].any()


def test_gradients_past_32_bits():
    announce("clip past 2^31 elements")
    g = torch.zeros((1 << 31) + 70001, dtype=torch.bfloat16, device="cuda")
    g[7], g[-1], g[1 << 31] = 3.0, 4.0, 12.0
    assert float(cresso_amd.clip_gradients(g, 6.5)) == 13.0
    assert g[7] == 1.5 and g[-1] == 2.0 and g[1 << 31] == 6.0 and int(g.count_nonzero()) == 3


def dual_calls():
    x, gate, up, down = make()
    w, r = cresso_amd.route_experts(x @ gate.t(), TOP)
    rows = cresso_amd.dispatch_rows(x, r)
    return {
        "route": (lambda t: cresso_amd.route_experts(t, TOP)[0], x @ gate.t()),
        "bias": (lambda t: cresso_amd.route_experts(x @ gate.t(), TOP, bias=t)[0], torch.zeros(EXPERTS).cuda()),
        "dispatch": (lambda t: cresso_amd.dispatch_rows(t, r), x),
        "combine": (lambda t: cresso_amd.combine_rows(t, r, w), rows),
        "combine weights": (lambda t: cresso_amd.combine_rows(rows, r, t), w),
        "product": (lambda t: cresso_amd.expert_product(t, up, r.offsets), rows),
        "product weight": (lambda t: cresso_amd.expert_product(rows, t, r.offsets), up),
        "norm": (lambda t: cresso_amd.gradient_norm([t]), x),
        "clip": (lambda t: cresso_amd.clip_gradients([t], 1.0, out=[torch.empty_like(x)]), x),
    }


@pytest.mark.parametrize("name", ["route", "bias", "dispatch", "combine", "combine weights", "product", "product weight", "norm", "clip"])
def test_dual_tensors_are_refused(name):
    call, x = dual_calls()[name]
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(fwad.make_dual(x.detach(), torch.ones_like(x)))
        call(x.detach())


@pytest.mark.parametrize("name", ["route", "bias", "dispatch", "combine", "combine weights", "product", "product weight", "norm", "clip"])
def test_negative_views_are_refused(name):
    """Their memory holds the negative of what they are."""
    call, x = dual_calls()[name]
    with pytest.raises(RuntimeError, match="negative of its memory"):
        call(torch._neg_view(x.detach()))
    call(torch._neg_view(x.detach()).resolve_neg())


def test_second_derivatives_are_refused():
    """The gradient of dispatch depends on what arrives alone; that of combine is taken to depend on its rows too."""
    x, gate, up, down = make()
    routing = cresso_amd.route_experts(x @ gate.t(), TOP)[1]
    cases = ((lambda t: cresso_amd.route_experts(t, TOP)[0], (x @ gate.t()).detach(), "differentiated twice"),
             (lambda t: cresso_amd.dispatch_rows(t, routing), x.detach(), "does not require grad"),
             (lambda t: cresso_amd.combine_rows(t, routing), rand((180, WIDTH)), "differentiated twice"))
    for fn, leaf, text in cases:
        leaf.requires_grad_(True)
        y = fn(leaf)
        (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)
        if text == "differentiated twice":
            with pytest.raises(RuntimeError, match=text):
                g.sum().backward()
        else:
            assert not g.requires_grad
        y = fn(leaf)
        (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y).requires_grad_(True), create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated twice"):
            g.sum().backward()


def test_weights_changed_in_place_are_noticed():
    x, gate, _, _ = make()
    z = (x @ gate.t()).detach().requires_grad_(True)
    w, _ = cresso_amd.route_experts(z, TOP)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.sum().backward()
    leaf = rand((4, 4)).requires_grad_(True)
    y = (leaf * leaf).sum()
    with torch.no_grad():
        cresso_amd.clip_gradients([leaf], 0.1)   # written behind autograd's back, but not unnoticed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()

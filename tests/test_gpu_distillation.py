"""Distillation under the output unit on the GPU, against float64."""

import math

import pytest
import torch

from alignment_reference import near
from distill_reference import distill
from test1_amd import linear_logps as limits
from test1_amd.distillation import linear_distill
from test1_amd.sampling import top_logps

pytestmark = pytest.mark.gpu

# tokens, hidden, vocabulary, words: tiles and their edges, odd hidden sizes, one token, every word, one word
SHAPES = [(1, 64, 512, 4), (1, 64, 1, 1), (3, 8, 5, 5), (7, 128, 257, 16), (33, 65, 1000, 128), (64, 64, 256, 128),
          (65, 128, 255, 1), (128, 192, 1021, 64), (129, 256, 4099, 33), (255, 64, 2048, 128), (256, 512, 128, 128),
          (257, 320, 777, 100), (300, 896, 1540, 17), (513, 128, 513, 65), (40, 1024, 50_257, 20)]
FORMS = [("forward", True), ("forward", False), ("reverse", True)]


def inputs(shape, dtype, dev, seed=0, near_by=False):
    n, h, v, k = shape
    g = torch.Generator(device=dev).manual_seed(seed + n + h + v)
    hidden = torch.randn(n, h, generator=g, device=dev).to(dtype)
    weight = (torch.randn(v, h, generator=g, device=dev) * (2.0 / math.sqrt(h))).to(dtype)
    z = hidden.float() @ weight.float().t()
    teacher = top_logps(z * 1.2 + torch.randn(n, v, generator=g, device=dev), k)
    ids, logps = teacher.ids.clone(), teacher.logps.clone()
    turn = torch.randperm(k, generator=g, device=dev)   # in any order
    ids, logps = ids[:, turn].contiguous(), logps[:, turn].contiguous()
    if n > 4 and k > 1:
        logps[1, k // 2:] = -math.inf
        ids[1, -1] = -7
        logps[2] = -math.inf
    mask = torch.rand(n, generator=g, device=dev) < 0.85
    mask[0] = True
    up = torch.randn(n, generator=g, device=dev) / n
    return hidden, weight, ids, logps, mask, up


def check(args, dtype, temperature=1.0, kind="forward", rest=True):
    hidden, weight, ids, logps, mask, up = args
    want, bound = distill(hidden, weight, ids, logps, mask, 1 / temperature, kind, rest, grad=up)
    with torch.no_grad():
        near(linear_distill(hidden, weight, ids, logps, mask, temperature, kind, rest), want[0], bound[0])
    hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = linear_distill(hr, wr, ids, logps, mask, temperature, kind, rest)
    gh, gw = torch.autograd.grad(loss, (hr, wr), up)
    assert gh.dtype == gw.dtype == dtype and loss.dtype == torch.float32
    for got, w, b in zip((loss.detach(), gh, gw), want, bound):
        near(got, w, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_float64(dev, shape, dtype):
    args = inputs(shape, dtype, dev)
    for kind, rest in FORMS:
        check(args, dtype, 1.0 if shape[0] % 2 else 1.5, kind, rest)


@pytest.mark.parametrize("share", [0.0, 0.3, 0.95, 1.0])
@pytest.mark.parametrize("shape,dtype", [((400, 2048, 50_000, 9), torch.bfloat16), ((300, 2048, 60_000, 128), torch.float16),
                                         ((4200, 2048, 12_000, 3), torch.bfloat16), ((700, 1536, 40_011, 20), torch.bfloat16)])
def test_masked_tokens_left_out_of_the_products(dev, shape, dtype, share):
    """Calls large enough that D has the rows of the tokens that count alone: a fraction, none, all of them
    masked; tokens without an upstream gradient, without words, with wrong ones."""
    hidden, weight, ids, logps, _, up = inputs(shape, dtype, dev)
    g = torch.Generator(device=dev).manual_seed(1)
    mask = torch.rand(shape[0], generator=g, device=dev) >= share
    up[5:9] = 0
    plain = linear_distill(hidden.clone().requires_grad_(True), weight, ids, logps, mask)
    want, bound = distill(hidden, weight, ids, logps, mask, 1.0, "forward", True, grad=up)
    near(plain.detach(), want[0], bound[0])
    hidden[~mask] = math.nan
    hr, wr = hidden.requires_grad_(True), weight.clone().requires_grad_(True)
    loss = linear_distill(hr, wr, ids, logps, mask)
    assert torch.equal(loss, plain)
    gh, gw = torch.autograd.grad(loss, (hr, wr), up, retain_graph=True)
    assert (gh[~mask] == 0).all() and (gh[5:9] == 0).all() and gh.isfinite().all() and gw.isfinite().all()
    again = torch.autograd.grad(loss, (hr, wr), up)   # made again
    for got, other, w, b in zip((gh, gw), again, want[1:], bound[1:]):
        near(got, w, b)
        near(other, w, b)
    assert torch.equal(torch.autograd.grad(linear_distill(hr, weight, ids, logps, mask), hr, up)[0], gh)
    assert torch.equal(torch.autograd.grad(linear_distill(hidden.detach(), wr, ids, logps, mask), wr, up)[0], gw)
    if share < 0.9:
        at = int(mask.nonzero()[20])
        ids = ids.clone()
        ids[at, 0] = -3
        logps[at, 0] = -1.0
        up[at] = 1.0
        loss = linear_distill(hr, wr, ids, logps, mask)
        gh, gw = torch.autograd.grad(loss, (hr, wr), up)
        assert loss[at].isnan() and gh[at].isnan().all() and gh[torch.arange(shape[0], device=dev) != at].isfinite().all()
        assert gw.isnan().all()


def test_words_in_one_tile_and_at_its_edges(dev):
    """A token's words all side by side, across a tile's end, in the last tile."""
    hidden, weight, ids, logps, mask, up = inputs((70, 64, 1000, 128), torch.bfloat16, dev)
    for i in range(70):
        first = [0, 128, 192, 250, 256, 700, 872][i % 7]
        ids[i] = torch.arange(first, first + 128, device=dev).flip(0)
    for kind, rest in FORMS:
        check((hidden, weight, ids, logps, mask, up), torch.bfloat16, 1.0, kind, rest)


def test_large_logits(dev):
    """Far beyond what exp takes: a student sure of a word that the teacher does not name,
    or of one it does."""
    hidden, weight, ids, logps, mask, up = inputs((70, 128, 600, 20), torch.bfloat16, dev)
    for dtype in (torch.bfloat16, torch.float32):
        for kind, rest in FORMS:
            check(((hidden * 100).to(dtype), weight.to(dtype), ids, logps, mask, up), dtype, 1.0, kind, rest)


def test_words_that_are_wrong(dev):
    for dtype, h in ((torch.bfloat16, 64), (torch.float32, 40)):
        hidden, weight, ids, logps, _, up = inputs((70, h, 300, 6), dtype, dev)
        ids[5, 0], ids[6, 1], ids[7, 2] = 300, -1, ids[7, 1]
        ids[8, 3] = 1 << 40
        logps[8, 3] = -math.inf   # no word
        logps[9, 0] = math.nan
        hidden.requires_grad_(True)
        weight.requires_grad_(True)
        wrong = [5, 6, 7, 9]
        right = [i for i in range(70) if i not in wrong]
        for kind, rest in FORMS:
            loss = linear_distill(hidden, weight, ids, logps, kind=kind, rest=rest)
            assert loss[wrong].isnan().all() and loss[right].isfinite().all() and loss[2] == 0
            gh, gw = torch.autograd.grad(loss.sum(), (hidden, weight))
            assert gh[wrong].isnan().all() and gh[right].isfinite().all() and (gh[2] == 0).all() and gw.isnan().all()
            # no gradient arrives at them
            up = torch.ones(70, device=dev)
            up[wrong] = 0
            gh, gw = torch.autograd.grad(linear_distill(hidden, weight, ids, logps, kind=kind, rest=rest), (hidden, weight), up)
            assert (gh[wrong] == 0).all() and gh.isfinite().all() and gw.isfinite().all()


def test_tokens_that_do_not_count_may_hold_anything(dev):
    for shape, dtype in (((300, 128, 900, 8), torch.bfloat16), ((90, 40, 300, 8), torch.float32), ((600, 256, 70_000, 8), torch.float16)):
        hidden, weight, ids, logps, mask, up = inputs(shape, dtype, dev)
        hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        loss = linear_distill(hr, wr, ids, logps, mask)
        want = (loss.detach(), *torch.autograd.grad(loss, (hr, wr), up))
        wild = hidden.clone()
        wild[~mask] = math.nan
        ids2, logps2 = ids.clone(), logps.clone()
        ids2[~mask], logps2[~mask] = -5, math.nan
        up2 = torch.where(mask, up, math.nan)
        hr = wild.requires_grad_(True)
        loss = linear_distill(hr, wr, ids2, logps2, mask)
        for a, b in zip((loss.detach(), *torch.autograd.grad(loss, (hr, wr), up2)), want):
            assert torch.equal(a, b)


def test_infinite_and_nan_logits_stay_in_their_row(dev):
    for dtype, h in ((torch.bfloat16, 64), (torch.float32, 40)):
        hidden, weight, ids, logps, _, _ = inputs((70, h, 300, 6), dtype, dev)
        hidden[4, 3], hidden[9, 5] = math.nan, math.inf
        loss = linear_distill(hidden, weight, ids, logps)
        assert loss[4].isnan() and not loss[9].isfinite()
        assert loss[[i for i in range(70) if i not in (4, 9)]].isfinite().all()


def test_strides_shapes_and_parts_of_the_gradient(dev):
    hidden, weight, ids, logps, mask, up = inputs((360, 128, 700, 9), torch.bfloat16, dev)
    flat = linear_distill(hidden, weight, ids, logps, mask)
    cut = lambda t: t.view(12, 30, *t.shape[1:])[:, :-1]  # noqa: E731
    a = linear_distill(cut(hidden), weight, cut(ids), cut(logps), cut(mask))
    assert a.shape == (12, 29) and torch.equal(a, cut(flat))
    assert torch.equal(linear_distill(hidden, weight, ids.t().contiguous().t(), logps.t().contiguous().t(), mask), flat)
    assert torch.equal(linear_distill(hidden, weight, ids, logps, torch.stack([mask, mask], 1)[:, 0]), flat)
    wide = torch.full((360, 30), 7, dtype=torch.int64, device=dev)
    wide[:, 5:14] = ids
    assert torch.equal(linear_distill(hidden, weight, wide[:, 5:14], logps, mask), flat)
    # one row for all tokens
    same = linear_distill(hidden, weight, ids[:1].expand(360, 9), logps[:1].expand(360, 9))
    assert torch.equal(same, linear_distill(hidden, weight, ids[:1].repeat(360, 1), logps[:1].repeat(360, 1)))
    hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    both = torch.autograd.grad(linear_distill(hr, wr, ids, logps, mask), (hr, wr), up)
    assert torch.equal(torch.autograd.grad(linear_distill(hr, weight, ids, logps, mask), hr, up)[0], both[0])
    assert torch.equal(torch.autograd.grad(linear_distill(hidden, wr, ids, logps, mask), wr, up)[0], both[1])
    shared = torch.autograd.grad(linear_distill(hr, wr, ids, logps).sum(), (hr, wr))   # an expanded gradient
    whole = torch.autograd.grad(linear_distill(hr, wr, ids, logps), (hr, wr), torch.ones(360, device=dev))
    assert all(torch.equal(x, y) for x, y in zip(shared, whole))
    # rows and columns of wider tensors, off 16-byte boundaries
    odd = torch.empty(360 * 128 + 1, dtype=torch.bfloat16, device=dev)[1:].view(360, 128).copy_(hidden)
    want, bound = distill(hidden, weight, ids, logps, mask)
    near(linear_distill(odd, weight, ids, logps, mask), want[0], bound[0])
    near(linear_distill(hidden, weight.t().contiguous().t(), ids, logps, mask), want[0], bound[0])


@pytest.mark.parametrize("shape,dtype", [((700, 128, 3000, 40), torch.bfloat16), ((700, 128, 3000, 40), torch.float16),
                                         ((90, 40, 500, 11), torch.bfloat16)])
def test_backward_in_pieces_and_again(dev, shape, dtype, monkeypatch):
    """Beyond what the forward keeps the product is made again, in pieces; so in a second
    backward of a retained graph."""
    args = inputs(shape, dtype, dev)
    hidden, weight, ids, logps, mask, up = args
    hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = linear_distill(hr, wr, ids, logps, mask)
    first = torch.autograd.grad(loss, (hr, wr), up, retain_graph=True)
    again = torch.autograd.grad(loss, (hr, wr), up)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    monkeypatch.setattr(limits, "_KEEP_BYTES", 0)
    monkeypatch.setattr(limits, "_AGAIN_BYTES", 2 * 200 * shape[2])
    check(args, dtype)
    check(args, dtype, 2.0, "reverse")


def test_once_differentiable_and_saved_elsewhere(dev):
    for shape, dtype in (((70, 64, 300, 6), torch.bfloat16), ((70, 40, 300, 6), torch.float32)):
        hidden, weight, ids, logps, mask, up = inputs(shape, dtype, dev)
        hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        g = torch.autograd.grad(linear_distill(hr, wr, ids, logps, mask).sum(), hr, create_graph=True)[0]
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.float().sum(), hr)
        want, bound = distill(hidden, weight, ids, logps, mask, grad=up)
        # what was saved comes back in another type: torch operations
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.double() if t.is_floating_point() else t, lambda t: t):
            loss = linear_distill(hr, wr, ids, logps, mask)
        for a, b, c in zip(torch.autograd.grad(loss, (hr, wr), up), want[1:], bound[1:]):
            near(a, b, c)
        # and from the host
        with torch.autograd.graph.save_on_cpu():
            loss = linear_distill(hr, wr, ids, logps, mask)
        for a, b, c in zip(torch.autograd.grad(loss, (hr, wr), up), want[1:], bound[1:]):
            near(a, b, c)


def test_graph_replays_with_an_eager_graph_alive(dev):
    """Forward and backward captured together while an eager graph of other leaves
    lives; replayed on new inputs."""
    hidden, weight, ids, logps, mask, up = inputs((300, 128, 5000, 16), torch.bfloat16, dev)
    he, we = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    hc, wc = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)

    def step(h, w):
        loss = linear_distill(h, w, ids, logps, mask)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(hc, wc)
    torch.cuda.current_stream().wait_stream(side)
    alive = linear_distill(he, we, ids, logps, mask)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(hc, wc)
    for seed in range(3):
        fresh = inputs((300, 128, 5000, 16), torch.bfloat16, dev, seed=seed + 1)
        with torch.no_grad():
            for to, t in zip((hc, wc, ids, logps, mask, up), fresh):
                to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(fresh[0].clone().requires_grad_(True), fresh[1].clone().requires_grad_(True))
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
    assert alive.isfinite().all()


@pytest.mark.parametrize("shape", [(4200, 2048, 12_000, 3), (400, 2048, 50_000, 9)])
def test_graph_replays_with_other_masks(dev, shape):
    """How many rows the products take is known on the device alone: a captured step replayed with more of
    them, fewer, none and all."""
    hidden, weight, ids, logps, mask, up = inputs(shape, torch.bfloat16, dev)
    hidden.requires_grad_(True), weight.requires_grad_(True)

    def step(h, w):
        loss = linear_distill(h, w, ids, logps, mask)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(hidden, weight)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(hidden, weight)
    g = torch.Generator(device=dev).manual_seed(2)
    for share in (0.5, 0.0, 1.0, 0.9, 0.1):
        mask.copy_(torch.rand(shape[0], generator=g, device=dev) >= share)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(hidden.detach().clone().requires_grad_(True), weight.detach().clone().requires_grad_(True))
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_transforms_take_torch_operations(dev):
    hidden, weight, ids, logps, mask, _ = inputs((12, 64, 300, 6), torch.float32, dev)
    out = torch.vmap(lambda h, i, l: linear_distill(h, weight, i, l))(hidden.view(3, 4, 64), ids.view(3, 4, 6), logps.view(3, 4, 6))
    want, bound = distill(hidden, weight, ids, logps)
    near(out.reshape(-1), want[0], bound[0])
    cpu = linear_distill(hidden.cpu(), weight.cpu(), ids.cpu(), logps.cpu(), mask.cpu())
    want, bound = distill(hidden, weight, ids, logps, mask)
    near(cpu.to(dev), want[0], bound[0])
